"""Host side of the microscaled operators: sizes, refusals and the oracle (no GPU)."""
import pytest
import torch

import mx_oracle as O
from lich_amd import _native as nat
from lich_amd import microscale as mx

P = 4096  # a fake, aligned, non-null address; never dereferenced (validation fails first)


@pytest.mark.parametrize("rows,n", [(1, 1), (3, 32), (5, 33), (64, 128), (10, 784), (7, 1531)])
@pytest.mark.parametrize("fmt", ["fp4", "int8"])
def test_sizes_agree_with_the_library(rows, n, fmt):
    codes, scales = mx.packed_shapes(rows, n, fmt)
    lib = nat.lib()
    assert codes[0] * codes[1] == lib.ipc_mx_code_bytes(rows, n, nat.MX_FORMATS[fmt])
    assert scales[0] * scales[1] * scales[2] == lib.ipc_mx_scale_bytes(rows, n)
    got = O.pack(torch.randn(rows, n, dtype=torch.float64), fmt)
    assert tuple(got[0].shape) == codes and tuple(got[1].shape) == scales
    packed = mx.new_packed(rows, n, fmt, "cpu")
    assert packed.codes.dtype == got[0].dtype and packed.scales.dtype == got[1].dtype


def test_sizes_that_are_refused():
    lib = nat.lib()
    assert lib.ipc_mx_code_bytes(0, 5, 0) == 0 and lib.ipc_mx_code_bytes(5, 5, 2) == 0
    assert lib.ipc_mx_code_bytes(1 << 24, 1, 0) == 0 and lib.ipc_mx_scale_bytes(1 << 24, 1) == 0  # padded: 2^31 values


@pytest.mark.parametrize("args,code,needle", [
    ((None, P, P, 64, 64, 1, 0, 0, 0, None), nat.ERR_NULL, "x"),
    ((P, None, P, 64, 64, 1, 0, 0, 0, None), nat.ERR_NULL, "packed"),
    ((P, P + 8, P, 64, 64, 1, 0, 0, 0, None), nat.ERR_ALIGN, "aligned"),
    ((P, P, P + 2, 64, 64, 1, 0, 0, 0, None), nat.ERR_ALIGN, "aligned"),
    ((P + 1, P, P, 64, 64, 1, 0, 1, 0, None), nat.ERR_ALIGN, "aligned"),
    ((P, P, P, 0, 64, 1, 0, 0, 0, None), nat.ERR_SHAPE, "dimensions"),
    ((P, P, P, 1 << 20, 4096, 1, 0, 0, 0, None), nat.ERR_SHAPE, "too large"),
    ((P, P, P, 1, 1 << 24, 0, 0, 0, 0, None), nat.ERR_SHAPE, "too large"),
    ((P, P, P, 64, 64, 2, 0, 0, 0, None), nat.ERR_CONFIG, "axis"),
    ((P, P, P, 64, 64, 1, 2, 0, 0, None), nat.ERR_DTYPE, "format"),
    ((P, P, P, 64, 64, 1, 0, 3, 0, None), nat.ERR_DTYPE, "storage"),
    ((P, P, P, 64, 64, 1, 0, 0, 6, None), nat.ERR_ACT, "activation"),
])
def test_quantize_validation(args, code, needle):
    assert nat.lib().ipc_mx_quantize(*args) == code
    assert needle in nat.last_error()


def test_other_entry_points_validate():
    lib = nat.lib()
    assert lib.ipc_mx_dequantize(P, P, None, 64, 64, 0, 0, None) == nat.ERR_NULL
    assert lib.ipc_mx_dequantize(P, None, P, 64, 64, 0, 0, None) == nat.ERR_NULL
    assert lib.ipc_mx_forward(P, P, P, P, None, 64, 64, 64, 0, None) == nat.ERR_NULL
    assert lib.ipc_mx_forward(P, P, P + 4, P, P, 64, 64, 64, 0, None) == nat.ERR_ALIGN
    assert lib.ipc_mx_forward(P, P, P, P, P, 64, -1, 64, 0, None) == nat.ERR_SHAPE
    assert lib.ipc_mx_pred_err(P, P, P, P, None, P, 64, 64, 64, 0, None) == nat.ERR_NULL
    assert "x_lower" in nat.last_error()
    assert lib.ipc_mx_infer_update(P, P, P, P, P, None, 64, 64, 64, 0.5, 0, 1, None) == nat.ERR_NULL
    assert lib.ipc_mx_infer_update(P, P, P, P, P, P, 64, 64, 64, 0.5, 0, 9, None) == nat.ERR_ACT
    assert lib.ipc_mx_weight_update(P, P, P, P, P, 64, 1 << 20, 1 << 20, 1e-4, 0, None) == nat.ERR_SHAPE
    assert lib.ipc_mx_predict(P, P, P, P, 1, 1, (1 << 20), 0, 0, None, 0, None) == nat.ERR_SHAPE
    assert lib.ipc_mx_predict(P, P, P, P + 1, 1, 1, 1, 1, 0, None, 0, None) == nat.ERR_ALIGN
    assert lib.ipc_mx_predict(P, P, P, P, 1, 1, 2, 1, 0, P + 8, 4096, None) == nat.ERR_ALIGN
    need = lib.ipc_mx_predict_workspace_bytes
    assert need(200, 1, 0) == 0 and need(200, 4, 0) == 0 and need(0, 17, 2) == 0
    assert need(200, 5, 0) == 3 * 5 * 256 * 2 and need(200, 17, 2) == 2 * 32 * 256 * 2
    assert lib.ipc_ckpt_weight_update(P, P, None, P, 64, 64, 64, 1e-4, 0, 0, 1, None, 0, None) == nat.ERR_NULL
    assert lib.ipc_ckpt_weight_update(P, P, P, P, 64, 64, 64, 1e-4, 1, 2, 1, None, 0, None) == nat.ERR_DTYPE
    assert lib.ipc_ckpt_weight_update(P, P, P, P, 64, 64, 64, 1e-4, 0, 0, 1, P + 8, 64, None) == nat.ERR_ALIGN
    assert lib.ipc_ckpt_weight_update(P, P, P, P, 64, 64, 64, 1e-4, 0, 0, 1, P, -1, None) == nat.ERR_SHAPE
    assert lib.ipc_ckpt_gradient(P, P, P + 4, P, P, 64, 64, 64, 0, 0, 1, None, 0, None) == nat.ERR_ALIGN
    assert lib.ipc_ckpt_gradient(P, P, P, P, None, 64, 64, 64, 0, 0, 1, None, 0, None) == nat.ERR_NULL
    assert lib.ipc_ckpt_gradient(P, P, P, P, P, 1 << 24, 64, 1, 0, 0, 1, None, 0, None) == nat.ERR_SHAPE
    assert lib.ipc_ckpt_gradient(P, P, P, P, P, 64, 64, 64, 2, 2, 1, P + 8, 64, None) == nat.ERR_ALIGN
    assert lib.ipc_ckpt_gradient_workspace_bytes(1001, 1000, 999, 2) == 2 * 1000 * (1008 + 1000)
    assert lib.ipc_ckpt_gradient_workspace_bytes(1000, 999, 998, 2) == 0


def test_builders_refuse():
    with pytest.raises(ValueError):
        mx.build_mx_quantize(4, 4, "relu", torch.float64)
    with pytest.raises(ValueError):
        mx.build_mx_quantize(4, 4, "relu", torch.float32, format="fp8")
    with pytest.raises(ValueError):
        mx.build_mx_quantize(4, 4, "softmax", torch.float32)
    with pytest.raises(ValueError):
        mx.build_mx_quantize(4, 0, "relu", torch.float32)
    with pytest.raises(ValueError):
        mx.build_mx_quantize(4, 4, "relu", torch.float32, axis=2)
    with pytest.raises(ValueError):
        mx.build_mx_forward(4, 4, -1)
    k = mx.build_mx_predict(4, 4, 1, "relu")
    with pytest.raises(ValueError, match="device"):
        k(torch.zeros(4, 1), mx.new_packed(4, 4, device="cpu"), torch.zeros(4, 1))


@pytest.mark.parametrize("fmt", ["fp4", "int8"])
def test_the_oracle_rounds_to_nearest(fmt):
    """No representable value of the block's scale is nearer."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(50, 64, generator=g, dtype=torch.float64) * 2.0 ** torch.randint(-20, 20, (50, 1), generator=g).double()
    code, byte = O.quantise(x, fmt)
    got = O.values(code, byte, 64, fmt)
    scale = (2.0 ** (byte[:, :2].double() - 127)).repeat_interleave(32, 1)
    grid = torch.cat([O.GRID, -O.GRID]) if fmt == "fp4" else torch.arange(-127, 128).double() / 64
    best = (x[..., None] - grid * scale[..., None]).abs().amin(-1)
    assert torch.equal((x - got).abs(), best)
    # ... and no block could have had a smaller scale without saturating past half a step
    top = x.view(50, 2, 32).abs().amax(-1) / 2.0 ** (byte[:, :2].double() - 127)
    assert bool((top < (7 if fmt == "fp4" else 255 / 128)).all()) and bool((top >= (3.5 if fmt == "fp4" else 255 / 256)).all())


def test_fast_calls_refuse():
    """What is no device tensor of the right kind is left to the checks with messages."""
    fast = pytest.importorskip("lich_amd._fast_call")
    spec = ((2, 3), torch.float32), ((2, 64), torch.uint8), ((1, 2, 4), torch.uint8)
    call = fast.Call("ipc_mx_quantize", 0, spec, (2, 3, 1, 0, 0, 1), lambda i: 0)
    x, p = torch.zeros(2, 3), mx.MXMatrix(torch.zeros(2, 64, dtype=torch.uint8), torch.zeros(1, 2, 4, dtype=torch.uint8))
    for given in ((), (x,), (x, p), (x, None), (x, (p.codes,)), (None, p), (x, p, None), (x, p, x), (p, x), (x, [*p])):
        assert call(*given) == 1
    assert call(x, p=p) == 1
    for bad in (("ipc_mx_nothing", 0, spec, (2, 3, 1, 0, 0, 1), None), ("ipc_mx_quantize", 0, spec[:2], (2, 3, 1, 0, 0, 1), None),
                ("ipc_mx_quantize", 0, spec, (2, 3, 1, 0, 0), None), ("ipc_mx_quantize", 0, spec, (2, 3, 1, 0, 0, 1.0), None),
                ("ipc_mx_quantize", 0, (spec[0], spec[1], ((1, 2, 3, 4), torch.uint8)), (2, 3, 1, 0, 0, 1), None)):
        with pytest.raises(ValueError):
            fast.Call(*bad)
    with pytest.raises(ValueError):
        fast.Packed((2, 64), torch.uint8, (1, 2, 4), torch.uint8, list)
    with pytest.raises(TypeError):
        fast.Packed((2, 64), torch.uint8, (1, 2, 4), torch.uint8, mx.MXMatrix)("cuda")


def test_quantiser_run_lies_inside_the_matrix(tmp_path):
    """The bound of the quantiser's 16-byte loads, as compiled from ipc_mx.h: no value
    of a run lies past the matrix's last one, down to rows of a single value."""
    import re
    import subprocess
    from pathlib import Path

    csrc = Path(__file__).resolve().parents[1] / "lich_amd" / "csrc"
    body = re.search(r"inline bool mx_run_inside\(.*?\n}\n", (csrc / "ipc_mx.h").read_text(), re.S).group(0)
    assert (csrc / "ipc_mx_quant.hip").read_text().count("mx_run_inside(") == 2  # rows, columns
    source = tmp_path / "inside.cpp"
    source.write_text(body + """
int main() {
  for (int rows = 1; rows <= 20; ++rows)
    for (int n = 1; n <= 20; ++n)
      for (int r = -2; r < rows + 3; ++r)
        for (int c = 0; c < 32; c += 4)
          for (int run = 4; run <= 8; run += 4) {
            const bool all = r >= 0 && r < rows && c < n && r * n + c + run <= rows * n;
            if (r >= 0 && mx_run_inside(rows - r, n, c, run) != all) return 1;
          }
  return mx_run_inside(1 << 24, 127, 120, 8) ? 0 : 2;
}
""")
    program = tmp_path / "inside"
    subprocess.run(["g++", "-std=c++17", "-o", str(program), str(source)], check=True)
    assert subprocess.run([str(program)]).returncode == 0


def test_rows_past_the_last_are_not_stored(tmp_path):
    """The limits of the tiles' buffers, as compiled from ipc_mx.h: loads reach every element,
    stores none past the last one, whatever the rows' length and the base's dword half."""
    import re
    import subprocess
    from pathlib import Path

    csrc = Path(__file__).resolve().parents[1] / "lich_amd" / "csrc"
    body = re.search(r"inline long long mx_rows_bytes\(.*?\n}\n", (csrc / "ipc_mx.h").read_text(), re.S).group(0)
    kernel = (csrc / "ipc_mx_gemm.h").read_text()
    assert "mx_rows_bytes(first, end, ES, mis, store)" in kernel and "dst(p.out, first, end, true)" in kernel
    source = tmp_path / "rows.cpp"
    source.write_text(body + """
int main() {
  for (int M = 1; M <= 70; ++M)
    for (int N = 1; N <= 70; ++N)
      for (int half = 0; half < 2; ++half)  // the base's element within its dword
        for (int row = 0; row < 128; row += 16)
          for (int col = 0; col < N; col += 32) {
            const long long first = (long long)row * N + col, end = (long long)M * N;
            const unsigned mis = (unsigned)((first + half) * 2) & 2u;
            const long long loads = mx_rows_bytes(first, end, 2, mis, false), stores = mx_rows_bytes(first, end, 2, mis, true);
            if (loads % 4 || loads < stores || loads - stores > 2) return 1;
            for (int r = 0; r < 16; ++r)
              for (int c = col; c < N && c < col + 32; ++c) {
                const unsigned at = (unsigned)(r * N + c - col) * 2u + mis;
                if ((at < stores) != (row + r < M)) return 2;
                if (row + r < M && at + 2 > loads) return 3;
              }
          }
  return mx_rows_bytes(5, 9, 4, 0, false) == 16 && mx_rows_bytes(9, 5, 4, 0, true) == 0 ? 0 : 4;
}
""")
    program = tmp_path / "rows"
    subprocess.run(["g++", "-std=c++17", "-O1", "-o", str(program), str(source)], check=True)
    assert subprocess.run([str(program)]).returncode == 0


def test_rows_past_the_last_do_not_come_round(tmp_path):
    """Offsets of a tile's 16 rows in 32 bits, as compiled from ipc_mx.h: with as many columns as
    are let through, no row past the tensor's end lands in it; with many more some do."""
    import re
    import subprocess
    from pathlib import Path

    csrc = Path(__file__).resolve().parents[1] / "lich_amd" / "csrc"
    body = re.search(r"inline bool mx_rows_fit\(.*?}\n", (csrc / "ipc_mx.h").read_text(), re.S).group(0)
    assert "mx_rows_fit(B, 4)" in (csrc / "ipc_abi.hip").read_text()
    source = tmp_path / "fit.cpp"
    source.write_text(body + """
static bool round(long long N, int rows) {  // a dropped row's offset inside the first `rows` rows
  for (int r = rows; r < 16; ++r)
    for (int c = 0; c < 256; ++c)
      if ((unsigned)((unsigned)r * (unsigned)N + c) * 4u < rows * N * 4) return true;
  return false;
}
int main() {
  long long most = 1;
  while (mx_rows_fit(most + 1, 4)) most += 1 + (most < 71000000 ? 1000 : 0);
  for (int rows = 1; rows < 8; ++rows)
    if (rows * most < 1LL << 29 && round(most, rows)) return 1;
  // sizes that the other limits let through: 2^26, one more row's offset; 2^28, the fifth row is the first
  if (round(1 << 26, 1) || !mx_rows_fit(1 << 26, 4) || !round(1 << 28, 1) || mx_rows_fit(1 << 28, 4)) return 2;
  return mx_rows_fit((1LL << 29) / 33, 4) && mx_rows_fit((1LL << 30) / 33, 2) && mx_rows_fit(1 << 24, 4) ? 0 : 3;
}
""")
    program = tmp_path / "fit"
    subprocess.run(["g++", "-std=c++17", "-O1", "-o", str(program), str(source)], check=True)
    assert subprocess.run([str(program)]).returncode == 0


@pytest.mark.parametrize("storage,operand,M,K,B,used", [
    ("float32", "float16", 4096, 4096, 1024, 0), ("float32", "bfloat16", 4096, 4096, 1024, 0),
    ("float32", "float32", 4096, 4096, 1024, 4 * 4096 * 1024), ("float32", "float32", 300, 300, 64, 0),
    ("float32", "float32", 4096, 4096, 8, 0), ("float32", "float32", 4096, 4099, 8, 4 * 4099 * 32),
    ("float32", "float32", 4096, 4096, 9, 4 * 4096 * 32),
    ("bfloat16", "bfloat16", 8192, 8192, 1, 0), ("float16", "float16", 8192, 8192, 5, 0),
    ("bfloat16", "bfloat16", 8192, 8192, 6, 2 * 8192 * 32), ("float16", "float16", 8192, 8192, 7, 2 * 2 * 8192 * 32),
])
def test_workspace_of_a_weight_update(storage, operand, M, K, B, used):
    """0 where no call of these sizes and types reads one."""
    lib, dts = nat.lib(), [nat.dtype_code(t) for t in (storage, operand)]
    act = nat.act_code("silu")
    assert lib.ipc_ckpt_weight_update_workspace_bytes(act, M, K, B, *dts) == used
    assert lib.ipc_ckpt_workspace_bytes(act, M, K, B, dts[0]) >= used
    k = mx.build_checkpoint_weight_update(M, K, B, "silu", storage, operand_dtype=operand)
    assert k.workspace_bytes == used or (storage != "float32" and B <= 5)
    if used == 0:
        assert k.new_workspace() is None


def test_workspace_queries_refuse():
    need = nat.lib().ipc_ckpt_weight_update_workspace_bytes
    assert need(4, 4096, 4096, 1024, 1, 1) > 0
    for bad in ((4, 0, 4096, 1024, 1, 1), (9, 4096, 4096, 1024, 1, 1), (4, 4096, 4096, 1024, 3, 3), (4, 4096, 4096, 1024, 1, 2)):
        assert need(*bad) == 0


def test_inline_assembly_names_m0():
    """Whatever writes m0 says so."""
    import re
    from pathlib import Path

    found = 0
    for path in (Path(__file__).resolve().parents[1] / "lich_amd" / "csrc").iterdir():
        for asm in re.findall(r"\basm\b[^;]*?\((.*?)\);", path.read_text(), re.S):
            if re.search(r"mov_b32 m0,", asm):
                found += 1
                assert '"m0"' in asm.rsplit(":", 1)[1], path.name
    assert found == 2


def test_tensors_on_different_devices_are_refused():
    """Also a workspace; tensors without storage, so that no such device is needed."""
    from torch._subclasses import FakeTensorMode

    def on(device, *shape, dtype=torch.float32):
        with FakeTensorMode():
            return torch.empty(shape, dtype=dtype, device=device)

    def packed(k, device):
        p = k._operands[1]
        return mx.MXMatrix(on(device, *p.codes, dtype=p.dtype), on(device, *p.scales, dtype=torch.uint8))

    k = mx.build_mx_predict(16, 256, 8, "relu")
    good = on("cuda:0", 256, 8), packed(k, "cuda:0"), on("cuda:0", 16, 8)
    for at, other in enumerate((on("cuda:1", 256, 8), packed(k, "cuda:1"), on("cuda:1", 16, 8))):
        with pytest.raises(ValueError, match="different devices .*cuda:0, cuda:1"):
            k(*good[:at], other, *good[at + 1:])
    codes, scales = good[1]
    with pytest.raises(ValueError, match="different devices"):
        k(good[0], mx.MXMatrix(codes, packed(k, "cuda:1").scales), good[2])
    with pytest.raises(ValueError, match="different devices"):
        k(*good, workspace=on("cuda:1", k.workspace_bytes, dtype=torch.uint8))
