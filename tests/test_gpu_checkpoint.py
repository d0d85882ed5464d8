"""Backward pass of a state kept in 8 bits, on the GPU, against its definition in
64 bits and against differences of the forward pass."""
import pytest
import torch

import mx_oracle as O
from lich_amd import _native as nat
from lich_amd import microscale as mx

pytestmark = pytest.mark.gpu
DT = O.DT
ACTS = ["identity", "relu", "tanh", "sigmoid", "silu", "gelu"]


def _rand(g, *shape, size=1.0, storage="fp32"):
    return (torch.randn(shape, generator=g, dtype=torch.float64) * size).to(DT[storage]).double()


def _dev(x, storage):
    return x.to(DT[storage]).cuda()


def _close(got, want, tol):
    d = (got.cpu().double() - want).abs()
    assert bool((d <= tol).all()), (float((d / tol).max()), int((d > tol).sum()))


def _keep(x, storage):
    save = mx.build_checkpoint_save(*x.shape, DT[storage])
    x8 = save.new_output()
    save(_dev(x, storage), x8)
    return x8, O.quantised(x, "int8")


# (storage, operand, unit of the operand's rounding)
TYPES = [("fp32", "fp32", 0.0), ("fp32", "bf16", 2.0 ** -8), ("fp32", "fp16", 2.0 ** -11), ("fp16", "fp16", 2.0 ** -11),
         ("bf16", "bf16", 2.0 ** -8)]
# few tiles, odd lengths, the k-chunk kernel's rows of odd length, the 16-bit products'
# and the LDS-DMA kernel's tiles with ragged edges, the tile kernel's (fp32 storage)
SHAPES = [(1, 1, 1), (10, 64, 128), (64, 784, 128), (33, 31, 65), (100, 200, 1), (130, 257, 300), (1000, 1531, 300),
          (1100, 2050, 192), (4100, 4000, 64)]


def _weight(M, K, B, storage, operand, unit, act, lend=False):
    g = torch.Generator().manual_seed(M + K + B)
    x = _rand(g, K, B, storage=storage)
    w, e = _rand(g, M, K, size=0.1, storage=storage), _rand(g, M, B, size=0.1, storage=storage)
    x8, xq = _keep(x, storage)
    fx = O.f(act, xq)
    acc = e @ fx.T
    wd = _dev(w, storage)
    k = mx.build_checkpoint_weight_update(M, K, B, act, DT[storage], 0.01, operand_dtype=DT[operand])
    ws = torch.empty(max(k.workspace_bytes, 16), dtype=torch.uint8, device="cuda") if lend else None
    k(wd, _dev(e, storage), x8, workspace=ws)
    alpha = float(torch.tensor(0.01, dtype=torch.float32))
    size = e.abs() @ fx.abs().T
    # operands rounded, f in fp32 (4 units and its cancellation, 2^-21), the sum, the epilogue, the result
    acc_tol = size * (2 * unit + unit * unit + 2.0 ** -21 + (B + 8) * 2.0 ** -23)
    if operand == "fp16":
        acc_tol = acc_tol + e.abs().sum(1, keepdim=True) * 2.0 ** -24
    want = w + alpha * acc
    tol = alpha * acc_tol + 2.0 ** -22 * (w.abs() + alpha * acc.abs())
    _close(wd, want, tol + O.UNIT[storage] * 1.01 * (want.abs() + tol) + 2.0 ** -25 * (storage == "fp16") + 2.0 ** -149)


def _gradient(M, K, B, storage, operand, unit, act):
    g = torch.Generator().manual_seed(M + K + B + 1)
    x = _rand(g, M, B, storage=storage)
    w, e = _rand(g, K, M, size=0.1, storage=storage), _rand(g, K, B, size=0.1, storage=storage)
    x8, xq = _keep(x, storage)
    up, d = w.T.contiguous() @ e, O.df(act, xq)
    k = mx.build_checkpoint_gradient(M, K, B, act, DT[storage], operand_dtype=DT[operand])
    if storage == "fp32" or (M % 2 == 0 and B % 2 == 0):
        assert k.new_workspace() is None
    size = w.T.abs().contiguous() @ e.abs()
    own = unit if storage == "fp32" else 0.0  # 16-bit tensors are operands as they are
    acc_tol = size * (2 * own + own * own + (K + 8) * 2.0 ** -23)
    if operand == "fp16":
        acc_tol = acc_tol + (w.abs().sum(0)[:, None] + e.abs().sum(0)[None]) * 2.0 ** -24
    want = d * up
    tol = d.abs() * acc_tol + 2.0 ** -20 * (up.abs() + acc_tol)  # f' in fp32: a few units of 1
    for workspace in (None, k.new_workspace()):
        out = torch.full((M, B), 7.0, dtype=DT[storage], device="cuda")
        k(_dev(w, storage), _dev(e, storage), x8, out, workspace=workspace)
        _close(out, want, tol + O.UNIT[storage] * 1.01 * (want.abs() + tol) + 2.0 ** -25 * (storage == "fp16") + 2.0 ** -149)


@pytest.mark.parametrize("storage,operand,unit", TYPES)
@pytest.mark.parametrize("M,K,B", SHAPES)
def test_weight_update(M, K, B, storage, operand, unit):
    _weight(M, K, B, storage, operand, unit, "tanh")


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("storage", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("M,K,B", [(1, 4, 1), (3, 65, 2), (64, 784, 4), (65, 260, 5), (130, 1028, 8), (2100, 1300, 3), (2101, 1303, 5)])
def test_weight_update_of_few_samples(M, K, B, storage, act):
    """Rank-B sums past W, operands not rounded where the samples are few enough."""
    few = B <= 8 and K % 4 == 0 if storage == "fp32" else B <= 5
    _weight(M, K, B, storage, storage, 0.0 if few or storage == "fp32" else O.UNIT[storage], act)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("storage,operand,unit", TYPES)
@pytest.mark.parametrize("M,K,B", [(33, 31, 65), (1100, 2050, 192)])
def test_weight_update_activations(M, K, B, storage, operand, unit, act):
    _weight(M, K, B, storage, operand, unit, act)


@pytest.mark.parametrize("storage,operand,unit", TYPES)
@pytest.mark.parametrize("M,K,B", SHAPES + [(4104, 64, 4000), (2048, 1088, 1096), (72, 32, 8), (1000, 96, 1040)])
def test_gradient(M, K, B, storage, operand, unit):
    _gradient(M, K, B, storage, operand, unit, "tanh")


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("storage,operand,unit", TYPES)
@pytest.mark.parametrize("M,K,B", [(33, 31, 65), (2048, 192, 1096), (4104, 64, 4000)])
def test_gradient_activations(M, K, B, storage, operand, unit, act):
    _gradient(M, K, B, storage, operand, unit, act)


@pytest.mark.parametrize("storage,operand,unit", TYPES[3:])
@pytest.mark.parametrize("M,K,B", [(1032, 1100, 32), (1100, 2050, 192), (4100, 4000, 64), (3000, 4104, 96), (1032, 1100, 2),
                                   (1032, 1100, 1), (1033, 1101, 63), (1100, 2050, 191), (1100, 2051, 190), (4101, 4000, 65),
                                   (4100, 4001, 66), (3000, 4104, 98), (512, 512, 2048), (700, 900, 2051), (700, 690, 257),
                                   (1000, 1030, 4002)])
def test_weight_update_widened_once(M, K, B, storage, operand, unit):
    """The 16-bit products on 64, 128 and 256 wide tiles."""
    k = mx.build_checkpoint_weight_update(M, K, B, "sigmoid", DT[storage])
    assert k.workspace_bytes == 2 * (K + (M if B % 2 else 0)) * (-(-B // 32) * 32)
    _weight(M, K, B, storage, operand, unit, "sigmoid", lend=True)


@pytest.mark.parametrize("act", ["identity", "relu", "tanh", "sigmoid"])
@pytest.mark.parametrize("M,K,B", [(300, 300, 4001), (1100, 2050, 192), (4100, 4000, 65), (4000, 4104, 300), (1000, 1531, 300)])
def test_fp32_weight_update(M, K, B, act):
    """fp32 products on 32, 64 and 128 wide tiles, the contraction's rests of 1 to 16, f(X)
    widened once where the call asks for it and from the codes."""
    k = mx.build_checkpoint_weight_update(M, K, B, act)
    padded = 4 * K * (-(-B // 32) * 32)
    assert k.workspace_bytes == (padded if M * K * B >= 2 ** (27 if act in ACTS[2:] else 32) else 0)
    for lend in (False, True):
        _weight(M, K, B, "fp32", "fp32", 0.0, act, lend=lend)


@pytest.mark.parametrize("M,K,B", [(65, 1, 65), (1, 4000, 1), (31, 16, 33), (1531, 1000, 300), (2050, 1100, 1000),
                                   (4001, 333, 4099), (4001, 17, 4099)])
def test_fp32_gradient(M, K, B):
    _gradient(M, K, B, "fp32", "fp32", 0.0, "silu")


@pytest.mark.parametrize("storage,operand,unit", TYPES[3:])
@pytest.mark.parametrize("M,K,B", [(2, 1, 2), (4, 33, 2), (65, 31, 64), (64, 40, 65), (1100, 513, 1002), (1101, 514, 1003),
                                   (2051, 333, 1000), (4098, 47, 4006), (4097, 65, 4001), (66, 1025, 34), (130, 1089, 70),
                                   (1000, 1026, 1000), (300, 4001, 301), (1, 4000, 301), (2, 5000, 2)])
def test_16_bit_gradient(M, K, B, storage, operand, unit):
    """Rows of even and odd lengths, contractions with a rest, on 64, 128 and 256 wide tiles."""
    pads = (M % 2 or B % 2) and M * K * B >= 2 ** 28 and (M % 2 == 0 or B >= 256)
    need = 2 * K * ((-(-M // 8) * 8 if M % 2 else 0) + (-(-B // 8) * 8 if B % 2 else 0)) if pads else 0
    assert mx.build_checkpoint_gradient(M, K, B, "silu", DT[storage]).workspace_bytes == need
    _gradient(M, K, B, storage, operand, unit, "silu")


@pytest.mark.parametrize("storage,operand,unit", TYPES)
@pytest.mark.parametrize("M,K,B", [(37, 50, 45), (40, 64, 72), (600, 1500, 1100), (1100, 2050, 190), (1101, 1201, 301)])
def test_not_a_number_stays_in_its_place(M, K, B, storage, operand, unit):
    """A load that reaches into the next row, or clears what a stage lacks, touches no
    other output."""
    g = torch.Generator().manual_seed(M)
    w, e = _rand(g, M, K, size=0.1, storage=storage), _rand(g, M, B, size=0.1, storage=storage)
    x = _rand(g, K, B, storage=storage)
    x8, _ = _keep(x, storage)
    nan, bad = float("nan"), float("inf")
    grad = mx.build_checkpoint_gradient(K, M, B, "tanh", DT[storage], operand_dtype=DT[operand])
    plain, hit = (torch.empty((K, B), dtype=DT[storage], device="cuda") for _ in range(2))
    ws = grad.new_workspace()
    grad(_dev(w, storage), _dev(e, storage), x8, plain, workspace=ws)
    w2, e2 = w.clone(), e.clone()
    w2[:, 0] = nan
    e2[:, 0] = bad
    grad(_dev(w2, storage), _dev(e2, storage), x8, hit, workspace=ws)
    assert bool(hit[0].isnan().all()) and bool((~hit[:, 0].isfinite()).all())
    assert torch.equal(hit[1:, 1:], plain[1:, 1:])
    update = mx.build_checkpoint_weight_update(M, K, B, "tanh", DT[storage], 0.01, operand_dtype=DT[operand])
    ws = torch.empty(max(update.workspace_bytes, 16), dtype=torch.uint8, device="cuda")
    e2 = e.clone()
    e2[5] = nan
    for lent in (None, ws):
        plain, hit = _dev(w, storage), _dev(w, storage)
        update(plain, _dev(e, storage), x8, workspace=lent)
        update(hit, _dev(e2, storage), x8, workspace=lent)
        assert bool(hit[5].isnan().all())
        keep = torch.arange(M, device="cuda") != 5
        assert torch.equal(hit[keep], plain[keep])


@pytest.mark.parametrize("storage", ["fp16", "bf16"])
@pytest.mark.parametrize("act", ["identity", "relu", "tanh", "gelu"])
def test_lent_workspaces(storage, act):
    """Wherever a call can use one (mode 1), the same results."""
    lib = nat.lib()
    unit = O.UNIT[storage]
    try:
        assert lib.ipc_set_s16_preactivate(1) == 0
        for M, K, B in ((33, 31, 65), (1100, 2050, 192), (130, 257, 300)):
            _weight(M, K, B, storage, storage, unit, act, lend=True)
    finally:
        lib.ipc_set_s16_preactivate(-1)


@pytest.mark.parametrize("act", ACTS[2:])
def test_against_differences(act):
    """L = sum(E * W f(X)): <dL/dX, D> and <dL/dW, D> against central differences
    in 64 bits, whose truncation is below h^2 times a third derivative of at
    most 4 and whose rounding is negligible."""
    M, K, B, h = 40, 70, 50, 1e-4
    g = torch.Generator().manual_seed(11)
    x = _rand(g, K, B)
    w, e = _rand(g, M, K, size=0.2), _rand(g, M, B)
    x8, xq = _keep(x, "fp32")
    grad = torch.empty((K, B), device="cuda")
    mx.build_checkpoint_gradient(K, M, B, act)(_dev(w, "fp32"), _dev(e, "fp32"), x8, grad)
    dw = torch.zeros((M, K), device="cuda")
    mx.build_checkpoint_weight_update(M, K, B, act, "float32", 1.0)(dw, _dev(e, "fp32"), x8)

    def loss(wv, xv):
        return float((e * (wv @ O.f(act, xv))).sum())

    for seed in range(3):
        dx, dww = _rand(torch.Generator().manual_seed(seed), K, B), _rand(torch.Generator().manual_seed(seed), M, K)
        up = (w.T.abs().contiguous() @ e.abs())
        fd = (loss(w, xq + h * dx) - loss(w, xq - h * dx)) / (2 * h)
        tol = float((up * (dx.abs() ** 3 * 4 * h * h + dx.abs() * (M + 16) * 2.0 ** -21)).sum()) + 1e-6
        assert abs(float((grad.cpu().double() * dx).sum()) - fd) <= tol
        fd = (loss(w + h * dww, xq) - loss(w - h * dww, xq)) / (2 * h)  # linear in W
        tol = float(((e.abs() @ O.f(act, xq).abs().T) * dww.abs()).sum()) * (B + 16) * 2.0 ** -21 + 1e-6
        assert abs(float((dw.cpu().double() * dww).sum()) - fd) <= tol


def test_a_lost_block_is_seen():
    """An infinity in a kept state reads back as NaN: its weight column and its own
    gradients are NaN, the others are not."""
    K, M, B = 70, 40, 64
    g = torch.Generator().manual_seed(2)
    x = _rand(g, K, B)
    x[5, 40] = float("inf")
    w, e = _rand(g, M, K), _rand(g, M, B)
    x8, _ = _keep(x, "fp32")
    wd, grad = _dev(w, "fp32"), torch.empty((K, B), device="cuda")
    mx.build_checkpoint_gradient(K, M, B, "tanh")(wd, _dev(e, "fp32"), x8, grad)
    mx.build_checkpoint_weight_update(M, K, B, "tanh")(wd, _dev(e, "fp32"), x8)
    want = torch.zeros((K, B), dtype=torch.bool)
    want[5, 32:] = True
    assert torch.equal(torch.isnan(grad).cpu(), want)
    assert bool(torch.isnan(wd[:, 5]).all()) and not bool(torch.isnan(wd[:, :5]).any())
    assert not bool(torch.isnan(wd[:, 6:]).any())


def test_refusals():
    update = mx.build_checkpoint_weight_update(16, 32, 64, "relu", torch.bfloat16)
    gradient = mx.build_checkpoint_gradient(32, 16, 64, "relu", torch.bfloat16)
    w, e = (torch.zeros(s, device="cuda", dtype=torch.bfloat16) for s in ((16, 32), (16, 64)))
    x8, g = mx.new_packed(32, 64, "int8"), torch.empty(32, 64, device="cuda", dtype=torch.bfloat16)
    four = mx.new_packed(32, 64, "fp4")
    for bad in ((w.float(), e, x8), (w, e.T, x8), (w, e, four), (w, e, mx.MXMatrix(x8.codes, x8.scales[:, :-1].contiguous())),
                (w, e, g)):
        with pytest.raises(ValueError):
            update(*bad)
        with pytest.raises(ValueError):
            gradient(*bad, g)
    with pytest.raises(ValueError):
        gradient(w, e, x8, g.float())
    with pytest.raises(ValueError):
        mx.build_checkpoint_weight_update(16, 32, 64, "relu", torch.bfloat16, operand_dtype=torch.float32)
    with pytest.raises(ValueError, match="workspace"):
        update(w, e, x8, workspace=torch.empty(64))


def test_calls_in_a_graph():
    """Keeping a state, its gradient and its weight update with their workspaces, captured
    and replayed between eager work: the eager bits every time."""
    M, K, B = 1101, 1203, 301
    g = torch.Generator().manual_seed(9)
    for storage in ("bf16", "fp32"):
        x, w, e = (_dev(_rand(g, *s, storage=storage), storage) for s in ((K, B), (M, K), (M, B)))
        save, grad = mx.build_checkpoint_save(K, B, DT[storage]), mx.build_checkpoint_gradient(K, M, B, "silu", DT[storage])
        update = mx.build_checkpoint_weight_update(M, K, B, "silu", DT[storage], 0.01)
        x8, out, ws = save.new_output(), torch.empty_like(x), [k.new_workspace() for k in (grad, update)]
        assert ws[1] is not None and (ws[0] is not None) == (storage == "bf16")

        def calls():
            save(x, x8)
            grad(w, e, x8, out, workspace=ws[0])
            update(w, e, x8, workspace=ws[1])

        start = w.clone()
        want = []
        for _ in range(3):
            calls()
            want.append((out.clone(), w.clone()))
        w.copy_(start)
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            calls()
        for a, b in want:
            out.zero_()
            graph.replay()
            assert torch.equal(out, a) and torch.equal(w, b)
            torch.cuda.synchronize()
            save(x * 2, mx.new_packed(K, B, "int8"))


def test_no_storage_is_refused():
    from torch._subclasses import FakeTensorMode

    save = mx.build_checkpoint_save(64, 64)
    x8 = save.new_output()
    with FakeTensorMode():
        fake = torch.empty(64, 64, device="cuda")
    with pytest.raises((ValueError, RuntimeError)):
        save(fake, x8)
    with pytest.raises((ValueError, RuntimeError)):
        save(torch.zeros(64, 64).to_sparse().cuda(), x8)


@pytest.mark.parametrize("storage,operand,unit", TYPES)
@pytest.mark.parametrize("M,K,B", [(2, 33, 70), (4, 65, 2), (70, 34, 4), (2, 98, 2), (1, 17, 40), (40, 18, 1), (2, 33, 2), (1, 4001, 1),
                                   (1000, 2049, 2), (1000, 1026, 1)])
def test_gradient_of_rows_shorter_than_a_load(M, K, B, storage, operand, unit):
    """Contractions whose last rows are too few for a load from the row before them."""
    _gradient(M, K, B, storage, operand, unit, "silu")


@pytest.mark.parametrize("M,K,B", [(1, 1, 2 ** 28 + 4), (3, 2, 2 ** 27)])
def test_gradient_of_rows_past_two_to_the_26(M, K, B):
    """A row's offsets times 16 pass 32 bits."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x, e = torch.randn(M, B, device="cuda", generator=g), torch.randn(K, B, device="cuda", generator=g)
    w = torch.randn(K, M, device="cuda", generator=g)
    save = mx.build_checkpoint_save(M, B)
    x8, out = save.new_output(), torch.empty(M, B, device="cuda")
    save(x, x8)
    mx.build_checkpoint_gradient(M, K, B, "sigmoid")(w, e, x8, out)
    mx.build_mx_dequantize(M, B, format="int8")(x8, x)
    s = torch.sigmoid(x)
    s.mul_(1 - s)
    for row in range(M):  # f' in [0, 1 / 4] to a few units of 1, two products
        want, size = torch.zeros(B, device="cuda"), torch.zeros(B, device="cuda")
        for k in range(K):
            want += w[k, row] * e[k]
            size += (w[k, row] * e[k]).abs()
        assert bool(((out[row] - s[row] * want).abs() <= 2.0 ** -20 * size + 2.0 ** -149).all())


@pytest.mark.parametrize("storage,operand,unit", TYPES)
@pytest.mark.parametrize("M,K,B", [(1032, 1100, 1), (2052, 2052, 5), (2052, 2052, 6), (4096, 4096, 8), (4096, 4099, 8), (300, 300, 4),
                                   (1100, 2050, 192), (4100, 4000, 64)])
def test_the_workspace_asked_for_is_used(M, K, B, storage, operand, unit):
    """A lent workspace is written where new_workspace() gives one, and nowhere else."""
    k = mx.build_checkpoint_weight_update(M, K, B, "silu", DT[storage], operand_dtype=DT[operand])
    x8, _ = _keep(torch.ones(K, B, dtype=torch.float64), storage)
    w, e = torch.zeros(M, K, dtype=DT[storage], device="cuda"), torch.ones(M, B, dtype=DT[storage], device="cuda")
    lent = torch.full((4 * K * 192 + 2 * M * 192,), 77, dtype=torch.uint8, device="cuda")
    k(w, e, x8, workspace=lent)
    own = k.new_workspace()
    assert bool((lent == 77).all()) == (own is None)
    if own is not None:
        assert bool((lent[own.numel():] == 77).all())
