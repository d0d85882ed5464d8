"""Outputs that are views of a larger buffer: the microscaled products and the 8-bit backward
pass write their tensor and nothing beside it, from any element-aligned address."""
import pytest
import torch

import mx_oracle as O
from lich_amd import microscale as mx

pytestmark = pytest.mark.gpu
DT = O.DT
EDGE, GUARD = 64, 77.0  # elements kept on either side, and their value


def _view(rows, columns, dtype, start, fill):
    """A matrix `start` elements past a 16-byte boundary, and the buffer around it."""
    n = rows * columns
    buf = torch.full((EDGE + start + n + EDGE,), GUARD, dtype=dtype, device="cuda")
    out = buf[EDGE + start:EDGE + start + n].view(rows, columns)
    assert out.data_ptr() % 16 == start * out.element_size() % 16
    out.copy_(fill) if isinstance(fill, torch.Tensor) else out.fill_(fill)
    return out, buf


def _beside(out, buf, start, want):
    assert torch.equal(out, want)
    n = out.numel()
    assert bool((buf[:EDGE + start] == GUARD).all()) and bool((buf[EDGE + start + n:] == GUARD).all())


def _rand(g, *shape, dtype=torch.float32, size=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * size).to(dtype)


# output rows x columns, elements past the boundary: odd by odd from a whole dword, any from
# within one, rows not a multiple of 16; on 64, 128 and 256 wide tiles
SHAPES = [(1001, 1531, 0), (1000, 1531, 1), (1001, 1530, 1), (1601, 2049, 0), (1602, 2050, 1), (3001, 3101, 0), (3002, 3101, 1)]


@pytest.mark.parametrize("storage", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("M,N,start", SHAPES)
def test_products(M, N, start, storage):
    g, dt, K = torch.Generator(device="cuda").manual_seed(M + N), DT[storage], 130
    a, b = mx.new_packed(M, K), mx.new_packed(N, K)
    mx.build_mx_quantize(M, K)(_rand(g, M, K), a)
    mx.build_mx_quantize(N, K)(_rand(g, N, K), b)
    full, other = _rand(g, M, N, dtype=dt), _rand(g, M, N, dtype=dt)
    calls = [(mx.build_mx_forward(M, K, N, dt), lambda k, o: k(b, a, o)),
             (mx.build_mx_prediction_error(M, K, N, dt), lambda k, o: k(b, a, other, o)),
             (mx.build_mx_inference_update(M, K, N, "tanh", dt), lambda k, o: k(o, other, a, b)),
             (mx.build_mx_weight_update(M, N, K, dt, 0.01), lambda k, o: k(o, a, b))]
    for kernel, call in calls:
        want = full.clone()
        call(kernel, want)
        out, buf = _view(M, N, dt, start, full)
        call(kernel, out)
        _beside(out, buf, start, want)


@pytest.mark.parametrize("storage", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("M,N,start", SHAPES[:5] + [(3301, 3305, 0), (4098, 3602, 1)])
def test_backward(M, N, start, storage):
    """The weight update (W [M, N]) and the state gradient (G [M, N])."""
    g, dt, C = torch.Generator(device="cuda").manual_seed(M * N), DT[storage], 192
    full, e = _rand(g, M, N, dtype=dt, size=0.1), _rand(g, M, C, dtype=dt, size=0.1)
    save = mx.build_checkpoint_save(N, C, dt)
    x8 = save.new_output()
    save(_rand(g, N, C, dtype=dt), x8)
    update = mx.build_checkpoint_weight_update(M, N, C, "sigmoid", dt, 0.01)
    ws = update.new_workspace()
    assert ws is not None
    want = full.clone()
    update(want, e, x8, workspace=ws)
    out, buf = _view(M, N, dt, start, full)
    update(out, e, x8, workspace=ws)
    _beside(out, buf, start, want)

    save = mx.build_checkpoint_save(M, N, dt)
    x8 = save.new_output()
    save(full, x8)
    w, e = _rand(g, C, M, dtype=dt, size=0.1), _rand(g, C, N, dtype=dt)
    gradient = mx.build_checkpoint_gradient(M, C, N, "tanh", dt)
    ws = gradient.new_workspace()
    want = torch.empty_like(full)
    gradient(w, e, x8, want, workspace=ws)
    out, buf = _view(M, N, dt, start, 7.0)
    gradient(w, e, x8, out, workspace=ws)
    _beside(out, buf, start, want)
