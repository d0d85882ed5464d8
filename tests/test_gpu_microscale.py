"""Microscaled operators on the GPU against their definition in 64 bits."""
import pytest
import torch

import mx_oracle as O
from lich_amd import microscale as mx

pytestmark = pytest.mark.gpu
DT = O.DT


def _rand(g, *shape, size=1.0):
    return torch.randn(shape, generator=g, dtype=torch.float64) * size


def _dev(x, storage):
    return x.to(DT[storage]).cuda()


def _up(t):
    return t.cpu().double()


def _pack4(x):
    """Packed rows of a host matrix, by the oracle."""
    return mx.MXMatrix(*(t.cuda() for t in O.pack(x, "fp4")))


# ------------------------------------------------------------------ storage
@pytest.mark.parametrize("fmt", ["fp4", "int8"])
@pytest.mark.parametrize("storage", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("axis", [0, 1])
@pytest.mark.parametrize("R,C", [(1, 1), (1, 33), (33, 1), (5, 31), (32, 32), (64, 784), (65, 129), (127, 130),
                                 (256, 200), (300, 1531), (200, 64), (400, 513), (513, 400)])
def test_quantize_is_the_definition(R, C, axis, storage, fmt):
    """Codes and scales equal, blocks of very different sizes among them."""
    g = torch.Generator().manual_seed(R * 7919 + C + axis)
    x = _rand(g, R, C) * 2.0 ** torch.randint(-12, 12, (R, C // 40 + 1), generator=g).double().repeat_interleave(40, 1)[:, :C]
    xd = _dev(x, storage)
    x = _up(xd)
    k = mx.build_mx_quantize(R, C, "identity", DT[storage], format=fmt, axis=axis)
    out = k.new_output()
    for t in out:
        t.fill_(77)
    k(xd, out)
    codes, scales = O.pack(x if axis == 1 else x.T.contiguous(), fmt)
    assert torch.equal(out.scales.cpu(), scales)
    got = out.codes.cpu()
    if fmt == "fp4":  # a value that rounds to zero may keep its sign
        got = torch.stack([got & 15, got >> 4], -1)
        codes = torch.stack([codes & 15, codes >> 4], -1)
        got, codes = (torch.where(t == 8, 0, t) for t in (got, codes))
    assert torch.equal(got, codes)


@pytest.mark.parametrize("fmt", ["fp4", "int8"])
@pytest.mark.parametrize("storage", ["fp32", "bf16"])
@pytest.mark.parametrize("R,C", [(10, 1), (9, 2), (257, 2), (10, 3), (66, 5), (7, 7), (129, 9)])
def test_quantize_of_narrow_matrices(R, C, storage, fmt):
    """A load of 16 bytes spans several rows: both axes, what comes back against the oracle."""
    g = torch.Generator().manual_seed(R * 31 + C)
    xd = _dev(_rand(g, R, C), storage)
    x = _up(xd)
    for axis in (0, 1):
        k = mx.build_mx_quantize(R, C, "identity", DT[storage], format=fmt, axis=axis)
        out = k.new_output()
        k(xd, out)
        codes, scales = O.pack(x if axis == 1 else x.T.contiguous(), fmt)
        assert torch.equal(out.scales.cpu(), scales)
        back, want = (torch.empty(k.rows, k.length, dtype=DT[storage], device="cuda") for _ in range(2))
        restore = mx.build_mx_dequantize(k.rows, k.length, DT[storage], format=fmt)
        restore(out, back)
        restore(mx.MXMatrix(codes.cuda(), scales.cuda()), want)
        assert torch.equal(back, want)


@pytest.mark.parametrize("fmt", ["fp4", "int8"])
@pytest.mark.parametrize("axis", [0, 1])
def test_quantize_ties_edges_and_specials(fmt, axis):
    """Midpoints and their neighbours, the largest and smallest floats, zeros,
    infinities and NaN, in every lane of a block."""
    rows = []
    step = 0.25 if fmt == "fp4" else 1 / 128
    for base in (2.0 ** -120, 1.0, 2.0 ** 100):
        for top in (4.0, 5.0, 6.0, 6.5, 6.99, 7.0, 7.01, 7.99):
            v = torch.arange(32, dtype=torch.float64) * step * (1 if fmt == "fp4" else 4)
            v = v.clamp(max=top) * torch.where(torch.arange(32) % 2 == 0, 1.0, -1.0)
            v[int(top * 4) % 32] = top
            rows += [v * base, (v * base * (1 + 2.0 ** -20)), (v * base * (1 - 2.0 ** -20))]
    fmax = torch.finfo(torch.float32).max
    for special in (0.0, -0.0, fmax, -fmax, 2.0 ** -126, 2.0 ** -149, -2.0 ** -140, 2.0 ** -124, float("inf"),
                    float("-inf"), float("nan")):
        for at in (0, 13, 31):
            v = torch.zeros(32, dtype=torch.float64)
            v[at] = special
            rows.append(v)
            w = torch.ones(32, dtype=torch.float64) * 2.0 ** -130
            w[at] = special
            rows.append(w)
    x = torch.stack(rows).float()
    x = torch.cat([x, x.flip(1), x.roll(5, 0), x.roll(11, 0), x], 1).contiguous()
    R, C = x.shape
    xin = x if axis == 1 else x.T.contiguous()
    k = mx.build_mx_quantize(*xin.shape, "identity", torch.float32, format=fmt, axis=axis)
    out = k.new_output()
    k(xin.cuda(), out)
    codes, scales = O.pack(x.double(), fmt)
    assert torch.equal(out.scales.cpu(), scales)
    y = torch.empty((R, C), device="cuda")
    mx.build_mx_dequantize(R, C, torch.float32, format=fmt)(out, y)
    want = O.quantised(x.double(), fmt)
    got = _up(y)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    off = torch.nan_to_num(got, nan=0.0) != torch.nan_to_num(want, nan=0.0)
    assert not bool(off.any()), [(float(x[i, j]), float(got[i, j]), float(want[i, j])) for i, j in off.nonzero()[:8]]


@pytest.mark.parametrize("act", ["relu", "tanh", "sigmoid", "silu", "gelu"])
@pytest.mark.parametrize("axis", [0, 1])
def test_quantize_applies_the_activation(act, axis):
    """Each value within half an element's step of f(x) (of 2^-20 more for f in
    fp32), padding zero although f(0) may not be."""
    g = torch.Generator().manual_seed(3)
    x = _rand(g, 70, 150, size=2.0).float()
    for fmt, step in (("fp4", 1.0), ("int8", 1 / 64)):
        k = mx.build_mx_quantize(70, 150, act, torch.float32, format=fmt, axis=axis)
        out = k.new_output()
        k(x.cuda(), out)
        y = torch.empty((k.rows, k.length), device="cuda")
        mx.build_mx_dequantize(k.rows, k.length, torch.float32, format=fmt)(out, y)
        want = O.f(act, x.double())
        want = want if axis == 1 else want.T
        scale = 2.0 ** (out.scales.cpu().transpose(0, 1).reshape(k.rows, -1).double() - 127)
        half = (scale * step * (1.0 if fmt == "fp4" else 0.5)).repeat_interleave(32, 1)[:, :k.length]
        assert bool(((_up(y) - want).abs() <= half + 2.0 ** -20 * (1 + want.abs())).all())
        code = out.codes.cpu()
        assert int(code[:, -(-k.length // 2) if fmt == "fp4" else k.length:].abs().sum() if fmt == "int8" else
                   code[:, -(-k.length // 2):].long().sum()) == 0


@pytest.mark.parametrize("fmt", ["fp4", "int8"])
@pytest.mark.parametrize("storage", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("R,C", [(1, 1), (3, 37), (64, 128), (65, 200), (130, 1031)])
def test_dequantize_every_code(R, C, storage, fmt):
    g = torch.Generator().manual_seed(R + C)
    (r, width), (groups, _, four) = mx.packed_shapes(R, C, fmt)
    codes = torch.randint(0, 256, (r, width), generator=g, dtype=torch.int64)
    codes = codes.to(torch.uint8) if fmt == "fp4" else (codes - 128).clamp(min=-127).to(torch.int8)
    scales = torch.randint(118, 134, (groups, R, four), generator=g).to(torch.uint8)
    out = torch.empty((R, C), dtype=DT[storage], device="cuda")
    mx.build_mx_dequantize(R, C, DT[storage], format=fmt)(mx.MXMatrix(codes.cuda(), scales.cuda()), out)
    byte = scales.transpose(0, 1).reshape(R, -1).long()
    c = torch.stack([codes & 15, codes >> 4], -1).reshape(R, -1).long() if fmt == "fp4" else codes.long()
    full = torch.zeros((R, groups * 128), dtype=torch.int64)
    full[:, :c.shape[1]] = c
    want = O.values(full, byte, C, fmt)
    assert torch.equal(_up(out), want.to(DT[storage]).double())


# ------------------------------------------------------------------ products
SHAPES = [(1, 1, 1), (16, 10, 1), (64, 784, 128), (33, 129, 31), (100, 257, 40), (31, 500, 97), (300, 130, 200),
          (129, 384, 1025), (1000, 300, 1531), (130, 2000, 70), (2048, 640, 1600), (1601, 130, 2049),
          (3000, 200, 3001), (3001, 400, 2900)]


def _close(got, want, bound, storage):
    """Within the bound of the fp32 sum and one rounding of the result."""
    u = O.UNIT[storage]
    tol = bound * (1 + u) + u * (want.abs() + bound) * 1.01 + 2.0 ** -149
    if storage == "fp16":
        tol = tol + 2.0 ** -25
    bad = (_up(got) - want).abs() > tol
    assert not bool(bad.any()), (float(((_up(got) - want).abs() / tol).max()), int(bad.sum()))


@pytest.mark.parametrize("storage", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("M,K,B", SHAPES)
def test_forward_and_prediction_error(M, K, B, storage):
    g = torch.Generator().manual_seed(M + K + B)
    w, x = _rand(g, M, K, size=K ** -0.5), _rand(g, B, K)
    xl = _up(_rand(g, M, B).to(DT[storage]))
    w4, x4 = _pack4(w), _pack4(x)
    wq, xq = O.quantised(w, "fp4"), O.quantised(x, "fp4").T.contiguous()
    want, bound = wq @ xq, O.product_bound(wq, xq, K)
    out = torch.full((M, B), 7.0, dtype=DT[storage], device="cuda")
    mx.build_mx_forward(M, K, B, DT[storage])(x4, w4, out)
    _close(out, want, bound, storage)
    mx.build_mx_prediction_error(M, K, B, DT[storage])(x4, w4, _dev(xl, storage), out)
    _close(out, xl - want, bound + 2.0 ** -23 * (xl.abs() + want.abs()), storage)


@pytest.mark.parametrize("act", ["identity", "relu", "tanh", "sigmoid", "silu", "gelu"])
@pytest.mark.parametrize("storage", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("M,K,B", [(1, 1, 1), (33, 129, 31), (64, 10, 128), (1100, 300, 1025), (2048, 640, 1600), (1601, 130, 2049),
                                   (3000, 200, 3001), (3001, 130, 2900)])
def test_inference_update(M, K, B, storage, act):
    g = torch.Generator().manual_seed(M + K + B)
    x, e = (_up(_rand(g, M, B, size=s).to(DT[storage])) for s in (1.0, 0.1))
    wt, et = _rand(g, M, K, size=K ** -0.5), _rand(g, B, K, size=0.1)
    wq, eq = O.quantised(wt, "fp4"), O.quantised(et, "fp4").T.contiguous()
    up, bound = wq @ eq, O.product_bound(wq, eq, K)
    d = O.df(act, x)
    want = x + 0.5 * (d * up - e)
    xd = _dev(x, storage)
    mx.build_mx_inference_update(M, K, B, act, DT[storage], 0.5)(xd, _dev(e, storage), _pack4(wt), _pack4(et))
    # f' in fp32: a few units of 1; four roundings of the epilogue
    bound = 0.5 * (bound * d.abs() + 2.0 ** -20 * up.abs()) + 2.0 ** -22 * (x.abs() + e.abs() + (d * up).abs())
    _close(xd, want, bound, storage)


@pytest.mark.parametrize("storage", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("M,K,B", [(1, 1, 1), (10, 64, 128), (33, 31, 300), (1000, 1531, 300), (2100, 2048, 129), (3000, 3001, 40)])
def test_weight_update(M, K, B, storage):
    g = torch.Generator().manual_seed(M + K + B)
    w = _up(_rand(g, M, K, size=0.1).to(DT[storage]))
    e, a = _rand(g, M, B, size=0.1), _rand(g, K, B)
    eq, aq = O.quantised(e, "fp4"), O.quantised(a, "fp4").T.contiguous()
    acc, bound = eq @ aq, O.product_bound(eq, aq, B)
    wd = _dev(w, storage)
    k = mx.build_mx_weight_update(M, K, B, DT[storage], 0.01)
    alpha = float(torch.tensor(0.01, dtype=torch.float32))
    k(wd, _pack4(e), _pack4(a))
    _close(wd, w + alpha * acc, alpha * bound + 2.0 ** -22 * (w.abs() + alpha * acc.abs()), storage)


@pytest.mark.parametrize("M,K,B", [(70, 300, 90), (700, 300, 600), (2048, 300, 1600), (3000, 300, 3001)])
def test_a_nan_block_reaches_its_row_and_column_only(M, K, B):
    """The direct kernel and the three tiles."""
    g = torch.Generator().manual_seed(5)
    w, x = _rand(g, M, K), _rand(g, B, K)
    w[3, 40] = float("inf")
    x[5, 299] = float("nan")
    out = torch.empty((M, B), device="cuda")
    mx.build_mx_forward(M, K, B)(_pack4(x), _pack4(w), out)
    bad = torch.isnan(out).cpu()
    want = torch.zeros((M, B), dtype=torch.bool)
    want[3, :] = True
    want[:, 5] = True
    assert torch.equal(bad, want)
    out1 = torch.empty((M, B), device="cuda")
    mx.build_mx_predict(M, K, B, "identity")(x.T.contiguous().float().cuda(), _pack4(w), out1)
    assert torch.equal(torch.isnan(out1).cpu(), want)


@pytest.mark.parametrize("M,K,B", [(130, 130, 130), (700, 130, 600), (2048, 130, 1600), (3000, 130, 3001)])
def test_zero_rows_and_far_scales(M, K, B):
    """Blocks of zeros, and scales at both ends of their range that cancel."""
    w, x = torch.zeros(M, K, dtype=torch.float64), torch.zeros(B, K, dtype=torch.float64)
    w[1:] = 2.0 ** 90
    x[1:] = 2.0 ** -100
    out = torch.empty((M, B), device="cuda")
    mx.build_mx_forward(M, K, B)(_pack4(x), _pack4(w), out)
    want = torch.zeros(M, B, dtype=torch.float64)
    want[1:, 1:] = K * 2.0 ** -10
    assert torch.equal(_up(out), want)


# ------------------------------------------------------------------ few samples
@pytest.mark.parametrize("storage", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("M,K,B", [(1, 1, 1), (10, 64, 1), (16, 784, 3), (64, 784, 4), (33, 129, 5), (100, 1531, 16),
                                   (47, 300, 17), (130, 2100, 33), (64, 64, 100),
                                   (8200, 300, 2), (8197, 140, 20), (8192, 130, 40)])
@pytest.mark.parametrize("act", ["identity", "tanh", "sigmoid"])
def test_predict(M, K, B, storage, act):
    g = torch.Generator().manual_seed(M + K + B)
    w, x = _rand(g, M, K, size=K ** -0.5), _up(_rand(g, K, B).to(DT[storage]))
    wq, fx = O.quantised(w, "fp4"), O.f(act, x)
    want = wq @ fx
    out = torch.full((M, B), 7.0, dtype=DT[storage], device="cuda")
    k = mx.build_mx_predict(M, K, B, act, DT[storage])
    # f in fp32 (4 units), its terms (2^-17 of it for 16-bit states), the sum
    term = (2.0 ** -21 if storage == "fp32" else 2.0 ** -16) * (wq.abs() @ fx.abs())
    for workspace in (None, k.new_workspace()):
        out.fill_(7.0)
        k(_dev(x, storage), _pack4(w), out, workspace=workspace)
        _close(out, want, O.product_bound(wq, fx, 3 * K) + term, storage)


# ------------------------------------------------------------------ streams, graphs, repeats
def test_calls_follow_torchs_stream_and_capture():
    """Quantiser, product and serving product in a graph, replayed between eager
    work, each replay equal to the eager result."""
    M, K, B = 300, 784, 128
    g = torch.Generator().manual_seed(9)
    w = _pack4(_rand(g, M, K))
    x = torch.randn(K, B, device="cuda", dtype=torch.bfloat16)
    one = torch.randn(K, 1, device="cuda", dtype=torch.bfloat16)
    out, out1 = torch.empty(M, B, device="cuda", dtype=torch.bfloat16), torch.empty(M, 1, device="cuda", dtype=torch.bfloat16)
    q = mx.build_mx_quantize(K, B, "relu", torch.bfloat16, axis=0)
    x4 = q.new_output()
    forward, predict = mx.build_mx_forward(M, K, B, torch.bfloat16), mx.build_mx_predict(M, K, 1, "relu", torch.bfloat16)

    def calls():
        q(x, x4)
        forward(x4, w, out)
        predict(one, w, out1)

    calls()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        calls()
    for seed in range(4):
        x.copy_(torch.randn(K, B, generator=torch.Generator().manual_seed(seed)))
        one.copy_(torch.randn(K, 1, generator=torch.Generator().manual_seed(seed)))
        out.zero_(), out1.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone(), out1.clone()
        calls()
        torch.cuda.synchronize()
        assert torch.equal(got[0], out) and torch.equal(got[1], out1)


def test_refusals():
    k = mx.build_mx_quantize(64, 96, "relu", torch.bfloat16)
    x, out = torch.zeros(64, 96, device="cuda", dtype=torch.bfloat16), k.new_output()
    for bad in ((x.float(), out), (x.T, out), (x[:, :95].contiguous(), out), (x.cpu(), out),
                (x, mx.MXMatrix(out.codes[:, :-1].contiguous(), out.scales)), (x, out.codes),
                (x, mx.MXMatrix(out.codes.to(torch.int8), out.scales)), (x, mx.MXMatrix(out.codes, out.scales.cpu()))):
        with pytest.raises(ValueError):
            k(*bad)
    shifted = torch.empty(out.codes.numel() + 4, dtype=torch.uint8, device="cuda")[4:].view_as(out.codes)
    with pytest.raises(ValueError, match="aligned"):
        k(x, mx.MXMatrix(shifted, out.scales))


def test_fast_and_checked_calls_agree():
    """The extension's calls and those through ctypes: the same results, on the stream that
    is current; a tensor that is not what it has to be is refused either way."""
    assert mx._fast_call is not None
    M, K, B = 96, 200, 40
    g = torch.Generator().manual_seed(5)
    x, w = (torch.randn(s, generator=g).cuda() for s in ((K, B), (M, K)))
    e = torch.randn((M, B), generator=g).cuda()
    got = []
    for fast in (True, False):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            def run(k, *a, **kw):
                before, k._run = k._run, k._run if fast else mx._no_fast_call
                try:
                    k(*a, **kw)
                finally:
                    k._run = before

            qx, qw, qt, qe = (mx.build_mx_quantize(K, B, "relu", axis=0), mx.build_mx_quantize(M, K), mx.build_mx_quantize(M, K, axis=0),
                              mx.build_mx_quantize(M, B, axis=0))
            x4, w4, wt, et = (k.new_output("cuda") for k in (qx, qw, qt, qe))
            for k, t, o in ((qx, x, x4), (qw, w, w4), (qt, w, wt), (qe, e, et)):
                run(k, t, o)
            save, x8 = mx.build_checkpoint_save(K, B), mx.new_packed(K, B, "int8")
            run(save, x, x8)
            out = [torch.empty_like(e), torch.empty_like(e), x.clone(), w.clone(), torch.empty_like(e), w.clone(),
                   torch.empty_like(x), torch.empty_like(x)]
            e4, a4 = mx.build_mx_quantize(M, B), mx.build_mx_quantize(K, B)
            er, ar = e4.new_output(), a4.new_output()
            run(e4, e, er)
            run(a4, x, ar)
            run(mx.build_mx_prediction_error(M, K, B), x4, w4, e, out[0])
            run(mx.build_mx_forward(M, K, B), x4, w4, out[1])
            run(mx.build_mx_inference_update(K, M, B, "tanh"), out[2], x, wt, et)
            run(mx.build_mx_weight_update(M, K, B), out[3], er, ar)
            predict = mx.build_mx_predict(M, K, B, "silu")
            run(predict, x, w4, out[4], workspace=predict.new_workspace())
            run(mx.build_checkpoint_weight_update(M, K, B, "gelu"), out[5], e, x8)
            run(mx.build_checkpoint_gradient(K, M, B, "gelu"), w, e, x8, out[6])
            run(mx.build_mx_dequantize(K, B, format="int8"), x8, out[7])
        side.synchronize()
        got.append(out)
    for a, b in zip(*got):
        assert bool(a.isfinite().all()) and torch.equal(a, b)
    for bad in (x.half(), x[:, :-1], x.T.contiguous().T, x.cpu(), None):
        with pytest.raises((ValueError, TypeError)):
            qx(bad, x4)
    for bad in ((x4.codes, x4.scales[:1]), (x4.codes.cpu(), x4.scales), [*x4], (x4.codes,)):
        with pytest.raises((ValueError, TypeError)):
            qx(x, bad)


@pytest.mark.parametrize("M,K,B", [(40, 200, 1), (40, 200, 3), (8200, 200, 2), (40, 200, 12), (100, 1531, 17)])
@pytest.mark.parametrize("size", [2.0 ** 127, 2.0 ** -100])
def test_predict_of_states_near_the_ends_of_fp32(M, K, B, size):
    """Finite states past the largest bf16 among them, zero weights in their way: the sum's
    bound and that of the terms as for any other states."""
    g = torch.Generator().manual_seed(K + B)
    w = _rand(g, M, K, size=2.0 ** -16)
    w[::3] = 0
    x = (torch.rand(K, B, generator=g, dtype=torch.float64) * 2 - 1) * 2 * size
    x[:4] = torch.tensor([1.0, -1.0, 1 - 2.0 ** -10, 1 - 2.0 ** -23], dtype=torch.float64)[:, None] * (2 - 2.0 ** -23) * size
    x = x.float().double()
    assert bool(x.isfinite().all())
    wq = O.quantised(w, "fp4")
    want = wq @ x
    k = mx.build_mx_predict(M, K, B, "identity")
    for workspace in (None, k.new_workspace()):
        out = torch.full((M, B), 7.0, device="cuda")
        k(_dev(x, "fp32"), _pack4(w), out, workspace=workspace)
        _close(out, want, O.product_bound(wq, x, 3 * K) + 2.0 ** -21 * (wq.abs() @ x.abs()), "fp32")


@pytest.mark.parametrize("storage", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("B", [1, 3, 12, 17])
def test_predict_carries_infinities_and_nan(B, storage):
    """They reach the outputs that a sum of products would give: infinite by a weight's sign,
    NaN by a zero weight, by two of different signs, by NaN, and the others stay finite."""
    M, K = 40, 200
    g = torch.Generator().manual_seed(B)
    w, x = _rand(g, M, K), _rand(g, K, B)
    w[7, 96:128] = 0
    x[100, 0] = float("inf")
    if B > 1:
        x[5, 1] = float("nan")
        x[130, 2], x[150, 2] = float("inf"), float("-inf")
    x = _up(x.to(DT[storage]))
    wq = O.quantised(w, "fp4")
    want = sum(wq[:, k:k + 1] * x[k:k + 1] for k in range(K))
    k = mx.build_mx_predict(M, K, B, "identity", DT[storage])
    for workspace in (None, k.new_workspace()):
        out = torch.full((M, B), 7.0, dtype=DT[storage], device="cuda")
        k(_dev(x, storage), _pack4(w), out, workspace=workspace)
        got = _up(out)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isfinite(), want.isfinite())
        assert torch.equal(got[want.isinf()], want[want.isinf()])


@pytest.mark.parametrize("fmt", ["fp4", "int8"])
@pytest.mark.parametrize("storage", ["fp32", "bf16"])
@pytest.mark.parametrize("axis", [0, 1])
def test_quantize_at_the_bottom_of_the_range(axis, storage, fmt):
    """Blocks under the smallest scale, 2^-126, whose values are subnormal floats: the codes of
    the definition, and back the subnormals they stand for."""
    g = torch.Generator().manual_seed(8)
    x = _rand(g, 64, 160) * 2.0 ** torch.randint(-132, -122, (64, 5), generator=g).double().repeat_interleave(32, 1)
    x[:8, :32] = torch.linspace(2.0 ** -128, 2.0 ** -126, 32, dtype=torch.float64)
    x[8, :32] = 2.0 ** -128  # halfway to the first code
    x[9, :32] = 2.0 ** -128 * (1 + 2.0 ** -7)
    xd = _dev(x if axis == 1 else x.T.contiguous(), storage)
    x = _up(xd if axis == 1 else xd.T.contiguous())
    k = mx.build_mx_quantize(*xd.shape, "identity", DT[storage], format=fmt, axis=axis)
    out = k.new_output()
    k(xd, out)
    codes, scales = O.pack(x, fmt)
    assert bool((scales == 1).any()) and torch.equal(out.scales.cpu(), scales)
    back = torch.empty(x.shape, dtype=DT[storage], device="cuda")
    mx.build_mx_dequantize(*x.shape, DT[storage], format=fmt)(out, back)
    want = O.quantised(x, fmt)
    assert bool((want.abs() == 2.0 ** -127).any()) and torch.equal(_up(back), want.to(DT[storage]).double())


@pytest.mark.parametrize("M,K,B", [(64, 160, 40), (1100, 160, 1025)])
def test_products_read_the_bottom_of_the_range(M, K, B):
    """Weights of 2^-127 to 2^-122 against states of 2^100: exact codes and scales in the product
    and in the prediction."""
    g = torch.Generator().manual_seed(M)
    w = _rand(g, M, K) * 2.0 ** torch.randint(-127, -122, (M, K // 32), generator=g).double().repeat_interleave(32, 1)
    x = _rand(g, B, K, size=2.0 ** 100)
    wq, xq = O.quantised(w, "fp4"), O.quantised(x, "fp4").T.contiguous()
    out = torch.full((M, B), 7.0, device="cuda")
    mx.build_mx_forward(M, K, B)(_pack4(x), _pack4(w), out)
    _close(out, wq @ xq, O.product_bound(wq, xq, K), "fp32")
    predict = mx.build_mx_predict(M, K, B, "identity")
    for workspace in (None, predict.new_workspace()):
        out.fill_(7.0)
        xs = x.T.contiguous().float()
        predict(xs.cuda(), _pack4(w), out, workspace=workspace)
        _close(out, wq @ xs.double(), O.product_bound(wq, xs.double(), 3 * K) + 2.0 ** -21 * (wq.abs() @ xs.double().abs()), "fp32")
