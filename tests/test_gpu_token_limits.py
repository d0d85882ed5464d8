"""Softmax calls over tokens where their plans change: states near an operand's limit, short last
pieces, against their definitions in 64 bits on the device (bounds: those of test_gpu_tokens.py)."""
import pytest
import torch

from lich_amd import tokens
from tests import token_oracle as O
from tests.helpers import DEV
from tests.test_gpu_tokens import H, TYPES, half_step, run_update, softmax_bounds, softmax_case

pytestmark = pytest.mark.gpu


def large_case(V, D, B, dt, padded=0.1):
    g = torch.Generator(device=DEV).manual_seed(V + D + B)
    x = torch.randn((D, B), generator=g, device=DEV).to(dt)
    w = (torch.randn((V, D), generator=g, device=DEV) * (2.0 / D ** 0.5)).to(dt)
    t = torch.randint(0, V, (B,), generator=g, device=DEV)
    return x, w, torch.where(torch.rand(B, generator=g, device=DEV) < padded, -1, t)


def check(got, want, bound, what):
    assert bool(torch.isfinite(got).all()), what
    over = ((got.double() - want).abs() - bound).max()
    assert float(over) <= 0, f"{what}: {float(over):.3e} over a bound of {float(bound.max()):.3e} at most"


def check_update(x, w, t, activation, alpha):
    (D, B), V = x.shape, w.shape[0]
    loss, g, wn = run_update(x, w, t, activation, alpha)
    r = O.softmax(x, w, t, activation)
    bl, bg, bw = softmax_bounds(r, w, x.dtype, V, D, B, activation, alpha)
    check(loss, r["loss"], bl, "loss")
    check(g, r["g"], bg, "g")
    check(wn, w.double() + alpha * r["dw"], bw, "w")
    padded = t < 0
    assert bool((loss[padded] == 0).all()) and bool((g[:, padded] == 0).all())


# G in 16 bits is the rounding of a sum that is good to a few H, where errors rounded to 16 bits would leave u in a whole
# column: it may differ from the exact sum's rounding only where that lies within the sum's bound of a tie.  e, per element:
# p's own error (the logits' two or three terms of f(X), exp, the sum of V exponentials in a tree of parts, as for the weights
# of test_gpu_tokens.py) and what is left of two terms, u^2 of it.  A matrix instruction adds 16 products to a sum at once:
# D / 16 steps of three terms in a logit, V / 16 of two in G, and within a step's products 16 H.
def gradient_bounds(r, x, w, V, D, dt):
    u, half = half_step(dt), dt == torch.float16
    exact, small, wa, ea = not bool((r["f"].to(dt).double() != r["f"]).any()), 2.0 ** -25 * half, w.double().abs(), r["e"].abs()
    dz = (r["size"] * ((0.0 if exact else 18 * H) + (3 * D / 16 + 64) * H)).max(0).values + small * 2.0 ** -11 * wa.sum(1).max()
    de = r["p"] * ((2 * dz).expm1() + 8 * H * (1 + r["p"].clamp(min=1e-300).log().abs()) + 256 * H) + (u * u + 4 * H) * ea + 2.0 ** -34 * half
    return r["df"].abs() * (wa.T @ de + (V / 8 + 64) * H * (wa.T @ ea)) + 16 * H * (wa.T @ ea) + 2 * H * r["g"].abs()


@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("V,D,B,activation", [(2, 200, 400, "relu"), (90, 70, 40, "tanh"), (400, 60, 90, "identity"), (100, 600, 70, "gelu"), (300, 130, 40, "relu"),
                                              (700, 90, 130, "silu"), (600, 300, 300, "relu"), (3000, 8, 12, "tanh"), (500, 400, 20, "sigmoid"),
                                              (700, 1100, 70, "relu"), (600, 1200, 33, "identity")])
def test_state_gradients_round_as_the_exact_sums(V, D, B, activation, name):
    dt = TYPES[name]
    x, w, t = softmax_case(V, D, B, dt, V + D)
    got = run_update(x.to(DEV), w.to(DEV), t.to(DEV), activation, 0.25)[1].cpu()
    r = O.softmax(x, w, t, activation)
    bound = gradient_bounds(r, x, w, V, D, dt)
    low, high = (r["g"] - bound).to(dt), (r["g"] + bound).to(dt)
    assert bool(((got >= low) & (got <= high)).all()), int(((got < low) | (got > high)).sum())
    # (errors rounded to 16 bits would not pass; but at D = 1200 a logit's bound, 289 H of magnitudes of 44 in all, lets p
    # be off by 2^-9 of itself, more than fp16's half step)
    plain = (r["df"] * (w.double().T @ r["e"].to(dt).double())).to(dt)
    assert D > 1000 or bool(((plain < low) | (plain > high)).any())


# Large updates: the target's error in fp32, the others, probabilities of a large vocabulary, rounded to the type (and kept as
# fp16 times 2^15 of their part's largest): a_v each at most, of either sign, so that a sum of them passes 8 sqrt(sum a_v^2 W^2)
# once in 10^13 (Hoeffding's bound).  f(X) is exact here.
@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("V,D,B,activation", [(524301, 8, 17, "relu"), (700001, 5, 13, "identity"), (5000, 33, 1700, "relu"), (6000, 300, 1500, "relu")])
def test_state_gradients_of_large_updates(V, D, B, activation, name):
    dt = TYPES[name]
    u, half = half_step(dt), dt == torch.float16
    x, w, t = (v.to(DEV) for v in softmax_case(V, D, B, dt, V + D))
    got = run_update(x, w, t, activation, 0.25)[1]
    r = O.softmax(x, w, t, activation)
    hot = torch.zeros((V, B), dtype=torch.bool, device=DEV)
    real = (t >= 0) & (t < V)
    hot[t[real], real.nonzero()[:, 0]] = True
    wa, p = w.double().abs(), r["p"]
    dz = (r["size"] * (D / 16 + 64) * H).max(0).values
    de = p * ((2 * dz).expm1() + 8 * H * (1 + p.clamp(min=1e-300).log().abs()) + 256 * H) + 4 * H * r["e"].abs()
    rounded = torch.where(hot, 0.0, (u + 2.0 ** -11) * p + 2.0 ** -38 + 2.0 ** -35 * half)
    back = wa.T @ de + 8 * ((wa ** 2).T @ rounded ** 2).sqrt() + (V / 16 + 64) * H * (wa.T @ r["e"].abs())
    bound = r["df"].abs() * back + 2 * H * r["g"].abs()
    low, high = (r["g"] - bound).to(dt), (r["g"] + bound).to(dt)
    assert bool(((got >= low) & (got <= high)).all()), int(((got < low) | (got > high)).sum())
    plain = (r["df"] * (w.double().T @ r["e"].to(dt).double())).to(dt)
    assert V > 10000 or bool(((plain < low) | (plain > high)).any())


# Infinities by the definition, in every form that a call takes by its size: a small layer, few samples, one tile, tiles and pieces of
# exponentials.  A weight of -inf gives a logit of the sign of its state: -inf, a masked word, or inf, a loss of NaN.
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("activation", ["identity", "tanh"])
@pytest.mark.parametrize("V,D,B", [(10, 20, 30), (700, 70, 2), (60, 33, 90), (300, 50, 40), (1000, 600, 130), (5000, 17, 260)])
def test_infinities(V, D, B, activation, name):
    dt = TYPES[name]
    x, w, t = softmax_case(V, D, B, dt, V + D + B, padded=0.1)
    t[0], t[1] = 1, V - 1
    some = w.clone()
    some[V - 1, 3] = -float("inf")
    many = x.clone()
    many[5, 0] = float("inf")
    up = w.clone()
    up[2] = float("inf")
    for states, weights in ((x, some), (many, w), (x, up)):
        if states is many and activation == "tanh":
            continue  # (f is finite)
        want = O.softmax(states, weights, t, activation)["loss"]
        k, loss = tokens.build_token_loss(V, D, B, activation, dt), torch.zeros(B, device=DEV)
        k(states.to(DEV), weights.to(DEV), t.to(DEV), loss, workspace=k.new_workspace(DEV))
        got = loss.cpu().double()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got == float("inf"), want == float("inf"))
        if states is many:
            trained, g, _ = run_update(states.to(DEV), weights.to(DEV), t.to(DEV), activation, 0.25)
            assert bool(trained[0].isnan()) and bool(trained[1:].isfinite().all()) and bool(g[:, 1:].isfinite().all())
        fine = want.isfinite()
        assert bool(fine.any()) or weights is up
        # (what a masked word adds is 0; its row is left out of the bounds)
        kept = weights.clone()
        kept[weights.isinf()] = 0.0
        r = O.softmax(x, kept, t, activation)
        assert bool(((got - want).abs() <= softmax_bounds(r, kept, dt, V, D, B, activation, 0.0, False)[0])[fine].all())


@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_losses_of_huge_logits_are_not_negative(name):
    """Logits of thousands, which rounding f(X) moves by some: a loss corrected to first order stays a loss."""
    dt, V, D, B = TYPES[name], 9000, 300, 2000
    x, w, t = (v.to(DEV) for v in softmax_case(V, D, B, dt, 4, padded=0.0, wscale=600.0 if name == "f16" else 100.0))
    t[:] = (w.double() @ torch.tanh(x.double())).argmax(0)
    loss = run_update(x, w, t, "tanh", 0.0)[0]
    assert bool(torch.isfinite(loss).all()) and float(loss.min()) >= 0.0
    want = O.softmax(x, w, t, "tanh")["loss"]
    off = (w.double() @ (torch.tanh(x.double()) - torch.tanh(x.double()).to(dt).double())).abs().amax(0)
    # (rounding moves the logits by `off` at most, and a loss by twice that; the correction moves it by as much again)
    assert bool(((loss.double() - want).abs() <= 4 * off + 2.0 ** -10).all())


# states that fit an operand in two terms but not in three; the last three in fp16, which takes two
@pytest.mark.parametrize("V,D,B,activation,name", [(200, 10000, 40000, "tanh", "bf16"), (2, 8200, 50000, "relu", "bf16"), (1, 500, 800000, "gelu", "bf16"),
                                                   (300, 16384, 24576, "silu", "bf16"), (40, 20000, 20000, "tanh", "f16"), (3, 30000, 20000, "relu", "f16")])
def test_updates_of_large_states(V, D, B, activation, name):
    check_update(*large_case(V, D, B, TYPES[name]), activation, 0.5)


# vocabularies in pieces whose last one has fewer stages of 32 rows than a whole one has slices
@pytest.mark.parametrize("V,D,B,name", [(524298, 64, 1000, "bf16"), (524289, 8, 1000, "f16"), (131073, 300, 4096, "f16"), (21770, 8192, 64, "f32"), (91793, 1949, 118, "f32")])
def test_short_last_pieces(V, D, B, name):
    check_update(*large_case(V, D, B, TYPES[name]), "tanh", 0.5)


def off(t, by):
    """The same values `by` elements behind a 256-byte boundary."""
    base = torch.zeros(t.numel() + by, dtype=t.dtype, device=DEV)
    view = base[by:].view(t.shape)
    view.copy_(t)
    return view


# every form of a call: a small layer, few samples, one tile, two launches at the end, slices, large products, two pieces
FORMS = [(10, 64, 128), (900, 72, 2), (60, 34, 92), (300, 52, 40), (20, 40, 1000), (1000, 600, 130), (3001, 36, 64), (6000, 300, 1500), (9000, 33, 1000), (524298, 8, 1000)]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("V,D,B", FORMS)
def test_softmax_calls_on_tensors_off_their_boundaries(V, D, B, name):
    """The same bits; a loss corrected by sums of other parts within 8 H of what the sums hold."""
    dt = TYPES[name]
    x, w, t = large_case(V, D, B, dt)
    k = tokens.build_token_update(V, D, B, "tanh", dt, 0.3)
    score = tokens.build_token_loss(V, D, B, "tanh", dt)
    ws, ws2 = k.new_workspace(DEV), score.new_workspace(DEV)
    got = []
    for by in (0, 1, 2, 3, 6):
        by_w = by if dt == torch.float32 or D % 2 else by // 2 * 2  # (rows of an even length lie on 4 bytes)
        a, v, loss, g, alone = off(x, by), off(w, by_w), off(torch.zeros(B, device=DEV), by), off(torch.zeros_like(x), by + 1), off(torch.zeros(B, device=DEV), by)
        score(a, v, t, alone, workspace=ws2)
        k(a, v, t, loss, g, workspace=ws)
        got.append((alone, g, v, loss))
    for other in got[1:]:
        assert all(torch.equal(p, q) for p, q in zip(got[0][:3], other[:3]))
        assert float((got[0][3] - other[3]).abs().max()) <= 8 * H * 64
    assert bool(torch.isfinite(got[0][3]).all())


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("V,D,C,B", [(50, 64, 3, 1), (50, 64, 3, 4), (50, 64, 3, 40), (700, 36, 2, 300), (700, 131, 1, 600)])
def test_embedding_calls_on_tensors_off_their_boundaries(V, D, C, B, name):
    dt = TYPES[name]
    g = torch.Generator(device=DEV).manual_seed(V + D)
    table, e = torch.randn((V, D), generator=g, device=DEV).to(dt), torch.randn((C * D, B), generator=g, device=DEV).to(dt)
    ids = torch.randint(-1, V, (C, B), generator=g, device=DEV)
    look, learn = tokens.build_embedding(V, D, C, B, dt, 1.5), tokens.build_embedding_update(V, D, C, B, dt, 0.1)
    ws, got = learn.new_workspace(DEV), []
    for by in (0, 1, 2, 3, 6):
        x, rows = off(torch.zeros_like(e), by + 1), off(table, by)
        look(off(ids, by), rows, x)
        learn(rows, ids, off(e, by), workspace=ws)
        got.append((x, rows))
    for other in got[1:]:
        assert all(torch.equal(p, q) for p, q in zip(got[0], other))


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("V,D,B", FORMS)
def test_targets_that_are_all_padded(V, D, B, name):
    dt = TYPES[name]
    x, w, _ = large_case(V, D, B, dt)
    x[0] = float("nan")
    loss, g, wn = run_update(x, w, torch.full((B,), -1, device=DEV), "gelu", 0.5)
    assert bool((loss == 0).all()) and bool((g == 0).all()) and torch.equal(wn, w)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("V,D,B", FORMS[5:])
def test_large_calls_in_a_graph(V, D, B, name):
    """Replays between eager calls, both in one workspace, give the eager bits."""
    dt = TYPES[name]
    x, w, t = large_case(V, D, B, dt)
    k = tokens.build_token_update(V, D, B, "silu", dt, 0.3)
    ws = k.new_workspace(DEV)

    def new():
        return w.clone(), torch.empty(B, device=DEV), torch.empty_like(x)

    eager, kept, side = new(), new(), torch.cuda.Stream()
    warm = new()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        k(x, warm[0], t, *warm[1:], workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        k(x, kept[0], t, *kept[1:], workspace=ws)
    for _ in range(3):
        k(x, eager[0], t, *eager[1:], workspace=ws)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, kept))


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("V,D,B", FORMS[3:9])
def test_one_target_in_every_column(V, D, B, name):
    x, w, t = large_case(V, D, B, TYPES[name])
    check_update(x, w, torch.full_like(t, V - 1), "relu", 0.25 / B)


@pytest.mark.parametrize("name", TYPES)
def test_calls_on_two_streams_at_once(name):
    """Each with a workspace of its own."""
    dt, V, D, B = TYPES[name], 6000, 300, 1500
    x, w, t = large_case(V, D, B, dt)
    k = tokens.build_token_update(V, D, B, "gelu", dt, 0.3)
    want = run_update(x, w, t, "gelu", 0.3)
    streams, calls = [torch.cuda.Stream() for _ in range(3)], []
    for _ in streams:
        calls.append((k.new_workspace(DEV), w.clone(), torch.empty(B, device=DEV), torch.empty_like(x)))
    torch.cuda.synchronize()
    for s, (ws, v, loss, g) in zip(streams, calls):
        with torch.cuda.stream(s):
            k(x, v, t, loss, g, workspace=ws)
    torch.cuda.synchronize()
    for _, v, loss, g in calls:
        assert torch.equal(v, want[2]) and torch.equal(loss, want[0]) and torch.equal(g, want[1])
