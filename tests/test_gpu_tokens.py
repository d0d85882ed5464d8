"""Operators over tokens against their definitions in 64 bits.

Tolerances: u is half a step of the storage type (bf16 2^-8, fp16 2^-11, fp32 2^-24), H = 2^-24 the
fp32 arithmetic's.  Bounds are per element and worst case: a sum of n products of
magnitudes summing to S is off by at most (n + 2) H S; the activations are within
16 H of theirs, relative."""
import pytest
import torch

from lich_amd import tokens
from tests import token_oracle as O
from tests.helpers import DEV, gen

pytestmark = pytest.mark.gpu

H = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def check(got, want, bound, what):
    got, want, bound = got.detach().cpu().double(), want.cpu(), bound.cpu()
    assert bool(torch.isfinite(got).all()), what
    over = ((got - want).abs() - bound).max()
    assert float(over) <= 0, f"{what}: {float(over):.3e} over a bound of {float(bound.max()):.3e} at most"


def randn(shape, g, dtype, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def some_ids(V, shape, g, padded=0.2):
    """Ids with many repeats of a few, and padded places of three kinds."""
    ids = torch.where(torch.rand(shape, generator=g) < 0.5, torch.randint(0, V, shape, generator=g),
                      torch.randint(0, min(V, 3), shape, generator=g))
    bad = torch.tensor([-1, V, 2 ** 40])[torch.randint(0, 3, shape, generator=g)]
    return torch.where(torch.rand(shape, generator=g) < padded, bad, ids)


# ------------------------------------------------------------------ embedding
SIZES = [(1, 1, 1, 1), (5, 3, 1, 1), (7, 1030, 3, 1), (40, 17, 2, 3), (11, 1029, 1, 4), (64, 33, 5, 9), (100, 260, 2, 16),
         (130, 65, 3, 17), (1000, 64, 8, 64), (333, 129, 4, 131), (3000, 131, 5, 301)]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("V,D,C,B", SIZES)
def test_embedding(V, D, C, B, name):
    dt, g = TYPES[name], gen(V + D)
    ids, table = some_ids(V, (C, B), g), randn((V, D), g, dt)
    x = torch.full((C * D, B), float("nan"), dtype=dt, device=DEV)
    tokens.build_embedding(V, D, C, B, dt, 1.7)(ids.to(DEV), table.to(DEV), x)
    want = O.embedding(ids, table, torch.tensor(1.7, dtype=torch.float32).item())
    # the product rounded to fp32, then to the type
    check(x, want, (half_step(dt) + 2 * H) * want.abs() + 2.0 ** -25 * (dt == torch.float16), "x")


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("V,D,C,B", SIZES + [(3, 20, 1, 513), (1, 7, 2, 700), (70000, 5, 3, 1000), (600000, 4, 1, 520), (50, 1100, 1, 600)])
def test_embedding_update(V, D, C, B, name):
    dt, gn = TYPES[name], gen(V + D + 1)
    ids, table, g = some_ids(V, (C, B), gn), randn((V, D), gn, dt), randn((C * D, B), gn, dt)
    k = tokens.build_embedding_update(V, D, C, B, dt, 0.3)
    assert (k.workspace_bytes > 0) == (C * B >= 513)
    t = table.to(DEV)
    k(t, ids.to(DEV), g.to(DEV), workspace=k.new_workspace(DEV))
    total, size, many = O.embedding_sums(ids, g, V)
    alpha = torch.tensor(0.3, dtype=torch.float32).item()
    want = table.double() + alpha * total
    bound = half_step(dt) * want.abs() + 2.0 ** -25 * (dt == torch.float16) + (many[:, None] + 4) * H * alpha * size + 4 * H * (table.double().abs() + want.abs())
    check(t, want, bound * 1.01, "table")
    unused = many == 0
    assert torch.equal(t.cpu()[unused], table[unused])


def test_embedding_update_gives_the_same_bits():
    V, D, C, B = 1000, 96, 3, 700
    g = gen(4)
    ids, table, e = some_ids(V, (C, B), g).to(DEV), randn((V, D), g, torch.float32).to(DEV), randn((C * D, B), g, torch.float32).to(DEV)
    k = tokens.build_embedding_update(V, D, C, B, "float32", 0.1)
    got = []
    for _ in range(3):
        t = table.clone()
        k(t, ids, e, workspace=k.new_workspace(DEV))
        got.append(t)
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


def test_embedding_update_of_padded_places_only():
    V, D, C, B = 100, 9, 2, 400
    table = torch.randn((V, D), device=DEV)
    t = table.clone()
    k = tokens.build_embedding_update(V, D, C, B, "float32", 0.1)
    k(t, torch.full((C, B), -1, device=DEV), torch.full((C * D, B), float("nan"), device=DEV), workspace=k.new_workspace(DEV))
    assert torch.equal(t, table)


# -------------------------------------------------------------------- dropout
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("M,B,p", [(1, 1, 0.5), (3, 5, 0.0), (7, 9, 0.1), (64, 33, 0.25), (129, 8, 0.9), (40, 64, 65535 / 65536)])
def test_dropout(M, B, p, name):
    dt, g = TYPES[name], gen(M + B)
    seed, step, site = 0x123456789ABCDEF, -3, 7
    x = randn((M, B), g, dt)
    x[0, 0] = float("inf")
    rng, xd = torch.tensor([seed, step], device=DEV), x.to(DEV)
    out = torch.full_like(xd, float("nan"))
    k = tokens.build_dropout(M, B, dt, p, site=site)
    k(xd, rng, out)
    dropped = round(p * 65536)
    keep = O.kept(M * B, seed, step, site, dropped).reshape(M, B)
    want = torch.where(keep, x.double() * 65536 / (65536 - dropped), torch.zeros((), dtype=torch.float64))
    # share, product and result are rounded; at the type's end the result may be infinite
    top = torch.finfo(dt).max
    fine = want.abs() <= top
    got = out.cpu().double()
    assert torch.equal(got == 0, (want == 0) | ~keep)
    assert bool(((got - want).abs()[fine] <= (half_step(dt) + 3 * H) * want.abs()[fine] + 2.0 ** -25 * (dt == torch.float16)).all())
    assert bool(torch.isinf(got[~fine]).all())
    k(xd, rng, xd)  # in place
    assert torch.equal(torch.nan_to_num(xd), torch.nan_to_num(out))


def test_dropout_of_a_view_off_16_bytes():
    M, B = 33, 31
    base = torch.randn(M * B + 1, device=DEV)
    rng = torch.tensor([5, 6], device=DEV)
    k = tokens.build_dropout(M, B, "float32", 0.5)
    want, out = torch.empty((M, B), device=DEV), torch.full((M * B + 2,), 9.0, device=DEV)
    k(base[1:].reshape(M, B).clone(), rng, want)
    k(base[1:].reshape(M, B), rng, out[1:-1].reshape(M, B))
    assert torch.equal(out[1:-1].reshape(M, B), want) and float(out[0]) == float(out[-1]) == 9.0


# ------------------------------------------- tensors of more than 2^32 bytes
def test_rows_behind_four_gigabytes():
    V, D, C, B = 1100000, 1944, 2, 300
    table = torch.empty((V, D), dtype=torch.bfloat16, device=DEV)
    last = 700
    table[:last].normal_()
    table[-last:].normal_()
    ids = torch.cat([torch.randint(0, last, (1, B), device=DEV), torch.randint(V - last, V, (1, B), device=DEV)])
    x = torch.empty((C * D, B), dtype=torch.bfloat16, device=DEV)
    tokens.build_embedding(V, D, C, B, "bfloat16", 1.0)(ids, table, x)
    assert torch.equal(x.reshape(C, D, B).transpose(1, 2), table[ids])
    far, near = table[-last:].clone(), table[:last].clone()
    k = tokens.build_embedding_update(V, D, C, B, "bfloat16", 0.5)
    k(table, ids, x, workspace=k.new_workspace(DEV))
    for part, old, rows in ((ids[0], near, table[:last]), (ids[1] - (V - last), far, table[-last:])):
        want = old.clone()
        small = tokens.build_embedding_update(last, D, 1, B, "bfloat16", 0.5)
        # (the same sums in other runs: one more rounding each of at most 300 fp32 additions)
        small(want, part.reshape(1, B), old[part].t().contiguous(), workspace=small.new_workspace(DEV))
        assert bool(((want.double() - rows.double()).abs() <= 2 * half_step(torch.bfloat16) * rows.double().abs() + 2.0 ** -12).all())


def test_dropout_behind_four_gigabytes():
    M, B = 40001, 53001
    x = torch.empty((M, B), dtype=torch.bfloat16, device=DEV)
    x[-1] = 1.0
    tokens.build_dropout(M, B, "bfloat16", 0.5, site=3)(x, torch.tensor([9, 8], device=DEV), x)
    got = x[-1].cpu()
    for i in (M * B - 1, M * B - 100, M * B - B):
        word = O.philox((i // 8, 3, 8, 0), (9, 0))[i % 8 // 2]
        assert float(got[i - (M - 1) * B]) == (2.0 if (word >> (16 * (i % 2))) & 0xFFFF >= 32768 else 0.0)


# -------------------------------------------------------------------- softmax
def softmax_bounds(r, w, dt, V, D, B, activation, alpha, update=True):
    """Per element: what loss, G and W may be off by."""
    u, half, f32 = half_step(dt), dt == torch.float16, dt == torch.float32
    exact = activation in ("identity", "relu") and not f32
    # f rounded to the type (identity, relu: exact); fp32: three bf16 terms, six of nine products
    df = 0.0 if exact else 17 * H if f32 else u + 17 * H
    products = 6 if f32 else 1
    wa, fa, ea = w.double().abs(), r["f"].abs(), r["e"].abs()
    small = 2.0 ** -25 * half  # half of fp16's smallest number
    sums = (8 * H if f32 else 0) + (products * D + 4) * H
    dz = (r["size"] * (df + sums)).max(0).values + small * wa.sum(1).max()
    near = 2.0 ** -19  # exp and log: the exponent's own rounding, 2^-24 of at most 32 where a result counts
    de = r["p"] * ((2 * dz).expm1() + near + (V + 64) * H) + (u if not f32 else H) * ea + (2.0 ** -35 if half else H)
    if not f32:  # kept as fp16 times 2^15 of a part's largest
        de = de + r["p"] * 2.0 ** -11 + 2.0 ** -39
    n = (V + 64) * products
    back = wa.T @ de + n * H * (wa.T @ ea)
    g = r["df"].abs() * back + (u + 20 * H) * r["g"].abs() + 16 * H * (wa.T @ ea) + small
    # the loss: f in two terms, or corrected to first order by back's sums
    df2 = df if exact or f32 else 17 * H + u * u
    dz2 = (r["size"] * (df2 + sums + H)).max(0).values + small * 2.0 ** -11 * wa.sum(1).max()
    loss = 2 * dz2 + near * (1 + r["loss"].abs()) + (V + 64) * H
    if update and not exact and not f32:
        loss = loss + dz ** 2 * (2 * dz).exp() + ((back + D * H * (wa.T @ ea)) * (fa * u + small)).sum(0) + 20 * H * (wa.T @ ea * fa).sum(0)
    dw = de @ fa.T + ea @ (fa * df).T + (B * products + 8) * H * (ea @ fa.T) + small * ea.sum(1, keepdim=True)
    new = w.double() + alpha * r["dw"]
    return loss * 1.01, g * 1.01, (alpha * dw + (u + 2 * H) * new.abs() + 4 * H * w.double().abs() + small) * 1.01


def softmax_case(V, D, B, dt, seed, padded=0.15, wscale=None):
    g = gen(seed)
    x, w = randn((D, B), g, dt), randn((V, D), g, dt, wscale if wscale is not None else 2.0 / D ** 0.5)
    return x, w, some_ids(V, (B,), g, padded)


def run_update(x, w, targets, activation, alpha):
    (D, B), V, dt = x.shape, w.shape[0], x.dtype
    k = tokens.build_token_update(V, D, B, activation, dt, alpha)
    w = w.clone()
    loss, g = torch.full((B,), float("nan"), device=DEV), torch.full((D, B), float("nan"), dtype=dt, device=DEV)
    ws = k.new_workspace(DEV)
    ws.fill_(255)  # (a NaN in every type)
    k(x, w, targets, loss, g, workspace=ws)
    return loss, g, w


SOFTMAX = [(1, 1, 1), (2, 1, 1), (1, 5, 3), (10, 64, 128), (3, 33, 2), (17, 31, 65), (65, 40, 64), (257, 96, 33), (1000, 37, 130),
           (130, 515, 77), (2001, 300, 257), (5003, 64, 300), (300, 1100, 1), (4100, 70, 5)]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("V,D,B", SOFTMAX)
def test_token_update(V, D, B, name):
    dt = TYPES[name]
    activation = ["identity", "relu", "tanh", "sigmoid", "silu", "gelu"][(V + D + B) % 6]
    x, w, t = softmax_case(V, D, B, dt, V + D + B)
    alpha = 0.25
    loss, g, wn = run_update(x.to(DEV), w.to(DEV), t.to(DEV), activation, alpha)
    r = O.softmax(x, w, t, activation)
    bl, bg, bw = softmax_bounds(r, w, dt, V, D, B, activation, alpha)
    check(loss, r["loss"], bl, "loss")
    check(g, r["g"], bg, "g")
    check(wn, w.double() + alpha * r["dw"], bw, "w")
    padded = (t < 0) | (t >= V)
    assert bool((loss.cpu()[padded] == 0).all()) and bool((g.cpu()[:, padded] == 0).all())


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("activation", ["identity", "relu", "tanh", "sigmoid", "silu", "gelu"])
def test_token_loss(activation, name):
    dt = TYPES[name]
    for V, D, B in ((10, 64, 128), (999, 77, 3), (300, 130, 90)):
        x, w, t = softmax_case(V, D, B, dt, V)
        k = tokens.build_token_loss(V, D, B, activation, dt)
        loss, wd = torch.full((B,), float("nan"), device=DEV), w.to(DEV)
        k(x.to(DEV), wd, t.to(DEV), loss, workspace=k.new_workspace(DEV))
        r = O.softmax(x, w, t, activation)
        check(loss, r["loss"], softmax_bounds(r, w, dt, V, D, B, activation, 0.0, False)[0], "loss")
        assert torch.equal(wd.cpu(), w)


# vocabularies whose errors take more than a piece, or (the last) whose exponentials do not fit beside them
@pytest.mark.parametrize("V,D,B,name", [(140003, 24, 4000, "bf16"), (131075, 7, 4200, "f16"), (45000, 16, 4001, "f32"),
                                        (120000, 8, 1000, "f32")])
def test_token_update_in_pieces(V, D, B, name):
    dt = TYPES[name]
    x, w, t = (v.to(DEV) for v in softmax_case(V, D, B, dt, V + D + B))
    loss, g, wn = run_update(x, w, t, "tanh", 2.0)
    r = O.softmax(x, w, t, "tanh")
    bl, bg, bw = softmax_bounds(r, w, dt, V, D, B, "tanh", 2.0)
    check(loss, r["loss"], bl, "loss")
    check(g, r["g"], bg, "g")
    check(wn, w.double() + 2.0 * r["dw"], bw, "w")


# Weights in 16 bits are the roundings of sums that are good to a few H, where an operand rounded to
# 16 bits would leave u: a weight may differ from the exact sum's rounding only where that
# lies within the sums' bound of a tie.  e: of small calls as fp32, of large ones (the last two) that of the
# targets alone; the others are probabilities of a large vocabulary.  Sums over the
# vocabulary are trees of parts: 256 H.
@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("V,D,B,activation", [(400, 6, 9, "relu"), (3000, 8, 12, "gelu"), (90, 7, 40, "silu"), (524301, 8, 17, "relu"),
                                              (700001, 6, 13, "tanh")])
def test_weights_round_as_the_exact_sums(V, D, B, activation, name):
    dt, alpha = TYPES[name], 0.25
    u, half, few = half_step(dt), dt == torch.float16, V * B <= 1 << 23
    x, w, t = softmax_case(V, D, B, dt, V + D)
    got = run_update(x.to(DEV), w.to(DEV), t.to(DEV), activation, alpha)[2].cpu()
    r = O.softmax(x, w, t, activation)
    hot = torch.zeros((V, B), dtype=torch.bool)
    real = (t >= 0) & (t < V)
    hot[t[real], real.nonzero()[:, 0]] = True
    exact = activation in ("identity", "relu")
    fa, ea, p, small = r["f"].abs(), r["e"].abs(), r["p"], 2.0 ** -25 * half
    fine_df = 0.0 if exact else 18 * H + (0.0 if few else u * u)
    logit_df = fine_df if few else 0.0 if exact else u + 17 * H
    dz = (r["size"] * (logit_df + (3 * D + 4) * H)).max(0).values + small * w.double().abs().sum(1).max()
    de = p * ((2 * dz).expm1() + 8 * H * (1 + p.clamp(min=1e-300).log().abs()) + 256 * H) + 4 * H * ea + 2.0 ** -34 * half + 2.0 ** -38 * (not few)
    if not few:
        de = de + torch.where(hot, 0.0, (u + 2.0 ** -11) * ea)
    left = torch.where(hot | few, fine_df, 0.0 if exact else u + 17 * H)
    new = w.double() + alpha * r["dw"]
    bound = alpha * (de @ fa.T + (ea * left) @ fa.T + (3 * B + 10) * H * (ea @ fa.T) + small * ea.sum(1, keepdim=True)) + 2 * H * (new.abs() + (alpha * r["dw"]).abs())
    low, high = (new - bound).to(dt), (new + bound).to(dt)
    assert bool(((got >= low) & (got <= high)).all()), int(((got < low) | (got > high)).sum())
    # (operands rounded to 16 bits would not pass, but where they are e of nearly 1 and an exact f)
    plain = (w.double() + alpha * (r["e"].to(dt).double() @ r["f"].to(dt).double().T)).to(dt)
    assert bool(((plain < low) | (plain > high)).any()) or (not few and exact)


# a few samples: every number of them, rows that end inside 16 bytes, one piece of a row or many
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("V,D,B", [(9, 8, 1), (1000, 9, 2), (700, 15, 1), (257, 129, 3), (40, 513, 4), (6001, 701, 3), (2500, 2055, 4), (513, 520, 5),
                                   (90, 1021, 7), (3, 300, 8), (33, 36000, 1), (20000, 16, 2)])
def test_a_few_samples(V, D, B, name):
    dt = TYPES[name]
    activation = ["tanh", "identity", "gelu", "relu", "silu", "sigmoid"][(V + D + B) % 6]
    x, w, t = softmax_case(V, D, B, dt, V + D + B, padded=0.0 if B == 1 else 0.3)
    loss, g, wn = run_update(x.to(DEV), w.to(DEV), t.to(DEV), activation, 0.25)
    r = O.softmax(x, w, t, activation)
    bl, bg, bw = softmax_bounds(r, w, dt, V, D, B, activation, 0.25)
    check(loss, r["loss"], bl, "loss")
    check(g, r["g"], bg, "g")
    check(wn, w.double() + 0.25 * r["dw"], bw, "w")
    k, alone = tokens.build_token_loss(V, D, B, activation, dt), torch.full((B,), float("nan"), device=DEV)
    k(x.to(DEV), w.to(DEV), t.to(DEV), alone, workspace=k.new_workspace(DEV))
    check(alone, r["loss"], softmax_bounds(r, w, dt, V, D, B, activation, 0.0, False)[0], "the loss alone")


# a vocabulary within one tile, and the first that is not
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("V,D,B", [(64, 300, 200), (63, 33, 1000), (2, 3001, 40), (100, 90, 65), (128, 512, 33), (127, 7, 700), (128, 513, 40), (129, 60, 70), (6, 73, 3026), (329, 3, 2059), (480, 33, 900),
                                   (1, 400, 100)])
def test_a_vocabulary_within_a_tile(V, D, B, name):
    dt = TYPES[name]
    activation = ["silu", "sigmoid", "tanh", "identity", "gelu", "relu"][(V + D + B) % 6]
    x, w, t = softmax_case(V, D, B, dt, V + D + B, padded=0.2)
    loss, g, wn = run_update(x.to(DEV), w.to(DEV), t.to(DEV), activation, 0.25)
    r = O.softmax(x, w, t, activation)
    bl, bg, bw = softmax_bounds(r, w, dt, V, D, B, activation, 0.25)
    check(loss, r["loss"], bl, "loss")
    check(g, r["g"], bg, "g")
    check(wn, w.double() + 0.25 * r["dw"], bw, "w")
    k, alone = tokens.build_token_loss(V, D, B, activation, dt), torch.full((B,), float("nan"), device=DEV)
    k(x.to(DEV), w.to(DEV), t.to(DEV), alone, workspace=k.new_workspace(DEV))
    check(alone, r["loss"], softmax_bounds(r, w, dt, V, D, B, activation, 0.0, False)[0], "the loss alone")
    padded = (t < 0) | (t >= V)
    for got in (loss, alone, g):
        assert bool((got.cpu()[..., padded] == 0).all())


# large products: few words (bf16 as small calls), targets' rows made good, the widest tiles
@pytest.mark.parametrize("V,D,B,name", [(600, 4000, 1000, "bf16"), (601, 3999, 1001, "f16"), (3000, 1500, 600, "bf16"), (6000, 700, 1030, "f16"),
                                        (4000, 500, 1000, "f16"), (2000, 1030, 500, "f32")])
def test_token_update_of_large_products(V, D, B, name):
    dt = TYPES[name]
    x, w, t = (v.to(DEV) for v in softmax_case(V, D, B, dt, V + D + B))
    loss, g, wn = run_update(x, w, t, "gelu", 0.5)
    r = O.softmax(x, w, t, "gelu")
    bl, bg, bw = softmax_bounds(r, w, dt, V, D, B, "gelu", 0.5)
    check(loss, r["loss"], bl, "loss")
    check(g, r["g"], bg, "g")
    check(wn, w.double() + 0.5 * r["dw"], bw, "w")


# weights of more than a piece under few columns
@pytest.mark.parametrize("V,D,B,name", [(300001, 2001, 1, "bf16"), (600001, 2000, 2, "f16"), (14001, 40001, 1, "bf16"), (30000, 40000, 1, "f16")])
def test_token_update_of_a_large_table_and_one_sample(V, D, B, name):
    dt = TYPES[name]
    g = torch.Generator(device=DEV).manual_seed(V)
    x, t = torch.randn((D, B), generator=g, device=DEV).to(dt), torch.tensor([V - 1, 5][:B], device=DEV)
    w = torch.empty((V, D), dtype=dt, device=DEV).normal_(generator=g).mul_(2.0 / D ** 0.5)
    loss, gx, wn = run_update(x, w, t, "silu", 0.5)
    r = O.softmax(x, w, t, "silu")
    bl, bg, bw = softmax_bounds(r, w, dt, V, D, B, "silu", 0.5)
    check(loss, r["loss"], bl, "loss")
    check(gx, r["g"], bg, "g")
    for rows in (slice(0, 2000), slice(V // 2, V // 2 + 2000), slice(V - 2000, V)):
        check(wn[rows], w[rows].double() + 0.5 * r["dw"][rows], bw[rows], "w")
    assert bool(torch.isfinite(wn).all())


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("V,D,B", [(10, 64, 128), (1000, 37, 130), (2001, 300, 257), (33000, 40, 7)])
def test_padded_columns_hold_anything(V, D, B, name):
    """NaN and infinities in padded columns reach nothing."""
    dt = TYPES[name]
    x, w, t = (v.to(DEV) for v in softmax_case(V, D, B, dt, V, padded=0.3))
    padded = (t < 0) | (t >= V)
    if not bool(padded.any()):
        padded[0], t[0] = True, -1
    want = run_update(torch.where(padded[None], 0, x), w, t, "gelu", 0.5)
    for junk in (float("nan"), float("inf"), -float("inf"), torch.finfo(dt).min):
        y = torch.where(padded[None], junk, x.float()).to(dt)
        got = run_update(y, w, t, "gelu", 0.5)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        k = tokens.build_token_loss(V, D, B, "gelu", dt)
        loss = torch.empty(B, device=DEV)
        k(y, w, t, loss, workspace=k.new_workspace(DEV))
        assert bool(torch.isfinite(loss).all()) and bool((loss[padded] == 0).all())


@pytest.mark.parametrize("name", TYPES)
def test_words_masked_by_their_weights(name):
    """Rows of W at the type's lowest value or at -inf under positive states: words of probability 0."""
    dt, V, D, B = TYPES[name], 300, 50, 40
    x, w, t = softmax_case(V, D, B, dt, 3, padded=0.0)
    t = t % 200
    for low in (torch.finfo(dt).min / 64, -float("inf")):
        wm = w.clone()
        wm[200:] = low
        k = tokens.build_token_loss(V, D, B, "sigmoid", dt)
        loss = torch.full((B,), float("nan"), device=DEV)
        k(x.to(DEV), wm.to(DEV), t.to(DEV), loss, workspace=k.new_workspace(DEV))
        r = O.softmax(x, w[:200], t, "sigmoid")
        check(loss, r["loss"], softmax_bounds(r, w[:200], dt, V, D, B, "sigmoid", 0.0, False)[0], "loss")
    wm[200:] = torch.finfo(dt).min / 64
    loss, g, wn = run_update(x.to(DEV), wm.to(DEV), t.to(DEV), "sigmoid", 0.5)
    assert bool(torch.isfinite(g).all()) and torch.equal(wn[200:].cpu(), wm[200:])


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("V,D,B", [(12, 9, 30), (300, 50, 2), (70000, 70, 1), (100, 60, 90), (5000, 40, 11)])
def test_words_masked_by_their_weights_in_every_size(V, D, B, name):
    dt, some = TYPES[name], V - V // 3
    x, w, t = softmax_case(V, D, B, dt, 5, padded=0.0)
    t = t % some
    for low in (torch.finfo(dt).min / 64, -float("inf")):
        wm = w.clone()
        wm[some:] = low
        k = tokens.build_token_loss(V, D, B, "sigmoid", dt)
        loss = torch.full((B,), float("nan"), device=DEV)
        k(x.to(DEV), wm.to(DEV), t.to(DEV), loss, workspace=k.new_workspace(DEV))
        r = O.softmax(x, w[:some], t, "sigmoid")
        check(loss, r["loss"], softmax_bounds(r, w[:some], dt, V, D, B, "sigmoid", 0.0, False)[0], "loss")
    wm[some:] = torch.finfo(dt).min / 64
    loss, g, wn = run_update(x.to(DEV), wm.to(DEV), t.to(DEV), "sigmoid", 0.5)
    bl, bg, _ = softmax_bounds(r, w[:some], dt, V, D, B, "sigmoid", 0.5)
    check(loss, r["loss"], bl, "loss")
    check(g, r["g"], bg, "g")
    assert torch.equal(wn[some:].cpu(), wm[some:])


@pytest.mark.parametrize("name", TYPES)
def test_calls_of_few_samples_in_a_graph(name):
    """A few samples, one tile, slices of a long batch: replays that share a workspace give the eager bits."""
    dt = TYPES[name]
    cases = []
    for V, D, B in ((900, 70, 2), (100, 60, 90), (20, 40, 1000)):
        x, w, t = (v.to(DEV) for v in softmax_case(V, D, B, dt, V))
        k = tokens.build_token_update(V, D, B, "tanh", dt, 0.3)
        cases.append((k, x, w, t))
    ws = torch.empty(max(k.workspace_bytes for k, *_ in cases), dtype=torch.uint8, device=DEV)

    def new():
        return [(w.clone(), torch.empty(x.shape[1], device=DEV), torch.empty_like(x)) for _, x, w, _ in cases]

    def run(state):
        for (k, x, _, t), (w, loss, g) in zip(cases, state):
            k(x, w, t, loss, g, workspace=ws)

    eager, kept, side = new(), new(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        run(new())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        run(kept)
    for _ in range(3):
        run(eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager, kept):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


@pytest.mark.parametrize("name", TYPES)
def test_large_and_confident_logits(name):
    """Logits of a few hundred, columns whose target has all the probability."""
    dt, V, D, B = TYPES[name], 400, 64, 65
    x, w, t = softmax_case(V, D, B, dt, 9, padded=0.0, wscale=4.0)
    t[:32] = (w.double() @ x.double()).argmax(0)[:32]
    loss, g, wn = run_update(x.to(DEV), w.to(DEV), t.to(DEV), "identity", 0.5)
    r = O.softmax(x, w, t, "identity")
    bl, bg, bw = softmax_bounds(r, w, dt, V, D, B, "identity", 0.5)
    check(loss, r["loss"], bl, "loss")
    check(g, r["g"], bg, "g")
    check(wn, w.double() + 0.5 * r["dw"], bw, "w")


def test_gradients_against_differences():
    """G and the change of W, by central differences of the loss itself (fp32: a step of 2^-5 has an error of
    h^2 / 6 of a third derivative of at most |w|^3 or |f|^3, and a rounding of 2^-22 of the loss over 2 h)."""
    V, D, B, h = 50, 12, 6, 2.0 ** -5
    x, w, t = (v.to(DEV) for v in softmax_case(V, D, B, torch.float32, 2, padded=0.0))
    k = tokens.build_token_loss(V, D, B, "tanh", "float32")
    ws = k.new_workspace(DEV)

    def total(x, w):
        loss = torch.empty(B, device=DEV)
        k(x, w, t, loss, workspace=ws)
        return float(loss.double().sum())

    _, g, wn = run_update(x, w, t, "tanh", 1.0)
    rounding = 2.0 ** -22 * total(x, w) / h
    for d, b in ((0, 0), (5, 3), (11, 5)):
        up, down = x.clone(), x.clone()
        up[d, b] += h
        down[d, b] -= h
        slope = (total(up, w) - total(down, w)) / (2 * h)
        assert abs(slope + float(g[d, b])) <= h * h * (float(w.abs().max()) + 2) ** 3 + rounding
    for v, d in ((0, 0), (1, 7), (49, 11)):
        up, down = w.clone(), w.clone()
        up[v, d] += h
        down[v, d] -= h
        slope = (total(x, up) - total(x, down)) / (2 * h)
        assert abs(slope + float((wn - w)[v, d])) <= h * h * B + rounding


@pytest.mark.parametrize("name", TYPES)
def test_calls_in_a_graph_and_on_another_stream(name):
    """Replays of all five calls with changing inputs give the eager calls' bits; two graphs share a workspace."""
    dt, V, D, C, B = TYPES[name], 700, 40, 4, 150
    g = gen(1)
    ids, t = some_ids(V, (C, B), g).to(DEV), some_ids(V, (B,), g).to(DEV)
    table0, w0 = randn((V, D), g, dt).to(DEV), randn((V, C * D), g, dt, 0.1).to(DEV)
    rng = torch.tensor([11, 0], device=DEV)
    look, drop = tokens.build_embedding(V, D, C, B, dt, 2.0), tokens.build_dropout(C * D, B, dt, 0.2, site=1)
    learn, update = tokens.build_embedding_update(V, D, C, B, dt, 0.1), tokens.build_token_update(V, C * D, B, "tanh", dt, 0.1)
    score = tokens.build_token_loss(V, C * D, B, "tanh", dt)
    ws = torch.empty(max(learn.workspace_bytes, update.workspace_bytes, score.workspace_bytes), dtype=torch.uint8, device=DEV)

    class Step:
        def __init__(self):
            self.table, self.w = table0.clone(), w0.clone()
            self.x = torch.empty((C * D, B), dtype=dt, device=DEV)
            self.g, self.loss, self.after = torch.empty_like(self.x), torch.empty(B, device=DEV), torch.empty(B, device=DEV)

        def run(self):
            look(ids, self.table, self.x)
            drop(self.x, rng, self.x)
            update(self.x, self.w, t, self.loss, self.g, workspace=ws)
            score(self.x, self.w, t, self.after, workspace=ws)
            drop(self.g, rng, self.g)
            learn(self.table, ids, self.g, workspace=ws)

    eager, one, two = Step(), Step(), Step()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        Step().run()
    torch.cuda.synchronize()
    graphs = []
    for s in (one, two):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            s.run()
        graphs.append(graph)
    for step in range(4):
        rng[1] = step
        ids.copy_(some_ids(V, (C, B), g))
        eager.run()
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for s in (one, two):
            for a, b in ((s.table, eager.table), (s.w, eager.w), (s.x, eager.x), (s.g, eager.g), (s.loss, eager.loss), (s.after, eager.after)):
                assert torch.equal(a, b), step
    assert float(eager.loss.mean()) != float(eager.after.mean())


# --------------------------------------------------- nothing written beside the tensors
class Fenced:
    """Tensors inside one larger buffer with a known value between and behind them."""

    def __init__(self, parts, room):
        offsets, at = [], room
        for shape, dtype in parts:
            size = torch.empty((), dtype=dtype).element_size()
            n = 1
            for v in shape:
                n *= v
            at = -(-at // 256) * 256
            offsets.append((at, n * size))
            at += n * size + room
        self.buffer = torch.full((at,), 0x5A, dtype=torch.uint8, device=DEV)
        self.views = [self.buffer[o:o + b].view(dtype).reshape(shape) for (o, b), (shape, dtype) in zip(offsets, parts)]
        self.mine = torch.zeros(at, dtype=torch.bool, device=DEV)
        for o, b in offsets:
            self.mine[o:o + b] = True

    def intact(self):
        return bool((self.buffer[~self.mine] == 0x5A).all())


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("activation", ["identity", "tanh"])
@pytest.mark.parametrize("V,D,B", [(2, 1, 1), (10, 64, 128), (999, 77, 3), (300, 131, 90), (26240, 1, 70), (7001, 65, 1), (700, 200, 300),
                                   (164, 2, 188), (5000, 35, 520), (1000, 9, 2), (6001, 701, 3), (520, 130, 8), (100, 90, 65), (33, 100, 300)])
def test_softmax_calls_stay_inside_their_tensors(V, D, B, activation, name):
    """Also inside the workspace's stated size; room behind each as large as the workspace itself."""
    dt = TYPES[name]
    x, w, t = softmax_case(V, D, B, dt, V + D)
    k, score = tokens.build_token_update(V, D, B, activation, dt, 0.1), tokens.build_token_loss(V, D, B, activation, dt)
    for call, inputs in ((k, 5), (score, 4)):
        f = Fenced([((D, B), dt), ((V, D), dt), ((B,), torch.int64), ((B,), torch.float32), ((D, B), dt),
                    ((call.workspace_bytes,), torch.uint8)], max(4096, call.workspace_bytes))
        for view, value in zip(f.views, (x, w, t)):
            view.copy_(value)
        call(*f.views[:inputs], workspace=f.views[5])
        assert f.intact()
        assert bool(torch.isfinite(f.views[3]).all())


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("V,D,C,B", [(5, 3, 1, 1), (130, 65, 3, 17), (47, 2, 12, 290), (300, 1, 3, 500), (3000, 131, 5, 301), (70, 64, 3, 400)])
def test_embedding_calls_stay_inside_their_tensors(V, D, C, B, name):
    dt, g = TYPES[name], gen(V)
    k = tokens.build_embedding_update(V, D, C, B, dt, 0.1)
    f = Fenced([((V, D), dt), ((C, B), torch.int64), ((C * D, B), dt), ((k.workspace_bytes,), torch.uint8)], max(4096, k.workspace_bytes))
    f.views[0].copy_(randn((V, D), g, dt))
    f.views[1].copy_(some_ids(V, (C, B), g))
    tokens.build_embedding(V, D, C, B, dt, 2.0)(f.views[1], f.views[0], f.views[2])
    assert f.intact()
    k(f.views[0], f.views[1], f.views[2], workspace=f.views[3])
    assert f.intact()
    rng = torch.tensor([1, 2], device=DEV)
    tokens.build_dropout(C * D, B, dt, 0.3)(f.views[2], rng, f.views[2])
    assert f.intact()
