"""Softmax calls over tokens where their plans change: states near an operand's limit, short last
pieces, against their definitions in 64 bits on the device (bounds: those of test_gpu_tokens.py)."""
import pytest
import torch

from tests import token_oracle as O
from tests.helpers import DEV
from tests.test_gpu_tokens import TYPES, run_update, softmax_bounds

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


# states that fit an operand in two terms but not in three; the last three in fp16, which takes two
@pytest.mark.parametrize("V,D,B,activation,name", [(200, 10000, 40000, "tanh", "bf16"), (2, 8200, 50000, "relu", "bf16"), (1, 500, 800000, "gelu", "bf16"),
                                                   (300, 16384, 24576, "silu", "bf16"), (40, 20000, 20000, "tanh", "f16"), (3, 30000, 20000, "relu", "f16")])
def test_updates_of_large_states(V, D, B, activation, name):
    check_update(*large_case(V, D, B, TYPES[name]), activation, 0.5)


# vocabularies in pieces whose last one has fewer stages of 32 rows than a whole one has slices
@pytest.mark.parametrize("V,D,B,name", [(524298, 64, 1000, "bf16"), (524289, 8, 1000, "f16"), (131073, 300, 4096, "f16"), (21770, 8192, 64, "f32"), (91793, 1949, 118, "f32")])
def test_short_last_pieces(V, D, B, name):
    check_update(*large_case(V, D, B, TYPES[name]), "tanh", 0.5)
