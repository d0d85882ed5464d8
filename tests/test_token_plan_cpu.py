"""How softmax calls over tokens are planned (``ipc_token_plan.h``, compiled for the CPU): what every
accepted plan has to hold, so that no kernel reads what none has written or past an operand's end."""
import itertools
import random
import subprocess
from pathlib import Path

import pytest

from lich_amd import _native as nat

ROOT = Path(__file__).resolve().parents[1]
F32, F16, BF16 = 0, 1, 2
IDENTITY, TANH = 0, 2
OPERAND = 2 ** 31 - 1
FIELDS = ("taken terms Dp Bk copy ways fine mend fix ft_terms f_terms e_terms keep one tail cut rows Vp tile unit grad_tile grad_ways "
          "slices f ft et kept ws part stats bytes last last_slices").split()


class Plan:
    def __init__(self, case, values):
        self.V, self.D, self.B, self.storage, self.act, self.update = case
        self.case = dict(zip("V D B storage act update".split(), case))
        for name, value in zip(FIELDS, values):
            setattr(self, name, value)


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    """plans(cases): the accepted ones of (V, D, B, storage, activation, update)."""
    at = tmp_path_factory.mktemp("plan")
    values = ", (long long)o.".join(["(long long)taken"] + FIELDS[1:-2]) + ", last, ipc::token_piece_slices(o, last)"
    (at / "plan.cpp").write_text("""
#include <cstdio>
namespace ipc { enum { DT_F32 = 0, DT_F16 = 1, DT_BF16 = 2 }; enum { ACT_IDENTITY = 0, ACT_RELU = 1 }; }
#include "%s"
int main() {
  int V, D, B, storage, act, update;
  while (scanf("%%d %%d %%d %%d %%d %%d", &V, &D, &B, &storage, &act, &update) == 6) {
    ipc::TokenPlan o;
    const bool taken = ipc::plan_token(V, D, B, storage, act, update != 0, o);
    const int last = taken ? (V - 1) %% o.rows + 1 : 0;  // rows of the last piece
    const long long all[] = {%s};
    for (long long v : all) printf("%%lld ", v);
    printf("\\n");
  }
}
""" % (ROOT / "lich_amd" / "csrc" / "ipc_token_plan.h", values))
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-o", str(at / "plan"), str(at / "plan.cpp")], check=True)

    def run(cases):
        cases = list(cases)
        text = "\n".join(" ".join(str(int(v)) for v in c) for c in cases)
        out = subprocess.run([str(at / "plan")], input=text, capture_output=True, text=True, check=True).stdout.splitlines()
        assert len(out) == len(cases)
        got = [Plan(c, map(int, line.split())) for c, line in zip(cases, out)]
        return [p for p in got if p.taken]

    return run


def size(rng, low, high):
    v = int(round(low * (high / low) ** rng.random()))
    return v // 64 * 64 if rng.random() < 0.5 and v >= 64 else v


def some_cases():
    """Sizes of every kind, those with states near an operand's limit in one, two or three terms among them."""
    rng = random.Random(3)
    yield from itertools.product((1, 2, 47, 64, 65, 128, 300, 481, 2048, 2049, 32000, 262144), (1, 8, 60, 513, 2260, 16384),
                                 (1, 9, 128, 4096, 24576, 164689, 8000000), (F32, F16, BF16), (IDENTITY, TANH), (0, 1))
    for _ in range(40000):
        V, D = size(rng, 1, 1 << 20), size(rng, 1, 1 << 15)
        B = size(rng, 1, 1 << 20) if rng.random() < 0.5 else int((2 ** 30 / rng.uniform(0.9, 4)) / D)
        if V * D <= OPERAND and V * B <= OPERAND and 1 <= D * B <= OPERAND:
            yield V, D, B, rng.choice((F32, F16, BF16)), rng.choice((IDENTITY, TANH)), rng.random() < 0.7


@pytest.fixture(scope="module")
def accepted(plans):
    got = plans(c for c in some_cases() if c[0] * c[1] <= OPERAND and c[0] * c[2] <= OPERAND and c[1] * c[2] <= OPERAND)
    assert len(got) > 20000
    return got


def test_as_many_terms_are_laid_out_as_multiplied(accepted):
    """f(X)'s launch writes ft_terms terms of it in one order and the first f_terms of these in the other."""
    for p in accepted:
        if p.storage == F32:
            assert (p.ways, p.ft_terms, p.terms, p.fine, p.mend) == (1, 3, 3, 0, 0), p.case
            assert not p.update or (p.f_terms == p.e_terms == 3 and p.grad_ways == 1), p.case
            continue
        assert p.ft_terms >= p.ways, p.case
        if p.update:
            assert p.f_terms <= p.ft_terms and p.f_terms == p.e_terms, p.case
            assert p.fine != p.mend and p.grad_ways == 1 + p.fine, p.case
            most = 2 if p.storage == F16 else 3
            assert (p.ways, p.ft_terms, p.f_terms) == ((most,) * 3 if p.fine else (1, 2 if p.fix else 1, 1)), p.case


def test_every_plan_has_its_kernels(accepted):
    """The forms that ipc_token_one, _keep and _stats instantiate."""
    for p in accepted:
        one = {F32: 1, F16: 2, BF16: 3}[p.storage]
        if p.one:
            assert p.ways == one and p.V <= 128 and p.rows == p.V, p.case
        elif p.keep:
            assert p.ways in (1, one), p.case
        else:
            assert p.ways in {F32: (1,), F16: (1, 2), BF16: (1, 2, 3)}[p.storage], p.case
            assert not p.update or p.ways == 1, p.case  # (the errors' form)


def test_operands_lie_below_their_limit(accepted):
    for p in accepted:
        state = 2 * p.Dp * p.Bk
        assert state * p.ft_terms <= OPERAND and state * p.f_terms <= OPERAND, p.case
        assert 2 * p.Vp * (p.terms * p.Dp if p.copy else p.D) <= OPERAND, p.case
        assert not p.update or 2 * p.e_terms * p.Bk * p.Vp <= OPERAND, p.case


@pytest.mark.parametrize("V,D,B", [(124, 10304, 42179), (200, 10000, 40000), (47, 2260, 164689), (300, 16384, 24576), (1, 60, 8000000)])
def test_updates_whose_states_fit_in_two_terms_alone(plans, V, D, B):
    """bf16, few words: not in three terms, so not as a small call."""
    p, = plans([(V, D, B, BF16, TANH, 1)])
    assert (p.fine, p.mend, p.ways, p.ft_terms, p.f_terms, p.e_terms) == (0, 1, 1, 2, 1, 1)


def slices_of(p):
    """First stage and the one behind the last of each slice of the last piece, as product_tile has them."""
    stages = (p.last + 31) // 32
    return [(stages * s // p.last_slices, stages * (s + 1) // p.last_slices) for s in range(p.last_slices)]


def test_every_slice_of_every_piece_has_a_stage(plans, accepted):
    """A whole piece has eight stages a slice and more; the last one may be of a single row."""
    in_pieces = [(V, D, B, storage, TANH, 1) for V in (151936, 256128, 262144, 131073, 524298, 21770, 91793) for D in (64, 1024, 1949, 2048, 4096, 4192, 8192)
                 for B in (9, 64, 118, 128, 256, 1000, 4096) for storage in (F32, F16, BF16) if V * D <= OPERAND]
    short = 0
    for p in plans(in_pieces) + [p for p in accepted if p.update]:
        if p.tail:
            continue
        assert 1 <= p.slices <= max(1, p.Vp // 32 // 8), p.case
        assert 1 <= p.last_slices <= p.slices, p.case
        for begin, end in slices_of(p):
            assert 0 <= begin < end <= (p.last + 31) // 32, p.case
        short += p.rows < p.V and p.last_slices < p.slices
    assert short > 20


P = 4096  # a fake, aligned, non-null address; never dereferenced (validation fails first)


@pytest.mark.parametrize("V,D,C,B", [(10, 1, 1 << 24, 1), (10, 1, 1 << 24, 3), (5, 2, 1 << 25, 17), (100, 1, 1, 1 << 30), (100, 1, 2, 1 << 29)])
def test_embeddings_of_too_many_places_for_a_launch_are_refused(V, D, C, B):
    """2^32 work-items and more: before any of an update's launches has run."""
    lib, big = nat.lib(), 1 << 50
    for storage in (F32, F16, BF16):
        if B < 1 << 29:
            assert lib.ipc_embedding(P, P, P, V, D, C, B, 1.0, storage, None) == nat.ERR_SHAPE and "launch" in nat.last_error()
        assert lib.ipc_embedding_update(P, P, P, V, D, C, B, 1.0, storage, P, big, None) == nat.ERR_SHAPE and "launch" in nat.last_error()
        assert lib.ipc_embedding_update_workspace_bytes(V, D, C, B, storage) == 0


def test_updates_of_too_many_samples_for_a_launch_are_refused(plans):
    lib = nat.lib()
    for V, D, B in ((1, 8, 1 << 24), (3, 30, 20000000), (100, 2, 17000000)):
        for storage in (F16, BF16):
            assert lib.ipc_token_update_workspace_bytes(V, D, B, storage, TANH) == 0
            assert lib.ipc_token_update(P, P, P, P, P, V, D, B, 1.0, storage, TANH, P, 1 << 50, None) == nat.ERR_SHAPE
            assert "too large" in nat.last_error()
    assert len(plans([(1, 8, 1 << 24, BF16, IDENTITY, 0), (1, 60, 8000000, BF16, TANH, 1)])) == 2


def test_no_launch_has_too_many_work_items(accepted):
    for p in accepted:
        if p.keep and not p.one:
            runs = 1 if p.Vp <= 8192 else (p.Vp + 2047) // 2048
            assert 256 * p.Bk * runs < 1 << 32, p.case
        if p.mend:
            assert 256 * (-(-p.D // 64) * -(-p.B // 64) + p.B * -(-p.Dp // 256)) < 1 << 32, p.case


@pytest.mark.parametrize("storage", [F32, F16, BF16])
def test_pieces_bound_what_a_large_vocabulary_takes(plans, storage):
    """Errors and laid-out weights of a piece 1 GiB each, whatever the vocabulary."""
    got = plans((V, 64, B, storage, TANH, 1) for V, B in ((1 << 19, 4095), (1 << 20, 2047), (1 << 24, 127), (1 << 24, 33)))
    assert len(got) == 4 and all(p.rows < p.V and 1 << 30 < p.bytes < 3 << 30 for p in got), [(p.case, p.rows, p.bytes) for p in got]
