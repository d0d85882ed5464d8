"""Nets in microscaled storage against the same steps in 64 bits, and the command."""
import pytest
import torch

import mx_oracle as O
from lich_amd import cli
from lich_amd.compact import CompactNet, FourBitSteps

pytestmark = pytest.mark.gpu
DIMS, B = (10, 65, 96, 200), 70


def _inputs(seed):
    g = torch.Generator().manual_seed(seed)
    w = [(torch.rand(m, k, generator=g, dtype=torch.float64) * 2 - 1) * (6 / (m + k)) ** 0.5 for m, k in zip(DIMS, DIMS[1:])]
    x = torch.rand(DIMS[-1], B, generator=g, dtype=torch.float64)
    y = torch.nn.functional.one_hot(torch.randint(0, 10, (B,), generator=g), 10).T.double().contiguous()
    return [t.float().double() for t in w], x.float().double(), y


@pytest.mark.parametrize("act", ["relu", "tanh", "gelu"])
def test_a_training_step(act):
    """The weights after one step: fp32 sums over at most 200 terms through three
    layers, a code of a state that turns (its value within 2^-20 of the middle
    of two) moves one gradient by a 128th at most; the step is 0.1 / 70 of it."""
    w, x, y = _inputs(1)
    net = CompactNet(DIMS, B, act, rate=0.1, weights=w)
    net.step(x.float().cuda(), y.float().cuda())
    state, kept = x, []
    for l in (2, 1, 0):
        kept.insert(0, O.quantised(state, "int8"))
        state = w[l] @ O.f(act, state)
    e, want = y - state, []
    for l in range(3):
        want.append(w[l] + 0.1 / B * (e @ O.f(act, kept[l]).T.contiguous()))
        e = O.df(act, kept[l]) * (w[l].T.contiguous() @ e)
    for got, ref, w0 in zip(net.w, want, w):
        moved = (ref - w0).abs().max()
        assert float((got.cpu().double() - ref).abs().max()) <= 0.02 * float(moved) + 2.0 ** -23
    packed, full = net.bytes_kept()
    assert packed < 0.4 * full


@pytest.mark.parametrize("n", [1, 7, 64, 130])
def test_answers_with_packed_weights(n):
    w, x, _ = _inputs(2)
    net = CompactNet(DIMS, B, "relu", weights=w)
    got = net.predict(x[:, :1].repeat(1, n).float().cuda() if n > B else x[:, :n].float().cuda())
    state = x[:, :1].repeat(1, n) if n > B else x[:, :n]
    for l in (2, 1, 0):
        f = O.f("relu", state)
        f = f if n <= 64 else O.quantised(f.T.contiguous(), "fp4").T.contiguous()
        state = O.quantised(w[l], "fp4") @ f
    # fp32 sums; for a batch a code that turns moves its state by a quarter at most, of some forty that count
    tol = 1e-5 if n <= 64 else 0.05
    assert float((got.cpu().double() - state).abs().max()) <= tol * float(state.abs().max())


def test_four_bit_steps():
    """One iPC step on 4-bit operands (relu: nothing rounds differently before the
    products)."""
    w, x, y = _inputs(3)
    states = [x]
    for l in (2, 1, 0):
        states.insert(0, (w[l] @ O.f("relu", states[0])).float().double())
    states[0] = y
    q = O.quantised
    steps = FourBitSteps([t.float().cuda() for t in states], [t.float().cuda() for t in w], "relu", 1e-2, 0.1)
    steps.step()
    e = [states[l] - q(w[l], "fp4") @ q(O.f("relu", states[l + 1]).T.contiguous(), "fp4").T for l in range(3)]
    for l in range(3):
        assert float((steps.e[l].cpu().double() - e[l]).abs().max()) <= 1e-5 * float(1 + e[l].abs().max())
    # the updates quantise the errors the GPU computed
    ge = [t.cpu().double() for t in steps.e]
    nx = list(states)
    for l in (1, 2):
        up = q(w[l - 1].T.contiguous(), "fp4") @ q(ge[l - 1].T.contiguous(), "fp4").T
        nx[l] = states[l] + 0.1 * (-ge[l] + O.df("relu", states[l]) * up)
        assert float((steps.x[l].cpu().double() - nx[l]).abs().max()) <= 1e-5 * float(1 + nx[l].abs().max())
    gx = [t.cpu().double() for t in steps.x]
    for l in range(3):
        nw = w[l] + 1e-2 * (q(ge[l], "fp4") @ q(O.f("relu", gx[l + 1]), "fp4").T)
        assert float((steps.w[l].cpu().double() - nw).abs().max()) <= 1e-5 * float(1 + nw.abs().max())
    assert abs(steps.energy() - sum(float((t ** 2).sum()) for t in ge) / 2) <= 1e-9 * steps.energy()


def test_the_command(capsys):
    """Eight epochs of eight batches learn the synthetic classes (the same loop in
    plain torch, scored with weights and states rounded to 4 bits: 0.99)."""
    assert cli.main(["compact", "--synthetic", "1024"]) == 0
    out = capsys.readouterr().out
    assert "epoch=008" in out and "first sample" in out and "energies" in out
    assert float(out.split("epoch=008")[1].split("train_acc (4-bit weights)=")[1].split()[0]) > 0.9


def test_refusals():
    with pytest.raises(ValueError, match="dims"):
        CompactNet((10, 20), 4, weights=[torch.zeros(10, 21)])
    with pytest.raises(ValueError, match="state"):
        FourBitSteps([torch.zeros(4, 2)], [torch.zeros(4, 4)])


def test_answers_after_a_step():
    """The weights of the last step answer, not those that an answer before it packed."""
    w, x, y = _inputs(4)
    xd, yd = x.float().cuda(), y.float().cuda()
    net = CompactNet(DIMS, B, "tanh", rate=2.0, weights=w)
    before = net.predict(xd)
    for _ in range(2):
        net.step(xd, yd)
        got = net.predict(xd)
        fresh = CompactNet(DIMS, B, "tanh", weights=[t.clone() for t in net.w])
        assert torch.equal(got, fresh.predict(xd)) and not torch.equal(got, before)
        before = got
