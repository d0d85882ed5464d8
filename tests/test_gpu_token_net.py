"""A net over tokens against the same step in 64 bits, and the command."""
import pytest
import torch

from lich_amd import cli
from lich_amd.token_net import TokenNet
from tests import mx_oracle, token_oracle as O
from tests.helpers import gen

pytestmark = pytest.mark.gpu
V, C, D, HIDDEN, B = 90, 3, 20, (48, 40), 70


def _net(dtype=torch.float32, p=0.0, rate=0.5):
    g = gen(5)
    dims = (V, *HIDDEN, C * D)
    w = [torch.randn((m, k), generator=g) / k ** 0.5 for m, k in zip(dims, dims[1:])]
    table = torch.randn((V, D), generator=g) / D ** 0.5
    ids = torch.randint(-1, V, (C, B), generator=g)
    targets = torch.randint(-1, V, (B,), generator=g)
    net = TokenNet(V, C, D, HIDDEN, B, "tanh", dtype, rate, p, seed=3, weights=[t.clone() for t in w], table=table.clone())
    return net, [t.double() for t in w], table.double(), ids, targets


@pytest.mark.parametrize("p", [0.0, 0.25])
def test_a_training_step(p):
    """fp32 sums over at most 90 terms through three layers (2^-15 of the largest change with room);
    a code of a kept state that turns, its value within 2^-20 of the middle of two, moves
    one gradient by a 128th at most: a fiftieth of the change in all, as for the net
    over images."""
    net, w, table, ids, targets = _net(p=p)
    loss = net.step(ids.cuda(), targets.cuda())
    assert int(net.rng[1]) == 1
    masks = [None] * 4
    dropped = round(p * 65536)
    for l, n in enumerate((V, *HIDDEN, C * D)):
        masks[l] = O.kept(n * B, 3, 0, l, dropped).reshape(n, B).double() * 65536 / (65536 - dropped)
    state = O.embedding(ids, table, D ** 0.5) * masks[3]
    kept = [None] * 3
    for l in (2, 1):
        kept[l] = mx_oracle.quantised(state, "int8")
        state = (w[l] @ O.act("tanh", state)) * masks[l]
    r = O.softmax(state, w[0], targets, "tanh")
    rate = 0.5 / B
    want = [w[0] + rate * r["dw"]]
    e = r["g"]
    for l in (1, 2):
        e = e * masks[l]
        want.append(w[l] + rate * e @ O.act("tanh", kept[l]).T.contiguous())
        e = O.dact("tanh", kept[l]) * (w[l].T.contiguous() @ e)
    moved = O.embedding_sums(ids, e * masks[3], V)[0]
    want_table = table + rate * D ** 0.5 * moved
    assert float((loss.cpu().double() - r["loss"]).abs().max()) <= 2.0 ** -15 * float(r["loss"].max())
    for got, ref, old in zip(net.w + [net.table], want + [want_table], w + [table]):
        change = (ref - old).abs().max()
        assert float(change) > 0
        assert float((got.cpu().double() - ref).abs().max()) <= 0.02 * float(change) + 2.0 ** -22


def test_losses_and_answers():
    net, w, table, ids, targets = _net()
    state = O.embedding(ids, table, D ** 0.5)
    exact = state.clone()
    for l in (2, 1):
        exact = w[l] @ O.act("tanh", exact)
    want = O.softmax(exact, w[0], targets, "tanh")["loss"]
    got = net.losses(ids.cuda(), targets.cuda())
    assert float((got.cpu().double() - want).abs().max()) <= 2.0 ** -16 * float(want.max())
    for l in (2, 1, 0):
        state = mx_oracle.quantised(w[l], "fp4") @ O.act("tanh", state)
    few = net.predict(ids[:, :5].cuda().contiguous())
    assert float((few.cpu().double() - state[:, :5]).abs().max()) <= 1e-5 * float(state.abs().max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_steps_in_16_bits(dtype):
    net, w, table, ids, targets = _net(dtype, p=0.1)
    first = net.step(ids.cuda(), targets.cuda())
    for _ in range(3):
        loss = net.step(ids.cuda(), targets.cuda())
    assert bool(torch.isfinite(loss).all()) and bool((loss[targets.cuda() < 0] == 0).all())
    assert not torch.equal(first, loss)


def test_the_command(capsys, tmp_path):
    assert cli.main(["tokens", "--synthetic", "3000", "--vocab", "50", "--epochs", "2", "--dropout", "0.1", "--batch", "64"]) == 0
    out = capsys.readouterr().out
    assert "epoch=002" in out and "4-bit weights" in out
    text = tmp_path / "text.txt"
    text.write_text("one two three two one three three one two " * 40)
    assert cli.main(["tokens", "--text", str(text), "--words", "2", "--epochs", "1", "--depth", "0", "--dtype", "bfloat16"]) == 0
    assert cli.main(["tokens", "--text", str(text), "--epochs", "1", "--depth", "2", "--hidden", "33"]) == 0
