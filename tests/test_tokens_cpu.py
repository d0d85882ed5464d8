"""Operators over tokens: refusals, workspaces, the generator and the data (no GPU)."""
import numpy as np
import pytest
import torch

from lich_amd import _native as nat
from lich_amd import cli, tokens
from lich_amd.data import TokenDataset, load_tokens, synthetic_tokens
from lich_amd.token_net import TokenNet
from tests import token_oracle as O

P = 4096  # a fake, aligned, non-null address; never dereferenced (validation fails first)
BIG = 1 << 40


@pytest.mark.parametrize("entry,args,code,needle", [
    ("ipc_embedding", (None, P, P, 10, 4, 2, 3, 1.0, 0, None), nat.ERR_NULL, "ids"),
    ("ipc_embedding", (P, None, P, 10, 4, 2, 3, 1.0, 0, None), nat.ERR_NULL, "table"),
    ("ipc_embedding", (P, P, P + 2, 10, 4, 2, 3, 1.0, 0, None), nat.ERR_ALIGN, "x"),
    ("ipc_embedding", (P + 4, P, P, 10, 4, 2, 3, 1.0, 0, None), nat.ERR_ALIGN, "ids"),
    ("ipc_embedding", (P, P, P, 0, 4, 2, 3, 1.0, 0, None), nat.ERR_SHAPE, "dimensions"),
    ("ipc_embedding", (P, P, P, 1 << 20, 1 << 12, 2, 3, 1.0, 0, None), nat.ERR_SHAPE, "too large"),
    ("ipc_embedding", (P, P, P, 10, 1 << 10, 1 << 11, 1 << 11, 1.0, 0, None), nat.ERR_SHAPE, "too large"),
    ("ipc_embedding", (P, P, P, 10, 4, 2, 3, 1.0, 3, None), nat.ERR_DTYPE, "dtype"),
    ("ipc_embedding_update", (P, P, None, 10, 4, 2, 3, 1.0, 0, None, 0, None), nat.ERR_NULL, "g"),
    ("ipc_embedding_update", (P, P, P, 10, 4, 2, 300, 1.0, 0, None, 0, None), nat.ERR_NULL, "workspace"),
    ("ipc_embedding_update", (P, P, P, 10, 4, 2, 300, 1.0, 0, P, 100, None), nat.ERR_SHAPE, "workspace of 100"),
    ("ipc_embedding_update", (P, P, P, 10, 4, 2, 300, 1.0, 0, P + 8, BIG, None), nat.ERR_ALIGN, "workspace"),
    ("ipc_embedding_update", (P, P, P, 10, 4, 2, 300, 1.0, 0, P, -1, None), nat.ERR_SHAPE, "workspace"),
    ("ipc_dropout", (P, None, P, 4, 4, 100, 0, 0, None), nat.ERR_NULL, "rng"),
    ("ipc_dropout", (P, P, P, 4, 4, 65536, 0, 0, None), nat.ERR_CONFIG, "dropped"),
    ("ipc_dropout", (P, P, P, 4, 4, -1, 0, 0, None), nat.ERR_CONFIG, "dropped"),
    ("ipc_dropout", (P, P, P, 1 << 16, 1 << 16, 1, 0, 0, None), nat.ERR_SHAPE, "too large"),
    ("ipc_token_loss", (P, P, None, P, 10, 4, 3, 0, 0, P, BIG, None), nat.ERR_NULL, "targets"),
    ("ipc_token_loss", (P, P, P, P, 10, 4, 3, 0, 9, P, BIG, None), nat.ERR_ACT, "activation"),
    ("ipc_token_loss", (P, P, P, P, 10, 4, 3, 0, 0, None, 0, None), nat.ERR_NULL, "workspace"),
    ("ipc_token_loss", (P, P, P, P, 10, 4, 3, 0, 0, P, 16, None), nat.ERR_SHAPE, "workspace of 16"),
    ("ipc_token_loss", (P, P + 2, P, P, 10, 4, 3, 2, 0, P, BIG, None), nat.ERR_ALIGN, "4-byte"),
    ("ipc_token_loss", (P, P, P, P, 1, 40000, 40000, 2, 0, P, BIG, None), nat.ERR_SHAPE, "too large"),
    ("ipc_token_update", (P, P, P, P, None, 10, 4, 3, 1.0, 0, 0, P, BIG, None), nat.ERR_NULL, "g"),
    ("ipc_token_update", (P, P, P, P, P, 10, 0, 3, 1.0, 0, 0, P, BIG, None), nat.ERR_SHAPE, "dimensions"),
    ("ipc_token_update", (P, P, P, P, P, 10, 4, 3, 1.0, 0, 0, P, 16, None), nat.ERR_SHAPE, "workspace of 16"),
])
def test_entry_points_refuse(entry, args, code, needle):
    assert getattr(nat.lib(), entry)(*args) == code
    assert needle in nat.last_error()


def test_workspaces():
    lib = nat.lib()
    assert lib.ipc_embedding_update_workspace_bytes(10, 4, 2, 256, 0) == 0
    n = lib.ipc_embedding_update_workspace_bytes(10, 4, 2, 300, 0)
    assert n >= 600 * (4 + 4 + 16)
    assert lib.ipc_embedding_update_workspace_bytes(10, 4, 2, 300, 5) == 0
    loss, update = lib.ipc_token_loss_workspace_bytes, lib.ipc_token_update_workspace_bytes
    for storage in (0, 1, 2):
        assert 0 < loss(1000, 64, 32, storage, 2) < update(1000, 64, 32, storage, 2)
    for bad in ((0, 64, 32, 0, 0), (10, 64, 32, 3, 0), (10, 64, 32, 0, 6), (10, 1 << 16, 1 << 16, 0, 0)):
        assert loss(*bad) == update(*bad) == 0
    # pieces bound what a large vocabulary takes
    assert update(1 << 20, 64, 4096, 2, 0) < 3 << 30


@pytest.mark.parametrize("storage", [0, 1, 2])
@pytest.mark.parametrize("V,D,B", [(300001, 2001, 1), (14001, 40001, 1), (30000, 40000, 1), (700001, 2000, 1), (1 << 20, 2047, 1), (1, 1, 1 << 22), (2, 8, 1 << 21), (1, 60, 8000000)])
def test_calls_of_few_products_over_large_tensors_are_taken(V, D, B, storage):
    """A vocabulary whose weights take more than a piece, and states that do not fit in three terms."""
    lib = nat.lib()
    fits = storage != 0 or D * B < 1 << 28
    assert (lib.ipc_token_update_workspace_bytes(V, D, B, storage, 2) > 0) == fits
    assert (lib.ipc_token_loss_workspace_bytes(V, D, B, storage, 2) > 0) == fits


def test_builders_refuse():
    for bad in (dict(p=1.0), dict(p=-0.1), dict(p=1 - 2.0 ** -18), dict(p=float("nan")), dict(site=-1), dict(site=2 ** 31)):
        with pytest.raises(ValueError):
            tokens.build_dropout(4, 4, "float32", **{"p": 0.5, **bad})
    for build, sizes in ((tokens.build_embedding, (5, 0, 1, 1)), (tokens.build_embedding_update, (5, 1, 0, 1)),
                         (tokens.build_token_loss, (0, 3, 1)), (tokens.build_token_update, (5, 3, -1)), (tokens.build_dropout, (0, 3))):
        with pytest.raises(ValueError, match="invalid shape"):
            build(*sizes)
    with pytest.raises(ValueError, match="activation"):
        tokens.build_token_loss(4, 4, 4, "swish")
    with pytest.raises(ValueError, match="dtype"):
        tokens.build_embedding(4, 4, 1, 4, "float64")


def test_tensors_that_do_not_fit_are_refused():
    x, w, t, loss = torch.zeros(4, 3), torch.zeros(10, 4), torch.zeros(3, dtype=torch.int64), torch.zeros(3)
    k = tokens.build_token_loss(10, 4, 3)
    with pytest.raises(ValueError, match="X must be a device tensor"):
        k(x, w, t, loss)
    from torch._subclasses import FakeTensorMode

    def on(device, *shape, dtype=torch.float32):
        with FakeTensorMode():
            return torch.empty(shape, dtype=dtype, device=device)

    good = [on("cuda:0", 4, 3), on("cuda:0", 10, 4), on("cuda:0", 3, dtype=torch.int64), on("cuda:0", 3)]
    for at, other, why in ((0, on("cuda:0", 4, 4), "shape"), (1, on("cuda:0", 10, 4, dtype=torch.float16), "dtype"),
                           (2, on("cuda:0", 3, dtype=torch.int32), "TARGETS has dtype"), (3, on("cuda:1", 3), "different devices"),
                           (0, on("cuda:0", 3, 4).t(), "contiguous")):
        with pytest.raises(ValueError, match=why):
            k(*good[:at], other, *good[at + 1:])
    with pytest.raises(ValueError, match="different devices"):
        k(*good, workspace=on("cuda:1", k.workspace_bytes, dtype=torch.uint8))


def test_the_generator_gives_its_published_words():
    """Philox 4x32-10's known answers (the published test vectors of its authors)."""
    assert O.philox((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    f = 0xFFFFFFFF
    assert O.philox((f, f, f, f), (f, f)) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert O.philox((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0)) == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def test_token_data(tmp_path):
    d = TokenDataset(np.arange(10), 10)
    got = list(d.batches(4, 3, shuffle=False))
    assert len(got) == 3 and all(ids.shape == (3, 4) and t.shape == (4,) for ids, t in got)
    assert got[0][0][:, 0].tolist() == [-1, -1, -1] and got[0][0][:, 2].tolist() == [-1, 0, 1]
    assert got[1][0][:, 1].tolist() == [2, 3, 4] and int(got[1][1][1]) == 5
    assert got[2][1].tolist() == [8, 9, -1, -1] and got[2][0][:, 2].tolist() == [-1, -1, -1]
    seen = torch.cat([t for _, t in d.batches(4, 3, seed=1)])
    assert sorted(seen.tolist()) == [-1, -1] + list(range(10))
    path = tmp_path / "t.txt"
    path.write_text("b a b c b a")
    assert load_tokens(path).tokens.tolist() == [ord(c) for c in "b a b c b a"]
    words = load_tokens(path, words=2)
    assert words.tokens.tolist() == [0, 1, 0, -1, 0, 1] and words.vocab == 2 and words.names == ["b", "a"]
    s = synthetic_tokens(500, vocab=30, seed=2)
    assert len(s) == 500 and 0 <= s.tokens.min() and s.tokens.max() < 30
    assert np.array_equal(s.tokens, synthetic_tokens(500, vocab=30, seed=2).tokens)


def test_net_and_command_refuse(capsys):
    with pytest.raises(ValueError, match="weights"):
        TokenNet(10, 2, 4, (6,), 8, weights=[torch.zeros(10, 6), torch.zeros(6, 7)], device="cpu")
    with pytest.raises(ValueError, match="table"):
        TokenNet(10, 2, 4, (6,), 8, weights=[torch.zeros(10, 6), torch.zeros(6, 8)], table=torch.zeros(9, 4), device="cpu")
    for argv in (["tokens"], ["tokens", "--synthetic", "10", "--text", "x"]):
        with pytest.raises(SystemExit):
            cli.main(argv)
    assert "either --text" in capsys.readouterr().err
