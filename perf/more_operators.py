"""The calls of the token operators (``lich_amd.tokens``) by which their speed is judged.

Nets whose input and target are tokens: the input state is a context of rows of
a learnt table, the target one of V words under a softmax.  States are
``[features, batch]`` and weights ``[out, in]``, as everywhere in the package.

Five calls, each in its plain form (elementary torch operations in 32 bits) and,
with ``own`` set, through the package's entry points:

* ``embed``         X = scale * TABLE[ids], the rows of a context under each other;
* ``embed_update``  TABLE[v] += alpha * scale * sum of G over the places of v;
* ``dropout``       OUT = m X / (1 - p), m from a counter-based generator; on an
                    error, with the same counters, its backward pass;
* ``loss``          -log softmax(W f(X)) at the target, a column each;
* ``update``        that loss, e = onehot - softmax(W f(X)), W += alpha e f(X)^T
                    and G = f'(X) W^T e with the W from before.

An id or target outside 0 .. V - 1 marks a padded place: zeros in X, nothing in
TABLE, loss 0, no share of W and zeros in G.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
ACTIVATIONS = ("identity", "relu", "tanh", "sigmoid", "silu", "gelu")
SITE = 3  # a layer's number: its part of the dropout counter
PADDED = 0.03


# ------------------------------------------------------------------ the cases
def _embed(name, kind, V, D, C, B, storage):
    return {"name": name, "kind": kind, "vocab": V, "width": D, "context": C, "batch": B, "storage": storage}


def _dropout(name, M, B, storage, p):
    return {"name": name, "kind": "dropout", "M": M, "batch": B, "storage": storage, "p": p}


def _softmax(name, kind, V, D, B, storage, activation):
    return {"name": name, "kind": kind, "vocab": V, "width": D, "batch": B, "storage": storage, "activation": activation}


def listed():
    return [
        # The context of one sample, answered online: latency.
        _embed("embed_one", "embed", 10007, 64, 8, 1, "fp32"),
        # The input state of the wide net (4096 rows, batch 1024) from contexts of eight words.
        _embed("embed_context", "embed", 32000, 512, 8, 1024, "bf16"),
        # What that batch teaches the table; the commonest words come hundreds of times.
        _embed("embed_update_context", "embed_update", 32000, 512, 8, 1024, "bf16"),
        # A small vocabulary at odd sizes, everything in fp32.
        _embed("embed_update_ragged", "embed_update", 1531, 131, 5, 301, "fp32"),
        # A hidden state of a large net.
        _dropout("dropout_wide", 4096, 4096, "bf16", 0.1),
        # Odd sizes in fp32.
        _dropout("dropout_ragged", 1531, 301, "fp32", 0.5),
        # One sample scored under a large vocabulary: bound by the weights' bytes.
        _softmax("loss_one", "loss", 32000, 4096, 1, "bf16", "tanh"),
        # A validation batch scored.
        _softmax("loss_batch", "loss", 32000, 1024, 1024, "fp16", "gelu"),
        # The output layer of the image nets as a softmax: launches and latency.
        _softmax("update_classes", "update", 10, 64, 128, "fp32", "tanh"),
        # A ragged batch in fp32.
        _softmax("update_ragged", "update", 10007, 515, 77, "fp32", "silu"),
        # The output layer of the wide net over words, a training batch.
        _softmax("update_words", "update", 32000, 4096, 1024, "bf16", "relu"),
        # A vocabulary whose logits would take half a gigabyte.  The largest work there is.
        _softmax("update_large", "update", 128000, 2048, 2048, "fp16", "tanh"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    limit = work(listed()[-1])["flops"]
    while True:
        kind = rng.choice(("embed", "embed_update", "embed_update", "dropout", "loss", "update", "update", "update"))
        storage = rng.choice(("fp32", "fp16", "bf16", "bf16"))
        even = rng.random() < 0.5  # half of the sizes are as even as real nets are

        def size(lo, hi):
            v = _log_int(rng, lo, hi)
            return max(lo, v // 64 * 64) if even else v

        if kind in ("embed", "embed_update"):
            case = _embed("", kind, size(16, 200000), size(1, 2048), rng.randint(1, 16), size(1, 4096), storage)
            if case["width"] * case["context"] * case["batch"] > 1 << 26:
                continue
        elif kind == "dropout":
            case = _dropout("", size(1, 8192), size(1, 8192), storage, rng.choice((0.0, 0.1, 0.25, 0.5, 0.9)))
        else:
            case = _softmax("", kind, size(2, 131072), size(1, 8192), size(1, 4096), storage, rng.choice(ACTIVATIONS))
            if work(case)["flops"] > limit / 2 or case["vocab"] * case["width"] > 1 << 28:
                continue
        del case["name"]
        return case


# ------------------------------------------------------------------ inputs
def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    dt, B = DTYPES[case["storage"]], case["batch"]

    def normal(rows, cols, size=1.0):
        return (torch.randn((rows, cols), generator=g, device="cuda") * size).to(dt)

    def words(V, *shape):  # frequencies near 1 / rank, as words have; a few padded places
        u = torch.rand(shape, generator=g, device="cuda", dtype=torch.float64)
        rank = torch.floor(torch.exp(u * math.log(V + 1.0))).long() - 1
        ids = (rank.clamp(0, V - 1) * 7919) % V if math.gcd(7919, V) == 1 else rank.clamp(0, V - 1)
        return torch.where(torch.rand(shape, generator=g, device="cuda") < PADDED, -1, ids)

    if case["kind"] == "dropout":
        rng = torch.randint(0, 2 ** 62, (2,), generator=g, device="cuda")
        return {"x": normal(case["M"], B), "rng": rng}
    V, D = case["vocab"], case["width"]
    if case["kind"] in ("embed", "embed_update"):
        s = {"table": normal(V, D, 0.1), "ids": words(V, case["context"], B)}
        if case["kind"] == "embed_update":  # errors a tenth of the states
            s["g"] = normal(case["context"] * D, B, 0.1)
        return s
    # trained weights: logits of a standard deviation of about three
    return {"x": normal(D, B), "w": normal(V, D, 3.0 / math.sqrt(D)), "targets": words(V, B)}


def _scale(case):
    return math.sqrt(case["width"])


def _alpha(case):
    return 0.5 / case["batch"] if case["kind"] == "update" else 0.1


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["kind"] == "embed":
        s["out"] = torch.empty((case["context"] * case["width"], case["batch"]), dtype=DTYPES[case["storage"]], device="cuda")
    elif case["kind"] == "dropout":
        s["out"] = torch.empty_like(s["x"])
    elif case["kind"] in ("loss", "update"):
        s["loss"] = torch.empty((case["batch"],), dtype=torch.float32, device="cuda")
        if case["kind"] == "update":
            s["grad"] = torch.empty_like(s["x"])
    return s


# ------------------------------------------------------------------ plain forms
def _f(name, x):
    if name == "relu":
        return torch.clamp(x, min=0)
    if name == "tanh":
        return torch.tanh(x)
    if name == "sigmoid":
        return torch.sigmoid(x)
    if name == "silu":
        return x * torch.sigmoid(x)
    if name == "gelu":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))
    return x


def _df(name, x):
    if name == "relu":
        return (x > 0).to(x.dtype)
    if name == "tanh":
        return 1 - torch.tanh(x) ** 2
    if name == "sigmoid":
        s = torch.sigmoid(x)
        return s * (1 - s)
    if name == "silu":
        s = torch.sigmoid(x)
        return s * (1 + x * (1 - s))
    if name == "gelu":
        k = math.sqrt(2 / math.pi)
        t = torch.tanh(k * (x + 0.044715 * x ** 3))
        return 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * k * (1 + 3 * 0.044715 * x * x)
    return torch.ones_like(x)


LOW = 0xFFFFFFFF


def _random_words(rng, blocks):
    """The four 32-bit words of the counters (block, SITE, step) under the key `seed`:
    the generator Philox 4x32-10 of Salmon, Moraes, Dror and Shaw (2011), in 64-bit whole numbers."""
    def product(a, m):  # high and low halves of a * m, both below 2^32
        low, high = a * (m & 0xFFFF), a * (m >> 16)
        t = (low >> 16) + high
        return (t >> 16) & LOW, ((t & 0xFFFF) << 16) | (low & 0xFFFF)

    c0 = torch.arange(blocks, device=rng.device)
    c1, c2, c3 = torch.full_like(c0, SITE), (rng[1] & LOW).expand_as(c0), ((rng[1] >> 32) & LOW).expand_as(c0)
    k0, k1 = rng[0] & LOW, (rng[0] >> 32) & LOW
    for _ in range(10):
        h0, l0 = product(c0, 0xD2511F53)
        h1, l1 = product(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & LOW, (k1 + 0xBB67AE85) & LOW
    return torch.stack([c0, c1, c2, c3], -1)


def _run_plain(s):
    case = s["case"]
    if case["kind"] == "dropout":
        x, below = s["x"].float(), round(case["p"] * 65536)
        words = _random_words(s["rng"], (x.numel() + 7) // 8)
        draws = torch.stack([words & 0xFFFF, words >> 16], -1).reshape(-1)[:x.numel()].reshape(x.shape)
        s["out"].copy_(torch.where(draws >= below, x * (65536 / (65536 - below)), 0))
        return s["out"]
    V, D = case["vocab"], case["width"]
    if case["kind"] in ("embed", "embed_update"):
        ids, C, B = s["ids"], case["context"], case["batch"]
        real = (ids >= 0) & (ids < V)
        if case["kind"] == "embed":
            rows = s["table"][ids.clamp(0, V - 1)].float() * _scale(case) * real[..., None]
            s["out"].copy_(rows.transpose(1, 2).reshape(C * D, B))
            return s["out"]
        g = s["g"].reshape(C, D, B).transpose(1, 2)[real].float()
        total = torch.zeros((V, D), device=g.device).index_add_(0, ids[real], g)
        s["table"].copy_(s["table"].float() + (_alpha(case) * _scale(case)) * total)
        return s["table"]
    x, w, t = s["x"].float(), s["w"].float(), s["targets"]
    real = (t >= 0) & (t < V)
    f = _f(case["activation"], x)
    z = w @ f
    top = z.amax(0)
    u = torch.exp(z - top)
    total = u.sum(0)
    at = t.clamp(0, V - 1)[None]
    s["loss"].copy_(torch.where(real, torch.log(total) + top - z.gather(0, at)[0], 0))
    if case["kind"] == "loss":
        return s["loss"]
    e = u.mul_(-1 / total)
    e.scatter_add_(0, at, torch.ones_like(at, dtype=e.dtype))
    e.mul_(real)
    s["grad"].copy_(_df(case["activation"], x) * (w.T @ e))
    s["w"].copy_(w + _alpha(case) * (e @ f.T))
    return {"loss": s["loss"], "grad": s["grad"], "w": s["w"]}


# ------------------------------------------------------------------ the package's calls
def _run_own(s):
    from lich_amd import tokens

    case, dt, B = s["case"], DTYPES[s["case"]["storage"]], s["case"]["batch"]
    if case["kind"] == "dropout":
        tokens.build_dropout(case["M"], B, dt, case["p"], site=SITE)(s["x"], s["rng"], s["out"])
        return s["out"]
    V, D = case["vocab"], case["width"]
    if case["kind"] == "embed":
        tokens.build_embedding(V, D, case["context"], B, dt, _scale(case))(s["ids"], s["table"], s["out"])
        return s["out"]
    if case["kind"] == "embed_update":
        k = tokens.build_embedding_update(V, D, case["context"], B, dt, _alpha(case) * _scale(case))
        k(s["table"], s["ids"], s["g"], workspace=k.new_workspace(s["g"].device))
        return s["table"]
    if case["kind"] == "loss":
        k = tokens.build_token_loss(V, D, B, case["activation"], dt)
        k(s["x"], s["w"], s["targets"], s["loss"], workspace=k.new_workspace(s["x"].device))
        return s["loss"]
    k = tokens.build_token_update(V, D, B, case["activation"], dt, _alpha(case))
    k(s["x"], s["w"], s["targets"], s["loss"], s["grad"], workspace=k.new_workspace(s["x"].device))
    return {"loss": s["loss"], "grad": s["grad"], "w": s["w"]}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------ what they cost
def _distinct(V, n):
    """How many different words n places hold, on average."""
    edges = np.log(np.arange(1, V + 2)) / math.log(V + 1.0)
    return float((1 - (1 - np.diff(edges)) ** n).sum())


def work(case):
    size = 4 if case["storage"] == "fp32" else 2
    if case["kind"] == "dropout":
        return {"bytes": 2 * size * case["M"] * case["batch"], "flops": 0}
    V, D, B = case["vocab"], case["width"], case["batch"]
    if case["kind"] in ("embed", "embed_update"):
        n = case["context"] * B
        rows = _distinct(V, n * (1 - PADDED))
        if case["kind"] == "embed":
            return {"bytes": size * D * (rows + n) + 8 * n, "flops": n * D}
        return {"bytes": size * D * (2 * rows + n) + 8 * n, "flops": n * D}
    if case["kind"] == "loss":
        return {"bytes": size * (V * D + D * B) + 12 * B, "flops": 2.0 * V * D * B}
    return {"bytes": size * (2 * V * D + 2 * D * B) + 12 * B, "flops": 6.0 * V * D * B}


# ------------------------------------------------------------------ the same in 64 bits
def _mask(seed, step, count, p):
    """Which of `count` values are kept, by the generator's definition on 64-bit words."""
    u64 = np.uint64
    word = np.arange((count + 7) // 8, dtype=u64)
    c = [word, np.full_like(word, SITE), np.full_like(word, step & LOW), np.full_like(word, step >> 32)]
    key = [seed & LOW, seed >> 32]
    for _ in range(10):
        a, b = c[0] * u64(0xD2511F53), c[2] * u64(0xCD9E8D57)  # whole in 64 bits
        c = [(b >> u64(32)) ^ c[1] ^ u64(key[0]), b & u64(LOW), (a >> u64(32)) ^ c[3] ^ u64(key[1]), a & u64(LOW)]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    halves = np.empty((len(word), 8), dtype=np.int64)
    for j in range(4):
        halves[:, 2 * j], halves[:, 2 * j + 1] = c[j] & u64(0xFFFF), c[j] >> u64(16)
    return halves.reshape(-1)[:count] >= round(p * 65536)


def exact(case, seed):
    v = _inputs(case, seed)
    if case["kind"] == "dropout":
        kept = _mask(int(v["rng"][0]), int(v["rng"][1]), v["x"].numel(), case["p"])
        share = 1 - round(case["p"] * 65536) / 65536
        return v["x"].double() / share * torch.from_numpy(kept).to(v["x"].device).reshape(v["x"].shape)
    V, D, B = case["vocab"], case["width"], case["batch"]
    if case["kind"] in ("embed", "embed_update"):
        ids, C = v["ids"], case["context"]
        padded = torch.cat([v["table"].double(), torch.zeros((1, D), dtype=torch.float64, device="cuda")])
        place = torch.where((ids < 0) | (ids >= V), V, ids)  # the row of zeros
        if case["kind"] == "embed":
            return torch.cat([padded[place[c]].T * math.sqrt(D) for c in range(C)])
        for c in range(C):
            padded.index_add_(0, place[c], 0.1 * math.sqrt(D) * v["g"][c * D:(c + 1) * D].double().T.contiguous())
        return padded[:V].contiguous()
    x, w, t = v["x"].double(), v["w"].double(), v["targets"]
    f = _f(case["activation"], x)
    z = torch.mm(w, f)
    logs = z - torch.logsumexp(z, 0, keepdim=True)
    del z
    hot = torch.arange(V, device="cuda")[:, None] == t[None]  # a padded column has none
    real = hot.any(0)
    loss = -(logs * hot).sum(0)
    if case["kind"] == "loss":
        return loss
    e = (hot.double() - logs.exp_()) * real
    return {"loss": loss, "grad": _df(case["activation"], x) * torch.mm(w.T.contiguous(), e),
            "w": w + 0.5 / B * torch.mm(e, f.T.contiguous())}
