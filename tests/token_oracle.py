"""The operators over tokens by their definitions, in 64 bits (test infrastructure)."""
import math

import numpy as np
import torch

F64 = torch.float64


def act(name, x):
    if name == "relu":
        return torch.where(x > 0, x, torch.zeros_like(x))
    if name == "tanh":
        return torch.tanh(x)
    if name == "sigmoid":
        return 1 / (1 + torch.exp(-x))
    if name == "silu":
        return x / (1 + torch.exp(-x))
    if name == "gelu":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))
    return x.clone()


def dact(name, x):
    if name == "relu":
        return (x > 0).to(x.dtype)
    if name == "tanh":
        return 1 - torch.tanh(x) ** 2
    if name == "sigmoid":
        s = 1 / (1 + torch.exp(-x))
        return s * (1 - s)
    if name == "silu":
        s = 1 / (1 + torch.exp(-x))
        return s + x * s * (1 - s)
    if name == "gelu":
        k = math.sqrt(2 / math.pi)
        t = torch.tanh(k * (x + 0.044715 * x ** 3))
        return 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * k * (1 + 3 * 0.044715 * x * x)
    return torch.ones_like(x)


def embedding(ids, table, scale):
    (C, B), (V, D) = ids.shape, table.shape
    out = torch.zeros((C * D, B), dtype=F64)
    for c in range(C):
        for b in range(B):
            if 0 <= int(ids[c, b]) < V:
                out[c * D:(c + 1) * D, b] = scale * table[int(ids[c, b])].to(F64)
    return out


def embedding_sums(ids, g, V):
    """Sums of G's columns by id, sums of their magnitudes, places of each id."""
    C, B = ids.shape
    D = g.shape[0] // C
    total, size, many = torch.zeros((V, D), dtype=F64), torch.zeros((V, D), dtype=F64), torch.zeros(V, dtype=F64)
    g = g.to(F64).reshape(C, D, B).permute(0, 2, 1).reshape(C * B, D)
    ids = ids.reshape(-1)
    real = (ids >= 0) & (ids < V)
    total.index_add_(0, ids[real], g[real])
    size.index_add_(0, ids[real], g[real].abs())
    many.index_add_(0, ids[real], torch.ones(int(real.sum()), dtype=F64))
    return total, size, many


def philox(counter, key):
    """Philox 4x32-10 of one counter (four words) and key (two), in Python's whole numbers."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def kept(count, seed, step, site, dropped):
    out = np.zeros(count, dtype=bool)
    low = 0xFFFFFFFF
    for block in range((count + 7) // 8):
        words = philox((block, site, step & low, (step >> 32) & low), (seed & low, (seed >> 32) & low))
        for i in range(8):
            if block * 8 + i < count:
                out[block * 8 + i] = (words[i // 2] >> (16 * (i % 2))) & 0xFFFF >= dropped
    return torch.from_numpy(out)


def softmax(x, w, targets, name):
    """loss, e = onehot - softmax, G and the sum e f(X)^T, with what bounds need."""
    V = w.shape[0]
    real = (targets >= 0) & (targets < V)
    x = torch.where(real[None], x.to(F64), torch.zeros((), dtype=F64, device=x.device))
    w = w.to(F64)
    f = torch.where(real[None], act(name, x), torch.zeros((), dtype=F64, device=x.device))
    z = w @ f
    top = z.max(0).values
    u = torch.exp(z - top)
    total = u.sum(0)
    at = torch.where(real, targets, torch.zeros_like(targets))
    loss = torch.where(real, torch.log(total) + top - z.gather(0, at[None])[0], torch.zeros_like(total))
    p = u / total
    e = -p
    e.scatter_add_(0, at[None], torch.ones_like(at, dtype=F64)[None])
    e = e * real
    return {"loss": loss, "f": f, "p": p * real, "e": e, "g": dact(name, x) * (w.T @ e) * real, "dw": e @ f.T,
            "df": dact(name, x) * real, "size": w.abs() @ f.abs()}
