"""Operators of nets over tokens (HIP, gfx950).

The input of such a net is a context of C tokens, each a row of a learnt table,
the output one of V words under a softmax.  States are ``[features, batch]`` and
weights ``[out, in]``, as in ``lich_amd.kernels``; ids and targets are int64.  An
id or target outside 0 .. V - 1 marks a padded place, whatever stands in its
column of a state.

* ``build_embedding``, ``build_embedding_update``: the input state from the
  table, and the table's update by the input state's error direction, its places
  sorted by id.
* ``build_dropout``: a mask from a counter-based generator, never stored; the
  same call on an error is the backward pass.
* ``build_token_loss``, ``build_token_update``: softmax cross entropy of the
  output layer over the vocabulary in pieces, whose logits are kept for a few
  samples at most; the update also gives the state's error direction and changes
  the weights.

Each builder returns a callable that validates its tensors and enqueues on
torch's current stream, as in ``lich_amd.kernels``; nothing is allocated or
synchronised inside a call.  Directions point downhill, as the errors ``target -
prediction`` of the rest of the package: an update adds them.  The reference has no
counterpart.
"""
from __future__ import annotations

from functools import lru_cache

import torch

from . import _native as nat
from .kernels import _Kernel
from .microscale import _MXKernel, _sizes


class _TokenKernel(_MXKernel):
    workspace_bytes = 0

    new_workspace = _Kernel.new_workspace


class EmbeddingKernel(_TokenKernel):
    """``k(IDS[C, B], TABLE[V, D], X[C * D, B])``: ``X[c * D + d, b] = scale * TABLE[IDS[c, b], d]``,
    zeros in padded places."""

    def __init__(self, V, D, C, B, dtype, scale):
        super().__init__(dtype)
        _sizes(V=V, D=D, C=C, B=B)
        self.V, self.D, self.C, self.B, self.scale = int(V), int(D), int(C), int(B), float(scale)
        self._bind("ipc_embedding", (("IDS", (self.C, self.B), torch.int64), ("TABLE", (self.V, self.D), self.dtype),
                                     ("X", (self.C * self.D, self.B), self.dtype)),
                   self.V, self.D, self.C, self.B, self.scale, self.storage)

    def __call__(self, ids, table, x):
        rc = self._run(ids, table, x)
        if rc:
            self._checked(rc, ids, table, x)


class EmbeddingUpdateKernel(_TokenKernel):
    """``k(TABLE[V, D], IDS[C, B], G[C * D, B], *, workspace)``: ``TABLE[v] += alpha * sum of G's
    columns at the places of v``, the sum in fp32 in a fixed order, one rounding.
    ``workspace`` (caller-owned, ``new_workspace()``) is needed where
    ``workspace_bytes`` is not 0."""

    def __init__(self, V, D, C, B, dtype, alpha):
        super().__init__(dtype)
        _sizes(V=V, D=D, C=C, B=B)
        self.V, self.D, self.C, self.B, self.alpha = int(V), int(D), int(C), int(B), float(alpha)
        self._bind("ipc_embedding_update", (("TABLE", (self.V, self.D), self.dtype), ("IDS", (self.C, self.B), torch.int64),
                                            ("G", (self.C * self.D, self.B), self.dtype)),
                   self.V, self.D, self.C, self.B, self.alpha, self.storage, workspace=True)
        self.workspace_bytes = int(nat.lib().ipc_embedding_update_workspace_bytes(self.V, self.D, self.C, self.B, self.storage))

    def __call__(self, table, ids, g, *, workspace=None):
        rc = self._run(table, ids, g, workspace)
        if rc:
            self._checked(rc, table, ids, g, workspace=workspace)


class DropoutKernel(_TokenKernel):
    """``k(X[M, B], RNG[2], OUT[M, B])``: ``OUT = m X / (1 - p)`` (OUT may be X).  RNG holds seed
    and step (int64) on the device, read when the call runs: a captured call draws anew
    once they change.  ``site`` tells the calls of one step apart.  p counts in
    65536ths; dropped values are 0 whatever they were."""

    def __init__(self, M, B, dtype, p, site):
        super().__init__(dtype)
        _sizes(M=M, B=B)
        self.M, self.B, self.p, self.site = int(M), int(B), float(p), int(site)
        if not 0.0 <= self.p < 1.0 or round(self.p * 65536) > 65535:
            raise ValueError(f"p must be in [0, 1), at most 65535 / 65536 (got {p})")
        if not 0 <= self.site < 2 ** 31:
            raise ValueError(f"site must be in [0, 2^31) (got {site})")
        self._bind("ipc_dropout", (("X", (self.M, self.B), self.dtype), ("RNG", (2,), torch.int64),
                                   ("OUT", (self.M, self.B), self.dtype)),
                   self.M, self.B, round(self.p * 65536), self.site, self.storage)

    def __call__(self, x, rng, out):
        rc = self._run(x, rng, out)
        if rc:
            self._checked(rc, x, rng, out)


class TokenLossKernel(_TokenKernel):
    """``k(X[D, B], W[V, D], TARGETS[B], LOSS[B], *, workspace)``: ``LOSS[b] = -log softmax(W f(X))``
    of column b at its target, in float32; 0 for a padded one.  ``workspace``
    (caller-owned, ``new_workspace()``) is needed."""

    def __init__(self, V, D, B, activation, dtype):
        super().__init__(dtype, activation)
        _sizes(V=V, D=D, B=B)
        self.V, self.D, self.B = int(V), int(D), int(B)
        self._bind("ipc_token_loss", (("X", (self.D, self.B), self.dtype), ("W", (self.V, self.D), self.dtype),
                                      ("TARGETS", (self.B,), torch.int64), ("LOSS", (self.B,), torch.float32)),
                   self.V, self.D, self.B, self.storage, self.act, workspace=True)
        self.workspace_bytes = int(nat.lib().ipc_token_loss_workspace_bytes(self.V, self.D, self.B, self.storage, self.act))

    def __call__(self, x, w, targets, loss, *, workspace=None):
        rc = self._run(x, w, targets, loss, workspace)
        if rc:
            self._checked(rc, x, w, targets, loss, workspace=workspace)


class TokenUpdateKernel(_TokenKernel):
    """``k(X[D, B], W[V, D], TARGETS[B], LOSS[B], G[D, B], *, workspace)``: the loss; with ``e = onehot
    - softmax(W f(X))`` also ``G = f'(X) * (W.T @ e)`` by the W from before and ``W += alpha *
    e @ f(X).T``.  Padded columns: loss 0, zeros in G, no share of W.  ``workspace``
    (caller-owned, ``new_workspace()``) is needed."""

    def __init__(self, V, D, B, activation, dtype, alpha):
        super().__init__(dtype, activation)
        _sizes(V=V, D=D, B=B)
        self.V, self.D, self.B, self.alpha = int(V), int(D), int(B), float(alpha)
        state = (self.D, self.B), self.dtype
        self._bind("ipc_token_update", (("X", *state), ("W", (self.V, self.D), self.dtype), ("TARGETS", (self.B,), torch.int64),
                                        ("LOSS", (self.B,), torch.float32), ("G", *state)),
                   self.V, self.D, self.B, self.alpha, self.storage, self.act, workspace=True)
        self.workspace_bytes = int(nat.lib().ipc_token_update_workspace_bytes(self.V, self.D, self.B, self.storage, self.act))

    def __call__(self, x, w, targets, loss, g, *, workspace=None):
        rc = self._run(x, w, targets, loss, g, workspace)
        if rc:
            self._checked(rc, x, w, targets, loss, g, workspace=workspace)


@lru_cache(maxsize=256)
def build_embedding(V: int, D: int, C: int, B: int, dtype="float32", scale: float = 1.0):
    """``X[c * D + d, b] = scale * TABLE[IDS[c, b], d]``."""
    return EmbeddingKernel(V, D, C, B, dtype, scale)


@lru_cache(maxsize=256)
def build_embedding_update(V: int, D: int, C: int, B: int, dtype="float32", alpha: float = 1e-4):
    """``TABLE[v] += alpha *`` the sum of G's columns at the places of v (alpha: the step
    times the lookup's scale)."""
    return EmbeddingUpdateKernel(V, D, C, B, dtype, alpha)


@lru_cache(maxsize=256)
def build_dropout(M: int, B: int, dtype="float32", p: float = 0.1, *, site: int = 0):
    """``OUT = m X / (1 - p)`` with a mask that is never stored."""
    return DropoutKernel(M, B, dtype, p, site)


@lru_cache(maxsize=256)
def build_token_loss(V: int, D: int, B: int, activation: str = "identity", dtype="float32"):
    """``LOSS = -log softmax(W f(X))`` at the targets."""
    return TokenLossKernel(V, D, B, activation, dtype)


@lru_cache(maxsize=256)
def build_token_update(V: int, D: int, B: int, activation: str = "identity", dtype="float32", alpha: float = 1e-4):
    """The loss, ``G = f'(X) * (W.T @ e)`` and ``W += alpha * e @ f(X).T``, ``e = onehot - softmax``."""
    return TokenUpdateKernel(V, D, B, activation, dtype, alpha)
