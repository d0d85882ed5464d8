"""Nets over tokens: the operators of ``lich_amd.tokens`` together.

``TokenNet`` predicts a token from the C before it: rows of a learnt table under
each other are the input state, a ``CompactNet`` (states kept in 8 bits, trained by
back-propagation) the layers, a softmax over the vocabulary the output, with
dropout on every state.  ``predict`` answers with 4-bit weights, ``losses`` scores
with the weights as they are.  The reference has no nets over tokens.
"""
from __future__ import annotations

import torch

from . import tokens
from .compact import CompactNet
from .kernels import build_forward


class TokenNet(CompactNet):
    """``vocab`` words, ``context`` of them before the one to predict, rows of ``width``
    features in the table, ``hidden`` widths from the output's side to the input's; ``p`` the
    share of dropped values, ``rate`` the step of the mean gradient over a batch.  A batch
    is ids ``[context, batch]`` and targets ``[batch]`` (int64); padded places hold -1."""

    def __init__(self, vocab: int, context: int, width: int, hidden=(), batch: int = 128, activation: str = "tanh",
                 dtype=torch.float32, rate: float = 0.1, p: float = 0.0, *, device=None, seed: int = 0, weights=None,
                 table=None):
        super().__init__((vocab, *hidden, context * width), batch, activation, dtype, rate, device=device, seed=seed,
                         weights=weights)
        self.context, self.width, self.scale = int(context), int(width), float(width) ** 0.5
        if table is None:
            g = torch.Generator().manual_seed(int(seed) + 1)
            table = torch.randn((vocab, width), generator=g) / self.scale
        if tuple(table.shape) != (vocab, width):
            raise ValueError(f"the table has shape {tuple(table.shape)}, the net expects {(vocab, width)}")
        self.table = table.to(self.device, dtype).contiguous()
        self.rng = torch.tensor([int(seed), 0], device=self.device)  # seed and step of the dropout masks
        d, B = self.dims, self.batch
        step = float(rate) / B
        self._learn = tokens.build_embedding_update(vocab, width, context, B, dtype, step * self.scale)
        self._output = tokens.build_token_update(vocab, d[1], B, activation, dtype, step)
        self._drop = [tokens.build_dropout(n, B, dtype, p, site=l) if p > 0 else None for l, n in enumerate(d)]
        most = max(self._learn.workspace_bytes, self._output.workspace_bytes,
                   0 if self._workspace is None else self._workspace.numel())
        self._workspace = torch.empty(most, dtype=torch.uint8, device=self.device)

    def _dropped(self, l: int, state: torch.Tensor) -> torch.Tensor:
        """State (or its error) of layer l under this step's mask, in place."""
        if self._drop[l] is not None:
            self._drop[l](state, self.rng, state)
        return state

    def embed(self, ids: torch.Tensor) -> torch.Tensor:
        """Input states ``[context * width, n]`` of ids ``[context, n]``."""
        n = int(ids.shape[1])
        x = self._state(self.dims[-1], n)
        tokens.build_embedding(self.dims[0], self.width, self.context, n, self.dtype, self.scale)(ids, self.table, x)
        return x

    def step(self, ids: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
        """One training step; returns the losses ``[batch]`` before it (0 for padded targets)."""
        L, d, B = len(self.w), self.dims, self.batch
        state = self._dropped(L, self.embed(ids))
        for l in range(L - 1, 0, -1):
            self._save[l](state, self.kept[l])
            out = self._state(d[l], B)
            self._forward[l](state, self.w[l], out)
            state = self._dropped(l, out)
        loss, e = torch.empty(B, device=self.device), self._state(d[1], B)
        self.w4 = None
        self._output(state, self.w[0], targets, loss, e, workspace=self._workspace)
        for l in range(1, L):
            e = self._dropped(l, e)
            below = self._state(d[l + 1], B)
            self._gradient[l](self.w[l], e, self.kept[l], below, workspace=self._workspace)  # before W[l] changes
            self._update[l](self.w[l], e, self.kept[l], workspace=self._workspace)
            e = below
        self._learn(self.table, ids, self._dropped(L, e), workspace=self._workspace)
        self.rng[1] += 1
        return loss

    def losses(self, ids: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
        """Losses ``[n]`` of ids ``[context, n]`` and targets ``[n]``, nothing dropped."""
        n, state = int(ids.shape[1]), self.embed(ids)
        for l in range(len(self.w) - 1, 0, -1):
            out = self._state(self.dims[l], n)
            build_forward(self.dims[l], self.dims[l + 1], n, self.activation, self.dtype)(state, self.w[l], out)
            state = out
        loss = torch.empty(n, device=self.device)
        k = tokens.build_token_loss(self.dims[0], self.dims[1], n, self.activation, self.dtype)
        k(state, self.w[0], targets, loss, workspace=k.new_workspace(self.device))
        return loss

    def predict(self, ids: torch.Tensor) -> torch.Tensor:
        """Logits ``[vocab, n]`` of ids ``[context, n]`` with the packed weights."""
        return super().predict(self.embed(ids))


def train(dataset, *, context=4, width=32, hidden=(64,), batch=128, epochs=4, rate=0.5, p=0.0, activation="tanh",
          dtype=torch.float32, seed=0, device=None, log=print):
    """Trains a ``TokenNet`` on a ``TokenDataset``; returns (records, net)."""
    device = torch.device("cuda", 0) if device is None else torch.device(device)
    net = TokenNet(dataset.vocab, context, width, hidden, batch, activation, dtype, rate, p, device=device, seed=seed)
    records = []
    for epoch in range(epochs):
        total, count = torch.zeros((), device=device, dtype=torch.float64), 0
        for ids, targets in dataset.batches(batch, context, seed=seed, epoch=epoch):
            total += net.step(ids.to(device), targets.to(device)).double().sum()
            count += int((targets >= 0).sum())
        records.append({"epoch": epoch + 1, "loss": float(total) / max(count, 1), "tokens": count})
        log(f"epoch={epoch + 1:03d} loss={records[-1]['loss']:.4f} tokens={count}")
    return records, net
