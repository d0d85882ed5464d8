"""Nets in microscaled storage: the operators of ``lich_amd.microscale`` together.

``CompactNet`` is the trainer's MLP, ``x[l] = W[l] f(x[l+1])`` with ``x[L]`` the
input, trained by back-propagation: the forward pass keeps every layer's state
in 8 bits, the backward pass reads it there, and two full-width states are
alive at any time.  ``pack`` lays its weights out in 4 bits, ``predict`` answers
with them: the states in 4 bits too for a batch, as they are for few samples.

``FourBitSteps`` takes iPC steps (the reference's ``reference.py:35-59``) whose
three products run on 4-bit operands, over full-width master states and weights.

The reference trains neither way; both share its layout (``[features, batch]``,
``W[l]: f(x[l+1]) -> x[l]``).
"""
from __future__ import annotations

import torch

from . import microscale as mx
from .kernels import build_forward
from .trainer import HipIPC, IPCConfig

FEW = 64  # samples that ``CompactNet.predict`` answers without quantising the states


def _weights(dims, seed, device, dtype):
    """The trainer's initial weights of these sizes."""
    model = HipIPC(IPCConfig(dims=tuple(dims), init="xavier_uniform"), device=device, seed=seed)
    return [w.to(dtype).contiguous() for w in model.w]


class CompactNet:
    """``dims`` = (classes, hidden ..., features), ``dtype`` the type of states and
    weights, ``rate`` the step of the mean gradient over a batch.  ``weights`` are the
    net's own from then on: where they have its type and device they are not copied,
    and ``step`` updates them in place."""

    def __init__(self, dims, batch: int, activation: str = "relu", dtype=torch.float32, rate: float = 0.01, *,
                 device=None, seed: int = 0, weights=None):
        self.dims, self.batch, self.activation, self.dtype = tuple(dims), int(batch), activation, dtype
        self.device = torch.device(device or "cuda")
        self.w = ([w.to(self.device, dtype).contiguous() for w in weights] if weights is not None
                  else _weights(self.dims, seed, self.device, dtype))
        L, d, B = len(self.w), self.dims, self.batch
        if L != len(d) - 1 or any(tuple(w.shape) != (d[l], d[l + 1]) for l, w in enumerate(self.w)):
            raise ValueError(f"weights do not match dims {d}")
        self._save = [mx.build_checkpoint_save(d[l + 1], B, dtype) for l in range(L)]
        self._forward = [build_forward(d[l], d[l + 1], B, activation, dtype) for l in range(L)]
        self._gradient = [mx.build_checkpoint_gradient(d[l + 1], d[l], B, activation, dtype) for l in range(L)]
        self._update = [mx.build_checkpoint_weight_update(d[l], d[l + 1], B, activation, dtype, float(rate) / B)
                        for l in range(L)]
        self.kept = [k.new_output(self.device) for k in self._save]  # x[l + 1] of layer l
        most = max((k.workspace_bytes for k in self._update + self._gradient), default=0)
        self._workspace = torch.empty(most, dtype=torch.uint8, device=self.device) if most else None
        self.w4 = None

    def _state(self, rows: int, columns: int) -> torch.Tensor:
        return torch.empty((rows, columns), dtype=self.dtype, device=self.device)

    def step(self, x: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
        """One training step on ``x [features, batch]`` and targets ``y [classes,
        batch]``; returns the error ``y - x[0]`` before it.  The packed weights are
        laid out anew by the next ``predict``."""
        if tuple(y.shape) != (self.dims[0], self.batch):
            raise ValueError(f"targets have shape {tuple(y.shape)}, the net expects {(self.dims[0], self.batch)}")
        state = x.to(self.dtype).contiguous()
        for l in range(len(self.w) - 1, -1, -1):
            self._save[l](state, self.kept[l])
            out = self._state(self.dims[l], self.batch)
            self._forward[l](state, self.w[l], out)
            state = out
        error = e = (y.to(self.dtype) - state).contiguous()
        self.w4 = None
        for l in range(len(self.w)):
            below = None
            if l + 1 < len(self.w):  # before W[l] changes
                below = self._state(self.dims[l + 1], self.batch)
                self._gradient[l](self.w[l], e, self.kept[l], below, workspace=self._workspace)
            self._update[l](self.w[l], e, self.kept[l], workspace=self._workspace)
            e = below
        return error

    def pack(self) -> None:
        """Lays the weights out in 4 bits for ``predict``, which does so itself after a
        ``step``; for a program that changes ``w``."""
        self.w4 = []
        for w in self.w:
            k = mx.build_mx_quantize(*w.shape, "identity", self.dtype)
            self.w4.append(k.new_output(self.device))
            k(w, self.w4[-1])

    def predict(self, x: torch.Tensor) -> torch.Tensor:
        """Outputs ``[classes, n]`` of ``x [features, n]`` with the packed weights."""
        if self.w4 is None:
            self.pack()
        state, n, d = x.to(self.dtype).contiguous(), x.shape[1], self.dims
        for l in range(len(self.w4) - 1, -1, -1):
            out = self._state(d[l], n)
            if n <= FEW:
                k = mx.build_mx_predict(d[l], d[l + 1], n, self.activation, self.dtype)
                k(state, self.w4[l], out, workspace=k.new_workspace(self.device))
            else:
                q = mx.build_mx_quantize(d[l + 1], n, self.activation, self.dtype, axis=0)
                state4 = q.new_output(self.device)
                q(state, state4)
                mx.build_mx_forward(d[l], d[l + 1], n, self.dtype)(state4, self.w4[l], out)
            state = out
        return state

    def bytes_kept(self) -> tuple[int, int]:
        """Bytes of the kept states, and of the same states at full width."""
        packed = sum(t.numel() * t.element_size() for k in self.kept for t in k)
        width = torch.empty((), dtype=self.dtype).element_size()
        return packed, sum(self.dims[1:]) * self.batch * width


class FourBitSteps:
    """iPC steps on 4-bit operands: ``x`` (L + 1 states) and ``w`` (L weights), all of
    one type, are the masters and are updated in place."""

    def __init__(self, x, w, activation: str = "tanh", alpha: float = 1e-4, gamma: float = 0.5):
        self.x, self.w = list(x), list(w)
        self.activation, self.alpha, self.gamma = activation, float(alpha), float(gamma)
        self.dtype, self.batch = self.x[0].dtype, int(self.x[0].shape[1])
        if len(self.x) != len(self.w) + 1:
            raise ValueError("one state more than weights")
        self.e = [torch.empty_like(t) for t in self.x[:-1]]

    def _packed(self, t, axis, activation="identity"):
        k = mx.build_mx_quantize(*t.shape, activation, self.dtype, axis=axis)
        out = k.new_output(t.device)
        k(t, out)
        return out

    def step(self) -> None:
        x, w, e, L, B, dt, act = self.x, self.w, self.e, len(self.w), self.batch, self.dtype, self.activation
        for l in range(L):
            M, K = w[l].shape
            mx.build_mx_prediction_error(M, K, B, dt)(self._packed(x[l + 1], 0, act), self._packed(w[l], 1), x[l], e[l])
        for l in range(1, L):
            K, M = w[l - 1].shape
            mx.build_mx_inference_update(M, K, B, act, dt, self.gamma)(x[l], e[l], self._packed(w[l - 1], 0),
                                                                       self._packed(e[l - 1], 0))
        for l in range(L):
            M, K = w[l].shape
            mx.build_mx_weight_update(M, K, B, dt, self.alpha)(w[l], self._packed(e[l], 1), self._packed(x[l + 1], 1, act))

    def energy(self) -> float:
        """Half the squared prediction errors of the last step."""
        return float(sum((t.double() ** 2).sum() for t in self.e)) / 2


def train(dataset, *, hidden=64, depth=2, batch=128, epochs=8, rate=0.01, activation="relu", dtype=torch.float32,
          seed=0, device=None, log=print):
    """Trains a ``CompactNet`` on an ``ArrayDataset`` and scores it with its packed
    weights after every epoch; returns (records, net)."""
    device = torch.device(device or "cuda", 0)
    net = CompactNet((dataset.num_classes,) + (hidden,) * depth + (dataset.features,), batch, activation, dtype, rate,
                     device=device, seed=seed)
    records = []
    for epoch in range(epochs):
        loss, total, right = torch.zeros((), device=device, dtype=torch.float64), 0, torch.zeros((), device=device)
        batches = list(dataset.batches(batch, seed=seed, epoch=epoch))
        for images, labels in batches:
            x = images.reshape(batch, -1).T.contiguous().to(device)
            y = torch.nn.functional.one_hot(labels, dataset.num_classes).T.to(device, torch.float32)
            loss += (net.step(x, y).double() ** 2).sum() / 2
            total += batch
        net.pack()
        for images, labels in batches:
            x = images.reshape(batch, -1).T.contiguous().to(device)
            right += (net.predict(x).float().argmax(0) == labels.to(device)).sum()
        packed, full = net.bytes_kept()
        records.append({"epoch": epoch + 1, "loss": float(loss) / max(total, 1), "train_acc_4bit": float(right) / max(total, 1),
                        "samples": total, "state_bytes": packed, "state_bytes_full": full})
        log(f"epoch={epoch + 1:03d} loss={records[-1]['loss']:.4f} train_acc (4-bit weights)="
            f"{records[-1]['train_acc_4bit']:.4f} states kept in {packed} bytes of {full}")
    return records, net
