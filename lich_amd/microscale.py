"""Microscaled operators: 4-bit products and 8-bit checkpoints (HIP, gfx950).

Microscaled storage (OCP MX) keeps 32 consecutive values of a row under one
power-of-two scale.  ``fp4`` (E2M1) carries weights and product operands,
``int8`` carries states that a backward pass reads again.  A packed matrix is an
``MXMatrix`` of two tensors whose layout ``include/ipc_hip.h`` states; the
quantiser's ``new_output()`` allocates one.

* ``build_mx_quantize`` / ``build_mx_dequantize``: a matrix, with f applied, into
  packed rows (``axis=1``) or packed columns (``axis=0``) and back.
* ``build_mx_prediction_error``, ``build_mx_forward``, ``build_mx_inference_update``,
  ``build_mx_weight_update``: the kernel families of ``lich_amd.kernels`` with
  both operands in fp4.
* ``build_mx_predict``: fp4 weights, states in their own type, few samples.
* ``build_checkpoint_save``, ``build_checkpoint_weight_update``,
  ``build_checkpoint_gradient``: a layer's state kept in int8 and the backward
  pass that reads it there.

Each builder returns a callable that validates its tensors and enqueues on
torch's current stream, as in ``lich_amd.kernels``; nothing is allocated or
synchronised inside a call.  The reference has no counterpart.
"""
from __future__ import annotations

from ctypes import c_float, c_int, c_void_p, cast
from functools import lru_cache
from typing import NamedTuple

import torch

from . import _native as nat
from .kernels import _check, _Kernel, _storage_dtype

try:
    from . import _fast_call
except ImportError:  # not built: the calls go through ctypes
    _fast_call = None

BLOCK, GROUP = 32, 128  # values per scale, per four scale bytes


class MXMatrix(NamedTuple):
    """Packed rows: ``codes`` [rows, bytes of a row], ``scales`` [groups of 128, rows, 4]."""

    codes: torch.Tensor
    scales: torch.Tensor


def _format(name: str) -> str:
    if name not in nat.MX_FORMATS:
        raise ValueError(f"unknown microscaled format {name!r}; expected 'fp4' or 'int8'")
    return name


def packed_shapes(rows: int, n: int, format: str = "fp4"):
    """Shapes of the codes and scales of ``rows`` packed rows of ``n`` values."""
    groups = -(-n // GROUP)
    width = groups * GROUP // 2 if _format(format) == "fp4" else -(-n // BLOCK) * BLOCK
    return (rows, width), (groups, rows, 4)


def new_packed(rows: int, n: int, format: str = "fp4", device=None) -> MXMatrix:
    """An uninitialised packed matrix of ``rows`` rows of ``n`` values."""
    return _Packed("packed", rows, n, format).new(device)


class _Packed:
    """Checks of a packed operand; the call gives its pointers."""

    def __init__(self, name: str, rows: int, n: int, format: str = "fp4"):
        self.name, self.format = name, _format(format)
        self.codes, self.scales = packed_shapes(rows, n, format)
        self.dtype = torch.uint8 if format == "fp4" else torch.int8

    def __call__(self, m):
        if not isinstance(m, tuple) or len(m) != 2:
            raise ValueError(f"{self.name} must be an MXMatrix (codes, scales)")
        return (_pointer(m[0], f"{self.name}.codes", self.codes, self.dtype),
                _pointer(m[1], f"{self.name}.scales", self.scales, torch.uint8))

    def new(self, device=None) -> MXMatrix:
        device = device or torch.device("cuda")
        return MXMatrix(torch.empty(self.codes, dtype=self.dtype, device=device),
                        torch.empty(self.scales, dtype=torch.uint8, device=device))


def _pointer(t, name: str, shape: tuple, dtype: torch.dtype) -> int:
    """The address of a tensor that passes ``_check``."""
    _check(t, name, shape, dtype)
    return t.data_ptr()


def _sizes(**sizes) -> None:
    if min(sizes.values()) < 1:
        raise ValueError("invalid shape " + " ".join(f"{k}={v}" for k, v in sizes.items()))


class _Operator:
    """A call of a library entry point whose arguments are pointers, constants, for some a
    lent workspace, and the stream.  ``_run(*operands[, workspace])`` makes it where
    every operand is what it has to be and returns 0; else ``_checked`` finds out why
    not and raises."""

    def _bind(self, entry: str, operands: tuple, *constants, workspace: bool = False) -> None:
        """``operands``: of each argument a ``_Packed`` or (name, shape, dtype)."""
        self._entry, self._operands, self._lends = getattr(nat.lib(), entry), operands, workspace
        self._constants = tuple(c_float(v) if isinstance(v, float) else c_int(v) for v in constants)
        self._run = _no_fast_call
        if _fast_call is not None and nat._raw_stream is not None:
            parts = []
            for o in operands:
                parts += [(o.codes, o.dtype), (o.scales, torch.uint8)] if isinstance(o, _Packed) else [tuple(o[1:])]
            self._run = _fast_call.Call(entry, cast(self._entry, c_void_p).value, tuple(parts), constants, nat._raw_stream)

    def _checked(self, rc: int, *given, workspace=None) -> None:
        if rc < 0:
            nat.check(rc)
        flat = [t for g in (*given, workspace) for t in (g if isinstance(g, tuple) else (g,))]
        devices = {t.device for t in flat if isinstance(t, torch.Tensor) and t.device.type == "cuda"}
        if len(devices) > 1:
            raise ValueError(f"tensors on different devices ({', '.join(sorted(map(str, devices)))})")
        pointers = []
        for o, t in zip(self._operands, given):
            pointers += o(t) if isinstance(o, _Packed) else (_pointer(t, *o),)
        first = given[0] if isinstance(given[0], torch.Tensor) else given[0][0]
        lent = _Kernel._ws(workspace) if self._lends else ()
        nat.check(self._entry(*pointers, *self._constants, *lent, nat.current_stream_handle(first.get_device())))


def _no_fast_call(*_) -> int:
    return 1


class _MXKernel(_Operator):
    def __init__(self, dtype, activation: str = "identity"):
        self.dtype = _storage_dtype(dtype)
        self.storage = nat.dtype_code(self.dtype)
        self.activation = str(activation).lower()
        self.act = nat.act_code(self.activation)


class MXQuantizeKernel(_MXKernel):
    """``k(X[R, C], packed)``: f(X) into packed rows (axis 1) or columns (axis 0)."""

    def __init__(self, R, C, activation, dtype, format, axis):
        super().__init__(dtype, activation)
        _sizes(R=R, C=C)
        if axis not in (0, 1):
            raise ValueError(f"axis must be 0 or 1 (got {axis})")
        self.R, self.C, self.axis, self.format = int(R), int(C), int(axis), _format(format)
        self.rows, self.length = (self.R, self.C) if axis == 1 else (self.C, self.R)
        packed = _Packed("packed", self.rows, self.length, format)
        self._bind("ipc_mx_quantize", (("X", (self.R, self.C), self.dtype), packed), self.R, self.C, self.axis,
                   nat.MX_FORMATS[format], self.storage, self.act)
        self._new = packed.new
        if _fast_call is not None:
            self._new = _fast_call.Packed(packed.codes, packed.dtype, packed.scales, torch.uint8, MXMatrix)

    def new_output(self, device=None) -> MXMatrix:
        return self._new(torch.device(device) if isinstance(device, (str, int)) else device)

    def __call__(self, x, packed):
        rc = self._run(x, packed)
        if rc:
            self._checked(rc, x, packed)


class MXDequantizeKernel(_MXKernel):
    """``k(packed, OUT[R, C])``: the values of R packed rows of C."""

    def __init__(self, R, C, dtype, format):
        super().__init__(dtype)
        _sizes(R=R, C=C)
        self.R, self.C, self.format = int(R), int(C), _format(format)
        self._bind("ipc_mx_dequantize", (_Packed("packed", self.R, self.C, format), ("OUT", (self.R, self.C), self.dtype)),
                   self.R, self.C, nat.MX_FORMATS[format], self.storage)

    def __call__(self, packed, out):
        rc = self._run(packed, out)
        if rc:
            self._checked(rc, packed, out)


class _MXProduct(_MXKernel):
    def __init__(self, M, K, B, dtype, activation="identity"):
        super().__init__(dtype, activation)
        _sizes(M=M, K=K, B=B)
        self.M, self.K, self.B = int(M), int(K), int(B)


class MXPredictionErrorKernel(_MXProduct):
    """``k(X4, W4, X_lower[M, B], E[M, B])``: ``E = X_lower - W f(X_upper)``; W [M, K]
    packed by rows, f(X_upper) [K, B] by columns."""

    def __init__(self, *a):
        super().__init__(*a)
        out = (self.M, self.B), self.dtype
        self._bind("ipc_mx_pred_err", (_Packed("X_upper", self.B, self.K), _Packed("W", self.M, self.K), ("X_lower", *out),
                                       ("E", *out)), self.M, self.K, self.B, self.storage)

    def __call__(self, x4, w4, x_lower, e):
        rc = self._run(x4, w4, x_lower, e)
        if rc:
            self._checked(rc, x4, w4, x_lower, e)


class MXForwardKernel(_MXProduct):
    """``k(X4, W4, OUT[M, B])``: ``OUT = W f(X_upper)``, operands as for the prediction error."""

    def __init__(self, *a):
        super().__init__(*a)
        self._bind("ipc_mx_forward", (_Packed("X_upper", self.B, self.K), _Packed("W", self.M, self.K),
                                      ("OUT", (self.M, self.B), self.dtype)), self.M, self.K, self.B, self.storage)

    def __call__(self, x4, w4, out):
        rc = self._run(x4, w4, out)
        if rc:
            self._checked(rc, x4, w4, out)


class MXInferenceUpdateKernel(_MXProduct):
    """``k(X[M, B], E[M, B], WT4, ET4)``: ``X += gamma(-E + f'(X) W_lower^T E_lower)``;
    W_lower [K, M] and E_lower [K, B] packed by columns."""

    def __init__(self, M, K, B, activation, dtype, gamma):
        super().__init__(M, K, B, dtype, activation)
        self.gamma = float(gamma)
        out = (self.M, self.B), self.dtype
        self._bind("ipc_mx_infer_update", (("X", *out), ("E", *out), _Packed("W_lower", self.M, self.K),
                                           _Packed("E_lower", self.B, self.K)),
                   self.M, self.K, self.B, self.gamma, self.storage, self.act)

    def __call__(self, x, e, wt4, et4):
        rc = self._run(x, e, wt4, et4)
        if rc:
            self._checked(rc, x, e, wt4, et4)


class MXWeightUpdateKernel(_MXProduct):
    """``k(W[M, K], E4, A4)``: ``W += alpha E A^T``; E [M, B] and A = f(X_upper) [K, B]
    packed by rows."""

    def __init__(self, M, K, B, dtype, alpha):
        super().__init__(M, K, B, dtype)
        self.alpha = float(alpha)
        self._bind("ipc_mx_weight_update", (("W", (self.M, self.K), self.dtype), _Packed("E", self.M, self.B),
                                            _Packed("A", self.K, self.B)),
                   self.M, self.K, self.B, self.alpha, self.storage)

    def __call__(self, w, e4, a4):
        rc = self._run(w, e4, a4)
        if rc:
            self._checked(rc, w, e4, a4)


class MXPredictKernel(_MXProduct):
    """``k(X[K, B], W4, OUT[M, B], *, workspace=None)``: ``OUT = W f(X)``, W [M, K] packed
    by rows, the states not quantised.  ``workspace`` (optional, caller-owned,
    ``new_workspace()``) lets a call of several samples evaluate f(X) once."""

    def __init__(self, M, K, B, activation, dtype):
        super().__init__(M, K, B, dtype, activation)
        self._bind("ipc_mx_predict", (("X", (self.K, self.B), self.dtype), _Packed("W", self.M, self.K),
                                      ("OUT", (self.M, self.B), self.dtype)),
                   self.M, self.K, self.B, self.storage, self.act, workspace=True)
        self.workspace_bytes = int(nat.lib().ipc_mx_predict_workspace_bytes(self.K, self.B, self.storage))

    new_workspace = _Kernel.new_workspace

    def __call__(self, x, w4, out, *, workspace=None):
        rc = self._run(x, w4, out, workspace)
        if rc:
            self._checked(rc, x, w4, out, workspace=workspace)


class CheckpointWeightUpdateKernel(_Operator, _Kernel):
    """``k(W[M, K], E[M, B], X8, *, workspace=None)``: ``W += alpha E f(X)^T``, X [K, B] kept
    in 8 bits.  ``workspace`` (optional, caller-owned, ``new_workspace()``) lets a
    large call evaluate f(X) once.  ``workspace_bytes`` is enough for it, in 16-bit storage also
    where a call of few samples reads none and ``new_workspace()`` gives None."""

    workspace_bytes = 0

    def __init__(self, *a, alpha, **kw):
        super().__init__("weight", *a, **kw)
        self.alpha = float(alpha)
        self._bind("ipc_ckpt_weight_update", (("W", (self.M, self.K), self.dtype), ("E", (self.M, self.B), self.dtype),
                                              _Packed("X", self.K, self.B, "int8")),
                   self.M, self.K, self.B, self.alpha, self.storage, self.operand, self.act, workspace=True)
        sizes = self.act, self.M, self.K, self.B, self.storage
        self._used = int(nat.lib().ipc_ckpt_weight_update_workspace_bytes(*sizes, self.operand))
        self.workspace_bytes = self._used if self.storage == nat.DT_F32 else int(nat.lib().ipc_ckpt_workspace_bytes(*sizes))

    def new_workspace(self, device=None) -> torch.Tensor | None:
        return super().new_workspace(device) if self._used else None

    def __call__(self, w, e, x8, *, workspace=None):
        rc = self._run(w, e, x8, workspace)
        if rc:
            self._checked(rc, w, e, x8, workspace=workspace)


class CheckpointGradientKernel(_Operator, _Kernel):
    """``k(W_lower[K, M], E_lower[K, B], X8, G[M, B], *, workspace=None)``:
    ``G = f'(X) W_lower^T E_lower``, X [M, B] kept in 8 bits.  ``workspace`` (optional,
    caller-owned, ``new_workspace()``) lets a 16-bit call lay out rows of an odd length once."""

    workspace_bytes = 0

    def __init__(self, *a, **kw):
        super().__init__("gradient", *a, **kw)
        self._bind("ipc_ckpt_gradient", (("W_lower", (self.K, self.M), self.dtype), ("E_lower", (self.K, self.B), self.dtype),
                                         _Packed("X", self.M, self.B, "int8"), ("G", (self.M, self.B), self.dtype)),
                   self.M, self.K, self.B, self.storage, self.operand, self.act, workspace=True)
        self.workspace_bytes = int(nat.lib().ipc_ckpt_gradient_workspace_bytes(self.M, self.K, self.B, self.storage))

    def __call__(self, w_lower, e_lower, x8, g, *, workspace=None):
        rc = self._run(w_lower, e_lower, x8, g, workspace)
        if rc:
            self._checked(rc, w_lower, e_lower, x8, g, workspace=workspace)


@lru_cache(maxsize=256)
def build_mx_quantize(R: int, C: int, activation: str = "identity", dtype="float32", *, format: str = "fp4",
                      axis: int = 1):
    """f(X [R, C]) into a packed matrix: R rows of C (``axis=1``) or C rows of R (``axis=0``)."""
    return MXQuantizeKernel(R, C, activation, dtype, format, axis)


@lru_cache(maxsize=256)
def build_mx_dequantize(R: int, C: int, dtype="float32", *, format: str = "fp4"):
    """A packed matrix of R rows of C values into OUT [R, C]."""
    return MXDequantizeKernel(R, C, dtype, format)


@lru_cache(maxsize=256)
def build_mx_prediction_error(M: int, K: int, B: int, dtype="float32"):
    """``E = X_lower - W f(X_upper)`` on fp4 operands."""
    return MXPredictionErrorKernel(M, K, B, dtype)


@lru_cache(maxsize=256)
def build_mx_forward(M: int, K: int, B: int, dtype="float32"):
    """``OUT = W f(X_upper)`` on fp4 operands."""
    return MXForwardKernel(M, K, B, dtype)


@lru_cache(maxsize=256)
def build_mx_inference_update(M: int, K: int, B: int, activation: str, dtype="float32", gamma: float = 0.5):
    """``X += gamma*(-E + f'(X)*W.T@E_lower)`` on fp4 operands."""
    return MXInferenceUpdateKernel(M, K, B, activation, dtype, gamma)


@lru_cache(maxsize=256)
def build_mx_weight_update(M: int, K: int, B: int, dtype="float32", alpha: float = 1e-4):
    """``W += alpha * E @ A.T`` on fp4 operands."""
    return MXWeightUpdateKernel(M, K, B, dtype, alpha)


@lru_cache(maxsize=256)
def build_mx_predict(M: int, K: int, B: int, activation: str, dtype="float32"):
    """``OUT = W f(X)`` with fp4 weights and states in ``dtype``."""
    return MXPredictKernel(M, K, B, activation, dtype)


def build_checkpoint_save(K: int, B: int, dtype="float32", activation: str = "identity"):
    """X [K, B] (or f(X), for a weight update built with ``identity``) into an 8-bit checkpoint."""
    return build_mx_quantize(K, B, activation, dtype, format="int8", axis=1)


@lru_cache(maxsize=256)
def build_checkpoint_weight_update(M: int, K: int, B: int, activation: str, dtype="float32", alpha: float = 1e-4, *,
                                   operand_dtype=None):
    """``W += alpha * E @ f(X).T`` with X [K, B] kept in 8 bits."""
    return CheckpointWeightUpdateKernel(M, K, B, activation, dtype, None, operand_dtype, alpha=alpha)


@lru_cache(maxsize=256)
def build_checkpoint_gradient(M: int, K: int, B: int, activation: str, dtype="float32", *, operand_dtype=None):
    """``G = f'(X) * (W_lower.T @ E_lower)`` with X [M, B] kept in 8 bits."""
    return CheckpointGradientKernel(M, K, B, activation, dtype, None, operand_dtype)
