"""lich_amd: MI355X-native (gfx950) iPC training step.

Hand-written HIP kernels behind the C ABI of ``include/ipc_hip.h``
(``libipc_hip.so``, built in-tree by ``lich_amd.build``), with a Python host
surface that mirrors the reference's ``ipc_tilelang`` package: kernel
builders (``lich_amd.kernels``), layer batching, the small-batch weight
update, the trainer (``IPCConfig``, ``HipIPC``/``TileLangIPC``,
``prepare_batch``) and graph capture.
"""
from .kernels import (KernelConfig, build_forward, build_inference_update, build_prediction_error,
                      build_weight_update, build_weight_update_outer)
from .microscale import (MXMatrix, build_checkpoint_gradient, build_checkpoint_save, build_checkpoint_weight_update,
                         build_mx_dequantize, build_mx_forward, build_mx_inference_update, build_mx_predict,
                         build_mx_prediction_error, build_mx_quantize, build_mx_weight_update)
from .tokens import (build_dropout, build_embedding, build_embedding_update, build_token_loss, build_token_update)
from .trainer import HipIPC, IPCConfig, TileLangIPC, prepare_batch

__all__ = [
    "KernelConfig", "build_prediction_error", "build_inference_update", "build_weight_update",
    "build_weight_update_outer", "build_forward", "IPCConfig", "HipIPC", "TileLangIPC", "prepare_batch",
    "MXMatrix", "build_mx_quantize", "build_mx_dequantize", "build_mx_forward", "build_mx_prediction_error",
    "build_mx_inference_update", "build_mx_weight_update", "build_mx_predict", "build_checkpoint_save",
    "build_checkpoint_gradient", "build_checkpoint_weight_update", "build_embedding", "build_embedding_update",
    "build_dropout", "build_token_loss", "build_token_update",
]
__version__ = "0.1.0"
