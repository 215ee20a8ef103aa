"""B200-native (sm_100a) sparse-pooling layer: a drop-in for the reference
``sparse_pooling`` package's Mode-A fp32 hot path.

About 10^8 logical neurons each compute ``act(b + sum_{k<8} w_k x[idx_k])``
and are pooled into contiguous groups without materialising the [B, H]
hidden tensor; backward gives dX, dW, db; ``FusedAdamW`` applies the
optimizer in one pass.  Dense operators for the layers around it (``linear_act``,
``group_norm_act``, 8-bit activation checkpoints) are in ``dense``.  All GPU work runs in the in-tree library
``_lib/libgranule_b200.so`` through the C ABI of ``include/granule_b200.h``.
"""
from .dense import (Activation8, GroupNormAct, LinearAct, decode_activation, encode_activation, group_norm_act,
                    linear_act)
from .config import LevelSpec, PhysicalPlan, PoolingConfig
from .layer import SparsePoolingLayer
from .layout import SparseLayout, init_parameters
from .optim import FusedAdamW

__all__ = ["SparsePoolingLayer", "PoolingConfig", "LevelSpec", "PhysicalPlan", "SparseLayout", "init_parameters",
           "FusedAdamW", "linear_act", "LinearAct", "group_norm_act", "GroupNormAct", "encode_activation",
           "decode_activation", "Activation8"]
