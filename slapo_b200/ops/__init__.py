"""Modules and functions that schedules swap into models."""
from .linear import (FusedQKV, LinearWithAct, LinearWithDropout,  # noqa: F401
                     LinearWithSeparateBias, LinearWithSyncFunc)
from .adamw import (FusedAdamW, dequantize_moment, multi_tensor_adamw,  # noqa: F401
                    quantize_moment)
from .attention import FlashAttention, FlashAttentionOp  # noqa: F401
from .cross_entropy import ParallelCrossEntropy  # noqa: F401
from .embedding import FusedEmbedding  # noqa: F401
from .mlp import FusedMLP  # noqa: F401
from .norm import FusedDropoutAddLayerNorm, FusedLayerNorm, FusedRMSNorm  # noqa: F401
from .paged import PagedKVCache  # noqa: F401
from .rotary import RotaryEmbedding, rotary_table  # noqa: F401
from .sampling import sample  # noqa: F401
from .utils import Print  # noqa: F401
