from ._ext import get_ext, have_ext
from .attention import flash_attention_packed
from .norms import (FusedLayerNorm, FusedRMSNorm, FusedBlockNorm,
                    fused_block_norm)
from .linear import MFMALinear
from .optim import FusedAdamW, FusedSGD
from .bn import FusedBN2d
from .ce import fused_cross_entropy
from .clip import clip_grad_norm_, grad_norm
from .elementwise import fused_rope_axes
from .embedding import FusedEmbedding

__all__ = ["get_ext", "have_ext", "FusedLayerNorm", "FusedRMSNorm",
           "MFMALinear", "FusedAdamW", "FusedSGD", "FusedBN2d", "fused_cross_entropy", "FusedEmbedding",
           "flash_attention_packed", "fused_rope_axes", "FusedBlockNorm",
           "fused_block_norm", "clip_grad_norm_", "grad_norm"]
