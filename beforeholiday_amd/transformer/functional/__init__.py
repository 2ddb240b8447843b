from .fused_attention import attention_dropout_keep, fused_grouped_attention
from .fused_dropout import dropout_keep, fused_dropout
from .fused_rope import fused_qk_norm_rope, rotary_tables
from .fused_softmax import FusedScaleMaskSoftmax, GenericFusedScaleMaskSoftmax

__all__ = ["FusedScaleMaskSoftmax", "GenericFusedScaleMaskSoftmax", "attention_dropout_keep", "dropout_keep",
           "fused_dropout", "fused_grouped_attention", "fused_qk_norm_rope", "rotary_tables"]
