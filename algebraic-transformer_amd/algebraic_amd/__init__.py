"""MI355X-native algebraic attention and fused algebraic LM head.

Public entry points keep the reference's signatures:
``algebraic_amd.kernels.flash.flash_attention`` (src/algebraic/kernels/flash.py:763) and
``algebraic_amd.kernels.fused_head.fused_head`` (src/algebraic/kernels/fused_head.py:260).
"""

from .kernels.embedding import token_embedding  # noqa: F401
from .kernels.flash import flash_attention, make_variant  # noqa: F401
from .kernels.fused_head import fused_head  # noqa: F401
from .kernels.norm import add_rms_norm, add_rms_norm_fp8, rms_norm  # noqa: F401
from .kernels.packed import packed_flash_attention  # noqa: F401
from .kernels.paged import paged_append, paged_flash_attention  # noqa: F401
from .kernels.paged_fp8 import paged_append_fp8, paged_flash_attention_fp8, paged_read_fp8  # noqa: F401
from .kernels.sample import head_logits, head_sample  # noqa: F401
