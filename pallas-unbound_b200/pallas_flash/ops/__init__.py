from .interface import pallas_flash_attention
from .rotary import qk_norm_rope, rotary_frequencies

__all__ = ["pallas_flash_attention", "qk_norm_rope", "rotary_frequencies"]
