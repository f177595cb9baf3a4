"""FlashMoBA for AMD Instinct MI355X (gfx950): the reference's Python API over hand-written HIP kernels."""
__version__ = "2.0.0+mi355x"

from flash_moba.flash_moba_interface import (  # noqa: F401
    flash_topk_varlen_func,
    flash_moba_attn_varlen_func,
    flash_moba_varlen_func,
)
from flash_moba.rotary import flash_moba_rotary_func  # noqa: F401
from flash_moba.kv_cache import (  # noqa: F401
    MobaKVCache,
    flash_moba_cache_append_func,
    flash_moba_cache_attn_func,
    flash_moba_cache_evict_func,
    flash_moba_with_cache_func,
)
