"""pa_int8 -- paged-attention decode for one AMD MI355X (gfx950).

FP16, per-token INT8 and 4-bit KV decode kernels, quantize + paged-cache write
kernels and block tables built on the device, hand-written in HIP, behind the
C ABI of include/pa_mi355x.h and a thin torch extension with the reference's
op names.
"""

from .registry import (  # noqa: F401
    KIND,
    VARIANTS,
    VARIANTS_INT4,
    VARIANTS_INT8,
    decode,
    decode_plan,
    extend_block_tables,
    gather_cache_int4,
    paged_decode_attention,
    reshape_and_cache,
    reshape_and_cache_int4,
    reshape_and_cache_int8,
    reshape_and_cache_int8_static,
)
from .paged_cache import PagedKVCache  # noqa: F401
from ._loader import capi, ext  # noqa: F401
