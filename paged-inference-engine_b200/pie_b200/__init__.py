"""B200 (sm_100a) paged-attention hot path: ctypes front end of libpaged_attn_b200.so."""
from ._lib import LIB_PATH, PagedAttnError, load  # noqa: F401
from .ops import (beam_select, compact_blocks, copy_blocks, paged_attention, reorder_beams,  # noqa: F401
                  write_kv)

__version__ = "0.1.0"
