"""B200-native (sm_100a) int8 weight-only linear for vladimirfilip/llm-serving-engine.

The compute path is liblse_int8.so (hand-written CUDA for sm_100a, C ABI in
include/lse_int8.h); this package is its host side: the ctypes binding (`_lib`), the
torch-facing ops (`ops`), the drop-in modules and the model hook (`int8_linear`), the
on-disk int8 checkpoint (`checkpoint`), the 8-bit K/V cache and token log-probabilities (`ops`), the output-column split over ranks (`parallel`)
and the seeded inputs (`inputs`).
"""

from .checkpoint import load_int8_checkpoint_, save_int8_checkpoint  # noqa: F401
from .int8_linear import FusedInt8QKV, Int8Linear, Int8LlamaMLP, int8_weight_bytes, quantize_llama_  # noqa: F401
from .ops import (ALGO_AUTO, ALGO_GEMV, ALGO_SKINNY, ALGO_TCGEN05, Kv8Cache, TokenLogprobs, device_status,  # noqa: F401
                  int8_linear, int8_linear_packed, kv8_cache, kv8_decode_attention, kv8_paged_attention, kv8_read,
                  kv8_rope_append, pack_weight, quantize_per_channel, token_logprobs)

__version__ = "0.1.0"
