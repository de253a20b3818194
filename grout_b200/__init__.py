"""grout_b200 — B200-native (sm_100a) attention hot path of the Grout engine.

The compute lives in libgrout_attn.so (CUDA C++ kernels behind the C ABI in
include/grout_attn.h); this package is its host-side mirror of the
reference's op interface (attn.py), the seeded input generator (synth.py)
and the build script (build.py).
"""
from .attn import (  # noqa: F401
    GroutError,
    add_rms_norm,
    attention_decode,
    attention_decode_fused,
    attention_decode_paged,
    attention_decode_paged_fp8,
    attention_decode_paged_window,
    attention_decode_window,
    attention_prefill,
    attention_prefill_paged,
    attention_prefill_paged_window,
    attention_prefill_splitk,
    attention_prefill_varlen,
    attention_prefill_varlen_window,
    check_device_error,
    decode_splits,
    decode_window_splits,
    decode_window_workspace_bytes,
    decode_workspace_bytes,
    init,
    inv_freq,
    kv_read_paged_fp8,
    lib,
    prefill_window_splits,
    prefill_window_workspace_bytes,
    qk_norm_rope_kv_decode,
    qk_norm_rope_kv_decode_paged,
    qk_norm_rope_kv_decode_paged_fp8,
    qk_norm_rope_kv_prefill,
    qk_norm_rope_kv_prefill_paged,
    qk_norm_rope_kv_prefill_paged_fp8,
    qkv_proj_norm_rope_kv_prefill,
    rope_table,
    silu_mul,
)

__version__ = "0.1.0"
