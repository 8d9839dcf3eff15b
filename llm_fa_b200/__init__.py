"""llm_fa_b200: FlashAttention forward (bf16, head dim 128, non-causal) for B200, and
attention over a paged 4-bit key/value cache (kv4).

The compute path is the sm_100a kernel in libllm_fa_b200.so behind the C ABI
of include/llm_fa_b200.h; this package is the host-side mirror of the
reference's Python surface (`llm_fa.mod.llm_fa_forward`, `llm_fa.forward`).
"""
from .attention import (HEAD_DIM, attention_flops, attention_forward, build_info,
                        device_status, launch_plan, max_active_clusters, reset_device_status,
                        selftest_wait_timeout, set_wait_timeout_ms, workspace_size)
from .kv4 import (KV4Cache, kv4_append, kv4_attention, kv4_evict_move, kv4_evict_select,
                  kv4_expand)

__all__ = [
    "HEAD_DIM", "attention_flops", "attention_forward", "build_info", "device_status",
    "launch_plan",
    "max_active_clusters", "reset_device_status", "selftest_wait_timeout", "set_wait_timeout_ms",
    "workspace_size",
    "KV4Cache", "kv4_append", "kv4_attention", "kv4_evict_move", "kv4_evict_select", "kv4_expand",
]
__version__ = "0.1.0"
