"""B200-native (sm_100a) DeepSeek sparse attention over a paged MLA latent cache.

Drop-in for the reference operator `kernel(q_nope, q_pe, ckv_cache, kpe_cache,
sparse_indices, sm_scale) -> (output, lse)` (solution/triton/kernel.py:138-182)
plus the FP8 lightning indexer and exact top-k that feed it, and the operators
around them in a serving step: block tables and slot maps (`step_layout`), rotary
positions (`apply_rope`), the latent-cache writer (`latent_cache_append`) and dense
attention behind a shared prefix (`shared_prefix_attention`).  All compute runs
in libdsa_b200.so (hand-written CUDA for sm_100a, C ABI in include/dsa_b200.h).
"""
from .kernel import (get_options, kernel, kernel_splitk, kernel_splitk_v2, options,  # noqa: F401
                     read_device_error, set_options, workspace_size)
from .latent_cache import latent_cache_append  # noqa: F401
from .layout import StepLayout, step_layout  # noqa: F401
from .prefix import prefix_workspace_size, read_prefix_error, shared_prefix_attention  # noqa: F401
from .rope import apply_rope, rope_frequencies  # noqa: F401

__all__ = ["kernel", "kernel_splitk", "kernel_splitk_v2", "read_device_error", "options",
           "set_options", "get_options", "workspace_size", "step_layout", "StepLayout", "apply_rope",
           "rope_frequencies", "latent_cache_append", "shared_prefix_attention", "prefix_workspace_size",
           "read_prefix_error"]
