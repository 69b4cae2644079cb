"""kvbridge-b200: B200-native (sm_100a) paged INT8-KV grouped-query split-K
decode attention, drop-in for the kvbridge attention library.

The product is the C++/CUDA library ``libkvbridge_b200.so`` behind the C ABI
of ``include/kvbridge_c.h``; this package binds it with ctypes and mirrors the
reference's interface names (``Shape``, ``DeviceInput``, ``launch_attention``,
``merge_attention``, ...).
"""
from .api import (  # noqa: F401
    AppendInput,
    AppendShape,
    append_kv,
    append_shape_error,
    BatchInput,
    BatchShape,
    DeviceInput,
    Shape,
    attention_b200_supported,
    attention_mma_supported,
    attention_partitions,
    attention_shape_error,
    attention_shape_valid,
    batch_shape_error,
    batch_workspace_bytes,
    kSplitTokens,
    launch_attention,
    launch_attention_batched,
    launch_attention_ex,
    launch_attention_mma,
    launch_attention_partials,
    merge_attention,
    merge_attention_ex,
    merge_attention_shards,
    merge_attention_shards_ex,
    merge_attention_peers,
    debug_copy_to_device,
    peer_buffer_alloc,
    peer_buffer_bytes,
    peer_buffer_close,
    peer_buffer_free,
    peer_buffer_open,
    peer_slot,
    set_wait_limit_ns,
    wait_limit_ns,
    debug_fail_launch,
    debug_skip_stage,
    launch_attention_noalloc,
    set_decode_kernel,
    decode_kernel,
    KERNEL_AUTO,
    KERNEL_WARP_MMA,
    KERNEL_TCGEN05,
    KERNEL_GENERAL,
    output_numerator_elements,
    output_scalar_elements,
    preload_attention_kernels,
    preload_attention_mma_kernels,
    preload_attention_reference_kernels,
    read_device_status,
    read_wait_failure,
    schedule_cta_of,
    scratch_elements,
    split_count,
    validate_shape,
)
from ._lib import LIB_PATH, LibraryMissing  # noqa: F401

# The 4-bit cache (kv4.py) takes torch tensors; torch is imported with it.
_KV4 = (
    "EvictPlan",
    "Kv4Pool",
    "Kv4Query",
    "Kv4Rows",
    "accumulate_weights_kv4",
    "append_kv4",
    "attention_kv4_workspace_bytes",
    "compact_kv4",
    "launch_attention_kv4",
    "load_kv4",
    "select_tokens",
)


def __getattr__(name):
    if name not in _KV4:
        raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
    from . import kv4

    for known in _KV4:
        globals()[known] = getattr(kv4, known)
    return globals()[name]


def __dir__():
    return sorted({*globals(), *_KV4})
