"""B200-native (sm_100a) Continuum Attention.

Public API (mirrors the reference project's operator):
    continuum_attention(q, k, v, log_gain, query_tile=64)   learned per-head gain (S/H)
    continuum_attention_fixed_tau(q, k, v, tau=0.30)        fixed temperature (P)
    ContinuumAttentionFunction                              the torch.autograd.Function
    use_impl("simt" | "tcgen05" | "auto")                   kernel-family override
    deterministic_backward(True)                            bitwise-reproducible dQ (also
                                                            under torch.use_deterministic_algorithms)
    continuum_attention_paged(q, k_cache, v_cache, ...)     new tokens over a paged cache (serving)
    PagedKVCache                                            the cache's pages and page table
    rotary_qkv / rotary_append / RotaryTable                rotary positions in general form

The kernels live in the native library libca_b200.so (C ABI in
include/continuum_attention_b200.h); build it with
``python -m continuum_attention_b200.build``.
"""
from .attention import (ContinuumAttentionFunction, backward_raw, continuum_attention,
                        continuum_attention_fixed_tau, deterministic_backward, forward_raw, use_impl,
                        workspace_bytes)
from .paged import PagedKVCache, PagedStep, continuum_attention_paged, paged_workspace_bytes
from .rotary import RotaryTable, rotary_append, rotary_qkv
from ._native import CANativeError, LIB_PATH, lib

__all__ = ["continuum_attention", "continuum_attention_fixed_tau", "ContinuumAttentionFunction",
           "use_impl", "deterministic_backward", "forward_raw", "backward_raw", "workspace_bytes",
           "continuum_attention_paged", "paged_workspace_bytes", "PagedKVCache", "PagedStep", "RotaryTable",
           "rotary_qkv", "rotary_append", "CANativeError", "LIB_PATH", "lib"]
