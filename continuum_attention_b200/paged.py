"""Continuum Attention over a paged key/value cache: prompts in pieces and single tokens.

``continuum_attention_paged`` answers packed new tokens of many sequences against a cache
whose keys and values lie in fixed-size pages (``ca_paged_forward``); ``rotary.rotary_append``
fills the cache.  ``PagedKVCache`` owns the pages of every layer and hands out, per step, the
page table, lengths and row ranges that both take.

The operator is that of ``attention.continuum_attention`` (scores, piecewise-linear
trajectories, half caps on the first and on the row's own key), so a prompt fed in pieces, or a
token at a time, gives the rows that one call over the whole sequence gives.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Sequence

import torch
from torch.autograd import forward_ad

from . import _native
from .attention import _DTYPE_CODE, on_device, raw_stream


def refuse_gradients(what, *tensors):
    """The serving operators drop no gradient without a word."""
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} has no backward; call it under torch.no_grad()")
    refuse_tangents(what, *tensors)


def refuse_tangents(what, *tensors):
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what} has no forward-mode gradient")


class _NoBackward(torch.autograd.Function):
    """An output of parameters that ask for a gradient: a backward pass through it says that there is none."""

    @staticmethod
    def forward(ctx, out, log_gain):
        ctx.mark_dirty(out)      # not a view: it may be changed in place
        return out

    @staticmethod
    def backward(ctx, grad):
        raise RuntimeError("continuum_attention_paged has no backward, for log_gain neither; call it under "
                           "torch.no_grad()")


def check_cache(what, k_cache, v_cache, page_table, kv_lens, q_starts, dtype, device):
    """Checks of the cache arguments, shared with ``rotary.rotary_append``; returns (pages, kv_heads,
    page_size, D).  Values on the device (lengths, pages) are checked by the kernels."""
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ValueError(f"{what}: k_cache and v_cache must share one shape [pages, kv_heads, page_size, D]; got "
                         f"{tuple(k_cache.shape)}, {tuple(v_cache.shape)}")
    if k_cache.dtype != dtype or v_cache.dtype != dtype:
        raise ValueError(f"{what}: new tokens and cache must share dtype; got {dtype}, {k_cache.dtype}, "
                         f"{v_cache.dtype}")
    P, G, page, D = k_cache.shape
    if G < 1 or page < 1:
        raise ValueError(f"{what}: the cache needs kv_heads and page_size >= 1; got {tuple(k_cache.shape)}")
    strides = k_cache.stride()
    if strides != v_cache.stride():
        raise ValueError(f"{what}: k_cache and v_cache must share strides")
    unit = 16 // k_cache.element_size()
    if strides[3] != 1 or strides[0] % unit or strides[1] % unit or strides[2] % unit \
            or k_cache.data_ptr() % 16 or v_cache.data_ptr() % 16:
        raise ValueError(f"{what}: the cache's D values must be contiguous, its strides and start multiples of "
                         "16 bytes")
    S = kv_lens.numel()
    if page_table.dim() != 2 or kv_lens.dim() != 1 or q_starts.dim() != 1 \
            or page_table.shape[0] != S or q_starts.numel() != S + 1:
        raise ValueError(f"{what}: expected page_table [S, pages], kv_lens [S], q_starts [S+1]; got "
                         f"{tuple(page_table.shape)}, {tuple(kv_lens.shape)}, {tuple(q_starts.shape)}")
    if page_table.dtype != torch.int32 or kv_lens.dtype != torch.int32 or q_starts.dtype != torch.int32:
        raise TypeError(f"{what}: page_table, kv_lens and q_starts must be int32")
    if not (kv_lens.is_contiguous() and q_starts.is_contiguous()) or \
            (not page_table.is_contiguous() and ((page_table.shape[1] > 1 and page_table.stride(1) != 1) or
                                                 (S > 1 and page_table.stride(0) < page_table.shape[1]))):
        raise ValueError(f"{what}: page_table rows, kv_lens and q_starts must be contiguous")
    if device.type != "cuda":
        raise RuntimeError("continuum_attention_b200 runs on CUDA tensors only (no CPU fallback)")
    if not (k_cache.device == v_cache.device == page_table.device == kv_lens.device == q_starts.device == device):
        raise RuntimeError(f"{what}: every tensor must be on {device}")
    return P, G, page, D


def paged_workspace_bytes(num_seqs, max_q_len, heads, kv_heads, head_dim, dtype) -> int:
    return int(_native.lib().ca_paged_workspace_size(num_seqs, max_q_len, heads, kv_heads, head_dim,
                                                     _DTYPE_CODE[dtype]))


def continuum_attention_paged(q, k_cache, v_cache, page_table, kv_lens, q_starts, log_gain, *, max_q_len: int,
                              out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None):
    """Continuum Attention of packed new tokens q [N, H, D] over the paged cache; returns [N, H, D].

    k_cache, v_cache   [pages, G, page_size, D] of q's dtype (f32, bf16, f16), H a multiple of G,
                       D a multiple of 8 up to 128; strided views are fine
    page_table         int32 [S, pages_per_seq]: key j of sequence s is slot j % page_size of page
                       page_table[s, j // page_size]; entries no key needs are not used
    kv_lens            int32 [S]: keys of each sequence, its new tokens among them
    q_starts           int32 [S+1]: rows q_starts[s] .. q_starts[s+1] - 1 are sequence s's new
                       tokens, the last of them at position kv_lens[s] - 1
    log_gain           per-head log score gain [H]
    max_q_len          the new tokens of the longest sequence (1 for decoding): chooses the kernel;
                       a wrong one costs time only

    A row at a negative position (more rows than keys) sees nothing and gives zeros.  Rows behind
    ``q_starts[S]`` are left as they were in ``out`` (undefined without it).  Lengths and pages
    that are out of range give NaN rows and are recorded in the library's device status word, and so
    do calls of more tiles (16 to 128 rows of a key head by 32 or 64 keys) than 2^31, as in a prompt of
    a million tokens of 16 key heads.
    ``workspace`` (uint8, ``paged_workspace_bytes``) is allocated per call if not given; calls that
    may overlap need one each.  Serving only: q and caches that require a gradient are refused outside
    ``torch.no_grad()``; with a ``log_gain`` that does, a backward pass through the output raises.
    """
    if q.dim() != 3:
        raise ValueError(f"continuum_attention_paged expects q [N, H, D]; got {tuple(q.shape)}")
    refuse_gradients("continuum_attention_paged", q, k_cache, v_cache)
    refuse_tangents("continuum_attention_paged", log_gain)
    N, H, D = q.shape
    if q.dtype not in _DTYPE_CODE:
        raise TypeError(f"CA supports float32, bfloat16 and float16 inputs, not {q.dtype}")
    P, G, page, Dc = check_cache("continuum_attention_paged", k_cache, v_cache, page_table, kv_lens, q_starts, q.dtype,
                                 q.device)
    if Dc != D or H < 1 or H % G:
        raise ValueError(f"continuum_attention_paged: q has {H} heads of {D}, the cache {G} of {Dc}")
    if D % 8 or not 8 <= D <= 128:
        raise ValueError(f"continuum_attention_paged: head dim {D} must be a multiple of 8 and <= 128")
    if log_gain.dim() != 1 or log_gain.shape[0] != H:
        raise ValueError(f"log_gain must have shape [H]=[{H}], got {tuple(log_gain.shape)}")
    if int(max_q_len) < 1:
        raise ValueError(f"max_q_len must be >= 1, got {max_q_len}")
    lg = log_gain.detach()
    if lg.dtype != torch.float32 or lg.device != q.device or not lg.is_contiguous():
        lg = lg.to(device=q.device, dtype=torch.float32).contiguous()
    unit = 16 // q.element_size()
    if q.stride(2) != 1 or q.stride(0) % unit or q.stride(1) % unit or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    if out is None:
        out = torch.empty(N, H, D, dtype=q.dtype, device=q.device)
    elif out.shape != (N, H, D) or out.dtype != q.dtype or out.device != q.device or not out.is_contiguous() \
            or out.data_ptr() % 16:
        raise ValueError(f"continuum_attention_paged: out must be a contiguous, 16-byte aligned {q.dtype} "
                         f"[{N}, {H}, {D}] on {q.device}")
    S = kv_lens.numel()
    if N == 0 or S == 0:
        return out
    lib = _native.lib()
    code = _DTYPE_CODE[q.dtype]
    max_q_len = min(int(max_q_len), N)
    with on_device(q.device):
        nbytes = lib.ca_paged_workspace_size(S, max_q_len, H, G, D, code)
        if workspace is None:
            workspace = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
            given = nbytes
        else:
            given = workspace.numel() * workspace.element_size()
            if workspace.device != q.device or given < nbytes or not workspace.is_contiguous():
                raise ValueError(f"continuum_attention_paged: workspace must be {nbytes} contiguous bytes on {q.device}")
        ks, ps, ss, _ = k_cache.stride()
        st = lib.ca_paged_forward(
            q.data_ptr(), q.stride(0), q.stride(1), k_cache.data_ptr(), v_cache.data_ptr(), ks, ps, ss,
            page_table.data_ptr(), page_table.stride(0), kv_lens.data_ptr(), q_starts.data_ptr(), lg.data_ptr(),
            out.data_ptr(), workspace.data_ptr(), given, N, S, max_q_len, H, G, D, P, page, page_table.shape[1], code,
            raw_stream(q.device))
    _native.check("ca_paged_forward", st)
    return _NoBackward.apply(out.detach(), log_gain) if log_gain.requires_grad and torch.is_grad_enabled() else out


@dataclass
class PagedStep:
    """What one step passes to ``rotary_append`` and ``continuum_attention_paged``."""
    page_table: torch.Tensor    # int32 [S, pages_per_seq]
    kv_lens: torch.Tensor       # int32 [S], the step's new tokens among them
    q_starts: torch.Tensor      # int32 [S+1]
    max_q_len: int


class PagedKVCache:
    """Pages of keys and values for every layer, and the pages that each sequence holds.

    ``k`` and ``v`` are [layers, pages, kv_heads, page_size, head_dim]; one page table serves all
    layers.  Sequences are numbered 0 .. max_seqs-1 and start empty.
    """

    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, *, max_seqs: int,
                 max_len: int, dtype=torch.bfloat16, device="cuda"):
        if min(layers, pages, page_size, kv_heads, head_dim, max_seqs, max_len) < 1:
            raise ValueError("layers, pages, page_size, kv_heads, head_dim, max_seqs and max_len must be >= 1")
        self.page_size, self.max_len = page_size, max_len
        self.k = torch.zeros(layers, pages, kv_heads, page_size, head_dim, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        width = -(-max_len // page_size)
        self._table = torch.full((max_seqs, width), -1, dtype=torch.int32)   # host copy
        self._free = list(range(pages - 1, -1, -1))
        self.lens = [0] * max_seqs
        self._held = [0] * max_seqs          # pages of each sequence

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _grow(self, what: str, keys: Sequence[int]) -> None:
        """Pages for keys[s] keys of each sequence; raises, and changes nothing, when they do not suffice."""
        if max(keys) > self.max_len:
            raise ValueError(f"{what}: a sequence of {max(keys)} tokens exceeds the cache's max_len={self.max_len}")
        need = [max(-(-a // self.page_size), h) for a, h in zip(keys, self._held)]
        more = sum(need) - sum(self._held)
        if more > len(self._free):
            raise RuntimeError(f"{what}: the cache is out of pages: {more} needed, {len(self._free)} free")
        for s, (a, b) in enumerate(zip(self._held, need)):
            for j in range(a, b):
                self._table[s, j] = self._free.pop()
        self._held = need

    def reserve(self, keys: Sequence[int]) -> None:
        """Hold pages for keys[s] keys of each sequence in advance, so that the page tables of later steps
        (one captured into a graph, say) cover them."""
        if len(keys) != len(self.lens):
            raise ValueError(f"reserve takes one length for each of {len(self.lens)} sequences")
        self._grow("reserve", keys)

    def step(self, new: Sequence[int]) -> PagedStep:
        """Make room for new[s] more tokens of each sequence s; the step that appends them.  Raises, and
        changes nothing, when a sequence would pass ``max_len`` or the pages do not suffice."""
        if len(new) != len(self.lens) or min(new) < 0:
            raise ValueError(f"step takes one count >= 0 for each of {len(self.lens)} sequences")
        after = [a + n for a, n in zip(self.lens, new)]
        self._grow("step", after)
        self.lens = after
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        # one copy to the device for the three
        host = torch.cat((self._table.flatten(), torch.tensor(after + starts, dtype=torch.int32)))
        dev = host.to(self.k.device)
        S, width = self._table.shape
        return PagedStep(dev[:S * width].view(S, width), dev[S * width:S * width + S], dev[S * width + S:],
                         max(max(new), 1))

    def release(self, seq: int) -> None:
        """Empty a sequence: its pages return to the free ones."""
        for j in range(self._held[seq]):
            self._free.append(int(self._table[seq, j]))
        self._table[seq] = -1
        self._held[seq] = self.lens[seq] = 0
