"""Rotary positions in general form: layouts, part of the head, stretched contexts, paged caches.

``rope.rope_qkv`` is the decoder's own case (interleaved pairs of the whole head, as many
key heads as query heads, positions 0 .. T-1).  Here:

* ``RotaryTable`` holds the cosines and sines of every position, computed in 64 bits and
  rounded once (in 32 bits the angle of position 100,000 is off by several thousandths),
  with the frequencies stretched for contexts longer than trained:
  ``"linear"`` divides every position by ``factor``; ``"ntk"`` raises the base to
  ``theta * factor ** (R / (R - 2))``, which keeps the fastest pair and divides the slowest
  by ``factor``; ``"yarn"`` (Peng et al., 2023) keeps pairs that turn more than 32 times
  within ``original_positions``, divides those that turn less than once by ``factor``, ramps
  between (over the pairs' numbers, from whole pair to whole pair) and scales cosine and sine by
  ``0.1 ln(factor) + 1``.
* ``rotary_qkv`` splits a projection output into turned q, k and v for training, with its
  gradient (``ca_rotary_qkv_forward`` / ``_backward``).
* ``rotary_append`` turns new tokens at their cache positions and writes keys and values
  into the paged cache that ``paged.continuum_attention_paged`` reads (``ca_rotary_append``).

``layout`` is ``"interleaved"`` (pairs (2p, 2p+1), the reference's apply_rope,
cuda/continuum_attention.py:825-835) or ``"half"`` (pairs (p, p + R/2)).
"""
from __future__ import annotations

import math
import threading
from typing import Optional

import torch

from . import _native
from .attention import _DTYPE_CODE, on_device, raw_stream
from .paged import check_cache, refuse_gradients
from .rope import settled

_LAYOUTS = {"interleaved": _native.CA_ROTARY_INTERLEAVED, "half": _native.CA_ROTARY_HALF}
SCALINGS = (None, "linear", "ntk", "yarn")


def rotary_frequencies(rotary_dim: int, theta: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                       original_positions: Optional[int] = None):
    """(angle per position of each pair, float64 [R/2]; the factor on cosine and sine)."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and >= 2, got {rotary_dim}")
    if not theta > 1:
        raise ValueError(f"theta must be > 1, got {theta}")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}, got {scaling!r}")
    if scaling is not None and not factor >= 1:
        raise ValueError(f"factor must be >= 1, got {factor}")
    R = rotary_dim
    base = float(theta)
    if scaling == "ntk" and R > 2:
        base *= factor ** (R / (R - 2))
    freq = base ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    if scaling == "linear":
        return freq / factor, 1.0
    if scaling == "yarn":
        if original_positions is None or original_positions < 1:
            raise ValueError("scaling 'yarn' needs original_positions")

        def pair_of(turns):    # the (real) index of the pair that turns this often in the original length
            return R * math.log(original_positions / (turns * 2 * math.pi)) / (2 * math.log(base))

        # the upper end may lie behind the last pair, R / 2 - 1, which then turns more than once and is not divided whole
        low, high = max(math.floor(pair_of(32)), 0), min(math.ceil(pair_of(1)), R - 1)
        ramp = ((torch.arange(R // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
        return freq / factor * ramp + freq * (1 - ramp), 0.1 * math.log(factor) + 1.0
    return freq, 1.0


class RotaryTable:
    """Cosines and sines of positions 0 .. ``max_positions`` - 1: ``cos_sin`` float32
    [max_positions, R/2, 2].  Build it once per model and device and pass it to every call."""

    def __init__(self, rotary_dim: int, max_positions: int, *, theta: float = 10000.0,
                 scaling: Optional[str] = None, factor: float = 1.0, original_positions: Optional[int] = None,
                 device="cuda"):
        if max_positions < 1:
            raise ValueError(f"max_positions must be >= 1, got {max_positions}")
        freq, scale = rotary_frequencies(rotary_dim, theta, scaling, factor, original_positions)
        with torch.inference_mode(False), torch.no_grad():    # training may save a table that serving made
            phase = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * freq.to(device)
            self.cos_sin = torch.stack((phase.cos() * scale, phase.sin() * scale), -1).float().contiguous()

    @classmethod
    def from_cos_sin(cls, cos_sin: torch.Tensor) -> "RotaryTable":
        """A table of the caller's own making, float32 [positions, R/2, 2] (such as ``rope.cos_sin_table``)."""
        if cos_sin.dim() != 3 or cos_sin.shape[2] != 2 or cos_sin.dtype != torch.float32 or cos_sin.shape[0] < 1 \
                or cos_sin.shape[1] < 1:
            raise ValueError("cos_sin must be float32 [positions, R/2, 2]; got "
                             f"{cos_sin.dtype} {tuple(cos_sin.shape)}")
        self = cls.__new__(cls)
        self.cos_sin = _aligned(cos_sin.contiguous())
        return self

    @property
    def rotary_dim(self) -> int:
        return 2 * self.cos_sin.shape[1]

    @property
    def positions(self) -> int:
        return self.cos_sin.shape[0]


_tables = {}
_tables_lock = threading.Lock()


def _capturing(device: torch.device) -> bool:
    if device.type != "cuda":
        return False
    with torch.cuda.device(device):
        return torch.cuda.is_current_stream_capturing()


def rotary_table(rotary_dim: int, max_positions: int, theta: float, scaling: Optional[str], factor: float,
                 original_positions: Optional[int], device) -> RotaryTable:
    """The ``RotaryTable`` of these settings, made once per device; not while a CUDA graph is captured."""
    device = torch.device(device)
    if device.type == "cuda" and device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    key = (rotary_dim, max_positions, float(theta), scaling, float(factor), original_positions, str(device))
    table = _tables.get(key)
    if table is None:
        with _tables_lock:
            table = _tables.get(key)
            if table is None:
                if _capturing(device):
                    raise RuntimeError("rotary_table: the table of these settings has to be made before a CUDA graph "
                                       "that uses it is captured (one call outside does)")
                table = RotaryTable(rotary_dim, max_positions, theta=theta, scaling=scaling, factor=factor,
                                    original_positions=original_positions, device=device)
                settled(table.cos_sin)
                _tables[key] = table
    return table


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy that starts on 16 bytes."""
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _head_dim(what, width, heads, kv_heads, dtype, device, table, layout):
    """Checks that rotary_qkv and rotary_append share; returns D."""
    if heads < 1 or kv_heads < 1:
        raise ValueError(f"{what}: heads={heads} and kv_heads={kv_heads} must be >= 1")
    if layout not in _LAYOUTS:
        raise ValueError(f"{what}: layout must be one of {sorted(_LAYOUTS)}, got {layout!r}")
    if dtype not in _DTYPE_CODE:
        raise TypeError(f"{what} supports float32, bfloat16 and float16, not {dtype}")
    if width % (heads + 2 * kv_heads):
        raise ValueError(f"{what}: {width} values a token are not heads + 2 kv_heads = {heads + 2 * kv_heads} heads")
    D = width // (heads + 2 * kv_heads)
    if D % 8 or not 8 <= D <= 256:
        raise ValueError(f"{what}: head dim {D} must be a multiple of 8 and <= 256")
    if table.rotary_dim > D:
        raise ValueError(f"{what}: the table turns {table.rotary_dim} values, a head has {D}")
    if device.type != "cuda":
        raise RuntimeError("continuum_attention_b200 runs on CUDA tensors only (no CPU fallback)")
    if table.cos_sin.device != device:
        raise RuntimeError(f"{what}: the table is on {table.cos_sin.device}, the input on {device}")
    return D


class RotaryQKVFunction(torch.autograd.Function):
    """qkv [B,T,(H+2G)D] -> q [B,H,T,D], k, v [B,G,T,D], q and k turned; native both ways."""

    @staticmethod
    def forward(ctx, qkv, cos_sin, positions, heads, kv_heads, layout):
        B, T, width = qkv.shape
        D = width // (heads + 2 * kv_heads)
        if not qkv.is_contiguous() or qkv.data_ptr() % 16:
            qkv = _aligned(qkv.contiguous())
        q = qkv.new_empty(B, heads, T, D)
        k, v = qkv.new_empty(B, kv_heads, T, D), qkv.new_empty(B, kv_heads, T, D)
        stride = 0 if positions is None or positions.dim() == 1 else positions.stride(0)
        with on_device(qkv.device):
            st = _native.lib().ca_rotary_qkv_forward(
                qkv.data_ptr(), width, cos_sin.data_ptr(), None if positions is None else positions.data_ptr(),
                stride, q.data_ptr(), k.data_ptr(), v.data_ptr(), B, T, heads, kv_heads, D, 2 * cos_sin.shape[1],
                cos_sin.shape[0], layout, _DTYPE_CODE[qkv.dtype], raw_stream(qkv.device))
        _native.check("ca_rotary_qkv_forward", st)
        ctx.save_for_backward(cos_sin, positions)
        ctx.meta = (B, T, heads, kv_heads, D, stride, layout, qkv.dtype)
        ctx.set_materialize_grads(False)
        return q, k, v

    @staticmethod
    def backward(ctx, dq, dk, dv):
        if torch.is_grad_enabled():
            raise RuntimeError("rotary_qkv supports first-order gradients only")
        cos_sin, positions = ctx.saved_tensors
        B, T, heads, kv_heads, D, stride, layout, dtype = ctx.meta
        device = cos_sin.device
        grads = []
        for g, h in ((dq, heads), (dk, kv_heads), (dv, kv_heads)):
            if g is None:
                g = torch.zeros((B, h, T, D), dtype=dtype, device=device)
            elif g.dtype != dtype or not g.is_contiguous() or g.data_ptr() % 16:
                g = _aligned(g.to(dtype).contiguous())
            grads.append(g)
        dqkv = grads[0].new_empty(B, T, (heads + 2 * kv_heads) * D)
        with on_device(device):
            st = _native.lib().ca_rotary_qkv_backward(
                grads[0].data_ptr(), grads[1].data_ptr(), grads[2].data_ptr(), cos_sin.data_ptr(),
                None if positions is None else positions.data_ptr(), stride, dqkv.data_ptr(), B, T, heads, kv_heads,
                D, 2 * cos_sin.shape[1], cos_sin.shape[0], layout, _DTYPE_CODE[dtype], raw_stream(device))
        _native.check("ca_rotary_qkv_backward", st)
        return dqkv, None, None, None, None, None


def rotary_qkv(qkv: torch.Tensor, heads: int, table: RotaryTable, *, kv_heads: Optional[int] = None,
               layout: str = "interleaved", positions: Optional[torch.Tensor] = None):
    """Split [B, T, (heads + 2 kv_heads) D] into turned q [B,heads,T,D], k and plain v [B,kv_heads,T,D].

    ``positions`` int32 [T] or [B,T] (default 0 .. T-1).  A position outside the table turns its
    token's values into NaN and is recorded in the library's device status word.  The gradient is
    qkv's; the table is a constant.
    """
    kv_heads = heads if kv_heads is None else kv_heads
    if qkv.dim() != 3:
        raise ValueError(f"rotary_qkv expects [B, T, width]; got {tuple(qkv.shape)}")
    if table.cos_sin.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("rotary_qkv: the table is a constant and gets no gradient; detach its cos_sin")
    B, T, width = qkv.shape
    _head_dim("rotary_qkv", width, heads, kv_heads, qkv.dtype, qkv.device, table, layout)
    if positions is None:
        if T > table.positions:
            raise ValueError(f"rotary_qkv: {T} positions, a table of {table.positions}")
    else:
        if positions.dtype != torch.int32 or tuple(positions.shape) not in ((T,), (B, T)):
            raise ValueError(f"rotary_qkv: positions must be int32 [{T}] or [{B}, {T}]; got {positions.dtype} "
                             f"{tuple(positions.shape)}")
        if positions.device != qkv.device:
            raise RuntimeError("rotary_qkv: positions must be on qkv's device")
        positions = positions.contiguous()
    return RotaryQKVFunction.apply(qkv, table.cos_sin, positions, heads, kv_heads, _LAYOUTS[layout])


def rotary_append(qkv: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                  kv_lens: torch.Tensor, q_starts: torch.Tensor, table: RotaryTable, *, heads: int,
                  layout: str = "interleaved", out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Turn new tokens at their cache positions, store keys and values in the cache, return q [N, heads, D].

    ``qkv`` [N, (heads + 2 kv_heads) D] packs the new tokens of all sequences; the cache arguments are
    those of ``paged.continuum_attention_paged``, and ``kv_lens`` already counts the new tokens.  Keys and
    values are written in place; no two tokens may share a slot.  Rows behind the last sequence are left
    as they were in ``out`` (undefined without it).  Serving only: no gradient.
    """
    if qkv.dim() != 2:
        raise ValueError(f"rotary_append expects qkv [N, width]; got {tuple(qkv.shape)}")
    refuse_gradients("rotary_append", qkv, k_cache, v_cache, table.cos_sin)
    P, G, page, D = check_cache("rotary_append", k_cache, v_cache, page_table, kv_lens, q_starts, qkv.dtype,
                                qkv.device)
    if _head_dim("rotary_append", qkv.shape[1], heads, G, qkv.dtype, qkv.device, table, layout) != D:
        raise ValueError(f"rotary_append: {qkv.shape[1]} values a token are not {heads} + 2 * {G} heads of {D}")
    N = qkv.shape[0]
    if qkv.stride(1) != 1 or qkv.stride(0) < qkv.shape[1] or (qkv.stride(0) * qkv.element_size()) % 16 \
            or qkv.data_ptr() % 16:
        qkv = qkv.clone(memory_format=torch.contiguous_format)
    if out is None:
        out = torch.empty(N, heads, D, dtype=qkv.dtype, device=qkv.device)
    elif out.shape != (N, heads, D) or out.dtype != qkv.dtype or out.device != qkv.device \
            or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError(f"rotary_append: out must be a contiguous, 16-byte aligned {qkv.dtype} "
                         f"[{N}, {heads}, {D}] on {qkv.device}")
    cs = table.cos_sin
    with on_device(qkv.device):
        st = _native.lib().ca_rotary_append(
            qkv.data_ptr(), qkv.stride(0), cs.data_ptr(), out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
            k_cache.stride(0), k_cache.stride(1), k_cache.stride(2), page_table.data_ptr(), page_table.stride(0),
            kv_lens.data_ptr(), q_starts.data_ptr(), N, kv_lens.shape[0], heads, G, D, table.rotary_dim, cs.shape[0],
            P, page, page_table.shape[1], _LAYOUTS[layout], _DTYPE_CODE[qkv.dtype], raw_stream(qkv.device))
    _native.check("ca_rotary_append", st)
    return out
