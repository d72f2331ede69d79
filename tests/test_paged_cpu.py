"""Refusals of the paged and rotary entry points, and the page bookkeeping, without a GPU."""
import ctypes

import pytest
import torch

from continuum_attention_b200 import (PagedKVCache, RotaryTable, _native, continuum_attention_paged, rotary_append,
                                      rotary_qkv)
from continuum_attention_b200.rotary import rotary_frequencies
from paged_testlib import arguments, make_case

FAKE = ctypes.c_void_p(256)


def _msg():
    return _native.lib().ca_last_error().decode()


def paged_args(**kw):
    a = dict(q=FAKE, qt=256, qh=64, k=FAKE, v=FAKE, ps=2048, hs=1024, ss=64, table=FAKE, ts=8, lens=FAKE, starts=FAKE,
             gain=FAKE, o=FAKE, ws=FAKE, wsb=1 << 40, rows=4, seqs=2, maxq=2, H=4, G=2, D=64, pages=16, page=16, pps=8,
             dtype=1)
    a.update(kw)
    return [*a.values(), None]


@pytest.mark.parametrize("change,status,text", [
    (dict(dtype=7), 1, "dtype"), (dict(rows=-1), 1, "negative"), (dict(page=0), 1, "page_size"),
    (dict(D=72 + 4), 2, "multiple of 8"), (dict(D=136), 2, "<= 128"), (dict(G=3), 1, "multiple of kv_heads"),
    (dict(G=0), 1, "multiple of kv_heads"), (dict(maxq=0), 1, "max_q_len"), (dict(q=None), 1, "null"),
    (dict(o=None), 1, "null"), (dict(table=None), 1, "null"), (dict(k=None), 1, "null"),
    (dict(q=ctypes.c_void_p(264)), 1, "aligned"), (dict(qt=260), 1, "strides"), (dict(ss=60), 1, "strides"),
    (dict(ts=7), 1, "page table"), (dict(pps=1 << 25, ts=1 << 25, page=64), 2, "2^30"),
    (dict(rows=1 << 31), 2, "2^31-1"), (dict(seqs=2049), 2, "2048"), (dict(maxq=1, rows=1 << 28, H=16), 2, "2^31-1"),
])
def test_paged_forward_refusals(change, status, text):
    assert _native.lib().ca_paged_forward(*paged_args(**change)) == status
    assert text in _msg()


def test_paged_forward_workspace_and_empty_calls():
    lib = _native.lib()
    assert lib.ca_paged_forward(*paged_args(rows=0)) == 0
    assert lib.ca_paged_forward(*paged_args(seqs=0)) == 0
    assert lib.ca_paged_workspace_size(0, 1, 4, 2, 64, 1) == 0
    need = lib.ca_paged_workspace_size(2, 2, 4, 2, 64, 1)
    if need:
        assert need % 256 == 0
        assert lib.ca_paged_forward(*paged_args(wsb=need - 1)) == 4
        assert lib.ca_paged_forward(*paged_args(ws=None)) == 4
        assert lib.ca_paged_forward(*paged_args(ws=ctypes.c_void_p(16))) == 1 and "workspace" in _msg()


@pytest.mark.parametrize("change,status,text", [
    (dict(dtype=3), 1, "dtype"), (dict(layout=2), 1, "layout"), (dict(D=12), 2, "multiple of 8"),
    (dict(D=264), 2, "<= 256"), (dict(R=3), 1, "even"), (dict(R=66), 1, "even"), (dict(R=0), 1, "even"),
    (dict(rows=3), 1, "table"), (dict(rows=0), 1, "table"), (dict(stride=500), 1, "row stride"),
    (dict(stride=516), 1, "row stride"), (dict(q=None), 1, "null"), (dict(k=ctypes.c_void_p(8)), 1, "aligned"),
    (dict(B=1 << 20, T=1 << 20, rows=1 << 30), 2, "2^31-1"), (dict(H=(1 << 20) + 1, stride=1 << 40), 2, "heads"),
])
def test_rotary_qkv_refusals(change, status, text):
    a = dict(x=FAKE, stride=512, cs=FAKE, pos=None, poss=0, q=FAKE, k=FAKE, v=FAKE, B=1, T=4, H=4, G=2, D=64, R=64,
             rows=4, layout=0, dtype=1)
    a.update(change)
    assert _native.lib().ca_rotary_qkv_forward(*a.values(), None) == status
    assert text in _msg()


@pytest.mark.parametrize("change,status,text", [
    (dict(n=-1), 1, "negative"), (dict(page=0), 1, "page_size"), (dict(lens=None), 1, "null"),
    (dict(kc=None), 1, "null"), (dict(hs=1028), 1, "strides"), (dict(R=1), 1, "even"), (dict(dtype=9), 1, "dtype"),
])
def test_rotary_append_refusals(change, status, text):
    a = dict(x=FAKE, stride=512, cs=FAKE, q=FAKE, kc=FAKE, vc=FAKE, ps=2048, hs=1024, ss=64, table=FAKE, ts=8,
             lens=FAKE, starts=FAKE, n=4, S=2, H=4, G=2, D=64, R=64, rows=128, pages=16, page=16, pps=8, layout=0,
             dtype=1)
    a.update(change)
    assert _native.lib().ca_rotary_append(*a.values(), None) == status
    assert text in _msg()


def test_python_refusals():
    c = make_case("bf16", 4, 2, 64, 16, [(1, 20), (2, 5)], device="cpu")
    args = arguments(c)
    with pytest.raises(RuntimeError, match="CUDA"):
        continuum_attention_paged(*args, max_q_len=2)

    def refused(exc, match, i, value):
        bad = list(args)
        bad[i] = value
        with pytest.raises(exc, match=match):
            continuum_attention_paged(*bad, max_q_len=2)

    refused(ValueError, "expects q", 0, c["q"][0])
    refused(TypeError, "supports", 0, c["q"].double())
    refused(ValueError, "share dtype", 0, c["q"].float())
    refused(ValueError, "one shape", 2, c["v_cache"][:1])
    refused(ValueError, "page_table", 3, c["page_table"][:1])
    refused(TypeError, "int32", 3, c["page_table"].long())
    refused(TypeError, "int32", 4, c["kv_lens"].long())
    refused(ValueError, "q_starts", 5, c["q_starts"][:-1])
    refused(ValueError, "strides", 1, c["k_cache"].transpose(2, 3).contiguous().transpose(2, 3))
    qkv = torch.zeros(3, 8 * 64, dtype=torch.bfloat16)
    table = RotaryTable(64, 32, device="cpu")
    cache = args[1:6]
    with pytest.raises(RuntimeError, match="CUDA"):
        rotary_append(qkv, *cache, table, heads=4)
    with pytest.raises(ValueError, match="N, width"):
        rotary_append(qkv[0], *cache, table, heads=4)
    with pytest.raises(RuntimeError, match="CUDA"):
        rotary_qkv(qkv[None], 4, table, kv_heads=2)
    with pytest.raises(ValueError, match="layout"):
        rotary_qkv(qkv[None], 4, table, kv_heads=2, layout="quarter")
    with pytest.raises(ValueError, match="heads"):
        rotary_qkv(qkv[None], 4, table, kv_heads=3)
    with pytest.raises(ValueError, match="turns"):
        rotary_qkv(qkv[None], 8, table, kv_heads=4)
    with pytest.raises(TypeError, match="supports"):
        rotary_qkv(qkv[None].double(), 4, table, kv_heads=2)


def test_rotary_frequencies_and_table():
    base, one = rotary_frequencies(8)
    assert one == 1.0 and torch.allclose(base, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64))
    lin, _ = rotary_frequencies(8, scaling="linear", factor=4.0)
    assert torch.equal(lin, base / 4)
    ntk, _ = rotary_frequencies(8, scaling="ntk", factor=4.0)
    assert ntk[0] == 1 and torch.allclose(ntk[-1], base[-1] / 4, rtol=1e-12)       # ends: kept, divided
    yarn, scale = rotary_frequencies(64, scaling="yarn", factor=8.0, original_positions=2048)
    plain, _ = rotary_frequencies(64)
    turns = 2048 * plain / (2 * torch.pi)
    assert torch.equal(yarn[turns > 40], plain[turns > 40])
    assert torch.allclose(yarn[turns < 0.7], plain[turns < 0.7] / 8, rtol=1e-12)
    assert (yarn <= plain).all() and (yarn >= plain / 8 * 0.999999).all() and scale == pytest.approx(1.20794415)
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, scaling="cubic"), dict(rotary_dim=8, theta=1),
                dict(rotary_dim=8, scaling="linear", factor=0.5), dict(rotary_dim=8, scaling="yarn", factor=2.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)
    t = RotaryTable(8, 100001, device="cpu")
    assert t.rotary_dim == 8 and t.positions == 100001 and t.cos_sin.dtype == torch.float32
    # the last angle to half a step of 32 bits, where a 32-bit angle would be off by 1e-3
    want = torch.stack(((100000 * base).cos(), (100000 * base).sin()), -1)
    assert (t.cos_sin[-1].double() - want).abs().max() < 2.0 ** -24
    again = RotaryTable.from_cos_sin(t.cos_sin)
    assert again.positions == 100001
    with pytest.raises(ValueError):
        RotaryTable.from_cos_sin(t.cos_sin.double())
    with pytest.raises(ValueError):
        RotaryTable(8, 0, device="cpu")


def test_cache_pages():
    c = PagedKVCache(2, 6, 4, 1, 8, max_seqs=3, max_len=16, dtype=torch.float32, device="cpu")
    assert c.k.shape == (2, 6, 1, 4, 8) and c.free_pages == 6
    s = c.step([5, 0, 1])
    assert s.kv_lens.tolist() == [5, 0, 1] and s.q_starts.tolist() == [0, 5, 5, 6] and s.max_q_len == 5
    used = s.page_table[0, :2].tolist() + s.page_table[2, :1].tolist()
    assert len(set(used)) == 3 and c.free_pages == 3 and (s.page_table[1] == -1).all()
    s2 = c.step([3, 0, 1])                                  # fits the pages held
    assert c.free_pages == 3 and s2.kv_lens.tolist() == [8, 0, 2] and torch.equal(s2.page_table, s.page_table)
    with pytest.raises(RuntimeError, match="out of pages"):
        c.step([0, 16, 0])
    with pytest.raises(ValueError, match="max_len"):
        c.step([9, 0, 0])
    with pytest.raises(ValueError, match="count"):
        c.step([1, 1])
    assert c.lens == [8, 0, 2] and c.free_pages == 3        # a refused step changes nothing
    c.release(0)
    assert c.free_pages == 5 and c.lens == [0, 0, 2]
    s3 = c.step([0, 16, 0])
    assert c.free_pages == 1 and s3.kv_lens.tolist() == [0, 16, 2] and s3.max_q_len == 16
    assert len(set(s3.page_table[1, :4].tolist() + s3.page_table[2, :1].tolist())) == 5


def test_cache_reserve():
    c = PagedKVCache(1, 5, 4, 1, 8, max_seqs=2, max_len=16, dtype=torch.float32, device="cpu")
    c.reserve([9, 2])
    assert c.free_pages == 1 and c.lens == [0, 0]
    s = c.step([1, 1])
    assert c.free_pages == 1 and (s.page_table[0, :3] >= 0).all() and s.kv_lens.tolist() == [1, 1]
    c.step([8, 0])                                          # within what is reserved
    assert c.free_pages == 1
    with pytest.raises(RuntimeError, match="out of pages"):
        c.reserve([16, 16])
    with pytest.raises(ValueError, match="max_len"):
        c.reserve([17, 0])
    c.release(0)
    assert c.free_pages == 4 and c.lens == [0, 1]


def test_decoder_options():
    from continuum_attention_b200.decoder import ContinuumDecoderConfig
    small = dict(d_model=64, n_heads=2)
    assert not ContinuumDecoderConfig(**small).rope_general
    assert ContinuumDecoderConfig(rope_dim=16, **small).rope_general
    table = ContinuumDecoderConfig(rope_dim=16, rope_scaling="linear", rope_factor=2.0, block_size=10, **small).rope_table(
        torch.device("cpu"))
    assert table.rotary_dim == 16 and table.positions == 10
    for bad in (dict(rope_layout="x"), dict(rope_dim=15), dict(rope_dim=34), dict(rope_scaling="y"),
                dict(rope_scaling="yarn", rope_factor=2.0), dict(rope_scaling="linear", rope_factor=0.5)):
        with pytest.raises(ValueError):
            ContinuumDecoderConfig(**small, **bad)
