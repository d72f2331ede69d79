"""Edges of the paged and rotary operators and of the decoder's answering that need no GPU."""
import ctypes
import math

import pytest
import torch

from continuum_attention_b200 import (RotaryTable, _native, continuum_attention_paged, rotary, rotary_append,
                                      rotary_qkv)
from continuum_attention_b200.decoder import ContinuumDecoderConfig, ContinuumDecoderLM
from continuum_attention_b200.rope import cos_sin_table
from continuum_attention_b200.rotary import rotary_frequencies, rotary_table
from paged_testlib import arguments, make_case

FAKE = ctypes.c_void_p(256)


@pytest.mark.parametrize("page", [1 << 31, 1 << 32, (1 << 32) + 16])
def test_page_sizes_beyond_32_bits(page):
    """A table without columns, so that no product with the page size is too large."""
    lib = _native.lib()
    assert lib.ca_paged_forward(FAKE, 256, 64, FAKE, FAKE, 2048, 1024, 64, None, 0, FAKE, FAKE, FAKE, FAKE, FAKE,
                                1 << 40, 4, 2, 2, 4, 2, 64, 16, page, 0, 1, None) == 2
    assert "page_size" in lib.ca_last_error().decode()
    assert lib.ca_rotary_append(FAKE, 512, FAKE, FAKE, FAKE, FAKE, 2048, 1024, 64, None, 0, FAKE, FAKE, 4, 2, 4, 2, 64,
                                64, 128, 16, page, 0, 0, 1, None) == 2
    assert "page_size" in lib.ca_last_error().decode()


class _Saves(torch.autograd.Function):
    """What the rotary operators do with their table: keep it for the gradient."""

    @staticmethod
    def forward(ctx, x, table):
        ctx.save_for_backward(table)
        return x * 2

    @staticmethod
    def backward(ctx, g):
        return g * 2 + ctx.saved_tensors[0].sum() * 0, None


@pytest.mark.parametrize("make", [
    lambda: rotary_table(8, 11, 4321.0, "linear", 2.0, None, "cpu").cos_sin,
    lambda: cos_sin_table(13, 8, 4321.0, "cpu"),
    lambda: RotaryTable(8, 7, device="cpu").cos_sin,
])
def test_tables_first_made_in_inference_mode_serve_training(make):
    with torch.inference_mode():
        make()
        first = make()
    assert not first.is_inference()
    x = torch.ones(3, requires_grad=True)
    for table in (first, make()):
        _Saves.apply(x, table).sum().backward()
    assert x.grad.tolist() == [4.0] * 3


# the ends of the ramp by hand: 20 and 33, 45 and 70, 4 and 8, 22 and 35, 8 and 21
@pytest.mark.parametrize("R,original,factor,last", [
    (64, 65536, 4.0, 1 - 11 / 13 * 3 / 4), (128, 131072, 4.0, 1 - 18 / 25 * 3 / 4), (16, 32768, 4.0, 1 - 3 / 4 * 3 / 4),
    (64, 131072, 8.0, 1 - 9 / 13 * 7 / 8), (64, 2048, 8.0, 1 / 8)])
def test_yarn_where_the_slowest_pair_turns_more_than_once(R, original, factor, last):
    """What is left of each pair's frequency, from the ramp's two ends: the pairs (as real numbers) that turn 32
    times and once within the original length, to whole pairs outwards, in 0 .. R - 1."""
    plain, _ = rotary_frequencies(R)
    freq, _ = rotary_frequencies(R, scaling="yarn", factor=factor, original_positions=original)
    kept = (freq / plain).tolist()
    # 10000^(-2 p / R) original / (2 pi) = turns
    ends = [R / 2 * math.log10(original / (2 * math.pi * turns)) / 4 for turns in (32, 1)]
    low, high = max(math.floor(ends[0]), 0), min(math.ceil(ends[1]), R - 1)
    for p, k in enumerate(kept):
        t = min(max((p - low) / (high - low), 0.0), 1.0)
        assert k == pytest.approx(1 - t + t / factor, rel=1e-12)
    assert kept[-1] == pytest.approx(last, rel=1e-9)


def small_decoder(**kw):
    cfg = ContinuumDecoderConfig(vocab_size=50, block_size=32, d_model=64, n_heads=2, n_layers=2)
    return ContinuumDecoderLM(cfg, **kw)


def test_a_model_with_another_attention_does_not_answer_with_the_default():
    m = small_decoder(attention_fn=lambda q, k, v, gain, tile: v)
    cache = m.make_cache(1)
    with pytest.raises(ValueError, match="attention_fn"):
        m.forward_paged(torch.tensor([1, 2]), cache, cache.step([2]))
    with pytest.raises(ValueError, match="attention_fn"):
        m.generate([[1, 2]], 2)


def test_serving_operators_refuse_gradients():
    c = make_case("bf16", 4, 2, 64, 16, [(1, 20), (2, 5)], device="cpu")
    args = arguments(c)
    qkv, table = torch.zeros(3, 8 * 64, dtype=torch.bfloat16), RotaryTable(64, 32, device="cpu")
    for i in (0, 1, 2):
        asks = [t.detach().requires_grad_() if j == i else t for j, t in enumerate(args)]
        with pytest.raises(RuntimeError, match="no backward"):
            continuum_attention_paged(*asks, max_q_len=2)
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):       # as far as the device
            continuum_attention_paged(*asks, max_q_len=2)
    for x, cache in [(qkv.detach().requires_grad_(), args[1:6]),
                     (qkv, [args[1].detach().requires_grad_(), *args[2:6]]),
                     (qkv, [args[1], args[2].detach().requires_grad_(), *args[3:6]])]:
        with pytest.raises(RuntimeError, match="no backward"):
            rotary_append(x, *cache, table, heads=4)
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
            rotary_append(x, *cache, table, heads=4)
    with torch.autograd.forward_ad.dual_level():
        for i in (0, 1, 2, 6):
            dual = torch.autograd.forward_ad.make_dual(args[i], torch.ones_like(args[i]))
            with torch.no_grad(), pytest.raises(RuntimeError, match="no forward-mode"):
                continuum_attention_paged(*args[:i], dual, *args[i + 1:], max_q_len=2)
        dual = torch.autograd.forward_ad.make_dual(qkv, torch.ones_like(qkv))
        with pytest.raises(RuntimeError, match="no forward-mode"):
            rotary_append(dual, *args[1:6], table, heads=4)
        with pytest.raises(RuntimeError, match="CUDA"):                          # plain inputs inside a level
            continuum_attention_paged(*args, max_q_len=2)


def test_rotary_qkv_refuses_a_table_that_asks_for_a_gradient():
    qkv = torch.zeros(1, 3, 8 * 64)
    table = RotaryTable.from_cos_sin(RotaryTable(64, 32, device="cpu").cos_sin.requires_grad_())
    with pytest.raises(RuntimeError, match="table is a constant"):
        rotary_qkv(qkv, 4, table, kv_heads=2)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):       # as far as the device
        rotary_qkv(qkv, 4, table, kv_heads=2)


def test_prompts_in_every_form():
    """A tensor of prompts is one prompt a row; a prompt of another shape and ids that the embedding does not have (a
    read behind it) are refused before anything runs."""
    m = small_decoder()
    for bad, match in (([[1, 50]], "0 .. 49"), ([[1], [-1]], "0 .. 49"), (torch.full((2, 3), 50), "0 .. 49"),
                       ([torch.tensor([[1, 2]])], "1-D"), (torch.tensor([1, 2]), "1-D"), ([[]], "one token"),
                       (torch.zeros(0, 3, dtype=torch.long), "one token"), ([[1.5]], "whole"),
                       (torch.zeros(2, 31), "whole")):
        with pytest.raises(ValueError, match=match):
            m.generate(bad, 2)
    for good in (torch.zeros(2, 3, dtype=torch.long), [(1, 2), [3]], [torch.tensor([49]), [0, 1]],
                 torch.zeros(2, 3, dtype=torch.uint8).numpy()):
        with pytest.raises(RuntimeError, match="CUDA"):                        # as far as the device
            m.generate(good, 2)


def test_temperature_that_is_no_number():
    with pytest.raises(ValueError, match="temperature"):
        small_decoder().generate([[1]], 2, temperature=float("nan"))


def test_a_cache_of_no_pages_is_refused():
    """It is not the default number of pages."""
    with pytest.raises(ValueError, match="pages"):
        small_decoder().make_cache(2, pages=0)
    assert small_decoder().make_cache(2, page_size=16).free_pages == 4


def test_tables_of_the_current_device_are_of_that_device(monkeypatch):
    """"cuda" without a number is another device after a switch: not the table that was made for the first."""
    made = []

    class Fake:
        def __init__(self, *a, device, **kw):
            made.append(torch.device(device))
            self.cos_sin = torch.zeros(1, 1, 2)

    monkeypatch.setattr(rotary, "RotaryTable", Fake)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(rotary, "_capturing", lambda device: False, raising=False)
    for current in (0, 1, 0):
        monkeypatch.setattr(torch.cuda, "current_device", lambda: current)
        for device in ("cuda", torch.device("cuda"), f"cuda:{current}"):
            rotary.rotary_table(8, 9, 1234.0, None, 1.0, None, device)
    assert made == [torch.device("cuda", 0), torch.device("cuda", 1)]


def test_as_many_rows_as_32_bits_index():
    """Rows are counted in whole tiles of 128: a call of nearly 2^31 would pass the index."""
    lib = _native.lib()
    for rows, heads in ((2 ** 31 - 2, 1), (2 ** 31 - 512, 1), ((2 ** 31 - 1) // 3, 3)):
        assert lib.ca_paged_forward(FAKE, 8, 8, FAKE, FAKE, 8, 8, 8, FAKE, 8, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 40, rows, 1,
                                    1, heads, heads, 8, 16, 16, 8, 1, None) == 2
        assert "2^31-1024" in lib.ca_last_error().decode()


def test_a_table_that_starts_anywhere():
    """The kernels read tables from 16-byte borders on: a slice that starts between two is copied."""
    full = RotaryTable(6, 40, device="cpu").cos_sin
    for first in range(4):
        table = RotaryTable.from_cos_sin(full[first:])
        assert table.cos_sin.data_ptr() % 16 == 0 and torch.equal(table.cos_sin, full[first:])
    assert RotaryTable.from_cos_sin(full).cos_sin.data_ptr() == full.data_ptr()
