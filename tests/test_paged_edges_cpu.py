"""Edges of the paged and rotary operators and of the decoder's answering that need no GPU."""
import ctypes

import pytest
import torch

from continuum_attention_b200 import RotaryTable, _native
from continuum_attention_b200.rope import cos_sin_table
from continuum_attention_b200.rotary import rotary_table

FAKE = ctypes.c_void_p(256)


@pytest.mark.parametrize("page", [1 << 31, 1 << 32, (1 << 32) + 16])
def test_page_sizes_beyond_32_bits(page):
    """A table without columns, so that no product with the page size is too large."""
    lib = _native.lib()
    assert lib.ca_paged_forward(FAKE, 256, 64, FAKE, FAKE, 2048, 1024, 64, None, 0, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 40,
                                4, 2, 2, 4, 2, 64, 16, page, 0, 1, None) == 2
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
