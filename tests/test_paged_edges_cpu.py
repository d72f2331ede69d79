"""Edges of the paged and rotary operators and of the decoder's answering that need no GPU."""
import ctypes

import pytest

from continuum_attention_b200 import _native

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
