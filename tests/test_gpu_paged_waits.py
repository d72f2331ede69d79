"""Paged attention whose device-side waits run out: the call ends, says so, and writes nothing but its own
buffers, whatever its workspace held before; the next call is right again."""
import pytest
import torch

from continuum_attention_b200 import _native, continuum_attention_paged, paged_workspace_bytes
from paged_testlib import DTYPES, arguments, make_case

pytestmark = pytest.mark.gpu

GUARD = 1 << 20

# heads, kv_heads, dim, sequences: which kernels of the 16-bit types answer; long enough that workers have more tiles
# than their shared memory holds
FORMS = {
    "decode": (8, 8, 64, [(1, 20000), (1, 700)] + [(1, 33)] * 20),
    "decode_wide": (4, 4, 128, [(1, 9000)] * 5),
    "decode_16_rows": (16, 1, 64, [(1, 20000)] * 9),
    "short_chunks": (4, 4, 64, [(40, 30000), (17, 17), (64, 900)]),
    "short_chunks_wide": (2, 2, 128, [(33, 30000), (17, 17), (64, 900)]),
    "tcgen05": (4, 4, 64, [(700, 5000), (128, 128), (129, 4000)]),
    "tcgen05_wide": (4, 2, 128, [(300, 9000), (90, 90)]),
    "tcgen05_units_of_one_tile": (64, 64, 64, [(100, 100)] + [(20, 20)] * 30),
    "mixed": (6, 2, 64, [(1, 3000), (200, 16000), (30, 500), (0, 10), (2, 1)]),
}


def guarded(nbytes):
    """(whole buffer, its middle): every byte 0x7f, which read as a record of pieces is two billion of them."""
    whole = torch.full((nbytes + 2 * GUARD,), 0x7F, dtype=torch.uint8, device="cuda")
    return whole, whole[GUARD:GUARD + nbytes]


def untouched(whole):
    return bool((whole[:GUARD] == 0x7F).all()) and bool((whole[-GUARD:] == 0x7F).all())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("form", FORMS)
def test_waits_that_run_out(dtype, form):
    H, G, D, seqs = FORMS[form]
    c = make_case(dtype, H, G, D, 16, seqs, seed=3)
    args, n = arguments(c), c["max_q_len"]
    want = continuum_attention_paged(*args, max_q_len=n)
    lib = _native.lib()
    assert lib.ca_device_status(1) == 0
    try:
        for limit_us in (0, 1, 0, 20, 0):
            assert lib.ca_selftest_paged_wait_limit(limit_us) == 0
            ws_all, ws = guarded(paged_workspace_bytes(len(seqs), n, H, G, D, DTYPES[dtype]))
            out_all, out = guarded(want.numel() * want.element_size())
            out = out.view(DTYPES[dtype]).view(want.shape)
            continuum_attention_paged(*args, max_q_len=n, out=out, workspace=ws)
            status = lib.ca_device_status(1)
            assert status == 5 if limit_us == 0 else status in (0, 5)
            assert untouched(ws_all) and untouched(out_all)
            if status == 0:
                assert torch.equal(out, want)
    finally:
        lib.ca_selftest_paged_wait_limit(-1)
    assert torch.equal(continuum_attention_paged(*args, max_q_len=n), want)
    assert lib.ca_device_status(0) == 0


def test_the_limits_range():
    lib = _native.lib()
    assert lib.ca_selftest_paged_wait_limit(10000001) == 1
    assert "limit_us" in lib.ca_last_error().decode()
    assert lib.ca_selftest_paged_wait_limit(-1) == 0
