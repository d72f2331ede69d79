"""Paged attention and the append at the ends of what their documentation allows."""
import pytest
import torch

from continuum_attention_b200 import RotaryTable, _native, continuum_attention_paged, rotary_append
from paged_testlib import DTYPES, WEIGHT_ERROR, make_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("news", [[1], [20], [100], [1, 100, 3], [5] * 40])
def test_more_tiles_than_a_call_takes(dtype, news):
    """2^30 keys (one slot, read again and again) for 256 key heads are 2^32 tiles or more: no row is left as it was,
    rows behind the last sequence are, and the next call is right."""
    H, D, L = 256, 8, 2 ** 30
    S, N = len(news), sum(news)
    k = torch.ones(1, H, 1, D, device="cuda", dtype=DTYPES[dtype]).expand(1, H, L, D)
    q = torch.ones(N + 2, H, D, device="cuda", dtype=DTYPES[dtype])
    starts = torch.tensor([sum(news[:s]) for s in range(S + 1)], dtype=torch.int32, device="cuda")
    table = torch.zeros(S, 1, dtype=torch.int32, device="cuda")
    lens = torch.full((S,), L, dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 2.0)
    gain = torch.zeros(H, device="cuda")
    lib = _native.lib()
    assert lib.ca_device_status(1) == 0
    continuum_attention_paged(q, k, k, table, lens, starts, gain, max_q_len=max(news), out=out)
    assert lib.ca_device_status(1) == 1
    assert torch.isnan(out[:N]).all() and (out[N:] == 2.0).all()
    lens.fill_(max(news))
    continuum_attention_paged(q, k, k, table, lens, starts, gain, max_q_len=max(news), out=out)
    assert lib.ca_device_status(1) == 0
    # a mean of ones: half a step, and the weights' error in numerator and normaliser
    assert ((out[:N].double() - 1).abs() <= torch.finfo(out.dtype).eps / 2 + 2 * WEIGHT_ERROR[dtype]).all()
    assert (out[N:] == 2.0).all()


@pytest.mark.parametrize("starts", [[0, 2, 3, 5], [0, 2, 3, 2 ** 31 - 1], [0, 2, 4, 9], [0, 2, 9, 4], [-1, 2, 3, 4]])
def test_append_of_rows_outside_the_buffer(starts):
    """Sequences that claim rows which the buffer does not have: recorded, and nothing of theirs is written."""
    c = make_case("bf16", 2, 1, 64, 16, [(2, 20), (1, 40), (1, 8)], seed=3)
    table = RotaryTable(64, 64)
    qkv = torch.randn(4, 4 * 64, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).bfloat16()
    lib = _native.lib()
    lib.ca_device_status(1)

    def go(ends):
        k, v = c["k_cache"].clone(), c["v_cache"].clone()
        out = torch.full((4, 2, 64), 3.0, device="cuda", dtype=torch.bfloat16)
        rotary_append(qkv, k, v, c["page_table"], c["kv_lens"], torch.tensor(ends, dtype=torch.int32, device="cuda"),
                      table, heads=2, out=out)
        return out, k, v

    good = go([0, 2, 3, 4])
    assert lib.ca_device_status(1) == 0
    got = go(starts)
    assert lib.ca_device_status(1) == 1
    pages = c["page_table"].cpu()
    for s, (n, L) in enumerate(c["seqs"]):
        inside = 0 <= starts[s] <= starts[s + 1] <= 4
        if inside and [starts[s], starts[s + 1]] != [[0, 2, 3, 4][s], [0, 2, 3, 4][s + 1]]:
            continue                                     # (in range, of another number of rows)
        rows = slice([0, 2, 3][s], [2, 3, 4][s])
        if inside:
            assert torch.equal(got[0][rows], good[0][rows])
        elif not any(0 <= starts[u] <= starts[u + 1] <= 4 and starts[u] <= r < starts[u + 1]
                     for u in range(3) for r in range(rows.start, rows.stop)):
            assert (got[0][rows] == 3.0).all()
        for j in range(L - n, L):
            at = (int(pages[s, j // 16]), 0, j % 16)
            for new, right, old in zip(got[1:], good[1:], (c["k_cache"], c["v_cache"])):
                want = right if inside else old
                assert torch.equal(torch.nan_to_num(new[at], 7.0), torch.nan_to_num(want[at], 7.0))
