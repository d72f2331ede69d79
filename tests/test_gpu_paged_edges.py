"""Paged attention and the append at the ends of what their documentation allows."""
import pytest
import torch

from continuum_attention_b200 import _native, continuum_attention_paged
from paged_testlib import DTYPES, WEIGHT_ERROR

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
