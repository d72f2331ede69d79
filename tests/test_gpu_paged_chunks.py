"""Chunks of more than 64 rows a head over a paged cache (units of 128 rows) against the float64 oracle: what
``test_gpu_paged.py`` asks of short ones, and units that end or start inside a tile, a page or a batch."""
import math
import random
import threading

import pytest
import torch

from continuum_attention_b200 import _native, continuum_attention_paged
from paged_testlib import DTYPES, arguments, check, exact, make_case

pytestmark = pytest.mark.gpu


def run(case, **kw):
    return continuum_attention_paged(*arguments(case), max_q_len=kw.pop("max_q_len", case["max_q_len"]), **kw)


def run_and_check(dtype, case):
    out = run(case)
    check(dtype, out, *exact(case), sum(n for n, _ in case["seqs"]))
    assert _native.lib().ca_device_status(0) == 0
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(2, 2, 64, 16), (8, 2, 64, 64), (6, 2, 56, 7), (5, 1, 8, 1),
                                                     (3, 3, 64, 128), (64, 1, 16, 32), (128, 1, 64, 16),
                                                     (2, 2, 128, 16), (6, 2, 80, 24), (4, 1, 120, 1)])
def test_shapes(dtype, heads, kv_heads, dim, page):
    case = make_case(dtype, heads, kv_heads, dim, page, [(70, 70), (129, 191), (1, 40), (127, 500)], seed=dim + page)
    run_and_check(dtype, case)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("seqs", [
    [(65, 65)] * 9,                                    # short units, two after one another in a worker
    [(80, L) for L in (0, 1, 2, 31, 32, 33, 63, 79)],   # rows before the first key, units of one tile
    [(300, 4096)],
    [(200, 200 + L) for L in (0, 1, 31, 32, 33, 95, 96, 97)],
])
@pytest.mark.parametrize("dim", [64, 128])
def test_lengths(dtype, dim, seqs):
    run_and_check(dtype, make_case(dtype, 2, 1, dim, 16, seqs, seed=len(seqs)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("seed,dims", [(s, (8, 24, 40, 64)) for s in range(6)] + [(s, (72, 80, 104, 128)) for s in range(6, 12)])
def test_random_batches(dtype, seed, dims):
    r = random.Random(seed)
    kv_heads = r.choice([1, 2, 3])
    heads = kv_heads * r.choice([1, 2, 3, 4, 7])
    dim, page = r.choice(dims), r.choice([1, 5, 16, 24, 64])
    seqs = []
    for _ in range(r.randint(1, 12)):
        n = r.choice([0, 1, 1, 3, r.randint(1, 40), r.randint(65, 260)])
        seqs.append((n, max(0, n + r.choice([-3, 0, 0, 1, 17, r.randint(0, 600)]))))
    seqs.append((r.randint(65, 200), 400))
    run_and_check(dtype, make_case(dtype, heads, kv_heads, dim, page, seqs, seed=seed, tail=r.choice([0, 3])))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (6, 2, 64), (4, 2, 96), (6, 2, 128)])
def test_neighbours_and_a_tail_do_not_reach_a_sequence(dtype, heads, kv_heads, dim):
    """A unit's rows go on behind its sequence's last in the buffer: what stands there stays out of the answers,
    and the rows behind the last sequence keep what they held."""
    case = make_case(dtype, heads, kv_heads, dim, 16, [(70, 100), (75, 90), (0, 5), (90, 90)], seed=11, tail=40)
    case["q"][70:145] = float("nan")
    case["q"][235:] = float("inf")
    out = torch.full_like(case["q"], 7.0)
    assert run(case, out=out) is out
    assert (out[235:] == 7.0).all()
    assert torch.isnan(out[70:145]).all()
    case["q"][70:145] = 0.0
    want, mag = exact(case)
    keep = torch.ones(235, dtype=torch.bool)
    keep[70:145] = False
    check(dtype, out[:235][keep], want[:235][keep], mag[:235][keep], 160)
    assert _native.lib().ca_device_status(0) == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 40, 128, 88])
def test_strided_cache_and_queries(dtype, dim):
    case = make_case(dtype, 4, 2, dim, 16, [(5, 77), (100, 130), (70, 70)], seed=5, cache_layout="psgd")
    want = exact(case)
    N, H, D = case["q"].shape
    wide = torch.full((N, 3 * H * D), float("nan"), dtype=case["q"].dtype, device="cuda")
    wide[:, :H * D] = case["q"].reshape(N, H * D)
    case["q"] = wide[:, :H * D].unflatten(1, (H, D))       # the query part of a projection row
    out = run(case)
    check(dtype, out, *want, N)
    case["q"] = case["q"].permute(1, 0, 2).contiguous().permute(1, 0, 2)     # head-major
    assert torch.equal(run(case), out)
    # a cache whose slots lie in wider rows, and pages with gaps between them
    pages, G, page, _ = case["k_cache"].shape
    for n in ("k_cache", "v_cache"):
        held = torch.full((pages, page + 1, G, D + 16), float("nan"), dtype=wide.dtype, device="cuda")
        view = held[:, :page, :, :D].permute(0, 2, 1, 3)
        view.copy_(case[n])
        case[n] = view
    assert torch.equal(run(case), out)
    # one head's keys and queries for all
    shared = {n: case[n][:, :1].expand(-1, G, -1, -1) for n in ("k_cache", "v_cache")}
    alone = {n: t.contiguous() for n, t in shared.items()}
    assert shared["k_cache"].stride(1) == 0
    same_q = case["q"][:, :1].expand(-1, H, -1)
    assert torch.equal(run({**case, **shared, "q": same_q}), run({**case, **alone, "q": same_q.contiguous()}))


def steepness(case, s):
    """Sum over the segments of the larger end's exponential, over the mass, for every row and head of sequence s."""
    n, L = case["seqs"][s]
    at = sum(m for m, _ in case["seqs"][:s])
    q, k = case["q"][at:at + n].double().cpu(), case["keys"][s].double()
    H, D = q.shape[1:]
    kk = k.permute(1, 0, 2).repeat_interleave(H // k.shape[1], 0)
    x = q.permute(1, 0, 2) @ kk.transpose(1, 2) * (case["log_gain"].double().cpu().exp() / math.sqrt(D))[:, None, None]
    sees = torch.arange(L)[None, :] <= torch.arange(L - n, L)[:, None]
    x = x.masked_fill(~sees, float("-inf"))
    x = x - x.amax(2, keepdim=True)
    top = torch.maximum(x[..., 1:], x[..., :-1]).exp() * sees[:, 1:]
    d = torch.where(sees[:, 1:], (x[..., 1:] - x[..., :-1]).abs(), torch.ones(()).double())
    mass = (top * -torch.expm1(-d) / d.clamp_min(1e-12)).sum(2) + 0.5 * x[..., 0].exp()
    return (top.sum(2) / mass).transpose(0, 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("qk_mag", [0.0, 1e-3, 6.0])
def test_flat_and_steep_scores(dtype, qk_mag):
    """Equal scores (every segment at the series' centre) and scores hundreds apart: the maximum moves often."""
    case = make_case(dtype, 4, 4, 64, 16, [(1, 200), (140, 400)], seed=6, qk_mag=qk_mag, gain=0.0)
    out = run(case)
    want, mag = exact(case)
    if qk_mag <= 1:
        check(dtype, out, want, mag, out.shape[0])
        return
    # scores up to |s| ~ 36 * 8 * 4 = 1152 in 32 bits are off by 1152 * 2^-23 + 64 products' sums, below 3e-4:
    # so are the weights
    got = out.double().cpu()
    bound = want.abs() * torch.finfo(DTYPES[dtype]).eps / 2 * 1.001 + 2 * (3e-4 + 4e-5) * mag + 2.0 ** -25
    # A steep segment of ends e >= e' at distance |d| > 1: M0 = (e - e') / d and M1 = (e - M0) / d carry the
    # reciprocal's 2^-23 and two roundings of 2^-24, 2^-22 of themselves, which are below e.  The weight
    # M0 - M1 of the segment's other key is only e / d^2 and takes e 2^-22 of it as an absolute error
    # (formed as M0 = e - d M1, the mass would as well).  Summed, over the mass: steepness * 2^-22, times
    # that key's |v| and, for the mass, |y|.
    top_v = max(v.abs().max().item() for v in case["values"])
    steep = torch.cat([steepness(case, s) for s in range(2)])
    bound += steep[..., None] * 2.0 ** -22 * 2 * top_v
    assert ((got - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_offsets_beyond_32_bits(dtype):
    """The used pages lie behind 2^31 elements of the cache."""
    dim, page, kv_heads = 64, 64, 2
    far = 2 ** 31 // (dim * page * kv_heads) + 1
    case = make_case(dtype, 2, kv_heads, dim, page, [(1, 150), (90, 200)], seed=8, far=far)
    assert case["k_cache"].numel() > 2 ** 31
    run_and_check(dtype, case)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_bad_lengths_and_pages_are_refused_by_the_kernel(dtype, dim):
    lib = _native.lib()
    lib.ca_device_status(1)
    base = make_case(dtype, 4, 2, dim, 16, [(1, 40), (90, 120), (2, 3), (70, 100)], seed=12)
    want, mag = exact(base)
    rows = slice(1, 91)
    for what in ("page", "page_neg", "len", "len_neg"):
        case = dict(base)
        case["page_table"], case["kv_lens"] = base["page_table"].clone(), base["kv_lens"].clone()
        if what == "page":
            case["page_table"][1, 2] = base["k_cache"].shape[0]
        elif what == "page_neg":
            case["page_table"][1, 0] = -1
        elif what == "len":
            case["kv_lens"][1] = base["page_table"].shape[1] * 16 + 1
        else:
            case["kv_lens"][1] = -1
        out = run(case)
        assert lib.ca_device_status(1) == 1, what
        # page 2 holds keys 32 .. 47: the rows at positions 30 and 31 do not see it
        assert torch.isnan(out[3:91] if what == "page" else out[rows]).all(), what
        keep = torch.ones(out.shape[0], dtype=torch.bool)
        keep[rows] = False
        check(dtype, out[keep], want[keep], mag[keep], int(keep.sum()))
    assert lib.ca_device_status(0) == 0


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_wrong_max_q_len(dtype):
    """max_q_len chooses the kernels; another value than the longest sequence's costs time only."""
    case = make_case(dtype, 2, 2, 64, 16, [(1, 40), (100, 150), (20, 30)], seed=13)
    want = exact(case)
    for wrong in (1, 9, 40, 70, 10 ** 6):
        check(dtype, run(case, max_q_len=wrong), *want, 121)
    assert _native.lib().ca_device_status(0) == 0


def test_graph_replays_follow_the_lengths():
    """A step captured once answers for other lengths when replayed; two graphs share a pool, and an eager call
    between them uses a workspace of its own."""
    def batch(seqs, seed):
        return make_case("bf16", 4, 2, 64, 16, seqs, seed=seed)
    case, other = batch([(80, 100), (1, 37), (90, 260)], 14), batch([(3, 16), (168, 250), (0, 1)], 15)
    P = max(c["k_cache"].shape[0] for c in (case, other))
    W = max(c["page_table"].shape[1] for c in (case, other))
    buf = {n: torch.zeros((P, *case["k_cache"].shape[1:]), dtype=torch.bfloat16, device="cuda")
           for n in ("k_cache", "v_cache")}
    buf.update({n: case[n].clone() for n in ("q", "log_gain", "kv_lens", "q_starts")},
               page_table=torch.zeros(3, W, dtype=torch.int32, device="cuda"))

    def load(c):
        for n in ("k_cache", "v_cache"):
            buf[n][:c[n].shape[0]] = c[n]
        for n in ("q", "log_gain", "kv_lens", "q_starts"):
            buf[n].copy_(c[n])
        buf["page_table"][:, :c["page_table"].shape[1]] = c["page_table"]

    load(case)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run({**buf, "max_q_len": 171})
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(run({**buf, "max_q_len": 171}))
        graphs.append(g)
    for c in (case, other, case):
        load(c)
        want = exact(c)
        for g, o in zip(graphs, outs):
            g.replay()
            eager = run({**buf, "max_q_len": 171})
            check("bf16", o, *want, 171)
            assert torch.equal(o, eager)
    assert _native.lib().ca_device_status(0) == 0


def test_two_streams_at_once():
    cases = [make_case("f16", 4, 2, 64, 16, [(150, 1000), (1, 40 + i), (70, 90)], seed=20 + i) for i in range(2)]
    want = [exact(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                outs[i].append(run(c))
    torch.cuda.synchronize()
    for got, w in zip(outs, want):
        for o in got:
            check("f16", o, *w, 221)
            assert torch.equal(o, got[0])               # same bits every time


def test_from_a_thread_that_never_called_cuda():
    """The same kernels, so the same bits, from a thread without a context of its own."""
    lib = _native.lib()
    case = make_case("bf16", 4, 2, 64, 16, [(150, 300), (1, 40)], seed=31)
    want = run(case)
    got = torch.zeros_like(want)
    q, kc, vc, table, lens, starts, gain = arguments(case)
    n = lib.ca_paged_workspace_size(2, 150, 4, 2, 64, 1)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    args = (q.data_ptr(), q.stride(0), q.stride(1), kc.data_ptr(), vc.data_ptr(), *kc.stride()[:3], table.data_ptr(),
            table.stride(0), lens.data_ptr(), starts.data_ptr(), gain.data_ptr(), got.data_ptr(), ws.data_ptr(), n,
            q.shape[0], 2, 150, 4, 2, 64, kc.shape[0], 16, table.shape[1], 1, 0)
    torch.cuda.synchronize()
    status = []
    t = threading.Thread(target=lambda: status.append(lib.ca_paged_forward(*args)))
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert status == [0]
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_short_sequence_alone_in_a_long_buffer(dtype):
    """max_q_len and the buffer say 100 rows, the sequence has three."""
    case = make_case(dtype, 4, 2, 64, 16, [(3, 50)], seed=32, tail=97)
    out = torch.full_like(case["q"], 7.0)
    run(case, max_q_len=100, out=out)
    check(dtype, out, *exact(case), 3)
    assert (out[3:] == 7.0).all()
    assert _native.lib().ca_device_status(0) == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_as_many_sequences_as_a_call_takes(dtype):
    seqs = [(1, 1 + s % 40) for s in range(1500)] + [(0, 3)] * 500 + [(2, 5)] * 46 + [(70, 100), (80, 80)]
    assert len(seqs) == 2048
    run_and_check(dtype, make_case(dtype, 2, 2, 16, 16, seqs, seed=33))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 20, 100])
def test_a_cache_without_pages(dtype, n):
    """No keys anywhere: every row is zero."""
    q = torch.randn(n, 4, 64, device="cuda").to(DTYPES[dtype])
    kc = torch.empty(0, 2, 16, 64, dtype=q.dtype, device="cuda")
    ints = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0], [0, n])]
    table = torch.empty(1, 0, dtype=torch.int32, device="cuda")
    out = continuum_attention_paged(q, kc, kc.clone(), table, *ints, torch.zeros(4, device="cuda"), max_q_len=n)
    assert (out == 0).all()
    assert _native.lib().ca_device_status(0) == 0
