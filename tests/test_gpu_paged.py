"""Continuum Attention over a paged cache against the float64 oracle: lengths from none to long, odd
pages, shared heads, strided buffers, stale slots, empty rows, bad pages, streams and graphs."""
import pytest
import torch

from continuum_attention_b200 import _native, continuum_attention, continuum_attention_paged, paged_workspace_bytes
from paged_testlib import DTYPES, arguments, check, exact, make_case

pytestmark = pytest.mark.gpu


def run(case, **kw):
    return continuum_attention_paged(*arguments(case), max_q_len=kw.pop("max_q_len", case["max_q_len"]), **kw)


def run_and_check(dtype, case):
    out = run(case)
    rows = sum(n for n, _ in case["seqs"])
    check(dtype, out, *exact(case), rows)
    assert _native.lib().ca_device_status(0) == 0
    return out


# decoding: one new token, lengths around every border of tiles (64 keys), pages and splits
DECODE_LENS = [1, 2, 3, 15, 16, 17, 31, 32, 63, 64, 65, 127, 128, 129, 191, 192, 193, 700]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 4, 64, 16), (8, 2, 64, 64), (3, 1, 128, 24), (5, 5, 8, 1),
                                                     (2, 1, 80, 7), (16, 1, 64, 128), (32, 1, 32, 16)])
def test_decode_lengths(dtype, heads, kv_heads, dim, page):
    case = make_case(dtype, heads, kv_heads, dim, page, [(1, L) for L in DECODE_LENS], seed=dim + page)
    run_and_check(dtype, case)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(2, 2, 64, 16), (6, 2, 64, 64), (4, 1, 128, 32), (3, 3, 40, 5)])
@pytest.mark.parametrize("n", [2, 5, 8, 9, 16, 17, 33, 63, 64, 65, 130])
def test_chunks(dtype, heads, kv_heads, dim, page, n):
    seqs = [(n, n), (n, n + 1), (n, n + 63), (n, n + 64), (n, n + 200)]
    case = make_case(dtype, heads, kv_heads, dim, page, seqs, seed=n)
    run_and_check(dtype, case)


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_context_of_one_sequence(dtype):
    case = make_case(dtype, 2, 1, 64, 16, [(1, 9001)], seed=3)
    run_and_check(dtype, case)
    case = make_case(dtype, 2, 2, 64, 64, [(70, 5003)], seed=4)
    run_and_check(dtype, case)


@pytest.mark.parametrize("dtype", DTYPES)
def test_ragged_with_empty_rows_and_a_tail(dtype):
    seqs = [(0, 5), (3, 0), (9, 4), (1, 1), (0, 0), (40, 200), (1, 333), (2, 3), (18, 18), (0, 64)]
    case = make_case(dtype, 4, 2, 64, 16, seqs, seed=11, tail=6)
    rows = sum(n for n, _ in seqs)
    out = torch.full_like(case["q"], 7.0)
    assert run(case, out=out) is out
    want, mag = exact(case)
    check(dtype, out, want, mag, rows)
    assert (out[rows:] == 7.0).all()                      # rows behind the last sequence
    assert (out[0:3] == 0).all() and (out[3:8] == 0).all()   # no keys at all, and rows before the first key
    assert _native.lib().ca_device_status(0) == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_cache_and_queries(dtype):
    case = make_case(dtype, 4, 2, 64, 16, [(5, 77), (1, 130), (30, 31)], seed=5, cache_layout="psgd")
    want = exact(case)
    N, H, D = case["q"].shape
    wide = torch.full((N, 3 * H * D), float("nan"), dtype=case["q"].dtype, device="cuda")
    wide[:, :H * D] = case["q"].reshape(N, H * D)
    case["q"] = wide[:, :H * D].unflatten(1, (H, D))       # the query part of a projection row
    assert not case["q"].is_contiguous()
    out = run(case)
    check(dtype, out, *want, N)
    case["q"] = case["q"].permute(1, 0, 2).contiguous().permute(1, 0, 2)     # head-major
    assert torch.equal(run(case), out)
    odd = torch.empty(case["q"].numel() + 1, dtype=case["q"].dtype, device="cuda")[1:].view(N, H, D)
    odd.copy_(case["q"])                                    # not on 16 bytes: copied by the call
    case["q"] = odd
    assert torch.equal(run(case), out)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("qk_mag", [0.0, 1e-3, 6.0])
def test_flat_and_steep_scores(dtype, qk_mag):
    """Equal scores (every segment at the series' centre) and scores hundreds apart."""
    case = make_case(dtype, 4, 4, 64, 16, [(1, 200), (40, 100)], seed=6, qk_mag=qk_mag, gain=0.0)
    out = run(case)
    want, mag = exact(case)
    rows = out.shape[0]
    if qk_mag <= 1:
        check(dtype, out, want, mag, rows)
    else:
        # scores up to |s| ~ 36 * 8 * 4 = 1152 in 32 bits are off by 1152 * 2^-23 + 64 products' sums,
        # below 3e-4: so are the weights
        got = out.double().cpu()
        bound = want.abs() * torch.finfo(DTYPES[dtype]).eps / 2 * 1.001 + 2 * (3e-4 + 4e-5) * mag + 2.0 ** -25
        assert ((got - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_offsets_beyond_32_bits(dtype):
    """The used pages lie behind 2^31 elements of the cache."""
    dim, page, kv_heads = 64, 64, 2
    far = 2 ** 31 // (dim * page * kv_heads) + 1
    case = make_case(dtype, 4, kv_heads, dim, page, [(1, 150), (20, 70)], seed=8, far=far)
    assert case["k_cache"].numel() > 2 ** 31
    run_and_check(dtype, case)


@pytest.mark.parametrize("dtype", DTYPES)
def test_equals_the_whole_sequence_operator(dtype):
    """A prompt fed in pieces and then by single tokens gives the rows of one call over all of it."""
    B, H, T, D, page = 2, 4, 150, 64, 16
    g = torch.Generator().manual_seed(9)
    q, k, v = (torch.randn(B, H, T, D, generator=g).to("cuda", DTYPES[dtype]) for _ in range(3))
    lg = torch.rand(H, generator=g).cuda()
    with torch.no_grad():
        whole = continuum_attention(q, k, v, lg)
    pages = -(-T // page)
    table = torch.arange(B * pages, dtype=torch.int32, device="cuda").view(B, pages)
    kc, vc = (torch.zeros(B * pages, H, page, D, dtype=q.dtype, device="cuda") for _ in range(2))
    for b in range(B):
        for j in range(pages):
            m = min(page, T - j * page)
            kc[b * pages + j, :, :m] = k[b, :, j * page:j * page + m]
            vc[b * pages + j, :, :m] = v[b, :, j * page:j * page + m]
    done, outs = 0, []
    for n in (1, 70, 33, 1, 1, 44):
        rows = q[:, :, done:done + n].permute(0, 2, 1, 3).reshape(B * n, H, D)
        done += n
        o = continuum_attention_paged(rows, kc, vc, table, torch.full((B,), done, dtype=torch.int32, device="cuda"),
                                      torch.tensor([0, n, 2 * n], dtype=torch.int32, device="cuda"), lg, max_q_len=n)
        outs.append(o.view(B, n, H, D))
    pieces = torch.cat(outs, 1).permute(0, 2, 1, 3)
    # each side within half a step and its weights' error of the exact answer
    step = torch.finfo(q.dtype).eps
    bound = step * whole.float().abs() + 2 * 2 * 4e-5 * 4.0
    assert ((pieces.float() - whole.float()).abs() <= bound).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_bad_lengths_and_pages_are_refused_by_the_kernel(dtype):
    lib = _native.lib()
    lib.ca_device_status(1)
    base = make_case(dtype, 4, 2, 64, 16, [(1, 40), (20, 50), (2, 3), (1, 100)], seed=12)
    want, mag = exact(base)
    rows = slice(1, 21)
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
        assert torch.isnan(out[3:21] if what == "page" else out[rows]).all(), what
        keep = torch.ones(out.shape[0], dtype=torch.bool)
        keep[rows] = False
        check(dtype, out[keep], want[keep], mag[keep], int(keep.sum()))
    assert lib.ca_device_status(0) == 0


def test_wrong_max_q_len_and_rows_outside_the_buffer():
    lib = _native.lib()
    lib.ca_device_status(1)
    case = make_case("bf16", 4, 2, 64, 16, [(1, 40), (20, 50), (2, 3)], seed=13)
    want, mag = exact(case)
    out = torch.full_like(case["q"], 3.0)
    for wrong in (1, 3, 8, 1000):
        check("bf16", run(case, max_q_len=wrong, out=out), want, mag, 23)
    assert lib.ca_device_status(0) == 0
    # the last sequence claims rows that q does not have: nothing of it is written
    starts = case["q_starts"].clone()
    starts[3] = out.shape[0] + 1
    out.fill_(3.0)
    continuum_attention_paged(*[starts if t is case["q_starts"] else t for t in arguments(case)], max_q_len=20, out=out)
    assert lib.ca_device_status(1) == 1
    assert (out[21:] == 3.0).all()
    check("bf16", out[:21], want[:21], mag[:21], 21)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_graph_replays_follow_the_lengths(dtype):
    """A decoding step captured once answers for other lengths and another page table when replayed, and
    two graphs that were captured with one pool do not disturb each other."""
    lens = [(1, 100), (1, 37), (1, 260)]
    case = make_case(dtype, 4, 2, 64, 16, lens, seed=14)
    other = make_case(dtype, 4, 2, 64, 16, [(1, 16), (1, 250), (1, 1)], seed=15)
    P = max(case["k_cache"].shape[0], other["k_cache"].shape[0])
    W = max(case["page_table"].shape[1], other["page_table"].shape[1])
    buf = {n: torch.zeros((P, *case["k_cache"].shape[1:]), dtype=case["q"].dtype, device="cuda")
           for n in ("k_cache", "v_cache")}
    buf.update(q=case["q"].clone(), log_gain=case["log_gain"].clone(), kv_lens=case["kv_lens"].clone(),
               q_starts=case["q_starts"].clone(),
               page_table=torch.zeros(3, W, dtype=torch.int32, device="cuda"))

    def load(c):
        for n in ("k_cache", "v_cache"):
            buf[n][:c[n].shape[0]] = c[n]
        for n in ("q", "log_gain", "kv_lens"):
            buf[n].copy_(c[n])
        buf["page_table"][:, :c["page_table"].shape[1]] = c["page_table"]

    load(case)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run({**buf, "max_q_len": 1})
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(run({**buf, "max_q_len": 1}))
        graphs.append(g)
    for c in (case, other, case):
        load(c)
        want = exact(c)
        for g, o in zip(graphs, outs):
            g.replay()
            check(dtype, o, *want, 3)
    assert _native.lib().ca_device_status(0) == 0


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_two_streams_at_once(dtype):
    cases = [make_case(dtype, 4, 2, 64, 16, [(1, 3000), (1, 40 + i)], seed=20 + i) for i in range(2)]
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
            check(dtype, o, *w, 2)
            assert torch.equal(o, got[0])               # same bits every time


def test_given_workspace_and_types():
    case = make_case("f16", 4, 2, 64, 16, [(1, 500), (3, 60)], seed=30)
    n = paged_workspace_bytes(2, 3, 4, 2, 64, torch.float16)
    ws = torch.full((max(n, 1),), 255, dtype=torch.uint8, device="cuda")
    a = run(case, workspace=ws)
    assert torch.equal(a, run(case))
    check("f16", a, *exact(case), 4)
    if n:
        with pytest.raises(ValueError, match="workspace"):
            run(case, workspace=ws[:n - 1])
    case["log_gain"] = case["log_gain"].double().requires_grad_()      # a parameter of another type
    assert torch.equal(run(case), a)


def test_nothing_to_do():
    case = make_case("bf16", 4, 2, 64, 16, [(1, 20)], seed=31)
    args = arguments(case)
    args[0] = case["q"][:0]
    assert continuum_attention_paged(*args, max_q_len=1).shape == (0, 4, 64)
    none = make_case("bf16", 4, 2, 64, 16, [], seed=31, tail=3)
    out = torch.full_like(none["q"], 2.0)
    run(none, out=out)
    assert (out == 2.0).all()
