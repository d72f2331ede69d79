"""Rotary positions in general form against complex multiplication in float64: both layouts, part of the
head, shared heads, far positions, gradients, and the append to a paged cache."""
import pytest
import torch

from continuum_attention_b200 import RotaryTable, _native, rotary_append, rotary_qkv
from continuum_attention_b200.rope import cos_sin_table, rope_qkv
from continuum_attention_b200.rotary import rotary_frequencies
from paged_testlib import DTYPES, make_case

pytestmark = pytest.mark.gpu


def turn(x, pos, freq, scale, half, back=False):
    """x [..., heads, D] float64 at positions pos [...]: pairs of the first R values times scale e^(i pos freq)."""
    R = 2 * freq.numel()
    y = x.clone()
    a, b = (slice(0, R // 2), slice(R // 2, R)) if half else (slice(0, R, 2), slice(1, R, 2))
    ang = pos.double()[..., None, None] * freq * (-1 if back else 1)
    z = torch.complex(x[..., a], x[..., b]) * torch.polar(torch.full_like(ang, scale), ang)
    y[..., a], y[..., b] = z.real, z.imag
    return y


def check(got, want, dtype, pair_norm):
    """Half a step of the output, and the table's rounding (half a step of 32 bits each for cosine and
    sine) and the two products' (one step each): together below 4 * 2^-24 of the pair's norm."""
    err = (got.double().cpu() - want).abs()
    bound = want.abs() * torch.finfo(DTYPES[dtype]).eps / 2 * 1.0001 + 4 * 2.0 ** -24 * pair_norm + 2.0 ** -25
    if dtype == "f32":
        bound -= 2.0 ** -25
    assert bool((err <= bound).all()), f"{(err / bound.clamp_min(1e-300)).max().item():.2f} times the bound"


SHAPES = [  # B, T, H, G, D, R
    (2, 37, 3, 3, 64, 64), (1, 1, 4, 2, 64, 64), (2, 5, 8, 1, 128, 64), (1, 33, 5, 5, 8, 8), (1, 19, 4, 4, 80, 40),
    (2, 7, 2, 1, 256, 256), (1, 12, 6, 2, 24, 2), (1, 9, 3, 3, 72, 6), (1, 40, 2, 2, 40, 36), (1, 3, 32, 8, 16, 12)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("shape", SHAPES)
def test_rotary_qkv(dtype, layout, shape):
    B, T, H, G, D, R = shape
    g = torch.Generator().manual_seed(T * 100 + D)
    table = RotaryTable(R, 64, scaling="yarn", factor=3.0, original_positions=16)
    freq, scale = rotary_frequencies(R, scaling="yarn", factor=3.0, original_positions=16)
    qkv = torch.randn(B, T, (H + 2 * G) * D, generator=g).to("cuda", DTYPES[dtype])
    grads = [torch.randn(B, h, T, D, generator=g).to("cuda", DTYPES[dtype]) for h in (H, G, G)]
    heads = qkv.double().cpu().view(B, T, H + 2 * G, D)
    gh = torch.cat([t.double().cpu().transpose(1, 2) for t in grads], 2)
    pos_b = torch.randint(0, 64, (B, T), generator=g, dtype=torch.int32)
    for pos in (None, pos_b[0], pos_b):
        where = torch.arange(T).expand(B, T) if pos is None else pos.expand(B, T)
        x = qkv.detach().requires_grad_()
        q, k, v = rotary_qkv(x, H, table, kv_heads=G, layout=layout, positions=None if pos is None else pos.cuda())
        assert q.shape == (B, H, T, D) and k.shape == v.shape == (B, G, T, D)
        want = turn(heads, where, freq, scale, layout == "half")
        check(torch.cat((q, k), 1).transpose(1, 2), want[:, :, :H + G], dtype, 2.5 * heads.abs().max())
        assert torch.equal(v, qkv.view(B, T, H + 2 * G, D)[:, :, H + G:].transpose(1, 2))
        (dx,) = torch.autograd.grad((q, k, v), x, grads)
        dwant = turn(gh, where, freq, scale, layout == "half", back=True)
        dx = dx.view(B, T, H + 2 * G, D)
        check(dx[:, :, :H + G], dwant[:, :, :H + G], dtype, 2.5 * gh.abs().max())
        assert torch.equal(dx[:, :, H + G:], grads[2].transpose(1, 2))
    assert _native.lib().ca_device_status(0) == 0


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_gradient_against_differences(layout):
    """The turn is linear: differences in float32 are exact to rounding at any step."""
    table = RotaryTable(12, 8, scaling="linear", factor=2.0)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(1, 3, (2 + 2) * 16, generator=g).cuda()
    w = [torch.randn(1, h, 3, 16, generator=g).cuda() for h in (2, 1, 1)]

    def f(t):
        return sum((a.double() * b.double()).sum() for a, b in
                   zip(rotary_qkv(t, 2, table, kv_heads=1, layout=layout), w))

    xr = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(f(xr), xr)
    for i in torch.randperm(x.numel(), generator=g)[:40].tolist():
        e = torch.zeros_like(x).flatten()
        e[i] = 1.0
        d = (f(x + e.view_as(x)) - f(x - e.view_as(x))) / 2
        # x +- 1 rounds by 2^-23 at most, times gradients of a few, over two outputs
        assert abs(float(d) - float(dx.flatten()[i])) < 40 * 2.0 ** -23


def test_partial_gradients_views_and_expanded_inputs():
    table = RotaryTable(64, 32)
    x = torch.randn(2, 9, 6 * 64, device="cuda", requires_grad=True)
    q, k, v = rotary_qkv(x, 4, table, kv_heads=1)
    full = torch.autograd.grad((q, k, v), x, [torch.ones_like(q), torch.zeros_like(k), torch.zeros_like(v)],
                               retain_graph=True)[0]
    assert torch.equal(torch.autograd.grad(q.sum(), x, retain_graph=True)[0], full)      # expanded gradient, None for k, v
    with pytest.raises(RuntimeError, match="first-order"):
        torch.autograd.grad(q.sum(), x, create_graph=True)
    wide = torch.randn(2, 9, 8 * 64 + 1, device="cuda")
    view = wide[..., 1:6 * 64 + 1]                                                     # strided and off 16 bytes
    for a, b in zip(rotary_qkv(view, 4, table, kv_heads=1), rotary_qkv(view.contiguous(), 4, table, kv_heads=1)):
        assert torch.equal(a, b)
    row = torch.randn(1, 9, 6 * 64, device="cuda").expand(3, 9, 6 * 64).requires_grad_()   # one row for all
    q, k, v = rotary_qkv(row, 4, table, kv_heads=1)
    assert torch.equal(q[0], q[2])


def test_equals_the_decoders_own_kernel():
    """Interleaved, whole head, the decoder's own table: the bits of rope_qkv."""
    x = torch.randn(2, 50, 3 * 4 * 64, device="cuda").bfloat16()
    table = RotaryTable.from_cos_sin(cos_sin_table(50, 64, 10000.0, x.device))
    for a, b in zip(rotary_qkv(x, 4, table), rope_qkv(x, 4, 10000.0)):
        assert torch.equal(a, b)


def test_positions_outside_the_table():
    lib = _native.lib()
    lib.ca_device_status(1)
    table = RotaryTable(32, 8)
    x = torch.randn(1, 4, 3 * 64, device="cuda")
    for bad in (8, -1, 2 ** 31 - 1, -2 ** 31):
        q, k, v = rotary_qkv(x, 1, table, positions=torch.tensor([0, bad, 7, 3], dtype=torch.int32, device="cuda"))
        assert lib.ca_device_status(1) == 1
        assert torch.isnan(q[0, 0, 1, :32]).all() and torch.isfinite(q[0, 0, [0, 2, 3]]).all()
        assert torch.equal(v[0, 0], x[0, :, 128:])
    with pytest.raises(ValueError, match="positions"):
        rotary_qkv(torch.zeros(1, 9, 192, device="cuda"), 1, table)
    with pytest.raises(ValueError, match="int32"):
        rotary_qkv(x, 1, table, positions=torch.arange(4, device="cuda"))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("heads,kv_heads,dim,rotary,page,cache_layout", [
    (4, 4, 64, 64, 16, "pgsd"), (8, 2, 128, 64, 7, "psgd"), (3, 1, 40, 12, 1, "pgsd"), (32, 8, 16, 16, 64, "pgsd")])
def test_append(dtype, layout, heads, kv_heads, dim, rotary, page, cache_layout):
    seqs = [(1, 1), (0, 9), (5, 40), (3, 0), (7, 4), (1, 130), (64, 64), (20, 97)]
    c = make_case(dtype, heads, kv_heads, dim, page, seqs, seed=dim, tail=4, cache_layout=cache_layout)
    rows = sum(n for n, _ in seqs)
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(rows + 4, (heads + 2 * kv_heads) * dim, generator=g).to("cuda", DTYPES[dtype])
    table = RotaryTable(rotary, 130, scaling="ntk", factor=2.0)
    freq, scale = rotary_frequencies(rotary, scaling="ntk", factor=2.0)
    out = torch.full((rows + 4, heads, dim), 5.0, dtype=qkv.dtype, device="cuda")
    before = [c["k_cache"].clone(), c["v_cache"].clone()]
    res = rotary_append(qkv, c["k_cache"], c["v_cache"], c["page_table"], c["kv_lens"], c["q_starts"], table,
                        heads=heads, layout=layout, out=out)
    assert res is out and _native.lib().ca_device_status(0) == 0
    assert (out[rows:] == 5.0).all()
    x = qkv.double().cpu().view(-1, heads + 2 * kv_heads, dim)
    at = 0
    written = torch.zeros(c["k_cache"].shape[0], page, dtype=torch.bool)
    for s, (n, L) in enumerate(seqs):
        for t in range(n):
            pos = L - n + t
            if pos < 0:
                assert (out[at + t] == 0).all()
                continue
            want = turn(x[at + t, :heads + kv_heads], torch.tensor(pos), freq, scale, layout == "half")
            p, slot = int(c["page_table"][s, pos // page]), pos % page
            written[p, slot] = True
            norm = 2 * x[at + t].abs().max()
            check(out[at + t], want[:heads], dtype, norm)
            check(c["k_cache"][p, :, slot], want[heads:], dtype, norm)
            assert torch.equal(c["v_cache"][p, :, slot], qkv[at + t].view(-1, dim)[heads + kv_heads:])
        at += n
    for old, new in zip(before, (c["k_cache"], c["v_cache"])):      # every other slot as it was (NaN among them)
        keep = ~written
        a, b = (t.permute(0, 2, 1, 3)[keep.to(t.device)] for t in (old, new))
        assert torch.equal(torch.nan_to_num(a, 77.0), torch.nan_to_num(b, 77.0))


def test_append_refuses_bad_pages_and_positions():
    lib = _native.lib()
    lib.ca_device_status(1)
    c = make_case("bf16", 2, 1, 64, 16, [(2, 20), (1, 40), (1, 8)], seed=3)
    table = RotaryTable(64, 40)
    qkv = torch.randn(4, 4 * 64, device="cuda").bfloat16()

    def go(**kw):
        a = {**c, **kw}
        before = a["k_cache"].clone()
        q = rotary_append(qkv, a["k_cache"], a["v_cache"], a["page_table"], a["kv_lens"], a["q_starts"],
                          a.get("table", table), heads=2)
        return q, torch.nan_to_num(before, 7.0), torch.nan_to_num(a["k_cache"], 7.0)

    pt = c["page_table"].clone()
    pt[1, 2] = c["k_cache"].shape[0]
    for kw, row in ((dict(page_table=pt), 2), (dict(table=RotaryTable(64, 39)), 2)):
        q, _, _ = go(**kw)
        assert lib.ca_device_status(1) == 1
        assert torch.isnan(q[row]).all() and torch.isfinite(q[[0, 1, 3]]).all()
    far = c["kv_lens"].clone()
    far[1] = c["page_table"].shape[1] * 16 + 5
    q, _, _ = go(kv_lens=far, table=RotaryTable(64, 4000))
    assert lib.ca_device_status(1) == 1 and torch.isnan(q[2]).all()
    with pytest.raises(RuntimeError, match="no backward"):
        rotary_append(qkv.requires_grad_(), c["k_cache"], c["v_cache"], c["page_table"], c["kv_lens"], c["q_starts"],
                      table, heads=2)


def test_captured_forward_and_backward():
    """The training pair captured into one graph (leaves of its own) and replayed on new data."""
    table = RotaryTable(32, 64)
    x = torch.randn(2, 30, 4 * 64, device="cuda", requires_grad=True)
    grads = [torch.randn(2, h, 30, 64, device="cuda") for h in (2, 1, 1)]

    def step():
        return torch.autograd.grad(rotary_qkv(x, 2, table, kv_heads=1, layout="half"), x, grads)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dx = step()
    for t in grads:
        t.normal_()
    graph.replay()
    assert torch.equal(dx, step())


def test_shared_tables_are_not_made_by_a_capture():
    """A table kept for later calls must not be one that only a graph's replay fills."""
    from continuum_attention_b200.rope import cos_sin_table
    from continuum_attention_b200.rotary import rotary_table
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        inside = cos_sin_table(57, 48, 777.0, torch.device("cuda", 0))
        with pytest.raises(RuntimeError, match="before a CUDA graph"):
            rotary_table(48, 57, 777.0, "ntk", 2.0, None, torch.device("cuda", 0))
    after = cos_sin_table(57, 48, 777.0, torch.device("cuda", 0))
    assert after is not inside and cos_sin_table(57, 48, 777.0, torch.device("cuda", 0)) is after
    graph.replay()
    assert torch.equal(inside, after)
    table = rotary_table(48, 57, 777.0, "ntk", 2.0, None, torch.device("cuda", 0))
    assert rotary_table(48, 57, 777.0, "ntk", 2.0, None, torch.device("cuda", 0)) is table
