"""Paged caches for the tests: random pages, stale slots, and the float64 answer.

``make_case`` scatters sequences over shuffled pages.  Everything no key needs (free slots of
a sequence's last page, pages of nobody) is NaN, and page-table entries no key needs are -1 or
far out of range, so a kernel that touches one shows it.
"""
from __future__ import annotations

import math

import torch

from oracle.ca_oracle import ca_weights_tile

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def make_case(dtype, heads, kv_heads, dim, page, seqs, *, seed=0, tail=0, gain=1.0, qk_mag=1.0, device="cuda",
              cache_layout="pgsd", far=0):
    """seqs: (new tokens, keys in all) of each sequence; far: pages in front of the first used one."""
    g = torch.Generator().manual_seed(seed)
    dt = DTYPES[dtype]
    need = [-(-L // page) for _, L in seqs]
    pages = sum(need) + 2 + far
    order = (torch.randperm(sum(need) + 2, generator=g) + far).tolist()
    width = max(max(need, default=0), 1) + 1
    table = torch.full((len(seqs), width), -1, dtype=torch.int32)
    table[:, 1::2] = 2 ** 31 - 1
    shape = {"pgsd": (pages, kv_heads, page, dim), "psgd": (pages, page, kv_heads, dim)}[cache_layout]
    caches = [torch.full(shape, float("nan"), dtype=dt, device=device) for _ in range(2)]
    if cache_layout == "psgd":
        caches = [c.permute(0, 2, 1, 3) for c in caches]
    keys, values = [], []
    at = 0
    for s, (n, L) in enumerate(seqs):
        k = (torch.randn(L, kv_heads, dim, generator=g) * qk_mag).to(dt)
        v = torch.randn(L, kv_heads, dim, generator=g).to(dt)
        keys.append(k)
        values.append(v)
        table[s, :need[s]] = torch.tensor(order[at:at + need[s]], dtype=torch.int32)
        at += need[s]
        for j in range(need[s]):
            rows = slice(j * page, min(L, (j + 1) * page))
            m = rows.stop - rows.start
            caches[0][table[s, j], :, :m] = k[rows].permute(1, 0, 2).to(device)
            caches[1][table[s, j], :, :m] = v[rows].permute(1, 0, 2).to(device)
    starts = [0]
    for n, _ in seqs:
        starts.append(starts[-1] + n)
    N = starts[-1] + tail
    q = (torch.randn(N, heads, dim, generator=g) * qk_mag).to(dt)
    log_gain = (torch.rand(heads, generator=g) - 0.3) * gain
    ints = dict(page_table=table, kv_lens=torch.tensor([L for _, L in seqs], dtype=torch.int32),
                q_starts=torch.tensor(starts, dtype=torch.int32))
    return {"q": q.to(device), "k_cache": caches[0], "v_cache": caches[1],
            **{n: t.to(device) for n, t in ints.items()}, "log_gain": log_gain.to(device),
            "max_q_len": max(max((n for n, _ in seqs), default=1), 1), "seqs": seqs, "keys": keys, "values": values}


def exact(case):
    """(answer, sum of w |v|) float64 on the CPU for the rows of all sequences; a row without keys is 0.
    The weights are the oracle's (pinned to the reference's own outputs)."""
    q, lg = case["q"].cpu().double(), case["log_gain"].cpu().double()
    N, H, D = q.shape
    out, mag = torch.zeros(N, H, D, dtype=torch.float64), torch.zeros(N, H, D, dtype=torch.float64)
    at = 0
    for (n, L), k, v in zip(case["seqs"], case["keys"], case["values"]):
        G = k.shape[1]
        skip = max(n - L, 0)      # rows at negative positions
        rows = slice(at + skip, at + n)
        at += n
        if n - skip == 0:
            continue
        kk = k.double().permute(1, 0, 2).repeat_interleave(H // G, 0)
        vv = v.double().permute(1, 0, 2).repeat_interleave(H // G, 0)
        x = q[rows].permute(1, 0, 2) * (lg.exp() / math.sqrt(D))[:, None, None]
        w = ca_weights_tile(x @ kk.transpose(1, 2), L - (n - skip))
        out[rows] = (w @ vv).permute(1, 0, 2)
        mag[rows] = (w @ vv.abs()).permute(1, 0, 2)
    return out, mag


# Weights off by a relative e move y by at most 2 e sum w |v| (numerator and normaliser).
# bf16: the two bf16 parts of a weight keep 16 bits (2^-16); moments 8e-6 (closed form at the
# series' border) and exponentials and scores, fp32 sums of at most 128 products and an argument of
# at most ~2^6, 64 * 2^-23: together below 4e-5.  f16 parts keep more, the rest is the same.
# f32: scores of at most 128 products summed in 32 bits, |q k| sums of at most ~40 in these
# cases: 128 * 2^-24 * 40 / 8 (errors of random sign over 8 partial sums) = 4e-5 at the very worst
# rows; the rows' own sums add below 1e-6.
WEIGHT_ERROR = {"f32": 4e-5, "bf16": 4e-5, "f16": 4e-5}


def check(dtype, out, want, mag, rows):
    """out [N,H,D] against the float64 answer: half a rounding step plus the weights' error."""
    got = out[:rows].double().cpu()
    assert torch.isfinite(got).all(), "non-finite output"
    bound = want[:rows].abs() * (torch.finfo(DTYPES[dtype]).eps / 2) * 1.0001 + 2 * WEIGHT_ERROR[dtype] * mag[:rows]
    # the smallest subnormal step of f16
    bound += 2.0 ** -25
    err = (got - want[:rows]).abs()
    worst = (err / bound.clamp_min(1e-300)).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"error {worst:.2f} times the bound, largest {err.max().item():.3e}"


def arguments(case):
    return [case[n] for n in ("q", "k_cache", "v_cache", "page_table", "kv_lens", "q_starts", "log_gain")]
