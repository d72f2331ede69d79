"""The serving and rotary operators as they are measured: cases, inputs, plain forms, exact values.

Three operators:

* ``attend``: Continuum Attention of new tokens over a paged cache.  Sequence s holds
  ``kv_lens[s]`` keys in pages listed by its row of ``page_table``; its last ``n_s`` keys
  belong to the new tokens, which are rows ``q_starts[s] .. q_starts[s+1]`` of q.  A single
  new token per sequence is the decoding step, more are a prompt or a part of one.
* ``append``: the rotary embedding of new tokens' queries and keys at their cache
  positions, with the rotated keys and the values written into the paged cache.
* ``rotate``: the rotary embedding of a projection output for training, with its gradient.

With ``own`` false ``run`` is the plain form (elementary torch operations in 32 bits, angles
in 64); with ``own`` true it makes the calls that a user of the package makes.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}


# ------------------------------------------------------------------ cases

def _attend(name, dtype, heads, kv_heads, dim, page, seqs, new_lo, new_hi, len_lo, len_hi, tail=0):
    """``seqs`` sequences with new_lo..new_hi new tokens over len_lo..len_hi keys in all (both
    spread evenly over their logarithm), ``tail`` unused rows behind the last sequence."""
    case = {"op": "attend", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "seqs": seqs, "new_lo": new_lo, "new_hi": new_hi, "len_lo": len_lo, "len_hi": len_hi, "tail": tail}
    return {"name": name, **case} if name else case


def _append(name, dtype, heads, kv_heads, dim, rotary, layout, scaling, factor, page, seqs, new_lo, new_hi,
            len_lo, len_hi, tail=0):
    case = {"op": "append", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotary": rotary,
            "layout": layout, "scaling": scaling, "factor": factor, "page": page, "seqs": seqs, "new_lo": new_lo,
            "new_hi": new_hi, "len_lo": len_lo, "len_hi": len_hi, "tail": tail}
    return {"name": name, **case} if name else case


def _rotate(name, dtype, heads, kv_heads, dim, rotary, layout, scaling, factor, batch, length, offset):
    """``offset``: the first position (0, or far into a long context)."""
    case = {"op": "rotate", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotary": rotary,
            "layout": layout, "scaling": scaling, "factor": factor, "batch": batch, "length": length,
            "offset": offset}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one user decoding at the end of the decoder's block of 2048 bytes: latency
        _attend("decode_one", "bf16", 16, 16, 64, 64, 1, 1, 1, 2048, 2048),
        # a serving batch of the decoder's head layout, from a first byte to long contexts
        _attend("decode_batch", "bf16", 16, 16, 64, 64, 64, 1, 1, 1, 8192),
        # two very long contexts with shared key heads and small pages: the long axis has to be split
        _attend("decode_long", "f16", 32, 8, 64, 16, 2, 1, 1, 90001, 131071),
        # wide heads, shared, several tokens a step (a draft being checked)
        _attend("decode_wide", "bf16", 32, 8, 128, 32, 17, 1, 4, 500, 20000),
        # whole prompts of the decoder's block size, no cache before them
        _attend("prompt", "bf16", 16, 16, 64, 64, 2, 2048, 2048, 2048, 2048),
        # a piece of a long prompt behind what the cache holds
        _attend("chunk_long", "f16", 16, 16, 64, 128, 1, 511, 511, 16001, 16001),
        # a step that mixes decoding, short pieces and empty sequences; rows behind the last one
        _attend("chunk_mixed", "bf16", 16, 4, 64, 16, 23, 0, 300, 0, 4000, tail=5),
        # the small model's heads and length in its own type
        _attend("chunk_f32", "f32", 4, 4, 64, 16, 8, 40, 192, 40, 192),
        # the decoding step's side of the projection: one token of each of 64 sequences
        _append("append_decode", "bf16", 16, 16, 64, 64, "interleaved", "none", 1.0, 64, 64, 1, 1, 1, 8192),
        # pieces of prompts at far positions: half layout, half the head, positions stretched
        _append("append_chunk", "f16", 32, 8, 128, 64, "half", "yarn", 8.0, 32, 5, 1, 1500, 9000, 60000, tail=3),
        # the decoder's training batch
        _rotate("train_decoder", "bf16", 16, 16, 64, 64, "interleaved", "none", 1.0, 8, 2048, 0),
        # the small model's heads in 32 bits, an odd length far into a stretched context, part of the head
        _rotate("train_part", "f32", 12, 4, 64, 48, "half", "ntk", 4.0, 3, 577, 100003),
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "rotate"])
    if op == "attend":
        dtype = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
        kv_heads = rng.choice([1, 2, 4, 8, 16])
        heads = kv_heads * rng.choice([g for g in (1, 2, 3, 4, 8) if kv_heads * g <= 32])
        dim = rng.choice([32, 64, 64, 64, 80, 128])
        page = rng.choice([1, 8, 16, 24, 64, 128])
        # keys in all and pairs of rows and keys that the largest listed cases have
        keys = 450000000 // (2 * kv_heads * dim * _BYTES[dtype])
        pairs = (130000000 if dtype != "f32" else 30000000) * 64 // (heads * max(dim, 64))
        if rng.random() < 0.5:
            seqs, hi_new = _spread(rng, 1, 64), rng.choice([1, 1, 2, 5])
            hi = max(8, min(_spread(rng, 16, 100000), keys // seqs, pairs // (seqs * hi_new)))
        else:
            hi_new = _spread(rng, 17, 1500)
            hi = max(hi_new, min(_spread(rng, 64, 16000), pairs // hi_new, keys))
            seqs = max(1, min(12, pairs // (hi * hi_new), keys // hi))
        return _attend(None, dtype, heads, kv_heads, dim, page, seqs, rng.choice([0, 1, hi_new]), hi_new,
                       rng.choice([0, 1, hi // 2, hi]), hi, rng.choice([0, 0, 7]))
    dtype = rng.choice(["bf16", "f16", "f32"])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    heads = kv_heads * rng.choice([g for g in (1, 2, 3, 4, 8) if kv_heads * g <= 32])
    dim = rng.choice([32, 64, 64, 80, 128])
    rotary = rng.choice([dim, dim, dim // 2, 16])
    layout = rng.choice(["interleaved", "half"])
    scaling = rng.choice(["none", "linear", "ntk", "yarn"])
    factor = 1.0 if scaling == "none" else round(rng.uniform(1.5, 16.0), 2)
    if op == "append":
        seqs = _spread(rng, 1, 64)
        hi_new = _spread(rng, 1, max(2, 6000 // seqs))
        hi = max(hi_new, min(_spread(rng, 16, 100000), 100000 // seqs))
        return _append(None, dtype, heads, kv_heads, dim, rotary, layout, scaling, factor,
                       rng.choice([1, 8, 16, 24, 64, 128]), seqs, rng.choice([0, 1, hi_new]), hi_new,
                       rng.choice([1, hi // 2, hi]), hi, rng.choice([0, 0, 7]))
    tokens = 400000000 // (4 * (heads + 2 * kv_heads) * dim * _BYTES[dtype])
    length = _spread(rng, 1, min(4000, tokens))
    return _rotate(None, dtype, heads, kv_heads, dim, rotary, layout, scaling, factor,
                   max(1, min(_spread(rng, 1, 32), tokens // length)), length, rng.choice([0, 0, 1000, 100003]))


# ------------------------------------------------------------------ what a case's sequences look like

def _sequences(case, seed):
    """(new tokens, keys in all) of each sequence.  A sequence has as many keys as new tokens at
    least, but where a range begins at 0: there one sequence is empty and one has more rows than
    keys, so that its first rows see nothing.  The seed gives their order alone, so that a case's
    work is the same for all."""
    rng = random.Random(f"{case['op']}/{case['seqs']}/{case['new_hi']}/{case['len_hi']}")
    pairs = []
    for s in range(case["seqs"]):
        n = _spread(rng, max(case["new_lo"], 1), max(case["new_hi"], 1))
        pairs.append((n, max(n, _spread(rng, max(case["len_lo"], 1), max(case["len_hi"], 1)))))
    pairs[-1] = (max(case["new_hi"], 1), max(case["len_hi"], case["new_hi"], 1))
    if case["new_lo"] == 0 and len(pairs) > 2:
        pairs[0] = (0, pairs[0][1])
    if case["len_lo"] == 0 and case["op"] == "attend" and len(pairs) > 4:
        pairs[1], pairs[2] = (min(3, case["new_hi"]), 0), (case["new_hi"], case["new_hi"] // 2)
    random.Random(seed).shuffle(pairs)
    return [n for n, _ in pairs], [L for _, L in pairs]


def work(case):
    e, D = _BYTES[case["dtype"]], case["dim"]
    H, G = case["heads"], case["kv_heads"]
    if case["op"] == "rotate":
        tokens = case["batch"] * case["length"]
        once = tokens * (H + 2 * G) * D * e
        # read and write of values and of gradients, and the rotation's angles
        return {"bytes": 4 * once, "flops": 2 * 3 * tokens * (H + G) * case["rotary"]}
    new, lens = _sequences(case, 0)
    tokens = sum(new)
    if case["op"] == "append":
        return {"bytes": 2 * tokens * (H + 2 * G) * D * e, "flops": 3 * tokens * (H + G) * case["rotary"]}
    pairs = sum(n * max(L - n, 0) + min(n, L) * (min(n, L) + 1) // 2 for n, L in zip(new, lens))
    keys = sum(L for n, L in zip(new, lens) if n)
    return {"bytes": (2 * keys * G + 2 * tokens * H) * D * e, "flops": 4 * pairs * H * D}


# ------------------------------------------------------------------ inputs

def _frequencies(case):
    """Angle per position of each pair, in 64 bits, and the factor on cosine and sine."""
    R, theta, f = case["rotary"], 10000.0, case["factor"]
    if case["scaling"] == "ntk" and R > 2:
        theta *= f ** (R / (R - 2))
    inv = theta ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    if case["scaling"] == "linear":
        return inv / f, 1.0
    if case["scaling"] == "yarn":
        # pairs that turn often within the original length keep their angle, slow ones are stretched
        def border(turns):
            return R * math.log(_ORIGINAL / (turns * 2 * math.pi)) / (2 * math.log(theta))
        low, high = max(math.floor(border(32)), 0), min(math.ceil(border(1)), R // 2 - 1)
        ramp = ((torch.arange(R // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
        return inv / f * ramp + inv * (1 - ramp), 0.1 * math.log(f) + 1.0
    return inv, 1.0


_ORIGINAL = 2048      # the length before it was stretched: the decoder's block


def _table(case, positions):
    from continuum_attention_b200.rotary import RotaryTable
    return RotaryTable(case["rotary"], positions, theta=10000.0,
                       scaling=None if case["scaling"] == "none" else case["scaling"], factor=case["factor"],
                       original_positions=_ORIGINAL, device="cuda")


def _paged_inputs(case, seed, st, gen):
    """Page table, lengths and a cache whose free pages and free slots hold stale values."""
    new, lens = _sequences(case, seed)
    page, G, D, dt = case["page"], case["kv_heads"], case["dim"], _TYPES[case["dtype"]]
    need = [-(-L // page) for L in lens]
    width = max(need) + 1
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    rows = torch.tensor(need, device="cuda")
    first = torch.cumsum(rows, 0) - rows
    col = torch.arange(width, device="cuda")
    index = (first[:, None] + col[None, :]).clamp(max=pages - 1)
    # entries that no key needs are -1
    table = torch.where(col[None, :] < rows[:, None], order[index], torch.full_like(order[index], -1))
    st["page_table"] = table.contiguous()
    st["kv_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    st["q_starts"] = torch.tensor([sum(new[:s]) for s in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    st["max_q_len"] = max(max(new), 1)
    st["new"], st["lens"] = new, lens
    shape = (pages, G, page, D)
    st["k_cache"] = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dt)
    st["v_cache"] = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dt)
    return sum(new) + case["tail"]


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(1000003 * seed + 17)
    dt, H, G, D = _TYPES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]
    st = {"case": case}

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)

    if case["op"] == "attend":
        rows = _paged_inputs(case, seed, st, gen)
        st["q"] = normal(rows, H, D).to(dt)
        # learned per-head gains between no sharpening and that of tau = 0.30
        st["log_gain"] = torch.rand(H, generator=gen, device="cuda") * 1.2
        st["out"] = torch.full((rows, H, D), 0.25, dtype=dt, device="cuda")
        return st
    freq, scale = _frequencies(case)
    st["freq"], st["scale"] = freq.cuda(), scale
    if case["op"] == "append":
        rows = _paged_inputs(case, seed, st, gen)
        st["qkv"] = normal(rows, (H + 2 * G) * D).to(dt)
        st["out"] = torch.full((rows, H, D), 0.25, dtype=dt, device="cuda")
        if own:
            st["table"] = _table(case, case["page"] * st["page_table"].shape[1])
        return st
    B, T = case["batch"], case["length"]
    st["qkv"] = normal(B, T, (H + 2 * G) * D).to(dt).requires_grad_()
    st["grads"] = [normal(B, h, T, D).to(dt) for h in (H, G, G)]
    st["positions"] = (torch.arange(T, device="cuda", dtype=torch.int32) + case["offset"]) if case["offset"] else None
    if own:
        st["table"] = _table(case, T + case["offset"])
    return st


# ------------------------------------------------------------------ plain forms

_J1 = [1 / 2, 1 / 3, 1 / 8, 1 / 30, 1 / 144, 1 / 840, 1 / 5760, 1 / 45360, 1 / 403200, 1 / 3991680]


def _plain_weights(s, visible):
    """Unnormalised weights of the keys of each row and their sum (32 bits).  s [.., rows, keys] are
    scores, visible [rows, keys] says which keys a row sees (a prefix of them)."""
    s = s.masked_fill(~visible, float("-inf"))
    m = s.amax(-1, keepdim=True)
    m = torch.where(torch.isfinite(m), m, torch.zeros_like(m))
    e = torch.exp(s - m)
    seg = visible[:, 1:]
    d = torch.where(seg, s[..., 1:] - s[..., :-1], torch.zeros_like(s[..., 1:]))
    a, b = e[..., :-1], e[..., 1:]
    series = torch.full_like(d, _J1[9])
    for c in _J1[8::-1]:
        series = series * d + c
    near = d.abs() < 1
    safe = torch.where(near, torch.ones_like(d), d)
    right = torch.where(near, a * series, (b - (b - a) / safe) / safe)
    left = torch.where(near, b - d * right, (b - a) / safe) - right
    right, left = (torch.where(seg, t, torch.zeros_like(t)) for t in (right, left))
    w = torch.zeros_like(e)
    w[..., 1:] += right
    w[..., :-1] += left
    w[..., 0] += 0.5 * e[..., 0]
    last = visible.sum(-1) - 1
    rows = torch.arange(s.shape[-2], device=s.device)
    ok = (last >= 0).to(e.dtype)
    w[..., rows, last.clamp(min=0)] += 0.5 * e[..., rows, last.clamp(min=0)] * ok
    return w, w.sum(-1, keepdim=True)


def _rows_of(cache, table, length, page):
    """The first ``length`` rows of a sequence: [kv_heads, length, D] in 32 bits."""
    pages = table[:-(-length // page)].long()
    x = cache[pages].permute(1, 0, 2, 3)
    return x.reshape(x.shape[0], -1, x.shape[-1])[:, :length].float()


def _run_attend(st):
    case, q, out = st["case"], st["q"], st["out"]
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    gain = torch.exp(st["log_gain"]) / math.sqrt(D)
    start = 0
    for s, (n, L) in enumerate(zip(st["new"], st["lens"])):
        if n == 0:
            continue
        rows = slice(start, start + n)
        start += n
        if L == 0:
            out[rows] = 0
            continue
        k = _rows_of(st["k_cache"], st["page_table"][s], L, case["page"])
        v = _rows_of(st["v_cache"], st["page_table"][s], L, case["page"])
        pos = torch.arange(L - n, L, device=q.device)
        visible = torch.arange(L, device=q.device)[None, :] <= pos[:, None]
        x = (q[rows].float() * gain[None, :, None]).permute(1, 0, 2).reshape(G, (H // G) * n, D)
        scores = torch.matmul(x, k.transpose(1, 2)).reshape(H, n, L)
        w, z = _plain_weights(scores, visible)
        y = torch.matmul(w.reshape(G, (H // G) * n, L), v).reshape(H, n, D)
        y = torch.where(z > 0, y / torch.where(z > 0, z, torch.ones_like(z)), torch.zeros_like(y))
        out[rows] = y.permute(1, 0, 2).to(out.dtype)
    return out


def _turn(x, cos, sin, case):
    """x [.., heads, D] in 32 bits with cos, sin [.., 1, R/2]: pairs of the first R values turned."""
    R = case["rotary"]
    part = x[..., :R]
    if case["layout"] == "interleaved":
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = part[..., :R // 2], part[..., R // 2:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., R:]), -1)


def _angles(st, positions):
    phase = positions.double()[:, None] * st["freq"]
    return (phase.cos() * st["scale"]).float()[:, None, :], (phase.sin() * st["scale"]).float()[:, None, :]


def _token_places(st):
    """(position, page, slot in page) of each new token, from lengths and page table on the device."""
    starts, page = st["q_starts"].long(), st["case"]["page"]
    token = torch.arange(sum(st["new"]), device="cuda")
    s = torch.searchsorted(starts, token, right=True) - 1
    pos = token - starts[s + 1] + st["kv_lens"].long()[s]
    return pos, st["page_table"][s, pos // page].long(), pos % page


def _run_append(st):
    case, out = st["case"], st["out"]
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    pos, page, slot = _token_places(st)
    n = pos.shape[0]
    x = st["qkv"][:n].float().reshape(n, H + 2 * G, D)
    cos, sin = _angles(st, pos)
    out[:n] = _turn(x[:, :H], cos, sin, case).to(out.dtype)
    st["k_cache"][page, :, slot] = _turn(x[:, H:H + G], cos, sin, case).to(out.dtype)
    st["v_cache"][page, :, slot] = x[:, H + G:].to(out.dtype)
    return out, st["k_cache"], st["v_cache"]


def _run_rotate(st):
    case, qkv = st["case"], st["qkv"].detach()
    B, T, H, G, D = case["batch"], case["length"], case["heads"], case["kv_heads"], case["dim"]
    pos = torch.arange(T, device="cuda") if st["positions"] is None else st["positions"]
    cos, sin = _angles(st, pos)
    x = qkv.float().reshape(B, T, H + 2 * G, D)
    turned = torch.cat((_turn(x[:, :, :H + G], cos, sin, case), x[:, :, H + G:]), 2).to(qkv.dtype)
    outs = [t.transpose(1, 2).contiguous() for t in turned.split([H, G, G], 2)]
    g = torch.cat([t.float().transpose(1, 2) for t in st["grads"]], 2)
    back = torch.cat((_turn(g[:, :, :H + G], cos, -sin, case), g[:, :, H + G:]), 2)
    return (*outs, back.reshape(B, T, -1).to(qkv.dtype))


# ------------------------------------------------------------------ one pass

def run(st):
    case = st["case"]
    if not own:
        return {"attend": _run_attend, "append": _run_append, "rotate": _run_rotate}[case["op"]](st)
    if case["op"] == "attend":
        from continuum_attention_b200 import continuum_attention_paged
        return continuum_attention_paged(st["q"], st["k_cache"], st["v_cache"], st["page_table"], st["kv_lens"],
                                         st["q_starts"], st["log_gain"], max_q_len=st["max_q_len"], out=st["out"])
    if case["op"] == "append":
        from continuum_attention_b200.rotary import rotary_append
        q = rotary_append(st["qkv"], st["k_cache"], st["v_cache"], st["page_table"], st["kv_lens"], st["q_starts"],
                          st["table"], heads=case["heads"], layout=case["layout"], out=st["out"])
        return q, st["k_cache"], st["v_cache"]
    from continuum_attention_b200.rotary import rotary_qkv
    q, k, v = rotary_qkv(st["qkv"], case["heads"], st["table"], kv_heads=case["kv_heads"], layout=case["layout"],
                         positions=st["positions"])
    (dqkv,) = torch.autograd.grad((q, k, v), st["qkv"], st["grads"])
    return q, k, v, dqkv


# ------------------------------------------------------------------ exact values

def _exact_row_weights(s, count):
    """Weights in 64 bits of the rows of s [rows, keys], row r seeing its first count[r] keys: every
    segment's two integrals of e^(s + u d) (1 - u) and e^(s + u d) u over u in [0, 1]."""
    keys = torch.arange(s.shape[-1], device=s.device)
    seen = keys[None, :] < count[:, None]
    top = torch.where(seen, s, torch.full_like(s, -1e300)).amax(-1, keepdim=True)
    e = torch.where(seen, torch.exp(torch.where(seen, s - top, torch.zeros_like(s))), torch.zeros_like(s))
    d = torch.where(seen[:, 1:], s[:, 1:] - s[:, :-1], torch.ones_like(s[:, 1:]))
    small = d.abs() < 2e-2
    ds = torch.where(small, torch.ones_like(d), d)
    # int u e^(ud) = (e^d (d - 1) + 1) / d^2 ; int (1 - u) e^(ud) = (e^d - 1 - d) / d^2
    up = torch.where(small, 1 / 2 + d / 3 + d ** 2 / 8 + d ** 3 / 30 + d ** 4 / 144 + d ** 5 / 840 + d ** 6 / 5760,
                     (1 + (ds - 1) * torch.exp(ds.clamp(max=0))) / ds ** 2)
    down = torch.where(small, 1 / 2 + d / 6 + d ** 2 / 24 + d ** 3 / 120 + d ** 4 / 720 + d ** 5 / 5040
                       + d ** 6 / 40320, (torch.expm1(ds.clamp(max=0)) - ds) / ds ** 2)
    # for rising scores the same integrals from the right end: u -> 1 - u, d -> -d
    rise = ~small & (d > 0)
    down_r = (1 + (-ds - 1) * torch.exp((-ds).clamp(max=0))) / ds ** 2
    up_r = (torch.expm1((-ds).clamp(max=0)) + ds) / ds ** 2
    base = torch.where(rise, e[:, 1:], e[:, :-1])
    left = torch.where(rise, down_r, down) * base
    right = torch.where(rise, up_r, up) * base
    left, right = (torch.where(seen[:, 1:], t, torch.zeros_like(t)) for t in (left, right))
    w = torch.nn.functional.pad(left, (0, 1)) + torch.nn.functional.pad(right, (1, 0))
    ends = (keys[None, :] == 0).double() + (keys[None, :] == count[:, None] - 1).double()
    return w + 0.5 * ends * e


def _exact_attend(st):
    case = st["case"]
    H, G, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out = st["out"].double()
    gain = torch.exp(st["log_gain"].double()) / math.sqrt(D)
    token = 0
    for s, (n, L) in enumerate(zip(st["new"], st["lens"])):
        out[token:token + n] = 0
        if n and L:
            key = torch.arange(L, device="cuda")
            where = (st["page_table"][s, key // page].long(), key % page)
            k, v = st["k_cache"][where[0], :, where[1]].double(), st["v_cache"][where[0], :, where[1]].double()
            count = torch.arange(L - n + 1, L + 1, device="cuda")
            empty = count <= 0
            for h in range(H):
                scores = gain[h] * (st["q"][token:token + n, h].double() @ k[:, h // (H // G)].T)
                w = _exact_row_weights(scores, count)
                y = (w / w.sum(-1, keepdim=True)) @ v[:, h // (H // G)]
                y[empty] = 0
                out[token:token + n, h] = y
        token += n
    return out


def _exact_turn(x, phase, scale, case, back=False):
    """x [.., heads, D] in 64 bits turned as complex numbers by e^(i phase) scale, phase [.., R/2]."""
    R = case["rotary"]
    pairs = x[..., :R].unflatten(-1, (R // 2, 2) if case["layout"] == "interleaved" else (2, R // 2))
    if case["layout"] == "half":
        pairs = pairs.transpose(-1, -2)
    turn = torch.polar(torch.full_like(phase, scale), -phase if back else phase)[..., None, :]
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    if case["layout"] == "half":
        z = z.transpose(-1, -2)
    y = x.clone()
    y[..., :R] = z.flatten(-2)
    return y


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "attend":
        return _exact_attend(st)
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        out, kc, vc = st["out"].double(), st["k_cache"].double(), st["v_cache"].double()
        token = 0
        for s, (n, L) in enumerate(zip(st["new"], st["lens"])):
            if n:
                pos = torch.arange(L - n, L, device="cuda")
                x = st["qkv"][token:token + n].double().reshape(n, H + 2 * G, D)
                y = _exact_turn(x[:, :H + G], pos[:, None].double() * st["freq"], st["scale"], case)
                pages, slots = st["page_table"][s, pos // case["page"]].long(), pos % case["page"]
                out[token:token + n] = y[:, :H]
                kc[pages, :, slots] = y[:, H:]
                vc[pages, :, slots] = x[:, H + G:]
            token += n
        return out, kc, vc
    B, T = case["batch"], case["length"]
    phase = (torch.arange(T, device="cuda") + case["offset"])[:, None].double() * st["freq"]
    x = st["qkv"].detach().double().reshape(B, T, H + 2 * G, D)
    q, k = _exact_turn(x[:, :, :H], phase, st["scale"], case), _exact_turn(x[:, :, H:H + G], phase, st["scale"], case)
    dq, dk, dv = (t.double().transpose(1, 2) for t in st["grads"])
    back = torch.cat((_exact_turn(dq, phase, st["scale"], case, True),
                      _exact_turn(dk, phase, st["scale"], case, True), dv), 2)
    return (q.transpose(1, 2).contiguous(), k.transpose(1, 2).contiguous(),
            x[:, :, H + G:].transpose(1, 2).contiguous(), back.reshape(B, T, -1))
