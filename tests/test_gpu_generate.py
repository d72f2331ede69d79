"""The decoder answering over the paged cache: rotary append, paged attention and the block's kernels in a
run, against the same model's forward over whole sequences."""
import pytest
import torch

from continuum_attention_b200 import _native
from continuum_attention_b200.decoder import ContinuumDecoderConfig, ContinuumDecoderLM

pytestmark = pytest.mark.gpu


def model(seed=0, **kw):
    torch.manual_seed(seed)
    cfg = ContinuumDecoderConfig(**{**dict(block_size=160, d_model=256, n_heads=4, n_layers=3), **kw})
    m = ContinuumDecoderLM(cfg).cuda()
    for b in m.blocks:
        torch.nn.init.uniform_(b.attn.log_qk_gain, -0.3, 0.5)
    return m


GENERAL = dict(rope_layout="half", rope_dim=32, rope_scaling="yarn", rope_factor=4.0, rope_original=40)


@pytest.mark.parametrize("kw", [{}, GENERAL, dict(rope_scaling="ntk", rope_factor=2.0), dict(rope_scaling="linear", rope_factor=3.0)])
def test_paged_steps_give_the_forwards_logits(kw):
    """Ragged pieces, then single tokens, in 32 bits: every row is the forward's row."""
    m = model(**kw)
    g = torch.Generator().manual_seed(1)
    lens = [150, 97, 33]
    ids = [torch.randint(0, 256, (n,), generator=g).cuda() for n in lens]
    with torch.no_grad():
        want = [m(i[None])["logits"][0] for i in ids]
    cache = m.make_cache(3, page_size=16)
    done, got = [0, 0, 0], [[], [], []]
    for news in ([1, 0, 20], [70, 60, 1], [1, 1, 1], [1, 1, 1], [77, 35, 10]):
        step = cache.step(news)
        out = m.forward_paged(torch.cat([i[d:d + n] for i, d, n in zip(ids, done, news)]), cache, step)
        for s, part in enumerate(out.split(news)):
            got[s].append(part)
            done[s] += news[s]
    assert done == lens
    for a, b in zip(got, want):
        a = torch.cat(a)
        # f32 products of two orders through three blocks: 1e-5 of the operator's bar in each, logits of size 1
        assert (a - b).abs().max() <= 1e-4 * b.abs().max()
    assert _native.lib().ca_device_status(0) == 0


@pytest.mark.parametrize("kw", [{}, GENERAL])
def test_generate_takes_the_forwards_tokens(kw):
    m = model(seed=3, **kw)
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 256, (n,), generator=g) for n in (1, 17, 64, 65)]
    new = m.generate(prompts, 20, page_size=16)
    assert new.shape == (4, 20)
    for p, n in zip(prompts, new):
        seq = torch.cat((p.cuda(), n))
        with torch.no_grad():
            logits = m(seq[None])["logits"][0]
        best = logits.amax(-1)
        chosen = logits.gather(1, seq.roll(-1)[:, None])[:, 0]
        rows = slice(len(p) - 1, len(seq) - 1)
        # the chosen token is the forward's best, or within the two sides' rounding of it
        assert (best[rows] - chosen[rows] <= 2e-4 * logits.abs().max()).all()
    assert torch.equal(m.generate(prompts, 20, page_size=16), new)
    assert _native.lib().ca_device_status(0) == 0


def test_generate_under_autocast_and_drawn():
    m = model(seed=4)
    prompts = [[1, 2, 3], [9] * 40]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert m.make_cache(1).k.dtype == torch.bfloat16
        a = m.generate(prompts, 8)
        gens = [torch.Generator("cuda").manual_seed(5) for _ in range(2)]
        b, c = (m.generate(prompts, 8, temperature=1.5, generator=g) for g in gens)
    assert a.shape == b.shape == (2, 8) and torch.equal(b, c) and ((a >= 0) & (a < 256)).all()
    assert m.generate(prompts, 1).shape == (2, 1)


def test_generate_refusals():
    m = model()
    for bad in (dict(prompts=[], max_new_tokens=3), dict(prompts=[[1], []], max_new_tokens=3),
                dict(prompts=[[1]], max_new_tokens=0), dict(prompts=[[1] * 150], max_new_tokens=12),
                dict(prompts=[[1]], max_new_tokens=3, temperature=-1.0)):
        with pytest.raises(ValueError):
            m.generate(**bad)
    with pytest.raises(ValueError, match="packed"):
        m.forward_paged(torch.zeros(1, 3, dtype=torch.long, device="cuda"), m.make_cache(1), None)


def test_training_with_general_rotary_positions():
    """Runs, and its gradient is that of differences along a random direction."""
    m = model(seed=6, **GENERAL)
    g = torch.Generator().manual_seed(7)
    ids = torch.randint(0, 256, (2, 60), generator=g).cuda()
    loss = m(ids, ids)["loss"]
    loss.backward()
    w = m.blocks[1].attn.qkv.weight
    direction = torch.randn(w.shape, generator=g).cuda() * w.grad.abs().mean().sqrt()
    slope = (w.grad.double() * direction.double()).sum().item()
    eps, values = 2e-2 / direction.norm().item(), []
    with torch.no_grad():
        for e in (eps, -eps):
            w.add_(direction, alpha=e)
            values.append(m(ids, ids)["loss"].double().item())
            w.add_(direction, alpha=-e)
    # a loss of 5.5 in 32 bits is good to 5e-7; the step's square to 1e-3 of the slope
    assert abs((values[0] - values[1]) / (2 * eps) - slope) <= 1e-6 / eps + 2e-2 * abs(slope)
