"""The decoder answering, in the ways around its plain run: grad modes, threads, prompts' forms."""
import threading

import pytest
import torch

from continuum_attention_b200 import _native, continuum_attention_paged
from continuum_attention_b200.decoder import ContinuumDecoderConfig, ContinuumDecoderLM
from paged_testlib import arguments, make_case

pytestmark = pytest.mark.gpu


def model(seed=0, **kw):
    torch.manual_seed(seed)
    cfg = ContinuumDecoderConfig(**{**dict(block_size=96, d_model=256, n_heads=4, n_layers=2), **kw})
    return ContinuumDecoderLM(cfg).cuda()


@pytest.mark.parametrize("kw", [dict(rope_theta=4321.0), dict(rope_theta=4321.0, rope_layout="half", rope_dim=32)])
def test_generate_in_inference_mode_then_training(kw):
    """The first use of a table is in inference mode, its second (a whole block) saves it for the gradient."""
    m = model(**kw)
    with torch.inference_mode():
        a = m.generate([[1, 2, 3], [4]], 5)
    ids = torch.arange(96, device="cuda")[None]
    m(ids, ids)["loss"].backward()
    assert all(torch.isfinite(p.grad).all() for p in m.parameters())
    assert torch.equal(m.generate([[1, 2, 3], [4]], 5), a)
    assert _native.lib().ca_device_status(0) == 0


def test_a_gain_that_asks_for_a_gradient():
    """Its output is the same, and a backward pass through it says that there is none."""
    c = make_case("bf16", 4, 2, 64, 16, [(1, 20), (2, 5)])
    args = arguments(c)
    plain = continuum_attention_paged(*args, max_q_len=2)
    assert not plain.requires_grad
    gain = args[6].clone().requires_grad_()
    out = torch.empty_like(plain)
    for kw in (dict(), dict(out=out)):
        y = continuum_attention_paged(*args[:6], gain, max_q_len=2, **kw)
        assert torch.equal(y.detach(), plain)
        assert y.data_ptr() == kw.get("out", y).data_ptr() and not out.requires_grad
        y += 0.0
        with pytest.raises(RuntimeError, match="no backward"):
            (y.float().sum() + gain.sum()).backward()
    assert torch.equal(out, plain)
    with torch.no_grad():
        assert not continuum_attention_paged(*args[:6], gain, max_q_len=2).requires_grad


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_generate_in_two_threads(temperature):
    """A capture in one thread bears the other's launches, allocations, copies and draws."""
    m = model(seed=2)
    prompts = [[[1, 2, 3], [4] * 20], [[7] * 9]]
    want = [m.generate(p, 12, page_size=16) for p in prompts]
    barrier, got, errors = threading.Barrier(2), [[], []], []

    def work(t):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(4):
                    barrier.wait(60)
                    got[t].append(m.generate(prompts[t], 12, page_size=16, temperature=temperature))
                torch.cuda.current_stream().synchronize()
        except BaseException as e:
            errors.append(e)
            barrier.abort()

    threads = [threading.Thread(target=work, args=(t,)) for t in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for t in range(2):
        assert len(got[t]) == 4
        for g in got[t]:
            assert g.shape == want[t].shape and ((g >= 0) & (g < 256)).all()
            if temperature == 0:
                assert torch.equal(g, want[t])
    assert _native.lib().ca_device_status(0) == 0


def test_prompts_as_a_tensor():
    m = model(seed=5)
    ids = torch.arange(12).view(3, 4)
    want = m.generate([p.tolist() for p in ids], 6)
    for form in (ids, ids.cuda(), ids.to(torch.uint8), ids.numpy(), list(ids.cuda())):
        assert torch.equal(m.generate(form, 6), want)


@pytest.mark.parametrize("autocast", [False, True])
def test_a_step_without_tokens(autocast):
    m = model(seed=6)
    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
        cache = m.make_cache(2, page_size=16)
        first = m.forward_paged(torch.tensor([1, 2, 3], device="cuda"), cache, cache.step([3, 0]))
        kept = cache.k.clone()
        none = m.forward_paged(torch.zeros(0, dtype=torch.long, device="cuda"), cache, cache.step([0, 0]))
    assert first.shape == (3, 256) and none.shape == (0, 256)
    assert torch.equal(cache.k, kept) and cache.lens == [3, 0]
    assert _native.lib().ca_device_status(0) == 0
