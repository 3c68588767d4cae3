"""The serving operators where a program uses them: the decoder with a sampler,
and several sequences with paged caches (examples/serve_paged.py) against the
one-sequence decoder."""

from __future__ import annotations

import importlib.util
import os

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HD64 = dict(n_layer=2, n_embd=512, n_ff=1024, n_head=8, n_head_kv=2, head_dim=64, n_vocab=1024,
            rope_base=500000.0, rms_eps=1e-5)


@pytest.fixture(scope="module")
def example(cuda_lib):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "serve_paged.py")
    spec = importlib.util.spec_from_file_location("serve_paged", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_decoder_with_sampler(cuda_lib, pkg):
    from llm_kv260_b200 import model
    m = model.synth_model(HD64, seed=5)
    prompt = model.random_prompt(6, HD64["n_vocab"], seed=6)
    dec = pkg.Decoder(m, device=0, ctx_max=32)
    want, _, _ = dec.generate(prompt, 12)
    u = np.random.default_rng(1).random(12).astype(np.float32)
    greedy, lp = dec.generate_sampled(prompt, 12, u, temperature=0.0)
    assert np.array_equal(greedy, want) and not lp.any()
    one, lp = dec.generate_sampled(prompt, 12, u, top_k=1)
    assert np.array_equal(one, want) and not lp.any()
    # the sampler reads the decoder's own logits
    assert np.array_equal(dec.logits_tensor().cpu().numpy()[0], dec.logits())
    a, la = dec.generate_sampled(prompt, 12, u, temperature=1.5, top_k=50, top_p=0.9)
    b, lb = dec.generate_sampled(prompt, 12, u, temperature=1.5, top_k=50, top_p=0.9)
    assert np.array_equal(a, b) and np.array_equal(la, lb) and (la <= 0).all()
    for bad in (dict(n_gen=12, u=u[:3]), dict(n_gen=40, u=np.zeros(40, np.float32))):
        with pytest.raises(ValueError):
            dec.generate_sampled(prompt, **bad)
    dec.close()


@pytest.mark.parametrize("page", [16, 7])
def test_paged_sequences_follow_the_decoder(cuda_lib, pkg, example, page):
    """Every sequence is fed its own decoder's greedy tokens; at each step the decoder's pick is the paged server's,
    or within the noise of activations rounded to 8 bits (a step of 1/127 of a block's largest, in a sum of
    independent terms: far below 5 percent of the logits' spread)."""
    import torch
    from llm_kv260_b200 import model
    m = model.synth_model(HD64, seed=9)
    batch, n = 3, 20
    prompts = np.stack([model.random_prompt(5, HD64["n_vocab"], seed=20 + b) for b in range(batch)])
    fed = []
    for b in range(batch):
        dec = pkg.Decoder(m, device=0, ctx_max=32)
        toks, _, _ = dec.generate(prompts[b], n)
        dec.close()
        fed.append(np.concatenate([prompts[b], toks]))
    fed = np.stack(fed)
    srv = example.PagedServer(m, batch, 5 + n, page=page)
    for i in range(5 + n - 1):
        logits = srv.step(torch.from_numpy(fed[:, i]).cuda())
        if i >= 4:
            x = logits.cpu().numpy()
            for b in range(batch):
                assert x[b].max() - x[b][fed[b, i + 1]] <= 0.05 * x[b].std()


def test_paged_sequences_within_a_budget(cuda_lib, pkg, example):
    """A budget that is not reached changes nothing; one that is holds the caches, and the run repeats to the bit."""
    from llm_kv260_b200 import model
    m = model.synth_model(HD64, seed=9)
    prompts = np.stack([model.random_prompt(12, HD64["n_vocab"], seed=30 + b) for b in range(4)])
    kw = dict(temperature=0.8, top_k=40, top_p=0.95, min_p=0.02, seed=3)
    free = example.PagedServer(m, 4, 40).generate(prompts, 24, **kw)
    wide = example.PagedServer(m, 4, 40, budget=39, recent=8, sinks=2).generate(prompts, 24, **kw)
    assert np.array_equal(free, wide)
    runs = []
    for _ in range(2):
        srv = example.PagedServer(m, 4, 21, budget=20, recent=8, sinks=2)
        runs.append(srv.generate(prompts, 24, **kw))
        for c in srv.caches:
            assert c["kv"].lengths.tolist() == [20] * 4 and c["seen"].tolist() == [35] * 4
            pos = c["positions"][:, :, :20].cpu().numpy()
            for b in range(4):
                for h in range(2):
                    have = set(pos[b, h].tolist())
                    assert len(have) == 20 and {0, 1} <= have and set(range(27, 35)) <= have
    assert np.array_equal(runs[0], runs[1])
    with pytest.raises(RuntimeError):
        example.PagedServer(m, 4, 10, page=2).generate(prompts, 2)
