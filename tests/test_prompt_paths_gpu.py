"""The operators of prompts in chunks where a program uses them: examples/serve_chunks.py against the one-sequence decoder."""

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
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "serve_chunks.py")
    spec = importlib.util.spec_from_file_location("serve_chunks", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("page", [16, 7])
def test_chunks_follow_the_decoder(cuda_lib, pkg, example, page):
    """Every sequence is fed its own decoder's greedy tokens, in chunks of different sizes; behind each chunk the decoder's
    pick is the server's, or within the noise of activations rounded to 8 bits (a step of 1/127 of a block's largest, in
    a sum of independent terms) and of 16-bit attention: far below 5 percent of the logits' spread."""
    from llm_kv260_b200 import model
    m = model.synth_model(HD64, seed=9)
    batch, n = 3, 40
    fed = []
    for b in range(batch):
        prompt = model.random_prompt(30, HD64["n_vocab"], seed=20 + b)
        dec = pkg.Decoder(m, device=0, ctx_max=80)
        toks, _, _ = dec.generate(prompt, n)
        dec.close()
        fed.append(np.concatenate([prompt, toks]).tolist())
    srv = example.ChunkServer(m, batch, pages=64, page=page, columns=16)
    at = [0] * batch
    plan = [(30, 10, 0), (1, 19, 31), (0, 1, 1), (7, 1, 5), (1, 1, 1), (25, 30, 1), (5, 0, 29)]
    for sizes in plan:
        chunks = [fed[b][at[b]:at[b] + s] for b, s in enumerate(sizes)]
        logits, granted = srv.step(chunks)
        assert granted.tolist() == list(sizes)
        x = logits.cpu().numpy()
        for b, s in enumerate(sizes):
            at[b] += s
            if s and at[b] >= 30:
                assert x[b].max() - x[b][fed[b][at[b]]] <= 0.05 * x[b].std()
    assert srv.lengths.tolist() == at
    assert srv.eng.status() == 0


def test_requests_share_a_pool(cuda_lib, pkg, example):
    """More requests than rows, and at times more than there are pages for: the greedy tokens do not depend on either, nor
    on the chunks' size, beyond the roundings' noise in a pick between near equals; all pages come back."""
    from llm_kv260_b200 import model
    m = model.synth_model(HD64, seed=4)
    prompts = [model.random_prompt(k, HD64["n_vocab"], seed=50 + k) for k in (33, 5, 60, 1, 17, 48)]
    runs = []
    for batch, pages, chunk in ((6, 200, 64), (2, 200, 16), (4, 13, 16)):
        srv = example.ChunkServer(m, batch, pages=pages, page=8, columns=16)
        runs.append(srv.serve(prompts, 10, chunk=chunk))
        assert int(srv.free_count) == pages and srv.lengths.tolist() == [0] * batch
        assert sorted(srv.free[:pages].tolist()) == list(range(pages))
    assert all(len(r) == 10 for run in runs for r in run)
    same = np.mean([a == b for x, y in ((0, 1), (0, 2)) for p in range(6) for a, b in zip(runs[x][p], runs[y][p])])
    assert same >= 0.5, same
    again = example.ChunkServer(m, 4, pages=13, page=8, columns=16).serve(prompts, 10, chunk=16)
    assert again == runs[2]                              # and repeat to the token
    with pytest.raises(RuntimeError):
        example.ChunkServer(m, 1, pages=3, page=8, columns=16).serve(prompts[:1], 2, chunk=64)
