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
    """More requests than rows, and at times more than there are pages for: every request gets its tokens, all pages come
    back, and a run repeats to the token."""
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
    again = example.ChunkServer(m, 4, pages=13, page=8, columns=16).serve(prompts, 10, chunk=16)
    assert again == runs[2]                              # and repeat to the token
    with pytest.raises(RuntimeError):
        example.ChunkServer(m, 1, pages=3, page=8, columns=16).serve(prompts[:1], 2, chunk=64)


def step_case(torch, pkg, seed, batch=5, hkv=2, h=4, d=64, page=16, cols=20, pages=60, n=120):
    """What a step of one layer holds: a pool with some pages handed out, tokens to come, and outputs of fixed size."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device="cuda").to(dtype)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    k = normal(pages, hkv, page, d, dtype=torch.float16)
    v = normal(pages, hkv, page, d, dtype=torch.float16)
    table = torch.full((batch, cols), -1, dtype=torch.int32, device="cuda")
    s = dict(cache=pkg.PagedKV(k, v, table, ints([0] * batch)), held=ints([0] * batch),
             free=torch.arange(pages, device="cuda", dtype=torch.int32), free_count=ints([pages]), new=ints([0] * batch),
             offsets=ints([0] * (batch + 1)), granted=ints([0] * batch), positions=ints([0] * n),
             slots=torch.zeros(n, dtype=torch.int64, device="cuda"), freqs=pkg.rope_freqs(d).cuda(),
             add=normal(n, h * d), x=normal(n, h * d), w=normal(h * d), q8=torch.zeros(n, h * d * 9 // 8, dtype=torch.uint8, device="cuda"),
             qkv=normal(n, h + 2 * hkv, d), q=torch.zeros(n, h, d, dtype=torch.float16, device="cuda"),
             out=torch.zeros(n, h, d, dtype=torch.float16, device="cuda"), lse=torch.zeros(n, h, device="cuda"), h=h, hkv=hkv)
    return s


def step_run(eng, s):
    h, hkv = s["h"], s["hkv"]
    eng.kv_plan(s["cache"], s["new"], s["held"], s["free"], s["free_count"], s["offsets"], slots=s["slots"],
                positions=s["positions"], granted=s["granted"])
    eng.rms_norm(s["add"], s["w"], residual=s["x"], q8=s["q8"])
    eng.rope(s["positions"], s["freqs"], q=s["qkv"][:, :h], q_out=s["q"], k=s["qkv"][:, h:h + hkv], kv=s["cache"],
             v=s["qkv"][:, h + hkv:], slots=s["slots"])
    eng.kv_attend_chunk(s["cache"], s["q"], s["out"], s["offsets"], lse=s["lse"])


STATE = ("held", "free", "free_count", "offsets", "granted", "positions", "slots", "x", "q8", "q", "out", "lse")


def step_state(s):
    return [s[k].clone() for k in STATE] + [s["cache"].k.clone(), s["cache"].v.clone(), s["cache"].table.clone(),
                                            s["cache"].lengths.clone()]


def test_a_recorded_step(cuda_lib, pkg):
    """A whole step recorded once and replayed with other requests gives what eager steps give, to the bit: prompts, single
    tokens, sequences that end, requests that find no page, fewer tokens than there is room for."""
    import torch
    eager, rec = (step_case(torch, pkg, 3) for _ in range(2))
    requests = [[40, 3, 0, 60, 17], [1, 1, 30, 1, 1], [200, -1, 1, 1, 1], [1, 100, -1, 1, 0], [0, 0, 0, 0, 0], [64, 20, 20, 15, 1]]
    e1, e2 = pkg.Engine(0), pkg.Engine(0)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        e2.set_stream(stream.cuda_stream)
        step_run(e2, rec)                                # no requests: every call once before it is recorded
        rec["x"].copy_(eager["x"])
        e2.capture_begin()
        step_run(e2, rec)
        g = e2.capture_end()
        for new in requests:
            rec["new"].copy_(torch.tensor(new))
            g.launch()
    stream.synchronize()
    for new in requests:
        eager["new"].copy_(torch.tensor(new))
        step_run(e1, eager)
    torch.cuda.synchronize()
    for name, a, b in zip(STATE + ("k", "v", "table", "lengths"), step_state(eager), step_state(rec)):
        assert torch.equal(a, b), name
    assert e1.status() == 0 and e2.status() == 0
    g.close()


def test_two_engines_at_once(cuda_lib, pkg):
    """Two engines on streams of their own, their steps side by side, as if alone."""
    import torch
    alone, a, b = (step_case(torch, pkg, 7) for _ in range(3))
    other = step_case(torch, pkg, 8)
    engines = [pkg.Engine(0) for _ in range(3)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    requests = [[100, 3, 1, 10, 5], [1, 60, 30, 1, 1], [7, 7, 7, 7, 7], [-1, 1, 90, 1, 2]] * 4
    torch.cuda.synchronize()
    for new in requests:
        alone["new"].copy_(torch.tensor(new))
        step_run(engines[2], alone)
    torch.cuda.synchronize()
    news = [[torch.tensor(r, dtype=torch.int32, device="cuda") for r in requests] for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(len(requests)):
        for e, st, s, n in zip(engines, streams, (a, other), news):
            with torch.cuda.stream(st):
                e.set_stream(st.cuda_stream)
                s["new"].copy_(n[i])
                step_run(e, s)
    torch.cuda.synchronize()
    for name, x, y in zip(STATE + ("k", "v", "table", "lengths"), step_state(alone), step_state(a)):
        assert torch.equal(x, y), name
