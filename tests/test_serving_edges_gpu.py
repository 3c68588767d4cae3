"""The serving operators where neighbouring work, unusual numbers or unusual
settings could change what they answer: other kernels beside a call, streams
that change, outliers, NaN and infinities, long heads, rows of equal logits."""

from __future__ import annotations

import numpy as np
import pytest

from test_serving_gpu import run_sample, sample_check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch_mod(cuda_lib):
    import torch
    torch.cuda.set_device(0)
    return torch


@pytest.fixture(scope="module")
def eng(pkg, torch_mod):
    e = pkg.Engine(0)
    yield e
    e.close()


def make_cache(torch, pkg, lens, hkv, d, page, dtype, seed):
    """A pool of random rows, every sequence's pages in random order."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    cols = max(1, max(-(-n // page) for n in lens))
    n_pages = len(lens) * cols
    k = torch.randn(n_pages, hkv, page, d, generator=gen, device="cuda").to(dtype)
    v = torch.randn(n_pages, hkv, page, d, generator=gen, device="cuda").to(dtype)
    table = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32).view(len(lens), cols)
    return pkg.PagedKV(k, v, table, torch.tensor(lens, dtype=torch.int32, device="cuda"))


def cache_rows(cache, b, n):
    """k and v of the first n slots of sequence b in 64 bits, [n_head_kv, n, head_dim]."""
    page = cache.page_size
    pages = cache.table[b, :-(-n // page)].long()
    return tuple(x[pages].double().transpose(0, 1).reshape(cache.n_head_kv, -1, cache.head_dim)[:, :n]
                 for x in (cache.k, cache.v))


def attend_ref(torch, cache, lens, q, scale=None):
    """softmax(scale q K^T) V and the log-sums in 64 bits."""
    b, h, d = q.shape
    out = torch.zeros(b, h, d, dtype=torch.float64, device="cuda")
    lse = torch.full((b, h), -np.inf, dtype=torch.float64, device="cuda")
    for i, n in enumerate(lens):
        if n == 0:
            continue
        k, v = cache_rows(cache, i, n)
        s = (scale or d ** -0.5) * (q[i].double().view(cache.n_head_kv, -1, d) @ k.transpose(1, 2))
        out[i] = (torch.softmax(s, 2) @ v).view(h, d)
        lse[i] = torch.logsumexp(s, 2).view(h)
    return out, lse


# ------------------------------------------------------------------ streams

def test_engine_opened_beside_a_busy_default_stream(torch_mod, pkg):
    """The first call does not wait for the legacy default stream, and the scratch it needs is ready."""
    torch = torch_mod
    lens = [5000, 3000]
    cache = make_cache(torch, pkg, lens, 2, 64, 16, torch.float16, seed=1)
    q = torch.randn(2, 8, 64, device="cuda")
    want, _ = attend_ref(torch, cache, lens, q)
    out, stream = torch.zeros_like(q), torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(100_000_000)              # of clock cycles: some 50 ms
    e = pkg.Engine(0, stream=stream.cuda_stream)
    for _ in range(3):
        e.kv_attend(cache, q, out)
    e.sync()
    torch.cuda.synchronize()
    assert (out.double() - want).abs().max() < 1e-5
    e.close()


def test_calls_on_two_streams_follow_one_another(torch_mod, pkg):
    """One engine, two caches, a stream each: the second stream's call waits for the first one's, whose scratch it
    shares; the same with the first call in a graph."""
    torch = torch_mod
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    e = pkg.Engine(0, stream=streams[0].cuda_stream)
    lens = [[9000, 70], [20000, 12, 5000]]      # heads that are split over CTAs
    caches = [make_cache(torch, pkg, n, 2, 64, 16, torch.float16, seed=i) for i, n in enumerate(lens)]
    qs = [torch.randn(len(n), 8, 64, device="cuda") for n in lens]
    want = [attend_ref(torch, c, n, q)[0] for c, n, q in zip(caches, lens, qs)]
    outs = [torch.zeros_like(q) for q in qs]
    ws = [torch.zeros(c.batch, 2, c.capacity, device="cuda") for c in caches]

    def call(i):
        e.kv_attend(caches[i], qs[i], outs[i], weights_out=ws[i])

    torch.cuda.synchronize()
    call(1), call(0)
    e.sync()
    e.capture_begin()
    call(0)
    g = e.capture_end()
    for first in (lambda: call(0), g.launch):
        for turn in range(5):
            for t in outs:
                t.zero_()
            torch.cuda.synchronize()
            with torch.cuda.stream(streams[0]):
                torch.cuda._sleep(20_000_000)   # of clock cycles: some 10 ms
            e.set_stream(streams[0].cuda_stream)
            first()
            e.set_stream(streams[1].cuda_stream)
            call(1)
            ended = torch.cuda.Event()
            ended.record(streams[1])
            assert not ended.query()            # it waits for the sleeping stream's call
            torch.cuda.synchronize()
            for o, w in zip(outs, want):
                assert (o.double() - w).abs().max() < 1e-5
    # recording on a stream that the engine comes to in the middle
    e.set_stream(streams[0].cuda_stream)
    call(0)
    graph = torch.cuda.CUDAGraph()
    outs[1].zero_()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=streams[1]):
        e.set_stream(streams[1].cuda_stream)
        call(1)
    e.set_stream(streams[0].cuda_stream)
    call(0)
    e.sync()
    graph.replay()
    torch.cuda.synchronize()
    assert (outs[1].double() - want[1]).abs().max() < 1e-5
    g.close()
    e.close()


def test_generate_sampled_leaves_the_engine_on_its_stream(torch_mod, pkg):
    """Also where it ends with an error."""
    from llm_kv260_b200 import model
    torch = torch_mod
    m = model.synth_model(dict(n_layer=1, n_embd=512, n_ff=1024, n_head=8, n_head_kv=2, head_dim=64, n_vocab=1024,
                               rope_base=500000.0, rms_eps=1e-5), seed=5)
    dec = pkg.Decoder(m, device=0, ctx_max=16)
    e = pkg.Engine(0, stream=torch.cuda.Stream().cuda_stream)
    at = e.stream
    u = np.full(3, 0.5, np.float32)
    a, _ = dec.generate_sampled([1, 2], 3, u, engine=e)
    assert e.stream == at != torch.cuda.current_stream().cuda_stream
    with pytest.raises(pkg.B200Error):
        dec.generate_sampled([1, 1 << 30], 3, u, engine=e)     # no such token
    assert e.stream == at
    b, _ = dec.generate_sampled([1, 2], 3, u)
    assert np.array_equal(a, b)
    e.close()
    dec.close()


# ------------------------------------------------------------------ workspace

def wide_cache(torch, pkg, batch, columns, hkv=8):
    """Sequences of one page each under tables of many columns: little memory, a large workspace with weights."""
    k = torch.randn(batch, hkv, 16, 64, device="cuda").half()
    table = torch.full((batch, columns), -1, dtype=torch.int32, device="cuda")
    table[:, 0] = torch.arange(batch, device="cuda")
    cache = pkg.PagedKV(k, torch.randn_like(k), table, torch.full((batch,), 16, dtype=torch.int32, device="cuda"))
    return cache, torch.zeros(batch, hkv, cache.capacity, device="cuda")


def test_a_grown_workspace_replaces_the_smaller_one(torch_mod, pkg):
    """Without graphs an engine holds little more than its largest call needs."""
    import ctypes
    torch = torch_mod
    e = pkg.Engine(0, stream=torch.cuda.Stream().cuda_stream)
    batch, h = 16, 32
    q = torch.randn(batch, h, 64, device="cuda")
    outs = [torch.zeros_like(q) for _ in range(3)]
    calls = [wide_cache(torch, pkg, batch, columns) for columns in (1000, 1010, 1100)]
    for cache, _ in calls:
        cache.k.copy_(calls[0][0].k), cache.v.copy_(calls[0][0].v)
    need = pkg.lib().b200_kv_attend_workspace(ctypes.byref(calls[2][0].c), h, 1)
    assert need > 32 << 20
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for out, (cache, w) in zip(outs, calls):
        e.kv_attend(cache, q, out, weights_out=w)
    e.sync()
    assert torch.cuda.memory_allocated() - before <= 1.25 * need
    want, _ = attend_ref(torch, calls[0][0], [16] * batch, q)
    for out in outs:
        assert (out.double() - want).abs().max() < 1e-5
    e.close()


def test_a_workspace_does_not_grow_in_a_capture(torch_mod, pkg):
    """A recorded call that needs more than the engine has is refused, and the recording goes on."""
    torch = torch_mod
    stream = torch.cuda.Stream()
    e = pkg.Engine(0, stream=stream.cuda_stream)
    (small, w0), (large, w1) = wide_cache(torch, pkg, 2, 10), wide_cache(torch, pkg, 64, 3000)
    q0, q1 = torch.randn(2, 32, 64, device="cuda"), torch.randn(64, 32, 64, device="cuda")
    out0, out1 = torch.zeros_like(q0), torch.zeros_like(q1)
    torch.cuda.synchronize()
    e.kv_attend(small, q0, out0, weights_out=w0)
    e.sync()
    want = out0.clone()
    out0.zero_()
    torch.cuda.synchronize()
    e.capture_begin()
    e.kv_attend(small, q0, out0, weights_out=w0)
    with pytest.raises(RuntimeError, match="captur"):
        e.kv_attend(large, q1, out1, weights_out=w1)
    g = e.capture_end()
    e.kv_attend(large, q1, out1, weights_out=w1)
    filler = [torch.full((1 << 20,), 7.0, device="cuda") for _ in range(16)]      # what would take a freed workspace
    torch.cuda.synchronize()
    g.launch()
    e.sync()
    assert torch.equal(out0, want)
    assert all(bool((f == 7.0).all()) for f in filler)
    assert (out1.double() - attend_ref(torch, large, [16] * 64, q1)[0]).abs().max() < 1e-5
    g.close()
    e.close()


# ------------------------------------------------------------------ append

LOW, HIGH = -2 ** 31, 2 ** 31 - 1


@pytest.mark.parametrize("offsets", [[LOW, 2, 4, HIGH, 10], [HIGH] * 5, [LOW] * 5, [5, 5, 6, 6, 6], [-HIGH, -7, 3, 3, 4],
                                     [LOW, LOW, LOW, LOW, HIGH], [0, 9, 9, 9, 7], [0, 3, 3, 7, 8]])
@pytest.mark.parametrize("in_place", [False, True])
def test_append_offsets_out_of_range(torch_mod, pkg, eng, offsets, in_place):
    """Offsets below 0 or past the rows: what there is of each sequence's rows is appended, nothing else written."""
    torch = torch_mod
    n, b, page, hkv, d = 8, 4, 16, 2, 64
    lens = [0, 31, 40, 2]                       # of 32 slots: the second sequence has one free, the third none
    table = torch.arange(2 * b, dtype=torch.int32, device="cuda").view(b, 2)
    k = torch.randn(2 * b, hkv, page, d, device="cuda").half()
    v = torch.randn_like(k)
    cache = pkg.PagedKV(k, v, table, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    kn, vn = torch.randn(n, hkv, d, device="cuda").half(), torch.randn(n, hkv, d, device="cuda").half()
    seen = torch.tensor([7, 8, 9, 10], dtype=torch.int32, device="cuda")
    pos = torch.full((b, hkv, 32), -9, dtype=torch.int32, device="cuda")
    w = torch.full((b, hkv, 32), -9.0, device="cuda")
    off = [min(max(x, 0), n) for x in offsets]
    want_k, want_v, want_pos, want_w = k.clone(), v.clone(), pos.clone(), w.clone()
    want_len, want_seen = [], []
    for i in range(b):
        at, m = min(lens[i], 32), max(off[i + 1] - off[i], 0)
        want_len.append(min(at + m, 32))
        want_seen.append(7 + i + m)
        for j in range(m):
            if at + j < 32:
                pg, s = 2 * i + (at + j) // page, (at + j) % page
                want_k[pg, :, s], want_v[pg, :, s] = kn[off[i] + j], vn[off[i] + j]
                want_pos[i, :, at + j], want_w[i, :, at + j] = 7 + i + j, 0.0
    out = {} if in_place else dict(lengths_out=torch.zeros_like(seen), seen_out=torch.zeros_like(seen))
    torch.cuda.synchronize()
    eng.kv_append(cache, kn, vn, offsets=torch.tensor(offsets, dtype=torch.int32, device="cuda"), seen=seen,
                  positions=pos, weights=w, **out)
    eng.sync()
    assert torch.equal(k, want_k) and torch.equal(v, want_v)
    assert torch.equal(pos, want_pos) and torch.equal(w, want_w)
    assert out.get("lengths_out", cache.lengths).tolist() == want_len
    assert out.get("seen_out", seen).tolist() == want_seen


# ------------------------------------------------------------------ attention

@pytest.mark.parametrize("ratio", [1.0, 128.0, 4096.0, 30000.0])
def test_attend_with_outliers_among_the_query(torch_mod, pkg, eng, ratio):
    """A float32 query whose largest element, in a channel where all keys are 0, is `ratio` times the others: the
    others keep their bits. A score is a float32 dot product: off by (d + 16) half units of sum |q k| at most, of the
    channels that are not 0."""
    torch = torch_mod
    lens, d = [400, 1000], 128
    cache = make_cache(torch, pkg, lens, 2, d, 16, torch.float16, seed=11)
    cache.k[..., 17] = 0.0
    gen = torch.Generator(device="cuda").manual_seed(3)
    q = 1.5 * torch.randn(2, 8, d, generator=gen, device="cuda")
    q[..., 17] = 3.0 * ratio * torch.where(torch.arange(8, device="cuda") % 2 == 0, 1.0, -1.0)
    out, lse = torch.empty_like(q), torch.empty(2, 8, device="cuda")
    torch.cuda.synchronize()
    eng.kv_attend(cache, q, out, lse, scale=1.0)
    eng.sync()
    want, want_lse = attend_ref(torch, cache, lens, q, scale=1.0)
    for i, n in enumerate(lens):
        k, v = cache_rows(cache, i, n)
        sabs = (q[i].double().abs().view(2, 4, d) @ k.abs().transpose(1, 2)).amax(2).view(8)
        eps = (d + 16) * 2.0 ** -24 * sabs
        assert bool(((lse[i].double() - want_lse[i]).abs() <= eps + 2.0 ** -22 * want_lse[i].abs()).all())
        tol = v.abs().max() * (2 * eps + (64 + n / 16) * 2.0 ** -24 + 2.0 ** -20)
        assert bool(((out[i].double() - want[i]).abs() <= tol[:, None] + 2.0 ** -23 * want[i].abs()).all())


TYPES = {"f32_f16": ("float32", "float16"), "f16": ("float16", "float16"), "bf16": ("bfloat16", "bfloat16"),
         "f32": ("float32", "float32")}


@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("lens", [[1, 40], [9, 5000]])
def test_attend_with_a_query_that_is_not_a_number(torch_mod, pkg, eng, types, value, lens):
    """Scores that are NaN make the head NaN, and only that head: it does not look like an empty cache. (An infinite
    query element meets positive keys: scores of +infinity.)"""
    torch = torch_mod
    qt, kt = (getattr(torch, t) for t in TYPES[types])
    cache = make_cache(torch, pkg, lens, 2, 64, 16, kt, seed=12)
    q = torch.randn(2, 8, 64, device="cuda").to(qt)
    want, want_lse = attend_ref(torch, cache, lens, q)
    q[0, 1, 5] = q[1, 7, 63] = value
    if value == float("inf"):
        cache.k[..., 5] = cache.k[..., 63] = 1.0
        want, want_lse = attend_ref(torch, cache, lens, q)
    out, lse = torch.zeros_like(q), torch.zeros(2, 8, device="cuda")
    w = torch.zeros(2, 2, cache.capacity, device="cuda")
    torch.cuda.synchronize()
    eng.kv_attend(cache, q, out, lse, weights_out=w)
    eng.sync()
    bad = torch.zeros(2, 8, dtype=torch.bool, device="cuda")
    bad[0, 1] = bad[1, 7] = True
    assert bool(out[bad].isnan().all()) and bool(lse[bad].isnan().all())
    assert bool(((out.double() - want)[~bad].abs() <= 0.02).all()) and bool(((lse.double() - want_lse)[~bad].abs() <= 0.02).all())
    # the weights of the cache heads that the two query heads read are NaN, the others are not
    for i, n in enumerate(lens):
        assert bool(w[i, i, :n].isnan().all()) and bool(w[i, 1 - i, :n].isfinite().all())


@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("lens", [[17, 64], [3000, 77]])
def test_attend_with_infinite_keys(torch_mod, pkg, eng, types, lens):
    """A key row with an infinite element (a value that float16 does not hold) has a score of -infinity where the
    query's element is of the other sign: it weighs nothing and the head is that of the other rows. Where it is of the
    same sign the head is not a number; where a row's infinities cancel, too."""
    torch = torch_mod
    qt, kt = (getattr(torch, t) for t in TYPES[types])
    cache = make_cache(torch, pkg, lens, 1, 64, 16, kt, seed=13)
    q = torch.randn(2, 4, 64, device="cuda").to(qt)
    q[..., 7] = 1.0
    q[..., 9] = -0.5
    rows = {0: [3, lens[0] - 1], 1: [0, 15, 40]}

    def place(i, s):
        return cache.table[i, s // 16].item(), 0, s % 16

    for i, slots in rows.items():
        for s in slots:
            cache.k[place(i, s)][7] = -float("inf")
            cache.k[place(i, s)][9] = float("inf")
    out, lse = torch.zeros_like(q), torch.zeros(2, 4, device="cuda")
    w = torch.zeros(2, 1, cache.capacity, device="cuda")
    torch.cuda.synchronize()
    eng.kv_attend(cache, q, out, lse, weights_out=w)
    eng.sync()
    tol = 2e-5 if types == "f32_f16" or types == "f32" else 2e-3 if types == "f16" else 1.6e-2
    for i, n in enumerate(lens):
        k, v = cache_rows(cache, i, n)
        live = torch.ones(n, dtype=torch.bool, device="cuda")
        live[rows[i]] = False
        s = 0.125 * (q[i].double().view(1, 4, 64) @ k[:, live].transpose(1, 2))
        want = (torch.softmax(s, 2) @ v[:, live])[0]
        assert bool(((out[i].double() - want).abs() <= tol).all())
        assert bool(((lse[i].double() - torch.logsumexp(s, 2)[0]).abs() <= 2e-5).all())
        assert bool((w[i, 0, :n][~live] == 0).all()) and bool((w[i, 0, :n][live] > 0).all())
    cache.k[place(0, 5)][7] = float("inf")      # a score of +infinity
    cache.k[place(1, 15)][9] = -float("inf")    # -infinity and infinity
    torch.cuda.synchronize()
    eng.kv_attend(cache, q, out, lse)
    eng.sync()
    assert bool(out.isnan().all()) and bool(lse.isnan().all())


def test_attend_16_bit_outputs_of_long_heads_lean_to_neither_side(torch_mod, pkg, eng):
    """131072 slots of positive values and so many heads that few are split: over some thousand units added up by a warp
    float16 outputs are as often above the exact ones as below. (Sums that are cut off at each unit pull all of them down,
    by a fifth of a unit.) Scores spread by 2 leave some 2400 slots that count, so outputs differ by several units
    between heads and round independently: the mean error of 32768 of them is below 2^-17 of the values, over five times
    what the rounding leaves (a unit / sqrt(12 * 32768)); the weights' 22 bits and the 32-bit sums are far below."""
    torch = torch_mod
    b, hkv, n, d, page = 64, 8, 131072, 64, 1024
    k = torch.randn(n // page, hkv, page, d, device="cuda").half()
    v = (1.2 + 0.3 * torch.rand(hkv, 1, d, device="cuda") + 0.5 * torch.rand(n // page, hkv, page, d, device="cuda")).half()
    table = torch.arange(n // page, dtype=torch.int32, device="cuda").repeat(b, 1)
    cache = pkg.PagedKV(k, v, table, torch.full((b,), n, dtype=torch.int32, device="cuda"))
    q = (2 * torch.randn(b, hkv, d, device="cuda")).half()
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    eng.kv_attend(cache, q, out)
    eng.sync()
    kk, vv = (x.double().transpose(0, 1).reshape(hkv, n, d) for x in (k, v))
    lean = 0.0
    for i in range(0, b, 8):
        s = 0.125 * (q[i:i + 8].double().transpose(0, 1) @ kk.transpose(1, 2))      # head, sequence, slot
        want = (torch.softmax(s, 2) @ vv).transpose(0, 1)
        lean += float(((out[i:i + 8].double() - want) / want).mean()) * 8 / b
    assert abs(lean) <= 2.0 ** -17


def test_attend_float32_error_over_many_units(torch_mod, pkg, eng):
    """32 heads of 8000 float32 slots: the error's norm against 64 bits is below 1e-6 of the output's, which sums that
    are cut off instead of rounded miss (2.0e-6)."""
    torch = torch_mod
    lens = [8000] * 8
    cache = make_cache(torch, pkg, lens, 4, 128, 64, torch.float32, seed=14)
    q = 1.5 * torch.randn(8, 16, 128, device="cuda")
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    eng.kv_attend(cache, q, out)
    eng.sync()
    want, _ = attend_ref(torch, cache, lens, q)
    err = float((out.double() - want).norm() / want.norm())
    assert err <= 1e-6


# ------------------------------------------------------------------ eviction

@pytest.mark.parametrize("kv,q", [("float16", "float32"), ("bfloat16", "bfloat16"), ("float32", "float32")])
@pytest.mark.parametrize("page", [16, 7])
def test_attention_after_evictions_is_that_over_the_kept_tokens(torch_mod, pkg, eng, kv, q, page):
    """Append, attend with weights and evict in turn, as a server does: each attention is the softmax over the tokens
    whose positions are left, from rows kept aside as they were appended; and those are the ones the weights name."""
    torch = torch_mod
    kt, qt = getattr(torch, kv), getattr(torch, q)
    b, hkv, h, d, budget, recent, sinks = 3, 2, 8, 64, 40, 9, 3
    cols = -(-(budget + 60) // page)
    gen = torch.Generator(device="cuda").manual_seed(page)
    k = torch.zeros(b * cols, hkv, page, d, dtype=kt, device="cuda")
    table = torch.randperm(b * cols, generator=gen, device="cuda").to(torch.int32).view(b, cols)
    cache = pkg.PagedKV(k, torch.zeros_like(k), table, torch.zeros(b, dtype=torch.int32, device="cuda"))
    seen = torch.zeros(b, dtype=torch.int32, device="cuda")
    w = torch.zeros(b, hkv, cache.capacity, device="cuda")
    pos = torch.zeros(b, hkv, cache.capacity, dtype=torch.int32, device="cuda")
    rows = [[torch.zeros(0, hkv, d, dtype=kt, device="cuda")] * b for _ in "kv"]       # every token's, in order
    tol = 2e-5 if qt == torch.float32 else 1.6e-2
    for news in ([60, 3, 41], [1, 1, 1], [0, 50, 1], [7, 1, 30], [1, 1, 1]):
        off = torch.tensor(np.concatenate([[0], np.cumsum(news)]), dtype=torch.int32, device="cuda")
        kn, vn = (torch.randn(sum(news), hkv, d, generator=gen, device="cuda").to(kt) for _ in "kv")
        qq = (1.5 * torch.randn(b, h, d, generator=gen, device="cuda")).to(qt)
        out, lse = torch.zeros_like(qq), torch.zeros(b, h, device="cuda")
        torch.cuda.synchronize()
        eng.kv_append(cache, kn, vn, offsets=off, seen=seen, positions=pos, weights=w)
        eng.kv_attend(cache, qq, out, lse, weights=w, weights_out=w, decay=0.9)
        eng.sync()
        old_pos, old_w, lens = pos.clone(), w.clone(), cache.lengths.tolist()
        for i in range(b):
            for side, new in zip(rows, (kn, vn)):
                side[i] = torch.cat([side[i], new[off[i]:off[i + 1]]])
            for j in range(hkv):
                at = pos[i, j, :lens[i]].long()
                kk, vv = (side[i][at, j].double() for side in rows)
                s = d ** -0.5 * (qq[i, 4 * j:4 * j + 4].double() @ kk.T)
                assert bool(((out[i, 4 * j:4 * j + 4].double() - torch.softmax(s, 1) @ vv).abs() <= tol).all())
                assert bool(((lse[i, 4 * j:4 * j + 4].double() - torch.logsumexp(s, 1)).abs() <= 2e-5).all())
        eng.kv_evict(cache, w, pos, seen, budget, recent=recent, sinks=sinks)
        eng.sync()
        for i in range(b):
            n, m = lens[i], min(lens[i], budget)
            assert cache.lengths[i].item() == m and seen[i].item() == rows[0][i].shape[0]
            for j in range(hkv):
                at, weight = old_pos[i, j, :n], old_w[i, j, :n]
                fixed = (at >= seen[i] - recent) | (at < sinks)
                order = torch.sort(torch.where(fixed, np.inf, weight), descending=True, stable=True).indices[:m]
                kept = dict(zip(at[order].tolist(), weight[order].tolist()))
                assert kept == dict(zip(pos[i, j, :m].tolist(), w[i, j, :m].tolist()))


# ------------------------------------------------------------------ sampling

@pytest.mark.parametrize("n", [20000, 50257, 128256])
def test_sample_beside_other_kernels(torch_mod, pkg, n):
    """CTAs of a cluster that start at different times, on SMs that other kernels keep busy: the tokens are those of
    a GPU that does nothing else. A row of 20000 float32 has two CTAs and more."""
    torch = torch_mod
    gen = torch.Generator(device="cuda").manual_seed(n)
    b = 96
    x = 2.5 * torch.randn(b, n, generator=gen, device="cuda")
    u = torch.rand(b, generator=gen, device="cuda")
    rows = torch.arange(b, device="cuda")
    kw = dict(temperature=torch.where(rows % 4 == 0, 0.0, 0.9), top_k=torch.where(rows % 4 == 1, 50, 0).int(),
              top_p=torch.where(rows % 4 == 2, 0.8, 1.0), min_p=torch.zeros(b, device="cuda"))
    stream, busy = torch.cuda.Stream(), torch.cuda.Stream()
    e = pkg.Engine(0, stream=stream.cuda_stream)
    quiet, lp = torch.empty(b, dtype=torch.int32, device="cuda"), torch.empty(b, device="cuda")
    torch.cuda.synchronize()
    e.sample(x, u, quiet, lp, **kw)
    e.sync()
    assert torch.equal(quiet[0::4].long(), x[0::4].argmax(1))
    y = torch.randn(1 << 22, device="cuda")
    token = torch.empty(20, b, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(busy):
        for _ in range(200):
            y = y * 1.0001
    for i in range(20):
        e.sample(x, u, token[i], lp, **kw)
    torch.cuda.synchronize()
    assert all(torch.equal(t, quiet) for t in token)
    e.close()


def equal_logits(kind, n, rng):
    """Rows in which many logits are equal: more of them than a list of candidates holds."""
    if kind == "all":
        return np.full(n, -1.25, np.float32)
    if kind == "all_but_few":                   # a few above the rest, a few far below
        x = np.full(n, 0.5, np.float32)
        x[rng.choice(n, 3, replace=False)] = [2.0, 2.0, 0.75]
        x[rng.choice(n, 9, replace=False)] = -30.0
        return x
    if kind == "three":
        return rng.choice(np.array([1.0, 0.0, -1.5], np.float32), n)
    if kind == "five_near":                     # within one bin of distance from the top, and one bit of each other
        return rng.choice(np.array([3.0, np.nextafter(np.float32(3), np.float32(4)), 2.9999, 2.99, -8.0], np.float32), n)
    if kind == "infinite":
        x = rng.standard_normal(n).astype(np.float32)
        x[rng.random(n) < 0.4] = np.inf
        x[rng.random(n) < 0.1] = -np.inf
        return x
    x = np.where(rng.random(n) < 0.5, -np.inf, 0.0).astype(np.float32)     # "masked"
    x[rng.random(n) < 0.1] = np.nan
    return x


@pytest.mark.parametrize("kind", ["all", "all_but_few", "three", "five_near", "infinite", "masked"])
@pytest.mark.parametrize("n,dtype", [(50257, "f32"), (50257, "bf16"), (128256, "f32")])
@pytest.mark.parametrize("k", [0, 5, 40, 2048, 2049, 30000])
def test_sample_rows_of_equal_logits(torch_mod, eng, kind, n, dtype, k):
    """The cut falls among more equal logits than a list of candidates holds: of those, the lowest indexes stay."""
    rng = np.random.default_rng(n + k)
    settings = [(p, m, t) for p in (1.0, 0.5, 0.97) for m in (0.0, 0.3) for t in (1.0, 0.6)]
    b = 2 * len(settings)
    p, m, t = (np.array([s[j] for s in settings] * 2, np.float32) for j in range(3))
    x = np.stack([equal_logits(kind, n, rng) for _ in range(b)])
    u = rng.random(b).astype(np.float32)
    u[0], u[1] = 0.0, np.float32(1 - 2.0 ** -24)
    got = run_sample(torch_mod, eng, x, u, t, [k] * b, p, m, dtype, stride=3)
    for i in range(b):
        sample_check(got[0][i], t[i], k, p[i], m[i], u[i], int(got[1][i]), got[2][i])
    again = run_sample(torch_mod, eng, x, u, t, [k] * b, p, m, dtype, stride=3)
    assert np.array_equal(got[1], again[1]) and np.array_equal(got[2], again[2])
