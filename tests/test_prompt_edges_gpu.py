"""The operators that a prompt passes through where neighbouring work, unusual numbers or unusual settings could change
what they answer."""

from __future__ import annotations

import math

import pytest

from test_prompt_gpu import DT, TYPES, U, chunk_case, chunk_exact, chunk_run
from test_prompt_paths_gpu import STATE, step_case, step_run, step_state

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


# ------------------------------------------------------------------ streams

def test_calls_of_a_step_on_two_streams_follow_one_another(torch_mod, pkg):
    """One engine whose stream changes between any two calls of a step: each waits for the one before, whose stream sleeps,
    and reads what it wrote."""
    torch = torch_mod
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    e = pkg.Engine(0, stream=streams[0].cuda_stream)
    s = step_case(torch, pkg, 21)
    h, hkv = s["h"], s["hkv"]
    logits = torch.randn(4, 1000, device="cuda")
    u, token = torch.rand(4, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    s["new"].copy_(torch.tensor([40, 3, 30, 30, 17]))
    calls = (
        lambda: e.kv_plan(s["cache"], s["new"], s["held"], s["free"], s["free_count"], s["offsets"], slots=s["slots"],
                          positions=s["positions"], granted=s["granted"]),
        lambda: e.rms_norm(s["add"], s["w"], residual=s["x"], q8=s["q8"]),
        lambda: e.rope(s["positions"], s["freqs"], q=s["qkv"][:, :h], q_out=s["q"], k=s["qkv"][:, h:h + hkv], kv=s["cache"],
                       v=s["qkv"][:, h + hkv:], slots=s["slots"]),
        lambda: e.kv_attend_chunk(s["cache"], s["q"], s["out"], s["offsets"], lse=s["lse"]),
        lambda: e.sample(logits, u, token))
    live = [s[k] for k in STATE] + [s["cache"].k, s["cache"].v, s["cache"].table, s["cache"].lengths, token]
    fresh = [t.clone() for t in live]
    torch.cuda.synchronize()
    for call in calls:
        call()
    e.sync()
    want = [t.clone() for t in live]
    for asleep in range(len(calls)):
        for t, old in zip(live, fresh):
            t.copy_(old)
        torch.cuda.synchronize()
        for i, call in enumerate(calls):
            stream = streams[i % 2]
            e.set_stream(stream.cuda_stream)
            if i == asleep:
                with torch.cuda.stream(stream):
                    torch.cuda._sleep(20_000_000)        # of clock cycles: some 10 ms
            call()
            if i == asleep + 1:
                ended = torch.cuda.Event()
                ended.record(stream)
                assert not ended.query(), i              # it waits for the sleeping stream's call
        torch.cuda.synchronize()
        for name, a, b in zip(STATE + ("k", "v", "table", "lengths", "token"), live, want):
            assert torch.equal(a, b), (asleep, name)
    assert e.status() == 0
    e.close()


# ------------------------------------------------------------------ values that are not finite

@pytest.mark.parametrize("q,kv", TYPES)
@pytest.mark.parametrize("new,old,low,slots", [
    (200, 100, 0, (20, 150, 299)),       # a unit that all rows see; units that some rows see
    (9, 20000, 10000, (10, 5000)),       # parts of a split tile in which no slot has a weight beside the others'
])
def test_chunk_seen_values_count_however_small_their_weight(torch_mod, pkg, eng, q, kv, new, old, low, slots):
    """A value that is not finite spoils its element in every row that sees it, with a weight of e^-250 beside 1, which
    float32 rounds to 0, as with any other: whichever unit, stretch or part of a tile it falls into."""
    torch = torch_mod
    c = chunk_case(torch, pkg, [new], [old], 4, 2, 64, 16, q, kv, seed=22)
    k, v, table = c["cache"].k, c["cache"].v, c["table"][0]
    c["q"].fill_(1.0)
    k.zero_()
    for s in list(slots) + list(range(low)):
        k[int(table[s // 16]), :, s % 16] = -250.0 / 64      # exact in every type
    for i, (s, what) in enumerate(zip(slots, (math.nan, math.inf, -math.inf))):
        v[int(table[s // 16]), i % 2, s % 16, 5 + i] = what
    chunk_run(torch, eng, c, scale=1.0)
    assert not torch.isfinite(c["out"][:new, 0, 5]).any() and torch.isfinite(c["out"][:new, 0, 0]).all()


@pytest.mark.parametrize("q,kv", TYPES)
@pytest.mark.parametrize("rising", [False, True])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 7), (256, 64)])
def test_chunk_rows_are_the_same_whatever_comes_behind_them(torch_mod, pkg, eng, q, kv, d, page, rising):
    """To the bit: later tokens' keys and values of other sizes, infinite or NaN leave earlier rows as they are, also where
    a row's largest score grows from unit to unit."""
    torch = torch_mod
    # enough heads that a stretch holds a tile's units, not one of them
    c = chunk_case(torch, pkg, [300, 40], [500, 90], 64, 32, d, page, q, kv, seed=27)
    k, v, lens = c["cache"].k, c["cache"].v, c["lens"]
    if rising:
        for b in range(2):
            for s in range(lens[b]):
                k[int(c["table"][b, s // page]), :, s % page] *= 1 + s / 100
    want, wl = chunk_run(torch, eng, c)
    cut = {0: 690, 1: 111}                   # first slot that changes
    rows = torch.cat([torch.arange(300)[:690 - 500], 300 + torch.arange(40)[:111 - 90]]).cuda()
    for what in (60.0, -3.0, math.nan, math.inf, -math.inf):
        for b, first in cut.items():
            for s in range(first, lens[b]):
                for pool in (k, v):
                    row = pool[int(c["table"][b, s // page]), :, s % page]
                    row.copy_(row.nan_to_num(0.5, 1.0, -1.0) * what if math.isfinite(what) else torch.full_like(row, what))
        got, gl = chunk_run(torch, eng, c, check=False)
        assert torch.equal(got[rows], want[rows]), what
        assert torch.equal(gl[rows], wl[rows]), what


# ------------------------------------------------------------------ small weights, small elements of queries

SINK = [("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "f32")]


@pytest.mark.parametrize("q,kv", SINK)
@pytest.mark.parametrize("below", [15, 18, 20, 22, 24, 30, 60])
@pytest.mark.parametrize("new,old", [(5, 4000), (700, 0), (60, 0)])
def test_chunk_beside_a_slot_without_value(torch_mod, pkg, eng, q, kv, below, new, old):
    """One slot holds nearly all weight and the value 0, so that all of the output comes from weights of e^-15 to e^-60
    beside 1, in units with that slot and without. With float32 queries they are as exact as any; with float16 ones a
    weight is within 2^-35 of the row's largest, so the output within 2^-35 of the values' sum."""
    torch = torch_mod
    c = chunk_case(torch, pkg, [new], [old], 4, 2, 64, 16, q, kv, seed=23)
    k, v, table = c["cache"].k, c["cache"].v, c["table"][0]
    c["q"].fill_(1.0)
    k.fill_(-below / 64)                     # exact in every type
    v.copy_(64 * v.abs() + 32)
    k[int(table[0]), :, 0] = 0.0
    v[int(table[0]), :, 0] = 0.0
    chunk_run(torch, eng, c, scale=1.0, check=False)
    out, lse, tol, ltol = chunk_exact(torch, c, 1.0)
    if q == "f16":
        tol = tol + 2.0 ** -35 * (old + new) * v.max().double()
    got, n = c["out"].double(), new
    bad = ~((got - out).abs() <= tol)[:n]
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}: worst {float(((got - out).abs() / tol)[:n][bad].max())} at {bad.nonzero()[0].tolist()}"
    assert ((c["lse"].double() - lse).abs() <= ltol)[:n].all()


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("j", [20, 26, 30, 34])
def test_chunk_small_elements_of_a_query(torch_mod, pkg, eng, kv, j):
    """A query whose one large element meets keys of 0: the scores come from elements of 2^-j of it."""
    torch = torch_mod
    c = chunk_case(torch, pkg, [70], [200], 4, 2, 64, 16, "f32", kv, seed=24)
    c["cache"].k.mul_(256.0)
    c["cache"].k[..., 7] = 0.0
    c["q"].mul_(2.0 ** -8)
    c["q"][..., 7] = 2.0 ** (j - 8)
    chunk_run(torch, eng, c)


# ------------------------------------------------------------------ rows that share memory

def test_rows_of_an_output_that_meet_are_refused(torch_mod, pkg, eng):
    """Also in place, where a broadcast row would be turned, or normed, again for each that reads it."""
    torch = torch_mod
    eng.set_stream(torch.cuda.current_stream().cuda_stream)
    one = torch.randn(1, 1, 64, device="cuda")
    q, pos, freqs = torch.randn(5, 2, 64, device="cuda"), torch.arange(5, dtype=torch.int32, device="cuda"), pkg.rope_freqs(64).cuda()
    before = one.clone()
    for out in (one.expand(5, 2, 64), q[:1].expand(5, 2, 64), q[:, :1].expand(5, 2, 64),
                q.view(-1).as_strided((5, 2, 64), (32, 320, 1))):
        for kw in (dict(q=out), dict(k=out), dict(q=q.clone(), q_out=out), dict(k=q.clone(), k_out=out)):
            with pytest.raises(pkg.B200Error):
                eng.rope(pos, freqs, **kw)
    x, w = one.view(1, 64), torch.ones(64, device="cuda")
    y, half = torch.randn(5, 64, device="cuda"), torch.randn(5, 128, device="cuda").half()
    for kw in (dict(x=x.expand(5, 64), out=x.expand(5, 64)), dict(x=y, out=x.expand(5, 64)),
               dict(x=y, residual=x.expand(5, 64), out=y), dict(x=y, residual=y.clone(), residual_out=x.expand(5, 64)),
               dict(x=y, residual=torch.randn(5, 128, device="cuda")[:, :64], residual_out=y.view(-1).as_strided((5, 64), (32, 1))),
               # the sum of 32 bits over an input of 16, over rows of other strides, and where the norm goes
               dict(x=half[:, :64], residual=y, residual_out=half.view(torch.float32)),
               dict(x=y, residual=half.float()[:, :64], residual_out=y, out=y)):
        with pytest.raises(pkg.B200Error):
            eng.rms_norm(weight=w, **kw)
    torch.cuda.synchronize()
    assert torch.equal(one, before)
    # inputs may be broadcast, and one row may lie anywhere
    a, b = torch.empty(5, 2, 64, device="cuda"), torch.empty(5, 2, 64, device="cuda")
    eng.rope(pos, freqs, q=one.expand(5, 2, 64), q_out=a)
    eng.rope(pos, freqs, q=one.expand(5, 2, 64).contiguous(), q_out=b)
    assert torch.equal(a, b)
    u, v = torch.empty_like(y), torch.empty_like(y)
    eng.rms_norm(x.expand(5, 64), w, out=u, residual=y, residual_out=v)
    eng.rms_norm(x.expand(5, 64).contiguous(), w, out=y, residual=y.clone())
    assert torch.equal(u, y)


# ------------------------------------------------------------------ packed rows

@pytest.mark.parametrize("x,res", [("f32", None), ("f32", "f32"), ("bf16", None), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("n,k", [(1, 2048), (33, 256), (2050, 4096), (2049, 2080), (3, 32736)])
def test_norm_q8_of_all_types(torch_mod, eng, x, res, n, k):
    """The packed rows are b200_quantize_q8_0's of the float32 norm, to the bit, from inputs of any type, with a residual
    and without, with one, two and four units of eight elements a thread."""
    torch = torch_mod
    eng.set_stream(torch.cuda.current_stream().cuda_stream)
    gen = torch.Generator(device="cuda").manual_seed(n + k)
    a = torch.randn(n, k, generator=gen, device="cuda").to(getattr(torch, DT[x]))
    r = None if res is None else (3 * torch.randn(n, k, generator=gen, device="cuda")).to(getattr(torch, DT[res]))
    w = torch.rand(k, generator=gen, device="cuda") + 0.5
    q8 = torch.full((n, k + k // 8), 99, dtype=torch.uint8, device="cuda")
    s = a.float() if r is None else r.float() + a.float()
    y, again = torch.empty(n, k, device="cuda"), torch.empty(n, k, dtype=a.dtype, device="cuda")
    eng.rms_norm(s, w, out=y)                # the same sums in the same order
    eng.rms_norm(a, w, residual=r, out=again, q8=q8)
    assert torch.equal(again, y.to(a.dtype))
    if r is not None:
        assert torch.equal(r, s.to(r.dtype))
    want = torch.zeros(n, (k + k // 8 + 15) // 16 * 16, dtype=torch.uint8, device="cuda")
    for i in range(n):
        eng.quantize(y[i], want[i], k)
    assert torch.equal(q8, want[:, :k + k // 8])


# ------------------------------------------------------------------ engines

def test_two_engines_at_once_leave_each_other_alone(torch_mod, pkg):
    """Two engines on streams of their own, their steps side by side: both to the bit as alone."""
    torch = torch_mod
    requests = [[100, 3, 1, 10, 5], [1, 60, 30, 1, 1], [7, 7, 7, 7, 7], [-1, 1, 90, 1, 2]] * 4
    streams = [torch.cuda.Stream() for _ in range(2)]
    engines = [pkg.Engine(0, stream=s.cuda_stream) for s in streams]
    alone, both = ([step_case(torch, pkg, seed) for seed in (7, 8)] for _ in range(2))
    news = [torch.tensor(r, dtype=torch.int32, device="cuda") for r in requests]
    torch.cuda.synchronize()
    for e, st, s in zip(engines, streams, alone):
        with torch.cuda.stream(st):
            for new in news:
                s["new"].copy_(new)
                step_run(e, s)
        torch.cuda.synchronize()
    for new in news:
        for e, st, s in zip(engines, streams, both):
            with torch.cuda.stream(st):
                s["new"].copy_(new)
                step_run(e, s)
    torch.cuda.synchronize()
    for i in range(2):
        for name, x, y in zip(STATE + ("k", "v", "table", "lengths"), step_state(alone[i]), step_state(both[i])):
            assert torch.equal(x, y), (i, name)
        assert engines[i].status() == 0
        engines[i].close()


# ------------------------------------------------------------------ single tokens

@pytest.mark.parametrize("q,kv", SINK)
@pytest.mark.parametrize("below", [15, 18, 20, 22, 24, 30])
@pytest.mark.parametrize("old", [40, 4000])
def test_attend_beside_a_slot_without_value(torch_mod, pkg, eng, q, kv, below, old):
    """kv_attend where one slot holds nearly all weight and the value 0. A float16 cache's weights are within 2^-48 of the
    row's largest, or to 22 bits."""
    torch = torch_mod
    eng.set_stream(torch.cuda.current_stream().cuda_stream)
    c = chunk_case(torch, pkg, [1], [old], 4, 2, 64, 16, q, kv, seed=25)
    k, v, table = c["cache"].k, c["cache"].v, c["table"][0]
    c["q"].fill_(1.0)
    k.fill_(-below / 64)
    v.copy_(64 * v.abs() + 32)
    k[int(table[0]), :, 0] = 0.0
    v[int(table[0]), :, 0] = 0.0
    out, lse = torch.empty(1, 4, 64, dtype=c["q"].dtype, device="cuda"), torch.empty(1, 4, device="cuda")
    eng.kv_attend(c["cache"], c["q"][:1].contiguous(), out, lse=lse, scale=1.0)
    want, wl, tol, ltol = (t[:1] for t in chunk_exact(torch, c, 1.0))
    # weights keep 22 bits, not half a step of the cache's type
    tol = tol - (U[kv] if q != "f32" else 0) * want.abs() + 2.0 ** -16 * want.abs()
    if kv == "f16":
        tol = tol + 2.0 ** -48 * (old + 1) * v.max().double()
    assert ((out.double() - want).abs() <= tol).all(), float(((out.double() - want).abs() / tol).max())
    assert ((lse.double() - wl).abs() <= ltol).all()


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("j", [20, 26, 30, 34])
def test_attend_small_elements_of_a_query(torch_mod, pkg, eng, kv, j):
    """A query whose one large element meets keys of 0: the scores come from elements of 2^-j of it."""
    torch = torch_mod
    eng.set_stream(torch.cuda.current_stream().cuda_stream)
    c = chunk_case(torch, pkg, [1], [200], 4, 2, 64, 16, "f32", kv, seed=26)
    c["cache"].k.mul_(256.0)
    c["cache"].k[..., 7] = 0.0
    c["q"].mul_(2.0 ** -8)
    c["q"][..., 7] = 2.0 ** (j - 8)
    out = torch.empty(1, 4, 64, device="cuda")
    eng.kv_attend(c["cache"], c["q"][:1].contiguous(), out)
    want, _, tol, _ = (t[:1] for t in chunk_exact(torch, c, 0.125))
    assert ((out.double() - want).abs() <= tol).all(), float(((out.double() - want).abs() / tol).max())
