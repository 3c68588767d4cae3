"""The operators that a prompt passes through (b200_kv_plan, b200_rope,
b200_rms_norm, b200_kv_attend_chunk) against plain implementations in 64 bits,
at the sizes, layouts and masks where they can go wrong."""

from __future__ import annotations

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

DT = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}
U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}      # half a step, relative to the value


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


# ------------------------------------------------------------ chunk attention

def chunk_case(torch, pkg, new, old, h, hkv, d, page, q, kv, seed=0, layout="head", garbage=None, absent=(), extra=0, spread=1.5):
    """Caches of old[b] + new[b] slots in pages of random order, and queries whose rows lie in a wider tensor. `absent`
    names (sequence, column) pairs whose page is not there; rows not in use hold `garbage`."""
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lens = [a + b for a, b in zip(new, old)]
    need = [-(-n // page) for n in lens]
    cols, n_pages = max(1, max(need)) + extra, sum(need) + 3
    dt = getattr(torch, DT[kv])
    shape = (n_pages, hkv, page, d) if layout == "head" else (n_pages, page, hkv, d)
    k = torch.randn(shape, generator=gen, device="cuda").to(dt)
    v = torch.randn(shape, generator=gen, device="cuda").to(dt)
    if layout != "head":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    perm = rng.permutation(n_pages)
    table = np.full((len(lens), cols), -1, np.int32)
    at = 0
    for b, c in enumerate(need):
        table[b, :c] = perm[at:at + c]
        at += c
    if garbage is not None:
        used = torch.zeros(n_pages, page, dtype=torch.bool, device="cuda")
        for b, n in enumerate(lens):
            for s in range(0, n, page):
                used[table[b, s // page], :min(page, n - s)] = True
        k[~used[:, None, :].expand(-1, hkv, -1)] = garbage
        v[~used[:, None, :].expand(-1, hkv, -1)] = garbage
    for b, c in absent:
        table[b, c] = -1 if (b + c) % 2 else n_pages + 7
    cache = pkg.PagedKV(k, v, torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"))
    off = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    n = int(off[-1])
    wide = (spread * torch.randn(n + 2, h + 1, d, generator=gen, device="cuda")).to(getattr(torch, DT[q]))
    out = torch.full((n + 2, h, d), 7.0, dtype=wide.dtype, device="cuda")
    return dict(cache=cache, table=table, q=wide[:, 1:], out=out, lse=torch.full((n + 2, h), 7.0, device="cuda"), n=n,
                offsets=torch.from_numpy(off).cuda(), new=list(new), lens=lens, h=h, hkv=hkv, d=d, page=page, dt=q, kv=kv)


def chunk_exact(torch, c, scale, window=0):
    """out and lse in 64 bits, and with A = sum p |v| and S the largest sum |q k| scale of a row the bounds of their
    errors. A sum of n products in float32 is off by at most n 2^-23 of the sum of their sizes where additions are cut
    off, so a score by (d + 8) 2^-23 S, a weight by twice that and the rounding of its exponent (t log2 e, |t| <= S +
    |lse|), a sum of weights by (n + 64) 2^-23; then the rounding of the weight and of the output to 16 bits."""
    h, hkv, d, page, cache = c["h"], c["hkv"], c["d"], c["page"], c["cache"]
    dev = "cuda"
    n_all = c["q"].shape[0]
    out = torch.zeros(n_all, h, d, dtype=torch.float64, device=dev)
    lse = torch.full((n_all, h), -math.inf, dtype=torch.float64, device=dev)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    at = 0
    e = 2.0 ** -23
    for b, (n, length) in enumerate(zip(c["new"], c["lens"])):
        if n and length > 0:
            slot = torch.arange(length, device=dev)
            pages = torch.from_numpy(c["table"][b]).cuda()[slot // page].long()
            there = (pages >= 0) & (pages < cache.n_pages)
            pg = torch.where(there, pages, 0)
            row = torch.arange(length - n, length, device=dev)[:, None]
            seen = (slot <= row) & there
            if window:
                seen &= slot > row - window
            for j in range(hkv):
                k = cache.k[pg, j, slot % page].double()
                v = cache.v[pg, j, slot % page].double()
                for x in range(j * h // hkv, (j + 1) * h // hkv):
                    q = c["q"][at:at + n, x].double()
                    s = (q @ k.T * scale).masked_fill_(~seen, -math.inf)
                    big = (q.abs() @ k.abs().T * abs(scale)).masked_fill_(~seen, 0).nan_to_num(0, 0, 0).amax(1)
                    z = torch.logsumexp(s, 1)
                    p = torch.exp(s - z.clamp(min=-1e30)[:, None])
                    p = torch.where(seen, p, 0.0)
                    vv = torch.where(seen.any(0)[:, None], v, 0.0)
                    # a value that is not finite and not seen by a row stays out of its sum
                    bad = ~torch.isfinite(vv)
                    o = p @ vv.masked_fill(bad, 0.0)
                    if bad.any():
                        o = torch.where((seen.double() @ bad.double()) > 0, math.nan, o)
                    a = p @ vv.masked_fill(bad, 0.0).abs()
                    rel = (2 * (d + 8) + 8) * e * big + 4 * e * z.abs().nan_to_num(0, 0, 0) + (length + 64) * e
                    rel = rel + (U[c["kv"]] if c["dt"] != "f32" else 0)
                    out[at:at + n, x], lse[at:at + n, x] = o, z
                    tol[at:at + n, x] = U[c["dt"]] * o.abs().nan_to_num(0) + a * rel[:, None] + 1e-37 + (6e-8 if c["dt"] == "f16" else 0)
                    ltol[at:at + n, x] = (d + 8) * e * big + (length + 64) * e + 4 * e * z.abs().nan_to_num(0, 0, 0)
        at += n
    return out, lse, tol, ltol


def chunk_check(torch, c, scale, window=0):
    out, lse, tol, ltol = chunk_exact(torch, c, scale, window)
    n = c["n"]
    got, gl = c["out"][:n].double(), c["lse"][:n].double()
    out, lse, tol, ltol = out[:n], lse[:n], tol[:n], ltol[:n]
    fin = torch.isfinite(out)
    bad = fin & ~((got - out).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}: worst {float(((got - out).abs() / tol)[bad].max())} at {bad.nonzero()[0].tolist()}"
    assert not torch.isfinite(got[~fin]).any()
    empty = torch.isinf(lse) & (lse < 0)
    assert (got[empty] == 0).all() and (gl[empty] == -math.inf).all()
    ok = torch.isfinite(lse)
    assert ((gl - lse).abs() <= ltol)[ok].all(), float(((gl - lse).abs() / ltol)[ok].max())
    assert torch.isnan(gl[torch.isnan(lse)]).all()
    assert (c["out"][n:] == 7).all() and (c["lse"][n:] == 7).all()      # rows behind the last sequence


def chunk_run(torch, eng, c, scale=None, window=0, check=True):
    eng.set_stream(torch.cuda.current_stream().cuda_stream)
    n = c["n"]
    eng.kv_attend_chunk(c["cache"], c["q"], c["out"], c["offsets"], lse=c["lse"], scale=scale, window=window)
    assert eng.status() == 0             # no wait inside the kernel ran out
    if check:
        chunk_check(torch, c, c["d"] ** -0.5 if scale is None else scale, window)
    return c["out"][:n].clone(), c["lse"][:n].clone()


TYPES = [("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "f32")]


@pytest.mark.parametrize("q,kv", TYPES)
@pytest.mark.parametrize("new,old,h,hkv,d,page,window", [
    ([1], [0], 1, 1, 64, 16, 0),                       # one token, one slot
    ([1, 1, 1], [0, 5, 300], 4, 2, 64, 16, 0),         # single tokens
    ([5], [600], 32, 8, 64, 16, 0),
    ([64], [0], 8, 2, 128, 64, 0),
    ([130, 0, 7, 1], [0, 9, 250, 127], 8, 2, 128, 41, 0),
    ([257], [500], 6, 2, 96, 7, 0),                    # groups that do not divide a tile
    ([33, 500], [64, 0], 5, 1, 80, 1, 0),              # pages of one slot
    ([300], [300], 7, 1, 192, 33, 0),
    ([200, 3], [100, 700], 8, 4, 256, 64, 0),
    ([40, 90], [10, 20], 3, 3, 8, 16, 0),
    ([129], [0], 40, 1, 16, 128, 0),
    ([300, 20], [0, 400], 8, 2, 64, 16, 1),            # only itself
    ([300, 20, 9], [0, 400, 3], 8, 2, 64, 16, 37),
    ([513], [700], 4, 1, 128, 64, 256),
    ([200], [1000], 3, 1, 72, 50, 5000),               # wider than the cache
])
def test_chunk(torch_mod, pkg, eng, q, kv, new, old, h, hkv, d, page, window):
    c = chunk_case(torch_mod, pkg, new, old, h, hkv, d, page, q, kv, seed=d + page, garbage=math.nan)
    chunk_run(torch_mod, eng, c, window=window)


@pytest.mark.parametrize("q,kv", TYPES)
def test_chunk_layouts_and_absent_pages(torch_mod, pkg, eng, q, kv):
    """Pages [row][head], pages that are not there (at the start, inside, at the last slots), an infinite garbage."""
    c = chunk_case(torch_mod, pkg, [70, 30, 20], [200, 0, 40], 4, 2, 128, 16, q, kv, seed=3, layout="row", garbage=math.inf,
                   absent=[(0, 0), (0, 5), (1, 0), (1, 1), (2, 3)], extra=4)
    chunk_run(torch_mod, eng, c)
    chunk_run(torch_mod, eng, c, scale=0.02, window=50)


@pytest.mark.parametrize("q,kv", TYPES)
def test_chunk_long_axis_is_split_and_repeats(torch_mod, pkg, eng, q, kv):
    """Few rows over a long axis, which many CTAs share: the same bits on every run."""
    c = chunk_case(torch_mod, pkg, [9], [20000], 4, 2, 128, 64, q, kv, seed=4)
    a, la = chunk_run(torch_mod, eng, c)
    for _ in range(3):
        b, lb = chunk_run(torch_mod, eng, c, check=False)
        assert torch_mod.equal(a, b) and torch_mod.equal(la, lb)


@pytest.mark.parametrize("q,kv", TYPES)
def test_chunk_rising_scores(torch_mod, pkg, eng, q, kv):
    """The running maximum rises by far more than any slack, again and again, and falls."""
    torch = torch_mod
    c = chunk_case(torch, pkg, [140], [900], 4, 2, 64, 16, q, kv, seed=5)
    up = torch.linspace(0.0, 30.0, 1040, device="cuda")
    for pages in c["table"][:1]:
        for s in range(1040):
            c["cache"].k[int(pages[s // 16]), 0, s % 16] = up[s]
            c["cache"].k[int(pages[s // 16]), 1, s % 16] = 30.0 - up[s]
    c["q"].fill_(1.0)
    chunk_run(torch, eng, c, scale=0.25)


@pytest.mark.parametrize("q,kv", TYPES)
def test_chunk_lengths_below_the_new_tokens(torch_mod, pkg, eng, q, kv):
    """A length smaller than the number of rows (a sequence that got no slots, or was cut): rows at p < 0 see nothing."""
    torch = torch_mod
    c = chunk_case(torch, pkg, [100, 50, 20], [0, 0, 60], 4, 2, 64, 16, q, kv, seed=6)
    c["lens"] = [30, 0, 80]
    c["cache"].lengths.copy_(torch.tensor([30, -5, 80]))
    chunk_run(torch, eng, c)


@pytest.mark.parametrize("q,kv", TYPES)
@pytest.mark.parametrize("window", [0, 60])
def test_chunk_values_not_seen_do_not_matter(torch_mod, pkg, eng, q, kv, window):
    """Infinities and NaN in the values and keys of later tokens leave the earlier ones alone; who sees a value that is not
    finite gets one, in that element only."""
    torch = torch_mod
    c = chunk_case(torch, pkg, [200], [100], 4, 2, 64, 16, q, kv, seed=7)
    cache, table = c["cache"], c["table"]
    for slot, j, col, what in ((150, 0, 3, math.inf), (231, 0, slice(None), math.nan), (299, 0, 10, -math.inf),
                               (120, 1, 63, math.nan)):
        cache.v[int(table[0, slot // 16]), j, slot % 16, col] = what
    chunk_run(torch, eng, c, window=window)
    cache.k[int(table[0, 250 // 16]), 1, 250 % 16] = math.nan
    cache.v.nan_to_num_(0.5, 0.5, 0.5)
    chunk_run(torch, eng, c, window=window)


@pytest.mark.parametrize("q,kv", TYPES)
def test_chunk_scores_that_are_not_finite(torch_mod, pkg, eng, q, kv):
    """-infinity weighs nothing; +infinity and NaN make the row NaN."""
    torch = torch_mod
    c = chunk_case(torch, pkg, [40], [30], 2, 1, 64, 16, q, kv, seed=8)
    k, table = c["cache"].k, c["table"]
    c["q"][:, 0].abs_()
    c["q"][:, 1] = -c["q"][:, 1].abs() - 0.1
    k[int(table[0, 0]), 0, 3] = -math.inf              # head 0: -infinity; head 1: +infinity
    chunk_run(torch, eng, c)
    assert torch.isnan(c["out"][:40, 1]).all() and torch.isfinite(c["out"][:40, 0]).all()


def test_chunk_many_sequences(torch_mod, pkg, eng):
    """More sequences than a CTA has threads, most of them without rows."""
    rng = np.random.default_rng(9)
    new = [int(x) if i % 3 == 0 else 0 for i, x in enumerate(rng.integers(0, 9, 1500))]
    old = rng.integers(0, 40, 1500).tolist()
    for q in ("bf16", "f32"):
        c = chunk_case(torch_mod, pkg, new, old, 4, 2, 64, 16, q, "bf16" if q == "bf16" else "f32", seed=9)
        chunk_run(torch_mod, eng, c)


def test_chunk_many_tiles(torch_mod, pkg, eng):
    """More tiles than a CTA has threads, an axis of several thousand slots, causal."""
    for q, kv, n in (("bf16", "bf16", 30000), ("f32", "f16", 9000)):
        c = chunk_case(torch_mod, pkg, [n], [0], 8, 1, 64, 64, q, kv, seed=10)
        chunk_run(torch_mod, eng, c, check=False)
        # rows of all kinds against the definition
        rows = sorted({0, 1, 63, 64, n // 2, n - 1} | set(np.random.default_rng(1).integers(0, n, 40).tolist()))
        pages = torch_mod.from_numpy(c["table"][0]).cuda().long()
        k = c["cache"].k[pages, 0].reshape(-1, 64).double()
        v = c["cache"].v[pages, 0].reshape(-1, 64).double()
        for r in rows:
            s = c["q"][r].double() @ k[:r + 1].T / 8
            p = torch_mod.softmax(s, 1)
            want = p @ v[:r + 1]
            # half a step of the output, of each weight, and of sums of up to n terms
            tol = U[q] * want.abs() + (p @ v[:r + 1].abs()) * ((U[kv] if q != "f32" else 0) + 2.0 ** -23 * (n + 64 + 80 * 40))
            assert ((c["out"][r].double() - want).abs() <= tol).all(), r


@pytest.mark.parametrize("q,kv", TYPES)
@pytest.mark.parametrize("d,window", [(64, 0), (128, 0), (128, 90), (256, 0)])
def test_chunk_short_and_long_in_turn(torch_mod, pkg, eng, q, kv, d, window):
    """Single tokens beside chunks of several tiles, so that a CTA has one after another of both kinds."""
    new = [1, 150, 3, 70, 1, 1, 260, 2] * 5
    old = [int(x) for x in np.random.default_rng(14).integers(0, 700, len(new))]
    c = chunk_case(torch_mod, pkg, new, old, 32, 8, d, 16, q, kv, seed=14, garbage=math.nan)
    chunk_run(torch_mod, eng, c, window=window)


def test_chunk_equals_single_tokens(torch_mod, pkg, eng):
    """Chunks of one token are kv_attend's call."""
    torch = torch_mod
    for q, kv in TYPES:
        c = chunk_case(torch, pkg, [1] * 6, [0, 3, 100, 17, 2000, 640], 8, 2, 128, 16, q, kv, seed=11)
        chunk_run(torch, eng, c)
        one, lse = torch.empty_like(c["out"][:6]), torch.empty(6, 8, device="cuda")
        eng.kv_attend(c["cache"], c["q"][:6].contiguous(), one, lse=lse)
        _, _, tol, ltol = chunk_exact(torch, c, 128 ** -0.5)
        assert ((one.double() - c["out"][:6].double()).abs() <= 2 * tol[:6]).all()
        assert ((lse - c["lse"][:6]).abs() <= 2 * ltol[:6]).all()


def test_chunk_in_a_graph_on_another_stream(torch_mod, pkg):
    """Recorded and replayed on a stream of its own, with lengths, offsets, tables and queries that change between the
    launches; eager calls on another stream in between."""
    torch = torch_mod
    e = pkg.Engine(0)
    s = torch.cuda.Stream()
    c = chunk_case(torch, pkg, [60, 30], [100, 40], 4, 2, 64, 16, "bf16", "bf16", seed=12, extra=3)
    d = chunk_case(torch, pkg, [10], [3000], 8, 2, 128, 64, "f16", "f16", seed=13)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        e.set_stream(s.cuda_stream)
        e.kv_attend_chunk(c["cache"], c["q"], c["out"], c["offsets"], lse=c["lse"])
        e.capture_begin()
        e.kv_attend_chunk(c["cache"], c["q"], c["out"], c["offsets"], lse=c["lse"])
        g = e.capture_end()
        for new, lens in (([60, 30], [160, 70]), ([10, 80], [50, 70]), ([0, 90], [0, 90 - 20])):
            c["new"], c["lens"] = new, lens
            c["cache"].lengths.copy_(torch.tensor(lens))
            c["offsets"].copy_(torch.tensor([0, new[0], sum(new)]))
            c["q"].normal_()
            c["out"].fill_(7.0)
            c["lse"].fill_(7.0)
            g.launch()
            chunk_run(torch, e, d)
            c["table"] = c["cache"].table.cpu().numpy()
            chunk_check(torch, c, 0.125)
    g.close()
    e.sync()
    e.close()


# ------------------------------------------------------------ rotary positions

def rope_exact(torch, x, positions, freqs, interleaved, mscale):
    """In 64 bits, with the frequencies' whole numbers: a phase is exact."""
    half = freqs.numel()
    phase = (positions.cpu().numpy().astype(np.int64)[:, None].astype(np.uint64) * freqs.numpy().view(np.uint64)[None])
    angle = torch.from_numpy(phase.view(np.int64).astype(np.float64) * (2.0 * math.pi / 2.0 ** 64)).cuda()[:, None]
    c, s = torch.cos(angle) * mscale, torch.sin(angle) * mscale
    y = x.double().clone()
    i = torch.arange(half, device="cuda")
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    u, v = x.double()[..., a], x.double()[..., b]
    y[..., a], y[..., b] = u * c - v * s, v * c + u * s
    size = y.abs().clone()
    size[..., a] = size[..., b] = (u.abs() + v.abs()) * abs(mscale)
    return y, size


# the cosine is off by 2^-28 turns (2^-25.3), an ulp or two of its own and its product with mscale, each product and
# the sum by half a step: in all below 8 half steps of the sizes' sum
def rope_close(torch, got, want, size, dt):
    assert ((got.double() - want).abs() <= 8 * 2.0 ** -24 * size + U[dt] * want.abs() + (3e-8 if dt == "f16" else 0)).all()


@pytest.mark.parametrize("src,dst", [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("n,h,hkv,d,rot", [(1, 1, 1, 8, 2), (3, 4, 2, 64, 64), (5, 32, 8, 128, 128), (1030, 3, 3, 80, 32),
                                            (17, 2, 1, 96, 20), (9, 5, 5, 256, 254), (1025, 8, 2, 64, 48)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope(torch_mod, pkg, eng, src, dst, n, h, hkv, d, rot, interleaved):
    torch = torch_mod
    gen = torch.Generator(device="cuda").manual_seed(n + d)
    eng.set_stream(torch.cuda.current_stream().cuda_stream)
    wide = torch.randn(n, h + 2 * hkv, d, generator=gen, device="cuda").to(getattr(torch, DT[src]))
    q, k, v = wide[:, :h], wide[:, h:h + hkv], wide[:, h + hkv:]
    pos = torch.randint(-5, 1 << 20, (n,), generator=gen, device="cuda", dtype=torch.int32)
    pos[0] = 0
    freqs = pkg.rope_freqs(rot, 10000.0)
    out = dict(dtype=getattr(torch, DT[dst]), device="cuda")
    qo, ko = torch.empty(n, h, d, **out), torch.empty(n, hkv, d, **out)
    m = 1.25
    eng.rope(pos, freqs.cuda(), q=q, q_out=qo, k=k, k_out=ko, interleaved=interleaved, mscale=m)
    for x, y in ((q, qo), (k, ko)):
        want, size = rope_exact(torch, x, pos, freqs, interleaved, m)
        rope_close(torch, y, want, size, dst)
        if rot < d:
            assert torch.equal(y[..., rot:], x[..., rot:].to(y.dtype))
    # into a cache, with tokens that have no slot; other rows keep what they hold
    page, n_pages = 7, n // 7 + 4
    kp, vp = (torch.randn(n_pages, page, hkv, d, generator=gen, device="cuda").to(out["dtype"]).transpose(1, 2)
              for _ in range(2))
    cache = pkg.PagedKV(kp, vp, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"))
    slots = torch.randperm(n_pages * page, generator=gen, device="cuda")[:n]
    slots[::5] = -1
    if n > 3:
        slots[3] = n_pages * page
    k0, v0 = kp.clone(), vp.clone()
    keep = q.clone()
    eng.rope(pos, freqs.cuda(), k=k, kv=cache, v=v, slots=slots, interleaved=interleaved, mscale=m)
    assert torch.equal(q, keep)
    ok = (slots >= 0) & (slots < n_pages * page)
    pg, row = slots[ok] // page, slots[ok] % page
    assert torch.equal(kp[pg, :, row], ko[ok]) and torch.equal(vp[pg, :, row], v[ok].to(out["dtype"]))
    k0[pg, :, row], v0[pg, :, row] = ko[ok], v[ok].to(out["dtype"])
    assert torch.equal(kp, k0) and torch.equal(vp, v0)
    if src == dst:                                       # in place
        eng.rope(pos, freqs.cuda(), q=q, k=k, interleaved=interleaved, mscale=m)
        assert torch.equal(q, qo) and torch.equal(k, ko)


def test_rope_far_positions_and_other_layouts(torch_mod, pkg, eng):
    """Positions up to the largest: the angle is the product of whole numbers; q alone, heads before tokens."""
    torch = torch_mod
    eng.set_stream(torch.cuda.current_stream().cuda_stream)
    pos = torch.tensor([0, 1, 1 << 20, (1 << 31) - 1, -(1 << 31), -1, 123456789], dtype=torch.int32, device="cuda")
    freqs = pkg.rope_freqs(64, 500000.0)
    x = torch.randn(3, 7, 64, device="cuda").transpose(0, 1)
    y = torch.empty(7, 3, 64, device="cuda")
    eng.rope(pos, freqs.cuda(), q=x, q_out=y)
    want, size = rope_exact(torch, x, pos, freqs, False, 1.0)
    rope_close(torch, y, want, size, "f32")
    eng.rope(pos[:0], freqs.cuda(), q=x[:0], q_out=y[:0])


# ------------------------------------------------------------ the norm

@pytest.mark.parametrize("x,res,out", [("f32", "f32", "f32"), ("f32", "f32", "bf16"), ("f32", None, "f16"),
                                       ("bf16", "bf16", "bf16"), ("bf16", "f32", "bf16"), ("f16", "f16", "f16"),
                                       ("f16", None, "f16")])
@pytest.mark.parametrize("n,k", [(1, 8), (1, 2048), (3, 2056), (7, 4096), (2050, 4096), (2, 8192), (5, 32768), (2049, 264),
                                 (4, 11008)])
def test_norm(torch_mod, eng, x, res, out, n, k):
    torch = torch_mod
    eng.set_stream(torch.cuda.current_stream().cuda_stream)
    gen = torch.Generator(device="cuda").manual_seed(n + k)
    wide = torch.randn(n, k + 8, generator=gen, device="cuda").to(getattr(torch, DT[x]))
    a, w = wide[:, 8:], 1 + 0.3 * torch.randn(k, generator=gen, device="cuda")
    r = None if res is None else (3 * torch.randn(n, k, generator=gen, device="cuda")).to(getattr(torch, DT[res]))
    ro = None if res is None else torch.empty_like(r)
    y = torch.empty(n, k, dtype=getattr(torch, DT[out]), device="cuda")
    eng.rms_norm(a, w, out=y, eps=1e-5, residual=r, residual_out=ro)
    s = a.double() if r is None else a.double() + r.double()
    want = s / torch.sqrt(s.square().mean(1, keepdim=True) + 1e-5) * w.double()
    # half a step for the residual's sum, of the sum of squares (k / threads + 40 terms in a row), of root, two products
    tol = ((2 + (k / 256 + 48) / 2 + 4) * 2.0 ** -24 + U[out]) * want.abs() + (3e-8 if out == "f16" else 0)
    assert ((y.double() - want).abs() <= tol).all()
    if r is not None:
        assert ((ro.double() - s).abs() <= U[res] * s.abs()).all()
        eng.rms_norm(a, w, residual=r)                   # in place, the residual alone
        assert torch.equal(r, ro)
    if x == out and res is None:
        eng.rms_norm(a, w, out=a, eps=1e-5)
        assert torch.equal(a, y)


@pytest.mark.parametrize("n,k", [(1, 32), (1, 2048), (5, 2080), (33, 256), (2, 8192), (3, 32736)])
def test_norm_q8_is_the_engines(torch_mod, pkg, eng, n, k):
    """The packed rows are b200_quantize_q8_0's of the float32 output, to the bit, and feed gemv_q8; both rounding rules;
    blocks of zeros."""
    torch = torch_mod
    eng.set_stream(torch.cuda.current_stream().cuda_stream)
    gen = torch.Generator(device="cuda").manual_seed(k)
    x, w = torch.randn(n, k, generator=gen, device="cuda"), torch.rand(k, generator=gen, device="cuda") + 0.5
    w[:32] = 0
    mode = eng.config()["round_mode"]
    try:
        for m in (0, 1):
            eng.configure(round_mode=m)
            y = torch.empty(n, k, device="cuda")
            q8 = torch.full((n, k + k // 8), 99, dtype=torch.uint8, device="cuda")
            eng.rms_norm(x, w, out=y, q8=q8)
            want = torch.zeros((k + k // 8 + 15) // 16 * 16, dtype=torch.uint8, device="cuda")
            for i in range(n):
                eng.quantize(y[i].clone(), want, k)
                assert torch.equal(q8[i], want[:k + k // 8])
    finally:
        eng.configure(round_mode=mode)
    if k % 256 == 0 and k <= 8192:
        from llm_kv260_b200 import model
        rows = model.synth_model(dict(n_layer=1, n_embd=k, n_ff=256, n_head=4, n_head_kv=4, head_dim=64, n_vocab=64,
                                      rope_base=1e4, rms_eps=1e-5), seed=1)["token_embd"] if k <= 2048 else None
        if rows is not None:
            W = eng.repack(pkg.QMat.from_numpy(rows, 0))
            a, b = torch.empty(64, device="cuda"), torch.empty(64, device="cuda")
            eng.rms_norm(x, w, q8=q8, out=y)
            eng.gemv_q8(W, q8[0], a)
            eng.gemv_f32(W, y[0], b)
            assert torch.equal(a, b)


# ------------------------------------------------------------ pages and slots

def plan_exact(page, n_pages, table, free, count, length, new, held, seen, n_tokens, room):
    """Request by request, as a host program would."""
    cols = table.shape[1]
    table, free = table.copy(), free.copy()
    length = [min(max(x, 0), cols * page) for x in length]
    held = [min(max(x, 0), cols) for x in held]
    count = min(max(count, 0), room)
    want = [0 if n < 0 else -(-(x + n) // page) if x + n <= cols * page else c for x, n, c in zip(length, new, held)]
    for b in range(len(new)):
        for c in range(want[b], held[b]):
            if count < room:
                free[count] = table[b, c]
                count += 1
    left, asked, given = count, 0, []
    for b in range(len(new)):
        need = max(want[b] - held[b], 0)
        asked += need
        ok = (new[b] < 0 or length[b] + new[b] <= cols * page) and (need == 0 or asked <= count)
        given.append(ok)
        if ok:
            for c in range(held[b], want[b]):
                left -= 1
                table[b, c] = free[left]
    got = [n if ok and n > 0 else 0 for n, ok in zip(new, given)]
    off, slots, pos, seq = [0], [], [], []
    for b, n in enumerate(new):
        for i in range(max(n, 0)):
            if len(slots) == n_tokens:
                break
            s = length[b] + i
            p = table[b, s // page] if given[b] else -1
            slots.append(int(p) * page + s % page if 0 <= p < n_pages else -1)
            pos.append(seen[b] + i)
            seq.append(b)
        off.append(len(slots))
    pad = n_tokens - len(slots)
    return dict(table=table, free=free, free_count=[left], held=[w if ok else c for w, c, ok in zip(want, held, given)],
                lengths=[0 if n < 0 else x + g for x, n, g in zip(length, new, got)],
                seen=[0 if n < 0 else x + g for x, n, g in zip(seen, new, got)], granted=got, offsets=off,
                slots=slots + [-1] * pad, positions=pos + [-1] * pad, sequences=seq + [-1] * pad)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("batch,page,max_new,max_len,spare,pad", [
    (1, 16, 1, 0, 2.0, 0), (1, 1, 5, 3, 1.0, 3), (7, 16, 40, 100, 1.0, 0), (64, 16, 1, 500, 0.5, 0), (33, 41, 900, 300, 0.6, 9),
    (1500, 8, 3, 30, 0.7, 0), (3000, 3, 20, 9, 0.3, 50), (20, 64, 3000, 2000, 0.8, 1000), (5, 2, 60000, 10, 1.0, 0)])
def test_plan(torch_mod, pkg, eng, in_place, batch, page, max_new, max_len, spare, pad):
    torch = torch_mod
    eng.set_stream(torch.cuda.current_stream().cuda_stream)
    rng = np.random.default_rng(batch + page)
    length = rng.integers(0, max_len + 1, batch)
    new = np.where(rng.random(batch) < 0.2, -1, rng.integers(0, max_new + 1, batch))
    new[rng.integers(batch)] = max_new
    held = -(-length // page) + np.where(rng.random(batch) < 0.1, rng.integers(0, 4, batch), 0)
    want = np.where(new < 0, 0, -(-(length + np.maximum(new, 0)) // page))
    cols = max(int(np.quantile(np.maximum(want, held), 0.99)) if batch > 50 else int(max(want.max(), held.max())), 1)
    held = np.minimum(held, cols)
    length = np.minimum(length, held * page)
    free = max(int(spare * np.maximum(want - held, 0).sum()), 1)
    n_pages = int(held.sum()) + free
    perm = rng.permutation(n_pages).astype(np.int32)
    table = np.full((batch, cols), -7, np.int32)
    at = 0
    for b in range(batch):
        table[b, :held[b]] = perm[at:at + held[b]]
        at += held[b]
    room = n_pages - 1 if batch == 33 else n_pages       # once a stack with no room for the last page
    stack = np.full(max(room, 1), -3, np.int32)
    stack[:min(free, room)] = perm[at:at + min(free, room)]
    seen = length + rng.integers(0, 50, batch)
    n_tokens = int(np.maximum(new, 0).sum()) + pad
    if batch == 64:
        n_tokens -= 5                                    # fewer tokens than asked for
    want_all = plan_exact(page, n_pages, table, stack, free, length.tolist(), new.tolist(), held.tolist(), seen.tolist(), n_tokens, len(stack))

    def dev(a, dt=torch.int32):
        return torch.tensor(np.asarray(a), device="cuda").to(dt).contiguous()

    k = torch.empty(n_pages, 1, page, 8, dtype=torch.float16, device="cuda")
    cache = pkg.PagedKV(k, k, dev(table), dev(length))
    t = dict(new=dev(new), held=dev(held), free=dev(stack), free_count=dev([free]),
             offsets=torch.full((batch + 1,), 9, dtype=torch.int32, device="cuda"), seen=dev(seen),
             slots=torch.full((n_tokens,), 9, dtype=torch.int64, device="cuda"), granted=dev(new),
             positions=torch.full((n_tokens,), 9, dtype=torch.int32, device="cuda"),
             sequences=torch.full((n_tokens,), 9, dtype=torch.int32, device="cuda"))
    if in_place:
        eng.kv_plan(cache, **t)
        got = dict(table=cache.table, lengths=cache.lengths, **t)
        runs = 1
    else:
        outs = dict(lengths_out=torch.empty_like(cache.lengths), held_out=torch.empty_like(t["held"]),
                    free_count_out=torch.empty_like(t["free_count"]), seen_out=torch.empty_like(t["seen"]))
        runs = 2
    for _ in range(runs):
        if not in_place:
            eng.kv_plan(cache, **t, **outs)
            got = dict(t, table=cache.table, lengths=outs["lengths_out"], held=outs["held_out"], seen=outs["seen_out"],
                       free_count=outs["free_count_out"])
        for name, value in want_all.items():
            assert np.array_equal(got[name].cpu().numpy(), np.asarray(value)), name
    # no page has two owners, and none is lost
    if in_place and batch not in (33,):
        h, f = got["held"].cpu().numpy(), int(got["free_count"])
        pages = np.concatenate([got["table"].cpu().numpy()[b, :h[b]] for b in range(batch)] + [got["free"].cpu().numpy()[:f]])
        assert np.array_equal(np.sort(pages), np.arange(n_pages))


def test_plan_odd_inputs(torch_mod, pkg, eng):
    """Lengths, counts and pages out of range are clamped or passed over; outputs that are not wanted stay out."""
    torch = torch_mod
    eng.set_stream(torch.cuda.current_stream().cuda_stream)

    def dev(a):
        return torch.tensor(a, dtype=torch.int32, device="cuda")

    k = torch.empty(6, 1, 4, 8, dtype=torch.float16, device="cuda")
    cache = pkg.PagedKV(k, k, dev([[0, -1, -1], [99, 2, -1], [3, -1, -1]]), dev([-4, 100, 3]))
    held, free, count, off = dev([9, -2, 1]), dev([5, 70, 1, 4]), dev([77]), torch.zeros(4, dtype=torch.int32, device="cuda")
    slots = torch.zeros(8, dtype=torch.int64, device="cuda")
    want = plan_exact(4, 6, cache.table.cpu().numpy(), free.cpu().numpy(), 77, [-4, 100, 3], [2, 0, 4], held.tolist(), [0, 12, 3], 8, 4)
    eng.kv_plan(cache, dev([2, 0, 4]), held, free, count, off, slots=slots)
    for name, got in (("held", held), ("free", free), ("free_count", count), ("offsets", off), ("slots", slots),
                      ("table", cache.table), ("lengths", cache.lengths)):
        assert np.array_equal(got.cpu().numpy(), np.asarray(want[name])), name
    eng.kv_plan(cache, dev([1, 1, -1]), held, free, count, off)
    assert cache.lengths.tolist()[2] == 0 and off.tolist() == [0, 1, 2, 2]


# ------------------------------------------------------------ refusals

def test_refusals(torch_mod, pkg, eng):
    """Arguments that a call cannot use are errors, from Python's checks or the library's, and nothing is launched."""
    torch = torch_mod
    eng.set_stream(torch.cuda.current_stream().cuda_stream)

    def i32(*a):
        return torch.zeros(*a, dtype=torch.int32, device="cuda")

    def f(*a, dt=torch.float16):
        return torch.zeros(*a, dtype=dt, device="cuda")

    cache = pkg.PagedKV(f(4, 2, 16, 64), f(4, 2, 16, 64), i32(3, 2), i32(3))
    off, bad = i32(4), (ValueError, pkg.B200Error)
    q, out = f(5, 4, 64), f(5, 4, 64)

    def chunk(q=q, out=out, offsets=off, **kw):
        eng.kv_attend_chunk(cache, q, out, offsets, **kw)

    chunk()
    for kw in (dict(q=f(5, 3, 64), out=f(5, 3, 64)), dict(q=f(5, 4, 32), out=f(5, 4, 32)), dict(out=f(5, 4, 64, dt=torch.float32)),
               dict(q=f(5, 4, 64, dt=torch.bfloat16), out=f(5, 4, 64, dt=torch.bfloat16)), dict(offsets=i32(3)),
               dict(offsets=off.long()), dict(offsets=off.cpu()), dict(window=-1), dict(scale=math.inf), dict(scale=math.nan), dict(scale=0.0), dict(scale=-0.1),
               dict(lse=f(5, 4)), dict(lse=f(4, 4, dt=torch.float32)), dict(out=out.cpu()),
               dict(q=f(5, 4, 65)[..., 1:]), dict(q=f(5, 4, 128)[..., ::2]), dict(q=f(5, 4, 68)[..., :64]),
               dict(out=f(5 * 4 * 64 + 8)[4:5 * 4 * 64 + 4].view(5, 4, 64))):
        with pytest.raises(bad):
            chunk(**kw)
    wide = pkg.PagedKV(f(4, 2, 16, 64, dt=torch.float32), f(4, 2, 16, 64, dt=torch.float32), i32(3, 2), i32(3))
    with pytest.raises(bad):
        eng.kv_attend_chunk(wide, q, out, off)

    pos, freqs, slots = i32(5), pkg.rope_freqs(64).cuda(), torch.zeros(5, dtype=torch.int64, device="cuda")
    k = f(5, 2, 64)
    eng.rope(pos, freqs, q=q, k=k, kv=cache, v=k, slots=slots)
    for kw in (dict(), dict(q=q, positions=i32(4)), dict(q=q, positions=pos.long()), dict(q=q, freqs=freqs.int()),
               dict(q=q, freqs=pkg.rope_freqs(128).cuda()), dict(q=q, freqs=freqs[:0]), dict(q=q, v=k), dict(q=q, slots=slots),
               dict(q=q, k=f(5, 2, 32)), dict(q=q, k=f(4, 2, 64)), dict(q=q, k=f(5, 2, 64, dt=torch.float32)),
               dict(q=q, q_out=f(5, 4, 64, dt=torch.float32)), dict(q=q, q_out=f(5, 3, 64)), dict(q=q, kv=cache),
               dict(k=k, kv=cache), dict(k=k, kv=cache, slots=slots.int()), dict(k=k, kv=cache, slots=slots[:4]),
               dict(k=f(5, 3, 64), kv=cache, slots=slots), dict(k=f(5, 2, 64, dt=torch.bfloat16), kv=cache, slots=slots),
               dict(k=k, kv=cache, slots=slots, v=f(5, 2, 32)), dict(q=q, mscale=math.nan), dict(q=f(5, 4, 64, dt=torch.int16)),
               dict(q=f(5, 4, 68)[..., :64]), dict(q=q.cpu()), dict(q=f(5, 4 * 64))):
        kw = dict(dict(positions=pos, freqs=freqs), **kw)
        with pytest.raises(bad):
            eng.rope(**kw)

    x, w = f(3, 64, dt=torch.float32), f(64, dt=torch.float32)
    q8 = torch.zeros(3, 72, dtype=torch.uint8, device="cuda")
    eng.rms_norm(x, w, out=x, q8=q8)
    for kw in (dict(), dict(out=f(3, 32, dt=torch.float32)), dict(out=f(3, 64, dt=torch.int32)), dict(out=x, weight=w[:32]),
               dict(out=x, weight=w.half()), dict(out=x, residual=f(3, 64)), dict(out=x, residual_out=x), dict(out=x, eps=-1.0),
               dict(out=x, eps=math.nan), dict(out=x, eps=math.inf), dict(q8=q8[:, :64]), dict(q8=q8.int()), dict(out=x.cpu()),
               dict(x=f(3, 40, dt=torch.float32), weight=w[:40], q8=torch.zeros(3, 45, dtype=torch.uint8, device="cuda")),
               dict(x=f(3, 60, dt=torch.float32), weight=w[:60], out=f(3, 60, dt=torch.float32)),
               dict(x=f(3, 66, dt=torch.float32)[:, :64], out=x), dict(x=f(3, 64), out=x), dict(x=f(2, 3, 64), out=x),
               dict(x=f(1, 32776), weight=f(32776, dt=torch.float32), out=f(1, 32776))):
        with pytest.raises(bad):
            eng.rms_norm(**dict(dict(x=x, weight=w), **kw))

    a = dict(new=i32(3), held=i32(3), free=i32(9), free_count=i32(1), offsets=off)
    eng.kv_plan(cache, **a)
    for kw in (dict(new=i32(2)), dict(held=i32(4)), dict(held=i32(3).long()), dict(free=i32(3, 3)), dict(free_count=i32(2)),
               dict(offsets=i32(3)), dict(slots=i32(7)), dict(slots=slots, positions=i32(4)), dict(sequences=slots),
               dict(positions=i32(2, 2)), dict(seen_out=i32(3)), dict(seen=i32(2)), dict(granted=i32(2)), dict(lengths_out=i32(4)),
               dict(free_count_out=i32(0)), dict(new=i32(3).cpu())):
        with pytest.raises(bad):
            eng.kv_plan(cache, **dict(a, **kw))


def test_empty_calls(torch_mod, pkg, eng):
    """No tokens at all."""
    torch = torch_mod
    eng.set_stream(torch.cuda.current_stream().cuda_stream)
    c = chunk_case(torch, pkg, [0, 0], [5, 0], 4, 2, 64, 16, "f16", "f16")
    eng.kv_attend_chunk(c["cache"], c["q"][:0], c["out"][:0], c["offsets"], lse=c["lse"][:0])
    chunk_run(torch, eng, c)                             # rows that no sequence has
    x, w = torch.zeros(0, 64, device="cuda"), torch.ones(64, device="cuda")
    eng.rms_norm(x, w, out=x, residual=x)
    s = torch.zeros(0, dtype=torch.int64, device="cuda")
    eng.rope(s.int(), pkg.rope_freqs(64).cuda(), q=c["q"][:0], k=c["q"][:0, :2], kv=c["cache"], v=c["q"][:0, :2], slots=s)


def test_rows_in_place_that_would_move(torch_mod, pkg, eng):
    """Rows that would be written over others still to be read are refused; a row's own place in another type is not."""
    torch = torch_mod
    eng.set_stream(torch.cuda.current_stream().cuda_stream)
    g = torch.Generator().manual_seed(5)
    buf = torch.randn(6, 4, 64, generator=g).cuda()
    before, pos, freqs = buf.clone(), torch.arange(5, dtype=torch.int32).cuda(), pkg.rope_freqs(64).cuda()
    half = buf.view(torch.float16)[:5, :, :64]           # as many bytes apart, of another type
    apart = buf.as_strided((5, 2, 64), (2 * 256 // 2, 128, 1))
    for q, out in ((buf[:5], half), (buf[:5, :2], buf.as_strided((5, 2, 64), (128, 64, 1))), (buf[:5, :2], apart)):
        for kw in (dict(q=q, q_out=out), dict(k=q, k_out=out)):
            with pytest.raises(pkg.B200Error):
                eng.rope(pos, freqs, **kw)
    x, w = buf.view(6, 256)[:, :64], torch.ones(64, device="cuda")
    dense, res = buf.as_strided((6, 64), (64, 1)), torch.zeros(6, 256, device="cuda")
    for kw in (dict(out=dense), dict(out=buf.view(torch.float16).as_strided((6, 64), (256, 1))),
               dict(residual=res[:, :64], residual_out=res.as_strided((6, 64), (64, 1)))):
        with pytest.raises(pkg.B200Error):
            eng.rms_norm(x, w, **kw)
    torch.cuda.synchronize()
    assert torch.equal(buf, before)
    # one row has no strides to differ by, and a row may change its type where it stands
    want, got = torch.empty(1, 2, 64, device="cuda"), before[:1, :2].clone()
    eng.rope(pos[3:4], freqs, q=before[:1, :2], q_out=want)
    eng.rope(pos[3:4], freqs, q=got, q_out=got.as_strided((1, 2, 64), (256, 64, 1)))
    assert torch.equal(got, want)
    y = torch.empty(6, 64, dtype=torch.float16, device="cuda")
    eng.rms_norm(x, w, out=y)
    own = buf.view(torch.float16).view(6, 512)[:, :64]
    eng.rms_norm(x, w, out=own)
    assert torch.equal(own, y)
