"""The serving operators (b200_kv_append, b200_kv_attend, b200_kv_evict,
b200_sample) against plain implementations in 64 bits, at the sizes, layouts
and masks where they can go wrong, and their refusals."""

from __future__ import annotations

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

DT = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}


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


def make_cache(torch, pkg, lens, hkv, d, page, kv, seed, layout="head", extra_cols=0, garbage=None):
    """A pool with every sequence's pages in random order; rows not in use hold `garbage` where it is given."""
    rng = np.random.default_rng(seed)
    dt = getattr(torch, DT[kv])
    need = [-(-n // page) for n in lens]
    cols = max(1, max(need)) + extra_cols
    n_pages = sum(need) + 3
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if layout == "head":
        k = torch.randn(n_pages, hkv, page, d, generator=gen, device="cuda").to(dt)
        v = torch.randn(n_pages, hkv, page, d, generator=gen, device="cuda").to(dt)
    else:                              # [page][row][head][d]
        k = torch.randn(n_pages, page, hkv, d, generator=gen, device="cuda").to(dt).transpose(1, 2)
        v = torch.randn(n_pages, page, hkv, d, generator=gen, device="cuda").to(dt).transpose(1, 2)
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
    cache = pkg.PagedKV(k, v, torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"))
    return cache, table


def cache_rows(cache, table, b, h, n, pool):
    """Rows 0..n of one head as float64 numpy, NaN rows where the page is not there; and which are there."""
    page = cache.page_size
    rows = np.zeros((n, cache.head_dim))
    there = np.zeros(n, bool)
    p = pool[:, h].double().cpu().numpy()
    for s in range(n):
        pg = table[b, s // page]
        if 0 <= pg < cache.n_pages:
            rows[s], there[s] = p[pg, s % page], True
    return rows, there


# ------------------------------------------------------------------ attention

ATTEND = {
    # name: batch lengths, heads, cache heads, head size, page, q, kv, layout
    "one_slot": ([1], 4, 2, 64, 16, "f32", "f16", "head"),
    "empty_and_not": ([0, 5, 0, 17], 8, 2, 64, 16, "f16", "f16", "head"),
    "all_empty": ([0, 0], 4, 4, 128, 32, "bf16", "bf16", "head"),
    "group3_long": ([4352, 4097], 24, 8, 128, 32, "f32", "f16", "head"),
    "group4": ([200, 199, 16, 15], 32, 8, 64, 16, "f32", "f16", "row"),
    "group5_odd_page": ([333, 1, 90], 20, 4, 96, 41, "f32", "f32", "head"),
    "group8": ([1000, 31], 64, 8, 128, 64, "bf16", "bf16", "row"),
    "group7_d80": ([257, 256, 255], 14, 2, 80, 16, "f16", "f16", "row"),
    "mqa16": ([700], 16, 1, 128, 128, "bf16", "bf16", "head"),
    "mqa40_page1": ([77, 3], 40, 1, 64, 1, "f16", "f16", "head"),
    "d256": ([130, 515], 8, 2, 256, 16, "bf16", "bf16", "head"),
    "d256_f32": ([130, 70], 4, 2, 256, 16, "f32", "f32", "row"),
    "d8": ([50, 9], 4, 2, 8, 16, "f32", "f16", "head"),
    "d192_f32q": ([600], 6, 2, 192, 48, "f32", "f16", "head"),
    "d64_f32_group8": ([1023], 16, 2, 64, 64, "f32", "f32", "head"),
    "mha": ([129] * 3, 6, 6, 64, 7, "bf16", "bf16", "head"),
    "one_long": ([20011], 8, 2, 128, 64, "f32", "f16", "head"),
    "many_short": (list(range(1, 70)), 4, 2, 64, 16, "f32", "f16", "head"),
    "d256_group8": ([300, 77], 16, 2, 256, 16, "bf16", "bf16", "head"),
    "d256_f32_group6": ([210, 800], 12, 2, 256, 33, "f32", "f32", "head"),
    "batch_of_300_short": ([(7 * i) % 100 for i in range(300)], 3, 1, 64, 16, "f32", "f16", "head"),
    "batch_of_200_mixed": ([(37 * i) % 97 * (20 if i % 50 == 3 else 1) for i in range(200)], 2, 1, 64, 32, "bf16", "bf16",
                           "head"),
    "heads_of_640_and_641": ([640, 640], 8, 2, 128, 16, "f16", "f16", "head"),
    "one_head_over": ([641, 3, 640], 8, 2, 128, 16, "f16", "f16", "head"),
}


def attend_ref(cache, table, lens, q, scale):
    """In 64 bits: out, lse, the softmax's weights summed over a cache head's query heads, and per (batch, head) the
    largest sum of |scale q_i k_i| and largest |v| that bound the rounding."""
    b, h, d = q.shape
    g = h // cache.n_head_kv
    qd = q.double().cpu().numpy()
    out = np.zeros((b, h, d))
    lse = np.full((b, h), -np.inf)
    wsum = np.zeros((b, cache.n_head_kv, cache.capacity))
    sabs, vmax = np.zeros((b, h)), np.zeros((b, h))
    for i, n in enumerate(lens):
        n = min(n, cache.capacity)
        for j in range(cache.n_head_kv):
            k, there = cache_rows(cache, table, i, j, n, cache.k)
            v, _ = cache_rows(cache, table, i, j, n, cache.v)
            if not there.any():
                continue
            for x in range(j * g, (j + 1) * g):
                s = np.where(there, scale * (k @ qd[i, x]), -np.inf)
                m = s.max()
                p = np.exp(s - m)
                lse[i, x] = m + np.log(p.sum())
                p /= p.sum()
                out[i, x] = p @ np.where(there[:, None], v, 0)
                wsum[i, j, :n] += p
                sabs[i, x] = abs(scale) * (np.abs(k[there]) @ np.abs(qd[i, x])).max()
                vmax[i, x] = np.abs(v[there]).max()
    return out, lse, wsum, sabs, vmax


def attend_tol(d, n, kv, qtype, sabs):
    """Rounding that the formulas allow, of 32-bit sums: a score differs by eps_dot at most, which is (d + 16) half
    units of the sum of |q k| (16: q split in two 16-bit parts of 22 bits together); a softmax weight held in two
    16-bit parts keeps 2^-20 (float16, tf32) or 2^-15 (bfloat16) of itself; sums over n slots run in 16 parts or more."""
    eps_dot = (d + 16) * 2.0 ** -24 * sabs
    eps_sum = (64 + n / 16) * 2.0 ** -24
    eps_p = 2.0 ** -15 if kv == "bf16" else 2.0 ** -20
    ulp = {"f32": 2.0 ** -23, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[qtype]
    return eps_dot, eps_sum, eps_p, ulp


def check_attend(torch, eng, cache, table, lens, h, qtype, kv, seed, scale=None, with_weights=False, decay=1.0,
                 weights_in=True, in_place=False, qstride=False):
    b, d = cache.batch, cache.head_dim
    gen = torch.Generator(device="cuda").manual_seed(seed)
    q = (1.5 * torch.randn(b, h, d, generator=gen, device="cuda")).to(getattr(torch, DT[qtype]))
    out = torch.full_like(q, 7.0)
    if qstride:                        # heads before sequences, rows 8 elements apart, in both
        q = torch.empty(h, b, d + 8, dtype=q.dtype, device="cuda")[:, :, :d].transpose(0, 1).copy_(q)
        out = torch.full((h, b, d + 24), 7.0, dtype=q.dtype, device="cuda")[:, :, 8:8 + d].transpose(0, 1)
    lse = torch.full((b, h), 7.0, device="cuda")
    kw = {}
    if with_weights:
        w0 = torch.rand(b, cache.n_head_kv, cache.capacity + 5, generator=gen, device="cuda")
        win = w0.clone()
        wout = win if in_place else torch.full_like(w0, -3.0)
        kw = dict(weights=win if weights_in else None, weights_out=wout, decay=decay)
    torch.cuda.synchronize()
    eng.kv_attend(cache, q, out, lse, scale=scale, **kw)
    eng.sync()
    sc = d ** -0.5 if scale is None else scale
    r_out, r_lse, r_w, sabs, vmax = attend_ref(cache, table, lens, q, sc)
    n = max(lens) if lens else 0
    eps_dot, eps_sum, eps_p, ulp = attend_tol(d, n, kv, qtype, sabs)
    got = out.double().cpu().numpy()
    tol = (vmax * (2 * eps_dot + eps_sum + eps_p))[..., None] + ulp * np.abs(r_out)
    assert np.isfinite(got).all()
    assert (np.abs(got - r_out) <= tol).all(), np.max(np.abs(got - r_out) - tol)
    gl = lse.double().cpu().numpy()
    empty = np.isneginf(r_lse)
    assert (np.isneginf(gl) == empty).all()
    ltol = eps_dot + eps_sum + 2.0 ** -22 * (1 + np.abs(np.where(empty, 0, r_lse)))
    assert (np.abs(np.where(empty, 0, gl) - np.where(empty, 0, r_lse)) <= ltol).all()
    if with_weights:
        g = h // cache.n_head_kv
        used = np.zeros((b, 1, cache.capacity + 5), bool)
        for i, x in enumerate(lens):
            used[i, :, :min(x, cache.capacity)] = True
        base = w0.double().cpu().numpy() * (decay if weights_in else 0.0)
        want = base.copy()
        want[:, :, :cache.capacity] += r_w
        worst = eps_dot.reshape(b, cache.n_head_kv, g).max(2)[..., None]
        wtol = np.zeros_like(want)
        wtol[:, :, :cache.capacity] = r_w * (2 * worst + eps_sum + 2.0 ** -20)
        wtol += 2.0 ** -22 * np.abs(want) + 1e-30
        gw = wout.double().cpu().numpy()
        old = (w0 if in_place else torch.full_like(w0, -3.0)).double().cpu().numpy()
        assert np.array_equal(np.where(used, 0, gw), np.where(used, 0, old))      # slots not in use are left alone
        assert (np.where(used, np.abs(gw - want), 0) <= wtol).all()
    return out, lse


@pytest.mark.parametrize("name", list(ATTEND))
def test_attend_matches_the_formula(torch_mod, pkg, eng, name):
    lens, h, hkv, d, page, qtype, kv, layout = ATTEND[name]
    cache, table = make_cache(torch_mod, pkg, lens, hkv, d, page, kv, seed=len(name), layout=layout)
    check_attend(torch_mod, eng, cache, table, lens, h, qtype, kv, seed=7)


@pytest.mark.parametrize("name", ["empty_and_not", "group3_long", "group5_odd_page", "group8", "mqa40_page1", "d256",
                                  "many_short"])
@pytest.mark.parametrize("mode", ["beside", "in_place", "from_zero"])
def test_attend_adds_up_the_weights(torch_mod, pkg, eng, name, mode):
    lens, h, hkv, d, page, qtype, kv, layout = ATTEND[name]
    cache, table = make_cache(torch_mod, pkg, lens, hkv, d, page, kv, seed=3, layout=layout, extra_cols=1)
    check_attend(torch_mod, eng, cache, table, lens, h, qtype, kv, seed=8, with_weights=True,
                 decay=0.75 if mode == "in_place" else 1.0, weights_in=mode != "from_zero", in_place=mode == "in_place")


@pytest.mark.parametrize("garbage", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("name", ["empty_and_not", "group4", "group5_odd_page", "group7_d80", "d256"])
def test_attend_reads_nothing_of_unused_rows(torch_mod, pkg, eng, name, garbage):
    lens, h, hkv, d, page, qtype, kv, layout = ATTEND[name]
    cache, table = make_cache(torch_mod, pkg, lens, hkv, d, page, kv, seed=4, layout=layout, garbage=garbage)
    check_attend(torch_mod, eng, cache, table, lens, h, qtype, kv, seed=9, with_weights=True)


@pytest.mark.parametrize("kv,qtype", [("f16", "f32"), ("bf16", "bf16"), ("f32", "f32")])
def test_attend_skips_pages_that_are_not_there(torch_mod, pkg, eng, kv, qtype):
    torch = torch_mod
    lens = [100, 64, 33, 5000]                  # the last one passes its columns
    cache, table = make_cache(torch, pkg, [100, 64, 33, 112], 2, 64, 16, kv, seed=5)
    table[0, 2], table[0, 3], table[1, :], table[3, 0] = -1, cache.n_pages, -7, 2 ** 31 - 1
    cache.table.copy_(torch.from_numpy(table))
    cache.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
    check_attend(torch, eng, cache, table, lens, 8, qtype, kv, seed=10, with_weights=True)
    cache.lengths.copy_(torch.tensor([-5, 0, -2 ** 31, 3], dtype=torch.int32))
    table[3, 0] = 0
    cache.table.copy_(torch.from_numpy(table))
    check_attend(torch, eng, cache, table, [0, 0, 0, 3], 8, qtype, kv, seed=11, with_weights=True)


def test_attend_strides_scale_and_large_scores(torch_mod, pkg, eng):
    lens, h, hkv, d, page, qtype, kv, layout = ATTEND["group4"]
    cache, table = make_cache(torch_mod, pkg, lens, hkv, d, page, kv, seed=6, layout=layout)
    check_attend(torch_mod, eng, cache, table, lens, h, qtype, kv, seed=12, qstride=True)
    check_attend(torch_mod, eng, cache, table, lens, h, "f16", kv, seed=12, qstride=True)
    check_attend(torch_mod, eng, cache, table, lens, h, qtype, kv, seed=12, scale=2.0)       # scores of +-60
    check_attend(torch_mod, eng, cache, table, lens, h, qtype, kv, seed=12, scale=0.0)       # all weights equal
    check_attend(torch_mod, eng, cache, table, lens, h, qtype, kv, seed=12, scale=-0.3)


def test_attend_small_and_large_queries(torch_mod, pkg, eng):
    """float32 queries whose size float16 does not hold: scores are those of the float32 values."""
    torch = torch_mod
    cache, table = make_cache(torch, pkg, [90, 300], 2, 64, 16, "f16", seed=13)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for size in (1e-12, 1e12):
        q = size * torch.randn(2, 8, 64, generator=gen, device="cuda")
        out, lse = torch.empty_like(q), torch.empty(2, 8, device="cuda")
        torch.cuda.synchronize()
        eng.kv_attend(cache, q, out, lse, scale=1.0 / size / 8)
        eng.sync()
        r_out, r_lse, _, sabs, vmax = attend_ref(cache, table, [90, 300], q, float(np.float32(1.0 / size / 8)))
        eps_dot, eps_sum, eps_p, ulp = attend_tol(64, 300, "f16", "f32", sabs)
        assert (np.abs(out.double().cpu().numpy() - r_out)
                <= (vmax * (2 * eps_dot + eps_sum + eps_p))[..., None] + ulp * np.abs(r_out)).all()
        assert (np.abs(lse.double().cpu().numpy() - r_lse) <= eps_dot + eps_sum + 2.0 ** -22 * (1 + np.abs(r_lse))).all()


def test_attend_offsets_past_32_bits(torch_mod, pkg, eng):
    """Pages at more than 2^32 bytes into the pool."""
    torch = torch_mod
    hkv, d, page, n_pages = 8, 128, 64, 40000                   # 5.2 GB a pool
    k = torch.empty(n_pages, hkv, page, d, dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    lens = [130, 70]
    table = np.array([[39999, 1, 33333], [0, 38000, -1]], np.int32)
    for p in (39999, 1, 33333, 0, 38000):
        k[p].normal_()
        v[p].normal_()
    cache = pkg.PagedKV(k, v, torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"))
    gen = torch.Generator(device="cuda").manual_seed(2)
    q = torch.randn(2, 16, d, generator=gen, device="cuda")
    out, lse = torch.empty_like(q), torch.empty(2, 16, device="cuda")
    torch.cuda.synchronize()
    eng.kv_attend(cache, q, out, lse)
    eng.sync()
    for i, n in enumerate(lens):
        idx = torch.tensor([table[i, s // page] for s in range(n)], device="cuda").long()
        sl = torch.arange(n, device="cuda") % page
        kk, vv = k[idx, :, sl].double(), v[idx, :, sl].double()           # n hkv d
        s = torch.einsum("hgd,nhd->hgn", q[i].double().view(hkv, 2, d), kk) / math.sqrt(d)
        want = torch.einsum("hgn,nhd->hgd", torch.softmax(s, 2), vv).reshape(16, d)
        assert (out[i].double() - want).abs().max() < 1e-4
        assert (lse[i].double() - torch.logsumexp(s, 2).reshape(16)).abs().max() < 1e-4


def test_attend_repeats_to_the_bit_and_in_a_graph(torch_mod, pkg):
    """The same call gives the same bits again, on a stream of its own and replayed from a graph, also after lengths
    changed under it."""
    torch = torch_mod
    stream = torch.cuda.Stream()
    e = pkg.Engine(0, stream=stream.cuda_stream)
    lens = [3000, 0, 77, 1500]
    cache, table = make_cache(torch, pkg, lens, 4, 128, 32, "bf16", seed=20)
    q = torch.randn(4, 16, 128, device="cuda", dtype=torch.bfloat16)
    out, lse = torch.zeros_like(q), torch.zeros(4, 16, device="cuda")
    w = torch.zeros(4, 4, cache.capacity, device="cuda")
    torch.cuda.synchronize()

    def call():
        e.kv_attend(cache, q, out, lse, weights_out=w)

    call()
    e.sync()
    first = [t.clone() for t in (out, lse, w)]
    e.capture_begin()
    call()
    g = e.capture_end()
    for n in (lens, [5, 6, 0, 2999], lens):
        cache.lengths.copy_(torch.tensor(n, dtype=torch.int32))
        for t in (out, lse, w):
            t.zero_()
        torch.cuda.synchronize()
        g.launch()
        e.sync()
    assert all(torch.equal(a, b) for a, b in zip(first, (out, lse, w)))
    g.close()
    e.close()


def test_attend_graph_outlives_a_larger_call(torch_mod, pkg):
    """A captured call keeps its workspace when a later call needs a larger one."""
    torch = torch_mod
    stream = torch.cuda.Stream()
    e = pkg.Engine(0, stream=stream.cuda_stream)
    cache, _ = make_cache(torch, pkg, [700, 90], 2, 64, 16, "f16", seed=21)
    q = torch.randn(2, 8, 64, device="cuda")
    out, w = torch.zeros_like(q), torch.zeros(2, 2, cache.capacity, device="cuda")
    torch.cuda.synchronize()
    e.kv_attend(cache, q, out, weights_out=w)
    e.sync()
    first = [out.clone(), w.clone()]
    e.capture_begin()
    e.kv_attend(cache, q, out, weights_out=w)
    g = e.capture_end()
    big, _ = make_cache(torch, pkg, [3000] * 40, 2, 128, 16, "f16", seed=22)
    q2 = torch.randn(40, 16, 128, device="cuda")
    out2, w2 = torch.empty_like(q2), torch.empty(40, 2, big.capacity, device="cuda")
    torch.cuda.synchronize()
    e.kv_attend(big, q2, out2, weights_out=w2)
    filler = [torch.full((1 << 20,), 7.0, device="cuda") for _ in range(16)]      # what would take a freed workspace
    out.zero_(), w.zero_()
    torch.cuda.synchronize()
    g.launch()
    e.sync()
    assert torch.equal(first[0], out) and torch.equal(first[1], w)
    assert all(bool((f == 7.0).all()) for f in filler)
    g.close()
    e.close()


# ------------------------------------------------------------------ append

@pytest.mark.parametrize("src,kv", [("f32", "f16"), ("f32", "bf16"), ("f32", "f32"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("news", ["one", "ragged", "none"])
@pytest.mark.parametrize("layout", ["head", "row"])
def test_append_puts_rows_behind_the_slots_in_use(torch_mod, pkg, eng, src, kv, news, layout):
    torch = torch_mod
    hkv, d, page = 3, 40, 7
    lens = [0, 5, 13, 20, 7]
    new = {"one": [1] * 5, "ragged": [3, 0, 11, 1, 30], "none": [0] * 5}[news]
    cache, table = make_cache(torch, pkg, [a + b for a, b in zip(lens, new)], hkv, d, page, kv, seed=1, layout=layout)
    cache.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
    n = sum(new)
    kn = torch.randn(n, hkv, d + 8, device="cuda").to(getattr(torch, DT[src]))[:, :, :d]
    vn = torch.randn(n, hkv, d + 8, device="cuda").to(getattr(torch, DT[src]))[:, :, :d]
    off = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda")
    seen = torch.tensor([10, 20, 30, 40, 50], dtype=torch.int32, device="cuda")
    pos = torch.full((5, hkv, cache.capacity + 2), -9, dtype=torch.int32, device="cuda")
    w = torch.full((5, hkv, cache.capacity + 2), -9.0, device="cuda")
    want_k, want_v, want_pos, want_w = cache.k.clone(), cache.v.clone(), pos.clone(), w.clone()
    t = 0
    for b in range(5):
        for i in range(new[b]):
            s = lens[b] + i
            want_k[table[b, s // page], :, s % page] = kn[t].to(cache.k.dtype)
            want_v[table[b, s // page], :, s % page] = vn[t].to(cache.v.dtype)
            want_pos[b, :, s] = 10 * (b + 1) + i
            want_w[b, :, s] = 0.0
            t += 1
    torch.cuda.synchronize()
    eng.kv_append(cache, kn, vn, offsets=None if news == "one" else off, seen=seen, positions=pos, weights=w)
    eng.sync()
    assert torch.equal(cache.k, want_k) and torch.equal(cache.v, want_v)
    assert torch.equal(pos, want_pos) and torch.equal(w, want_w)
    assert cache.lengths.tolist() == [a + b for a, b in zip(lens, new)]
    assert seen.tolist() == [10 * (b + 1) + new[b] for b in range(5)]


def test_append_drops_what_does_not_fit(torch_mod, pkg, eng):
    """Rows past the last slot or in pages that are not there are dropped; the lengths stay within the slots."""
    torch = torch_mod
    cache, table = make_cache(torch, pkg, [30, 30, 30], 2, 64, 16, "f16", seed=2)
    table[1, 1] = cache.n_pages
    cache.table.copy_(torch.from_numpy(table))
    cache.lengths.copy_(torch.tensor([30, 14, 2 ** 31 - 1], dtype=torch.int32))
    kn, vn = torch.randn(10, 2, 64, device="cuda"), torch.randn(10, 2, 64, device="cuda")
    off = torch.tensor([0, 4, 8, 10], dtype=torch.int32, device="cuda")
    want_k, want_v = cache.k.clone(), cache.v.clone()
    for want, new in ((want_k, kn), (want_v, vn)):
        want[table[0, 1], :, 14:16] = new[0:2].transpose(0, 1).half()
        want[table[1, 0], :, 14:16] = new[4:6].transpose(0, 1).half()
    out, seen_out = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    eng.kv_append(cache, kn, vn, offsets=off, lengths_out=out, seen_out=seen_out)
    eng.sync()
    assert torch.equal(cache.k, want_k) and torch.equal(cache.v, want_v)
    assert out.tolist() == [32, 18, 32] and seen_out.tolist() == [34, 18, 34]
    assert cache.lengths.tolist() == [30, 14, 2 ** 31 - 1]


def test_append_many_tokens_in_place_lengths(torch_mod, pkg, eng):
    """Lengths replaced while thousands of CTAs read them."""
    torch = torch_mod
    new = [5000, 1, 0, 7777, 300]
    lens = [3, 100, 50, 0, 9]
    cache, table = make_cache(torch, pkg, [a + b for a, b in zip(lens, new)], 2, 64, 64, "bf16", seed=3)
    cache.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
    n = sum(new)
    kn = torch.randn(n, 2, 64, device="cuda").bfloat16()
    off = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda")
    for turn in range(3):                       # the ticket is ready again for the next call
        cache.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
        cache.k.zero_()
        torch.cuda.synchronize()
        eng.kv_append(cache, kn, kn, offsets=off)
        eng.sync()
        assert cache.lengths.tolist() == [a + b for a, b in zip(lens, new)]
        for b in range(5):
            s = torch.arange(lens[b], lens[b] + new[b], device="cuda")
            pg = torch.from_numpy(table[b]).cuda().long()[s // 64]
            assert torch.equal(cache.k[pg, :, s % 64], kn[int(off[b]):int(off[b + 1])])


# ------------------------------------------------------------------ eviction

def evict_ref(cache, table, lens, w, pos, seen, budget, recent, sinks):
    """By the definition, one (sequence, head) at a time: new k, v, weights, positions, lengths."""
    page = cache.page_size
    k, v = cache.k.clone(), cache.v.clone()
    wo, po = {}, {}
    for b, n in enumerate(lens):
        for h in range(cache.n_head_kv):
            ww, pp = w[b, h, :n].copy(), pos[b, h, :n].copy()
            if n > budget:
                fixed = (pp >= seen[b] - recent) | (pp < sinks)
                score = np.where(np.isnan(ww), -np.inf, ww.astype(np.float64))
                nan = np.isnan(ww)
                order = sorted(range(n), key=lambda i: (not fixed[i], nan[i] and not fixed[i],
                                                        0 if fixed[i] else -score[i], i))
                kept = np.zeros(n, bool)
                kept[order[:budget]] = True
                frm = [i for i in range(budget, n) if kept[i]]
                to = [i for i in range(budget) if not kept[i]]
                assert len(frm) == len(to)
                for f, t in zip(frm, to):
                    ww[t], pp[t] = ww[f], pp[f]
                    pf, pt = table[b, f // page], table[b, t // page]
                    k[pt, h, t % page] = cache.k[pf, h, f % page]
                    v[pt, h, t % page] = cache.v[pf, h, f % page]
            wo[b, h], po[b, h] = ww[:budget], pp[:budget]
    return k, v, wo, po, [min(n, budget) for n in lens]


EVICT = {
    # lengths, heads, head size, page, type, budget, recent, sinks, weights
    "step": ([65, 65, 64, 3, 0], 3, 64, 16, "f16", 64, 8, 2, "random"),
    "prompt": ([700, 333, 90], 2, 128, 64, "bf16", 100, 30, 4, "random"),
    "odd_page_f32": ([130, 129], 2, 40, 7, "f32", 33, 0, 0, "random"),
    "ties": ([200, 150], 2, 64, 16, "f16", 70, 5, 3, "ties"),
    "all_equal": ([300], 2, 64, 16, "f16", 77, 10, 0, "equal"),
    "nan_inf": ([120, 60], 2, 64, 16, "f16", 40, 4, 2, "nan"),
    "negative_zero": ([64], 1, 64, 16, "f16", 20, 0, 0, "zero"),
    "budget_is_recent": ([100, 40], 2, 64, 16, "f16", 30, 30, 0, "random"),
    "budget_one": ([50, 1, 0, 2], 2, 64, 16, "f16", 1, 0, 0, "random"),
    "all_but_one": ([2, 1000], 1, 64, 128, "bf16", 999, 100, 1, "random"),
    "more_moves_than_one_list": ([9000], 1, 64, 64, "f16", 4400, 2500, 0, "random"),
    "long": ([70000], 1, 8, 64, "f16", 30000, 1000, 4, "random"),
    "longer_than_shared_memory": ([300000, 5000], 1, 8, 64, "f16", 1500, 100, 4, "random"),
}


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("name", list(EVICT))
def test_evict_keeps_what_the_definition_keeps(torch_mod, pkg, eng, name, in_place):
    torch = torch_mod
    lens, hkv, d, page, kv, budget, recent, sinks, kind = EVICT[name]
    rng = np.random.default_rng(len(name))
    cache, table = make_cache(torch, pkg, lens, hkv, d, page, kv, seed=5, layout="row" if hkv == 3 else "head")
    cap = cache.capacity + 3
    w = np.exp(rng.standard_normal((len(lens), hkv, cap))).astype(np.float32)
    if kind == "ties":
        w = rng.integers(0, 4, w.shape).astype(np.float32)
    elif kind == "equal":
        w[:] = 2.5
    elif kind == "nan":
        w[rng.random(w.shape) < 0.3] = np.nan
        w[rng.random(w.shape) < 0.2] = np.inf
        w[rng.random(w.shape) < 0.2] = -np.inf
    elif kind == "zero":
        w = np.where(rng.random(w.shape) < 0.5, np.float32(-0.0), np.float32(0.0))
    pos = np.zeros((len(lens), hkv, cap), np.int32)
    for b, n in enumerate(lens):
        for h in range(hkv):
            pos[b, h, :n] = rng.permutation(n)
    k, v, wo, po, new = evict_ref(cache, table, lens, w, pos, lens, budget, recent, sinks)
    tw, tp = torch.from_numpy(w).cuda(), torch.from_numpy(pos).cuda()
    seen = torch.tensor(lens, dtype=torch.int32, device="cuda")
    kw = {}
    if not in_place:
        kw = dict(weights_out=torch.full_like(tw, -3.0), positions_out=torch.full_like(tp, -3),
                  lengths_out=torch.full_like(seen, -3))
    torch.cuda.synchronize()
    eng.kv_evict(cache, tw, tp, seen, budget, recent=recent, sinks=sinks, **kw)
    eng.sync()
    assert torch.equal(cache.k, k) and torch.equal(cache.v, v)
    gw = kw.get("weights_out", tw).cpu().numpy()
    gp = kw.get("positions_out", tp).cpu().numpy()
    assert kw.get("lengths_out", cache.lengths).tolist() == new
    for b, n in enumerate(lens):
        m = min(n, budget)
        for h in range(hkv):
            assert np.array_equal(gw[b, h, :m].view(np.uint32), wo[b, h].view(np.uint32))
            assert np.array_equal(gp[b, h, :m], po[b, h])
            old_w, old_p = (w, pos) if in_place else (np.full_like(w, -3), np.full_like(pos, -3))
            assert np.array_equal(gw[b, h, m:], old_w[b, h, m:], equal_nan=True)     # nothing past the new length
            assert np.array_equal(gp[b, h, m:], old_p[b, h, m:])


def test_evict_with_more_kept_positions_than_budget_and_missing_pages(torch_mod, pkg, eng):
    """Positions that repeat, a `seen` out of step, pages that are not there: the count still comes out, and rows
    only move between pages that are there."""
    torch = torch_mod
    lens = [90, 80]
    cache, table = make_cache(torch, pkg, lens, 2, 64, 16, "f16", seed=6)
    table[0, 4], table[1, 0] = -1, cache.n_pages + 5
    cache.table.copy_(torch.from_numpy(table))
    w = np.random.default_rng(1).random((2, 2, cache.capacity)).astype(np.float32)
    pos = np.full(w.shape, 1000, np.int32)
    order = np.arange(cache.capacity)
    before_k = cache.k.clone()
    tw, tp = torch.from_numpy(w).cuda(), torch.from_numpy(pos).cuda()
    torch.cuda.synchronize()
    eng.kv_evict(cache, tw, tp, torch.zeros(2, dtype=torch.int32, device="cuda"), 40, recent=10)
    eng.sync()
    # every token counts as recent: the lower slots stay, nothing moves
    assert cache.lengths.tolist() == [40, 40]
    assert torch.equal(cache.k, before_k)
    assert np.array_equal(tw.cpu().numpy(), w) and order.size == cache.capacity
    cache.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
    pos[:] = order
    w[:, :, :] = order                     # the upper slots win: 50..89 -> 0..39 and 40..79 -> 0..39
    tw, tp = torch.from_numpy(w).cuda(), torch.from_numpy(pos).cuda()
    torch.cuda.synchronize()
    eng.kv_evict(cache, tw, tp, torch.tensor(lens, dtype=torch.int32, device="cuda"), 40)
    eng.sync()
    assert np.array_equal(tw.cpu().numpy()[0, 0, :40], np.arange(50, 90, dtype=np.float32))
    assert np.array_equal(tp.cpu().numpy()[1, 1, :40], np.arange(40, 80))
    want = before_k.clone()
    for b, shift in ((0, 50), (1, 40)):
        for t in range(40):
            pf, pt = table[b, (t + shift) // 16], table[b, t // 16]
            if 0 <= pf < cache.n_pages and 0 <= pt < cache.n_pages:
                want[pt, :, t % 16] = before_k[pf, :, (t + shift) % 16]
    assert torch.equal(cache.k, want)


# ------------------------------------------------------------------ sampling

def sample_check(x, t, k, p, m, u, token, logprob):
    """The token is one that the definition gives in 64 bits, and its log-probability is near. A weight in 32 bits is
    off by up to 2^-23 of its exponent's size (40 at most) and 2 units of exp2, so by eps = 4e-6 of itself: the
    prefix sums where top-p and u fall, and min-p's edge, may differ by that much."""
    eps = 4e-6
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    top = x.max()
    if top == -np.inf:
        assert token == -1 and logprob == -np.inf
        return
    if not t > 0:
        assert token == int(np.argmax(x)) and logprob == 0
        return
    if top == np.inf:
        w = (x == np.inf).astype(np.float64)
    else:
        with np.errstate(invalid="ignore"):
            w = np.where(x == -np.inf, 0.0, np.exp((x - top) / t))
    w[w < 2.0 ** -40 * (1 - eps)] = 0.0
    order = np.argsort(-x, kind="stable")
    ws = w[order]
    kk = k if 0 < k < x.size else x.size
    c = np.cumsum(ws[:kk])
    cuts = set()
    for e in (-eps, 0.0, eps):
        n = kk
        if p < 1:
            n = min(kk, int((c < max(p, 0.0) * (1 + e) * c[-1]).sum()) + 1)
        nm = kk
        if m > 0:
            nm = max(1, int((ws >= m * (1 + e)).sum())) if m <= 1 else 1
        cuts.add(max(1, min(n, nm)))
    for n in range(min(cuts), max(cuts) + 1):
        kept = np.zeros_like(w)
        kept[order[:n]] = ws[:n]
        cum = np.cumsum(kept)
        if kept[token] <= 0:
            continue
        lo, hi = (cum[token] - kept[token]) / cum[-1], cum[token] / cum[-1]
        uu = min(max(u if u == u else 0.0, 0.0), 1.0)
        want = np.log(kept[token] / cum[-1])
        if lo - eps <= uu <= hi + eps and abs(logprob - want) <= 2e-5 + 1e-6 * abs(want):
            return
    raise AssertionError(f"token {token} is none that the definition gives")


def run_sample(torch, eng, x, u, t=None, k=None, p=None, m=None, dtype="f32", stride=0):
    b, n = x.shape
    tx = torch.empty(b, n + stride, dtype=getattr(torch, DT[dtype]), device="cuda")[:, :n]
    tx.copy_(torch.from_numpy(x))
    dev = {}
    for name, a, ty in (("temperature", t, np.float32), ("top_k", k, np.int32), ("top_p", p, np.float32),
                        ("min_p", m, np.float32)):
        dev[name] = None if a is None else torch.from_numpy(np.asarray(a, ty)).cuda()
    token = torch.full((b,), -77, dtype=torch.int32, device="cuda")
    lp = torch.full((b,), 77.0, device="cuda")
    torch.cuda.synchronize()
    eng.sample(tx, torch.from_numpy(np.asarray(u, np.float32)).cuda(), token, lp, **dev)
    eng.sync()
    return tx.float().cpu().numpy(), token.cpu().numpy(), lp.cpu().numpy()


FILTERS = {"none": (1.0, 0, 1.0, 0.0), "k": (0.8, 40, 1.0, 0.0), "p": (1.0, 0, 0.9, 0.0), "m": (1.2, 0, 1.0, 0.05),
           "kp": (0.9, 100, 0.95, 0.0), "kpm": (0.7, 50, 0.9, 0.02), "pm": (1.5, 0, 0.99, 0.001), "k1": (1.0, 1, 1.0, 0.0),
           "k_all_but_one": (2.0, -1, 1.0, 0.0), "tiny_p": (1.0, 0, 1e-6, 0.0), "p0": (1.0, 0, 0.0, 0.0),
           "hot": (50.0, 0, 0.999, 0.0), "cold": (0.01, 0, 0.9, 0.0)}


@pytest.mark.parametrize("name", list(FILTERS))
@pytest.mark.parametrize("n,dtype", [(1, "f32"), (33, "f16"), (1000, "f32"), (50257, "bf16"), (128256, "f32")])
def test_sample_matches_the_definition(torch_mod, eng, name, n, dtype):
    t, k, p, m = FILTERS[name]
    if k < 0:
        k = n - 1
    rng = np.random.default_rng(n + len(name))
    b = 6
    x = (2.5 * rng.standard_normal((b, n))).astype(np.float32)
    u = rng.random(b).astype(np.float32)
    u[0], u[1] = 0.0, np.float32(1 - 2.0 ** -24)
    got = run_sample(torch_mod, eng, x, u, [t] * b, [k] * b, [p] * b, [m] * b, dtype, stride=3)
    for i in range(b):
        sample_check(got[0][i], np.float32(t), k, np.float32(p), np.float32(m), u[i], int(got[1][i]), got[2][i])


def test_sample_each_row_has_settings_of_its_own(torch_mod, eng):
    rng = np.random.default_rng(3)
    b, n = 64, 4999
    x = (3 * rng.standard_normal((b, n))).astype(np.float32)
    t = rng.choice([0.0, -1.0, np.nan, 0.5, 1.0, 2.0], b).astype(np.float32)
    k = rng.choice([-3, 0, 1, 7, 500, n, n + 5], b).astype(np.int32)
    p = rng.choice([0.2, 0.9, 1.0, 1.5, -0.5], b).astype(np.float32)
    m = rng.choice([0.0, -1.0, 0.1, 1.0, 3.0], b).astype(np.float32)
    u = rng.random(b).astype(np.float32)
    got = run_sample(torch_mod, eng, x, u, t, k, p, m)
    for i in range(b):
        sample_check(got[0][i], t[i], int(k[i]), p[i], m[i], u[i], int(got[1][i]), got[2][i])
    got2 = run_sample(torch_mod, eng, x, u, t, k, p, m)
    assert np.array_equal(got[1], got2[1]) and np.array_equal(got[2], got2[2])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sample_masks_infinities_and_ties(torch_mod, eng, dtype):
    rng = np.random.default_rng(4)
    n = 3001
    low = -3.0e38
    rows = [np.full(n, -np.inf), np.full(n, np.nan), np.zeros(n), np.full(n, low)]
    a = rng.standard_normal(n)
    a[::2] = -np.inf
    rows.append(a)
    a = rng.standard_normal(n)
    a[::3] = low
    rows.append(a)
    a = rng.standard_normal(n)
    a[[5, 900, 2999]] = np.inf
    rows.append(a)
    a = rng.standard_normal(n)
    a[rng.integers(0, n, 500)] = np.nan
    rows.append(a)
    rows.append(np.round(2 * rng.standard_normal(n)))           # few values, many ties
    a = np.full(n, -np.inf)
    a[1234] = -5.0
    rows.append(a)
    rows.append(np.where(np.arange(n) % 2, 0.0, -0.0))
    x = np.stack(rows).astype(np.float32)
    b = x.shape[0]
    for t, k, p, m in [(1.0, 0, 1.0, 0.0), (1.0, 10, 1.0, 0.0), (0.7, 0, 0.5, 0.0), (1.0, 100, 0.8, 0.3), (0.0, 0, 1.0, 0.0),
                       (1.0, 2990, 0.9, 0.0)]:
        for u in (0.0, 0.31, 0.77, 1 - 2.0 ** -24):
            got = run_sample(torch_mod, eng, x, [u] * b, [t] * b, [k] * b, [p] * b, [m] * b, dtype)
            for i in range(b):
                sample_check(got[0][i], t, k, np.float32(p), np.float32(m), np.float32(u), int(got[1][i]), got[2][i])


def test_sample_ties_at_the_edge_go_to_the_lowest_indexes(torch_mod, eng):
    """Equal logits and top-k 5: tokens 0..4 share the draw evenly."""
    x = np.zeros((10, 777), np.float32)
    u = (np.arange(10) + 0.5) / 10
    _, token, lp = run_sample(torch_mod, eng, x, u, k=[5] * 10)
    assert token.tolist() == [0, 0, 1, 1, 2, 2, 3, 3, 4, 4]
    assert np.allclose(lp, -np.log(5), atol=1e-6)
    _, token, _ = run_sample(torch_mod, eng, x, u, p=[4.5 / 777] * 10)
    assert token.tolist() == [0, 0, 1, 1, 2, 2, 3, 3, 4, 4]


def test_sample_odd_numbers_and_extreme_temperatures(torch_mod, eng):
    rng = np.random.default_rng(6)
    x = rng.standard_normal((6, 999)).astype(np.float32)
    u = np.array([np.nan, -1.0, 2.0, np.inf, -np.inf, 1e-30], np.float32)
    got = run_sample(torch_mod, eng, x, u)
    for i in range(6):
        sample_check(x[i], 1.0, 0, 1.0, 0.0, u[i], int(got[1][i]), got[2][i])
    t = np.array([1e-45, np.inf, 3e38, 1e-38, 1e-3, 1e3], np.float32)
    u = rng.random(6).astype(np.float32)
    got = run_sample(torch_mod, eng, x, u, t=t)
    assert got[1][0] == np.argmax(x[0]) and got[1][3] == np.argmax(x[3])
    assert got[1][1] == int(u[1] * 999) and got[1][2] == int(u[2] * 999)
    for i in (4, 5):
        sample_check(x[i], t[i], 0, 1.0, 0.0, u[i], int(got[1][i]), got[2][i])


def test_sample_large_vocabulary(torch_mod, eng):
    rng = np.random.default_rng(7)
    x = (2 * rng.standard_normal((3, 1_000_003))).astype(np.float32)
    u = np.array([0.2, 0.5, 0.999], np.float32)
    for k, p in ((0, 1.0), (1000, 0.9), (0, 0.95)):
        got = run_sample(torch_mod, eng, x, u, k=[k] * 3, p=[p] * 3)
        for i in range(3):
            sample_check(x[i], 1.0, k, np.float32(p), 0.0, u[i], int(got[1][i]), got[2][i])


def test_sample_follows_the_distribution(torch_mod, eng):
    """u on an even grid: each token comes as often as its share of the grid."""
    rng = np.random.default_rng(8)
    x1 = (1.5 * rng.standard_normal(50)).astype(np.float32)
    g = 4096
    x = np.broadcast_to(x1, (g, 50)).copy()
    _, token, _ = run_sample(torch_mod, eng, x, (np.arange(g) + 0.5) / g)
    p = np.exp(x1.astype(np.float64))
    p /= p.sum()
    assert (np.abs(np.bincount(token, minlength=50) - g * p) <= 1.01).all()


# ------------------------------------------------------------------ refusals

def test_refusals(torch_mod, pkg, eng):
    import copy
    import ctypes
    torch, capi, lib = torch_mod, pkg.capi, pkg.lib()
    cache, _ = make_cache(torch, pkg, [40, 20], 2, 64, 16, "f16", seed=1)
    q = torch.zeros(2, 4, 64, device="cuda")
    lse = torch.zeros(2, 4, device="cuda")
    aux = torch.zeros(2, 2, cache.capacity, device="cuda")
    pos = torch.zeros(2, 2, cache.capacity, dtype=torch.int32, device="cuda")
    seen = torch.zeros(2, dtype=torch.int32, device="cuda")
    new = torch.zeros(2, 2, 64, device="cuda")
    ap = capi.b200_kv_append_t(new.data_ptr(), new.data_ptr(), 0, 2, 128, 64, 0, 0, 0, 0, 0, 0, 0)
    ws = torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")
    at = capi.b200_kv_attend_t(q.data_ptr(), q.data_ptr(), 0, 4, 256, 64, 256, 64, 0.125, lse.data_ptr(), 0, 0, 0, 1.0,
                               ws.data_ptr(), ws.numel())
    ev = capi.b200_kv_evict_t(aux.data_ptr(), aux.data_ptr(), pos.data_ptr(), pos.data_ptr(), cache.capacity,
                              seen.data_ptr(), 0, 8, 2, 1)
    sm = capi.b200_sample_t(q.data_ptr(), 0, 2, 256, 256, 0, 0, 0, 0, lse.data_ptr(), seen.data_ptr(), 0)

    def refused(call, kv, arg, **change):
        kv, arg = copy.copy(kv), copy.copy(arg)
        for key, val in change.items():
            if key.startswith("kv_"):
                setattr(kv, key[3:], val)
            else:
                setattr(arg, key, val)
        rc = call(eng.h, ctypes.byref(kv), ctypes.byref(arg)) if kv is not None else call(eng.h, ctypes.byref(arg))
        assert rc == -22, (change, rc)
        assert lib.b200_last_error()

    # as they are, the calls are taken: each refusal below is of its one change
    for call, arg in ((lib.b200_kv_append, ap), (lib.b200_kv_attend, at), (lib.b200_kv_evict, ev)):
        assert call(eng.h, ctypes.byref(cache.c), ctypes.byref(arg)) == 0
    assert lib.b200_sample(eng.h, ctypes.byref(sm)) == 0
    eng.sync()
    kvs = [dict(kv_dtype=3), dict(kv_dtype=-1), dict(kv_batch=0), dict(kv_n_pages=0), dict(kv_page_size=0),
           dict(kv_head_dim=60), dict(kv_head_dim=0), dict(kv_head_dim=264), dict(kv_n_head_kv=0), dict(kv_table_cols=0),
           dict(kv_table_cols=1 << 20), dict(kv_table_stride=1), dict(kv_k=0), dict(kv_v=0), dict(kv_table=0),
           dict(kv_lengths=0), dict(kv_k=cache.c.k + 8), dict(kv_row_stride=65), dict(kv_page_stride=-64)]
    for call, arg in ((lib.b200_kv_append, ap), (lib.b200_kv_attend, at), (lib.b200_kv_evict, ev)):
        for change in kvs:
            refused(call, cache.c, arg, **change)
        assert call(eng.h, None, ctypes.byref(arg)) == -22
        assert call(eng.h, ctypes.byref(cache.c), None) == -22
        assert call(None, ctypes.byref(cache.c), ctypes.byref(arg)) == -22
    for change in (dict(dtype=2), dict(n_tokens=-1), dict(n_tokens=3), dict(k_new=0), dict(v_new=new.data_ptr() + 4),
                   dict(token_stride=129), dict(head_stride=-64), dict(positions=pos.data_ptr(), aux_stride=3),
                   dict(seen=seen.data_ptr() + 2)):
        refused(lib.b200_kv_append, cache.c, ap, **change)
    for change in (dict(dtype=2), dict(n_head=3), dict(n_head=0), dict(q=0), dict(out=0), dict(q=q.data_ptr() + 2),
                   dict(scale=float("nan")), dict(scale=float("inf")), dict(q_head_stride=-1),
                   dict(weights=aux.data_ptr()),
                   dict(weights_out=aux.data_ptr(), aux_stride=1), dict(workspace=0), dict(workspace_bytes=3),
                   dict(workspace=ws.data_ptr() + 8),
                   dict(weights_out=aux.data_ptr(), aux_stride=cache.capacity,
                        workspace_bytes=lib.b200_kv_attend_workspace(ctypes.byref(cache.c), 4, 0)),
                   dict(n_head=2 * 257), dict(kv_dtype=2), dict(kv_dtype=0, dtype=1)):
        refused(lib.b200_kv_attend, cache.c, at, **change)
    for change in (dict(weights=0), dict(weights_out=0), dict(positions=0), dict(positions_out=0), dict(seen=0),
                   dict(budget=0), dict(recent=-1), dict(sinks=-1), dict(recent=8), dict(aux_stride=2),
                   dict(weights=aux.data_ptr() + 1)):
        refused(lib.b200_kv_evict, cache.c, ev, **change)
    for change in (dict(logits=0), dict(u=0), dict(token=0), dict(dtype=7), dict(batch=0), dict(n_vocab=0),
                   dict(n_vocab=(1 << 22) + 1), dict(row_stride=255), dict(logits=q.data_ptr() + 1),
                   dict(top_k=seen.data_ptr() + 3)):
        refused(lib.b200_sample, None, sm, **change)
    assert lib.b200_sample(None, ctypes.byref(sm)) == -22 and lib.b200_sample(eng.h, None) == -22
    # the Python layer's own checks
    f16 = torch.float16
    with pytest.raises(ValueError):
        pkg.PagedKV(cache.k, cache.v.float(), cache.table, cache.lengths)
    with pytest.raises(ValueError):
        pkg.PagedKV(cache.k.cpu(), cache.v.cpu(), cache.table, cache.lengths)
    with pytest.raises(ValueError):
        pkg.PagedKV(cache.k, cache.v, cache.table.long(), cache.lengths)
    with pytest.raises(ValueError):
        pkg.PagedKV(cache.k, cache.v, cache.table, cache.lengths[:1])
    with pytest.raises(ValueError):
        pkg.PagedKV(cache.k.transpose(2, 3), cache.v.transpose(2, 3), cache.table, cache.lengths)
    with pytest.raises(ValueError):
        eng.kv_attend(cache, q, q.to(f16))
    with pytest.raises(ValueError):
        eng.kv_attend(cache, q[:1], q[:1])
    with pytest.raises(ValueError):
        eng.kv_attend(cache, q, torch.empty_like(q), weights_out=aux[:, :, :-1].contiguous())
    with pytest.raises(pkg.B200Error):
        eng.kv_attend(cache, q.bfloat16(), q.bfloat16())
    with pytest.raises(ValueError):
        eng.kv_append(cache, new, new.to(f16))
    with pytest.raises(ValueError):
        eng.kv_append(cache, new, new, positions=pos.float())
    with pytest.raises(ValueError):
        eng.kv_evict(cache, aux, pos.float(), seen, 8)
    with pytest.raises(pkg.B200Error):
        eng.kv_evict(cache, aux, pos, seen, 8, recent=9)
    with pytest.raises(ValueError):
        eng.sample(q[0], lse[0], seen)
    with pytest.raises(ValueError):
        eng.sample(q[:, 0], lse[:, 0].contiguous(), seen.float())
    eng.sync()
