"""The host side of the operators that a prompt passes through, without a GPU."""

from __future__ import annotations

import math
from decimal import Decimal, getcontext

import numpy as np
import pytest

TWO64 = 2.0 ** 64


def turns(t):
    """rope_freqs' whole numbers as turns a position."""
    return t.numpy().view(np.uint64).astype(np.float64) / TWO64


@pytest.mark.parametrize("rot,base", [(2, 10000.0), (64, 10000.0), (80, 500000.0), (256, 1.5)])
def test_frequencies(pkg, rot, base):
    """To a part in 2^50 of a turn: the double's own rounding."""
    want = base ** (-2.0 * np.arange(rot // 2) / rot) / (2 * math.pi)
    assert np.abs(turns(pkg.rope_freqs(rot, base)) - want).max() < 2.0 ** -50
    assert np.abs(turns(pkg.rope_freqs(rot, base, scaling="linear", factor=4.0)) - want / 4).max() < 2.0 ** -50
    f = np.linspace(1.0, 8.0, rot // 2).astype(np.float32)
    assert np.abs(turns(pkg.rope_freqs(rot, base, factors=f)) - want / f).max() < 2.0 ** -50


def test_frequencies_for_long_contexts(pkg):
    rot, base = 64, 500000.0
    inv = base ** (-2.0 * np.arange(rot // 2) / rot)
    got = turns(pkg.rope_freqs(rot, base, scaling="bands", factor=8.0, context=8192, low=1.0, high=4.0))
    n = 8192 * inv / (2 * math.pi)
    for i in range(rot // 2):
        keep = min(max((n[i] - 1) / 3, 0), 1)
        assert abs(got[i] - (inv[i] * keep + inv[i] / 8 * (1 - keep)) / (2 * math.pi)) < 2.0 ** -50
    assert (n > 4).any() and (n < 1).any()
    got = turns(pkg.rope_freqs(rot, base, scaling="yarn", factor=16.0, context=4096, low=1.0, high=32.0))

    def index(x):
        return rot * math.log(4096 / (x * 2 * math.pi)) / (2 * math.log(base))

    lo, hi = math.floor(index(32.0)), math.ceil(index(1.0))
    assert 0 < lo < hi < rot // 2
    for i in range(rot // 2):
        slow = min(max((i - lo) / (hi - lo), 0), 1)
        assert abs(got[i] - inv[i] * (1 - slow + slow / 16) / (2 * math.pi)) < 2.0 ** -50


def exact_turns(rot, base, factor=1):
    """Turns a position of each pair, to 45 digits."""
    getcontext().prec = 50
    pi = Decimal("3.14159265358979323846264338327950288419716939937510582097494459")
    return [(Decimal(base).ln() * (-2 * i) / rot).exp() / (2 * pi * Decimal(factor)) for i in range(rot // 2)]


@pytest.mark.parametrize("rot,base,factor", [(64, 10000.0, 1.0), (128, 500000.0, 1.0), (80, 10000.0, 40.0), (256, 1.5, 3.0)])
def test_frequencies_carry_the_farthest_position(pkg, rot, base, factor):
    """Times 2^31 - 1, the last position, to 2^-28 of a turn: a frequency to 2^-59, where a double's 53 bits would not do."""
    got = pkg.rope_freqs(rot, base, scaling=None if factor == 1 else "linear", factor=factor).numpy().view(np.uint64)
    for i, want in enumerate(exact_turns(rot, base, factor)):
        off = (Decimal(int(got[i])) / 2 ** 64 - want % 1) * (2 ** 31 - 1)
        assert abs(off) < Decimal(2) ** -28, (i, float(off))


def test_stretched_frequencies_carry_the_farthest_position(pkg):
    """The same for bands and for the ramp over a pair's index."""
    rot, base, factor, context = 64, 500000.0, 8.0, 8192
    plain = exact_turns(rot, base)
    got = pkg.rope_freqs(rot, base, scaling="bands", factor=factor, context=context, low=1.0, high=4.0).numpy().view(np.uint64)
    for i, f in enumerate(plain):
        keep = min(max((context * f - 1) / 3, Decimal(0)), Decimal(1))
        off = (Decimal(int(got[i])) / 2 ** 64 - f * (keep + (1 - keep) / 8)) * (2 ** 31 - 1)
        assert abs(off) < Decimal(2) ** -28, (i, float(off))
    got = pkg.rope_freqs(rot, base, scaling="yarn", factor=factor, context=context, low=1.0, high=32.0).numpy().view(np.uint64)

    def index(x):
        return rot * math.log(context / (x * 2 * math.pi)) / (2 * math.log(base))

    lo, hi = math.floor(index(32.0)), math.ceil(index(1.0))
    for i, f in enumerate(plain):
        slow = min(max(Decimal(i - lo) / (hi - lo), Decimal(0)), Decimal(1))
        off = (Decimal(int(got[i])) / 2 ** 64 - f * (1 - slow + slow / 8)) * (2 ** 31 - 1)
        assert abs(off) < Decimal(2) ** -28, (i, float(off))


def test_frequencies_refused(pkg):
    for kw in (dict(rot_dim=0), dict(rot_dim=7), dict(rot_dim=258), dict(base=0.0), dict(base=-1.0), dict(base=math.nan),
               dict(scaling="linear", factor=0.0), dict(scaling="bands", factor=2.0), dict(scaling="other"),
               dict(scaling="bands", factor=2.0, context=100.0, low=4.0, high=4.0), dict(factors=[1.0, 0.0] * 16),
               dict(scaling="yarn", factor=2.0, context=100.0, base=1.0), dict(factors=[1.0])):
        with pytest.raises((ValueError, pkg.B200Error)):
            pkg.rope_freqs(**dict(dict(rot_dim=64), **kw))


def test_workspace_of_unusable_sizes(pkg):
    import ctypes
    lib, t = pkg.lib(), pkg.capi.b200_kv_t
    good = dict(k=256, v=256, dtype=1, n_pages=4, page_size=16, n_head_kv=2, head_dim=64, page_stride=2048, head_stride=1024,
                row_stride=64, table=256, table_stride=2, table_cols=2, lengths=256, batch=1)
    for change, dtype, n_head in ((dict(head_dim=60), 1, 4), (dict(batch=0), 1, 4), (dict(k=0), 1, 4), ({}, 2, 4), ({}, 1, 3),
                                  ({}, 1, 1), (dict(dtype=0), 1, 4), (dict(dtype=2), 0, 4), (dict(page_size=0), 1, 4)):
        kv = t(**dict(good, **change))
        assert lib.b200_kv_chunk_workspace(ctypes.byref(kv), dtype, n_head) == 0


def test_workspace_of_too_many_heads(pkg):
    """0 where the call refuses: more than 4096 query heads to a cache head, none, fewer than none."""
    import ctypes
    kv = pkg.capi.b200_kv_t(k=256, v=256, dtype=1, n_pages=4, page_size=16, n_head_kv=2, head_dim=64, page_stride=2048,
                            head_stride=1024, row_stride=64, table=256, table_stride=2, table_cols=2, lengths=256, batch=1)
    lib = pkg.lib()
    for dtype in (0, 1):
        assert lib.b200_kv_chunk_workspace(ctypes.byref(kv), dtype, 2 * 4096) > 0
        for n_head in (2 * 4097, 1 << 30, 0, -2):
            assert lib.b200_kv_chunk_workspace(ctypes.byref(kv), dtype, n_head) == 0


def test_arguments_refused_before_any_call(pkg, monkeypatch):
    """Python's own checks, with a stand-in for the library that must not be reached."""
    import torch
    from llm_kv260_b200 import engine

    from test_serving_host import FakeLib, FakeTensor

    calls = []
    lib = FakeLib()
    lib.on_call = lambda name, c: calls.append(name)
    monkeypatch.setattr(engine, "lib", lambda: lib)
    eng = pkg.Engine(0, stream=0)

    def t(*shape, dt=torch.float16, at=4096):
        return FakeTensor(at, shape, dt)

    class Cache:
        batch, n_head_kv, head_dim, n_pages, page_size, capacity = 3, 2, 64, 4, 16, 32
        lengths, ref, workspace = t(3, dt=torch.int32), None, {}

    kv, i32 = Cache(), torch.int32
    del calls[:]
    q, off, pos, slots = t(5, 4, 64), t(4, dt=i32), t(5, dt=i32), t(5, dt=torch.int64)
    freqs, new, free = t(32, dt=torch.int64), t(3, dt=i32), t(9, dt=i32)
    x, w = t(3, 64, dt=torch.float32), t(64, dt=torch.float32)
    for f in (lambda: eng.kv_attend_chunk(kv, t(5, 4), q, off), lambda: eng.kv_attend_chunk(kv, q, t(5, 4, 64, dt=torch.float32), off),
              lambda: eng.kv_attend_chunk(kv, t(5, 4, 32), t(5, 4, 32), off), lambda: eng.kv_attend_chunk(kv, q, q, t(3, dt=i32)),
              lambda: eng.kv_attend_chunk(kv, q, q, t(4, dt=torch.int64)), lambda: eng.kv_attend_chunk(kv, q, q, off, lse=t(5, 4)),
              lambda: eng.rope(pos, freqs), lambda: eng.rope(t(4, dt=i32), freqs, q=q), lambda: eng.rope(pos, t(32, dt=i32), q=q),
              lambda: eng.rope(pos, freqs, q=q, k=t(4, 2, 64)), lambda: eng.rope(pos, freqs, q=q, v=q),
              lambda: eng.rope(pos, freqs, q=q, slots=slots), lambda: eng.rope(pos, freqs, q=q, q_out=t(5, 3, 64)),
              lambda: eng.rope(pos, freqs, k=t(5, 2, 64), kv=kv, v=t(5, 2, 64, dt=torch.float32), slots=slots),
              lambda: eng.rope(pos, t(4, 8, dt=torch.int64), q=q), lambda: eng.rms_norm(t(64), w, out=x),
              lambda: eng.rms_norm(x, t(32, dt=torch.float32), out=x), lambda: eng.rms_norm(x, w, out=t(2, 64, dt=torch.float32)),
              lambda: eng.rms_norm(x, w, residual_out=x), lambda: eng.rms_norm(x, w, residual=t(3, 64), residual_out=x),
              lambda: eng.kv_plan(kv, t(2, dt=i32), new, free, t(1, dt=i32), off), lambda: eng.kv_plan(kv, new, new, t(3, 3, dt=i32), t(1, dt=i32), off),
              lambda: eng.kv_plan(kv, new, new, free, t(2, dt=i32), off), lambda: eng.kv_plan(kv, new, new, free, t(1, dt=i32), off, slots=pos),
              lambda: eng.kv_plan(kv, new, new, free, t(1, dt=i32), off, slots=slots, positions=t(4, dt=i32)),
              lambda: eng.kv_plan(kv, new, new, free, t(1, dt=i32), off, sequences=t(5, 1, dt=i32))):
        with pytest.raises(ValueError):
            f()
    assert not [c for c in calls if c != "b200_kv_chunk_workspace"]
    eng.kv_plan(kv, new, new, free, t(1, dt=i32), off, slots=slots, positions=pos)
    assert calls[-1] == "b200_kv_plan"
