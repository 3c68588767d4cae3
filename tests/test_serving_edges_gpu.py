"""The serving operators where neighbouring work, unusual numbers or unusual
settings could change what they answer: other kernels beside a call, streams
that change, outliers, NaN and infinities, long heads, rows of equal logits."""

from __future__ import annotations

import numpy as np
import pytest

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
