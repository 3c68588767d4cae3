"""examples/serve_chunks.py: what it refuses before any step, without a GPU."""

from __future__ import annotations

import importlib.util
import os
from types import SimpleNamespace

import pytest


@pytest.fixture(scope="module")
def example(pkg):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "serve_chunks.py")
    spec = importlib.util.spec_from_file_location("serve_chunks", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def server(example):
    """A server whose steps must not be reached: they would hand out logits of nothing, without end."""
    import torch
    srv = example.ChunkServer.__new__(example.ChunkServer)
    srv.torch, srv.dev, srv.batch, srv.page, srv.hp = torch, "cpu", 2, 16, dict(n_vocab=8)
    srv.free, srv.table = torch.zeros(40, dtype=torch.int32), torch.zeros(2, 10, dtype=torch.int32)
    srv.eng = SimpleNamespace(sample=lambda *a, **k: None)

    def step(chunks):
        raise AssertionError(f"step({chunks})")

    srv.step = step
    return srv


@pytest.mark.parametrize("prompts,n,chunk", [([[1, 2]], 0, 64), ([[1, 2]], -3, 64), ([[1], []], 4, 64), ([[1, 2]], 4, 0)])
def test_requests_that_never_end_are_refused(example, prompts, n, chunk):
    with pytest.raises(ValueError):
        server(example).serve(prompts, n, chunk=chunk)


def test_no_requests(example):
    srv = server(example)
    srv.step = lambda chunks: None
    assert srv.serve([], 4) == []
