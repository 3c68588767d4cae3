"""The host side of the serving calls (Engine in Python), without a GPU: the C
library is a stand-in that keeps what it was called with."""

from __future__ import annotations

import threading

import pytest


class FakeTensor:
    """What Engine asks of a CUDA tensor."""
    is_cuda = True

    def __init__(self, at, shape, dtype):
        self.at, self.shape, self.dtype = at, tuple(shape), dtype

    def dim(self):
        return len(self.shape)

    def stride(self, i=None):
        st = [1] * len(self.shape)
        for k in reversed(range(len(st) - 1)):
            st[k] = st[k + 1] * self.shape[k + 1]
        return tuple(st) if i is None else st[i]

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return self.at


class FakeLib:
    def __init__(self):
        self.on_call = lambda name, c: None

    def __getattr__(self, name):
        def call(*args):
            self.on_call(name, args[-1]._obj if hasattr(args[-1], "_obj") else None)
            return 0
        return call


@pytest.fixture
def fake(pkg, monkeypatch):
    from llm_kv260_b200 import engine
    lib = FakeLib()
    monkeypatch.setattr(engine, "lib", lambda: lib)
    return lib


def test_a_thread_does_not_overwrite_the_arguments_of_another(pkg, fake):
    """The C call reads its arguments with the interpreter's lock given up: a call of another thread on the same engine
    in the meantime leaves them alone."""
    import torch
    eng = pkg.Engine(0, stream=0)
    seen, inside, done = [], threading.Event(), threading.Event()

    def on_call(name, c):
        if name != "b200_sample":
            return
        if threading.current_thread() is first:
            inside.set()
            done.wait(0.5)                      # the other thread's call, or its wait for this one
        seen.append((c.logits, c.n_vocab, c.batch, c.u, c.token))

    fake.on_call = on_call

    def call(at, batch, vocab):
        eng.sample(FakeTensor(at, (batch, vocab), torch.float32), FakeTensor(at + 1, (batch,), torch.float32),
                   FakeTensor(at + 2, (batch,), torch.int32))

    def second():
        inside.wait(5)
        call(2000, 7, 99)
        done.set()

    first = threading.Thread(target=call, args=(1000, 3, 50))
    other = threading.Thread(target=second)
    first.start(), other.start()
    first.join(10), other.join(10)
    assert sorted(seen) == [(1000, 50, 3, 1001, 1002), (2000, 99, 7, 2001, 2002)]
