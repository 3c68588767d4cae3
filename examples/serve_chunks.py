"""A server that takes prompts in chunks beside single tokens of other sequences, from one Q4_0 Llama-shaped model, with
key-value caches whose pages come from one pool.

    python examples/serve_chunks.py --batch 4 --requests 12 --chunk 64 --pages 40 --temperature 0.8

Every step hands pages out for all new tokens (kv_plan), and takes them through the layers together: norms with Q8_0
rows (rms_norm) in front of the Q4_0 matrices, rotary positions with the store into the cache (rope), attention of each
sequence's new tokens (kv_attend_chunk). The matrices run through the engine's GEMV, a token after another. The model is
the seeded random one of llm-kv260_b200/model.py, so the tokens mean nothing; at temperature 0 they are the one-sequence
Decoder's.
"""

from __future__ import annotations

import argparse
import os
import sys

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)
from __graft_entry__ import load_package  # noqa: E402

load_package()
import llm_kv260_b200 as k26  # noqa: E402


def dequantize(rows: np.ndarray) -> np.ndarray:
    """Q4_0 rows (18-byte blocks: float16 scale, 16 nibble bytes) as float32."""
    blocks = rows.reshape(rows.shape[0], -1, 18)
    d = blocks[:, :, :2].copy().view(np.float16).astype(np.float32)
    n = blocks[:, :, 2:]
    q = np.concatenate([n & 15, n >> 4], axis=2).astype(np.float32) - 8.0
    return (q * d).reshape(rows.shape[0], -1)


class ChunkServer:
    """A model, and caches of up to `batch` sequences at once out of a pool of `pages` pages a layer. A sequence is a row of
    the table with `columns` pages at most."""

    def __init__(self, model: dict, batch: int, pages: int, page: int = 16, columns: int = 64, device: int = 0):
        import torch
        self.torch, self.hp, self.batch, self.page = torch, model, batch, page
        self.dev = f"cuda:{device}"
        self.eng = k26.Engine(device)

        def mat(*parts):
            rows = np.concatenate([np.ascontiguousarray(p) for p in parts])
            return self.eng.repack(k26.QMat.from_numpy(rows, device))

        def vec(a):
            return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).to(self.dev)

        self.layers = [dict(qkv=mat(L["attn_q"], L["attn_k"], L["attn_v"]), o=mat(L["attn_output"]),
                            gate_up=mat(L["ffn_gate"], L["ffn_up"]), down=mat(L["ffn_down"]),
                            attn_norm=vec(L["attn_norm"]), ffn_norm=vec(L["ffn_norm"])) for L in model["layers"]]
        self.embd = vec(dequantize(model["token_embd"]))
        self.head, self.out_norm = mat(model["token_embd"]), vec(model["output_norm"])
        hkv, d = model["n_head_kv"], model["head_dim"]
        self.table = torch.full((batch, columns), -1, dtype=torch.int32, device=self.dev)
        self.lengths, self.held = self._ints(batch), self._ints(batch)
        # the layers' pools differ, but not who owns which page of them
        self.caches = []
        for _ in model["layers"]:
            k = torch.zeros(pages, hkv, page, d, dtype=torch.float16, device=self.dev)
            self.caches.append(k26.PagedKV(k, torch.zeros_like(k), self.table, self.lengths))
        self.free = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=self.dev)
        self.free_count = torch.full((1,), pages, dtype=torch.int32, device=self.dev)
        self.offsets, self.granted = self._ints(batch + 1), self._ints(batch)
        self.freqs = k26.rope_freqs(d, model["rope_base"], factors=model.get("rope_freqs")).to(self.dev)

    def _ints(self, n: int):
        return self.torch.zeros(n, dtype=self.torch.int32, device=self.dev)

    def _gemv(self, mat, q8):
        """y[t] = W x[t] for packed rows, a call per token."""
        y = self.torch.empty(q8.shape[0], mat.rows, device=self.dev)
        for t in range(q8.shape[0]):
            self.eng.gemv_q8(mat, q8[t], y[t])
        return y

    def _pack(self, x):
        """Q8_0 rows of x as it is."""
        q8 = self.torch.empty(x.shape[0], x.shape[1] * 9 // 8, dtype=self.torch.uint8, device=self.dev)
        for t in range(x.shape[0]):
            self.eng.quantize(x[t], q8[t], x.shape[1])
        return q8

    def step(self, chunks):
        """chunks: for each sequence the tokens it gets (none: it waits), or None: it is done and its pages are free.
        Returns the logits behind the last token of each sequence that got tokens, float32 [batch, n_vocab], and
        how many of its tokens each got pages for, int32 [batch] (all of them or none)."""
        torch, hp, eng = self.torch, self.hp, self.eng
        eng.set_stream(torch.cuda.current_stream().cuda_stream)
        new = torch.tensor([-1 if c is None else len(c) for c in chunks], dtype=torch.int32, device=self.dev)
        tokens = torch.tensor([t for c in chunks for t in (c if c is not None else ())], device=self.dev)
        n, h, hkv, d = tokens.numel(), hp["n_head"], hp["n_head_kv"], hp["head_dim"]
        slots, positions = torch.empty(n, dtype=torch.int64, device=self.dev), self._ints(n)
        eng.kv_plan(self.caches[0], new, self.held, self.free, self.free_count, self.offsets, slots=slots,
                    positions=positions, granted=self.granted)
        logits = torch.zeros(self.batch, hp["n_vocab"], device=self.dev)
        if n == 0:
            return logits, self.granted
        x = self.embd[tokens.long()]
        q8 = torch.empty(n, hp["n_embd"] * 9 // 8, dtype=torch.uint8, device=self.dev)
        add = None                                 # what the last matrix adds to the residual stream x
        q = torch.empty(n, h, d, dtype=torch.float16, device=self.dev)
        out = torch.empty_like(q)

        def norm(w):
            if add is None:
                eng.rms_norm(x, w, eps=hp["rms_eps"], q8=q8)
            else:
                eng.rms_norm(add, w, eps=hp["rms_eps"], residual=x, q8=q8)

        for L, kv in zip(self.layers, self.caches):
            norm(L["attn_norm"])
            qkv = self._gemv(L["qkv"], q8).view(n, h + 2 * hkv, d)
            eng.rope(positions, self.freqs, q=qkv[:, :h], q_out=q, k=qkv[:, h:h + hkv], kv=kv, v=qkv[:, h + hkv:],
                     slots=slots, interleaved=True)
            eng.kv_attend_chunk(kv, q, out, self.offsets)
            add = self._gemv(L["o"], self._pack(out.view(n, h * d).float()))
            norm(L["ffn_norm"])
            gu = self._gemv(L["gate_up"], q8)
            g, u = gu[:, :hp["n_ff"]], gu[:, hp["n_ff"]:]
            add = self._gemv(L["down"], self._pack((g * torch.sigmoid(g) * u).contiguous()))
        norm(self.out_norm)
        last = 0
        for b, c in enumerate(chunks):
            if c is not None and len(c):
                last += len(c)
                eng.gemv_q8(self.head, q8[last - 1], logits[b])
        return logits, self.granted

    def serve(self, prompts, n: int, chunk: int = 64, temperature: float = 0.0, top_p: float = 1.0, seed: int = 0):
        """n tokens (a list) behind each of any number of prompts: as many at a time as there are rows, prompts `chunk`
        tokens a step beside the others' single tokens. A request begins when the pool can hold all of it beside those
        that run."""
        torch = self.torch
        if n < 1 or chunk < 1 or any(len(p) == 0 for p in prompts):
            raise ValueError("every request needs a prompt and at least one token behind it, every step a token of its prompt")
        gen = torch.Generator(device=self.dev).manual_seed(seed)
        out, waiting, rows = [[] for _ in prompts], list(range(len(prompts))), [None] * self.batch
        pages = [-(-(len(p) + n - 1) // self.page) for p in prompts]
        pool = self.free.numel()
        if max(pages, default=0) > min(pool, self.table.shape[1]):
            raise RuntimeError("a request needs more pages than there are")
        pick, lp = self._ints(self.batch), torch.empty(self.batch, device=self.dev)
        kw = dict(temperature=torch.full((self.batch,), temperature, device=self.dev),
                  top_p=torch.full((self.batch,), top_p, device=self.dev))
        ended = [False] * self.batch               # the row's pages come back with this step
        while waiting or any(r is not None for r in rows):
            for b in range(self.batch):
                if rows[b] is None and not ended[b] and waiting:
                    if sum(pages[r["i"]] for r in rows if r is not None) + pages[waiting[0]] > pool:
                        break
                    i = waiting.pop(0)
                    rows[b] = dict(i=i, left=[int(t) for t in prompts[i]])
            logits, granted = self.step([None if r is None else r["left"][:chunk] for r in rows])
            u = torch.rand(self.batch, generator=gen, device=self.dev)
            self.eng.sample(logits, u, pick, lp, **kw)
            got, picks = granted.tolist(), pick.tolist()
            ended = [False] * self.batch
            for b, r in enumerate(rows):
                if r is None:
                    continue
                r["left"] = r["left"][got[b]:]
                if not r["left"]:                  # the prompt's end, or a token that was drawn before
                    out[r["i"]].append(picks[b])
                    r["left"] = [picks[b]]
                    if len(out[r["i"]]) == n:
                        rows[b], ended[b] = None, True
        self.step([None] * self.batch)
        return out


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--batch", type=int, default=4, help="sequences at a time")
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=100, help="tokens of the longest (random) prompt")
    ap.add_argument("--tokens", type=int, default=16, help="tokens to generate per request")
    ap.add_argument("--chunk", type=int, default=64, help="tokens of a prompt a step")
    ap.add_argument("--page", type=int, default=16)
    ap.add_argument("--pages", type=int, default=40)
    ap.add_argument("--temperature", type=float, default=0.8)
    ap.add_argument("--top-p", type=float, default=0.95)
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args()
    from llm_kv260_b200 import model
    hp = dict(n_layer=4, n_embd=1024, n_ff=2048, n_head=16, n_head_kv=4, head_dim=64, n_vocab=32000,
              rope_base=500000.0, rms_eps=1e-5)
    m = model.synth_model(hp, seed=a.seed)
    srv = ChunkServer(m, a.batch, a.pages, a.page)
    rng = np.random.default_rng(a.seed)
    prompts = [model.random_prompt(int(rng.integers(1, a.prompt + 1)), hp["n_vocab"], seed=a.seed + 1 + i)
               for i in range(a.requests)]
    out = srv.serve(prompts, a.tokens, a.chunk, a.temperature, a.top_p, a.seed)
    for i, row in enumerate(out):
        print(f"request {i} ({len(prompts[i])} tokens): {' '.join(map(str, row))}")
    print(f"free pages: {int(srv.free_count)} of {a.pages}")


if __name__ == "__main__":
    main()
