"""Several sequences at once from one Q4_0 Llama-shaped model: paged key-value
caches cut to a budget by accumulated attention weight, and a sampler.

    python examples/serve_paged.py --batch 4 --tokens 32 --budget 48 --temperature 0.8 --top-p 0.9

The matrices run through the engine's Q4_0 GEMV, one sequence after another;
kv_append, kv_attend, kv_evict and sample take all sequences in a call. The
model is the seeded random one of llm-kv260_b200/model.py, so the tokens mean
nothing; with the budget off and temperature 0 they are the one-sequence
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


class PagedServer:
    """A model and the caches of `batch` sequences. `step` takes every
    sequence's next token and gives the logits of the one after it."""

    def __init__(self, model: dict, batch: int, slots: int, page: int = 16, budget: int = 0, recent: int = 0,
                 sinks: int = 0, device: int = 0):
        import torch
        self.torch, self.hp, self.batch = torch, model, batch
        self.budget, self.recent, self.sinks, self.page = budget, recent, sinks, page
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
        # every sequence owns pages for `slots` slots; a server would hand them out from one pool as they are needed
        cols = -(-slots // page)
        hkv, d = model["n_head_kv"], model["head_dim"]
        table = torch.randperm(batch * cols, device=self.dev).to(torch.int32).view(batch, cols).contiguous()
        self.caches, self.used = [], 0
        for _ in model["layers"]:
            k = torch.empty(batch * cols, hkv, page, d, dtype=torch.float16, device=self.dev)
            c = dict(kv=k26.PagedKV(k, torch.empty_like(k), table, torch.zeros(batch, dtype=torch.int32, device=self.dev)),
                     seen=torch.zeros(batch, dtype=torch.int32, device=self.dev))
            if budget:
                c["weights"] = torch.zeros(batch, hkv, cols * page, device=self.dev)
                c["positions"] = torch.zeros(batch, hkv, cols * page, dtype=torch.int32, device=self.dev)
            self.caches.append(c)
        self.slots, self.pos = cols * page, 0
        self.logits = torch.empty(batch, model["n_vocab"], device=self.dev)
        self.picks = torch.empty(batch, dtype=torch.int32, device=self.dev)
        self.logprob = torch.empty(batch, device=self.dev)
        half = np.arange(0, d, 2, dtype=np.float32)
        inv = np.float32(model["rope_base"]) ** (-half / np.float32(d))
        if model.get("rope_freqs") is not None:
            inv = inv / np.asarray(model["rope_freqs"], np.float32)
        self.inv = vec(inv)

    def _gemv(self, mat, x):
        """y[b] = W x[b], a call per sequence."""
        y = self.torch.empty(x.shape[0], mat.rows, device=self.dev)
        for b in range(x.shape[0]):
            self.eng.gemv_f32(mat, x[b], y[b])
        return y

    def _norm(self, x, w):
        s = x.double().square().mean(1, keepdim=True).float()
        return (x / (s + self.hp["rms_eps"]).sqrt() * w).contiguous()

    def _rope(self, x):
        theta = self.pos * self.inv
        c, s = theta.cos(), theta.sin()
        a, b = x[..., 0::2], x[..., 1::2]
        return self.torch.stack([a * c - b * s, a * s + b * c], dim=-1).flatten(-2)

    def step(self, tokens):
        """tokens: int tensor [batch]. Returns the logits, float32 [batch, n_vocab]."""
        torch, hp = self.torch, self.hp
        self.eng.set_stream(torch.cuda.current_stream().cuda_stream)
        if self.used == self.slots:
            raise RuntimeError("the caches are full")
        h, hkv, d = hp["n_head"], hp["n_head_kv"], hp["head_dim"]
        x = self.embd[tokens.long()]
        self.used += 1
        cut = self.budget and self.used > self.budget
        for L, c in zip(self.layers, self.caches):
            qkv = self._gemv(L["qkv"], self._norm(x, L["attn_norm"])).view(self.batch, h + 2 * hkv, d)
            q, k = self._rope(qkv[:, :h]), self._rope(qkv[:, h:h + hkv])
            self.eng.kv_append(c["kv"], k, qkv[:, h + hkv:].contiguous(), seen=c["seen"], positions=c.get("positions"),
                               weights=c.get("weights"))
            out = torch.empty_like(q)
            self.eng.kv_attend(c["kv"], q, out, weights=c.get("weights"), weights_out=c.get("weights"))
            if cut:
                self.eng.kv_evict(c["kv"], c["weights"], c["positions"], c["seen"], self.budget, recent=self.recent,
                                  sinks=self.sinks)
            x = x + self._gemv(L["o"], out.view(self.batch, h * d))
            gu = self._gemv(L["gate_up"], self._norm(x, L["ffn_norm"]))
            g, u = gu[:, :hp["n_ff"]], gu[:, hp["n_ff"]:]
            x = x + self._gemv(L["down"], (g * torch.sigmoid(g) * u).contiguous())
        if cut:
            self.used = self.budget
        self.pos += 1
        x = self._norm(x, self.out_norm)
        for b in range(self.batch):
            self.eng.gemv_f32(self.head, x[b], self.logits[b])
        return self.logits

    def generate(self, prompts, n: int, temperature=None, top_k=None, top_p=None, min_p=None, seed: int = 0):
        """n tokens per sequence (int32 [batch, n], on the host) behind prompts of one length, [batch, length]."""
        torch = self.torch
        gen = torch.Generator(device=self.dev).manual_seed(seed)
        prompts = torch.as_tensor(np.asarray(prompts), device=self.dev)
        for i in range(prompts.shape[1]):
            self.step(prompts[:, i])

        def per_row(v, dtype):
            return None if v is None else torch.full((self.batch,), v, dtype=dtype, device=self.dev)

        kw = dict(temperature=per_row(temperature, torch.float32), top_k=per_row(top_k, torch.int32),
                  top_p=per_row(top_p, torch.float32), min_p=per_row(min_p, torch.float32))
        out = torch.empty(self.batch, n, dtype=torch.int32, device=self.dev)
        for i in range(n):
            u = torch.rand(self.batch, generator=gen, device=self.dev)
            self.eng.sample(self.logits, u, self.picks, self.logprob, **kw)
            out[:, i] = self.picks
            if i + 1 < n:
                self.step(self.picks)
        return out.cpu().numpy()


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=24, help="tokens of each (random) prompt")
    ap.add_argument("--tokens", type=int, default=32, help="tokens to generate per sequence")
    ap.add_argument("--budget", type=int, default=0, help="slots each head keeps (0: all)")
    ap.add_argument("--recent", type=int, default=16)
    ap.add_argument("--sinks", type=int, default=4)
    ap.add_argument("--page", type=int, default=16)
    ap.add_argument("--temperature", type=float, default=0.8)
    ap.add_argument("--top-k", type=int, default=0)
    ap.add_argument("--top-p", type=float, default=0.95)
    ap.add_argument("--min-p", type=float, default=0.0)
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args()
    from llm_kv260_b200 import model
    hp = dict(n_layer=4, n_embd=1024, n_ff=2048, n_head=16, n_head_kv=4, head_dim=64, n_vocab=32000,
              rope_base=500000.0, rms_eps=1e-5)
    m = model.synth_model(hp, seed=a.seed)
    slots = (a.budget + 1) if a.budget else a.prompt + a.tokens
    srv = PagedServer(m, a.batch, slots, a.page, a.budget, a.recent, a.sinks)
    prompts = np.stack([model.random_prompt(a.prompt, hp["n_vocab"], seed=a.seed + 1 + b) for b in range(a.batch)])
    out = srv.generate(prompts, a.tokens, a.temperature, a.top_k, a.top_p, a.min_p, a.seed)
    for b, row in enumerate(out):
        print(f"sequence {b}: {' '.join(map(str, row))}")
    print(f"slots in use: {srv.caches[0]['kv'].lengths.tolist()} of {srv.slots}")


if __name__ == "__main__":
    main()
