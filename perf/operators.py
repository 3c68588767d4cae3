"""What is timed of the serving operators: a paged key-value cache (append,
single-token attention, eviction by accumulated attention weight) and the
sampler that turns logits into the next token.

A case is a dict of plain values. `prepare` makes what a serving program holds
before the call, `run` makes one call -- in plain torch operations where `own`
is false, through the library's Engine where it is true -- and `exact` gives
the same outputs from the definitions in 64 bits. Nothing a call reads is
changed by it, so that it can be repeated: the accumulated weights, positions
and lengths go to buffers of their own, and eviction moves rows only out of
slots at or past the budget into slots below it.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
ESIZE = {"f16": 2, "bf16": 2, "f32": 4}
LOG2E = 1.4426950408889634
ONE = 1 << 40                      # the sampler's weight of the largest logit


# ---------------------------------------------------------------- the cases

def listed() -> list[dict]:
    return [
        # One user of the 1B model early in an answer: the latency of a call.
        dict(name="attend_one_short", op="attend", batch=1, n_head=32, n_head_kv=8, head_dim=64, page=16,
             min_len=200, max_len=200, q="f32", kv="f16", weights=False, lens=1),
        # One user with a very long document in the 3B model's cache.
        dict(name="attend_one_long", op="attend", batch=1, n_head=24, n_head_kv=8, head_dim=128, page=64,
             min_len=131071, max_len=131071, q="f32", kv="f16", weights=False, lens=2),
        # A full server: users anywhere between their first token and a long context, bfloat16 throughout.
        dict(name="attend_batch", op="attend", batch=32, n_head=32, n_head_kv=8, head_dim=128, page=64,
             min_len=1, max_len=16384, q="bf16", kv="bf16", weights=False, lens=3),
        # The 3B model's 4096-token context with the weights kept for eviction.
        dict(name="attend_weights", op="attend", batch=8, n_head=24, n_head_kv=8, head_dim=128, page=32,
             min_len=4096, max_len=4352, q="f32", kv="f16", weights=True, lens=4),
        # The cache in float32, pages of an odd size, a head size that is no power of two.
        dict(name="attend_f32_odd", op="attend", batch=5, n_head=20, n_head_kv=4, head_dim=96, page=41,
             min_len=0, max_len=6000, q="f32", kv="f32", weights=False, lens=5),
        # One new token of each user of a full server goes into the cache.
        dict(name="append_step", op="append", batch=64, n_head_kv=8, head_dim=64, page=16, new_min=1, new_max=1,
             max_len=4096, src="f32", kv="f16", lens=6),
        # Prompts of different lengths go into the cache at once.
        dict(name="append_prompts", op="append", batch=12, n_head_kv=8, head_dim=128, page=64, new_min=1,
             new_max=4096, max_len=2048, src="bf16", kv="bf16", lens=7),
        # Every user's cache is one token over its budget: the step of a running server.
        dict(name="evict_step", op="evict", batch=16, n_head_kv=8, head_dim=64, page=16, min_len=1025, max_len=1025,
             budget=1024, recent=128, sinks=4, kv="f16", lens=8),
        # Prompts cut down to the budget after they were read.
        dict(name="evict_prompts", op="evict", batch=8, n_head_kv=8, head_dim=128, page=64, min_len=900,
             max_len=16000, budget=1000, recent=256, sinks=4, kv="bf16", lens=9),
        # One user's next token, with the filters that chat programs set.
        dict(name="sample_one", op="sample", batch=1, n_vocab=128256, dtype="f32", spread=2.5, top_k=40, top_p=0.95,
             min_p=0.05, temperature=0.8, mixed=False),
        # A small server without filters, a vocabulary of odd size, logits of 16 bits with their ties.
        dict(name="sample_plain_odd", op="sample", batch=24, n_vocab=50257, dtype="bf16", spread=3.0, top_k=0,
             top_p=1.0, min_p=0.0, temperature=1.0, mixed=False),
        # A full server whose users each set filters of their own, some none, some greedy.
        dict(name="sample_batch", op="sample", batch=256, n_vocab=128256, dtype="f32", spread=2.5, top_k=100,
             top_p=0.9, min_p=0.02, temperature=0.9, mixed=True),
    ]


def _log(rng: random.Random, lo: float, hi: float) -> int:
    return max(int(lo), min(int(hi), int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random) -> dict:
    op = rng.choice(["attend", "attend", "attend", "append", "evict", "sample", "sample"])
    lens = rng.randrange(1 << 30)
    if op == "sample":
        n_vocab = _log(rng, 1000, 200000)
        batch = _log(rng, 1, max(1, min(256, 256 * 128256 // n_vocab)))
        return dict(op=op, batch=batch, n_vocab=n_vocab, dtype=rng.choice(["f32", "f32", "bf16", "f16"]),
                    spread=round(rng.uniform(1.5, 3.5), 3), top_k=rng.choice([0, 0, _log(rng, 1, 2000)]),
                    top_p=rng.choice([1.0, round(rng.uniform(0.3, 0.999), 4)]),
                    min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.2), 4)]),
                    temperature=round(rng.uniform(0.4, 1.3), 3), mixed=rng.random() < 0.5)
    head_dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256])
    n_head_kv = rng.choice([1, 2, 4, 8, 8, 8, 16])
    page = rng.choice([16, 32, 64, 128, rng.randrange(1, 200)])
    kv = rng.choice(["f16", "bf16", "bf16", "f32"])
    row = 2 * n_head_kv * head_dim * ESIZE[kv]            # bytes of one token in the cache
    if op == "attend":
        max_len = _log(rng, 1, 131072)
        most = max(1, int((512 << 20) // (row * max_len)))
        max_len = min(max_len, (512 << 20) // row)
        batch = _log(rng, 1, min(64, most))
        q = {"f16": rng.choice(["f16", "f32"]), "bf16": "bf16", "f32": "f32"}[kv]
        return dict(op=op, batch=batch, n_head=n_head_kv * rng.choice([1, 2, 3, 4, 4, 5, 7, 8]), n_head_kv=n_head_kv,
                    head_dim=head_dim, page=page, min_len=rng.choice([0, 1, max_len]), max_len=max_len, q=q, kv=kv,
                    weights=rng.random() < 0.3, lens=lens)
    if op == "append":
        new_max = rng.choice([1, _log(rng, 1, 4096)])
        max_len = _log(rng, 1, 4096)
        batch = _log(rng, 1, max(1, min(128, (384 << 20) // (row * (new_max + max_len)))))
        return dict(op=op, batch=batch, n_head_kv=n_head_kv, head_dim=head_dim, page=page,
                    new_min=rng.choice([0, 1, new_max]), new_max=new_max, max_len=max_len,
                    src=rng.choice([kv, "f32"]), kv=kv, lens=lens)
    max_len = _log(rng, 64, 32768)
    max_len = min(max_len, (384 << 20) // row)
    batch = _log(rng, 1, max(1, min(64, (384 << 20) // (row * max_len))))
    budget = rng.choice([max_len - 1, _log(rng, max_len / 16, max_len - 1)])
    recent = rng.randrange(0, budget // 2 + 1)
    return dict(op=op, batch=batch, n_head_kv=n_head_kv, head_dim=head_dim, page=page,
                min_len=rng.choice([0, max_len // 2, max_len]), max_len=max_len, budget=budget, recent=recent,
                sinks=rng.choice([0, min(4, budget - recent)]), kv=kv, lens=lens)


def _lengths(case: dict) -> list[int]:
    """The slots in use per sequence: part of the case, so that its work is known."""
    rng = random.Random(case["lens"])
    lo = case.get("min_len", 0)
    lens = [rng.randint(lo, case["max_len"]) for _ in range(case["batch"])]
    if case["op"] != "append":
        lens[rng.randrange(len(lens))] = case["max_len"]
    return lens


def _news(case: dict) -> list[int]:
    rng = random.Random(case["lens"] + 1)
    news = [rng.randint(case["new_min"], case["new_max"]) for _ in range(case["batch"])]
    news[rng.randrange(len(news))] = case["new_max"]
    return news


def work(case: dict) -> dict:
    if case["op"] == "sample":
        n = case["batch"] * case["n_vocab"]
        return {"bytes": n * ESIZE[case["dtype"]] + 28 * case["batch"], "flops": 4 * n}
    hkv, d, b, lens = case["n_head_kv"], case["head_dim"], case["batch"], _lengths(case)
    es = ESIZE[case["kv"]]
    if case["op"] == "attend":
        n = sum(lens)
        by = n * hkv * d * 2 * es + 2 * b * case["n_head"] * d * ESIZE[case["q"]] + 4 * b * case["n_head"]
        by += 4 * sum(-(-x // case["page"]) for x in lens) + 4 * b
        if case["weights"]:
            by += 8 * n * hkv
        return {"bytes": by, "flops": 4 * n * case["n_head"] * d}
    if case["op"] == "append":
        n = sum(_news(case))
        return {"bytes": n * hkv * d * 2 * (es + ESIZE[case["src"]]) + n * hkv * 8 + 16 * b, "flops": 0}
    # evict: the weights and positions in and out; a row moves when it is kept and lies past the budget
    by, keep = 8 * b, case["recent"] + case["sinks"]
    for x in lens:
        over = x - case["budget"]
        by += hkv * 8 * x + hkv * 8 * min(x, case["budget"])
        if over > 0:
            moved = min(case["recent"], over)
            moved += max(0, over - case["recent"]) * (case["budget"] - keep) / max(1, x - keep)
            by += int(hkv * moved * 2 * 2 * d * es)
    return {"bytes": by, "flops": sum(hkv * x for x in lens)}


# ---------------------------------------------------------------- the inputs

def prepare(case: dict, seed: int) -> dict:
    st = _inputs(case, seed)
    if own:                                    # the handle that a program opens once, and its view of the cache
        from __graft_entry__ import load_package
        pkg = load_package()
        st["eng"] = pkg.Engine(torch.cuda.current_device())
        if "k" in st:
            st["cache"] = pkg.PagedKV(st["k"], st["v"], st["table"], st["lengths"])
    return st


def _inputs(case: dict, seed: int) -> dict:
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device=dev, dtype=dtype)

    st = {"case": case}
    if case["op"] == "sample":
        b, n = case["batch"], case["n_vocab"]
        x = normal(b, n) * case["spread"]
        # the few tokens that a trained model makes likely
        x.scatter_add_(1, torch.randint(n, (b, 8), generator=gen, device=dev), 3 * case["spread"] + 2 * normal(b, 8))
        st["logits"] = x.to(DTYPES[case["dtype"]])
        st["u"] = torch.rand(b, generator=gen, device=dev)
        t = torch.full((b,), case["temperature"], device=dev)
        k = torch.full((b,), case["top_k"], device=dev, dtype=torch.int32)
        p = torch.full((b,), case["top_p"], device=dev)
        m = torch.full((b,), case["min_p"], device=dev)
        if case["mixed"]:
            rows = torch.arange(b, device=dev)
            k[rows % 2 == 1] = 0
            p[rows % 3 == 1] = 1.0
            m[rows % 5 != 0] = 0.0
            t[rows % 16 == 5] = 0.0
        st.update(temperature=t, top_k=k, top_p=p, min_p=m,
                  token=torch.empty(b, dtype=torch.int32, device=dev), logprob=torch.empty(b, device=dev))
        return st

    b, hkv, d, page, lens = case["batch"], case["n_head_kv"], case["head_dim"], case["page"], _lengths(case)
    dt = DTYPES[case["kv"]]
    most = max(lens) if case["op"] != "append" else max(x + n for x, n in zip(lens, _news(case)))
    cols = max(1, -(-most // page))
    held = [-(-x // page) for x in lens]
    if case["op"] == "append":
        held = [-(-(x + n) // page) for x, n in zip(lens, _news(case))]
    n_pages = sum(held) + 1
    # pages in the order in which a running server hands them out: any
    perm = torch.randperm(n_pages, generator=gen, device=dev).to(torch.int32)
    table = torch.zeros(b, cols, dtype=torch.int32, device=dev)
    at = 0
    for i, c in enumerate(held):
        table[i, :c] = perm[at:at + c]
        at += c
    st["k"] = normal(n_pages, hkv, page, d, dtype=dt)
    st["v"] = normal(n_pages, hkv, page, d, dtype=dt)
    st["table"] = table
    st["lengths"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    cap = cols * page
    if case["op"] == "attend":
        h = case["n_head"]
        st["q"] = (1.5 * normal(b, h, d)).to(DTYPES[case["q"]])
        st["out"] = torch.empty_like(st["q"])
        st["lse"] = torch.empty(b, h, device=dev)
        if case["weights"]:
            st["weights"] = torch.exp(normal(b, hkv, cap))
            st["weights_out"] = torch.zeros(b, hkv, cap, device=dev)
    elif case["op"] == "append":
        news = _news(case)
        n = sum(news)
        off = [0]
        for x in news:
            off.append(off[-1] + x)
        st["k_new"] = normal(n, hkv, d).to(DTYPES[case["src"]])
        st["v_new"] = normal(n, hkv, d).to(DTYPES[case["src"]])
        st["offsets"] = torch.tensor(off, dtype=torch.int32, device=dev)
        st["seen"] = st["lengths"] + torch.randint(0, 1000, (b,), generator=gen, device=dev, dtype=torch.int32)
        st["positions"] = torch.zeros(b, hkv, cap, dtype=torch.int32, device=dev)
        st["weights"] = torch.ones(b, hkv, cap, device=dev)
        st["lengths_out"] = torch.empty_like(st["lengths"])
        st["seen_out"] = torch.empty_like(st["seen"])
    else:
        st["weights"] = torch.exp(1.5 * normal(b, hkv, cap))
        # a cache that was cut before holds its positions in any order, the newest last
        pos = torch.rand(b, hkv, cap, generator=gen, device=dev)
        pos = pos.masked_fill_(torch.arange(cap, device=dev) >= (st["lengths"] - 1).view(b, 1, 1), 2.0)
        pos = torch.argsort(torch.argsort(pos, dim=2, stable=True), dim=2, stable=True).to(torch.int32)
        st["positions"] = pos
        st["seen"] = st["lengths"].clone()
        st["weights_out"] = torch.zeros_like(st["weights"])
        st["positions_out"] = torch.zeros_like(pos)
        st["lengths_out"] = torch.empty_like(st["lengths"])
    return st


# ---------------------------------------------------------------- one pass

def run(st: dict):
    case = st["case"]
    if not own:
        return {"sample": _sample, "attend": _attend, "append": _append, "evict": _evict}[case["op"]](st)
    eng = st["eng"]
    eng.set_stream(torch.cuda.current_stream().cuda_stream)
    if case["op"] == "sample":
        eng.sample(st["logits"], st["u"], st["token"], st["logprob"], temperature=st["temperature"],
                   top_k=st["top_k"], top_p=st["top_p"], min_p=st["min_p"])
        return {"token": st["token"], "logprob": st["logprob"]}
    if case["op"] == "attend":
        eng.kv_attend(st["cache"], st["q"], st["out"], st["lse"], weights=st.get("weights"),
                      weights_out=st.get("weights_out"))
        out = {"out": st["out"], "lse": st["lse"]}
        if case["weights"]:
            out["weights"] = st["weights_out"]
        return out
    if case["op"] == "append":
        eng.kv_append(st["cache"], st["k_new"], st["v_new"], offsets=st["offsets"], seen=st["seen"],
                      positions=st["positions"], weights=st["weights"], lengths_out=st["lengths_out"],
                      seen_out=st["seen_out"])
        return {"k": st["k"], "v": st["v"], "positions": st["positions"], "weights": st["weights"],
                "lengths": st["lengths_out"], "seen": st["seen_out"]}
    eng.kv_evict(st["cache"], st["weights"], st["positions"], st["seen"], case["budget"], recent=case["recent"],
                 sinks=case["sinks"], weights_out=st["weights_out"], positions_out=st["positions_out"],
                 lengths_out=st["lengths_out"])
    return {"k": st["k"], "v": st["v"], "weights": st["weights_out"], "positions": st["positions_out"],
            "lengths": st["lengths_out"]}


def _rows(st: dict, n: int):
    """Page and slot within it of every sequence's first n cache slots."""
    slot = torch.arange(n, device=st["table"].device)
    page = st["case"]["page"]
    return st["table"][:, slot // page].long(), (slot % page).expand(st["table"].shape[0], n)


def _attend(st: dict):
    """softmax(q K^T / sqrt(d)) V over each sequence's slots; no slots: zeros and a log-sum of -inf."""
    case = st["case"]
    b, h, hkv, d = case["batch"], case["n_head"], case["n_head_kv"], case["head_dim"]
    n = case["max_len"]
    pg, sl = _rows(st, n)
    k = st["k"][pg, :, sl].float().permute(0, 2, 3, 1)              # b hkv d n
    v = st["v"][pg, :, sl].float().permute(0, 2, 1, 3)              # b hkv n d
    q = st["q"].float().view(b, hkv, h // hkv, d)
    dead = (torch.arange(n, device=q.device) >= st["lengths"].view(b, 1)).view(b, 1, 1, n)
    s = (q @ k * (1.0 / math.sqrt(d))).masked_fill_(dead, -math.inf)
    m = s.amax(3, keepdim=True)
    p = torch.exp(s - m.clamp(min=-3e38))
    z = p.sum(3, keepdim=True)
    p = torch.where(z > 0, p / z, 0.0)
    v = v.masked_fill_(dead.view(b, 1, n, 1), 0.0)
    out = {"out": (p @ v).view(b, h, d).to(st["q"].dtype), "lse": (m + torch.log(z)).view(b, h)}
    if case["weights"]:
        w = st["weights_out"][:, :, :n]
        w.copy_(torch.where(dead.view(b, 1, n), w, st["weights"][:, :, :n] + p.sum(2)))
        out["weights"] = st["weights_out"]
    return out


def _append(st: dict):
    """Row i of a sequence's new rows goes to slot length + i, its position is seen + i, its weight 0."""
    case = st["case"]
    off = st["offsets"].long()
    n = st["k_new"].shape[0]
    row = torch.arange(n, device=off.device)
    b = torch.searchsorted(off, row, right=True) - 1
    i = row - off[b]
    slot = st["lengths"].long()[b] + i
    pg, sl = st["table"][b, slot // case["page"]].long(), slot % case["page"]
    st["k"][pg, :, sl] = st["k_new"].to(st["k"].dtype)
    st["v"][pg, :, sl] = st["v_new"].to(st["v"].dtype)
    st["positions"][b, :, slot] = (st["seen"].long()[b] + i).to(torch.int32).view(n, 1)
    st["weights"][b, :, slot] = 0.0
    new = (off[1:] - off[:-1]).to(torch.int32)
    return {"k": st["k"], "v": st["v"], "positions": st["positions"], "weights": st["weights"],
            "lengths": st["lengths"] + new, "seen": st["seen"] + new}


def _evict(st: dict):
    """Per sequence and head, keep the newest `recent` tokens, the first `sinks` and the largest weights (the lower
    slot where weights are equal), `budget` slots in all; the i-th kept slot at or past the budget moves into the
    i-th slot below it that was given up."""
    case = st["case"]
    b, hkv, n, budget = case["batch"], case["n_head_kv"], case["max_len"], case["budget"]
    w, pos = st["weights"][:, :, :n], st["positions"][:, :, :n]
    length, seen = st["lengths"].view(b, 1, 1), st["seen"].view(b, 1, 1)
    slot = torch.arange(n, device=w.device)
    live = (slot < length).expand(b, hkv, n)
    fixed = (pos >= seen - case["recent"]) | (pos < case["sinks"])
    rank = torch.where(fixed, math.inf, w).masked_fill(~live, -math.inf)
    order = torch.sort(rank, dim=2, descending=True, stable=True).indices
    kept = torch.zeros_like(live).scatter_(2, order, (slot < budget).expand(b, hkv, n)) & live
    over = (length > budget).expand(b, hkv, 1)
    src = kept & (slot >= budget) & over
    dst = ~kept & (slot < budget) & over
    moved_from, moved_to = src.nonzero(), dst.nonzero()               # both in (sequence, head, slot) order: pairs
    bb, hh, sf, sto = moved_from[:, 0], moved_from[:, 1], moved_from[:, 2], moved_to[:, 2]
    page, table = case["page"], st["table"].long()
    pf, pt = table[bb, sf // page], table[bb, sto // page]
    st["k"][pt, hh, sto % page] = st["k"][pf, hh, sf % page]
    st["v"][pt, hh, sto % page] = st["v"][pf, hh, sf % page]
    lo = (slot < torch.clamp(length, max=budget)).expand(b, hkv, n)
    w_out, p_out = st["weights_out"], st["positions_out"]
    w_out[:, :, :n] = torch.where(lo, w, w_out[:, :, :n])
    p_out[:, :, :n] = torch.where(lo, pos, p_out[:, :, :n])
    w_out[bb, hh, sto], p_out[bb, hh, sto] = w[bb, hh, sf], pos[bb, hh, sf]
    return {"k": st["k"], "v": st["v"], "weights": w_out, "positions": p_out,
            "lengths": torch.clamp(st["lengths"], max=budget)}


def _part(frac, total):
    """floor(frac * total / 2^24) for whole numbers frac <= 2^24 and total < 2^62."""
    return (total >> 24) * frac + (((total & 0xffffff) * frac) >> 24)


def _sample(st: dict):
    """Weights 2^((x - max) log2(e) / T) in units of 2^-40, cut down; the token whose weight, added up in the order
    of the vocabulary, passes the share u of the whole. Filters keep a prefix of the logits in falling order (the
    lower index where equal): top-k its first k, top-p the fewest of those whose weight reaches p of theirs, min-p
    what weighs at least min_p of the largest. Temperature 0: the largest logit."""
    x = st["logits"].float()
    b, n = x.shape
    x = torch.where(torch.isnan(x), -math.inf, x)
    top = x.amax(1, keepdim=True)
    first = (x == top).int().argmax(1)
    t = st["temperature"].view(b, 1)
    greedy = ~(t > 0)
    c = torch.tensor(LOG2E, device=x.device) / torch.where(greedy, 1.0, t)
    y = (x - top) * c
    e = torch.exp2(y)
    w = (e * float(ONE)).long()
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    ws, es = w.gather(1, order), e.gather(1, order)
    rank = torch.arange(n, device=x.device)
    k = st["top_k"].view(b, 1).long()
    ws = torch.where(rank < torch.where(k > 0, k, n), ws, 0)
    upto = torch.cumsum(ws, 1)
    frac = torch.round(st["top_p"].view(b, 1) * 16777216.0).long().clamp(0, 1 << 24)
    need = _part(frac, upto[:, -1:])
    need = need + ((frac * (upto[:, -1:] & 0xffffff)) & 0xffffff).ne(0)
    keep = (upto - ws < need.clamp(min=1)) & ((es >= st["min_p"].view(b, 1)) | (rank == 0))
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ws, 0))
    upto = torch.cumsum(kept, 1)
    total = upto[:, -1:]
    share = (st["u"].view(b, 1) * 16777216.0).long().clamp(0, (1 << 24) - 1)
    token = (upto <= _part(share, total)).sum(1)
    token = torch.where(greedy.view(b), first, token)
    lp = y.gather(1, token.view(b, 1)) * math.log(2.0) - torch.log(total.float() / float(ONE))
    return {"token": token.to(torch.int32), "logprob": torch.where(greedy, 0.0, lp).view(b)}


# ---------------------------------------------------------------- in 64 bits

def exact(case: dict, seed: int):
    st = _inputs(case, seed)
    if case["op"] == "sample":
        return _exact_sample(st)
    if case["op"] == "attend":
        return _exact_attend(st)
    # rows, positions and counts are moved, not computed; the rounding of a new row is torch's
    return None


def _exact_attend(st: dict):
    case = st["case"]
    h, hkv, d, page = case["n_head"], case["n_head_kv"], case["head_dim"], case["page"]
    g = h // hkv
    out = torch.zeros(case["batch"], h, d, dtype=torch.float64, device=st["k"].device)
    lse = torch.full((case["batch"], h), -math.inf, dtype=torch.float64, device=out.device)
    acc = st["weights_out"].double() if case["weights"] else None
    for i, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        pages = st["table"][i, :-(-n // page)].long()
        for j in range(hkv):
            k = st["k"][pages, j].double().reshape(-1, d)[:n]
            v = st["v"][pages, j].double().reshape(-1, d)[:n]
            s = torch.einsum("hd,nd->hn", st["q"][i, j * g:(j + 1) * g].double(), k) / d ** 0.5
            lse[i, j * g:(j + 1) * g] = torch.logsumexp(s, 1)
            p = torch.softmax(s, 1)
            out[i, j * g:(j + 1) * g] = torch.einsum("hn,nd->hd", p, v)
            if acc is not None:
                acc[i, j, :n] = st["weights"][i, j, :n].double() + p.sum(0)
    res = {"out": out, "lse": lse}
    if acc is not None:
        res["weights"] = acc
    return res


def _exact_sample(st: dict):
    case = st["case"]
    token, lp = [], []
    for i in range(case["batch"]):
        x = st["logits"][i].double()
        t, k = float(st["temperature"][i]), int(st["top_k"][i])
        if t <= 0:
            token.append(torch.nonzero(x == x.max())[0, 0])
            lp.append(torch.zeros((), dtype=torch.float64, device=x.device))
            continue
        w = torch.exp((x - x.max()) / t)
        value, order = torch.sort(w, descending=True, stable=True)
        if k > 0:
            value, order = value[:k], order[:k]
        c = torch.cumsum(value, 0)
        # the first of the prefix sums that reaches p of the whole ends what top-p keeps
        n = min(value.numel(), int((c < float(st["top_p"][i]) * c[-1]).sum()) + 1)
        n = max(1, min(n, int((value >= float(st["min_p"][i])).sum())))
        kept = torch.zeros_like(w)
        kept[order[:n]] = value[:n]
        c = torch.cumsum(kept, 0)
        j = torch.searchsorted(c, float(st["u"][i]) * c[-1], right=True).clamp(max=x.numel() - 1)
        token.append(j)
        lp.append(torch.log(kept[j] / c[-1]))
    return {"token": torch.stack(token).to(torch.int32), "logprob": torch.stack(lp)}
