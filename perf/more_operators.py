"""What is timed of the operators that a prompt needs on its way through a
server of several sequences: pages and slots for the new tokens (kv_plan),
rotary positions with the store into the cache (rope), the norm in front of a
matrix (rms_norm) and attention of a chunk of new tokens over the paged cache
(kv_attend_chunk).

A case is a dict of plain values. `prepare` makes what a serving program holds
before the call, `run` makes one call -- in plain torch operations where `own`
is false, through the library's Engine where it is true -- and `exact` gives
the same outputs from the definitions in 64 bits. Nothing a call reads is
changed by it, so that it can be repeated: counts and lengths go to buffers of
their own, pages are handed out of the free list without a change to it, and
rotated rows go to other rows than they come from.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
ESIZE = {"f16": 2, "bf16": 2, "f32": 4}
MAX_FLOPS = 560e9                  # of a drawn attention case in 16 bits, and
MAX_FLOPS_F32 = 40e9               # with float32 queries


# ---------------------------------------------------------------- the cases

def listed() -> list[dict]:
    return [
        # One user of the 1B model asks a short follow-up question: the latency of a call.
        dict(name="chunk_short", op="chunk", batch=1, n_head=32, n_head_kv=8, head_dim=64, page=16, min_new=11,
             max_new=11, min_len=600, max_len=600, q="f16", kv="f16", window=0, lens=1),
        # One long prompt read from its start: bound by arithmetic.
        dict(name="chunk_prompt", op="chunk", batch=1, n_head=32, n_head_kv=8, head_dim=128, page=64, min_new=8192,
             max_new=8192, min_len=0, max_len=0, q="bf16", kv="bf16", window=0, lens=2),
        # A step of a full server: chunks of prompts and single tokens, some users far into a long context.
        dict(name="chunk_mixed", op="chunk", batch=24, n_head=32, n_head_kv=8, head_dim=128, page=64, min_new=1,
             max_new=1024, min_len=0, max_len=8192, q="bf16", kv="bf16", window=0, lens=3),
        # A question of 200 tokens about a very long document: few rows, a long axis.
        dict(name="chunk_long", op="chunk", batch=1, n_head=24, n_head_kv=8, head_dim=128, page=64, min_new=200,
             max_new=200, min_len=120000, max_len=120000, q="f16", kv="f16", window=0, lens=4),
        # float32 queries of the engine's matrices over its float16 cache, pages of an odd size.
        dict(name="chunk_f32q", op="chunk", batch=4, n_head=24, n_head_kv=8, head_dim=128, page=41, min_new=100,
             max_new=333, min_len=0, max_len=2000, q="f32", kv="f16", window=0, lens=5),
        # One new token of each user of a full server, from the matrices' float32 into a float16 cache, with the
        # frequencies of a model whose context was stretched by bands.
        dict(name="rope_step", op="rope", n=64, n_head=32, n_head_kv=8, head_dim=64, rot=64, page=16, pairs="next",
             scaling="bands", base=500000.0, max_pos=131072, src="f32", out="f16", store=True),
        # A long prompt in bfloat16, positions from 0.
        dict(name="rope_prompt", op="rope", n=16384, n_head=32, n_head_kv=8, head_dim=128, rot=128, page=64,
             pairs="half", scaling="none", base=10000.0, max_pos=16384, src="bf16", out="bf16", store=False),
        # A model that rotates only part of a head of an odd size, stretched to a long context, into the cache.
        dict(name="rope_part", op="rope", n=3001, n_head=24, n_head_kv=24, head_dim=80, rot=32, page=41, pairs="half",
             scaling="yarn", base=10000.0, max_pos=1000000, src="f16", out="f16", store=True),
        # One token's residual stream of the 1B model in front of a Q4_0 matrix: 8 bits out.
        dict(name="norm_step", op="norm", n=1, k=2048, x="f32", res="f32", out="none", q8=True),
        # A chunk of prompts in bfloat16.
        dict(name="norm_prompt", op="norm", n=16384, k=4096, x="bf16", res="bf16", out="bf16", q8=False),
        # A full server's next token each: now and then a user needs a page, and some are done.
        dict(name="plan_step", op="plan", batch=256, page=16, max_new=1, max_len=4096, ended=0.03, spare=1.0, lens=11),
        # Prompts come in, and not all of them find pages.
        dict(name="plan_prompts", op="plan", batch=61, page=16, max_new=4000, max_len=2000, ended=0.2, spare=0.7,
             lens=12),
    ]


def _log(rng: random.Random, lo: float, hi: float) -> int:
    return max(int(lo), min(int(hi), int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random) -> dict:
    op = rng.choice(["chunk", "chunk", "chunk", "chunk", "rope", "rope", "norm", "norm", "plan"])
    lens = rng.randrange(1 << 30)
    page = rng.choice([16, 32, 64, 128, rng.randrange(1, 200)])
    head_dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256])
    n_head_kv = rng.choice([1, 2, 4, 8, 8, 8, 16])
    if op == "chunk":
        kv = rng.choice(["f16", "bf16", "bf16", "f32"])
        q = {"f16": rng.choice(["f16", "f16", "f32"]), "bf16": "bf16", "f32": "f32"}[kv]
        window = rng.choice([0, 0, 0, _log(rng, 16, 8192)])
        max_new, max_len, batch = _log(rng, 1, 8192), rng.choice([0, _log(rng, 1, 120000)]), _log(rng, 1, 48)
        case = dict(op=op, batch=batch, n_head=n_head_kv * rng.choice([1, 2, 3, 4, 4, 5, 7, 8]), n_head_kv=n_head_kv,
                    head_dim=head_dim, page=page, min_new=rng.choice([0, 1, max_new]), max_new=max_new,
                    min_len=rng.choice([0, max_len]), max_len=max_len, q=q, kv=kv, window=window, lens=lens)
        most = MAX_FLOPS_F32 if q == "f32" else MAX_FLOPS
        while work(case)["flops"] > most or work(case)["bytes"] > 512 << 20:      # fewer users, then shorter ones
            if case["batch"] > 1:
                case["batch"] = (case["batch"] + 1) // 2
            else:
                key = "max_len" if case["max_len"] > 4 * case["max_new"] else "max_new"
                case[key] = case[key] * 3 // 4
                low = "min" + key[3:]
                case[low] = min(case[low], case[key])
        return case
    if op == "rope":
        n = _log(rng, 1, 16384)
        src = rng.choice(["f32", "f16", "bf16", "bf16"])
        rot = rng.choice([head_dim, head_dim, 2 * rng.randrange(1, head_dim // 2 + 1)])
        return dict(op=op, n=min(n, 16384 * 10240 // (head_dim * 10 * n_head_kv)), n_head=n_head_kv * rng.choice([1, 2, 4, 8]),
                    n_head_kv=n_head_kv, head_dim=head_dim, rot=rot, page=page, pairs=rng.choice(["half", "half", "next"]),
                    scaling=rng.choice(["none", "linear", "bands", "yarn"]), base=rng.choice([10000.0, 500000.0]),
                    max_pos=_log(rng, n, 1000000), src=src, out=rng.choice(["f16", "bf16", "f32"]) if src == "f32" else src,
                    store=rng.random() < 0.6)
    if op == "norm":
        k = rng.choice([1024, 2048, 4096, 8192, 32 * _log(rng, 2, 256)])
        n = _log(rng, 1, min(16384, 16384 * 4096 // k))
        x = rng.choice(["f32", "bf16", "bf16", "f16"])
        out, q8 = rng.choice([(x, False), (x, False), ("none", True), (x, True)])
        return dict(op=op, n=n, k=k, x=x, res=rng.choice([x, "f32", "none"]), out=out, q8=q8)
    max_new = rng.choice([1, _log(rng, 1, 4000)])
    batch = _log(rng, 1, 2000 if max_new == 1 else min(2000, max(1, 128000 // max_new)))
    return dict(op=op, batch=batch, page=page, max_new=max_new, max_len=_log(rng, 1, 4096),
                ended=round(rng.uniform(0, 0.3), 3), spare=round(rng.uniform(0.3, 1.2), 3), lens=lens)


def _chunks(case: dict) -> tuple[list[int], list[int]]:
    """New tokens and slots in use before them, per sequence: part of the case, so that its work is known."""
    rng = random.Random(case["lens"])
    new = [rng.randint(case["min_new"], case["max_new"]) for _ in range(case["batch"])]
    new[rng.randrange(len(new))] = case["max_new"]
    old = [rng.randint(case["min_len"], case["max_len"]) for _ in range(case["batch"])]
    old[rng.randrange(len(old))] = case["max_len"]
    return new, old


def _requests(case: dict) -> tuple[list[int], list[int], list[int], list[int]]:
    """Per sequence its slots in use, the tokens it wants to add (-1: it is done), the pages it holds and the tokens
    it has had. Pages are held for what is in use; some sequences were cut and hold more."""
    rng = random.Random(case["lens"])
    length = [rng.randint(0, case["max_len"]) for _ in range(case["batch"])]
    new = [-1 if rng.random() < case["ended"] else rng.randint(min(1, case["max_new"]), case["max_new"]) for _ in length]
    held = [-(-x // case["page"]) for x in length]
    for i in range(len(held)):
        if rng.random() < 0.05:
            held[i] += rng.randint(0, 8)
    seen = [x + (rng.randint(0, 1000) if rng.random() < 0.2 else 0) for x in length]
    return length, new, held, seen


def _pool(case: dict) -> tuple[int, int, int]:
    """Columns of the table, pages of the pool and how many of them are free: enough for a part of what is wanted."""
    length, new, held, _ = _requests(case)
    page = case["page"]
    want = [-(-(x + n) // page) if n >= 0 else 0 for x, n in zip(length, new)]
    cols = max(max(want), max(held), 1)
    need = sum(max(w - h, 0) for w, h in zip(want, held))
    free = int(case["spare"] * need) + 1
    return cols, sum(held) + free, free


def work(case: dict) -> dict:
    if case["op"] == "chunk":
        new, old = _chunks(case)
        h, hkv, d = case["n_head"], case["n_head_kv"], case["head_dim"]
        pairs, rows = 0, 0
        for n, x in zip(new, old):
            w = case["window"] or n + x
            full = max(0, min(n, w - x))             # rows that see fewer slots than the window holds
            pairs += full * x + full * (full + 1) // 2 + (n - full) * w
            rows += min(n + x, w + n - 1) if n else 0   # slots that some row sees
        by = rows * hkv * d * 2 * ESIZE[case["kv"]] + sum(new) * h * (2 * d * ESIZE[case["q"]] + 4)
        return {"bytes": by, "flops": 4 * pairs * h * d}
    if case["op"] == "rope":
        n, d = case["n"], case["head_dim"]
        heads = case["n_head"] + case["n_head_kv"] * (2 if case["store"] else 1)
        by = n * d * heads * (ESIZE[case["src"]] + ESIZE[case["out"]]) + n * (12 if case["store"] else 4)
        return {"bytes": by, "flops": n * (case["n_head"] + case["n_head_kv"]) * case["rot"] * 3}
    if case["op"] == "norm":
        n, k = case["n"], case["k"]
        by = ESIZE[case["x"]] + 2 * ESIZE.get(case["res"], 0) + ESIZE.get(case["out"], 0) + (1.125 if case["q8"] else 0)
        return {"bytes": int(n * k * by) + 4 * k, "flops": 5 * n * k}
    length, new, held, _ = _requests(case)
    cols, n_pages, free = _pool(case)
    tokens = sum(max(n, 0) for n in new)
    moved = sum(abs(-(-(x + n) // case["page"]) - h) if n >= 0 else h for x, n, h in zip(length, new, held))
    return {"bytes": 40 * case["batch"] + 16 * tokens + 8 * moved, "flops": tokens + moved}


# ---------------------------------------------------------------- the inputs

def _frequencies(case: dict) -> torch.Tensor:
    """Radians a position for each pair, float64, on the host: the model's, stretched for a longer context."""
    rot, base, kind = case["rot"], case["base"], case["scaling"]
    i = torch.arange(rot // 2, dtype=torch.float64)
    inv = base ** (-2.0 * i / rot)
    if kind == "linear":
        return inv / 4.0
    if kind == "bands":                       # slow pairs by 8, quick ones as they are, from wavelength to wavelength
        turns = 8192 * inv / (2 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return inv * keep + inv / 8.0 * (1 - keep)
    if kind == "yarn":                        # the same between two pairs, named by the turns they make
        def pair(turns):
            return rot * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), rot - 1)
        slow = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return inv / 16.0 * slow + inv * (1 - slow)
    return inv


def _mscale(case: dict) -> float:
    return 0.1 * math.log(16.0) + 1.0 if case["scaling"] == "yarn" else 1.0


def prepare(case: dict, seed: int) -> dict:
    st = _inputs(case, seed)
    if own:                                    # the handle that a program opens once, and what it keeps beside
        from __graft_entry__ import load_package
        pkg = load_package()
        st["eng"] = pkg.Engine(torch.cuda.current_device())
        if "k_pool" in st:
            st["cache"] = pkg.PagedKV(st["k_pool"], st["v_pool"], st["table"], st["lengths"])
        if case["op"] == "rope":
            kw = {"none": {}, "linear": dict(scaling="linear", factor=4.0),
                  "bands": dict(scaling="bands", factor=8.0, context=8192, low=1.0, high=4.0),
                  "yarn": dict(scaling="yarn", factor=16.0, context=4096, low=1.0, high=32.0)}[case["scaling"]]
            st["freqs"] = pkg.rope_freqs(case["rot"], case["base"], **kw).to(st["positions"].device)
    return st


def _inputs(case: dict, seed: int) -> dict:
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device=dev, dtype=dtype)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=dev)

    st = {"case": case}
    if case["op"] == "norm":
        n, k, dt = case["n"], case["k"], DTYPES[case["x"]]
        # a residual stream has a few large channels, what a layer adds to it is small
        wide = 1 + 8 * (torch.rand(k, generator=gen, device=dev) < 0.01)
        x = normal(n, k) * wide
        if case["res"] == "none":
            st["x"] = x.to(dt)
        else:
            st["x"], st["res"] = (0.3 * normal(n, k)).to(dt), x.to(DTYPES[case["res"]])
            st["res_out"] = torch.empty_like(st["res"])
        st["w"] = 1 + 0.2 * normal(k)
        if case["out"] != "none":
            st["out"] = torch.empty(n, k, dtype=DTYPES[case["out"]], device=dev)
        if case["q8"]:
            st["q8"] = torch.empty(n, k + k // 8, dtype=torch.uint8, device=dev)
        return st
    if case["op"] == "rope":
        n, h, hkv, d, page = case["n"], case["n_head"], case["n_head_kv"], case["head_dim"], case["page"]
        src, out = DTYPES[case["src"]], DTYPES[case["out"]]
        st["q"], st["k"] = normal(n, h, d).to(src), normal(n, hkv, d).to(src)
        # a step's tokens are anywhere, a prompt's in a row
        first = torch.randint(max(case["max_pos"] - n, 0) + 1, (1,), generator=gen, device=dev)
        st["positions"] = (first + torch.arange(n, device=dev)).to(torch.int32)
        if n <= 256:
            st["positions"] = torch.randint(case["max_pos"], (n,), generator=gen, device=dev, dtype=torch.int32)
        st["q_out"] = torch.empty(n, h, d, dtype=out, device=dev)
        if case["store"]:
            st["v"] = normal(n, hkv, d).to(src)
            n_pages = -(-n // page) + 4
            perm = torch.randperm(n_pages * page, generator=gen, device=dev)[:n] if n <= 256 else \
                (torch.randperm(n_pages, generator=gen, device=dev)[:-(-n // page), None] * page
                 + torch.arange(page, device=dev)).flatten()[:n]
            st["slots"] = perm.long().contiguous()
            st["k_pool"], st["v_pool"] = normal(n_pages, hkv, page, d).to(out), normal(n_pages, hkv, page, d).to(out)
            st["table"], st["lengths"] = ints([[0]]), ints([0])
        else:
            st["k_out"] = torch.empty(n, hkv, d, dtype=out, device=dev)
        return st
    page = case["page"]
    if case["op"] == "plan":
        length, new, held, seen = _requests(case)
        cols, n_pages, free = _pool(case)
        b, n = case["batch"], sum(max(x, 0) for x in new)
        perm = torch.randperm(n_pages, generator=gen, device=dev).to(torch.int32)
        table = torch.full((b, cols), -1, dtype=torch.int32, device=dev)
        starts = torch.cumsum(torch.tensor([0] + held, device=dev), 0)[:-1, None]
        col = torch.arange(cols, device=dev)
        own_pages = col < torch.tensor(held, device=dev)[:, None]
        table[own_pages] = perm[(starts + col)[own_pages]]
        # the free list's end is what is handed out next; behind it there is room for what comes back
        st["free"] = torch.cat([perm[sum(held):], torch.full((sum(held),), -1, dtype=torch.int32, device=dev)])
        st.update(lengths=ints(length), new=ints(new), held=ints(held), seen=ints(seen), table=table,
                  free_count=ints([free]), k_pool=torch.empty(n_pages, 1, page, 8, dtype=torch.float16, device=dev),
                  v_pool=torch.empty(n_pages, 1, page, 8, dtype=torch.float16, device=dev))
        for name in ("lengths_out", "held_out", "seen_out", "granted"):
            st[name] = torch.empty(b, dtype=torch.int32, device=dev)
        st["free_count_out"] = torch.empty(1, dtype=torch.int32, device=dev)
        st["offsets"] = torch.empty(b + 1, dtype=torch.int32, device=dev)
        st["slots"] = torch.empty(n, dtype=torch.int64, device=dev)
        st["positions"] = torch.empty(n, dtype=torch.int32, device=dev)
        st["sequences"] = torch.empty(n, dtype=torch.int32, device=dev)
        return st
    new, old = _chunks(case)
    h, hkv, d, dt = case["n_head"], case["n_head_kv"], case["head_dim"], DTYPES[case["kv"]]
    total = [x + n for x, n in zip(old, new)]
    pages = [-(-x // page) for x in total]
    n_pages, cols = sum(pages) + 1, max(1, max(pages))
    # pages in the order in which a running server hands them out: any
    perm = torch.randperm(n_pages, generator=gen, device=dev).to(torch.int32)
    table = torch.zeros(case["batch"], cols, dtype=torch.int32, device=dev)
    at = 0
    for i, c in enumerate(pages):
        table[i, :c] = perm[at:at + c]
        at += c
    off = [0]
    for n in new:
        off.append(off[-1] + n)
    st.update(k_pool=normal(n_pages, hkv, page, d, dtype=dt), v_pool=normal(n_pages, hkv, page, d, dtype=dt), table=table,
              lengths=ints(total), offsets=ints(off))
    st["q"] = (1.5 * normal(off[-1], h, d)).to(DTYPES[case["q"]])
    st["out"] = torch.empty_like(st["q"])
    st["lse"] = torch.empty(off[-1], h, device=dev)
    return st


# ---------------------------------------------------------------- one pass

def run(st: dict):
    case = st["case"]
    if not own:
        return {"chunk": _chunk, "rope": _rope, "norm": _norm, "plan": _plan}[case["op"]](st)
    eng = st["eng"]
    eng.set_stream(torch.cuda.current_stream().cuda_stream)
    if case["op"] == "chunk":
        eng.kv_attend_chunk(st["cache"], st["q"], st["out"], st["offsets"], lse=st["lse"], window=case["window"])
        return {"out": st["out"], "lse": st["lse"]}
    if case["op"] == "rope":
        kw = dict(interleaved=case["pairs"] == "next", mscale=_mscale(case))
        if case["store"]:
            eng.rope(st["positions"], st["freqs"], q=st["q"], q_out=st["q_out"], k=st["k"], kv=st["cache"], v=st["v"],
                     slots=st["slots"], **kw)
            return {"q": st["q_out"], "k_pool": st["k_pool"], "v_pool": st["v_pool"]}
        eng.rope(st["positions"], st["freqs"], q=st["q"], q_out=st["q_out"], k=st["k"], k_out=st["k_out"], **kw)
        return {"q": st["q_out"], "k": st["k_out"]}
    if case["op"] == "norm":
        eng.rms_norm(st["x"], st["w"], out=st.get("out"), eps=1e-5, residual=st.get("res"),
                     residual_out=st.get("res_out"), q8=st.get("q8"))
        res = {}
        if "res" in st:
            res["residual"] = st["res_out"]
        if "out" in st:
            res["out"] = st["out"]
        if case["q8"]:                        # the packed rows as the values that they stand for
            n, k = case["n"], case["k"]
            code = st["q8"][:, :k].view(torch.int8).view(n, k // 32, 32)
            res["q8"] = (code * st["q8"][:, k:].view(torch.float32).unsqueeze(2)).view(n, k)
        return res
    eng.kv_plan(st["cache"], st["new"], st["held"], st["free"], st["free_count"], st["offsets"], slots=st["slots"],
                positions=st["positions"], sequences=st["sequences"], granted=st["granted"], seen=st["seen"],
                lengths_out=st["lengths_out"], held_out=st["held_out"], free_count_out=st["free_count_out"],
                seen_out=st["seen_out"])
    return {name: st[name] for name in PLAN_OUTPUTS}


PLAN_OUTPUTS = ("table", "free", "free_count_out", "held_out", "lengths_out", "seen_out", "granted", "offsets", "slots",
                "positions", "sequences")


def _chunk(st: dict):
    """softmax(q K^T / sqrt(d)) V: the new token at slot p sees slots 0 up to p, or the last `window` of them."""
    case = st["case"]
    h, hkv, d, page = case["n_head"], case["n_head_kv"], case["head_dim"], case["page"]
    g = h // hkv
    out, lse = torch.empty_like(st["q"]), torch.empty_like(st["lse"])
    at = 0
    for i, (n, old) in enumerate(zip(*_chunks(case))):
        if n == 0:
            continue
        first = max(0, old + 1 - case["window"]) if case["window"] else 0
        slot = torch.arange(first, old + n, device=out.device)
        pages, rows = st["table"][i, slot // page].long(), slot % page
        dead = slot > (old + torch.arange(n, device=out.device)).view(n, 1)
        if case["window"]:
            dead |= slot <= (old - case["window"] + torch.arange(n, device=out.device)).view(n, 1)
        side = max(1, min(hkv, (1 << 28) // (g * n * slot.numel())))        # cache heads at a time
        for j in range(0, hkv, side):
            e = min(hkv, j + side)
            k = st["k_pool"][pages, j:e, rows].float().permute(1, 2, 0)                       # heads d slots
            v = st["v_pool"][pages, j:e, rows].float().permute(1, 0, 2)
            q = st["q"][at:at + n, j * g:e * g].float().view(n, e - j, g, d).permute(1, 2, 0, 3)   # heads g n d
            s = (q.reshape(e - j, g * n, d) @ k).view(e - j, g, n, -1)
            s.mul_(1.0 / math.sqrt(d)).masked_fill_(dead, -math.inf)
            m = s.amax(3, keepdim=True)
            p = s.sub_(m).exp_()
            z = p.sum(3, keepdim=True)
            o = (p.view(e - j, g * n, -1) @ v).view(e - j, g, n, d) / z
            out[at:at + n, j * g:e * g] = o.permute(2, 0, 1, 3).reshape(n, -1, d).to(out.dtype)
            lse[at:at + n, j * g:e * g] = (m + torch.log(z)).view(e - j, g, n).permute(2, 0, 1).reshape(n, -1)
        at += n
    return {"out": out, "lse": lse}


def _rope(st: dict):
    """The pairs of a head's first elements (neighbours, or i and i + half) turned by position times frequency."""
    case = st["case"]
    rot, m = case["rot"], _mscale(case)
    angle = st["positions"].double().view(-1, 1) * _frequencies(case).to(st["positions"].device)
    c, s = (torch.cos(angle).float() * m).unsqueeze(1), (torch.sin(angle).float() * m).unsqueeze(1)

    def turn(x):
        y = x.float().clone()
        a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if case["pairs"] == "next" else (y[..., :rot // 2], y[..., rot // 2:rot])
        a_new, b_new = a * c - b * s, b * c + a * s
        a.copy_(a_new)
        b.copy_(b_new)
        return y.to(DTYPES[case["out"]])

    q, k = turn(st["q"]), turn(st["k"])
    if not case["store"]:
        return {"q": q, "k": k}
    pages, rows = st["slots"] // case["page"], st["slots"] % case["page"]
    st["k_pool"][pages, :, rows] = k
    st["v_pool"][pages, :, rows] = st["v"].to(k.dtype)
    return {"q": q, "k_pool": st["k_pool"], "v_pool": st["v_pool"]}


def _norm(st: dict):
    """r = residual + x; y = w r / sqrt(mean(r^2) + eps); in 8 bits: per 32 values a scale of the largest / 127, kept in
    16 bits, and codes rounded to nearest, halves away from 0."""
    case = st["case"]
    n, k = case["n"], case["k"]
    r = st["x"].float()
    res = {}
    if "res" in st:
        r = r + st["res"].float()
        res["residual"] = r.to(st["res"].dtype)
    y = r * torch.rsqrt(r.square().mean(1, keepdim=True) + 1e-5) * st["w"]
    if "out" in st:
        res["out"] = y.to(st["out"].dtype)
    if case["q8"]:
        y = y.view(n, k // 32, 32)
        scale = y.abs().amax(2, keepdim=True) / 127.0
        inv = torch.where(scale == 0, 0.0, 1.0 / scale)
        code = torch.sign(y) * torch.floor((y * inv).abs() + 0.5)
        res["q8"] = (code * scale.half().float()).view(n, k)
    return res


def _plan(st: dict):
    """Pages that a sequence no longer needs go back to the end of the free list, in the order of sequences and columns;
    then each takes what it needs from that end, in the same order, while all up to it find enough."""
    case = st["case"]
    page, b = case["page"], case["batch"]
    n_pages, cols, dev = st["k_pool"].shape[0], st["table"].shape[1], st["table"].device
    length, new, held = st["lengths"].long(), st["new"].long(), st["held"].long()
    done, add = new < 0, new.clamp(min=0)
    total = torch.where(done, 0, length + add)
    fits = total <= cols * page
    want = torch.where(fits, (total + page - 1) // page, held)
    back, need = (held - want).clamp(min=0), (want - held).clamp(min=0)
    col = torch.arange(cols, device=dev)
    table, free = st["table"], st["free"]
    dump = torch.cat([free, free.new_zeros(1)])
    at = st["free_count"].long() + (torch.cumsum(back, 0) - back).view(b, 1) + col - want.view(b, 1)
    leaves = (col >= want.view(b, 1)) & (col < held.view(b, 1))
    dump[torch.where(leaves, at, free.numel())] = table
    free.copy_(dump[:-1])
    count = st["free_count"].long() + back.sum()
    upto = torch.cumsum(need, 0)
    given = fits & ((need == 0) | (upto <= count))
    take = torch.where(given, need, 0)
    at = count - 1 - (upto - need).view(b, 1) - (col - held.view(b, 1))
    comes = given.view(b, 1) & (col >= held.view(b, 1)) & (col < want.view(b, 1))
    table.copy_(torch.where(comes, free[at.clamp(0, free.numel() - 1)], table))
    granted = torch.where(given & ~done, add, 0)
    offsets = torch.cat([add.new_zeros(1), torch.cumsum(add, 0)])
    t = torch.arange(st["slots"].numel(), device=dev)
    seq = torch.searchsorted(offsets, t, right=True) - 1
    i = t - offsets[seq]
    slot = length[seq] + i
    where = table[seq, (slot // page).clamp(max=cols - 1)].long()
    there = given[seq] & (where >= 0) & (where < n_pages)
    i32 = torch.int32
    return {"table": table, "free": free, "free_count_out": (count - take.sum()).to(i32).view(1),
            "held_out": torch.where(given, want, held).to(i32),
            "lengths_out": torch.where(done, 0, length + granted).to(i32),
            "seen_out": torch.where(done, 0, st["seen"].long() + granted).to(i32), "granted": granted.to(i32),
            "offsets": offsets.to(i32), "slots": torch.where(there, where * page + slot % page, -1),
            "positions": (st["seen"].long()[seq] + i).to(i32), "sequences": seq.to(i32)}


# ---------------------------------------------------------------- in 64 bits

def exact(case: dict, seed: int):
    st = _inputs(case, seed)
    return {"chunk": _exact_chunk, "rope": _exact_rope, "norm": _exact_norm, "plan": _exact_plan}[case["op"]](st)


def _exact_chunk(st: dict):
    case = st["case"]
    h, hkv, d, page = case["n_head"], case["n_head_kv"], case["head_dim"], case["page"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    lse = torch.full(st["lse"].shape, -math.inf, dtype=torch.float64, device=out.device)
    offsets = st["offsets"].tolist()
    for i, length in enumerate(st["lengths"].tolist()):
        lo, hi = offsets[i], offsets[i + 1]
        if lo == hi:
            continue
        pages = st["table"][i, :-(-length // page)].long()
        for j in range(hkv):
            k = st["k_pool"][pages, j].reshape(-1, d)[:length].double()
            v = st["v_pool"][pages, j].reshape(-1, d)[:length].double()
            for x in range(j * h // hkv, (j + 1) * h // hkv):
                for a in range(lo, hi, 4096):                       # rows a up to b, the last of them at slot `last`
                    b = min(a + 4096, hi)
                    last = length - (hi - b)
                    s = torch.einsum("nd,ld->nl", st["q"][a:b, x].double(), k[:last]) / d ** 0.5
                    row = torch.arange(last - (b - a), last, device=out.device)[:, None]
                    col = torch.arange(last, device=out.device)[None]
                    hidden = col > row
                    if case["window"]:
                        hidden = hidden | (row - col >= case["window"])
                    s[hidden] = -math.inf
                    lse[a:b, x] = torch.logsumexp(s, 1)
                    out[a:b, x] = torch.softmax(s, 1) @ v[:last]
    return {"out": out, "lse": lse}


def _exact_rope(st: dict):
    case = st["case"]
    rot = case["rot"]
    half = rot // 2
    first = torch.arange(half) * 2 if case["pairs"] == "next" else torch.arange(half)
    other = first + (1 if case["pairs"] == "next" else half)
    turn = torch.polar(torch.tensor(_mscale(case), dtype=torch.float64).expand(case["n"], half).contiguous(),
                       (st["positions"].cpu().double()[:, None] * _frequencies(case)[None]))
    turn = turn.to(st["q"].device)[:, None]
    res = []
    for x in (st["q"], st["k"]):
        y = x.double().clone()
        z = torch.complex(y[:, :, first], y[:, :, other]) * turn
        y[:, :, first], y[:, :, other] = z.real, z.imag
        res.append(y)
    if not case["store"]:
        return {"q": res[0], "k": res[1]}
    k_pool, v_pool = st["k_pool"].double(), st["v_pool"].double()
    for i, s in enumerate(st["slots"].tolist()):
        k_pool[s // case["page"], :, s % case["page"]] = res[1][i]
        v_pool[s // case["page"], :, s % case["page"]] = st["v"][i].double()
    return {"q": res[0], "k_pool": k_pool, "v_pool": v_pool}


def _exact_norm(st: dict):
    case = st["case"]
    r = st["x"].double()
    res = {}
    if "res" in st:
        r = r + st["res"].double()
        res["residual"] = r
    y = r / torch.sqrt(torch.mean(r * r, dim=1, keepdim=True) + 1e-5) * st["w"].double()
    if "out" in st:
        res["out"] = y
    if case["q8"]:
        b = y.reshape(case["n"], -1, 32)
        step = b.abs().max(dim=2, keepdim=True).values / 127
        code = torch.where(step > 0, b / step, torch.zeros_like(b))
        code = torch.where(code < 0, torch.ceil(code - 0.5), torch.floor(code + 0.5))
        res["q8"] = (code * step.to(torch.float16).double()).reshape(y.shape)
    return res


def _exact_plan(st: dict):
    """Request by request, with a list of free pages, as a host program would."""
    page = st["case"]["page"]
    table, free = st["table"].tolist(), st["free"].tolist()
    length, new, held, seen = (st[x].tolist() for x in ("lengths", "new", "held", "seen"))
    count, capacity, n_pages = int(st["free_count"]), len(table[0]) * page, st["k_pool"].shape[0]
    want = [0 if n < 0 else -(-(x + n) // page) if x + n <= capacity else c for x, n, c in zip(length, new, held)]
    for b, row in enumerate(table):
        for c in range(want[b], held[b]):
            free[count] = row[c]
            count += 1
    left, asked, given = count, 0, []
    for b, row in enumerate(table):
        need = max(want[b] - held[b], 0)
        asked += need
        given.append((new[b] < 0 or length[b] + new[b] <= capacity) and (need == 0 or asked <= count))
        if given[b]:
            for c in range(held[b], want[b]):
                left -= 1
                row[c] = free[left]
    offsets, slots, positions, sequences, granted = [0], [], [], [], []
    for b, row in enumerate(table):
        granted.append(new[b] if given[b] and new[b] > 0 else 0)
        for i in range(max(new[b], 0)):
            s = length[b] + i
            p = row[s // page] if given[b] else -1
            slots.append(p * page + s % page if 0 <= p < n_pages else -1)
            positions.append(seen[b] + i)
            sequences.append(b)
        offsets.append(len(slots))
    dev, i32 = st["table"].device, torch.int32
    res = {"table": table, "free": free, "free_count_out": [left],
           "held_out": [w if ok else c for w, c, ok in zip(want, held, given)],
           "lengths_out": [0 if n < 0 else x + m for x, n, m in zip(length, new, granted)],
           "seen_out": [0 if n < 0 else x + m for x, n, m in zip(seen, new, granted)],
           "granted": granted, "offsets": offsets, "slots": slots, "positions": positions, "sequences": sequences}
    return {name: torch.tensor(res[name], dtype=torch.int64 if name == "slots" else i32, device=dev)
            for name in PLAN_OUTPUTS}
