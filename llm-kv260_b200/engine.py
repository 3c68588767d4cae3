"""Python wrappers over the C ABI: the engine (b200_engine.h) and the
drop-in device interfaces (gemv_dev.h, gemv2_dev.h, udmabuf.h).

Device memory comes from torch (plumbing only); every computation is a call
into libb200gemv.so.
"""

from __future__ import annotations

import ctypes
from struct import Struct
from threading import Lock

from . import capi
from .capi import check, lib
from .paged import PagedKV, address, dtype_code, row_stride, rows

# native struct formats of the C ABI's field types
_FORMAT = {capi.c_u64: "Q", capi.c_i64: "q", capi.c_int: "i", ctypes.c_float: "f"}

QK = 32
BLOCK_BYTES = 18
LAYOUT_ROWS = 0    # GGUF rows (B200_LAYOUT_ROWS)
LAYOUT_TILES = 1   # the engine's re-laid tiles (B200_LAYOUT_TILES)


def _torch():
    import torch
    return torch


def dev_ptr(t) -> int:
    """Device address of a CUDA tensor (or an int address as is)."""
    if isinstance(t, int):
        return t
    if not t.is_cuda:
        raise ValueError("expected a CUDA tensor")
    if not t.is_contiguous():
        raise ValueError("expected a contiguous tensor")
    return int(t.data_ptr())


def current_stream_handle(device: int) -> int:
    torch = _torch()
    return int(torch.cuda.current_stream(device).cuda_stream)


def tiled_bytes(rows: int, k: int) -> int:
    return int(lib().b200_tiled_bytes(rows, k))


class QMat:
    """A Q4_0 matrix in device memory (b200_qmat_t): GGUF rows, or the
    engine's tiles (Engine.repack)."""

    def __init__(self, blocks, rows: int, k: int, layout: int = LAYOUT_ROWS):
        if k % QK:
            raise ValueError(f"in_features must be a multiple of {QK}, got {k}")
        nbytes = rows * (k // QK) * BLOCK_BYTES if layout == LAYOUT_ROWS else tiled_bytes(rows, k)
        if hasattr(blocks, "numel") and blocks.numel() * blocks.element_size() < nbytes:
            raise ValueError(f"blocks tensor is smaller than the {nbytes} bytes of a {rows}x{k} matrix")
        self.blocks = blocks          # keeps the allocation alive
        self.rows, self.k, self.layout = rows, k, layout
        self.c = capi.b200_qmat_t(dev_ptr(blocks), rows, k, layout)

    @classmethod
    def from_numpy(cls, blocks_np, device: int = 0) -> "QMat":
        torch = _torch()
        rows, rb = blocks_np.shape
        t = torch.from_numpy(blocks_np.reshape(-1).copy()).to(f"cuda:{device}")
        return cls(t, rows, rb // BLOCK_BYTES * QK)

    @property
    def nbytes(self) -> int:
        """Algorithmic weight bytes (18 per 32 weights), whatever the layout."""
        return self.rows * (self.k // QK) * BLOCK_BYTES


ROPE_SCALING = {None: 0, "linear": 1, "bands": 2, "yarn": 3}


def rope_freqs(rot_dim: int, base: float = 10000.0, factors=None, scaling: str | None = None, factor: float = 1.0,
               context: float = 0.0, low: float = 1.0, high: float = 32.0):
    """Frequencies for Engine.rope, an int64 tensor [rot_dim / 2] on the host in units of 2^-64 turns: base^(-2 i /
    rot_dim) radians divided by factors[i], and for long contexts "linear", "bands" or "yarn" (b200_rope_freqs)."""
    torch = _torch()
    if scaling not in ROPE_SCALING:
        raise ValueError(f"scaling must be one of {list(ROPE_SCALING)}")
    out = torch.empty(max(rot_dim // 2, 0), dtype=torch.int64)
    if factors is not None:
        factors = torch.as_tensor(factors, dtype=torch.float32, device="cpu").contiguous()
        if factors.shape != out.shape:
            raise ValueError(f"factors must hold rot_dim / 2 = {out.numel()} numbers")
    check(lib().b200_rope_freqs(out.data_ptr(), rot_dim, base, None if factors is None else factors.data_ptr(),
                                ROPE_SCALING[scaling], factor, context, low, high), "b200_rope_freqs")
    return out


class Engine:
    """b200_engine.h: the engine_t-level call (tp_llama.cpp:289-375). One thread at a time, as there; only the serving
    calls (kv_*, sample, rope, rms_norm) may come from several, on a stream that stays the same."""

    def __init__(self, device: int = 0, stream: int | None = None):
        self.device = device
        h = ctypes.c_void_p()
        check(lib().b200_engine_open(ctypes.byref(h), device), "b200_engine_open")
        self.h = h
        self._lock, self._structs = Lock(), {}
        self._ws, self._ws_at, self._ws_bytes, self._ws_old, self._ws_recorded = None, 0, 0, [], []
        self.set_stream(current_stream_handle(device) if stream is None else stream)

    def close(self) -> None:
        if self.h:
            lib().b200_engine_close(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def set_stream(self, stream: int | None) -> None:
        check(lib().b200_engine_set_stream(self.h, stream), "b200_engine_set_stream")

    @property
    def stream(self) -> int:
        return int(lib().b200_engine_stream(self.h) or 0)

    def config(self) -> dict:
        c = capi.b200_engine_config_t()
        check(lib().b200_engine_get_config(self.h, ctypes.byref(c)), "b200_engine_get_config")
        return {f: getattr(c, f) for f, _ in c._fields_}

    def configure(self, **kw) -> None:
        c = capi.b200_engine_config_t()
        check(lib().b200_engine_get_config(self.h, ctypes.byref(c)), "b200_engine_get_config")
        for k, v in kw.items():
            if not hasattr(c, k):
                raise KeyError(k)
            setattr(c, k, int(v))
        check(lib().b200_engine_set_config(self.h, ctypes.byref(c)), "b200_engine_set_config")

    def gemv_f32(self, W: QMat, x, y, next: QMat | None = None) -> None:
        check(lib().b200_gemv_f32(self.h, ctypes.byref(W.c), dev_ptr(x), dev_ptr(y),
                                  ctypes.byref(next.c) if next else None), "b200_gemv_f32")

    def gemv_q8(self, W: QMat, xpacked, y, next: QMat | None = None) -> None:
        check(lib().b200_gemv_q8(self.h, ctypes.byref(W.c), dev_ptr(xpacked), dev_ptr(y),
                                 ctypes.byref(next.c) if next else None), "b200_gemv_q8")

    def quantize(self, x, xpacked, k: int) -> None:
        check(lib().b200_quantize_q8_0(self.h, dev_ptr(x), dev_ptr(xpacked), k), "b200_quantize_q8_0")

    def repack(self, W: QMat) -> QMat:
        """GGUF rows -> a new tiled matrix on this engine's device (b200_repack_q4_0)."""
        torch = _torch()
        if W.layout != LAYOUT_ROWS:
            raise ValueError("repack takes a GGUF-row matrix")
        n = tiled_bytes(W.rows, W.k)
        if n == 0:
            raise ValueError(f"cannot tile a {W.rows}x{W.k} matrix")
        dst = torch.empty(n, dtype=torch.uint8, device=f"cuda:{self.device}")
        check(lib().b200_repack_q4_0(self.h, W.c.w, W.rows, W.k, dev_ptr(dst)), "b200_repack_q4_0")
        return QMat(dst, W.rows, W.k, LAYOUT_TILES)

    def gemv_argmax_f32(self, W: QMat, x, y, out, index_base: int = 0) -> None:
        """gemv_f32 with the greedy pick over y fused into it (out: int32 index + index_base, float32 value)."""
        check(lib().b200_gemv_argmax_f32(self.h, ctypes.byref(W.c), dev_ptr(x), dev_ptr(y), index_base, dev_ptr(out)),
              "b200_gemv_argmax_f32")

    def argmax(self, y, n: int, out, index_base: int = 0) -> None:
        """First index of the largest of y[:n] (+ index_base) and its value -> out (8 bytes: int32, float32)."""
        check(lib().b200_argmax_f32(self.h, dev_ptr(y), n, index_base, dev_ptr(out)), "b200_argmax_f32")

    def capture_begin(self) -> None:
        check(lib().b200_capture_begin(self.h), "b200_capture_begin")

    def capture_end(self) -> "Graph":
        g = ctypes.c_void_p()
        check(lib().b200_capture_end(self.h, ctypes.byref(g)), "b200_capture_end")
        return Graph(self, g)

    def copy_async(self, dst: int, src: int, nbytes: int) -> None:
        check(lib().b200_copy_async(self.h, dst, src, nbytes), "b200_copy_async")

    def prefetch(self, W: QMat) -> None:
        check(lib().b200_prefetch(self.h, ctypes.byref(W.c)), "b200_prefetch")

    def _call(self, name: str, struct, values, kv: PagedKV | None = None, may_lack_kv: bool = False) -> None:
        """The C call of that name with an argument struct of `values`. Another thread's call waits: the interpreter's
        lock is given up while C reads the struct."""
        with self._lock:
            self._queue(name, struct, values, kv, may_lack_kv)

    def _queue(self, name: str, struct, values, kv: PagedKV | None, may_lack_kv: bool = False) -> None:
        kept = self._structs.get(name)
        if kept is None:               # the struct is one per engine, filled anew each time
            buf = bytearray(ctypes.sizeof(struct))
            fmt = Struct("".join(_FORMAT[t] for _, t in struct._fields_))
            c = struct.from_buffer(buf)
            kept = self._structs[name] = (getattr(lib(), name), ctypes.byref(c), fmt.pack_into, buf)
        fn, ref, pack, buf = kept
        pack(buf, 0, *values)
        rc = fn(self.h, kv.ref, ref) if kv is not None else fn(self.h, None, ref) if may_lack_kv else fn(self.h, ref)
        if rc < 0:
            check(rc, name)

    def kv_append(self, kv: PagedKV, k_new, v_new, offsets=None, seen=None, positions=None, weights=None,
                  lengths_out=None, seen_out=None) -> None:
        """New rows k_new, v_new [tokens, n_head_kv, head_dim] (the cache's type or float32) behind the slots in use:
        one row per sequence, or rows offsets[b]:offsets[b + 1] for sequence b. Their positions seen[b] + i (lengths
        where seen is None) and weights of 0 go into `positions` and `weights`. The lengths, and seen, are
        advanced: in lengths_out and seen_out, by default in place."""
        n = k_new.shape[0]
        st = rows(k_new, "k_new", (n, kv.n_head_kv, kv.head_dim))
        if (v_new.shape != k_new.shape or v_new.stride() != k_new.stride() or v_new.dtype is not k_new.dtype
                or not v_new.is_cuda):
            raise ValueError("k_new and v_new must be alike in shape, type and strides")
        pos, stride = (0, 0) if positions is None else kv.aux(positions, "int32", "positions")
        w, stride2 = (0, stride) if weights is None else kv.aux(weights, "float32", "weights")
        if pos and stride != stride2:
            raise ValueError("weights and positions must have one shape")
        b = (kv.batch,)
        self._call("b200_kv_append", capi.b200_kv_append_t, (
            k_new.data_ptr(), v_new.data_ptr(), dtype_code(k_new, "k_new"), n, st[0], st[1],
            address(offsets, "int32", "offsets", (kv.batch + 1,)), address(seen, "int32", "seen", b), pos, w, stride2,
            address(kv.lengths if lengths_out is None else lengths_out, "int32", "lengths_out", b),
            address(seen if seen_out is None else seen_out, "int32", "seen_out", b)), kv)

    def kv_attend(self, kv: PagedKV, q, out, lse=None, scale: float | None = None, weights=None, weights_out=None,
                  decay: float = 1.0) -> None:
        """out = softmax(scale q K^T) V for one token per sequence: q and out [batch, n_head, head_dim], lse float32
        [batch, n_head]; scale 1 / sqrt(head_dim) by default. With weights_out, the softmax's weights summed over
        the query heads of a cache head are added to decay * weights (None: zeros)."""
        if q.dim() != 3 or q.dtype is not out.dtype:
            raise ValueError("q and out must be [batch, n_head, head_dim] of one type")
        n_head = q.shape[1]
        shape = (kv.batch, n_head, kv.head_dim)
        qs, os_ = rows(q, "q", shape), rows(out, "out", shape)
        wo, stride = (0, 0) if weights_out is None else kv.aux(weights_out, "float32", "weights_out")
        w, stride2 = (0, stride) if weights is None else kv.aux(weights, "float32", "weights")
        if wo and stride != stride2:
            raise ValueError("weights and weights_out must have one shape")
        ws_bytes = kv.workspace.get((n_head, wo != 0))
        if ws_bytes is None:
            ws_bytes = kv.workspace[n_head, wo != 0] = int(lib().b200_kv_attend_workspace(kv.ref, n_head, int(wo != 0)))
        self._call_ws("b200_kv_attend", capi.b200_kv_attend_t, ws_bytes, (
            q.data_ptr(), out.data_ptr(), dtype_code(q, "q"), n_head, qs[0], qs[1], os_[0], os_[1],
            kv.head_dim ** -0.5 if scale is None else scale, address(lse, "float32", "lse", (kv.batch, n_head)),
            w, wo, stride2, decay), kv)

    def kv_attend_chunk(self, kv: PagedKV, q, out, offsets, lse=None, scale: float | None = None, window: int = 0) -> None:
        """out = softmax(scale q K^T) V for new tokens that are in the cache already, rows offsets[b]:offsets[b + 1] for
        the last slots in use of sequence b: q and out [tokens, n_head, head_dim], lse float32 [tokens, n_head]. Each
        sees the slots up to its own, with a window the last `window` of them."""
        if q.dim() != 3 or q.dtype is not out.dtype:
            raise ValueError("q and out must be [tokens, n_head, head_dim] of one type")
        n, n_head, _ = q.shape
        shape = (n, n_head, kv.head_dim)
        qs, os_ = rows(q, "q", shape), rows(out, "out", shape)
        code = dtype_code(q, "q")
        ws_bytes = kv.workspace.get(("chunk", code, n_head))
        if ws_bytes is None:
            ws_bytes = kv.workspace["chunk", code, n_head] = int(lib().b200_kv_chunk_workspace(kv.ref, code, n_head))
        self._call_ws("b200_kv_attend_chunk", capi.b200_kv_chunk_t, ws_bytes, (
            q.data_ptr(), out.data_ptr(), code, n, n_head, qs[0], qs[1], os_[0], os_[1],
            address(offsets, "int32", "offsets", (kv.batch + 1,)), kv.head_dim ** -0.5 if scale is None else scale,
            window, address(lse, "float32", "lse", (n, n_head))), kv)

    def _call_ws(self, name: str, struct, ws_bytes: int, values, kv: PagedKV) -> None:
        """_call with the engine's workspace, at least ws_bytes of it, behind the values."""
        with self._lock:
            if self._ws_bytes < ws_bytes:
                self._grow(ws_bytes)
            self._queue(name, struct, (*values, self._ws_at, ws_bytes), kv)
            if self._ws_old:           # this call waits for all that used them
                on = self._torch_stream()
                for ws in self._ws_old:
                    ws.record_stream(on)
                self._ws_old.clear()

    def _torch_stream(self):
        torch = _torch()
        dev = torch.device("cuda", self.device)
        return torch.cuda.ExternalStream(self.stream, device=dev) if self.stream else torch.cuda.default_stream(dev)

    def _grow(self, nbytes: int) -> None:
        """A larger workspace, device memory of this engine's own for calls on its stream, with an eighth to spare. The
        smaller one is given up after the next call, or lives on with the engine where a graph holds its address."""
        torch, on = _torch(), self._torch_stream()
        with torch.cuda.stream(on):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"attention needs a workspace of {nbytes} bytes, which cannot be allocated in a capture: "
                                   "make the call once before it is captured")
            ws = torch.empty(nbytes + nbytes // 8, dtype=torch.uint8, device=on.device)
        if self._ws is not None:
            (self._ws_recorded if lib().b200_engine_recorded(self.h) else self._ws_old).append(self._ws)
        self._ws, self._ws_at, self._ws_bytes = ws, ws.data_ptr(), ws.numel()

    def kv_evict(self, kv: PagedKV, weights, positions, seen, budget: int, recent: int = 0, sinks: int = 0,
                 weights_out=None, positions_out=None, lengths_out=None) -> None:
        """Cut every sequence and head to `budget` slots: the `recent` newest of `seen` tokens, the first `sinks` and
        the largest weights stay. Rows move inside the cache, whose pages in use must all be there; weights, positions
        and lengths go to the outputs, by default in place."""
        w, stride = kv.aux(weights, "float32", "weights")
        wo, s1 = (w, stride) if weights_out is None else kv.aux(weights_out, "float32", "weights_out")
        p, s2 = kv.aux(positions, "int32", "positions")
        po, s3 = (p, s2) if positions_out is None else kv.aux(positions_out, "int32", "positions_out")
        if not stride == s1 == s2 == s3:
            raise ValueError("weights and positions must have one shape")
        b = (kv.batch,)
        self._call("b200_kv_evict", capi.b200_kv_evict_t, (
            w, wo, p, po, stride, address(seen, "int32", "seen", b),
            address(kv.lengths if lengths_out is None else lengths_out, "int32", "lengths_out", b), budget, recent,
            sinks), kv)

    def kv_plan(self, kv: PagedKV, new, held, free, free_count, offsets, slots=None, positions=None, sequences=None,
                granted=None, seen=None, lengths_out=None, held_out=None, free_count_out=None, seen_out=None) -> None:
        """Pages for new[b] tokens (int32 [batch], negative: the sequence is done) behind the slots in use: table rows of
        which held[b] columns are in use, and a stack of free pages, free[:free_count]. All or nothing for a sequence.
        Written are offsets [batch + 1], the tokens of each sequence; per token its slot in the pool (int64, -1: none), its
        position and its sequence (int32 [tokens]); granted, the tokens that got slots; and held, free_count, lengths
        and seen, by default in place."""
        n, b = None, (kv.batch,)
        for t in (slots, positions, sequences):
            if t is not None:
                if n is not None and t.shape != n:
                    raise ValueError("slots, positions and sequences must have one length")
                n = t.shape
        if n is not None and len(n) != 1:
            raise ValueError("slots, positions and sequences must be [tokens]")
        if free.dim() != 1:
            raise ValueError("free must be [pages]")
        self._call("b200_kv_plan", capi.b200_kv_plan_t, (
            address(new, "int32", "new", b), address(held, "int32", "held", b),
            address(held if held_out is None else held_out, "int32", "held_out", b),
            address(free, "int32", "free", free.shape), free.shape[0], address(free_count, "int32", "free_count", (1,)),
            address(free_count if free_count_out is None else free_count_out, "int32", "free_count_out", (1,)),
            address(offsets, "int32", "offsets", (kv.batch + 1,)), (0x7fffffff if n is None else n[0]),
            address(slots, "int64", "slots", n), address(positions, "int32", "positions", n),
            address(sequences, "int32", "sequences", n), address(granted, "int32", "granted", b),
            address(seen, "int32", "seen", b), address(seen if seen_out is None else seen_out, "int32", "seen_out", b),
            address(kv.lengths if lengths_out is None else lengths_out, "int32", "lengths_out", b)), kv)

    def rope(self, positions, freqs, q=None, q_out=None, k=None, k_out=None, interleaved: bool = False, mscale: float = 1.0,
             kv: PagedKV | None = None, v=None, slots=None) -> None:
        """Rotary positions (int32 [tokens]) for q [tokens, n_head, head_dim] and k [tokens, n_head_kv, head_dim], with the
        frequencies of rope_freqs on the device: to q_out and k_out, by default in place. With a cache, k's rows go to
        its rows slots[t] (int64, -1: nowhere) instead, and v's beside them."""
        some = k if q is None else q
        if some is None or some.dim() != 3:
            raise ValueError("q or k must be [tokens, heads, head_dim]")
        n, heads, d = some.shape
        code = dtype_code(some, "q")
        zero = (0, 0)
        qp = qo = h = kp = ko = hkv = vp = 0
        qs = qos = ks = kos = vs = zero
        out_code = code
        if q is not None:
            q_out = q if q_out is None else q_out
            h, qs, qos = heads, rows(q, "q", q.shape), rows(q_out, "q_out", q.shape)
            qp, qo, out_code = q.data_ptr(), q_out.data_ptr(), dtype_code(q_out, "q_out")
        if k is not None:
            if k.dim() != 3 or dtype_code(k, "k") != code:
                raise ValueError("k must be [tokens, n_head_kv, head_dim], of q's type")
            hkv = k.shape[1]
            kp, ks = k.data_ptr(), rows(k, "k", (n, hkv, d))
            if kv is None:
                k_out = k if k_out is None else k_out
                ko, kos = k_out.data_ptr(), rows(k_out, "k_out", k.shape)
                if q is not None and dtype_code(k_out, "k_out") != out_code:
                    raise ValueError("q_out and k_out must be of one type")
                out_code = dtype_code(k_out, "k_out")
        if kv is None and (v is not None or slots is not None):
            raise ValueError("v and slots need a cache")
        if v is not None:
            if k is None or v.dtype is not k.dtype:
                raise ValueError("v must be of k's type")
            vp, vs = v.data_ptr(), rows(v, "v", k.shape)
        if freqs.dim() != 1:
            raise ValueError("freqs must be [rot_dim / 2]")
        self._call("b200_rope", capi.b200_rope_t, (
            qp, qo, h, *qs, *qos, kp, ko, hkv, *ks, *kos, vp, *vs, code, out_code, n, d, 2 * freqs.shape[0], int(interleaved),
            address(positions, "int32", "positions", (n,)), address(freqs, "int64", "freqs", freqs.shape), mscale,
            address(slots, "int64", "slots", (n,))), kv, True)

    def rms_norm(self, x, weight, out=None, eps: float = 1e-5, residual=None, residual_out=None, q8=None) -> None:
        """r = residual + x (x alone without one), y = r / sqrt(mean(r^2) + eps) * weight (float32) for rows x [n, k]: r to
        residual_out, by default in place, y to out and, as Q8_0 rows that gemv_q8 reads, to q8 (uint8 [n, k + k / 8])."""
        if x.dim() != 2:
            raise ValueError("x must be [rows, k]")
        n, k = shape = x.shape
        code = dtype_code(x, "x")
        rp = ro = op = qp = rs = ros = os_ = qs = 0
        r_code = o_code = code
        xs = row_stride(x, "x", shape)
        if residual is not None:
            residual_out = residual if residual_out is None else residual_out
            if residual_out.dtype is not residual.dtype:
                raise ValueError("residual and residual_out must be of one type")
            rp, rs, r_code = residual.data_ptr(), row_stride(residual, "residual", shape), dtype_code(residual, "residual")
            ro, ros = residual_out.data_ptr(), row_stride(residual_out, "residual_out", shape)
        elif residual_out is not None:
            raise ValueError("residual_out without residual")
        if out is not None:
            op, os_, o_code = out.data_ptr(), row_stride(out, "out", shape), dtype_code(out, "out")
        if q8 is not None:
            if q8.element_size() != 1:
                raise ValueError("q8 must be bytes")
            qp, qs = q8.data_ptr(), row_stride(q8, "q8", (n, k + k // 8))
        self._call("b200_rms_norm", capi.b200_rms_norm_t, (
            x.data_ptr(), code, rp, ro, r_code, address(weight, "float32", "weight", (k,)), op, o_code, qp, n, k, xs, rs, ros,
            os_, qs, eps))

    def sample(self, logits, u, token, logprob=None, temperature=None, top_k=None, top_p=None, min_p=None) -> None:
        """token int32 [batch] (and the log of its probability) drawn from logits [batch, n_vocab] with the uniform
        numbers u float32 [batch]; temperature, top_p and min_p float32 [batch], top_k int32 [batch], None: off."""
        if logits.dim() != 2 or not logits.is_cuda or (logits.shape[1] > 1 and logits.stride(1) != 1):
            raise ValueError("logits must be a CUDA tensor [batch, n_vocab] with contiguous rows")
        n, vocab = logits.shape
        b = (n,)
        self._call("b200_sample", capi.b200_sample_t, (
            logits.data_ptr(), dtype_code(logits, "logits"), n, vocab, logits.stride(0),
            address(temperature, "float32", "temperature", b), address(top_k, "int32", "top_k", b),
            address(top_p, "float32", "top_p", b), address(min_p, "float32", "min_p", b), address(u, "float32", "u", b),
            address(token, "int32", "token", b), address(logprob, "float32", "logprob", b)))

    def sync(self, timeout_ms: int = 10000) -> None:
        check(lib().b200_engine_sync(self.h, timeout_ms), "b200_engine_sync")

    def status(self) -> int:
        s = ctypes.c_uint(0)
        check(lib().b200_engine_status(self.h, ctypes.byref(s)), "b200_engine_status")
        return int(s.value)

    def plan(self, rows: int, k: int, fused_f32: bool = False, layout: int = LAYOUT_TILES) -> tuple[int, int]:
        g, sm = ctypes.c_int(0), ctypes.c_int(0)
        check(lib().b200_gemv_plan(self.h, rows, k, layout, int(fused_f32), ctypes.byref(g), ctypes.byref(sm)),
              "b200_gemv_plan")
        return g.value, sm.value


class Graph:
    """A captured sequence of engine calls (b200_graph_t)."""

    def __init__(self, engine: Engine, handle):
        self.engine, self.h = engine, handle

    def launch(self) -> None:
        check(lib().b200_graph_launch(self.engine.h, self.h), "b200_graph_launch")

    def close(self) -> None:
        if self.h:
            lib().b200_graph_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class GemvDev:
    """gemv_dev.h: the reference's gemv_q4_0 engine interface (board/kv260gemv/gemv_dev.h)."""

    def __init__(self, name: str = "gemv_q4_0", quiet: bool = False):
        self.d = capi.gemv_dev_t()
        if lib().gemv_dev_open_named(ctypes.byref(self.d), name.encode(), int(quiet)) != 0:
            raise capi.B200Error(f"gemv_dev_open_named({name})", -1)

    def set_stream(self, stream: int | None) -> None:
        check(lib().gemv_dev_set_stream(ctypes.byref(self.d), stream), "gemv_dev_set_stream")

    def run(self, w: int, x: int, y: int, k: int, rows: int) -> None:
        check(lib().gemv_dev_run(ctypes.byref(self.d), w, x, y, k, rows), "gemv_dev_run")

    def start(self, w: int, x: int, y: int, k: int, rows: int) -> None:
        check(lib().gemv_dev_start(ctypes.byref(self.d), w, x, y, k, rows), "gemv_dev_start")

    def start4(self, w4, x: int, y: int, k: int, rows: int) -> None:
        arr = (ctypes.c_uint64 * 4)(*w4)
        check(lib().gemv_dev_start4(ctypes.byref(self.d), arr, x, y, k, rows), "gemv_dev_start4")

    def wait(self) -> None:
        check(lib().gemv_dev_wait(ctypes.byref(self.d)), "gemv_dev_wait")

    def close(self) -> None:
        lib().gemv_dev_close(ctypes.byref(self.d))


class Gemv2Dev:
    """gemv2_dev.h: fetch (L2 prefetch) + mac (GEMV) over the chunk-pair layout."""

    def __init__(self):
        self.d = capi.gemv2_dev_t()
        if lib().gemv2_dev_open(ctypes.byref(self.d)) != 0:
            raise capi.B200Error("gemv2_dev_open", -1)

    def fetch_start(self, w4, k: int, rows: int) -> None:
        arr = (ctypes.c_uint64 * 4)(*w4)
        check(lib().gemv2_fetch_start(ctypes.byref(self.d), arr, k, rows), "gemv2_fetch_start")

    def mac_start(self, x: int, y: int, k: int, rows: int) -> None:
        check(lib().gemv2_mac_start(ctypes.byref(self.d), x, y, k, rows), "gemv2_mac_start")

    def mac_wait(self) -> None:
        check(lib().gemv2_mac_wait(ctypes.byref(self.d)), "gemv2_mac_wait")

    def mac_idle(self) -> bool:
        return check(lib().gemv2_mac_idle(ctypes.byref(self.d)), "gemv2_mac_idle") == 1

    def drain(self) -> None:
        check(lib().gemv2_drain(ctypes.byref(self.d)), "gemv2_drain")

    def close(self) -> None:
        lib().gemv2_dev_close(ctypes.byref(self.d))


class Udmabuf:
    """udmabuf.h: device pool with a pinned host mirror (clean = H2D, invalidate = D2H)."""

    def __init__(self, name: str = "udmabuf0", size: int | None = None, device: int = 0):
        self.b = capi.udmabuf_t()
        if size is None:
            rc = lib().udmabuf_open(ctypes.byref(self.b), name.encode())
        else:
            rc = lib().udmabuf_open_size(ctypes.byref(self.b), name.encode(), size, device)
        if rc != 0:
            raise capi.B200Error(f"udmabuf_open({name})", rc)

    def alloc(self, size: int, align: int = 4096) -> int:
        """Host-mirror address of a new allocation (0 when the pool is full)."""
        return int(lib().udmabuf_alloc(ctypes.byref(self.b), size, align) or 0)

    def phys(self, host_addr: int) -> int:
        base = ctypes.cast(self.b.base, ctypes.c_void_p).value
        return self.b.phys + (host_addr - base)

    def view(self, host_addr: int, nbytes: int):
        """numpy uint8 view of the host mirror."""
        import numpy as np
        return np.ctypeslib.as_array((ctypes.c_uint8 * nbytes).from_address(host_addr))

    @staticmethod
    def clean(host_addr: int, nbytes: int) -> None:
        check(lib().udmabuf_clean(host_addr, nbytes), "udmabuf_clean")

    @staticmethod
    def invalidate(host_addr: int, nbytes: int) -> None:
        check(lib().udmabuf_invalidate(host_addr, nbytes), "udmabuf_invalidate")

    def close(self) -> None:
        lib().udmabuf_close(ctypes.byref(self.b))
