"""A paged key-value cache as the serving calls take it (b200_kv_t,
include/b200_engine.h): Engine.kv_append, kv_attend and kv_evict."""

from __future__ import annotations

import ctypes

from . import capi

_CODES: dict = {}          # torch dtype -> B200_F32, B200_F16, B200_BF16


def codes() -> dict:
    if not _CODES:
        import torch
        _CODES.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
        _CODES["int32"], _CODES["float32"] = torch.int32, torch.float32
    return _CODES


def dtype_code(t, name: str) -> int:
    code = (_CODES or codes()).get(t.dtype)
    if code is None:
        raise ValueError(f"{name} must be float32, float16 or bfloat16, not {t.dtype}")
    return code


def address(t, dtype: str, name: str, shape) -> int:
    """Device address of a contiguous CUDA tensor of that type ("int32" or "float32") and shape; 0 for None."""
    if t is None:
        return 0
    want = (_CODES or codes())[dtype]
    if t.dtype is want and t.is_cuda and t.shape == shape and t.is_contiguous():
        return t.data_ptr()
    if not t.is_cuda or t.dtype is not want:
        raise ValueError(f"{name} must be a CUDA {dtype} tensor")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {shape}, not {tuple(t.shape)}")
    raise ValueError(f"{name} must be contiguous")


def rows(t, name: str, shape) -> tuple[int, int]:
    """Strides of a tensor's first two dimensions, its last one contiguous."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {shape}, not {tuple(t.shape)}")
    s0, s1, s2 = t.stride()
    if s2 != 1 and shape[2] != 1:
        raise ValueError(f"{name}: a row must be contiguous")
    return s0, s1


class PagedKV:
    """Pools k and v, [n_pages, n_head_kv, page_size, head_dim] views of one
    type and the same strides, rows contiguous; table int32 [batch, columns],
    the pages of each sequence; lengths int32 [batch], its slots in use.

    The object holds the tensors, and reads nothing of them itself: a caller
    fills the table as it hands pages out, and the calls advance or cut the
    lengths."""

    def __init__(self, k, v, table, lengths):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.stride() != v.stride():
            raise ValueError("k and v must be [n_pages, n_head_kv, page_size, head_dim] alike in type and strides")
        if not (k.is_cuda and v.is_cuda):
            raise ValueError("k and v must be CUDA tensors")
        if k.stride(3) != 1:
            raise ValueError("a cache row must be contiguous")
        if not table.is_cuda or table.dtype is not codes()["int32"]:
            raise ValueError("table must be a CUDA int32 tensor")
        if table.dim() != 2 or (table.shape[1] > 1 and table.stride(1) != 1):
            raise ValueError("table must be [batch, columns] with contiguous rows")
        at = address(lengths, "int32", "lengths", (table.shape[0],))
        self.k, self.v, self.table, self.lengths = k, v, table, lengths
        self.n_pages, self.n_head_kv, self.page_size, self.head_dim = k.shape
        self.batch, cols = table.shape
        self.capacity = cols * self.page_size
        st = k.stride()
        self.c = capi.b200_kv_t(k.data_ptr(), v.data_ptr(), dtype_code(k, "k"), self.n_pages, self.page_size,
                                self.n_head_kv, self.head_dim, st[0], st[1], st[2], table.data_ptr(),
                                max(table.stride(0), cols), cols, at, self.batch)
        self.ref = ctypes.byref(self.c)
        self.workspace: dict = {}     # bytes that kv_attend needs, by (query heads, with weights)

    def aux(self, t, dtype: str, name: str) -> tuple[int, int]:
        """Address and head stride of a [batch, n_head_kv, >= capacity] tensor beside the cache (weights, positions)."""
        shape = t.shape
        if len(shape) != 3 or shape[2] < self.capacity:
            raise ValueError(f"{name} must be [{self.batch}, {self.n_head_kv}, >= {self.capacity}]")
        return address(t, dtype, name, (self.batch, self.n_head_kv, shape[2])), shape[2]
