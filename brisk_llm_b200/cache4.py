"""The paged key/value cache in 4 bits over device tensors: append, attention and read of include/brisk_cuda.h.

    cache = PagedCache.allocate(pages=512, kv_heads=8, head_dim=128)       # one layer's pool of pages
    rotary = Rotary(128, base=1e6, layout="half", device="cuda")           # once
    batch = Batch(context, tokens, page_table=table, query_start=starts, max_tokens=512, max_length=4096)
    q = cache.append(batch, q, k, v, rotary=rotary, q_norm=wq, k_norm=wk)   # norms, rotates, stores
    out = cache.attention(batch, q)

Tensors are torch tensors on the cache's device; work goes to that device's current stream and nothing here synchronises. What does
not fit together raises RuntimeError("cuda: ...") before anything is launched. A batch's context, page_table and query_start are
read on the device when the work runs: a captured call that is replayed sees what they hold then.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import abi

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
_ERR = 512


def _fail(message: str):
    raise RuntimeError("cuda: " + message)


class Rotary:
    """Rotation of the leading `width` values of a head (0: all of it). layout: "half" pairs value i with i + width / 2, "adjacent" 2 i with
    2 i + 1. The angle of pair i at position p is p * scale * base^(-2 i / width) / factors[i]; cos and sin are multiplied by
    attn_factor (brisk-llm src/model.cpp:880-892)."""

    def __init__(self, head_dim: int, base: float, layout: str = "half", width: int = 0, scale: float = 1.0, factors=None,
                 attn_factor: float = 1.0, device="cuda"):
        if layout not in ("half", "adjacent"):
            _fail("a rotation's layout is 'half' or 'adjacent'")
        self.width = width or head_dim
        if self.width > head_dim or self.width % 2:
            _fail("the rotated width must be even and at most the head size")
        self.adjacent, self.attn_factor = int(layout == "adjacent"), float(attn_factor)
        divisors = None
        if factors is not None:
            factors = torch.as_tensor(factors, dtype=torch.float32).cpu().contiguous()
            if factors.numel() != self.width // 2:
                _fail("rope factor count must be half the rotated width")
            divisors = C.cast(factors.data_ptr(), C.POINTER(C.c_float))
        turns = torch.empty(self.width // 2, dtype=torch.float64)
        err = C.create_string_buffer(_ERR)
        if abi.load_library().brisk_cuda_rope_turns(self.width, base, scale, divisors, C.cast(turns.data_ptr(), C.POINTER(C.c_double)), err, _ERR) != 0:
            raise RuntimeError(err.value.decode())
        self.turns = turns.to(device)


def _index(t, device, shape, what):
    if t.dtype != torch.int32 or t.device != device or not t.is_contiguous() or tuple(t.shape) != tuple(shape):
        _fail(f"{what} must be a contiguous int32 tensor of shape {tuple(shape)} on {device}")
    return t.data_ptr()


class Batch:
    """Tokens of several sequences one behind the other: token i of sequence s is row query_start[s] + i and stands at position
    context[s] + i. Without query_start every sequence has tokens / sequences of them; without a page_table column c of
    sequence s is page s * columns + c. max_tokens and max_length bound a sequence's tokens and its positions with them."""

    def __init__(self, context, tokens: int, page_table=None, query_start=None, columns: int = 0, max_tokens: int = 0, max_length: int = 0):
        self.context, self.page_table, self.query_start, self.device = context, page_table, query_start, context.device
        if context.device.type != "cuda" or context.dim() != 1:
            _fail("context must be a vector on a CUDA device")
        n = context.shape[0]
        s = self.c = abi.Cache4Batch()
        s.context = _index(context, self.device, (n,), "context")
        if page_table is not None:
            if page_table.dim() != 2:
                _fail("page_table must be [sequences, columns]")
            columns = page_table.shape[1]
            s.page_table = _index(page_table, self.device, (n, columns), "page_table")
        if query_start is not None:
            s.query_start = _index(query_start, self.device, (n + 1,), "query_start")
        for name, value in (("tokens", tokens), ("columns", columns), ("max_tokens", max_tokens), ("max_length", max_length)):
            if not 0 <= value <= 0x7fffffff:
                _fail(f"{name} must be from 0 to 2^31 - 1")
        s.sequences, s.table_columns, s.tokens, s.max_tokens, s.max_length = n, columns, tokens, max_tokens, max_length
        self.tokens = tokens


class PagedCache:
    """One layer's pool of pages: k_quants and v_quants [pages, kv_heads, page_size, head_dim / 2] bytes, k_scales and v_scales
    [pages, kv_heads, page_size, head_dim / 32] f16."""

    def __init__(self, k_quants, k_scales, v_quants, v_scales):
        if k_quants.dim() != 4 or k_quants.device.type != "cuda":
            _fail("the planes of a 4-bit cache are [pages, kv_heads, page_size, ...] on a CUDA device")
        pages, kv_heads, page_size, half = k_quants.shape
        self.device, self.kv_heads, self.head_dim, self.page_size, self.pages = k_quants.device, kv_heads, 2 * half, page_size, pages
        for name, t, dtype, last in (("k_quants", k_quants, torch.uint8, half), ("v_quants", v_quants, torch.uint8, half),
                                     ("k_scales", k_scales, torch.float16, half // 16), ("v_scales", v_scales, torch.float16, half // 16)):
            if t.dtype != dtype or t.device != self.device or tuple(t.shape) != (pages, kv_heads, page_size, last) or not t.is_contiguous():
                _fail(f"{name} must be a contiguous {dtype} tensor of shape {(pages, kv_heads, page_size, last)} on {self.device}")
        self.k_quants, self.k_scales, self.v_quants, self.v_scales = k_quants, k_scales, v_quants, v_scales
        self.c = abi.Cache4(k_quants.data_ptr(), k_scales.data_ptr(), v_quants.data_ptr(), v_scales.data_ptr(), pages, page_size, kv_heads, self.head_dim)
        self._lib = abi.load_library()

    @classmethod
    def allocate(cls, pages: int, kv_heads: int, head_dim: int, page_size: int = 64, device="cuda"):
        """Pages of zeros."""
        def plane(last, dtype):
            return torch.zeros((pages, kv_heads, page_size, last), dtype=dtype, device=device)

        return cls(plane(head_dim // 2, torch.uint8), plane(head_dim // 32, torch.float16), plane(head_dim // 2, torch.uint8),
                   plane(head_dim // 32, torch.float16))

    def _rows(self, t, batch, heads, what, dtype=None):
        """[tokens, heads, head_dim] with any stride between tokens; returns it."""
        if t.dim() != 3 or t.shape[0] != batch.tokens or (heads and t.shape[1] != heads) or t.shape[2] != self.head_dim or t.device != self.device:
            _fail(f"{what} must be [{batch.tokens}, {heads or 'heads'}, {self.head_dim}] on {self.device}")
        if (dtype is not None and t.dtype != dtype) or t.dtype not in _TYPES:
            _fail(f"{what} must be {dtype or 'float32, float16 or bfloat16'}")
        if t.shape[0] and (t.stride(2) != 1 or (t.shape[1] > 1 and t.stride(1) != self.head_dim) or (t.shape[0] > 1 and t.stride(0) < t.shape[1] * self.head_dim)):
            _fail(f"the heads of a token must lie side by side in {what}")
        return t

    @staticmethod
    def _stride(t):
        return max(t.stride(0), t.shape[1] * t.shape[2])  # of a single row any stride will do

    def _vector(self, t, n, what):
        if t is None:
            return None
        if t.dtype != torch.float32 or t.device != self.device or t.numel() != n or not t.is_contiguous():
            _fail(f"{what} must be {n} contiguous float32 values on {self.device}")
        return t.data_ptr()

    def _call(self, fn, *args):
        err = C.create_string_buffer(_ERR)
        index = self.device.index
        if torch.cuda.current_device() == index:
            rc = fn(self.c, *args, torch.cuda.current_stream(index).cuda_stream, err, _ERR)
        else:
            with torch.cuda.device(index):
                rc = fn(self.c, *args, torch.cuda.current_stream(index).cuda_stream, err, _ERR)
        if rc != 0:
            raise RuntimeError(err.value.decode())

    def _check(self, batch):
        if batch.device != self.device:
            _fail(f"the batch is on {batch.device}, the cache on {self.device}")

    def append(self, batch: Batch, q, k, v, rotary: Rotary | None = None, q_norm=None, k_norm=None, eps: float = 1e-6, q_bias=None, k_bias=None,
               v_bias=None, out=None):
        """Stores the batch's keys and values at their positions and returns its queries: biased, each head over its root mean square times
        its norm, rotated (the values only biased). q may be None: keys and values only. out may be q."""
        self._check(batch)
        dtype, kv, dim = k.dtype, self.kv_heads, self.head_dim
        self._rows(k, batch, kv, "k")
        self._rows(v, batch, kv, "v", dtype)
        r = abi.Cache4Rows()
        r.k, r.v, r.k_stride, r.v_stride = k.data_ptr(), v.data_ptr(), self._stride(k), self._stride(v)
        if q is not None:
            heads = self._rows(q, batch, 0, "q", dtype).shape[1]
            if out is None:
                out = torch.empty((batch.tokens, heads, dim), dtype=dtype, device=self.device)
            self._rows(out, batch, heads, "out", dtype)
            r.heads, r.q, r.q_out, r.q_stride, r.q_out_stride = heads, q.data_ptr(), out.data_ptr(), self._stride(q), self._stride(out)
            r.q_norm, r.q_bias = self._vector(q_norm, dim, "q_norm"), self._vector(q_bias, heads * dim, "q_bias")
        r.k_norm, r.k_bias, r.v_bias = self._vector(k_norm, dim, "k_norm"), self._vector(k_bias, kv * dim, "k_bias"), self._vector(v_bias, kv * dim, "v_bias")
        if rotary is not None:
            if rotary.turns.device != self.device:
                _fail(f"the rotation is on {rotary.turns.device}, the cache on {self.device}")
            r.rope_turns, r.rope_dim, r.rope_adjacent, r.rope_attn_factor = rotary.turns.data_ptr(), rotary.width, rotary.adjacent, rotary.attn_factor
        r.eps, r.type = eps, _TYPES[dtype]
        self._call(self._lib.brisk_cuda_cache4_append, batch.c, r)
        return out

    def attention(self, batch: Batch, q, scale: float = 0.0, window: int = 0, out=None):
        """softmax(scale * q k) v of every row over the positions it sees: up to its own, with a window the last `window` of them. scale 0:
        1 / sqrt(head_dim). Rows behind the last sequence's stay as they are in `out` (unset, where it is made here)."""
        self._check(batch)
        heads = self._rows(q, batch, 0, "q").shape[1]
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=self.device)
        self._rows(out, batch, heads, "out", q.dtype)
        if not 0 <= window <= 0x7fffffff:
            _fail("a window is from 0 to 2^31 - 1 positions")
        self._call(self._lib.brisk_cuda_cache4_attention, batch.c, _TYPES[q.dtype], q.data_ptr(), out.data_ptr(), self._stride(q), self._stride(out), heads,
                   scale, window)
        return out

    def read(self, batch: Batch, dtype=torch.float32, k_out=None, v_out=None):
        """The stored rows at the positions of the batch's tokens, as values: two tensors [tokens, kv_heads, head_dim]."""
        self._check(batch)
        if dtype not in _TYPES:
            _fail("a cache is read as float32, float16 or bfloat16")
        outs = []
        for t, what in ((k_out, "k_out"), (v_out, "v_out")):
            t = torch.empty((batch.tokens, self.kv_heads, self.head_dim), dtype=dtype, device=self.device) if t is None else t
            outs.append(self._rows(t, batch, self.kv_heads, what, dtype))
        k, v = outs
        self._call(self._lib.brisk_cuda_cache4_read, batch.c, _TYPES[dtype], k.data_ptr(), v.data_ptr(), self._stride(k), self._stride(v))
        return k, v
