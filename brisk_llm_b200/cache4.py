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
import math
import threading

import torch

from . import abi

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
_ERR = 512
_thread = threading.local()  # a buffer for messages, made once: a call's host part is a third of the shortest calls' time as it is
_device, _stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


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
        if self.attn_factor == 0.0 or not math.isfinite(self.attn_factor):
            _fail("a rotation's factor on cos and sin must be finite and not 0")
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
        self.ref = C.byref(s)


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
        self._lib, self._ref = abi.load_library(), C.byref(self.c)

    @classmethod
    def allocate(cls, pages: int, kv_heads: int, head_dim: int, page_size: int = 64, device="cuda"):
        """Pages of zeros."""
        def plane(last, dtype):
            return torch.zeros((pages, kv_heads, page_size, last), dtype=dtype, device=device)

        return cls(plane(head_dim // 2, torch.uint8), plane(head_dim // 32, torch.float16), plane(head_dim // 2, torch.uint8),
                   plane(head_dim // 32, torch.float16))

    def _rows(self, t, tokens, heads, what, dtype):
        """Checks [tokens, heads, head_dim] (heads 0: any number) with any stride between tokens; returns heads and that stride."""
        shape, dim = t.shape, self.head_dim
        if len(shape) != 3 or shape[0] != tokens or shape[2] != dim or (heads and shape[1] != heads) or t.device != self.device:
            _fail(f"{what} must be [{tokens}, {heads or 'heads'}, {dim}] on {self.device}")
        if t.dtype != dtype:
            _fail(f"{what} must be {dtype}")
        heads = shape[1]
        outer, middle, inner = t.stride()
        if tokens and (inner != 1 or (middle != dim and heads > 1) or (outer < heads * dim and tokens > 1)):
            _fail(f"the heads of a token must lie side by side in {what}")
        return heads, max(outer, heads * dim)  # of a single row any stride will do

    def _vector(self, t, n, what):
        if t is None:
            return None
        if t.dtype != torch.float32 or t.device != self.device or t.numel() != n or not t.is_contiguous():
            _fail(f"{what} must be {n} contiguous float32 values on {self.device}")
        return t.data_ptr()

    def _type(self, batch, t, what):
        if batch.device != self.device:
            _fail(f"the batch is on {batch.device}, the cache on {self.device}")
        number = _TYPES.get(t.dtype)
        if number is None:
            _fail(f"{what} must be float32, float16 or bfloat16")
        return number

    def _call(self, fn, *args):
        try:
            err = _thread.err
        except AttributeError:
            err = _thread.err = C.create_string_buffer(_ERR)
        index = self.device.index
        if _device() == index:
            rc = fn(self._ref, *args, _stream(index), err, _ERR)
        else:
            with torch.cuda.device(index):
                rc = fn(self._ref, *args, _stream(index), err, _ERR)
        if rc != 0:
            raise RuntimeError(err.value.decode())

    def append(self, batch: Batch, q, k, v, rotary: Rotary | None = None, q_norm=None, k_norm=None, eps: float = 1e-6, q_bias=None, k_bias=None,
               v_bias=None, out=None):
        """Stores the batch's keys and values at their positions and returns its queries: biased, each head over its root mean square times
        its norm, rotated (the values only biased). q may be None: keys and values only. out may be q."""
        kind, dtype, n, kv, dim = self._type(batch, k, "k"), k.dtype, batch.tokens, self.kv_heads, self.head_dim
        _, k_stride = self._rows(k, n, kv, "k", dtype)
        _, v_stride = self._rows(v, n, kv, "v", dtype)
        heads = q_stride = out_stride = 0
        q_at = out_at = q_bias_at = q_norm_at = turns = None
        if q is not None:
            heads, q_stride = self._rows(q, n, 0, "q", dtype)
            if out is None:
                out = q.new_empty((n, heads, dim))
            _, out_stride = self._rows(out, n, heads, "out", dtype)
            q_at, out_at = q.data_ptr(), out.data_ptr()
            q_norm_at, q_bias_at = self._vector(q_norm, dim, "q_norm"), self._vector(q_bias, heads * dim, "q_bias")
        width = adjacent = 0
        factor = 1.0
        if rotary is not None:
            if rotary.turns.device != self.device or rotary.width > dim:
                _fail(f"the rotation is of {rotary.width} values on {rotary.turns.device}, the cache's heads of {dim} on {self.device}")
            turns, width, adjacent, factor = rotary.turns.data_ptr(), rotary.width, rotary.adjacent, rotary.attn_factor
        rows = abi.Cache4Rows(q_at, k.data_ptr(), v.data_ptr(), out_at, q_stride, k_stride, v_stride, out_stride, q_bias_at,
                              self._vector(k_bias, kv * dim, "k_bias"), self._vector(v_bias, kv * dim, "v_bias"), q_norm_at,
                              self._vector(k_norm, dim, "k_norm"), turns, width, adjacent, factor, eps, heads, kind)
        self._call(self._lib.brisk_cuda_cache4_append, batch.ref, C.byref(rows))
        return out

    def attention(self, batch: Batch, q, scale: float = 0.0, window: int = 0, out=None):
        """softmax(scale * q k) v of every row over the positions it sees: up to its own, with a window the last `window` of them. scale 0:
        1 / sqrt(head_dim). Rows behind the last sequence's stay as they are in `out` (unset, where it is made here)."""
        kind = self._type(batch, q, "q")
        heads, q_stride = self._rows(q, batch.tokens, 0, "q", q.dtype)
        if out is None:
            out = q.new_empty(q.shape)
        _, out_stride = self._rows(out, batch.tokens, heads, "out", q.dtype)
        if not 0 <= window <= 0x7fffffff:
            _fail("a window is from 0 to 2^31 - 1 positions")
        self._call(self._lib.brisk_cuda_cache4_attention, batch.ref, kind, q.data_ptr(), out.data_ptr(), q_stride, out_stride, heads, scale, window)
        return out

    def read(self, batch: Batch, dtype=torch.float32, k_out=None, v_out=None):
        """The stored rows at the positions of the batch's tokens, as values: two tensors [tokens, kv_heads, head_dim]."""
        if dtype not in _TYPES:
            _fail("a cache is read as float32, float16 or bfloat16")
        shape = (batch.tokens, self.kv_heads, self.head_dim)
        k = torch.empty(shape, dtype=dtype, device=self.device) if k_out is None else k_out
        v = torch.empty(shape, dtype=dtype, device=self.device) if v_out is None else v_out
        kind = self._type(batch, k, "k_out")
        _, k_stride = self._rows(k, batch.tokens, self.kv_heads, "k_out", dtype)
        _, v_stride = self._rows(v, batch.tokens, self.kv_heads, "v_out", dtype)
        self._call(self._lib.brisk_cuda_cache4_read, batch.ref, kind, k.data_ptr(), v.data_ptr(), k_stride, v_stride)
        return k, v
