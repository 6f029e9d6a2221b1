"""The operators of a decoder layer with 8-bit floating-point weights (include/transmuter_hip.h, "decoder
layers in 8-bit floating point", and "drafted steps and sampling"): the residual's addition and the root-mean-square
norm, rows in 8 bits, the 8-bit product, a paged cache of keys and values with the attentions that read it, and tokens
drawn from logits.

Rows in 8 bits (`Rows8`) are f8_e4m3fn values with one f32 scale for each block of 128 columns. Every call is
asynchronous on `stream` (None: the context's); its operands must stay until its work is done. A call's answer is new
device memory, or `out`, of the same shapes and types, which a step that is recorded into a graph has to give
(nothing can be allocated there). No reference counterpart: the reference's norms and attention stay on the Nx backend.
"""

from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import numpy as np

from . import _lib
from ._lib import PagedCacheDesc, TmhArgumentError, lib
from .device import FLOAT_TYPES, NX_TO_NUMPY, NX_TO_TMH, Context, DeviceTensor

BLOCK = 128  # columns of a row, and of K in a weight, that share a scale


def _refuse(message: str):
    raise TmhArgumentError(_lib.ERR_INVALID, message)


def _rows(x: DeviceTensor, what: str) -> tuple[int, int]:
    if x.dtype not in FLOAT_TYPES:
        _refuse(f"{what} takes f32, f16 or bf16 rows, got {x.dtype}")
    if not x.shape:
        _refuse(f"{what} takes rows, got a scalar")
    return math.prod(x.shape[:-1]), x.shape[-1]


def _at(t: DeviceTensor, elements: int) -> ctypes.c_void_p:
    """The address of an element of t (NULL in a tensor of no bytes)."""
    if t.ptr is None or t.ptr.value is None:
        return ctypes.c_void_p(None)
    return ctypes.c_void_p(t.ptr.value + elements * np.dtype(NX_TO_NUMPY[t.dtype]).itemsize)


def _given(t: DeviceTensor | None, what: str) -> ctypes.c_void_p | None:
    """The address of an operand that a call may do without. (A freed one has none, which would leave it out.)"""
    if t is None:
        return None
    if t.ptr is None:
        _refuse(f"{what} has been freed")
    return t.ptr


def _out(out: DeviceTensor | None, ctx: Context, shape, dtype: str) -> DeviceTensor:
    """The answer's memory: `out`, if it has the answer's shape and type, or new."""
    if out is None:
        return ctx.empty(shape, dtype)
    _given(out, "out")
    if out.shape != tuple(shape) or out.dtype != dtype:
        _refuse(f"out must be {dtype} {tuple(shape)}, got {out.dtype} {out.shape}")
    return out


class Rows8(NamedTuple):
    """Rows [..., N] in 8 bits: value (t, n) is q[t, n] * scales[n // 128, t]."""

    q: DeviceTensor       # f8_e4m3fn [..., N]
    scales: DeviceTensor  # f32 [ceil(N / 128), rows]

    @classmethod
    def empty(cls, ctx: Context, shape) -> "Rows8":
        return cls._of(ctx, shape, None)

    @classmethod
    def _of(cls, ctx: Context, shape, out: "Rows8 | None") -> "Rows8":
        rows = math.prod(shape[:-1])
        return cls(_out(out.q if out is not None else None, ctx, shape, "f8_e4m3fn"),
                   _out(out.scales if out is not None else None, ctx, (-(-shape[-1] // BLOCK), rows), "f32"))


class Norm(NamedTuple):
    """What rms_norm answers; what was not asked for is None."""

    y: DeviceTensor | None
    rows: Rows8 | None
    sum: DeviceTensor | None


def rms_norm(x: DeviceTensor, gamma: DeviceTensor, residual: DeviceTensor | None = None, eps: float = 1e-6, *,
             y: bool = False, rows: bool = True, out: Norm | None = None, stream=None) -> Norm:
    """h * rsqrt(mean(h^2) + eps) * gamma over the rows of h = x + residual, in x's type (`y`), in 8 bits (`rows`),
    or both; `sum` is h, where there is a residual. Of `out` the parts that are asked for are used; its sum may be x
    or the residual itself."""
    t, n = _rows(x, "the norm")
    if gamma.shape != (n,):
        _refuse(f"the norm's gamma must be [{n}], got {gamma.shape}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        _refuse(f"the residual must be {x.dtype} {x.shape}, got {residual.dtype} {residual.shape}")
    ctx = x.ctx
    out = out or Norm(None, None, None)
    out = Norm(_out(out.y, ctx, x.shape, x.dtype) if y else None, Rows8._of(ctx, x.shape, out.rows) if rows else None,
               _out(out.sum, ctx, x.shape, x.dtype) if residual is not None else None)
    ctx.check(lib().tmh_rms_norm(
        ctx.handle, x.ptr, n, _given(residual, "the residual"), n, x.tmh_dtype, t, n, gamma.ptr,
        gamma.tmh_dtype, eps, out.sum.ptr if out.sum else None, n, out.y.ptr if out.y else None, n,
        out.rows.q.ptr if out.rows else None, n, out.rows.scales.ptr if out.rows else None, stream))
    return out


def quantize_rows(x: DeviceTensor, *, out: Rows8 | None = None, stream=None) -> Rows8:
    """x's rows in 8 bits."""
    t, n = _rows(x, "quantization")
    out = Rows8._of(x.ctx, x.shape, out)
    x.ctx.check(lib().tmh_quantize_rows(x.ctx.handle, x.ptr, n, None, 0, x.tmh_dtype, t, n, out.q.ptr, n,
                                        out.scales.ptr, stream))
    return out


def quantize_swiglu(gate_up: DeviceTensor, *, out: Rows8 | None = None, stream=None) -> Rows8:
    """gate * sigmoid(gate) * up in 8 bits, of a merged gate/up product [..., 2 N] (the gate's columns first)."""
    t, width = _rows(gate_up, "SwiGLU")
    if width % 2:
        _refuse(f"a merged gate/up product has two equal halves, got {width} columns")
    n = width // 2
    out = Rows8._of(gate_up.ctx, (*gate_up.shape[:-1], n), out)
    gate_up.ctx.check(lib().tmh_quantize_rows(gate_up.ctx.handle, _at(gate_up, n), width, gate_up.ptr, width,
                                              gate_up.tmh_dtype, t, n, out.q.ptr, n, out.scales.ptr, stream))
    return out


class Fp8Weight:
    """A weight [N, K] of f8_e4m3fn with a scale for each 128 x 128 block, laid out once on the device
    (tmh_fp8_weight)."""

    def __init__(self, ctx: Context, handle: ctypes.c_void_p, k: int, n: int):
        self.ctx, self.handle, self.k, self.n = ctx, handle, k, n

    @property
    def shape(self) -> tuple[int, int]:
        return (self.n, self.k)

    @classmethod
    def from_pointers(cls, ctx: Context, b, scales, k: int, n: int, stream=None) -> "Fp8Weight":
        """From device memory that other code holds: b [n, k] f8_e4m3fn, scales [ceil(n/128), ceil(k/128)] f32,
        both of which must stay until the stream's work is done."""
        handle = ctypes.c_void_p()
        ctx.check(lib().tmh_fp8_weight_prepare(ctx.handle, b, scales, k, n, stream, ctypes.byref(handle)))
        return cls(ctx, handle, k, n)

    @classmethod
    def prepare(cls, ctx: Context, b, scales) -> "Fp8Weight":
        """From b [N, K] (f8_e4m3fn, or a host array of its bytes) and scales [ceil(N/128), ceil(K/128)] f32."""
        if not isinstance(b, DeviceTensor):
            b = np.asarray(b)
            # (Values of floats would be cut to whole numbers and taken for bits. Signed bytes are bits all the same.)
            if b.dtype.kind not in "iu" or (b.dtype.itemsize > 1 and b.size and not 0 <= b.min() <= b.max() <= 255):
                _refuse(f"a host 8-bit weight is an array of f8_e4m3fn bytes, got {b.dtype}")
        b_t = b if isinstance(b, DeviceTensor) else ctx.put(b.astype(np.uint8), "f8_e4m3fn")
        s_t = scales if isinstance(scales, DeviceTensor) else ctx.put(np.asarray(scales, dtype=np.float32))
        try:
            if len(b_t.shape) != 2 or b_t.dtype != "f8_e4m3fn":
                _refuse(f"an 8-bit weight is f8_e4m3fn [N, K], got {b_t.dtype} {b_t.shape}")
            n, k = b_t.shape
            if s_t.shape != (-(-n // BLOCK), -(-k // BLOCK)) or s_t.dtype != "f32":
                _refuse(f"the scales of an 8-bit weight [{n}, {k}] are f32 [{-(-n // BLOCK)}, {-(-k // BLOCK)}], "
                        f"got {s_t.dtype} {s_t.shape}")
            w = cls.from_pointers(ctx, b_t.ptr, s_t.ptr, k, n)
            ctx.synchronize()
        finally:
            if b_t is not b:
                b_t.free()
            if s_t is not scales:
                s_t.free()
        return w

    def device_bytes(self) -> int:
        size = ctypes.c_size_t()
        _lib.check(lib().tmh_fp8_weight_info(self.handle, None, None, ctypes.byref(size)))
        return size.value

    def free(self) -> None:
        if self.handle:
            lib().tmh_fp8_weight_free(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass

    def __repr__(self) -> str:
        return f"Fp8Weight(N={self.n}, K={self.k})"


def matmul_fp8(a: Rows8, w: Fp8Weight, bias: DeviceTensor | None = None, *, y_type: str = "f16",
               out: DeviceTensor | None = None, stream=None) -> DeviceTensor:
    """Y = A . W^T (+ bias) of rows and a weight in 8 bits, in y_type."""
    ctx = w.ctx
    if a.q.shape[-1] != w.k:
        _refuse(f"the 8-bit product's A has {a.q.shape[-1]} columns, K is {w.k}")
    m = math.prod(a.q.shape[:-1])
    if a.q.dtype != "f8_e4m3fn" or a.scales.dtype != "f32" or a.scales.shape != (-(-w.k // BLOCK), m):
        _refuse(f"the 8-bit product's A must be f8_e4m3fn with f32 scales [{-(-w.k // BLOCK)}, {m}], got {a.q.dtype} with "
                f"{a.scales.dtype} {a.scales.shape}")
    if bias is not None and bias.shape != (w.n,):
        _refuse(f"the 8-bit product's bias must be [{w.n}], got {bias.shape}")
    if y_type not in FLOAT_TYPES:
        _refuse(f"the 8-bit product's y must be f32, f16 or bf16, got {y_type}")
    y = _out(out, ctx, (*a.q.shape[:-1], w.n), y_type)
    ctx.check(lib().tmh_matmul_fp8(ctx.handle, w.handle, a.q.ptr, m, w.k, a.scales.ptr,
                                   _given(bias, "the 8-bit product's bias"), bias.tmh_dtype if bias is not None else 0,
                                   y.ptr, y.tmh_dtype, w.n, stream))
    return y


class PagedCache:
    """Keys and values in pages (tmh_paged_cache), either [pages, page_size, kv_heads, head_dim] (order "token") or
    [pages, kv_heads, page_size, head_dim] (order "head"). Which pages hold a sequence is the caller's to keep."""

    def __init__(self, ctx: Context, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: str = "f16",
                 order: str = "token"):
        if order not in ("token", "head"):
            _refuse(f"a paged cache's order is \"token\" or \"head\", got {order!r}")
        if dtype not in FLOAT_TYPES:
            _refuse(f"a paged cache holds f32, f16 or bf16 values, got {dtype}")
        if min(pages, page_size, kv_heads, head_dim) < 1:
            _refuse(f"a paged cache's sizes must be positive, got {(pages, page_size, kv_heads, head_dim)}")
        self.ctx, self.pages, self.page_size = ctx, pages, page_size
        self.kv_heads, self.head_dim, self.dtype, self.order = kv_heads, head_dim, dtype, order
        inner = (page_size, kv_heads) if order == "token" else (kv_heads, page_size)
        self.k = ctx.empty((pages, *inner, head_dim), dtype)
        self.v = ctx.empty((pages, *inner, head_dim), dtype)
        token, head = (kv_heads * head_dim, head_dim) if order == "token" else (head_dim, page_size * head_dim)
        self.desc = PagedCacheDesc(k=self.k.ptr, v=self.v.ptr, dtype=NX_TO_TMH[dtype], kv_heads=kv_heads,
                                   head_dim=head_dim, page_size=page_size, pages=pages,
                                   page_stride=page_size * kv_heads * head_dim, token_stride=token, head_stride=head)

    def append(self, qkv: DeviceTensor, heads: int, slots: DeviceTensor, positions: DeviceTensor | None = None,
               cos: DeviceTensor | None = None, sin: DeviceTensor | None = None, *, interleaved: bool = False,
               q_norm: DeviceTensor | None = None, k_norm: DeviceTensor | None = None, eps: float = 1e-6,
               out: DeviceTensor | None = None, stream=None) -> DeviceTensor:
        """The keys and values of a merged q/k/v product [T, (heads + 2 kv_heads) * head_dim] into slots [T] (s64,
        page * page_size + place; outside the cache: not stored), its queries and keys turned by their positions [T]
        (s64) first where tables cos and sin [max_positions, rotary_dim / 2] are given. With q_norm or k_norm, gammas
        [head_dim], each query or key head is normed ahead of that: x * rsqrt(mean(x^2) + eps) * gamma. Returns the
        queries."""
        t, d, g = math.prod(qkv.shape[:-1]), self.head_dim, self.kv_heads
        width = (heads + 2 * g) * d
        if qkv.dtype != self.dtype or qkv.shape[-1] != width:
            _refuse(f"the cache appends {self.dtype} rows of {width} columns, got {qkv.dtype} {qkv.shape}")
        if slots.dtype != "s64" or slots.size != t:
            _refuse(f"a step of {t} tokens takes {t} s64 slots, got {slots.dtype} {slots.shape}")
        rotary = most = table = 0
        if cos is not None or sin is not None:
            if cos is None or sin is None or positions is None or cos.shape != sin.shape or cos.dtype != sin.dtype or len(cos.shape) != 2:
                _refuse("rotary positions take positions and tables cos and sin of one type and shape")
            if positions.dtype != "s64" or positions.size != t:
                _refuse(f"a step of {t} tokens takes {t} s64 positions, got {positions.dtype} {positions.shape}")
            most, rotary, table = cos.shape[0], 2 * cos.shape[1], cos.tmh_dtype
        gammas = [gamma for gamma in (q_norm, k_norm) if gamma is not None]
        if any(gamma.shape != (d,) or gamma.dtype != gammas[0].dtype for gamma in gammas):
            _refuse(f"the heads' norms take gammas [{d}] of one type, got {[(gamma.dtype, gamma.shape) for gamma in gammas]}")
        norm = (_given(q_norm, "q_norm"), _given(k_norm, "k_norm"), gammas[0].tmh_dtype, eps) if gammas else ()
        q = _out(out, self.ctx, (*qkv.shape[:-1], heads * d), self.dtype)
        self.ctx.check((lib().tmh_paged_append_norm if norm else lib().tmh_paged_append)(
            self.ctx.handle, qkv.ptr, width, _at(qkv, heads * d), width, _at(qkv, (heads + g) * d), width, t, heads, *norm,
            positions.ptr if rotary else None, cos.ptr if rotary else None, sin.ptr if rotary else None, table, most,
            rotary, int(interleaved), slots.ptr, ctypes.byref(self.desc), q.ptr, heads * d, stream))
        return q

    def attend(self, q: DeviceTensor, page_table: DeviceTensor, lengths: DeviceTensor, *, scale: float | None = None,
               window: int = 0, out: DeviceTensor | None = None, stream=None) -> DeviceTensor:
        """Attention of one token a sequence, q [B, heads * head_dim], over the first lengths[b] (s32) tokens of the
        pages page_table[b] (s32, [B, max_pages]), or the last `window` of them. The scale is 1 / sqrt(head_dim) by
        default."""
        if q.dtype != self.dtype or len(q.shape) != 2 or q.shape[1] % self.head_dim:
            _refuse(f"attention takes {self.dtype} queries [B, heads * {self.head_dim}], got {q.dtype} {q.shape}")
        b = q.shape[0]
        if page_table.dtype != "s32" or len(page_table.shape) != 2 or page_table.shape[0] != b:
            _refuse(f"the page table is s32 [{b}, pages], got {page_table.dtype} {page_table.shape}")
        if lengths.dtype != "s32" or lengths.shape != (b,):
            _refuse(f"the lengths are s32 [{b}], got {lengths.dtype} {lengths.shape}")
        y = _out(out, self.ctx, q.shape, q.dtype)
        scale = 1 / math.sqrt(self.head_dim) if scale is None else scale
        self.ctx.check(lib().tmh_paged_attention(
            self.ctx.handle, q.ptr, q.shape[1], b, q.shape[1] // self.head_dim, ctypes.byref(self.desc), page_table.ptr,
            page_table.shape[1], lengths.ptr, scale, window, y.ptr, y.shape[1], stream))
        return y

    def attend_tree(self, q: DeviceTensor, page_table: DeviceTensor, lengths: DeviceTensor, starts: DeviceTensor,
                    mask: DeviceTensor | None = None, *, scale: float | None = None, window: int = 0,
                    out: DeviceTensor | None = None, stream=None) -> DeviceTensor:
        """Attention of several new tokens a sequence: rows starts[b] .. starts[b + 1] - 1 (s32, [B + 1]) of q
        [T, heads * head_dim] are the last of sequence b's lengths[b] (s32) tokens, in the pages page_table[b] (s32,
        [B, max_pages]). A row sees its sequence's tokens before them, and of them those whose bits its row of mask
        [T, words] (s64) has: bit j % 64 of word j // 64 is the sequence's j-th row. Without a mask a row sees those up to
        itself (a chain of drafts, a prompt's chunk). With a window it sees the last `window` of these. The scale is
        1 / sqrt(head_dim) by default; rows behind the last sequence's are left as they are."""
        if q.dtype != self.dtype or len(q.shape) != 2 or q.shape[1] % self.head_dim:
            _refuse(f"attention takes {self.dtype} queries [T, heads * {self.head_dim}], got {q.dtype} {q.shape}")
        t = q.shape[0]
        if page_table.dtype != "s32" or len(page_table.shape) != 2:
            _refuse(f"the page table is s32 [B, pages], got {page_table.dtype} {page_table.shape}")
        b = page_table.shape[0]
        if lengths.dtype != "s32" or lengths.shape != (b,):
            _refuse(f"the lengths are s32 [{b}], got {lengths.dtype} {lengths.shape}")
        if starts.dtype != "s32" or starts.shape != (b + 1,):
            _refuse(f"the starts are s32 [{b + 1}], got {starts.dtype} {starts.shape}")
        if mask is not None and (mask.dtype != "s64" or len(mask.shape) != 2 or mask.shape[0] != t or mask.shape[1] < 1):
            _refuse(f"the mask is s64 [{t}, words], got {mask.dtype} {mask.shape}")
        y = _out(out, self.ctx, q.shape, q.dtype)
        scale = 1 / math.sqrt(self.head_dim) if scale is None else scale
        self.ctx.check(lib().tmh_paged_tree_attention(
            self.ctx.handle, q.ptr, q.shape[1], t, q.shape[1] // self.head_dim, ctypes.byref(self.desc), page_table.ptr, b,
            page_table.shape[1], lengths.ptr, starts.ptr, _given(mask, "the mask"), mask.shape[1] if mask is not None else 0,
            scale, window, y.ptr, y.shape[1], stream))
        return y

    def free(self) -> None:
        self.k.free()
        self.v.free()
        self.desc.k = self.desc.v = None  # (later calls are refused)

    def __repr__(self) -> str:
        return (f"PagedCache({self.pages} pages of {self.page_size}, {self.kv_heads} heads of {self.head_dim}, "
                f"{self.dtype}, {self.order})")


def sample(logits: DeviceTensor, random: DeviceTensor, *, temperature: DeviceTensor | None = None,
           top_k: DeviceTensor | None = None, top_p: DeviceTensor | None = None, min_p: DeviceTensor | None = None,
           out: DeviceTensor | None = None, stream=None) -> DeviceTensor:
    """One token (s64) for each row of logits [..., V], drawn by the row's random number in [0, 1) (f32). Each row has its
    own temperature (f32; 0: the largest logit), top_k (s32; 0: all), top_p (f32; 1: all) and min_p (f32; 0: all), None
    leaving that out for all rows: of the top_k largest logits' tokens the fewest whose probabilities sum to top_p, and of
    these those of at least min_p times the most probable one's. -1 for a row without a logit above -infinity."""
    t, v = _rows(logits, "sampling")
    for name, tensor, dtype in (("random", random, "f32"), ("temperature", temperature, "f32"), ("top_k", top_k, "s32"),
                                ("top_p", top_p, "f32"), ("min_p", min_p, "f32")):
        if tensor is not None and (tensor.dtype != dtype or tensor.size != t):
            _refuse(f"sampling {t} rows takes {t} {dtype} values of {name}, got {tensor.dtype} {tensor.shape}")
    ctx = logits.ctx
    out = _out(out, ctx, logits.shape[:-1], "s64")
    ctx.check(lib().tmh_sample(ctx.handle, logits.ptr, v, logits.tmh_dtype, t, v, _given(temperature, "temperature"),
                               _given(top_k, "top_k"), _given(top_p, "top_p"), _given(min_p, "min_p"), random.ptr, out.ptr,
                               stream))
    return out
