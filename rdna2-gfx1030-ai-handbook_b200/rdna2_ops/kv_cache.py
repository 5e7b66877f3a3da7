"""A paged key/value cache held in 8 bits, and attention over it.

  cache = PagedKVCache(num_pages, kv_heads, head_dim, page_size=64, code="int8")
  q = cache.append(k, v, lengths, table, q=q, angles=angles)   # rotate, quantize, store
  y = cache.attend(q, lengths, table)                           # read
  k, v = cache.read(pages)                                      # values of whole pages

A page holds page_size tokens of one sequence for every kv head: int8 or
float8_e4m3fn codes [page_size, head_dim] and one fp32 scale for each (page,
head), K and V apart; a value is code * scale.  The caller owns the paging:
table[b, i] is the page of sequence b's tokens [i * page_size, (i + 1) *
page_size), and lengths[b] counts its tokens, those of the call included.  A
call's tokens are packed, [tokens, heads, head_dim]: the same number for every
sequence, or rows offsets[b] .. offsets[b + 1], with offsets[0] = 0 and the
last one the number of tokens; a sequence's last row is at position
lengths[b] - 1.  lengths, table and offsets are int32 on the device and are
not read on the host: one lengths tensor serves every layer of a step.

Tokens at negative positions, past the table, or on a table entry outside the
cache (-1 marks an absent page) are not stored and not seen.  A page that a
call appends to must belong to one sequence only.

What attend relies on where a cache holds other data than append wrote: scales
are not negative, a value scale below 2**-100 counts as 2**-100 (append writes
none, and zero goes with codes of zero), and e4m3 codes are no NaN, but behind
the last token of a sequence.  A scale that is NaN or infinite shows in the rows
that see its block, in all of their channels, and in no others.

The workspace of attend is kept for each stream, so one cache may serve calls
on several; ordering its appends before the calls that read them is the
caller's, as for any tensor.
"""
from __future__ import annotations

import functools
import math

import torch

from . import _args
from . import _native as nat
from .rotary import LAYOUTS, angle_table

CODE_DTYPE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
_CODE_INDEX = {torch.int8: 0, torch.float8_e4m3fn: 1}
PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)


def _rows(x):
    """x [tokens, heads, dim] itself where the kernels can read its rows (channels
    contiguous, rows at multiples of 16 bytes), else a copy."""
    if x.data_ptr() % 16 == 0:
        step = 16 // x.element_size()
        if x.stride(2) == 1 and x.stride(0) % step == 0 and x.stride(1) % step == 0:
            return x
        if x.is_contiguous():  # the stride of a dimension of one entry is anything
            return x.as_strided(x.shape, (x.shape[1] * x.shape[2], x.shape[2], 1))
    return x.clone(memory_format=torch.contiguous_format)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(index, *shape):
    with torch.cuda.device(index):
        return nat.library().b2_kv_attention_workspace_bytes(*shape)


class PagedKVCache:
    """num_pages pages of page_size tokens for kv_heads heads of head_dim
    channels, all codes and scales zero."""

    def __init__(self, num_pages, kv_heads, head_dim, *, page_size=64, code="int8", device="cuda"):
        _args.require(code in CODE_DTYPE, ValueError, "code must be 'int8' or 'e4m3'")
        _args.require(num_pages >= 0 and kv_heads >= 1, ValueError, "num_pages and kv_heads must be positive")
        codes = (num_pages, kv_heads, page_size, head_dim)
        self._hold(*(torch.zeros(codes, device=device, dtype=torch.uint8).view(CODE_DTYPE[code]) for _ in range(2)),
                   *(torch.zeros(codes[:2], device=device, dtype=torch.float32) for _ in range(2)))

    @classmethod
    def wrap(cls, k_codes, v_codes, k_scale, v_scale):
        """A cache in the caller's own tensors: codes [pages, kv_heads,
        page_size, head_dim] int8 or float8_e4m3fn, scales [pages, kv_heads] fp32."""
        cache = cls.__new__(cls)
        cache._hold(k_codes, v_codes, k_scale, v_scale)
        return cache

    def _hold(self, k_codes, v_codes, k_scale, v_scale):
        _args.require(all(isinstance(t, torch.Tensor) for t in (k_codes, v_codes, k_scale, v_scale)), TypeError,
                      "A cache is made of tensors")
        _args.require(k_codes.dtype in _CODE_INDEX and v_codes.dtype == k_codes.dtype, TypeError,
                      "codes must both be int8 or both float8_e4m3fn")
        _args.require(k_scale.dtype == v_scale.dtype == torch.float32, TypeError, "scales must be fp32")
        _args.require(k_codes.ndim == 4 and v_codes.shape == k_codes.shape
                      and k_scale.shape == v_scale.shape == k_codes.shape[:2], ValueError,
                      "codes must be [pages, kv_heads, page_size, head_dim] and scales [pages, kv_heads]")
        _args.require(k_codes.shape[2] in PAGE_SIZES, ValueError, f"page_size must be one of {PAGE_SIZES}")
        _args.require(k_codes.shape[3] in HEAD_DIMS, ValueError, f"head_dim must be one of {HEAD_DIMS}")
        _args.require(all(t.is_contiguous() and t.device == k_codes.device
                          for t in (k_codes, v_codes, k_scale, v_scale)), ValueError,
                      "codes and scales must be contiguous on one device")
        self.k_codes, self.v_codes, self.k_scale, self.v_scale = k_codes, v_codes, k_scale, v_scale
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = k_codes.shape
        self.code = "int8" if k_codes.dtype == torch.int8 else "e4m3"
        self._workspaces = {}  # one for each stream: calls on one stream follow each other

    def _memory(self):
        """The codes and scales as the C entry points take them."""
        return (self.k_codes.data_ptr(), self.v_codes.data_ptr(), self.k_scale.data_ptr(), self.v_scale.data_ptr(),
                self.num_pages)

    # ------------------------------------------------------------- arguments
    def _call(self, x, name, lengths, table, offsets):
        """Checks a call's packed tokens and its paging; returns (device, tokens, batch, width)."""
        if not isinstance(x, torch.Tensor) or x.dtype not in _args.FLOAT_DTYPES:
            raise TypeError(f"{name} must be an fp32, fp16 or bf16 tensor")
        shape = x.shape
        if len(shape) != 3 or shape[2] != self.head_dim:
            raise ValueError(f"{name} must be [tokens, heads, {self.head_dim}], got {tuple(shape)}")
        dev = nat.require_device(self.k_codes, x, lengths, table, offsets)
        if lengths.dtype != torch.int32 or table.dtype != torch.int32 or (
                offsets is not None and offsets.dtype != torch.int32):
            raise TypeError("lengths, table and offsets must be int32")
        paging = table.shape
        if lengths.ndim != 1 or len(paging) != 2 or paging[0] != lengths.shape[0]:
            raise ValueError(f"lengths must be [batch] and table [batch, pages], got {tuple(lengths.shape)} "
                             f"and {tuple(paging)}")
        if not (lengths.is_contiguous() and table.is_contiguous()):
            raise ValueError("lengths and table must be contiguous")
        tokens, (batch, width) = shape[0], paging
        if offsets is None:
            if batch == 0 and tokens or batch and tokens % batch:
                raise ValueError(f"{tokens} tokens do not divide among {batch} sequences; pass offsets")
        elif offsets.shape != (batch + 1,) or not offsets.is_contiguous():
            raise ValueError(f"offsets must be contiguous [{batch + 1}], got {tuple(offsets.shape)}")
        return dev, tokens, batch, width

    # ---------------------------------------------------------------- append
    def append(self, k, v, lengths, table, *, offsets=None, q=None, angles=None, layout="half"):
        """Stores keys and values [tokens, kv_heads, head_dim] (fp32, fp16 or
        bf16) of the call's tokens.  With angles [positions, rotary_dim] (see
        rope_table; rotary_dim a multiple of 16) the keys are rotated to their
        positions first, and q [tokens, q_heads, head_dim], if given, is
        returned rotated.

        A block (page, head) gets the scale s = max(s_old if it holds earlier
        tokens, max|x| / top, 2**-100), top = 127 (int8) or 448 (e4m3), its
        earlier codes become rne(c * (s_old / s)) and its new ones
        rne(x * fp32(1 / s)).  A NaN or infinite x shows in its whole block."""
        dev, tokens, batch, width = self._call(k, "k", lengths, table, offsets)
        if layout not in LAYOUTS:
            raise ValueError("layout must be 'half' or 'interleaved'")
        if not isinstance(v, torch.Tensor) or v.shape != k.shape or v.dtype != k.dtype or v.device != dev:
            raise ValueError("k and v must have one shape, type and device")
        if k.shape[1] != self.kv_heads:
            raise ValueError(f"k and v must have {self.kv_heads} heads, got {k.shape[1]}")
        nat.eager_only(k, v, q)
        rotary_dim = rows = 0
        if angles is not None:
            angle_table(angles, self.head_dim, dev)
            rows, rotary_dim = angles.shape
            if rotary_dim % 16:
                raise ValueError(f"append needs a rotary_dim that is a multiple of 16, got {rotary_dim}")
        rotated = None
        if q is not None:
            if angles is None:
                raise ValueError("q is only rotated: pass angles with it")
            if not isinstance(q, torch.Tensor) or q.dtype != k.dtype or q.device != dev:
                raise TypeError("q must have k's type and device")
            if q.ndim != 3 or q.shape[0] != tokens or q.shape[2] != self.head_dim:
                raise ValueError(f"q must be [{tokens}, heads, {self.head_dim}], got {tuple(q.shape)}")
            rotated = torch.empty_like(q, memory_format=torch.contiguous_format)
            q = _rows(q) if q.numel() else None
        if tokens == 0:
            return rotated
        k, v = _rows(k), _rows(v)
        nat.launch(
            dev, "b2_kv_append", k.data_ptr(), v.data_ptr(), nat.DTYPE_CODE[k.dtype], tokens, self.kv_heads,
            self.head_dim, k.stride(0), k.stride(1), v.stride(0), v.stride(1), lengths.data_ptr(), nat.ptr(offsets),
            batch, table.data_ptr(), width, nat.ptr(q), 0 if q is None else q.shape[1],
            0 if q is None else q.stride(0), 0 if q is None else q.stride(1), nat.ptr(rotated), nat.ptr(angles), rows,
            rotary_dim, LAYOUTS[layout], _CODE_INDEX[self.k_codes.dtype], *self._memory(), self.page_size)
        return rotated

    # ---------------------------------------------------------------- attend
    def attend(self, q, lengths, table, *, offsets=None, max_new=None, causal=True, window=None, scale=None,
               return_lse=False):
        """Attention of q [tokens, q_heads, head_dim] (fp16 or bf16) over the
        cache; q_heads is a multiple of kv_heads, and head h reads kv head
        h // (q_heads // kv_heads).

        A row at position p sees the cached tokens j < lengths[b]; with causal
        only j <= p, with window only j > p - window.  scale defaults to
        head_dim ** -0.5.  max_new bounds the tokens of one sequence where
        offsets are given (default: all tokens of the call); it picks the
        kernel and has no other effect.  Returns out (q's shape and type) and,
        with return_lse, the logarithm of each row's sum of exponentials
        [tokens, q_heads] fp32.  A row that sees nothing gives 0 and -inf."""
        dev, tokens, batch, width = self._call(q, "q", lengths, table, offsets)
        if q.dtype == torch.float32:
            raise TypeError("q must be fp16 or bf16")
        heads = q.shape[1]
        if heads == 0 or heads % self.kv_heads:
            raise ValueError(f"q has {heads} heads, not a multiple of {self.kv_heads}")
        if window is not None and window < 1:
            raise ValueError(f"window must be at least 1, got {window}")
        scale = self.head_dim ** -0.5 if scale is None else float(scale)
        if not (scale > 0.0 and math.isfinite(scale)):
            raise ValueError(f"scale must be positive and finite, got {scale}")
        nat.eager_only(q)
        if offsets is None:
            max_new = tokens // batch if batch else 0
        elif max_new is None:
            max_new = tokens
        elif max_new < 1:
            raise ValueError(f"max_new must be at least 1, got {max_new}")
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        lse = torch.empty((tokens, heads), device=dev, dtype=torch.float32) if return_lse else None
        if tokens:
            q = _rows(q)
            stream = nat.stream_ptr(dev)
            need = _workspace_bytes(dev.index, tokens, batch, max_new, heads, self.kv_heads, self.head_dim, width,
                                    self.page_size, window or 0)
            work = self._workspaces.get(stream)
            if work is None or work.numel() < need:
                work = self._workspaces[stream] = torch.zeros(need, device=dev, dtype=torch.uint8)
            nat.launch(
                dev, "b2_kv_attention", q.data_ptr(), nat.DTYPE_CODE[q.dtype], tokens, heads, q.stride(0), q.stride(1),
                lengths.data_ptr(), nat.ptr(offsets), batch, max_new, table.data_ptr(), width,
                _CODE_INDEX[self.k_codes.dtype], *self._memory(), self.kv_heads, self.page_size, self.head_dim, scale,
                int(causal), window or 0, out.data_ptr(), nat.ptr(lse), work.data_ptr(), work.numel())
        return (out, lse) if return_lse else out

    # ------------------------------------------------------------------ read
    def read(self, pages, *, dtype=torch.bfloat16, return_scales=False):
        """Keys and values of whole pages [n] (int32), each [n, kv_heads,
        page_size, head_dim], and with return_scales their scales, each [n,
        kv_heads] fp32; NaN for a page outside the cache."""
        if dtype not in _args.FLOAT_DTYPES:
            raise TypeError(f"dtype must be fp32, fp16 or bf16, got {dtype}")
        dev = nat.require_device(self.k_codes, pages)
        if pages.dtype != torch.int32:
            raise TypeError("pages must be int32")
        if pages.ndim != 1 or not pages.is_contiguous():
            raise ValueError(f"pages must be contiguous [n], got {tuple(pages.shape)}")
        nat.eager_only()
        shape = (pages.shape[0], self.kv_heads, self.page_size, self.head_dim)
        k, v = torch.empty(shape, device=dev, dtype=dtype), torch.empty(shape, device=dev, dtype=dtype)
        scales = torch.empty((2, *shape[:2]), device=dev, dtype=torch.float32) if return_scales else None
        nat.launch(
            dev, "b2_kv_read", *self._memory()[:4], _CODE_INDEX[self.k_codes.dtype], self.num_pages, self.kv_heads,
            self.page_size, self.head_dim, pages.data_ptr(), shape[0], nat.DTYPE_CODE[dtype], k.data_ptr(),
            v.data_ptr(), nat.ptr(scales))
        return (k, v, *scales.unbind()) if return_scales else (k, v)
