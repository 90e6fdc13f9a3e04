"""A paged key-value cache in 4 bits: little more than a fourth of the memory of
PagedKVCache in 16-bit types, and of what attention reads.

  PagedKVCache4bit  append(): quantise and store new keys and values, the keys
                    rotated on the way; attend(): attention of one new token
                    per sequence; read(): the values that slots hold

The calls are those of decoding.PagedKVCache, on its terms (streams, capture
into CUDA graphs, errors, gradients).  They have no counterpart in PyFlame.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional

from . import _native as N
from .decoding import (RotaryEmbedding, _apart, _Bound, _call, _check, _code, _cuda, _extent, _model, _no_tangents, _other_strides,
                       _Plans)


class PagedKVCache4bit:
    """Keys and values of many sequences in 4 bits, in pages of `page_size`
    tokens.

    A head's values are cut into groups of `group_size` (32, 64 or 128; the
    last may be shorter), and a group is kept as 16 even steps from its least
    value on: value = low + step * code with low = bfloat16(least), step =
    bfloat16((greatest - low) * (1 / 15)) (0 below 2^-126) and code = (value -
    low) * (1 / step) rounded to the nearest (ties to even) of 0 to 15, each
    operation, 1 / 15 and 1 / step among them, rounded to float32.  A group
    that holds an infinity, a NaN or a value above 2^126 in size is kept as
    NaN.  head_dim: a multiple of 8, at most 256.

    `k`, `v` (codes, in an order of their own) and `k_scales`, `v_scales` are
    int32 [num_pages, num_heads, ...]: a page is moved by copying its rows of
    all four.  Values of two tokens share words, so a page of an odd size has
    room for one more.  Which pages a sequence owns is the caller's
    bookkeeping.  Keys, values and queries of a call are float32, float16 or
    bfloat16; the cache itself has no type.
    """

    def __init__(self, num_pages: int, page_size: int, num_heads: int, head_dim: int, group_size: int = 64, device="cuda"):
        import torch
        _Bound.load()
        pages, size, heads, dim, group = (int(s) for s in (num_pages, page_size, num_heads, head_dim, group_size))
        if min(pages, size, heads) < 1:
            raise ValueError("sizes must be positive")
        if pages * size > 0x7FFFFFFF or pages * size * heads >= 0xFFFFFFFF:
            raise ValueError("a cache holds fewer than 2^31 tokens, and fewer than 2^32 - 1 heads of them")
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError(f"device: must be a CUDA device, not {device}")
        codes, scales = C.c_int64(0), C.c_int64(0)
        N.check(N.lib().pfk_cache4_words(dim, group, C.byref(codes), C.byref(scales)))
        records, pairs = pages * heads * size, pages * heads * ((size + 1) // 2)
        with torch.inference_mode(False):  # a tensor made in that mode could not be written outside it
            # one memory for all, so that an output that lies in it is found by one comparison
            memory = torch.zeros(records * (codes.value + 2 * scales.value) + pairs * 2 * codes.value + 4 * 4, dtype=torch.int32,
                                 device=device)
            self._err = torch.zeros(1, dtype=torch.int32, device=device)
        parts, at = [], 0
        for rows, words in ((size, codes.value), ((size + 1) // 2, 2 * codes.value), (size, scales.value), (size, scales.value)):
            count = pages * heads * rows * words
            parts.append(memory[at:at + count].view(pages, heads, rows, words))
            at += -(-count // 4) * 4  # the next begins at a multiple of 16 bytes
        self.k, self.v, self.k_scales, self.v_scales = parts
        self.device = memory.device
        self.num_pages, self.page_size, self.num_heads, self.head_dim, self.group_size = pages, size, heads, dim, group
        self._start, self._end = memory.data_ptr(), memory.data_ptr() + memory.numel() * 4
        self._c = N.Cache4C(*(t.data_ptr() for t in parts), pages, size, heads, dim, group, self._err.data_ptr())
        self._plans = _Plans()
        self._no_rotary = N.RotaryC(None, 0, 0, 1.0)
        L = N.lib()
        self._append_fn, self._attend_fn, self._read_fn = L.pfk_cache4_append, L.pfk_cache4_attention, L.pfk_cache4_read

    def _apart_from_cache(self, name, to, size):
        if to < self._end and self._start < to + size:
            raise ValueError(f"{name}: shares memory with the cache")

    def append(self, k, v, slots, positions=None, rotary: Optional[RotaryEmbedding] = None, q=None, q_out=None):
        """Quantise and store new tokens: k, v [tokens, num_heads, head_dim] at
        `slots` (int64 [tokens], page * page_size + offset; negative: the token
        is skipped).  With `rotary`, keys and queries q [tokens, q_heads,
        head_dim] are rotated by `positions` (int64 [tokens]) first, the keys
        in 64 bits, rounded to float32 once; returns the rotated queries
        (`q_out`, which may be q and otherwise shares no memory with the
        inputs, or a new tensor, whose rows of skipped tokens are 0).  The
        slots of one call are distinct."""
        if _Bound.forward._current_level >= 0:  # inside forward-mode differentiation
            _no_tangents(k=k, v=v, q=q, q_out=q_out)
        key = (k.dtype, k.shape, k.stride(), k.get_device(), k.requires_grad, v.dtype, v.shape, v.stride(), v.get_device(),
               v.requires_grad, slots.dtype, slots.shape, slots.stride(), slots.get_device(),
               None if rotary is None else rotary._kind,
               None if positions is None else (positions.dtype, positions.shape, positions.stride(), positions.get_device()),
               None if q is None else (q.dtype, q.shape, q.stride(), q.get_device(), q.requires_grad),
               None if q_out is None else (q_out.dtype, q_out.shape, q_out.stride(), q_out.get_device(), q_out.requires_grad))
        plan = self._plans.get(key) or self._plans.keep(
            key, self._append_plan(k, v, slots, positions, rotary, q, q_out), k, v, q, q_out)
        p = N.Cache4AppendParamsC.from_buffer_copy(plan[0])
        p.k, p.v, p.slots = at_k, at_v, _ = k.data_ptr(), v.data_ptr(), slots.data_ptr()
        if rotary is not None:
            p.positions, p.rotary, p.factor = positions.data_ptr(), rotary._c, rotary.factor
        if q is not None:
            if q_out is None:
                q_out = q.new_zeros(q.shape)
            else:
                size_q, size_k, size_v, size, other = plan[1]
                at, to = q.data_ptr(), q_out.data_ptr()
                end = to + size
                if at == to:
                    if other:
                        raise ValueError("q_out: shares q's memory with other strides")
                elif to < at + size_q and at < end:
                    _apart("q_out", q_out, q=q)
                if to < at_k + size_k and at_k < end or to < at_v + size_v and at_v < end:
                    _apart("q_out", q_out, k=k, v=v)
                self._apart_from_cache("q_out", to, size)
            if p.q_heads:
                p.q, p.q_out = q.data_ptr(), q_out.data_ptr()
        _call(self._append_fn, self.device, C.byref(p))
        return q_out

    def _append_plan(self, k, v, slots, positions, rotary, q, q_out):
        import torch
        n, h, d = len(k), self.num_heads, self.head_dim
        code = _code(k.dtype)
        _check("k", k, (n, h, d), k.dtype, self.device)
        _check("v", v, (n, h, d), k.dtype, self.device)
        _check("slots", slots, (n,), torch.int64, self.device)
        if (rotary is None) != (positions is None):
            raise ValueError("positions and rotary go together")
        if rotary is not None:
            if rotary.head_dim != d or rotary.device != self.device:
                raise ValueError("rotary: is for another head_dim or device")
            _check("positions", positions, (n,), torch.int64, self.device)
        ks, vs, outputs = k.stride(), v.stride(), None
        p = N.Cache4AppendParamsC(self._c, code, n, None, ks[0], ks[1], None, vs[0], vs[1])
        p.rotary = self._no_rotary
        if q is not None:
            _check("q", q, (n, None, d), k.dtype, self.device)
            qs = os = q.stride()
            if q_out is not None:
                _check("q_out", q_out, q.shape, k.dtype, self.device, output=True)
                os = q_out.stride()
                outputs = _extent(q), _extent(k), _extent(v), _extent(q_out), _other_strides(q, q_out)
            else:
                os = torch.empty(q.shape, device="meta").stride()
            p.q_heads, p.q_st, p.q_sh, p.qo_st, p.qo_sh = q.shape[1], qs[0], qs[1], os[0], os[1]
        elif q_out is not None:
            raise ValueError("q_out without q")
        return p, outputs

    def read(self, slots, dtype=None):
        """(k, v): what the cache holds at `slots` (int64 [tokens]; negative:
        zeros), [tokens, num_heads, head_dim] in `dtype` (float32 by
        default)."""
        key = (dtype, slots.dtype, slots.shape, slots.stride(), slots.get_device())
        plan = self._plans.get(key) or self._plans.keep(key, self._read_plan(slots, dtype), slots)
        p = N.Cache4ReadParamsC.from_buffer_copy(plan[0])
        empty = _Bound.torch.empty_like
        k, v = empty(plan[1]), empty(plan[1])
        p.slots, p.k, p.v = slots.data_ptr(), k.data_ptr(), v.data_ptr()
        _call(self._read_fn, self.device, C.byref(p))
        return k, v

    def _read_plan(self, slots, dtype):
        import torch
        dtype = torch.float32 if dtype is None else dtype
        code = _code(dtype)
        _check("slots", slots, (None,), torch.int64, self.device)
        return (N.Cache4ReadParamsC(self._c, code, len(slots)), _model(self._err, (len(slots), self.num_heads, self.head_dim), dtype))

    def attend(self, q, block_table, seq_lens, scale: Optional[float] = None, window: int = 0, out=None,
               return_lse: bool = False):
        """Attention of one new token per sequence over the values that the
        cache holds, its own key among them: q [batch, q_heads, head_dim]
        (q_heads a multiple of num_heads; query head h reads key-value head h
        // (q_heads / num_heads)), block_table int32 [batch, pages], seq_lens
        int32 [batch].  `scale` (1/sqrt(head_dim) by default) multiplies the
        scores; `window` > 0: only a sequence's last `window` tokens are seen.
        A sequence of length 0 gives 0.  With return_lse also the natural
        logarithm of the sum of exp(score), float32 [batch, q_heads] (-inf for
        length 0).  `out` may be q and otherwise shares no memory with it or
        the cache.  An infinity or NaN in q or in a seen row may make the
        results that depend on it NaN."""
        if _Bound.forward._current_level >= 0:  # inside forward-mode differentiation
            _no_tangents(q=q, out=out)
        torch = _Bound.torch
        scale, window = None if scale is None else float(scale), min(int(window), 0x7FFFFFFF)
        key = (scale, window, return_lse, q.dtype, q.shape, q.stride(), q.get_device(), q.requires_grad, block_table.dtype,
               block_table.shape, block_table.stride(), block_table.get_device(), seq_lens.dtype, seq_lens.shape,
               seq_lens.stride(), seq_lens.get_device())
        if out is not None:
            key += (out.dtype, out.shape, out.stride(), out.get_device(), out.requires_grad)
        plan = self._plans.get(key) or self._plans.keep(
            key, self._attend_plan(q, block_table, seq_lens, scale, window, out, return_lse), q, out)
        if out is None:
            out = torch.empty_like(q) if plan[1] else q.new_empty(q.shape)
        at, to = q.data_ptr(), out.data_ptr()
        if plan[4] is not None:
            size_q, size, other = plan[4]
            if at == to:
                if other:
                    raise ValueError("out: shares q's memory with other strides")
            elif to < at + size_q and at < to + size:
                _apart("out", out, q=q)
            self._apart_from_cache("out", to, size)
        p = N.Cache4AttentionParamsC.from_buffer_copy(plan[0])
        p.q, p.out, p.block_table, p.seq_lens = at, to, block_table.data_ptr(), seq_lens.data_ptr()
        lse = None
        if return_lse:
            lse = torch.empty_like(plan[3])
            p.lse = lse.data_ptr()
        # a workspace per call, from torch's allocator: calls on several streams and captured graphs share none
        if plan[2]:
            work = torch.empty(plan[2], dtype=torch.uint8, device=self.device)
            p.workspace = work.data_ptr()
        _call(self._attend_fn, self.device, C.byref(p))
        return (out, lse) if return_lse else out

    def _attend_plan(self, q, block_table, seq_lens, scale, window, out, return_lse):
        import torch
        if len(q.shape) != 3:
            raise ValueError("q must be [batch, q_heads, head_dim]")
        batch, heads, d = q.shape
        code = _code(q.dtype)
        _check("q", q, (None, None, self.head_dim), q.dtype, self.device)
        if heads == 0 or heads % self.num_heads:
            raise ValueError(f"q: {heads} heads are not a multiple of {self.num_heads}")
        _check("block_table", block_table, (batch, None), torch.int32, self.device)
        _check("seq_lens", seq_lens, (batch,), torch.int32, self.device)
        if window < 0:
            raise ValueError("window must not be negative")
        scale = 1.0 / math.sqrt(d) if scale is None else scale
        if out is not None:
            _check("out", out, (batch, heads, d), q.dtype, self.device, output=True)
        qs = q.stride()
        os = torch.empty(q.shape, device="meta").stride() if out is None else out.stride()
        p = N.Cache4AttentionParamsC(self._c, code, batch, heads, None, qs[0], qs[1], None, os[0], os[1], None, None,
                                     block_table.stride(0), block_table.shape[1], None, window, scale)
        size = C.c_size_t(0)
        with torch.cuda.device(self.device):
            N.check(N.lib().pfk_cache4_attention_workspace(C.byref(p), C.byref(size)))
        p.workspace_bytes = size.value
        return (p, q.is_contiguous(), size.value, _model(self._err, (batch, heads), torch.float32) if return_lse else None,
                None if out is None else (_extent(q), _extent(out), _other_strides(q, out)))

    def check(self) -> None:
        """Wait for the device and raise PfcError if a call met a slot, page
        or length outside the cache since the last check."""
        _Bound.torch.cuda.synchronize(self.device)
        code = int(self._err.item())
        if code:
            self._err.zero_()
            # finished here: later, it would clear the flag of a call on another stream
            _Bound.torch.cuda.synchronize(self.device)
            raise N.PfcError(code, "a call met a slot, page or length outside the 4-bit paged cache")
