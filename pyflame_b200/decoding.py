"""Token generation over a paged key-value cache.

The steps of a decoder layer for new tokens, on CUDA tensors of torch, in
float32, float16 or bfloat16:

  Linear4bit        x W^T (+ bias) with 4-bit weights and group scales
  RotaryEmbedding   rotary positions of queries and keys, and their gradient
  PagedKVCache      append(): store new keys and values, rotated on the way;
                    attend(): attention of one new token per sequence

They are hand-written kernels of libpyflame_cuda.so (the pfk_* entry points of
include/pyflame_cuda.h).  Every call runs on torch's current stream of its
tensors' device, does not synchronise, and may be captured into a CUDA graph
(each captured call has its own workspace, from torch's allocator).  Arguments
are checked on the host; a wrong one raises ValueError or TypeError, a size or
layout that the kernels do not take PfcError.  Page numbers, slots and lengths
are device data: a kernel that meets a bad one skips it and sets the cache's
error flag, which `PagedKVCache.check()` raises.

A graph between them runs on the same memory by `CudaExecutor.execute_device`,
in their order if its `stream` is torch.cuda.current_stream() (without one it
runs on the executor's own stream, which waits for no other).

A handle (rotation, cache, layer) owns tables that its kernels read: keep it as
long as graphs that captured its calls.

The calls take part in no autograd graph of torch and refuse tensors that
require a gradient or carry a forward-mode tangent; RotaryEmbedding.backward is
the rotation's gradient.  They have no counterpart in PyFlame.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional

import numpy as np

from . import _native as N
from .ir import DType

_codes = None


def _code(dtype) -> int:
    """pfc_dtype of a torch dtype that the kernels take."""
    global _codes
    if _codes is None:
        import torch
        _codes = {torch.float32: int(DType.float32), torch.float16: int(DType.float16),
                  torch.bfloat16: int(DType.bfloat16)}
    c = _codes.get(dtype)
    if c is None:
        raise TypeError(f"dtype must be float32, float16 or bfloat16, not {dtype}")
    return c


def _check(name: str, t, shape, dtype, device, last_contiguous: bool = True, output: bool = False) -> None:
    """`shape` holds None where any size will do."""
    if t.dtype != dtype:
        raise TypeError(f"{name}: dtype must be {dtype}, not {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name}: is on {t.device}, not on {device}")
    if len(t.shape) != len(shape) or any(w is not None and w != s for w, s in zip(shape, t.shape)):
        raise ValueError(f"{name}: shape must be {[('any' if w is None else w) for w in shape]}, not {list(t.shape)}")
    if last_contiguous and t.shape and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}: the last axis must be contiguous")
    if t.requires_grad:
        import torch
        if torch.is_grad_enabled():
            raise RuntimeError(f"{name}: requires a gradient, which this call does not record (detach it)")
    if output and any(st == 0 and s > 1 for s, st in zip(t.shape, t.stride())):
        raise ValueError(f"{name}: an output may not have elements that share memory")


def _extent(t) -> int:
    """Bytes from a tensor's first element to behind its last."""
    return (1 + sum((n - 1) * st for n, st in zip(t.shape, t.stride()))) * t.element_size() if t.numel() else 0


class _Place:
    """The places of a tensor's elements, for numpy (which reads none of them)."""

    def __init__(self, t):
        size = t.element_size()
        self.__array_interface__ = {"version": 3, "typestr": f"|V{size}", "data": (t.data_ptr(), False), "shape": tuple(t.shape),
                                    "strides": tuple(st * size for st in t.stride())}


def _share(a, b) -> bool:
    """Whether two tensors have memory in common: exactly, also where rows of
    one lie between rows of the other."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    try:
        return np.shares_memory(np.asarray(_Place(a)), np.asarray(_Place(b)), max_work=1 << 20)
    except np.exceptions.TooHardError:  # strides that no slicing gives
        return True


def _apart(name: str, out, **others) -> None:
    """Refuses an output that shares memory with one of the others.  Callers
    ask where the extents of the two meet, which is not often."""
    for other, t in others.items():
        if _share(out, t):
            raise ValueError(f"{name}: shares memory with {other.replace('_', ' ')}")


def _no_tangents(**tensors) -> None:
    """Refuses dual tensors of forward-mode differentiation.  Not a matter of a
    call's kept checks: a tensor has a tangent or not, whatever its shape."""
    for name, t in tensors.items():
        if t is not None and _Bound.forward.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{name}: carries a tangent, which this call does not (detach it)")


def _cuda(t, name: str):
    if t.device.type != "cuda":
        raise ValueError(f"{name}: must be on a CUDA device, not on {t.device}")
    return t.device


class _Bound:
    """torch and the library's entry points, looked up once."""
    torch = forward = device = stream = rope = append = attend = linear = None

    @classmethod
    def load(cls):
        import torch
        import torch.autograd.forward_ad as forward
        L = N.lib()
        # what torch.cuda.current_device() and current_stream().cuda_stream read, without their 2 us of Python
        cls.device, cls.stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
        cls.rope, cls.append = L.pfk_rope, L.pfk_paged_append
        cls.attend, cls.linear = L.pfk_paged_attention, L.pfk_linear_w4
        cls.torch, cls.forward = torch, forward


def _call(fn, device, *args) -> None:
    """One entry point on torch's current stream of `device`."""
    index = device.index
    if _Bound.device() == index:
        rc = fn(*args, _Bound.stream(index))
    else:
        with _Bound.torch.cuda.device(device):
            rc = fn(*args, _Bound.stream(index))
    if rc:
        N.check(rc)


def _other_strides(a, b) -> bool:
    """Of two tensors of one shape: whether the same start means other places."""
    return any(n > 1 and s != r for n, s, r in zip(a.shape, a.stride(), b.stride())) and a.numel() > 0


def _model(memory, shape, dtype):
    """A tensor that outputs of known calls are made like (torch.empty_like
    takes half the time of torch.empty): one element of memory that the handle
    has anyway (int32), seen as the whole shape."""
    return memory.view(-1)[:1].view(dtype)[:1].expand(shape)


class _Plans(dict):
    """What a call's checks found, by everything about its tensors that they
    look at (types, shapes, strides, devices; never addresses or contents), so
    that a loop of like calls is checked once."""

    def keep(self, key, plan, *tensors):
        if not any(t.requires_grad for t in tensors if t is not None):  # refused or not by the grad mode of each call
            if len(self) >= 512:
                self.clear()
            self[key] = plan
        return plan


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------

def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[dict] = None):
    """(inv_freq, factor): the angle per position of each of rotary_dim / 2
    pairs, as float64, and the factor on cosines and sines.

    `scaling` stretches the positions of a model to longer contexts:
      {"type": "linear", "factor": f}   every frequency divided by f
      {"type": "ntk", "factor": f}      the base multiplied by f^(d / (d - 2)): the lowest frequency is divided by f,
                                        the highest kept
      {"type": "yarn", "factor": f, "original_max_position": n [, "beta_fast": 32, "beta_slow": 1,
       "attention_factor": 0.1 ln f + 1]}
                                        pairs that turn more than beta_fast times in n positions keep their frequency,
                                        those below beta_slow turns are divided by f, a ramp between them
    """
    if rotary_dim < 0 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and not negative")
    if not (base > 0 and math.isfinite(base)) or base == 1.0:
        raise ValueError("base must be positive, finite and not 1")
    i = np.arange(rotary_dim // 2, dtype=np.float64)
    factor = 1.0
    if scaling is None:
        return base ** (-2.0 * i / max(1, rotary_dim)), factor
    kind, f = scaling.get("type"), float(scaling.get("factor", 0.0))
    known = {"linear": {"type", "factor"}, "ntk": {"type", "factor"},
             "yarn": {"type", "factor", "original_max_position", "beta_fast", "beta_slow", "attention_factor"}}
    if kind not in known:
        raise ValueError(f"scaling type must be one of {sorted(known)}, not {kind!r}")
    if set(scaling) - known[kind]:
        raise ValueError(f"{kind} scaling has no {sorted(set(scaling) - known[kind])}")
    if not (f >= 1.0 and math.isfinite(f)):
        raise ValueError("scaling factor must be at least 1")
    if kind == "ntk":
        if rotary_dim <= 2:
            raise ValueError("ntk scaling needs rotary_dim above 2")
        base = base * f ** (rotary_dim / (rotary_dim - 2))
    inv = base ** (-2.0 * i / max(1, rotary_dim))
    if kind == "linear":
        inv = inv / f
    if kind == "yarn":
        n = float(scaling.get("original_max_position", 0))
        fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))
        if not n > 0 or not fast > slow > 0:
            raise ValueError("yarn scaling needs original_max_position > 0 and beta_fast > beta_slow > 0")

        def pair_of(turns):  # the pair that turns so often in n positions
            return rotary_dim * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(base))

        low, high = max(math.floor(pair_of(fast)), 0), min(math.ceil(pair_of(slow)), rotary_dim - 1)
        ramp = np.clip((i - low) / max(high - low, 0.001), 0.0, 1.0)
        inv = inv * (1.0 - ramp) + inv / f * ramp
        factor = float(scaling.get("attention_factor", 0.1 * math.log(f) + 1.0))
    return inv, factor


class RotaryEmbedding:
    """Rotary positions of the first `rotary_dim` values of a head.

    layout "half" turns the pairs (i, i + rotary_dim/2), "interleaved" the
    pairs (2i, 2i + 1), by position * inv_freq[i].  Angles are formed and
    reduced in two 64-bit numbers, so far positions (below 2^53) and small
    cosines lose nothing.  `inv_freq` (a sequence of rotary_dim / 2 numbers)
    replaces base and scaling (rotary_frequencies).
    """

    def __init__(self, head_dim: int, rotary_dim: Optional[int] = None, base: float = 10000.0, layout: str = "half",
                 scaling: Optional[dict] = None, inv_freq=None, factor: float = 1.0, device="cuda"):
        import torch
        _Bound.load()
        rotary_dim = head_dim if rotary_dim is None else int(rotary_dim)
        if not 1 <= head_dim <= 1024:
            raise ValueError("head_dim must be 1 to 1024")
        if not 0 <= rotary_dim <= head_dim or rotary_dim % 2:
            raise ValueError("rotary_dim must be even and at most head_dim")
        if layout not in ("half", "interleaved"):
            raise ValueError("layout must be 'half' or 'interleaved'")
        if inv_freq is None:
            inv_freq, scaled = rotary_frequencies(rotary_dim, base, scaling)
            factor = factor * scaled
        elif scaling is not None:
            raise ValueError("inv_freq and scaling exclude each other")
        inv_freq = np.asarray(inv_freq, dtype=np.float64)
        if inv_freq.shape != (rotary_dim // 2,):
            raise ValueError(f"inv_freq must hold {rotary_dim // 2} numbers")
        self.head_dim, self.rotary_dim, self.layout, self.factor = int(head_dim), rotary_dim, layout, float(factor)
        # a copy of the caller's: the device's table may not change with it
        self.inv_freq = torch.from_numpy(inv_freq.copy()).to(torch.device(device))
        _cuda(self.inv_freq, "device")
        self.device = self.inv_freq.device
        self._c = N.RotaryC(self.inv_freq.data_ptr(), rotary_dim, int(layout == "interleaved"), self.factor)
        self._plans = _Plans()
        self._kind = (self.head_dim, self.device.index)

    def _plan(self, x, positions, out, inverse: int):
        import torch
        _cuda(x, "x")
        dims = len(x.shape)
        if dims not in (3, 4):
            raise ValueError("x must be [tokens, heads, head_dim] or [batch, tokens, heads, head_dim]")
        code = _code(x.dtype)
        _check("x", x, (None,) * (dims - 1) + (self.head_dim,), x.dtype, self.device)
        batch, tokens, heads = (1,) * (4 - dims) + tuple(x.shape[:-1])
        if len(positions.shape) == 2 and dims == 4:
            _check("positions", positions, (batch, tokens), torch.int64, self.device, False)
            p_sb, p_st = positions.stride()
        else:
            _check("positions", positions, (tokens,), torch.int64, self.device, False)
            p_sb, p_st = 0, positions.stride(0)
        if out is not None:
            _check("out", out, x.shape, x.dtype, self.device, output=True)
        xs = x.stride()
        ys = torch.empty(x.shape, device="meta").stride() if out is None else out.stride()
        p = N.RopeParamsC(code, inverse, batch, tokens, heads, self.head_dim, xs[0] if dims == 4 else 0, xs[-3], xs[-2],
                          ys[0] if dims == 4 else 0, ys[-3], ys[-2], None, p_sb, p_st, self._c)
        if out is None:  # a new one meets nothing
            return p, x.is_contiguous(), 0, False
        return p, _extent(out), _extent(x), _other_strides(x, out)

    def _run(self, x, positions, out, inverse: int):
        if _Bound.forward._current_level >= 0:  # inside forward-mode differentiation
            _no_tangents(x=x, out=out)
        key = (inverse, x.dtype, x.shape, x.stride(), x.get_device(), x.requires_grad, positions.dtype, positions.shape,
               positions.stride(), positions.get_device())
        if out is not None:
            key += (out.dtype, out.shape, out.stride(), out.get_device(), out.requires_grad)
        plan = self._plans.get(key) or self._plans.keep(key, self._plan(x, positions, out, inverse), x, out)
        if out is None:
            out = _Bound.torch.empty_like(x) if plan[1] else x.new_empty(x.shape)
        at, to = x.data_ptr(), out.data_ptr()
        if at == to:
            if plan[3]:
                raise ValueError("out: shares x's memory with other strides")
        elif plan[2] and to < at + plan[2] and at < to + plan[1]:
            _apart("out", out, x=x)
        p = N.RopeParamsC.from_buffer_copy(plan[0])
        p.positions = positions.data_ptr()
        _call(_Bound.rope, self.device, at, to, C.byref(p))
        return out

    def apply(self, x, positions, out=None):
        """x rotated.  x: [tokens, heads, head_dim] or [batch, tokens, heads,
        head_dim], any strides with a contiguous head; positions: int64
        [tokens] (shared by a batch) or [batch, tokens].  `out` may be x, or
        shares no memory with it."""
        return self._run(x, positions, out, 0)

    def backward(self, dy, positions, out=None):
        """The gradient with respect to x, given the gradient dy with respect
        to apply(x, positions): the rotation by the negative angles."""
        return self._run(dy, positions, out, 1)


# ---------------------------------------------------------------------------
# paged cache
# ---------------------------------------------------------------------------

class PagedKVCache:
    """Keys and values of many sequences in pages of `page_size` tokens.

    `k` and `v` are [num_pages, page_size, num_heads, head_dim]; token i of a
    sequence is at offset i % page_size of page block_table[sequence, i //
    page_size].  Which pages a sequence owns is the caller's bookkeeping.
    """

    def __init__(self, num_pages: int, page_size: int, num_heads: int, head_dim: int, dtype=None, device="cuda"):
        import torch
        dtype = torch.float32 if dtype is None else dtype
        _code(dtype)
        shape = (int(num_pages), int(page_size), int(num_heads), int(head_dim))
        if any(s < 1 for s in shape):
            raise ValueError("sizes must be positive")
        self._take(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))

    @classmethod
    def from_tensors(cls, k, v) -> "PagedKVCache":
        """A cache in the caller's tensors, [num_pages, page_size, num_heads,
        head_dim] with the same strides and a contiguous head (heads stored
        before tokens: the permuted view).  Where they share memory, the cache
        can be attended to, not appended to."""
        self = cls.__new__(cls)
        self._take(k, v)
        return self

    def _take(self, k, v):
        import torch
        _Bound.load()
        _no_tangents(k=k, v=v)
        device = _cuda(k, "k")
        code = _code(k.dtype)
        _check("k", k, (None,) * 4, k.dtype, device, output=True)
        _check("v", v, tuple(k.shape), k.dtype, device, output=True)
        if k.stride() != v.stride():
            raise ValueError("k and v must have the same strides")
        if k.numel() == 0:
            raise ValueError("sizes must be positive")
        if k.shape[0] * k.shape[1] > 0x7FFFFFFF:
            raise ValueError("a cache holds fewer than 2^31 tokens")
        self.k, self.v, self.device, self.dtype = k, v, device, k.dtype
        self.num_pages, self.page_size, self.num_heads, self.head_dim = k.shape
        with torch.inference_mode(False):  # a tensor made in that mode could not be cleared outside it
            self._err = torch.zeros(1, dtype=torch.int32, device=device)
        self._c = N.PagedCacheC(code, k.data_ptr(), v.data_ptr(), *k.shape, *k.stride()[:3], self._err.data_ptr())
        # keys, values and what may lie between them
        self._start, self._end = min(k.data_ptr(), v.data_ptr()), max(t.data_ptr() + _extent(t) for t in (k, v))
        self._one_memory = _share(k, v)
        self._plans = _Plans()
        self._no_rotary = N.RotaryC(None, 0, 0, 1.0)

    def append(self, k, v, slots, positions=None, rotary: Optional[RotaryEmbedding] = None, q=None, q_out=None):
        """Store new tokens: k, v [tokens, num_heads, head_dim] at `slots`
        (int64 [tokens], page * page_size + offset; negative: the token is
        skipped).  With `rotary`, keys and queries q [tokens, q_heads,
        head_dim] are rotated by `positions` (int64 [tokens]); returns the
        rotated queries (`q_out`, which may be q and otherwise shares no memory
        with the inputs, or a new tensor, whose rows of skipped tokens are 0).
        The slots of one call are distinct; k, v and q may be rows of the
        cache, if the call's slots are not among them."""
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
        p = N.PagedAppendParamsC.from_buffer_copy(plan[0])
        p.k, p.v, p.slots = at_k, at_v, _ = k.data_ptr(), v.data_ptr(), slots.data_ptr()
        if rotary is not None:
            p.positions, p.rotary = positions.data_ptr(), rotary._c
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
                if (to < at_k + size_k and at_k < end or to < at_v + size_v and at_v < end
                        or to < self._end and self._start < end):
                    _apart("q_out", q_out, k=k, v=v, the_keys=self.k, the_values=self.v)
            if p.q_heads:
                p.q, p.q_out = q.data_ptr(), q_out.data_ptr()
        _call(_Bound.append, self.device, C.byref(p))
        return q_out

    def _append_plan(self, k, v, slots, positions, rotary, q, q_out):
        import torch
        n, h, d = len(k), self.num_heads, self.head_dim
        if self._one_memory:
            raise ValueError("the cache's keys share memory with its values")
        _check("k", k, (n, h, d), self.dtype, self.device)
        _check("v", v, (n, h, d), self.dtype, self.device)
        _check("slots", slots, (n,), torch.int64, self.device)
        if (rotary is None) != (positions is None):
            raise ValueError("positions and rotary go together")
        if rotary is not None:
            if rotary.head_dim != d or rotary.device != self.device:
                raise ValueError("rotary: is for another head_dim or device")
            _check("positions", positions, (n,), torch.int64, self.device)
        ks, vs, outputs = k.stride(), v.stride(), None
        p = N.PagedAppendParamsC(self._c, n, None, ks[0], ks[1], None, vs[0], vs[1])
        p.rotary = self._no_rotary
        if q is not None:
            _check("q", q, (n, None, d), self.dtype, self.device)
            qs = os = q.stride()
            if q_out is not None:
                _check("q_out", q_out, q.shape, self.dtype, self.device, output=True)
                os = q_out.stride()
                outputs = _extent(q), _extent(k), _extent(v), _extent(q_out), _other_strides(q, q_out)
            else:
                os = torch.empty(q.shape, device="meta").stride()
            p.q_heads, p.q_st, p.q_sh, p.qo_st, p.qo_sh = q.shape[1], qs[0], qs[1], os[0], os[1]
        elif q_out is not None:
            raise ValueError("q_out without q")
        return p, outputs

    def attend(self, q, block_table, seq_lens, scale: Optional[float] = None, window: int = 0, out=None,
               return_lse: bool = False):
        """Attention of one new token per sequence, its own key among the
        cached: q [batch, q_heads, head_dim] (q_heads a multiple of num_heads;
        query head h reads key-value head h // (q_heads / num_heads); head_dim
        a multiple of 8, at most 256), block_table int32 [batch, pages],
        seq_lens int32 [batch].  `scale` (1/sqrt(head_dim) by default)
        multiplies the scores; `window` > 0: only a sequence's last `window`
        tokens are seen.  A sequence of length 0 gives 0.  With return_lse also
        the natural logarithm of the sum of exp(score), float32 [batch,
        q_heads] (-inf for length 0).  `out` may be q and otherwise shares no
        memory with it or the cache.  An infinity or NaN in q or in a seen row
        may make the results that depend on it NaN."""
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
            if to < self._end and self._start < to + size:
                _apart("out", out, the_keys=self.k, the_values=self.v)
        p = N.PagedAttentionParamsC.from_buffer_copy(plan[0])
        p.q, p.out, p.block_table, p.seq_lens = at, to, block_table.data_ptr(), seq_lens.data_ptr()
        lse = None
        if return_lse:
            lse = torch.empty_like(plan[3])
            p.lse = lse.data_ptr()
        # a workspace per call, from torch's allocator: calls on several streams and captured graphs share none
        if plan[2]:
            work = torch.empty(plan[2], dtype=torch.uint8, device=self.device)
            p.workspace = work.data_ptr()
        _call(_Bound.attend, self.device, C.byref(p))
        return (out, lse) if return_lse else out

    def _attend_plan(self, q, block_table, seq_lens, scale, window, out, return_lse):
        import torch
        if len(q.shape) != 3:
            raise ValueError("q must be [batch, q_heads, head_dim]")
        batch, heads, d = q.shape
        _check("q", q, (None, None, self.head_dim), self.dtype, self.device)
        if heads == 0 or heads % self.num_heads:
            raise ValueError(f"q: {heads} heads are not a multiple of {self.num_heads}")
        _check("block_table", block_table, (batch, None), torch.int32, self.device)
        _check("seq_lens", seq_lens, (batch,), torch.int32, self.device)
        if window < 0:
            raise ValueError("window must not be negative")
        scale = 1.0 / math.sqrt(d) if scale is None else scale
        if out is not None:
            _check("out", out, (batch, heads, d), self.dtype, self.device, output=True)
        qs = q.stride()
        os = torch.empty(q.shape, device="meta").stride() if out is None else out.stride()
        p = N.PagedAttentionParamsC(self._c, batch, heads, None, qs[0], qs[1], None, os[0], os[1], None, None,
                                    block_table.stride(0), block_table.shape[1], None, window, scale)
        size = C.c_size_t(0)
        with torch.cuda.device(self.device):
            N.check(N.lib().pfk_paged_attention_workspace(C.byref(p), C.byref(size)))
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
            raise N.PfcError(code, "a call met a slot, page or length outside the paged cache")


# ---------------------------------------------------------------------------
# 4-bit weights
# ---------------------------------------------------------------------------

class Linear4bit:
    """y = x W^T + bias with W[n, k] = (q[n, k] - zeros[n, k // group]) *
    scales[n, k // group], q from 0 to 15.

    packed: uint8 [out_features, (in_features + 1) // 2], column 2i in the low
    half of byte i; scales: float16 or bfloat16 [out_features,
    ceil(in_features / group_size)]; zeros: uint8 of the same shape, 0 to 15,
    or None for 8; bias: [out_features] of the type of x, or None; group_size:
    32, 64 or a multiple of 128.  The constructor lays the weights out for the
    kernel once.  For single tokens and batches of up to some tens of rows;
    more rows read and unpack the weights again for every 48 (16 in float32).
    """

    def __init__(self, packed, scales, zeros=None, bias=None, in_features: Optional[int] = None, group_size: int = 128):
        import torch
        _Bound.load()
        _no_tangents(scales=scales, bias=bias)
        device = _cuda(packed, "packed")
        if len(packed.shape) != 2 or 0 in packed.shape:
            raise ValueError("packed must be [out_features, (in_features + 1) // 2]")
        n = packed.shape[0]
        k = 2 * packed.shape[1] if in_features is None else int(in_features)
        if k < 1 or group_size not in (32, 64) and (group_size < 128 or group_size % 128):
            raise ValueError("group_size must be 32, 64 or a multiple of 128, in_features positive")
        groups = -(-k // group_size)
        _check("packed", packed, (n, (k + 1) // 2), torch.uint8, device)
        if scales.dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"scales: dtype must be float16 or bfloat16, not {scales.dtype}")
        _check("scales", scales, (n, groups), scales.dtype, device)
        if zeros is not None:
            _check("zeros", zeros, (n, groups), torch.uint8, device)
            if int(zeros.max()) > 15:
                raise ValueError("zeros must be 0 to 15")
            zeros = zeros.contiguous()
        if bias is not None:
            _code(bias.dtype)
            _check("bias", bias, (n,), bias.dtype, device, False)
            bias = bias.contiguous()
        self.in_features, self.out_features, self.group_size = k, n, int(group_size)
        self.device, self.scales, self.zeros, self.bias = device, scales.contiguous(), zeros, bias
        self._bias_start, self._bias_end = (0, 0) if bias is None else (bias.data_ptr(), bias.data_ptr() + _extent(bias))
        blocks, row_blocks = -(-k // 128), -(-n // 16)
        self.weight = torch.empty((row_blocks, blocks, 256), dtype=torch.int32, device=device)
        self.meta = torch.empty((row_blocks, blocks * (128 // group_size) if group_size < 128 else groups, 16), dtype=torch.int32,
                                device=device)
        self._plans = _Plans()
        packed = packed.contiguous()
        p = N.W4ArrangeParamsC(k, n, self.group_size, packed.data_ptr(), self.scales.data_ptr(), _code(scales.dtype),
                               None if zeros is None else zeros.data_ptr(), self.weight.data_ptr(), self.meta.data_ptr())
        _call(N.lib().pfk_w4_arrange, device, C.byref(p))

    @classmethod
    def quantize(cls, weight, group_size: int = 128, bias=None, symmetric: bool = False, scale_dtype=None) -> "Linear4bit":
        """Weights [out_features, in_features] rounded to 4 bits: the nearest
        of 16 evenly spaced values that cover each group's range and 0
        (symmetric: 15 steps around 8).  Scales are float16, or bfloat16 where
        one is outside float16's normal range."""
        import torch
        _cuda(weight, "weight")
        if len(weight.shape) != 2 or 0 in weight.shape:
            raise ValueError("weight must be [out_features, in_features]")
        if group_size not in (32, 64) and (group_size < 128 or group_size % 128):
            raise ValueError("group_size must be 32, 64 or a multiple of 128")
        weight = weight.detach().float()
        if not bool(torch.isfinite(weight).all()):
            raise ValueError("weight: holds an infinity or NaN")
        n, k = weight.shape
        groups = -(-k // group_size)
        w = torch.zeros((n, groups * group_size), dtype=torch.float32, device=weight.device)
        w[:, :k] = weight
        w = w.view(n, groups, group_size)
        if symmetric:
            scale = w.abs().amax(-1) / 7.0
        else:
            low, high = w.amin(-1).clamp(max=0.0), w.amax(-1).clamp(min=0.0)
            scale = high / 15.0 - low / 15.0
        if scale_dtype is None:
            normal = (scale == 0) | ((scale >= 2.0 ** -14) & (scale <= 65504.0))
            scale_dtype = torch.float16 if bool(normal.all()) else torch.bfloat16
        scales = scale.to(scale_dtype)
        if not bool(torch.isfinite(scales).all()):
            raise ValueError(f"weight: too large for scales of {scale_dtype}")
        s = scales.float()
        step = torch.where(s > 0, s, torch.ones_like(s))
        zeros = None if symmetric else (-low / step).round().clamp(0, 15)
        z = 8.0 if symmetric else zeros[..., None]
        q = ((w / step[..., None]).round() + z).clamp(0, 15).to(torch.uint8).view(n, -1)[:, :(k + 1) // 2 * 2]
        packed = q[:, 0::2] | (q[:, 1::2] << 4)
        return cls(packed, scales, None if symmetric else zeros.to(torch.uint8), bias, k, group_size)

    def __call__(self, x, out=None):
        """x: [..., in_features]; `out`, [..., out_features], shares no memory
        with it.  Rows at one stride are read where they are."""
        if _Bound.forward._current_level >= 0:  # inside forward-mode differentiation
            _no_tangents(x=x, out=out)
        key = (x.dtype, x.shape, x.stride(), x.get_device(), x.requires_grad)
        if out is not None:
            key += (out.dtype, out.shape, out.stride(), out.get_device(), out.requires_grad)
        plan = self._plans.get(key) or self._plans.keep(key, self._plan(x, out), x, out)
        if plan[1]:
            x = x.reshape(-1, self.in_features)
        if out is None:
            out = _Bound.torch.empty_like(plan[2])
        else:
            at, to = x.data_ptr(), out.data_ptr()
            if at < to + plan[3] and to < at + plan[4]:
                _apart("out", out, x=x)
            if to < self._bias_end and self._bias_start < to + plan[3]:
                _apart("out", out, the_bias=self.bias)
        p = N.LinearW4ParamsC.from_buffer_copy(plan[0])
        p.x, p.y = x.data_ptr(), out.data_ptr()
        _call(_Bound.linear, self.device, C.byref(p))
        return out

    def _plan(self, x, out):
        _cuda(x, "x")
        code = _code(x.dtype)
        if len(x.shape) < 1:
            raise ValueError("x must be [..., in_features]")
        _check("x", x, (None,) * (len(x.shape) - 1) + (self.in_features,), x.dtype, self.device)
        if self.bias is not None and self.bias.dtype != x.dtype:
            raise TypeError(f"x: dtype must be the bias's, {self.bias.dtype}, not {x.dtype}")
        rows = x if len(x.shape) == 2 else x.reshape(-1, self.in_features)
        shape = tuple(x.shape[:-1]) + (self.out_features,)
        y_st = self.out_features
        if out is not None:
            _check("out", out, shape, x.dtype, self.device, output=True)
            try:
                y_st = (out if len(shape) == 2 else out.view(-1, self.out_features)).stride(0)
            except RuntimeError:
                raise ValueError("out: its rows must be at one stride") from None
        p = N.LinearW4ParamsC(code, rows.shape[0], self.in_features, self.out_features, self.group_size, None,
                              rows.stride(0), None, y_st, self.weight.data_ptr(), self.meta.data_ptr(),
                              None if self.bias is None else self.bias.data_ptr())
        return (p, len(x.shape) != 2, _model(self.weight, shape, x.dtype) if out is None else None,
                0 if out is None else _extent(out), _extent(rows))
