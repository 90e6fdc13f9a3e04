"""Low-rank adapters of many requests at once, beside a shared projection.

  LowRankAdapters  out = base + scale_i * B_i (A_i x), each row of x with the
                   adapter i that its request names

Hand-written kernels of libpyflame_cuda.so, on the terms of decoding.py
(streams, capture into CUDA graphs, errors, gradients).  They have no
counterpart in PyFlame.
"""
from __future__ import annotations

import ctypes as C

from . import _native as N
from .decoding import _apart, _Bound, _call, _check, _code, _extent, _model, _no_tangents, _other_strides, _Plans


class LowRankAdapters:
    """`num_adapters` adapters of one projection, in_features to out_features,
    of ranks up to `max_rank` (at most 256; the memory is that of the next
    multiple of 16).  An adapter is in place after load() and adds nothing
    before.

    Rows of x may come in any order.  Those of one request lie best together:
    32 neighbouring rows are worked on at once, and each adapter among them is
    read once for them.
    """

    def __init__(self, num_adapters: int, in_features: int, out_features: int, max_rank: int, dtype=None, device="cuda"):
        import torch
        _Bound.load()
        n, k, m, r = (int(s) for s in (num_adapters, in_features, out_features, max_rank))
        if min(n, k, m, r) < 1:
            raise ValueError("sizes must be positive")
        if r > 256:
            raise ValueError("max_rank must be at most 256")
        dtype = torch.float32 if dtype is None else dtype
        code = _code(dtype)
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError(f"device: must be a CUDA device, not {device}")
        self.num_adapters, self.in_features, self.out_features, self.max_rank, self.dtype = n, k, m, r, dtype
        rank, row = -(-r // 16) * 16, -(-k // 8) * 8
        with torch.inference_mode(False):  # a tensor made in that mode could not be written outside it
            self._a = torch.zeros((n, rank, row), dtype=dtype, device=device)
            self._b = torch.zeros((n, m, rank), dtype=dtype, device=device)
            self._scales = torch.zeros(n, dtype=torch.float32, device=device)
            self._err = torch.zeros(1, dtype=torch.int32, device=device)
        self.device = self._a.device
        self._base = N.AdaptersParamsC(code, 0, k, m, n, rank)
        p = self._base
        p.a, p.a_st, p.b, p.scales, p.err = self._a.data_ptr(), row, self._b.data_ptr(), self._scales.data_ptr(), self._err.data_ptr()
        self._plans = _Plans()
        self._fn = N.lib().pfk_adapters

    def load(self, i: int, a, b, scale: float = 1.0) -> None:
        """Puts an adapter in place `i`: a [rank, in_features], b
        [out_features, rank], copied on torch's current stream."""
        import torch
        if not 0 <= i < self.num_adapters:
            raise IndexError(f"adapter {i} of {self.num_adapters}")
        _no_tangents(a=a, b=b)
        if len(a.shape) != 2 or not 1 <= a.shape[0] <= self.max_rank:
            raise ValueError(f"a must be [rank, in_features] with a rank of 1 to {self.max_rank}")
        r = a.shape[0]
        a, b = a.detach(), b.detach()
        _check("a", a, (r, self.in_features), self.dtype, self.device, False)
        _check("b", b, (self.out_features, r), self.dtype, self.device, False)
        with torch.no_grad():
            mine_a, mine_b = self._a[i], self._b[i]
            mine_a[:r, :self.in_features].copy_(a)
            mine_b[:, :r].copy_(b)
            if r < len(mine_a):
                mine_a[r:].zero_()
                mine_b[:, r:].zero_()
            self._scales[i] = float(scale)

    def __call__(self, x, index, base=None, out=None):
        """base + the adapters' part: x [..., in_features], index int32
        [...] (negative: no adapter; one that is not there sets the flag of
        check(), and its row is as without), base [..., out_features] or None
        for 0.  Sums are held in float32 and the result is rounded once.  `out`
        may be base and otherwise shares no memory with the inputs.  Rows at
        one stride are read where they are.  An infinity or NaN in x or in an
        adapter may make the results that depend on it NaN."""
        if _Bound.forward._current_level >= 0:  # inside forward-mode differentiation
            _no_tangents(x=x, base=base, out=out)
        key = (x.dtype, x.shape, x.stride(), x.get_device(), x.requires_grad, index.dtype, index.shape, index.stride(),
               index.get_device(),
               None if base is None else (base.dtype, base.shape, base.stride(), base.get_device(), base.requires_grad),
               None if out is None else (out.dtype, out.shape, out.stride(), out.get_device(), out.requires_grad))
        plan = self._plans.get(key) or self._plans.keep(key, self._plan(x, index, base, out), x, base, out)
        p = N.AdaptersParamsC.from_buffer_copy(plan[0])
        if plan[1]:  # not rows yet; an input whose rows lie at several strides is copied
            x, index = x.reshape(-1, self.in_features), index.reshape(-1)
            if base is not None:
                rows = base.reshape(-1, self.out_features)
        else:
            rows = base
        if plan[2]:
            index = index.contiguous()
        if out is None:
            out = _Bound.torch.empty_like(plan[3])
        else:
            size, size_x, size_index, size_base, other = plan[4]
            to, at, at_i = out.data_ptr(), x.data_ptr(), index.data_ptr()
            if to < at + size_x and at < to + size or to < at_i + size_index and at_i < to + size:
                _apart("out", out, x=x, index=index)
            if base is not None:
                at = base.data_ptr()
                if at == to:
                    if other:
                        raise ValueError("out: shares base's memory with other strides")
                elif at < to + size and to < at + size_base:
                    _apart("out", out, base=base)
        p.x, p.index, p.out = x.data_ptr(), index.data_ptr(), out.data_ptr()
        if base is not None:
            p.base = rows.data_ptr()
        _call(self._fn, self.device, C.byref(p))
        return out

    def _plan(self, x, index, base, out):
        import torch
        if len(x.shape) < 1:
            raise ValueError("x must be [..., in_features]")
        lead = tuple(x.shape[:-1])
        _check("x", x, lead + (self.in_features,), self.dtype, self.device)
        _check("index", index, lead, torch.int32, self.device, False)
        shape = lead + (self.out_features,)
        flat = len(lead) != 1
        rows = x.reshape(-1, self.in_features) if flat else x
        p = N.AdaptersParamsC.from_buffer_copy(self._base)
        p.rows, p.x_st = rows.shape[0], rows.stride(0)
        size_base, other = 0, False
        if base is not None:
            _check("base", base, shape, self.dtype, self.device)
            p.base_st = (base.reshape(-1, self.out_features) if flat else base).stride(0)
            size_base = _extent(base)
        p.out_st = self.out_features
        if out is not None:
            _check("out", out, shape, self.dtype, self.device, output=True)
            try:
                p.out_st = (out.view(-1, self.out_features) if flat else out).stride(0)
            except RuntimeError:
                raise ValueError("out: its rows must be at one stride") from None
            if base is not None:
                other = _other_strides(base, out)
        i = index.reshape(-1)
        return (p, flat, i.numel() > 1 and i.stride(0) != 1, _model(self._err, shape, self.dtype) if out is None else None,
                None if out is None else (_extent(out), _extent(rows), 4 * i.numel(), size_base, other))

    def check(self) -> None:
        """Wait for the device and raise PfcError if a call met an index that
        names no adapter since the last check."""
        _Bound.torch.cuda.synchronize(self.device)
        code = int(self._err.item())
        if code:
            self._err.zero_()
            # finished here: later, it would clear the flag of a call on another stream
            _Bound.torch.cuda.synchronize(self.device)
            raise N.PfcError(code, "a call met an index that names no adapter")
