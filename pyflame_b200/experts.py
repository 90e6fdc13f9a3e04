"""A mixture-of-experts layer for a few tokens.

  MixtureOfExperts  router, choice of experts, and the chosen experts' gated
                    feed-forward products

Hand-written kernels of libpyflame_cuda.so, on the terms of decoding.py
(streams, capture into CUDA graphs, errors, gradients).  They have no
counterpart in PyFlame.
"""
from __future__ import annotations

import ctypes as C

from . import _native as N
from .decoding import _apart, _Bound, _call, _check, _code, _cuda, _extent, _model, _no_tangents, _other_strides, _Plans


class MixtureOfExperts:
    """y = sum over the top_k experts with the largest router logits of weight
    * down_e (act(gate_e x) * (up_e x)).

    router: [experts, width]; gate_up: [experts, 2 * inner, width], the gate's
    rows, then the other factor's; down: [experts, width, inner], of the type
    of x.  Logits are taken in 64 bits (ties go to the lower expert, a NaN
    counts as the lowest); weights are the softmax of the chosen logits, or,
    without `renormalize`, their part of the softmax over all experts.
    activation: "silu" or "gelu" (tanh form).  Up to 1024 experts, top_k up to
    32, width and inner up to 65536.

    The router is copied (as float32).  gate_up and down are used where they
    are, if they are dense and their rows multiples of 16 bytes, else copied
    once.  For the tokens of a decoding step: up to 8 tokens read their experts'
    weights once, more once for every 16 of the tokens that chose the expert
    (from L2 again where they are still there), 128 at a time.
    """

    def __init__(self, router, gate_up, down, top_k: int, renormalize: bool = True, activation: str = "silu"):
        import torch
        _Bound.load()
        _no_tangents(router=router, gate_up=gate_up, down=down)
        device = _cuda(gate_up, "gate_up")
        router, gate_up, down = router.detach(), gate_up.detach(), down.detach()
        code = _code(gate_up.dtype)
        if len(gate_up.shape) != 3 or gate_up.shape[1] % 2 or 0 in gate_up.shape:
            raise ValueError("gate_up must be [experts, 2 * inner, width]")
        e, f, d = gate_up.shape[0], gate_up.shape[1] // 2, gate_up.shape[2]
        _check("gate_up", gate_up, (e, 2 * f, d), gate_up.dtype, device, False)
        _check("down", down, (e, d, f), gate_up.dtype, device, False)
        _code(router.dtype)
        _check("router", router, (e, d), router.dtype, device, False)
        if activation not in ("silu", "gelu"):
            raise ValueError("activation must be 'silu' or 'gelu'")
        if not 1 <= top_k <= min(e, 32):
            raise ValueError("top_k must be 1 to 32 and at most the number of experts")
        if e > 1024:
            raise ValueError("at most 1024 experts")
        if max(d, f) > 65536:
            raise ValueError("width and inner must be at most 65536")
        self.num_experts, self.width, self.inner, self.top_k = e, d, f, int(top_k)
        self.dtype, self.device, self.renormalize, self.activation = gate_up.dtype, device, bool(renormalize), activation

        def rows(w, step):  # dense rows of multiples of `step`, zeros behind the values
            w = torch.nn.functional.pad(w, (0, -w.shape[-1] % step)) if w.shape[-1] % step else w.contiguous()
            return w if w.data_ptr() % 16 == 0 else w.clone()

        vec = 16 // gate_up.element_size()
        with torch.no_grad(), torch.cuda.device(device):
            self.router = rows(router.float().clone(), 4)
            self.gate_up, self.down = rows(gate_up, vec), rows(down, vec)
        self._base = N.ExpertsParamsC(code, int(activation == "gelu"), int(self.renormalize), 0, d, f, e, self.top_k)
        p = self._base
        p.router, p.router_st = self.router.data_ptr(), self.router.shape[-1]
        p.gate_up, p.gate_up_st = self.gate_up.data_ptr(), self.gate_up.shape[-1]
        p.down, p.down_st = self.down.data_ptr(), self.down.shape[-1]
        self._plans = _Plans()
        self._fn = N.lib().pfk_experts

    def __call__(self, x, out=None, return_routing: bool = False):
        """x: [..., width]; returns y like x, and with return_routing also the
        chosen experts, int32 [..., top_k], best first, and their weights,
        float32.  `out` may be x and otherwise shares no memory with it.  Rows
        at one stride are read where they are.  An infinity or NaN in x or in
        a chosen expert's weights may make the results that depend on it
        NaN."""
        if _Bound.forward._current_level >= 0:  # inside forward-mode differentiation
            _no_tangents(x=x, out=out)
        torch = _Bound.torch
        key = (return_routing, x.dtype, x.shape, x.stride(), x.get_device(), x.requires_grad)
        if out is not None:
            key += (out.dtype, out.shape, out.stride(), out.get_device(), out.requires_grad)
        plan = self._plans.get(key) or self._plans.keep(key, self._plan(x, out, return_routing), x, out)
        p = N.ExpertsParamsC.from_buffer_copy(plan[0])
        if out is None:
            out = torch.empty_like(plan[1])
        else:
            size_x, size, other = plan[3]
            at, to = x.data_ptr(), out.data_ptr()
            if at == to:
                if other:
                    raise ValueError("out: shares x's memory with other strides")
            elif to < at + size_x and at < to + size:
                _apart("out", out, x=x)
        rows = x.reshape(-1, self.width) if plan[2] else x
        p.x, p.y = rows.data_ptr(), out.data_ptr()
        chosen = weights = None
        if return_routing:
            chosen, weights = torch.empty_like(plan[4]), torch.empty_like(plan[5])
            p.chosen, p.weights = chosen.data_ptr(), weights.data_ptr()
        # a workspace per call, from torch's allocator: calls on several streams and captured graphs share none
        if p.workspace_bytes:
            work = torch.empty(p.workspace_bytes, dtype=torch.uint8, device=self.device)
            p.workspace = work.data_ptr()
        _call(self._fn, self.device, C.byref(p))
        return (out, chosen, weights) if return_routing else out

    def _plan(self, x, out, return_routing):
        import torch
        _cuda(x, "x")
        if len(x.shape) < 1:
            raise ValueError("x must be [..., width]")
        lead = tuple(x.shape[:-1])
        _check("x", x, lead + (self.width,), self.dtype, self.device)
        flat = len(lead) != 1
        rows = x.reshape(-1, self.width) if flat else x
        p = N.ExpertsParamsC.from_buffer_copy(self._base)
        p.tokens, p.x_st, p.y_st = rows.shape[0], rows.stride(0), self.width
        if out is not None:
            _check("out", out, x.shape, self.dtype, self.device, output=True)
            try:
                p.y_st = (out.view(-1, self.width) if flat else out).stride(0)
            except RuntimeError:
                raise ValueError("out: its rows must be at one stride") from None
        size = C.c_size_t(0)
        N.check(N.lib().pfk_experts_workspace(C.byref(p), C.byref(size)))
        p.workspace_bytes = size.value
        memory = self.router
        return (p, _model(memory, x.shape, self.dtype) if out is None else None, flat,
                None if out is None else (_extent(x), _extent(out), _other_strides(x, out)),
                _model(memory, lead + (self.top_k,), torch.int32) if return_routing else None,
                _model(memory, lead + (self.top_k,), torch.float32) if return_routing else None)
