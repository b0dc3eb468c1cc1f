"""The norms around the MoE layer, fused with the block's gate, residual scale
and residual add, with gradients (``csrc/norm.cuh``). No counterpart in the
reference, whose layer starts and ends inside the model's own block code.

    h = rms_norm(x, pre_weight)                       # the norm before the block
    y = moe_layer_forward(h, ...).out
    x, h = norm_gate_residual(y, x, post_weight, next_weight, gate=g, residual_scale=a)

where the last line is one launch: x + a * g * rmsnorm(y) * post_weight and, if
``next_weight`` is given, the norm before the next block of that sum.
``layer.moe_block_forward`` is the whole block."""

from __future__ import annotations

import ctypes

import torch

from dispatch_b200 import _lib as L


def _rows(t: torch.Tensor, h: int) -> tuple[torch.Tensor, int]:
    """``t`` (..., h) as rows with unit last stride, and their stride; copied
    only if its rows do not lie at one stride of at least h."""
    r = t.reshape(-1, h)
    if r.stride(1) != 1 and h > 1:
        r = r.contiguous()
    if r.shape[0] <= 1:
        return r, h
    if r.stride(0) < h:
        r = r.contiguous()
    return r, r.stride(0)


def _gate_mode(gate: torch.Tensor | None, y: torch.Tensor) -> int:
    if gate is None:
        return L.GATE_NONE
    if gate.shape == y.shape:
        return L.GATE_FULL
    if gate.shape == y.shape[-1:]:
        return L.GATE_CHANNEL
    if gate.dim() == y.dim() and gate.shape == (*y.shape[:-1], 1):
        return L.GATE_TOKEN
    raise ValueError(f"gate.shape {tuple(gate.shape)} must be one value per channel, per token or per value of "
                     f"{tuple(y.shape)}")


class _Call:
    """Checked arguments of one call, as the C ABI takes them."""

    def __init__(self, what, y, residual, post_weight, next_weight, gate, residual_scale, eps, norm_dtype, *grads):
        self.dev = L.require_cuda(y, residual, post_weight, next_weight, gate, *grads, what=what)
        if residual.dim() < 1 or residual.shape[-1] < 1:
            raise ValueError(f"{what}: expected (..., H) with H >= 1, got {tuple(residual.shape)}")
        if y is not None and y.shape != residual.shape:
            raise ValueError(f"{what}: y.shape {tuple(y.shape)} != residual.shape {tuple(residual.shape)}")
        self.shape, h = residual.shape, residual.shape[-1]
        for name, w in (("post_weight", post_weight), ("next_weight", next_weight)):
            if w is not None and w.shape != (h,):
                raise ValueError(f"{what}: {name}.shape {tuple(w.shape)} != ({h},)")
        if y is None and next_weight is None:
            raise ValueError(f"{what}: nothing to compute without y and next_weight")
        mode = _gate_mode(gate, residual)
        d = self.desc = L.MoeNormDesc()
        self.residual, d.res_stride = _rows(residual.detach(), h)
        d.T, d.H = self.residual.shape
        self.y = self.gate = None
        if y is not None:
            self.y, d.y_stride = _rows(y.detach(), h)
            d.y_dtype = L.dt(y)
        if gate is not None:
            d.gate_dtype = L.dt(gate)
            if mode == L.GATE_FULL:
                self.gate, d.gate_stride = _rows(gate.detach(), h)
            elif mode == L.GATE_TOKEN:
                self.gate = gate.detach().reshape(-1, 1)
                d.gate_stride = self.gate.stride(0)
            else:
                self.gate = gate.detach().contiguous()
        d.gate_mode = mode
        d.res_dtype = L.dt(residual)
        self.post = None if post_weight is None else post_weight.detach().contiguous()
        self.next = None if next_weight is None else next_weight.detach().contiguous()
        d.post_dtype = 0 if post_weight is None else L.dt(post_weight)
        d.next_dtype = 0 if next_weight is None else L.dt(next_weight)
        self.norm_dtype = norm_dtype or residual.dtype
        d.norm_dtype = L.dt(self.norm_dtype)
        d.residual_scale, d.eps = float(residual_scale), float(eps)

    def inputs(self):
        return L.ptr(self.y), self.residual.data_ptr(), L.ptr(self.post), L.ptr(self.next), L.ptr(self.gate)


def _forward(what, y, residual, post_weight, next_weight, gate, residual_scale, eps, norm_dtype):
    c = _Call(what, y, residual, post_weight, next_weight, gate, residual_scale, eps, norm_dtype)
    out = torch.empty(c.shape, dtype=residual.dtype, device=c.dev) if y is not None else None
    normed = torch.empty(c.shape, dtype=c.norm_dtype, device=c.dev) if next_weight is not None else None
    with L.device_guard(c.dev):
        rc = L.lib().moe_norm_gate_residual(ctypes.byref(c.desc), *c.inputs(), L.ptr(out), L.ptr(normed),
                                            L.stream_ptr(c.dev))
    L.check(rc, what)
    return out, normed


def _backward(what, d_out, d_normed, y, residual, post_weight, next_weight, gate, residual_scale, eps, needs):
    norm_dtype = residual.dtype if d_normed is None else d_normed.dtype
    c = _Call(what, y, residual, post_weight, next_weight, gate, residual_scale, eps, norm_dtype, d_out, d_normed)
    h = c.shape[-1]
    for name, g in (("d_out", d_out), ("d_normed", d_normed)):
        if g is not None and g.shape != c.shape:
            raise ValueError(f"{what}: {name}.shape {tuple(g.shape)} != {tuple(c.shape)}")
    if d_normed is not None and next_weight is None:
        raise ValueError(f"{what}: d_normed needs next_weight")
    s_out = s_normed = h
    if d_out is not None:
        d_out, s_out = _rows(d_out.detach().to(residual.dtype), h)
    if d_normed is not None:
        d_normed, s_normed = _rows(d_normed.detach(), h)
    like = (y, residual, post_weight, next_weight, gate)
    grads = [torch.empty(t.shape, dtype=t.dtype, device=c.dev) if t is not None and n else None
             for t, n in zip(like, needs)]
    ws = None
    if grads[2] is not None or grads[3] is not None or (grads[4] is not None and c.desc.gate_mode == L.GATE_CHANNEL):
        # per call, not cached: a captured graph then owns the workspace it replays on
        ws = torch.empty(L.lib().moe_norm_backward_workspace_bytes(c.desc.T, h), dtype=torch.uint8, device=c.dev)
    with L.device_guard(c.dev):
        rc = L.lib().moe_norm_gate_residual_backward(
            ctypes.byref(c.desc), L.ptr(d_out), s_out, L.ptr(d_normed), s_normed, *c.inputs(),
            *(L.ptr(g) for g in grads), L.ptr(ws), 0 if ws is None else ws.numel(), L.stream_ptr(c.dev),
        )
    L.check(rc, what)
    return tuple(grads)


class _NormGateResidual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, residual, post_weight, next_weight, gate, residual_scale, eps, norm_dtype):
        ctx.save_for_backward(y, residual, post_weight, next_weight, gate)
        ctx.residual_scale, ctx.eps = residual_scale, eps
        ctx.set_materialize_grads(False)
        return _forward("norm_gate_residual", y, residual, post_weight, next_weight, gate, residual_scale, eps,
                        norm_dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out, d_normed):
        if d_out is None and d_normed is None:
            return (None,) * 8
        grads = _backward("norm_gate_residual", d_out, d_normed, *ctx.saved_tensors, ctx.residual_scale, ctx.eps,
                          ctx.needs_input_grad[:5])
        return *grads, None, None, None


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps, out_dtype):
        ctx.save_for_backward(x, weight)
        ctx.eps = eps
        return _forward("rms_norm", None, x, None, weight, None, 1.0, eps, out_dtype)[1]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_normed):
        x, weight = ctx.saved_tensors
        need_x, need_w = ctx.needs_input_grad[:2]
        _, dx, _, dw, _ = _backward("rms_norm", None, d_normed, None, x, None, weight, None, 1.0, ctx.eps,
                                    (False, need_x, False, need_w, False))
        return dx, dw, None, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6,
             out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """x * rsqrt(mean(x^2) + eps) * weight over the last dimension, in f32,
    rounded once to ``out_dtype`` (default: x's type). x (..., H) and weight
    (H,) in bf16, f16 or f32 each, H up to 16384, rows at any stride.
    Differentiable in both."""
    if L.grad_wanted("rms_norm", x, weight):
        return _RmsNorm.apply(x, weight, eps, out_dtype)
    return _forward("rms_norm", None, x, None, weight, None, 1.0, eps, out_dtype)[1]


def rms_norm_backward(d_normed: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, *,
                      eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """The gradients (dx, dweight) of ``rms_norm``, in x's and weight's types."""
    _, dx, _, dw, _ = _backward("rms_norm_backward", None, d_normed, None, x, None, weight, None, 1.0, eps,
                                (False, True, False, True, False))
    return dx, dw


def norm_gate_residual(
    y: torch.Tensor, residual: torch.Tensor, post_weight: torch.Tensor | None = None,
    next_weight: torch.Tensor | None = None, *, gate: torch.Tensor | None = None, residual_scale: float = 1.0,
    eps: float = 1e-6, norm_dtype: torch.dtype | None = None,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """The end of a block, (out, normed), in one launch:

        out    = residual + residual_scale * gate * rmsnorm(y) * post_weight
        normed = rmsnorm(out) * next_weight

    all in f32, each output rounded once; the second norm reads the unrounded
    sum. y and residual (..., H), bf16, f16 or f32 each (a 16-bit branch on an
    f32 residual stream is fine); out has residual's type, normed
    ``norm_dtype`` (default: residual's). Without ``post_weight`` y is added
    as it is; without ``next_weight`` normed is None. ``gate``: (H,) per
    channel, (..., 1) per token or (..., H) per value. Differentiable in y,
    residual, the weights and the gate."""
    if y is None:
        raise ValueError("norm_gate_residual needs y; rms_norm is the norm alone")
    if L.grad_wanted("norm_gate_residual", y, residual, post_weight, next_weight, gate):
        return _NormGateResidual.apply(y, residual, post_weight, next_weight, gate, residual_scale, eps, norm_dtype)
    return _forward("norm_gate_residual", y, residual, post_weight, next_weight, gate, residual_scale, eps, norm_dtype)


def norm_gate_residual_backward(
    d_out: torch.Tensor | None, d_normed: torch.Tensor | None, y: torch.Tensor, residual: torch.Tensor,
    post_weight: torch.Tensor | None = None, next_weight: torch.Tensor | None = None, *,
    gate: torch.Tensor | None = None, residual_scale: float = 1.0, eps: float = 1e-6,
) -> tuple[torch.Tensor | None, ...]:
    """The gradients (dy, dresidual, dpost_weight, dnext_weight, dgate) of
    ``norm_gate_residual``, each in its input's type and shape, None for an
    absent input. ``d_out`` or ``d_normed`` may be None (zero). The column
    sums (weights, a gate per channel) are f32, in a fixed order."""
    if y is None:
        raise ValueError("norm_gate_residual_backward needs y; rms_norm_backward is the norm alone")
    return _backward("norm_gate_residual_backward", d_out, d_normed, y, residual, post_weight, next_weight, gate,
                     residual_scale, eps, (True,) * 5)
