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
    if t.is_contiguous():
        return t, h
    r = t.detach().reshape(-1, h)
    if (r.stride(1) != 1 and h > 1) or (r.shape[0] > 1 and r.stride(0) < h):
        r = r.contiguous()
    return r, r.stride(0) if r.shape[0] > 1 else h


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


def _describe(what, y, residual, post_weight, next_weight, gate, residual_scale, eps, norm_dtype, *grads):
    """The device, the descriptor and the (kept alive) inputs of one call, all
    checked, as the C ABI takes them."""
    dev = L.require_cuda(y, residual, post_weight, next_weight, gate, *grads, what=what)
    shape = residual.shape
    h = shape[-1] if len(shape) else 0
    if h < 1:
        raise ValueError(f"{what}: expected (..., H) with H >= 1, got {tuple(shape)}")
    if y is None:
        if next_weight is None:
            raise ValueError(f"{what}: nothing to compute without y and next_weight")
    elif y.shape != shape:
        raise ValueError(f"{what}: y.shape {tuple(y.shape)} != residual.shape {tuple(shape)}")
    for name, w in (("post_weight", post_weight), ("next_weight", next_weight)):
        if w is not None and w.shape != (h,):
            raise ValueError(f"{what}: {name}.shape {tuple(w.shape)} != ({h},)")
    mode = _gate_mode(gate, residual)
    d = L.MoeNormDesc()
    d.T, d.H = residual.numel() // h, h
    residual, d.res_stride = _rows(residual, h)
    d.res_dtype = L.dt(residual)
    if y is not None:
        y, d.y_stride = _rows(y, h)
        d.y_dtype = L.dt(y)
    if gate is not None:
        d.gate_dtype = L.dt(gate)
        if mode == L.GATE_FULL:
            gate, d.gate_stride = _rows(gate, h)
        elif mode == L.GATE_TOKEN:
            gate = gate.detach().reshape(-1, 1)
            d.gate_stride = gate.stride(0)
        else:
            gate = gate.contiguous()
        d.gate_mode = mode
    if post_weight is not None:
        post_weight = post_weight.contiguous()
        d.post_dtype = L.dt(post_weight)
    if next_weight is not None:
        next_weight = next_weight.contiguous()
        d.next_dtype = L.dt(next_weight)
    d.norm_dtype = d.res_dtype if norm_dtype is None else L.dt(norm_dtype)
    d.residual_scale, d.eps = residual_scale, eps
    return dev, d, (y, residual, post_weight, next_weight, gate)


def _forward(what, y, residual, post_weight, next_weight, gate, residual_scale, eps, norm_dtype):
    dev, d, inputs = _describe(what, y, residual, post_weight, next_weight, gate, residual_scale, eps, norm_dtype)
    shape = residual.shape
    out = torch.empty(shape, dtype=residual.dtype, device=dev) if y is not None else None
    normed = torch.empty(shape, dtype=norm_dtype or residual.dtype, device=dev) if next_weight is not None else None
    L.call(what, dev, L.lib().moe_norm_gate_residual, ctypes.byref(d), *map(L.ptr, inputs), L.ptr(out),
           L.ptr(normed), L.stream_ptr(dev))
    return out, normed


def _backward(what, d_out, d_normed, y, residual, post_weight, next_weight, gate, residual_scale, eps, needs):
    norm_dtype = None if d_normed is None else d_normed.dtype
    dev, d, inputs = _describe(what, y, residual, post_weight, next_weight, gate, residual_scale, eps, norm_dtype,
                               d_out, d_normed)
    shape, h = residual.shape, residual.shape[-1]
    for name, g in (("d_out", d_out), ("d_normed", d_normed)):
        if g is not None and g.shape != shape:
            raise ValueError(f"{what}: {name}.shape {tuple(g.shape)} != {tuple(shape)}")
    s_out = s_normed = h
    if d_out is not None:
        d_out, s_out = _rows(d_out if d_out.dtype == residual.dtype else d_out.detach().to(residual.dtype), h)
    if d_normed is not None:
        if next_weight is None:
            raise ValueError(f"{what}: d_normed needs next_weight")
        d_normed, s_normed = _rows(d_normed, h)
    grads = [torch.empty(t.shape, dtype=t.dtype, device=dev) if t is not None and n else None
             for t, n in zip((y, residual, post_weight, next_weight, gate), needs)]
    lib, ws, nbytes = L.lib(), None, 0
    if grads[2] is not None or grads[3] is not None or (grads[4] is not None and d.gate_mode == L.GATE_CHANNEL):
        # per call, not cached: a captured graph then owns the workspace it replays on
        nbytes = lib.moe_norm_backward_workspace_bytes(d.T, h)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    L.call(what, dev, lib.moe_norm_gate_residual_backward, ctypes.byref(d), L.ptr(d_out), s_out, L.ptr(d_normed),
           s_normed, *map(L.ptr, inputs), *map(L.ptr, grads), L.ptr(ws), nbytes, L.status_word(dev).data_ptr(),
           L.stream_ptr(dev))
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
