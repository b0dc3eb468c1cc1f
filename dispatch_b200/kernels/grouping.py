"""Token-to-expert grouping on the device (mirror of the reference's
src/dispatch/kernels/grouping.py).

``group_tokens_by_expert`` is a stable counting sort in two launches (no host
sync, no argsort); ``ungroup_and_combine`` is the deterministic weighted
combine (f32 sum in slot order, one rounding) instead of ``index_add_``.
``permute_tokens`` and ``combine_tokens`` are the same gather and combine for
training: differentiable, with their gradients also as plain calls.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from dispatch_b200 import _lib as L


@dataclass(frozen=True)
class TokenGrouping:
    """Row i of the grouped layout is token sorted_token_idx[i], weighted by
    sorted_weight[i]; the first group_sizes[0] rows belong to expert 0, and so
    on (reference grouping.py:15-22). The extra fields keep the grouping on the
    device: ``offsets`` (E+1) int32, ``pos`` (T*k) int32 with
    pos[t*k+s] = grouped row of (token t, slot s), and the flat f32 weights."""

    sorted_token_idx: torch.Tensor  # (num_tokens * top_k,) int64
    sorted_weight: torch.Tensor  # (num_tokens * top_k,)
    group_sizes: torch.Tensor  # (n_routed_experts,) int64
    offsets: torch.Tensor
    pos: torch.Tensor
    flat_weight: torch.Tensor
    top_k: int


def _group(topk_idx: torch.Tensor, topk_weight: torch.Tensor | None, n_experts: int,
           x: torch.Tensor | None = None, xs_dtype: torch.dtype | None = None,
           want_sorted: bool = True, sizes: torch.Tensor | None = None):
    dev = L.require_cuda(topk_idx, topk_weight, x, what="token grouping")
    t, k = topk_idx.shape
    idx = topk_idx.contiguous()
    if idx.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"topk_idx must be int32 or int64, got {idx.dtype}")
    w = None if topk_weight is None else topk_weight.contiguous().float()
    n = t * k
    counts = torch.empty(n_experts, dtype=torch.int32, device=dev)
    offsets = torch.empty(n_experts + 1, dtype=torch.int32, device=dev)
    pos = torch.empty(n, dtype=torch.int32, device=dev)
    sti = torch.empty(n, dtype=torch.int64, device=dev) if want_sorted else None
    sw = torch.empty(n, dtype=torch.float32, device=dev) if (want_sorted and w is not None) else None
    xs = None
    h = 0
    if x is not None:
        h = x.shape[1]
        xs = torch.empty(n, h, dtype=xs_dtype, device=dev)
    lib = L.lib()
    nbytes = lib.moe_group_workspace_bytes(t, k, n_experts)
    ws = L.workspace(dev, nbytes, "group")
    L.call(
        "group_tokens_by_expert", dev, lib.moe_group_tokens_sizes,
        idx.data_ptr(), L.dt(idx), L.ptr(w), t, k, n_experts, counts.data_ptr(), L.ptr(sizes), offsets.data_ptr(),
        pos.data_ptr(), L.ptr(sti), L.ptr(sw),
        L.ptr(x), L.dt(x) if x is not None else 0, h, L.ptr(xs), L.dt(xs_dtype) if xs is not None else 0,
        ws.data_ptr(), ws.numel(), L.status_word(dev).data_ptr(), L.stream_ptr(dev),
    )
    return counts, offsets, pos, sti, sw, w, xs


def group_tokens_by_expert(
    topk_idx: torch.Tensor, topk_weight: torch.Tensor, n_routed_experts: int
) -> TokenGrouping:
    """Reference: src/dispatch/kernels/grouping.py:25-41."""
    if topk_idx.shape != topk_weight.shape:
        raise ValueError(
            f"topk_idx.shape {tuple(topk_idx.shape)} != topk_weight.shape {tuple(topk_weight.shape)}"
        )
    # sizes and weights are made here, on the grouping's own stream: a caller who
    # reads them elsewhere can then protect them with record_stream, or keep them
    # for a captured graph
    sizes = torch.empty(n_routed_experts, dtype=torch.int64, device=topk_idx.device)
    _, offsets, pos, sti, sw, w, _ = _group(topk_idx, topk_weight, n_routed_experts, sizes=sizes)
    return TokenGrouping(
        sorted_token_idx=sti,
        sorted_weight=sw if sw.dtype == topk_weight.dtype else sw.to(topk_weight.dtype),
        group_sizes=sizes,
        offsets=offsets,
        pos=pos,
        flat_weight=w.reshape(-1),
        top_k=topk_idx.shape[1],
    )


def combine(y: torch.Tensor, pos: torch.Tensor, flat_weight: torch.Tensor, num_tokens: int, top_k: int,
            y_shared: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """out[t] = sum_s w[t,s] * y[pos[t*k+s]] (+ y_shared[t]) in f32, slot order."""
    dev = L.require_cuda(y, pos, flat_weight, y_shared, what="ungroup_and_combine")
    h = y.shape[-1]
    out = torch.empty(num_tokens, h, dtype=out_dtype or y.dtype, device=dev)
    ys = None if y_shared is None else y_shared.contiguous()
    if ys is not None and ys.dtype != y.dtype:
        ys = ys.to(y.dtype)
    y, flat_weight = y.contiguous(), flat_weight.contiguous()
    L.call(
        "ungroup_and_combine", dev, L.lib().moe_combine,
        y.data_ptr(), L.dt(y), pos.data_ptr(), flat_weight.data_ptr(), num_tokens,
        top_k, h, L.ptr(ys), out.data_ptr(), L.dt(out), L.status_word(dev).data_ptr(), L.stream_ptr(dev),
    )
    return out


def ungroup_and_combine(
    grouped_output: torch.Tensor, grouping: TokenGrouping, num_tokens: int
) -> torch.Tensor:
    """Reference: src/dispatch/kernels/grouping.py:44-61."""
    if grouped_output.shape[0] != grouping.sorted_token_idx.shape[0]:
        raise ValueError(
            f"grouped_output has {grouped_output.shape[0]} rows, "
            f"grouping describes {grouping.sorted_token_idx.shape[0]}"
        )
    return combine(grouped_output, grouping.pos, grouping.flat_weight, num_tokens, grouping.top_k)


# ---------------------------------------------------------------- with gradients
def _tokens(what: str, grouping: TokenGrouping, rows: torch.Tensor | None, tokens: int | None) -> int:
    """The token count of ``grouping``; raises if rows or tokens do not fit it."""
    n = grouping.pos.numel()
    t = n // grouping.top_k
    if tokens is not None and tokens != t:
        raise ValueError(f"{what}: {tokens} tokens, grouping describes {t}")
    if rows is not None and rows.shape[0] != n:
        raise ValueError(f"{what}: {rows.shape[0]} rows, grouping describes {n}")
    return t


def _row_view(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """``t`` (N, H) and its row stride, copied only if its rows cannot be read
    in 16-byte pieces where they lie (a last stride other than 1, unaligned or
    overlapping rows)."""
    if t.dim() != 2:
        raise ValueError(f"expected (rows, H), got {tuple(t.shape)}")
    h = t.shape[1]
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():
            return t, h
        if t.stride(1) == 1 and t.stride(0) % 8 == 0 and t.stride(0) >= h:
            return t, t.stride(0)
    c = t.detach().contiguous()
    return (c if c.data_ptr() % 16 == 0 else c.clone(memory_format=torch.contiguous_format)), h


def _weights(what: str, topk_weight: torch.Tensor | None, grouping: TokenGrouping) -> torch.Tensor:
    """The weights, (T, k) or flat, in their own type."""
    if topk_weight is None:
        return grouping.flat_weight
    n, k = grouping.pos.numel(), grouping.top_k
    if topk_weight.shape not in ((n // k, k), (n,)):
        raise ValueError(f"{what}: topk_weight.shape {tuple(topk_weight.shape)}, grouping describes ({n // k}, {k})")
    return topk_weight if topk_weight.is_contiguous() else topk_weight.detach().contiguous()


def _permute(x: torch.Tensor, grouping: TokenGrouping) -> torch.Tensor:
    dev = L.require_cuda(x, grouping.pos, what="permute_tokens")
    x, stride = _row_view(x)
    t = _tokens("permute_tokens", grouping, None, x.shape[0])
    h, k = x.shape[1], grouping.top_k
    xs = torch.empty(t * k, h, dtype=x.dtype, device=dev)
    L.call("permute_tokens", dev, L.lib().moe_permute_rows, x.data_ptr(), L.dt(x), stride, grouping.pos.data_ptr(),
           grouping.offsets.data_ptr(), t, k, grouping.offsets.numel() - 1, h, xs.data_ptr(),
           L.status_word(dev).data_ptr(), L.stream_ptr(dev))
    return xs


def _unpermute(what, rows, grouping, w, y_shared, out_dtype) -> torch.Tensor:
    dev = L.require_cuda(rows, grouping.pos, w, y_shared, what=what)
    rows, stride = _row_view(rows)
    t = _tokens(what, grouping, rows, None if y_shared is None else y_shared.shape[0])
    h = rows.shape[1]
    shared_stride = h
    if y_shared is not None:
        y_shared, shared_stride = _row_view(y_shared)
    out = torch.empty(t, h, dtype=out_dtype or rows.dtype, device=dev)
    L.call(what, dev, L.lib().moe_unpermute_rows, rows.data_ptr(), L.dt(rows), stride, grouping.pos.data_ptr(),
           L.ptr(w), 0 if w is None else L.dt(w), L.ptr(y_shared), shared_stride, t, grouping.top_k, h,
           out.data_ptr(), L.dt(out), L.status_word(dev).data_ptr(), L.stream_ptr(dev))
    return out


def permute_tokens_backward(dxs: torch.Tensor, grouping: TokenGrouping, *,
                            out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """dx[t] = sum over the token's slots of dxs[pos], in f32 in slot order,
    rounded once to ``out_dtype`` (default: dxs' type)."""
    return _unpermute("permute_tokens_backward", dxs, grouping, None, None, out_dtype)


class _Permute(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, grouping):
        ctx.grouping, ctx.dtype = grouping, x.dtype
        ctx.save_for_backward(grouping.pos)  # so that a change in place is noticed
        return _permute(x, grouping)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dxs):
        ctx.saved_tensors  # raises for what was changed in place
        return permute_tokens_backward(dxs, ctx.grouping, out_dtype=ctx.dtype), None


def permute_tokens(x: torch.Tensor, grouping: TokenGrouping) -> torch.Tensor:
    """xs[pos[t*k+s]] = x[t]: each token's row once per slot, in expert order
    (T*k, H), in x's type (bf16, f16 or f32; H a multiple of 8, k <= 32). Rows
    that no slot owns, at and after ``offsets[E]``, are zero. Differentiable
    in x."""
    if L.grad_wanted("permute_tokens", x):
        return _Permute.apply(x, grouping)
    return _permute(x, grouping)


def _combine(y, grouping, topk_weight, y_shared, out_dtype) -> torch.Tensor:
    w = _weights("combine_tokens", topk_weight, grouping)
    if y_shared is not None and y_shared.dtype != y.dtype:
        raise ValueError(f"dtype mismatch: y is {y.dtype}, y_shared is {y_shared.dtype}")
    if y_shared is not None and y_shared.shape[1:] != y.shape[1:]:
        raise ValueError(f"y_shared.shape {tuple(y_shared.shape)} does not match rows of {tuple(y.shape)}")
    return _unpermute("combine_tokens", y, grouping, w, y_shared, out_dtype)


def combine_tokens_backward(
    dout: torch.Tensor, y: torch.Tensor, grouping: TokenGrouping, topk_weight: torch.Tensor | None = None, *,
    need_y: bool = True, need_weight: bool = True,
) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """The gradients (dy, dweight) of ``combine_tokens``: dy[pos[f]] = w[f] *
    dout[f/k] in y's type, zero in rows that no slot owns; dweight =
    <dout[f/k], y[pos[f]]>, summed in f32, in topk_weight's type and shape
    ((T, k) f32 for the grouping's own weights). y_shared's gradient is dout
    itself."""
    what = "combine_tokens_backward"
    dev = L.require_cuda(dout, y, grouping.pos, topk_weight, what=what)
    y, y_stride = _row_view(y)
    dout, dout_stride = _row_view(dout)
    t = _tokens(what, grouping, y, dout.shape[0])
    h, k = y.shape[1], grouping.top_k
    if dout.shape[1] != h:
        raise ValueError(f"dout.shape {tuple(dout.shape)} does not match rows of {tuple(y.shape)}")
    w = _weights(what, topk_weight, grouping)
    dy = torch.empty(t * k, h, dtype=y.dtype, device=dev) if need_y else None
    dw = None
    if need_weight:
        dw = torch.empty((t, k) if topk_weight is None else topk_weight.shape, dtype=w.dtype, device=dev)
    L.call(what, dev, L.lib().moe_combine_backward, dout.data_ptr(), L.dt(dout), dout_stride, y.data_ptr(), L.dt(y),
           y_stride, grouping.pos.data_ptr(), grouping.offsets.data_ptr(), w.data_ptr(), L.dt(w), t, k,
           grouping.offsets.numel() - 1, h, L.ptr(dy), L.ptr(dw), L.status_word(dev).data_ptr(), L.stream_ptr(dev))
    return dy, dw


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, topk_weight, y_shared, grouping, out_dtype):
        # the grouping's own weights may be the caller's tensor: saved so that a change in place is noticed
        own = grouping.flat_weight if topk_weight is None else None
        ctx.save_for_backward(y, topk_weight, own, grouping.pos, grouping.offsets)
        ctx.grouping = grouping
        return _combine(y, grouping, topk_weight, y_shared, out_dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        y, topk_weight, *_ = ctx.saved_tensors
        need_y, need_w, need_shared = ctx.needs_input_grad[:3]
        dy = dw = None
        if need_y or need_w:
            dy, dw = combine_tokens_backward(dout, y, ctx.grouping, topk_weight, need_y=need_y, need_weight=need_w)
        return dy, dw, dout.to(y.dtype) if need_shared else None, None, None


def combine_tokens(
    y: torch.Tensor, grouping: TokenGrouping, topk_weight: torch.Tensor | None = None, *,
    y_shared: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """out[t] = sum_s topk_weight[t, s] * y[pos[t*k+s]] (+ y_shared[t]), in f32
    in slot order, rounded once to ``out_dtype`` (default: y's type): the
    reference's ungroup_and_combine with the weights as an argument, so that
    it is differentiable in y, topk_weight and y_shared. ``topk_weight``
    None: the weights the grouping was made with (no gradient for them)."""
    if L.grad_wanted("combine_tokens", y, topk_weight, y_shared):
        return _Combine.apply(y, topk_weight, y_shared, grouping, out_dtype)
    return _combine(y, grouping, topk_weight, y_shared, out_dtype)
