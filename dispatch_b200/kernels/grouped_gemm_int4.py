"""Expert products with 4-bit weights and group scales (``csrc/int4.cuh``), the
int8 contract of ``grouped_gemm_int8.py`` for ``Int4Tensor`` weights. No
reference counterpart.

Up to 128 rows per expert on average (48 with groups below 128) the codes
themselves are multiplied: they become 16-bit floats exactly on the way to the
tensor cores (warp-level MMAs for a few rows, tcgen05 for more) and each column
group's f32 sum is multiplied by its scale. Larger batches write the weights as
16-bit ones, some experts at a time, for the 16-bit tcgen05 kernels (one
rounding of code * scale per weight), unless the weights are marked ``exact``."""

from __future__ import annotations

import torch

from dispatch_b200 import _lib as L
from dispatch_b200.kernels.quantization import Int4StackedExpertWeights, Int4Tensor, _check_int4
from dispatch_b200.kernels.tile_schedule import TileSchedule, device_offsets


def refuse_gradients(what: str, *tensors: torch.Tensor | None) -> None:
    """4-bit weights are frozen and no product has a backward: raises for an
    input whose derivative would be lost."""
    L.refuse_tangents(what, *tensors)
    for t in tensors:
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{what}: int4 weights are for inference: call under torch.no_grad() or detach the inputs")


def _check_activations(x: torch.Tensor, q: Int4Tensor) -> None:
    if not (x.is_cuda and q.data.is_cuda and q.scale.is_cuda):
        raise ValueError("the B200 int4 grouped-GEMM kernels need CUDA tensors")
    _check_int4(q)
    if x.dim() != 2 or x.shape[1] != q.k:
        raise ValueError(f"K mismatch: x has {tuple(x.shape)}, qweight has K={q.k}")
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"dtype mismatch: activations must be bf16/f16, got {x.dtype}")
    refuse_gradients("the int4 products", x)


def _aligned(x: torch.Tensor) -> torch.Tensor:
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone(memory_format=torch.contiguous_format)


def _workspace(nbytes: int, device: torch.device) -> torch.Tensor | None:
    # per call, not cached: a captured graph then owns the workspace it replays on
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def grouped_matmul_int4(x: torch.Tensor, qweight: Int4Tensor, schedule: TileSchedule) -> torch.Tensor:
    """out[rows of e] = x[rows of e] @ (code[e] * scale[e]).T, f32 accumulation,
    in x's type (bf16 or f16). K a multiple of 8, any N; only
    ``schedule.group_offsets`` is read."""
    _check_activations(x, qweight)
    if schedule.block_m < 1:
        raise ValueError(f"schedule.block_m={schedule.block_m} must be positive")
    e = qweight.num_experts
    if len(schedule.group_offsets) != e + 1:
        raise ValueError("schedule.group_offsets does not match the number of experts")
    m = x.shape[0]
    if schedule.group_offsets[-1] != m:
        raise ValueError(f"schedule covers {schedule.group_offsets[-1]} rows, x has {m}")
    out = torch.empty(m, qweight.n, dtype=x.dtype, device=x.device)
    if m == 0:
        return out
    dev = L.require_cuda(x, qweight.data, qweight.scale)
    x = _aligned(x)
    offsets = device_offsets(schedule, dev)
    lib = L.lib()
    # without a workspace no weight is rounded
    need = 0 if qweight.exact else lib.moe_int4_workspace_bytes(m, e, qweight.n, qweight.k, qweight.group_size)
    ws = _workspace(need, dev)
    L.call(
        "grouped_matmul_int4", dev, lib.moe_grouped_gemm_int4,
        x.data_ptr(), L.dt(x), m, qweight.k, qweight.data.data_ptr(), qweight.scale.data_ptr(),
        L.dt(qweight.scale), qweight.group_size, e, qweight.n, offsets.data_ptr(), out.data_ptr(), qweight.n,
        L.ptr(ws), 0 if ws is None else ws.numel(), L.status_word(dev).data_ptr(), L.stream_ptr(dev),
    )
    return out


def expert_ffn_int4(xs: torch.Tensor, offsets: torch.Tensor, weights: Int4StackedExpertWeights) -> torch.Tensor:
    """y = down(silu(gate(xs)) * up(xs)) per expert group of grouped rows, the
    offsets (E+1) int32 on the device; gate and up in one launch with SwiGLU
    where they are joined. No weight is rounded if any of the three is ``exact``."""
    gate, up, down = weights.gate, weights.up, weights.down
    _check_activations(xs, gate)
    for q in (up, down):
        _check_int4(q)
        if (q.group_size, q.scale.dtype, q.num_experts) != (gate.group_size, gate.scale.dtype, gate.num_experts):
            raise ValueError("gate, up and down must share experts, group size and scale type")
    if (up.n, up.k) != (gate.n, gate.k) or (down.n, down.k) != (gate.k, gate.n):
        raise ValueError(f"K mismatch: gate ({gate.n}, {gate.k}), up ({up.n}, {up.k}), down ({down.n}, {down.k})")
    if offsets.dtype != torch.int32 or offsets.numel() != gate.num_experts + 1:
        raise ValueError("offsets must be (E+1,) int32")
    dev = L.require_cuda(xs, offsets, *(t for q in (gate, up, down) for t in (q.data, q.scale)),
                         what="the B200 int4 expert FFN")
    xs, offsets = _aligned(xs), offsets.contiguous()
    r, h, i, e = xs.shape[0], gate.k, gate.n, gate.num_experts
    y = torch.empty(r, h, dtype=xs.dtype, device=dev)
    lib = L.lib()
    # room for the intermediate rows alone: no weight is rounded
    exact = gate.exact or up.exact or down.exact
    ws = _workspace((r * i * 2 + 255) // 256 * 256 if exact else
                    lib.moe_ffn_int4_workspace_bytes(r, e, h, i, gate.group_size), dev)
    L.call(
        "expert_ffn_int4", dev, lib.moe_expert_ffn_int4,
        xs.data_ptr(), L.dt(xs), r, h, offsets.data_ptr(), e, i, gate.data.data_ptr(),
        gate.scale.data_ptr(), up.data.data_ptr(), up.scale.data_ptr(), down.data.data_ptr(),
        down.scale.data_ptr(), L.dt(gate.scale), gate.group_size, y.data_ptr(), L.ptr(ws),
        0 if ws is None else ws.numel(), L.status_word(dev).data_ptr(), L.stream_ptr(dev),
    )
    return y
