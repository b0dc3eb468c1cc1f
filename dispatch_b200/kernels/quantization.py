"""Weight-only int8 quantisation (mirror of the reference's
src/dispatch/kernels/quantization.py). The quantiser runs as a CUDA kernel
(bit-exact with the reference's f32 arithmetic); the expert kernels consume
the int8 data plus per-output-channel scales (f32, or bf16 as the BASELINE int8
config asks) and apply the scale once after the K loop.

Also 4-bit weights with one scale per row and group of columns
(``Int4Tensor``), which the reference does not have: half of int8's bytes per
decoded token. ``quantize_groupwise_int4`` makes them from float weights,
``pack_int4`` from codes and scales that were quantised elsewhere."""

from __future__ import annotations

from collections.abc import Callable
from dataclasses import dataclass

import torch

from dispatch_b200 import _lib as L
from dispatch_b200.kernels.tile_schedule import TileSchedule

INT8_MAX = 127


@dataclass(frozen=True)
class QuantizedTensor:
    """An (E, N, K) weight tensor quantised to int8, one scale per expert per
    output channel (E, N) (reference quantization.py:23-28)."""

    data: torch.Tensor
    scale: torch.Tensor


def quantize_per_channel_int8(weight: torch.Tensor, *, scale_dtype: torch.dtype = torch.float32) -> QuantizedTensor:
    """scale = absmax/127 in f32 (1.0 for an all-zero channel), q =
    clamp(round_half_even(w / scale), -127, 127) (reference quantization.py:31-50).
    ``scale_dtype=torch.bfloat16`` stores the f32 scale rounded to bf16."""
    dev = L.require_cuda(weight, what="quantize_per_channel_int8")
    w = weight.detach().contiguous()
    if w.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        w = w.float()
    k = w.shape[-1]
    rows = w.numel() // max(k, 1)
    q = torch.empty(w.shape, dtype=torch.int8, device=dev)
    scale = torch.empty(w.shape[:-1], dtype=scale_dtype, device=dev)
    rc = L.lib().moe_quantize_int8(w.data_ptr(), L.dt(w), rows, k, q.data_ptr(), scale.data_ptr(), L.dt(scale),
                                   L.stream_ptr(dev))
    L.check(rc, "quantize_per_channel_int8")
    return QuantizedTensor(data=q, scale=scale)


def dequantize_int8(qtensor: QuantizedTensor) -> torch.Tensor:
    """q * scale in f32 (reference quantization.py:53-54); a test helper."""
    return qtensor.data.to(torch.float32) * qtensor.scale.float().unsqueeze(-1)


@dataclass(frozen=True)
class QuantizedStackedExpertWeights:
    gate: QuantizedTensor
    up: QuantizedTensor
    down: QuantizedTensor

    @property
    def num_experts(self) -> int:
        return int(self.gate.data.shape[0])


QuantizedGroupedMatmul = Callable[[torch.Tensor, QuantizedTensor, TileSchedule], torch.Tensor]


def quantize_stacked_weights(weights, *, scale_dtype: torch.dtype = torch.float32) -> QuantizedStackedExpertWeights:
    return QuantizedStackedExpertWeights(
        gate=quantize_per_channel_int8(weights.gate, scale_dtype=scale_dtype),
        up=quantize_per_channel_int8(weights.up, scale_dtype=scale_dtype),
        down=quantize_per_channel_int8(weights.down, scale_dtype=scale_dtype),
    )


def grouped_moe_routed_quantized(
    x: torch.Tensor,
    topk_idx: torch.Tensor,
    topk_weight: torch.Tensor,
    weights: QuantizedStackedExpertWeights | Int4StackedExpertWeights,
    matmul: QuantizedGroupedMatmul | None = None,
    *,
    block_m: int = 16,
    shared=None,
) -> torch.Tensor:
    """Reference: quantization.py:92-107. Runs the fused int8 path (two tcgen05
    launches with in-smem dequantisation), with 4-bit weights the int4 path
    (grouped_gemm_int4.py), with ``StackedExpertWeights`` the 16-bit one,
    whatever ``matmul`` is given."""
    from dispatch_b200.kernels.moe_forward import _routed_forward  # noqa: PLC0415

    _check_matmul(matmul)
    if block_m <= 0:
        raise ValueError(f"block_m must be positive, got {block_m}")
    return _routed_forward(x, topk_idx, topk_weight, weights, shared)


def _check_matmul(matmul) -> None:
    from dispatch_b200.kernels.grouped_gemm import grouped_matmul  # noqa: PLC0415
    from dispatch_b200.kernels.grouped_gemm_int4 import grouped_matmul_int4  # noqa: PLC0415
    from dispatch_b200.kernels.grouped_gemm_int8 import grouped_matmul_int8  # noqa: PLC0415

    if matmul is not None and matmul not in (grouped_matmul, grouped_matmul_int8, grouped_matmul_int4):
        raise ValueError("the B200 layer path runs its own fused kernels; pass matmul=None or the b200 backend")


def stacked_weights_nbytes(weights) -> int:
    return sum(t.element_size() * t.nelement() for t in (weights.gate, weights.up, weights.down))


def quantized_stacked_weights_nbytes(weights: QuantizedStackedExpertWeights | Int4StackedExpertWeights) -> int:
    total = 0
    for qt in (weights.gate, weights.up, weights.down):
        total += qt.data.element_size() * qt.data.nelement()
        total += qt.scale.element_size() * qt.scale.nelement()
    return total


# ---------------------------------------------------------------- 4-bit weights, group scales
INT4_GROUP_SIZES = (32, 64, 128, 256)


@dataclass(frozen=True)
class Int4Tensor:
    """(E, N, K) weights as 4-bit codes -8..7 and one scale per row and group
    of ``group_size`` columns, laid out once for the product's kernels
    (``include/moe_b200.h``): ``data`` (E, ceil(N/16), ceil(K/64), 32, 4) int32,
    ``scale`` (E, ceil(N/16), ceil(K/group_size), 16) f32, bf16 or f16.

    Batches of more than 128 rows per expert on average (48 for groups below
    128) round each weight code * scale once to the activation type, in f16
    within f16's range, for the 16-bit kernels. ``exact``: no batch rounds a
    weight; the codes are multiplied and the scales act in f32 at any size."""

    data: torch.Tensor
    scale: torch.Tensor
    n: int
    k: int
    group_size: int
    exact: bool = False

    @property
    def num_experts(self) -> int:
        return int(self.data.shape[0])

    @property
    def groups(self) -> int:
        return -(-self.k // self.group_size)


@dataclass(frozen=True)
class Int4StackedExpertWeights:
    gate: Int4Tensor
    up: Int4Tensor
    down: Int4Tensor

    @property
    def num_experts(self) -> int:
        return self.gate.num_experts


def _check_group_size(group_size: int) -> None:
    if group_size not in INT4_GROUP_SIZES:
        raise ValueError(f"group size {group_size} must be one of {INT4_GROUP_SIZES}")


def _check_int4(q: Int4Tensor) -> None:
    _check_group_size(q.group_size)
    n16, kb = -(-q.n // 16), -(-q.k // 64)
    if q.data.dtype != torch.int32:
        raise ValueError(f"expected int32 int4 weight data, got {q.data.dtype}")
    if q.scale.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise ValueError(f"expected float32, bfloat16 or float16 scales, got {q.scale.dtype}")
    e = q.num_experts
    if q.data.shape != (e, n16, kb, 32, 4):
        raise ValueError(f"int4 data shape {tuple(q.data.shape)} does not match weight ({e}, {q.n}, {q.k}) laid out")
    if q.scale.shape != (e, n16, q.groups, 16):
        raise ValueError(f"scale shape {tuple(q.scale.shape)} does not match weight ({e}, {q.n}, {q.k}) "
                         f"in groups of {q.group_size}")
    if not (q.data.is_contiguous() and q.scale.is_contiguous()):
        raise ValueError("int4 data and scales must be contiguous")


def quantize_groupwise_int4(weight: torch.Tensor, *, group_size: int = 128,
                            scale_dtype: torch.dtype = torch.float32, exact: bool = False) -> Int4Tensor:
    """Per row and group of columns: scale = absmax / 7 in f32 (1.0 for a group
    of zeros) rounded to ``scale_dtype``, code = clamp(round_half_even(w /
    scale), -8, 7). weight (E, N, K); a last group of fewer columns is fine."""
    _check_group_size(group_size)
    if weight.dim() != 3:
        raise ValueError(f"expected (E, N, K) weights, got {tuple(weight.shape)}")
    dev = L.require_cuda(weight, what="quantize_groupwise_int4")
    w = weight.detach().contiguous()
    if w.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        w = w.float()
    e, n, k = w.shape
    data = torch.empty(e, -(-n // 16), -(-k // 64), 32, 4, dtype=torch.int32, device=dev)
    scale = torch.empty(e, -(-n // 16), -(-k // group_size), 16, dtype=scale_dtype, device=dev)
    L.call("quantize_groupwise_int4", dev, L.lib().moe_quantize_int4, w.data_ptr(), L.dt(w), e, n, k, group_size,
           data.data_ptr(), scale.data_ptr(), L.dt(scale), L.stream_ptr(dev))
    return Int4Tensor(data, scale, n, k, group_size, exact)


def pack_int4(codes: torch.Tensor, scale: torch.Tensor, group_size: int, *, exact: bool = False) -> Int4Tensor:
    """Lays out codes (E, N, K), integers -8..7, and their scales (E, N,
    ceil(K/group_size)): for weights quantised elsewhere. Runs once per weight,
    on the codes' device (CPU included)."""
    _check_group_size(group_size)
    if codes.dim() != 3 or scale.shape != (*codes.shape[:2], -(-codes.shape[2] // group_size)):
        raise ValueError(f"scale shape {tuple(scale.shape)} does not match codes {tuple(codes.shape)} "
                         f"in groups of {group_size}")
    if codes.is_floating_point() or (codes.numel() and (int(codes.min()) < -8 or int(codes.max()) > 7)):
        raise ValueError("int4 codes must be integers in -8..7")
    e, n, k = codes.shape
    n16, kb = -(-n // 16), -(-k // 64)
    u = torch.nn.functional.pad((codes.to(torch.int16) + 8).to(torch.uint8), (0, -k % 64, 0, -n % 16), value=8)
    # row 16 i + 8 half + g, column 64 b + 32 j + 8 q + 4 step + 2 pair + odd
    u = u.view(e, n16, 2, 8, kb, 2, 4, 2, 2, 2).permute(0, 1, 4, 3, 6, 5, 7, 9, 8, 2)
    data = (u[..., 0] | (u[..., 1] << 4)).reshape(e, n16, kb, 32, 16).contiguous().view(torch.int32)
    s = torch.nn.functional.pad(scale, (0, 0, 0, -n % 16), value=1.0)
    s = s.view(e, n16, 16, -1).transpose(2, 3).contiguous()
    return Int4Tensor(data, s, n, k, group_size, exact)


def unpack_int4(q: Int4Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The codes (E, N, K) int8 and scales (E, N, groups) of ``q``; the inverse
    of ``pack_int4``, on q's device."""
    _check_int4(q)
    e, n16, kb = q.data.shape[:3]
    b = q.data.view(torch.uint8).view(e, n16, kb, 8, 4, 2, 2, 2, 2)
    u = torch.stack((b & 15, b >> 4), dim=-1)  # (e, i, b, g, q, j, step, odd, pair, half)
    u = u.permute(0, 1, 9, 3, 2, 5, 4, 6, 8, 7).reshape(e, n16 * 16, kb * 64)
    codes = u[:, :q.n, :q.k].to(torch.int8) - 8
    scale = q.scale.transpose(2, 3).reshape(e, n16 * 16, -1)[:, :q.n]
    return codes, scale


def dequantize_int4(q: Int4Tensor) -> torch.Tensor:
    """code * scale in f32 (E, N, K)."""
    codes, scale = unpack_int4(q)
    return codes.float() * scale.float().repeat_interleave(q.group_size, dim=2)[..., :q.k]


def quantize_stacked_weights_int4(weights, *, group_size: int = 128,
                                  scale_dtype: torch.dtype = torch.float32,
                                  exact: bool = False) -> Int4StackedExpertWeights:
    """Each projection of a ``StackedExpertWeights`` in 4 bits."""
    return Int4StackedExpertWeights(*(
        quantize_groupwise_int4(w, group_size=group_size, scale_dtype=scale_dtype, exact=exact)
        for w in (weights.gate, weights.up, weights.down)
    ))
