"""The 4-bit weights' layout and the host checks around them, without a GPU."""

from __future__ import annotations

import dataclasses

import pytest
import torch

from dispatch_b200 import _lib as L
from dispatch_b200.kernels.backends import resolve_quantized_backend
from dispatch_b200.kernels.grouped_gemm_int4 import expert_ffn_int4, grouped_matmul_int4
from dispatch_b200.kernels.grouped_gemm_int8 import grouped_matmul_int8
from dispatch_b200.kernels.quantization import (
    Int4StackedExpertWeights,
    Int4Tensor,
    _check_int4,
    dequantize_int4,
    pack_int4,
    quantize_groupwise_int4,
    unpack_int4,
)
from dispatch_b200.kernels.tile_schedule import build_tile_schedule


def codes_and_scale(e, n, k, group, dtype=torch.float32):
    g = torch.Generator().manual_seed(n + k)
    codes = torch.randint(-8, 8, (e, n, k), generator=g).to(torch.int8)
    scale = (torch.rand(e, n, -(-k // group), generator=g) + 0.1).to(dtype)
    return codes, scale


@pytest.mark.parametrize(("e", "n", "k", "group"), [(1, 16, 64, 32), (2, 17, 72, 64), (3, 1, 8, 128), (2, 40, 520, 256)])
def test_layout_round_trip(e, n, k, group) -> None:
    codes, scale = codes_and_scale(e, n, k, group)
    q = pack_int4(codes, scale, group)
    assert q.data.shape == (e, -(-n // 16), -(-k // 64), 32, 4) and q.scale.shape == (e, -(-n // 16), -(-k // group), 16)
    back, s = unpack_int4(q)
    assert torch.equal(back, codes) and torch.equal(s, scale)
    want = codes.float() * scale.repeat_interleave(group, 2)[..., :k]
    assert torch.equal(dequantize_int4(q), want)


def test_layout_is_the_documented_one() -> None:
    """Every nibble's place, as include/moe_b200.h states it."""
    codes, scale = codes_and_scale(1, 32, 128, 64)
    q = pack_int4(codes, scale, 64)
    for i in range(2):
        for b in range(2):
            for lane in range(32):
                g, quad = divmod(lane, 4)
                for word in range(4):
                    j, s = divmod(word, 2)
                    v = int(q.data[0, i, b, lane, word]) & 0xFFFFFFFF
                    for h in range(2):
                        for p in range(2):
                            for c in range(2):
                                code = ((v >> (4 * h + 8 * p + 16 * c)) & 15) - 8
                                col = 64 * b + 32 * j + 8 * quad + 4 * s + 2 * p + c
                                assert code == int(codes[0, 16 * i + 8 * h + g, col])
    assert torch.equal(q.scale[0, 1, 1], scale[0, 16:32, 1])


def test_padding_holds_zeros() -> None:
    codes, scale = codes_and_scale(1, 5, 24, 32)
    q = pack_int4(codes, scale, 32)
    whole = dataclasses.replace(q, n=16, k=64, scale=torch.ones(1, 1, 2, 16))
    back, _ = unpack_int4(whole)
    assert not back[:, 5:].any() and not back[:, :, 24:].any()


def test_refusals() -> None:
    codes, scale = codes_and_scale(1, 16, 64, 64)
    with pytest.raises(ValueError, match="group size"):
        pack_int4(codes, scale, 48)
    with pytest.raises(ValueError, match="scale shape"):
        pack_int4(codes, scale[..., :0], 64)
    with pytest.raises(ValueError, match="-8..7"):
        pack_int4(codes + 8, scale, 64)
    with pytest.raises(ValueError, match="-8..7"):
        pack_int4(codes.float(), scale, 64)
    q = pack_int4(codes, scale, 64)
    for change, match in ((dict(data=q.data.long()), "int32"), (dict(scale=q.scale.double()), "scales"),
                          (dict(n=17), "data shape"), (dict(k=128), "data shape"), (dict(group_size=32), "scale shape"),
                          (dict(data=q.data.transpose(3, 4).contiguous().transpose(3, 4)), "contiguous")):
        with pytest.raises(ValueError, match=match):
            _check_int4(dataclasses.replace(q, **change))
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        grouped_matmul_int4(x, q, build_tile_schedule(torch.tensor([4]), 16))
    with pytest.raises(ValueError, match="CUDA"):
        expert_ffn_int4(x, torch.tensor([0, 4], dtype=torch.int32), Int4StackedExpertWeights(q, q, q))
    with pytest.raises(ValueError, match="CUDA"):
        quantize_groupwise_int4(torch.zeros(1, 16, 64))
    with pytest.raises(ValueError, match="group size"):
        quantize_groupwise_int4(torch.zeros(1, 16, 64), group_size=100)


def test_backends_and_workspaces() -> None:
    assert resolve_quantized_backend() is grouped_matmul_int8
    assert resolve_quantized_backend(4) is grouped_matmul_int4
    with pytest.raises(ValueError, match="bits"):
        resolve_quantized_backend(3)
    lib = L.lib()
    assert lib.moe_int4_workspace_bytes(128 * 8, 8, 1408, 2048, 128) == 0  # no 16-bit weights
    assert lib.moe_int4_workspace_bytes(48 * 8, 8, 1408, 2048, 32) == 0
    per_expert = 1408 * 2048 * 2
    assert lib.moe_int4_workspace_bytes(128 * 8 + 1, 8, 1408, 2048, 128) >= per_expert
    assert lib.moe_int4_workspace_bytes(48 * 8 + 1, 8, 1408, 2048, 64) >= per_expert
    assert lib.moe_int4_workspace_bytes(10**6, 64, 2048, 1408, 64) < 64 * per_expert  # made a few experts at a time
    assert lib.moe_int4_workspace_bytes(0, 8, 1408, 2048, 64) == 0
    assert lib.moe_ffn_int4_workspace_bytes(6, 64, 2048, 1408, 64) >= 6 * 1408 * 2
    assert isinstance(Int4Tensor(torch.empty(3, 1, 1, 32, 4, dtype=torch.int32), torch.empty(3, 1, 1, 16), 16, 64,
                                 64).num_experts, int)
