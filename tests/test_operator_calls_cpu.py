"""Calls of the operators around the layer that the host has to refuse, or to
let through, before anything runs on a GPU."""

from __future__ import annotations

import torch

from dispatch_b200.kernels.moe_forward import StackedExpertWeights
from dispatch_b200.kernels.quantization import Int4StackedExpertWeights, Int4Tensor, pack_int4

BF16 = torch.bfloat16
T, K, E, H, I = 6, 2, 4, 64, 32


def int4(e=E, n=I, k=H) -> Int4Tensor:
    return pack_int4(torch.zeros(e, n, k, dtype=torch.int8), torch.ones(e, n, -(-k // 32)), 32)


def weights(kind):
    if kind == "int4":
        return Int4StackedExpertWeights(int4(), int4(), int4(n=H, k=I))
    return StackedExpertWeights(torch.zeros(E, I, H, dtype=BF16), torch.zeros(E, I, H, dtype=BF16),
                                torch.zeros(E, H, I, dtype=BF16))


def topk(t=T, k=K):
    return torch.zeros(t, k, dtype=torch.int32), torch.ones(t, k)


# ------------------------------------------------------------------ weights


def test_the_exact_flag_travels_with_the_weights() -> None:
    assert not int4().exact
    codes, scale = torch.zeros(E, I, H, dtype=torch.int8), torch.ones(E, I, H // 32)
    assert pack_int4(codes, scale, 32, exact=True).exact
