"""Calls of the operators around the layer that the host has to refuse, or to
let through, before anything runs on a GPU."""

from __future__ import annotations

import copy
from types import SimpleNamespace

import pytest
import torch
from torch.autograd import forward_ad

from dispatch_b200 import _lib as L
from dispatch_b200.kernels.grouping import TokenGrouping, combine_tokens, combine_tokens_backward
from dispatch_b200.kernels.layer import RouterConfig, moe_block_forward, moe_layer_forward
from dispatch_b200.kernels.moe_forward import SharedExpertWeights, StackedExpertWeights, expert_ffn, grouped_moe_routed
from dispatch_b200.kernels.quantization import (
    Int4StackedExpertWeights,
    Int4Tensor,
    grouped_moe_routed_quantized,
    pack_int4,
)
from dispatch_b200.kernels.tile_schedule import build_tile_schedule, device_offsets

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


# ------------------------------------------------------------------ the caller's top-k
@pytest.mark.parametrize("kind", ["int4", "bf16"])
@pytest.mark.parametrize("pair", [topk(T, K - 1), topk(T, K + 1), topk(T - 1, K), topk(T + 1, K), topk(K, T),
                                  (topk()[0], topk(T, K - 1)[1]), (topk()[0].flatten(), topk()[1].flatten())])
def test_topk_of_another_shape_is_refused(kind, pair) -> None:
    x = torch.zeros(T, H, dtype=BF16)
    with pytest.raises(ValueError, match="topk"):
        moe_layer_forward(x, None, weights(kind), RouterConfig(top_k=K), topk=pair)
    with pytest.raises(ValueError, match="topk"):
        moe_block_forward(x, None, None, weights(kind), RouterConfig(top_k=K), normed=x, topk=pair)
    with pytest.raises(ValueError, match="CUDA"):  # the right one goes on to the device check
        moe_layer_forward(x, None, weights(kind), RouterConfig(top_k=K), topk=topk())


@pytest.mark.parametrize("kind", ["int4", "bf16"])
def test_fewer_rows_than_the_topk_names_are_refused(kind) -> None:
    call = grouped_moe_routed_quantized if kind == "int4" else grouped_moe_routed
    with pytest.raises(ValueError, match="topk_idx"):
        call(torch.zeros(T - 1, H, dtype=BF16), *topk(), weights(kind))


# ------------------------------------------------------------------ arguments of the C entries
@pytest.mark.parametrize("missing", ["gate_scale", "up_scale", "down_scale"])
def test_ffn_without_a_scale_is_refused(missing) -> None:
    """Before any launch, and before the device is looked at. The addresses are never read."""
    lib, at = L.lib(), 4096
    scale = {n: None if n == missing else at for n in ("gate_scale", "up_scale", "down_scale")}
    rc = lib.moe_expert_ffn_int4(at, L.DT_BF16, 8, H, at, E, I, at, scale["gate_scale"], at, scale["up_scale"], at,
                                 scale["down_scale"], L.DT_F32, 32, at, at,
                                 lib.moe_ffn_int4_workspace_bytes(8, E, H, I, 32), None, None)
    assert rc == L.MOE_ERR_INVALID_ARG and b"null" in lib.moe_last_error()


# ------------------------------------------------------------------ derivatives
def test_forward_mode_derivatives_are_refused() -> None:
    """A dual tensor does not require grad, and its tangent would be lost."""
    x = torch.ones(3)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3))
        assert not dual.requires_grad
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), pytest.raises(RuntimeError, match="forward-mode"):
                L.grad_wanted("op", None, dual)
        assert not L.grad_wanted("op", x)
        q = Int4StackedExpertWeights(int4(), int4(), int4(n=H, k=I))
        dual = forward_ad.make_dual(torch.zeros(T, H, dtype=BF16), torch.zeros(T, H, dtype=BF16))
        with pytest.raises(RuntimeError, match="forward-mode"):
            moe_layer_forward(dual, None, q, RouterConfig(top_k=K), topk=topk())
        with pytest.raises(RuntimeError, match="forward-mode"):
            grouped_moe_routed_quantized(dual, *topk(), q)
        with pytest.raises(RuntimeError, match="forward-mode"):
            moe_block_forward(dual, None, None, q, RouterConfig(top_k=K), normed=dual, topk=topk())
    assert not L.grad_wanted("op", x) and L.grad_wanted("op", x.clone().requires_grad_())


@pytest.mark.parametrize("which", ["x", "weight"])
def test_gradients_of_4_bit_layers_are_refused(which) -> None:
    x, (idx, w), q = torch.zeros(T, H, dtype=BF16), topk(), weights("int4")
    (x if which == "x" else w).requires_grad_()
    with pytest.raises(ValueError, match="inference"):
        moe_layer_forward(x, None, q, RouterConfig(top_k=K), topk=(idx, w))
    with pytest.raises(ValueError, match="inference"):
        grouped_moe_routed_quantized(x, idx, w, q)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        moe_layer_forward(x, None, q, RouterConfig(top_k=K), topk=(idx, w))
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        grouped_moe_routed_quantized(x, idx, w, q)


# ------------------------------------------------------------------ weights
def test_16_bit_weights_reach_the_quantised_call() -> None:
    with pytest.raises(ValueError, match="CUDA"):
        grouped_moe_routed_quantized(torch.zeros(T, H, dtype=BF16), *topk(), weights("bf16"))


@pytest.mark.parametrize("shared", [
    SharedExpertWeights(torch.zeros(8, H, dtype=BF16), torch.zeros(16, H, dtype=BF16), torch.zeros(H, 8, dtype=BF16)),
    SharedExpertWeights(torch.zeros(8, 32, dtype=BF16), torch.zeros(8, 32, dtype=BF16), torch.zeros(32, 8, dtype=BF16)),
    SharedExpertWeights(torch.zeros(8, H, dtype=BF16), torch.zeros(8, H, dtype=BF16), torch.zeros(8, H, dtype=BF16)),
    SharedExpertWeights(torch.zeros(8, H, dtype=BF16), torch.zeros(8, H), torch.zeros(H, 8, dtype=BF16)),
])
def test_a_shared_expert_that_does_not_fit_the_4_bit_ones_is_refused(shared) -> None:
    x = torch.zeros(T, H, dtype=BF16)
    off = torch.tensor([0, T, T, T, T], dtype=torch.int32)
    with pytest.raises(ValueError, match="shared expert"):
        expert_ffn(x, off, weights("int4"), shared, x)


def test_weights_of_another_order_are_refused() -> None:
    """(T, k) or flat: a transposed matrix has as many values."""
    i32 = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    grouping = TokenGrouping(torch.zeros(T * K, dtype=torch.int64), torch.ones(T * K), torch.zeros(E, dtype=torch.int64),
                             i32(E + 1), i32(T * K), torch.ones(T * K), K)
    y, dout = torch.zeros(T * K, H), torch.zeros(T, H)
    for w in (torch.ones(K, T), torch.ones(T, K, 1), torch.ones(1, T * K)):
        with pytest.raises(ValueError, match="topk_weight"):
            combine_tokens(y, grouping, w)
    for w in (torch.ones(T, K), torch.ones(T * K)):
        with pytest.raises(ValueError, match="CUDA"):
            combine_tokens(y, grouping, w)
        with pytest.raises(ValueError, match="CUDA"):
            combine_tokens_backward(dout, y, grouping, w)


# ------------------------------------------------------------------ schedules
def test_offsets_are_those_of_the_schedule_as_it_is() -> None:
    """What is uploaded is kept by value: a schedule whose offsets change is uploaded again."""
    cpu = torch.device("cpu")
    sched = SimpleNamespace(block_m=16, group_offsets=(0, 3, 7))
    first = device_offsets(sched, cpu)
    assert first.tolist() == [0, 3, 7] and device_offsets(sched, cpu) is first
    sched.group_offsets = (0, 5, 7)
    assert device_offsets(sched, cpu).tolist() == [0, 5, 7]
    sched.group_offsets = [0, 1, 7]
    assert device_offsets(sched, cpu).tolist() == [0, 1, 7]
    sched.group_offsets[1] = 2
    assert device_offsets(sched, cpu).tolist() == [0, 2, 7]
    again = copy.deepcopy(build_tile_schedule(torch.tensor([3, 4]), 16))
    assert device_offsets(again, cpu).tolist() == [0, 3, 7] and device_offsets(copy.deepcopy(again), cpu).tolist() == [0, 3, 7]


def test_the_exact_flag_travels_with_the_weights() -> None:
    assert not int4().exact
    codes, scale = torch.zeros(E, I, H, dtype=torch.int8), torch.ones(E, I, H // 32)
    assert pack_int4(codes, scale, 32, exact=True).exact
