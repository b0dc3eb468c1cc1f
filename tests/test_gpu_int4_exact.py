"""4-bit products whose weights are rounded at no batch size
(``Int4Tensor.exact``); tolerances as in test_gpu_int4.py."""

from __future__ import annotations

import dataclasses

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU hosts too
    pytest.skip("needs a CUDA device", allow_module_level=True)

from gpu_helpers import LayerWeights  # noqa: E402
from test_gpu_int4 import BF16, DEV, F16, F32, check, deep, exact_rows, ffn64, ffn_weights, make, weights64  # noqa: E402

from dispatch_b200 import _lib as L  # noqa: E402
from dispatch_b200.kernels.grouped_gemm_int4 import expert_ffn_int4, grouped_matmul_int4  # noqa: E402
from dispatch_b200.kernels.grouping import combine_tokens, group_tokens_by_expert, permute_tokens  # noqa: E402
from dispatch_b200.kernels.layer import CapturedLayer, RouterConfig, moe_layer_forward  # noqa: E402
from dispatch_b200.kernels.moe_forward import StackedExpertWeights  # noqa: E402
from dispatch_b200.kernels.quantization import (  # noqa: E402
    Int4StackedExpertWeights,
    pack_int4,
    quantize_groupwise_int4,
    quantize_stacked_weights_int4,
    unpack_int4,
)
from dispatch_b200.kernels.tile_schedule import build_tile_schedule  # noqa: E402


@pytest.fixture(autouse=True)
def _device_status_clean():
    yield
    L.check_device_status(DEV)


def check_exact(out, x, q, offsets):
    w = weights64(q)
    for e in range(q.num_experts):
        a, b = offsets[e], offsets[e + 1]
        if b > a:
            xe = x[a:b].double()
            check(out[a:b], xe @ w[e].t(), deep(q.k) * (xe.abs() @ w[e].t().abs()))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize(("sizes", "n", "k"), [
    ([5], 40, 136), ([129], 16, 64), ([300, 0, 1, 257], 136, 520), ([170, 0, 300], 17, 72), ([400, 330, 900], 512, 1408),
    ([0, 2000], 1, 8),
])
def test_no_weight_is_rounded(sizes, n, k, group, dtype) -> None:
    q, g = make(len(sizes), n, k, group)
    q = dataclasses.replace(q, exact=True)
    sched = build_tile_schedule(torch.tensor(sizes), 16)
    x = torch.randn(sum(sizes), k, generator=g, device=DEV).to(dtype)
    check_exact(grouped_matmul_int4(x, q, sched), x, q, sched.group_offsets)


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("rows", [5, 20, 60, 100, 150, 700])
def test_weights_outside_f16s_range(rows, group) -> None:
    """code * scale up to 80000 and down to 2^-20, with products that f16 holds."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    codes = torch.randint(-8, 8, (2, 48, 128), generator=g, device=DEV).to(torch.int8)
    scale = torch.full((2, 48, 128 // group), 1e4, device=DEV)
    scale[:, ::2] = 2.0**-20
    q = pack_int4(codes, scale, group, exact=True)
    x = torch.zeros(2 * rows, 128, device=DEV, dtype=F16)
    x[torch.arange(2 * rows), torch.randint(0, 128, (2 * rows,), generator=g.manual_seed(1), device=DEV)] = 2.0**-2
    out = grouped_matmul_int4(x, q, build_tile_schedule(torch.tensor([rows, rows]), 16))
    assert torch.isfinite(out).all()
    check_exact(out, x, q, [0, rows, 2 * rows])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize(("sizes", "i", "h", "group"), [([200, 0, 190], 104, 520, 128), ([140, 33, 100], 72, 264, 64),
                                                        ([90, 0, 100], 200, 264, 32)])
def test_expert_ffn(sizes, i, h, group, dtype) -> None:
    ws = ffn_weights(len(sizes), i, h, group)
    ws = Int4StackedExpertWeights(ws.gate, ws.up, dataclasses.replace(ws.down, exact=True))  # one of the three is enough
    assert sum(sizes) > exact_rows(group) * len(sizes)
    off = torch.tensor([0, *torch.tensor(sizes).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    xs = torch.randn(sum(sizes), h, generator=torch.Generator(device="cuda").manual_seed(7), device=DEV).to(dtype)
    # ffn64's weights follow the rounding above the limit: the formula itself comes from rows in small parts
    parts = [ffn64(xs[a:b], [0] * (e + 1) + [b - a] * (len(sizes) - e), ws, dtype)
             for e, (lo, hi) in enumerate(zip(off.tolist(), off.tolist()[1:])) for a in range(lo, hi, 40)
             for b in (min(hi, a + 40),)]
    check(expert_ffn_int4(xs, off, ws), torch.cat([y for y, _ in parts]), torch.cat([b for _, b in parts]))


def test_layer_and_captured_layer() -> None:
    h, i, e, k, t = 256, 192, 4, 2, 700
    w = LayerWeights(h, i, e)
    q = quantize_stacked_weights_int4(StackedExpertWeights(w.gate, w.up, w.down), group_size=64, exact=True)
    assert q.gate.exact and q.up.exact and q.down.exact and quantize_groupwise_int4(w.gate, exact=True).exact
    x = torch.randn(t, h, device=DEV).to(BF16)
    cfg = RouterConfig(top_k=k)
    got = moe_layer_forward(x, w.router, q, cfg)
    grouping = group_tokens_by_expert(got.topk_idx, got.topk_weight, e)
    y = expert_ffn_int4(permute_tokens(x, grouping), grouping.offsets, q)
    assert torch.equal(got.out, combine_tokens(y, grouping))
    assert torch.equal(CapturedLayer(x, w.router, q, cfg)(x), got.out)
    rounded = quantize_stacked_weights_int4(StackedExpertWeights(w.gate, w.up, w.down), group_size=64)
    assert not rounded.gate.exact and not torch.equal(moe_layer_forward(x, w.router, rounded, cfg).out, got.out)


def test_from_c_without_a_workspace() -> None:
    rows, n, k, group = 300, 40, 128, 128
    q, g = make(1, n, k, group)
    x = torch.randn(rows, k, generator=g, device=DEV).to(BF16)
    off = torch.tensor([0, rows], dtype=torch.int32, device=DEV)
    out = torch.empty(rows, n, device=DEV, dtype=BF16)
    need = L.lib().moe_int4_workspace_bytes(rows, 1, n, k, group)
    assert need > 0
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)

    def call(ptr, nbytes):
        return L.lib().moe_grouped_gemm_int4(
            x.data_ptr(), L.DT_BF16, rows, k, q.data.data_ptr(), q.scale.data_ptr(), L.DT_F32, group, 1, n,
            off.data_ptr(), out.data_ptr(), n, ptr, nbytes, L.status_word(DEV).data_ptr(), L.stream_ptr(DEV))

    assert call(None, 0) == L.MOE_OK
    check_exact(out, x, q, [0, rows])
    assert call(ws.data_ptr(), need - 1) == L.MOE_ERR_INVALID_ARG  # room that is too small is a mistake
    assert q.scale.dtype == F32


@pytest.mark.parametrize("scale_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_non_finite_weights_do_not_become_finite(bad, scale_dtype) -> None:
    """The quantiser's formula: their group's scale is not finite; every other group is as without them."""
    g = torch.Generator(device="cuda").manual_seed(0)
    w = torch.randn(2, 20, 200, generator=g, device=DEV)
    want = quantize_groupwise_int4(w, group_size=32, scale_dtype=scale_dtype)
    w[1, 17, 70] = bad  # of group 2
    got = quantize_groupwise_int4(w, group_size=32, scale_dtype=scale_dtype)
    scale, sane = unpack_int4(got)[1], unpack_int4(want)[1]
    hit = torch.zeros_like(scale, dtype=torch.bool)
    hit[1, 17, 2] = True
    assert not torch.isfinite(scale[hit]).any() and torch.equal(scale[~hit], sane[~hit])
    columns = hit.repeat_interleave(32, 2)[..., :200]
    assert torch.equal(unpack_int4(got)[0][~columns], unpack_int4(want)[0][~columns])
    x = torch.randn(6, 200, generator=g, device=DEV).to(BF16)
    out = grouped_matmul_int4(x, got, build_tile_schedule(torch.tensor([3, 3]), 16))
    assert not torch.isfinite(out[3:, 17]).any()
    out[3:, 17] = 0
    assert torch.isfinite(out).all()
