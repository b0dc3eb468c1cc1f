"""Calls of the operators around the layer as programs make them: graphs that
are replayed in any order, other streams and devices, empty batches."""

from __future__ import annotations

import dataclasses

import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU hosts too
    pytest.skip("needs a CUDA device", allow_module_level=True)

from gpu_helpers import LayerWeights  # noqa: E402

from dispatch_b200 import _lib as L  # noqa: E402
from dispatch_b200.kernels.block import norm_gate_residual, norm_gate_residual_backward, rms_norm  # noqa: E402
from dispatch_b200.kernels.grouped_gemm import grouped_matmul  # noqa: E402
from dispatch_b200.kernels.grouped_gemm_int4 import expert_ffn_int4, grouped_matmul_int4  # noqa: E402
from dispatch_b200.kernels.grouping import (  # noqa: E402
    combine_tokens,
    combine_tokens_backward,
    group_tokens_by_expert,
    permute_tokens,
    permute_tokens_backward,
)
from dispatch_b200.kernels.layer import RouterConfig, moe_layer_forward  # noqa: E402
from dispatch_b200.kernels.moe_forward import SharedExpertWeights, StackedExpertWeights, grouped_moe_routed  # noqa: E402
from dispatch_b200.kernels.quantization import (  # noqa: E402
    grouped_moe_routed_quantized,
    pack_int4,
    quantize_stacked_weights_int4,
)
from dispatch_b200.kernels.tile_schedule import build_tile_schedule  # noqa: E402

DEV = torch.device("cuda", 0)
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _device_status_clean():
    yield
    L.check_device_status(DEV)


def grouped(t=33, k=6, e=64, h=512, dev=DEV, wdtype=F32):
    g = torch.Generator().manual_seed(t)
    idx = torch.multinomial(torch.ones(t, e), k, generator=g).to(dev)
    w = torch.rand(t, k, generator=g).to(dev, wdtype)
    x = torch.randn(t, h, generator=g).to(dev, BF16)
    y = torch.randn(t * k, h, generator=g).to(dev, BF16)
    return x, y, w, idx, group_tokens_by_expert(idx, w, e)


# ------------------------------------------------------------------ graphs
def test_errors_of_graphs_captured_before_any_eager_call(monkeypatch) -> None:
    """Their status word is zero before any replay, keeps what one graph
    reports when another is replayed, and is cleared by the check alone."""
    x, _, _, _, good = grouped()
    pos = good.pos.clone()
    pos[3] = x.shape[0] * 6  # one past the last row
    bad = dataclasses.replace(good, pos=pos)
    permute_tokens(x, good)
    monkeypatch.setattr(L, "_status", {})
    monkeypatch.setattr(L, "_captured_status", {})
    graphs = []
    for grouping in (good, bad):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = permute_tokens(x, grouping)
        graphs.append((g, out))
    L.check_device_status(DEV)  # neither has run
    (ok, xs), (wrong, _) = graphs
    for order in ((wrong,), (wrong, ok), (ok, wrong)):
        for g in order:
            g.replay()
        with pytest.raises(L.MoeDeviceError, match="positions out of range"):
            L.check_device_status(DEV)
        L.check_device_status(DEV)
    ok.replay()
    L.check_device_status(DEV)
    assert torch.equal(xs, permute_tokens(x, good))


@pytest.mark.parametrize("first", ["captured", "eager"])
def test_products_in_a_graph_that_outlives_its_schedule(first) -> None:
    """The graph reads offsets that were copied before its replay and that
    nothing else is given; an eager call before the replay reads them too."""
    x = torch.randn(21, 64, device=DEV).to(BF16)
    w = torch.randn(4, 32, 64, device=DEV).to(BF16)
    codes = torch.randint(-8, 8, (4, 32, 64), device=DEV).to(torch.int8)
    q = pack_int4(codes, torch.ones(4, 32, 1, device=DEV) / 16, 64)
    sizes = torch.tensor([3, 0, 7, 11])
    want = grouped_matmul_int4(x, q, build_tile_schedule(sizes, 16)), grouped_matmul(x, w, build_tile_schedule(sizes, 16))
    sched = build_tile_schedule(sizes, 16)
    if first == "eager":
        assert torch.equal(grouped_matmul_int4(x, q, sched), want[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = grouped_matmul_int4(x, q, sched), grouped_matmul(x, w, sched)
    assert torch.equal(grouped_matmul_int4(x, q, sched), want[0])
    del sched
    for _ in range(200):
        torch.full((5,), -1, dtype=torch.int32, device=DEV)
    for _ in range(2):
        for t in got:
            t.zero_()
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------ streams
def test_a_schedule_used_on_another_stream() -> None:
    """Its offsets are copied behind whatever the first stream is doing, and the second stream waits for the copy."""
    x = torch.randn(21, 64, device=DEV).to(BF16)
    q = pack_int4(torch.ones(4, 32, 64, dtype=torch.int8, device=DEV), torch.ones(4, 32, 1, device=DEV) / 16, 64)
    sizes = torch.tensor([3, 0, 7, 11])
    want = grouped_matmul_int4(x, q, build_tile_schedule(sizes, 16))
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        sched = build_tile_schedule(sizes, 16)
        with torch.cuda.stream(a):
            torch.cuda._sleep(2_000_000)
            first = grouped_matmul_int4(x, q, sched)
        with torch.cuda.stream(b):
            second = grouped_matmul_int4(x, q, sched)
        del sched
        torch.cuda.synchronize()
        assert torch.equal(first, want) and torch.equal(second, want)


@pytest.mark.parametrize("wdtype", [F32, BF16])
def test_sizes_belong_to_the_stream_that_made_them(wdtype) -> None:
    """What a grouping holds is made when it is: reading it elsewhere launches
    nothing, so record_stream of what was read protects the memory itself."""
    _, _, w, idx, grouping = grouped(wdtype=wdtype)
    want = torch.bincount(idx.flatten(), minlength=64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = grouping.group_sizes, grouping.sorted_weight
    with torch.cuda.graph(torch.cuda.CUDAGraph()):  # never replayed
        captured = grouping.group_sizes, grouping.sorted_weight
    for a, b, c in zip(there, captured, (grouping.group_sizes, grouping.sorted_weight)):
        assert a is b and b is c
    assert there[0].dtype == torch.int64 and there[1].dtype == wdtype
    assert torch.equal(there[0], want)
    order = torch.sort(idx.flatten(), stable=True).indices
    assert torch.equal(there[1], w.flatten()[order])


def test_a_dropped_groupings_sizes_read_on_another_stream() -> None:
    want = torch.bincount(grouped()[3].flatten(), minlength=64)
    side = torch.cuda.Stream()
    for _ in range(20):
        grouping = grouped()[4]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(200_000)
            sizes = grouping.group_sizes
            sizes.record_stream(side)
            del grouping
            got = sizes + 0
            del sizes
        for _ in range(8):  # what the making stream allocates next
            torch.full((64,), -1, device=DEV)
            torch.full((64,), -1, device=DEV, dtype=torch.int32)
        side.synchronize()
        assert torch.equal(got, want)


# ------------------------------------------------------------------ derivatives
def test_forward_mode_derivatives_are_refused() -> None:
    x, y, w, _, grouping = grouped()
    weight = torch.ones(512, device=DEV)
    q = pack_int4(torch.zeros(1, 16, 512, dtype=torch.int8, device=DEV), torch.ones(1, 16, 4, device=DEV), 128)
    calls = [(lambda d: rms_norm(d, weight), x), (lambda d: rms_norm(x, d), weight),
             (lambda d: norm_gate_residual(x, d, weight), x), (lambda d: permute_tokens(d, grouping), x),
             (lambda d: combine_tokens(d, grouping, w), y), (lambda d: combine_tokens(y, grouping, d), w),
             (lambda d: grouped_matmul_int4(d, q, build_tile_schedule(torch.tensor([33]), 16)), x)]
    with forward_ad.dual_level():
        for call, t in calls:
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(forward_ad.make_dual(t, torch.ones_like(t)))
            call(t)  # an ordinary tensor inside the level


@pytest.mark.parametrize("what", ["weights", "grouping's weights", "positions", "rows"])
def test_inputs_changed_before_the_backward_are_noticed(what) -> None:
    x, y, w, _, grouping = grouped()
    y = y.requires_grad_()
    out = combine_tokens(y, grouping, w if what == "weights" else None)
    with torch.no_grad():
        {"weights": w, "grouping's weights": w, "positions": grouping.pos, "rows": y}[what].add_(0)
    with pytest.raises(RuntimeError, match="inplace operation"):
        out.sum().backward()
    x = x.requires_grad_()
    xs = permute_tokens(x, grouping)
    with torch.no_grad():
        x.add_(1)  # the gather's gradient does not need it
    xs.sum().backward()
    assert torch.equal(x.grad, torch.full_like(x, 6))


# ------------------------------------------------------------------ layers
def test_16_bit_weights_in_the_quantised_call() -> None:
    w = LayerWeights(256, 192, 16)
    weights = StackedExpertWeights(w.gate, w.up, w.down)
    x, _, wt, idx, _ = grouped(t=19, k=4, e=16, h=256)
    assert torch.equal(grouped_moe_routed_quantized(x, idx, wt, weights), grouped_moe_routed(x, idx, wt, weights))


def test_strided_weights() -> None:
    """Their copies live until the launch, each in memory of its own."""
    w = LayerWeights(256, 192, 16, 320)
    x, _, wt, idx, _ = grouped(t=19, k=4, e=16, h=256)
    strided = lambda t: t.transpose(-1, -2).contiguous().transpose(-1, -2)  # noqa: E731
    plain = StackedExpertWeights(w.gate, w.up, w.down), SharedExpertWeights(*w.shared)
    other = StackedExpertWeights(*map(strided, (w.gate, w.up, w.down))), SharedExpertWeights(*map(strided, w.shared))
    cfg = RouterConfig(top_k=4)
    for shared in (False, True):
        a, b = (moe_layer_forward(x, w.router, p[0], cfg, shared=p[1] if shared else None).out for p in (plain, other))
        assert torch.equal(a, b)
        a, b = (grouped_moe_routed(x, idx, wt, p[0], shared=p[1] if shared else None) for p in (plain, other))
        assert torch.equal(a, b)


def test_a_4_bit_layer_without_tokens() -> None:
    w = LayerWeights(256, 192, 16, 320)
    q = quantize_stacked_weights_int4(StackedExpertWeights(w.gate, w.up, w.down), group_size=64)
    x = torch.empty(0, 256, device=DEV, dtype=BF16)
    for shared in (None, SharedExpertWeights(*w.shared)):
        out = moe_layer_forward(x, w.router, q, RouterConfig(top_k=4), shared=shared)
        assert out.out.shape == (0, 256) and out.topk_idx.shape == (0, 4) and not out.group_offsets.any()


def test_ffn_with_strided_offsets(monkeypatch) -> None:
    """Their copy lives until the launch, whatever is allocated on the way to it."""
    w = LayerWeights(256, 192, 4)
    q = quantize_stacked_weights_int4(StackedExpertWeights(w.gate, w.up, w.down))
    x = torch.randn(21, 256, device=DEV).to(BF16)
    off = torch.tensor([0, 3, 3, 10, 21], dtype=torch.int32, device=DEV)
    want = expert_ffn_int4(x, off, q)
    word = L.status_word(DEV)
    made = []

    def allocate(device):
        made.extend(torch.full((5,), -1, dtype=torch.int32, device=DEV) for _ in range(500))
        return word

    monkeypatch.setattr(L, "status_word", allocate)
    assert torch.equal(expert_ffn_int4(x, off.repeat_interleave(2)[::2], q), want) and made


# ------------------------------------------------------------------ devices
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two devices")
def test_every_form_on_a_second_device() -> None:
    """The first device's calls come first, and it stays the current one."""
    results = []
    for dev in (torch.device("cuda", 0), torch.device("cuda", 1)):
        got = []
        g = torch.Generator().manual_seed(0)
        codes = torch.randint(-8, 8, (2, 48, 256), generator=g).to(torch.int8).to(dev)
        for group in (32, 128):
            q = pack_int4(codes, torch.ones(2, 48, 256 // group, device=dev) / 16, group)
            for rows in (3, 20, 60, 100, 300):
                x = torch.randn(2 * rows, 256, generator=g).to(dev, BF16)
                got.append(grouped_matmul_int4(x, q, build_tile_schedule(torch.tensor([rows, rows]), 16)))
        x, y, w, idx, grouping = grouped(dev=dev)
        got += [permute_tokens(x, grouping), combine_tokens(y, grouping, w), permute_tokens_backward(y, grouping),
                *combine_tokens_backward(x, y, grouping, w)]
        weight = torch.ones(512, device=dev)
        got += [*norm_gate_residual(x, x, weight, weight), *norm_gate_residual_backward(x, x, x, x, weight, weight)[:4]]
        stacked = StackedExpertWeights(*((torch.randn(64, a, b, generator=g) / 16).to(dev, BF16)
                                         for a, b in ((48, 512), (48, 512), (512, 48))))
        router_weight = torch.randn(64, 512, generator=g).to(dev, BF16)
        for weights in (stacked, quantize_stacked_weights_int4(stacked, group_size=64)):
            got.append(moe_layer_forward(x, router_weight, weights, RouterConfig(top_k=6)).out)
            got.append(moe_layer_forward(x, None, weights, RouterConfig(top_k=6), topk=(idx, w)).out)
        results.append([t.cpu() for t in got])
        L.check_device_status(dev)
    assert all(torch.equal(a, b) for a, b in zip(*results))
