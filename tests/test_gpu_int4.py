"""The 4-bit expert products against their formula in 64 bits.

Tolerances: an output is rounded once to its type (half a step of the value);
f32 accumulation in MMA steps of 16 columns, each off by at most one unit 2u =
2^-23 of the magnitudes added up so far, and a few products and joins: K / 8 +
64 times u = 2^-24 of sum |x w|. With many rows per expert each weight is rounded
once to x's type, which the formula's weights follow; else none is. The FFN's
intermediate rows are rounded to x's type: half a step of each, through the down
weights."""

from __future__ import annotations

import pytest
import torch
from test_gpu_surfaces import DeepseekStyleMoE

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU hosts too
    pytest.skip("needs a CUDA device", allow_module_level=True)

from gpu_helpers import LayerWeights, assert_int8_parity  # noqa: E402

from dispatch_b200 import _lib as L  # noqa: E402
from dispatch_b200.kernels.block import norm_gate_residual, rms_norm  # noqa: E402
from dispatch_b200.kernels.grouped_gemm_int4 import expert_ffn_int4, grouped_matmul_int4  # noqa: E402
from dispatch_b200.kernels.integration import patch_moe_infer_quantized  # noqa: E402
from dispatch_b200.kernels.layer import CapturedLayer, RouterConfig, moe_block_forward, moe_layer_forward  # noqa: E402
from dispatch_b200.kernels.moe_forward import SharedExpertWeights, StackedExpertWeights, grouped_moe_routed  # noqa: E402
from dispatch_b200.kernels.quantization import (  # noqa: E402
    Int4StackedExpertWeights,
    Int4Tensor,
    dequantize_int4,
    grouped_moe_routed_quantized,
    pack_int4,
    quantize_groupwise_int4,
    quantize_stacked_weights_int4,
    quantized_stacked_weights_nbytes,
    unpack_int4,
)
from dispatch_b200.kernels.tile_schedule import build_tile_schedule  # noqa: E402

DEV = torch.device("cuda", 0)
U = 2.0**-24
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _device_status_clean():
    yield
    L.check_device_status(DEV)


def deep(k):
    return (k / 8 + 64) * U


def make(e, n, k, group, scale_dtype=F32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(-8, 8, (e, n, k), generator=g, device=DEV).to(torch.int8)
    scale = ((torch.rand(e, n, -(-k // group), generator=g, device=DEV) + 0.3) / k**0.5).to(scale_dtype)
    return pack_int4(codes, scale, group), g


def exact_rows(group):
    """MOE_INT4_EXACT_ROWS: the codes themselves are multiplied up to this average."""
    return 128 if group >= 128 else 48


def weights64(q, rows=0, dtype=None):
    """The formula's weights for a product of `rows` rows."""
    codes, scale = unpack_int4(q)
    w = codes.double() * scale.double().repeat_interleave(q.group_size, 2)[..., :q.k]
    return w if rows <= exact_rows(q.group_size) * q.num_experts else w.to(dtype).double()


def check(actual, value, bound):
    half = torch.finfo(actual.dtype).eps / 2
    bound = half * value.abs() + (1 + half) * bound + (2.0**-25 if actual.dtype == F16 else 0.0)
    off = (actual.double() - value).abs()
    assert bool((off <= bound).all()), f"off by {off.max().item():.3g}, {((off / bound).max().item()):.3g} of the bound"


def check_product(out, x, q, offsets):
    w = weights64(q, x.shape[0], x.dtype)
    for e in range(q.num_experts):
        a, b = offsets[e], offsets[e + 1]
        if b > a:
            xe = x[a:b].double()
            check(out[a:b], xe @ w[e].t(), deep(q.k) * (xe.abs() @ w[e].t().abs()))


def run(sizes, n, k, group, dtype=BF16, scale_dtype=F32, seed=0):
    q, g = make(len(sizes), n, k, group, scale_dtype, seed)
    sched = build_tile_schedule(torch.tensor(sizes), 16)
    x = torch.randn(sum(sizes), k, generator=g, device=DEV).to(dtype)
    out = grouped_matmul_int4(x, q, sched)
    assert out.shape == (sum(sizes), n) and out.dtype == dtype
    check_product(out, x, q, sched.group_offsets)
    return x, q, sched, out


# ------------------------------------------------------------------ products
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize(("sizes", "n", "k"), [
    ([1], 16, 64), ([1], 1, 8), ([0, 1, 0], 17, 72), ([3, 0, 1, 8, 9], 100, 1416), ([1] * 6, 1408, 2048),
    ([5, 6, 0, 7], 250, 520), ([11, 33, 0, 2], 72, 264), ([23, 1], 48, 136), ([2, 0], 33, 4168),
])
def test_few_rows(sizes, n, k, group, dtype) -> None:
    assert sum(sizes) <= 12 * len(sizes)
    run(sizes, n, k, group, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize(("sizes", "n", "k"), [
    ([13], 16, 64), ([48], 1, 8), ([70, 1], 48, 136), ([0, 100, 0, 17], 17, 72), ([65, 0, 16, 30, 129], 100, 1416),
    ([40] * 3, 1408, 2048), ([300, 0, 1, 0, 2, 0, 5], 250, 520),
])
def test_tiles_of_64_rows(sizes, n, k, group, dtype) -> None:
    assert 12 * len(sizes) < sum(sizes) <= 48 * len(sizes)
    run(sizes, n, k, group, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("group", [128, 256])
@pytest.mark.parametrize(("sizes", "n", "k"), [
    ([65], 16, 64), ([49], 48, 136), ([128], 1, 8), ([0, 250], 17, 72), ([130, 0, 256, 33, 129], 100, 1416), ([100] * 3, 1408, 2048),
    ([300, 0, 1, 200], 250, 520),
])
def test_tiles_of_128_rows(sizes, n, k, group, dtype) -> None:
    assert 48 * len(sizes) < sum(sizes) <= exact_rows(group) * len(sizes)
    run(sizes, n, k, group, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize(("sizes", "n", "k", "group"), [
    ([65], 16, 64, 32), ([300, 0, 1, 257], 136, 520, 64), ([512, 512], 256, 264, 128), ([170, 0, 300], 17, 72, 256),
    ([400, 330, 900], 2048, 1408, 128), ([90, 40, 100], 72, 456, 32),
])
def test_many_rows(sizes, n, k, group, dtype) -> None:
    assert sum(sizes) > exact_rows(group) * len(sizes)
    run(sizes, n, k, group, dtype)


@pytest.mark.parametrize("scale_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("sizes", [[2, 5, 1], [90, 40, 3], [190, 40, 13], [300, 100]])
def test_scale_types(sizes, scale_dtype) -> None:
    for group in (32, 128):
        run(sizes, 80, 456, group, BF16, scale_dtype)
        run(sizes, 80, 456, group, F16, scale_dtype)


@pytest.mark.parametrize("group", [64, 128])
@pytest.mark.parametrize("rows", [6, 7, 12, 13, 48, 49, 128, 129])
def test_around_the_change_of_kernels(rows, group) -> None:
    run([rows] * 3, 96, 256, group)


def test_experts_made_in_several_chunks() -> None:
    """16-bit weights of 4 experts at most fit the workspace at a time."""
    sizes = [140, 0, 133, 270, 190, 1, 133, 160, 136]
    n, k = 8192, 4096
    ws = L.lib().moe_int4_workspace_bytes(sum(sizes), len(sizes), n, k, 128)
    assert 0 < ws < len(sizes) * n * k * 2
    run(sizes, n, k, 128)


def test_a_row_does_not_depend_on_its_batch() -> None:
    x, q, _, out = run([1, 4, 2], 144, 1096, 64, seed=4)
    one = x[4:5]  # of expert 1
    for sizes, at in (([0, 1, 0], 0), ([3, 9, 0], 7), ([8, 20, 8], 20), ([2, 32, 2], 30)):
        g = torch.Generator(device="cuda").manual_seed(sum(sizes))
        batch = torch.randn(sum(sizes), 1096, generator=g, device=DEV).to(BF16)
        batch[at] = one
        got = grouped_matmul_int4(batch, q, build_tile_schedule(torch.tensor(sizes), 16))
        assert torch.equal(got[at], out[4])


def test_every_code_and_non_finite_rows() -> None:
    k = 64
    codes = torch.arange(k).remainder(16).sub(8).repeat(1, 16, 1).to(torch.int8)
    codes[0, 1:] = codes[0, 1:].flip(1)
    scale = torch.ones(1, 16, 1)
    scale[0, 3] = 0.0
    q = pack_int4(codes.to(DEV), scale.to(DEV), 128)
    for dtype in (BF16, F16):
        x = torch.eye(k, device=DEV).to(dtype)  # column k of the weights, exactly
        for rows in (12, 48, 128, 192):
            x_rows = x.repeat(3, 1)[:rows]
            out = grouped_matmul_int4(x_rows, q, build_tile_schedule(torch.tensor([rows]), 16))
            assert torch.equal(out, (codes[0].float() * scale[0]).t().repeat(3, 1)[:rows].to(DEV, dtype))
        for rows in (5, 20, 100, 150):  # a row's infinities and NaN are its own
            x_rows = torch.ones(rows, k, device=DEV, dtype=dtype)
            x_rows[1, 3], x_rows[3, 60] = float("inf"), float("nan")
            out = grouped_matmul_int4(x_rows, q, build_tile_schedule(torch.tensor([rows]), 16))
            rest = [i for i in range(rows) if i not in (1, 3)]
            assert torch.isfinite(out[rest]).all() and torch.isnan(out[3]).all() and not torch.isfinite(out[1]).all()


@pytest.mark.parametrize("rows", [5, 20, 100, 150])
def test_rows_past_the_last_expert_are_left_alone(rows) -> None:
    q, g = make(1, 40, 128, 128)
    x = torch.randn(rows + 9, 128, generator=g, device=DEV).to(BF16)
    x[rows:] = float("nan")
    out = torch.full((rows + 9, 40), 7.0, device=DEV, dtype=BF16)
    off = torch.tensor([0, rows], dtype=torch.int32, device=DEV)
    ws = torch.empty(max(L.lib().moe_int4_workspace_bytes(rows + 9, 1, 40, 128, 128), 16), dtype=torch.uint8, device=DEV)
    rc = L.lib().moe_grouped_gemm_int4(
        x.data_ptr(), L.DT_BF16, rows + 9, 128, q.data.data_ptr(), q.scale.data_ptr(), L.DT_F32, 128, 1, 40,
        off.data_ptr(), out.data_ptr(), 40, ws.data_ptr(), ws.numel(), L.status_word(DEV).data_ptr(),
        L.stream_ptr(DEV))
    assert rc == L.MOE_OK
    w = weights64(q, rows + 9, BF16)[0]
    xe = x[:rows].double()
    check(out[:rows], xe @ w.t(), deep(128) * (xe.abs() @ w.t().abs()))
    assert bool((out[rows:] == 7.0).all())


def test_strided_and_unaligned_rows() -> None:
    q, g = make(2, 40, 128, 64)
    sched = build_tile_schedule(torch.tensor([3, 4]), 16)
    wide = torch.randn(7, 300, generator=g, device=DEV).to(BF16)
    for x in (wide[:, 8:136], wide[:, 3:131], wide.t().contiguous().t()[:, :128]):
        assert torch.equal(grouped_matmul_int4(x, q, sched), grouped_matmul_int4(x.clone(), q, sched))


def test_no_rows() -> None:
    q, _ = make(2, 40, 128, 64)
    assert grouped_matmul_int4(torch.empty(0, 128, device=DEV, dtype=BF16), q,
                               build_tile_schedule(torch.tensor([0, 0]), 16)).shape == (0, 40)


def test_weights_past_4_gib() -> None:
    """Byte offsets of the last experts' weights pass 32 bits."""
    e, n, k, group = 256, 4864, 7168, 256
    data = torch.randint(-2**31, 2**31 - 1, (e, n // 16, k // 64, 32, 4), dtype=torch.int32, device=DEV)
    assert data.numel() * 4 > 2**32
    scale = torch.full((e, n // 16, k // group, 16), 1 / 64, device=DEV, dtype=BF16)
    for last in (3, 4000):  # a few rows, and a batch of tiles
        sizes = [0] * e
        sizes[0], sizes[255] = 2, last
        x = torch.randn(sum(sizes), k, device=DEV).to(BF16)
        sched = build_tile_schedule(torch.tensor(sizes), 16)
        out = grouped_matmul_int4(x, Int4Tensor(data, scale, n, k, group), sched)
        for i, a, b in ((0, 0, 2), (255, 2, 2 + last)):
            one = Int4Tensor(data[i:i + 1], scale[i:i + 1], n, k, group)
            w = weights64(one)[0]
            check(out[a:b], x[a:b].double() @ w.t(), deep(k) * (x[a:b].double().abs() @ w.t().abs()))


def test_bad_offsets_are_reported() -> None:
    q, g = make(3, 40, 128, 128)
    for rows in (6, 100, 350, 500):
        x = torch.randn(rows, 128, generator=g, device=DEV).to(BF16)
        out = torch.full((rows, 40), 7.0, device=DEV, dtype=BF16)
        ws = torch.empty(max(L.lib().moe_int4_workspace_bytes(rows, 3, 40, 128, 128), 16), dtype=torch.uint8, device=DEV)
        for offsets in ([0, 2, 4, rows + 1], [0, 4, 2, rows], [-1, 2, 4, rows]):
            off = torch.tensor(offsets, dtype=torch.int32, device=DEV)
            rc = L.lib().moe_grouped_gemm_int4(
                x.data_ptr(), L.DT_BF16, rows, 128, q.data.data_ptr(), q.scale.data_ptr(), L.DT_F32, 128, 3, 40,
                off.data_ptr(), out.data_ptr(), 40, ws.data_ptr(), ws.numel(), L.status_word(DEV).data_ptr(),
                L.stream_ptr(DEV))
            assert rc == L.MOE_OK
            with pytest.raises(L.MoeDeviceError, match="offsets"):
                L.check_device_status(DEV)
            assert bool((out == 7.0).all())


# ------------------------------------------------------------------ quantiser
@pytest.mark.parametrize("scale_dtype", [F32, BF16, F16])
@pytest.mark.parametrize(("e", "n", "k", "group", "dtype"), [(2, 17, 72, 32, BF16), (1, 64, 1416, 128, F32),
                                                             (3, 30, 520, 64, F16), (1, 5, 264, 256, BF16)])
def test_quantiser_is_its_formula(e, n, k, group, dtype, scale_dtype) -> None:
    g = torch.Generator(device="cuda").manual_seed(0)
    w = torch.randn(e, n, k, generator=g, device=DEV).to(dtype)
    w[0, 0, :group] = 0
    q = quantize_groupwise_int4(w, group_size=group, scale_dtype=scale_dtype)
    groups = -(-k // group)
    padded = torch.nn.functional.pad(w.float(), (0, groups * group - k)).view(e, n, groups, group)
    top = padded.abs().amax(3)
    scale = torch.where(top == 0, torch.ones_like(top), top / torch.full_like(top, 7)).to(scale_dtype)
    codes = (padded / scale.float()[..., None]).round().clamp(-8, 7).view(e, n, -1)[..., :k]
    got, got_scale = unpack_int4(q)
    assert torch.equal(got_scale, scale) and torch.equal(got.float(), codes)
    again = pack_int4(got, got_scale, group)
    assert torch.equal(again.data, q.data)


# ------------------------------------------------------------------ FFN, layer, block
def ffn64(xs, offsets, ws, dtype):
    """y and its bound in 64 bits, with the intermediate rows' rounding."""
    rows = xs.shape[0]
    wg, wu, wd = (weights64(q, rows, dtype) for q in (ws.gate, ws.up, ws.down))
    half = torch.finfo(dtype).eps / 2
    y = torch.zeros(rows, ws.down.n, dtype=torch.float64, device=DEV)
    bound = torch.zeros_like(y)
    for e in range(ws.num_experts):
        a, b = offsets[e], offsets[e + 1]
        if a == b:
            continue
        x = xs[a:b].double()
        gate, up = x @ wg[e].t(), x @ wu[e].t()
        dk = deep(ws.gate.k)
        d_gate, d_up = dk * (x.abs() @ wg[e].t().abs()), dk * (x.abs() @ wu[e].t().abs())
        silu = gate * torch.sigmoid(gate)
        h = silu * up
        # |silu'| <= 1.1; exp in f32 is off by a few units of its argument: 2^-20
        d_h = (half + 2.0**-20) * h.abs() + 1.1 * d_gate * (up.abs() + d_up) + silu.abs() * d_up + 2.0**-25
        y[a:b] = h @ wd[e].t()
        bound[a:b] = d_h @ wd[e].t().abs() + deep(ws.down.k) * (h.abs() @ wd[e].t().abs())
    return y, bound


def ffn_weights(e, i, h, group, scale_dtype=F32):
    return Int4StackedExpertWeights(make(e, i, h, group, scale_dtype, 1)[0], make(e, i, h, group, scale_dtype, 2)[0],
                                    make(e, h, i, group, scale_dtype, 3)[0])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize(("sizes", "i", "h", "group"), [
    ([1, 0, 2], 24, 72, 32), ([6, 9, 0, 20], 136, 264, 64), ([1] * 6, 1408, 2048, 128), ([200, 0, 70], 104, 520, 128),
    ([3, 1], 40, 128, 256), ([40, 0, 100], 200, 264, 32), ([40, 0, 17, 100], 72, 520, 64), ([300, 133], 104, 264, 128),
])
def test_expert_ffn(sizes, i, h, group, dtype) -> None:
    ws = ffn_weights(len(sizes), i, h, group)
    off = torch.tensor([0, *torch.tensor(sizes).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    g = torch.Generator(device="cuda").manual_seed(7)
    xs = torch.randn(sum(sizes), h, generator=g, device=DEV).to(dtype)
    y, bound = ffn64(xs, off.tolist(), ws, dtype)
    check(expert_ffn_int4(xs, off, ws), y, bound)


def dense(ws, dtype=BF16):
    return StackedExpertWeights(*(dequantize_int4(q).to(dtype) for q in (ws.gate, ws.up, ws.down)))


@pytest.mark.parametrize("t", [1, 5, 37, 300])
@pytest.mark.parametrize("shared", [False, True])
def test_layer_matches_the_16_bit_layer_on_the_same_weights(t, shared) -> None:
    """The bar of the int8 layers: the 16-bit layer on the dequantised weights."""
    h, i, e, k = 256, 192, 16, 4
    w = LayerWeights(h, i, e, 320 if shared else 0)
    q = quantize_stacked_weights_int4(StackedExpertWeights(w.gate, w.up, w.down), group_size=64)
    sh = SharedExpertWeights(*w.shared) if shared else None
    g = torch.Generator(device="cuda").manual_seed(t)
    x = torch.randn(t, h, generator=g, device=DEV).to(BF16)
    cfg = RouterConfig(top_k=k, renormalize=True)
    got = moe_layer_forward(x, w.router, q, cfg, shared=sh)
    want = moe_layer_forward(x, w.router, dense(q), cfg, shared=sh)
    assert torch.equal(got.topk_idx, want.topk_idx) and torch.equal(got.group_offsets, want.group_offsets)
    assert_int8_parity(got.out, want.out)
    routed = grouped_moe_routed_quantized(x, got.topk_idx, got.topk_weight, q)
    assert_int8_parity(routed, grouped_moe_routed(x, got.topk_idx, got.topk_weight, dense(q)))
    f32 = moe_layer_forward(x.float(), None, q, cfg, topk=(got.topk_idx, got.topk_weight))
    assert f32.out.dtype == F32 and torch.equal(f32.out.to(BF16), routed)
    cap = CapturedLayer(x, w.router, q, cfg, shared=sh)
    assert torch.equal(cap(x), got.out)
    assert quantized_stacked_weights_nbytes(q) < 0.16 * 3 * e * h * i * 4


def test_two_graphs_of_one_stream_replayed_together() -> None:
    """Captured calls own their workspaces, those of the grouping included."""
    h, i, e, k = 256, 192, 16, 4
    w = LayerWeights(h, i, e)
    q = quantize_stacked_weights_int4(StackedExpertWeights(w.gate, w.up, w.down))
    cfg = RouterConfig(top_k=k)
    xs = [torch.randn(t, h, device=DEV).to(BF16) for t in (64, 700)]
    want = [moe_layer_forward(x, w.router, q, cfg).out for x in xs]
    graphs = []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        before = len(L._workspaces)
        with torch.cuda.graph(g):
            out = moe_layer_forward(x, w.router, q, cfg).out
        assert len(L._workspaces) == before
        graphs.append((g, out))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(10):
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for (_, out), v in zip(graphs, want):
        assert torch.equal(out, v)


def test_patched_model() -> None:
    torch.manual_seed(0)
    model = torch.nn.Sequential(DeepseekStyleMoE(256, 128, 16, 4)).to(DEV, BF16)
    ref = torch.nn.Sequential(DeepseekStyleMoE(256, 128, 16, 4)).to(DEV, BF16)
    ref.load_state_dict(model.state_dict())
    for ex in ref[0].experts:
        for name in ("gate_proj", "up_proj", "down_proj"):
            lin = getattr(ex, name)
            q = quantize_groupwise_int4(lin.weight.detach()[None], group_size=32)
            lin.weight = torch.nn.Parameter(dequantize_int4(q)[0].to(BF16), requires_grad=False)
    with pytest.raises(ValueError, match="bits"):
        patch_moe_infer_quantized(model, bits=3)
    assert patch_moe_infer_quantized(model, bits=4, group_size=32) == 1
    x = torch.randn(19, 256, device=DEV, dtype=BF16)
    with torch.no_grad():
        assert_int8_parity(model(x), ref(x))


@pytest.mark.parametrize("stream_dtype", [BF16, F32])
@pytest.mark.parametrize("t", [1, 50])
def test_block_is_its_parts(t, stream_dtype) -> None:
    h, i, e, k = 256, 192, 16, 4
    w = LayerWeights(h, i, e, 320)
    q = quantize_stacked_weights_int4(StackedExpertWeights(w.gate, w.up, w.down))
    sh, cfg = SharedExpertWeights(*w.shared), RouterConfig(top_k=k)
    x = torch.randn(t, h, device=DEV).to(stream_dtype)
    pre, post, nxt = (1 + 0.1 * torch.randn(h, device=DEV) for _ in range(3))
    gate = torch.rand(t, 1, device=DEV)
    b = moe_block_forward(x, pre, w.router, q, cfg, shared=sh, post_weight=post, next_weight=nxt, gate=gate,
                          residual_scale=0.5)
    n = rms_norm(x, pre, out_dtype=BF16)
    layer = moe_layer_forward(n, w.router, q, cfg, shared=sh)
    out, normed = norm_gate_residual(layer.out, x, post, nxt, gate=gate, residual_scale=0.5, norm_dtype=BF16)
    assert torch.equal(b.out, out) and torch.equal(b.normed, normed) and b.out.dtype == stream_dtype
    # the next block starts from normed
    c = moe_block_forward(b.out, None, w.router, q, cfg, shared=sh, normed=b.normed)
    layer = moe_layer_forward(b.normed, w.router, q, cfg, shared=sh)
    assert c.normed is None and torch.equal(c.out, norm_gate_residual(layer.out, b.out)[0])
    with pytest.raises(ValueError, match="normed"):
        moe_block_forward(x, pre, w.router, q, cfg, normed=n)
    with pytest.raises(ValueError, match="inference"):
        moe_block_forward(x.float().requires_grad_(), pre, w.router, q, cfg)


def test_refusals() -> None:
    q, _ = make(2, 40, 128, 64)
    sched = build_tile_schedule(torch.tensor([3, 4]), 16)
    x = torch.zeros(7, 128, device=DEV, dtype=BF16)
    with pytest.raises(ValueError, match="dtype mismatch"):
        grouped_matmul_int4(x.float(), q, sched)
    with pytest.raises(ValueError, match="K mismatch"):
        grouped_matmul_int4(x[:, :120], q, sched)
    with pytest.raises(ValueError, match="schedule covers 7"):
        grouped_matmul_int4(x[:6], q, sched)
    with pytest.raises(ValueError, match="number of experts"):
        grouped_matmul_int4(x, q, build_tile_schedule(torch.tensor([7]), 16))
    with pytest.raises(ValueError, match="inference"):
        grouped_matmul_int4(x.requires_grad_(), q, sched)
    x = x.detach()
    bad, _ = make(2, 40, 60, 64)  # K not a multiple of 8
    with pytest.raises(ValueError, match="K mismatch"):
        grouped_matmul_int4(torch.zeros(7, 60, device=DEV, dtype=BF16), bad, sched)
    off = torch.tensor([0, 3, 7], dtype=torch.int32, device=DEV)
    ws = ffn_weights(2, 40, 128, 64)
    with pytest.raises(ValueError, match="offsets"):
        expert_ffn_int4(x, off.long(), ws)
    with pytest.raises(ValueError, match="K mismatch"):
        expert_ffn_int4(x, off, Int4StackedExpertWeights(ws.gate, ws.up, ws.up))
    other, _ = make(2, 40, 128, 128)
    with pytest.raises(ValueError, match="share"):
        expert_ffn_int4(x, off, Int4StackedExpertWeights(ws.gate, other, ws.down))
