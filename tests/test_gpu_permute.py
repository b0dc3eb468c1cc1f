"""The differentiable sort and combine (kernels/grouping.py) against their
formulas in 64 bits. Tolerances: one rounding to the output's type (half a
step), after f32 sums that are off by at most u = 2^-24 per term deep of the
magnitudes added up (dw's sum over H: 32 values per thread, 5 shuffle steps, 8
warps; 64 covers it and the sums over k <= 32 slots)."""

from __future__ import annotations

import dataclasses

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU hosts too
    pytest.skip("needs a CUDA device", allow_module_level=True)

from dispatch_b200 import _lib as L  # noqa: E402
from dispatch_b200.kernels.grouping import (  # noqa: E402
    combine_tokens,
    combine_tokens_backward,
    group_tokens_by_expert,
    permute_tokens,
    permute_tokens_backward,
    ungroup_and_combine,
)

DEV = torch.device("cuda", 0)
U, DEEP = 2.0**-24, 64
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _device_status_clean():
    yield
    L.check_device_status(DEV)


def make(t, k, e, h, dtype, wdtype=F32, seed=0, distinct=True):
    g = torch.Generator().manual_seed(seed)
    if distinct:
        idx = torch.multinomial(torch.ones(t, e), k, generator=g) if t else torch.empty(0, k, dtype=torch.long)
    else:
        idx = torch.randint(0, e, (t, k), generator=g)  # a token may name one expert twice
    d = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=d, device=DEV)  # noqa: E731
    i = dict(x=rnd(t, h).to(dtype), y=rnd(t * k, h).to(dtype), w=rnd(t, k).to(wdtype), dout=rnd(t, h).to(dtype),
             dxs=rnd(t * k, h).to(dtype), y_shared=rnd(t, h).to(dtype))
    return i, group_tokens_by_expert(idx.to(DEV), i["w"], e), idx.to(DEV)


def check(name, actual, value, mag, dtype):
    assert actual.dtype == dtype and actual.shape == value.shape, name
    half = torch.finfo(dtype).eps / 2
    bound = half * value.abs() + (1 + half) * U * DEEP * mag + (2.0**-25 if dtype == F16 else 0.0)
    off = (actual.double() - value).abs()
    assert bool((off <= bound).all()), f"{name}: off by {off.max().item():.3g}"


def run_all(i, grouping, idx):
    t, k = idx.shape
    h = i["x"].shape[1]
    order = torch.sort(idx.flatten(), stable=True).indices
    pos = torch.empty_like(order)
    pos[order] = torch.arange(t * k, device=DEV)
    assert torch.equal(grouping.pos.long(), pos)
    xs = permute_tokens(i["x"], grouping)
    assert torch.equal(xs, i["x"][order // k])
    dxs = i["dxs"].double()[pos].view(t, k, h)
    check("dx", permute_tokens_backward(i["dxs"], grouping), dxs.sum(1), dxs.abs().sum(1), i["dxs"].dtype)
    y, w, dout = i["y"].double()[pos].view(t, k, h), i["w"].double(), i["dout"].double()
    terms = y * w[..., None]
    check("out", combine_tokens(i["y"], grouping, i["w"]), terms.sum(1), terms.abs().sum(1), i["y"].dtype)
    got = combine_tokens(i["y"], grouping, i["w"], y_shared=i["y_shared"], out_dtype=F32)
    sh = i["y_shared"].double()
    check("out with the shared row", got, terms.sum(1) + sh, terms.abs().sum(1) + sh.abs(), F32)
    dy, dw = combine_tokens_backward(i["dout"], i["y"], grouping, i["w"])
    want = dout[order // k] * w.flatten()[order][:, None]
    check("dy", dy, want, want.abs(), i["y"].dtype)
    terms = y * dout[:, None]
    check("dw", dw, terms.sum(2), terms.abs().sum(2), i["w"].dtype)
    assert combine_tokens_backward(i["dout"], i["y"], grouping, i["w"], need_weight=False)[1] is None
    only_dy, _ = combine_tokens_backward(i["dout"], i["y"], grouping, i["w"], need_weight=False)
    none, only_dw = combine_tokens_backward(i["dout"], i["y"], grouping, i["w"], need_y=False)
    assert none is None and torch.equal(only_dy, dy) and torch.equal(only_dw, dw)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize(("t", "k", "e", "h"), [(1, 1, 1, 8), (1, 6, 64, 2048), (7, 3, 5, 24), (64, 8, 256, 7168),
                                                (333, 6, 64, 264), (50, 32, 64, 64), (19, 9, 12, 2056),
                                                (4096, 2, 8, 512)])
def test_matches_the_formula(t, k, e, h, dtype) -> None:
    run_all(*make(t, k, e, h, dtype, seed=t))


@pytest.mark.parametrize("wdtype", [BF16, F16, F32])
def test_weight_types(wdtype) -> None:
    run_all(*make(40, 4, 16, 128, BF16, wdtype))


def test_the_same_expert_twice_for_one_token() -> None:
    run_all(*make(60, 5, 3, 80, BF16, distinct=False))


def test_no_tokens() -> None:
    i, grouping, _ = make(0, 4, 8, 64, BF16)
    assert permute_tokens(i["x"], grouping).shape == (0, 64)
    assert permute_tokens_backward(i["dxs"], grouping).shape == (0, 64)
    assert combine_tokens(i["y"], grouping, i["w"]).shape == (0, 64)
    dy, dw = combine_tokens_backward(i["dout"], i["y"], grouping, i["w"])
    assert dy.shape == (0, 64) and dw.shape == (0, 4)


def test_the_groupings_own_weights_and_the_references_combine() -> None:
    i, grouping, _ = make(77, 6, 64, 256, BF16)
    out = combine_tokens(i["y"], grouping)
    assert torch.equal(out, ungroup_and_combine(i["y"], grouping, 77))
    dy, dw = combine_tokens_backward(i["dout"], i["y"], grouping)
    dy2, dw2 = combine_tokens_backward(i["dout"], i["y"], grouping, i["w"])
    assert torch.equal(dy, dy2) and torch.equal(dw, dw2) and dw.dtype == F32


def test_strided_rows() -> None:
    i, grouping, idx = make(30, 3, 8, 512, BF16)
    i = {n: v[:, 128:256] if n != "w" else v for n, v in i.items()}
    run_all(i, grouping, idx)
    i = {n: v[:, 3:123] if n != "w" else v for n, v in i.items()}  # unaligned rows: copied
    run_all(i, grouping, idx)
    i = {n: v[:, :64].t().contiguous().t() if n != "w" else v for n, v in i.items()}
    run_all(i, grouping, idx)


def test_slots_without_a_row() -> None:
    """A dropped slot (pos -1) adds nothing and gets a zero gradient; the rows
    behind the last expert's are zeros, whatever memory they are made in."""
    t, k, e, h = 37, 4, 8, 136
    i, full, idx = make(t, k, e, h, F32)
    keep = torch.rand(t * k, generator=torch.Generator().manual_seed(3)).to(DEV) < 0.6
    keep[: k] = False  # a token without any row
    order = [f for f in torch.sort(idx.flatten(), stable=True).indices.tolist() if keep[f]]
    pos = torch.full((t * k,), -1, dtype=torch.int32, device=DEV)
    pos[order] = torch.arange(len(order), dtype=torch.int32, device=DEV)
    sizes = torch.bincount(idx.flatten()[order], minlength=e)
    offsets = torch.cat([torch.zeros(1, device=DEV), sizes.cumsum(0)]).int()
    grouping = dataclasses.replace(full, pos=pos, offsets=offsets)
    n = len(order)
    for _ in range(2):
        torch.full((t * k, h), float("nan"), device=DEV)  # freed: what the next allocation is likely to hold
        xs = permute_tokens(i["x"], grouping)
        assert torch.equal(xs[:n], i["x"][torch.tensor(order, device=DEV) // k]) and not xs[n:].any()
        torch.full((t * k, h), float("nan"), device=DEV)
        dy, dw = combine_tokens_backward(i["dout"], i["y"], grouping, i["w"])
        assert not dy[n:].any() and not dw.flatten()[~keep].any()
    rows = torch.where(keep[:, None], i["y"].double()[pos.clamp(min=0).long()], 0.0).view(t, k, h)
    terms = rows * i["w"].double()[..., None]
    check("out", combine_tokens(i["y"], grouping, i["w"]), terms.sum(1), terms.abs().sum(1), F32)
    terms = rows * i["dout"].double()[:, None]
    check("dw", dw, terms.sum(2), terms.abs().sum(2), F32)
    # what lies in rows of no slot does not matter
    i["dxs"][n:] = float("nan")
    rows = torch.where(keep[:, None], i["dxs"].double()[pos.clamp(min=0).long()], 0.0).view(t, k, h)
    check("dx", permute_tokens_backward(i["dxs"], grouping), rows.sum(1), rows.abs().sum(1), F32)


def test_a_position_out_of_range_is_reported() -> None:
    i, grouping, _ = make(8, 2, 4, 64, BF16)
    pos = grouping.pos.clone()
    pos[3] = 16  # one past the last row
    bad = dataclasses.replace(grouping, pos=pos)
    for call in (lambda: permute_tokens(i["x"], bad), lambda: permute_tokens_backward(i["dxs"], bad),
                 lambda: combine_tokens_backward(i["dout"], i["y"], bad, i["w"])):
        call()
        with pytest.raises(L.MoeDeviceError, match="positions out of range"):
            L.check_device_status(DEV)


def test_autograd_is_the_explicit_backward() -> None:
    i, grouping, _ = make(45, 6, 16, 320, BF16, wdtype=BF16)
    x = i["x"].clone().requires_grad_()
    (dx,) = torch.autograd.grad(permute_tokens(x, grouping), x, i["dxs"])
    assert torch.equal(dx, permute_tokens_backward(i["dxs"], grouping))
    y, w, sh = (i[n].clone().requires_grad_() for n in ("y", "w", "y_shared"))
    out = combine_tokens(y, grouping, w, y_shared=sh, out_dtype=F32)
    dout = i["dout"].float()
    got = torch.autograd.grad(out, (y, w, sh), dout)
    dy, dw = combine_tokens_backward(dout, i["y"], grouping, i["w"])
    assert torch.equal(got[0], dy) and torch.equal(got[1], dw) and torch.equal(got[2], i["dout"])
    assert got[1].dtype == BF16
    out = combine_tokens(i["y"], grouping, w)  # the weights alone
    (dw2,) = torch.autograd.grad(out, w, i["dout"])
    assert torch.equal(dw2, combine_tokens_backward(i["dout"], i["y"], grouping, i["w"])[1])


def test_gradients_are_adjoints() -> None:
    """The operators are linear in x and in y, so <d, f(v)> = <f'(d), v> up to
    the roundings of f32 sums."""
    i, grouping, _ = make(90, 4, 16, 104, F32)
    n = i["x"].double().abs().sum().item() * 4
    lhs = (permute_tokens(i["x"], grouping).double() * i["dxs"].double()).sum()
    rhs = (i["x"].double() * permute_tokens_backward(i["dxs"], grouping).double()).sum()
    assert abs((lhs - rhs).item()) < 8 * U * n * 4
    out = combine_tokens(i["y"], grouping, i["w"])
    dy, dw = combine_tokens_backward(i["dout"], i["y"], grouping, i["w"])
    lhs = (out.double() * i["dout"].double()).sum()
    assert abs((lhs - (i["y"].double() * dy.double()).sum()).item()) < 8 * U * n * 8
    assert abs((lhs - (i["w"].double() * dw.double()).sum()).item()) < 8 * U * n * 8


def test_in_a_graph_and_refused_autograd_in_one() -> None:
    i, grouping, _ = make(33, 6, 64, 512, BF16)

    def both():
        return (permute_tokens(i["x"], grouping), permute_tokens_backward(i["dxs"], grouping),
                combine_tokens(i["y"], grouping, i["w"]),
                *combine_tokens_backward(i["dout"], i["y"], grouping, i["w"]))

    both()
    g = torch.cuda.CUDAGraph()
    x = i["x"].clone().requires_grad_()
    with torch.cuda.graph(g):
        res = both()
        with pytest.raises(RuntimeError, match="capture"):
            permute_tokens(x, grouping)
    for n in ("x", "y", "dxs", "dout"):
        i[n].mul_(0.5)
    want = both()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, res))


def test_sizes_first_read_inside_a_capture_or_on_another_stream() -> None:
    idx = torch.randint(0, 4, (40, 2), device=DEV)
    w = torch.rand(40, 2, device=DEV).to(BF16)
    want = torch.bincount(idx.flatten(), minlength=4)
    for where in ("graph", "stream"):
        grouping = group_tokens_by_expert(idx, w, 4)
        if where == "graph":
            with torch.cuda.graph(torch.cuda.CUDAGraph()):  # never replayed
                grouping.group_sizes, grouping.sorted_weight
        else:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                assert torch.equal(grouping.group_sizes, want)
        first = grouping.group_sizes
        assert torch.equal(first, want) and grouping.group_sizes is first
        assert grouping.sorted_weight.dtype == BF16
        assert torch.equal(grouping.sorted_weight.sort().values, w.flatten().sort().values)


def test_first_call_on_a_device_captured(monkeypatch) -> None:
    """Its status word belongs to the graph; an eager call before the first replay has its own."""
    i, grouping, _ = make(33, 6, 64, 512, BF16)
    want = permute_tokens(i["x"], grouping)
    monkeypatch.setattr(L, "_status", {})
    monkeypatch.setattr(L, "_captured_status", {})
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        xs = permute_tokens(i["x"], grouping)
    assert torch.equal(permute_tokens(i["x"], grouping), want)
    g.replay()
    L.check_device_status(DEV)
    assert torch.equal(xs, want) and L._status[0] is not L._captured_status[0]


def test_refusals() -> None:
    i, grouping, _ = make(6, 2, 4, 64, BF16)
    with pytest.raises(ValueError, match="CUDA"):
        permute_tokens(i["x"].cpu(), grouping)
    with pytest.raises(ValueError, match="grouping describes 6"):
        permute_tokens(i["x"][:5], grouping)
    with pytest.raises(ValueError, match="grouping describes 12"):
        combine_tokens(i["y"][:11], grouping, i["w"])
    with pytest.raises(ValueError, match="topk_weight"):
        combine_tokens(i["y"], grouping, i["w"][:3])
    with pytest.raises(ValueError, match="dtype mismatch"):
        combine_tokens(i["y"], grouping, i["w"], y_shared=i["y_shared"].float())
    with pytest.raises(ValueError, match="y_shared.shape"):
        combine_tokens(i["y"], grouping, i["w"], y_shared=i["y_shared"][:, :32])
    with pytest.raises(ValueError, match="dout.shape"):
        combine_tokens_backward(i["dout"][:, :32], i["y"], grouping, i["w"])
    with pytest.raises(ValueError, match="multiple of 8"):
        permute_tokens(i["x"][:, :60], grouping)
    with pytest.raises(ValueError, match="bf16, f16 or f32"):
        permute_tokens(i["x"].int(), grouping)
