"""The block's norms (kernels/block.py) against their formulas in 64 bits.

Tolerances: an output is rounded once to its type (half a step, eps / 2 of
the value, or half the smallest f16 step), after f32 arithmetic whose error is
at most u = 2^-24 per operation of the magnitudes that enter: K operations deep
for a row (8 to 16 values per thread, 5 shuffle steps, 32 warps, rsqrt and the
products: K = 64), and one more per row for a sum over rows."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU hosts too
    pytest.skip("needs a CUDA device", allow_module_level=True)

from dispatch_b200.kernels.block import (  # noqa: E402
    norm_gate_residual,
    norm_gate_residual_backward,
    rms_norm,
    rms_norm_backward,
)

DEV = torch.device("cuda", 0)
U, K = 2.0**-24, 64
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def reference(y, res, post, nxt, gate, a, eps, d_out=None, d_normed=None):
    """{name: (value, magnitude of what is added up in f32)} in 64 bits."""
    h = res.shape[-1]
    one = torch.ones(1, dtype=torch.float64, device=DEV)
    f = lambda t: None if t is None else t.detach().double()  # noqa: E731
    y, res, post, nxt, gate, d_out, d_normed = map(f, (y, res, post, nxt, gate, d_out, d_normed))
    got = {}
    g = one if gate is None else gate
    if y is not None:
        r1 = one if post is None else (y.square().mean(-1, keepdim=True) + eps).rsqrt()
        w1 = one if post is None else post
        z = y * r1 * w1
        out, out_mag = res + a * g * z, res.abs() + abs(a) * (g * z).abs()
        got["out"] = out, out_mag
    else:
        out, out_mag = res, res.abs()
    r2 = (out.square().mean(-1, keepdim=True) + eps).rsqrt()
    # how much a relative error of out_mag weighs in r2
    rho = 1 + out_mag.square().sum(-1, keepdim=True) / (out.square().sum(-1, keepdim=True) + h * eps)
    if nxt is not None:
        got["normed"] = out * r2 * nxt, rho * out_mag * r2 * nxt.abs()
    if d_out is None and d_normed is None:
        return got
    df = torch.zeros_like(res) if d_out is None else d_out
    df_mag = df.abs()
    if d_normed is not None:
        c = (d_normed * nxt * out).mean(-1, keepdim=True)
        c_mag = (d_normed.abs() * nxt.abs() * out_mag).mean(-1, keepdim=True)
        df = df + r2 * (d_normed * nxt - out * r2.square() * c)
        df_mag = df_mag + rho * r2 * ((d_normed * nxt).abs() + out_mag * r2.square() * c_mag)
        got["dnext"] = (d_normed * out * r2).flatten(0, -2).sum(0), (rho * d_normed.abs() * out_mag * r2).flatten(0, -2).sum(0)
    elif nxt is not None:
        got["dnext"] = torch.zeros_like(nxt), torch.zeros_like(nxt)
    got["dresidual"] = df, df_mag
    if y is None:
        return got
    dz, dz_mag = a * g * df, abs(a) * g.abs() * df_mag
    if post is not None:
        got["dpost"] = (dz * y * r1).flatten(0, -2).sum(0), (dz_mag * (y * r1).abs()).flatten(0, -2).sum(0)
        c = (dz * w1 * y).mean(-1, keepdim=True)
        c_mag = (dz_mag * (w1 * y).abs()).mean(-1, keepdim=True)
        got["dy"] = (r1 * (dz * w1 - y * r1.square() * c),
                     r1 * (dz_mag * w1.abs() + y.abs() * r1.square() * c_mag))
    else:
        got["dy"] = dz, dz_mag
    if gate is not None:
        dg, dg_mag = a * z * df, abs(a) * z.abs() * df_mag
        if gate.shape == res.shape:
            pass
        elif gate.shape[-1] == 1 and gate.dim() == res.dim():
            dg, dg_mag = dg.sum(-1, keepdim=True), dg_mag.sum(-1, keepdim=True)
        else:
            dg, dg_mag = dg.flatten(0, -2).sum(0), dg_mag.flatten(0, -2).sum(0)
        got["dgate"] = dg, dg_mag
    return got


def check(name, actual, expected, rows=0):
    value, mag = expected
    assert actual.shape == value.shape, name
    half_step = torch.finfo(actual.dtype).eps / 2
    smallest = 2.0**-25 if actual.dtype == F16 else 0.0
    bound = half_step * value.abs() + (1 + half_step) * U * (K + rows) * mag + smallest
    off = (actual.double() - value).abs()
    worst = ((off - bound) / bound.clamp(min=1e-300)).max().item() if value.numel() else -1.0
    assert worst <= 0, f"{name}: {worst:.3g} over its bound"


def make(t, h, dtypes, gate, seed=0, shape=None):
    """Inputs in the types (y, residual, weights, gate)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    lead = shape or (t,)

    def rnd(*s, d=F32, k=1.0):
        return (torch.randn(*s, generator=g, device=DEV) * k).to(d)

    yd, rd, wd, gd = dtypes
    gs = dict(none=None, channel=(h,), token=(*lead, 1), full=(*lead, h))[gate]
    return dict(y=rnd(*lead, h, d=yd, k=0.5), residual=rnd(*lead, h, d=rd, k=2.0),
                post_weight=(1 + 0.2 * rnd(h)).to(wd), next_weight=(1 + 0.2 * rnd(h)).to(wd),
                gate=None if gs is None else rnd(*gs, d=gd), d_out=rnd(*lead, h, d=rd), d_normed=rnd(*lead, h, d=rd))


def run_all(i, a=0.7, eps=1e-6, post=True, nxt=True, rows=None):
    """Forward and backward of the inputs against the reference."""
    pw, nw = i["post_weight"] if post else None, i["next_weight"] if nxt else None
    dn = i["d_normed"] if nxt else None
    args, kw = (i["y"], i["residual"], pw, nw), dict(gate=i["gate"], residual_scale=a, eps=eps)
    a32 = torch.tensor(a, dtype=F32).item()  # the scale and eps reach the kernel in f32
    e32 = torch.tensor(eps, dtype=F32).item()
    want = reference(*args, i["gate"], a32, e32, i["d_out"], dn)
    out, normed = norm_gate_residual(*args, **kw)
    check("out", out, want["out"])
    assert (normed is None) == (not nxt)
    if nxt:
        check("normed", normed, want["normed"])
    rows = i["y"][..., 0].numel() if rows is None else rows
    grads = norm_gate_residual_backward(i["d_out"], dn, *args, **kw)
    for name, got in zip(("dy", "dresidual", "dpost", "dnext", "dgate"), grads):
        assert (got is None) == (name not in want), name
        if got is not None:
            check(name, got, want[name], rows if name in ("dpost", "dnext", "dgate") else 0)


# ------------------------------------------------------------------ sizes, gates, types
@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize(("t", "h"), [(1, 1), (1, 2048), (3, 7), (17, 256), (9, 264), (33, 1000), (5, 1001), (4, 4096),
                                      (3, 7168), (2, 8192), (700, 512)])
def test_matches_the_formula(t, h, gate) -> None:
    run_all(make(t, h, (BF16, BF16, BF16, BF16), gate, seed=t + h))


@pytest.mark.parametrize("dtypes", [(F16, F16, F16, F16), (F32, F32, F32, F32), (BF16, F32, F32, F32),
                                    (F32, BF16, F16, BF16), (F16, F32, BF16, F16)])
@pytest.mark.parametrize(("t", "h", "gate"), [(21, 520, "channel"), (6, 131, "full"), (40, 2048, "token")])
def test_types(t, h, gate, dtypes) -> None:
    run_all(make(t, h, dtypes, gate, seed=5))


def test_the_widest_row() -> None:
    run_all(make(3, 16384, (BF16, BF16, F32, BF16), "channel"))
    run_all(make(2, 16383, (F32, F32, F32, F32), "full"))


def test_more_rows_than_one_wave_of_ctas() -> None:
    run_all(make(5000, 64, (BF16, BF16, F32, BF16), "channel"))
    run_all(make(2500, 2048, (BF16, BF16, F32, BF16), "token"))


@pytest.mark.parametrize(("post", "nxt"), [(False, True), (True, False), (False, False)])
@pytest.mark.parametrize("gate", ["none", "channel", "token"])
def test_without_one_of_the_norms(post, nxt, gate) -> None:
    run_all(make(19, 776, (BF16, BF16, F32, F32), gate), post=post, nxt=nxt)


def test_leading_dimensions_and_strides() -> None:
    i = make(0, 264, (BF16, BF16, F32, F32), "full", shape=(3, 5))
    run_all(i)
    wide = make(11, 512, (BF16, F32, F32, F32), "full")
    for off, h in ((0, 256), (8, 256), (1, 255)):  # a slice of wider rows; the last one unaligned
        cut = {n: v[..., off:off + h] for n, v in wide.items()}
        assert cut["y"].stride(0) == 512
        run_all(cut)
    i = make(24, 40, (F16, F16, F16, F16), "token")
    for n in ("y", "residual", "d_out", "d_normed"):
        i[n] = i[n].t().contiguous().t()  # last stride not 1
    i["gate"] = i["gate"][:1].expand(24, 1)
    run_all(i)


def test_the_row_gradients_do_not_depend_on_the_batch() -> None:
    i = make(97, 1024, (BF16, BF16, F32, BF16), "full")
    one = {n: v[41:42] if v.dim() == 2 else v for n, v in i.items()}
    names = ("y", "residual", "post_weight", "next_weight")
    whole = norm_gate_residual(*(i[n] for n in names), gate=i["gate"])
    part = norm_gate_residual(*(one[n] for n in names), gate=one["gate"])
    assert torch.equal(whole[0][41:42], part[0]) and torch.equal(whole[1][41:42], part[1])
    whole = norm_gate_residual_backward(i["d_out"], i["d_normed"], *(i[n] for n in names), gate=i["gate"])
    again = norm_gate_residual_backward(i["d_out"], i["d_normed"], *(i[n] for n in names), gate=i["gate"])
    assert all(torch.equal(a, b) for a, b in zip(whole, again))
    part = norm_gate_residual_backward(one["d_out"], one["d_normed"], *(one[n] for n in names), gate=one["gate"])
    assert torch.equal(whole[0][41:42], part[0]) and torch.equal(whole[1][41:42], part[1])


# ------------------------------------------------------------------ values
def test_zero_rows_and_non_finite_rows_stay_apart() -> None:
    i = make(6, 512, (F32, F32, F32, F32), "token", seed=9)
    i["y"][1] = 0
    i["residual"][1] = 0  # both norms of a zero row: eps decides
    run_all(i)
    i["y"][3, 7] = float("inf")
    i["residual"][4, 9] = float("nan")
    args = [i[n] for n in ("y", "residual", "post_weight", "next_weight")]
    out, normed = norm_gate_residual(*args, gate=i["gate"])
    keep = [0, 1, 2, 5]
    want = reference(*[a[keep] if a.dim() == 2 else a for a in args], i["gate"][keep], 1.0,
                     torch.tensor(1e-6, dtype=F32).item())
    check("out", out[keep], want["out"])
    check("normed", normed[keep], want["normed"])
    assert not torch.isfinite(normed[3]).all() and torch.isnan(normed[4]).all()
    dy, dres, *_ = norm_gate_residual_backward(i["d_out"], i["d_normed"], *args, gate=i["gate"])
    assert torch.isfinite(dy[keep]).all() and torch.isfinite(dres[keep]).all()


@pytest.mark.parametrize("shape", [(0, 64), (2, 0, 64)])
def test_no_rows(shape) -> None:
    y = torch.empty(*shape, device=DEV, dtype=BF16)
    w = torch.ones(64, device=DEV)
    g = torch.ones(64, device=DEV)
    out, normed = norm_gate_residual(y, y, w, w, gate=g)
    assert out.shape == normed.shape == shape
    dy, dres, dpost, dnext, dgate = norm_gate_residual_backward(y, y, y, y, w, w, gate=g)
    assert dy.shape == dres.shape == shape
    assert not dpost.any() and not dnext.any() and not dgate.any()
    assert rms_norm(y, w).shape == shape


# ------------------------------------------------------------------ the norm alone, autograd
@pytest.mark.parametrize(("t", "h", "xd", "wd"), [(1, 2048, BF16, BF16), (300, 7168, F32, F32), (65, 999, F16, F32)])
def test_rms_norm(t, h, xd, wd) -> None:
    i = make(t, h, (xd, xd, wd, xd), "none")
    x, w, eps = i["residual"], i["next_weight"], 1e-5
    e32 = torch.tensor(eps, dtype=F32).item()
    want = reference(None, x, None, w, None, 1.0, e32, None, i["d_normed"])
    check("normed", rms_norm(x, w, eps=eps), want["normed"])
    dx, dw = rms_norm_backward(i["d_normed"], x, w, eps=eps)
    check("dx", dx, want["dresidual"])
    check("dw", dw, want["dnext"], t)
    assert rms_norm(x, w, out_dtype=F16).dtype == F16


def test_autograd_is_the_explicit_backward() -> None:
    i = make(12, 640, (BF16, F32, F32, F32), "channel", shape=(3, 4))
    names = ("y", "residual", "post_weight", "next_weight", "gate")
    leaves = [i[n].clone().requires_grad_() for n in names]
    out, normed = norm_gate_residual(*leaves[:4], gate=leaves[4], residual_scale=0.3)
    got = torch.autograd.grad((out, normed), leaves, (i["d_out"], i["d_normed"]))
    want = norm_gate_residual_backward(i["d_out"], i["d_normed"], *(i[n] for n in names[:4]), gate=i["gate"],
                                       residual_scale=0.3)
    for n, a, b in zip(names, got, want):
        assert torch.equal(a, b), n
    # one of the outputs only, and one of the inputs only
    only_y = i["y"].clone().requires_grad_()
    out, _ = norm_gate_residual(only_y, *(i[n] for n in names[1:4]), gate=i["gate"], residual_scale=0.3)
    (dy,) = torch.autograd.grad(out, only_y, i["d_out"])
    assert torch.equal(dy, norm_gate_residual_backward(i["d_out"], None, *(i[n] for n in names[:4]), gate=i["gate"],
                                                       residual_scale=0.3)[0])
    x, w = i["residual"].clone().requires_grad_(), i["next_weight"].clone().requires_grad_()
    got = torch.autograd.grad(rms_norm(x, w), (x, w), i["d_normed"])
    assert all(torch.equal(a, b) for a, b in zip(got, rms_norm_backward(i["d_normed"], i["residual"], i["next_weight"])))


def test_gradient_against_differences() -> None:
    """Along a random direction v, (f(x + s v) - f(x - s v)) / 2s in the
    kernel's own f32: off by s^2 / 6 of the third derivative and by u |f| / s."""
    i = make(4, 96, (F32, F32, F32, F32), "channel", seed=3)
    names = ("y", "residual", "post_weight", "next_weight", "gate")
    step = 2.0**-7
    grads = norm_gate_residual_backward(i["d_out"], i["d_normed"], *(i[n] for n in names[:4]), gate=i["gate"])

    def loss(**other):
        v = {**i, **other}
        out, normed = norm_gate_residual(*(v[n] for n in names[:4]), gate=v["gate"])
        return (out.double() * i["d_out"].double() + normed.double() * i["d_normed"].double()).sum().item()

    for n, g in zip(names, grads):
        v = torch.randn(i[n].shape, generator=torch.Generator(device="cuda").manual_seed(1), device=DEV)
        v = v / v.norm()
        diff = (loss(**{n: i[n] + step * v}) - loss(**{n: i[n] - step * v})) / (2 * step)
        # |f| is at most |d| |out|, each ~ sqrt(4 * 96) and a few: 1e3 u / step < 1e-2; third derivatives ~ 1e2
        assert abs(diff - (g.double() * v.double()).sum().item()) < 1e-2 + 1e2 * step**2 / 6, n


# ------------------------------------------------------------------ streams, graphs, refusals
def test_on_a_side_stream_and_in_a_graph() -> None:
    i = make(65, 2048, (BF16, BF16, F32, F32), "channel")
    names = ("y", "residual", "post_weight", "next_weight")

    def both():
        fwd = norm_gate_residual(*(i[n] for n in names), gate=i["gate"])
        return (*fwd, *norm_gate_residual_backward(i["d_out"], i["d_normed"], *(i[n] for n in names), gate=i["gate"]))

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graphs = []
    for _ in range(2):  # two graphs, replayed at the same time, share nothing
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = both()
        graphs.append((g, res))
    i["y"].mul_(1.5)
    want = both()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for _, res in graphs:
        assert all(torch.equal(a, b) for a, b in zip(want, res))


def test_autograd_is_refused_during_capture() -> None:
    x = torch.randn(4, 64, device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV)
    rms_norm(x, w)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="capture"):
            rms_norm(x, w)
        with torch.no_grad():
            out = rms_norm(x, w)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, rms_norm(x.detach(), w))


def test_refusals() -> None:
    y, w = torch.ones(4, 64, device=DEV), torch.ones(64, device=DEV)
    with pytest.raises(ValueError, match="CUDA"):
        rms_norm(y.cpu(), w.cpu())
    with pytest.raises(ValueError, match="one CUDA device|CUDA tensors"):
        rms_norm(y, w.cpu())
    with pytest.raises(ValueError, match="residual.shape"):
        norm_gate_residual(y, y[:2])
    with pytest.raises(ValueError, match="post_weight.shape"):
        norm_gate_residual(y, y, w[:32])
    with pytest.raises(ValueError, match="next_weight.shape"):
        norm_gate_residual(y, y, w, y)
    with pytest.raises(ValueError, match="gate.shape"):
        norm_gate_residual(y, y, gate=torch.ones(4, device=DEV))
    with pytest.raises(ValueError, match="unsupported dtype"):
        rms_norm(y.double(), w)
    with pytest.raises(ValueError, match="dtypes"):
        rms_norm(y.int(), w)
    with pytest.raises(ValueError, match="needs y"):
        norm_gate_residual(None, y, next_weight=w)
    with pytest.raises(ValueError, match="d_normed"):
        norm_gate_residual_backward(y, y, y, y, w)
    wide = torch.ones(1, 16385, device=DEV)
    with pytest.raises(ValueError, match="16384"):
        rms_norm(wide, wide[0])
