"""The cases that the operators around the MoE layer are measured on.

Three operators, each computed in two ways: in elementary torch operations
(``own`` false) and by this package's public calls (``own`` true).

``int4``  the experts' products with 4-bit weights and group scales:
          out[rows of e] = x[rows of e] @ (code[e] * scale[e])^T.
``sort``  tokens sorted by expert and back: the row gather, the weighted
          combine and, with ``train``, the gradients of both.
``norm``  the end of a block: out = residual + residual_scale * gate *
          rmsnorm(y) * post_weight, and the next block's input
          rmsnorm(out) * next_weight, with ``train`` the gradients of all inputs.
"""

from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6

# The largest drawn sizes: what the largest listed case of each operator costs.
MAX_WEIGHTS = 64 * 1408 * 2048
MAX_INT4_ROWS = 2048 * 6
MAX_SORT = 4096 * 6 * 2048
MAX_NORM = 8192 * 2048


def listed():
    return [
        # one decoded token's gate projection: 6 of 64 experts, one row each
        dict(name="int4 decode 1 token", op="int4", tokens=1, k=6, e=64, n=1408, kdim=2048, group=128,
             dtype="bf16", scale="bf16", skew=0.0),
        # a decode batch's down projection, f16 activations, small groups
        dict(name="int4 decode 16 tokens", op="int4", tokens=16, k=6, e=64, n=2048, kdim=1408, group=64,
             dtype="f16", scale="f32", skew=0.0),
        # a ragged batch between decode and prefill, one expert much busier than the rest
        dict(name="int4 mixed 93 tokens", op="int4", tokens=93, k=6, e=64, n=1408, kdim=2048, group=32,
             dtype="bf16", scale="f32", skew=1.2),
        # a prompt's down projection
        dict(name="int4 prompt 2048 tokens", op="int4", tokens=2048, k=6, e=64, n=2048, kdim=1408, group=128,
             dtype="bf16", scale="bf16", skew=0.0),
        # a decode batch: sort, gather and combine, no gradient
        dict(name="sort decode 4 tokens", op="sort", tokens=4, k=6, e=64, h=2048, dtype="bf16", weight="f32",
             train=False, skew=0.0),
        # a ragged training micro-batch of a small model in f32
        dict(name="sort train 1021 tokens", op="sort", tokens=1021, k=2, e=8, h=520, dtype="f32", weight="f32",
             train=True, skew=0.0),
        # a training micro-batch with skewed routing and weights in the activation type
        dict(name="sort train 4096 tokens", op="sort", tokens=4096, k=6, e=64, h=2048, dtype="bf16", weight="bf16",
             train=True, skew=1.2),
        # one decoded token between two blocks
        dict(name="norm decode 1 token", op="norm", tokens=1, h=2048, dtype="bf16", weight="bf16", gate="none",
             train=False),
        # a prompt on an f32 residual stream, a gate per token
        dict(name="norm prompt 1000 tokens", op="norm", tokens=1000, h=7168, dtype="f32", weight="f32",
             gate="token", train=False),
        # a training step at an odd width, a gate per value
        dict(name="norm train 517 tokens", op="norm", tokens=517, h=1001, dtype="f16", weight="f16", gate="full",
             train=True),
        # a training micro-batch, a learned scale per channel, f32 norm weights
        dict(name="norm train 8192 tokens", op="norm", tokens=8192, h=2048, dtype="bf16", weight="f32",
             gate="channel", train=True),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["int4", "sort", "norm"])
    if op == "int4":
        e = rng.choice([8, 16, 32, 64, 64, 128])
        k = rng.randint(1, min(8, e))
        tokens = _log_int(rng, 1, MAX_INT4_ROWS // k)
        n = _log_int(rng, 17, 4096)
        kdim = 8 * _log_int(rng, 8, min(7168, MAX_WEIGHTS // (e * n)) // 8)
        while tokens * k * n * kdim > MAX_INT4_ROWS * 2048 * 1408:
            tokens = (tokens + 1) // 2
        # skewed routing leaves most experts idle: for batches of decode size
        return dict(op=op, tokens=tokens, k=k, e=e, n=n, kdim=kdim, group=rng.choice([32, 64, 128]),
                    dtype=rng.choice(["bf16", "f16"]), scale=rng.choice(["f32", "bf16"]),
                    skew=rng.choice([0.0, 1.2]) if tokens <= 128 else 0.0)
    if op == "sort":
        e = rng.choice([2, 8, 33, 64, 256])
        k = rng.randint(1, min(8, e))
        h = 8 * _log_int(rng, 8, 896)
        tokens = _log_int(rng, 1, min(4096, MAX_SORT // (k * h)))
        dtype = rng.choice(["bf16", "f16", "f32"])
        if dtype == "f32":
            tokens = (tokens + 1) // 2
        return dict(op=op, tokens=tokens, k=k, e=e, h=h, dtype=dtype, weight=rng.choice(["f32", dtype]),
                    train=rng.random() < 0.7, skew=rng.choice([0.0, 1.2]))
    h = _log_int(rng, 32, 7168)
    if rng.random() < 0.7:
        h = (h + 7) // 8 * 8
    tokens = _log_int(rng, 1, min(8192, MAX_NORM // h))
    dtype = rng.choice(["bf16", "f16", "f32"])
    if dtype == "f32":
        tokens = (tokens + 1) // 2
    return dict(op=op, tokens=tokens, h=h, dtype=dtype, weight=rng.choice(["f32", dtype]),
                gate=rng.choice(["none", "channel", "token", "full"]), train=rng.random() < 0.6)


# ---------------------------------------------------------------- inputs
def _routing(case, seed):
    """tokens x k distinct experts, uniform or with 1 / rank^skew weights."""
    g = torch.Generator().manual_seed(seed)
    p = torch.arange(1, case["e"] + 1, dtype=torch.float32) ** -case["skew"]
    return torch.multinomial(p.expand(case["tokens"], -1), case["k"], replacement=False, generator=g)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _lay_out(codes):
    """Codes + 8 (E, N, K) uint8, two per byte in the order in which the
    product's warps read them: (E, N/16, K/64, 32 lanes, 4) int32."""
    e, n, k = codes.shape
    codes = torch.nn.functional.pad(codes, (0, -k % 64, 0, -n % 16), value=8)
    # n = 16 i + 8 half + lane / 4, k = 64 b + 32 j + 8 (lane % 4) + 4 step + 2 pair + odd
    c = codes.view(e, (n + 15) // 16, 2, 8, (k + 63) // 64, 2, 4, 2, 2, 2)
    c = c.permute(0, 1, 4, 3, 6, 5, 7, 9, 8, 2)
    data = c[..., 0] | (c[..., 1] << 4)
    return data.reshape(e, (n + 15) // 16, (k + 63) // 64, 32, 16).contiguous().view(torch.int32)


def _prepare_int4(case, seed, g):
    e, n, k, group = case["e"], case["n"], case["kdim"], case["group"]
    ids = _routing(case, seed).flatten()
    sizes = torch.bincount(ids, minlength=e)
    offsets = [0] + sizes.cumsum(0).tolist()
    codes = torch.empty(e, n, k, dtype=torch.uint8, device="cuda")
    for i in range(e):  # symmetric codes of normal weights, -7 .. 7, held with 8 added
        codes[i] = (_randn(g, n, k) * 2.4).round().clamp(-7, 7).add(8).to(torch.uint8)
    groups = (k + group - 1) // group
    scale = (0.3 + 0.2 * torch.rand(e, n, groups, generator=g, device="cuda")) / math.sqrt(k)
    scale = scale.to(DTYPES[case["scale"]])
    rows = sum(sizes.tolist())
    # the places of the rows in a padded (busy experts, most rows) layout
    busy = sizes.nonzero().flatten()
    row_e = torch.repeat_interleave(torch.arange(len(busy)), sizes[busy])
    row_i = torch.arange(rows) - torch.tensor(offsets)[busy][row_e]
    return dict(
        x=_randn(g, rows, k).to(DTYPES[case["dtype"]]),
        rows=codes[..., 0::2] | (codes[..., 1::2] << 4), row_scale=scale,
        data=_lay_out(codes),
        scale=torch.nn.functional.pad(scale, (0, 0, 0, -n % 16)).view(e, -1, 16, groups).transpose(2, 3).contiguous(),
        schedule=SimpleNamespace(block_m=16, group_offsets=tuple(offsets)),
        busy=busy.cuda(), row_e=row_e.cuda(), row_i=row_i.cuda(), most=int(sizes.max()))


def _prepare_sort(case, seed, g):
    dtype = DTYPES[case["dtype"]]
    t, k, h = case["tokens"], case["k"], case["h"]
    w = torch.rand(t, k, generator=g, device="cuda") + 0.1
    return dict(
        idx=_routing(case, seed).cuda(), w=(w / w.sum(1, keepdim=True)).to(DTYPES[case["weight"]]),
        x=_randn(g, t, h).to(dtype),
        y=_randn(g, t * k, h).to(dtype),  # the experts' rows, in grouped order
        dout=_randn(g, t, h).to(dtype), dxs=_randn(g, t * k, h).to(dtype))


def _prepare_norm(case, seed, g):
    dtype, wdtype = DTYPES[case["dtype"]], DTYPES[case["weight"]]
    t, h = case["tokens"], case["h"]
    shape = dict(none=None, channel=(h,), token=(t, 1), full=(t, h))[case["gate"]]
    # a residual stream has a few channels much larger than the rest
    channel = 1.0 + 8.0 * (torch.rand(h, generator=g, device="cuda") > 0.98)
    return dict(
        y=(_randn(g, t, h) * 0.4).to(dtype), residual=(_randn(g, t, h) * channel).to(dtype),
        post=(1 + 0.1 * _randn(g, h)).to(wdtype), next=(1 + 0.1 * _randn(g, h)).to(wdtype),
        gate=None if shape is None else torch.sigmoid(_randn(g, *shape)).to(dtype),
        dout=_randn(g, t, h).to(dtype), dnormed=_randn(g, t, h).to(dtype))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    made = dict(int4=_prepare_int4, sort=_prepare_sort, norm=_prepare_norm)[case["op"]](case, seed, g)
    return dict(case=case, **made)


# ---------------------------------------------------------------- plain forms
def _plain_int4(s):
    case = s["case"]
    n, k, group = case["n"], case["kdim"], case["group"]
    packed = s["rows"][s["busy"]]
    codes = torch.stack((packed & 15, packed >> 4), dim=-1).view(len(packed), n, k)
    scale = s["row_scale"][s["busy"]].float().repeat_interleave(group, dim=2)[..., :k]
    w = (codes.float() - 8.0) * scale
    xp = torch.zeros(len(packed), s["most"], k, dtype=torch.float32, device="cuda")
    xp[s["row_e"], s["row_i"]] = s["x"].float()
    y = torch.bmm(xp, w.transpose(1, 2))
    return y[s["row_e"], s["row_i"]].to(s["x"].dtype)


def _plain_sort(s):
    case = s["case"]
    t, k, h = case["tokens"], case["k"], case["h"]
    dtype = s["x"].dtype
    order = torch.sort(s["idx"].flatten(), stable=True).indices
    pos = torch.empty_like(order)
    pos[order] = torch.arange(t * k, device="cuda")
    xs = s["x"][order // k]
    y = s["y"][pos].float().view(t, k, h)
    w = s["w"].float()
    out = (y * w[..., None]).sum(1).to(dtype)
    if not case["train"]:
        return dict(xs=xs, out=out)
    dout = s["dout"].float()
    dy = (dout[order // k] * w.flatten()[order][:, None]).to(dtype)
    dw = (y * dout[:, None]).sum(2).to(s["w"].dtype)
    dx = s["dxs"][pos].float().view(t, k, h).sum(1).to(dtype)
    return dict(xs=xs, out=out, dy=dy, dw=dw, dx=dx)


def _plain_norm(s):
    case = s["case"]
    scale, h = _residual_scale(case), case["h"]
    y, res, post, nxt = (s[n].float() for n in ("y", "residual", "post", "next"))
    gate = torch.ones(1, device="cuda") if s["gate"] is None else s["gate"].float()
    yhat = y * torch.rsqrt((y * y).mean(1, keepdim=True) + EPS)
    z = yhat * post
    full = res + scale * gate * z
    r2 = torch.rsqrt((full * full).mean(1, keepdim=True) + EPS)
    fhat = full * r2
    dtype = s["y"].dtype
    got = dict(out=full.to(dtype), normed=(fhat * nxt).to(dtype))
    if not case["train"]:
        return got
    r1 = torch.rsqrt((y * y).mean(1, keepdim=True) + EPS)
    dn = s["dnormed"].float()
    dfhat = dn * nxt
    dfull = s["dout"].float() + r2 * (dfhat - fhat * (dfhat * fhat).mean(1, keepdim=True))
    dz = scale * gate * dfull
    dyhat = dz * post
    got.update(dnext=(dn * fhat).sum(0).to(s["next"].dtype), dresidual=dfull.to(dtype),
               dpost=(dz * yhat).sum(0).to(s["post"].dtype),
               dy=(r1 * (dyhat - yhat * (dyhat * yhat).mean(1, keepdim=True))).to(dtype))
    dgate = scale * z * dfull
    if case["gate"] == "channel":
        got["dgate"] = dgate.sum(0).to(dtype)
    elif case["gate"] == "token":
        got["dgate"] = dgate.sum(1, keepdim=True).to(dtype)
    elif case["gate"] == "full":
        got["dgate"] = dgate.to(dtype)
    return got


def _residual_scale(case):
    return 0.22 if case["gate"] == "none" else 1.0


# ---------------------------------------------------------------- the package's calls
def _own_int4(s):
    from dispatch_b200.kernels.grouped_gemm_int4 import grouped_matmul_int4
    from dispatch_b200.kernels.quantization import Int4Tensor

    case = s["case"]
    w = Int4Tensor(data=s["data"], scale=s["scale"], n=case["n"], k=case["kdim"], group_size=case["group"])
    return grouped_matmul_int4(s["x"], w, s["schedule"])


def _own_sort(s):
    from dispatch_b200.kernels import grouping as G

    grouping = G.group_tokens_by_expert(s["idx"], s["w"], s["case"]["e"])
    xs = G.permute_tokens(s["x"], grouping)
    out = G.combine_tokens(s["y"], grouping, s["w"])
    if not s["case"]["train"]:
        return dict(xs=xs, out=out)
    dy, dw = G.combine_tokens_backward(s["dout"], s["y"], grouping, s["w"])
    dx = G.permute_tokens_backward(s["dxs"], grouping)
    return dict(xs=xs, out=out, dy=dy, dw=dw, dx=dx)


def _own_norm(s):
    from dispatch_b200.kernels import block as B

    args = (s["y"], s["residual"], s["post"], s["next"])
    kw = dict(gate=s["gate"], residual_scale=_residual_scale(s["case"]), eps=EPS)
    out, normed = B.norm_gate_residual(*args, **kw)
    if not s["case"]["train"]:
        return dict(out=out, normed=normed)
    dy, dresidual, dpost, dnext, dgate = B.norm_gate_residual_backward(s["dout"], s["dnormed"], *args, **kw)
    got = dict(out=out, normed=normed, dnext=dnext, dresidual=dresidual, dpost=dpost, dy=dy)
    if dgate is not None:
        got["dgate"] = dgate
    return got


def run(state):
    op = state["case"]["op"]
    if own:
        return dict(int4=_own_int4, sort=_own_sort, norm=_own_norm)[op](state)
    return dict(int4=_plain_int4, sort=_plain_sort, norm=_plain_norm)[op](state)


# ---------------------------------------------------------------- what a pass needs
def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4}
    if case["op"] == "int4":
        n, k = case["n"], case["kdim"]
        rows = case["tokens"] * case["k"]
        p = torch.arange(1, case["e"] + 1, dtype=torch.float64) ** -case["skew"]
        p = p / p.sum()
        # experts with at least one row, on average
        busy = float((1 - (1 - (p * case["k"]).clamp(max=1)) ** case["tokens"]).sum())
        groups = (k + case["group"] - 1) // case["group"]
        weights = busy * n * (k / 2 + groups * size[case["scale"]])
        return {"bytes": weights + rows * (k + n) * 2, "flops": 2.0 * rows * n * k}
    if case["op"] == "sort":
        t, k, b = case["tokens"], case["k"], size[case["dtype"]]
        token, row = t * case["h"] * b, t * k * case["h"] * b
        ids = t * k * (8 + size[case["weight"]])
        passes = 2 * row + 2 * token  # x, out; the gathered rows, the experts' rows
        if case["train"]:
            passes += 2 * row + 2 * token  # dout, dx; dy and dxs (the experts' rows are read once)
        return {"bytes": float(ids + passes), "flops": (6.0 if case["train"] else 2.0) * t * k * case["h"]}
    b, values = size[case["dtype"]], case["tokens"] * case["h"]
    gate = dict(none=0, channel=case["h"], token=case["tokens"], full=values)[case["gate"]]
    arrays = 4 * values + gate + (4 * values + gate if case["train"] else 0)
    return {"bytes": float(arrays * b + 2 * case["h"] * size[case["weight"]]),
            "flops": (45.0 if case["train"] else 12.0) * values}


# ---------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "int4":
        out = torch.empty(len(s["x"]), case["n"], dtype=torch.float64, device="cuda")
        column = torch.arange(case["kdim"], device="cuda")
        offsets = s["schedule"].group_offsets
        for e in range(case["e"]):
            a, b = offsets[e], offsets[e + 1]
            if a == b:
                continue
            code = torch.bitwise_right_shift(s["rows"][e][:, column // 2], (4 * (column % 2)).to(torch.uint8)) % 16
            weight = (code.double() - 8) * s["row_scale"][e].double()[:, column // case["group"]]
            out[a:b] = s["x"][a:b].double() @ weight.t()
        return out
    if case["op"] == "sort":
        x, y, w = s["x"].double(), s["y"].double(), s["w"].double()
        x.requires_grad_()
        y.requires_grad_()
        w.requires_grad_()
        flat = s["idx"].flatten()
        n = len(flat)
        # rank of pair f: pairs of lower experts, and earlier pairs of its own
        key = flat * n + torch.arange(n, device="cuda")
        rank = torch.searchsorted(key.sort().values, key)
        token_of_row = torch.zeros(n, dtype=torch.long, device="cuda").index_put((rank,), torch.arange(n, device="cuda") // case["k"])
        xs = x.index_select(0, token_of_row)
        out = torch.zeros(case["tokens"], case["h"], dtype=torch.float64, device="cuda")
        for slot in range(case["k"]):
            out = out + w[:, slot, None] * y.index_select(0, rank.view(-1, case["k"])[:, slot])
        got = dict(xs=xs.detach(), out=out.detach())
        if case["train"]:
            got["dx"], = torch.autograd.grad(xs, x, s["dxs"].double())
            got["dy"], got["dw"] = torch.autograd.grad(out, (y, w), s["dout"].double())
        return got
    leaf = {n: s[n].double().requires_grad_() for n in ("y", "residual", "post", "next")}
    if s["gate"] is not None:
        leaf["gate"] = s["gate"].double().requires_grad_()

    def rms(v):
        return v / (v.pow(2).sum(1, keepdim=True) / case["h"] + EPS).sqrt()

    branch = rms(leaf["y"]) * leaf["post"] * _residual_scale(case)
    out = leaf["residual"] + (branch * leaf["gate"] if "gate" in leaf else branch)
    normed = rms(out) * leaf["next"]
    got = dict(out=out.detach(), normed=normed.detach())
    if case["train"]:
        grads = torch.autograd.grad((out, normed), list(leaf.values()), (s["dout"].double(), s["dnormed"].double()))
        got.update({"d" + name: grad for name, grad in zip(leaf, grads)})
    return got
