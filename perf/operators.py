"""Workloads of two training operators: the norms around a residual block's join (with the branch's gate and
residual scale, forward and backward) and the global gradient norm over many tensors with clipping.

`run` makes one pass: in elementary torch operations where `own` is false, through jirf_hip.train_ops where it is true.

residual_norm           u = post(f);  y = x + scale[b] * gate * u;  n = pre(y)
residual_norm_bwd       the gradients of that with respect to x, f, gate and both norms' parameters
grad_clip               total = ||grad_scale * (g_0, g_1, ...)||;  out = grad_scale * min(max_norm / (total + 1e-6), 1) * g

Norm kinds: 1 LayerNorm with bias, 2 LayerNorm without centring and bias ("BiasFree"), 3 root mean square; 0 none.
Gate kinds: 0 none, 1 one factor per channel, 2 one per image and channel.  Layouts: planar [B][C][P], tokens [B][P][C].
"""
import math
import os
import random
import sys

import torch

own = False
EPS = 1e-5
_DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    def fwd(name, layout, dtype, B, C, P, post, gate, scale, pre, train):
        return dict(name=name, op="residual_norm", layout=layout, dtype=dtype, B=B, C=C, P=P, post=post, gate=gate, scale=scale,
                    pre=pre, train=train)

    def bwd(name, layout, dtype, B, C, P, post, gate, scale, pre):
        return dict(name=name, op="residual_norm_bwd", layout=layout, dtype=dtype, B=B, C=C, P=P, post=post, gate=gate,
                    scale=scale, pre=pre)

    def clip(name, sizes, n, total, types, out, norm, max_norm, grad_scale):
        return dict(name=name, op="grad_clip", sizes=sizes, n=n, total=total, types=types, out=out, norm=norm,
                    max_norm=max_norm, grad_scale=grad_scale)

    return [
        # one token between two blocks of a step-by-step decoder, both norms and a layer scale: latency alone
        fwd("fwd_one_token", "tokens", "bf16", 1, 512, 1, 3, 1, False, 3, False),
        # AST level 0, two 256 x 256 crops: x + drop_path(attention), then norm2
        fwd("fwd_ast_level0", "planar", "fp32", 2, 32, 65536, 0, 0, True, 1, True),
        # odd channels and pixels, modulation per image, half precision
        fwd("fwd_ragged_planar", "planar", "fp16", 3, 97, 1237, 1, 2, False, 2, True),
        # a wide token model's training batch, norm on both sides of the block
        fwd("fwd_wide_tokens", "tokens", "bf16", 8, 4096, 4096, 3, 1, True, 3, True),
        # AST bottleneck, two 16 x 16 planes of 512 channels: few pixels, many channels
        bwd("bwd_ast_bottleneck", "planar", "fp32", 2, 512, 256, 0, 0, True, 1),
        # AST last decoder level, two 256 x 256 crops
        bwd("bwd_ast_decoder0", "planar", "fp32", 2, 64, 65536, 0, 0, True, 1),
        # a token model's training batch with everything on
        bwd("bwd_tokens", "tokens", "bf16", 4, 2048, 4096, 3, 1, True, 3),
        # odd sizes, modulation per image, fp32 tokens as the reference lays them out
        bwd("bwd_ragged_tokens", "tokens", "fp32", 5, 771, 333, 2, 2, False, 1),
        # a small head's gradients: latency alone
        clip("clip_small", "log", 24, 40_000, "fp32", "fp32", "2", 0.01, 1.0),
        # every gradient of the full AST (26.3 M), mean over 4 ranks on the way into the flat buffer
        clip("clip_ast", "ast", 0, 0, "fp32", "fp32", "2", 0.01, 0.25),
        # autocast gradients of three types and odd sizes, clipped by their largest value
        clip("clip_mixed", "log", 401, 60_000_000, "mixed", "fp32", "inf", 0.001, 0.0009765625),
        # half a billion bf16 gradients: beyond every cache
        clip("clip_large", "log", 160, 536_000_000, "bf16", "bf16", "2", 1.0, 1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["residual_norm", "residual_norm", "residual_norm_bwd", "residual_norm_bwd", "grad_clip"])
    if op == "grad_clip":
        types = rng.choice(["fp32", "bf16", "fp16", "mixed"])
        return dict(op=op, sizes="log", n=_log(rng, 1, 700), total=_log(rng, 1_000, 200_000_000), types=types,
                    out=rng.choice(["fp32", "bf16"] if types == "bf16" else ["fp32"]), norm=rng.choice(["2", "2", "inf"]),
                    max_norm=rng.choice([0.01, 0.1, 1.0]), grad_scale=2.0 ** -rng.randint(0, 10))
    layout = rng.choice(["planar", "tokens"])
    C = _log(rng, 16, 768) if layout == "planar" else _log(rng, 16, 8192)
    most = 60_000_000 if op == "residual_norm_bwd" else 100_000_000
    P = min(_log(rng, 1, 65536), most // C)
    B = max(1, min(_log(rng, 1, 16), most // (C * P)))
    post, pre, gate = rng.choice([0, 0, 1, 2, 3]), rng.choice([0, 1, 1, 2, 3, 3]), rng.choice([0, 1, 2])
    c = dict(op=op, layout=layout, dtype=rng.choice(["fp32", "bf16", "fp16"]), B=B, C=C, P=P, post=post, gate=gate,
             scale=rng.random() < 0.5, pre=pre)
    if op == "residual_norm":
        c["train"] = rng.random() < 0.5
    return c


def _sizes(case):
    """Element counts of the gradients, from the case alone."""
    if case["sizes"] == "ast":
        # embed_dim 32, two blocks per level, mlp_ratio 4: projections and feed-forward of each block, the resampling
        # convolutions between the levels (the token attention sits in the last five levels)
        out = [32 * 3 * 9, 32]
        for level, C in enumerate([32, 64, 128, 256, 512, 512, 256, 128, 64]):
            for _ in range(2):
                h, d = 4 * C, C // 4
                if level >= 4:
                    out += [C, C, 225 * (C // 32), 2, C * C, C, 2 * C * C, 2 * C, C * C, C]
                out += [C, C, d * d * 9, 2 * h * C, 2 * h, h * 9, h, C * h, C]
            if level < 4:
                out += [2 * C * C * 16, 2 * C]
            elif level < 8:
                out += [C * (C // 2 if level == 4 else C // 4) * 4, C // 2 if level == 4 else C // 4]
        return out + [3 * 64 * 9, 3]
    r = random.Random(case["n"] * 1_000_003 + case["total"])
    w = [math.exp(r.uniform(0.0, 9.0)) for _ in range(case["n"])]
    s = sum(w)
    return [max(1, int(case["total"] * v / s)) for v in w]


def _norm_params(kind, C, rnd):
    if kind == 0:
        return None, None
    return 1.0 + 0.2 * rnd(C), (0.1 * rnd(C) if kind == 1 else None)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if case["op"] == "grad_clip":
        kinds = {"fp32": ["fp32"], "bf16": ["bf16"], "fp16": ["fp16"], "mixed": ["bf16", "fp32", "fp16"]}[case["types"]]
        sizes = _sizes(case)
        # gradients of different tensors differ by orders of magnitude
        mags = (10.0 ** (-3.0 * torch.rand(len(sizes), generator=gen, device="cuda"))).tolist()
        grads = [rnd(n).mul_(m).to(_DT[kinds[i % len(kinds)]]) for i, (n, m) in enumerate(zip(sizes, mags))]
        flat = torch.empty(sum(sizes), dtype=_DT[case["out"]], device="cuda")
        st = dict(case=case, grads=grads, flat=flat)
        if own:
            # what a training program builds once for its parameters' gradients and keeps
            st["clip"] = _ops().GradientClip(grads, out=list(flat.split(sizes)))
        return st

    B, C, P, dt = case["B"], case["C"], case["P"], _DT[case["dtype"]]
    planar = case["layout"] == "planar"
    shape = (B, C, P) if planar else (B, P, C)
    st = dict(case=case)
    # a residual stream has a spread of channel levels, a few of them large
    level = rnd(C) * 0.5
    level[:: max(1, C // 3)] *= 8.0
    st["x"] = (rnd(*shape) * 1.5 + (level.view(1, C, 1) if planar else level)).to(dt)
    st["f"] = (rnd(*shape) * 0.7 + 0.1).to(dt)
    st["post_w"], st["post_b"] = _norm_params(case["post"], C, rnd)
    st["pre_w"], st["pre_b"] = _norm_params(case["pre"], C, rnd)
    st["gate"] = None if case["gate"] == 0 else 0.5 + 0.3 * (rnd(C) if case["gate"] == 1 else rnd(B, C))
    st["scale"] = None
    if case["scale"]:     # stochastic depth: 0 or 1 / keep_prob per sample, the first one kept
        keep = (torch.rand(B, generator=gen, device="cuda") >= 0.1).float()
        keep[0] = 1.0
        st["scale"] = keep / 0.9
    if case["op"] == "residual_norm_bwd":
        # what the forward left: y in the activations' type, the statistics in 32 bits
        st["dy"] = rnd(*shape).to(dt)
        st["dn"] = rnd(*shape).to(dt) if case["pre"] else None
        y, _, stats = _forward64(st)
        st["y"] = y.to(dt)
        st["stats"] = stats.to(torch.float32)
        del st["x"]
    return st


def _ops():
    """The framework's operators on torch tensors."""
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "image-restoration_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from jirf_hip import train_ops
    return train_ops


def run(st):
    case = st["case"]
    if own:
        return _run_own(st, case)
    if case["op"] == "grad_clip":
        return _plain_clip(st, case)
    if case["op"] == "residual_norm":
        return _plain_forward(st, case)
    return _plain_backward(st, case)


def _run_own(st, case):
    ops = _ops()
    if case["op"] == "grad_clip":
        stats = st["clip"].run(case["max_norm"], norm=float(case["norm"]), grad_scale=case["grad_scale"])
        return {"norm": stats[1:2], "flat": st["flat"]}
    post = (case["post"], st["post_w"], st["post_b"]) if case["post"] else None
    pre = (case["pre"], st["pre_w"], st["pre_b"]) if case["pre"] else None
    if case["op"] == "residual_norm":
        y, n, stats = ops.residual_norm(st["x"], st["f"], post=post, gate=st["gate"], scale=st["scale"], pre=pre,
                                        layout=case["layout"], eps=EPS, save_stats=case["train"])
        return {"y": y, "n": n, "stats": stats}
    g = ops.residual_norm_bwd(st["dy"], st["dn"], st["y"], st["f"], st["stats"], post=post, gate=st["gate"],
                              scale=st["scale"], pre=pre, layout=case["layout"])
    return g


# ---- the plain form -------------------------------------------------------------------------------------------------

def _chan(v, planar):
    """A [C] or [B, C] tensor against activations."""
    return v.unsqueeze(-1) if planar else v.unsqueeze(-2)


def _plain_norm(v, kind, w, b, planar):
    c = 1 if planar else 2
    if kind == 3:
        mu = torch.zeros_like(v.select(c, 0))
        rs = torch.rsqrt((v * v).mean(c) + EPS)
        return v * rs.unsqueeze(c) * _chan(w, planar), mu, rs
    mu = v.mean(c)
    d = v - mu.unsqueeze(c)
    rs = torch.rsqrt((d * d).mean(c) + EPS)
    if kind == 2:
        return v * rs.unsqueeze(c) * _chan(w, planar), mu, rs
    return d * rs.unsqueeze(c) * _chan(w, planar) + _chan(b, planar), mu, rs


def _plain_forward(st, case):
    planar, dt = case["layout"] == "planar", _DT[case["dtype"]]
    x, u = st["x"].float(), st["f"].float()
    none = torch.zeros(case["B"], case["P"], device="cuda") if case["train"] else None
    mu0 = rs0 = mu1 = rs1 = none
    if case["post"]:
        u, mu0, rs0 = _plain_norm(u, case["post"], st["post_w"], st["post_b"], planar)
    if st["gate"] is not None:
        u = u * _chan(st["gate"], planar)
    if st["scale"] is not None:
        u = u * st["scale"].view(-1, 1, 1)
    y = x + u
    n = None
    if case["pre"]:
        n, mu1, rs1 = _plain_norm(y, case["pre"], st["pre_w"], st["pre_b"], planar)
        n = n.to(dt)
    return {"y": y.to(dt), "n": n, "stats": torch.stack([mu0, rs0, mu1, rs1]) if case["train"] else None}


def _plain_norm_bwd(dout, v, mu, rs, kind, w, planar):
    """(dv, dw, db) of the norm of v, with the forward's statistics."""
    c = 1 if planar else 2
    rows = (0, 2) if planar else (0, 1)
    mu, rs = mu.unsqueeze(c), rs.unsqueeze(c)
    cent = (v - mu) * rs
    vh = cent if kind == 1 else v * rs
    g = dout * _chan(w, planar)
    dv = g - cent * (g * vh).mean(c, keepdim=True)
    if kind == 1:
        dv = dv - g.mean(c, keepdim=True)
    return dv * rs, (dout * vh).sum(rows), (dout.sum(rows) if kind == 1 else None)


def _plain_backward(st, case):
    planar, dt = case["layout"] == "planar", _DT[case["dtype"]]
    rows = (0, 2) if planar else (0, 1)
    d, f, s = st["dy"].float(), st["f"].float(), st["stats"]
    out = dict.fromkeys(("dx", "dbranch", "dgate", "dpost_w", "dpost_b", "dpre_w", "dpre_b"))
    if case["pre"]:
        dv, out["dpre_w"], out["dpre_b"] = _plain_norm_bwd(st["dn"].float(), st["y"].float(), s[2], s[3], case["pre"],
                                                           st["pre_w"], planar)
        d = d + dv
    out["dx"] = d.to(dt)
    du = d if st["scale"] is None else d * st["scale"].view(-1, 1, 1)
    if st["gate"] is not None:
        u = f
        if case["post"]:
            c = 1 if planar else 2
            u = f - s[0].unsqueeze(c) if case["post"] == 1 else f
            u = u * s[1].unsqueeze(c) * _chan(st["post_w"], planar)
            if case["post"] == 1:
                u = u + _chan(st["post_b"], planar)
        t = du * u
        out["dgate"] = t.sum(rows) if case["gate"] == 1 else t.sum(2 if planar else 1)
        du = du * _chan(st["gate"], planar)
    if case["post"]:
        du, out["dpost_w"], out["dpost_b"] = _plain_norm_bwd(du, f, s[0], s[1], case["post"], st["post_w"], planar)
    out["dbranch"] = du.to(dt)
    return out


def _plain_clip(st, case):
    flat = torch.cat([g.reshape(-1).float() for g in st["grads"]])
    # squares of many values of different magnitude: 64 bits
    total = flat.double().square().sum().sqrt() if case["norm"] == "2" else flat.abs().max().double()
    total = total * case["grad_scale"]
    k = case["grad_scale"] * torch.clamp(case["max_norm"] / (total + 1e-6), max=1.0)
    return {"norm": total.reshape(1), "flat": (flat * k.float()).to(_DT[case["out"]])}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def _last(t, case):
    """[B, P, C] in 64 bits whatever the layout."""
    return t.double().transpose(1, 2) if case["layout"] == "planar" else t.double()


def _back(t, case):
    return t.transpose(1, 2).contiguous() if case["layout"] == "planar" else t


def _norm64(v, kind, w, b):
    if kind == 3:
        mu = v.new_zeros(v.shape[:2])
        var = v.square().mean(-1)
    else:
        var, mu = torch.var_mean(v, dim=-1, unbiased=False)
    rs = (var + EPS).pow(-0.5)
    o = v * rs[..., None]
    if kind == 1:
        o -= (mu * rs)[..., None]
    o *= w.double()
    return (o + b.double() if b is not None else o), mu, rs


def _forward64(st):
    """y, n, statistics in 64 bits."""
    case = st["case"]
    u, z = _last(st["f"], case), torch.zeros(case["B"], case["P"], dtype=torch.float64, device="cuda")
    rows = [z, z, z, z]
    if case["post"]:
        u, rows[0], rows[1] = _norm64(u, case["post"], st["post_w"], st["post_b"])
    k = torch.ones(case["B"], case["C"], dtype=torch.float64, device="cuda")
    if st["gate"] is not None:
        k = k * st["gate"].double()
    if st["scale"] is not None:
        k = k * st["scale"].double()[:, None]
    y = torch.addcmul(_last(st["x"], case), u, k[:, None, :])
    n = None
    if case["pre"]:
        n, rows[2], rows[3] = _norm64(y, case["pre"], st["pre_w"], st["pre_b"])
        n = _back(n, case)
    return _back(y, case), n, torch.stack(rows)


def _row_dot(a, b):
    return (a * b).sum(-1)


def _norm64_bwd(d, v, mu, rs, kind, w):
    # derivative of w * (v - m) * rs(v), term by term: through the value, through the mean, through rs
    C = v.shape[-1]
    g = d * w.double()
    base = v - mu[..., None] if kind == 1 else v
    drs = _row_dot(g, base)
    dv = g * rs[..., None] - (v - mu[..., None]) * (drs * rs ** 3 / C)[..., None]
    if kind == 1:
        dv -= (g.sum(-1) * rs / C)[..., None]
    dw = torch.einsum("bpc,bpc,bp->c", d, base, rs)
    return dv, dw, d.sum((0, 1)) if kind == 1 else None


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "grad_clip":
        if case["norm"] == "2":
            total = torch.stack([g.double().square().sum() for g in st["grads"]]).sum().sqrt()
        else:
            total = torch.stack([g.abs().max().double() for g in st["grads"]]).max()
        total = total * case["grad_scale"]
        k = case["grad_scale"] * min(case["max_norm"] / (float(total) + 1e-6), 1.0)
        return {"norm": total.reshape(1), "flat": torch.cat([g.double() * k for g in st["grads"]])}
    if case["op"] == "residual_norm":
        y, n, stats = _forward64(st)
        return {"y": y, "n": n, "stats": stats if case["train"] else None}
    # the inputs are what the forward saved: y in the activations' type and the statistics as given
    s = st["stats"].double()
    out = dict.fromkeys(("dx", "dbranch", "dgate", "dpost_w", "dpost_b", "dpre_w", "dpre_b"))
    f, d = _last(st["f"], case), _last(st["dy"], case)
    if case["pre"]:
        dv, out["dpre_w"], out["dpre_b"] = _norm64_bwd(_last(st["dn"], case), _last(st["y"], case), s[2], s[3], case["pre"],
                                                       st["pre_w"])
        d = d + dv
    out["dx"] = _back(d, case)
    if st["scale"] is not None:
        d = d * st["scale"].double()[:, None, None]
    if st["gate"] is not None:
        u = f
        if case["post"]:
            u = (f - s[0][..., None] if case["post"] == 1 else f) * s[1][..., None] * st["post_w"].double()
            u = u + st["post_b"].double() if case["post"] == 1 else u
        per_image = torch.einsum("bpc,bpc->bc", d, u)
        out["dgate"] = per_image.sum(0) if case["gate"] == 1 else per_image
        k = st["gate"].double()
        d = d * (k if case["gate"] == 1 else k[:, None, :])
    if case["post"]:
        d, out["dpost_w"], out["dpost_b"] = _norm64_bwd(d, f, s[0], s[1], case["post"], st["post_w"])
    out["dbranch"] = _back(d, case)
    return out


def work(case):
    """Bytes and operations one pass cannot do without: each input read once, each output written once."""
    if case["op"] == "grad_clip":
        sizes = _sizes(case)
        es = {"fp32": [4], "bf16": [2], "fp16": [2], "mixed": [2, 4, 2]}[case["types"]]
        read = sum(n * es[i % len(es)] for i, n in enumerate(sizes))
        total = sum(sizes)
        return {"bytes": read + total * (4 if case["out"] == "fp32" else 2), "flops": 3.0 * total}
    B, C, P = case["B"], case["C"], case["P"]
    e = B * C * P
    es = 4 if case["dtype"] == "fp32" else 2
    post, pre, gate = case["post"] != 0, case["pre"] != 0, case["gate"] != 0
    params = 4 * C * (post + (case["post"] == 1) + pre + (case["pre"] == 1))
    g = 0 if not gate else 4 * C * (1 if case["gate"] == 1 else B)
    stats = 4 * B * P
    if case["op"] == "residual_norm":
        tensors = 3 + pre
        return {"bytes": tensors * e * es + params + g + (4 * stats if case["train"] else 0),
                "flops": float(e * (2 + 8 * (post + pre)))}
    tensors = 3 + 2 * pre + (1 if post or gate else 0)
    return {"bytes": tensors * e * es + 2 * (params + g) + 2 * stats * (post + pre), "flops": float(e * (2 + 4 * gate + 14 * (post + pre)))}
