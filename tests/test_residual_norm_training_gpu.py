"""The residual norm and the gradient clip as a training program uses them: in the AST optimisation step, and in a
chain of blocks built from the library's operators whose separate gradients are clipped into the flat buffer of the
Adam step.

Tolerances of whole chains: every gradient is a sum of products that each went through at most a few hundred 32-bit
roundings (2^-24 each), so 1e-4 of the largest element holds them with a factor of ten to spare."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

from jirf_hip import train_ops as T
from tests.gpu_util import call, ptr, stream
from tests.test_train_step_gpu import _cfg, _data, _oracle_grads, _state

pytestmark = pytest.mark.gpu
REL = 1e-4


def rel_err(got, want):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    return float(np.abs(got - want).max() / max(np.abs(want).max(), 1e-12))


def _scales(tr, B, seed):
    rng = np.random.default_rng(seed)
    out = {}
    for bl in tr._blocks():
        for branch in (("attn", "mlp") if bl["att"] else ("mlp",)):
            if bl["drop"] > 0:
                out[f"{bl['name']}.{branch}"] = ((rng.random(B) >= bl["drop"]) / (1 - bl["drop"])).astype(np.float32)
    return out


def test_ast_step_with_the_fused_join():
    """AstTrainStep(fuse_residual_norm=True): loss and every gradient against autograd over the oracle with the same
    DropPath factors, and against the step without it."""
    from jirf_hip.train import AstTrainStep
    cfg = dict(_cfg(), drop_path_rate=0.5)
    sd = _state(cfg, 21)
    lq, gt = _data(2, 128, 5)
    grads, losses = [], []
    for fuse in (False, True):
        tr = AstTrainStep(cfg, sd, coupled=True, fuse_residual_norm=fuse)
        tr.drop_scales = _scales(tr, 2, 9)
        tr.g.zero_()
        loss, _ = tr.forward_backward(torch.from_numpy(lq), torch.from_numpy(gt))
        torch.cuda.synchronize()
        losses.append(loss)
        grads.append(tr.grad_dict())
    loss_ref, _, g_ref = _oracle_grads(sd, lq, gt, cfg, drop_scales=tr.drop_scales)
    assert abs(losses[1] - loss_ref) < 1e-5 * abs(loss_ref) and abs(losses[1] - losses[0]) < 1e-6 * abs(losses[0])
    for k, g in g_ref.items():
        assert rel_err(grads[1][k], g) < 1e-3, k           # the bound of the step's other comparisons with the oracle
        if np.abs(grads[0][k]).max() > 0:
            assert rel_err(grads[1][k], grads[0][k]) < REL, k


def test_captured_ast_step_with_the_fused_join():
    """The replayed step equals the one queued kernel by kernel, bit for bit, over several steps."""
    from jirf_hip.train import AstTrainStep
    cfg = _cfg()
    sd = _state(cfg, 22)
    eager = AstTrainStep(cfg, sd, use_graph=False, fuse_residual_norm=True, seed=3)
    graph = AstTrainStep(cfg, sd, use_graph=True, fuse_residual_norm=True, seed=3)
    for it in range(1, 6):
        lq, gt = _data(2, 128, 40 + it)
        a = eager.optimize_parameters(torch.from_numpy(lq), torch.from_numpy(gt), it)
        b = graph.optimize_parameters(torch.from_numpy(lq), torch.from_numpy(gt), it)
        assert a == b and torch.equal(eager.p, graph.p) and torch.equal(eager.g, graph.g), it
    assert graph._graph is not None


def _norm(v, kind, w, b):
    mu = v.mean(1, keepdim=True) if kind != 3 else 0.0
    rs = ((v - mu).square().mean(1, keepdim=True) + 1e-5) ** -0.5
    o = ((v - mu) if kind == 1 else v) * rs * w[:, None]
    return o + b[:, None] if b is not None else o


@pytest.mark.parametrize("post,pre,gate", [(3, 3, 1), (1, 1, 2), (0, 2, 1)])
def test_blocks_forward_backward_clip_and_step(post, pre, gate):
    """Three blocks y <- y + scale gate post(W n), n <- pre(y); the branch is the library's 1x1 convolution, all gradients
    are separate tensors, GradientClip lays them clipped into the flat buffer, jirf_train_adam_step updates.  Against
    autograd in 64 bits and the same update."""
    B, C, H, blocks, max_norm = 2, 32, 16, 3, 0.05
    P = H * H
    g = torch.Generator().manual_seed(31 + post)
    rnd = lambda *s: torch.randn(*s, generator=g)                                       # noqa: E731
    names, params = [], []
    for i in range(blocks):
        for n, t in ((f"{i}.W", rnd(C, C) * C ** -0.5), (f"{i}.gate", 0.7 + 0.2 * (rnd(C) if gate == 1 else rnd(B, C))),
                     (f"{i}.post.w", 1 + 0.2 * rnd(C)), (f"{i}.post.b", 0.1 * rnd(C)), (f"{i}.pre.w", 1 + 0.2 * rnd(C)),
                     (f"{i}.pre.b", 0.1 * rnd(C))):
            if (n.endswith(".b") and (post if "post" in n else pre) != 1) or ("post" in n and not post):
                continue
            names.append(n)
            params.append(t)
    x0, target = rnd(B, C, P), rnd(B, C, P)
    scale = torch.tensor([1.0 / 0.9, 0.0])
    # 64 bits
    p64 = {n: t.double().requires_grad_(True) for n, t in zip(names, params)}
    y = x0.double()
    n = y
    for i in range(blocks):
        f = torch.matmul(p64[f"{i}.W"], n)
        u = _norm(f, post, p64[f"{i}.post.w"], p64.get(f"{i}.post.b")) if post else f
        k = p64[f"{i}.gate"][:, None] if gate == 1 else p64[f"{i}.gate"][:, :, None]
        y = y + scale.double()[:, None, None] * k * u
        n = _norm(y, pre, p64[f"{i}.pre.w"], p64.get(f"{i}.pre.b"))
    F.smooth_l1_loss(n, target.double()).backward()
    g64 = {k: v.grad for k, v in p64.items()}
    # the library
    sizes = [t.numel() for t in params]
    flat_p = torch.cat([t.reshape(-1) for t in params]).cuda()
    p = dict(zip(names, [v.view(t.shape) for v, t in zip(flat_p.split(sizes), params)]))
    grads = {k: None for k in names}
    scale, tgt = scale.cuda(), target.cuda()
    spec = lambda i, w, kind: (kind, p[f"{i}.{w}.w"], p.get(f"{i}.{w}.b")) if kind else None          # noqa: E731
    y = x0.cuda()
    n, saved = y, []
    for i in range(blocks):
        f = torch.empty_like(y)
        call("jirf_train_conv", ptr(n), 0, ptr(p[f"{i}.W"]), 0, None, None, 0, ptr(f), 0, B, C, C, H, H, 1, 1, 0, 0, stream())
        r = T.residual_norm(y, f, post=spec(i, "post", post), gate=p[f"{i}.gate"], scale=scale, pre=spec(i, "pre", pre),
                            save_stats=True)
        saved.append((n, f, r))
        y, n = r.y, r.n
    dn, loss = torch.empty_like(n), torch.zeros(1, dtype=torch.float64, device="cuda")
    call("jirf_train_smooth_l1", ptr(n), ptr(tgt), ptr(dn), n.numel(), 1.0, ptr(loss), None, stream())
    dy = None
    for i in reversed(range(blocks)):
        n_in, f, r = saved[i]
        d = T.residual_norm_bwd(dy, dn, r.y, f, r.stats, post=spec(i, "post", post), gate=p[f"{i}.gate"], scale=scale,
                                pre=spec(i, "pre", pre))
        grads[f"{i}.gate"] = d["dgate"]
        for w in ("post", "pre"):
            for q in ("w", "b"):
                if f"{i}.{w}.{q}" in grads:
                    grads[f"{i}.{w}.{q}"] = d[f"d{w}_{q}"]
        grads[f"{i}.W"] = torch.empty_like(p[f"{i}.W"])
        call("jirf_train_linear_bwd_weight", ptr(d["dbranch"]), ptr(n_in), ptr(grads[f"{i}.W"]), None, B, C, C, P, 0, stream())
        dn = torch.empty_like(n_in)
        call("jirf_train_conv", ptr(d["dbranch"]), 0, ptr(p[f"{i}.W"]), 1, None, None, 0, ptr(dn), 0, B, C, C, H, H, 1, 1, 0, 0, stream())
        dy = d["dx"]
    for k in names:
        assert rel_err(grads[k].cpu().numpy(), g64[k].numpy()) < REL, k
    flat = torch.empty(sum(sizes), device="cuda")
    stats = T.GradientClip([grads[k] for k in names], out=list(flat.split(sizes))).run(max_norm)
    total = float(torch.cat([v.reshape(-1) for v in g64.values()]).norm())
    assert total > max_norm and abs(float(stats[1]) - total) < REL * total
    m, v = torch.zeros_like(flat), torch.zeros_like(flat)
    before = flat_p.clone()
    call("jirf_train_adam_step", ptr(flat_p), ptr(flat), ptr(m), ptr(v), flat.numel(), None, 0.0, 1.0, 1e-3, 0.9, 0.999, 1e-8, 1, 1,
         stream())
    want = torch.cat([(g64[k] * min(max_norm / (total + 1e-6), 1.0)).reshape(-1) for k in names])
    # the first step of Adam moves by -lr g / (|g| + eps) whatever the gradient's size: compared where it is not noise
    step = -1e-3 * want / (want.abs() + 1e-8)
    big = want.abs() > 1e-3 * want.abs().max()
    got = (flat_p - before).double().cpu()
    assert (got - step)[big].abs().max() < 1e-3 * 1e-3 + 2.0 ** -23 * float(before.abs().max())
    assert rel_err(flat.cpu().numpy(), want.numpy()) < 3 * REL
