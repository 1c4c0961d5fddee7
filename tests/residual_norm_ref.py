"""The residual join with its norms (jirf_train_residual_norm and its backward) restated in 64 bits, together with a
bound on what 32-bit arithmetic may lose.

Every fp32 value of the kernels comes out of a chain of at most K roundings (K counts the longest sum of one thread, the
additions across threads and the operations around them), so its error is at most K 2^-24 M to first order, with M the
same formula evaluated on absolute values.  The reciprocal deviation carries the cancellation of v - mu: its relative
error is at most K 2^-24 kappa, kappa = 1 + rms(|v| + mean |v|) / deviation (1 for the root mean square, which
subtracts nothing).  The store adds half a step of its type: 2^-8 (bf16), 2^-11 (fp16) or 2^-24 (fp32) of the value
(fp16: at least half its smallest step, 2^-25)."""
import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
U = 2.0 ** -24


def tokens_last(t, layout):
    """[B, P, C] float64 on the host."""
    t = t.detach().double().cpu()
    return t.flatten(2).transpose(1, 2) if layout == "planar" else t


def chain(C, layout):
    """Roundings of a sum over the channels: at least four threads share a planar pixel, at least eight channels'
    worth of lanes a token."""
    return C // 4 + 40 if layout == "planar" else C // 8 + 40


class Norm:
    """One norm of v [B, P, C] in 64 bits: the value `out`, the statistics, and the bound's magnitudes."""

    def __init__(self, v, mag, kind, w, b, eps, stats=None):
        # mag: magnitude of v's own error (|terms| that v was added up from)
        self.kind, self.v, self.w = kind, v, w
        self.mu = v.mean(-1) if kind != 3 else torch.zeros(v.shape[:2], dtype=torch.float64)
        var = (v - self.mu[..., None]).square().mean(-1)
        self.rs = (var + eps) ** -0.5
        if stats is not None:
            self.mu, self.rs = stats
        m, rs = self.mu[..., None], self.rs[..., None]
        am = mag + mag.mean(-1, keepdim=True) if kind != 3 else mag
        self.kappa = (1 + am.square().mean(-1, keepdim=True).sqrt() * rs) if kind != 3 else 1 + mag.square().mean(-1, keepdim=True).sqrt() * rs
        self.vh = (v - m) * rs if kind == 1 else v * rs
        self.cent = (v - m) * rs
        self.vh_mag = self.kappa * am * rs
        self.out = self.vh * w + (b if b is not None else 0)
        self.out_mag = self.vh_mag * w.abs() + (b.abs() if b is not None else 0)

    def backward(self, dout, dmag):
        """dv, dw, db of dout and their magnitudes."""
        rs = self.rs[..., None]
        g, gm = dout * self.w, dmag * self.w.abs()
        s2 = (g * self.vh).mean(-1, keepdim=True)
        s2m = (gm * self.vh_mag).mean(-1, keepdim=True)
        dv = g - self.cent * s2
        dvm = gm + self.vh_mag * s2m
        if self.kind == 1:
            dv = dv - g.mean(-1, keepdim=True)
            dvm = dvm + gm.mean(-1, keepdim=True)
        return dv * rs, dvm * rs, dout * self.vh, dmag * self.vh_mag, dout, dmag


def host(t):
    return None if t is None else t.detach().double().cpu()


def factors(B, C, gate, scale):
    k = torch.ones(B, 1, C, dtype=torch.float64)
    s = torch.ones(B, 1, 1, dtype=torch.float64)
    if gate is not None:
        g = host(gate)
        k = (g if g.dim() == 2 else g.expand(B, C)).reshape(B, 1, C)
    if scale is not None:
        s = host(scale).reshape(B, 1, 1)
    return k, s


def forward(x, f, post, gate, scale, pre, layout, eps):
    """{"y", "n", "stats"}: (value, magnitude) pairs, [B, P, C] and [4, B, P]."""
    x, f = tokens_last(x, layout), tokens_last(f, layout)
    B, P, C = x.shape
    k, s = factors(B, C, gate, scale)
    u, um, st = f, f.abs(), [torch.zeros(B, P, dtype=torch.float64)] * 4
    sm = list(st)
    if post is not None:
        N = Norm(f, f.abs(), post[0], host(post[1]), host(post[2]), eps)
        u, um = N.out, N.out_mag
        st[0], st[1] = N.mu, N.rs
        sm[0], sm[1] = f.abs().mean(-1), N.rs * N.kappa[..., 0]
    y, ym = x + s * k * u, x.abs() + (s * k).abs() * um
    n = nm = None
    if pre is not None:
        N = Norm(y, ym, pre[0], host(pre[1]), host(pre[2]), eps)
        n, nm = N.out, N.out_mag
        st[2], st[3] = N.mu, N.rs
        sm[2], sm[3] = ym.mean(-1), N.rs * N.kappa[..., 0]
    return {"y": (y, ym), "n": (n, nm), "stats": (torch.stack(st), torch.stack(sm))}


def backward(dy, dn, y, f, stats, post, gate, scale, pre, layout, eps):
    """(value, magnitude) of every gradient; y and the statistics are what the forward saved."""
    like = dy if dy is not None else dn
    lt = tokens_last(like, layout)
    B, P, C = lt.shape
    k, s = factors(B, C, gate, scale)
    st = host(stats)
    out = dict.fromkeys(("dx", "dbranch", "dgate", "dpost_w", "dpost_b", "dpre_w", "dpre_b"))
    d = tokens_last(dy, layout) if dy is not None else torch.zeros_like(lt)
    dm = d.abs()
    if pre is not None:
        v, dnl = tokens_last(y, layout), tokens_last(dn, layout)
        N = Norm(v, v.abs(), pre[0], host(pre[1]), host(pre[2]), eps, (st[2], st[3]))
        dv, dvm, dw, dwm, db, dbm = N.backward(dnl, dnl.abs())
        d, dm = d + dv, dm + dvm
        out["dpre_w"] = (dw.sum((0, 1)), dwm.sum((0, 1)))
        if pre[0] == 1 and pre[2] is not None:
            out["dpre_b"] = (db.sum((0, 1)), dbm.sum((0, 1)))
    out["dx"] = (d, dm)
    du, dum = d * s, dm * s.abs()
    N = None
    if post is not None:
        v = tokens_last(f, layout)
        N = Norm(v, v.abs(), post[0], host(post[1]), host(post[2]), eps, (st[0], st[1]))
    if gate is not None:
        u, um = (N.out, N.out_mag) if N is not None else (tokens_last(f, layout), tokens_last(f, layout).abs())
        t, tm = du * u, dum * um
        out["dgate"] = (t.sum((0, 1)), tm.sum((0, 1))) if gate.dim() == 1 else (t.sum(1), tm.sum(1))
    du, dum = du * k, dum * k.abs()
    if N is not None:
        dv, dvm, dw, dwm, db, dbm = N.backward(du, dum)
        out["dpost_w"] = (dw.sum((0, 1)), dwm.sum((0, 1)))
        if post[0] == 1 and post[2] is not None:
            out["dpost_b"] = (db.sum((0, 1)), dbm.sum((0, 1)))
        du, dum = dv, dvm
    out["dbranch"] = (du, dum)
    return out


def check(name, got, want, K, layout=None):
    """got (a device tensor) against (value, magnitude): every element within half a step of its type plus K 2^-24 M."""
    value, mag = want
    g = host(got) if layout is None else tokens_last(got, layout)
    assert g.shape == value.shape, f"{name}: shape {tuple(g.shape)}, expected {tuple(value.shape)}"
    tol = HALF[got.dtype] * (value.abs() + K * U * mag) + K * U * mag + (2.0 ** -25 if got.dtype == torch.float16 else 1e-37)
    err = (g - value).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} outside the bound, worst error / bound "
                           f"{float((err / tol)[bad].max()):.3g}")
