"""The backward of the residual join against the definition in 64 bits, with the bound that holds once the statistics are
given.

The backward reads mean and reciprocal deviation as they are, so the cancellation of their own computation is not in it:
a centred value v - mean is one rounding of its own size, and (v - mean) rs a second one.  In place of the general bound's
kappa (|v| + mean |v|) rs (tests/residual_norm_ref.py) the magnitude of a normalised value is therefore the value itself, and
so it is of a centred one.  Everything else of that bound stays.  `bounded` also asks that no bound is so wide that any
number would pass: the part of it that is not the store's own rounding stays below a hundredth of the largest value or of
one unit.  (A single channel has no deviation, its gradients are differences of equal numbers times eps^-1/2: test_one_channel.)"""
import pytest
import torch

from jirf_hip import train_ops as T
from tests import residual_norm_ref as R
from tests import test_residual_norm_gpu as G

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
EPS = G.EPS


class GivenStats(R.Norm):
    def __init__(self, v, mag, kind, w, b, eps, stats=None):
        assert stats is not None
        super().__init__(v, mag, kind, w, b, eps, stats)
        self.vh_mag = self.vh.abs()
        self.out_mag = self.vh_mag * w.abs() + (b.abs() if b is not None else 0)

    def backward(self, dout, dmag):
        dv, _, dw, dwm, db, dbm = super().backward(dout, dmag)
        rs, gm = self.rs[..., None], dmag * self.w.abs()
        dvm = gm + self.cent.abs() * (gm * self.vh_mag).mean(-1, keepdim=True)
        if self.kind == 1:
            dvm = dvm + gm.mean(-1, keepdim=True)
        return dv, dvm * rs, dw, dwm, db, dbm


@pytest.fixture(autouse=True)
def given(monkeypatch):
    monkeypatch.setattr(R, "Norm", GivenStats)


def reference(d, y, stats, layout):
    return R.backward(d["dy"], d["dn"] if d["pre"] is not None else None, y, d["f"], stats, d["post"], d["gate"], d["scale"], d["pre"],
                      layout, EPS)


def bounded(name, value, mag, K, limit=0.01):
    assert float((K * R.U * mag).max()) <= limit * max(1.0, float(value.abs().max())), f"{name}: a bound that says nothing"


def run(d, layout, C):
    kw = dict(post=d["post"], gate=d["gate"], scale=d["scale"], pre=d["pre"], layout=layout)
    r = T.residual_norm(d["x"], d["f"], eps=EPS, save_stats=True, **kw)
    g = T.residual_norm_bwd(d["dy"], d["dn"], r.y, d["f"], r.stats, **kw)
    K = 2 * R.chain(C, layout) + 40
    for k, w in reference(d, r.y, r.stats, layout).items():
        assert (g[k] is None) == (w is None), k
        if w is not None:
            if C > 1:
                bounded(k, *w, K)
            R.check(k, g[k], w, K, layout if k in ("dx", "dbranch") else None)
    return r, g


@pytest.mark.parametrize("layout,size", [(lay, s) for lay in G.SHAPES for s in G.SHAPES[lay]])
def test_sizes(layout, size):
    B, C, P = size
    for i, (post, gate, pre, scale) in enumerate(G.FORMS + [(1, 1, 1, True)]):
        for dtype in (F32, BF16, F16):
            d = G.make(layout, dtype, B, C, P, post, gate, pre, scale, seed=i)
            try:
                run(d, layout, C)
            except AssertionError as e:
                raise AssertionError(f"{layout} B{B} C{C} P{P} {dtype} post {post} gate {gate} pre {pre} scale {scale}: {e}") from e


@pytest.mark.parametrize("layout", ["planar", "tokens"])
@pytest.mark.parametrize("kind", [1, 2, 3])
@pytest.mark.parametrize("C", [24, 300])
def test_one_channel_far_above_the_others(layout, kind, C):
    d = G.make(layout, F32, 2, C, 40, kind, 1, kind, True, seed=40)
    for t in (d["x"], d["f"]):
        (t[:, 0] if layout == "planar" else t[..., 0]).add_(1000.0)
    run(d, layout, C)


@pytest.mark.parametrize("layout", ["planar", "tokens"])
@pytest.mark.parametrize("C", [1, 24, 300])
def test_constant_rows(layout, C):
    """No deviation: rs is eps^-1/2 and every normalised value a rounding of zero."""
    d = G.make(layout, F32, 2, C, 20, 1, 0, 1, True, seed=10)
    d["x"].zero_()
    d["f"].fill_(0.5)
    r, g = run(d, layout, C)
    rs = EPS ** -0.5
    dsum = R.tokens_last(g["dx"], layout).mul(R.host(d["scale"]).reshape(-1, 1, 1))
    # the mean of C halves is off by the roundings of its sum, then of its division
    off = (C // 4 + 10) * R.U * 0.5
    assert (R.host(g["dpost_w"]).abs() <= rs * off * dsum.abs().sum((0, 1)) * 1.01).all()
    assert ((R.host(g["dpost_b"]) - dsum.sum((0, 1))).abs() <= 64 * R.U * dsum.abs().sum((0, 1))).all()
    # the stream itself constant: n is the bias, off by that mean
    r = T.residual_norm(d["f"], torch.zeros_like(d["f"]), pre=d["pre"], layout=layout, eps=EPS, save_stats=True)
    w, b = R.host(d["pre"][1]), R.host(d["pre"][2])
    assert ((R.tokens_last(r.n, layout) - b).abs() <= rs * off * w.abs() * 1.01 + 2 * R.U * b.abs()).all()
    g = T.residual_norm_bwd(d["dy"], d["dn"], r.y, None, r.stats, pre=d["pre"], layout=layout)
    dn = R.tokens_last(d["dn"], layout)
    assert (R.host(g["dpre_w"]).abs() <= rs * off * dn.abs().sum((0, 1)) * 1.01).all()
    assert ((R.host(g["dpre_b"]) - dn.sum((0, 1))).abs() <= 64 * R.U * dn.abs().sum((0, 1))).all()


@pytest.mark.parametrize("layout", ["planar", "tokens"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,P", [(1, 1), (3, 70), (300, 5)])
def test_one_channel(layout, dtype, B, P):
    """A single channel is its own mean: the centred norm gives its bias, the normalised value is zero, and no gradient passes
    but the rounding of dn w, times eps^-1/2.  (In 16 bits y is rounded and the saved mean is not: vh of y is no zero there.)"""
    d = G.make(layout, dtype, B, 1, P, 1, 1, 1, True, seed=41)
    r, g = run(d, layout, 1)
    assert torch.equal(r.n, d["pre"][2].to(dtype).expand_as(r.n))
    assert not g["dpost_w"].any()
    if dtype is F32:
        assert not g["dpre_w"].any()
        dy, dn = R.host(d["dy"]), R.host(d["dn"])
        off = 4 * R.U * EPS ** -0.5 * (dn * float(d["pre"][1])).abs() * 1.01
        dx = R.host(g["dx"])
        assert ((dx - dy).abs() <= off + R.U * dx.abs()).all()
        du = dx * R.host(d["scale"]).reshape(-1, 1, 1) * float(d["gate"]) * float(d["post"][1])
        assert (R.host(g["dbranch"]).abs() <= 4 * R.U * EPS ** -0.5 * du.abs() * 1.01).all()
