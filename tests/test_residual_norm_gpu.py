"""The residual join with its norms, forward and backward, through the C ABI against the definition in 64 bits
(tests/residual_norm_ref.py, where the bounds are derived), at the sizes, layouts, types and strides where it can go
wrong; against central differences; against the operators it stands in for; captured and replayed; on two streams."""
import itertools

import pytest
import torch

import jirf_hip
from jirf_hip import train_ops as T
from tests import residual_norm_ref as R
from tests.gpu_util import call, ptr, stream

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
EPS = 1e-5


def gen(seed):
    return torch.Generator().manual_seed(seed)


def make(layout, dtype, B, C, P, post, gate, pre, scale, seed=0, offset=0):
    """Inputs on the device; offset: elements by which each activation is shifted from its allocation's start."""
    g = gen(seed * 7919 + B * 131 + C * 17 + P)
    rnd = lambda *s: torch.randn(*s, generator=g)                      # noqa: E731

    def act(t):
        buf = torch.empty(t.numel() + offset, dtype=dtype, device="cuda")
        v = buf[offset:].view(t.shape)
        v.copy_(t)
        return v

    shape = (B, C, P) if layout == "planar" else (B, P, C)
    level = rnd(C)
    d = dict(x=act(rnd(*shape) * 1.5 + (level[:, None] if layout == "planar" else level)), f=act(rnd(*shape) * 0.7 + 0.1),
             dy=act(rnd(*shape)), dn=act(rnd(*shape)))
    norm = lambda k: None if k == 0 else (k, (1 + 0.2 * rnd(C)).cuda(), (0.1 * rnd(C)).cuda() if k == 1 else None)   # noqa: E731
    d["post"], d["pre"] = norm(post), norm(pre)
    d["gate"] = None if gate == 0 else ((0.5 + 0.3 * rnd(C)).cuda() if gate == 1 else (0.5 + 0.3 * rnd(B, C)).cuda())
    d["scale"] = None
    if scale:
        s = torch.where(torch.rand(B, generator=g) < 0.3, 0.0, 1 / 0.7)
        s[0] = 1 / 0.7
        d["scale"] = s.cuda()
    return d


def run_both(d, layout, K, backward=True, eps=EPS):
    kw = dict(post=d["post"], gate=d["gate"], scale=d["scale"], pre=d["pre"], layout=layout)
    r = T.residual_norm(d["x"], d["f"], eps=eps, save_stats=True, **kw)
    want = R.forward(d["x"], d["f"], d["post"], d["gate"], d["scale"], d["pre"], layout, eps)
    R.check("y", r.y, want["y"], K, layout)
    if d["pre"] is not None:
        R.check("n", r.n, want["n"], K, layout)
    else:
        assert r.n is None
    R.check("stats", r.stats, want["stats"], K)
    if not backward:
        return r
    g = T.residual_norm_bwd(d["dy"], d["dn"], r.y, d["f"], r.stats, **kw)
    want = R.backward(d["dy"], d["dn"] if d["pre"] is not None else None, r.y, d["f"], r.stats, d["post"], d["gate"],
                      d["scale"], d["pre"], layout, eps)
    for k, w in want.items():
        assert (g[k] is None) == (w is None), k
        if w is not None:
            R.check(k, g[k], w, 2 * K + 40, layout if k in ("dx", "dbranch") else None)
    return r, g


SHAPES = {
    "planar": [(1, 1, 1), (2, 3, 5), (2, 32, 64), (1, 48, 1000), (3, 97, 127), (2, 128, 65), (1, 192, 33), (1, 384, 130),
               (2, 512, 256), (1, 771, 61), (70, 16, 9), (300, 32, 16), (1, 1030, 37), (2, 2100, 11)],
    "tokens": [(1, 1, 1), (2, 3, 5), (4, 32, 70), (1, 48, 333), (3, 97, 127), (2, 128, 64), (1, 255, 40), (1, 256, 33), (300, 257, 1),
               (1, 512, 1), (2, 771, 33), (1, 1024, 37), (5, 1537, 7), (2, 4096, 9), (1, 5000, 6), (1, 8192, 5), (3, 8197, 2),
               (2, 16400, 3)],
}
# (post, gate, pre, scale)
FORMS = [(0, 0, 1, True), (3, 1, 3, False), (1, 2, 2, True), (2, 1, 0, True), (0, 0, 0, False), (0, 2, 3, False), (3, 0, 1, True)]


@pytest.mark.parametrize("layout,size", [(lay, s) for lay in SHAPES for s in SHAPES[lay]])
def test_sizes(layout, size):
    B, C, P = size
    for i, (post, gate, pre, scale) in enumerate(FORMS):
        for dtype in (F32, BF16, F16):
            d = make(layout, dtype, B, C, P, post, gate, pre, scale, seed=i)
            try:
                run_both(d, layout, R.chain(C, layout))
            except AssertionError as e:
                raise AssertionError(f"{layout} B{B} C{C} P{P} {dtype} post {post} gate {gate} pre {pre} scale {scale}: {e}") from e


@pytest.mark.parametrize("layout", ["planar", "tokens"])
def test_every_combination_of_norms_and_gates(layout):
    for post, gate, pre, scale in itertools.product(range(4), range(3), range(4), (False, True)):
        d = make(layout, F32, 3, 40, 21, post, gate, pre, scale, seed=3)
        try:
            run_both(d, layout, R.chain(40, layout))
        except AssertionError as e:
            raise AssertionError(f"post {post} gate {gate} pre {pre} scale {scale}: {e}") from e


@pytest.mark.parametrize("layout", ["planar", "tokens"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("offset", [1, 2, 3])
def test_any_alignment(layout, dtype, offset):
    """Views that start one to three elements into an allocation, with rows that are no multiple of a vector."""
    for C, P in ((64, 62), (33, 131), (256, 64)):
        run_both(make(layout, dtype, 2, C, P, 1, 1, 1, True, offset=offset), layout, R.chain(C, layout))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_large_batch_of_images(dtype):
    """More pixels than all workgroups take at once: every worker walks over many tiles."""
    run_both(make("planar", dtype, 5, 64, 9001, 1, 2, 1, True), "planar", R.chain(64, "planar"))
    run_both(make("tokens", dtype, 3, 96, 12007, 3, 2, 3, True), "tokens", R.chain(96, "tokens"))
    run_both(make("tokens", dtype, 20011, 40, 1, 3, 2, 1, True), "tokens", R.chain(40, "tokens"))


@pytest.mark.parametrize("layout", ["planar", "tokens"])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_batch_strides_and_untouched_neighbours(layout, dtype):
    """Inputs and outputs as image-contiguous views of wider buffers; what lies between the images stays as it was."""
    B, C, P, gap = 3, 40, 50, 7
    d = make(layout, dtype, B, C, P, 3, 1, 1, True, seed=5)
    shape, n = d["x"].shape, C * P

    def wide(t=None, fill=7.0):
        buf = torch.full((B, n + gap), fill, dtype=dtype, device="cuda")
        v = buf[:, :n].unflatten(1, shape[1:])
        if t is not None:
            v.copy_(t)
        return buf, v

    (_, xs), (_, fs) = wide(d["x"]), wide(d["f"])
    (yb, ys), (nb, ns) = wide(), wide()
    kw = dict(post=d["post"], gate=d["gate"], scale=d["scale"], pre=d["pre"], layout=layout)
    a = T.residual_norm(d["x"], d["f"], save_stats=True, **kw)
    b = T.residual_norm(xs, fs, out=ys, norm_out=ns, save_stats=True, **kw)
    assert torch.equal(a.y, ys) and torch.equal(a.n, ns) and torch.equal(a.stats, b.stats)
    assert (yb[:, n:] == 7).all() and (nb[:, n:] == 7).all()
    (_, dys), (_, dns) = wide(d["dy"]), wide(d["dn"])
    g = T.residual_norm_bwd(d["dy"], d["dn"], a.y, d["f"], a.stats, **kw)
    h = T.residual_norm_bwd(dys, dns, ys, fs, a.stats, **kw)
    for k in g:
        assert (g[k] is None) == (h[k] is None) and (g[k] is None or torch.equal(g[k], h[k])), k


@pytest.mark.parametrize("layout,C,P", [("planar", 64, 70), ("planar", 1300, 9), ("tokens", 96, 70), ("tokens", 9000, 3)])
def test_in_place(layout, C, P):
    """y into x and n into f."""
    d = make(layout, F32, 2, C, P, 1, 1, 1, True, seed=6)
    kw = dict(post=d["post"], gate=d["gate"], scale=d["scale"], pre=d["pre"], layout=layout)
    a = T.residual_norm(d["x"], d["f"], **kw)
    x, f = d["x"].clone(), d["f"].clone()
    T.residual_norm(x, f, out=x, norm_out=f, **kw)
    assert torch.equal(a.y, x) and torch.equal(a.n, f)


def test_image_planes_and_missing_stream_gradient():
    """[B, C, H, W] activations; dy None is a zero gradient over the residual stream."""
    d = make("planar", F32, 2, 32, 12 * 10, 0, 1, 2, True, seed=8)
    x4, f4 = d["x"].view(2, 32, 12, 10), d["f"].view(2, 32, 12, 10)
    kw = dict(gate=d["gate"], scale=d["scale"], pre=d["pre"])
    r = T.residual_norm(x4, f4, save_stats=True, **kw)
    assert r.y.shape == x4.shape and torch.equal(r.y.flatten(2), T.residual_norm(d["x"], d["f"], **kw).y)
    g = T.residual_norm_bwd(None, d["dn"].view_as(x4), r.y, f4, r.stats, **kw)
    h = T.residual_norm_bwd(torch.zeros_like(x4), d["dn"].view_as(x4), r.y, f4, r.stats, **kw)
    assert all((g[k] is None and h[k] is None) or torch.equal(g[k], h[k]) for k in g)


@pytest.mark.parametrize("layout", ["planar", "tokens"])
@pytest.mark.parametrize("kind", [1, 2, 3])
def test_one_channel_far_above_the_others(layout, kind):
    """A channel a thousand deviations out: the variance is formed about the mean, not about any one channel."""
    C, P = 128, 40
    d = make(layout, F32, 2, C, P, kind, 1, kind, False, seed=9)
    for t in (d["x"], d["f"]):
        (t[:, 0] if layout == "planar" else t[..., 0]).add_(1000.0)
    run_both(d, layout, R.chain(C, layout))


@pytest.mark.parametrize("layout", ["planar", "tokens"])
@pytest.mark.parametrize("C", [1, 24, 300])
def test_constant_rows(layout, C):
    """No deviation at all: the reciprocal is eps^-1/2 and the normalised value 0 (kind 1); also all zeros."""
    d = make(layout, F32, 2, C, 20, 1, 0, 1, True, seed=10)
    d["x"].zero_()
    d["f"].fill_(0.5)
    run_both(d, layout, R.chain(C, layout))
    d["f"].zero_()
    r = run_both(d, layout, R.chain(C, layout), backward=False)
    assert torch.equal(r.stats[1], torch.full_like(r.stats[1], float(torch.tensor(EPS).double() ** -0.5)))


@pytest.mark.parametrize("layout", ["planar", "tokens"])
def test_not_a_number_stays_in_its_token(layout):
    B, C, P = 3, 64, 90
    d = make(layout, F32, B, C, P, 1, 1, 1, True, seed=11)
    kw = dict(post=d["post"], gate=d["gate"], scale=d["scale"], pre=d["pre"], layout=layout)
    a = T.residual_norm(d["x"], d["f"], save_stats=True, **kw)
    ga = T.residual_norm_bwd(d["dy"], d["dn"], a.y, d["f"], a.stats, **kw)
    pick = lambda t, b, p: t[b, :, p] if layout == "planar" else t[b, p]            # noqa: E731
    bad = [(0, 3, float("nan")), (1, 89, float("inf")), (2, 0, float("-inf"))]
    for b, p, v in bad:
        pick(d["f"], b, p)[5] = v
    n = T.residual_norm(d["x"], d["f"], save_stats=True, **kw)
    gb = T.residual_norm_bwd(d["dy"], d["dn"], n.y, d["f"], n.stats, **kw)
    hit = torch.zeros(B, P, dtype=torch.bool)
    for b, p, _ in bad:
        hit[b, p] = True
        assert not torch.isfinite(pick(n.n, b, p)).all()
    last = lambda t: t.transpose(1, 2) if layout == "planar" else t                  # noqa: E731
    keep = ~hit.cuda()
    for u, v in ((a.y, n.y), (a.n, n.n), (ga["dx"], gb["dx"]), (ga["dbranch"], gb["dbranch"])):
        assert torch.equal(last(u)[keep], last(v)[keep])


def test_accumulate_adds_to_the_parameter_gradients():
    B, C, P = 2, 50, 70
    d = make("planar", F32, B, C, P, 1, 2, 1, True, seed=12)
    kw = dict(post=d["post"], gate=d["gate"], scale=d["scale"], pre=d["pre"])
    r = T.residual_norm(d["x"], d["f"], save_stats=True, **kw)
    g = T.residual_norm_bwd(d["dy"], d["dn"], r.y, d["f"], r.stats, **kw)
    names = ("dpost_w", "dpost_b", "dgate", "dpre_w", "dpre_b")
    base = {k: torch.randn(g[k].shape, generator=gen(4)).cuda() for k in names}
    acc = {k: v.clone() for k, v in base.items()}
    dx, df = torch.empty_like(d["x"]), torch.empty_like(d["x"])
    work = torch.empty(jirf_hip.lib().jirf_train_residual_norm_bwd_work_floats(0, 0, 1, 2, 1, B, C, P), device="cuda")
    call("jirf_train_residual_norm_bwd", ptr(d["dy"]), 0, ptr(d["dn"]), 0, ptr(r.y), 0, ptr(d["f"]), 0, ptr(r.stats), 0, 0, 1,
         ptr(d["post"][1]), ptr(d["post"][2]), 2, ptr(d["gate"]), ptr(d["scale"]), 1, ptr(d["pre"][1]), ptr(dx), 0, ptr(df), 0,
         *[ptr(acc[k]) for k in names], 1, ptr(work), B, C, P, stream())
    for k in names:
        # the sum is rounded once more: one rounding of each addend and of the result
        tol = 2.0 ** -23 * (g[k].abs() + base[k].abs() + acc[k].abs())
        assert ((acc[k] - (g[k] + base[k])).abs() <= tol).all(), k
    assert torch.equal(dx, g["dx"]) and torch.equal(df, g["dbranch"])


def test_parameter_gradients_may_be_left_out():
    B, C, P = 2, 50, 70
    d = make("planar", F32, B, C, P, 1, 1, 1, True, seed=13)
    kw = dict(post=d["post"], gate=d["gate"], scale=d["scale"], pre=d["pre"])
    r = T.residual_norm(d["x"], d["f"], save_stats=True, **kw)
    g = T.residual_norm_bwd(d["dy"], d["dn"], r.y, d["f"], r.stats, **kw)
    names = ("dpost_w", "dpost_b", "dgate", "dpre_w", "dpre_b")
    work = torch.empty(jirf_hip.lib().jirf_train_residual_norm_bwd_work_floats(0, 0, 1, 1, 1, B, C, P), device="cuda")
    for wanted in ((), ("dpre_w",), ("dgate",), ("dpost_b", "dpre_b")):
        out = {k: torch.full((C,), 7.0, device="cuda") for k in wanted}
        dx, df = torch.empty_like(d["x"]), torch.empty_like(d["x"])
        call("jirf_train_residual_norm_bwd", ptr(d["dy"]), 0, ptr(d["dn"]), 0, ptr(r.y), 0, ptr(d["f"]), 0, ptr(r.stats), 0, 0, 1,
             ptr(d["post"][1]), ptr(d["post"][2]), 1, ptr(d["gate"]), ptr(d["scale"]), 1, ptr(d["pre"][1]), ptr(dx), 0, ptr(df), 0,
             *[ptr(out[k]) if k in wanted else None for k in names], 0, ptr(work), B, C, P, stream())
        assert torch.equal(dx, g["dx"]) and torch.equal(df, g["dbranch"])
        for k in wanted:
            assert torch.equal(out[k], g[k]), k


@pytest.mark.parametrize("layout", ["planar", "tokens"])
@pytest.mark.parametrize("post,gate,pre", [(1, 1, 1), (2, 2, 3), (3, 1, 2)])
def test_gradients_against_differences(layout, post, gate, pre):
    """<gradient, direction> against the central difference of the 64-bit forward, per input.  The difference's own
    error: h^2 times a third derivative (h = 1e-4) and 2^-53 |L| / h, both under 1e-6 of the bound below, which is the
    kernel's: K 2^-24 of the gradient's magnitude along the direction."""
    B, C, P = 2, 24, 15
    d = make(layout, F32, B, C, P, post, gate, pre, True, seed=14)
    kw = dict(post=d["post"], gate=d["gate"], scale=d["scale"], pre=d["pre"], layout=layout)
    r = T.residual_norm(d["x"], d["f"], save_stats=True, **kw)
    g = T.residual_norm_bwd(d["dy"], d["dn"], r.y, d["f"], r.stats, **kw)
    dy, dn = R.tokens_last(d["dy"], layout), R.tokens_last(d["dn"], layout)

    def loss(delta, h):
        q = {k: R.host(v) for k, v in (("x", d["x"]), ("f", d["f"]), ("gate", d["gate"]))}
        norms = {k: [d[k][0], R.host(d[k][1]), R.host(d[k][2])] for k in ("post", "pre")}
        for k, v in delta.items():
            if k in q:
                q[k] = q[k] + h * v
            else:
                norms[k[:-2]][1 if k.endswith("w") else 2] += h * v
        o = R.forward(q["x"], q["f"], norms["post"], q["gate"], d["scale"], norms["pre"], layout, EPS)
        return float((o["y"][0] * dy).sum() + (o["n"][0] * dn).sum())

    at = {"x": "dx", "f": "dbranch", "gate": "dgate", "post_w": "dpost_w", "post_b": "dpost_b", "pre_w": "dpre_w", "pre_b": "dpre_b"}
    K = 2 * R.chain(C, layout) + 40
    want = R.backward(d["dy"], d["dn"], r.y, d["f"], r.stats, d["post"], d["gate"], d["scale"], d["pre"], layout, EPS)
    for k, name in at.items():
        if g[name] is None:
            continue
        v = torch.randn(g[name].shape, generator=gen(5)).double()
        h = 1e-4
        diff = (loss({k: v}, h) - loss({k: v}, -h)) / (2 * h)
        mag = want[name][1]
        vl = R.tokens_last(v, layout) if name in ("dx", "dbranch") else v
        got = float((R.host(g[name]) * v).sum())
        tol = float((mag * vl.abs()).sum()) * K * R.U + 1e-6 * float((mag * vl.abs()).sum())
        assert abs(got - diff) <= tol, f"{name}: {got} against {diff}, bound {tol}"


def test_against_the_operators_it_stands_in_for():
    """x + drop_path(branch), then the next norm, and back: jirf_train_scale_add + jirf_train_layernorm(_bwd).  Both sides
    round in 32 bits, so they agree within twice the bound of one."""
    B, C, P = 2, 64, 1024
    d = make("planar", F32, B, C, P, 0, 0, 1, True, seed=15)
    _, w, b = d["pre"]
    r = T.residual_norm(d["x"], d["f"], scale=d["scale"], pre=d["pre"], save_stats=True)
    y, n = torch.empty_like(d["x"]), torch.empty_like(d["x"])
    call("jirf_train_scale_add", ptr(d["x"]), 0, ptr(d["f"]), 0, ptr(d["scale"]), ptr(y), 0, B, C * P, stream())
    call("jirf_train_layernorm", ptr(y), 0, ptr(w), ptr(b), ptr(n), 0, B, C, P, 1, stream())
    K = 2 * R.chain(C, "planar")
    want = R.forward(d["x"], d["f"], None, None, d["scale"], d["pre"], "planar", EPS)
    R.check("y", y, (R.tokens_last(r.y, "planar"), want["y"][1]), K, "planar")
    R.check("n", n, (R.tokens_last(r.n, "planar"), want["n"][1]), K, "planar")
    dx, df, dw, db = torch.empty_like(d["x"]), torch.empty_like(d["x"]), torch.empty_like(w), torch.empty_like(b)
    call("jirf_train_layernorm_bwd", ptr(y), 0, ptr(d["dn"]), 0, ptr(w), ptr(d["dy"]), 0, ptr(dx), 0, ptr(dw), ptr(db), B, C, P, 1, 0,
         stream())
    call("jirf_train_scale_add", None, 0, ptr(dx), 0, ptr(d["scale"]), ptr(df), 0, B, C * P, stream())
    g = T.residual_norm_bwd(d["dy"], d["dn"], r.y, None, r.stats, scale=d["scale"], pre=d["pre"])
    want = R.backward(d["dy"], d["dn"], r.y, None, r.stats, None, None, d["scale"], d["pre"], "planar", EPS)
    for k, t in (("dx", dx), ("dbranch", df), ("dpre_w", dw), ("dpre_b", db)):
        lay = "planar" if k in ("dx", "dbranch") else None
        R.check(k, t, (R.tokens_last(g[k], "planar") if lay else R.host(g[k]), want[k][1]), 2 * K + 80, lay)


def test_same_bits_every_time_and_on_two_streams():
    d = make("planar", BF16, 4, 96, 5000, 1, 2, 1, True, seed=16)
    kw = dict(post=d["post"], gate=d["gate"], scale=d["scale"], pre=d["pre"])
    one = T.residual_norm(d["x"], d["f"], save_stats=True, **kw)
    g = T.residual_norm_bwd(d["dy"], d["dn"], one.y, d["f"], one.stats, **kw)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    res = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            r = T.residual_norm(d["x"], d["f"], save_stats=True, **kw)
            res.append((r, T.residual_norm_bwd(d["dy"], d["dn"], r.y, d["f"], r.stats, **kw)))
    torch.cuda.synchronize()
    for r, h in res:
        assert torch.equal(r.y, one.y) and torch.equal(r.n, one.n)
        assert all(g[k] is None or torch.equal(g[k], h[k]) for k in g)


def test_captured_and_replayed():
    d = make("planar", F32, 2, 64, 3000, 1, 2, 1, True, seed=17)
    kw = dict(post=d["post"], gate=d["gate"], scale=d["scale"], pre=d["pre"])

    def step():
        r = T.residual_norm(d["x"], d["f"], save_stats=True, **kw)
        return r, T.residual_norm_bwd(d["dy"], d["dn"], r.y, d["f"], r.stats, **kw)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r, g = step()
    for i in range(4):
        d["x"].copy_(torch.randn(d["x"].shape, generator=gen(100 + i)))
        d["dn"].copy_(torch.randn(d["x"].shape, generator=gen(200 + i)))
        graph.replay()
        torch.cuda.synchronize()
        er, eg = step()
        torch.cuda.synchronize()
        assert torch.equal(r.y, er.y) and torch.equal(r.n, er.n) and torch.equal(r.stats, er.stats)
        assert all(eg[k] is None or torch.equal(g[k], eg[k]) for k in eg)


def test_offsets_past_32_bits():
    """2.3 G elements of one tensor: the second image's last pixel lies past 2^31 elements and 2^32 bytes."""
    B, C, P = 2, 64, 18_000_064
    x = torch.zeros(B, C, P, dtype=BF16, device="cuda")
    f = torch.zeros(B, C, P, dtype=BF16, device="cuda")
    tail = torch.randn(C, 70, generator=gen(18)).to(BF16).cuda()
    x[1, :, P - 70:], f[1, :, P - 70:] = tail, -0.5 * tail
    w = torch.ones(C, device="cuda")
    r = T.residual_norm(x, f, pre=(3, w, None))
    small = T.residual_norm(tail[None], (-0.5 * tail)[None], pre=(3, w, None))
    assert torch.equal(r.y[1, :, P - 70:], small.y[0]) and torch.equal(r.n[1, :, P - 70:], small.n[0])
    assert not r.y[0].any() and not r.n[1, :, : P - 70].any()


@pytest.mark.parametrize("layout,C", [("planar", 48), ("planar", 2100), ("tokens", 200), ("tokens", 9000)])
def test_without_a_pre_norm_dx_is_dy(layout, C):
    """The stream's gradient passes through unchanged and uncopied; written where the caller of the C entry asks for it."""
    B, P = 2, 30
    d = make(layout, F32, B, C, P, 0, 1, 0, True, seed=19)
    kw = dict(gate=d["gate"], scale=d["scale"], layout=layout)
    g = T.residual_norm_bwd(d["dy"], None, None, d["f"], None, **kw)
    assert g["dx"] is d["dy"]
    assert all(T.residual_norm_bwd(d["dy"], None, None, None, None, layout=layout)[k] is d["dy"] for k in ("dx", "dbranch"))
    lay = T.LAYOUTS[layout]
    work = torch.empty(jirf_hip.lib().jirf_train_residual_norm_bwd_work_floats(0, lay, 0, 1, 0, B, C, P), device="cuda")
    for want in (False, True):
        dx, df, dg = torch.full_like(d["dy"], 7.0), torch.empty_like(d["dy"]), torch.empty(C, device="cuda")
        call("jirf_train_residual_norm_bwd", ptr(d["dy"]), 0, None, 0, None, 0, ptr(d["f"]), 0, None, 0, lay, 0, None, None, 1,
             ptr(d["gate"]), ptr(d["scale"]), 0, None, ptr(dx) if want else None, 0, ptr(df), 0, None, None, ptr(dg), None, None, 0,
             ptr(work), B, C, P, stream())
        assert torch.equal(df, g["dbranch"]) and torch.equal(dg, g["dgate"])
        assert torch.equal(dx, d["dy"]) if want else (dx == 7).all()


@pytest.mark.parametrize("layout", ["planar", "tokens"])
def test_an_image_past_32_bits(layout):
    """4.6 GB in one image: every byte offset past 2^32, forward and backward; all but the last pixels are zero, so the
    parameter gradients are those of the last pixels alone (summed in another order: the bound of each side)."""
    C, P, n = 64, 18_000_064, 70
    shape = (1, C, P) if layout == "planar" else (1, P, C)
    last = (lambda t: t[..., P - n:]) if layout == "planar" else (lambda t: t[:, P - n:])          # noqa: E731
    g = gen(20)
    small = {k: torch.randn((1, C, n) if layout == "planar" else (1, n, C), generator=g).cuda() for k in ("x", "f", "dy", "dn")}
    big = {}
    for k, t in small.items():
        big[k] = torch.zeros(shape, device="cuda")
        last(big[k]).copy_(t)
    w, gate = (1 + 0.2 * torch.randn(C, generator=g)).cuda(), torch.randn(C, generator=g).cuda()
    kw = dict(post=(3, w, None), gate=gate, pre=(1, w, None), layout=layout)
    R1 = T.residual_norm(big["x"], big["f"], save_stats=True, **kw)
    r = T.residual_norm(small["x"], small["f"], save_stats=True, **kw)
    K = R.chain(C, layout)
    want = R.forward(small["x"], small["f"], kw["post"], gate, None, kw["pre"], layout, EPS)
    for got, name in ((last(R1.y), "y"), (last(R1.n), "n")):
        R.check(name, got, want[name], K, layout)
    assert not R1.y.flatten()[: 10_000_000].any()
    d = T.residual_norm_bwd(big["dy"], big["dn"], R1.y, big["f"], R1.stats, **kw)
    want = R.backward(small["dy"], small["dn"], r.y, small["f"], r.stats, kw["post"], gate, None, kw["pre"], layout, EPS)
    for k in ("dx", "dbranch"):
        R.check(k, last(d[k]), want[k], 4 * K + 80, layout)
    for k in ("dgate", "dpost_w", "dpre_w"):
        R.check(k, d[k], want[k], 4 * K + 80)


@pytest.mark.parametrize("layout,dtype,C,P", [("planar", F32, 5, 9), ("planar", BF16, 70, 131), ("tokens", F32, 9, 6),
                                              ("tokens", BF16, 9, 6), ("tokens", F16, 523, 6), ("tokens", F32, 2051, 3)])
def test_an_infinity_where_vectors_meet(layout, dtype, C, P):
    """Near a ragged end two threads hold the same element, and one of them owns it: an infinity there counts once (inf, not
    inf - inf or inf * 0) and leaves every other channel's gradient as it is."""
    d = make(layout, dtype, 2, C, P, 0, 1, 0, False, seed=21)
    kw = dict(gate=d["gate"], layout=layout)
    d["dy"].abs_().add_(0.5)
    clean = T.residual_norm_bwd(d["dy"], None, None, d["f"], None, **kw)["dgate"]
    for back in range(1, 9):
        f = d["f"].clone()
        c, p = (C // 2, P - back) if layout == "planar" else (C - back, P // 2)
        (f[1, c] if layout == "planar" else f[1, :, c])[p] = float("inf")
        dg = T.residual_norm_bwd(d["dy"], None, None, f, None, **kw)["dgate"]
        assert dg[c] == float("inf"), (back, float(dg[c]))
        others = torch.arange(C, device="cuda") != c
        assert torch.equal(dg[others], clean[others])
        # a gradient dn of infinity: the same pattern of infinities and NaN as the formula gives
        w = (1 + 0.1 * torch.arange(C, device="cuda") / C).float()
        r = T.residual_norm(d["x"], d["f"], pre=(3, w, None), layout=layout, save_stats=True)
        dn = d["dn"].clone()
        (dn[1, c] if layout == "planar" else dn[1, :, c])[p] = float("inf")
        g = T.residual_norm_bwd(d["dy"], dn, r.y, None, r.stats, pre=(3, w, None), layout=layout)
        want = R.backward(d["dy"], dn, r.y, None, r.stats, None, None, None, (3, w, None), layout, EPS)
        for k in ("dx", "dpre_w"):
            got, ref = (R.tokens_last(g[k], layout) if k == "dx" else R.host(g[k])), want[k][0]
            assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(torch.isinf(got), torch.isinf(ref)), (back, k)


@pytest.mark.parametrize("dtype,C,P", [(BF16, 2048, 34000), (F32, 2051, 17000), (F16, 4100, 17000), (BF16, 4096, 33000)])
def test_calls_larger_than_the_cache(dtype, C, P):
    """Token rows whose operands (and, in the last case, outputs) are streamed past the caches: bit for bit what shorter
    calls give row by row, and parameter gradients equal to the shorter calls' sum (each within its bound: the sums of
    absolute terms at 32-bit roundings)."""
    g = torch.Generator(device="cuda").manual_seed(22)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")                        # noqa: E731
    x, f, dy, dn = (rnd(1, P, C).to(dtype) for _ in range(4))
    w, gate = 1 + 0.2 * rnd(C), rnd(C)
    kw = dict(post=(3, w, None), gate=gate, pre=(1, w, None), layout="tokens")
    big = T.residual_norm(x, f, save_stats=True, **kw)
    gb = T.residual_norm_bwd(dy, dn, big.y, f, big.stats, **kw)
    cut, sums, mags = 4000, {}, {}
    for p in range(0, P, cut):
        s = slice(p, min(P, p + cut))
        part = [t[:, s].contiguous() for t in (x, f, dy, dn)]
        r = T.residual_norm(part[0], part[1], save_stats=True, **kw)
        assert torch.equal(r.y, big.y[:, s]) and torch.equal(r.n, big.n[:, s]) and torch.equal(r.stats, big.stats[:, :, s])
        d = T.residual_norm_bwd(part[2], part[3], r.y, part[1], r.stats, **kw)
        assert torch.equal(d["dx"], gb["dx"][:, s]) and torch.equal(d["dbranch"], gb["dbranch"][:, s])
        for k in ("dgate", "dpost_w", "dpre_w"):
            sums[k] = sums.get(k, 0) + d[k].double()
    # |terms| <= |dn| |vh| and so on are of order one each, so the sum of their magnitudes is at most about P; a worker adds
    # at most P / 256 rows in 32 bits
    for k, v in sums.items():
        assert (gb[k].double() - v).abs().max() <= (P / 256 + 60) * 2.0 ** -24 * 8 * P, k


# fp32 planes of more than 128 channels, forward: eight, four and two pixel lanes; ragged channels and pixels; the last two
# with more tiles than workers
@pytest.mark.parametrize("B,C,P", [(9, 131, 1003), (64, 300, 130), (4, 511, 2055), (300, 257, 5), (2, 700, 50), (1, 1024, 9),
                                   (3, 1025, 21), (1, 2047, 401), (1, 2048, 4), (8, 512, 2055), (33, 131, 2011)])
def test_planes_of_many_channels(B, C, P):
    for i, (post, gate, pre, scale) in enumerate([(1, 2, 1, True), (3, 1, 2, False), (0, 0, 3, True)][:1 if B * C * P > 5e6 else 3]):
        d = make("planar", F32, B, C, P, post, gate, pre, scale, seed=30 + i)
        r = run_both(d, "planar", R.chain(C, "planar"), backward=False)
        kw = dict(post=d["post"], gate=d["gate"], scale=d["scale"], pre=d["pre"])
        x, f = d["x"].clone(), d["f"].clone()
        T.residual_norm(x, f, out=x, norm_out=f, **kw)
        assert torch.equal(x, r.y) and torch.equal(f, r.n)
        # a pixel of infinities is nobody else's: every other pixel keeps its bits
        for back in (1, 3, 4, 5):
            if back > P:
                continue
            x = d["x"].clone()
            x[:, :, P - back] = float("inf")
            s = T.residual_norm(x, d["f"], **kw)
            others = torch.arange(P, device="cuda") != P - back
            assert torch.equal(s.y[..., others], r.y[..., others]) and torch.equal(s.n[..., others], r.n[..., others])
            assert torch.isinf(s.y[..., P - back]).all()
