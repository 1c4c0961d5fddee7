"""The residual norm at the far ends of the sizes it takes: counts next to 2^31, calls beyond the cache."""
import pytest
import torch

from jirf_hip import train_ops as T

pytestmark = pytest.mark.gpu


def test_parameter_gradients_of_the_most_images():
    """2^31 - 1 images of one token and one channel: the last worker's images end past 31 bits unless counted in 64.  All but
    the first and the last two images are zero, so each gradient is a sum of three small whole numbers, exact in any order;
    with mean 0 and reciprocal deviation 1 as the statistics, vh is y."""
    B = 2**31 - 1
    at = torch.tensor([0, B - 2, B - 1], device="cuda")
    dn, y = (torch.zeros(B, 1, 1, dtype=torch.float16, device="cuda") for _ in range(2))
    dn[at, 0, 0] = torch.tensor([1.0, 2.0, 4.0], dtype=torch.float16, device="cuda")
    y[at, 0, 0] = torch.tensor([3.0, 5.0, 7.0], dtype=torch.float16, device="cuda")
    stats = torch.zeros(4, B, 1, device="cuda")
    stats[3] = 1.0
    pre = (1, torch.ones(1, device="cuda"), torch.zeros(1, device="cuda"))
    g = T.residual_norm_bwd(None, dn, y, None, stats, pre=pre, scale=None, layout="tokens")
    assert float(g["dpre_b"]) == 1 + 2 + 4
    assert float(g["dpre_w"]) == 1 * 3 + 2 * 5 + 4 * 7


def _stream(tensors, outputs, nbytes):
    """How a token call with rows of more than 512 channels treats the 256 MB cache: 0 through it, 1 operands read past it,
    2 outputs written past it too (the forward alone)."""
    return 0 if nbytes * tensors <= 256 << 20 else 2 if outputs * nbytes > 256 << 20 else 1


# each type with eight and with sixteen channels per thread; in 16-bit types the backward of a branch with a norm or gate has
# sixteen from 2049 channels on
STREAMED = [(torch.float32, 1030), (torch.float32, 5003), (torch.bfloat16, 1030), (torch.bfloat16, 2600), (torch.bfloat16, 5003),
            (torch.float16, 1030), (torch.float16, 2600), (torch.float16, 5003)]


@pytest.mark.parametrize("dtype,C", STREAMED)
@pytest.mark.parametrize("mib,stream", [(96, 1), (160, 2)])
def test_calls_beyond_the_cache_in_each_form(dtype, C, mib, stream):
    """Tensors of 96 MiB, whose operands alone go past the cache, and of 160 MiB, whose outputs do too; without a branch norm,
    with one, with a gate per image: bit for bit what short calls give, which stay in the cache.  A parameter gradient is a sum
    of the same terms in another order: a worker adds at most ceil(B P / 256) rows in 32 bits, about the magnitudes' sum."""
    B, es = 2, torch.empty((), dtype=dtype).element_size()
    P = (mib << 20) // (B * C * es)
    nbytes, cut = B * C * P * es, -(-P // 6)
    assert _stream(4, 2, nbytes) == stream and _stream(6, 3, nbytes) > 0 and _stream(6, 3, B * C * cut * es) == 0
    g = torch.Generator(device="cuda").manual_seed(C)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")                        # noqa: E731
    x, f, dy, dn = (rnd(B, P, C).to(dtype) for _ in range(4))
    w0, w1, b0, b1 = 1 + 0.2 * rnd(C), 1 + 0.2 * rnd(C), 0.1 * rnd(C), 0.1 * rnd(C)
    scale = torch.tensor([1.25, 0.5], device="cuda")
    for kw in (dict(pre=(1, w1, b1)), dict(post=(3, w0, None), gate=rnd(C), pre=(1, w1, b1)),
               dict(post=(1, w0, b0), gate=rnd(B, C), pre=(3, w1, None))):
        kw.update(scale=scale, layout="tokens")
        big = T.residual_norm(x, f, save_stats=True, **kw)
        gb = T.residual_norm_bwd(dy, dn, big.y, f, big.stats, **kw)
        sums, mags = {}, {}
        for p in range(0, P, cut):
            s = slice(p, min(P, p + cut))
            px, pf, pdy, pdn = (t[:, s].contiguous() for t in (x, f, dy, dn))
            r = T.residual_norm(px, pf, save_stats=True, **kw)
            assert torch.equal(r.y, big.y[:, s]) and torch.equal(r.n, big.n[:, s]) and torch.equal(r.stats, big.stats[:, :, s])
            d = T.residual_norm_bwd(pdy, pdn, r.y, pf, r.stats, **kw)
            assert torch.equal(d["dx"], gb["dx"][:, s]) and torch.equal(d["dbranch"], gb["dbranch"][:, s])
            # the magnitudes of the terms, from the gradients as stored (within 2^-8 of what was summed)
            st = r.stats[..., None]
            vh1 = ((r.y.float() - st[2]) * st[3]).abs()
            vh0 = ((pf.float() - st[0]) * st[1]).abs()
            sd = d["dx"].float().abs() * scale[:, None, None]
            m = dict(dpre_w=(pdn.float().abs() * vh1).sum((0, 1)), dpre_b=pdn.float().abs().sum((0, 1)))
            if kw.get("post"):
                gate = kw["gate"].abs()
                per = (sd * vh0).sum(1), sd.sum(1)
                u = per[0] * w0.abs() + (per[1] * b0.abs() if kw["post"][2] is not None else 0)
                m.update(dgate=u if gate.dim() == 2 else u.sum(0), dpost_w=(per[0] * gate).sum(0), dpost_b=(per[1] * gate).sum(0))
            for k, v in d.items():
                if v is not None and k[:4] in ("dpos", "dpre", "dgat"):
                    sums[k], mags[k] = sums.get(k, 0) + v.double(), mags.get(k, 0) + m[k].double()
        for k, v in sums.items():
            tol = (2 * -(-B * P // 256) + 60) * 2.0 ** -24 * mags[k] * 1.02
            assert ((gb[k].double() - v).abs() <= tol).all(), (k, float(((gb[k].double() - v).abs() / tol).max()))
