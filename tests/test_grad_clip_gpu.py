"""The global gradient norm over many tensors and clipping by it, through the C ABI, against 64 bits.

Bounds: squares and sums are 64-bit, a chain of fewer than 2^20 roundings, so the norm is within 2^-33 of the value;
the stored gradient is g * fl32(k) in fp32, rounded once more to the output's type: three roundings of 2^-24 and half a
step of the type."""
import math

import numpy as np
import pytest
import torch

import jirf_hip
from jirf_hip import train_ops as T
from tests.gpu_util import call, ptr, stream

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 2.0 ** -150, BF16: 2.0 ** -134, F16: 2.0 ** -25}      # half the smallest step


def grads(sizes, dtypes, seed=0, scale=1e-2):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * scale * 10.0 ** (-2 * float(torch.rand(1, generator=g)))).to(dtypes[i % len(dtypes)]).cuda()
            for i, n in enumerate(sizes)]


def reference(ts, max_norm, norm, grad_scale):
    flat = torch.cat([t.detach().double().cpu().reshape(-1) for t in ts])
    raw = float(flat.square().sum()) if norm == 2 else (float(flat.abs().max()) if flat.numel() else 0.0)
    total = grad_scale * (math.sqrt(raw) if norm == 2 else raw)
    k = grad_scale * (min(max_norm / (total + 1e-6), 1.0) if max_norm > 0 else 1.0)
    return raw, total, k


def check_out(out, src, k):
    for i, (o, s) in enumerate(zip(out, src)):
        want = s.double() * k
        tol = want.abs() * (HALF[o.dtype] + 3 * 2.0 ** -24) * (1 + 2.0 ** -7) + TINY[o.dtype] + 2.0 ** -149
        bad = ~((o.double() - want).abs() <= tol)
        assert not bad.any(), f"tensor {i} ({s.dtype} -> {o.dtype}, {s.numel()}): {int(bad.sum())} outside the bound"


def check_stats(stats, want, exact):
    got = stats.cpu().numpy()
    if exact:
        assert got[0] == want[0] and got[1] == want[1]
    assert np.all(np.abs(got - np.array(want)) <= 2.0 ** -33 * np.abs(want)), (got, want)


SIZES = {
    "one value": [1],
    "small": [3, 1, 0, 48, 7, 4096, 2048, 2047, 2049, 33],
    "a network": [27 * 32, 32, 9216, 3, 1, 225 * 16, 2, 262144, 512, 65537, 1_000_003, 8191],
    "one large": [5_000_011],
    "many": [1 + (i * 37) % 301 for i in range(1500)],
}


@pytest.mark.parametrize("norm", [2, math.inf])
@pytest.mark.parametrize("name", list(SIZES))
@pytest.mark.parametrize("types", [[F32], [BF16], [F16], [BF16, F32, F16]])
def test_sizes_and_types(name, types, norm):
    src = grads(SIZES[name], types, seed=1)
    want = reference(src, 0.01, norm, 0.125)
    flat = torch.full((sum(SIZES[name]) + 2,), 7.0, device="cuda")
    out = list(flat[1:-1].split(SIZES[name]))                        # packed tight: any alignment of four bytes
    keep = [t.clone() for t in src]
    stats = T.GradientClip(src, out=out).run(0.01, norm=norm, grad_scale=0.125)
    check_stats(stats, want, norm == math.inf)
    check_out(out, src, float(stats[2]))
    assert flat[0] == 7 and flat[-1] == 7 and all(torch.equal(a, b) for a, b in zip(src, keep))
    # in place, and the norm alone
    assert torch.equal(T.GradientClip(src, out=False).run(0.01, norm=norm, grad_scale=0.125), stats)
    assert all(torch.equal(a, b) for a, b in zip(src, keep))
    again = T.GradientClip(src).run(0.01, norm=norm, grad_scale=0.125)
    assert torch.equal(again, stats)
    check_out(src, keep, float(stats[2]))


@pytest.mark.parametrize("src_t", [F32, BF16, F16])
@pytest.mark.parametrize("dst_t", [F32, BF16, F16])
@pytest.mark.parametrize("off_s,off_d", [(0, 0), (1, 0), (0, 3), (5, 2)])
def test_every_pair_of_types_at_any_alignment(src_t, dst_t, off_s, off_d):
    g = torch.Generator().manual_seed(2)
    n = 70_001
    src = torch.randn(n + off_s, generator=g).to(src_t).cuda()[off_s:]
    buf = torch.full((n + off_d + 3,), 7.0, dtype=dst_t, device="cuda")
    dst = buf[off_d:off_d + n]
    stats = T.GradientClip([src], out=[dst]).run(1.5)
    check_stats(stats, reference([src], 1.5, 2, 1.0), False)
    check_out([dst], [src], float(stats[2]))
    assert (buf[:off_d] == 7).all() and (buf[off_d + n:] == 7).all()


def test_no_clipping_leaves_every_bit():
    """Below the limit, in place with factor 1, and into the flat buffer; max_norm <= 0 clips nothing."""
    src = grads([1000, 77, 300_000], [F32, BF16, F16], seed=3)
    keep = [t.clone() for t in src]
    flat = torch.empty(301_077, device="cuda")
    for max_norm in (1e9, 0.0, -1.0, math.inf):
        stats = T.GradientClip(src).run(max_norm)
        assert float(stats[2]) == 1.0
        assert all(torch.equal(a, b) for a, b in zip(src, keep))
        flat.fill_(7.0)
        T.GradientClip(src, out=list(flat.split([1000, 77, 300_000]))).run(max_norm)
        assert torch.equal(flat, torch.cat([k.float() for k in keep]))


def test_all_zero_and_no_elements():
    z = [torch.zeros(5000, device="cuda"), torch.zeros(3, dtype=BF16, device="cuda")]
    for norm in (2, math.inf):
        s = T.GradientClip(z).run(0.01, norm=norm)
        assert s.tolist() == [0.0, 0.0, 1.0] and not z[0].any()
        e = T.GradientClip([torch.empty(0, device="cuda"), torch.empty(0, dtype=F16, device="cuda")]).run(0.01, norm=norm, grad_scale=0.5)
        assert e.tolist() == [0.0, 0.0, 0.5]


@pytest.mark.parametrize("norm", [2, math.inf])
@pytest.mark.parametrize("where", [0, 70_000, 2_000_000])
def test_not_a_number_and_infinity(norm, where):
    n = 2_000_001
    for v, total in ((float("nan"), float("nan")), (float("inf"), float("inf")), (float("-inf"), float("inf"))):
        src = [torch.ones(17, device="cuda"), torch.full((n,), 0.5, device="cuda")]
        src[1][where] = v
        s = T.GradientClip(src).run(0.01, norm=norm).cpu()
        if math.isnan(total):
            assert torch.isnan(s).all() and torch.isnan(src[0]).all() and torch.isnan(src[1]).all()
        else:
            assert s[1] == total and s[2] == 0 and not src[0].any()
            assert torch.isnan(src[1][where]) and int(torch.isnan(src[1]).sum()) == 1 and int((src[1] == 0).sum()) == n - 1


def test_values_whose_squares_overflow_32_bits():
    src = [torch.full((1000,), 3e30, device="cuda"), torch.full((1000,), 1e-30, device="cuda")]
    want = reference(src, 1.0, 2, 1.0)
    s = T.GradientClip(src).run(1.0)
    check_stats(s, want, False)
    assert abs(float(src[0].double().square().sum().sqrt()) - 1.0) < 1e-6


def test_small_tensors_beside_a_large_one():
    """Summed in 32 bits the small tensor would vanish: (2^12)^2 * 2^24 + 2^-8."""
    src = [torch.full((1 << 24,), 4096.0, device="cuda"), torch.full((1,), 0.0625, device="cuda")]
    s = T.GradientClip(src, out=False).run(0.0)
    assert float(s[0]) == 4096.0 ** 2 * 2 ** 24 + 0.0625 ** 2


def test_a_tensor_listed_twice_counts_twice():
    t = torch.full((300,), 2.0, device="cuda")
    out = [torch.empty(300, device="cuda"), torch.empty(300, dtype=BF16, device="cuda")]
    s = T.GradientClip([t, t], out=out).run(0.0)
    assert float(s[0]) == 2 * 300 * 4.0 and (out[0] == 2).all() and (out[1] == 2).all()
    with pytest.raises(jirf_hip.JirfError, match="overlaps"):
        T.GradientClip([t, t])


def test_many_workgroups_and_past_32_bits():
    """2.2 G bf16 values, more than 2^31 elements and 2^32 bytes in one tensor."""
    n = 2_200_000_007
    t = torch.zeros(n, dtype=BF16, device="cuda")
    t[-3:] = torch.tensor([3.0, 4.0, 12.0]).to(BF16)
    t[n // 2] = 84.0
    s = T.GradientClip([t]).run(8.5)
    assert float(s[0]) == 169.0 + 84.0 ** 2 and float(s[1]) == 85.0
    k = float(s[2])
    assert abs(k - 0.1) < 1e-8
    check_out([t[-3:], t[n // 2: n // 2 + 1]], [torch.tensor([3.0, 4.0, 12.0]).cuda(), torch.tensor([84.0]).cuda()], k)


def test_the_clipped_buffer_feeds_the_adam_step():
    """The flat buffer and stats[0] in the places of jirf_train_sumsq's: the same update as from a flat gradient."""
    sizes = [4096, 77, 30_000]
    src = grads(sizes, [F32], seed=6)
    n = sum(sizes)
    flat = torch.empty(n, device="cuda")
    stats = T.GradientClip(src, out=list(flat.split(sizes))).run(0.0)          # gathered, not yet clipped
    ss = torch.zeros(1, dtype=torch.float64, device="cuda")
    call("jirf_train_sumsq", ptr(flat), n, ptr(ss), None, stream())
    assert abs(float(stats[0]) - float(ss)) <= 2.0 ** -33 * float(ss)
    outs = []
    for sumsq in (stats, ss):
        p, m, v = (torch.zeros(n, device="cuda") for _ in range(3))
        call("jirf_train_adam_step", ptr(p), ptr(flat), ptr(m), ptr(v), n, ptr(sumsq), 0.01, 1.0, 2e-4, 0.9, 0.999, 1e-8, 1, 0, stream())
        outs.append(p)
    assert torch.allclose(outs[0], outs[1], rtol=1e-5, atol=0)
    # clipped here, or there: one rounding of each gradient and of the factor apart
    clipped = torch.empty(n, device="cuda")
    T.GradientClip(src, out=list(clipped.split(sizes))).run(0.01)
    p, m, v = (torch.zeros(n, device="cuda") for _ in range(3))
    call("jirf_train_adam_step", ptr(p), ptr(clipped), ptr(m), ptr(v), n, None, 0.0, 1.0, 2e-4, 0.9, 0.999, 1e-8, 1, 0, stream())
    assert torch.allclose(p, outs[1], rtol=1e-4, atol=0)


def test_captured_and_replayed_and_on_two_streams():
    src = grads([70_000, 13, 500_000], [F32, BF16], seed=7)
    flat = [torch.empty(570_013, device="cuda") for _ in range(2)]
    plans = [T.GradientClip(src, out=list(f.split([70_000, 13, 500_000]))) for f in flat]
    plans[0].run(0.01)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        stats = plans[0].run(0.01, grad_scale=0.5)
    for i in range(4):
        for t in src:
            t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        eager = plans[1].run(0.01, grad_scale=0.5)
        torch.cuda.synchronize()
        assert torch.equal(stats, eager) and torch.equal(flat[0], flat[1])
    # one plan on two streams at once: the runs share no workspace
    streams = [torch.cuda.Stream() for _ in range(2)]
    want = plans[0].run(0.01).clone()
    norm_only = T.GradientClip(src, out=False)
    torch.cuda.synchronize()
    got = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            got.append(norm_only.run(0.01))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("types", [[F32], [BF16], [BF16, F32]])
@pytest.mark.parametrize("sizes,value,max_norm", [([5], 1e38, 0.01), ([100, 3], 1e38, 1e-4), ([300_001, 7], 1e38, 0.01),
                                                  ([1_000_003, 17], 3e38, 0.01), ([1_000_003, 17], 3e38, 1e-7), ([40], 3e38, 1e-12)])
def test_factors_below_the_normal_range_of_32_bits(types, sizes, value, max_norm):
    """Gradients so large that the factor is far below 2^-126: it keeps its digits, into fp32 and in place.  The
    factor's leading digits and the product are rounded to 24 digits each and scaled by a power of two (half a smallest step
    where that leaves the normal range), so the bound of the other tests holds."""
    src = [(torch.arange(n, device="cuda") % 7 - 3.0).div_(3.0).mul_(value).to(types[i % len(types)]) for i, n in enumerate(sizes)]
    src[0][0] = value                                                                   # (never all zero)
    keep = [t.clone() for t in src]
    for norm in (2, math.inf):
        want = reference(keep, max_norm, norm, 1.0)
        assert 0 < want[2] < 2.0 ** -126
        out = [torch.empty(n, device="cuda") for n in sizes]
        stats = T.GradientClip(src, out=out).run(max_norm, norm=norm)
        check_stats(stats, want, norm == math.inf)
        check_out(out, keep, want[2])
    T.GradientClip(src).run(max_norm)
    check_out(src, keep, reference(keep, max_norm, 2, 1.0)[2])


@pytest.mark.parametrize("sizes", [[11], [300_001, 7]])
@pytest.mark.parametrize("value,grad_scale", [(1e-30, 2.0 ** 160), (2.0 ** -149, 2.0 ** 200), (3e38, 2.0 ** -200), (1.0, 1e-60), (3e38, 2.0 ** -270),
                                              (2.0 ** -120, 3e70)])
def test_scales_outside_the_range_of_32_bits(sizes, value, grad_scale):
    """grad_scale may be any positive finite number of 64 bits; the scaled gradients are what 64 bits give, rounded to fp32."""
    src = [torch.full((n,), value, device="cuda") for n in sizes]
    out = [torch.empty(n, device="cuda") for n in sizes]
    stats = T.GradientClip(src, out=out).run(0.0, grad_scale=grad_scale)
    assert float(stats[2]) == grad_scale
    check_out(out, src, grad_scale)
