"""What the residual norm and the gradient clip refuse, on the host: the library's argument checks return before any
launch, so no GPU is needed (addresses are made up and never read), and the Python layer's raise before the library."""
import ctypes as C
import math

import pytest
import torch

import jirf_hip
from jirf_hip import train_ops as T

A, B_, D, E = (0x1000_0000 * i for i in (1, 2, 3, 4))      # four far apart, aligned addresses
EINVAL = -1


def fwd(**kw):
    a = dict(x=A, x_bs=0, f=B_, f_bs=0, dtype=0, layout=0, post=0, post_w=None, post_b=None, gate_kind=0, gate=None, scale=None,
             pre=0, pre_w=None, pre_b=None, eps=1e-5, y=D, y_bs=0, n=None, n_bs=0, stats=None, B=2, C=8, P=16, stream=None)
    assert not set(kw) - set(a)
    a.update(kw)
    return jirf_hip.lib().jirf_train_residual_norm(*a.values())


def bwd(**kw):
    a = dict(dy=A, dy_bs=0, dn=None, dn_bs=0, y=None, y_bs=0, f=None, f_bs=0, stats=None, dtype=0, layout=0, post=0, post_w=None,
             post_b=None, gate_kind=0, gate=None, scale=None, pre=0, pre_w=None, dx=D, dx_bs=0, df=E, df_bs=0, dpost_w=None,
             dpost_b=None, dgate=None, dpre_w=None, dpre_b=None, accumulate=0, work=None, B=2, C=8, P=16, stream=None)
    assert not set(kw) - set(a)
    a.update(kw)
    return jirf_hip.lib().jirf_train_residual_norm_bwd(*a.values())


BAD_COMMON = [dict(dtype=1), dict(dtype=3), dict(dtype=6), dict(dtype=-1), dict(layout=2), dict(layout=-1), dict(post=4, post_w=A),
              dict(post=-1), dict(pre=4, pre_w=A), dict(gate_kind=3, gate=A), dict(gate_kind=-1), dict(B=0), dict(C=0), dict(P=0),
              dict(B=-1), dict(gate_kind=1), dict(gate_kind=2)]


@pytest.mark.parametrize("kw", BAD_COMMON + [
    dict(x=None), dict(f=None), dict(y=None), dict(post=1), dict(pre=1, n=E), dict(pre=1, pre_w=A), dict(eps=-1.0), dict(eps=math.nan),
    dict(eps=math.inf), dict(x_bs=127), dict(y_bs=-128), dict(f_bs=1), dict(x=A + 2), dict(dtype=4, f=B_ + 1), dict(y=D + 1),
    dict(pre=1, pre_w=A, n=E, n_bs=100), dict(y=A + 64), dict(y=B_), dict(pre=3, pre_w=A, n=D), dict(pre=3, pre_w=A, n=A)])
def test_forward_refuses(kw):
    assert fwd(**kw) == EINVAL and "residual_norm" in jirf_hip.last_error()


@pytest.mark.parametrize("kw", BAD_COMMON + [
    dict(dx=None, pre=1, pre_w=A, dn=B_, y=B_, stats=B_, work=A), dict(df=None), dict(dy=None), dict(pre=1, pre_w=A, y=B_, stats=B_, work=A), dict(pre=1, pre_w=A, dn=B_, stats=B_, work=A),
    dict(pre=1, pre_w=A, dn=B_, y=B_, work=A), dict(pre=1, dn=B_, y=B_, stats=B_, work=A), dict(post=1, post_w=A, stats=B_, work=A),
    dict(gate_kind=1, gate=A, work=A), dict(post=2, post_w=A, f=B_, work=A), dict(dpost_w=A, work=A), dict(dgate=A, work=A),
    dict(dpre_w=A, work=A), dict(dpre_b=A, work=A), dict(post=2, post_w=A, f=B_, stats=B_, dpost_b=A, work=A),
    dict(pre=3, pre_w=A, dn=B_, y=B_, stats=B_, dpre_b=A, work=A), dict(gate_kind=1, gate=A, f=B_, dgate=A), dict(dy_bs=5),
    dict(dx_bs=127), dict(df_bs=-3), dict(dx=D + 1), dict(df=D), dict(dx=A), dict(df=A + 256)])
def test_backward_refuses(kw):
    assert bwd(**kw) == EINVAL and "residual_norm_bwd" in jirf_hip.last_error()


def test_backward_work_size():
    size = jirf_hip.lib().jirf_train_residual_norm_bwd_work_floats
    assert size(0, 0, 1, 2, 1, 2, 64, 1000) > 0
    for bad in ((1, 0, 0, 0, 0, 1, 1, 1), (0, 2, 0, 0, 0, 1, 1, 1), (0, 0, 4, 0, 0, 1, 1, 1), (0, 0, 0, 3, 0, 1, 1, 1),
                (0, 0, 0, 0, 5, 1, 1, 1), (0, 0, 0, 0, 0, 0, 1, 1), (0, 0, 0, 0, 0, 1, -1, 1), (0, 0, 0, 0, 0, 1, 1, 0)):
        assert size(*bad) < 0, bad


def plan(src, sdt, dst, ddt, count, n=None):
    n = len(src) if n is None else n
    k = max(1, len(src))
    out = C.c_void_p()
    rc = jirf_hip.lib().jirf_train_grad_clip_plan_create(
        n, (C.c_void_p * k)(*src), (C.c_int * k)(*sdt), None if dst is None else (C.c_void_p * k)(*dst),
        None if ddt is None else (C.c_int * k)(*ddt), (C.c_long * k)(*count), C.byref(out))
    assert rc != 0 and not out.value
    return rc


@pytest.mark.parametrize("args", [
    ([], [], None, None, []),                                                # no tensors
    ([A], [1], None, None, [4]), ([A], [0], [D], [3], [4]), ([A], [9], None, None, [4]),          # types
    ([None], [0], None, None, [4]), ([A], [0], [None], [0], [4]), ([A], [0], None, None, [-1]),   # addresses, sizes
    ([A], [0], [D], None, [4]),                                              # destinations without types
    ([A + 1], [4], None, None, [4]), ([A + 2], [0], None, None, [4]), ([A], [0], [D + 2], [0], [4]), ([A], [0], [D + 1], [4], [4]),
    ([A, B_], [0, 0], [D, D], [0, 0], [4, 4]), ([A, B_], [0, 0], [D, D + 12], [0, 0], [4, 4]),    # overlapping destinations
    ([A, B_], [0, 0], [D, A], [0, 0], [4, 4]), ([A, A], [0, 0], [A, D], [0, 0], [4, 4]),          # onto another's source
    ([A], [0], [A + 4], [0], [4]), ([A], [0], [A], [4], [4]), ([A, A], [0, 0], [A, A], [0, 0], [4, 4]),   # onto a part of itself
    ([A, D], [0, 0], [B_, E], [0, 0], [0x1000_0000, 4]),                     # a long one across its neighbours
])
def test_clip_plan_refuses(args):
    assert plan(*args) == EINVAL and "grad_clip" in jirf_hip.last_error()


def test_clip_run_refuses_null():
    L = jirf_hip.lib()
    assert L.jirf_train_grad_clip_run(None, 0, 1.0, 1.0, A, A, None) == EINVAL
    assert L.jirf_train_grad_clip_work_doubles(None) < 0
    L.jirf_train_grad_clip_plan_destroy(None)


def test_python_layer_refuses():
    x = torch.zeros(2, 8, 4)
    with pytest.raises(ValueError, match="no CPU path"):
        T.residual_norm(x, x)
    with pytest.raises(ValueError, match="layout"):
        T.residual_norm(x, x, layout="rows")
    with pytest.raises(ValueError, match="dy or dn"):
        T.residual_norm_bwd(None, None, None, None, None)
    with pytest.raises(ValueError, match="no CPU path"):
        T.residual_norm_bwd(x, None, None, None, None)
    with pytest.raises(ValueError, match="no tensors"):
        T.GradientClip([])
    with pytest.raises(ValueError, match="one GPU"):
        T.GradientClip([x])
    with pytest.raises(ValueError, match="2 tensors, 1 outputs"):
        T.GradientClip([x, x], out=[x])


def test_python_layer_refuses_strides():
    """Images that overlap (an expanded batch), or are not contiguous themselves."""
    one = torch.zeros(1, 8, 6)
    like = torch.zeros(3, 8, 6)
    assert T._bs("x", like, like) == 0 and T._bs("x", torch.zeros(3, 16, 6)[:, :8], like) == 96
    for bad in (one.expand(3, 8, 6), torch.zeros(3, 6, 8).transpose(1, 2), torch.zeros(3, 8, 12)[..., ::2],
                torch.zeros(100).as_strided((3, 8, 6), (8, 6, 1))):
        with pytest.raises(ValueError, match="contiguous"):
            T._bs("x", bad, like)
    for bad in (torch.zeros(3, 8, 7), torch.zeros(3, 8, 6, dtype=torch.float16)):
        with pytest.raises(ValueError, match="expected"):
            T._bs("x", bad, like)


def test_python_layer_refuses_parameters():
    like = torch.zeros(3, 8, 6)
    good = torch.zeros(8)
    assert T._norm("pre", ("WithBias", good, good), 8, like)[0] == 1 and T._norm("pre", ("RMS", good, None), 8, like)[0] == 3
    assert T._gate(good, 3, 8, like)[0] == 1 and T._gate(torch.zeros(3, 8), 3, 8, like)[0] == 2 and T._gate(None, 3, 8, like) == (0, None)
    for spec in ((4, good, None), ("LayerNorm", good, None), ("RMS", good, good), (2, good, good), (1, torch.zeros(7), None),
                 (1, good.half(), None), (1, good, torch.zeros(9)), (3, torch.zeros(16)[::2], None)):
        with pytest.raises(ValueError):
            T._norm("pre", spec, 8, like)
    for gate in (torch.zeros(6), torch.zeros(2, 8), torch.zeros(3, 8, 6), good.bfloat16()):
        with pytest.raises(ValueError):
            T._gate(gate, 3, 8, like)


@pytest.mark.parametrize("layout,shape", [("planar", (1, 1, 2**16, 2**16 + 5)), ("planar", (1, 1, 2**31)), ("tokens", (1, 2**32 + 5, 1)),
                                          ("planar", (2**32 + 5, 1, 1)), ("tokens", (1, 1, 2**31))])
def test_sizes_past_31_bits_are_refused_not_cut_off(layout, shape):
    x = torch.empty(shape, dtype=torch.float16, device="meta")

    class OnGpu:
        is_cuda, dtype, numel = True, x.dtype, x.numel
    OnGpu.shape = x.shape
    with pytest.raises(ValueError, match="31 bits"):
        T._sizes(OnGpu, layout)


def test_the_largest_size_of_31_bits_is_taken():
    class OnGpu:
        is_cuda, dtype, shape = True, torch.float16, torch.Size((1, 2, 2**31 - 1))

        @staticmethod
        def numel():
            return 2 * (2**31 - 1)
    assert T._sizes(OnGpu, "planar")[:3] == (1, 2, 2**31 - 1)


MOST_C = 2**31 - 512       # channel indices step by up to 256 past the last channel in 32 bits


@pytest.mark.parametrize("dtype,layout", [(4, 1), (5, 1), (0, 1), (4, 0), (0, 0)])
def test_more_channels_than_an_index_holds_are_refused(dtype, layout):
    """Where (C + 7) / 8 no longer fits 32 bits, a kernel for 32 channels would be chosen; refused from 256 steps before."""
    size = jirf_hip.lib().jirf_train_residual_norm_bwd_work_floats
    for C_ in (MOST_C + 1, 2**31 - 8, 2**31 - 7, 2**31 - 1):
        assert fwd(dtype=dtype, layout=layout, B=1, C=C_, P=1, f=D, y=0x100_0000_0000) == EINVAL, C_
        assert "channels" in jirf_hip.last_error()
        assert bwd(dtype=dtype, layout=layout, B=1, C=C_, P=1, dx=None, df=0x100_0000_0000) == EINVAL, C_
        assert "channels" in jirf_hip.last_error()
        assert size(dtype, layout, 0, 0, 1, 1, C_, 1) < 0, C_
    # the kernel for any number of channels up to there: two row sums per pixel, four rows of partial sums
    for C_ in (16384 + 1, 2**28, 2**30 + 3, MOST_C):
        assert size(dtype, layout, 0, 0, 1, 1, C_, 1) == 2 + 4 * C_, C_


@pytest.mark.parametrize("layout", [0, 1])
def test_parameter_gradients_of_more_channels_than_a_grid_holds_are_refused(layout):
    """The sums over the rows take 64 threads per channel in one grid of fewer than 2^32 threads; without parameter gradients
    there is no such launch."""
    far = 0x100_0000_0000
    for C_ in (2**26 - 15, 2**26, MOST_C):
        kw = dict(layout=layout, pre=2, pre_w=A, dy=None, dn=A, y=B_, stats=D, work=D, dx=far, df=2 * far, dpre_w=E, B=1, C=C_, P=1)
        assert bwd(**kw) == EINVAL and "parameter gradients" in jirf_hip.last_error(), C_
        assert bwd(**dict(kw, pre=0, gate_kind=1, gate=A, f=A, dy=A, dn=None, dx=None, dpre_w=None, dgate=E)) == EINVAL
        assert "parameter gradients" in jirf_hip.last_error(), C_
    if not torch.cuda.is_available():        # nothing to launch on: the arguments themselves are taken
        assert bwd(**dict(kw, dpre_w=None)) != EINVAL
        assert bwd(**dict(kw, C=2**26 - 16)) != EINVAL


def test_a_clip_plan_of_more_elements_than_any_memory_is_refused_before_its_table():
    """2^46 elements would take 2^30 chunks, a table of 25 GB on the host; from 2^26 chunks on they are refused by their
    number, with no table made."""
    import resource
    before = resource.getrusage(resource.RUSAGE_SELF).ru_maxrss
    for src, count in (([A], [2**42]), ([A], [2**46]), ([A, A], [2**45, 2**45]), ([A], [2**62]), ([A] * 3, [2**45, 1, 2**45])):
        assert plan(src, [0] * len(src), None, None, count) == EINVAL and "grad_clip" in jirf_hip.last_error()
    assert resource.getrusage(resource.RUSAGE_SELF).ru_maxrss - before < 1 << 20        # (KiB)


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: only where there is nothing to launch on")
@pytest.mark.parametrize("dtype", [0, 4, 5])
@pytest.mark.parametrize("layout", [0, 1])
def test_every_size_has_a_kernel(dtype, layout):
    """Sizes on both sides of every choice of form: the arguments are taken and a kernel is found for them (the launch itself
    fails, without a device).  A form without a kernel is an error, never a call that does nothing."""
    Cs = sorted({c + d for c in (1, 4, 8, 16, 32, 64, 128, 256, 512, 1024, 2048, 4096, 8192, 16384) for d in (-1, 0, 1) if c + d > 0})
    for C_ in Cs:
        for P in (1, 2, 3, 4, 5, 7, 8, 9, 16, 31, 33, 64, 130, 1000, 8200, 300_001):
            for B in (1, 3, 300):
                b = dict(dtype=dtype, layout=layout, B=B, C=C_, P=P)
                far = dict(x=1 << 44, f=2 << 44, y=3 << 44)
                assert fwd(**b, **far) != EINVAL, (b, jirf_hip.last_error())
                far = dict(dy=1 << 44, f=2 << 44, dx=3 << 44, df=4 << 44)
                for gate in ({}, dict(gate_kind=1, gate=A), dict(gate_kind=2, gate=A)):
                    assert bwd(**b, **far, **gate) != EINVAL, (b, gate, jirf_hip.last_error())


def test_python_layer_refuses_tensors_of_an_autograd_graph():
    """There is no graph through these operators: outputs of tracked inputs would be cut off from it without a word."""
    like = torch.zeros(3, 8, 6)
    tracked, w = torch.zeros(3, 8, 6, requires_grad=True), torch.zeros(8, requires_grad=True)
    calls = [lambda: T._bs("x", tracked, tracked), lambda: T._bs("branch", tracked * 2, like), lambda: T._gate(w, 3, 8, like),
             lambda: T._gate(torch.zeros(3, 8, requires_grad=True), 3, 8, like), lambda: T._norm("pre", (1, w, None), 8, like),
             lambda: T._norm("post", (1, torch.zeros(8), w), 8, like), lambda: T._param("scale", torch.zeros(3, requires_grad=True), (3,), like)]
    for call in calls:
        with pytest.raises(ValueError, match="no autograd graph"):
            call()
        with torch.no_grad():
            call()
    assert T._bs("x", tracked.detach(), like) == 0
