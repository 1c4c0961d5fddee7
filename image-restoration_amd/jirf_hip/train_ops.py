"""Two training operators on torch tensors: the residual join of a block with the norms around it (forward and
backward), and the global gradient norm over many tensors with clipping.  Thin over the C ABI
(jirf_train_residual_norm*, jirf_train_grad_clip*, include/jirf_hip.h), for callers that hold their activations and
gradients as torch tensors; `jirf_hip.train.AstTrainStep` is the whole step for AST.

Everything runs asynchronously on the current stream of the tensors' device and can be captured into a graph (plans are
made outside a capture); workspaces come from torch's allocator per call, so calls on several streams do not share
any.  There is no CPU path and no autograd graph: the backward is called by name, as everywhere in jirf_hip.train, and tensors
that require gradients are refused except under torch.no_grad().
"""
from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple, Optional, Sequence, Tuple

import torch

from jirf_hip import check, lib

LAYOUTS = {"planar": 0, "tokens": 1}
NORM_KINDS = {"WithBias": 1, "BiasFree": 2, "RMS": 3, 1: 1, 2: 2, 3: 3}
_DTYPES = {torch.float32: 0, torch.bfloat16: 4, torch.float16: 5}
# the current stream's handle without the stream object around it
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else \
    lambda index: torch.cuda.current_stream(index).cuda_stream
Norm = Tuple[object, torch.Tensor, Optional[torch.Tensor]]


class ResidualNorm(NamedTuple):
    y: torch.Tensor
    n: Optional[torch.Tensor]
    stats: Optional[torch.Tensor]


def _sizes(x: torch.Tensor, layout: str):
    """B, C, P, layout tag, dtype tag"""
    lay = LAYOUTS.get(layout)
    if lay is None:
        raise ValueError(f"layout {layout!r}: 'planar' ([B, C, ...]) or 'tokens' ([B, P, C])")
    if not x.is_cuda:
        raise ValueError("residual_norm needs GPU tensors: there is no CPU path")
    dtype = _DTYPES.get(x.dtype)
    if dtype is None:
        raise ValueError(f"dtype {x.dtype}: only float32, bfloat16 and float16")
    shape, n = x.shape, x.numel()
    if len(shape) < 3 or (lay and len(shape) != 3):
        raise ValueError(f"{layout} activations are [B, C, ...] / [B, P, C], got shape {tuple(shape)}")
    if n == 0:
        raise ValueError(f"empty activation {tuple(shape)}")
    B, Cn, P = (shape[0], shape[2], shape[1]) if lay else (shape[0], shape[1], n // (shape[0] * shape[1]))
    if n >> 31 and (B >> 31 or Cn >> 31 or P >> 31):        # a C int would keep the low bits
        raise ValueError(f"{layout} activation {tuple(shape)}: images, channels and pixels have to fit 31 bits each")
    return B, Cn, P, lay, dtype


def _refuse_tracked(name: str):
    if torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, and there is no autograd graph through these operators: detach it, or call "
                         "under torch.no_grad() and take the gradients from the backward by name")


def _bs(name: str, t: torch.Tensor, like: torch.Tensor) -> int:
    """Batch stride (0: dense) of an activation that has to match `like`."""
    if t is not like and (t.shape != like.shape or t.dtype is not like.dtype or t.get_device() != like.get_device()):
        raise ValueError(f"{name}: {tuple(t.shape)} {t.dtype} on {t.device}, expected {tuple(like.shape)} {like.dtype} on {like.device}")
    if t.requires_grad:
        _refuse_tracked(name)
    if t.is_contiguous():
        return 0
    bs = t.stride(0)
    if not t[0].is_contiguous() or bs < t[0].numel():
        raise ValueError(f"{name}: each image has to be contiguous and apart from the others (strides {t.stride()})")
    return bs


def _param(name: str, t: torch.Tensor, shape, like: torch.Tensor) -> int:
    if t.dtype is not torch.float32 or t.shape != shape or t.get_device() != like.get_device() or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous float32 tensor {shape} on {like.device} is needed, got {tuple(t.shape)} {t.dtype} "
                         f"on {t.device}")
    if t.requires_grad:
        _refuse_tracked(name)
    return t.data_ptr()


def _norm(name: str, spec: Optional[Norm], Cn: int, like: torch.Tensor):
    """(kind, weight address, bias address)"""
    if spec is None:
        return 0, None, None
    kind, w, b = spec
    k = NORM_KINDS.get(kind)
    if k is None:
        raise ValueError(f"{name}: norm kind {kind!r}, one of {list(NORM_KINDS)}")
    if b is None:
        return k, _param(name, w, (Cn,), like), None
    if k != 1:
        raise ValueError(f"{name}: only the WithBias norm takes a bias")
    return k, _param(name, w, (Cn,), like), _param(name, b, (Cn,), like)


def _gate(gate: Optional[torch.Tensor], B: int, Cn: int, like: torch.Tensor):
    if gate is None:
        return 0, None
    if gate.dim() == 1:
        return 1, _param("gate", gate, (Cn,), like)
    return 2, _param("gate", gate, (B, Cn), like)


def _new(x: torch.Tensor, dense: bool) -> torch.Tensor:
    return torch.empty_like(x) if dense else x.new_empty(x.shape)


def residual_norm(x: torch.Tensor, branch: torch.Tensor, *, post: Optional[Norm] = None, gate: Optional[torch.Tensor] = None,
                  scale: Optional[torch.Tensor] = None, pre: Optional[Norm] = None, layout: str = "planar", eps: float = 1e-5,
                  save_stats: bool = False, out: Optional[torch.Tensor] = None,
                  norm_out: Optional[torch.Tensor] = None) -> ResidualNorm:
    """y = x + scale[b] * gate * post(branch) and n = pre(y), in one pass.

    x, branch: [B, C, ...] (layout "planar") or [B, P, C] ("tokens"), float32 / bfloat16 / float16, each image
    contiguous.  post, pre: (kind, weight [C], bias [C] or None) with kind "WithBias", "BiasFree" or "RMS" (or 1, 2, 3),
    or None.  gate: [C], [B, C] or None.  scale: [B] (a sample's DropPath factor) or None.  Parameters are float32.
    save_stats: keep what residual_norm_bwd needs ([4, B, P] float32).  out, norm_out: where y and n go (out may be x,
    norm_out may be branch)."""
    B, Cn, P, lay, dtype = _sizes(x, layout)
    index = x.get_device()
    if index != torch.cuda.current_device():
        with torch.cuda.device(x.device):
            return residual_norm(x, branch, post=post, gate=gate, scale=scale, pre=pre, layout=layout, eps=eps,
                                 save_stats=save_stats, out=out, norm_out=norm_out)
    xb, fb = _bs("x", x, x), _bs("branch", branch, x)
    k0, w0, b0 = _norm("post", post, Cn, x)
    k1, w1, b1 = _norm("pre", pre, Cn, x)
    gk, gp = _gate(gate, B, Cn, x)
    sp = None if scale is None else _param("scale", scale, (B,), x)
    if norm_out is not None and not k1:
        raise ValueError("norm_out without a pre norm")
    y = _new(x, xb == 0) if out is None else out
    n = (_new(x, xb == 0) if norm_out is None else norm_out) if k1 else None
    stats = x.new_empty((4, B, P), dtype=torch.float32) if save_stats else None
    check(lib().jirf_train_residual_norm(
        x.data_ptr(), xb, branch.data_ptr(), fb, dtype, lay, k0, w0, b0, gk, gp, sp, k1, w1,
        b1, eps, y.data_ptr(), 0 if out is None else _bs("out", y, x), n.data_ptr() if k1 else None,
        0 if norm_out is None else _bs("norm_out", n, x), stats.data_ptr() if save_stats else None, B, Cn, P,
        _raw_stream(index)))
    return ResidualNorm(y, n, stats)


def residual_norm_bwd(dy: Optional[torch.Tensor], dn: Optional[torch.Tensor], y: Optional[torch.Tensor],
                      branch: Optional[torch.Tensor], stats: Optional[torch.Tensor], *, post: Optional[Norm] = None,
                      gate: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None, pre: Optional[Norm] = None,
                      layout: str = "planar") -> dict:
    """Gradients of residual_norm: {"dx", "dbranch", "dgate", "dpost_w", "dpost_b", "dpre_w", "dpre_b"}, None where
    there is no such input.  dy: gradient of y (None: zero), dn: gradient of n (not read without a pre norm: there is no
    n); y, stats: the forward's; branch: the forward's input (needed with a post norm or a gate).  Without a pre norm dx is
    dy itself, not a copy, and so is dbranch where the branch has no norm, gate or scale either: clone it before adding to
    it in place."""
    like = dy if dy is not None else dn
    if like is None:
        raise ValueError("residual_norm_bwd: dy or dn is needed")
    B, Cn, P, lay, dtype = _sizes(like, layout)
    index = like.get_device()
    if index != torch.cuda.current_device():
        with torch.cuda.device(like.device):
            return residual_norm_bwd(dy, dn, y, branch, stats, post=post, gate=gate, scale=scale, pre=pre, layout=layout)
    k0, w0, b0 = _norm("post", post, Cn, like)
    k1, w1, b1 = _norm("pre", pre, Cn, like)
    gk, gp = _gate(gate, B, Cn, like)
    sp = None if scale is None else _param("scale", scale, (B,), like)
    if k1 and (dn is None or y is None):
        raise ValueError("residual_norm_bwd: the pre norm needs dn and y")
    use_f = k0 or gk
    if use_f and branch is None:
        raise ValueError("residual_norm_bwd: a post norm or gate needs the branch")
    if (k0 or k1) and stats is None:
        raise ValueError("residual_norm_bwd: a norm needs the forward's stats (save_stats=True)")
    if dy is None and not k1:
        raise ValueError("residual_norm_bwd: without a pre norm dy is needed")
    st = _param("stats", stats, (4, B, P), like) if k0 or k1 else None
    if not (k0 or gk or k1 or sp):
        return dict(dx=dy, dbranch=dy, dgate=None, dpost_w=None, dpost_b=None, dpre_w=None, dpre_b=None)
    L = lib()
    dense = like.is_contiguous()
    dx, df = _new(like, dense) if k1 else dy, _new(like, dense)
    # the [C] gradients: rows of one tensor where there are several
    rows = [None] * 5
    wanted = [i for i, on in enumerate((k0, b0 is not None, gk == 1, k1, b1 is not None)) if on]
    if len(wanted) < 3:
        for i in wanted:
            rows[i] = like.new_empty(Cn, dtype=torch.float32)
    else:
        for i, t in zip(wanted, like.new_empty((len(wanted), Cn), dtype=torch.float32).unbind()):
            rows[i] = t
    if gk == 2:
        rows[2] = like.new_empty((B, Cn), dtype=torch.float32)
    need = L.jirf_train_residual_norm_bwd_work_floats(dtype, lay, k0, gk, k1, B, Cn, P)
    work = like.new_empty(max(1, need), dtype=torch.float32)
    p = [None if t is None else t.data_ptr() for t in rows]
    check(L.jirf_train_residual_norm_bwd(
        None if dy is None else dy.data_ptr(), 0 if dy is None else _bs("dy", dy, like), dn.data_ptr() if k1 else None,
        _bs("dn", dn, like) if k1 else 0, y.data_ptr() if k1 else None, _bs("y", y, like) if k1 else 0,
        branch.data_ptr() if use_f else None, _bs("branch", branch, like) if use_f else 0, st, dtype, lay, k0, w0, b0, gk, gp, sp,
        k1, w1, dx.data_ptr() if k1 else None, 0, df.data_ptr(), 0, p[0], p[1], p[2], p[3], p[4], 0, work.data_ptr(), B, Cn, P,
        _raw_stream(index)))
    return dict(dx=dx, dbranch=df, dgate=rows[2], dpost_w=rows[0], dpost_b=rows[1], dpre_w=rows[3], dpre_b=rows[4])


class GradientClip:
    """The global norm of a fixed list of gradient tensors, and clipping by it.

    tensors: contiguous float32 / bfloat16 / float16 tensors on one GPU, any number of elements (0 too).  out: None to clip
    in place, a list of as many tensors (any of the three types, e.g. slices of a flat float32 buffer), or False for the
    norm alone.  The object keeps the tensors; make a new one when a gradient moves to other memory.  It is made and dropped
    outside captures, and kept as long as a graph that holds one of its runs: every replay reads its table."""

    def __init__(self, tensors: Sequence[torch.Tensor], out=None):
        self._plan = None
        tensors = list(tensors)
        if not tensors:
            raise ValueError("GradientClip: no tensors")
        dst = tensors if out is None else None if out is False else list(out)
        if dst is not None and len(dst) != len(tensors):
            raise ValueError(f"GradientClip: {len(tensors)} tensors, {len(dst)} outputs")
        self.device = tensors[0].device
        for t in tensors + (dst or []):
            if not t.is_cuda or t.device != self.device:
                raise ValueError("GradientClip: all tensors on one GPU (there is no CPU path)")
            if t.dtype not in _DTYPES or not t.is_contiguous():
                raise ValueError(f"GradientClip: contiguous float32, bfloat16 or float16 tensors, got {t.dtype} with strides {t.stride()}")
        for t, d in zip(tensors, dst or []):
            if t.numel() != d.numel():
                raise ValueError(f"GradientClip: output of {d.numel()} elements for a gradient of {t.numel()}")
        n = len(tensors)
        self.tensors, self.out = tensors, dst
        self._lib = lib()
        vp, ci = C.c_void_p * n, C.c_int * n
        plan = C.c_void_p()
        with torch.cuda.device(self.device):
            check(self._lib.jirf_train_grad_clip_plan_create(
                n, vp(*[t.data_ptr() for t in tensors]), ci(*[_DTYPES[t.dtype] for t in tensors]),
                None if dst is None else vp(*[t.data_ptr() for t in dst]),
                None if dst is None else ci(*[_DTYPES[t.dtype] for t in dst]),
                (C.c_long * n)(*[t.numel() for t in tensors]), C.byref(plan)))
        self._plan = plan
        self._work = self._lib.jirf_train_grad_clip_work_doubles(plan)

    def run(self, max_norm: float, *, norm: float = 2.0, grad_scale: float = 1.0) -> torch.Tensor:
        """Queues one pass on the current stream and returns a float64 tensor of three on the device: the sum of squares (or
        the maximum) of the gradients as stored, the norm of grad_scale * gradients, and the factor applied,
        grad_scale * min(max_norm / (norm + 1e-6), 1) (max_norm <= 0: grad_scale).  norm: 2 or math.inf."""
        if norm not in (2, math.inf):
            raise ValueError(f"GradientClip: norm {norm}: 2 or inf")
        index = self.device.index
        if index != torch.cuda.current_device():
            with torch.cuda.device(self.device):
                return self.run(max_norm, norm=norm, grad_scale=grad_scale)
        stats = torch.empty(3 + self._work, dtype=torch.float64, device=self.device)
        p = stats.data_ptr()
        check(self._lib.jirf_train_grad_clip_run(self._plan, 0 if norm == 2 else 1, max_norm, grad_scale, p,
                                                 p + 24 if self._work else None, _raw_stream(index)))
        return stats[:3] if self._work else stats

    def __del__(self):
        if getattr(self, "_plan", None) is not None:
            self._lib.jirf_train_grad_clip_plan_destroy(self._plan)
            self._plan = None
