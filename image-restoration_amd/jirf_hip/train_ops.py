"""Two training operators on torch tensors: the residual join of a block with the norms around it (forward and
backward), and the global gradient norm over many tensors with clipping.  Thin over the C ABI
(jirf_train_residual_norm*, jirf_train_grad_clip*, include/jirf_hip.h), for callers that hold their activations and
gradients as torch tensors; `jirf_hip.train.AstTrainStep` is the whole step for AST.

Everything runs asynchronously on the current stream of the tensors' device and can be captured into a graph (plans are
made outside a capture); workspaces come from torch's allocator per call, so calls on several streams do not share
any.  There is no CPU path and no autograd graph: the backward is called by name, as everywhere in jirf_hip.train.
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
Norm = Tuple[object, torch.Tensor, Optional[torch.Tensor]]


class ResidualNorm(NamedTuple):
    y: torch.Tensor
    n: Optional[torch.Tensor]
    stats: Optional[torch.Tensor]


def _sizes(x: torch.Tensor, layout: str):
    if layout not in LAYOUTS:
        raise ValueError(f"layout {layout!r}: 'planar' ([B, C, ...]) or 'tokens' ([B, P, C])")
    if not x.is_cuda:
        raise ValueError("residual_norm needs GPU tensors: there is no CPU path")
    if x.dtype not in _DTYPES:
        raise ValueError(f"dtype {x.dtype}: only float32, bfloat16 and float16")
    if x.dim() < 3 or (layout == "tokens" and x.dim() != 3):
        raise ValueError(f"{layout} activations are [B, C, ...] / [B, P, C], got shape {tuple(x.shape)}")
    if x.numel() == 0:
        raise ValueError(f"empty activation {tuple(x.shape)}")
    if layout == "planar":
        B, Cn = x.shape[0], x.shape[1]
        return B, Cn, x.numel() // (B * Cn)
    return x.shape[0], x.shape[2], x.shape[1]


def _bs(name: str, t: torch.Tensor, like: torch.Tensor) -> int:
    """Batch stride (0: dense) of an activation that has to match `like`."""
    if t.shape != like.shape or t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{name}: {tuple(t.shape)} {t.dtype} on {t.device}, expected {tuple(like.shape)} {like.dtype} on {like.device}")
    if t.is_contiguous():
        return 0
    if not t[0].is_contiguous():
        raise ValueError(f"{name}: each image has to be contiguous (strides {t.stride()})")
    return t.stride(0)


def _param(name: str, t: torch.Tensor, shape, like: torch.Tensor) -> int:
    if tuple(t.shape) != shape or t.dtype != torch.float32 or t.device != like.device or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous float32 tensor {shape} on {like.device} is needed, got {tuple(t.shape)} {t.dtype} "
                         f"on {t.device}")
    return t.data_ptr()


def _norm(name: str, spec: Optional[Norm], Cn: int, like: torch.Tensor):
    """(kind, weight address, bias address)"""
    if spec is None:
        return 0, None, None
    kind, w, b = spec
    if kind not in NORM_KINDS:
        raise ValueError(f"{name}: norm kind {kind!r}, one of {list(NORM_KINDS)}")
    kind = NORM_KINDS[kind]
    if b is not None and kind != 1:
        raise ValueError(f"{name}: only the WithBias norm takes a bias")
    return kind, _param(name + " weight", w, (Cn,), like), None if b is None else _param(name + " bias", b, (Cn,), like)


def _gate(gate: Optional[torch.Tensor], B: int, Cn: int, like: torch.Tensor):
    if gate is None:
        return 0, None
    if gate.dim() == 1:
        return 1, _param("gate", gate, (Cn,), like)
    return 2, _param("gate", gate, (B, Cn), like)


def _stream(dev: torch.device) -> int:
    return torch.cuda.current_stream(dev).cuda_stream


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
    B, Cn, P = _sizes(x, layout)
    fb = _bs("branch", branch, x)
    k0, w0, b0 = _norm("post", post, Cn, x)
    k1, w1, b1 = _norm("pre", pre, Cn, x)
    gk, gp = _gate(gate, B, Cn, x)
    sp = None if scale is None else _param("scale", scale, (B,), x)
    if norm_out is not None and not k1:
        raise ValueError("norm_out without a pre norm")
    dev = x.device
    with torch.cuda.device(dev):
        y = torch.empty(x.shape, dtype=x.dtype, device=dev) if out is None else out
        n = (torch.empty(x.shape, dtype=x.dtype, device=dev) if norm_out is None else norm_out) if k1 else None
        stats = torch.empty((4, B, P), dtype=torch.float32, device=dev) if save_stats else None
        check(lib().jirf_train_residual_norm(
            x.data_ptr(), _bs("x", x, x), branch.data_ptr(), fb, _DTYPES[x.dtype], LAYOUTS[layout], k0, w0, b0, gk, gp, sp, k1, w1,
            b1, eps, y.data_ptr(), 0 if out is None else _bs("out", y, x), n.data_ptr() if k1 else None,
            0 if norm_out is None else _bs("norm_out", n, x), stats.data_ptr() if save_stats else None, B, Cn, P, _stream(dev)))
    return ResidualNorm(y, n, stats)


def residual_norm_bwd(dy: Optional[torch.Tensor], dn: Optional[torch.Tensor], y: Optional[torch.Tensor],
                      branch: Optional[torch.Tensor], stats: Optional[torch.Tensor], *, post: Optional[Norm] = None,
                      gate: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None, pre: Optional[Norm] = None,
                      layout: str = "planar") -> dict:
    """Gradients of residual_norm: {"dx", "dbranch", "dgate", "dpost_w", "dpost_b", "dpre_w", "dpre_b"}, None where
    there is no such input.  dy: gradient of y (None: zero), dn: gradient of n; y, stats: the forward's; branch: the
    forward's input (needed with a post norm or a gate)."""
    like = dy if dy is not None else dn
    if like is None:
        raise ValueError("residual_norm_bwd: dy or dn is needed")
    B, Cn, P = _sizes(like, layout)
    k0, w0, b0 = _norm("post", post, Cn, like)
    k1, w1, b1 = _norm("pre", pre, Cn, like)
    gk, gp = _gate(gate, B, Cn, like)
    sp = None if scale is None else _param("scale", scale, (B,), like)
    if k1 and (dn is None or y is None):
        raise ValueError("residual_norm_bwd: the pre norm needs dn and y")
    if (k0 or gk) and branch is None:
        raise ValueError("residual_norm_bwd: a post norm or gate needs the branch")
    if (k0 or k1) and stats is None:
        raise ValueError("residual_norm_bwd: a norm needs the forward's stats (save_stats=True)")
    st = None if not (k0 or k1) else _param("stats", stats, (4, B, P), like)
    use_f = bool(k0 or gk)
    dev = like.device
    L = lib()
    with torch.cuda.device(dev):
        dx = torch.empty(like.shape, dtype=like.dtype, device=dev)
        df = torch.empty(like.shape, dtype=like.dtype, device=dev)
        # one allocation for the parameter gradients and the workspace
        new = lambda *s: torch.empty(s, dtype=torch.float32, device=dev)     # noqa: E731
        dgate = None if gk == 0 else (new(Cn) if gk == 1 else new(B, Cn))
        dpost_w, dpost_b = new(Cn) if k0 else None, new(Cn) if b0 is not None else None
        dpre_w, dpre_b = new(Cn) if k1 else None, new(Cn) if b1 is not None else None
        work = new(max(1, L.jirf_train_residual_norm_bwd_work_floats(_DTYPES[like.dtype], LAYOUTS[layout], k0, gk, k1, B, Cn, P)))
        ptr = lambda t: None if t is None else t.data_ptr()                  # noqa: E731
        check(L.jirf_train_residual_norm_bwd(
            ptr(dy), 0 if dy is None else _bs("dy", dy, like), ptr(dn) if k1 else None, _bs("dn", dn, like) if k1 else 0,
            ptr(y) if k1 else None, _bs("y", y, like) if k1 else 0, ptr(branch) if use_f else None,
            _bs("branch", branch, like) if use_f else 0, st, _DTYPES[like.dtype], LAYOUTS[layout], k0, w0, b0, gk, gp, sp, k1, w1,
            dx.data_ptr(), 0, df.data_ptr(), 0, ptr(dpost_w), ptr(dpost_b), ptr(dgate), ptr(dpre_w), ptr(dpre_b), 0,
            work.data_ptr(), B, Cn, P, _stream(dev)))
    return dict(dx=dx, dbranch=df, dgate=dgate, dpost_w=dpost_w, dpost_b=dpost_b, dpre_w=dpre_w, dpre_b=dpre_b)


class GradientClip:
    """The global norm of a fixed list of gradient tensors, and clipping by it.

    tensors: contiguous float32 / bfloat16 / float16 tensors on one GPU, any number of elements (0 too).  out: None to clip
    in place, a list of as many tensors (any of the three types, e.g. slices of a flat float32 buffer), or False for the
    norm alone.  The object keeps the tensors; make a new one when a gradient moves to other memory."""

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
        with torch.cuda.device(self.device):
            stats = torch.empty(3 + self._work, dtype=torch.float64, device=self.device)
            p = stats.data_ptr()
            check(self._lib.jirf_train_grad_clip_run(self._plan, 0 if norm == 2 else 1, max_norm, grad_scale, p, p + 24,
                                                     _stream(self.device)))
        return stats[:3]

    def __del__(self):
        if getattr(self, "_plan", None) is not None:
            self._lib.jirf_train_grad_clip_plan_destroy(self._plan)
            self._plan = None
