"""Group normalisation + activation over channels-last maps: a normalisation whose statistics do not depend on the batch, for training
with few images per GPU, next to the network's BatchNorm + SiLU (ops.bn_act, ops.bn_silu_backward).

    z, saved = group_norm_act(x, groups, weight, bias, act="silu", keep="e4m3")      # x (N, C, *spatial), channels last
    dx, dweight, dbias = group_norm_act_backward(dz, saved)
    layer = GroupNormAct(groups, channels, keep="e4m3")                              # the same as a module, with autograd

`keep` says what the forward leaves for the backward: None (inference: nothing), "x" (the input itself, not copied), or "e4m3" / "int8"
(the input in 8 bits, written in the same pass; act8.py has the form). From the 8-bit form the backward takes the gradient at the values
that were kept, with the forward's mean and rstd; x itself can be freed or overwritten. Statistics are right to f32's rounding for
finite inputs up to half of the type's largest, whatever their spread, and joined in f64 in a fixed order. Types: float32, bfloat16, float16 for x / z / dz / dx; weight and bias are read as float32, their gradients are float32.
"""
import torch
import torch.nn as nn
from torch.autograd import forward_ad

from . import _lib
from ._lib import Y5MError, c_float, c_int, c_int64, c_size_t, c_void_p, register
from .act8 import DTYPES, FORMATS, Act8, empty_rows, new_act8, on_device_of, rows_of, same_device

register("y5m_gn_act_workspace_bytes", c_size_t, [c_int64, c_int64, c_int, c_int])
register("y5m_gn_act_bwd_workspace_bytes", c_size_t, [c_int64, c_int64, c_int, c_int])
register("y5m_gn_act", c_int, [c_void_p, c_int64, c_int64, c_void_p, c_void_p, c_int64, c_int64, c_int, c_int, c_float, c_int, c_void_p, c_int64,
                               c_int64, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_int, c_void_p, c_size_t, c_int, c_void_p])
register("y5m_gn_act_bwd", c_int, [c_void_p, c_int64, c_int64, c_void_p, c_int64, c_int64, c_void_p, c_int, c_void_p, c_int, c_void_p, c_void_p,
                                   c_void_p, c_void_p, c_int64, c_int64, c_int, c_int, c_int, c_void_p, c_int64, c_int64, c_void_p, c_void_p,
                                   c_void_p, c_size_t, c_int, c_void_p])

_ACTS = {None: 0, "none": 0, "silu": 1}


class GroupNormSaved:
    """what a forward leaves for its backward: `kept` (the input tensor or an Act8), `mean`, `rstd` (N, groups) f32 (one tensor, `stat`),
    the parameters"""
    __slots__ = ("kept", "stat", "groups", "act", "weight", "bias")

    @property
    def mean(self):
        return self.stat[0]

    @property
    def rstd(self):
        return self.stat[1]


def _param(t, c, name, x):
    if t is None:
        return None
    if tuple(t.shape) != (c,):
        raise Y5MError(f"{name}: expected ({c},), got {tuple(t.shape)}")
    if not t.dtype.is_floating_point:
        raise Y5MError(f"{name}: a floating-point tensor, got {t.dtype}")
    if t.device != x.device:
        raise Y5MError(f"{name} is on {t.device}, expected {x.device}")
    return t if t.dtype == torch.float32 and t.is_contiguous() else t.detach().float().contiguous()


def _ptr(t):
    return t.data_ptr() if t is not None else None


def group_norm_act(x, groups, weight=None, bias=None, eps=1e-5, act="silu", keep=None):
    """z = act(weight * (x - mean) / sqrt(var + eps) + bias), mean and (biased) variance per sample and group of C / groups
    consecutive channels. Returns (z, saved); saved is None without `keep`. Autograd does not record the call: z carries no gradient,
    group_norm_act_backward(dz, saved) gives them (weight and bias are read again there: change them only behind it). GroupNormAct is
    the form that autograd records."""
    _lib.require_cuda(x)
    n, s, c, sn, sr = rows_of(x, "x")
    if not isinstance(groups, int) or groups < 1 or c % groups:
        raise Y5MError(f"groups = {groups} must divide the {c} channels")
    if act not in _ACTS:
        raise Y5MError(f"act {act!r}: \"silu\" or None")
    if keep == "none":
        keep = None
    if keep is not None and keep != "x" and keep not in FORMATS:
        raise Y5MError(f"keep {keep!r}: None, \"x\" or one of {sorted(FORMATS)}")
    if not eps > 0:
        raise Y5MError(f"eps = {eps} must be positive")
    w, b = _param(weight, c, "weight", x), _param(bias, c, "bias", x)
    L = _lib.lib()
    with on_device_of(x):
        z = empty_rows(x.shape, x.dtype, x.device)
        a = new_act8(x, keep) if keep in FORMATS else None
        # mean, rstd and the workspace in one allocation where nobody keeps the statistics
        ng = n * groups
        wsb, sb = L.y5m_gn_act_workspace_bytes(n, s, c, groups), (8 * ng + 255) // 256 * 256
        if keep is None:
            mem = torch.empty(sb + wsb, dtype=torch.uint8, device=x.device)
            mean, ws = mem.data_ptr(), mem.data_ptr() + sb
        else:
            stat = torch.empty((2, n, groups), dtype=torch.float32, device=x.device)
            mem = torch.empty(wsb, dtype=torch.uint8, device=x.device)
            mean, ws = stat.data_ptr(), mem.data_ptr()
        _lib.check(L.y5m_gn_act(x.data_ptr(), sn, sr, _ptr(w), _ptr(b), n, s, c, groups, eps, _ACTS[act], z.data_ptr(), s * c, c,
                                mean, mean + 4 * ng, a.q.data_ptr() if a else None, a.q.shape[1] if a else 0,
                                a.scale.data_ptr() if a else None, FORMATS[keep] if a else 0, ws, wsb, DTYPES[x.dtype],
                                _lib.stream_ptr()), "y5m_gn_act")
    if keep is None:
        return z, None
    sv = GroupNormSaved()
    sv.kept = a if a else x.detach()
    sv.stat, sv.groups, sv.act, sv.weight, sv.bias = stat, groups, act, w, b
    return z, sv


def group_norm_act_backward(dz, saved):
    """dz (N, C, *spatial), channels last -> dx (dense, channels last, dz's type), dweight, dbias (C,) f32"""
    kept = saved.kept
    a = kept if isinstance(kept, Act8) else None
    ref = a.q if a else kept
    same_device(ref, dz=dz)
    if dz.shape != kept.shape or dz.dtype != kept.dtype:
        raise Y5MError(f"dz: expected {kept.dtype} {tuple(kept.shape)}, got {dz.dtype} {tuple(dz.shape)}")
    n, s, c, dn, dr = rows_of(dz, "dz")
    xn = xr = 0
    if a is None:
        _, _, _, xn, xr = rows_of(kept, "x")
    L = _lib.lib()
    with on_device_of(dz):
        dx = empty_rows(dz.shape, dz.dtype, dz.device)
        grads = torch.empty((2, c), dtype=torch.float32, device=dz.device)
        mean, dgamma = saved.stat.data_ptr(), grads.data_ptr()
        wsb = L.y5m_gn_act_bwd_workspace_bytes(n, s, c, saved.groups)
        ws = torch.empty(wsb, dtype=torch.uint8, device=dz.device)
        _lib.check(L.y5m_gn_act_bwd(dz.data_ptr(), dn, dr, None if a else kept.data_ptr(), xn, xr, a.q.data_ptr() if a else None,
                                    a.q.shape[1] if a else 0, a.scale.data_ptr() if a else None, FORMATS[a.fmt] if a else 0, _ptr(saved.weight),
                                    _ptr(saved.bias), mean, mean + 4 * n * saved.groups, n, s, c, saved.groups, _ACTS[saved.act],
                                    dx.data_ptr(), s * c, c, dgamma, dgamma + 4 * c, ws.data_ptr(), wsb, DTYPES[dz.dtype],
                                    _lib.stream_ptr()), "y5m_gn_act_bwd")
    return (dx, *grads.unbind(0))


class _GroupNormActFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act, keep):
        z, sv = group_norm_act(x, groups, weight, bias, eps, act, keep)
        if isinstance(sv.kept, Act8):
            ctx.save_for_backward(sv.kept.q, sv.kept.scale, sv.stat, weight, bias)
            ctx.act8 = (sv.kept.shape, sv.kept.dtype, sv.kept.fmt)
        else:
            ctx.save_for_backward(x, None, sv.stat, weight, bias)      # (autograd notices if x is overwritten meanwhile)
            ctx.act8 = None
        ctx.meta = (groups, act)
        return z

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dz):
        k, scale, stat, weight, bias = ctx.saved_tensors
        sv = GroupNormSaved()
        sv.kept = Act8(k, scale, *ctx.act8) if ctx.act8 else k
        sv.stat = stat
        sv.groups, sv.act = ctx.meta
        c = sv.kept.shape[1]
        sv.weight, sv.bias = _param(weight, c, "weight", stat), _param(bias, c, "bias", stat)
        try:
            rows_of(dz, "dz")
        except Y5MError:                                       # autograd hands over what the consumer produced: lay it out
            n, _, *sp = dz.shape
            dz = empty_rows(dz.shape, dz.dtype, dz.device).copy_(dz)
        dx, dw, db = group_norm_act_backward(dz, sv)
        return (dx, dw.to(weight.dtype) if weight is not None else None, db.to(bias.dtype) if bias is not None else None, None, None, None, None)


class GroupNormAct(nn.Module):
    """GroupNorm + activation of a channels-last map as one autograd node. `keep` as in group_norm_act ("x", "e4m3", "int8"); in a pass
    that needs no gradient nothing is kept. Parameters have nn.GroupNorm's names and initial values."""

    def __init__(self, groups, channels, eps=1e-5, act="silu", keep="x", affine=True):
        super().__init__()
        if not isinstance(groups, int) or groups < 1 or channels % groups:
            raise Y5MError(f"groups = {groups} must divide the {channels} channels")
        if act not in _ACTS:
            raise Y5MError(f"act {act!r}: \"silu\" or None")
        if keep != "x" and keep not in FORMATS:
            raise Y5MError(f"keep {keep!r}: \"x\" or one of {sorted(FORMATS)}")
        self.groups, self.channels, self.eps, self.act, self.keep = groups, channels, eps, act, keep
        self.weight = nn.Parameter(torch.ones(channels)) if affine else None
        self.bias = nn.Parameter(torch.zeros(channels)) if affine else None

    def forward(self, x):
        needs = torch.is_grad_enabled() and (x.requires_grad or (self.weight is not None and (self.weight.requires_grad or self.bias.requires_grad)))
        if not needs:
            if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in (x, self.weight, self.bias)):
                raise Y5MError("GroupNormAct has no forward-mode derivative: its output would carry no tangent")
            return group_norm_act(x, self.groups, self.weight, self.bias, self.eps, self.act)[0]
        return _GroupNormActFn.apply(x, self.weight, self.bias, self.groups, self.eps, self.act, self.keep)

    def extra_repr(self):
        return f"{self.groups}, {self.channels}, eps={self.eps}, act={self.act!r}, keep={self.keep!r}"
