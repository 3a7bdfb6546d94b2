"""Activations kept in 8 bits between a forward pass and its backward: written, read back, and used in a weight gradient.

    kept = act8_store(x, "e4m3")            # x (N, C, *spatial), channels last in memory; f32, bf16 or fp16
    y = act8_load(kept)                     # the values it stands for, x's shape and type
    dw, db = act8_wgrad(dy, kept)           # pointwise convolution: dw (Cout, C), from the 8-bit form directly

Every 32 consecutive channels of a row share one scale 2^e (one byte), e the smallest exponent >= -117 that holds the block's largest
magnitude; the codes are e4m3 (3 mantissa bits: relative error <= 2^-4 down to 2^-13 of the block's maximum) or int8 (absolute error
<= 1/127 of the block's maximum), rounded to nearest even; both where e is above -117. 1 + 1/32 bytes per element. Magnitudes above 1.875 * 2^E (E the largest
exponent of x's type) are held as that value; a block with a NaN or an infinity reads back as NaN throughout.

The rows of a tensor are its positions (n, *spatial), each C consecutive values: torch.channels_last tensors, (N, L, C) token tensors
as x.transpose(1, 2), and channel slices of wider buffers. A tensor laid out otherwise is refused, not copied.
"""
import contextlib
import math

import torch

from . import _lib
from ._lib import Y5MError, c_int, c_int64, c_size_t, c_void_p, register

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}     # Y5M_F32, Y5M_BF16, Y5M_F16
FORMATS = {"e4m3": 1, "int8": 2}                                     # Y5M_KEEP_E4M3, Y5M_KEEP_INT8

register("y5m_act8_store", c_int, [c_void_p, c_int64, c_int64, c_int64, c_int64, c_int, c_void_p, c_int, c_void_p, c_int, c_int, c_void_p])
register("y5m_act8_load", c_int, [c_void_p, c_int, c_void_p, c_int64, c_int, c_void_p, c_int64, c_int, c_int, c_void_p])
register("y5m_act8_wgrad_workspace_bytes", c_size_t, [c_int64, c_int, c_int])
register("y5m_act8_wgrad", c_int, [c_void_p, c_int64, c_int64, c_int64, c_int64, c_int, c_void_p, c_int, c_void_p, c_int, c_int, c_void_p,
                                   c_void_p, c_void_p, c_size_t, c_int, c_void_p])

_HERE = contextlib.nullcontext()


def on_device_of(t):
    """context in which launches go to t's device (its current stream), whatever the current device is"""
    if t.is_cuda and t.get_device() != torch.cuda.current_device():
        return torch.cuda.device(t.device)
    return _HERE


def same_device(first, **others):
    _lib.require_cuda(first, *others.values())
    for name, t in others.items():
        if t is not None and t.device != first.device:
            raise Y5MError(f"{name} is on {t.device}, expected {first.device}")


def rows_of(t, name):
    """(N, S, C, batch stride, row stride) of a channels-last (N, C, *spatial) tensor, strides in elements"""
    if t.dtype not in DTYPES:
        raise Y5MError(f"{name}: float32, bfloat16 or float16, got {t.dtype}")
    shape, st = t.shape, t.stride()
    if len(shape) < 2:
        raise Y5MError(f"{name}: expected (N, C, *spatial), got shape {tuple(shape)}")
    n, c = shape[0], shape[1]
    if c == 0:
        raise Y5MError(f"{name}: no channels")
    if t.numel() == 0:                                               # (strides mean nothing)
        return n, math.prod(shape[2:]), c, 0, c
    s, row, pitch = 1, None, 0
    for d in range(len(shape) - 1, 1, -1):
        size = shape[d]
        s *= size
        if size == 1:
            continue
        if row is None:
            row = st[d]
        elif st[d] != pitch:
            raise Y5MError(f"{name}: the positions must lie at one distance from each other (channels last); strides {tuple(st)} of "
                           f"shape {tuple(shape)}: use .contiguous(memory_format=torch.channels_last)")
        pitch = st[d] * size
    if c > 1 and st[1] != 1:
        raise Y5MError(f"{name}: channels must be the dense dimension (channels last); strides {tuple(st)} of shape {tuple(shape)}: "
                       "use .contiguous(memory_format=torch.channels_last)")
    return n, s, c, st[0], (c if row is None else row)


def empty_rows(shape, dtype, device):
    """an uninitialised (N, C, *spatial) tensor, dense and channels last"""
    c = shape[1]
    st, run = [1] * len(shape), c
    for d in range(len(shape) - 1, 1, -1):
        st[d] = run
        run *= shape[d]
    st[0] = run
    return torch.empty_strided(shape, st, dtype=dtype, device=device)


class Act8:
    """An activation in 8 bits: `q` uint8 (rows, C rounded up to 8) codes, `scale` uint8 (rows, ceil(C / 32)) exponents + 127, the
    `shape` and `dtype` of what was stored, `fmt` "e4m3" or "int8"."""
    __slots__ = ("q", "scale", "shape", "dtype", "fmt")

    def __init__(self, q, scale, shape, dtype, fmt):
        shape = torch.Size(shape)
        if fmt not in FORMATS:
            raise Y5MError(f"8-bit format {fmt!r}: one of {sorted(FORMATS)}")
        if dtype not in DTYPES:
            raise Y5MError(f"dtype {dtype}: float32, bfloat16 or float16")
        if len(shape) < 2 or shape[1] == 0:
            raise Y5MError(f"shape {tuple(shape)}: expected (N, C, *spatial)")
        c = shape[1]
        m = shape.numel() // c
        for name, t, w in (("q", q, -(-c // 8) * 8), ("scale", scale, -(-c // 32))):
            if t.dtype != torch.uint8 or tuple(t.shape) != (m, w) or not t.is_contiguous():
                raise Y5MError(f"{name}: contiguous uint8 of shape {(m, w)}, got {t.dtype} {tuple(t.shape)}")
        if q.device != scale.device:
            raise Y5MError("q and scale are on different devices")
        self.q, self.scale, self.shape, self.dtype, self.fmt = q, scale, shape, dtype, fmt

    @property
    def nbytes(self):
        return self.q.numel() + self.scale.numel()


def new_act8(x, fmt):
    """an Act8 for x whose contents a kernel is about to write"""
    c = x.shape[1]
    m = x.numel() // c
    a = Act8.__new__(Act8)
    a.q = torch.empty((m, -(-c // 8) * 8), dtype=torch.uint8, device=x.device)
    a.scale = torch.empty((m, -(-c // 32)), dtype=torch.uint8, device=x.device)
    a.shape, a.dtype, a.fmt = x.shape, x.dtype, fmt
    return a


def _format(fmt):
    if fmt not in FORMATS:
        raise Y5MError(f"8-bit format {fmt!r}: one of {sorted(FORMATS)}")
    return FORMATS[fmt]


def act8_store(x, fmt="e4m3"):
    """x (N, C, *spatial) -> Act8"""
    f = _format(fmt)
    _lib.require_cuda(x)
    n, s, c, sn, sr = rows_of(x, "x")
    with on_device_of(x):
        a = new_act8(x, fmt)
        _lib.check(_lib.lib().y5m_act8_store(x.data_ptr(), sn, sr, n, s, c, a.q.data_ptr(), a.q.shape[1], a.scale.data_ptr(), f,
                                             DTYPES[x.dtype], _lib.stream_ptr()), "y5m_act8_store")
    return a


def act8_load(kept):
    """the values an Act8 stands for, in the type it was stored from, dense and channels last"""
    _lib.require_cuda(kept.q)
    with on_device_of(kept.q):
        y = empty_rows(kept.shape, kept.dtype, kept.q.device)
        c = kept.shape[1]
        _lib.check(_lib.lib().y5m_act8_load(kept.q.data_ptr(), kept.q.shape[1], kept.scale.data_ptr(), kept.q.shape[0], c, y.data_ptr(), c,
                                            FORMATS[kept.fmt], DTYPES[kept.dtype], _lib.stream_ptr()), "y5m_act8_load")
    return y


def act8_wgrad(dy, kept, bias=False):
    """weight gradient of a pointwise convolution (or linear layer) whose input was kept in 8 bits: dy (N, Cout, *spatial) over the
    same positions, channels last -> dw (Cout, C) f32, db (Cout,) f32 or None. Sums run over the values that were kept, products are
    exact, accumulation is f32 (joined in f64); dy may be of another type than what was stored, and infinite: dw is what the sums are then."""
    same_device(kept.q, dy=dy)
    n, s, cout, dn, dr = rows_of(dy, "dy")
    if dy.shape[0] != kept.shape[0] or dy.shape[2:] != kept.shape[2:]:
        raise Y5MError(f"dy: positions {(dy.shape[0], *dy.shape[2:])}, the kept input has {(kept.shape[0], *kept.shape[2:])}")
    c = kept.shape[1]
    L = _lib.lib()
    with on_device_of(dy):
        dw = torch.empty((cout, c), dtype=torch.float32, device=dy.device)
        db = torch.empty(cout, dtype=torch.float32, device=dy.device) if bias else None
        wsb = L.y5m_act8_wgrad_workspace_bytes(n * s, cout, c)
        ws = torch.empty(wsb, dtype=torch.uint8, device=dy.device)
        _lib.check(L.y5m_act8_wgrad(dy.data_ptr(), dn, dr, n, s, cout, kept.q.data_ptr(), kept.q.shape[1], kept.scale.data_ptr(), c,
                                    FORMATS[kept.fmt], dw.data_ptr(), db.data_ptr() if bias else None, ws.data_ptr(), wsb, DTYPES[dy.dtype],
                                    _lib.stream_ptr()), "y5m_act8_wgrad")
    return dw, db
