"""Activations kept in 8 bits (yolov5m_amd/act8.py): the stored form and its read-back bit for bit against the definition in 64 bits,
the weight gradient against a 64-bit product of the same values. tests/test_emu_act8.py runs the same functions on the CPU executor."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U = 2.0 ** -24                                  # half a step of f32, relative


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def rows_tensor(shape, dtype, seed, scale=1.0, offset=0.0):
    """random (N, C, *spatial), channels last, with channels of different spread"""
    n, c, *sp = shape
    g = _gen(seed)
    x = torch.randn((n, *sp, c), generator=g) * torch.exp(0.7 * torch.randn(c, generator=g)) * scale + offset * torch.randn(c, generator=g)
    return x.to(DT[dtype]).movedim(-1, 1).to(DEV)


def stored_values(x, fmt):
    """definition in 64 bits, by channels-last rows: (N, *spatial, C) values and (N, *spatial, blocks) exponents"""
    limit = 1.875 * 2.0 ** (15 if x.dtype == torch.float16 else 127)
    top = 448.0 if fmt == "e4m3" else 127.0
    v = x.detach().cpu().movedim(1, -1).double()
    out, exps = [], []
    for c0 in range(0, v.shape[-1], 32):
        b = v[..., c0:c0 + 32]
        bad = ~torch.isfinite(b).all(-1, keepdim=True)
        b = torch.nan_to_num(b, nan=0.0).clamp(-limit, limit)
        big = b.abs().amax(-1, keepdim=True)
        e = torch.full_like(big, -117.0)
        for t in range(-116, 122):
            e = torch.where(big > top * 2.0 ** (t - 1), torch.full_like(e, float(t)), e)
        s = torch.exp2(e)
        q = b / s
        if fmt == "e4m3":
            step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
            q = torch.round(q / step) * step
        else:
            q = torch.round(q)
        out.append(torch.where(bad, torch.full_like(q, float("nan")), q * s))
        exps.append(torch.where(bad, torch.full_like(e, 128.0), e))
    return torch.cat(out, -1), torch.cat(exps, -1)


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0))


SHAPES = [(1, 1, 1, 1), (1, 8, 1, 1), (2, 32, 3, 5), (3, 33, 7, 1), (2, 100, 4, 4), (1, 255, 2, 3), (5, 3, 3, 3), (2, 48, 5, 9), (2, 96, 17), (4, 64),
          (1, 2056, 2, 2), (0, 16, 4, 4), (2, 16, 0, 4)]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_stored_form_is_the_definition(shape, dtype, fmt):
    from yolov5m_amd.act8 import act8_load, act8_store
    x = rows_tensor(shape, dtype, 1)
    a = act8_store(x, fmt)
    y = act8_load(a)
    val, ex = stored_values(x, fmt)
    assert y.shape == x.shape and y.dtype == x.dtype and same(y.cpu().movedim(1, -1).double(), val.to(DT[dtype]).double())
    # the codes and scales themselves, and the zero padding of a row's last piece
    c, m = shape[1], x.numel() // shape[1]
    assert torch.equal(a.scale.cpu().double() - 127, ex.reshape(m, ex.shape[-1]))
    q = a.q.cpu()
    code = q[:, :c].view(torch.int8).double() if fmt == "int8" else q[:, :c].view(torch.float8_e4m3fn).double()
    s = torch.exp2(a.scale.cpu().double() - 127).repeat_interleave(32, 1)[:, :c]
    assert same(code * s, val.reshape(m, c)) and not q[:, c:].any()
    assert a.nbytes == a.q.numel() + a.scale.numel()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "fp16"])
def test_special_values(dtype, fmt):
    """zeros, the smallest subnormal, the largest value, signed zero, the borders between two exponents, and blocks that are not finite"""
    from yolov5m_amd.act8 import act8_load, act8_store
    t = DT[dtype]
    fi = torch.finfo(t)
    x = torch.zeros(10, 64, dtype=t)
    x[1, 0] = fi.smallest_normal * 2.0 ** -5
    x[2, :3] = torch.tensor([fi.max, -fi.max, fi.max / 2], dtype=t)
    x[3, 5] = -0.0
    top = 448.0 if fmt == "e4m3" else 127.0
    x[4, :4] = torch.tensor([top, top / 2, -top, 1.0], dtype=t)                    # exactly the top: scale 1
    x[5, :4] = torch.tensor([top * 1.01, 1.0, -3.0, 0.3], dtype=t)                 # just above: scale 2
    x[6, 40] = float("inf")
    x[6, 3] = 2.0
    x[7, 1] = float("nan")
    x[7, 35] = -1.0
    x[8, 31] = float("-inf")
    x[8, 32] = 5.0
    x[9] = torch.linspace(-3, 3, 64).to(t)
    xd = x.to(DEV)
    a = act8_store(xd, fmt)
    y = act8_load(a).cpu().double()
    val, ex = stored_values(xd, fmt)
    assert same(y, val.to(t).double())
    assert torch.isfinite(y[2]).all() and float(y[2, 0]) >= 0.93 * float(fi.max)
    assert torch.isnan(y[6, 32:]).all() and torch.isfinite(y[6, :32]).all()
    assert torch.isnan(y[7, :32]).all() and float(y[7, 35]) == -1.0
    assert int(a.scale[4, 0]) == 127 and int(a.scale[5, 0]) == 128 and int(a.scale[7, 0]) == 255


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_views_of_wider_buffers_and_token_tensors(dtype):
    """a channel slice, a slice that starts off a 16-byte border, (N, L, C) tokens, every second image, a broadcast image"""
    from yolov5m_amd.act8 import act8_load, act8_store
    wide = rows_tensor((4, 128, 5, 6), dtype, 2)
    tokens = torch.randn(3, 11, 40, generator=_gen(3)).to(DT[dtype]).to(DEV)
    for x in (wide[:, 32:96], wide[:, 3:72], wide[::2], wide[:1].expand(3, -1, -1, -1), tokens.transpose(1, 2), wide[:, :, 1:4], wide[:, :, :, 2:3], wide[..., ::2]):
        for fmt in ("e4m3", "int8"):
            y = act8_load(act8_store(x, fmt))
            assert same(y.cpu().movedim(1, -1).double(), stored_values(x, fmt)[0].to(DT[dtype]).double())


def test_offsets_beyond_32_bits():
    """rows whose element offsets pass 2^31 in the source (a broadcast of one buffer with a large batch stride costs no memory to check)"""
    if DEV != "cuda":
        pytest.skip("a 5 GiB buffer")
    from yolov5m_amd.act8 import act8_load, act8_store
    base = torch.zeros(2 ** 31 + 4096, dtype=torch.bfloat16, device=DEV)
    base[2 ** 31 + 64:2 ** 31 + 64 + 320] = torch.randn(320, device=DEV)
    base[:320] = torch.randn(320, device=DEV)
    x = base.as_strided((2, 32, 10), (2 ** 31 + 64, 1, 32))
    y = act8_load(act8_store(x, "int8"))
    assert same(y.cpu().movedim(1, -1).double(), stored_values(x, "int8")[0].bfloat16().double())


# ---- the weight gradient -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "fp16"])
@pytest.mark.parametrize("case", [(1, 8, 8, (1, 1)), (1, 1, 1, (3,)), (2, 48, 96, (7, 9)), (3, 100, 255, (5, 4)), (2, 130, 129, (8, 8)), (1, 33, 7, (1, 1)),
                                  (5, 16, 200, (13, 3)), (1, 256, 128, (300,)), (4, 300, 20, (5, 7)), (0, 8, 8, (2, 2))])
def test_wgrad_is_the_product_of_the_kept_values(case, dtype, fmt):
    """dw = dy^T x8, db = sum dy against float64. Products are exact, sums f32 per row range: a chain of at most (rows of a range) / 32
    matrix instructions of 32 products each plus the final rounding; ranges here are below 2048 rows, so at most 64 + 32 roundings of
    partial sums that are each at most the sum of magnitudes: |err| <= 96 u sum |dy| |x|. For db: chains of at most 2048 / 16 rows a
    thread + 16 threads."""
    from yolov5m_amd.act8 import act8_load, act8_store, act8_wgrad
    n, c, cout, sp = case
    x = rows_tensor((n, c, *sp), "bf16" if dtype == "bf16" else "f32", 4)
    dy = rows_tensor((n, cout, *sp), dtype, 5, scale=0.1, offset=0.02)
    kept = act8_store(x, fmt)
    dw, db = act8_wgrad(dy, kept, bias=True)
    xv = act8_load(kept).cpu().double().movedim(1, -1).reshape(-1, c)
    dv = dy.cpu().double().movedim(1, -1).reshape(-1, cout)
    assert dw.dtype == torch.float32 and tuple(dw.shape) == (cout, c) and tuple(db.shape) == (cout,)
    assert ((dw.cpu().double() - dv.t() @ xv).abs() <= 96 * U * (dv.abs().t() @ xv.abs())).all()
    assert ((db.cpu().double() - dv.sum(0)).abs() <= 160 * U * dv.abs().sum(0)).all()
    dw2, none = act8_wgrad(dy, kept)
    assert none is None and torch.equal(dw, dw2)                       # one result per input


def test_wgrad_long_sum_and_strided_gradient():
    """a range of rows per workgroup and their join; dy a channel slice of a wider buffer"""
    from yolov5m_amd.act8 import act8_load, act8_store, act8_wgrad
    rows = 40000 if DEV == "cuda" else 3000
    x = rows_tensor((2, 24, rows // 2), "bf16", 6)
    wide = rows_tensor((2, 64, rows // 2), "bf16", 7)
    kept = act8_store(x, "e4m3")
    xv = act8_load(kept).cpu().double().movedim(1, -1).reshape(-1, 24)
    for dy in (wide[:, 16:56], wide[:, 5:50]):
        dw, db = act8_wgrad(dy, kept, bias=True)
        dv = dy.cpu().double().movedim(1, -1).reshape(rows, -1)
        assert ((dw.cpu().double() - dv.t() @ xv).abs() <= 96 * U * (dv.abs().t() @ xv.abs())).all()
        assert ((db.cpu().double() - dv.sum(0)).abs() <= 160 * U * dv.abs().sum(0)).all()


def test_wgrad_nan_block_reaches_the_gradient_and_nothing_else():
    from yolov5m_amd.act8 import act8_store, act8_wgrad
    x = rows_tensor((1, 96, 5, 5), "bf16", 8)
    x[0, 40, 2, 2] = float("inf")
    dy = rows_tensor((1, 16, 5, 5), "bf16", 9)
    dw, _ = act8_wgrad(dy, act8_store(x, "int8"))
    assert torch.isnan(dw[:, 32:64]).all() and torch.isfinite(dw[:, :32]).all() and torch.isfinite(dw[:, 64:]).all()


def test_refusals():
    from yolov5m_amd._lib import Y5MError
    from yolov5m_amd.act8 import Act8, act8_load, act8_store, act8_wgrad
    x = rows_tensor((2, 16, 4, 4), "f32", 10)
    with pytest.raises(Y5MError, match="8-bit format"):
        act8_store(x, "fp8")
    with pytest.raises(Y5MError, match="channels last"):
        act8_store(x.contiguous())
    with pytest.raises(Y5MError, match="channels last"):
        act8_store(x[..., :3])                              # three of four columns: rows at two distances
    with pytest.raises(Y5MError, match="float32"):
        act8_store(x.double())
    with pytest.raises(Y5MError, match="no channels"):
        act8_store(x[:, :0])
    with pytest.raises(Y5MError, match=r"\(N, C"):
        act8_store(x[0, 0, 0])
    k = act8_store(x)
    with pytest.raises(Y5MError, match="positions"):
        act8_wgrad(rows_tensor((2, 16, 4, 5), "f32", 11), k)
    with pytest.raises(Y5MError, match="channels last"):
        act8_wgrad(x.contiguous(), k)
    with pytest.raises(Y5MError, match="scale"):
        Act8(k.q, k.scale[:-1], k.shape, k.dtype, k.fmt)
    with pytest.raises(Y5MError, match="q"):
        Act8(k.q[:, :8], k.scale, k.shape, k.dtype, k.fmt)
    with pytest.raises(Y5MError, match="format"):
        Act8(k.q, k.scale, k.shape, k.dtype, "int4")
    assert torch.equal(act8_load(Act8(k.q, k.scale, k.shape, k.dtype, k.fmt)), act8_load(k))


def test_c_entry_refuses_what_it_cannot_run():
    """argument checks of the C entry points return an error code, launch nothing and leave the outputs alone"""
    from yolov5m_amd import _lib
    import yolov5m_amd.act8  # noqa: F401
    L = _lib.lib()
    x = rows_tensor((1, 16, 2, 2), "f32", 12)
    q = torch.full((4, 16), 7, dtype=torch.uint8, device=DEV)
    s = torch.full((4, 1), 7, dtype=torch.uint8, device=DEV)
    st = _lib.stream_ptr()
    assert L.y5m_act8_store(x.data_ptr(), 64, 16, 1, 4, 16, q.data_ptr(), 12, s.data_ptr(), 1, 0, st) != 0      # ldq
    assert L.y5m_act8_store(x.data_ptr(), 64, 16, 1, 4, 16, q.data_ptr(), 16, s.data_ptr(), 3, 0, st) != 0      # format
    assert L.y5m_act8_store(x.data_ptr(), 64, 16, 1, 4, 16, q.data_ptr(), 16, s.data_ptr(), 1, 7, st) != 0      # dtype
    assert L.y5m_act8_store(x.data_ptr(), 64, 16, 1, 4, 16, q.data_ptr() + 1, 16, s.data_ptr(), 1, 0, st) != 0  # alignment
    assert L.y5m_act8_load(q.data_ptr(), 16, s.data_ptr(), 4, 16, x.data_ptr(), 8, 1, 0, st) != 0               # overlapping rows
    dw = torch.full((16, 16), 3.0, device=DEV)
    need = L.y5m_act8_wgrad_workspace_bytes(4, 16, 16)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    assert L.y5m_act8_wgrad(x.data_ptr(), 64, 16, 1, 4, 16, q.data_ptr(), 16, s.data_ptr(), 16, 1, dw.data_ptr(), None, ws.data_ptr(), need - 1, 0, st) != 0
    assert b"workspace" in L.y5m_last_error()
    torch.cuda.synchronize()
    assert (q == 7).all() and (s == 7).all() and (dw == 3.0).all()
    assert isinstance(ctypes.c_size_t(need).value, int)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "fp16"])
def test_one_row_per_image_and_rows_apart(dtype):
    """(N, C) matrices cut out of wider ones, batches that do not follow each other at the rows' distance: stored form and gradient"""
    from yolov5m_amd.act8 import act8_load, act8_store, act8_wgrad
    flat = torch.randn(70, 256, generator=_gen(11)).to(DT[dtype]).to(DEV)
    maps = rows_tensor((3, 160, 9, 8), dtype, 12)
    for x, dy in ((flat[:, 8:72], flat[:, 128:168]), (flat[:, 3:72], flat[:, 101:150]), (maps[:, :72, 1:8], maps[:, 72:136, 1:8]), (maps[::2, 5:60], maps[::2, 64:160])):
        kept = act8_store(x, "int8")
        assert same(act8_load(kept).cpu().movedim(1, -1).double(), stored_values(x, "int8")[0].to(DT[dtype]).double())
        dw, db = act8_wgrad(dy, kept, bias=True)
        xv = stored_values(x, "int8")[0].reshape(-1, x.shape[1])
        dv = dy.cpu().double().movedim(1, -1).reshape(-1, dy.shape[1])
        assert ((dw.cpu().double() - dv.t() @ xv).abs() <= 96 * U * (dv.abs().t() @ xv.abs())).all()
        assert ((db.cpu().double() - dv.sum(0)).abs() <= 160 * U * dv.abs().sum(0)).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", [(1, 100, 5, 5), (1, 160, 40)])
def test_wgrad_nan_in_any_block(shape, dtype):
    """e4m3: a block that is not finite reaches its own columns only, the last (short) block as well; a NaN of dy its own rows only"""
    from yolov5m_amd.act8 import act8_store, act8_wgrad
    c = shape[1]
    for ch in (2, 70, c - 1):
        x, dy = rows_tensor(shape, "bf16", 13), rows_tensor((1, 72, *shape[2:]), dtype, 14)
        x[(0, ch) + (2,) * (len(shape) - 2)] = float("nan")
        dw, _ = act8_wgrad(dy, act8_store(x, "e4m3"))
        bad = torch.zeros(c, dtype=torch.bool, device=DEV)
        bad[ch // 32 * 32:ch // 32 * 32 + 32] = True
        assert torch.isnan(dw[:, bad]).all() and torch.isfinite(dw[:, ~bad]).all()
    x = rows_tensor(shape, "bf16", 13)
    dy[(0, 37) + (1,) * (len(shape) - 2)] = float("nan")
    dw, db = act8_wgrad(dy, act8_store(x, "e4m3"), bias=True)
    rows = torch.arange(72, device=DEV) == 37
    assert torch.isnan(dw[rows]).all() and torch.isfinite(dw[~rows]).all() and torch.isnan(db[rows]).all() and torch.isfinite(db[~rows]).all()


def test_large_tensors_read_back():
    """more than 64 MB: stored past the caches, by kernels of their own"""
    if DEV != "cuda":
        pytest.skip("36 million elements")
    from yolov5m_amd.act8 import act8_load, act8_store
    x = rows_tensor((2, 72, 500, 501), "bf16", 15)
    for fmt in ("e4m3", "int8"):
        assert same(act8_load(act8_store(x, fmt)).cpu().movedim(1, -1).double(), stored_values(x, fmt)[0])


def test_wgrad_rows_far_apart():
    """rows of dy at a distance that one range's 32-bit offsets cannot hold"""
    if DEV != "cuda":
        pytest.skip("6 GB")
    from yolov5m_amd.act8 import act8_load, act8_store, act8_wgrad
    wide = torch.empty((3000, 1 << 20), dtype=torch.bfloat16, device=DEV)
    dy = wide[:, 1 << 19:(1 << 19) + 160].t()[None]
    dy.copy_(rows_tensor((1, 160, 3000), "bf16", 16))
    kept = act8_store(rows_tensor((1, 200, 3000), "bf16", 17), "e4m3")
    dw, db = act8_wgrad(dy, kept, bias=True)
    xv, dv = act8_load(kept).cpu().double()[0].t(), dy.cpu().double()[0].t()
    assert ((dw.cpu().double() - dv.t() @ xv).abs() <= 96 * U * (dv.abs().t() @ xv.abs())).all()
    assert ((db.cpu().double() - dv.sum(0)).abs() <= 160 * U * dv.abs().sum(0)).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "fp16"])
@pytest.mark.parametrize("cout", [1, 2, 3, 4, 5, 7, 63, 65, 67])
def test_wgrad_of_few_and_odd_channels(cout, dtype):
    """pieces that end with the row, rows of less than one piece; rows at one distance and images apart"""
    from yolov5m_amd.act8 import act8_load, act8_store, act8_wgrad
    maps, wide = rows_tensor((3, 40, 9, 8), dtype, 18), rows_tensor((3, 80, 9, 8), dtype, 19, scale=0.1)
    for x, dy in ((maps, wide[:, 3:3 + cout].contiguous(memory_format=torch.channels_last)), (maps, wide[:, 3:3 + cout]), (maps[:, :, 1:8], wide[:, 8:8 + cout, 1:8])):
        kept = act8_store(x, "e4m3")
        dw, db = act8_wgrad(dy, kept, bias=True)
        xv = act8_load(kept).cpu().double().movedim(1, -1).reshape(-1, 40)
        dv = dy.cpu().double().movedim(1, -1).reshape(-1, cout)
        assert ((dw.cpu().double() - dv.t() @ xv).abs() <= 96 * U * (dv.abs().t() @ xv.abs())).all()
        assert ((db.cpu().double() - dv.sum(0)).abs() <= 160 * U * dv.abs().sum(0)).all()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "fp16"])
@pytest.mark.parametrize("case", [(16, 24, 9), (96, 136, 40), (20, 33, 40), (72, 3, 40)])
def test_wgrad_of_the_largest_kept_values(case, dtype, fmt):
    """blocks up to the largest magnitude that is held (a scale of 2^121 in int8), rows of ordinary and of tiny blocks beside them: the products
    are those of the values read back. At most 40 rows: two instructions of 32 products, 34 roundings"""
    from yolov5m_amd.act8 import act8_load, act8_store, act8_wgrad
    c, cout, s = case
    x = rows_tensor((1, c, s), "f32", 120)
    big = torch.finfo(torch.float32).max
    x[0, :, 1] = big
    x[0, ::3, 1] = -big / 3
    x[0, :, 2] = big / 2.0 ** 0.75 * torch.linspace(-1, 1, c).to(DEV)
    x[0, :, 4] = 2.0 ** -110
    dy = rows_tensor((1, cout, s), dtype, 121)
    dy[0, :, 1:3] = dy[0, :, 1:3] * 2.0 ** -8
    kept = act8_store(x, fmt)
    dw, _ = act8_wgrad(dy, kept)
    xv, dv = act8_load(kept).cpu().double()[0], dy.cpu().double()[0]
    assert torch.isfinite(xv).all() and float(xv.abs().max()) > 0.9 * big
    assert ((dw.cpu().double() - dv @ xv.t()).abs() <= 34 * U * (dv.abs() @ xv.abs().t())).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "fp16"])
@pytest.mark.parametrize("case", [(40, 64, 70), (40, 65, 70), (96, 3, 70), (160, 136, 70)])
def test_wgrad_of_large_and_infinite_gradients(case, dtype):
    """dy with the largest finite values of its type, infinities and a NaN, over all ways in which rows are read: a product that is finite in 64
    bits is finite and right (70 rows: three instructions of 32 products, 36 roundings), an infinity gives the signed infinity, or NaN against
    a zero or another sign, as in 64 bits; db alike"""
    from yolov5m_amd.act8 import act8_load, act8_store, act8_wgrad
    c, cout, s = case
    x = rows_tensor((1, c, s), "f32", 122) * 2.0 ** -12
    dy = rows_tensor((1, cout, s), dtype, 123)
    big = torch.finfo(DT[dtype]).max
    dy[0, 0, 5], dy[0, 0, 40] = big, -big
    dy[0, 1, 33] = big * (1 - 2.0 ** -9)
    inf = float("inf")
    dy[0, 2, 7] = inf
    x[0, 1, 7] = 0.0
    if cout > 8:
        dy[0, 3, 9] = -inf
        dy[0, 4, 9], dy[0, 4, 69] = inf, -inf
        dy[0, 5, 0] = float("nan")
        dy[0, cout - 1, 69] = -big
    kept = act8_store(x, "e4m3")
    dw, db = act8_wgrad(dy, kept, bias=True)
    xv, dv = act8_load(kept).cpu().double()[0], dy.cpu().double()[0]
    want, mag, sums = dv @ xv.t(), dv.abs() @ xv.abs().t(), dv.sum(1)
    assert not torch.isfinite(want[2]).any() and torch.isfinite(want[:2]).all()
    for got, ref, tol in ((dw, want, 36 * U * mag), (db, sums, 20 * U * dv.abs().sum(1))):
        got, fin = got.cpu().double(), torch.isfinite(ref)
        assert same(got[~fin], ref[~fin])
        ok = fin & (ref.abs() + tol < 0.9 * torch.finfo(torch.float32).max) & (tol < big)
        assert ((got - ref).abs() <= tol)[ok].all()


@pytest.mark.parametrize("dtype", ["f32", "fp16"])
def test_wgrad_of_infinite_gradients_at_any_strides(dtype):
    """the same where samples and rows lie at two distances; db of every row once"""
    from yolov5m_amd.act8 import act8_load, act8_store, act8_wgrad
    x = rows_tensor((3, 40, 21), "f32", 124)
    dy = rows_tensor((6, 20, 21), dtype, 125)[::2]
    dy[1, 2, 7], dy[2, 3, 20] = float("inf"), torch.finfo(DT[dtype]).max
    kept = act8_store(x, "int8")
    dw, db = act8_wgrad(dy, kept, bias=True)
    xv, dv = (t.cpu().double().movedim(1, -1).flatten(0, 1) for t in (act8_load(kept), dy))
    want, fin = dv.t() @ xv, torch.arange(20) != 2
    assert same(dw.cpu().double()[2], want[2]) and float(db[2]) == float("inf")
    ok = torch.isfinite(want.float())
    assert ((dw.cpu().double() - want).abs() <= 36 * U * (dv.abs().t() @ xv.abs()))[fin][ok[fin]].all()
    assert ((db.cpu().double() - dv.sum(0)).abs() <= 20 * U * dv.abs().sum(0))[fin].all()
