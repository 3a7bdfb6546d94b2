"""Group normalisation + activation over channels-last maps (yolov5m_amd/group_norm.py) against the formulas in 64 bits: every type,
group width and kept form, views, single rows, empty batches; gradients also against differences, through autograd, in a captured
graph and inside the CBL block that uses them. tests/test_emu_act8.py runs the same functions on the CPU executor."""
import pytest
import torch
import torch.nn.functional as F

from test_gpu_act8 import DT, U, rows_tensor, stored_values

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _rows(*a, **k):
    return rows_tensor(*a, **k).to(DEV)


def _params(c, seed):
    g = torch.Generator().manual_seed(seed)
    return (1 + 0.3 * torch.randn(c, generator=g)).to(DEV), (0.3 * torch.randn(c, generator=g)).to(DEV)


class Exact:
    """the formulas in 64 bits, with the error bounds of a computation that rounds to f32 (u = 2^-24) at every step.
    Sums run in chains of at most ~300 f32 additions before they are joined in f64; errors of such a chain grow like its square root
    (17 u), the pivot of the squares may double that: 64 u of the summed magnitudes. In xhat = (x - mean) rstd the mean's own rounding
    counts u |mean| rstd; act' <= 1.1 carries t's error on, and the exponential adds u |t|, |t| <= 20 here, of the value."""

    def __init__(self, x, groups, gamma, beta, eps, act, kept=None, dz=None):
        d = lambda t: t.detach().cpu().double()
        v = d(x).movedim(1, -1)
        n, c = v.shape[0], v.shape[-1]
        v = v.reshape(n, -1, groups, c // groups)
        ga = (d(gamma) if gamma is not None else torch.ones(c).double()).view(groups, -1)
        be = (d(beta) if beta is not None else torch.zeros(c).double()).view(groups, -1)
        mean = v.mean((1, 3), keepdim=True)
        rstd = 1 / torch.sqrt(((v - mean) ** 2).mean((1, 3), keepdim=True) + eps)
        self.mean, self.rstd = mean.flatten(), rstd.flatten()
        mabs = v.abs().mean((1, 3), keepdim=True)
        xh = (v - mean) * rstd
        t = xh * ga + be
        mag = (xh * ga).abs() + be.abs() + mabs * rstd * ga.abs()
        self.z = t * torch.sigmoid(t) if act == "silu" else t
        self.z_tol = 64 * U * mag * 1.1
        self.shape = x.shape
        if dz is None:
            return
        k = v if kept is None else kept.reshape(v.shape)
        xh = (k - mean) * rstd
        xm = xh.abs() + mabs * rstd
        t = xh * ga + be
        g = d(dz).movedim(1, -1).reshape(v.shape)
        s = torch.sigmoid(t)
        dt = g * (s * (1 + t * (1 - s)) if act == "silu" else 1.0)
        dtm = g.abs() * (1.1 + (0.5 * (xm * ga.abs() + be.abs()) if act == "silu" else 0.0))     # |dt| and 0.5 >= |act''| times t's magnitude
        self.dgamma, self.dgamma_tol = (dt * xh).sum((0, 1)).flatten(), 64 * U * (dtm * xm).sum((0, 1)).flatten()
        self.dbeta, self.dbeta_tol = dt.sum((0, 1)).flatten(), 64 * U * dtm.sum((0, 1)).flatten()
        w, wm = dt * ga, dtm * ga.abs()
        A, B = w.mean((1, 3), keepdim=True), (w * xh).mean((1, 3), keepdim=True)
        Am, Bm = wm.mean((1, 3), keepdim=True), (wm * xm).mean((1, 3), keepdim=True)
        self.dx = rstd * (w - A - xh * B)
        self.dx_tol = 64 * U * rstd * (wm + Am + xm * Bm)

    def check(self, got, what):
        want, tol = getattr(self, what), getattr(self, what + "_tol")
        g = got.detach().cpu().double()
        if what in ("z", "dx"):
            g = g.movedim(1, -1).reshape(want.shape)
        half = torch.finfo(got.dtype).eps / 2
        small = torch.finfo(got.dtype).smallest_normal * half * 2         # half a subnormal step
        bad = (g - want).abs() > tol + half * (want.abs() + tol) + small
        assert not bad.any(), (what, int(bad.sum()), float((g - want).abs().max()), float(tol.max()))


CASES = [((1, 8, 1, 1), 1), ((2, 4, 1, 1), 4), ((1, 1, 3, 3), 1), ((2, 96, 5, 7), 32), ((3, 36, 6, 5), 12), ((2, 255, 3, 4), 15), ((1, 64, 17, 13), 1),
         ((4, 40, 9, 2), 5), ((2, 33, 11), 33), ((5, 24), 3), ((1, 2056, 3, 1), 8), ((2, 192, 40, 33), 32), ((1, 768, 20, 20), 32), ((70, 16, 2, 2), 2)]


@pytest.mark.parametrize("act", ["silu", None])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "fp16"])
@pytest.mark.parametrize("case", CASES)
def test_forward(case, dtype, act):
    from yolov5m_amd.group_norm import group_norm_act
    shape, groups = case
    x = _rows(shape, dtype, 1, offset=0.5)
    ga, be = _params(shape[1], 2)
    ref = Exact(x, groups, ga, be, 1e-3, act)
    z, saved = group_norm_act(x, groups, ga, be, eps=1e-3, act=act)
    assert saved is None and z.dtype == x.dtype and z.shape == x.shape
    ref.check(z, "z")
    # what a training forward keeps does not change its result; mean and rstd come with it
    z2, saved = group_norm_act(x, groups, ga, be, eps=1e-3, act=act, keep="x")
    assert torch.equal(z, z2)
    assert ((saved.mean.cpu().double().flatten() - ref.mean).abs() <= 64 * U * (ref.mean.abs() + 1 / ref.rstd)).all()
    assert ((saved.rstd.cpu().double().flatten() - ref.rstd).abs() <= 64 * U * ref.rstd).all()


@pytest.mark.parametrize("keep", ["x", "e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "fp16"])
@pytest.mark.parametrize("case", CASES)
def test_backward_from_what_was_kept(case, dtype, keep):
    from yolov5m_amd.act8 import act8_load
    from yolov5m_amd.group_norm import group_norm_act, group_norm_act_backward
    shape, groups = case
    x = _rows(shape, dtype, 3, offset=0.5)
    dz = _rows(shape, dtype, 4, scale=0.1)
    ga, be = _params(shape[1], 5)
    kept = None if keep == "x" else stored_values(x, keep)[0]
    ref = Exact(x, groups, ga, be, 1e-3, "silu", kept, dz)
    z, saved = group_norm_act(x, groups, ga, be, eps=1e-3, keep=keep)
    ref.check(z, "z")
    if keep != "x":
        assert torch.equal(act8_load(saved.kept).cpu().movedim(1, -1).double(), kept.to(DT[dtype]).double())
        x.fill_(float("nan"))                                             # the input is no longer needed
    dx, dg, db = group_norm_act_backward(dz, saved)
    assert dx.dtype == x.dtype and dg.dtype == db.dtype == torch.float32
    ref.check(dx, "dx")
    ref.check(dg, "dgamma")
    ref.check(db, "dbeta")
    again = group_norm_act_backward(dz, saved)
    assert all(torch.equal(a, b) for a, b in zip((dx, dg, db), again))    # one result per input


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_no_parameters_no_activation_and_views(dtype):
    """weight and bias absent, act none; x and dz as channel slices of wider buffers (on and off 16-byte borders) and as tokens"""
    from yolov5m_amd.group_norm import group_norm_act, group_norm_act_backward
    wide, gwide = _rows((3, 128, 6, 5), dtype, 6, offset=1.0), _rows((3, 128, 6, 5), dtype, 7)
    tok, gtok = _rows((3, 48, 19), dtype, 8), _rows((3, 48, 19), dtype, 9)
    for x, dz, groups in ((wide[:, 32:96], gwide[:, 64:128], 8), (wide[:, 3:75], gwide[:, 1:73], 6), (tok, gtok, 48),
                          (wide[::2], gwide[1:], 16), (wide[:1].expand(3, -1, -1, -1), gwide, 4)):
        for keep in ("x", "int8"):
            kept = None if keep == "x" else stored_values(x, keep)[0]
            ref = Exact(x, groups, None, None, 1e-5, None, kept, dz)
            z, saved = group_norm_act(x, groups, act=None, keep=keep)
            ref.check(z, "z")
            dx, dg, db = group_norm_act_backward(dz, saved)
            ref.check(dx, "dx")
            ref.check(dg, "dgamma")
            ref.check(db, "dbeta")


def test_far_from_zero_and_an_outlier_row():
    """a mean of 300 spreads and a first row of 1000: the squares are summed about a pivot, so neither cancels. The mean itself is f32:
    |mean| rstd u is in the bounds"""
    from yolov5m_amd.group_norm import group_norm_act
    for seed in (10, 11):
        x = torch.randn((2, 40, 30, 48), generator=torch.Generator().manual_seed(seed))
        if seed == 10:
            x = x + 300.0
        else:
            x[:, 0, 0] = 1000.0
        x = x.movedim(-1, 1).to(DEV)
        ref = Exact(x, 6, None, None, 1e-5, None)
        z, saved = group_norm_act(x, 6, act=None, keep="x")
        ref.check(z, "z")
        assert ((saved.rstd.cpu().double().flatten() - ref.rstd).abs() <= 64 * U * ref.rstd).all()


def test_constant_groups_and_single_values():
    """variance zero: rstd = 1 / sqrt(eps), z = act(bias) and dx = 0 up to rounding, for one value per group and for constant maps"""
    from yolov5m_amd.group_norm import group_norm_act, group_norm_act_backward
    ga, be = _params(16, 12)
    for x, groups in ((_rows((3, 16, 1, 1), "f32", 13), 16), (torch.full((2, 5, 5, 16), 3.7, device=DEV).movedim(-1, 1), 4)):
        z, saved = group_norm_act(x, groups, ga, be, eps=1e-5, act=None, keep="x")
        assert (z.movedim(1, -1) - be).abs().max() <= 1e-4            # (f32 mean of equal values: xhat <= u |x| / sqrt(eps) = 7e-5)
        assert torch.allclose(saved.rstd, torch.full_like(saved.rstd, 1e-5 ** -0.5), rtol=1e-6)
        dz = _rows(x.shape, "f32", 14)
        dx, dg, db = group_norm_act_backward(dz, saved)
        Exact(x, groups, ga, be, 1e-5, None, None, dz).check(dx, "dx")


def test_empty_inputs():
    from yolov5m_amd.group_norm import group_norm_act, group_norm_act_backward
    ga, be = _params(16, 15)
    for shape in ((0, 16, 4, 4), (2, 16, 0, 4)):
        for keep in ("x", "e4m3"):
            x = torch.zeros((shape[0], *shape[2:], 16), device=DEV).movedim(-1, 1)
            z, saved = group_norm_act(x, 4, ga, be, keep=keep)
            dx, dg, db = group_norm_act_backward(x, saved)
            assert z.shape == dx.shape == x.shape and not dg.any() and not db.any()


def test_a_value_that_is_not_finite_stays_in_its_group():
    from yolov5m_amd.group_norm import group_norm_act, group_norm_act_backward
    for bad in (float("inf"), float("nan")):
        for keep in ("x", "e4m3", "int8"):
            x = _rows((3, 64, 5, 5), "bf16", 16)
            x[1, 20, 2, 3] = bad                                     # group 1 of 4 (channels 16..31) of image 1
            z, saved = group_norm_act(x, 4, keep=keep)
            dx, dg, db = group_norm_act_backward(_rows((3, 64, 5, 5), "bf16", 17), saved)
            hit = torch.zeros_like(z, dtype=torch.bool)
            hit[1, 16:32] = True
            assert not torch.isfinite(z[hit]).any() and torch.isfinite(z[~hit]).all()
            # (in 8 bits the whole block of 32 channels reads back as NaN, so the block's other group has it in the backward too)
            first = 16 if keep == "x" else 0
            hit[1, first:32] = True
            assert torch.isnan(dx[hit]).all() and torch.isfinite(dx[~hit]).all()
            assert torch.isnan(dg[first:32]).all() and torch.isfinite(dg[:first]).all() and torch.isfinite(dg[32:]).all()


def test_gradient_against_differences():
    """d/dx, d/dgamma, d/dbeta of sum(z w) by central differences of the 64-bit formula: step h, truncation h^2 |f'''| / 6 < 1e-6"""
    from yolov5m_amd.group_norm import group_norm_act, group_norm_act_backward
    x, w = _rows((1, 8, 3, 2), "f32", 18), _rows((1, 8, 3, 2), "f32", 19, scale=0.3)
    ga, be = _params(8, 20)

    def f(xv, gv, bv):
        return float((Exact(xv, 2, gv, bv, 1e-3, "silu").z.reshape(1, 3, 2, 8).movedim(-1, 1) * w.cpu().double()).sum())
    _, saved = group_norm_act(x, 2, ga, be, eps=1e-3, keep="x")
    dx, dg, db = group_norm_act_backward(w, saved)
    h = 1e-4
    args = [t.detach().cpu().double() for t in (x, ga, be)]
    for which, got in ((0, dx), (1, dg), (2, db)):
        for idx in torch.cartesian_prod(*[torch.arange(n) for n in args[which].shape]).reshape(-1, args[which].dim()).tolist():
            d = []
            for sgn in (1, -1):
                a = [t.clone() for t in args]
                a[which][tuple(idx)] += sgn * h
                d.append(f(*a))
            num = (d[0] - d[1]) / (2 * h)
            assert abs(num - float(got[tuple(idx)])) <= 2e-5, (which, idx, num, float(got[tuple(idx)]))


@pytest.mark.parametrize("keep", ["x", "int8"])
def test_module_and_autograd(keep):
    """GroupNormAct inside a torch graph: gradients of input and parameters; a gradient that arrives in another layout (NCHW, a broadcast)
    is laid out; nn.GroupNorm's parameter names"""
    from yolov5m_amd.group_norm import GroupNormAct
    layer = GroupNormAct(6, 48, eps=1e-3, keep=keep).to(DEV)
    assert set(layer.state_dict()) == set(torch.nn.GroupNorm(6, 48).state_dict())
    with torch.no_grad():
        layer.weight.copy_(_params(48, 21)[0])
        layer.bias.copy_(_params(48, 21)[1])
    x = _rows((2, 48, 7, 5), "f32", 22).requires_grad_()
    w = torch.randn(2, 48, 7, 5, generator=torch.Generator().manual_seed(23)).to(DEV)          # NCHW
    z = layer(x)
    (z * w).sum().backward()
    kept = None if keep == "x" else stored_values(x, keep)[0]
    ref = Exact(x, 6, layer.weight, layer.bias, 1e-3, "silu", kept, w)
    ref.check(z, "z")
    ref.check(x.grad, "dx")
    ref.check(layer.weight.grad, "dgamma")
    ref.check(layer.bias.grad, "dbeta")
    layer.zero_grad()
    layer(x).sum().backward()                                                                    # dz: one value, broadcast
    Exact(x, 6, layer.weight, layer.bias, 1e-3, "silu", kept, torch.ones_like(w)).check(layer.bias.grad, "dbeta")
    with torch.no_grad():
        assert not layer(x).requires_grad
    if keep == "x":
        y = layer(x * 1.0)
        inp = (x * 1.0)
        y = layer(inp)
        with torch.no_grad():
            inp.zero_()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_rows_between_and_behind_the_output_are_left_alone():
    """the C entry points with padded rows: elements between the rows of z / dx, and the workspace's neighbours, keep what they hold"""
    import yolov5m_amd.group_norm  # noqa: F401
    from yolov5m_amd import _lib
    L = _lib.lib()
    n, s, c, g = 2, 37, 24, 3
    for ld, odd in ((40, 0), (29, 1)):
        x = torch.randn(n, s, c, generator=torch.Generator().manual_seed(24)).to(DEV)
        z = torch.full((n, s + 1, ld), 7.0, device=DEV)
        dx = torch.full((n, s + 1, ld), 7.0, device=DEV)
        stat = torch.full((2 * n * g + 4,), 7.0, device=DEV)
        wsb = L.y5m_gn_act_workspace_bytes(n, s, c, g)
        ws = torch.full((wsb + 64,), 7, dtype=torch.uint8, device=DEV)
        p = stat.data_ptr()
        _lib.check(L.y5m_gn_act(x.data_ptr(), s * c, c, None, None, n, s, c, g, 1e-5, 1, z.data_ptr() + 4 * odd, (s + 1) * ld, ld, p, p + 4 * n * g, None, 0,
                                None, 0, ws.data_ptr(), wsb, 0, _lib.stream_ptr()), "y5m_gn_act")
        assert (ws[wsb:] == 7).all() and (stat[2 * n * g:] == 7.0).all()
        wsb = L.y5m_gn_act_bwd_workspace_bytes(n, s, c, g)
        ws = torch.full((wsb + 64,), 7, dtype=torch.uint8, device=DEV)
        gr = torch.full((2 * c + 4,), 7.0, device=DEV)
        _lib.check(L.y5m_gn_act_bwd(x.data_ptr(), s * c, c, x.data_ptr(), s * c, c, None, 0, None, 0, None, None, p, p + 4 * n * g, n, s, c, g, 1,
                                    dx.data_ptr() + 4 * odd, (s + 1) * ld, ld, gr.data_ptr(), gr.data_ptr() + 4 * c, ws.data_ptr(), wsb, 0, _lib.stream_ptr()),
                   "y5m_gn_act_bwd")
        assert (ws[wsb:] == 7).all() and (gr[2 * c:] == 7.0).all()
        xt = x.transpose(1, 2)
        ref = Exact(xt, g, None, None, 1e-5, "silu", None, xt)
        for t, what in ((z, "z"), (dx, "dx")):
            ref.check(t[:, :s, odd:c + odd].transpose(1, 2), what)
            assert (t[:, s] == 7.0)[:, odd:].all() and (t[:, :s, c + odd:] == 7.0).all() and (odd == 0 or (t[0, 0, :odd] == 7.0).all())


@pytest.mark.parametrize("shape", [(2, 90, 40), (1, 2000, 136)])
def test_in_place_at_the_c_entry(shape):
    """z over x, dx over dz"""
    import yolov5m_amd.group_norm  # noqa: F401
    from yolov5m_amd import _lib
    L = _lib.lib()
    (n, s, c), g = shape, 4
    x, dz = (torch.randn(n, s, c, generator=torch.Generator().manual_seed(k)).to(DEV) for k in (25, 26))
    xt = x.clone().transpose(1, 2)
    ref = Exact(xt, g, None, None, 1e-5, "silu", None, dz.clone().transpose(1, 2))
    stat = torch.empty(2 * n * g, device=DEV)
    wsb = L.y5m_gn_act_bwd_workspace_bytes(n, s, c, g)
    ws = torch.empty(wsb, dtype=torch.uint8, device=DEV)
    keep = x.clone()
    p = stat.data_ptr()
    _lib.check(L.y5m_gn_act(x.data_ptr(), s * c, c, None, None, n, s, c, g, 1e-5, 1, x.data_ptr(), s * c, c, p, p + 4 * n * g,
                            None, 0, None, 0, ws.data_ptr(), wsb, 0, _lib.stream_ptr()), "y5m_gn_act")
    ref.check(x.transpose(1, 2), "z")
    _lib.check(L.y5m_gn_act_bwd(dz.data_ptr(), s * c, c, keep.data_ptr(), s * c, c, None, 0, None, 0, None, None, p, p + 4 * n * g, n, s, c, g, 1,
                                dz.data_ptr(), s * c, c, None, None, ws.data_ptr(), wsb, 0, _lib.stream_ptr()), "y5m_gn_act_bwd")
    ref.check(dz.transpose(1, 2), "dx")


def test_refusals():
    from yolov5m_amd._lib import Y5MError
    from yolov5m_amd.group_norm import GroupNormAct, group_norm_act, group_norm_act_backward
    x = _rows((2, 16, 4, 4), "f32", 26)
    for kw, msg in ((dict(groups=3), "divide"), (dict(groups=0), "divide"), (dict(groups=4, act="relu"), "act"), (dict(groups=4, keep="int4"), "keep"),
                    (dict(groups=4, eps=0.0), "eps"), (dict(groups=4, weight=torch.ones(8, device=DEV)), "weight"),
                    (dict(groups=4, bias=torch.ones(16, device=DEV, dtype=torch.int32)), "bias")):
        with pytest.raises(Y5MError, match=msg):
            group_norm_act(x, **kw)
    with pytest.raises(Y5MError, match="channels last"):
        group_norm_act(x.contiguous(), 4)
    with pytest.raises(Y5MError, match="float32"):
        group_norm_act(x.double(), 4)
    _, saved = group_norm_act(x, 4, keep="x")
    with pytest.raises(Y5MError, match="dz"):
        group_norm_act_backward(x[:1], saved)
    with pytest.raises(Y5MError, match="dz"):
        group_norm_act_backward(x.bfloat16(), saved)
    with pytest.raises(Y5MError, match="channels last"):
        group_norm_act_backward(x.contiguous(), saved)
    with pytest.raises(Y5MError, match="divide"):
        GroupNormAct(5, 16)
    with pytest.raises(Y5MError, match="keep"):
        GroupNormAct(4, 16, keep=None)


def test_other_stream_and_captured_graph():
    """forward, 8-bit form, backward and weight gradient on a side stream, and captured: every replay, with new inputs and eager calls
    of the same operators between the replays, equals the eager result"""
    if DEV != "cuda":
        pytest.skip("streams and graphs")
    from yolov5m_amd.act8 import act8_wgrad
    from yolov5m_amd.group_norm import group_norm_act, group_norm_act_backward
    shape, groups = (4, 96, 20, 20), 32
    ga, be = _params(96, 27)
    x, dz = _rows(shape, "bf16", 28), _rows(shape, "bf16", 29)

    def step(x, dz):
        z, saved = group_norm_act(x, groups, ga, be, keep="e4m3")
        dx, dg, db = group_norm_act_backward(dz, saved)
        dw, dwb = act8_wgrad(dz, saved.kept, bias=True)
        return z, dx, dg, db, dw, dwb
    want = step(x, dz)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x, dz)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    g = torch.cuda.CUDAGraph()
    xs, dzs = x.clone(), dz.clone()
    with torch.cuda.graph(g):
        out = step(xs, dzs)
    for seed in (30, 31, 32):
        xs.copy_(_rows(shape, "bf16", seed))
        dzs.copy_(_rows(shape, "bf16", seed + 50))
        g.replay()
        want = step(xs, dzs)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, out)), seed


@pytest.mark.parametrize("keep", ["x", "e4m3", "int8"])
@pytest.mark.parametrize("case", [(16, 32, 1, 1), (16, 24, 3, 1), (16, 32, 3, 2), (3, 16, 3, 1)])
def test_cbl_with_group_norm(case, keep):
    """conv + GroupNorm + SiLU of model.CBL as a training step, forward and every gradient, against the same block in 64 bits whose kept
    tensors are replaced by what their 8-bit form stands for. f32 convolutions: chains of at most 144 products, 64 u of the magnitudes;
    the norm multiplies by rstd * gamma (<= 16 here) and its gradient passes on to the convolution's: 2e-4 of each tensor's largest"""
    from yolov5m_amd.model import CBL
    cin, cout, k, s = case
    torch.manual_seed(33)
    m = CBL(cin, cout, k, s, k // 2, norm_groups=8, keep=keep).to(DEV)
    with torch.no_grad():
        m.cbl[1].weight.copy_(_params(cout, 34)[0])
        m.cbl[1].bias.copy_(_params(cout, 34)[1])
    x = torch.randn(2, cin, 10, 6, generator=torch.Generator().manual_seed(35)).to(DEV).requires_grad_()
    z = m(x)
    w = torch.randn(z.shape, generator=torch.Generator().manual_seed(36)).to(DEV)
    (z * w).sum().backward()
    xd, wd = x.detach().cpu().double(), m.cbl[0].weight.detach().cpu().double()
    y = F.conv2d(xd, wd, stride=s, padding=k // 2)
    nhwc = lambda t: t.contiguous(memory_format=torch.channels_last)
    # (the stored form of the layer's own f32 convolution output: a code border may fall between it and the 64-bit one)
    from yolov5m_amd.model import _ConvKeptFn
    yd = _ConvKeptFn.apply(x.detach(), m.cbl[0].weight.detach(), m)
    kept = None if keep == "x" else stored_values(yd, keep)[0]
    ref = Exact(nhwc(y), 8, m.cbl[1].weight, m.cbl[1].bias, 1e-3, "silu", kept, w)

    def close(a, b, what):
        a = a.detach().cpu().double()
        assert (a - b).abs().max() <= 2e-4 * b.abs().max(), (what, float((a - b).abs().max()), float(b.abs().max()))
    sh = (2, *y.shape[2:], cout)
    close(z, ref.z.reshape(sh).movedim(-1, 1), "z")
    close(m.cbl[1].weight.grad, ref.dgamma, "dgamma")
    close(m.cbl[1].bias.grad, ref.dbeta, "dbeta")
    dy = ref.dx.reshape(sh).movedim(-1, 1)
    xk = xd if keep == "x" else stored_values(nhwc(x.detach()), keep)[0].movedim(-1, 1)
    close(x.grad, torch.nn.grad.conv2d_input(xd.shape, wd, dy, stride=s, padding=k // 2), "dx")
    close(m.cbl[0].weight.grad, torch.nn.grad.conv2d_weight(xk, wd.shape, dy, stride=s, padding=k // 2), "dw")


def test_c3_block_trains_with_group_norm_and_kept_activations():
    """a whole C3 block (7 convolutions, residuals, concat) with norm_groups: runs forward and backward, every parameter gets a finite
    gradient, a group-norm C3 in f32 with keep="x" agrees with torch's group_norm block in 64 bits"""
    from yolov5m_amd.model import C3, CBL
    torch.manual_seed(37)
    m = C3(16, 16, width_multiple=0.5, depth=2, norm_groups=4, keep="int8").to(DEV)
    x = torch.randn(2, 16, 6, 8).to(DEV)
    m(x).square().sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().sum() > 0 for p in m.parameters())
    m = C3(16, 16, width_multiple=0.5, depth=1, norm_groups=4).to(DEV)

    def cbl(mod, t):
        conv, norm = mod.cbl[0], mod.cbl[1]
        assert isinstance(mod, CBL)
        t = F.conv2d(t, conv.weight.detach().cpu().double(), padding=conv.padding[0])
        return F.silu(F.group_norm(t, 4, norm.weight.detach().cpu().double(), norm.bias.detach().cpu().double(), 1e-3))
    xd = x.detach().cpu().double()
    a = cbl(m.c1, xd)
    b = m.seq[0]
    a = cbl(b.c2, cbl(b.c1, a)) + a
    want = cbl(m.c_out, torch.cat([a, cbl(m.c_skipped, xd)], 1))
    got = m(x).detach().cpu().double()
    assert (got - want).abs().max() <= 2e-4 * want.abs().max()


@pytest.mark.parametrize("keep", ["x", "int8"])
@pytest.mark.parametrize("case", [((3, 8200), 1), ((3, 8200), 8), ((300, 24), 3), ((2, 40, 3), 40)])
def test_samples_of_few_rows(case, keep):
    """one row per sample (tokens, class logits), rows wider than a workgroup holds, groups of one channel"""
    from yolov5m_amd.group_norm import group_norm_act, group_norm_act_backward
    shape, groups = case
    x, dz = _rows(shape, "bf16", 60, offset=0.5), _rows(shape, "bf16", 61, scale=0.1)
    ga, be = _params(shape[1], 62)
    kept = None if keep == "x" else stored_values(x, keep)[0]
    ref = Exact(x, groups, ga, be, 1e-3, "silu", kept, dz)
    z, saved = group_norm_act(x, groups, ga, be, eps=1e-3, keep=keep)
    ref.check(z, "z")
    for got, what in zip(group_norm_act_backward(dz, saved), ("dx", "dgamma", "dbeta")):
        ref.check(got, what)


def test_more_samples_than_one_grid_dimension():
    """33000 samples (the launches fold them over two dimensions of the grid), each long enough for the split form"""
    if DEV != "cuda":
        pytest.skip("34 million elements")
    from yolov5m_amd.group_norm import group_norm_act, group_norm_act_backward
    shape = (33000, 8, 128)
    x, dz = _rows(shape, "bf16", 63, offset=0.5), _rows(shape, "bf16", 64, scale=0.1)
    ga, be = _params(8, 65)
    z, saved = group_norm_act(x, 2, ga, be, eps=1e-3, keep="x")
    dx, dg, db = group_norm_act_backward(dz, saved)
    ref = Exact(x, 2, ga, be, 1e-3, "silu", None, dz)
    for got, what in ((z, "z"), (dx, "dx"), (dg, "dgamma"), (db, "dbeta")):
        ref.check(got, what)


@pytest.mark.parametrize("keep", ["x", "e4m3"])
def test_outputs_larger_than_the_caches(keep):
    """above 64 MB outputs are stored past the caches, by kernels of their own; the gradient in place of dz as well"""
    if DEV != "cuda":
        pytest.skip("34 million elements")
    from yolov5m_amd import _lib
    from yolov5m_amd.group_norm import group_norm_act, group_norm_act_backward
    shape = (3, 96, 340, 351)
    x, dz = _rows(shape, "bf16", 66, offset=0.5), _rows(shape, "bf16", 67, scale=0.1)
    ga, be = _params(96, 68)
    kept = None if keep == "x" else stored_values(x, keep)[0]
    z, saved = group_norm_act(x, 32, ga, be, eps=1e-3, keep=keep)
    dx, dg, db = group_norm_act_backward(dz, saved)
    ref = Exact(x, 32, ga, be, 1e-3, "silu", kept, dz)
    for got, what in ((z, "z"), (dx, "dx"), (dg, "dgamma"), (db, "dbeta")):
        ref.check(got, what)
    if keep == "x":
        return
    L, s, a = _lib.lib(), 340 * 351, saved.kept
    ws = torch.empty(L.y5m_gn_act_bwd_workspace_bytes(3, s, 96, 32), dtype=torch.uint8, device=DEV)
    _lib.check(L.y5m_gn_act_bwd(dz.data_ptr(), s * 96, 96, None, 0, 0, a.q.data_ptr(), a.q.shape[1], a.scale.data_ptr(), 1, ga.data_ptr(), be.data_ptr(),
                                saved.mean.data_ptr(), saved.rstd.data_ptr(), 3, s, 96, 32, 1, dz.data_ptr(), s * 96, 96, None, None, ws.data_ptr(),
                                ws.numel(), 1, _lib.stream_ptr()), "y5m_gn_act_bwd")
    assert torch.equal(dz, dx)


def test_offsets_beyond_32_bits():
    """elements past 2^31: in the strides of the input and of dz, and in dense tensors (output, codes, gradient)"""
    if DEV != "cuda":
        pytest.skip("30 GB")
    from yolov5m_amd.act8 import act8_load, act8_wgrad
    from yolov5m_amd.group_norm import group_norm_act, group_norm_act_backward
    ga, be = _params(64, 69)
    wide = torch.empty((20000, 110000), dtype=torch.bfloat16, device=DEV)
    x, dz = wide[:, 64:128].t()[None], wide[:, 109936:].t()[None]
    x.copy_(_rows((1, 64, 20000), "bf16", 70, offset=0.5))
    dz.copy_(_rows((1, 64, 20000), "bf16", 71, scale=0.1))
    z, saved = group_norm_act(x, 4, ga, be, eps=1e-3, keep="x")
    ref = Exact(x, 4, ga, be, 1e-3, "silu", None, dz)
    ref.check(z, "z")
    for got, what in zip(group_norm_act_backward(dz, saved), ("dx", "dgamma", "dbeta")):
        ref.check(got, what)
    del wide, x, dz, z, saved

    shape = (140, 96, 400, 400)
    ga, be = _params(96, 72)
    big = lambda: torch.empty((140, 400, 400, 96), dtype=torch.bfloat16, device=DEV).normal_().movedim(-1, 1)
    x, dz = big(), big()
    z, saved = group_norm_act(x, 32, ga, be, eps=1e-3, keep="int8")
    dx, dg, db = group_norm_act_backward(dz, saved)
    y = act8_load(saved.kept)
    for n in (0, 139):
        kept = stored_values(x[n:n + 1], "int8")[0]
        assert torch.equal(y[n:n + 1].cpu().movedim(1, -1).double(), kept)
        ref = Exact(x[n:n + 1], 32, ga, be, 1e-3, "silu", kept, dz[n:n + 1])
        ref.check(z[n:n + 1], "z")
        ref.check(dx[n:n + 1], "dx")
    # 22.4 million rows in 512 ranges of at most 43776: a wave's chain is a quarter of that in steps of 32, plus 32 products each
    dw, dwb = act8_wgrad(dz, saved.kept, bias=True)
    want, mag, sums, smag = (torch.zeros(s, dtype=torch.float64, device=DEV) for s in ((96, 96), (96, 96), (96,), (96,)))
    for n in range(140):
        d, v = dz[n].movedim(0, -1).reshape(-1, 96).double(), y[n].movedim(0, -1).reshape(-1, 96).double()
        want += d.t() @ v
        mag += d.abs().t() @ v.abs()
        sums += d.sum(0)
        smag += d.abs().sum(0)
    assert ((dw.double() - want).abs() <= (342 + 32 + 8) * U * mag).all()
    assert ((dwb.double() - sums).abs() <= (43776 // 16 + 16) * U * smag).all()


def test_two_streams_at_once():
    """the same operators on two streams at a time, several times over: each call has its own workspace, results equal the first ones"""
    if DEV != "cuda":
        pytest.skip("streams")
    from yolov5m_amd.act8 import act8_wgrad
    from yolov5m_amd.group_norm import group_norm_act, group_norm_act_backward
    ga, be = _params(96, 73)

    def step(x, dz):
        z, saved = group_norm_act(x, 32, ga, be, keep="e4m3")
        return (z, *group_norm_act_backward(dz, saved), *act8_wgrad(dz, saved.kept, bias=True))
    data = [(_rows((n, 96, 80, 80), "bf16", 74 + n), _rows((n, 96, 80, 80), "bf16", 90 + n)) for n in (2, 8)]
    want = [step(*d) for d in data]
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(4):
        for s, d in zip(side, data):
            with torch.cuda.stream(s):
                got.append(step(*d))
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(want[i % 2], out)), i


def test_empty_maps_of_any_layout():
    from yolov5m_amd.act8 import act8_load, act8_store
    from yolov5m_amd.group_norm import group_norm_act
    for x in (torch.zeros((2, 8, 5, 0), device=DEV), torch.zeros((2, 8, 5, 0), device=DEV).contiguous(memory_format=torch.channels_last), torch.zeros((0, 8, 3), device=DEV)):
        assert group_norm_act(x, 4)[0].shape == act8_load(act8_store(x)).shape == x.shape


def test_a_kept_form_needs_group_norm():
    from yolov5m_amd._lib import Y5MError
    from yolov5m_amd.model import CBL
    with pytest.raises(Y5MError, match="norm_groups"):
        CBL(8, 8, 1, 1, 0, keep="int8")


SPLIT = [((5, 36, 21, 37), 12, "fp16"), ((3, 29, 121, 63), 29, "bf16"), ((1, 96, 80, 80), 32, "bf16"), ((2, 768, 30, 30), 1, "bf16"), ((1, 1386, 31, 5), 2, "f32"),
         ((1, 2112, 12, 11), 3, "bf16"), ((9, 64, 40, 40), 64, "f32")]


@pytest.mark.parametrize("keep", ["x", "int8"])
@pytest.mark.parametrize("case", SPLIT)
def test_few_and_many_sums_to_join(case, keep):
    """maps too long for one workgroup: sums joined by the apply pass, by 256 and by 1024 threads a group, groups across column tiles"""
    from yolov5m_amd.group_norm import group_norm_act, group_norm_act_backward
    shape, groups, dtype = case
    if DEV != "cuda" and shape[0] * shape[1] * shape[2] * shape[3] > 10 ** 6:
        pytest.skip("long on the executor")
    x, dz = _rows(shape, dtype, 100, offset=0.5), _rows(shape, dtype, 101, scale=0.1)
    ga, be = _params(shape[1], 102)
    kept = None if keep == "x" else stored_values(x, keep)[0]
    ref = Exact(x, groups, ga, be, 1e-3, "silu", kept, dz)
    z, saved = group_norm_act(x, groups, ga, be, eps=1e-3, keep=keep)
    ref.check(z, "z")
    assert ((saved.mean.cpu().double().flatten() - ref.mean).abs() <= 64 * U * (ref.mean.abs() + 1 / ref.rstd)).all()
    assert ((saved.rstd.cpu().double().flatten() - ref.rstd).abs() <= 64 * U * ref.rstd).all()
    for got, what in zip(group_norm_act_backward(dz, saved), ("dx", "dgamma", "dbeta")):
        ref.check(got, what)


@pytest.mark.parametrize("case", SPLIT)
def test_captured_split_forms(case):
    """captured, replayed with new inputs and eager calls between the replays: equal to the eager result"""
    if DEV != "cuda":
        pytest.skip("graphs")
    from yolov5m_amd.group_norm import group_norm_act, group_norm_act_backward
    shape, groups, dtype = case
    ga, be = _params(shape[1], 103)

    def step(x, dz):
        z, saved = group_norm_act(x, groups, ga, be, keep="e4m3")
        return (z, *group_norm_act_backward(dz, saved))
    x, dz = _rows(shape, dtype, 104), _rows(shape, dtype, 105)
    step(x, dz)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(x, dz)
    for seed in (106, 107, 108):
        x.copy_(_rows(shape, dtype, seed))
        dz.copy_(_rows(shape, dtype, seed + 50))
        g.replay()
        want = step(x, dz)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, out)), seed


def near(ref, got, what):
    """Exact.check, which a NaN passes (no comparison with it is true), of an output that has to be finite"""
    assert torch.isfinite(got).all(), (what, int((~torch.isfinite(got)).sum()))
    ref.check(got, what)


@pytest.mark.parametrize("keep", ["x", "e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "fp16"])
def test_every_output_is_finite(dtype, keep):
    from yolov5m_amd.group_norm import group_norm_act, group_norm_act_backward
    for shape, groups in CASES:
        x, dz = _rows(shape, dtype, 115, offset=0.5), _rows(shape, dtype, 116, scale=0.1)
        for act in ("silu", None):
            z, saved = group_norm_act(x, groups, *_params(shape[1], 117), eps=1e-3, act=act, keep=keep)
            assert all(torch.isfinite(t).all() for t in (z, saved.mean, saved.rstd, *group_norm_act_backward(dz, saved))), (shape, groups, act)


# (samples, channels, rows, groups): long enough for the split form, one chunk with many rows side by side where there are few channels
OUTLIER = [((1, 8, 25600), 1), ((1, 8, 5000), 4), ((1, 16, 25600), 4), ((1, 48, 25600), 6), ((1, 768, 2600), 1)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", OUTLIER)
def test_an_outlier_first_row_at_every_width(case, dtype):
    """a first row of 1000 before N(0, 1): whatever shares a chunk with it, the statistics and outputs stay within the bounds of a computation
    that sums about the mean (rstd: the f64 sums leave the rounding to f32, two u)"""
    from yolov5m_amd.group_norm import group_norm_act
    shape, groups = case
    if DEV != "cuda" and shape[1] > 100:
        pytest.skip("long on the executor")
    x = torch.randn((shape[0], shape[2], shape[1]), generator=torch.Generator().manual_seed(110))
    x[:, 0] = 1000.0
    x = x.to(DT[dtype]).movedim(-1, 1).to(DEV)
    ref = Exact(x, groups, None, None, 1e-5, None)
    z, saved = group_norm_act(x, groups, act=None, keep="x")
    near(ref, z, "z")
    assert ((saved.rstd.cpu().double().flatten() - ref.rstd).abs() <= 8 * U * ref.rstd).all()
    assert ((saved.mean.cpu().double().flatten() - ref.mean).abs() <= 8 * U * (ref.mean.abs() + 1 / ref.rstd)).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 50, 100, 5000])
def test_statistics_over_the_whole_range_of_the_type(rows, dtype):
    """finite inputs whose squares leave f32: a first row of 1e17 / 1e18 / 1e30 before N(0, 1), maps around 1e18 and 3e37, and one of 1e-25 (its
    squares are below f32, as its eps is). Held and split form alike, within the bounds of ordinary inputs"""
    from yolov5m_amd.group_norm import group_norm_act
    for first, scale, offset, eps in ((1e17, 1.0, 0.0, 1e-5), (1e18, 1.0, 0.0, 1e-5), (1e30, 1.0, 0.0, 1e-5), (None, 1e17, 1e18, 1e-5), (None, 3e37, 0.0, 1e-5),
                                      (None, 1e-25, 0.0, 1e-37)):
        x = torch.randn((2, rows, 16), generator=torch.Generator().manual_seed(111)).clamp(-4, 4) * scale + offset
        if first is not None:
            x[:, 0] = first
        x = x.to(DT[dtype]).movedim(-1, 1).to(DEV)
        ref = Exact(x, 4, None, None, eps, None)
        z, saved = group_norm_act(x, 4, act=None, eps=eps, keep="x")
        assert ((saved.rstd.cpu().double().flatten() - ref.rstd).abs() <= 64 * U * ref.rstd).all(), (first, scale)
        near(ref, z, "z")


@pytest.mark.parametrize("keep", ["x", "e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [3, 50, 5000])
def test_gradients_of_very_large_inputs(rows, dtype, keep):
    """inputs from 1e12 to 1e30, where rstd^2 and sums of dz x leave f32: the gradients are those of the normalised values, within the bounds of
    ordinary inputs"""
    from yolov5m_amd.group_norm import group_norm_act, group_norm_act_backward
    for scale, offset in ((1e12, 0.0), (1e25, 0.0), (1e30, 0.0), (1e20, 1e21)):
        x = (torch.randn((2, rows, 16), generator=torch.Generator().manual_seed(112)) * scale + offset).to(DT[dtype]).movedim(-1, 1).to(DEV)
        dz = (_rows((2, 16, rows), "f32", 113) * 1e10).to(DT[dtype])
        ga, be = _params(16, 114)
        kept = None if keep == "x" else stored_values(x, keep)[0]
        ref = Exact(x, 4, ga, be, 1e-3, "silu", kept, dz)
        z, saved = group_norm_act(x, 4, ga, be, eps=1e-3, keep=keep)
        near(ref, z, "z")
        for got, what in zip(group_norm_act_backward(dz, saved), ("dx", "dgamma", "dbeta")):
            near(ref, got, what)


@pytest.mark.parametrize("keep", ["e4m3", "int8"])
def test_cbl_keeps_nothing_where_no_gradient_is_wanted(keep, monkeypatch):
    """no_grad, inference_mode and a frozen weight store no input in 8 bits; results are those of a training forward, up to the order in which the
    statistics are summed (a slice is cut at whole blocks only where codes are written): each is within 64 u of |xhat| + |mean| rstd <= 6 + 1
    of the formula, so the two within 128 u 7 = 5.4e-5"""
    from yolov5m_amd import act8
    from yolov5m_amd.model import CBL
    real, calls = act8.act8_store, []
    monkeypatch.setattr(act8, "act8_store", lambda *a, **k: (calls.append(1), real(*a, **k))[1])
    m = CBL(16, 24, 3, 1, 1, norm_groups=8, keep=keep).to(DEV)
    x = torch.randn(2, 16, 6, 5, generator=torch.Generator().manual_seed(118)).to(DEV)
    want = m(x)
    assert len(calls) == 1
    m.eval()
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            assert (m(x) - want).abs().max() <= 5.4e-5
    assert len(calls) == 1
    m.cbl[0].weight.requires_grad_(False)
    m(x).sum().backward()                                             # (the norm's parameters still train)
    assert len(calls) == 1 and m.cbl[1].weight.grad is not None


@pytest.mark.parametrize("frozen", [True, False])
def test_forward_mode_is_refused(frozen):
    """a tangent is never dropped silently: with frozen parameters (no autograd node) and with trained ones"""
    import torch.autograd.forward_ad as fw
    from yolov5m_amd.group_norm import GroupNormAct
    layer = GroupNormAct(4, 16).to(DEV).requires_grad_(not frozen)
    x = _rows((2, 16, 3, 3), "f32", 119)
    with fw.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError), match="forward|jvp"):
            layer(fw.make_dual(x, torch.ones_like(x)))
        assert fw.unpack_dual(layer(x)).tangent is None


@pytest.mark.parametrize("case", [((16384, 768), 32, True), ((3, 64, 5, 5), 4, True), ((1, 768, 20, 20), 32, False), ((2, 24, 37), 3, True), ((2, 96, 130, 50), 32, False),
                                  ((1, 8, 5000), 1, False)])
def test_workspace_of_the_form_that_runs(case):
    """maps that one launch holds need no workspace forward, and none is touched; a null pointer is taken there. Longer ones, and the backward,
    write within what the size functions say, whatever the alignment and the kept form. (One 20 x 20 x 768 map is held without an 8-bit form
    only: with one its slices are whole blocks, lcm(24, 32) = 96 channels wide, and eight workgroups are too few for 16 rows a thread.)"""
    import yolov5m_amd.group_norm  # noqa: F401
    from yolov5m_amd import _lib
    from yolov5m_amd.act8 import FORMATS
    L = _lib.lib()
    (n, c, *sp), g, held = case
    s = 1
    for v in sp:
        s *= v
    wsb, bwb = L.y5m_gn_act_workspace_bytes(n, s, c, g), L.y5m_gn_act_bwd_workspace_bytes(n, s, c, g)
    assert (wsb == 0) == held and bwb >= 8 * n * c
    if held:
        assert bwb <= 8 * n * (c + g)
    if DEV != "cuda" and n * c * s > 10 ** 6:
        return
    ldq, cb = -(-c // 8) * 8, -(-c // 32)
    for odd in (0, 1):
        buf = torch.randn(n * s * c + odd, generator=torch.Generator().manual_seed(128)).to(DEV)
        x = buf[odd:].view(n, s, c)
        ref = Exact(x.transpose(1, 2), g, None, None, 1e-5, "silu", None, x.transpose(1, 2))
        for fmt in (0, *FORMATS.values()):
            z, dx = torch.empty((n, s, c), device=DEV), torch.empty((n, s, c), device=DEV)
            stat = torch.empty(2 * n * g, device=DEV)
            q, sc = torch.empty((n * s, ldq), dtype=torch.uint8, device=DEV), torch.empty((n * s, cb), dtype=torch.uint8, device=DEV)
            ws, bw = (torch.full((b + 64,), 7, dtype=torch.uint8, device=DEV) for b in (wsb, bwb))
            p = stat.data_ptr()
            _lib.check(L.y5m_gn_act(x.data_ptr(), s * c, c, None, None, n, s, c, g, 1e-5, 1, z.data_ptr(), s * c, c, p, p + 4 * n * g, q.data_ptr() if fmt else None,
                                    ldq, sc.data_ptr() if fmt else None, fmt, None if held else ws.data_ptr(), wsb, 0, _lib.stream_ptr()), "y5m_gn_act")
            near(ref, z.transpose(1, 2), "z")
            _lib.check(L.y5m_gn_act_bwd(x.data_ptr(), s * c, c, x.data_ptr(), s * c, c, q.data_ptr() if fmt else None, ldq, sc.data_ptr() if fmt else None, fmt, None,
                                        None, p, p + 4 * n * g, n, s, c, g, 1, dx.data_ptr(), s * c, c, None, None, bw.data_ptr(), bwb, 0, _lib.stream_ptr()),
                       "y5m_gn_act_bwd")
            if fmt == 0:
                near(ref, dx.transpose(1, 2), "dx")
            assert (ws[wsb:] == 7).all() and (bw[bwb:] == 7).all()
    # one byte too few is refused
    if not held:
        assert L.y5m_gn_act(x.data_ptr(), s * c, c, None, None, n, s, c, g, 1e-5, 1, z.data_ptr(), s * c, c, p, p + 4 * n * g, None, 0, None, 0, ws.data_ptr(), wsb - 1, 0,
                            _lib.stream_ptr()) != 0
    assert L.y5m_gn_act_bwd(x.data_ptr(), s * c, c, x.data_ptr(), s * c, c, None, 0, None, 0, None, None, p, p + 4 * n * g, n, s, c, g, 1, dx.data_ptr(), s * c, c, None,
                            None, bw.data_ptr(), bwb - 1, 0, _lib.stream_ptr()) != 0


@pytest.mark.parametrize("keep", ["x", "e4m3", "int8"])
@pytest.mark.parametrize("case", [(16, 32, 1, 1), (16, 24, 3, 1), (16, 32, 3, 2), (3, 16, 3, 1)])
def test_cbl_with_group_norm_in_bf16(case, keep):
    """the block's bf16 path, stage by stage against 64 bits on the operands that the stage before left: convolution output (bf16: half a step,
    2^-8, of sums of at most 288 products in f32, 300 u), norm and its gradient (Exact's bounds), and the convolution's gradients, whose bounds
    carry the error of the bf16 dy on: sum |err dy| |operand| + 300 u sum |dy| |operand|, and half a step where the result is bf16 (dx)"""
    from yolov5m_amd.model import CBL, _ConvKeptFn
    cin, cout, k, s = case
    torch.manual_seed(129)
    m = CBL(cin, cout, k, s, k // 2, norm_groups=8, keep=keep).to(DEV)
    m.compute_dtype = "bf16"
    with torch.no_grad():
        m.cbl[1].weight.copy_(_params(cout, 130)[0])
        m.cbl[1].bias.copy_(_params(cout, 130)[1])
    x = torch.randn(2, cin, 10, 6, generator=torch.Generator().manual_seed(131)).to(DEV).requires_grad_()
    z = m(x)
    w = torch.randn(z.shape, generator=torch.Generator().manual_seed(132)).to(DEV)
    (z * w).sum().backward()
    half, conv = 2.0 ** -8, dict(stride=s, padding=k // 2)
    b64 = lambda t: t.detach().cpu().bfloat16().double()
    xd, wd = b64(x), b64(m.cbl[0].weight)
    y = _ConvKeptFn.apply(x.detach(), m.cbl[0].weight.detach(), m)
    ref = F.conv2d(xd, wd, **conv)
    assert y.dtype == torch.bfloat16
    assert ((y.cpu().double() - ref).abs() <= half * ref.abs() + (1 + half) * 300 * U * F.conv2d(xd.abs(), wd.abs(), **conv)).all()
    nhwc = lambda t: t.contiguous(memory_format=torch.channels_last)
    norm = Exact(y, 8, m.cbl[1].weight, m.cbl[1].bias, 1e-3, "silu", None if keep == "x" else stored_values(y, keep)[0], w.bfloat16())
    near(norm, z.detach().bfloat16(), "z")
    assert torch.equal(z.detach().bfloat16().float(), z.detach())
    near(norm, m.cbl[1].weight.grad, "dgamma")
    near(norm, m.cbl[1].bias.grad, "dbeta")
    img = lambda t: t.reshape(2, *y.shape[2:], cout).movedim(-1, 1)
    dy, err = img(norm.dx), img(norm.dx_tol + half * (norm.dx.abs() + norm.dx_tol))
    xk = xd if keep == "x" else stored_values(nhwc(x.detach().bfloat16()), keep)[0].movedim(-1, 1)
    for got, op, grad, rnd in ((x.grad, wd, lambda o, d: torch.nn.grad.conv2d_input(xd.shape, o, d, **conv), half),
                               (m.cbl[0].weight.grad, xk, lambda o, d: torch.nn.grad.conv2d_weight(o, wd.shape, d, **conv), 0.0)):
        want = grad(op, dy)
        tol = grad(op.abs(), err + 300 * U * dy.abs())
        assert ((got.cpu().double() - want).abs() <= tol + rnd * (want.abs() + tol)).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [4, 50, 5000])
def test_half_of_the_largest_value(rows, dtype):
    """maps of +-1.6e38: rstd is below f32's normal range (its step there, 2^-149 of 6e-39, is 4 u) and z is +-1"""
    from yolov5m_amd.group_norm import group_norm_act, group_norm_act_backward
    x = torch.full((2, rows, 16), 1.6e38)
    x[:, ::2, ::3] = -1.6e38
    x[:, 1::2, 1::3] = -1.6e38
    x = x.to(DT[dtype]).movedim(-1, 1).to(DEV)
    dz = (_rows((2, 16, rows), "f32", 133) * 1e20).to(DT[dtype])
    ref = Exact(x, 4, None, None, 1e-5, None, None, dz)
    z, saved = group_norm_act(x, 4, act=None, keep="x")
    near(ref, z, "z")
    assert ((saved.rstd.cpu().double().flatten() - ref.rstd).abs() <= 8 * U * ref.rstd).all()
    for got, what in zip(group_norm_act_backward(dz, saved), ("dx", "dgamma", "dbeta")):
        near(ref, got, what)


@pytest.mark.parametrize("rows", [1, 40, 5000])
def test_equal_values_far_from_zero(rows):
    """groups of one value in 16 bits: xhat is 0 and z = act(bias) to the type's rounding, however large the value and rstd are"""
    from yolov5m_amd.group_norm import group_norm_act
    ga, be = _params(16, 134)
    for dtype, value, eps in (("bf16", 1e10, 1e-5), ("bf16", -1e37, 1e-5), ("bf16", 1.5e38, 1e-3), ("fp16", 6e4, 1e-12), ("bf16", 300.0, 1e-14)):
        x = torch.full((2, rows, 16), value).to(DT[dtype]).movedim(-1, 1).to(DEV)
        z, _ = group_norm_act(x, 4, ga, be, eps=eps, act=None)
        b = be.to(DT[dtype]).view(1, 16, 1).expand(2, 16, rows)
        assert torch.equal(z, b), (dtype, value, float((z - b).abs().max()))
