"""The channels-last group normalisation and the 8-bit kept activations, as cases to be timed and compared.

`run` makes ONE pass through an operator: in its plain form (elementary torch operations in 32 bits, rounded once at the end) or,
where `own` is true, through the framework's own entry points. `exact` computes the same outputs from the definitions in 64 bits.

Four kinds of case:
  norm   group norm + activation, forward only (inference)
  step   group norm + activation forward, then its backward from what the forward kept: the input itself, or the input in 8 bits
  keep   an activation stored in 8 bits and read back
  wgrad  a pointwise convolution's input stored in 8 bits, then its weight (and bias) gradient from the stored form

Tensors are (N, C, H, W) with channels last in memory: rows of C values, N * H * W of them.

An 8-bit stored activation: each row is cut into blocks of 32 consecutive channels (the last one of a row may be shorter). A block has
one power-of-two scale 2^e, e the smallest integer with max|x| <= top * 2^e, at least -117; top is 448 for "e4m3" and 127 for "int8".
A value is held as x / 2^e rounded to the nearest value of the format, ties to even. Values are first limited to 1.875 * 2^E, E the
largest exponent of x's type, so that nothing read back overflows; a block with a value that is not finite reads back as NaN.
"""
import math

import torch

own = False

EPS = 1e-3                        # the eps of the network's normalisations
_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "fp16": 2}
_LIMIT = {torch.float32: 1.875 * 2.0 ** 127, torch.bfloat16: 1.875 * 2.0 ** 127, torch.float16: 1.875 * 2.0 ** 15}


# ---------------------------------------------------------------------------------------------- the cases
def _case(name, kind, n, c, h, w, dtype, groups=0, act="silu", keep="none", cout=0, bias=False):
    return {"name": name, "kind": kind, "n": n, "c": c, "h": h, "w": w, "dtype": dtype, "groups": groups, "act": act, "keep": keep,
            "cout": cout, "bias": bias}


def listed():
    return [
        # one image at inference, the deepest stage of the 640 x 640 network: the call's latency is what counts
        _case("norm_image_20", "norm", 1, 768, 20, 20, "bf16", groups=32),
        # the forward benchmark's batch of 32 at the first wide stage: 3 channels a group, larger than the caches hold at once
        _case("norm_batch_160", "norm", 32, 96, 160, 160, "bf16", groups=32),
        # a rectangular image's head map: 255 channels, rows that no vector load divides, no activation
        _case("norm_odd_f32", "norm", 3, 255, 13, 19, "f32", groups=15, act="none"),
        # training at batch 64: the 40 x 40 stage with its input kept in 8 bits
        _case("step_40_e4m3", "step", 64, 384, 40, 40, "bf16", groups=32, keep="e4m3"),
        # training at batch 64 with the input kept whole
        _case("step_80_whole", "step", 64, 192, 80, 80, "bf16", groups=32, keep="x"),
        # the widest maps, where 8 bits save the most memory
        _case("step_160_int8", "step", 64, 96, 160, 160, "bf16", groups=32, keep="int8"),
        # a small odd map in half precision
        _case("step_odd_fp16", "step", 5, 36, 21, 37, "fp16", groups=12, keep="e4m3"),
        # a whole training activation written in 8 bits and read back
        _case("keep_160_e4m3", "keep", 64, 96, 160, 160, "bf16", keep="e4m3"),
        # a short odd one in single precision
        _case("keep_odd_f32", "keep", 2, 100, 31, 33, "f32", keep="int8"),
        # the pooling block's output convolution: the largest pointwise weight
        _case("wgrad_20_e4m3", "wgrad", 64, 1536, 20, 20, "bf16", keep="e4m3", cout=768),
        # the narrowest pointwise layer over the widest maps: many rows, a small weight
        _case("wgrad_160_int8", "wgrad", 64, 96, 160, 160, "bf16", keep="int8", cout=48),
        # a head convolution with its bias, odd sizes, single precision
        _case("wgrad_odd_f32", "wgrad", 3, 100, 11, 17, "f32", keep="e4m3", cout=255, bias=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    top_bytes = max(work(c)["bytes"] for c in listed())
    top_flops = max(work(c)["flops"] for c in listed())
    while True:
        kind = rng.choice(["norm", "norm", "step", "step", "keep", "wgrad"])
        c = _log_int(rng, 8, 1536)
        n = _log_int(rng, 1, 64)
        h, w = _log_int(rng, 1, 160), _log_int(rng, 1, 160)
        if rng.random() < 0.5:
            c = max(8, c // 8 * 8)          # half of the widths are whole vectors, as the network's are
        groups = 0
        if kind in ("norm", "step"):
            groups = rng.choice([g for g in range(1, min(c, 64) + 1) if c % g == 0])
            if c // groups * h * w < 8:     # (a mean over fewer values says little)
                continue
        case = {"kind": kind, "n": n, "c": c, "h": h, "w": w, "dtype": rng.choice(["bf16", "bf16", "fp16", "f32"]), "groups": groups,
                "act": rng.choice(["silu", "silu", "none"]),
                "keep": {"norm": "none", "step": rng.choice(["x", "e4m3", "int8"])}.get(kind, rng.choice(["e4m3", "int8"])),
                "cout": _log_int(rng, 1, 768) if kind == "wgrad" else 0, "bias": kind == "wgrad" and rng.random() < 0.5}
        wk = work(case)
        if wk["bytes"] <= top_bytes and wk["flops"] <= top_flops:
            return case


def work(case):
    """bytes and operations that one pass cannot do without: each input read once, each output written once; what is kept between a
    forward and its backward is written once and read once"""
    m, c, sz = case["n"] * case["h"] * case["w"], case["c"], _SIZE[case["dtype"]]
    kept = m * c + m * ((c + 31) // 32)
    if case["kind"] == "norm":
        return {"bytes": 2 * m * c * sz + 8 * c, "flops": 12 * m * c}
    if case["kind"] == "step":
        # forward: x, z, the kept form (nothing is written where x itself is kept); backward: the kept form, dz, dx
        k = m * c * sz if case["keep"] == "x" else 2 * kept
        return {"bytes": 4 * m * c * sz + k + 24 * c, "flops": 40 * m * c}
    if case["kind"] == "keep":
        return {"bytes": 2 * m * c * sz + 2 * kept, "flops": 6 * m * c}
    n = case["cout"]
    return {"bytes": m * c * sz + 2 * kept + m * n * sz + 4 * n * c + (4 * n if case["bias"] else 0), "flops": 2 * m * n * c}


def prepare(case, seed):
    """what a training or serving program has in hand: maps whose channels differ in mean and spread, as a convolution's outputs do"""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    n, c, h, w, dt = case["n"], case["c"], case["h"], case["w"], _DT[case["dtype"]]

    def rows(ch, scale, offset):
        t = torch.randn((n, h, w, ch), generator=g, device="cuda", dtype=torch.float32)
        return t.mul_(scale).add_(offset).to(dt).movedim(-1, 1)

    spread = torch.exp(0.5 * torch.randn(c, generator=g, device="cuda"))
    centre = 0.5 * torch.randn(c, generator=g, device="cuda")
    st = {"case": case, "x": rows(c, spread, centre)}
    if case["kind"] in ("norm", "step"):
        st["gamma"] = 1.0 + 0.2 * torch.randn(c, generator=g, device="cuda")
        st["beta"] = 0.2 * torch.randn(c, generator=g, device="cuda")
    if case["kind"] == "step":
        st["dz"] = rows(c, torch.full((c,), 0.05, device="cuda"), 0.0)
    if case["kind"] == "wgrad":
        st["dy"] = rows(case["cout"], torch.full((case["cout"],), 0.05, device="cuda"), 0.0)
    return st


# ---------------------------------------------------------------------------------------------- plain forms (32 bits)
def _plain_round_trip(x, fmt):
    """(N, C, H, W) -> float32 (N, H, W, C): the values that the 8-bit form of x stands for"""
    xr = x.movedim(1, -1).float()
    c = xr.shape[-1]
    xb = torch.nn.functional.pad(xr, (0, -c % 32)).unflatten(-1, (-1, 32))
    bad = ~torch.isfinite(xb).all(-1, keepdim=True)
    xb = xb.clamp(-_LIMIT[x.dtype], _LIMIT[x.dtype])
    m, k = torch.frexp(xb.abs().amax(-1, keepdim=True))
    e = torch.where(m > 0.875, k - 8, k - 9) if fmt == "e4m3" else torch.where(m > 127.0 / 128.0, k - 6, k - 7)
    e = e.clamp(min=-117)
    v = torch.ldexp(xb, -e)
    v = v.to(torch.float8_e4m3fn).float() if fmt == "e4m3" else torch.round(v)
    v = torch.where(bad, torch.full_like(v, float("nan")), torch.ldexp(v, e))
    return v.flatten(-2)[..., :c]


def _plain_norm(x, gamma, beta, groups, act):
    """-> z (rounded, (N, C, H, W)), mean and rstd (N, 1, 1, G, 1) in float32"""
    xg = x.movedim(1, -1).float().unflatten(-1, (groups, -1))
    mean = xg.mean((1, 2, 4), keepdim=True)
    rstd = torch.rsqrt((xg - mean).square().mean((1, 2, 4), keepdim=True) + EPS)
    t = ((xg - mean) * rstd).flatten(-2) * gamma + beta
    z = t * (1.0 / (1.0 + torch.exp(-t))) if act == "silu" else t
    return z.to(x.dtype).movedim(-1, 1), mean, rstd


def _plain_norm_grad(dz, xk, mean, rstd, gamma, beta, groups, act, dtype):
    """dz (N, C, H, W); xk: the kept input, float32 (N, H, W, C) -> dx, dgamma, dbeta"""
    xhat = (xk.unflatten(-1, (groups, -1)) - mean) * rstd
    dt = dz.movedim(1, -1).float()
    if act == "silu":
        t = xhat.flatten(-2) * gamma + beta
        s = 1.0 / (1.0 + torch.exp(-t))
        dt = dt * (s * (1.0 + t * (1.0 - s)))
    dgamma = (dt * xhat.flatten(-2)).sum((0, 1, 2))
    dbeta = dt.sum((0, 1, 2))
    d = (dt * gamma).unflatten(-1, (groups, -1))
    dx = rstd * (d - d.mean((1, 2, 4), keepdim=True) - xhat * (d * xhat).mean((1, 2, 4), keepdim=True))
    return dx.flatten(-2).to(dtype).movedim(-1, 1), dgamma, dbeta


def _run_plain(st):
    case, x = st["case"], st["x"]
    if case["kind"] == "norm":
        return _plain_norm(x, st["gamma"], st["beta"], case["groups"], case["act"])[0]
    if case["kind"] == "step":
        z, mean, rstd = _plain_norm(x, st["gamma"], st["beta"], case["groups"], case["act"])
        xk = x.movedim(1, -1).float() if case["keep"] == "x" else _plain_round_trip(x, case["keep"])
        dx, dg, db = _plain_norm_grad(st["dz"], xk, mean, rstd, st["gamma"], st["beta"], case["groups"], case["act"], x.dtype)
        return {"z": z, "dx": dx, "dgamma": dg, "dbeta": db}
    if case["kind"] == "keep":
        return _plain_round_trip(x, case["keep"]).to(x.dtype).movedim(-1, 1)
    xk = _plain_round_trip(x, case["keep"]).flatten(0, 2)
    dy = st["dy"].movedim(1, -1).flatten(0, 2).float()
    out = {"dw": dy.t() @ xk}
    if case["bias"]:
        out["db"] = dy.sum(0)
    return out


# ---------------------------------------------------------------------------------------------- the framework's operators
def _run_own(st):
    from yolov5m_amd.act8 import act8_load, act8_store, act8_wgrad
    from yolov5m_amd.group_norm import group_norm_act, group_norm_act_backward
    case, x = st["case"], st["x"]
    if case["kind"] == "norm":
        z, _ = group_norm_act(x, case["groups"], st["gamma"], st["beta"], eps=EPS, act=case["act"])
        return z
    if case["kind"] == "step":
        z, saved = group_norm_act(x, case["groups"], st["gamma"], st["beta"], eps=EPS, act=case["act"], keep=case["keep"])
        dx, dg, db = group_norm_act_backward(st["dz"], saved)
        return {"z": z, "dx": dx, "dgamma": dg, "dbeta": db}
    kept = act8_store(x, case["keep"])
    if case["kind"] == "keep":
        return act8_load(kept)
    dw, db = act8_wgrad(st["dy"], kept, bias=case["bias"])
    return {"dw": dw, "db": db} if case["bias"] else {"dw": dw}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------------- the definitions, in 64 bits
def _exact_stored(x, fmt, limit):
    """float64 (rows, C) -> what the 8-bit form stands for: the scale by trial against the definition, the rounding by the
    format's spacing around each value"""
    top = 448.0 if fmt == "e4m3" else 127.0
    out = torch.empty_like(x)
    for c0 in range(0, x.shape[1], 32):
        b = x[:, c0:c0 + 32]
        bad = ~torch.isfinite(b).all(1, keepdim=True)
        b = torch.minimum(torch.maximum(b, b.new_tensor(-limit)), b.new_tensor(limit))
        big = b.abs().max(1, keepdim=True).values
        e = torch.floor(torch.log2(big.clamp(min=2.0 ** -200))) - 12
        for _ in range(14):                                   # up to the first exponent that holds the block's largest value
            e = torch.where(big > top * torch.exp2(e), e + 1, e)
        e = torch.maximum(e, e.new_tensor(-117.0))
        v = b / torch.exp2(e)
        if fmt == "e4m3":                                     # 3 mantissa bits down to 2^-6, then the subnormal spacing 2^-9
            step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
        else:
            step = torch.ones_like(v)
        v = torch.round(v / step) * step * torch.exp2(e)
        out[:, c0:c0 + 32] = torch.where(bad, v.new_tensor(float("nan")), v)
    return out


def exact(case, seed):
    st = prepare(case, seed)
    x = st["x"]
    n, c = x.shape[:2]
    limit = _LIMIT[x.dtype]
    rows = x.movedim(1, -1).reshape(n, -1, c)                     # (N, S, C)
    if case["kind"] == "keep":
        out = torch.empty(rows.shape, dtype=torch.float64, device=x.device)
        for i in range(n):
            out[i] = _exact_stored(rows[i].double(), case["keep"], limit)
        return out.reshape(n, *x.shape[2:], c).movedim(-1, 1)
    if case["kind"] == "wgrad":
        dy = st["dy"].movedim(1, -1).reshape(n, -1, case["cout"])
        dw = torch.zeros((case["cout"], c), dtype=torch.float64, device=x.device)
        db = torch.zeros(case["cout"], dtype=torch.float64, device=x.device)
        for i in range(n):
            d = dy[i].double()
            dw += d.t() @ _exact_stored(rows[i].double(), case["keep"], limit)
            db += d.sum(0)
        return {"dw": dw, "db": db} if case["bias"] else {"dw": dw}
    groups, gamma, beta = case["groups"], st["gamma"].double(), st["beta"].double()
    per = c // groups
    z = torch.empty(rows.shape, dtype=torch.float64, device=x.device)
    grad = case["kind"] == "step"
    if grad:
        dzr = st["dz"].movedim(1, -1).reshape(n, -1, c)
        dx = torch.empty_like(z)
        dg, db = torch.zeros_like(gamma), torch.zeros_like(gamma)
    for i in range(n):
        v = rows[i].double()
        s = v.shape[0]
        mean = (v.sum(0).view(groups, per).sum(1) / (s * per)).repeat_interleave(per)
        var = ((v - mean) ** 2).sum(0).view(groups, per).sum(1) / (s * per)
        r = (1.0 / torch.sqrt(var + EPS)).repeat_interleave(per)
        t = (v - mean) * r * gamma + beta
        z[i] = t * torch.sigmoid(t) if case["act"] == "silu" else t
        if grad:
            k = v if case["keep"] == "x" else _exact_stored(v, case["keep"], limit)
            xh = (k - mean) * r
            d = dzr[i].double()
            if case["act"] == "silu":
                t = xh * gamma + beta
                s_ = torch.sigmoid(t)
                d = d * s_ * (1 + t * (1 - s_))
            dg += (d * xh).sum(0)
            db += d.sum(0)
            a = ((d * gamma).sum(0).view(groups, per).sum(1) / (s * per)).repeat_interleave(per)
            b = ((d * gamma * xh).sum(0).view(groups, per).sum(1) / (s * per)).repeat_interleave(per)
            dx[i] = r * (d * gamma - a - xh * b)

    def whole(t):
        return t.reshape(n, *x.shape[2:], c).movedim(-1, 1)
    return {"z": whole(z), "dx": whole(dx), "dgamma": dg, "dbeta": db} if grad else whole(z)
