"""The layers behind the large actor's sensor preparation, for timing and comparison.

Three operators: group norm with an activation over channels-last planes (the
convolution stems), the routing of tokens to experts with the order of their
choices by expert, and products in microscaled 4-bit floating point (the
experts' weights while acting).  `run` with `own` false is their plain form,
with `own` true the calls of turbinator_c_amd.layers; `exact` restates them in
64 bits.
"""
import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5
BLOCK, PAD = 32, 128  # values that share a scale; k is padded to whole 64-byte rows of codes


def listed():
    return [
        # One environment acting: its LiDAR planes (16 x 128 bins) behind the
        # first convolution.
        {"name": "norm_act_1", "entry": "norm", "n": 1, "p": 2048, "c": 64, "g": 8, "pitch": 64,
         "act": "silu", "dtype": "f32"},
        # A training batch of 1,024 environments' four cameras (64 x 64,
        # halved by the convolution's stride).
        {"name": "norm_cameras_4096", "entry": "norm", "n": 4096, "p": 1024, "c": 64, "g": 8,
         "pitch": 64, "act": "silu", "dtype": "bf16"},
        # Planes with odd sizes, a slice of wider rows (two stems written
        # side by side).
        {"name": "norm_odd_257", "entry": "norm", "n": 257, "p": 1023, "c": 48, "g": 6,
         "pitch": 52, "act": "gelu", "dtype": "f32"},
        # The backward pass at the trainer's default batch, and of a training
        # batch of LiDAR planes.
        {"name": "norm_back_32", "entry": "norm_back", "n": 32, "p": 512, "c": 128, "g": 8,
         "pitch": 128, "act": "silu", "dtype": "f32"},
        {"name": "norm_back_1024", "entry": "norm_back", "n": 1024, "p": 2048, "c": 64, "g": 8,
         "pitch": 64, "act": "silu", "dtype": "bf16"},
        # The ten tokens of each of 32 environments to two of eight experts.
        {"name": "route_320", "entry": "route", "t": 320, "e": 8, "k": 2, "groups": 1, "kept": 1,
         "score": "softmax", "bias": False, "renorm": True, "padded": False, "dtype": "f32"},
        # The tokens of 16,384 environments to four of 64 experts in groups,
        # with a balance bias and padding tokens.
        {"name": "route_163840", "entry": "route", "t": 163840, "e": 64, "k": 4, "groups": 8,
         "kept": 4, "score": "sigmoid", "bias": True, "renorm": True, "padded": True,
         "dtype": "bf16"},
        # The gradient of the routing weights for a training batch.
        {"name": "route_back_40961", "entry": "route_back", "t": 40961, "e": 128, "k": 8,
         "score": "softmax", "renorm": False, "dtype": "bf16"},
        # A training batch's activations to 4 bits and back (an odd width).
        {"name": "mx4_round_40960", "entry": "round", "m": 40960, "k": 2000, "dtype": "bf16"},
        # One environment's ten tokens through one layer.
        {"name": "mx4_product_10", "entry": "product", "m": 10, "n": 2048, "k": 2048,
         "experts": 1, "top": 1, "act": "none", "bias": True, "dtype": "bf16"},
        # Two of eight experts for 410 environments' tokens.
        {"name": "mx4_experts_4100", "entry": "product", "m": 4100, "n": 2048, "k": 1024,
         "experts": 8, "top": 2, "act": "silu", "bias": True, "dtype": "bf16"},
        # A full batch of tokens through one wide layer.
        {"name": "mx4_product_16384", "entry": "product", "m": 16384, "n": 4096, "k": 4096,
         "experts": 1, "top": 1, "act": "none", "bias": False, "dtype": "bf16"},
    ]


def _size(rng, least, most):
    return min(most, int(math.exp(rng.uniform(math.log(least), math.log(most + 1)))))


def draw(rng):
    entry = rng.choice(["norm", "norm", "norm_back", "route", "route", "route_back", "round",
                        "product", "product"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    if entry in ("norm", "norm_back"):
        per, g = rng.choice([1, 2, 3, 4, 6, 8, 8, 16, 32]), rng.choice([1, 2, 4, 6, 8, 16, 32])
        c = per * g
        # At least 16 values to a group: with fewer the gradient all but cancels.
        p = max(_size(rng, 1, 16384), -(-16 // per))
        most = (1 << 28) if entry == "norm" else (1 << 27)
        if dtype == "f32":
            most //= 2
        n = _size(rng, 1, max(1, min(4096, most // (p * c))))
        pitch = c if rng.random() < 0.7 else c + rng.choice([1, 4, 8, 64])
        return {"entry": entry, "n": n, "p": p, "c": c, "g": g, "pitch": pitch,
                "act": rng.choice(["none", "silu", "silu", "gelu"]), "dtype": dtype}
    if entry in ("route", "route_back"):
        e = rng.choice([2, 4, 7, 8, 16, 24, 32, 64, 96, 128, 160, 256])
        k = rng.randint(1, min(8, e))
        limit = 10485760 if entry == "route" else 5242880
        t = _size(rng, 1, min(163840, limit // e))
        score, renorm = rng.choice(["softmax", "sigmoid"]), rng.random() < 0.6
        if entry == "route_back":
            return {"entry": entry, "t": t, "e": e, "k": k, "score": score, "renorm": renorm,
                    "dtype": dtype}
        groups = rng.choice([d for d in (1, 1, 2, 4, 8) if e % d == 0])
        kept = rng.randint(min(groups, -(-k * groups // e)), groups)
        return {"entry": entry, "t": t, "e": e, "k": k, "groups": groups, "kept": kept,
                "score": score, "bias": rng.random() < 0.5, "renorm": renorm,
                "padded": rng.random() < 0.3, "dtype": dtype}
    if entry == "round":
        k = _size(rng, 16, 8192)
        return {"entry": entry, "m": _size(rng, 1, min(163840, 81920000 // k)), "k": k,
                "dtype": dtype}
    n, k = _size(rng, 64, 4096), _size(rng, 64, 4096)
    experts = rng.choice([1, 1, 4, 8, 16])
    return {"entry": entry, "m": _size(rng, 1, 16384 if experts == 1 else 8192), "n": n, "k": k,
            "experts": experts, "top": 1 if experts == 1 else rng.randint(1, 2),
            "act": rng.choice(["none", "silu", "gelu"]), "bias": rng.random() < 0.5,
            "dtype": dtype}


# --------------------------------------------------------------------------
# Inputs


def _gen(seed):
    return torch.Generator(DEVICE).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, device=DEVICE, generator=g)


def _rand(g, *shape):
    return torch.rand(shape, device=DEVICE, generator=g)


def _planes(g, case):
    """[n, p, pitch] of a convolution's outputs: every channel with a mean and a size of its own."""
    n, p, pitch, dt = case["n"], case["p"], case["pitch"], TYPES[case["dtype"]]
    size, mean = 0.3 + 1.4 * _rand(g, pitch), 0.6 * _randn(g, pitch)
    out = torch.empty((n, p, pitch), dtype=dt, device=DEVICE)
    step = max(1, (1 << 25) // (p * pitch))
    for i in range(0, n, step):
        part = out[i:i + step]
        part.copy_(_randn(g, *part.shape) * size + mean)
    return out


def _norm_state(case, seed):
    g, c = _gen(seed), case["c"]
    s = {"x": _planes(g, case)[..., :c], "gamma": 1 + 0.2 * _randn(g, c),
         "beta": 0.2 * _randn(g, c)}
    if case["entry"] == "norm_back":
        s["dy"] = (_planes(g, {**case, "pitch": c}) * 0.01).contiguous()
        x = s["x"]
        mean = torch.empty((case["n"], case["g"]), device=DEVICE)
        rstd = torch.empty_like(mean)
        step = max(1, (1 << 25) // (case["p"] * c))
        for i in range(0, case["n"], step):
            v = x[i:i + step].double().reshape(-1, case["p"], case["g"], c // case["g"])
            mean[i:i + step] = v.mean(dim=(1, 3))
            rstd[i:i + step] = 1 / torch.sqrt(v.var(dim=(1, 3), unbiased=False) + EPS)
        s["mean"], s["rstd"] = mean, rstd
    return s


def _logits(g, t, e, dt):
    return (1.2 * _randn(g, t, e) + 0.5 * _randn(g, e)).to(dt)


def _close_call(case, logits, bias):
    """Rows whose order of biased scores hangs on less than 2e-6, a few
    roundings of their 32-bit sums."""
    e, k, groups, kept = case["e"], case["k"], case["groups"], case["kept"]
    x = logits.double()
    s = torch.softmax(x, dim=1) if case["score"] == "softmax" else torch.sigmoid(x)
    key = (s + bias.double()).view(-1, groups, e // groups)
    close = torch.zeros(len(logits), dtype=torch.bool, device=DEVICE)
    if kept < groups:
        best = key.sort(dim=2, descending=True).values[..., :2].sum(dim=2)
        order = best.sort(dim=1, descending=True)
        close |= order.values[:, kept - 1] - order.values[:, kept] < 2e-6
        keep = torch.zeros_like(best, dtype=torch.bool).scatter_(1, order.indices[:, :kept], True)
        key = torch.where(keep[..., None], key, -math.inf)
    top = key.reshape(-1, e).sort(dim=1, descending=True).values[:, :k + 1]
    return close | (top[:, :-1] - top[:, 1:] < 2e-6).any(dim=1)


def _route_state(case, seed):
    g, t, e = _gen(seed), case["t"], case["e"]
    dt = TYPES[case["dtype"]]
    s = {"logits": _logits(g, t, e, dt)}
    if case["entry"] == "route_back":
        best = s["logits"].float().sort(dim=1, descending=True, stable=True).indices
        s["experts"] = best[:, :case["k"]].to(torch.int32).contiguous()
        s["dw"] = 0.01 * _randn(g, t, case["k"])
        return s
    s["bias"] = None
    if case["bias"]:
        # As a balancing rule leaves it: whole steps of 0.001.
        s["bias"] = torch.round(20 * _randn(g, e)) * 0.001
        close = torch.cat([_close_call(case, s["logits"][i:i + 16384], s["bias"])
                           for i in range(0, t, 16384)])
        good = (~close).nonzero()[:, 0]
        if len(good):
            bad = close.nonzero()[:, 0]
            s["logits"][bad] = s["logits"][good[torch.arange(len(bad), device=DEVICE) % len(good)]]
        else:
            s["logits"].copy_(torch.arange(e, 0, -1, device=DEVICE) * 0.01)
            s["bias"].zero_()
    s["valid"] = None
    if case["padded"]:
        s["valid"] = (_rand(g, t) < 0.95).to(torch.uint8)
        s["logits"][s["valid"] == 0] = math.nan  # never read: padding holds what it holds
    return s


def _activations(g, m, k, dt):
    """Rows of a block's activations: a few channels far larger than the rest."""
    size = torch.exp(0.5 * _randn(g, k)) * torch.where(_rand(g, k) < 0.01, 20.0, 1.0)
    out = torch.empty((m, k), dtype=dt, device=DEVICE)
    for i in range(0, m, 16384):
        part = out[i:i + 16384]
        part.copy_(_randn(g, *part.shape) * size)
    return out


def _product_state(case, seed):
    g, m, n, k, experts = _gen(seed), case["m"], case["n"], case["k"], case["experts"]
    s = {"x": _activations(g, m, k, TYPES[case["dtype"]]), "rows": None, "offsets": None,
         "bounds": [0, m], "row_scale": None}
    w = _randn(g, experts * n, k) / math.sqrt(k)
    s["codes"], s["scales"] = _encode(w)
    s["bias"] = 0.1 * _randn(g, experts, n) if case["bias"] else None
    if experts > 1:
        # The routing of m tokens to `top` experts each, some experts liked
        # more than others, and the order of the choices by expert.
        liked = _randn(g, m, experts) + 0.5 * _randn(g, experts)
        choice = liked.topk(case["top"], dim=1).indices
        order = choice.reshape(-1).sort(stable=True)
        s["rows"] = (order.indices // case["top"]).to(torch.int32)
        count = torch.bincount(order.values, minlength=experts)
        s["offsets"] = torch.cat([count.new_zeros(1), count.cumsum(0)]).to(torch.int32)
        s["bounds"] = s["offsets"].tolist()
        s["row_scale"] = _rand(g, len(s["rows"]))
    return s


def prepare(case, seed):
    entry = case["entry"]
    if entry in ("norm", "norm_back"):
        s = _norm_state(case, seed)
    elif entry in ("route", "route_back"):
        s = _route_state(case, seed)
    elif entry == "round":
        s = {"x": _activations(_gen(seed), case["m"], case["k"], TYPES[case["dtype"]])}
    else:
        s = _product_state(case, seed)
    s["case"] = case
    if own:
        from turbinator_c_amd import layers
        s["layers"], s["stream"] = layers, torch.cuda.current_stream()
        if entry in ("norm", "norm_back"):
            need = layers.group_norm_workspace_bytes(case["n"], case["p"], case["c"], case["g"],
                                                     layers.DTYPES[s["x"].dtype],
                                                     entry == "norm_back")
            s["workspace"] = torch.empty(max(need, 1), dtype=torch.uint8, device=DEVICE)
        elif entry == "route":
            need = layers.expert_order_workspace_bytes(case["t"], case["e"], case["k"])
            s["workspace"] = torch.empty(max(need, 1), dtype=torch.uint8, device=DEVICE)
    return s


# --------------------------------------------------------------------------
# Plain forms, in 32 bits


def _sigmoid(x):
    return 1 / (1 + torch.exp(-x))


def _act(z, act):
    if act == "silu":
        return z * _sigmoid(z)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _act_slope(z, act):
    if act == "silu":
        s = _sigmoid(z)
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return (0.5 * (1 + torch.erf(z * math.sqrt(0.5))) +
                z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi)))
    return torch.ones_like(z)


def _grouped(v, groups):
    return v.reshape(*v.shape[:-1], groups, v.shape[-1] // groups)


def _plain_norm(s):
    case, x = s["case"], s["x"].float()
    v = _grouped(x, case["g"])
    mean = v.mean(dim=(1, 3), keepdim=True)
    d = v - mean
    rstd = 1 / torch.sqrt((d * d).mean(dim=(1, 3), keepdim=True) + EPS)
    z = (d * rstd).reshape(x.shape) * s["gamma"] + s["beta"]
    return {"y": _act(z, case["act"]).to(s["x"].dtype), "mean": mean.reshape(case["n"], -1),
            "rstd": rstd.reshape(case["n"], -1)}


def _plain_norm_back(s):
    case, x, groups = s["case"], s["x"].float(), s["case"]["g"]
    mean, rstd = s["mean"][:, None, :, None], s["rstd"][:, None, :, None]
    xh = (_grouped(x, groups) - mean) * rstd
    z = xh.reshape(x.shape) * s["gamma"] + s["beta"]
    dz = s["dy"].float() * _act_slope(z, case["act"])
    dxh = _grouped(dz * s["gamma"], groups)
    dx = rstd * (dxh - dxh.mean(dim=(1, 3), keepdim=True) -
                 xh * (dxh * xh).mean(dim=(1, 3), keepdim=True))
    return {"dx": dx.reshape(x.shape).to(s["x"].dtype),
            "dgamma": (dz * xh.reshape(x.shape)).sum(dim=(0, 1)), "dbeta": dz.sum(dim=(0, 1))}


def _scores(x, score):
    if score == "sigmoid":
        return _sigmoid(x)
    ex = torch.exp(x - x.max(dim=1, keepdim=True).values)
    return ex / ex.sum(dim=1, keepdim=True)


def _choose(case, x, bias, valid):
    """Experts and weights of each row of logits x, in x's precision."""
    t, e, k, groups, kept = len(x), case["e"], case["k"], case["groups"], case["kept"]
    s = _scores(x, case["score"])
    key = x if bias is None else s + bias.to(x.dtype)
    key = torch.where(x == -math.inf, -math.inf, key)
    if kept < groups:
        v = key.view(t, groups, e // groups)
        best = v.max(dim=2).values
        if bias is not None and e // groups > 1:
            second = v.sort(dim=2, descending=True).values[..., 1]
            best = best + torch.where(second == -math.inf, 0.0, second)
        keep = best.sort(dim=1, descending=True, stable=True).indices[:, :kept]
        mask = torch.zeros_like(best, dtype=torch.bool).scatter_(1, keep, True)
        key = torch.where(mask[..., None], v, -math.inf).view(t, e)
    order = key.sort(dim=1, descending=True, stable=True)
    experts, gone = order.indices[:, :k], order.values[:, :k] == -math.inf
    if valid is not None:
        gone = gone | (valid == 0)[:, None]
    w = torch.where(gone, 0.0, s.gather(1, experts))
    if case["renorm"]:
        total = w.sum(dim=1, keepdim=True)
        w = torch.where(total == 0, 0.0, w / total)
    return torch.where(gone, -1, experts), w * 2.5


def _order(experts, weights, e):
    """The choices sorted by expert: offsets, token and weight of each row, row of each choice."""
    t, k = experts.shape
    flat = experts.reshape(-1)
    # Dropped choices (-1) go behind every expert's.
    order = torch.where(flat < 0, e, flat).sort(stable=True)
    live = order.values < e
    tokens = torch.where(live, order.indices // k, -1)
    rows = torch.arange(t * k, device=DEVICE)
    positions = torch.empty_like(flat).scatter_(0, order.indices, torch.where(live, rows, -1))
    count = torch.zeros(e + 1, dtype=torch.int64, device=DEVICE)
    count.scatter_add_(0, order.values, torch.ones_like(order.values))
    offsets = torch.cat([count.new_zeros(1), count[:e].cumsum(0)])
    row_weights = torch.where(live, weights.reshape(-1)[order.indices], 0.0)
    return {"offsets": offsets.to(torch.int32), "tokens": tokens.to(torch.int32),
            "positions": positions.view(t, k).to(torch.int32), "row_weights": row_weights}


def _plain_route(s):
    experts, weights = _choose(s["case"], s["logits"].float(), s["bias"], s["valid"])
    return {"experts": experts.to(torch.int32), "weights": weights,
            **_order(experts, weights, s["case"]["e"])}


def _plain_route_back(s):
    case, x = s["case"], s["logits"].float()
    at, g = s["experts"].long(), 2.5 * s["dw"]
    sc = _scores(x, case["score"])
    if case["renorm"]:
        chosen = sc.gather(1, at)
        total = chosen.sum(dim=1, keepdim=True)
        w = chosen / total
        g = (g - (g * w).sum(dim=1, keepdim=True)) / total
    ds = torch.zeros_like(sc).scatter_(1, at, g)
    if case["score"] == "sigmoid":
        dl = ds * sc * (1 - sc)
    else:
        dl = sc * (ds - (ds * sc).sum(dim=1, keepdim=True))
    return {"dlogits": dl.to(s["logits"].dtype)}


def _blocks(x):
    m, k = x.shape
    kp = -(-k // PAD) * PAD
    if kp > k:
        x = torch.cat([x, x.new_zeros((m, kp - k))], dim=1)
    return x.view(m, kp // BLOCK, BLOCK)


def _quantised(x):
    """Magnitude codes, signs and scale codes of rows x (32 bits), blocks of 32."""
    v = _blocks(x)
    bits = v.abs().amax(dim=2).view(torch.int32) >> 23
    scale = torch.where(bits == 255, 255, (bits - 2).clamp(min=0))
    # 2^(127 - scale) from its bits; scale 255 stands for NaN, whose codes are 0.
    inverse = torch.where(scale == 255, 0, (254 - scale) << 23).to(torch.int32).view(torch.float32)
    u = torch.where((scale == 255)[..., None], 0.0, v.abs() * inverse[..., None])
    code = ((u > 0.25).int() + (u >= 0.75) + (u > 1.25) + (u >= 1.75) + (u > 2.5) + (u >= 3.5) +
            (u > 5))
    return code, torch.signbit(v) & (scale != 255)[..., None], scale


def _encode(x):
    """codes [rows, kp / 2] (the even value in the low half) and scales [rows, kp / 32]."""
    code, sign, scale = _quantised(x.float())
    full = (code + 8 * sign.int()).view(len(x), -1, 2)
    return ((full[..., 0] + 16 * full[..., 1]).to(torch.uint8).contiguous(),
            scale.to(torch.uint8).contiguous())


def _power(scale):
    """2^(scale - 127) of scale codes, exactly; NaN for 255."""
    scale = scale.int()
    bits = torch.where(scale == 0, 1 << 22, scale << 23)
    return torch.where(scale == 255, math.nan, bits.to(torch.int32).view(torch.float32))


_HALVES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _rounded(x):
    """The values that the 4-bit form of rows x stands for, in 32 bits."""
    code, sign, scale = _quantised(x.float())
    v = torch.tensor(_HALVES, device=DEVICE)[code.long()]
    v = torch.where(sign, -v, v) * _power(scale)[..., None]
    return v.reshape(len(x), -1)[:, :x.shape[1]]


def _decoded(codes, scales, k, dtype=torch.float32):
    table = torch.tensor(_HALVES + [-h for h in _HALVES], dtype=dtype, device=DEVICE)
    c = torch.stack([codes & 15, codes >> 4], dim=2).view(len(codes), -1, BLOCK)
    v = table[c.int()] * _power(scales).to(dtype)[..., None]
    return v.view(len(codes), -1)[:, :k]


def _plain_round(s):
    return {"values": _rounded(s["x"]).to(s["x"].dtype)}


def _products(s, a, w):
    """act(a w^T + bias) row_scale per expert's rows, in the operands' precision."""
    case, n, bounds = s["case"], s["case"]["n"], s["bounds"]
    rows = a if s["rows"] is None else a[s["rows"].long()]
    out = rows.new_empty((len(rows), n))
    for x in range(case["experts"]):
        lo, hi = bounds[x], bounds[x + 1]
        if hi > lo:
            z = rows[lo:hi] @ w[x * n:(x + 1) * n].T
            out[lo:hi] = z if s["bias"] is None else z + s["bias"][x].to(z.dtype)
    out = _act(out, case["act"])
    return out if s["row_scale"] is None else out * s["row_scale"].to(out.dtype)[:, None]


def _plain_product(s):
    w = _decoded(s["codes"], s["scales"], s["case"]["k"])
    return {"y": _products(s, _rounded(s["x"]), w).to(s["x"].dtype)}


# --------------------------------------------------------------------------
# The framework's calls


def _empty(like, *shape, dtype=None):
    return torch.empty(shape, dtype=dtype or like.dtype, device=DEVICE)


def _strides(x):
    return x.stride(0) * x.element_size(), x.stride(1) * x.element_size()


def _check(ok):
    if ok != 1:
        raise RuntimeError("the call was refused")


def _own_norm(s):
    c, x, layers = s["case"], s["x"], s["layers"]
    y = _empty(x, *x.shape)
    mean, rstd = (_empty(x, c["n"], c["g"], dtype=torch.float32) for _ in range(2))
    _check(layers.group_norm_device(x, *_strides(x), s["gamma"], s["beta"], y, mean, rstd,
                                    s["workspace"], c["n"], c["p"], c["c"], c["g"], EPS,
                                    layers.ACTS[c["act"]], layers.DTYPES[x.dtype], s["stream"]))
    return {"y": y, "mean": mean, "rstd": rstd}


def _own_norm_back(s):
    c, x, dy, layers = s["case"], s["x"], s["dy"], s["layers"]
    dx = _empty(x, *x.shape)
    dgamma, dbeta = (_empty(x, c["c"], dtype=torch.float32) for _ in range(2))
    _check(layers.group_norm_backward_device(
        x, *_strides(x), dy, *_strides(dy), s["gamma"], s["beta"], s["mean"], s["rstd"], dx,
        dgamma, dbeta, s["workspace"], c["n"], c["p"], c["c"], c["g"], layers.ACTS[c["act"]],
        layers.DTYPES[x.dtype], s["stream"]))
    return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}


def _own_route(s):
    c, x, layers = s["case"], s["logits"], s["layers"]
    t, e, k = c["t"], c["e"], c["k"]
    experts, positions = (_empty(x, t, k, dtype=torch.int32) for _ in range(2))
    weights, row_weights = (_empty(x, *n, dtype=torch.float32) for n in ((t, k), (t * k,)))
    offsets, tokens = (_empty(x, n, dtype=torch.int32) for n in (e + 1, t * k))
    _check(layers.route_device(x, e * x.element_size(), s["bias"], s["valid"], experts, weights,
                               t, e, k, c["groups"], c["kept"], layers.SCORES[c["score"]],
                               c["renorm"], 2.5, layers.DTYPES[x.dtype], s["stream"]))
    _check(layers.expert_order_device(experts, weights, offsets, tokens, positions, row_weights,
                                      s["workspace"], t, e, k, s["stream"]))
    return {"experts": experts, "weights": weights, "offsets": offsets, "tokens": tokens,
            "positions": positions, "row_weights": row_weights}


def _own_route_back(s):
    c, x, layers = s["case"], s["logits"], s["layers"]
    dl = _empty(x, *x.shape)
    _check(layers.route_backward_device(x, c["e"] * x.element_size(), s["experts"], s["dw"], dl,
                                        c["t"], c["e"], c["k"], layers.SCORES[c["score"]],
                                        c["renorm"], 2.5, layers.DTYPES[x.dtype], s["stream"]))
    return {"dlogits": dl}


def _own_quantise(s):
    x, layers = s["x"], s["layers"]
    m, k = x.shape
    kp = layers.mx4_padded(k)
    codes = _empty(x, m, kp // 2, dtype=torch.uint8)
    scales = _empty(x, m, kp // BLOCK, dtype=torch.uint8)
    _check(layers.mx4_quantise_device(x, k * x.element_size(), codes, scales, m, k,
                                      layers.DTYPES[x.dtype], s["stream"]))
    return codes, scales


def _own_round(s):
    x, layers = s["x"], s["layers"]
    codes, scales = _own_quantise(s)
    values = _empty(x, *x.shape)
    _check(layers.mx4_values_device(codes, scales, values, len(x), x.shape[1],
                                    layers.DTYPES[x.dtype], s["stream"]))
    return {"values": values}


def _own_product(s):
    c, x, layers = s["case"], s["x"], s["layers"]
    codes, scales = _own_quantise(s)
    m = c["m"] if s["rows"] is None else len(s["rows"])
    y = _empty(x, m, c["n"])
    _check(layers.mx4_product_device(codes, scales, c["m"], s["rows"], s["codes"], s["scales"],
                                     s["offsets"], s["bias"], s["row_scale"], y, m, c["n"],
                                     c["k"], c["experts"], layers.ACTS[c["act"]],
                                     layers.DTYPES[x.dtype], s["stream"]))
    return {"y": y}


def run(state):
    entry = state["case"]["entry"]
    if own:
        return {"norm": _own_norm, "norm_back": _own_norm_back, "route": _own_route,
                "route_back": _own_route_back, "round": _own_round,
                "product": _own_product}[entry](state)
    return {"norm": _plain_norm, "norm_back": _plain_norm_back, "route": _plain_route,
            "route_back": _plain_route_back, "round": _plain_round,
            "product": _plain_product}[entry](state)


def work(case):
    entry, b = case["entry"], BYTES[case["dtype"]]
    if entry == "norm":
        v = case["n"] * case["p"] * case["c"]
        return {"bytes": 2 * b * v + 8 * case["n"] * case["g"] + 8 * case["c"], "flops": 12 * v}
    if entry == "norm_back":
        v = case["n"] * case["p"] * case["c"]
        return {"bytes": 3 * b * v + 8 * case["n"] * case["g"] + 16 * case["c"], "flops": 24 * v}
    if entry == "route":
        t, e, k = case["t"], case["e"], case["k"]
        # Logits, bias and mask in; experts, weights, positions, and tokens
        # and weights by expert out.
        return {"bytes": t * e * b + 20 * t * k + 4 * (e + 1) + 4 * e * case["bias"] +
                t * case["padded"], "flops": 4 * t * e}
    if entry == "route_back":
        t, e, k = case["t"], case["e"], case["k"]
        # Renormalised weights depend on the chosen logits alone.
        read = t * k if case["renorm"] or case["score"] == "sigmoid" else t * e
        return {"bytes": (read + t * e) * b + 8 * t * k, "flops": 4 * read}
    if entry == "round":
        return {"bytes": 2 * case["m"] * case["k"] * b, "flops": 6 * case["m"] * case["k"]}
    m, n, k = case["m"] * case["top"], case["n"], case["k"]
    kp = -(-k // PAD) * PAD
    weights = case["experts"] * n * kp * 17 // 32
    if case["experts"] > 1:
        weights = min(weights, m * n * kp * 17 // 32)
    return {"bytes": case["m"] * k * b + weights + m * n * b, "flops": 2 * m * n * k}


# --------------------------------------------------------------------------
# The definitions in 64 bits


def _exact_norm(s, x):
    case = s["case"]
    v = x.reshape(case["n"], case["p"], case["g"], -1).permute(0, 2, 1, 3)
    v = v.reshape(case["n"], case["g"], -1)
    var, mean = torch.var_mean(v, dim=2, unbiased=False)
    rstd = (var + EPS) ** -0.5
    z = (v - mean[..., None]) * rstd[..., None]
    z = z.reshape(case["n"], case["g"], case["p"], -1).permute(0, 2, 1, 3).reshape(x.shape)
    z = torch.addcmul(s["beta"].double(), z, s["gamma"].double())
    if case["act"] == "silu":
        z = torch.nn.functional.silu(z)
    elif case["act"] == "gelu":
        z = torch.nn.functional.gelu(z)
    return z, mean, rstd


def _exact_norm_back(s):
    step = max(1, (1 << 26) // (s["case"]["p"] * s["case"]["c"]))
    gamma = s["gamma"].double().requires_grad_()
    beta = s["beta"].double().requires_grad_()
    parts = []
    for i in range(0, s["case"]["n"], step):
        x = s["x"][i:i + step].double().requires_grad_()
        part = {"case": {**s["case"], "n": len(x)}, "gamma": gamma, "beta": beta}
        _exact_norm(part, x)[0].backward(s["dy"][i:i + step].double())
        parts.append(x.grad)
    return {"dx": torch.cat(parts), "dgamma": gamma.grad, "dbeta": beta.grad}


def _exact_order(experts, weights, e):
    """By one pass over the choices for each expert."""
    t, k = experts.shape
    flat = experts.reshape(-1)
    rows = [(flat == x).nonzero()[:, 0] for x in range(e)]
    ends = [0]
    for r in rows:
        ends.append(ends[-1] + len(r))
    rows = torch.cat(rows)
    tokens, positions = (torch.full((t * k,), -1, dtype=torch.int32, device=DEVICE)
                         for _ in range(2))
    row_weights = torch.zeros(t * k, dtype=weights.dtype, device=DEVICE)
    tokens[:len(rows)] = torch.div(rows, k, rounding_mode="floor").to(torch.int32)
    positions[rows] = torch.arange(len(rows), dtype=torch.int32, device=DEVICE)
    row_weights[:len(rows)] = weights.reshape(-1)[rows]
    return {"offsets": torch.tensor(ends, dtype=torch.int32, device=DEVICE), "tokens": tokens,
            "positions": positions.view(t, k), "row_weights": row_weights}


def _exact_route(s):
    """By repeated selection instead of sorting."""
    case, x = s["case"], s["logits"].double()
    t, e, groups = case["t"], case["e"], case["groups"]
    s64 = torch.softmax(x, dim=1) if case["score"] == "softmax" else torch.sigmoid(x)
    key = x.clone() if s["bias"] is None else s64 + s["bias"].double()
    lane = torch.arange(max(e, groups), device=DEVICE)

    def best(v):
        """Highest value of each row, its lowest index; v without it."""
        top = v.max(dim=1, keepdim=True).values
        at = torch.where(v == top, lane[:v.shape[1]], e).min(dim=1).values
        return top[:, 0], at, v.masked_fill(lane[:v.shape[1]] == at[:, None], -math.inf)

    if s["valid"] is not None:
        key = torch.where((s["valid"] == 0)[:, None], 0.0, key)
    if case["kept"] < groups:
        v = key.reshape(t * groups, e // groups)
        total, _, rest = best(v)
        if s["bias"] is not None and e > groups:
            total = total + best(rest)[0]
        total = total.view(t, groups)
        keep = torch.zeros((t, groups), dtype=torch.bool, device=DEVICE)
        for _ in range(case["kept"]):
            _, at, total = best(total)
            keep[torch.arange(t, device=DEVICE), at] = True
        key = key.masked_fill(~keep.repeat_interleave(e // groups, dim=1), -math.inf)
    picks = []
    for _ in range(case["k"]):
        _, at, key = best(key)
        picks.append(at)
    experts = torch.stack(picks, dim=1)
    w = torch.stack([s64[torch.arange(t, device=DEVICE), at] for at in picks], dim=1)
    if case["renorm"]:
        w = w / w.sum(dim=1, keepdim=True)
    w = 2.5 * w
    if s["valid"] is not None:
        live = (s["valid"] != 0)[:, None]
        experts, w = torch.where(live, experts, -1), torch.where(live, w, 0.0)
    return {"experts": experts.to(torch.int32), "weights": w, **_exact_order(experts, w, e)}


def _exact_route_back(s):
    case = s["case"]
    x = s["logits"].double().requires_grad_()
    sc = torch.softmax(x, dim=1) if case["score"] == "softmax" else torch.sigmoid(x)
    w = sc.gather(1, s["experts"].long())
    if case["renorm"]:
        w = w / w.sum(dim=1, keepdim=True)
    (2.5 * w).backward(s["dw"].double())
    return {"dlogits": x.grad}


def _exact_rounded(x):
    """By the nearest of the form's values, the even code at a tie."""
    m, k = x.shape
    out = torch.empty((m, k), dtype=torch.float64, device=DEVICE)
    for i in range(0, m, 8192):
        v = _blocks(x[i:i + 8192].double())
        top = v.abs().amax(dim=2, keepdim=True)
        # frexp's mantissa lies in [0.5, 1).
        power = (torch.frexp(top).exponent - 3).clamp(min=-127)
        unit = torch.ldexp(torch.ones_like(top), power)
        u = (v.abs() / unit).clamp(max=6.0)
        step = torch.where(u < 2, 0.5, torch.where(u < 4, 1.0, 2.0))
        v = torch.sign(v) * torch.round(u / step) * step * unit
        out[i:i + 8192] = v.view(len(v), -1)[:, :k]
    return out


def _exact_product(case, s):
    n, k, a = case["n"], case["k"], _exact_rounded(s["x"])
    low, high = s["codes"] % 16, s["codes"] // 16
    code = torch.stack([low, high], dim=2).flatten(1).double()
    sign, size = torch.where(code >= 8, -1.0, 1.0), code % 8
    power, half = torch.floor(size / 2), size % 2 / 2
    # Codes 0 and 1 are 0 and one half, then two values to each power of two.
    size = torch.where(power == 0, half, (1 + half) * torch.exp2(power - 1))
    unit = torch.exp2(s["scales"].double() - 127).repeat_interleave(BLOCK, dim=1)
    w = (sign * size * unit)[:, :k].view(case["experts"], n, k)
    expert = torch.zeros(len(a), dtype=torch.long, device=DEVICE)
    if s["rows"] is not None:
        at = torch.arange(len(s["rows"]), device=DEVICE)
        expert = (at[:, None] >= s["offsets"][None, 1:-1]).sum(dim=1)
        a = a[s["rows"].long()]
    z = torch.zeros((len(a), n), dtype=torch.float64, device=DEVICE)
    for x in range(case["experts"]):
        mine = (expert == x).nonzero()[:, 0]
        bias = None if s["bias"] is None else s["bias"][x].double()
        z[mine] = torch.nn.functional.linear(a[mine], w[x], bias)
    if case["act"] == "silu":
        z = torch.nn.functional.silu(z)
    elif case["act"] == "gelu":
        z = torch.nn.functional.gelu(z)
    return z if s["row_scale"] is None else z * s["row_scale"].double()[:, None]


def exact(case, seed):
    entry = case["entry"]
    if entry in ("norm", "norm_back"):
        s = {**_norm_state(case, seed), "case": case}
        if entry == "norm_back":
            return _exact_norm_back(s)
        parts, step = [], max(1, (1 << 26) // (case["p"] * case["c"]))
        for i in range(0, case["n"], step):
            x = s["x"][i:i + step].double()
            parts.append(_exact_norm({**s, "case": {**case, "n": len(x)}}, x))
        return dict(zip(("y", "mean", "rstd"), (torch.cat(v) for v in zip(*parts))))
    if entry in ("route", "route_back"):
        s = {**_route_state(case, seed), "case": case}
        return _exact_route(s) if entry == "route" else _exact_route_back(s)
    if entry == "round":
        x = _activations(_gen(seed), case["m"], case["k"], TYPES[case["dtype"]])
        return {"values": _exact_rounded(x)}
    return {"y": _exact_product(case, _product_state(case, seed))}
