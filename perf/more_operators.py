"""Tokens on their way to experts and back, embeddings, and 8-bit products, for timing and comparison.

Three groups of operators: tokens copied into their experts' order and summed
back with the routing's weights, each with its gradients; embedding lookup with
its gradient; rows in 8-bit integers with a scale each, and their products,
dense or per expert.  `run` with `own` false is their plain form, with `own`
true the calls of turbinator_c_amd.layers; `exact` restates them in 64 bits.
"""
import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
PAD = 128  # 8-bit rows are padded to whole 128s
LEAST = 2.0 ** -126


def listed():
    return [
        # One environment acting: its 256 patches (four cameras), two of eight
        # experts each.
        {"name": "rows_256", "entry": "rows", "t": 256, "e": 8, "k": 2, "d": 256, "pitch": 256,
         "weighted": False, "padded": False, "dtype": "bf16"},
        # A training batch of 256 environments' patches, four of 64 experts.
        {"name": "rows_65536", "entry": "rows", "t": 65536, "e": 64, "k": 4, "d": 2048,
         "pitch": 2048, "weighted": False, "padded": False, "dtype": "bf16"},
        # Gradient of the tokens and of weights applied on the way in; odd
        # sizes, tokens a slice of wider rows, some of them padding.
        {"name": "rows_back_odd", "entry": "rows_back", "t": 20483, "e": 24, "k": 3, "d": 1001,
         "pitch": 1030, "weighted": True, "padded": True, "dtype": "f32"},
        # A single token's eight experts summed back, added to the token.
        {"name": "sum_1", "entry": "sum", "t": 1, "e": 64, "k": 8, "d": 4096, "pitch": 4096,
         "weighted": True, "padded": False, "residual": True, "dtype": "bf16"},
        # The weighted sum's gradients in training.
        {"name": "sum_back_40960", "entry": "sum_back", "t": 40960, "e": 16, "k": 2, "d": 1024,
         "pitch": 1024, "weighted": True, "padded": False, "dtype": "bf16"},
        # Activations to 8 bits and back, rows of no whole vectors.
        {"name": "eight_round_odd", "entry": "round", "m": 40959, "k": 1999, "dtype": "bf16"},
        # One token through a layer: the weights are what is read.
        {"name": "eight_1", "entry": "product", "m": 1, "n": 4096, "k": 4096, "experts": 1,
         "top": 1, "act": "none", "bias": True, "dtype": "f16"},
        # Experts' first matrices over a batch of routed tokens.
        {"name": "eight_experts_8192", "entry": "product", "m": 8192, "n": 2048, "k": 1024,
         "experts": 8, "top": 2, "act": "silu", "bias": True, "dtype": "bf16"},
        # A dense layer over a training batch's tokens.
        {"name": "eight_16384", "entry": "product", "m": 16384, "n": 4096, "k": 4096,
         "experts": 1, "top": 1, "act": "gelu", "bias": True, "dtype": "bf16"},
        # Tokens of a large vocabulary, added to what they already hold.
        {"name": "embed_40961", "entry": "embed", "t": 40961, "v": 65536, "d": 1024,
         "base": True, "spread": "skewed", "dtype": "bf16"},
        # Gradient of 64 patch places over four environments acting.
        {"name": "embed_back_1024", "entry": "embed_back", "t": 1024, "v": 64, "d": 256,
         "spread": "even", "dtype": "f32"},
        # Gradient of a large vocabulary, a few entries in a third of the tokens.
        {"name": "embed_back_163840", "entry": "embed_back", "t": 163840, "v": 32768, "d": 1024,
         "spread": "skewed", "dtype": "bf16"},
    ]


def _size(rng, low, high):
    """Spread over the logarithm, odd and even alike."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))
    return min(high, max(low, n))


def draw(rng):
    entry = rng.choice(["rows", "rows_back", "sum", "sum_back", "round", "product", "product",
                        "embed", "embed_back", "embed_back"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    if entry in ("rows", "rows_back", "sum", "sum_back"):
        k, d = rng.randint(1, 8), _size(rng, 16, 4096)
        if rng.random() < 0.4:
            d = d // 8 * 8
        limit = 536870912 if entry in ("rows", "sum") else 201326592
        t = _size(rng, 1, min(163840, limit * 2 // BYTES[dtype] // (k * d)))
        return {"entry": entry, "t": t, "e": rng.randint(k, 256), "k": k, "d": d,
                "pitch": d + rng.choice([0, 0, 1, 8, 30]), "weighted": rng.random() < 0.6,
                "padded": rng.random() < 0.4, "residual": rng.random() < 0.5, "dtype": dtype}
    if entry == "round":
        k = _size(rng, 16, 8192)
        return {"entry": entry, "m": _size(rng, 1, min(163840, 81920000 // k)), "k": k,
                "dtype": dtype}
    if entry == "product":
        n, k = _size(rng, 64, 4096), _size(rng, 64, 4096)
        experts = rng.choice([1, 1, 4, 8, 16])
        return {"entry": entry, "m": _size(rng, 1, 16384 if experts == 1 else 8192), "n": n,
                "k": k, "experts": experts, "top": 1 if experts == 1 else rng.randint(1, 2),
                "act": rng.choice(["none", "silu", "gelu"]), "bias": rng.random() < 0.5,
                "dtype": dtype}
    d = _size(rng, 16, 4096)
    if rng.random() < 0.6:
        d = d // 8 * 8
    size = 2 // BYTES[dtype] or 1
    case = {"entry": entry, "t": _size(rng, 1, min(163840, 83886080 * size // d)),
            "v": _size(rng, 1, min(262144, 33554432 // d)), "d": d,
            "spread": rng.choice(["even", "skewed", "skewed", "one"]), "dtype": dtype}
    if entry == "embed":
        case["base"] = rng.random() < 0.5
    return case


# --------------------------------------------------------------------------
# Inputs


def _gen(seed):
    return torch.Generator(DEVICE).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, device=DEVICE, generator=g)


def _rand(g, *shape):
    return torch.rand(shape, device=DEVICE, generator=g)


def _activations(g, m, k, dt, pitch=None):
    """Rows of a block's activations: a few channels far larger than the rest."""
    pitch = pitch or k
    size = torch.exp(0.5 * _randn(g, pitch)) * torch.where(_rand(g, pitch) < 0.01, 20.0, 1.0)
    out = torch.empty((m, pitch), dtype=dt, device=DEVICE)
    for i in range(0, m, 16384):
        part = out[i:i + 16384]
        part.copy_(_randn(g, *part.shape) * size)
    return out[:, :k]


def _routing(g, t, e, k, padded):
    """k different experts for each token, none for padding, and the order of
    the choices by expert: offsets [e + 1], positions [t, k]."""
    liked = _randn(g, t, e) + 0.5 * _randn(g, e)
    experts = liked.sort(dim=1, descending=True).indices[:, :k]
    if padded:
        experts = torch.where((_rand(g, t) < 0.95)[:, None], experts, e)
    order = experts.reshape(-1).sort(stable=True)
    live = order.values < e
    at = torch.arange(t * k, device=DEVICE)
    positions = torch.empty_like(at).scatter_(0, order.indices, torch.where(live, at, -1))
    count = torch.bincount(order.values, minlength=e + 1)[:e]
    offsets = torch.cat([count.new_zeros(1), count.cumsum(0)])
    return offsets.to(torch.int32), positions.view(t, k).to(torch.int32)


def _expert_state(case, seed):
    g, entry = _gen(seed), case["entry"]
    t, k, d, dt = case["t"], case["k"], case["d"], TYPES[case["dtype"]]
    s = {"residual": None, "weights": None}
    s["offsets"], s["positions"] = _routing(g, t, case["e"], k, case["padded"])
    if case["weighted"]:
        w = _rand(g, t, k)
        s["weights"] = 2.5 * w / w.sum(dim=1, keepdim=True)
    # Tokens, or their gradient; the experts' rows, or theirs.
    s["x"] = _activations(g, t, d, dt, case["pitch"])
    if entry == "sum":
        s["residual"] = s["x"] if case["residual"] else None
    if entry != "rows":
        s["rows"] = _activations(g, t * k, d, dt)
        if case["padded"]:
            # Behind the last expert's rows nothing is read.
            s["rows"].masked_fill_((torch.arange(t * k, device=DEVICE) >= s["offsets"][-1])
                                   [:, None], math.nan)
    return s


def _encode(x):
    """codes [rows, kp] and scales [rows] of rows x, padded with zeros."""
    q, scale = _quantised(x.float())
    m, k = q.shape
    codes = torch.zeros((m, -(-k // PAD) * PAD), dtype=torch.int8, device=DEVICE)
    codes[:, :k] = q.to(torch.int8)
    return codes, scale


def _product_state(case, seed):
    g, m, n, k, experts = _gen(seed), case["m"], case["n"], case["k"], case["experts"]
    s = {"x": _activations(g, m, k, TYPES[case["dtype"]]), "rows": None, "offsets": None,
         "bounds": [0, m], "row_scale": None}
    s["codes"], s["scales"] = _encode(_randn(g, experts * n, k) / math.sqrt(k))
    s["bias"] = 0.1 * _randn(g, experts, n) if case["bias"] else None
    if experts > 1:
        s["offsets"], positions = _routing(g, m, experts, case["top"], False)
        rows = torch.empty(m * case["top"], dtype=torch.int32, device=DEVICE)
        token = torch.arange(m * case["top"], device=DEVICE) // case["top"]
        rows[positions.reshape(-1).long()] = token.to(torch.int32)
        s["rows"], s["bounds"] = rows, s["offsets"].tolist()
        s["row_scale"] = _rand(g, len(rows))
    return s


def _embed_state(case, seed):
    g, t, v, d, dt = _gen(seed), case["t"], case["v"], case["d"], TYPES[case["dtype"]]
    if case["spread"] == "even":
        ids = torch.randint(0, v, (t,), device=DEVICE, generator=g)
    elif case["spread"] == "skewed":
        # As words are spread: each entry about in proportion to 1 / its rank.
        rank = torch.exp(_rand(g, t) * math.log(v + 1)).long().clamp(1, v) - 1
        ids = torch.randperm(v, device=DEVICE, generator=g)[rank]
    else:
        ids = torch.full((t,), int(seed) % v, dtype=torch.int64, device=DEVICE)
    # Some tokens are padding and have no entry.
    ids = torch.where(_rand(g, t) < 0.02, -1, ids)
    s = {"ids": ids.to(torch.int32), "scale": math.sqrt(d)}
    if case["entry"] == "embed":
        s["table"] = (_randn(g, v, d) / math.sqrt(d)).to(dt)
        s["base"] = _activations(g, t, d, dt) if case["base"] else None
    else:
        s["dout"] = (_activations(g, t, d, torch.float32) * 0.01).to(dt)
    return s


def _inputs(case, seed):
    entry = case["entry"]
    if entry in ("rows", "rows_back", "sum", "sum_back"):
        return _expert_state(case, seed)
    if entry == "round":
        return {"x": _activations(_gen(seed), case["m"], case["k"], TYPES[case["dtype"]])}
    return _product_state(case, seed) if entry == "product" else _embed_state(case, seed)


def prepare(case, seed):
    s = {**_inputs(case, seed), "case": case}
    if own:
        from turbinator_c_amd import layers
        s["layers"], s["stream"] = layers, torch.cuda.current_stream()
        if case["entry"] == "embed_back":
            # Kept by a training program from step to step.
            need = max(layers.embed_order_workspace_bytes(case["t"], case["v"]),
                       layers.embed_backward_workspace_bytes(case["t"], case["v"], case["d"]), 1)
            s["workspace"] = torch.empty(need, dtype=torch.uint8, device=DEVICE)
    return s


# --------------------------------------------------------------------------
# Plain forms, in 32 bits


def _act(z, act):
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * torch.special.erfc(-z * math.sqrt(0.5))
    return z


def _weighted(s, v):
    return v if s["weights"] is None else v * s["weights"][..., None]


def _scattered(s, v):
    """v [t, k, d], 32 bits, at the rows of its choices; the other rows 0."""
    rows = torch.zeros((v.shape[0] * v.shape[1], v.shape[2]), dtype=s["x"].dtype, device=DEVICE)
    live = s["positions"] >= 0
    rows[s["positions"][live].long()] = v[live].to(rows.dtype)
    return rows


def _gathered(s):
    """The choices' rows [t, k, d] in 32 bits, 0 for choices without one."""
    v = s["rows"][s["positions"].clamp(min=0).long()].float()
    return torch.where((s["positions"] >= 0)[..., None], v, 0.0)


def _plain_rows(s):
    x = s["x"].float()[:, None, :].expand(-1, s["case"]["k"], -1)
    return {"rows": _scattered(s, _weighted(s, x))}


def _plain_rows_back(s):
    v = _gathered(s)
    return {"dx": _weighted(s, v).sum(dim=1).to(s["x"].dtype),
            "dweights": (v * s["x"].float()[:, None, :]).sum(dim=2)}


def _plain_sum(s):
    out = _weighted(s, _gathered(s)).sum(dim=1)
    if s["residual"] is not None:
        out = out + s["residual"].float()
    return {"out": out.to(s["x"].dtype)}


def _plain_sum_back(s):
    dout = s["x"].float()[:, None, :]
    return {"dweights": (_gathered(s) * dout).sum(dim=2),
            "drows": _scattered(s, _weighted(s, dout.expand(-1, s["case"]["k"], -1)))}


def _quantised(x):
    """Codes (32-bit floats) and scales of rows x, each step rounded to 32 bits."""
    most = x.abs().amax(dim=1)
    # A divisor on the device: torch multiplies by a plain number's inverse.
    scale = (most / torch.full_like(most, 127.0)).clamp(min=LEAST)
    return torch.round(x * (1 / scale)[:, None]), scale


def _plain_round(s):
    q, scale = _quantised(s["x"].float())
    return {"values": (q * scale[:, None]).to(s["x"].dtype)}


def _plain_product(s):
    case, n, bounds = s["case"], s["case"]["n"], s["bounds"]
    q, scale = _quantised(s["x"].float())
    if s["rows"] is not None:
        q, scale = q[s["rows"].long()], scale[s["rows"].long()]
    w = s["codes"][:, :case["k"]].float()
    z = q.new_empty((len(q), n))
    for x in range(case["experts"]):
        lo, hi = bounds[x], bounds[x + 1]
        if hi > lo:
            part = q[lo:hi] @ w[x * n:(x + 1) * n].T
            part = part * scale[lo:hi, None] * s["scales"][x * n:(x + 1) * n]
            z[lo:hi] = part if s["bias"] is None else part + s["bias"][x]
    z = _act(z, case["act"])
    if s["row_scale"] is not None:
        z = z * s["row_scale"][:, None]
    return {"y": z.to(s["x"].dtype)}


def _plain_embed(s):
    ids = s["ids"].long()
    out = s["table"][ids.clamp(min=0)].float() * s["scale"]
    out = torch.where((ids >= 0)[:, None], out, 0.0)
    if s["base"] is not None:
        out = out + s["base"].float()
    return {"out": out.to(s["table"].dtype)}


def _plain_embed_back(s):
    live = s["ids"] >= 0
    total = torch.zeros((s["case"]["v"], s["case"]["d"]), device=DEVICE)
    total.index_add_(0, s["ids"][live].long(), s["dout"][live].float())
    return {"dtable": total * s["scale"]}


# --------------------------------------------------------------------------
# The framework's calls


def _empty(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device=DEVICE)


def _stride(x):
    return x.stride(0) * x.element_size()


def _check(ok):
    if ok != 1:
        raise RuntimeError("the call was refused")


def _own_rows(s):
    c, x, layers = s["case"], s["x"], s["layers"]
    rows = _empty(c["t"] * c["k"], c["d"], dtype=x.dtype)
    _check(layers.expert_rows_device(x, _stride(x), s["offsets"], s["positions"], s["weights"],
                                     rows, c["t"], c["e"], c["k"], c["d"],
                                     layers.DTYPES[x.dtype], s["stream"]))
    return {"rows": rows}


def _own_rows_back(s):
    c, x, drows, layers = s["case"], s["x"], s["rows"], s["layers"]
    dx, dweights = _empty(c["t"], c["d"], dtype=x.dtype), _empty(c["t"], c["k"])
    _check(layers.expert_rows_backward_device(drows, _stride(drows), x, _stride(x),
                                              s["positions"], s["weights"], dx, dweights, c["t"],
                                              c["k"], c["d"], layers.DTYPES[x.dtype],
                                              s["stream"]))
    return {"dx": dx, "dweights": dweights}


def _own_sum(s):
    c, rows, residual, layers = s["case"], s["rows"], s["residual"], s["layers"]
    out = _empty(c["t"], c["d"], dtype=rows.dtype)
    _check(layers.expert_sum_device(rows, _stride(rows), s["positions"], s["weights"], residual,
                                    0 if residual is None else _stride(residual), out, c["t"],
                                    c["k"], c["d"], layers.DTYPES[rows.dtype], s["stream"]))
    return {"out": out}


def _own_sum_back(s):
    c, dout, rows, layers = s["case"], s["x"], s["rows"], s["layers"]
    drows, dweights = _empty(*rows.shape, dtype=rows.dtype), _empty(c["t"], c["k"])
    _check(layers.expert_sum_backward_device(dout, _stride(dout), rows, _stride(rows),
                                             s["offsets"], s["positions"], s["weights"], drows,
                                             dweights, c["t"], c["e"], c["k"], c["d"],
                                             layers.DTYPES[rows.dtype], s["stream"]))
    return {"drows": drows, "dweights": dweights}


def _own_quantise(s):
    x, layers = s["x"], s["layers"]
    m, k = x.shape
    codes = _empty(m, layers.int8_padded(k), dtype=torch.int8)
    scales = _empty(m)
    _check(layers.int8_quantise_device(x, _stride(x), codes, scales, m, k,
                                       layers.DTYPES[x.dtype], s["stream"]))
    return codes, scales


def _own_round(s):
    x, layers = s["x"], s["layers"]
    codes, scales = _own_quantise(s)
    values = _empty(*x.shape, dtype=x.dtype)
    _check(layers.int8_values_device(codes, scales, values, len(x), x.shape[1],
                                     layers.DTYPES[x.dtype], s["stream"]))
    return {"values": values}


def _own_product(s):
    c, x, layers = s["case"], s["x"], s["layers"]
    codes, scales = _own_quantise(s)
    m = c["m"] if s["rows"] is None else len(s["rows"])
    y = _empty(m, c["n"], dtype=x.dtype)
    _check(layers.int8_product_device(codes, scales, c["m"], s["rows"], s["codes"], s["scales"],
                                      s["offsets"], s["bias"], s["row_scale"], y, m, c["n"],
                                      c["k"], c["experts"], layers.ACTS[c["act"]],
                                      layers.DTYPES[x.dtype], s["stream"]))
    return {"y": y}


def _own_embed(s):
    c, table, base, layers = s["case"], s["table"], s["base"], s["layers"]
    out = _empty(c["t"], c["d"], dtype=table.dtype)
    _check(layers.embed_device(s["ids"], table, _stride(table), base,
                               0 if base is None else _stride(base), s["scale"], out, c["t"],
                               c["v"], c["d"], layers.DTYPES[table.dtype], s["stream"]))
    return {"out": out}


def _own_embed_back(s):
    c, dout, layers = s["case"], s["dout"], s["layers"]
    order, ranges = _empty(c["t"], dtype=torch.int32), _empty(c["v"], 2, dtype=torch.int32)
    dtable = _empty(c["v"], c["d"])
    _check(layers.embed_order_device(s["ids"], order, ranges, s["workspace"], c["t"], c["v"],
                                     s["stream"]))
    _check(layers.embed_backward_device(dout, _stride(dout), s["ids"], order, ranges, s["scale"],
                                        dtable, s["workspace"], c["t"], c["v"], c["d"],
                                        layers.DTYPES[dout.dtype], s["stream"]))
    return {"dtable": dtable}


def run(state):
    entry = state["case"]["entry"]
    if own:
        return {"rows": _own_rows, "rows_back": _own_rows_back, "sum": _own_sum,
                "sum_back": _own_sum_back, "round": _own_round, "product": _own_product,
                "embed": _own_embed, "embed_back": _own_embed_back}[entry](state)
    return {"rows": _plain_rows, "rows_back": _plain_rows_back, "sum": _plain_sum,
            "sum_back": _plain_sum_back, "round": _plain_round, "product": _plain_product,
            "embed": _plain_embed, "embed_back": _plain_embed_back}[entry](state)


def work(case):
    entry, b = case["entry"], BYTES[case["dtype"]]
    if entry in ("rows", "rows_back", "sum", "sum_back"):
        t, k, d = case["t"], case["k"], case["d"]
        token, rows = t * d * b, t * k * d * b
        choices = t * k * (8 if case["weighted"] else 4)
        if entry == "rows":
            return {"bytes": token + rows + choices, "flops": t * k * d}
        if entry == "sum":
            return {"bytes": token * (2 if case["residual"] else 1) + rows + choices,
                    "flops": 2 * t * k * d}
        return {"bytes": (2 * token + rows if entry == "rows_back" else token + 2 * rows) +
                choices + 4 * t * k, "flops": 4 * t * k * d}
    if entry == "round":
        return {"bytes": 2 * case["m"] * case["k"] * b, "flops": 4 * case["m"] * case["k"]}
    if entry == "product":
        m, n, k = case["m"] * case["top"], case["n"], case["k"]
        weights = case["experts"] * n * (k + 4)
        if case["experts"] > 1:
            weights = min(weights, m * n * (k + 4))
        return {"bytes": case["m"] * k * b + weights + m * n * b, "flops": 2 * m * n * k}
    t, v, d = case["t"], case["v"], case["d"]
    if entry == "embed":
        read = min(t, v) * d * b + (t * d * b if case["base"] else 0)
        return {"bytes": read + t * d * b + 4 * t, "flops": 2 * t * d}
    return {"bytes": t * d * b + 4 * t + 4 * v * d, "flops": t * d + v * d}


# --------------------------------------------------------------------------
# The definitions in 64 bits


def _exact_expert(case, s):
    entry, t, k, d = case["entry"], case["t"], case["k"], case["d"]
    x = s["x"].double()
    rows = torch.zeros((t * k, d), dtype=torch.float64, device=DEVICE)
    total = torch.zeros((t, d), dtype=torch.float64, device=DEVICE)
    dots = torch.zeros((t, k), dtype=torch.float64, device=DEVICE)
    if entry == "sum" and s["residual"] is not None:
        total += s["residual"].double()
    for j in range(k):
        at = s["positions"][:, j].long()
        have = (at >= 0).nonzero()[:, 0]
        at = at[have]
        w = s["weights"][have, j, None].double() if case["weighted"] else 1.0
        if entry in ("rows", "sum_back"):
            rows[at] = w * x[have]
        if entry != "rows":
            mine = s["rows"][at].double()
            total[have] += w * mine
            if entry != "sum":
                dots[have, j] = torch.linalg.vecdot(mine, x[have])
    return {"rows": {"rows": rows}, "sum": {"out": total},
            "rows_back": {"dx": total, "dweights": dots},
            "sum_back": {"drows": rows, "dweights": dots}}[entry]


def _exact_codes(x):
    """The rule's roundings to 32 bits, of quotients and products taken in 64."""
    x = x.double()
    top = torch.maximum(x.max(dim=1).values, -x.min(dim=1).values)
    scale = torch.maximum(top / 127, torch.full_like(top, LEAST)).float().double()
    inverse = (1 / scale).float().double()
    u = torch.einsum("mk,m->mk", x, inverse).float().double()
    low = torch.floor(u)
    over = u - low
    up = (over > 0.5) | ((over == 0.5) & (low % 2 == 1))
    return low + up, scale


def _exact_product(case, s):
    n, k, experts = case["n"], case["k"], case["experts"]
    q, scale = _exact_codes(s["x"])
    w = (s["codes"][:, :k].double() * s["scales"].double()[:, None]).view(experts, n, k)
    expert = torch.zeros(len(q), dtype=torch.long, device=DEVICE)
    if s["rows"] is not None:
        at = torch.arange(len(s["rows"]), device=DEVICE)
        expert = (at[:, None] >= s["offsets"][None, 1:-1]).sum(dim=1)
        q, scale = q[s["rows"].long()], scale[s["rows"].long()]
    z = torch.zeros((len(q), n), dtype=torch.float64, device=DEVICE)
    for x in range(experts):
        mine = (expert == x).nonzero()[:, 0]
        bias = None if s["bias"] is None else s["bias"][x].double()
        z[mine] = torch.nn.functional.linear(q[mine] * scale[mine, None], w[x], bias)
    if case["act"] == "silu":
        z = torch.nn.functional.silu(z)
    elif case["act"] == "gelu":
        z = torch.nn.functional.gelu(z)
    return z if s["row_scale"] is None else z * s["row_scale"].double()[:, None]


def _exact_embed(case, s):
    live = (s["ids"] >= 0).nonzero()[:, 0]
    ids = s["ids"][live].long()
    if case["entry"] == "embed":
        out = torch.zeros((case["t"], case["d"]), dtype=torch.float64, device=DEVICE)
        out[live] = s["scale"] * s["table"].double()[ids]
        return {"out": out if s["base"] is None else out + s["base"].double()}
    # By running sums over the tokens in their entries' order.
    order = ids.sort(stable=True)
    ends = torch.searchsorted(order.values, torch.arange(case["v"] + 1, device=DEVICE))
    total = torch.zeros((len(live) + 1, case["d"]), dtype=torch.float64, device=DEVICE)
    torch.cumsum(s["dout"].double()[live[order.indices]], dim=0, out=total[1:])
    return {"dtable": s["scale"] * (total[ends[1:]] - total[ends[:-1]])}


def exact(case, seed):
    entry, s = case["entry"], _inputs(case, seed)
    if entry in ("rows", "rows_back", "sum", "sum_back"):
        return _exact_expert(case, s)
    if entry == "round":
        q, scale = _exact_codes(s["x"])
        return {"values": q * scale[:, None]}
    if entry == "product":
        return {"y": _exact_product(case, s)}
    return _exact_embed(case, s)
