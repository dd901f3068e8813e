"""Operators of networks with 4-bit weights and of the optimiser beside them: cases, plain forms and values in 64 bits.

A 4-bit weight W [N, K] is held as codes [N, P / 2] (bytes; low nibble = even column, P = K rounded up to a whole group) and scales
[P / group, N]: W[n, k] = scales[k // group, n] * (code[n, k] - 8).  The operators:

  linear    y = x W^T + b
  interval  bounds of the same over boxes of x (centre and radius)
  rows      z = A W: a coefficient row pushed back through the layer
  train     linear with the gradients of x and b (the weight is frozen)
  quantise  codes and scales of a given weight
  adamw     one step over many tensors, moments in 32 bits, or in 8 with an exponent for each 256 of them

`own` selects between the plain forms here (elementary torch operations) and the package's operators.
"""
import torch

own = False

LR, BETAS, EPS, DECAY, STEPS = 1e-3, (0.9, 0.999), 1e-8, 0.01, 20
BLOCK = 256
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


def listed():
    return [
        # one input of a small image classifier's first layer, bounded: what a verifier asks for first; latency
        {"name": "bounds_one_input", "op": "interval", "rows": 1, "n": 512, "k": 784, "group": 32, "type": "fp32"},
        # four subdomains through a wide layer: the weights come from memory
        {"name": "bounds_wide_layer", "op": "interval", "rows": 4, "n": 8192, "k": 8192, "group": 128, "type": "fp32"},
        # nine sampled points through a layer whose sizes fit no tile
        {"name": "points_ragged", "op": "linear", "rows": 9, "n": 4001, "k": 4090, "group": 64, "type": "fp32"},
        # one token through the largest layer
        {"name": "one_token_large", "op": "linear", "rows": 1, "n": 16384, "k": 16384, "group": 128, "type": "bf16"},
        # the nine margins of a ten-class network, pushed back through a layer
        {"name": "margin_rows", "op": "rows", "rows": 9, "n": 4096, "k": 4096, "group": 128, "type": "fp32"},
        # sixteen tokens of a fine-tuning step around a frozen layer: output, gradient of the input and of the bias
        {"name": "train_frozen", "op": "train", "rows": 16, "n": 8192, "k": 4096, "group": 128, "type": "bf16"},
        # a small classifier's layer and a large model's, quantised
        {"name": "quantise_small", "op": "quantise", "n": 512, "k": 784, "group": 32, "type": "fp32"},
        {"name": "quantise_large", "op": "quantise", "n": 8192, "k": 8192, "group": 128, "type": "bf16"},
        # every weight and bias of a five-layer classifier: ten small tensors, latency
        {"name": "step_classifier", "op": "adamw", "bits": 32, "tensors": 10, "total": 1195018, "param": "fp32", "grad": "fp32"},
        # full-precision parameters with 16-bit gradients, forty tensors
        {"name": "step_large", "op": "adamw", "bits": 32, "tensors": 40, "total": 64000000, "param": "fp32", "grad": "bf16"},
        # moments in 8 bits: adapters beside frozen layers, of odd sizes
        {"name": "step8_adapters", "op": "adamw", "bits": 8, "tensors": 33, "total": 3300333, "param": "fp32", "grad": "fp32"},
        # moments in 8 bits where memory is what they save
        {"name": "step8_large", "op": "adamw", "bits": 8, "tensors": 40, "total": 64000000, "param": "bf16", "grad": "bf16"},
    ]


def draw(rng):
    spread = lambda lo, hi: int(round(lo * (hi / lo) ** rng.random()))  # noqa: E731
    op = rng.choice(["linear", "linear", "interval", "rows", "train", "quantise", "adamw", "adamw"])
    if op == "adamw":
        param = rng.choice(["fp32", "fp32", "bf16"])
        return {"op": op, "bits": rng.choice([32, 8]), "tensors": spread(1, 40), "total": spread(20000, 64000000), "param": param,
                "grad": rng.choice(["fp32", "bf16"]) if param == "fp32" else param}
    kind = "fp32" if op == "interval" else rng.choice(["fp32", "bf16", "fp16"])
    group, n = rng.choice([32, 64, 128]), spread(64, 16384)
    k = spread(64, 16384)
    if op == "quantise":
        return {"op": op, "n": n, "k": max(64, min(k, (1 << 26) // n)), "group": group, "type": kind}
    rows = spread(1, 64)
    return {"op": op, "rows": rows, "n": n, "k": max(64, min(k, (1 << 29) // (n * rows), (1 << 28) // n)), "group": group, "type": kind}


def _padded(case):
    return -(-case["k"] // case["group"]) * case["group"]


def _sizes(case):
    """Element counts of the tensors: layers and their biases, small beside large, whatever is left in the last."""
    count, total = case["tensors"], case["total"]
    parts = [(1 + (i * 37) % 11) * (40 if i % 2 == 0 else 1) for i in range(count)]
    sizes = [max(1, total * p // sum(parts)) for p in parts]
    sizes[-1] += max(0, total - sum(sizes))
    return sizes


def _flat(sizes):
    """Where each tensor's moments lie: at whole blocks of one buffer."""
    return [-(-s // BLOCK) * BLOCK for s in sizes]


def _inputs(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    if case["op"] == "adamw":
        sizes = _sizes(case)
        padded = sum(_flat(sizes))
        live = torch.cat([torch.arange(-(-s // BLOCK) * BLOCK, device="cuda") < s for s in sizes])  # behind each tensor's end there is nothing
        spread = torch.exp2(3 * normal(padded)) * live  # magnitudes of gradients differ by orders
        m, v = 1e-3 * spread * normal(padded), 1e-6 * spread.square() * normal(padded).square()
        d = {"sizes": sizes, "params": [(0.02 * normal(s)).to(TYPES[case["param"]]) for s in sizes],
             "grads": [(1e-3 * normal(s)).to(TYPES[case["grad"]]) for s in sizes]}
        if case["bits"] == 32:
            return d | {"m": m, "v": v}
        code = lambda top: torch.randint(0, top, (padded,), generator=g, device="cuda", dtype=torch.uint8)  # noqa: E731
        sign = 128 * torch.randint(0, 2, (padded,), generator=g, device="cuda", dtype=torch.uint8)
        exponent = lambda lo, hi: torch.randint(lo, hi, (padded // BLOCK,), generator=g, device="cuda", dtype=torch.uint8)  # noqa: E731
        return d | {"m": (code(128) + sign) * live, "v": (64 + code(192)) * live, "me": exponent(112, 120), "ve": exponent(100, 110)}
    n, k = case["n"], case["k"]
    if case["op"] == "quantise":
        return {"weight": (normal(n, k) * (2.0 / k) ** 0.5).to(TYPES[case["type"]])}
    padded, kind = _padded(case), TYPES[case["type"]]
    d = {"codes": torch.randint(0, 256, (n, padded // 2), generator=g, device="cuda", dtype=torch.uint8),
         "scales": (0.5 + torch.rand((padded // case["group"], n), generator=g, device="cuda")) * (0.25 * (2.0 / k) ** 0.5)}
    if case["op"] == "rows":
        return d | {"x": normal(case["rows"], n).to(kind)}
    x = normal(case["rows"], k)
    d["bias"] = (0.1 * normal(n)).to(kind)
    if case["op"] == "interval":
        r = 0.1 * torch.rand(x.shape, generator=g, device="cuda")
        return d | {"x": x - r, "upper": x + r}
    if case["op"] == "train":
        d["dy"] = normal(case["rows"], n).to(kind)
    return d | {"x": x.to(kind)}


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if case["op"] == "adamw":
        state["step"] = STEPS
        if own:
            from boundflow_b200.optim import AdamW

            opt = AdamW(state["params"], lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=case["bits"])
            moments = {"exp_avg": state["m"], "exp_avg_sq": state["v"]}
            if case["bits"] == 8:
                moments.update(exp_avg_exponent=state["me"], exp_avg_sq_exponent=state["ve"])
            opt.load_flat_moments(STEPS, **moments)
            for p, grad in zip(state["params"], state["grads"]):
                if p.dtype == grad.dtype:
                    p.grad = grad
            state["optimizer"] = opt
    elif own and case["op"] != "quantise":
        from boundflow_b200.weights4 import Weight4

        state["weight"] = Weight4(state["codes"], state["scales"], case["k"])
    if case["op"] == "train":
        state["x"].requires_grad_()
        state["bias"].requires_grad_()
    return state


def _run_own(state):
    from boundflow_b200 import weights4

    case = state["case"]
    op = case["op"]
    if op == "adamw":
        opt = state["optimizer"]
        opt.step(grads=None if case["param"] == case["grad"] else state["grads"])
        return state["params"] + list(opt.flat_moments())
    if op == "quantise":
        w = weights4.quantise_weight4(state["weight"], group=case["group"])
        return [w.integers(), w.scales]
    if op == "linear":
        return weights4.linear4(state["x"], state["weight"], state["bias"])
    if op == "interval":
        return list(weights4.interval_linear4(state["x"], state["upper"], state["weight"], state["bias"]))
    if op == "rows":
        return weights4.rows_times_weight4(state["x"], state["weight"])
    y = weights4.linear4(state["x"], state["weight"], state["bias"])
    return [y.detach(), *torch.autograd.grad(y, (state["x"], state["bias"]), state["dy"])]


# ---- plain forms -------------------------------------------------------------
def _dense(state):
    codes, scales, case = state["codes"], state["scales"], state["case"]
    q = torch.stack((codes & 15, codes >> 4), dim=2).float() - 8
    return (q.view(case["n"], -1, case["group"]) * scales.t().unsqueeze(2)).view(case["n"], -1)[:, : case["k"]]


def _decode(code, exponent, fields):
    """Magnitudes of 8-bit moments: `fields` of exponent and mantissa codes below their block's exponent."""
    e = exponent.int().repeat_interleave(BLOCK)
    bits = (code + ((e - fields) << 3)) << 20
    value = torch.where(code == 0, torch.zeros_like(bits), bits).view(torch.float32)
    return torch.where(e == 255, torch.full_like(value, float("nan")), value)


def _encode(value, noise, fields):
    """Codes and block exponents of non-negative moments: the bits behind the third of the mantissa are rounded up or down at random."""
    bits = value.view(torch.int32).long()
    top = bits.view(-1, BLOCK).amax(1)
    e = ((top + 0xFFFFF) >> 23).clamp(fields + 1, 254)
    e = torch.where(top >= 0x7F800000, torch.full_like(e, 255), e)
    rel = ((bits + noise) >> 20) - ((e - fields) << 3).repeat_interleave(BLOCK)
    return rel.clamp(0, 8 * fields + 7), e.to(torch.uint8)


def _mix(at, step):
    x = (at ^ (step * 0x9E3779B1)) & 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * 0x9BC84D59) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x7641A5C5) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _moments8(state):
    m, v = state["m"].int(), state["v"].int()
    size = _decode(m & 127, state["me"], 15)
    return torch.where(m >= 128, -size, size), _decode(v, state["ve"], 31)


def _adamw(state):
    case, sizes = state["case"], state["sizes"]
    slots = _flat(sizes)
    state["step"] += 1
    step = state["step"]
    m, v = (state["m"], state["v"]) if case["bits"] == 32 else _moments8(state)
    ms, vs = ([x[:s] for x, s in zip(t.split(slots), sizes)] for t in (m, v))
    p = [t.float() for t in state["params"]]
    grads = [t.float() for t in state["grads"]]
    torch._foreach_mul_(ms, BETAS[0])
    torch._foreach_add_(ms, torch._foreach_mul(grads, 1 - BETAS[0]))
    square = torch._foreach_mul(torch._foreach_mul(grads, 1 - BETAS[1]), grads)
    torch._foreach_mul_(vs, BETAS[1])
    torch._foreach_add_(vs, square)
    low = torch._foreach_div(torch._foreach_sqrt(vs), (1 - BETAS[1] ** step) ** 0.5)
    torch._foreach_add_(low, EPS)
    torch._foreach_mul_(p, 1 - LR * DECAY)
    torch._foreach_add_(p, torch._foreach_mul(torch._foreach_div(ms, low), -LR / (1 - BETAS[0] ** step)))
    torch._foreach_copy_(state["params"], p)
    if case["bits"] == 32:
        return state["params"] + [m, v]
    noise = _mix(torch.arange(m.numel(), device=m.device), step)
    code, state["me"] = _encode(m.abs(), noise & 0xFFFFF, 15)
    state["m"] = (code + 128 * ((m < 0) & (code > 0))).to(torch.uint8)
    code, state["ve"] = _encode(v, noise >> 12, 31)
    state["v"] = torch.where(v > 0, code.clamp(min=1), code).to(torch.uint8)
    return state["params"] + [t.bfloat16() for t in _moments8(state)]


def _quantise(state):
    case, w = state["case"], state["weight"].float()
    w = torch.nn.functional.pad(w, (0, _padded(case) - case["k"])).view(case["n"], -1, case["group"])
    scale = w.abs().amax(2) / 7
    q = torch.round(w / scale.unsqueeze(2)).clamp(-7, 7)
    q = torch.where(scale.unsqueeze(2) > 0, q, torch.zeros_like(q))
    return [q.view(case["n"], -1)[:, : case["k"]].to(torch.int8), scale.t().contiguous()]


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "adamw":
        return _adamw(state)
    if op == "quantise":
        return _quantise(state)
    with torch.no_grad():
        x, w = state["x"].float(), _dense(state)
        if op == "rows":
            return (x @ w).to(state["x"].dtype)
        bias = state["bias"].float()
        if op == "interval":
            c, r = (x + state["upper"]) / 2, (state["upper"] - x) / 2
            c, r = c @ w.t() + bias, r @ w.abs().t()
            return [c - r, c + r]
        y = (x @ w.t() + bias).to(state["x"].dtype)
        if op == "linear":
            return y
        dy = state["dy"].float()
        return [y, (dy @ w).to(y.dtype), dy.sum(0).to(y.dtype)]


def work(case):
    if case["op"] == "adamw":
        total, state = case["total"], 8 if case["bits"] == 32 else 2
        # 8-bit moments come back as the values that they stand for, in 16 bits
        per = 2 * BYTES[case["param"]] + BYTES[case["grad"]] + 2 * state + (4 if case["bits"] == 8 else 0)
        return {"bytes": total * per, "flops": 15 * total}
    n, k = case["n"], case["k"]
    groups = _padded(case) // case["group"]
    weight = n * k / 2 + 4 * n * groups
    if case["op"] == "quantise":
        return {"bytes": n * k * (BYTES[case["type"]] + 1) + 4 * n * groups, "flops": 3 * n * k}
    rows, b = case["rows"], BYTES[case["type"]]
    if case["op"] == "rows":
        return {"bytes": weight + b * rows * (n + k), "flops": 2 * rows * n * k}
    if case["op"] == "train":
        return {"bytes": weight + b * (2 * rows * (n + k) + 2 * n), "flops": 4 * rows * n * k}
    two = 2 if case["op"] == "interval" else 1
    return {"bytes": weight + b * (two * rows * (n + k) + n), "flops": 2 * two * rows * n * k}


# ---- values in 64 bits ---------------------------------------------------------
def exact(case, seed):
    data = _inputs(case, seed)
    if case["op"] == "adamw":
        return _exact_step(case, data)
    if case["op"] == "quantise":
        return _exact_codes(case, data["weight"].double())
    n, k, group = case["n"], case["k"], case["group"]
    column = torch.arange(k, device="cuda")
    byte = data["codes"][:, column // 2].int()
    q = torch.where(column % 2 == 1, byte >> 4, byte & 15)
    w = (q - 8).double()
    for j in range(data["scales"].shape[0]):
        w[:, j * group : (j + 1) * group] *= data["scales"][j].double()[:, None]
    x = data["x"].double()
    if case["op"] == "rows":
        return torch.matmul(x, w)
    bias = data["bias"].double()
    if case["op"] == "interval":
        up = data["upper"].double()
        plus, minus = w.clamp(min=0), w.clamp(max=0)
        return [x @ plus.t() + up @ minus.t() + bias, up @ plus.t() + x @ minus.t() + bias]
    y = torch.addmm(bias, x, w.t())
    if case["op"] == "linear":
        return y
    dy = data["dy"].double()
    return [y, dy @ w, torch.ones(1, dy.shape[0], dtype=torch.float64, device="cuda").matmul(dy).flatten()]


def _exact_codes(case, w):
    """A scale is a 32-bit number by definition, and so is what is rounded to a code: the quotient, rounded once."""
    codes, scales = [], []
    for first in range(0, case["k"], case["group"]):
        part = w[:, first : first + case["group"]]
        scale = (part.abs().max(dim=1).values / 7).float().double()
        quotient = (part / scale[:, None]).float().double()
        codes.append(torch.where(scale[:, None] > 0, quotient.round().clamp(-7, 7), torch.zeros_like(part)).to(torch.int8))
        scales.append(scale)
    return [torch.cat(codes, dim=1), torch.stack(scales)]


def _exact_step(case, data):
    """Moments are 32-bit numbers by definition, and each product and sum of theirs is rounded once; 8-bit ones follow from those."""
    once = lambda t: t.float().double()  # noqa: E731
    f32 = lambda x: float(torch.tensor(x, dtype=torch.float32))  # noqa: E731
    b1, b2, t = f32(BETAS[0]), f32(BETAS[1]), STEPS + 1
    params, moments, at = [], ([], []), 0
    for p, grad, size in zip(data["params"], data["grads"], data["sizes"]):
        slot = -(-size // BLOCK) * BLOCK
        here, g = slice(at, at + slot), torch.zeros(slot, dtype=torch.float64, device="cuda")
        g[:size] = grad.double()
        if case["bits"] == 32:
            m, v = data["m"][here].double(), data["v"][here].double()
        else:
            blocks = slice(at // BLOCK, (at + slot) // BLOCK)
            mc, vc = data["m"][here].double(), data["v"][here].double()
            m = _exact_value(mc % 128, data["me"][blocks], 15) * torch.where(mc >= 128, -1.0, 1.0)
            v = _exact_value(vc, data["ve"][blocks], 31)
        m1 = once(once(b1 * m) + once(f32(1 - BETAS[0]) * g))
        v1 = once(once(b2 * v) + once(once(f32(1 - BETAS[1]) * g) * g))
        step = (m1 / (1 - BETAS[0] ** t)) / ((v1 / (1 - BETAS[1] ** t)).sqrt() + EPS)
        params.append(p.double() * (1 - LR * DECAY) - LR * step[:size])
        if case["bits"] == 8:
            noise = _mix(torch.arange(at, at + slot, device="cuda"), t)
            m1 = _exact_coded(m1.abs(), noise % 2**20, 15, False) * m1.sign()
            v1 = _exact_coded(v1, noise // 2**12, 31, True)
        moments[0].append(m1)
        moments[1].append(v1)
        at += slot
    return params + [torch.cat(m) for m in moments]


def _exact_value(code, exponent, fields):
    """(1 + mantissa / 8) 2^(exponent - fields + code // 8 - 127), and zero for the code zero."""
    e = exponent.double().repeat_interleave(BLOCK) - fields + torch.floor(code / 8) - 127
    return torch.where(code > 0, (1 + code % 8 / 8) * torch.exp2(e), torch.zeros_like(code))


def _exact_coded(value, noise, fields, keep):
    """What the code of a moment stands for: eighths of a power of two, the rest carried up where it and 20 random bits reach one."""
    mantissa, e = torch.frexp(value)  # value = mantissa 2^e, mantissa in [1/2, 1)
    eighths = mantissa * 16 - 8  # of 2^(e - 1)
    low = torch.floor(eighths)
    up = low + ((eighths - low) * 2**20 + noise >= 2**20)
    place = torch.where(value > 0, 8 * (e.double() + 126) + up, torch.zeros_like(value))  # biased exponent and mantissa as one number
    top = value.view(-1, BLOCK).amax(1)
    mantissa, e = torch.frexp(top)
    shared = torch.where(top > 0, e.double() + 126 + (mantissa * 16 > 15), torch.zeros_like(top)).clamp(fields + 1, 254).repeat_interleave(BLOCK)
    code = (place - 8 * (shared - fields)).clamp(0, 8 * fields + 7)
    if keep:
        code = torch.where(value > 0, code.clamp(min=1), code)
    return torch.where(code > 0, (1 + code % 8 / 8) * torch.exp2(shared - fields + torch.floor(code / 8) - 127), torch.zeros_like(code))
