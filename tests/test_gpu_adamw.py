"""AdamW over many tensors against its definition.

Moments are compared bit for bit: a product of two float32 values is exact in float64, so rounding to float32 behind each operation gives that operation's
float32 result.  Parameters: three operations of the decay and the sum, and a step that is off by a handful of 2^-24 of itself; 16 of them are allowed for
it, and half a step of the parameter's type.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
PAIRS = [("fp32", "fp32"), ("fp32", "bf16"), ("fp32", "fp16"), ("bf16", "bf16"), ("fp16", "fp16")]
BLOCK = 256


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from boundflow_b200.csrc import build

    build.build()
    return torch.device("cuda", 0)


def f32(x):
    return float(torch.tensor(x, dtype=torch.float32))


def once(t):
    return t.float().double()


def moments(m, v, g, betas):
    m1 = once(once(f32(betas[0]) * m) + once(f32(1 - betas[0]) * g))
    v1 = once(once(f32(betas[1]) * v) + once(once(f32(1 - betas[1]) * g) * g))
    return m1, v1


def check_params(got, before, m, v, t, lr, wd, betas, eps):
    old = before.double()
    move = lr * (m / (1 - betas[0] ** t)) / ((v / (1 - betas[1] ** t)).sqrt() + eps)
    want = old * (1 - lr * wd) - move
    half = torch.finfo(got.dtype).eps / 2
    tol = (half * 1.01 + 3 * 2.0 ** -24) * (old.abs() + move.abs()) + 16 * 2.0 ** -24 * move.abs() + torch.finfo(got.dtype).tiny
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"worst {float((err / tol).max()):.2f} of the tolerance"


def make(sizes, kinds, dev, seed):
    g = torch.Generator("cpu").manual_seed(seed)
    params = [torch.randn(s, generator=g).to(TYPES[kinds[0]]).to(dev) for s in sizes]
    grads = [(torch.randn(s, generator=g) * torch.exp2(2 * torch.randn(s, generator=g))).to(TYPES[kinds[1]]).to(dev) for s in sizes]
    return params, grads


# an independent statement of the 8-bit format, value by value
def stands_for(code, e, fields):
    e = e.double().repeat_interleave(BLOCK)
    value = torch.where(code > 0, (1 + code % 8 / 8) * torch.exp2(e - fields + torch.floor(code / 8) - 127), torch.zeros_like(code))
    return torch.where(e == 255, torch.full_like(value, math.nan), value)


def coded(value, noise, fields, keep):
    mantissa, e = torch.frexp(value)
    eighths = mantissa * 16 - 8
    low = torch.floor(eighths)
    up = low + ((eighths - low) * 2 ** 20 + noise >= 2 ** 20)
    place = torch.where(value > 0, 8 * (e.double() + 126) + up, torch.zeros_like(value))
    mantissa, e = torch.frexp(value.view(-1, BLOCK).amax(1))
    shared = torch.where(mantissa > 0, e.double() + 126 + (mantissa * 16 > 15), torch.zeros_like(mantissa)).clamp(fields + 1, 254)
    code = (place - 8 * (shared.repeat_interleave(BLOCK) - fields)).clamp(0, 8 * fields + 7)
    return (torch.where(value > 0, code.clamp(min=1), code) if keep else code), shared


def noise_of(at, step):
    x = (at ^ (step * 0x9E3779B1)) & 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * 0x9BC84D59) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x7641A5C5) & 0xFFFFFFFF
    return x ^ (x >> 16)


@pytest.mark.parametrize("kinds", PAIRS)
@pytest.mark.parametrize("sizes", [[1], [5, 0, 255, 256, 257], [2048, 2049, 4099, 3], [70000]])
def test_step32(dev, kinds, sizes):
    from boundflow_b200.optim import AdamW

    params, grads = make(sizes, kinds, dev, sum(sizes))
    opt = AdamW(params, lr=3e-3, betas=(0.8, 0.95), eps=1e-6, weight_decay=0.1)
    m, v = ([torch.zeros(s, dtype=torch.float64, device=dev) for s in sizes] for _ in range(2))
    for t in (1, 2, 3):
        before = [p.clone() for p in params]
        opt.step(grads)
        for k, s in enumerate(sizes):
            at = opt.moment_offsets[k]
            m[k], v[k] = moments(m[k], v[k], grads[k].double(), (0.8, 0.95))
            assert torch.equal(opt.exp_avg[at:at + s].double(), m[k]) and torch.equal(opt.exp_avg_sq[at:at + s].double(), v[k])
            check_params(params[k], before[k], m[k], v[k], t, 3e-3, 0.1, (0.8, 0.95), 1e-6)
    assert opt.steps == 3


@pytest.mark.parametrize("kinds", PAIRS)
@pytest.mark.parametrize("sizes", [[1], [5, 0, 255, 256, 257], [2048, 2049, 4099, 3], [70000]])
def test_step8(dev, kinds, sizes):
    from boundflow_b200.optim import AdamW

    params, grads = make(sizes, kinds, dev, 1 + sum(sizes))
    betas = (0.9, 0.999)
    opt = AdamW(params, lr=3e-3, state_bits=8)
    m, v = (torch.zeros_like(opt.exp_avg, dtype=torch.float64) for _ in range(2))
    place = torch.arange(m.numel(), device=dev)
    for t in (1, 2, 3, 4):
        before = [p.clone() for p in params]
        opt.step(grads)
        for k, s in enumerate(sizes):
            at = slice(opt.moment_offsets[k], opt.moment_offsets[k] + s)
            m[at], v[at] = moments(m[at], v[at], grads[k].double(), betas)
            check_params(params[k], before[k], m[at], v[at], t, 3e-3, 1e-2, betas, 1e-8)
        noise = noise_of(place, t)
        mc, me = coded(m.abs(), noise % 2 ** 20, 15, False)
        vc, ve = coded(v, noise // 2 ** 12, 31, True)
        used = m.view(-1, BLOCK).any(1) | v.view(-1, BLOCK).any(1)
        m, v = stands_for(mc, me, 15) * m.sign(), stands_for(vc, ve, 31)
        assert torch.equal(opt.exp_avg_exponent[used].double(), me[used]) and torch.equal(opt.exp_avg_sq_exponent[used].double(), ve[used])
        assert torch.equal((opt.exp_avg & 127).double(), mc) and torch.equal(opt.exp_avg_sq.double(), vc)
        got_m, got_v = opt.flat_moments()
        assert torch.equal(got_m.double(), m) and torch.equal(got_v.double(), v)


def test_8_bit_moments_follow_32_bit_ones(dev):
    """Codes are an eighth apart, a step moves the second moment by a thousandth: the mean over many elements has to follow all the same.  A code is off by
    at most 1/8 of its value each time, the part that remains of it decays by beta: a random walk of variance (1/8)^2 / 4 / (1 - beta^2) at most, so the mean
    over n elements is within 6 / 8 / 2 / sqrt((1 - beta^2) n) of that of the 32-bit moments."""
    from boundflow_b200.optim import AdamW

    n = 1 << 18
    g = torch.Generator("cuda").manual_seed(5)
    opts = [AdamW([torch.zeros(n, device=dev)], lr=0.0, betas=(0.9, 0.99), state_bits=b) for b in (32, 8)]
    for t in range(300):
        grad = torch.randn(n, generator=g, device=dev) * (1.0 if t < 100 else 4.0) + 1.0
        for o in opts:
            o.step([grad])
    (m, v), (m8, v8) = (o.flat_moments() for o in opts)
    assert abs(float(m8.double().mean() / m.double().mean()) - 1) < 0.375 / math.sqrt((1 - 0.81) * n) * float(m.abs().double().mean() / m.double().mean()) + 1e-3
    assert abs(float(v8.double().mean() / v.double().mean()) - 1) < 0.375 / math.sqrt((1 - 0.9801) * n) + 1e-3
    assert float((v8.double() > 0).double().mean()) == 1.0


@pytest.mark.parametrize("bits", [32, 8])
def test_views_many_tensors_groups_and_missing_gradients(dev, bits):
    """Over 512 tensors (several launches), parameters off a 16-byte boundary, strided gradients, two groups, tensors without a gradient, mixed types: as a
    step for each tensor alone."""
    from boundflow_b200.optim import AdamW

    g = torch.Generator("cpu").manual_seed(9)
    sizes = [1 + int(x) for x in torch.randint(0, 600, (700,), generator=g)]
    buf = torch.randn(sum(sizes) + 1, generator=g).to(dev)
    params = [t for t in buf[1:].split(sizes)]
    params[10], params[11] = params[10].bfloat16(), params[11].half()
    grads = [torch.randn(2 * s, generator=g).to(dev)[::2] for s in sizes]
    grads[10], grads[11], grads[12], grads[13] = grads[10].bfloat16(), grads[11].half(), grads[12].bfloat16(), None
    for k in (10, 11, 12):
        assert grads[k].numel() == sizes[k]
    before = [p.clone() for p in params]
    scale = torch.tensor([0.5], device=dev)
    opt = AdamW([{"params": params[:300], "lr": 0.01}, {"params": params[300:], "lr": 0.02, "weight_decay": 0.0}], weight_decay=0.5, state_bits=bits)
    for t in (1, 2):
        opt.step(grads, grad_scale=scale)
    assert opt.steps == 2 and torch.equal(params[13], before[13])
    for k in (0, 10, 11, 12, 299, 300, 511, 512, 699):
        m = v = torch.zeros(sizes[k], dtype=torch.float64, device=dev)
        gk, now = 0.5 * grads[k].double(), before[k]
        alone = AdamW([now], lr=0.01 if k < 300 else 0.02, weight_decay=0.5 if k < 300 else 0.0)
        for t in (1, 2):
            alone.step([grads[k]], grad_scale=scale)
        m, v = alone.flat_moments()
        if bits == 32:
            at = slice(opt.moment_offsets[k], opt.moment_offsets[k] + sizes[k])
            assert torch.equal(opt.exp_avg[at], m[: sizes[k]]) and torch.equal(opt.exp_avg_sq[at], v[: sizes[k]]) and torch.equal(params[k], now)
        else:  # an eighth of the first moment and of the second is what one rounding can change of the second step
            lr = 0.01 if k < 300 else 0.02
            assert bool(((params[k].double() - now.double()).abs() <= 0.3 * lr * 2 + 2 ** -7 * now.double().abs()).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_infinities_and_nan_stay_in_their_place(dev, bits):
    from boundflow_b200.optim import AdamW

    p = torch.ones(3 * BLOCK, device=dev)
    grad = torch.linspace(-1, 1, 3 * BLOCK, device=dev)
    grad[BLOCK + 3], grad[2 * BLOCK + 1] = float("nan"), float("inf")
    opt = AdamW([p], state_bits=bits)
    opt.step([grad])
    bad = torch.zeros(3 * BLOCK, dtype=torch.bool, device=dev)
    bad[BLOCK + 3] = bad[2 * BLOCK + 1] = True
    assert torch.equal(p.isnan(), bad)  # inf / inf
    opt.step([torch.zeros_like(grad)])
    if bits == 8:
        bad[BLOCK:] = True  # the block's exponent is gone
    assert torch.equal(p.isnan(), bad)


def test_zero_gradients_and_smallest_values(dev):
    """No gradient at all moves a parameter by its decay alone; gradients whose square is below the normal range do not divide by zero."""
    from boundflow_b200.optim import AdamW

    for bits in (32, 8):
        p = torch.ones(300, device=dev)
        AdamW([p], lr=0.1, weight_decay=0.5, state_bits=bits).step([torch.zeros(300, device=dev)])
        assert torch.allclose(p, torch.full_like(p, 0.95), rtol=2 ** -22, atol=0)
        p = torch.zeros(300, device=dev)
        opt = AdamW([p], lr=0.1, weight_decay=0.0, state_bits=bits)
        for _ in range(3):
            opt.step([torch.full((300,), 1e-25, device=dev)])
        assert p.isfinite().all() and float(p.abs().max()) <= 3 * 0.1 * 1e-15


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_counts(dev, bits):
    from boundflow_b200.optim import AdamW

    params, grads = make([1000, 77], ("fp32", "fp32"), dev, 3)
    other = [p.clone() for p in params]
    a, b = AdamW(params, state_bits=bits), AdamW(other, state_bits=bits)
    a.step(grads)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step(grads)
    for _ in range(3):
        graph.replay()
    for _ in range(4):
        b.step(grads)
    assert a.steps == b.steps == 4
    assert all(torch.equal(x, y) for x, y in zip(params + list(a.flat_moments()), other + list(b.flat_moments())))


@pytest.mark.parametrize("bits", [32, 8])
def test_state_round_trip_versions_and_refusals(dev, bits):
    from boundflow_b200.optim import AdamW

    params, grads = make([100, 300], ("fp32", "fp32"), dev, 4)
    opt = AdamW(params, state_bits=bits)
    for p, g in zip(params, grads):
        p.grad = g
    versions = [p._version for p in params]
    opt.step()
    opt.step()
    assert all(p._version > v for p, v in zip(params, versions))
    copies = [p.clone() for p in params]
    again = AdamW(copies, lr=0.5, state_bits=bits)
    again.load_state_dict(opt.state_dict())
    assert again.param_groups[0]["lr"] == opt.param_groups[0]["lr"]
    opt.step()
    again.step(grads)
    assert again.steps == 3 and all(torch.equal(x, y) for x, y in zip(params, copies))
    opt.zero_grad()
    now = [p.clone() for p in params]
    opt.step()  # no gradient anywhere: nothing happens
    assert opt.steps == 3 and all(torch.equal(x, y) for x, y in zip(params, now))
    for call, error in [
        (lambda: opt.step([grads[0]]), ValueError), (lambda: opt.step([grads[1], grads[0]]), ValueError), (lambda: opt.step([g.double() for g in grads]), TypeError),
        (lambda: opt.step([g.cpu() for g in grads]), ValueError), (lambda: opt.step(grads, grad_scale=torch.ones(2, device=dev)), ValueError),
        (lambda: opt.step(grads, grad_scale=torch.ones(1)), ValueError), (lambda: AdamW([params[0], params[0][5:]]), ValueError),
        (lambda: AdamW([params[1].view(30, 10).t()]), ValueError), (lambda: AdamW([params[0].bfloat16()]).step([grads[0]]), TypeError),
        (lambda: again.load_state_dict(AdamW([params[0]], state_bits=bits).state_dict()), ValueError),
        (lambda: opt.load_flat_moments(1, exp_avg=opt.exp_avg), ValueError),
    ]:
        with pytest.raises(error):
            call()
    moved = torch.zeros(10, device=dev)
    left = AdamW([moved], state_bits=bits)
    moved.data = moved.data.cpu()
    with pytest.raises(ValueError):
        left.step([torch.zeros(10)])
    moved.data = torch.zeros(5, device=dev)
    with pytest.raises(ValueError):
        left.step([torch.zeros(5, device=dev)])
    with pytest.raises(ValueError):
        left.step([torch.zeros(5, device=dev).to_sparse()])
    opt.param_groups[0]["lr"] = -1.0
    with pytest.raises(ValueError):
        opt.step(grads)
