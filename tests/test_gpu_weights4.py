"""Products with 4-bit weights against the same in 64 bits.

Tolerances: every product x * q is exact in the tensor cores' or the FMA's 32-bit sums up to their rounding, so an output is off by at most
(terms + a few) * 2^-24 of the sum of the magnitudes it adds up; T below allows 2^-24 * (K / 8 + 32) of that sum (partial sums of a few terms each, added
pairwise or in short chains), and half a step of the output's type where that is shorter than 32 bits.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from boundflow_b200.csrc import build

    build.build()
    return torch.device("cuda", 0)


def make(n, k, group, dev, seed=0):
    from boundflow_b200.weights4 import Weight4

    g = torch.Generator("cpu").manual_seed(seed + 1000 * n + k + group)
    padded = -(-k // group) * group
    codes = torch.randint(0, 256, (n, padded // 2), generator=g, dtype=torch.uint8)
    scales = torch.rand((padded // group, n), generator=g) + 0.25
    q = torch.stack((codes & 15, codes >> 4), dim=2).reshape(n, padded).double() - 8
    w = (q * scales.double().t().repeat_interleave(group, dim=1))[:, :k]
    return Weight4(codes.to(dev), scales.to(dev), k), w.to(dev), g


def check(got, want, size, terms, dtype):
    """`size`: the sum of magnitudes behind each output."""
    eps = torch.finfo(dtype).eps if dtype != torch.float32 else 0.0
    tol = 2.0 ** -24 * (terms / 8 + 32) * size + eps / 2 * want.abs() * 1.01 + (torch.finfo(dtype).tiny if eps else 0.0)
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"worst {float((err / tol.clamp(min=1e-300)).max()):.2f} of the tolerance"


SHAPES = [(1, 1, 32), (3, 31, 32), (16, 64, 64), (17, 33, 32), (40, 128, 128), (100, 257, 64), (129, 500, 128), (512, 784, 32), (33, 1000, 256), (1000, 1111, 128),
          (48, 3000, 32), (2050, 640, 64), (5, 9000, 128), (9, 200, 512)]
ROWS = [1, 2, 3, 5, 8, 9, 16, 17, 40]


@pytest.mark.parametrize("n,k,group", SHAPES)
@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
def test_linear(dev, n, k, group, kind):
    from boundflow_b200.weights4 import linear4

    W, w, g = make(n, k, group, dev)
    for m in ROWS:
        x = torch.randn(m, k, generator=g).to(TYPES[kind]).to(dev)
        b = torch.randn(n, generator=g).to(dev)
        got = linear4(x, W, b)
        assert got.shape == (m, n) and got.dtype == x.dtype
        xd = x.double()
        check(got, xd @ w.t() + b.double(), xd.abs() @ w.abs().t() + b.double().abs(), k, x.dtype)
    check(linear4(x, W), xd @ w.t(), xd.abs() @ w.abs().t(), k, x.dtype)


@pytest.mark.parametrize("n,k,group", SHAPES)
def test_interval(dev, n, k, group):
    from boundflow_b200.weights4 import interval_linear4

    W, w, g = make(n, k, group, dev, 1)
    b = torch.randn(n, generator=g).to(dev)
    for m in ROWS:
        x, r = torch.randn(m, k, generator=g).to(dev), torch.rand(m, k, generator=g).to(dev)
        for relu in (False, True):
            lo, up = x - r, x + r
            yl, yu = interval_linear4(lo, up, W, b, relu_in=relu)
            l, u = (t.double().clamp(min=0) if relu else t.double() for t in (lo, up))
            plus, minus = w.clamp(min=0), w.clamp(max=0)
            size = (l.abs() + u.abs()) @ w.abs().t() + b.double().abs()
            check(yl, l @ plus.t() + u @ minus.t() + b.double(), size, k, torch.float32)
            check(yu, u @ plus.t() + l @ minus.t() + b.double(), size, k, torch.float32)


@pytest.mark.parametrize("n,k,group", SHAPES)
@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
def test_rows(dev, n, k, group, kind):
    """16-bit rows times a 32-bit scale are held in two bfloat16 parts: off by 2^-17 of each term beside the rounding of the result."""
    from boundflow_b200.weights4 import rows_times_weight4

    W, w, g = make(n, k, group, dev, 2)
    for m in ROWS:
        a = torch.randn(m, n, generator=g).to(TYPES[kind]).to(dev)
        got = rows_times_weight4(a, W)
        assert got.shape == (m, k) and got.dtype == a.dtype
        size = a.double().abs() @ w.abs()
        tol_terms = n if kind == "fp32" else n + 8 * 2 ** 7
        check(got, a.double() @ w, size, tol_terms, a.dtype)


@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("m,n,k,group", [(1, 7, 40, 32), (4, 130, 300, 64), (19, 65, 129, 128)])
def test_linear_gradients(dev, kind, m, n, k, group):
    from boundflow_b200.weights4 import linear4

    W, w, g = make(n, k, group, dev, 3)
    x = torch.randn(2, m, k, generator=g).to(TYPES[kind]).to(dev).requires_grad_()
    b = torch.randn(n, generator=g).to(TYPES[kind]).to(dev).requires_grad_()
    dy = torch.randn(2, m, n, generator=g).to(TYPES[kind]).to(dev)
    y = linear4(x, W, b)
    assert y.shape == (2, m, n)
    gx, gb = torch.autograd.grad(y, (x, b), dy)
    assert gx.dtype == x.dtype and gb.dtype == b.dtype and gx.shape == x.shape
    d = dy.double()
    check(gx, d @ w, d.abs() @ w.abs(), n if kind == "fp32" else n + 8 * 2 ** 7, x.dtype)
    check(gb, d.sum((0, 1)), d.abs().sum((0, 1)), 2 * m * 8, b.dtype)


def test_gradients_of_gradients(dev):
    """d / d dy of (dx . v) is v W^T, and d / d a of (a W . v) the same: products with the weight again."""
    from boundflow_b200.weights4 import linear4, rows_times_weight4

    W, w, g = make(70, 90, 32, dev, 8)
    x, b = torch.randn(3, 90, generator=g).to(dev).requires_grad_(), torch.randn(70, generator=g).to(dev).requires_grad_()
    dy, v, u = torch.randn(3, 70, generator=g).to(dev).requires_grad_(), torch.randn(3, 90, generator=g).to(dev), torch.randn(70, generator=g).to(dev)
    gx, gb = torch.autograd.grad(linear4(x, W, b), (x, b), dy, create_graph=True)
    got, = torch.autograd.grad((gx, gb), dy, (v, u))
    check(got, v.double() @ w.t() + u.double(), v.double().abs() @ w.abs().t() + u.double().abs(), 90, torch.float32)
    a = torch.randn(2, 2, 70, generator=g).to(dev).requires_grad_()
    got, = torch.autograd.grad(rows_times_weight4(a, W), a, v[:2].expand(2, 2, 90))
    check(got, (v[:2].double() @ w.t()).expand(2, 2, 70), (v[:2].double().abs() @ w.abs().t()).expand(2, 2, 70), 90, torch.float32)


@pytest.mark.parametrize("m,n,k,group", [(1, 7, 40, 32), (4, 130, 300, 64), (19, 65, 129, 128)])
def test_interval_gradients(dev, m, n, k, group):
    """Against the formula and against differences: the bounds are linear in lower and upper while W keeps its signs, so a difference of any length is exact."""
    from boundflow_b200.weights4 import interval_linear4

    W, w, g = make(n, k, group, dev, 4)
    lo = torch.randn(m, k, generator=g).to(dev).requires_grad_()
    up = (lo.detach() + torch.rand(m, k, generator=g).to(dev)).requires_grad_()
    b = torch.randn(n, generator=g).to(dev).requires_grad_()
    dl, du = torch.randn(m, n, generator=g).to(dev), torch.randn(m, n, generator=g).to(dev)
    yl, yu = interval_linear4(lo, up, W, b)
    gl, gu, gb = torch.autograd.grad((yl, yu), (lo, up, b), (dl, du))
    plus, minus = w.clamp(min=0), w.clamp(max=0)
    d, e = dl.double(), du.double()
    size = (d.abs() + e.abs()) @ w.abs()
    check(gl, d @ plus + e @ minus, size, n, torch.float32)
    check(gu, e @ plus + d @ minus, size, n, torch.float32)
    check(gb, d.sum(0) + e.sum(0), d.abs().sum(0) + e.abs().sum(0), 8 * m, torch.float32)
    step = torch.randn(m, k, generator=g).to(dev)
    with torch.no_grad():
        zl, zu = interval_linear4(lo + step, up + step.abs() + step, W, b)  # upper stays above lower
        moved = ((zl - yl).double() * d + (zu - yu).double() * e).sum()
    told = (gl.double() * step.double()).sum() + (gu.double() * (step.abs() + step).double()).sum()
    scale = float((((lo.abs() + up.abs() + 3 * step.abs()).detach().double() @ w.abs().t() + 1) * (d.abs() + e.abs())).sum())
    assert abs(float(moved - told)) <= 2.0 ** -24 * (k / 8 + n / 8 + 64) * scale


@pytest.mark.parametrize("n,k,group", [(1, 1, 32), (7, 45, 32), (64, 784, 64), (130, 1025, 128), (33, 300, 512)])
@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
def test_quantise(dev, n, k, group, kind):
    from boundflow_b200.weights4 import quantise_weight4

    g = torch.Generator("cpu").manual_seed(n + k)
    W = (torch.randn(n, k, generator=g) * 0.3).to(TYPES[kind])
    W[0, : min(k, group)] = 0                      # a group of zeros
    if n > 3:
        W[1, 0], W[2, k - 1] = float("nan"), float("inf")   # groups that hold what no scale can
        W[3] = torch.tensor(7 / 2.0).to(TYPES[kind])        # ties: w / scale = 7 at the largest, all equal
    got = quantise_weight4(W.to(dev), group)
    padded = -(-k // group) * group
    blocks = torch.nn.functional.pad(W.double(), (0, padded - k)).view(n, -1, group)
    scale = (blocks.abs().amax(2) * float(torch.tensor(1.0) / 7)).float().double()
    q = (blocks / scale.unsqueeze(2)).float().double().round().clamp(-7, 7)
    fine = scale.isfinite()
    q = torch.where((scale > 0).unsqueeze(2) & fine.unsqueeze(2), q, torch.zeros_like(q))
    s = got.scales.t().double().cpu()
    assert torch.equal(s[fine], scale[fine]) and not s[~fine].isfinite().any()
    assert torch.equal(got.integers().cpu(), q.view(n, -1)[:, :k].to(torch.int8))
    dense = got.dense().cpu().double()
    want = (q * s.unsqueeze(2)).view(n, -1)[:, :k].float().double()
    assert torch.equal(dense.isnan(), want.isnan()) and torch.equal(dense[~want.isnan()], want[~want.isnan()])
    # within half a code of the weight
    ok = fine.unsqueeze(2).expand(-1, -1, group).reshape(n, -1)[:, :k]
    half = (0.5 + 1e-6) * scale.unsqueeze(2).expand(-1, -1, group).reshape(n, -1)[:, :k] + 2.0 ** -22 * W.double().abs()
    assert bool(((dense - W.double()).abs() <= half)[ok].all())


def test_empty_strides_and_places(dev):
    """No rows, rows that are views with other strides or off a 16-byte boundary, a leading shape, CPU tensors, another stream."""
    from boundflow_b200.weights4 import interval_linear4, linear4, rows_times_weight4

    W, w, g = make(37, 70, 32, dev, 5)
    assert linear4(torch.empty(0, 70, device=dev), W).shape == (0, 37)
    assert rows_times_weight4(torch.empty(0, 37, device=dev), W).shape == (0, 70)
    assert interval_linear4(torch.empty(0, 70, device=dev), torch.empty(0, 70, device=dev), W)[0].shape == (0, 37)
    x = torch.randn(3, 5, 71, generator=g).to(dev)
    want = linear4(x[..., 1:].contiguous().clone(), W)
    assert torch.equal(linear4(x[..., 1:], W), want) and want.shape == (3, 5, 37)
    flat = torch.randn(1 + 4 * 70, generator=g).to(dev)
    assert torch.equal(linear4(flat[1:].view(4, 70), W), linear4(flat[1:].clone().view(4, 70), W))
    one = linear4(x[0, 0, 1:], W)
    assert one.shape == (37,) and torch.equal(one, linear4(x[0, 0, 1:].unsqueeze(0).contiguous(), W)[0])
    t = torch.randn(70, 6, generator=g).to(dev)
    assert torch.equal(linear4(t.t(), W), linear4(t.t().contiguous(), W))
    c = linear4(x[0, :, 1:].cpu(), W.to("cpu"))
    assert c.device.type == "cpu" and torch.equal(c, linear4(x[0, :, 1:], W).cpu())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = linear4(x[0, :, 1:], W)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, linear4(x[0, :, 1:], W))


def test_special_values(dev):
    """Infinities and NaN of the input reach the outputs that read them, and no others; what lies in a row's padding reaches none."""
    from boundflow_b200.weights4 import Weight4, interval_linear4, linear4, rows_times_weight4

    n, k, group = 50, 200, 64
    W, w, g = make(n, k, group, dev, 6)
    x = torch.randn(12, k, generator=g).to(dev)
    clean = linear4(x, W)
    x2 = x.clone()
    x2[3, 17], x2[5, 199] = float("nan"), float("inf")
    got = linear4(x2, W)
    keep = [i for i in range(12) if i not in (3, 5)]
    assert torch.equal(got[keep], clean[keep]) and got[3].isnan().all()
    q = w[:, 199]
    assert got[5][q == 0].isnan().all() and (got[5][q > 0] == float("inf")).all() and (got[5][q < 0] == -float("inf")).all()
    codes = W.codes.clone()
    codes[:, 100:] = 0xFF   # the padding behind column 199
    assert torch.equal(linear4(x, Weight4(codes, W.scales, k)), clean)
    a = torch.randn(4, n, generator=g).to(dev)
    assert torch.equal(rows_times_weight4(a, Weight4(codes, W.scales, k)), rows_times_weight4(a, W))
    a2 = a.clone()
    a2[1, 49] = float("nan")
    z, z2 = rows_times_weight4(a, W), rows_times_weight4(a2, W)
    assert z2[1].isnan().all() and torch.equal(z2[[0, 2, 3]], z[[0, 2, 3]])
    lo, up = x - 0.1, x + 0.1
    yl, yu = interval_linear4(lo, up, W)
    lo2 = lo.clone()
    lo2[0, 0] = float("nan")
    zl, zu = interval_linear4(lo2, up, W)
    assert zl[0].isnan().all() and torch.equal(zl[1:], yl[1:]) and torch.equal(zu[1:], yu[1:])
    tiny = torch.full((1, k), 1e-40, device=dev)  # below the normal range: at most lost, never garbage
    assert float(linear4(tiny, W).abs().max()) <= 1e-35


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5])
def test_16_bit_rows_of_all_magnitudes(dev, kind, m):
    """Few 16-bit rows are counted in units of 2^-30 of the largest of 128 columns: off by half a unit, beside the rounding of the result.  Magnitudes over the whole
    range of the type, its largest and smallest, zeros, and rows of infinities and NaN."""
    from boundflow_b200.weights4 import linear4

    n, k, group = 70, 700, 64
    W, w, g = make(n, k, group, dev, 9)
    t = TYPES[kind]
    span = 30 if kind == "bf16" else 5
    x = (torch.randn(m, k, generator=g) * torch.exp2(span * torch.randn(m, k, generator=g).clamp(-3, 3))).clamp(-6e4, 6e4).to(t).to(dev)
    x[0, :128] = torch.finfo(t).tiny / 2   # a whole chunk below the normal range
    x[0, 128:256] = 0
    x[m - 1, 300], x[m - 1, 301] = 60000.0, -torch.finfo(t).tiny
    xd = x.double()
    top = torch.nn.functional.pad(xd.abs(), (0, 68)).view(m, -1, 128).amax(2).repeat_interleave(128, dim=1)[:, :k].clamp(min=2.0 ** -97)
    want, size = xd @ w.t(), xd.abs() @ w.abs().t()
    got = linear4(x * 1.0, W)
    unit = (top * 2.0 ** -30) @ w.abs().t()
    half = torch.finfo(t).eps / 2
    tol = unit + 2.0 ** -24 * (k / 8 + 32) * size + half * 1.01 * want.abs() + torch.finfo(t).tiny
    fine = want.abs() <= torch.finfo(t).max
    assert bool(((got.double() - want).abs() <= tol)[fine].all())
    assert (got.double().abs()[~fine] >= torch.finfo(t).max).all()
    y = x.clone()
    y[m - 1, 17] = float("inf")
    out, q = linear4(y, W)[m - 1], w[:, 17]
    assert out[q == 0].isnan().all() and (out[q > 0] == float("inf")).all() and (out[q < 0] == -float("inf")).all()
    y[m - 1, 400] = float("nan")
    out = linear4(y, W)
    assert out[m - 1].isnan().all() and torch.equal(out[: m - 1], got[: m - 1])


def test_same_bits_again_and_in_a_graph(dev):
    """Fixed sums: the same call twice gives the same bits, also replayed, also beside a call on other data on another stream."""
    from boundflow_b200.weights4 import interval_linear4, linear4, rows_times_weight4

    W, w, g = make(700, 900, 128, dev, 7)
    x, a = torch.randn(3, 900, generator=g).to(dev), torch.randn(9, 700, generator=g).to(dev)

    def all_three():
        return (linear4(x, W), *interval_linear4(x - 1, x + 1, W), rows_times_weight4(a, W))

    first = all_three()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(3):
            linear4(x * 2, W)
    assert all(torch.equal(p, q) for p, q in zip(first, all_three()))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = all_three()
    x.mul_(0.5)
    a.add_(1.0)
    graph.replay()
    assert all(torch.equal(p, q) for p, q in zip(out, all_three()))
