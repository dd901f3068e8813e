"""Products of many rows with 4-bit weights against the same in 64 bits.

Tolerances.  x W^T: products are exact, sums of 32 bits: 2^-24 * (terms / 8 + 32) of the sum of magnitudes, as for few rows.  a W: the weight scale * (code - 8) is rounded to
32 bits (2^-24) and held in three bfloat16 parts for fp32 rows (what is left out is below 2^-26), in two for 16-bit rows (2^-17, and for halves, which are two parts themselves, 2^-18
for the product of second parts): 2^-16 of the sum of magnitudes covers both.  Beside that half a step of the output's type.
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


@pytest.fixture(autouse=True)
def many(monkeypatch):
    """These kernels at every size, not only where they are the faster ones."""
    from boundflow_b200 import weights4

    monkeypatch.setattr(weights4, "_many_pays", lambda *a: True)


def make(n, k, group, dev, seed=0):
    from boundflow_b200.weights4 import Weight4

    g = torch.Generator("cpu").manual_seed(seed + 1000 * n + k + group)
    padded = -(-k // group) * group
    codes = torch.randint(0, 256, (n, padded // 2), generator=g, dtype=torch.uint8)
    scales = (torch.rand((padded // group, n), generator=g) + 0.25) * torch.where(torch.rand((padded // group, n), generator=g) < 0.2, -1.0, 1.0)
    q = torch.stack((codes & 15, codes >> 4), dim=2).reshape(n, padded).double() - 8
    w = (q * scales.double().t().repeat_interleave(group, dim=1))[:, :k]
    return Weight4(codes.to(dev), scales.to(dev), k), w.to(dev), g


def check(got, want, size, terms, dtype, extra=0.0):
    eps = torch.finfo(dtype).eps if dtype != torch.float32 else 0.0
    tol = (2.0 ** -24 * (terms / 8 + 32) + extra) * size + eps / 2 * want.abs() * 1.01 + (torch.finfo(dtype).tiny if eps else 0.0)
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"worst {float((err / tol.clamp(min=1e-300)).max()):.2f} of the tolerance"


SHAPES = [(1, 1, 32), (3, 31, 32), (130, 33, 32), (129, 500, 128), (512, 784, 32), (257, 1000, 256), (300, 1111, 64), (48, 3000, 32), (2050, 640, 64), (5, 9000, 128), (9, 200, 512),
          (4096, 320, 128)]
ROWS = [64, 65, 128, 200, 300, 1025]


@pytest.mark.parametrize("n,k,group", SHAPES)
@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
def test_linear(dev, n, k, group, kind):
    from boundflow_b200.weights4 import linear4

    W, w, g = make(n, k, group, dev)
    b = torch.randn(n, generator=g).to(dev)
    for m in ROWS:
        x = torch.randn(m, k, generator=g).to(TYPES[kind]).to(dev)
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
    from boundflow_b200.weights4 import rows_times_weight4

    W, w, g = make(n, k, group, dev, 2)
    for m in ROWS:
        a = torch.randn(m, n, generator=g).to(TYPES[kind]).to(dev)
        got = rows_times_weight4(a, W)
        assert got.shape == (m, k) and got.dtype == a.dtype
        check(got, a.double() @ w, a.double().abs() @ w.abs(), n, a.dtype, 0.0 if kind == "fp32" else 2.0 ** -16)


@pytest.mark.parametrize("m,n,k,group", [(70, 130, 300, 64), (257, 65, 129, 128), (129, 300, 100, 32)])
def test_gradients(dev, m, n, k, group):
    from boundflow_b200.weights4 import interval_linear4, linear4

    W, w, g = make(n, k, group, dev, 3)
    x = torch.randn(m, k, generator=g).to(dev).requires_grad_()
    b = torch.randn(n, generator=g).to(dev).requires_grad_()
    dy, dz = (torch.randn(m, n, generator=g).to(dev) for _ in range(2))
    gx, gb = torch.autograd.grad(linear4(x, W, b), (x, b), dy)
    check(gx, dy.double() @ w, dy.double().abs() @ w.abs(), n, torch.float32)
    check(gb, dy.double().sum(0), dy.double().abs().sum(0), m, torch.float32)
    lo, up = (x.detach() - 0.1).requires_grad_(), (x.detach() + 0.1).requires_grad_()
    gl, gu = torch.autograd.grad(interval_linear4(lo, up, W, b.detach()), (lo, up), (dy, dz))
    plus, minus = w.clamp(min=0), w.clamp(max=0)
    size = (dy.double().abs() + dz.double().abs()) @ w.abs()
    check(gl, dy.double() @ plus + dz.double() @ minus, size, n, torch.float32)
    check(gu, dz.double() @ plus + dy.double() @ minus, size, n, torch.float32)


@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
def test_infinities_and_nan(dev, kind):
    """What is not finite reaches the outputs that a weight other than zero ties to it, as infinity, or as NaN where a weight is zero or signs meet."""
    from boundflow_b200.weights4 import linear4, rows_times_weight4

    W, w, g = make(70, 200, 64, dev, 4)
    for call, width, mat in ((linear4, 200, w.t()), (rows_times_weight4, 70, w)):
        x = torch.randn(80, width, generator=g).to(TYPES[kind])
        x[3, 5], x[7, 1], x[7, 60], x[9, 2] = float("inf"), float("-inf"), float("inf"), float("nan")
        x = x.to(dev)
        got, want = call(x, W).double(), x.double() @ mat
        odd = torch.zeros(80, dtype=torch.bool)
        odd[[3, 7, 9]] = True
        assert bool(torch.isfinite(got[~odd]).all())
        assert torch.equal(torch.isnan(got[odd]), torch.isnan(want[odd]))
        inf = torch.isinf(want[odd])
        assert torch.equal(got[odd][inf], want[odd][inf])


def test_large_and_small_numbers(dev):
    """Near the type's ends: parts that would round to infinity, subnormal numbers."""
    from boundflow_b200.weights4 import Weight4, linear4, rows_times_weight4

    codes = torch.full((64, 32), 0x99, dtype=torch.uint8, device=dev)  # ones
    W = Weight4(codes, torch.ones(1, 64, device=dev), 64)
    x = torch.zeros(64, 64, device=dev)
    x[0, 3], x[1, 4], x[2, 63] = 3.4e38, -3.4028e38, 2.0 ** -126
    for call in (linear4, rows_times_weight4):
        got = call(x, W)
        assert torch.equal(got, x.sum(1, keepdim=True).expand(64, 64))


def test_strided_empty_and_flat_inputs_and_streams(dev):
    from boundflow_b200.weights4 import linear4

    W, w, g = make(200, 300, 64, dev, 5)
    x = torch.randn(4, 300, 33, generator=g).to(dev).transpose(1, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = linear4(x, W)
    torch.cuda.current_stream().wait_stream(side)
    xd = x.double()
    check(y, xd @ w.t(), xd.abs() @ w.abs().t(), 300, torch.float32)
    shifted = torch.randn(100 * 300 + 1, generator=g).to(dev)[1:].view(100, 300)  # off its boundary
    check(linear4(shifted, W), shifted.double() @ w.t(), shifted.double().abs() @ w.abs().t(), 300, torch.float32)


def test_results_do_not_depend_on_the_other_rows(dev):
    """A row's result is the same bits in calls of other sizes that take the same kernel."""
    from boundflow_b200.weights4 import linear4, rows_times_weight4

    W, _, g = make(500, 700, 128, dev, 6)
    x, a = torch.randn(400, 700, generator=g).to(dev), torch.randn(400, 500, generator=g).to(dev)
    y, z = linear4(x, W), rows_times_weight4(a, W)
    for m in (64, 129, 300):
        assert torch.equal(linear4(x[:m], W), y[:m]) and torch.equal(rows_times_weight4(a[:m], W), z[:m])
    assert torch.equal(linear4(x, W), y)


def test_captured_calls_share_nothing(dev):
    """Two captured products, replayed at the same time on two streams."""
    from boundflow_b200.weights4 import linear4, rows_times_weight4

    W, w, g = make(300, 400, 128, dev, 7)
    x, a = torch.randn(96, 400, generator=g).to(dev), torch.randn(96, 300, generator=g).to(dev)
    graphs, outs, streams = [], [], []
    for call, t in ((linear4, x), (rows_times_weight4, a)):
        call(t, W)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(t, W))
        graphs.append(graph)
        streams.append(torch.cuda.Stream())
    x.copy_(torch.randn(96, 400, generator=g))
    a.copy_(torch.randn(96, 300, generator=g))
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    check(outs[0], x.double() @ w.t(), x.double().abs() @ w.abs().t(), 400, torch.float32)
    check(outs[1], a.double() @ w, a.double().abs() @ w.abs(), 300, torch.float32)


def test_refusals(dev):
    from boundflow_b200 import _lib

    lib = _lib.load()
    t = torch.zeros(4096, device=dev)
    p = t.data_ptr()
    assert lib.bf_w4_linear_many(p, 0, p, p, None, 0, p, 64, 32, 4, 32, None, None) == _lib.BF_E_INVALID      # no workspace
    assert lib.bf_w4_linear_many(p, 0, p, p, None, 0, p, 64, 32, 4, 32, p + 64, None) == _lib.BF_E_INVALID    # its boundary
    assert lib.bf_w4_rows_many(p, 0, p, p, p, 0, 32, 4, 32, p, None) == _lib.BF_E_INVALID                     # no rows
    assert lib.bf_w4_interval_many(p, p, 2, 0, p, p, None, p, p, 64, 32, 4, 32, p, None) == _lib.BF_E_INVALID  # unknown mode
    assert lib.bf_w4_interval_grad_many(p, None, p, p, p, p, 64, 32, 4, 32, p, None) == _lib.BF_E_INVALID
    assert lib.bf_w4_workspace_bytes(64, 32, 9) == 0 and lib.bf_w4_workspace_bytes(0, 32, 0) == 0
    assert 0 < lib.bf_w4_workspace_bytes(2 ** 31 - 1, 2 ** 14, 0) < 2 ** 29
    assert 256 * 2 ** 20 * 6 < lib.bf_w4_workspace_bytes(2 ** 31 - 1, 2 ** 20, 0) < 257 * 2 ** 20 * 6  # (256 rows at least)
    assert [lib.bf_w4_many_pays(m, 8192, 8192, 128, 1, 0, 0) for m in (0, 1, 16, 4096)] == [0, 0, 0, 1]


def test_both_kinds_of_kernels_agree_and_launch(dev, monkeypatch):
    """The choice between them is made for the sizes alone; the tensor cores' tiles count as such."""
    from boundflow_b200 import _lib, weights4

    W, w, g = make(1024, 2048, 128, dev, 8)
    x = torch.randn(2000, 2048, generator=g).to(dev)
    monkeypatch.undo()
    before = _lib.load().bf_tc_launch_count()
    y = weights4.linear4(x, W)
    assert _lib.load().bf_tc_launch_count() == before + 1
    monkeypatch.setattr(weights4, "_many_pays", lambda *a: False)
    size = x.double().abs() @ w.abs().t()
    check(y, x.double() @ w.t(), size, 2048, torch.float32)
    check(weights4.linear4(x, W), x.double() @ w.t(), size, 2048, torch.float32)


def test_column_sums_of_many_rows(dev):
    from boundflow_b200 import weights4

    g = torch.Generator("cpu").manual_seed(9)
    for m, n in ((65, 1), (64, 40), (127, 33), (128, 500), (1000, 129)):
        a = torch.randn(m, n, generator=g).to(dev)
        check(weights4._column_sums(a, torch.float32), a.double().sum(0), a.double().abs().sum(0), m, torch.float32)


def test_more_rows_than_the_workspace_holds(dev):
    """Slab by slab through one workspace: rows at the ends of the first and second slab, an infinity in the second."""
    from boundflow_b200 import _lib, weights4

    W, w, g = make(40, 4096, 128, dev, 10)
    m = 12000  # 4096 columns in three parts: 24 KB a row, 10752 rows a slab
    assert _lib.load().bf_w4_workspace_bytes(m, 4096, 0) < m * 4096 * 6
    x = torch.randn(m, 4096, generator=g).to(dev)
    picked = torch.tensor([0, 1, 10495, 10751, 10752, 10753, 11000, m - 1], device=dev)
    xd = x[picked].double()
    check(weights4.linear4(x, W)[picked], xd @ w.t(), xd.abs() @ w.abs().t(), 4096, torch.float32)
    lower, upper = weights4.interval_linear4(x - 0.5, x + 0.5, W)
    l, u = (x - 0.5)[picked].double(), (x + 0.5)[picked].double()
    plus, minus = w.clamp(min=0), w.clamp(max=0)
    check(lower[picked], l @ plus.t() + u @ minus.t(), (l.abs() + u.abs()) @ w.abs().t(), 4096, torch.float32)
    check(upper[picked], u @ plus.t() + l @ minus.t(), (l.abs() + u.abs()) @ w.abs().t(), 4096, torch.float32)
    V, v, g = make(4096, 40, 32, dev, 11)
    x[11000, 17] = float("inf")
    z = weights4.rows_times_weight4(x, V)[picked]
    want = x[picked].double() @ v
    keep = torch.tensor([True] * 6 + [False, True], device=dev)
    check(z[keep], want[keep], xd[keep].abs() @ v.abs(), 4096, torch.float32)
    assert torch.equal(torch.isnan(z[~keep]), torch.isnan(want[~keep])) and torch.equal(z[~keep].double()[torch.isinf(want[~keep])], want[~keep][torch.isinf(want[~keep])])
