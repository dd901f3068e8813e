"""Networks whose Linear layers are held in 4 bits, bounded by the functions that bound dense ones, and trained around: every bound is held against the same
function on the dense weights that the codes stand for (tests/helpers.py: 1e-4 + 1e-5 of the bound)."""
import pytest
import torch

from tests.helpers import assert_close

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from boundflow_b200.csrc import build

    build.build()
    return torch.device("cuda", 0)


def network(dev, widths=(45, 70, 66, 10), group=32, skip=False, seed=0):
    """(module with 4-bit weights, the same with dense ones); `skip`: the second hidden value is added to the third."""
    from boundflow_b200.ir import BFTaskModule, BoundTask, TaskKind, TaskOp
    from boundflow_b200.weights4 import quantise_weight4

    g = torch.Generator("cpu").manual_seed(seed)
    ops, packed, dense, cur = [], {}, {}, "x"
    for i, (a, b) in enumerate(zip(widths, widths[1:])):
        last = i + 2 == len(widths)
        w4 = quantise_weight4((torch.randn(b, a, generator=g) * (2 / a) ** 0.5).to(dev), group)
        bias = torch.randn(b, generator=g).to(dev) * 0.1
        packed[f"W{i}"], dense[f"W{i}"] = w4, w4.dense()
        packed[f"b{i}"] = dense[f"b{i}"] = bias
        ops.append(TaskOp("linear", f"l{i}", [cur, f"W{i}", f"b{i}"], [f"h{i}"]))
        cur = f"h{i}"
        if skip and i == 1:
            ops.append(TaskOp("add", "skip", [cur, "r0"], ["s1"]))
            cur = "s1"
        if not last:
            ops.append(TaskOp("relu", f"relu{i}", [cur], [f"r{i}"]))
            cur = f"r{i}"
    task = BoundTask(task_id="t", kind=TaskKind.INTERVAL_IBP, ops=ops, input_values=["x"], output_values=[cur])
    return BFTaskModule([task], "t", {"params": packed}), BFTaskModule([task], "t", {"params": dense})


def boxes(dev, B, n, seed=1):
    from boundflow_b200.ir import InputSpec

    g = torch.Generator("cpu").manual_seed(seed)
    x = torch.rand(B, n, generator=g).to(dev)
    return InputSpec.box(value_name="x", lower=x - 0.03, upper=x + 0.03), x


@pytest.mark.parametrize("skip", [False, True])
@pytest.mark.parametrize("B", [1, 7, 40])
def test_ibp_and_crown(dev, skip, B):
    from boundflow_b200.crown import run_crown_ibp_mlp
    from boundflow_b200.executor import CudaTaskExecutor

    m4, m32 = network(dev, widths=(45, 70, 70, 10) if skip else (45, 70, 66, 10), skip=skip)
    spec, x = boxes(dev, B, 45)
    C = torch.eye(10, device=dev)[:9] - torch.eye(10, device=dev)[1:]
    for run in (lambda m: CudaTaskExecutor().run_ibp(m, spec), lambda m: run_crown_ibp_mlp(m, spec), lambda m: run_crown_ibp_mlp(m, spec, linear_spec_C=C)):
        a, b = run(m4), run(m32)
        assert_close(a.lower, b.lower, "lower")
        assert_close(a.upper, b.upper, "upper")
        assert bool((a.lower <= a.upper).all())


@pytest.mark.parametrize("p", ["l2", "l1"])
def test_balls(dev, p):
    from boundflow_b200.crown import run_crown_ibp_mlp
    from boundflow_b200.executor import CudaTaskExecutor
    from boundflow_b200.ir import InputSpec

    m4, m32 = network(dev)
    _, x = boxes(dev, 5, 45)
    spec = getattr(InputSpec, p)(value_name="x", center=x, eps=0.1)
    for run in (lambda m: CudaTaskExecutor().run_ibp(m, spec), lambda m: run_crown_ibp_mlp(m, spec)):
        a, b = run(m4), run(m32)
        assert_close(a.lower, b.lower, p)
        assert_close(a.upper, b.upper, p)


@pytest.mark.parametrize("skip", [False, True])
@pytest.mark.parametrize("per_batch", [True, False])
def test_alpha_beta(dev, skip, per_batch):
    """Two steps of lr 0.05: Adam divides by the root of a gradient's own square, so that a gradient near zero may turn a rounding into a step; what the loop
    returns is compared through the bounds at its own alpha, on the dense weights."""
    from boundflow_b200.crown import run_alpha_beta_crown_mlp, run_crown_ibp_mlp

    m4, m32 = network(dev, widths=(45, 70, 70, 10) if skip else (45, 70, 66, 10), skip=skip, seed=2)
    spec, _ = boxes(dev, 6, 45)
    got, alpha, _, _ = run_alpha_beta_crown_mlp(m4, spec, steps=2, lr=0.05, per_batch_params=per_batch)
    plain = run_crown_ibp_mlp(m4, spec)
    at = run_crown_ibp_mlp(m32, spec, relu_alpha=alpha.alpha_by_relu_input)
    assert_close(got.lower, at.lower, "lower at the returned alpha")
    assert bool((got.lower <= plain.upper + 1e-4).all())


def test_splits_certificate_and_query_runtime_refusals(dev):
    from boundflow_b200.crown import first_layer_certificate, forward_ibp_trace_mlp, run_crown_ibp_mlp
    from boundflow_b200.executor import CudaIntervalDomain
    from boundflow_b200.ir import IntervalState

    m4, m32 = network(dev)
    spec, _ = boxes(dev, 4, 45)
    _, pre = forward_ibp_trace_mlp(m32, spec)
    name = list(pre)[0]
    split = ((pre[name].lower < 0) & (pre[name].upper > 0)).to(torch.int8)
    split[:, 20:] = 0
    a, b = (run_crown_ibp_mlp(m, spec, relu_split_state={name: split}) for m in (m4, m32))
    assert_close(a.lower, b.lower, "split lower")
    for p, q in zip(first_layer_certificate(m4, spec, {name: split}), first_layer_certificate(m32, spec, {name: split})):
        assert p.shape == q.shape
    W = m4.bindings["params"]["W0"]
    state = IntervalState(lower=torch.zeros(2, 45, 3, 3, device=dev), upper=torch.ones(2, 45, 3, 3, device=dev))
    with pytest.raises(NotImplementedError):
        CudaIntervalDomain().affine_transformer(state, W, None, op="conv2d")
    box = IntervalState(lower=torch.zeros(2, 3, 45, device=dev), upper=torch.ones(2, 3, 45, device=dev))
    got = CudaIntervalDomain().affine_transformer(box, W, m4.bindings["params"]["b0"].cpu(), op="linear", relu_in=True)
    want = CudaIntervalDomain().affine_transformer(box, W.dense(), m4.bindings["params"]["b0"], op="linear", relu_in=True)
    assert got.lower.shape == (2, 3, 70)
    assert_close(got.lower, want.lower, "domain lower")
    assert_close(got.upper, want.upper, "domain upper")


@pytest.mark.parametrize("bits", [32, 8])
def test_train_around_frozen_layers_then_bound(dev, bits):
    """All operators together, as they are used: a layer is quantised and frozen, gradients of a loss on points and on interval bounds flow through it to the
    layers around it, AdamW moves those, and the bounds of the new network are those of its dense twin.  The gradients are the dense twin's."""
    from boundflow_b200.crown import run_crown_ibp_mlp
    from boundflow_b200.executor import CudaTaskExecutor
    from boundflow_b200.ir import BFTaskModule, BoundTask, TaskKind, TaskOp
    from boundflow_b200.optim import AdamW
    from boundflow_b200.weights4 import interval_linear4, linear4, quantise_weight4

    g = torch.Generator("cpu").manual_seed(11)
    rand = lambda *s: (torch.randn(s, generator=g) * (1 / s[-1]) ** 0.5).to(dev)  # noqa: E731
    frozen = quantise_weight4(rand(64, 50), 32)
    dense = frozen.dense()
    params = [rand(50, 20).requires_grad_(), rand(50).requires_grad_(), rand(64).requires_grad_(), rand(10, 64).requires_grad_(), rand(10).requires_grad_()]
    opt = AdamW(params, lr=1e-2, state_bits=bits)
    x = torch.rand(16, 20, generator=g).to(dev)
    y = torch.randint(0, 10, (16,), generator=g).to(dev)

    def loss(product, bounds):
        w1, b1, b2, w3, b3 = params
        h = torch.relu(x @ w1.t() + b1)
        out = torch.relu(product(h, b2)) @ w3.t() + b3
        r = (0.01 * w1.abs().sum(1)).expand_as(h)
        lo, up = bounds(torch.relu(h - r), torch.relu(h + r), b2)
        return torch.nn.functional.cross_entropy(out, y) + 0.1 * (torch.relu(up) - torch.relu(lo)).mean()

    def dense_bounds(lo, up, b):
        plus, minus = dense.clamp(min=0), dense.clamp(max=0)
        return lo @ plus.t() + up @ minus.t() + b, up @ plus.t() + lo @ minus.t() + b

    for _ in range(5):
        opt.zero_grad()
        loss(lambda h, b: linear4(h, frozen, b), lambda lo, up, b: interval_linear4(lo, up, frozen, b)).backward()
        want = torch.autograd.grad(loss(lambda h, b: h @ dense.t() + b, dense_bounds), params)
        for p, w in zip(params, want):
            assert_close(p.grad, w, "gradient", atol=1e-5 * float(w.abs().max()), rtol=1e-4)
        opt.step()
    assert opt.steps == 5
    ops = [TaskOp("linear", "l1", ["x", "w1", "b1"], ["h1"]), TaskOp("relu", "a1", ["h1"], ["r1"]), TaskOp("linear", "l2", ["r1", "w2", "b2"], ["h2"]),
           TaskOp("relu", "a2", ["h2"], ["r2"]), TaskOp("linear", "l3", ["r2", "w3", "b3"], ["out"])]
    task = BoundTask(task_id="t", kind=TaskKind.INTERVAL_IBP, ops=ops, input_values=["x"], output_values=["out"])
    spec, _ = boxes(dev, 16, 20)
    sides = []
    for w2 in (frozen, dense):
        module = BFTaskModule([task], "t", {"params": dict(zip(["w1", "b1", "b2", "w3", "b3"], params)) | {"w2": w2}})
        sides.append((CudaTaskExecutor().run_ibp(module, spec), run_crown_ibp_mlp(module, spec)))
    for a, b in zip(*sides):
        assert_close(a.lower, b.lower, "lower")
        assert_close(a.upper, b.upper, "upper")


def test_gradients_of_several_rows_of_one_leaf_in_a_graph(dev):
    """A forward and backward pass captured into a graph, with tensors made for it, and replayed on new inputs."""
    from boundflow_b200.weights4 import linear4, quantise_weight4

    g = torch.Generator("cpu").manual_seed(12)
    W = quantise_weight4(torch.randn(96, 160, generator=g).to(dev), 32)
    x, dy = torch.randn(4, 160, generator=g).to(dev), torch.randn(4, 96, generator=g).to(dev)

    def both():
        leaf = x.detach().requires_grad_()
        return torch.autograd.grad(linear4(leaf, W), leaf, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    dy.mul_(-2.0)
    graph.replay()
    assert torch.equal(out, both())
