"""What is NaN stays NaN through a ReLU (max(NaN, 0) of the C library is 0): the bounds of weights that hold one, and of a product whose wait on the device ran out, are no bounds."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from boundflow_b200.csrc import build

    build.build()
    return torch.device("cuda", 0)


def module(params, skip=False):
    from boundflow_b200.ir import BFTaskModule, BoundTask, TaskKind, TaskOp

    ops = [TaskOp("linear", "l1", ["x", "w1"], ["h1"]), TaskOp("relu", "a1", ["h1"], ["r1"]), TaskOp("linear", "l2", ["r1", "w2"], ["h2"]), TaskOp("relu", "a2", ["h2"], ["r2"]),
           TaskOp("linear", "l3", ["r2", "w3"], ["out"])]
    task = BoundTask(task_id="t", kind=TaskKind.INTERVAL_IBP, ops=ops, input_values=["x"], output_values=["out"])
    return BFTaskModule([task], "t", {"params": params})


def sizes(dev):
    g = torch.Generator("cpu").manual_seed(0)
    ws = [torch.randn(64, 40, generator=g), torch.randn(48, 64, generator=g), torch.randn(5, 48, generator=g)]
    return [w.to(dev) for w in ws]


def box(dev, B=3):
    from boundflow_b200.ir import InputSpec

    x = torch.rand(B, 40, generator=torch.Generator("cpu").manual_seed(1)).to(dev)
    return InputSpec.box(value_name="x", lower=x - 0.1, upper=x + 0.1)


def test_relu_of_bounds(dev):
    from boundflow_b200.executor import CudaIntervalDomain
    from boundflow_b200.ir import IntervalState

    t = torch.tensor([[float("nan"), -1.0, 2.0, float("inf"), -float("inf"), -0.0]], device=dev)
    got = CudaIntervalDomain().relu_transformer(IntervalState(lower=t, upper=t + 1))
    assert torch.equal(got.lower[0].isnan(), t[0].isnan()) and got.upper[0, 0].isnan()
    assert torch.equal(got.lower[0, 1:], t[0, 1:].clamp(min=0)) and torch.equal(got.upper[0, 1:], (t + 1)[0, 1:].clamp(min=0))


@pytest.mark.parametrize("shape", ["linear", "batched", "conv"])
def test_clamped_inputs(dev, shape):
    from boundflow_b200.executor import CudaIntervalDomain
    from boundflow_b200.ir import IntervalState

    g = torch.Generator("cpu").manual_seed(2)
    if shape == "conv":
        x, w, op = torch.randn(2, 3, 8, 8, generator=g), torch.randn(4, 3, 3, 3, generator=g), "conv2d"
    else:
        x, w, op = torch.randn(2, 36, generator=g), torch.randn(*((5, 36) if shape == "linear" else (2, 5, 36)), generator=g), "linear"
    x, w = x.to(dev), w.to(dev)
    clean = CudaIntervalDomain().affine_transformer(IntervalState(lower=x, upper=x + 1), w, None, op=op, relu_in=True)
    y = x.clone()
    y.view(2, -1)[1] = float("nan")
    got = CudaIntervalDomain().affine_transformer(IntervalState(lower=y, upper=y + 1), w, None, op=op, relu_in=True)
    for a, b in ((got.lower, clean.lower), (got.upper, clean.upper)):
        assert a[1].isnan().all() and torch.equal(a[0], b[0])


@pytest.mark.parametrize("where", ["w1", "w2"])
def test_a_4_bit_weight_that_holds_a_nan(dev, where):
    from boundflow_b200.crown import run_crown_ibp_mlp
    from boundflow_b200.executor import CudaTaskExecutor
    from boundflow_b200.weights4 import quantise_weight4

    ws = dict(zip(["w1", "w2", "w3"], sizes(dev)))
    ws[where][:, 7] = float("nan")
    params = {k: quantise_weight4(w, 32) for k, w in ws.items()}
    for run in (lambda m: CudaTaskExecutor().run_ibp(m, box(dev)), lambda m: run_crown_ibp_mlp(m, box(dev))):
        got = run(module(params))
        assert not got.lower.isfinite().any() and not got.upper.isfinite().any()


def test_an_expired_wait_gives_no_bounds(dev, monkeypatch):
    """The products' sign of a wait that ran out is NaN in the results concerned."""
    from boundflow_b200 import weights4
    from boundflow_b200.crown import run_crown_ibp_mlp
    from boundflow_b200.executor import CudaTaskExecutor

    params = {k: weights4.quantise_weight4(w, 32) for k, w in zip(["w1", "w2", "w3"], sizes(dev))}
    good = CudaTaskExecutor().run_ibp(module(params), box(dev))
    interval = weights4._interval

    def expired(*args):
        lower, upper = interval(*args)
        if lower.shape[1] == 64:
            lower[1], upper[1] = float("nan"), float("nan")
        return lower, upper

    monkeypatch.setattr(weights4, "_interval", expired)
    for run in (lambda m: CudaTaskExecutor().run_ibp(m, box(dev)), lambda m: run_crown_ibp_mlp(m, box(dev))):
        got = run(module(params))
        assert not got.lower[1].isfinite().any() and not got.upper[1].isfinite().any()
        assert got.lower[[0, 2]].isfinite().all() and got.upper[[0, 2]].isfinite().all()
    assert torch.equal(CudaTaskExecutor().run_ibp(module(params), box(dev)).lower[[0, 2]], good.lower[[0, 2]])
