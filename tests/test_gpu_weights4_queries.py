"""Whole queries on networks with 4-bit layers beyond the sizes of single sweeps: the query runtime, the entry points that refuse them, and batches whose rows take the kernels
for many.  Bounds are held against the same function on the dense weights that the codes stand for (tests/helpers.py: 1e-4 + 1e-5 of the bound)."""
from types import SimpleNamespace

import pytest
import torch

from tests.helpers import assert_close
from tests.test_gpu_weights4_networks import boxes, dev, network  # noqa: F401

pytestmark = pytest.mark.gpu


def test_entry_points_that_read_dense_weights_refuse(dev):
    from boundflow_b200.crown import bound_split_domains, ibp_trace, run_crown_intermediate_mlp

    m4, _ = network(dev)
    spec, _ = boxes(dev, 2, 45)
    C = torch.eye(10, device=dev)
    for call in (lambda: bound_split_domains(m4, spec, linear_spec_C=C, relu_split_state=None), lambda: run_crown_intermediate_mlp(m4, spec),
                 lambda: run_crown_intermediate_mlp(m4, spec, chunk_rows=0), lambda: ibp_trace(m4, spec)):
        with pytest.raises(NotImplementedError, match="held in 4 bits"):
            call()


@pytest.mark.parametrize("method", ["alpha-CROWN", "alpha-beta-CROWN"])
def test_query_runtime(dev, method):
    """Nodes of one batch, one of them with an empty split; the bounds are those of plain CROWN on the dense weights or better, and hold for points of the boxes."""
    from boundflow_b200.crown import forward_ibp_trace_mlp, run_crown_ibp_mlp
    from boundflow_b200.ir import InputSpec
    from boundflow_b200.query_runtime import CudaQueryRuntime

    m4, m32 = network(dev, seed=4)
    g = torch.Generator("cpu").manual_seed(5)
    x = torch.rand(3, 45, generator=g).to(dev)
    specs = [InputSpec.box(value_name="x", lower=x[i : i + 1] - 0.02, upper=x[i : i + 1] + 0.02) for i in range(3)]
    _, pre = forward_ibp_trace_mlp(m32, specs[0])
    names = list(pre)
    options = {"alpha_steps": 4, "alpha_lr": 0.1, "alpha_init": 0.5, "beta_init": 0.0}

    def request(i, split):
        payload = SimpleNamespace(input_spec=specs[i], linear_spec_c=None, split_by_relu_input=split, warm_alpha_by_relu_input={}, warm_beta_by_relu_input={})
        return SimpleNamespace(query=SimpleNamespace(query_id=f"q{i}", bound_method=method, execution_options=options), payload=payload)

    def free():
        return {n: torch.zeros(pre[n].lower[0].numel(), dtype=torch.int8, device=dev) for n in names}

    impossible = free()
    lower = pre[names[0]].lower[0]
    positive = int(torch.nonzero(forward_ibp_trace_mlp(m32, specs[1])[1][names[0]].lower[0].flatten() > 0)[0])
    impossible[names[0]][positive] = -1
    assert lower.numel() == 70
    requests = [request(0, free()), request(1, impossible), request(2, free())]
    got4 = dict(CudaQueryRuntime().execute(m4, requests))
    assert [got4[f"q{i}"].status for i in range(3)] == ["ok", "infeasible" if method == "alpha-beta-CROWN" else "rejected", "ok"]
    for i in (0, 2):
        plain = run_crown_ibp_mlp(m32, specs[i], relu_alpha={n: torch.full_like(pre[n].lower, 0.5) for n in names})
        mean = lambda t: float(t.mean())  # noqa: E731
        assert mean(got4[f"q{i}"].lower) >= mean(plain.lower) - 1e-4
        at = run_crown_ibp_mlp(m32, specs[i], relu_alpha={n: a.reshape(1, -1) for n, a in got4[f"q{i}"].alpha_by_relu_input.items()})
        assert_close(got4[f"q{i}"].lower, at.lower, "lower at the returned alpha")


@pytest.mark.parametrize("B", [300, 1200])
def test_batches_that_take_the_kernels_for_many_rows(dev, B):
    """Nine specs of each box: 2700 and 10800 coefficient rows a side, interval products of 300 and 1200.  Which kernels run is asked of the library."""
    from boundflow_b200 import _lib
    from boundflow_b200.crown import run_alpha_beta_crown_mlp, run_crown_ibp_mlp
    from boundflow_b200.executor import CudaTaskExecutor

    m4, m32 = network(dev, widths=(784, 1024, 512, 10), group=64, seed=6)
    spec, _ = boxes(dev, B, 784)
    C = torch.eye(10, device=dev)[:9] - torch.eye(10, device=dev)[1:]
    lib = _lib.load()
    layers = [(784, 1024), (1024, 512), (512, 10)]
    intervals = sum(lib.bf_w4_many_pays(B, i, o, 64, 0, 0, 1) for i, o in layers)
    rows = sum(lib.bf_w4_many_pays(9 * B, i, o, 64, 0, 1, 0) for i, o in layers)
    assert rows > 0 and (intervals > 0) == (B == 1200)
    before = lib.bf_tc_launch_count()
    a = CudaTaskExecutor().run_ibp(m4, spec)
    assert lib.bf_tc_launch_count() - before == 2 * intervals  # (two products a pair)
    b = CudaTaskExecutor().run_ibp(m32, spec)
    assert_close(a.lower, b.lower, "interval lower")
    assert_close(a.upper, b.upper, "interval upper")
    before = lib.bf_tc_launch_count()
    a = run_crown_ibp_mlp(m4, spec, linear_spec_C=C)
    assert lib.bf_tc_launch_count() - before >= 2 * intervals + rows
    b = run_crown_ibp_mlp(m32, spec, linear_spec_C=C)
    assert_close(a.lower, b.lower, "lower")
    assert_close(a.upper, b.upper, "upper")
    got, alpha, _, _ = run_alpha_beta_crown_mlp(m4, spec, linear_spec_C=C, steps=2, lr=0.05, per_batch_params=True)
    at = run_crown_ibp_mlp(m32, spec, linear_spec_C=C, relu_alpha=alpha.alpha_by_relu_input)
    assert_close(got.lower, at.lower, "lower at the returned alpha")
