"""Uses of 4-bit weights that are refused, by name and not by a wrong or missing result: no GPU is needed for any of them."""
import pytest
import torch
from torch.autograd import forward_ad


def weight(n=4, k=40, group=32):
    from boundflow_b200.weights4 import Weight4

    padded = -(-k // group) * group
    return Weight4(torch.zeros(n, padded // 2, dtype=torch.uint8), torch.zeros(padded // group, n), k)


def test_forward_mode_tangents_are_refused():
    from boundflow_b200.weights4 import interval_linear4, linear4, rows_times_weight4

    w, x, a, b = weight(), torch.zeros(2, 40), torch.zeros(2, 4), torch.zeros(4)
    with forward_ad.dual_level():
        dx, da, db = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, a, b))
        for call in (lambda: linear4(dx, w), lambda: linear4(x, w, db), lambda: interval_linear4(dx, x, w), lambda: interval_linear4(x, dx, w), lambda: interval_linear4(x, x, w, db),
                     lambda: rows_times_weight4(da, w)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def chain():
    from boundflow_b200.ir import BFTaskModule, BoundTask, TaskKind, TaskOp

    ops = [TaskOp("linear", "l1", ["x", "W"], ["y"])]
    task = BoundTask(task_id="t", kind=TaskKind.INTERVAL_IBP, ops=ops, input_values=["x"], output_values=["y"])
    return BFTaskModule([task], "t", {"params": {"W": weight()}})


def test_chains_say_what_takes_a_4_bit_weight():
    from boundflow_b200.csrc import build
    from boundflow_b200.network import CudaChain

    build.build()
    with pytest.raises(NotImplementedError, match="bound_split_domains.*run_crown_intermediate_mlp.*run_alpha_beta_crown_mlp"):
        CudaChain(chain(), (40,), torch.device("cuda", 0))


def test_fused_regions_refuse_a_4_bit_weight():
    from types import SimpleNamespace

    from boundflow_b200.csrc import build
    from boundflow_b200.fused import CudaFusedCrownExecutor

    build.build()
    rows, line = torch.zeros(1, 2, 4), torch.zeros(1, 4)
    request = SimpleNamespace(kind="linear", A_u=rows, A_l=rows, alpha_u=line, alpha_l=line, beta_u=line, beta_l=line, weight=weight(), bias=None, input_shape=(40,), output_shape=(4,),
                              attrs={})
    executor = CudaFusedCrownExecutor()
    assert executor.supports(request, SimpleNamespace()) is False
    with pytest.raises(NotImplementedError, match="4 bits"):
        executor.run(request)


def test_sizes_beyond_32_bits_are_refused():
    """The library takes 32-bit counts: 2^32 + 5 rows would be 5.  (Expanded tensors: no memory behind them.)"""
    from boundflow_b200.weights4 import interval_linear4, linear4, quantise_weight4, rows_times_weight4

    w, many = weight(), 2 ** 32 + 5
    x, a = torch.zeros(1, 40).expand(many, 40), torch.zeros(1, 4).expand(many, 4)
    for call in (lambda: linear4(x, w), lambda: linear4(x.unsqueeze(0), w), lambda: interval_linear4(x, x, w), lambda: rows_times_weight4(a, w),
                 lambda: linear4(torch.zeros(1, 40).expand(2 ** 31, 40), w)):
        with pytest.raises(ValueError, match="at most 2.31 - 1"):
            call()
    for shape in ((many, 40), (40, many), (2 ** 30 + 1, 1)):
        with pytest.raises(ValueError, match="at most 2.30"):
            quantise_weight4(torch.zeros(1, 1).expand(shape))
