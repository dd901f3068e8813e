"""Refusals of the 4-bit weights and of AdamW, by the library and by the Python layer: no GPU is needed for any of them."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from boundflow_b200 import _lib
    from boundflow_b200.csrc import build

    build.build()
    return _lib.load()


def _weight(n=4, k=40, group=32):
    from boundflow_b200.weights4 import Weight4

    padded = -(-k // group) * group
    return Weight4(torch.zeros(n, padded // 2, dtype=torch.uint8), torch.zeros(padded // group, n), k)


def test_weight4_describes_itself():
    w = _weight()
    assert w.shape == (4, 40) and w.group == 32 and w.dim() == 2 and w.to("cpu") is w and "groups of 32" in repr(w)


@pytest.mark.parametrize("codes,scales,k,error", [
    (torch.zeros(4, 32), torch.zeros(2, 4), 40, TypeError),
    (torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(2, 4, dtype=torch.float16), 40, TypeError),
    (torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(2, 5), 40, ValueError),      # another number of rows
    (torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(2, 4), 32, ValueError),      # a whole group of padding
    (torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(2, 4), 65, ValueError),      # more columns than codes
    (torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(2, 4), 0, ValueError),
    (torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 4), 64, ValueError),      # groups of 16
    (torch.zeros(4, 48, dtype=torch.uint8), torch.zeros(1, 4), 96, ValueError),      # groups of 96
    (torch.zeros(4, 48, dtype=torch.uint8), torch.zeros(0, 4), 96, ValueError),
    (torch.zeros(0, 32, dtype=torch.uint8), torch.zeros(2, 0), 64, ValueError),
    (torch.zeros(64, dtype=torch.uint8), torch.zeros(2, 4), 64, ValueError),
    (torch.zeros(8, 32, dtype=torch.uint8)[::2], torch.zeros(2, 4), 64, ValueError),  # strided
    (torch.zeros(129, dtype=torch.uint8)[1:].view(4, 32), torch.zeros(2, 4), 64, ValueError),  # off its boundary
])
def test_weight4_refuses(codes, scales, k, error):
    from boundflow_b200.weights4 import Weight4

    with pytest.raises(error):
        Weight4(codes, scales, k)


def test_products_refuse_before_any_device():
    from boundflow_b200.weights4 import interval_linear4, linear4, quantise_weight4, rows_times_weight4

    w = _weight()
    x = torch.zeros(2, 40)
    for call, error in [
        (lambda: linear4(x, torch.zeros(4, 40)), TypeError), (lambda: linear4(x.double(), w), TypeError), (lambda: linear4(x[:, :39], w), ValueError),
        (lambda: linear4(torch.tensor(1.0), w), ValueError), (lambda: linear4(x, w, torch.zeros(5)), ValueError), (lambda: linear4(x, w, torch.zeros(4, dtype=torch.int32)), TypeError),
        (lambda: interval_linear4(x, x[:1], w), ValueError), (lambda: interval_linear4(x.bfloat16(), x.bfloat16(), w), TypeError),
        (lambda: interval_linear4(x, x, w, torch.zeros(4).half()), TypeError), (lambda: interval_linear4(x, x[:, :39], w), ValueError),
        (lambda: rows_times_weight4(x, w), ValueError), (lambda: rows_times_weight4(torch.zeros(2, 4), torch.zeros(4, 40)), TypeError),
        (lambda: quantise_weight4(torch.zeros(4, 40).double()), TypeError), (lambda: quantise_weight4(torch.zeros(4)), ValueError),
        (lambda: quantise_weight4(torch.zeros(4, 40), 48), ValueError), (lambda: quantise_weight4(torch.zeros(4, 40), 16), ValueError),
        (lambda: quantise_weight4(torch.zeros(0, 40)), ValueError),
    ]:
        with pytest.raises(error):
            call()


def test_a_device_is_needed():
    if torch.cuda.is_available():
        pytest.skip("there is one")
    from boundflow_b200.weights4 import linear4

    with pytest.raises(RuntimeError):
        linear4(torch.zeros(2, 40), _weight())


def test_library_refuses(lib):
    from boundflow_b200 import _lib

    p = 1 << 20  # never read: every call is refused before a launch
    bad = _lib.BF_E_INVALID
    assert lib.bf_w4_linear(p, 0, None, p, None, 0, p, 1, 64, 4, 32, None) == bad
    assert lib.bf_w4_linear(None, 0, p, p, None, 0, p, 1, 64, 4, 32, None) == bad
    assert lib.bf_w4_linear(p, 3, p, p, None, 0, p, 1, 64, 4, 32, None) == bad      # unknown type
    assert lib.bf_w4_linear(p, 0, p, p, p, 7, p, 1, 64, 4, 32, None) == bad
    assert lib.bf_w4_linear(p, 0, p, p, None, 0, p, 0, 64, 4, 32, None) == bad      # no rows
    assert lib.bf_w4_linear(p, 0, p, p, None, 0, p, 1, 64, 4, 48, None) == bad      # group
    assert lib.bf_w4_linear(p, 0, p, p, None, 0, p, 1, 64, 4, 16, None) == bad
    assert lib.bf_w4_linear(p, 0, p + 8, p, None, 0, p, 1, 64, 4, 32, None) == bad  # boundary
    assert b"16-byte" in lib.bf_last_error_string()
    assert lib.bf_w4_linear(p, 0, p, p, None, 0, p, 1, 0, 4, 32, None) == bad
    assert lib.bf_w4_interval(p, p, 1, 1, p, p, None, p, p, 1, 64, 4, 32, None) == bad  # relu_in of a midpoint
    assert lib.bf_w4_interval(p, p, 2, 0, p, p, None, p, p, 1, 64, 4, 32, None) == bad
    assert lib.bf_w4_interval(p, None, 0, 0, p, p, None, p, p, 1, 64, 4, 32, None) == bad
    assert lib.bf_w4_rows(p, 5, p, p, p, 1, 64, 4, 32, None) == bad
    assert lib.bf_w4_interval_grad(p, p, p, p, None, p, 1, 64, 4, 32, None) == bad
    assert lib.bf_w4_linear_grad(p, 9, p, p, p, None, 0, 1, 64, 4, 32, None) == bad and lib.bf_w4_linear_grad(p, 0, p, p, None, p, 9, 1, 64, 4, 32, None) == bad
    assert lib.bf_w4_quantise(p, 4, p, p, 4, 64, 32, None) == bad
    assert lib.bf_w4_integers(p, None, 4, 64, 32, None) == bad
    assert lib.bf_w4_dense(p, p, None, 4, 64, 32, None) == bad
    assert lib.bf_rows_dot(p, None, p, 0, 1, 1, None) == bad
    assert lib.bf_column_sums(p, 0, p, 9, 1, 1, None) == bad
    entry = (ctypes.c_byte * 40)()
    assert lib.bf_adamw_step(None, 1, 0, 0, 32, p, p, None, None, 0.9, 0.99, 1e-8, None, p, 1, None) == bad
    assert lib.bf_adamw_step(entry, -1, 0, 0, 32, p, p, None, None, 0.9, 0.99, 1e-8, None, p, 1, None) == bad
    assert lib.bf_adamw_step(entry, 1, 0, 0, 16, p, p, None, None, 0.9, 0.99, 1e-8, None, p, 1, None) == bad
    assert lib.bf_adamw_step(entry, 1, 0, 0, 8, p, p, None, p, 0.9, 0.99, 1e-8, None, p, 1, None) == bad
    assert lib.bf_adamw_step(entry, 1, 0, 0, 32, p + 4, p, None, None, 0.9, 0.99, 1e-8, None, p, 1, None) == bad
    assert lib.bf_adamw_step(entry, 1, 0, 0, 32, p, p, None, None, 1.0, 0.99, 1e-8, None, p, 1, None) == bad
    assert lib.bf_adamw_step(entry, 1, 0, 0, 32, p, p, None, None, 0.9, 0.99, -1.0, None, p, 1, None) == bad
    ctypes.cast(entry, ctypes.POINTER(ctypes.c_longlong))[2] = 5  # five elements at null pointers
    assert lib.bf_adamw_step(entry, 1, 0, 0, 32, p, p, None, None, 0.9, 0.99, 1e-8, None, p, 1, None) == bad
    ctypes.cast(entry, ctypes.POINTER(ctypes.c_longlong))[2] = 0
    ctypes.cast(entry, ctypes.POINTER(ctypes.c_longlong))[3] = 100  # not a whole block
    assert lib.bf_adamw_step(entry, 1, 0, 0, 32, p, p, None, None, 0.9, 0.99, 1e-8, None, p, 1, None) == bad
    ctypes.cast(entry, ctypes.POINTER(ctypes.c_longlong))[3] = 0
    assert lib.bf_adamw_step(entry, 1, 1, 0, 32, p, p, None, None, 0.9, 0.99, 1e-8, None, p, 1, None) == _lib.BF_E_UNSUPPORTED  # bf16 beside fp32 gradients
    assert lib.bf_adamw_moments(p, p, p, p, p, p, 100, None) == bad


def test_adamw_refuses():
    from boundflow_b200.optim import AdamW

    p = torch.zeros(4)
    for call, error in [
        (lambda: AdamW([]), ValueError), (lambda: AdamW([p]), RuntimeError), (lambda: AdamW([p.double()]), TypeError), (lambda: AdamW([p], state_bits=16), ValueError),
        (lambda: AdamW([p], betas=(1.0, 0.9)), ValueError), (lambda: AdamW([p], eps=-1.0), ValueError), (lambda: AdamW([{"params": [p], "betas": (0.5, 0.5)}]), ValueError),
        (lambda: AdamW([p], eps=float("nan")), ValueError),
    ]:
        with pytest.raises(error):
            call()


def test_chains_refuse_4_bit_weights_and_graphs_take_them():
    from boundflow_b200.crown import needs_graph_path
    from boundflow_b200.ir import BFTaskModule, BoundTask, TaskKind, TaskOp

    ops = [TaskOp("linear", "l1", ["x", "W"], ["y"])]
    task = BoundTask(task_id="t", kind=TaskKind.INTERVAL_IBP, ops=ops, input_values=["x"], output_values=["y"])
    assert needs_graph_path(BFTaskModule([task], "t", {"params": {"W": _weight()}}))
    assert not needs_graph_path(BFTaskModule([task], "t", {"params": {"W": torch.zeros(4, 40)}}))
    assert not needs_graph_path(BFTaskModule([task], "t", {}))
