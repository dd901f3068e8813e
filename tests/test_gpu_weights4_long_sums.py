"""Products back through 4-bit weights of many outputs: accumulators of matrix instructions truncate, always in the same direction, so a sum of n terms may not stay in one.

Tolerance, of the sum of magnitudes, which for positive rows and weights is the result itself.  A matrix instruction adds 16 products to an accumulator and cuts off less than one
unit in the last place (2^-23) of it.  Kernels for many rows: at most 48 instructions a sum, then one rounding (2^-24) for each of the n / 128 sums, the weight's own roundings below 2^-22:
2^-23 * 48 + 2^-24 * (n / 128 + 8).  Kernels for few rows: as many instructions, or 6 and an addition for every 32 of a warp's outputs, of which each of 8 warps has a share, then sums over warps and
blocks: 2^-23 * 48 + 2^-24 * (n / 256 + 24).
"""
import pytest
import torch

from tests.test_gpu_weights4_many import dev  # noqa: F401

pytestmark = pytest.mark.gpu


def positive(n, k, group, dev, seed):
    from boundflow_b200.weights4 import Weight4

    g = torch.Generator("cpu").manual_seed(seed)
    q = torch.randint(9, 16, (n, k), generator=g, dtype=torch.uint8)
    scales = torch.rand((k // group, n), generator=g) + 0.25
    w = (q.double() - 8) * scales.double().t().repeat_interleave(group, dim=1)
    return Weight4((q[:, ::2] | (q[:, 1::2] << 4)).contiguous().to(dev), scales.to(dev), k), w.to(dev), g


@pytest.mark.parametrize("n", [4096, 8192, 20000])
@pytest.mark.parametrize("m", [64, 300])
def test_many_rows(dev, n, m, monkeypatch):
    from boundflow_b200 import weights4

    monkeypatch.setattr(weights4, "_many_pays", lambda *a: True)
    W, w, g = positive(n, 256, 128, dev, n + m)
    a = torch.rand(m, n, generator=g).to(dev)
    want = a.double() @ w
    worst = float(((weights4.rows_times_weight4(a, W).double() - want).abs() / want).max())
    assert worst <= 2.0 ** -23 * 48 + 2.0 ** -24 * (n / 128 + 8), worst
    lo, up = torch.zeros(m, 256, device=dev).requires_grad_(), torch.ones(m, 256, device=dev).requires_grad_()
    gl, gu = torch.autograd.grad(weights4.interval_linear4(lo, up, W), (lo, up), (a, a))  # W >= 0: both are a W
    for got in (gl, gu):
        worst = float(((got.double() - want).abs() / want).max())
        assert worst <= 2.0 ** -23 * 48 + 2.0 ** -24 * (n / 128 + 8), worst


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [2, 8, 100])
@pytest.mark.parametrize("n", [9000, 20000])
def test_few_rows(dev, m, n, group, monkeypatch):
    """100 rows through 4096 columns fill the chip by themselves: a block has all outputs unless sums of many ask for more blocks."""
    from boundflow_b200 import weights4

    monkeypatch.setattr(weights4, "_many_pays", lambda *a: False)
    W, w, g = positive(n, 4096, group, dev, n + m + group)
    a = torch.rand(m, n, generator=g).to(dev)
    want = a.double() @ w
    tol = 2.0 ** -23 * 48 + 2.0 ** -24 * (n / 256 + 24)
    worst = float(((weights4.rows_times_weight4(a, W).double() - want).abs() / want).max())
    assert worst <= tol, worst
    lo, up = torch.zeros(m, 4096, device=dev).requires_grad_(), torch.ones(m, 4096, device=dev).requires_grad_()
    gl, gu = torch.autograd.grad(weights4.interval_linear4(lo, up, W), (lo, up), (a, a))
    for got in (gl, gu):
        assert float(((got.double() - want).abs() / want).max()) <= tol
