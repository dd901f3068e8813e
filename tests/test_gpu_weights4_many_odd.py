"""Many rows times a 4-bit weight where many of them hold infinities and NaN, as gradients do in the step in which a loss scale overflows: the kernels for many rows against
64 bits, with the infinities and NaN where those have them.  Tolerance of what stays finite: that of the rows without (2^-24 * (terms / 8 + 32) of the sum of magnitudes, 2^-16 of
it beside 16-bit rows, half a step of the output's type)."""
import pytest
import torch

from tests.test_gpu_weights4_many import TYPES, check, dev, make, many  # noqa: F401

pytestmark = pytest.mark.gpu


def compare(got, want, size, terms, kind):
    assert torch.equal(got.isnan(), want.isnan())
    inf = want.isinf()
    assert torch.equal(got.isinf(), inf) and torch.equal(got.double()[inf], want[inf])
    fine = want.isfinite()
    check(got[fine], want[fine], size[fine], terms, TYPES[kind], 0.0 if kind == "fp32" else 2.0 ** -16)


def product(a, w):
    """a w in 64 bits, on the CPU: elementwise products and sums keep infinities and NaN where they belong.  Magnitudes of the finite ones."""
    a, w = a.double().cpu(), w.cpu()
    return (a @ w), (torch.where(a.isfinite(), a, torch.zeros_like(a)).abs() @ w.abs())


@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("m,n,k,group", [(64, 70, 200, 64), (300, 130, 257, 32), (129, 2500, 300, 128), (257, 4200, 130, 512)])
def test_infinities_in_every_row(dev, kind, m, n, k, group):
    from boundflow_b200.weights4 import rows_times_weight4

    W, w, g = make(n, k, group, dev, 20)
    w = w.cpu()
    a = torch.randn(m, n, generator=g).to(TYPES[kind])
    places = torch.randint(0, n, (m,), generator=g)
    for i in range(m):
        a[i, places[i]] = float("inf") if i % 3 else -float("inf")
    a[::7, n - 1] = float("inf")
    a[5, 0] = float("nan")
    a[40:44] = torch.randn(4, n, generator=g).to(TYPES[kind])  # and some rows without
    want, size = product(a, w)
    got = rows_times_weight4(a.to(dev), W).cpu()
    compare(got, want, size, n, kind)
    every = torch.full((m, n), float("-inf"), dtype=TYPES[kind], device=dev)  # nothing else
    compare(rows_times_weight4(every, W).cpu(), *product(every, w), n, kind)


@pytest.mark.parametrize("m,n,k,group", [(80, 70, 200, 64), (130, 2300, 140, 128)])
def test_infinite_gradients_of_bounds(dev, m, n, k, group):
    """The two products of a pair meet as the formula has them: (sum - difference) / 2 and (sum + difference) / 2."""
    from boundflow_b200.weights4 import interval_linear4

    W, w, g = make(n, k, group, dev, 21)
    w = w.cpu()
    dl, du = torch.randn(m, n, generator=g), torch.randn(m, n, generator=g)
    dl[::2, 3], du[::3, n - 2], dl[7, 1], du[8, 2] = float("inf"), float("-inf"), float("nan"), float("inf")
    lo = torch.zeros(m, k, device=dev).requires_grad_()
    up = torch.ones(m, k, device=dev).requires_grad_()
    gl, gu = torch.autograd.grad(interval_linear4(lo, up, W), (lo, up), (dl.to(dev), du.to(dev)))
    s, size_s = product(dl + du, w)
    d, size_d = product(du - dl, w.abs())
    compare(gl.cpu(), 0.5 * (s - d), size_s + size_d, n, "fp32")
    compare(gu.cpu(), 0.5 * (s + d), size_s + size_d, n, "fp32")


def test_rows_of_infinities_take_no_other_order_of_time(dev):
    """An infinity in every row of every stage costs a second pass over the images, a few times the product and not hundreds of times."""
    from boundflow_b200.weights4 import rows_times_weight4

    W, _, g = make(4096, 2048, 128, dev, 22)
    a = torch.randn(256, 4096, generator=g).to(torch.bfloat16).to(dev)
    b = a.clone()
    b[:, ::64] = float("inf")

    def us(rows):
        rows_times_weight4(rows, W)
        best = float("inf")
        for _ in range(5):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            rows_times_weight4(rows, W)
            end.record()
            end.synchronize()
            best = min(best, 1e3 * begin.elapsed_time(end))
        return best

    assert us(b) < 40 * us(a)
