"""Products of one to five 16-bit rows with 4-bit weights where the numbers of a row differ by more than any fixed count of bits holds: the result may not depend on
how many rows a call has, nor on what lies beside a weight of zero.

Tolerance: products are exact, sums of 32 bits: 2^-24 * (terms / 8 + 32) of the sum of magnitudes |x| |w| (which leaves out what a zero weight meets), and half a step of the
output's type, 2^-8 (bf16) or 2^-11 (fp16) of it, or the type's smallest normal number.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from boundflow_b200.csrc import build

    build.build()
    return torch.device("cuda", 0)


def weight(n, k, group, dev, zeros, seed=0):
    """Random codes; columns `zeros` are zero in every other output."""
    from boundflow_b200.weights4 import Weight4

    g = torch.Generator("cpu").manual_seed(seed + 1000 * n + k + group)
    padded = -(-k // group) * group
    q = torch.randint(0, 16, (n, padded), generator=g, dtype=torch.uint8)
    for c in zeros:
        q[::2, c] = 8
    scales = torch.rand((padded // group, n), generator=g) + 0.25
    w = ((q.double() - 8) * scales.double().t().repeat_interleave(group, dim=1))[:, :k]
    return Weight4((q[:, ::2] | (q[:, 1::2] << 4)).contiguous().to(dev), scales.to(dev), k), w.to(dev), g


def check(got, x, w):
    t = x.dtype
    xd = x.double()
    want, size = xd @ w.t(), xd.abs() @ w.abs().t()
    tol = 2.0 ** -24 * (x.shape[1] / 8 + 32) * size + torch.finfo(t).eps / 2 * 1.01 * want.abs() + torch.finfo(t).tiny
    fine = want.abs() <= torch.finfo(t).max
    err = (got.double() - want).abs()
    assert bool((err <= tol)[fine].all()), f"worst {float((err / tol)[fine].max()):.3g} of the tolerance"
    assert bool((got.double().abs()[~fine] >= torch.finfo(t).max).all())


@pytest.mark.parametrize("kind,large", [("bf16", 1e10), ("bf16", -3e30), ("bf16", 7e5), ("fp16", 6e4)])
@pytest.mark.parametrize("n,k,group", [(70, 700, 64), (33, 130, 32), (40, 1000, 128), (16, 600, 512), (300, 5000, 128)])
def test_a_large_number_beside_a_weight_of_zero(dev, kind, large, n, k, group):
    from boundflow_b200.weights4 import linear4

    columns = [0, 37, 127, k - 1] if k > 128 else [0, k - 1]
    W, w, g = weight(n, k, group, dev, columns)
    for m in (1, 2, 3, 4, 5):
        x = torch.randn(m, k, generator=g) * (1e-3 if kind == "fp16" else 1.0)
        x[m - 1, columns] = large
        x = x.to(TYPES[kind]).to(dev)
        check(linear4(x, W), x, w)


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("group", [32, 64, 128, 256])
def test_all_magnitudes_and_many_zero_weights(dev, kind, group):
    """Magnitudes over the type's whole range, subnormal numbers and rows of nothing else among them, beside weights a half of which are zero."""
    from boundflow_b200.weights4 import Weight4, linear4

    n, k = 90, 1000
    g = torch.Generator("cpu").manual_seed(group)
    padded = -(-k // group) * group
    q = torch.randint(0, 16, (n, padded), generator=g, dtype=torch.uint8)
    q = torch.where(torch.rand(n, padded, generator=g) < 0.5, torch.full_like(q, 8), q)
    scales = torch.rand((padded // group, n), generator=g) + 0.25
    w = ((q.double() - 8) * scales.double().t().repeat_interleave(group, dim=1))[:, :k].to(dev)
    W = Weight4((q[:, ::2] | (q[:, 1::2] << 4)).contiguous().to(dev), scales.to(dev), k)
    low, high = (-133.0, 100.0) if kind == "bf16" else (-24.0, 15.0)
    for m in (1, 2, 3, 4, 5):
        x = torch.randn(m, k, generator=g).sign() * torch.exp2(low + (high - low) * torch.rand(m, k, generator=g))
        x[0, 128:256] = 2.0 ** low * torch.randint(0, 4, (128,), generator=g)
        x[m - 1, 300:500] = 0
        x = x.to(TYPES[kind]).to(dev)
        got = linear4(x, W)
        check(got, x, w)
        assert torch.equal(linear4(x[:1], W), got[:1]) or m == 5  # the same bits alone and beside other rows


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("n,k,group", [(60, 200, 32), (60, 200, 64), (61, 300, 128), (60, 700, 512)])
def test_several_infinities_in_a_group(dev, kind, n, k, group):
    """Infinity times zero is NaN and so are infinities of both signs in one sum, whatever else the group holds; the rows beside are as they are without."""
    from boundflow_b200.weights4 import linear4

    W, w, g = weight(n, k, group, dev, [3, 9])
    places = [{1: "inf", 2: "inf"}, {1: "inf", 2: "-inf"}, {3: "inf", 4: "inf"}, {3: "-inf", 9: "inf", k - 1: "inf"}, {5: "inf", 6: "nan"}, {c: "inf" for c in range(k)},
              {c: "-inf" for c in range(20, 31)}, {40: "inf"}]
    for m in (1, 2, 3, 4, 5):
        x = torch.randn(m, k, generator=g).to(TYPES[kind]).to(dev)
        clean = linear4(x, W)
        for row in range(m):
            for place in places:
                y = x.clone()
                for c, v in place.items():
                    y[row, c] = float(v)
                got, want = linear4(y, W), (y.double().cpu() @ w.t().cpu()).to(dev)
                assert torch.equal(got[row].isnan(), want[row].isnan()), (m, row, place)
                inf = want[row].isinf()
                assert torch.equal(got[row][inf].double(), want[row][inf]) and bool((got[row].isnan() | got[row].isinf()).all())
                others = [i for i in range(m) if i != row]
                assert torch.equal(got[others], clean[others])
