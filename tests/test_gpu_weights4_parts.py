"""16-bit rows back through 4-bit weights whose products cancel, so that what the parts of a product leave out shows beside the rounding of the result.

Tolerance: each product is held to 2^-17 (a product's first bfloat16 part is off by at most half its step, 2^(E - 8) for a number from 2^E on, so that the second is below that and off by at most
2^(E - 17)); sums of few terms in 32 bits, cut off after each of at most 8 instructions (2^-23) and rounded when they are added (2^-24 * 8); half a step of the result's type, or of its
smallest normal number.
"""
import pytest
import torch

from tests.test_gpu_weights4_many import TYPES, dev, make  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("many", [True, False])
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("n,k,group", [(2, 3000, 32), (13, 1198, 512), (30, 700, 64)])
def test_products_that_cancel(dev, monkeypatch, many, kind, n, k, group):
    from boundflow_b200 import weights4

    monkeypatch.setattr(weights4, "_many_pays", lambda *a: many)
    W, w, g = make(n, k, group, dev, 30)
    for m in (40, 113):
        x = torch.randn(m, n, generator=g) * torch.exp2(4 * torch.rand(m, n, generator=g))
        x = x.to(TYPES[kind]).to(dev)
        # the last output's row cancels what the others come to in a column of its own, as nearly as its type can
        column = torch.arange(m, device=dev) * 5 % k
        rest = (x[:, :-1].double() @ w[:-1])[torch.arange(m, device=dev), column]
        last = w[-1, column]
        x[:, -1] = torch.where(last != 0, -rest / last, torch.zeros_like(rest)).clamp(-1e4, 1e4).to(TYPES[kind])
        want, size = x.double() @ w, x.double().abs() @ w.abs()
        got = weights4.rows_times_weight4(x, W)
        t = torch.finfo(TYPES[kind])
        tol = (2.0 ** -17 + 8 * 2.0 ** -23 + 8 * 2.0 ** -24) * size + t.eps / 2 * 1.01 * want.abs() + t.tiny * t.eps
        worst = float(((got.double() - want).abs() / tol).max())
        assert worst <= 1, worst
