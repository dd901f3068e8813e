"""The quotients of the quantisation, at every mantissa that a largest weight can have: a code is w / scale rounded to 32 bits and then to the nearest even whole number, and numbers at
and beside the half-way points show any quotient that is off by its last bit.  (A quotient of 32-bit numbers formed in 64 bits and rounded is the rounded one: 53 >= 2 * 24 + 2.)"""
import pytest
import torch

from tests.test_gpu_weights4_many import dev  # noqa: F401

pytestmark = pytest.mark.gpu


def test_every_mantissa(dev):
    from boundflow_b200.weights4 import quantise_weight4

    g = torch.Generator("cuda").manual_seed(0)
    seventh = torch.tensor(1.0, device=dev) / 7
    per = 1 << 18
    for part in range(32):
        bits = (torch.arange(per, device=dev, dtype=torch.int32) + part * per) | ((90 + 3 * part) << 23)
        top = bits.view(torch.float32)
        scale = top * seventh
        half = (torch.randint(-7, 7, (per, 32), generator=g, device=dev) + 0.5) * scale[:, None]
        aside = torch.randint(-2, 3, (per, 32), generator=g, device=dev, dtype=torch.int32)
        w = (half.view(torch.int32) + aside).view(torch.float32)
        w[:, 0] = torch.where(torch.arange(per, device=dev) % 2 == 0, top, -top)
        assert bool((w.abs() <= top[:, None]).all())
        got = quantise_weight4(w, 32)
        assert torch.equal(got.scales[0], scale)
        want = (w.double() / scale.double()[:, None]).float().round()
        assert torch.equal(got.integers(), want.to(torch.int8))
