"""AdamW where numbers leave the normal range (second moments below it, an eps that does not cover them), and states that are refused.  The moments are taken from the optimiser (they are tested bit for bit
elsewhere); the step from them is formed in 64 bits, with the tolerance of `check_params`."""
import pytest
import torch

from tests.test_gpu_adamw import check_params, dev  # noqa: F401

pytestmark = pytest.mark.gpu


def test_roundings_of_a_step_with_32_bit_moments(dev):
    """From p = 0, with lr and both corrections powers of two, a step is three roundings of at most 2^-24 each: sqrt(v), that plus eps, and the quotient."""
    from boundflow_b200.optim import AdamW

    g = torch.Generator("cpu").manual_seed(3)
    grad = (torch.randn(200000, generator=g) * torch.exp2(20 * torch.rand(200000, generator=g) - 10)).to(dev)
    p = torch.zeros_like(grad)
    AdamW([p], lr=2.0 ** -8, betas=(0.5, 0.75), eps=2.0 ** -30, weight_decay=0.0).step([grad])  # 1 / (1 - 0.5) = 2, 1 / sqrt(1 - 0.75) = 2
    x = grad.double()
    v = ((0.25 * x).float().double() * x).float().double()
    want = -(2.0 ** -7) * (0.5 * x) / (2 * v.sqrt() + 2.0 ** -30)
    assert float(((p.double() - want) / want).abs().max()) <= 3.0 * 2.0 ** -24 * 1.000001


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [1.1e-18, 2e-18, 1e-16, 1e-13, 1e-8])
@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.5, 0.9999), (0.0, 0.0)])
def test_second_moments_below_the_normal_range(dev, bits, eps, betas):
    from boundflow_b200.optim import AdamW

    grad = torch.cat([torch.full((256,), g) for g in (3.4e-18, 1e-18, 3e-17, 1e-15, 1e-10, 2e-19)]).to(dev)
    p = torch.zeros_like(grad)
    opt = AdamW([p], lr=1.0, betas=betas, eps=eps, weight_decay=0.0, state_bits=bits)
    before = p.clone()
    opt.step([grad])
    eps32, g = float(torch.tensor(eps)), grad.double()
    c1, c2 = (float(torch.tensor(1 - b)) for b in betas)
    m = (c1 * g).float().double()
    v = ((c2 * g).float().double() * g).float().double()  # each product rounded by itself
    check_params(p, before, m, v, 1, 1.0, 0.0, betas, eps32)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_refused_state_changes_nothing(dev, bits):
    from boundflow_b200.optim import AdamW

    def fresh():
        g = torch.Generator("cpu").manual_seed(7)
        p = torch.randn(500, generator=g).to(dev)
        opt = AdamW([p], lr=0.01, state_bits=bits)
        opt.step([torch.randn(500, generator=g).to(dev)])
        return opt

    opt, twin = fresh(), fresh()
    good = opt.state_dict()
    moments = {k: v.clone() for k, v in good["moments"].items()}
    wrong = dict(moments, exp_avg=moments["exp_avg"][:256])
    for change in ({"moments": wrong, "betas": (0.1, 0.2), "eps": 1.0}, {"betas": (0.5, 1.5)}, {"betas": (0.5, float("nan"))}, {"eps": -1.0, "betas": (0.1, 0.2)},
                   {"step": -1, "betas": (0.1, 0.2)}, {"groups": [{"lr": -1.0, "weight_decay": 0.0}], "betas": (0.1, 0.2)}, {"moments": {}, "eps": 1.0}):
        with pytest.raises(ValueError):
            opt.load_state_dict(dict(good, **change))
        assert (opt.betas, opt.eps, opt.param_groups[0]["lr"]) == (twin.betas, twin.eps, twin.param_groups[0]["lr"])
    grad = torch.linspace(-1, 1, 500, device=dev)
    opt.step([grad])
    twin.step([grad])
    assert torch.equal(opt.param_groups[0]["params"][0], twin.param_groups[0]["params"][0])
    assert all(torch.equal(a, b) for a, b in zip(opt.flat_moments(), twin.flat_moments()))
