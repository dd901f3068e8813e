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
