"""The AdamW step of gradients so small that the second moment is a subnormal number.

Tolerances, u = 2^-24: the moments by the same float32 operations in numpy; of the update
the square root and the quotient 1 ulp each (2 u), three products and a sum; p is rounded
twice."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("beta2", (0.9, 0.99, 0.9999))
@pytest.mark.parametrize("eps", (0.0, 1e-40, 1e-30, 1e-20, 1e-14, 1e-11, 1e-8))
@pytest.mark.parametrize("bits", (8, 32))
def test_second_moments_below_the_normal_numbers(bits, eps, beta2):
    from gemmaedge_amd import head as H

    f = np.float32
    n = 700
    rng = np.random.default_rng(5)
    g = (10.0 ** rng.uniform(-20.3, -17.0, n) * rng.choice([-1, 1], n)).astype(f)
    p0 = rng.uniform(-0.05, 0.05, n).astype(f)
    p = torch.from_numpy(p0.copy()).cuda()
    opt = H.AdamW([p], [torch.from_numpy(g).cuda()], lr=1e-2, beta1=0.9, beta2=beta2, eps=eps, weight_decay=0.0, state_bits=bits)
    opt.step()
    with np.errstate(under="ignore"):
        m = g * f(1 - 0.9)
        v = g * g * f(1 - beta2)
    live = v > 0
    denom = np.sqrt(v.astype(np.float64)) / np.sqrt(1 - beta2) + eps
    upd = np.where(live, m / np.where(live, denom, 1.0) * (1e-2 / (1 - 0.9)), 0.0)
    got = p.cpu().numpy()[live].astype(np.float64)
    assert live.sum() > 400 and (v[live] < 2.0 ** -126).sum() > 100
    err = 10 * U * np.abs(upd) + 2 * U * (np.abs(p0) + np.abs(upd))
    bad = ~(np.abs(got - (p0 - upd)[live]) <= err[live])
    assert not bad.any(), (int(bad.sum()), got[bad][:4], (p0 - upd)[live][bad][:4])
