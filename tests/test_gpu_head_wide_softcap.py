"""Softcaps of every size. Where the cap is far above the logits the capped logit is the
logit itself, and its error has to be relative to the logit, not to the cap.

Tolerances, u = 2^-24, as in the loss's own tests, but for the softcap: 4e-7 of the cap up
to 64, above that 1e-6 of the logit (exp2, its sum with 1 and the reciprocal 2.9e-7 of
1 / (exp(2 x) + 1) at x = 1 / 4, where tanh is 0.245, less beyond; a series below)."""
import pytest
import torch

import test_gpu_head_loss as L

pytestmark = pytest.mark.gpu

U = L.U


def reference(h, w, t, grad, cap, dtype):
    h, w, grad = h.double(), w.double(), grad.double()
    n, d = h.shape
    v = w.shape[0]
    z = h @ w.t()
    y = torch.tanh(z / cap)
    l = cap * y
    lse = torch.logsumexp(l, 1)
    kept = (t >= 0) & (t < v)
    at = t.clamp(0, v - 1).long()
    loss = torch.where(kept, lse - l.gather(1, at[:, None])[:, 0], 0.0)
    slope = 1 - y * y
    S = float((h.abs() @ w.abs().t()).max())
    e_l = slope * (2 * d + 4) * U * S + (4e-7 * cap if cap <= 64 else 1e-6 * l.abs())
    e_lse = e_l.amax(1) + 2e-5 + 4 * U * lse.abs()
    p = torch.exp(l - lse[:, None])
    one = torch.zeros_like(p)
    one[torch.arange(n), at] = 1.0
    g = (grad * kept)[:, None]
    dz = g * (p - one) * slope
    rz = torch.finfo(dtype).eps / 2 if dtype == torch.bfloat16 else 4 * U
    e_dz = g * p * (e_l + e_lse[:, None] + 1e-6) + dz.abs() * rz
    e_dz = e_dz + g * (p - one).abs() * (2 * y.abs() * (e_l / cap + slope * 8 * U) + 4 * U)
    dh, dw = dz @ w, dz.t() @ h
    e_dh = e_dz @ w.abs() + 2 * (6 * v / 32 + 64) * U * (dz.abs() @ w.abs())
    e_dw = e_dz.t() @ h.abs() + 2 * (6 * n / 32 + 64) * U * (dz.abs().t() @ h.abs())
    return dict(loss=(loss, e_l.amax(1) + e_lse), lse=(lse, e_lse), dh=(dh, e_dh), dw=(dw, e_dw))


@pytest.mark.parametrize("cap", (39.0, 41.0, 50.0, 64.0, 65.0, 100.0, 300.0, 1e4, 1e6, 1e8, 1e20, 1e30, 1e37, 3e38))
@pytest.mark.parametrize("dt", ("bf16", "f32"))
@pytest.mark.parametrize("rows,dim,vocab,scale", [(5, 64, 300, 3.0), (100, 72, 1003, 20.0), (300, 64, 600, 0.05)])
def test_softcaps_above_the_logits(rows, dim, vocab, scale, dt, cap):
    from gemmaedge_amd import head as H

    h, w, t, grad = L.inputs(rows, dim, vocab, L.DT[dt], seed=rows, scale=scale)
    hd = H.Head(rows, dim, vocab, dtype=L.DT[dt], train=True)
    loss, lse = hd.loss(h, w, t, softcap=cap)
    dh, dw = hd.loss_backward(grad, h, w, t, lse, softcap=cap)
    ref = reference(h, w, t, grad, cap, L.DT[dt])
    for k, got in dict(loss=loss, lse=lse, dh=dh, dw=dw).items():
        L.close(got, ref[k], k)


def test_one_word_above_the_others():
    # One logit of 5, the others 0: at a cap far above it nothing is capped.
    from gemmaedge_amd import head as H

    w = torch.zeros(300, 64, device="cuda", dtype=torch.bfloat16)
    w[17, 0] = 5.0
    h = torch.zeros(1, 64, device="cuda", dtype=torch.bfloat16)
    h[0, 0] = 1.0
    t = torch.full((1,), 17, device="cuda", dtype=torch.int32)
    hd = H.Head(1, 64, 300)
    want = float(torch.log(torch.exp(torch.tensor(5.0, dtype=torch.float64)) + 299.0))
    for cap in (1e5, 1e8, 3e38):
        loss, lse = hd.loss(h, w, t, softcap=cap)
        assert abs(float(lse) - want) < 2e-5 + 6e-6 and abs(float(loss) - (want - 5.0)) < 2e-5 + 12e-6, cap
