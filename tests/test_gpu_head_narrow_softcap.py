"""Softcaps so small that their reciprocals are past float32's range: a logit of 0 stays 0
with a slope of 1, every other one is the cap with a slope of 0."""
import pytest
import torch

import test_gpu_head_loss as L

pytestmark = pytest.mark.gpu


def rows_of(ref, at):
    # an expected value and its tolerance, which may be one number for all rows
    return tuple(x[at] if torch.is_tensor(x) else x for x in ref)


@pytest.mark.parametrize("cap", (1e-30, 5e-39, 1e-39, 1e-42))
@pytest.mark.parametrize("dt", ("bf16", "f32"))
@pytest.mark.parametrize("rows,dim,vocab", [(5, 64, 300), (100, 72, 1000), (300, 64, 600)])
def test_softcaps_below_every_number(rows, dim, vocab, dt, cap):
    from gemmaedge_amd import head as H

    h, w, t, grad = L.inputs(rows, dim, vocab, L.DT[dt], seed=rows, ignored=0.0)
    h[::2] = 0.0
    hd = H.Head(rows, dim, vocab, dtype=L.DT[dt], train=True)
    loss, lse = hd.loss(h, w, t, softcap=cap)
    dh, dw = hd.loss_backward(grad, h, w, t, lse, softcap=cap)
    ref = L.reference(h, w, t, grad, cap, L.DT[dt])
    for k, got in dict(loss=loss, lse=lse, dh=dh).items():
        L.close(got[::2], rows_of(ref[k], slice(None, None, 2)), k)
    assert not dh[1::2].any() and not dw.any()
    for got in (loss, lse):  # all logits are the cap or its negative
        assert ((got[1::2].double() - torch.log(torch.tensor(float(vocab), dtype=torch.float64))).abs() < 2.5e-5).all()
