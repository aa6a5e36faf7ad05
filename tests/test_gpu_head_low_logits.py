"""Logits that lie far below zero as a whole: a constant offset of a row's logits changes
no probability, so the loss and its gradients stay what they are. exp(-lse) is past
float32's range here, and the vocabulary ends inside a unit of 8 words.

References and tolerances are those of the loss's own tests (float64)."""
import pytest
import torch

import test_gpu_head_loss as L

pytestmark = pytest.mark.gpu


def low_inputs(rows, dim, vocab, dt, level):
    """Logits near `level`, a few apart."""
    h, w, t, grad = L.inputs(rows, dim, vocab, dt, seed=rows + vocab, scale=1.0)
    h = (1.0 + 0.1 * h.float()).to(dt)
    w = (level / dim + 0.3 * w.float()).to(dt)
    grad[0] = 0.0
    return h, w, t, grad


@pytest.mark.parametrize("cap", (0.0, 400.0))
@pytest.mark.parametrize("dt", ("bf16", "f32"))
@pytest.mark.parametrize("rows,dim,vocab,level", [(1, 64, 9, -100.0), (3, 64, 1001, -150.0), (40, 64, 1002, -200.0), (64, 72, 131, -120.0),
                                                  (100, 64, 515, -100.0), (128, 33, 1003, -150.0), (200, 64, 260, -150.0),
                                                  (300, 128, 1005, -200.0), (260, 64, 774, -150.0), (513, 64, 2055, -100.0)])
def test_logits_far_below_zero(rows, dim, vocab, level, dt, cap):
    from gemmaedge_amd import head as H

    h, w, t, grad = low_inputs(rows, dim, vocab, L.DT[dt], level)
    hd = H.Head(rows, dim, vocab, dtype=L.DT[dt], train=True)
    loss, lse = hd.loss(h, w, t, softcap=cap)
    dh, dw = hd.loss_backward(grad, h, w, t, lse, softcap=cap)
    ref = L.reference(h, w, t, grad, cap, L.DT[dt])
    assert float(ref["lse"][0].max()) < -80.0
    for k, got in dict(loss=loss, lse=lse, dh=dh, dw=dw).items():
        L.close(got, ref[k], k)
    assert not dh[0].any()
