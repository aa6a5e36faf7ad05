"""Rows without a loss may hold anything: uninitialised padding adds nothing to a gradient,
not NaN either, and their own gradient is 0. References and tolerances are those of the
loss's own tests (float64)."""
import pytest
import torch

import test_gpu_head_loss as L

pytestmark = pytest.mark.gpu


def rows_of(ref, at):
    # an expected value and its tolerance, which may be one number for all rows
    return tuple(x[at] if torch.is_tensor(x) else x for x in ref)


@pytest.mark.parametrize("cap", (0.0, 30.0))
@pytest.mark.parametrize("dt", ("bf16", "f32"))
@pytest.mark.parametrize("rows,dim,vocab,pad", [(2, 64, 9, 0), (40, 64, 300, 0), (64, 33, 257, 0), (100, 72, 515, 8), (128, 1001, 130, 0),
                                                (200, 64, 260, 0), (300, 136, 1005, 3), (513, 256, 700, 0), (3, 33, 70001, 0),
                                                (70001, 64, 9, 0)])
def test_values_that_are_no_numbers_in_rows_without_a_loss(rows, dim, vocab, pad, dt, cap):
    from gemmaedge_amd import head as H

    h, w, t, grad = L.inputs(rows, dim, vocab, L.DT[dt], seed=rows, pad=pad, ignored=0.3)
    t[-1], t[0] = -1, 0
    ignored = ((t < 0) | (t >= vocab)).nonzero()[:, 0]
    clean = h.clone()
    clean[ignored] = 0.0
    for i, r in enumerate(ignored.tolist()):
        h[r, (7 * i) % dim] = (float("nan"), float("inf"), -float("inf"))[i % 3]
    h[ignored[-1]] = float("nan")
    before = h.clone()
    hd = H.Head(rows, dim, vocab, dtype=L.DT[dt], train=True)
    loss, lse = hd.loss(h, w, t, softcap=cap)
    dh, dw = hd.loss_backward(grad, h, w, t, lse, softcap=cap)
    assert not dh[ignored].any() and not loss[ignored].any()
    kept = (t >= 0) & (t < vocab)
    ref = L.reference(clean, w, t, grad, cap, L.DT[dt])
    for k, got in dict(loss=loss, lse=lse, dh=dh).items():
        L.close(got[kept], rows_of(ref[k], kept), k)
    L.close(dw, ref["dw"], "dw")
    only = hd.loss_backward(grad, h, w, t, lse, softcap=cap, need_hidden=False)[1]
    assert torch.equal(only, dw) and torch.equal(h.view(torch.uint8), before.view(torch.uint8))


@pytest.mark.parametrize("dt", ("bf16", "f32"))
@pytest.mark.parametrize("rows", (20, 100, 300))
def test_weights_that_are_no_numbers_leave_rows_without_a_loss_alone(rows, dt):
    from gemmaedge_amd import head as H

    h, w, t, grad = L.inputs(rows, 64, 300, L.DT[dt], seed=rows, ignored=0.5)
    t[-1] = -1
    w[7, 3], w[299, 60] = float("nan"), float("inf")
    hd = H.Head(rows, 64, 300, dtype=L.DT[dt], train=True)
    loss, lse = hd.loss(h, w, t)
    dh, _ = hd.loss_backward(grad, h, w, t, lse)
    ignored = (t < 0) | (t >= 300)
    assert not dh[ignored].any() and not loss[ignored].any()
