"""The answer head where its kernels change shape: tiles, lane groups, strides with
foreign values between the rows, long offsets, replayed graphs, and the operators
together in a training loop. References and tolerances are those of the operators'
own tests (float64)."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

import test_gpu_head_loss as L  # noqa: E402
import test_gpu_head_norm as N  # noqa: E402

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.mark.parametrize("cap", (0.0, 30.0, 50.0))
@pytest.mark.parametrize("dt", ("bf16", "f32"))
@pytest.mark.parametrize("rows,dim,vocab", [(31, 64, 256), (32, 72, 129), (33, 128, 257), (64, 136, 511), (65, 192, 512), (96, 64, 513),
                                            (97, 200, 300), (128, 64, 128), (129, 256, 1025), (192, 320, 256), (193, 64, 300),
                                            (256, 960, 700), (257, 64, 1300), (385, 128, 600)])
def test_loss_at_the_tiles_borders(rows, dim, vocab, dt, cap):
    L.check(rows, dim, vocab, dt, cap, seed=rows + dim)


@pytest.mark.parametrize("dt", ("bf16", "f32"))
@pytest.mark.parametrize("rows,dim,vocab", [(20, 64, 300), (100, 72, 300), (300, 33, 520)])
def test_foreign_values_between_the_rows(rows, dim, vocab, dt):
    from gemmaedge_amd import head as H

    h, w, t, grad = L.inputs(rows, dim, vocab, DT[dt], seed=3)
    wide_h = torch.full((rows, dim + 24), float("nan"), dtype=DT[dt], device="cuda")
    wide_w = torch.full((vocab, dim + 40), float("nan"), dtype=DT[dt], device="cuda")
    wide_h[:, 8:8 + dim], wide_w[:, 16:16 + dim] = h, w
    h, w = wide_h[:, 8:8 + dim], wide_w[:, 16:16 + dim]
    hd = H.Head(rows, dim, vocab, dtype=DT[dt], train=True)
    loss, lse = hd.loss(h, w, t, softcap=30.0)
    dh, dw = hd.loss_backward(grad, h, w, t, lse, softcap=30.0)
    ref = L.reference(h, w, t, grad, 30.0, DT[dt])
    for k, got in dict(loss=loss, lse=lse, dh=dh, dw=dw).items():
        L.close(got, ref[k], k)


@pytest.mark.parametrize("dt", ("bf16", "f32"))
def test_row_weights_of_every_size(dt):
    from gemmaedge_amd import head as H

    h, w, t, grad = L.inputs(80, 64, 300, DT[dt], seed=6)
    hd = H.Head(80, 64, 300, dtype=DT[dt], train=True)
    _, lse = hd.loss(h, w, t)
    for g in (torch.full_like(grad, 1 / 80), grad, grad * 1e-30, grad * 10.0 ** torch.arange(-20, 20, 0.5, device="cuda"),
              torch.zeros_like(grad)):
        dh, dw = hd.loss_backward(g, h, w, t, lse)
        ref = L.reference(h, w, t, g, 0.0, DT[dt])
        L.close(dh, ref["dh"], "dh")
        L.close(dw, ref["dw"], "dw")
        mh, mw = hd.loss_backward(-g, h, w, t, lse)  # the reference's tolerances are those of weights above zero
        L.close(-mh, ref["dh"], "dh of negative weights")
        L.close(-mw, ref["dw"], "dw of negative weights")
    # a weight that is no number stays with its row, and with no row at all if that carries no loss
    kept = (t >= 0) & (t < 300)
    bad, ignored = int(kept.nonzero()[0]), int((~kept).nonzero()[0])
    g = grad.clone()
    g[bad], g[ignored] = float("nan"), float("nan")
    dh, _ = hd.loss_backward(g, h, w, t, lse)
    ok = torch.ones(80, dtype=torch.bool, device="cuda")
    ok[bad] = False
    assert torch.isnan(dh[bad]).all() and not dh[ignored].any()
    ref = L.reference(h, w, t, torch.where(torch.isnan(g), 0.0, g), 0.0, DT[dt])
    L.close(dh[ok], tuple(x[ok] for x in ref["dh"]), "dh")


def test_equal_row_weights_are_not_rounded_to_the_gradients_type():
    # The logits' gradient is held in 8 bits; 1 / n for all rows is a common factor outside of them. One row of one
    # token: p - 1 is -1 / 2 exactly, so dhidden is half the other's row less half the target's, rounded once.
    from gemmaedge_amd import head as H

    w = torch.zeros(2, 64, device="cuda", dtype=torch.bfloat16)
    w[0] = 1.0
    h = torch.zeros(1, 64, device="cuda", dtype=torch.bfloat16)
    t = torch.zeros(1, dtype=torch.int32, device="cuda")
    g = torch.full((1,), 1 / 1021, device="cuda")
    hd = H.Head(1, 64, 2, train=True)
    _, lse = hd.loss(h, w, t)
    dh, _ = hd.loss_backward(g, h, w, t, lse)
    want = (-0.5 * g.double()).item()
    assert ((dh.double() - want).abs() <= abs(want) * (2.0 ** -8 + 1e-5)).all()


@pytest.mark.parametrize("dt", ("bf16", "f32"))
def test_offsets_past_31_bits(dt):
    from gemmaedge_amd import head as H

    vocab, dim, stride = 40000, 64, 65536  # 2.6 thousand million elements apart at the end
    h, small, t, grad = L.inputs(70, dim, vocab, DT[dt], seed=12)
    wide = torch.empty(vocab, stride, dtype=DT[dt], device="cuda")
    w = wide[:, :dim]
    w.copy_(small)
    out = torch.empty(vocab, stride, dtype=DT[dt], device="cuda")[:, 8:8 + dim]
    hd = H.Head(70, dim, vocab, dtype=DT[dt], train=True)
    loss, lse = hd.loss(h, w, t)
    dh, dw = hd.loss_backward(grad, h, w, t, lse, dweight=out)
    loss2, lse2 = hd.loss(h, small, t)
    dh2, dw2 = hd.loss_backward(grad, h, small, t, lse2)
    for a, b in ((loss, loss2), (lse, lse2), (dh, dh2), (dw, dw2)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("center", (True, False))
@pytest.mark.parametrize("dt,wdt", [("f32", "f32"), ("bf16", "f32")])
@pytest.mark.parametrize("dim", (4, 63, 64, 65, 127, 128, 129, 256, 257, 511, 512, 513, 1023, 1024, 1025, 1026, 2047, 2049, 4096, 4097, 4098,
                                 8190, 8191, 8192))
def test_norm_at_the_groups_borders(dim, dt, wdt, center):
    x, w, b, dy = N.inputs(23, dim, DT[dt], DT[wdt], seed=dim, pad=6)
    h = N.head(23, dim, DT[dt])
    y, mean, rstd = h.norm(x, w, b, eps=1e-5, center=center)
    dx, dw, db = h.norm_backward(dy, x, w, mean, rstd, bias=True)
    ref = N.reference(x, w, b, dy, 1e-5, center)
    for k, got in dict(y=y, rstd=rstd, dx=dx, dw=dw, db=db).items():
        N.close(got, ref[k], k)


@pytest.mark.parametrize("rows,dim", [(511, 640), (513, 640), (4099, 40), (8200, 24), (1025, 1100)])
def test_norm_of_many_rows(rows, dim):
    # More rows than the workgroups take at once, so that each adds up several.
    x, w, b, dy = N.inputs(rows, dim, torch.float32, torch.float32, seed=rows)
    h = N.head(rows, dim, torch.float32)
    y, mean, rstd = h.norm(x, w, b, eps=1e-5)
    dx, dw, db = h.norm_backward(dy, x, w, mean, rstd, bias=True)
    again = h.norm_backward(dy, x, w, mean, rstd, bias=True)
    ref = N.reference(x, w, b, dy, 1e-5, True)
    for k, got in dict(y=y, mean=mean, rstd=rstd, dx=dx, dw=dw, db=db).items():
        N.close(got, ref[k], k)
    for a, c in zip((dx, dw, db), again):
        assert torch.equal(a, c)


def test_replayed_training_step():
    from gemmaedge_amd import head as H

    rows, dim, vocab = 140, 128, 900
    dt = torch.bfloat16
    h, w, t, grad = L.inputs(rows, dim, vocab, dt, seed=2)
    nw = torch.rand(dim, device="cuda") + 0.5
    hd = H.Head(rows, dim, vocab, dtype=dt, train=True)
    empty = lambda *s, d=torch.float32: torch.empty(*s, dtype=d, device="cuda")  # noqa: E731
    out = dict(y=empty(rows, dim, d=dt), mean=empty(rows), rstd=empty(rows), loss=empty(rows), lse=empty(rows),
               dy=empty(rows, dim, d=dt), dw=empty(vocab, dim, d=dt), dx=empty(rows, dim, d=dt), dn=empty(dim))

    def step(o):
        hd.norm(h, nw, y=o["y"], mean=o["mean"], rstd=o["rstd"])
        hd.loss(o["y"], w, t, softcap=30.0, loss=o["loss"], lse=o["lse"])
        hd.loss_backward(grad, o["y"], w, t, o["lse"], softcap=30.0, dhidden=o["dy"], dweight=o["dw"])
        hd.norm_backward(o["dy"], h, nw, o["mean"], o["rstd"], dx=o["dx"], dweight=o["dn"])

    step(out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(out)
    for k in range(4):
        h2, w2, t2, g2 = L.inputs(rows, dim, vocab, dt, seed=20 + k)
        h.copy_(h2), w.copy_(w2), t.copy_(t2), grad.copy_(g2)
        graph.replay()
        torch.cuda.synchronize()
        got = {n: x.clone() for n, x in out.items()}
        step(out)  # the program's own work between two replays
        torch.cuda.synchronize()
        for n, x in out.items():
            assert torch.equal(x, got[n]), (k, n)


@pytest.mark.parametrize("bits", (32, 8))
def test_training_loop_learns(bits):
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import train_head

    losses = train_head.train(steps=60, rows=512, dim=256, vocab=1003, state_bits=bits)
    # near log(vocab) = 6.9 at first; the directions are far apart against the noise
    assert 6.0 < losses[0] < 8.0 and losses[-1] < 0.5 * losses[0], (losses[0], losses[-1])
