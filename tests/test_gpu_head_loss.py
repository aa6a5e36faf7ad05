"""The vocabulary's cross entropy and its gradients on the GPU against float64.

Tolerances, u = 2^-24. A logit is a float32 sum of D exact products (float32
operands: of the plane products, which leave out 4 u of each): off by at most
2 D u (twice the sum's own bound, for adders inside the matrix cores that
truncate) + 4 u times S, the largest sum of |h w|. The softcap's hardware exp2
and reciprocal add 4e-7 of the cap, exp2 and the log 2e-5 to the lse. dz is off by
p g times the errors of l and lse and is rounded once to its type; the products
add 32 terms at a time (six times as often for float32 operands), 2 u of the sum of
magnitudes for each addition and 128 u for what an instruction adds up itself;
outputs are rounded once."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def inputs(rows, dim, vocab, dt, seed=1, pad=0, scale=3.0, ignored=0.2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.randn(max(rows, 1), dim + pad, generator=g, device="cuda").to(dt)[:rows, :dim]
    w = (torch.randn(vocab, dim + pad, generator=g, device="cuda") * scale / dim ** 0.5).to(dt)[:, :dim]
    t = torch.randint(vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    skip = torch.rand(rows, generator=g, device="cuda") < ignored
    out = torch.tensor([-1, -100, vocab, 2 ** 31 - 1, -2 ** 31], device="cuda", dtype=torch.int32)
    t = torch.where(skip, out[torch.arange(rows, device="cuda") % 5], t)
    grad = torch.rand(rows, generator=g, device="cuda") + 0.5
    return h, w, t, grad


def reference(h, w, t, grad, cap, dtype):
    h, w, grad = h.double(), w.double(), grad.double()
    n, d = h.shape
    v = w.shape[0]
    z = h @ w.t()
    l = cap * torch.tanh(z / cap) if cap > 0 else z
    lse = torch.logsumexp(l, 1)
    kept = (t >= 0) & (t < v)
    at = t.clamp(0, v - 1).long()
    loss = torch.where(kept, lse - l.gather(1, at[:, None])[:, 0], 0.0)
    S = float((h.abs() @ w.abs().t()).max()) if n else 0.0
    e_l = (2 * d + 4) * U * S + 4e-7 * max(cap, 0.0)
    e_lse = e_l + 2e-5 + 4 * U * float(lse.abs().max() if n else 0)
    p = torch.exp(l - lse[:, None])
    slope = 1 - (l / cap) ** 2 if cap > 0 else torch.ones_like(l)
    one = torch.zeros_like(p)
    one[torch.arange(n), at] = 1.0
    g = (grad * kept)[:, None]
    dz = g * (p - one) * slope
    r = torch.finfo(dtype).eps / 2
    rz = r if dtype == torch.bfloat16 else 4 * U
    e_dz = g * p * (e_l + e_lse + 1e-6) + dz.abs() * rz
    if cap > 0:
        e_dz = e_dz + g * (p - one).abs() * (2 * l.abs() / cap * e_l / cap + 4 * U)
    a = lambda x: x.abs()  # noqa: E731
    dh, dw = dz @ w, dz.t() @ h
    e_dh = e_dz @ a(w) + 2 * (6 * v / 32 + 64) * U * (a(dz) @ a(w))
    e_dw = e_dz.t() @ a(h) + 2 * (6 * n / 32 + 64) * U * (a(dz).t() @ a(h))
    return dict(loss=(loss, e_l + e_lse), lse=(lse, e_lse), dh=(dh, e_dh), dw=(dw, e_dw))


def close(got, ref, what):
    want, err = ref
    tol = err + torch.finfo(got.dtype).eps / 2 * (want.abs() + err) + 1e-37
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {float((off / tol).max()):.3g} tolerances"


def check(rows, dim, vocab, dt, cap, pad=0, seed=1, handle=None, **kw):
    from gemmaedge_amd import head as H

    h, w, t, grad = inputs(rows, dim, vocab, DT[dt], seed=seed, pad=pad, **kw)
    hd = handle or H.Head(rows, dim, vocab, dtype=DT[dt], train=True)
    loss, lse = hd.loss(h, w, t, softcap=cap)
    dh, dw = hd.loss_backward(grad, h, w, t, lse, softcap=cap)
    torch.cuda.synchronize()
    ref = reference(h, w, t, grad, cap, DT[dt])
    for k, got in dict(loss=loss, lse=lse, dh=dh, dw=dw).items():
        close(got, ref[k], k)
    ignored = (t < 0) | (t >= vocab)
    assert not loss[ignored].any() and not dh[ignored].any()
    return hd


@pytest.mark.parametrize("cap", (0.0, 30.0))
@pytest.mark.parametrize("dt", ("bf16", "f32"))
@pytest.mark.parametrize("rows,dim,vocab,pad", [(1, 1, 1, 0), (1, 8, 2, 0), (2, 64, 127, 0), (7, 33, 255, 0), (16, 72, 256, 8),
                                                (17, 100, 257, 4), (33, 64, 1000, 1), (64, 136, 1003, 0), (65, 64, 512, 64),
                                                (129, 200, 300, 0), (255, 96, 5003, 0), (256, 64, 256, 0), (257, 328, 999, 0),
                                                (300, 1001, 700, 0), (600, 257, 2049, 3)])
def test_loss(rows, dim, vocab, pad, dt, cap):
    check(rows, dim, vocab, dt, cap, pad)


@pytest.mark.parametrize("dt", ("bf16", "f32"))
def test_smaller_calls_on_a_larger_handle(dt):
    from gemmaedge_amd import head as H

    hd = H.Head(700, 512, 6000, dtype=DT[dt], train=True)
    for rows, dim, vocab in ((700, 512, 6000), (3, 40, 5000), (65, 512, 77), (1, 7, 6000), (200, 129, 300)):
        check(rows, dim, vocab, dt, 30.0, handle=hd, seed=rows)


def test_pieces_of_the_vocabulary():
    # 256 MB hold the gradient of 32,768 logits for each of 4,096 rows: two pieces here.
    check(4096, 64, 40000, "bf16", 30.0, seed=9)


@pytest.mark.parametrize("dt", ("bf16", "f32"))
def test_packed_pieces_of_the_weights(dt):
    # Rows of 1,001 elements are packed, 32,768 of the vocabulary at a time.
    check(5, 1001, 33333, dt, 0.0, seed=4)


def test_large_logits_and_certain_targets():
    # Logits of hundreds: probabilities of 0 and 1, sums that overflow without the largest taken out.
    check(40, 128, 600, "bf16", 0.0, scale=100.0)
    check(90, 128, 600, "f32", 30.0, scale=100.0)


def test_every_row_ignored():
    from gemmaedge_amd import head as H

    h, w, t, grad = inputs(70, 64, 300, torch.bfloat16)
    t.fill_(-1)
    hd = H.Head(70, 64, 300, train=True)
    loss, lse = hd.loss(h, w, t)
    dh, dw = hd.loss_backward(grad, h, w, t, lse)
    assert not loss.any() and not dh.any() and not dw.any() and torch.isfinite(lse).all()


def test_no_rows():
    from gemmaedge_amd import head as H

    h, w, t, grad = inputs(0, 65, 300, torch.float32)
    hd = H.Head(70, 65, 300, dtype=torch.float32, train=True)
    loss, lse = hd.loss(h, w, t)
    dw = torch.full((300, 65), 7.0, device="cuda")
    dh, dw = hd.loss_backward(grad, h, w, t, lse, dweight=dw)
    assert loss.numel() == 0 and dh.shape == (0, 65) and not dw.any()


def test_gradient_against_differences():
    from gemmaedge_amd import head as H

    h, w, t, grad = inputs(5, 24, 60, torch.float32, seed=8)
    hd = H.Head(5, 24, 60, dtype=torch.float32, train=True)
    _, lse = hd.loss(h, w, t, softcap=5.0)
    dh, dw = hd.loss_backward(grad, h, w, t, lse, softcap=5.0)
    kept = (t >= 0) & (t < 60)

    def value(h, w):
        l = 5.0 * torch.tanh(h @ w.t() / 5.0)
        loss = torch.logsumexp(l, 1) - l.gather(1, t.clamp(0, 59).long()[:, None])[:, 0]
        return (loss * grad.double())[kept].sum()

    args = [h.double(), w.double()]
    for k, got in enumerate((dh, dw)):
        flat = args[k].reshape(-1)
        for i in range(0, flat.numel(), 11):
            step = torch.zeros_like(flat)
            step[i] = 1e-5
            up, down = list(args), list(args)
            up[k], down[k] = (flat + step).view_as(args[k]), (flat - step).view_as(args[k])
            want = float(value(*up) - value(*down)) / 2e-5
            # the quotient's own error is near 1e-9; float32 results to 1e-5
            assert abs(float(got.reshape(-1)[i]) - want) < 5e-5 * (1 + abs(want))


def test_non_finite_rows_stay_to_themselves():
    from gemmaedge_amd import head as H

    for dt in (torch.bfloat16, torch.float32):
        h, w, t, grad = inputs(70, 64, 300, dt, ignored=0.0)
        h[3, 5], h[66, 63] = float("nan"), float("inf")
        hd = H.Head(70, 64, 300, dtype=dt, train=True)
        loss, lse = hd.loss(h, w, t)
        dh, dw = hd.loss_backward(grad, h, w, t, lse)
        ok = torch.ones(70, dtype=torch.bool, device="cuda")
        ok[3] = ok[66] = False
        assert torch.isfinite(lse[ok]).all() and torch.isfinite(dh[ok]).all()
        assert torch.isnan(lse[~ok]).all() and torch.isnan(loss[~ok]).all()


def test_only_what_is_wanted():
    from gemmaedge_amd import head as H

    h, w, t, grad = inputs(130, 264, 3000, torch.bfloat16)
    hd = H.Head(130, 264, 3000, train=True)
    _, lse = hd.loss(h, w, t)
    dh, dw = hd.loss_backward(grad, h, w, t, lse)
    a = hd.loss_backward(grad, h, w, t, lse, need_weight=False)
    assert a[1] is None and torch.equal(a[0], dh)
    a = hd.loss_backward(grad, h, w, t, lse, need_hidden=False)
    assert a[0] is None and torch.equal(a[1], dw)
    wide = torch.full((3000, 300), 9.0, dtype=torch.bfloat16, device="cuda")
    tall = torch.full((130, 301), 9.0, dtype=torch.bfloat16, device="cuda")
    hd.loss_backward(grad, h, w, t, lse, dhidden=tall[:, 5:269], dweight=wide[:, 3:267])
    assert torch.equal(tall[:, 5:269], dh) and torch.equal(wide[:, 3:267], dw)
    for x, a, b in ((tall, 5, 269), (wide, 3, 267)):
        assert (x[:, :a] == 9).all() and (x[:, b:] == 9).all()


def test_same_bits_twice_and_on_another_stream():
    from gemmaedge_amd import head as H

    h, w, t, grad = inputs(513, 256, 4100, torch.bfloat16)
    hd = H.Head(513, 256, 4100, train=True)

    def both():
        loss, lse = hd.loss(h, w, t, softcap=30.0)
        return (loss, lse) + hd.loss_backward(grad, h, w, t, lse, softcap=30.0)

    first = both()
    again = both()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        third = both()
    side.synchronize()
    for a, b, c in zip(first, again, third):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_refusals():
    from gemmaedge_amd import head as H
    from gemmaedge_amd import sampler as S

    h, w, t, grad = inputs(8, 64, 300, torch.bfloat16)
    hd = H.Head(8, 64, 300)
    loss, lse = hd.loss(h, w, t)
    for bad in (lambda: hd.loss(h.float(), w, t), lambda: hd.loss(h, w.float(), t), lambda: hd.loss(h, w[:, :63], t),
                lambda: hd.loss(h, w, t.long()), lambda: hd.loss(h, w, t[:7]), lambda: hd.loss(h.cpu(), w, t),
                lambda: hd.loss(h, w.t(), t), lambda: hd.loss(h, w, t, lse=lse[:3]), lambda: hd.loss(h[0], w, t),
                lambda: hd.loss_backward(grad.double(), h, w, t, lse)):
        with pytest.raises(ValueError):
            bad()
    for bad, code in ((lambda: hd.loss_backward(grad, h, w, t, lse), S.GE_ERR_CAPACITY),
                      (lambda: hd.loss(torch.cat([h, h]), w, torch.cat([t, t])), S.GE_ERR_CAPACITY),
                      (lambda: hd.loss(h, torch.cat([w, w]), t), S.GE_ERR_CAPACITY),
                      (lambda: hd.loss(h, w, t, softcap=float("nan")), S.GE_ERR_INVALID_ARG),
                      (lambda: hd.loss(h, w[:0], t), S.GE_ERR_INVALID_ARG)):
        with pytest.raises(S.SamplerError) as e:
            bad()
        assert e.value.code == code
