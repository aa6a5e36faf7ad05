"""Calls on a stream other than the current one: tensors that the program drops right
after a call keep their memory until the stream has passed it."""
import gc

import pytest
import torch

import test_gpu_head_loss as L
import test_gpu_head_norm as N

pytestmark = pytest.mark.gpu


def dropped(make, call, setup=lambda *made: None):
    """Whether new tensors of the sizes of make()'s get the memory of those that call() used, while its stream is busy.
    Nothing runs on the current stream meanwhile: two streams may share a queue, and a copy would wait for the other's work."""
    side = torch.cuda.Stream()
    made = make()
    call(side, setup(*made), *made)  # what a first call loads
    del made
    gc.collect()  # handles that other tests left: to free their memory waits for the device
    gc.disable()
    try:
        made = make()
        ready = setup(*made)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(200_000_000)
        call(side, ready, *made)
        where = {t.data_ptr() for t in made}
        like = [(t.shape, t.dtype) for t in made]
        del made, ready
        seen, again = [], []
        for shape, dtype in like:  # an allocation that finds no memory at hand may wait for the device
            again.append(torch.empty(shape, dtype=dtype, device="cuda"))
            if not side.query():
                seen.append(again[-1].data_ptr() in where)
        side.synchronize()
    finally:
        gc.enable()
    if not seen:
        pytest.skip("the stream was done before the tensors were made: nothing to see")
    return any(seen)


def test_loss_inputs_dropped_after_the_call():
    from gemmaedge_amd import head as H

    hd = H.Head(300, 256, 4100, train=True)

    def both(side, _, h, w, t, grad):
        loss, lse = hd.loss(h, w, t, stream=side)
        hd.loss_backward(grad, h, w, t, lse, stream=side)

    assert not dropped(lambda: L.inputs(300, 256, 4100, torch.bfloat16), both)


def test_norm_inputs_dropped_after_the_call():
    hd = N.head(700, 2048, torch.bfloat16)

    def both(side, _, x, w, b, dy):
        _, mean, rstd = hd.norm(x, w, b, stream=side)
        hd.norm_backward(dy, x, w, mean, rstd, stream=side)

    assert not dropped(lambda: N.inputs(700, 2048, torch.bfloat16, torch.bfloat16), both)


@pytest.mark.parametrize("bits", (32, 8))
def test_optimiser_dropped_after_the_step(bits):
    from gemmaedge_amd import head as H

    def make():
        return [torch.zeros(700_000 + 5 * i, device="cuda") for i in range(2)]

    assert not dropped(make, lambda side, opt, p, g: opt.step(stream=side),
                       lambda p, g: H.AdamW([p[:600_000]], [g[:600_000]], state_bits=bits))


def test_results_on_a_stream_given_in_any_form():
    from gemmaedge_amd import head as H

    h, w, t, grad = L.inputs(130, 64, 900, torch.bfloat16)
    hd = H.Head(130, 64, 900, train=True)
    loss, lse = hd.loss(h, w, t)
    want = (loss, lse) + hd.loss_backward(grad, h, w, t, lse)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for s in (side, side.cuda_stream, torch.cuda.ExternalStream(side.cuda_stream), torch.cuda.current_stream()):
        loss, lse = hd.loss(h, w, t, stream=s)
        got = (loss, lse) + hd.loss_backward(grad, h, w, t, lse, stream=s)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
