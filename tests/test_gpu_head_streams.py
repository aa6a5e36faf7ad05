"""Calls on a stream other than the current one: tensors that the program drops right
after a call keep their memory until the stream has passed it."""
import pytest
import torch

import test_gpu_head_loss as L
import test_gpu_head_norm as N

pytestmark = pytest.mark.gpu


def dropped(make, call):
    """Whether new tensors of the sizes of make()'s get the memory of those that call(*) used, while its stream is busy."""
    side = torch.cuda.Stream()
    call(side, *make())  # what a first call loads
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)
    made = make()
    side.wait_stream(torch.cuda.current_stream())
    keep = call(side, *made)
    where = {t.data_ptr() for t in made}
    like = [(t.shape, t.dtype) for t in made]
    del made
    again = [torch.empty(shape, dtype=dtype, device="cuda") for shape, dtype in like]
    busy = not side.query()
    shared = [t for t in again if t.data_ptr() in where]
    side.synchronize()
    del keep
    assert busy, "the stream was done before the tensors were made"
    return bool(shared)


def test_loss_inputs_dropped_after_the_call():
    from gemmaedge_amd import head as H

    hd = H.Head(300, 256, 4100, train=True)

    def both(side, h, w, t, grad):
        loss, lse = hd.loss(h, w, t, stream=side)
        hd.loss_backward(grad, h, w, t, lse, stream=side)

    assert not dropped(lambda: L.inputs(300, 256, 4100, torch.bfloat16), both)


def test_norm_inputs_dropped_after_the_call():
    hd = N.head(700, 2048, torch.bfloat16)

    def both(side, x, w, b, dy):
        _, mean, rstd = hd.norm(x, w, b, stream=side)
        hd.norm_backward(dy, x, w, mean, rstd, stream=side)

    assert not dropped(lambda: N.inputs(700, 2048, torch.bfloat16, torch.bfloat16), both)


@pytest.mark.parametrize("bits", (32, 8))
def test_optimiser_dropped_after_the_step(bits):
    from gemmaedge_amd import head as H

    def make():
        return [torch.zeros(700_000 + 5 * i, device="cuda") for i in range(2)]

    def step(side, p, g):
        opt = H.AdamW([p[:600_000]], [g[:600_000]], state_bits=bits)
        side.wait_stream(torch.cuda.current_stream())
        opt.step(stream=side)

    assert not dropped(make, step)


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
