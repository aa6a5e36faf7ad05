"""What a failed creation leaves behind."""
import pytest
import torch

import test_gpu_head_loss as L

pytestmark = pytest.mark.gpu


def test_a_handle_that_does_not_fit_leaves_no_error_behind():
    from gemmaedge_amd import head as H
    from gemmaedge_amd import sampler as S

    h, w, t, grad = L.inputs(8, 64, 300, torch.bfloat16)
    p, g = torch.zeros(300, device="cuda"), torch.zeros(300, device="cuda")
    hd, opt = H.Head(8, 64, 300, train=True), H.AdamW([p], [g])
    nw = torch.ones(64, device="cuda")

    def calls():
        hd.norm(h, nw)
        loss, lse = hd.loss(h, w, t)
        hd.loss_backward(grad, h, w, t, lse)
        opt.step()

    calls()
    for call in (lambda: hd.norm(h, nw), lambda: hd.loss(h, w, t), opt.step):
        with pytest.raises(S.SamplerError) as e:
            H.Head(1 << 22, 65536, 8)  # 550 GB of packed hidden states
        assert e.value.code == S.GE_ERR_DEVICE
        call()
    calls()
    torch.cuda.synchronize()
