"""A call of more tiles than one launch's 2^32 threads: 2^20 rows over a vocabulary of
2^20 words. Rows do not depend on the batch that they come in."""
import pytest
import torch

import test_gpu_head_loss as L

pytestmark = pytest.mark.gpu


def test_more_tiles_than_a_launch():
    from gemmaedge_amd import head as H

    n = 1 << 20
    h, w, t, _ = L.inputs(n, 8, n, torch.bfloat16, seed=3)
    hd = H.Head(n, 8, n)
    loss, lse = torch.full((n,), -7.0, device="cuda"), torch.full((n,), -7.0, device="cuda")
    hd.loss(h, w, t, loss=loss, lse=lse)
    for at in (0, n // 2 - 100, n - 300):
        some = slice(at, at + 300)
        want_loss, want_lse = hd.loss(h[some], w, t[some].contiguous())
        ref = torch.logsumexp(h[some].double() @ w.double().t(), 1)
        assert ((want_lse.double() - ref).abs() < 1e-4).all()
        assert ((lse[some] - want_lse).abs() < 1e-5).all() and ((loss[some] - want_loss).abs() < 2e-5).all()
