"""The norm's mean without centring: a buffer that is passed in for it does not turn the
backward pass into that of the centred norm. References and tolerances are those of the
norm's own tests (float64)."""
import pytest
import torch

import test_gpu_head_norm as N

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("center", (True, False))
@pytest.mark.parametrize("dt", ("bf16", "f32"))
@pytest.mark.parametrize("rows,dim", [(3, 40), (20, 1152), (5, 8200)])
def test_a_buffer_for_the_mean(rows, dim, dt, center):
    x, w, b, dy = N.inputs(rows, dim, N.DT[dt], torch.float32, seed=dim)
    h = N.head(rows, dim, N.DT[dt])
    buf = torch.full((rows,), 9.0, device="cuda")
    y, mean, rstd = h.norm(x, w, b, eps=1e-5, center=center, mean=buf)
    assert mean is (buf if center else None)
    dx, dw, db = h.norm_backward(dy, x, w, mean, rstd, bias=True)
    ref = N.reference(x, w, b, dy, 1e-5, center)
    for k, got in dict(y=y, mean=buf, rstd=rstd, dx=dx, dw=dw, db=db).items():
        N.close(got, ref[k], k)
