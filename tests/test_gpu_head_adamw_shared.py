"""AdamW refuses tensors that share memory which a step writes: two workgroups would
update it at once."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def tensors(n=3, size=600):
    return [torch.zeros(size, device="cuda") for _ in range(n)]


def test_memory_that_is_shared():
    from gemmaedge_amd import head as H

    p, g, z = tensors(), tensors(), tensors(1, 2000)[0]
    codes = torch.zeros(600, dtype=torch.float8_e4m3fn, device="cuda")
    for bad in (lambda: H.AdamW([p[0], p[1], p[0]], g), lambda: H.AdamW([z[:600], z[599:1199], p[0]], g),
                lambda: H.AdamW([z[:1200], z[300:600]], [z.new_zeros(1200), g[0][:300]]), lambda: H.AdamW(p, [g[0], g[1], p[1]]),
                lambda: H.AdamW(p, g, masters=[None, p[0], None]), lambda: H.AdamW(p, g, masters=[None, z[:600], z[10:610]]),
                lambda: H.AdamW(p, g, m=[z[:600], z[600:1200], z[1199:1799]]), lambda: H.AdamW(p, g, m=tensors(), v=p),
                lambda: H.AdamW(p, g, state_bits=8, m=[codes] * 3),
                lambda: H.AdamW(p, g, state_bits=8, m_scale=[z[:3], z[3:6], z[6:9]], v_scale=[z[8:11], z[11:14], z[14:17]])):
        with pytest.raises(ValueError, match="shares memory"):
            bad()


def test_memory_that_may_be_shared():
    from gemmaedge_amd import head as H

    p, g, z = tensors(), tensors(), tensors(1, 4000)[0]
    H.AdamW([z[:600], z[600:1200], z[1200:1800]], [g[0], g[0], g[0]], m=[z[1800:2400], z[2400:3000], z[3000:3600]])
    H.AdamW([z[:0], z[:600], z[300:300]], [z[:0], g[0], z[5:5]])
    g[0].fill_(1.0)
    opt = H.AdamW(p, g, masters=[p[0], None, None], lr=0.5, weight_decay=0.0)  # its own master
    opt.step()
    assert ((p[0] + 0.5).abs() < 1e-6).all()
