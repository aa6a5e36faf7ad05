"""Parameters of an optimiser step in device memory pass the checks that the host's pass,
before they are copied: the launch that reads them has no way to refuse them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_parameters_for_the_device_are_checked():
    from gemmaedge_amd import head as H
    from gemmaedge_amd import sampler as S

    p, g = torch.zeros(300, device="cuda"), torch.ones(300, device="cuda")
    opt = H.AdamW([p], [g])
    hp = opt.device_params()
    before = hp.clone()
    for kw in (dict(lr=float("inf")), dict(lr=float("nan")), dict(grad_scale=float("nan"))):
        with pytest.raises(S.SamplerError) as e:
            opt.device_params(out=hp, **kw)
        assert e.value.code == S.GE_ERR_INVALID_ARG
    opt.beta2 = 1.0
    with pytest.raises(S.SamplerError):
        opt.device_params()
    opt.beta2 = 0.999
    for out in (torch.empty(56, device="cuda"), hp[:55], torch.empty(56, dtype=torch.uint8), torch.empty(112, dtype=torch.uint8, device="cuda")[::2]):
        with pytest.raises(ValueError):
            opt.device_params(out=out)
    assert opt.steps == 1 and torch.equal(hp, before)
    opt.device_params(out=hp)
    opt.step(device_params=hp)
    assert opt.steps == 2 and (p < 0).all()
