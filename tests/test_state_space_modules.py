"""What the state space modules refuse when they are made (no GPU)."""
import pytest
import torch

from subq_audio import SubQFp8Linear, SubQRMSNorm, SubQSelectiveStateSpace, SubQStateSpaceBlock


@pytest.mark.parametrize("k", [{"state_size": 0}, {"state_size": 129}, {"conv_width": 1}, {"conv_width": 5}, {"groups": 0}, {"groups": 7}, {"dt_min": 0.0},
                               {"dt_min": 0.2, "dt_max": 0.1}])
def test_shapes_that_no_kernel_takes(k):
    with pytest.raises(ValueError):
        SubQSelectiveStateSpace(64, **k)


def test_norm_widths():
    for n in (0, 16385):
        with pytest.raises(ValueError):
            SubQRMSNorm(n)


def test_quantised_widths():
    for n, m in ((0, 4), (16385, 4), (4, 0)):
        with pytest.raises(ValueError):
            SubQFp8Linear(n, m)


def test_quantised_weights_stay_bytes():
    m = SubQStateSpaceBlock(64).quantize()
    lin = m.mixer.in_proj
    assert isinstance(lin, SubQFp8Linear) and isinstance(m.mixer.out_proj, SubQFp8Linear)
    before = lin.weight_bytes.clone(), lin.scale_bytes.clone()
    m.to(torch.bfloat16)
    assert torch.equal(lin.weight_bytes, before[0]) and torch.equal(lin.scale_bytes, before[1])
    assert m.quantize().mixer.in_proj is lin
    back = lin.weight_bytes.view(torch.float8_e4m3fn)[:, :64].float() * lin.scale_bytes.view(torch.float32)[0, 0]
    assert back.shape == (256, 64) and float(back.abs().max()) > 0
    # step sizes start between dt_min and dt_max
    size = torch.nn.functional.softplus(SubQSelectiveStateSpace(64).dt_bias)
    assert 0.0009 < float(size.min()) and float(size.max()) < 0.101
