"""How the block operators' calls take their arguments (no GPU: the checks run before any launch)."""
import inspect

import pytest
import torch

from subq_audio import ops

CALLS = ["causal_conv_forward", "causal_conv_backward", "selective_scan_forward", "selective_scan_backward", "rms_norm", "rms_norm_fp8", "quantize_fp8",
         "rms_norm_backward", "scaled_matmul"]


@pytest.mark.parametrize("name", CALLS)
def test_every_argument_has_its_name(name):
    """A call by names gets as far as the same call by places: the refusal of CPU tensors."""
    call = getattr(ops, name)
    params = inspect.signature(call).parameters
    need = [k for k, p in params.items() if p.default is p.empty]
    x = torch.zeros(2, 8, 4)
    with pytest.raises(RuntimeError) as by_place:
        call(*[x for _ in need])
    with pytest.raises(RuntimeError) as by_name:
        call(**{k: x for k in need})
    assert str(by_name.value) == str(by_place.value)
    with pytest.raises((TypeError, RuntimeError)):
        call(x, **{k: x for k in need})  # the first one twice
    with pytest.raises(TypeError):
        call()
