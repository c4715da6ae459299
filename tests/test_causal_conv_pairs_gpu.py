"""The convolution's backward at channel counts that go in fours, in twos and not at all, with and without masks.

Tolerances as in test_causal_conv_gpu (3e-6 for gradients, half a step of a rounded one).
"""
import pytest
import torch

from subq_audio import ops
from test_causal_conv_gpu import BWD, T, definition, half, inputs, rel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("D", [64, 66, 126, 127])
def test_channels_in_twos(D, W, dtype):
    x, w, b, S, dout, dS = inputs(3, 150, D, W, dtype)
    mask = torch.arange(150)[None, :] < torch.tensor([[150], [33], [0]])
    mask[0, 40:44] = False
    for m in (None, mask.cuda()):
        got = ops.causal_conv_backward(x, w, dout, b, mask=m, state=S, dstate=dS, need_dstate=True)
        for name, a, e in zip(("dx", "dw", "db", "dstate"), got, definition(x, w, b, S, "silu", m, dout, dS)):
            assert rel(a, e) < BWD + half(a.dtype), name
