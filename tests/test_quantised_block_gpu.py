"""Quantised blocks as they come: nothing set by hand, whatever type the module had before and gets after.

Tolerance as in test_state_space_gpu: 0.1 for two projections of 8 bits (4 significant bits of inputs and weights), and 3e-2 where the
tensors between the operators have 16 bits.
"""
import pytest
import torch

from subq_audio import SubQRMSNorm, SubQStateSpaceBlock
from subq_audio.cache import run_layers
from test_state_space_gpu import rel

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def stack(seed=2):
    torch.manual_seed(seed)
    return torch.nn.ModuleList([SubQStateSpaceBlock(256) for _ in range(2)]).cuda(), SubQRMSNorm(256).cuda()


@pytest.mark.parametrize("before", [F32, F16, BF16])
@pytest.mark.parametrize("after", [None, F32, F16, BF16])
def test_types_before_and_after(before, after):
    blocks, last = stack()
    kind = before if after is None else after
    x = torch.randn(2, 40, 256, device="cuda", dtype=kind)
    with torch.no_grad():
        want = last(*run_layers(blocks, x.float())[0])[0]
        blocks.to(before)
        for b in blocks:
            b.quantize()
        if after is not None:
            blocks.to(after)
        (branch, stream), states = run_layers(blocks, x)
        assert branch.dtype == stream.dtype == kind
        assert rel(last(branch, stream)[0], want) < 0.1 + (3e-2 if F16 in (before, kind) or BF16 in (before, kind) else 0)
        # prompts, then single tokens
        pair, st = run_layers(blocks, x[:, :39])
        pair, st = run_layers(blocks, x[:, 39:], past_key_values=st)
        assert pair[0].dtype == kind and rel(last(*pair)[0], want[:, 39:]) < 0.1 + (3e-2 if F16 in (before, kind) or BF16 in (before, kind) else 0)


@pytest.mark.parametrize("auto", [F16, BF16])
def test_under_autocast(auto):
    blocks, last = stack()
    x = torch.randn(2, 40, 256, device="cuda")
    with torch.no_grad():
        want = last(*run_layers(blocks, x)[0])[0]
        for b in blocks:
            b.quantize()
        with torch.autocast("cuda", auto):
            (branch, stream), _ = run_layers(blocks, x)
            assert branch.dtype == auto and stream.dtype == F32
            assert rel(last(branch, stream)[0], want) < 0.1 + 3e-2
