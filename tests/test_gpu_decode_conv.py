"""Pools of stacks whose convolutions do not have four taps: tokens and beams go on them, prompts are refused before anything is written."""
import pytest
import torch
from torch import nn

from tests.helpers import RefShapedBlock
from tests.test_gpu_decode import DEV, Norm, close, cu_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d_conv", [2, 3, 5, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tokens_but_no_prompts(d_conv, dtype):
    import types
    import mamba_b200
    from mamba_b200 import mamba
    torch.manual_seed(d_conv)
    layer = nn.Module()
    layer.mixer, layer.norm = RefShapedBlock(32, d_conv=d_conv), Norm(32, torch.Generator().manual_seed(1))
    s = types.SimpleNamespace(layers=nn.ModuleList([layer]).to(DEV, dtype))
    pool = mamba_b200.StatePool(s, 5, dtype=dtype)
    slots = torch.tensor([3, 0, 9], device=DEV)
    with pytest.raises(RuntimeError, match="d_conv 4"):
        pool.prompts(torch.randn(6, 32, device=DEV, dtype=dtype), cu_of([2, 3, 1]), slots)
    assert not any(t.any() for t in pool.pools())
    cache = (None, torch.zeros(2, 64, d_conv - 1, dtype=dtype, device=DEV))
    with torch.no_grad():
        for _ in range(2 * d_conv):
            x = torch.randn(3, 32, device=DEV, dtype=dtype)
            y = pool.step(x, slots)
            normed = mamba_b200.rms_norm(x[:2], layer.norm.weight, layer.norm.eps)
            want, cache = mamba.step(layer.mixer, normed, cache)
            # sums in another order; in bfloat16 five values on the way (both halves of in_proj, delta, y, the output) may each round the other way, 2^-8
            # of their size, and the sum with x once more
            bound = (1e-4 if dtype == torch.float32 else 6 * 2 ** -8) * (want + x[:2]).abs().max()
            assert ((y[:2] - (want + x[:2])).abs() <= bound).all()
        pool.reorder(torch.tensor([[3, 0]], device=DEV), torch.tensor([[1, 1]], device=DEV))
    states, windows = pool.caches[0]
    assert torch.equal(states[3], states[0]) and torch.equal(windows[3], windows[0]) and not states[[1, 2, 4]].any()
