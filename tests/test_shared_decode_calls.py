"""Calls of shared decode attention beside those of a serving step: what is refused, long batches, plans."""

import pytest
import torch
from torch.autograd import forward_ad

from opsagent_amd import ops

gpu = pytest.mark.gpu
DEVICE = "cuda" if torch.cuda.is_available() else "cpu"


def _small():
    gen = torch.Generator().manual_seed(1)
    caches = [torch.randn(6, 8, 2, 64, generator=gen).to(DEVICE, torch.bfloat16) for _ in range(2)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEVICE)  # noqa: E731
    return dict(q=torch.randn(2, 4, 64, generator=gen).to(DEVICE, torch.bfloat16), k_cache=caches[0],
                v_cache=caches[1], block_table=i32([[0, 1, 2], [0, 3, 4]]), seq_lens=i32([20, 13]),
                leaders=i32([0, 0]), shared=i32([1, 1]))


@pytest.mark.parametrize("name", ["q", "k_cache", "v_cache"])
def test_gradients_of_either_mode_are_refused(name):
    """On the CPU as on the GPU: nothing is left out of a derivative without an error."""
    c = _small()
    want = ops.attention_decode_shared(**c)
    leaf = {**c, name: c[name].clone().requires_grad_()}
    with pytest.raises(RuntimeError, match="gradients"):
        ops.attention_decode_shared(**leaf)
    with torch.no_grad():
        assert torch.equal(ops.attention_decode_shared(**leaf), want)
    with forward_ad.dual_level():
        dual = {**c, name: forward_ad.make_dual(c[name], torch.ones_like(c[name]))}
        with pytest.raises(RuntimeError, match="gradients"):
            ops.attention_decode_shared(**dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="gradients"):
            ops.attention_decode_shared(**dual)
        assert torch.equal(ops.attention_decode_shared(**c), want)
