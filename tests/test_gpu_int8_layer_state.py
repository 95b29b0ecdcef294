"""GPU tests of what an 8-bit layer keeps between calls: it answers with its planes and bias as
they are, whatever happened to the module since the last call."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _layer(seed, **kw):
    from rpfq_review_b200 import PackedPhaseLinear
    from rpfq_review_b200.packing import random_packed
    return PackedPhaseLinear.from_packed(random_packed(96, 64, seed=seed, device="cuda"), compute="int8", **kw)


def _x(rows=5):
    return torch.randn(rows, 128, generator=torch.Generator().manual_seed(0)).to("cuda")


def test_two_moves_with_other_planes(cuda):
    """Off, loaded, back on, run, again and again: the allocator hands the same addresses out."""
    layer, x = _layer(0), _x()
    layer(x)
    for seed in (1, 2, 3, 4):
        layer.cpu()
        other = _layer(seed)
        planes = {k: v.cpu() for k, v in other.state_dict().items() if k != "bias"}
        layer.load_state_dict(planes, strict=False)
        layer.to(cuda)
        other.bias.copy_(layer.bias)
        assert torch.equal(layer(x), other(x)), seed
