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


@pytest.mark.parametrize("compute", ["int8", "fp16"])
def test_two_moves_with_another_bias(cuda, compute):
    from rpfq_review_b200 import PackedPhaseLinear
    from rpfq_review_b200.packing import random_packed
    layer, x = PackedPhaseLinear.from_packed(random_packed(96, 64, seed=0, device=cuda), compute=compute), _x()
    layer.bias.zero_()
    y = layer(x)
    for step in (1.0, 2.0, 4.0, 8.0):
        layer.cpu()
        layer.bias.fill_(step)
        layer.to(cuda)
        # y + step in fp32 rounds once more than the epilogue: 2^-24 of values below 256
        assert (layer(x) - (y + step)).abs().max() <= 2.0 ** -14, step


def test_first_call_inside_a_capture(cuda):
    """A layer whose first call is captured: eager calls before the first replay have their own
    codes and bias, and the replay follows planes loaded after the capture."""
    layer, x = _layer(1), _x()
    want = _layer(1)(x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = layer(x)
    assert torch.equal(layer(x), want)
    g.replay()
    assert torch.equal(y, want)
    layer.load_state_dict(_layer(2).state_dict())
    g.replay()
    assert torch.equal(y, _layer(2)(x)) and torch.equal(layer(x), y)
