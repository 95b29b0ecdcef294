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


SLEEP = 40_000_000  # clock cycles: about 20 ms, far longer than what runs beside it


def test_codes_are_ready_for_every_stream(cuda):
    """Made behind other work of one stream, used at once by another."""
    for seed in range(3):
        layer, x, want = _layer(seed), _x(), _layer(seed)(_x())
        a, b = torch.cuda.Stream(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(a):
            torch.cuda._sleep(SLEEP)
            ya = layer(x)
        with torch.cuda.stream(b):
            yb = layer(x)
        torch.cuda.synchronize()
        assert torch.equal(ya, want) and torch.equal(yb, want)


def test_codes_in_use_are_not_overwritten(cuda):
    """Planes loaded while a call on another stream still waits to read the old codes."""
    layer, other, x = _layer(1), _layer(2), _x()
    old, new = layer(x), other(x)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(SLEEP)
        y = layer(x)
    layer.load_state_dict(other.state_dict())
    z = layer(x)
    torch.empty(1 << 24, dtype=torch.uint8, device=cuda).fill_(17)
    torch.cuda.synchronize()
    assert torch.equal(y, old) and torch.equal(z, new)


def test_graph_reads_the_codes_of_loaded_planes(cuda):
    """A captured call reads the kept codes: they stay where they are when planes are loaded."""
    layer, x = _layer(1), _x()
    layer(x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = layer(x)
    for seed in (2, 3):
        layer.load_state_dict(_layer(seed).state_dict())
        want = layer(x)
        noise = [torch.full_like(layer.codes8, 17), torch.full_like(layer.scale8, 3.0), torch.full_like(want[0], 5.0)]
        g.replay()
        assert torch.equal(y, want) and torch.equal(want, _layer(seed)(x)), (seed, len(noise))


def test_layer_made_in_inference_mode(cuda):
    x = _x()
    with torch.inference_mode():
        layer = _layer(1)
        assert torch.equal(layer(x), _layer(1)(x))
        layer.load_state_dict(_layer(2).state_dict())
    assert torch.equal(layer(x), _layer(2)(x))
    with torch.inference_mode():
        layer.load_state_dict(_layer(3).state_dict())
        assert torch.equal(layer(x), _layer(3)(x))
        layer.u_s0.codes.fill_(0)
        layer.prepack()
        other = _layer(3)
        other.u_s0.codes.fill_(0)
        assert torch.equal(layer(x), other(x))


def test_planes_of_other_types_places_and_shapes_are_refused(cuda):
    """A cast module, a plane left on the CPU, one of another size or order: the decoder would
    read their bytes as something else."""
    from rpfq_review_b200 import PackedPhaseLinear
    from rpfq_review_b200.packing import random_packed
    x = _x()
    layer = lambda: PackedPhaseLinear.from_packed(random_packed(96, 64, seed=1, device=cuda), compute="int8")  # noqa: E731
    want = layer()(x)
    for cast in (torch.float32, torch.bfloat16):
        other = layer()
        other.to(cast)
        with pytest.raises(ValueError, match="float16"):
            other(x)
        other.to(torch.float16)
        assert cast == torch.bfloat16 or torch.equal(other(x), want)
    for name, value in (("gamma_real", lambda t: t.cpu()), ("codes", lambda t: t.cpu()), ("codes", lambda t: t[:-1]),
                        ("gamma_imag", lambda t: t[:-1]), ("codes", lambda t: t.t().contiguous().t()),
                        ("codes", lambda t: t.view(torch.int8))):
        other = layer()
        plane = other.w_s1
        plane._buffers[name] = value(plane._buffers[name])
        with pytest.raises(ValueError, match=f"w_s1.{name}"):
            other(x)
