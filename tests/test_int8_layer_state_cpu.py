"""What an 8-bit layer keeps between calls, on the CPU: the decoder, the row quantizer and the
product are stand-ins on CPU tensors (the layer's own bookkeeping is the tested code)."""

import copy
import pickle

import numpy as np
import pytest
import torch

from rpfq_review_b200 import PackedPhaseLinear, layers, ops
from rpfq_review_b200.packing import random_packed


@pytest.fixture
def calls(monkeypatch):
    """Stand-ins: the "dense matrix" is the first plane's codes as fp32, its "codes" their low
    seven bits, and the product returns the codes, scales and bias that the layer passes."""
    made = []

    def prepack(packed, rounding="rne"):
        made.append(1)
        return packed.planes["u_s0"][0].float()

    monkeypatch.setattr(ops, "prepack", prepack)
    monkeypatch.setattr(ops, "quantize_rows", lambda w: ((w % 128).to(torch.int8), w.amax(1).float()))
    monkeypatch.setattr(ops, "linear_int8", lambda x, w, w_scale, bias, *more: (w.clone(), w_scale.clone(), bias.clone()))
    return made


def _layer(seed=0, **kw):
    return PackedPhaseLinear.from_packed(random_packed(8, 8, seed=seed), compute="int8", **kw)


def _run(layer):
    return layer(torch.zeros(1, layer.in_features))


def _same(got, layer):
    w = layer.u_s0.codes.float()
    return torch.equal(got[0], (w % 128).to(torch.int8)) and torch.equal(got[1], w.amax(1))


class Pool:
    """An allocator that hands the same addresses out again: a tensor moved to it lands where the
    tensor of that name landed before (its memory there is taken to be free)."""

    def __init__(self):
        self.memory = {}

    def move(self, module):
        for name, plane in module.named_modules():
            for key, t in list(plane._buffers.items()):
                if t is None:
                    continue
                at = self.memory.setdefault((name, key), np.empty(t.numel() * t.element_size() + 64, np.uint8))
                new = torch.from_numpy(at[: t.numel() * t.element_size()]).view(t.dtype).view(t.shape)
                at[: t.numel() * t.element_size()] = t.detach().contiguous().view(-1).view(torch.uint8).numpy()
                plane._buffers[key] = new


def test_codes_follow_planes_that_move_over_the_same_addresses(calls):
    """Off, loaded, back on, run, twice: the second time the planes lie where they lay, in new
    tensors of the same version."""
    layer, pool = _layer(), Pool()
    for seed in (1, 2, 3):
        other = _layer(seed)
        for name, t in layer.named_buffers():
            if name.endswith(("codes", "gamma_real", "gamma_imag")):
                t.copy_(dict(other.named_buffers())[name])
        pool.move(layer)
        assert _same(_run(layer), layer), f"codes of older planes with seed {seed}"
        before = len(calls)
        assert _same(_run(layer), layer)
        assert len(calls) == before, "unchanged planes are not decoded again"


def test_codes_follow_writes_casts_and_assignments(calls):
    layer = _layer()
    _run(layer)
    layer.u_s0.codes.add_(1)
    assert _same(_run(layer), layer)
    layer.u_s0.codes = layer.u_s0.codes.clone().add_(3)
    assert _same(_run(layer), layer)
    layer.u_s0.codes.data = layer.u_s0.codes.clone().add_(5)
    assert _same(_run(layer), layer)
    layer.load_state_dict(_layer(4).state_dict())
    assert _same(_run(layer), layer)
    layer.load_state_dict(_layer(5).state_dict(), assign=True)
    assert _same(_run(layer), layer)
    layer.half()
    got = _run(layer)
    assert _same(got, layer) and got[1].dtype == torch.float32


def test_bias_follows_moves_over_the_same_addresses(calls):
    layer, pool = _layer(), Pool()
    for step in (1, 2, 3):
        layer.bias.fill_(step)
        pool.move(layer)
        assert (_run(layer)[2] == step).all()
    layer.bias.fill_(7)
    assert (_run(layer)[2] == 7).all()


def test_nothing_made_inside_a_capture_is_kept(calls, monkeypatch):
    """What a captured call makes is written when its graph is replayed, into the graph's memory."""
    layer = _layer()
    monkeypatch.setattr(layers, "_capturing", lambda t: True)
    assert _same(_run(layer), layer) and layer.codes8 is None and layer._bias32 is None
    layer.prepack()
    assert layer.codes8 is None
    monkeypatch.undo()


def test_codes_keep_their_memory(calls):
    """New planes of the same shape are quantized into the tensors that graphs may read."""
    layer = _layer()
    _run(layer)
    layer.bias.fill_(1)
    _run(layer)
    kept = layer.codes8, layer.scale8, layer._bias_f32()
    layer.u_s0.codes.add_(1)
    layer.bias.fill_(2)
    assert _same(_run(layer), layer)
    assert all(a is b for a, b in zip(kept, (layer.codes8, layer.scale8, layer._bias_f32()))) and (kept[2] == 2).all()


def test_layer_made_in_inference_mode(calls):
    """Its planes keep no version: calls run, in and outside of the mode, and loads are followed."""
    with torch.inference_mode():
        layer = _layer(1)
        assert _same(_run(layer), layer)
    assert _same(_run(layer), layer) and len(calls) == 1
    for seed in (2, 3):
        with torch.inference_mode():
            layer.load_state_dict(_layer(seed).state_dict())
            layer.bias.fill_(seed)
        got = _run(layer)
        assert _same(got, layer) and (got[2] == seed).all()
    outside = _layer(4)
    with torch.inference_mode():
        assert _same(_run(outside), outside)
    outside.u_s0.codes.add_(1)
    outside.bias.fill_(9)
    got = _run(outside)
    assert _same(got, outside) and (got[2] == 9).all()


def test_copies_make_their_own_codes(calls):
    layer = _layer(1)
    _run(layer)
    for other in (copy.deepcopy(layer), pickle.loads(pickle.dumps(layer))):
        other.u_s0.codes.add_(1)
        other.bias.fill_(3)
        got = _run(other)
        assert _same(got, other) and (got[2] == 3).all()
        assert _same(_run(layer), layer) and layer._bias_f32().ne(3).any()


def test_prepack_after_writes_that_raise_no_version(calls):
    layer = _layer(1)
    _run(layer)
    layer.u_s0.codes.data.add_(1)
    layer.bias.data.fill_(5)
    layer.prepack()
    got = _run(layer)
    assert _same(got, layer) and (got[2] == 5).all()


def test_fp32_bias_stays_the_callers(calls):
    """A bias that is fp32 already is copied, not kept itself and written over later."""
    layer = _layer(1)
    first = torch.full((16,), 2.0)
    layer.bias = first
    assert (_run(layer)[2] == 2).all()
    layer.bias = torch.full((16,), 3.0)
    assert (_run(layer)[2] == 3).all() and (first == 2).all()
    layer.bias.fill_(4)
    assert (_run(layer)[2] == 4).all()
    version, kept = layer.bias._version, layer._bias32
    assert (_run(layer)[2] == 4).all() and layer.bias._version == version and layer._bias32 is kept
