"""CPU tests of the 8-bit linear path and the rotary positions: the C entry
points reject bad arguments before any device work, the Python entry points
reject what they can see without a GPU, and the host-side tables are right."""

import ctypes
import math

import pytest
import torch

from rpfq_review_b200 import PackedPhaseLinear, _lib, ops
from rpfq_review_b200.packing import random_packed
from rpfq_review_b200.vit import DEIT_S16, VIT_B16, PackedViT, grid_positions

A = 4096  # a 16-byte aligned address; nothing is read


def test_struct_sizes():
    assert ctypes.sizeof(_lib.RpfqGemmI8Args) == 8 * 12 + 4 * 6 + 8 * 2
    assert ctypes.sizeof(_lib.RpfqRotaryArgs) == 8 * 13 + 4 * 10


def _gemm(**kw):
    a = dict(x=A, ldx=64, x_scale=A, w=A, ldw=64, w_scale=A, bias=None, residual=None, ldr=0, y=2 * A, ldy=32, m=4, n=32,
             k=60, activation=0, flags=0)
    a.update(kw)
    return _lib.lib().rpfq_gemm_i8_sm100(ctypes.byref(_lib.RpfqGemmI8Args(**a)), None)


@pytest.mark.parametrize("bad", [
    dict(m=-1), dict(n=0), dict(k=0), dict(k=-4), dict(x=None), dict(w=None), dict(y=None), dict(x_scale=None),
    dict(w_scale=None), dict(ldx=48), dict(ldx=72), dict(ldw=48), dict(ldw=60), dict(x=A + 8), dict(w=A + 1),
    dict(ldy=31), dict(residual=A, ldr=31), dict(y=2 * A + 1), dict(y=2 * A + 2, flags=1), dict(bias=A + 1),
    dict(bias=A + 2, flags=4), dict(residual=A + 1, ldr=32), dict(x_scale=A + 2), dict(w_scale=A + 1),
    dict(flags=32), dict(flags=24), dict(activation=2), dict(activation=-1),
    dict(block_n=96), dict(block_n=-1), dict(split_k=9), dict(split_k=-1), dict(block_n=256, split_k=2),
    dict(flags=8, x=A + 1), dict(flags=16, x=A + 2), dict(flags=8, ldx=59), dict(flags=8, m=9),
    dict(flags=8, m=9, scratch=A + 4, scratch_bytes=1 << 20), dict(flags=8, m=9, scratch=A, scratch_bytes=9 * 68 - 1)])
def test_gemm_i8_rejects(bad):
    assert _gemm(**bad) == _lib.RPFQ_ERR_INVALID
    assert _lib.lib().rpfq_last_error()


def test_gemm_i8_refuses_an_output_over_its_input():
    """x [4, 60] int8 at A, rows of 64 bytes: y over its range, its tail, around it; columns
    beside x in rows of the same stride pass this check (and fail later, without a GPU)."""
    for y, ldy, n in ((A, 32, 32), (A + 192, 32, 32), (A - 64, 32, 8), (A + 56, 32, 8), (A + 30, 32, 4)):
        assert _gemm(y=y, ldy=ldy, n=n) == _lib.RPFQ_ERR_INVALID
        assert b"overlap" in _lib.lib().rpfq_last_error()
    wide = dict(ldx=128, ldy=64)  # rows of 128 bytes: x in the first 60, y in the last 64
    for y, n in ((A + 64, 32), (A + 60, 34)):
        assert _gemm(y=y, n=n, **wide) == _lib.RPFQ_OK or b"overlap" not in _lib.lib().rpfq_last_error()
    assert _gemm(y=A + 64, n=33, **wide) == _lib.RPFQ_ERR_INVALID and b"overlap" in _lib.lib().rpfq_last_error()
    assert _gemm(y=A + 58, n=8, **wide) == _lib.RPFQ_ERR_INVALID and b"overlap" in _lib.lib().rpfq_last_error()


def test_gemm_i8_unsupported_and_empty():
    assert _gemm(k=131072, ldx=131072, ldw=131072) == _lib.RPFQ_ERR_UNSUPPORTED
    assert b"131071" in _lib.lib().rpfq_last_error()
    assert _gemm(m=2 ** 31) == _lib.RPFQ_ERR_UNSUPPORTED
    assert _gemm(residual=A, ldr=32, flags=1) == _lib.RPFQ_ERR_UNSUPPORTED  # fp16 residual, fp32 output
    assert _gemm(residual=A, ldr=32, flags=2) == _lib.RPFQ_ERR_UNSUPPORTED
    # few rows are quantized inside the launch: no scratch
    assert [_lib.lib().rpfq_gemm_i8_scratch_bytes(m, 60) for m in (0, 1, 8, 9)] == [0, 0, 0, 9 * 68]
    assert _lib.lib().rpfq_gemm_i8_scratch_bytes(8, 100000) == 8 * 100004
    assert _gemm(m=0, x=None, y=None, x_scale=None) == _lib.RPFQ_OK
    assert _lib.lib().rpfq_gemm_i8_sm100(None, None) == _lib.RPFQ_ERR_INVALID


@pytest.mark.parametrize("bad", [dict(m=-1), dict(k=0), dict(x=None), dict(q=None), dict(scale=None), dict(ldx=7),
                                 dict(ldq=7), dict(x=A + 1), dict(x=A + 2, f32=1), dict(scale=A + 2)])
def test_quantize_rows_rejects(bad):
    a = dict(x=A, f32=0, ldx=8, q=A, ldq=8, scale=A, m=2, k=8)
    a.update(bad)
    L = _lib.lib()
    assert L.rpfq_quantize_rows_sm100(a["x"], a["f32"], a["ldx"], a["q"], a["ldq"], a["scale"], a["m"], a["k"],
                                      None) == _lib.RPFQ_ERR_INVALID
    assert L.rpfq_quantize_rows_sm100(None, 0, 0, None, 0, None, 0, 8, None) == _lib.RPFQ_OK


def _rotary(**kw):
    a = dict(x=A, x_batch=640, x_token=128, x_head=64, y=2 * A, y_batch=640, y_token=128, y_head=64, positions=A,
             position_batch=0, inv_freq=A, batch=2, length=5, heads=2, dim=64, pairs=32, axes=1, position_type=0,
             f32=0, interleaved=0, transpose=0, magnitude=1.0)
    a.update(kw)
    return _lib.lib().rpfq_rotary_sm100(ctypes.byref(_lib.RpfqRotaryArgs(**a)), None)


@pytest.mark.parametrize("bad", [
    dict(batch=-1), dict(length=-1), dict(heads=-1), dict(dim=0), dict(pairs=0), dict(pairs=33), dict(pairs=-1),
    dict(axes=0), dict(axes=3), dict(axes=2, pairs=31), dict(position_type=4), dict(position_type=-1), dict(x=None),
    dict(y=None), dict(positions=None), dict(inv_freq=None), dict(x=A + 1), dict(y=A + 2, f32=1),
    dict(positions=A + 2), dict(positions=A + 4, position_type=1), dict(inv_freq=A + 4),
    dict(y=A, y_token=256), dict(y=A, y_head=128), dict(y=A, y_batch=0)])
def test_rotary_rejects(bad):
    assert _rotary(**bad) == _lib.RPFQ_ERR_INVALID
    assert _lib.lib().rpfq_last_error()


def test_rotary_unsupported_and_empty():
    assert _rotary(dim=8192, pairs=2049) == _lib.RPFQ_ERR_UNSUPPORTED
    assert _rotary(heads=(1 << 24) + 1) == _lib.RPFQ_ERR_UNSUPPORTED
    for empty in (dict(batch=0), dict(length=0), dict(heads=0)):
        assert _rotary(x=None, y=None, positions=None, inv_freq=None, **empty) == _lib.RPFQ_OK


def test_python_entries_refuse_cpu_tensors_and_types():
    x8, s = torch.zeros(2, 16, dtype=torch.int8), torch.ones(2)
    for call in (lambda: ops.gemm_int8(x8, s, x8, s), lambda: ops.linear_int8(torch.zeros(2, 16), x8, s),
                 lambda: ops.quantize_rows(torch.zeros(2, 16)),
                 lambda: ops.rotary(torch.zeros(2, 1, 4), torch.zeros(2), torch.zeros(2, dtype=torch.float64))):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_rotary_frequencies_refusals():
    for kw in (dict(rot_dim=0), dict(rot_dim=7), dict(rot_dim=6, axes=2), dict(rot_dim=8, axes=3),
               dict(rot_dim=8, base=0.0), dict(rot_dim=8, factor=0.5), dict(rot_dim=8, scaling="cubic"),
               dict(rot_dim=2, scaling="base", factor=2.0), dict(rot_dim=8, scaling="parts", factor=2.0),
               dict(rot_dim=8, scaling="parts", original_length=64, low=4.0, high=4.0)):
        with pytest.raises(ValueError):
            ops.rotary_frequencies(**kw)


def test_rotary_frequencies_values():
    f, mag = ops.rotary_frequencies(64)
    assert mag == 1.0 and f.dtype == torch.float64
    assert all(math.isclose(f[j].item(), 10000.0 ** (-2 * j / 64), rel_tol=1e-14) for j in range(32))
    assert torch.equal(ops.rotary_frequencies(64, scaling="linear", factor=4)[0], f / 4)
    b = ops.rotary_frequencies(64, scaling="base", factor=8)[0]
    assert b[0] == 1.0 and math.isclose(b[-1].item(), f[-1].item() / 8, rel_tol=1e-12)
    p, mag = ops.rotary_frequencies(64, scaling="parts", factor=8, original_length=4096)
    assert math.isclose(mag, 0.1 * math.log(8) + 1) and p[0] == f[0] and math.isclose(p[-1].item(), f[-1].item() / 8)
    turns = 4096 * f / (2 * math.pi)
    inside = (turns > 1) & (turns < 32)
    assert inside.any() and ((p[inside] < f[inside]) & (p[inside] > f[inside] / 8)).all()
    two = ops.rotary_frequencies(64, 100.0, axes=2)[0]
    assert torch.equal(two[:16], two[16:]) and torch.equal(two[:16], ops.rotary_frequencies(32, 100.0)[0])


def test_grid_positions():
    for cfg, prefix in ((VIT_B16, 1), (DEIT_S16, 2)):
        at = grid_positions(cfg)
        assert at.shape == (cfg.tokens, 2) and at.dtype == torch.int32
        assert torch.count_nonzero(at[:prefix]) == 0
        assert at[prefix + 14 * 3 + 5].tolist() == [3, 5] and at[-1].tolist() == [13, 13]


def test_layer_and_model_refusals():
    layer = random_packed(8, 8, seed=0)
    for kw, word in ((dict(compute="int4"), "compute"), (dict(compute="int8", enable_act_quant=True), "act_quant"),
                     (dict(compute="int8", cache_dense=False), "cache_dense")):
        with pytest.raises(ValueError, match=word):
            PackedPhaseLinear.from_packed(layer, **kw)
    with pytest.raises(ValueError, match="act_bits"):
        PackedViT(VIT_B16, "cpu", compute="int8", act_bits=4)
    assert "compute=int8" in repr(PackedPhaseLinear.from_packed(layer, compute="int8"))
