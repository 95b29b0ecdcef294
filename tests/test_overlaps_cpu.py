"""CPU tests: the C entry points of the 8-bit path and the rotary positions refuse outputs over
what they read. Addresses are invented; every call here is refused before any device work."""

import ctypes

import pytest

from rpfq_review_b200 import _lib

MB = 1 << 20


def _gemm(**kw):
    """x [4, 60] in rows of 64, w [32, 60] in rows of 64, y and residual fp16 [4, 32] in rows of
    32, all apart."""
    a = dict(x=MB, ldx=64, x_scale=2 * MB, w=3 * MB, ldw=64, w_scale=4 * MB, bias=5 * MB, residual=6 * MB, ldr=32,
             y=7 * MB, ldy=32, m=4, n=32, k=60, activation=0, flags=0)
    a.update(kw)
    rc = _lib.lib().rpfq_gemm_i8_sm100(ctypes.byref(_lib.RpfqGemmI8Args(**a)), None)
    return rc, _lib.lib().rpfq_last_error()


@pytest.mark.parametrize("bad,word", [
    (dict(y=MB), b"overlap x"), (dict(y=MB - 4 * 64 + 64), b"overlap x"), (dict(y=MB + 4 * 64 - 8), b"overlap x"),
    (dict(y=3 * MB), b"with w"), (dict(y=3 * MB + 31 * 64 + 58), b"with w"), (dict(y=3 * MB - 3 * 64 - 62), b"with w"),
    (dict(y=4 * MB + 126), b"w_scale"), (dict(y=4 * MB - 254), b"w_scale"), (dict(y=2 * MB + 14), b"x_scale"),
    (dict(y=5 * MB + 62), b"bias"), (dict(y=5 * MB + 126, flags=4), b"bias"),
    (dict(y=6 * MB + 2), b"residual"), (dict(y=6 * MB - 64), b"residual"), (dict(y=6 * MB, ldy=40), b"residual"),
    (dict(y=6 * MB + 64), b"residual"), (dict(y=6 * MB, ldr=64, ldy=32), b"residual"),
    (dict(residual=7 * MB + 62, ldr=64, ldy=64), b"residual"), (dict(residual=7 * MB + 66, ldr=64, ldy=64), b"residual"),
    (dict(flags=8, m=9, x_scale=None, scratch=7 * MB, scratch_bytes=MB), b"scratch"),
    (dict(flags=8, m=9, x_scale=None, scratch=MB - 16, scratch_bytes=MB), b"scratch"),
    # w in y's rows of another stride, and the other way round
    (dict(x=MB, y=3 * MB + 60, ldy=64), b"with w"), (dict(w=7 * MB + 64, ldw=128), b"with w")])
def test_gemm_i8_refuses_an_output_over_an_operand(bad, word):
    rc, message = _gemm(**bad)
    assert rc == _lib.RPFQ_ERR_INVALID and word in message, message


def test_gemm_i8_invented_addresses_are_refused():
    """Columns beside x whose rows reach into w (x, w and the scales at one address)."""
    for y, n in ((4096 + 64, 32), (4096 + 60, 34)):
        rc, message = _gemm(x=4096, x_scale=4096, w=4096, w_scale=4096, bias=None, residual=None, ldr=0, y=y, n=n,
                            ldx=128, ldy=64)
        assert rc == _lib.RPFQ_ERR_INVALID and b"with w" in message


def _rotary(**kw):
    """x and y [2, 5, 2, 64] fp16 in rows of 128, apart; positions int32 [5], 32 frequencies."""
    a = dict(x=MB, x_batch=640, x_token=128, x_head=64, y=2 * MB, y_batch=640, y_token=128, y_head=64, positions=3 * MB,
             position_batch=0, inv_freq=4 * MB, batch=2, length=5, heads=2, dim=64, pairs=32, axes=1, position_type=0,
             f32=0, interleaved=0, transpose=0, magnitude=1.0)
    a.update(kw)
    rc = _lib.lib().rpfq_rotary_sm100(ctypes.byref(_lib.RpfqRotaryArgs(**a)), None)
    return rc, _lib.lib().rpfq_last_error()


@pytest.mark.parametrize("bad,word", [
    (dict(y=MB + 2), b"overlap x"), (dict(y=MB + 128), b"overlap x"), (dict(y=MB - 128), b"overlap x"),
    (dict(y=MB + 256), b"overlap x"), (dict(y=MB + 1280), b"overlap x"), (dict(y=MB + 2 * 1280 - 2), b"overlap x"),
    (dict(y=MB - 2 * 1280 + 2), b"overlap x"), (dict(y=MB + 2, x_token=256, x_batch=1280), b"overlap x"),
    (dict(x_token=192, y_token=192, x_batch=960, y_batch=960, y=MB + 128), b"overlap x"),
    (dict(x=MB, y=MB + 130, x_token=128, y_token=128, heads=1), b"overlap x"),
    (dict(y=3 * MB - 2 * 1280 + 2), b"positions"), (dict(y=3 * MB + 18), b"positions"),
    (dict(y=3 * MB + 38, position_batch=5), b"positions"), (dict(y=4 * MB + 254), b"inv_freq"),
    (dict(y=4 * MB - 2 * 1280 + 2), b"inv_freq")])
def test_rotary_refuses_an_output_over_what_it_reads(bad, word):
    rc, message = _rotary(**bad)
    assert rc == _lib.RPFQ_ERR_INVALID and word in message, message


@pytest.mark.parametrize("batch,length", [(2 ** 62 + 1, 4), (2 ** 62, 4), (2 ** 32, 2 ** 32 + 1), (2 ** 31, 1), (1, 2 ** 31),
                                          (2 ** 16, 2 ** 15)])
def test_rotary_refuses_more_tokens_than_it_counts(batch, length):
    """Products past 2^64 among them, which would come out small."""
    rc, message = _rotary(batch=batch, length=length, x_batch=0, y_batch=128)
    assert rc == _lib.RPFQ_ERR_UNSUPPORTED and b"tokens" in message, message


@pytest.mark.parametrize("m,k", [(2 ** 61 + 1, 8), (2 ** 59 + 1, 8), (2 ** 56 + 1, 8), (2 ** 40, 8), (2, 2 ** 31 - 1)])
def test_quantize_rows_refuses_more_rows_than_it_counts(m, k):
    rc = _lib.lib().rpfq_quantize_rows_sm100(MB, 0, 2 ** 31 - 1, 2 * MB, 2 ** 31 - 1, 3 * MB, m, k, None)
    assert rc == _lib.RPFQ_ERR_UNSUPPORTED and b"too large" in _lib.lib().rpfq_last_error()
    assert _lib.lib().rpfq_gemm_i8_scratch_bytes(9, 2 ** 31 - 1) == 9 * (2 ** 31 + 4)


@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("bad,word", [
    (dict(q=MB), b"q shares"), (dict(q=MB + 8), b"q shares"), (dict(q=MB - 3 * 32 - 7), b"q shares"),
    (dict(scale=MB + 4), b"scale shares"), (dict(scale=MB - 12), b"scale shares"),
    (dict(scale=2 * MB + 4), b"q and scale"), (dict(q=3 * MB + 15), b"q and scale")])
def test_quantize_rows_refuses_outputs_over_what_is_read(f32, bad, word):
    """x [4, 8] in rows of 32 bytes, q in rows of 32, scale [4]."""
    a = dict(x=MB, q=2 * MB, scale=3 * MB)
    a.update(bad)
    L = _lib.lib()
    assert L.rpfq_quantize_rows_sm100(a["x"], f32, 8 if f32 else 16, a["q"], 32, a["scale"], 4, 8,
                                      None) == _lib.RPFQ_ERR_INVALID
    assert word in L.rpfq_last_error()


@pytest.mark.parametrize("strides", [dict(y_token=0), dict(y_head=0), dict(y_batch=0), dict(y_head=63), dict(y_token=-63),
                                     dict(y_batch=1)])
def test_rotary_refuses_an_output_over_itself(strides):
    rc, message = _rotary(**strides)
    assert rc == _lib.RPFQ_ERR_INVALID and b"itself" in message, message
    rc, message = _rotary(y=MB, **dict(strides, **{k.replace("y", "x"): v for k, v in strides.items()}))
    assert rc == _lib.RPFQ_ERR_INVALID and b"itself" in message, message
