"""GPU tests: outputs beside what a call reads, in one buffer, are answered; outputs over it are
refused."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [1, 4, 40, 1200])
def test_int8_output_beside_its_operands(cuda, m):
    from rpfq_review_b200 import ops
    n, k = 48, 64
    w, ws = ops.quantize_rows(torch.randn(n, k, device=cuda))
    x, xs = ops.quantize_rows(torch.randn(m, k, device=cuda))
    res = torch.randn(m, n, device=cuda).half()
    want = ops.gemm_int8(x, xs, w, ws, residual=res)
    buf = torch.zeros(m, 3 * n, dtype=torch.float16, device=cuda)
    for out_at, res_at in ((0, n), (2 * n, 0), (n, 2 * n), (n, 0), (n, n)):
        r, out = buf[:, res_at:res_at + n], buf[:, out_at:out_at + n]
        r.copy_(res)
        assert torch.equal(ops.gemm_int8(x, xs, w, ws, residual=r, out=out), want)
        assert out_at == res_at or torch.equal(r, res)
    # rows of w and of the output in one matrix, of the same stride
    both = torch.zeros(max(m, n), 64 + 96, dtype=torch.int8, device=cuda)
    both[:n, :k] = w
    out = both[:m, 64:].view(torch.float16)
    assert torch.equal(ops.gemm_int8(x, xs, both[:n, :k], ws, residual=res, out=out), want)
    assert torch.equal(both[:n, :k], w)


def test_int8_output_over_its_operands_is_refused(cuda):
    from rpfq_review_b200 import ops
    m, n, k = 40, 48, 64
    w, ws = ops.quantize_rows(torch.randn(n, k, device=cuda))
    x, xs = ops.quantize_rows(torch.randn(m, k, device=cuda))
    buf = torch.zeros(m + 1, 2 * n, dtype=torch.float16, device=cuda)
    flat = torch.zeros(m * n + 1, device=cuda).half()
    bias = torch.zeros(m * n, device=cuda)
    for residual, out, more in ((buf[:m, :n], buf[:m, 8:n + 8], {}), (buf[:m, :n], buf[1:, :n], {}),
                                (flat[1:].view(m, n), flat[:-1].view(m, n), {}),
                                (None, bias.view(m, n), dict(bias=bias[:n]))):
        with pytest.raises(ValueError, match="shares memory"):
            ops.gemm_int8(x, xs, w, ws, residual=residual, out=out, **more)
    with pytest.raises(ValueError, match="with w"):
        ops.gemm_int8(x[:10], xs[:10], w, ws, out=w.view(-1)[:10 * n * 2].view(torch.float16).view(10, n))


@pytest.mark.parametrize("D", [64, 20, 7])
def test_rotary_output_beside_its_input(cuda, D):
    """Query heads into the place of the key heads of the same rows, heads and tokens of one
    buffer in turn, an expanded input: answered. Shifted by a head, a token or a value: refused."""
    from rpfq_review_b200 import ops
    B, L, H, P = 2, 9, 3, D // 2
    f = ops.rotary_frequencies(2 * P, device=cuda)[0]
    pos = torch.arange(L, device=cuda)
    x = torch.randn(B, L, H, D, device=cuda).half()
    want = ops.rotary(x, pos, f)
    rows = torch.zeros(B, L, 3 * H, D, dtype=torch.float16, device=cuda)
    tokens = torch.zeros(B, 2 * L, H, D, dtype=torch.float16, device=cuda)
    for src, out in ((rows[:, :, :H], rows[:, :, H:2 * H]), (rows[:, :, 2 * H:], rows[:, :, :H]),
                     (rows[:, :, 0:2 * H:2], rows[:, :, 1:2 * H:2]), (tokens[:, ::2], tokens[:, 1::2]),
                     (tokens[:, L:], tokens[:, :L]), (rows[:, :, :H], rows[:, :, :H])):
        src.copy_(x)
        assert torch.equal(ops.rotary(src, pos, f, out=out), want)
        assert out.data_ptr() == src.data_ptr() or torch.equal(src, x)
    one = x[:1].expand(B, L, H, D)
    assert torch.equal(ops.rotary(one, pos, f, out=rows[:, :, :H]), ops.rotary(x[:1], pos, f).expand(B, L, H, D))
    flat = torch.zeros(B * L * H * D + 8, dtype=torch.float16, device=cuda)
    for src, out in ((rows[:, :, :H], rows[:, :, 1:H + 1]), (tokens[:, :L], tokens[:, 1:L + 1]),
                     (flat[:-8].view(B, L, H, D), flat[1:-7].view(B, L, H, D)),
                     (flat[8:].view(B, L, H, D), flat[:-8].view(B, L, H, D))):
        with pytest.raises(ValueError, match="overlap"):
            ops.rotary(src, pos, f, out=out)
    shared = torch.zeros(64, dtype=torch.float64, device=cuda)
    with pytest.raises(ValueError, match="inv_freq"):
        ops.rotary(x[0, :1, :1], pos[:1], shared[:P], out=shared.view(torch.float16)[:D].view(1, 1, D))


def test_codes_beside_their_rows(cuda):
    """The codes and scales of rows into the same buffer, beside them: through the C entry."""
    from rpfq_review_b200 import _lib, ops
    m, k = 5000, 64
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(0)).half().to(cuda)
    buf = torch.zeros(m, 2 * k + k + 16, dtype=torch.uint8, device=cuda)
    rows, codes = buf[:, :2 * k].view(torch.float16), buf[:, 2 * k:3 * k].view(torch.int8)
    rows.copy_(x)
    scale = torch.empty(m, device=cuda)
    _lib.check(_lib.lib().rpfq_quantize_rows_sm100(rows.data_ptr(), 0, buf.stride(0) // 2, codes.data_ptr(), buf.stride(0),
                                                   scale.data_ptr(), m, k, torch.cuda.current_stream().cuda_stream),
               "rpfq_quantize_rows_sm100")
    want = ops.quantize_rows(x)
    assert torch.equal(codes, want[0]) and torch.equal(scale, want[1]) and torch.equal(rows, x)
    assert (buf[:, 3 * k:] == 0).all()


def test_rotary_output_over_itself_is_refused(cuda):
    from rpfq_review_b200 import ops
    f, pos = ops.rotary_frequencies(16, device=cuda)[0], torch.arange(6, device=cuda)
    x, flat = torch.randn(6, 2, 16, device=cuda), torch.zeros(400, device=cuda)
    for strides in ((8, 64, 1), (32, 15, 1), (0, 16, 1)):
        with pytest.raises(ValueError):
            ops.rotary(x, pos, f, out=flat.as_strided((6, 2, 16), strides))
    out = flat.as_strided((6, 2, 16), (16, 96, 1))  # heads outermost
    assert torch.equal(ops.rotary(x, pos, f, out=out), ops.rotary(x, pos, f))
    one = flat.as_strided((1, 1, 16), (0, 0, 1))  # strides that no step uses
    assert torch.equal(ops.rotary(x[:1, :1], pos[:1], f, out=one), ops.rotary(x[:1, :1], pos[:1], f))
