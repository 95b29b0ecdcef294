"""GPU tests of the 8-bit product at the ends of its ranges."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 2, 4, 9])
def test_rows_of_very_many_columns(cuda, rows):
    """n so large that three times n passes 2^31: the last columns equal a small call's, with a
    residual in place, and nothing behind a row is written."""
    from rpfq_review_b200 import _lib, ops
    n, k = 720_000_003, 16
    w = torch.empty(n, k, dtype=torch.int8, device=cuda)  # 11.5 GB
    for part in w.split(1 << 27):
        part.random_(-127, 128)
    ws = torch.rand(n, device=cuda)
    x, xs = torch.randint(-127, 128, (rows, k), dtype=torch.int8, device=cuda), torch.rand(rows, device=cuda)
    wide = torch.full((rows, n + 5), 3.0, dtype=torch.float16, device=cuda)
    y = wide[:, :n]
    ends = [slice(0, 70), slice(536_870_900, 536_870_970), slice(n - 70, n)]
    small = [ops.gemm_int8(x, xs, w[e], ws[e], activation="gelu", residual=y[:, e].clone()) for e in ends]
    ops.gemm_int8(x, xs, w, ws, activation="gelu", residual=y, out=y)
    for e, want in zip(ends, small):
        assert torch.equal(y[:, e], want)
    assert (wide[:, n:] == 3.0).all()
    ops.gemm_int8(x, xs, w, ws, out=y)
    assert torch.equal(y[:, ends[2]], ops.gemm_int8(x, xs, w[ends[2]], ws[ends[2]])) and (wide[:, n:] == 3.0).all()
    assert _lib.device_error() == 0


def test_gelu_error(cuda):
    """y = max(v, 0) - a 2^Q(a), a = |v|: Q is within 0.75 x 2^-24 |v| of its place (shown on the
    CPU), the hardware's 2^x is off by 2^-22 of a Phi(-a), and the fused last step rounds y once:
    (0.75 + 4 Phi(-a)) 2^-24 a + 2^-24 |y|; results below the normal range may be flushed."""
    from rpfq_review_b200 import ops
    g = torch.Generator().manual_seed(0)
    v = torch.cat([torch.linspace(-14, 14, 400001), torch.randn(400000, generator=g) * 2, -torch.logspace(-6, 1.2, 100000),
                   torch.logspace(-6, 1.2, 100000)]).to(cuda)
    one = torch.ones(9, 1, dtype=torch.int8, device=cuda)
    w = torch.ones(v.numel(), 1, dtype=torch.int8, device=cuda)
    x = v.double()
    a, ref = x.abs(), x * torch.special.ndtr(x)
    bound = 2.0 ** -24 * ((0.75 + 4 * torch.special.ndtr(-a)) * a + ref.abs()) + 2.0 ** -126 * 64
    for rows in (1, 9):
        y = ops.gemm_int8(one[:rows], torch.ones(rows, device=cuda), w, v, activation="gelu", out_dtype=torch.float32)
        d = (y[-1].double() - ref).abs()
        assert (d <= bound).all(), (d / bound).max().item()
