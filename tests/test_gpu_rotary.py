"""GPU tests of the rotary positions (``rotary``) against float64.

Bound per element: with u = 2^-24, cos and sin (2 ulp of the function, one
rounding of the reduced angle's head and of the correction, one of the
magnitude) are off by at most 8 u, the two products and their sum by 3 u of
(|a| + |b|): 11 u c (|a| + |b|), taken as 16 u; the fp64 angle itself by
2^-52 |angle| c (|a| + |b|); an fp16 output adds half a step, 2^-11 |y| (2^-25
for subnormals)."""

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _ref(x, positions, inv_freq, layout, axes, magnitude, transpose):
    """Value and bound, float64 on the CPU."""
    x, pos, f = x.detach().cpu(), positions.cpu().double(), inv_freq.cpu()
    dtype, P = x.dtype, f.numel()
    x = x.double()
    if axes == 1:
        pos = pos.unsqueeze(-1)
    axis = torch.arange(P) * axes // P
    angle = (pos[..., axis] * f).unsqueeze(-2)
    c, s = magnitude * torch.cos(angle), magnitude * torch.sin(angle) * (-1.0 if transpose else 1.0)
    i = torch.arange(P) * (1 if layout == "half" else 2)
    j = i + (P if layout == "half" else 1)
    a, b = x[..., i], x[..., j]
    y, err = x.clone(), torch.zeros_like(x)
    y[..., i], y[..., j] = a * c - b * s, b * c + a * s
    size = (a.abs() + b.abs()) * magnitude * (16 * U + 2.0 ** -52 * angle.abs())
    err[..., i] = size
    err[..., j] = size
    if dtype == torch.float16:
        turned = torch.zeros(x.shape[-1])
        turned[i], turned[j] = 1.0, 1.0
        err = (err + 2.0 ** -11 * (y.abs() + err) + 2.0 ** -25) * turned
    return y, err + 1e-37 * (err > 0)


def _check(got, ref):
    y, err = ref
    d = (got.detach().cpu().double() - y).abs()
    assert torch.isfinite(d).all()
    assert (d <= err).all(), f"worst {(d / (err + 1e-300)).max().item():.3g} of the bound"


def _freq(P, axes=1, base=10000.0):
    from rpfq_review_b200 import ops
    return ops.rotary_frequencies(2 * P, base, axes=axes, device="cuda")[0]


CASES = [  # B, L, H, D, pairs, axes
    (1, 1, 1, 2, 1, 1), (16, 1, 32, 128, 64, 1), (2, 197, 6, 64, 32, 2), (3, 50, 5, 80, 20, 1), (1, 700, 3, 96, 36, 2),
    (2, 33, 2, 256, 128, 1), (2, 5, 3, 37, 9, 1), (1, 9, 4, 64, 3, 1), (5, 17, 1, 72, 36, 1), (1, 3, 2, 4096, 2048, 1)]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("B,L,H,D,P,axes", CASES)
def test_rotary_matches_fp64(cuda, B, L, H, D, P, axes, dtype, layout):
    from rpfq_review_b200 import ops
    g = torch.Generator().manual_seed(B + L + D)
    x = torch.randn(B, L, H, D, generator=g).to(dtype).to(cuda)
    f = _freq(P, axes)
    tail = (axes,) if axes > 1 else ()
    shared = torch.randint(0, 2000, (L, *tail), generator=g, dtype=torch.int32).to(cuda)
    own = torch.randint(-500, 100000, (B, L, *tail), generator=g).to(cuda)
    for pos, mag, t in ((shared, 1.0, False), (own, 1.25, False), (own, 1.25, True)):
        y = ops.rotary(x, pos, f, layout=layout, axes=axes, magnitude=mag, transpose=t)
        assert y.shape == x.shape and y.dtype == dtype and y.is_contiguous()
        _check(y, _ref(x, pos, f, layout, axes, mag, t))
    if B == 1:
        assert torch.equal(ops.rotary(x[0], shared, f, layout=layout, axes=axes),
                           ops.rotary(x, shared, f, layout=layout, axes=axes)[0])
    inplace = x.clone()
    assert ops.rotary(inplace, own, f, layout=layout, axes=axes, magnitude=1.25, out=inplace) is inplace
    assert torch.equal(inplace, ops.rotary(x, own, f, layout=layout, axes=axes, magnitude=1.25))


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, torch.float32, torch.float64])
def test_rotary_position_types_and_far_positions(cuda, dtype):
    """Far positions keep their angle: 2^24 - 1 in fp32, near 2^31 in int32, 2^40 in the
    64-bit types; fractions in the floating ones."""
    from rpfq_review_b200 import ops
    far = {torch.int32: 2 ** 31 - 9, torch.float32: 2 ** 24 - 1}.get(dtype, 2 ** 40 + 3)
    pos = torch.tensor([0, 1, 7, far, -far, far - 5], dtype=torch.float64).to(dtype)
    if dtype.is_floating_point:
        pos[1] = 0.375
    x = torch.randn(6, 3, 64, generator=torch.Generator().manual_seed(0)).to(cuda)
    f = _freq(32)
    _check(ops.rotary(x, pos.to(cuda), f), _ref(x, pos, f, "half", 1, 1.0, False))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_strides(cuda, dtype, layout):
    """Heads inside wider rows, [B, H, L, D] order, odd offsets and strides,
    expanded inputs; an output inside a wider buffer leaves the rest alone."""
    from rpfq_review_b200 import ops
    g = torch.Generator().manual_seed(9)
    B, L, H, D, P = 2, 37, 3, 48, 16
    f, pos = _freq(P), torch.arange(L, device=cuda, dtype=torch.int32)
    flat = torch.randn(B * L * (3 * H * D + 7) + 64, generator=g).to(dtype).to(cuda)
    views = [flat[:B * L * 3 * H * D].view(B, L, 3 * H, D)[:, :, :2 * H],
             flat[:B * L * H * D].view(B, H, L, D).transpose(1, 2),
             flat[1:1 + B * L * H * D].view(B, L, H, D),
             flat[4:4 + B * L * (3 * H * D + 7)].view(B, L, -1)[:, :, 3:3 + H * D].unflatten(-1, (H, D)),
             flat[:L * H * D].view(1, L, H, D).expand(B, L, H, D),
             flat[:B * L * H * 2 * D].view(B, L, H, 2 * D)[..., ::2]]
    for x in views:
        _check(ops.rotary(x, pos, f, layout=layout), _ref(x, pos, f, layout, 1, 1.0, False))
    for off in (0, 1):
        buf = torch.full((B, L + 1, H + 1, D + 8), 3.0, dtype=dtype, device=cuda)
        out = buf[:, :L, 1:, off:off + D]
        x = views[0][:, :, :H]
        assert ops.rotary(x, pos, f, layout=layout, out=out) is out
        _check(out, _ref(x, pos, f, layout, 1, 1.0, False))
        out.fill_(3.0)
        assert (buf == 3.0).all()
    # in place on query and key heads: the value heads and the unrotated part keep their bits
    rows = views[0].new_empty(B, L, 3 * H, D).copy_(flat[:B * L * 3 * H * D].view(B, L, 3 * H, D))
    before = rows.clone()
    qk = rows[:, :, :2 * H]
    ops.rotary(qk, pos, f, layout=layout, out=qk)
    _check(qk, _ref(before[:, :, :2 * H], pos, f, layout, 1, 1.0, False))
    assert torch.equal(rows[:, :, 2 * H:], before[:, :, 2 * H:]) and torch.equal(rows[..., 2 * P:], before[..., 2 * P:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_transpose_is_the_gradient(cuda, layout):
    """<w, R(x + h e) - R(x - h e)> / 2h against the transposed map of w, in fp32: R is
    linear, so the difference quotient is exact up to rounding (11 u of each output's
    operands over h, here h = 1)."""
    from rpfq_review_b200 import ops
    g = torch.Generator().manual_seed(2)
    L, H, D, P = 11, 2, 24, 10
    f, pos = _freq(P), torch.arange(L, device=cuda) * 37
    x, w = torch.randn(L, H, D, generator=g).to(cuda), torch.randn(L, H, D, generator=g).to(cuda)
    call = lambda v, t=False: ops.rotary(v, pos, f, layout=layout, magnitude=1.5, transpose=t)  # noqa: E731
    grad = call(w, True)
    for at in ((0, 0, 0), (3, 1, 7), (10, 0, 19), (5, 1, 23)):
        e = torch.zeros_like(x)
        e[at] = 1.0
        num = (w.double() * (call(x + e).double() - call(x - e).double())).sum() / 2
        size = w.double().abs().sum(-1)[at[0], at[1]] * (x.abs().max().double() + 1) * 2 * 1.5
        assert abs(num - grad[at].double()) <= 16 * U * size
    xd, f64 = x.detach().cpu().double().requires_grad_(), f.cpu()
    angle = (pos.cpu().double().unsqueeze(-1) * f64).unsqueeze(-2)
    i = torch.arange(P) * (1 if layout == "half" else 2)
    j = i + (P if layout == "half" else 1)
    a, b, c, s = xd[..., i], xd[..., j], 1.5 * torch.cos(angle), 1.5 * torch.sin(angle)
    wd = w.cpu().double()
    ((a * c - b * s) * wd[..., i] + (b * c + a * s) * wd[..., j]).sum().backward()
    want = xd.grad + torch.cat([torch.zeros(L, H, 2 * P, dtype=torch.float64), wd[..., 2 * P:]], -1)
    ref = _ref(w, pos, f, layout, 1, 1.5, True)
    assert torch.allclose(ref[0], want, rtol=0, atol=1e-12)
    _check(grad, ref)


def test_rotary_relative_positions(cuda):
    """Scores of turned queries and keys depend on the difference of positions only."""
    from rpfq_review_b200 import ops
    g = torch.Generator().manual_seed(4)
    q, k = torch.randn(40, 1, 64, generator=g).to(cuda), torch.randn(40, 1, 64, generator=g).to(cuda)
    f, pos = _freq(32), torch.arange(40, device=cuda)
    score = lambda s: (ops.rotary(q, pos + s, f)[:, 0].double() @ ops.rotary(k, pos + s, f)[:, 0].double().t())  # noqa: E731
    size = q[:, 0].double().norm(dim=1)[:, None] * k[:, 0].double().norm(dim=1) * 2
    assert ((score(0) - score(100003)).abs() <= 64 * U * size).all()


def test_rotary_graph_and_large_offsets(cuda):
    """A captured call replays on new values and positions; elements past 2^31 are reached."""
    from rpfq_review_b200 import _lib, ops
    x = torch.randn(3, 8, 2, 64, device=cuda).half()
    pos, f = torch.arange(8, device=cuda, dtype=torch.int32), _freq(32)
    ops.rotary(x, pos, f)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.rotary(x, pos, f)
    x.normal_()
    pos.add_(1000)
    g.replay()
    assert torch.equal(y, ops.rotary(x, pos, f))
    B, L, H, D = 2, 70000, 1, 64
    wide = torch.empty(B, L, 17600, dtype=torch.float16, device=cuda)  # 2.5e9 elements, 4.9 GB
    far = wide[:, :, 17536:].unsqueeze(2)
    far.normal_()
    pos = torch.arange(L, device=cuda)
    y = ops.rotary(far, pos, f)
    assert torch.equal(y, ops.rotary(far.contiguous(), pos, f))
    ops.rotary(far, pos, f, out=far)
    assert torch.equal(far, y)
    torch.cuda.synchronize()
    assert _lib.device_error() == 0


def test_rotary_refusals(cuda):
    from rpfq_review_b200 import ops
    x, pos, f = torch.randn(2, 5, 3, 16, device=cuda), torch.arange(5, device=cuda), _freq(8)
    bad = [
        lambda: ops.rotary(x.double(), pos, f), lambda: ops.rotary(x.bfloat16(), pos, f), lambda: ops.rotary(x[0, 0], pos, f),
        lambda: ops.rotary(x, pos.cpu(), f), lambda: ops.rotary(x, pos.half(), f), lambda: ops.rotary(x, pos[:4], f),
        lambda: ops.rotary(x, pos.expand(3, 5), f), lambda: ops.rotary(x[0], pos.expand(1, 5), f),
        lambda: ops.rotary(x, pos, f.float()), lambda: ops.rotary(x, pos, f.cpu()), lambda: ops.rotary(x, pos, _freq(9)),
        lambda: ops.rotary(x, pos, f[:0]), lambda: ops.rotary(x, pos, f, axes=2), lambda: ops.rotary(x, pos, f, axes=3),
        lambda: ops.rotary(x, pos[:, None].expand(5, 2), f[:7], axes=2), lambda: ops.rotary(x, pos, f, layout="pairs"),
        lambda: ops.rotary(x, pos, f, out=x.half()), lambda: ops.rotary(x, pos, f, out=x[:, :, :2]),
        lambda: ops.rotary(x, pos, f, out=x[:1].expand(2, 5, 3, 16)), lambda: ops.rotary(x[..., ::2], pos, f[:4], out=x[..., ::2]),
        lambda: ops.rotary(x.clone().requires_grad_(), pos, f)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"case {i} was accepted")
    for empty in (x[:0], x[:, :0], x[:, :, :0]):
        assert ops.rotary(empty, pos[: empty.shape[1]], f).shape == empty.shape
    y = torch.ops.rpfq.rotary(x, pos, f, "interleaved", 1, 1.5, True)
    assert torch.equal(y, ops.rotary(x, pos, f, layout="interleaved", magnitude=1.5, transpose=True))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("B,L,H,D,P", [(1, 3000, 32, 64, 32), (700, 3, 2, 32, 16), (1, 9000, 1, 8, 4), (3, 400, 40, 128, 32),
                                       (1, 2, 3, 2100, 300), (1, 70, 300, 16, 8)])
def test_rotary_many_tokens_and_heads(cuda, layout, B, L, H, D, P):
    """Tokens over many blocks, heads beyond a thread's copies in flight, heads of more
    pieces than a block has threads."""
    from rpfq_review_b200 import ops
    g = torch.Generator().manual_seed(L)
    f, pos = _freq(P), torch.randint(0, 5000, (B, L), generator=g).to(cuda)
    for dtype in (torch.float16, torch.float32):
        x = torch.randn(B, L, H, D, generator=g).to(dtype).to(cuda)
        ref = _ref(x, pos, f, layout, 1, 1.0, False)
        _check(ops.rotary(x, pos, f, layout=layout), ref)
        odd = torch.zeros(B, L, H, D + 1, dtype=dtype, device=cuda)[..., 1:]
        odd.copy_(x)
        _check(ops.rotary(odd, pos, f, layout=layout), ref)
        ops.rotary(x, pos, f, layout=layout, out=x)
        _check(x, ref)
