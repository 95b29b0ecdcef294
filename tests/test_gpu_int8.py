"""GPU tests of the 8-bit linear path: ``quantize_rows``, ``gemm_int8``,
``linear_int8`` and the layers that run on them.

Codes and scales are compared bit for bit with the same fp32 steps in numpy.
Products are compared element by element with float64: the int32 sum S is
exact, so with u = 2^-24 (half a step of fp32) the value before the activation,
v = fl(fl(fl(S) w_scale) x_scale + bias), is off by at most
3 u |S w_scale x_scale| + u |v|; exact GELU passes that on times at most 1.13 and
its own evaluation adds at most 2^-20 |v| (erf to 1.5e-7, the rest fp32 steps on
values below 5); a residual adds u |y|, an fp16 output half a step, 2^-11 |y|
(2^-25 for subnormals)."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _codes_ref(x: np.ndarray):
    """quantize_rows in numpy, fp32 steps."""
    x = x.astype(np.float32)
    with np.errstate(invalid="ignore", over="ignore"):
        bad = ~np.isfinite(x).all(axis=1)
        t = np.maximum(np.where(bad, np.float32(1), np.abs(x).max(axis=1)), np.float32(1e-30)).astype(np.float32)
        s = (np.float32(1) / t * np.float32(127)).astype(np.float32)
        q = np.rint((x * s[:, None]).astype(np.float32))
    q[bad] = 0
    scale = (t / np.float32(127)).astype(np.float32)
    scale[bad] = np.nan
    return q.astype(np.int8), scale


def _product_ref(xq, xs, wq, ws, bias, act, residual, out_dtype):
    """Value and error bound in float64, on the CPU."""
    f = lambda t: t.detach().cpu().double()  # noqa: E731
    S = f(xq) @ f(wq).t()
    main = S * f(xs).reshape(-1, 1) * f(ws)
    v = main + (f(bias) if bias is not None else 0.0)
    err = 3 * U * main.abs() + U * v.abs()
    if act == "gelu":
        err = 1.13 * err + 2.0 ** -20 * v.abs()
        v = v * torch.special.ndtr(v)
    if residual is not None:
        v = v + f(residual)
        err = err + U * v.abs()
    if out_dtype == torch.float16:
        err = err + 2.0 ** -11 * (v.abs() + err) + 2.0 ** -25
    return v, err + 1e-37


def _check(y, ref):
    v, err = ref
    d = (y.detach().cpu().double().reshape(v.shape) - v).abs()
    assert torch.isfinite(d).all()
    worst = (d / err).max().item() if d.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3g} of the bound"


def _operands(dev, m, n, k, seed=0, full_range=False):
    g = torch.Generator().manual_seed(seed)
    lo, hi = (-128, 128) if full_range else (-127, 128)
    xq = torch.randint(lo, hi, (m, k), generator=g, dtype=torch.int8)
    wq = torch.randint(lo, hi, (n, k), generator=g, dtype=torch.int8)
    xs = (torch.rand(m, generator=g) + 0.5) * 0.02
    ws = (torch.rand(n, generator=g) + 0.5) * (0.5 / (73 * k ** 0.5))
    return xq.to(dev), xs.to(dev), wq.to(dev), ws.to(dev)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 16), (3, 7), (5, 8), (9, 100), (33, 768), (2, 4096), (300, 1003), (4, 20011),
                                 (5003, 64), (4801, 33), (2500, 1024), (2501, 516), (1301, 2048), (1301, 1030), (1300, 2056),
                                 (5000, 1), (4900, 7), (4900, 62), (2500, 129), (2500, 1017), (1300, 4090), (1300, 1999),
                                 (1300, 4097)])
def test_quantize_rows_bit_exact(cuda, dtype, m, k):
    from rpfq_review_b200 import ops
    g = torch.Generator().manual_seed(m * 31 + k)
    x = (torch.randn(m, k, generator=g) * torch.logspace(-3, 2, m).unsqueeze(1)).to(dtype)
    q, scale = ops.quantize_rows(x.to(cuda))
    assert q.shape == x.shape and q.dtype == torch.int8 and scale.shape == (m,) and scale.dtype == torch.float32
    want_q, want_s = _codes_ref(x.float().numpy())
    assert np.array_equal(q.cpu().numpy(), want_q)
    assert np.array_equal(scale.cpu().numpy(), want_s)
    back = q.cpu().double() * scale.cpu().double().unsqueeze(1)
    # half a code, and the fp32 roundings of x s (|x s| <= 127) and of the scale
    bound = scale.cpu().double().unsqueeze(1) * (0.5 + 127 * 4 * U)
    assert ((back - x.double()).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_quantize_rows_off_the_grid(cuda, dtype):
    """Rows that start at every offset from 16 bytes, with strides of every remainder."""
    from rpfq_review_b200 import ops
    g = torch.Generator().manual_seed(0)
    flat = torch.randn(5000 * 90, generator=g).to(dtype)
    flat[7::1013] = float("nan")
    dev = flat.to(cuda)
    for k in (1, 5, 30, 64, 67):
        for stride in range(k, k + 9):
            for start in (0, 1, 3):
                want_q, want_s = _codes_ref(flat.as_strided((4800, k), (stride, 1), start).float().numpy())
                q, s = ops.quantize_rows(dev.as_strided((4800, k), (stride, 1), start))
                assert np.array_equal(q.cpu().numpy(), want_q) and np.array_equal(s.cpu().numpy(), want_s, equal_nan=True)


def test_quantize_rows_edges_and_strides(cuda):
    """Zeros, single peaks, ties, values below the floor, non-finite rows; rows
    with a stride, a column offset that breaks the 16-byte alignment, expanded rows."""
    from rpfq_review_b200 import ops
    k = 130
    x = torch.zeros(9, k)
    x[1, 5] = -3.0
    x[2] = torch.arange(k) * 0.5 - 31.75   # ties at amax 127 / 4 ...
    x[2, 0] = 127.0
    x[3, :3] = torch.tensor([1e-38, -1e-40, 3e-39])
    x[4, 7] = float("inf")
    x[5, 9] = float("nan")
    x[6] = 65504.0
    x[7, -1] = -3.0e38
    x[8, 0], x[8, 1:5] = 254.0, torch.tensor([1.0, 3.0, 5.0, -1.0])  # halves: to even
    q, s = ops.quantize_rows(x.to(cuda))
    want_q, want_s = _codes_ref(x.numpy())
    assert np.array_equal(q.cpu().numpy(), want_q) and np.array_equal(s.cpu().numpy(), want_s, equal_nan=True)
    assert torch.isnan(s[4]) and torch.isnan(s[5]) and torch.count_nonzero(q[4:6]) == 0 and torch.count_nonzero(q[0]) == 0
    assert q[8, 1:5].tolist() == [0, 2, 2, 0]
    g = torch.Generator().manual_seed(3)
    for dtype in (torch.float16, torch.float32):
        base = torch.randn(40, 3 * k + 5, generator=g).to(dtype).to(cuda)
        for view in (base[:, 1:1 + k], base[::3, 2 * k:3 * k], base[:, : 2 * k: 2], base[:1, :k].expand(6, k)):
            q, s = ops.quantize_rows(view)
            want_q, want_s = _codes_ref(view.cpu().float().numpy())
            assert np.array_equal(q.cpu().numpy(), want_q) and np.array_equal(s.cpu().numpy(), want_s)
    q, s = ops.quantize_rows(torch.randn(2, 3, 5, k, generator=g).to(cuda))
    assert q.shape == (2, 3, 5, k) and s.shape == (2, 3, 5)
    q, s = ops.quantize_rows(torch.empty(0, k, device=cuda))
    assert q.shape == (0, k) and s.shape == (0,)


SHAPES = [(1, 1, 1), (1, 8, 16), (1, 1000, 768), (2, 64, 33), (4, 129, 257), (7, 130, 128), (16, 96, 1024),
          (17, 300, 390), (63, 1001, 100), (128, 128, 128), (129, 257, 1003), (197, 768, 384), (255, 64, 4099),
          (300, 1000, 96), (1571, 77, 515)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("out_dtype", [torch.float16, torch.float32])
def test_gemm_int8_matches_fp64(cuda, m, n, k, out_dtype):
    from rpfq_review_b200 import ops
    xq, xs, wq, ws = _operands(cuda, m, n, k, seed=m + n + k, full_range=True)
    g = torch.Generator().manual_seed(5)
    bias = torch.randn(n, generator=g).to(cuda)
    res = torch.randn(m, n, generator=g).to(out_dtype).to(cuda)
    for b, act, r in ((None, "none", None), (bias.half(), "gelu", None), (bias, "none", res), (bias, "gelu", res)):
        y = ops.gemm_int8(xq, xs, wq, ws, bias=b, residual=r, activation=act, out_dtype=out_dtype)
        assert y.dtype == out_dtype and y.shape == (m, n)
        _check(y, _product_ref(xq, xs, wq, ws, b, act, r, out_dtype))


# enough 256 x 256 tiles for CTA pairs on 148 SMs: whole waves, last waves cut into two
# and four column pieces, ragged rows and columns, one k-block and several
MANY_ROWS = [(9500, 512, 200), (4900, 1000, 144), (6600, 1001, 96), (18900, 250, 33), (9473, 1000, 640)]


@pytest.mark.parametrize("m,n,k", MANY_ROWS)
@pytest.mark.parametrize("out_dtype", [torch.float16, torch.float32])
def test_gemm_int8_many_rows(cuda, m, n, k, out_dtype):
    from rpfq_review_b200 import _lib, ops
    xq, xs, wq, ws = _operands(cuda, m, n, k, seed=m + n + k)
    g = torch.Generator().manual_seed(6)
    bias = torch.randn(n, generator=g).to(cuda)
    res = torch.randn(m, n, generator=g).to(out_dtype).to(cuda)
    for b, act, r in ((bias, "none", None), (bias.half(), "gelu", res)):
        y = ops.gemm_int8(xq, xs, wq, ws, bias=b, residual=r, activation=act, out_dtype=out_dtype)
        _check(y, _product_ref(xq, xs, wq, ws, b, act, r, out_dtype))
    # rows that TMA can store but not load and the other way round, in place too
    wide = torch.full((m, n + 24), 5.0, dtype=out_dtype, device=cuda)
    want = y
    for out_off, res_off in ((8, 1), (1, 8)):
        rv = wide.clone()[:, res_off:res_off + n]
        rv.copy_(res)
        buf = wide.clone()
        out = buf[:, out_off:out_off + n]
        ops.gemm_int8(xq, xs, wq, ws, bias=bias.half(), residual=rv, activation="gelu", out=out)
        assert torch.equal(out, want)
        out.fill_(5.0)
        assert torch.equal(buf, wide)
        ops.gemm_int8(xq, xs, wq, ws, bias=bias.half(), residual=rv, activation="gelu", out=rv)
        assert torch.equal(rv, want)
    torch.cuda.synchronize()
    assert _lib.device_error() == 0


def test_gemm_int8_largest_sums(cuda):
    """k = 131071 codes of -128 reach 2^31 - 2^14: no overflow; one more is refused."""
    from rpfq_review_b200 import ops
    k = ops.GEMM_INT8_MAX_K
    x = torch.full((3, k), -128, dtype=torch.int8, device=cuda)
    x[1] = 127
    w = torch.full((5, k), -128, dtype=torch.int8, device=cuda)
    one = torch.ones(5, device=cuda)
    y = ops.gemm_int8(x, one[:3], w, one, out_dtype=torch.float32).cpu()
    assert (y[0] == torch.tensor(float(128 * 128 * k))).all() and (y[1] == torch.tensor(float(-127 * 128 * k))).all()
    with pytest.raises(NotImplementedError, match="131071"):
        ops.gemm_int8(torch.zeros(1, k + 1, dtype=torch.int8, device=cuda), one[:1],
                      torch.zeros(1, k + 1, dtype=torch.int8, device=cuda), one[:1])


@pytest.mark.parametrize("out_dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("m,n,k", [(5, 37, 48), (200, 130, 144), (1300, 256, 64)])
def test_gemm_int8_strides(cuda, m, n, k, out_dtype):
    """Rows with a stride, rows off the 16-byte grid, an output inside a wider
    buffer (its surroundings untouched), in-place residual, leading dimensions."""
    from rpfq_review_b200 import ops
    xq, xs, wq, ws = _operands(cuda, m, n, k, seed=7)
    wide_x = torch.zeros(m, 2 * k + 16, dtype=torch.int8, device=cuda)
    wide_w = torch.zeros(n, 2 * k + 16, dtype=torch.int8, device=cuda)
    for off in (16, 3):
        xv, wv = wide_x[:, off:off + k], wide_w[:, off:off + k]
        xv.copy_(xq)
        wv.copy_(wq)
        ref = _product_ref(xq, xs, wq, ws, None, "none", None, out_dtype)
        _check(ops.gemm_int8(xv, xs, wv, ws, out_dtype=out_dtype), ref)
    for pad, off in ((32, 8), (3, 1), (4, 2)):
        buf = torch.full((m + 2, n + pad + off), 7.0, dtype=out_dtype, device=cuda)
        out = buf[1:m + 1, off:off + n]
        assert ops.gemm_int8(xq, xs, wq, ws, out=out) is out
        _check(out, ref)
        keep = buf.clone()
        keep[1:m + 1, off:off + n] = 7.0
        assert (keep == 7.0).all()
        stream = torch.randn(m, n, generator=torch.Generator().manual_seed(1)).to(out_dtype)
        out.copy_(stream)
        ops.gemm_int8(xq, xs, wq, ws, residual=out, out=out)
        _check(out, _product_ref(xq, xs, wq, ws, None, "none", stream, out_dtype))
    if m % 5 == 0:
        y = ops.gemm_int8(xq.view(5, m // 5, k), xs.view(5, -1), wq, ws, out_dtype=out_dtype)
        assert y.shape == (5, m // 5, n)
        _check(y, ref)
    assert ops.gemm_int8(xq[:0], xs[:0], wq, ws).shape == (0, n)
    row = ops.gemm_int8(xq[:1].expand(9, k), xs[:1].expand(9), wq, ws, out_dtype=out_dtype)
    assert all(torch.equal(row[i], row[0]) for i in range(9))


@pytest.mark.parametrize("out_dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("m,n,k", [(4, 3, 15), (31, 63, 130), (300, 255, 63), (513, 1001, 300)])
def test_gemm_int8_inside_wider_rows(cuda, m, n, k, out_dtype):
    """Operands, residual and output as columns of wider rows on the 16-byte grid, n and
    k off it: what lies beside them is neither read nor written, by any schedule."""
    from rpfq_review_b200 import ops
    xq, xs, wq, ws = _operands(cuda, m, n, k, seed=19)
    g = torch.Generator().manual_seed(19)
    residual = torch.randn(m, n, generator=g).to(out_dtype)
    ref = _product_ref(xq, xs, wq, ws, None, "none", None, out_dtype)
    ref_res = _product_ref(xq, xs, wq, ws, None, "none", residual, out_dtype)

    def inside(t, step, beside):
        buf = torch.full((t.shape[0] + 1, -(-t.shape[1] // step) * step + 2 * step), beside, dtype=t.dtype, device=cuda)
        view = buf[:-1, step:step + t.shape[1]]
        view.copy_(t)
        return view

    xv, wv = inside(xq, 16, 113), inside(wq, 16, 127)
    rv = inside(residual.to(cuda), 16, float("nan"))
    for block_n in (0, 64, 128, 256):
        for res, want in ((None, ref), (rv, ref_res)):
            out = inside(torch.zeros(m, n, dtype=out_dtype, device=cuda), 16, 7.0)
            ops.gemm_int8(xv, xs, wv, ws, residual=res, out=out, block_n=block_n)
            _check(out, want)
            out.fill_(7.0)
            assert (out._base == 7.0).all(), f"written beside the output with block_n={block_n}"


def test_gemm_int8_nan_scale_stays_in_its_row(cuda):
    from rpfq_review_b200 import ops
    for m in (4, 140, 1000):
        x = torch.randn(m, 64, device=cuda)
        x[2, 3] = float("nan")
        w, ws = ops.quantize_rows(torch.randn(24, 64, device=cuda))
        y = ops.linear_int8(x, w, ws)
        assert torch.isnan(y[2]).all()
        y[2] = 0
        assert torch.isfinite(y).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("m,n,k", [(1, 768, 768), (3, 50, 33), (8, 1000, 200), (197, 640, 390), (2000, 264, 130)])
def test_linear_int8_is_quantize_then_product(cuda, dtype, m, n, k):
    from rpfq_review_b200 import ops
    g = torch.Generator().manual_seed(k)
    x = torch.randn(m, k, generator=g).to(dtype).to(cuda)
    w, ws = ops.quantize_rows((torch.randn(n, k, generator=g) * 0.05).to(cuda))
    bias = torch.randn(n, generator=g).to(cuda)
    res = torch.randn(m, n, generator=g).to(dtype).to(cuda)
    y = ops.linear_int8(x, w, ws, bias, res, "gelu", out_dtype=dtype)
    xq, xs = ops.quantize_rows(x)
    assert torch.equal(y, ops.gemm_int8(xq, xs, w, ws, bias, res, "gelu", out_dtype=dtype))
    _check(y, _product_ref(xq, xs, w, ws, bias, "gelu", res, dtype))
    # against the unquantized product: each operand is off by at most half a code
    exact = x.double() @ (w.double() * ws.double().unsqueeze(1)).t()
    plain = ops.linear_int8(x, w, ws, out_dtype=torch.float32).double()
    bound = 0.5 * (1 + 1e-4) * xs.double().unsqueeze(1) * (w.double().abs() * ws.double().unsqueeze(1)).sum(1)
    assert ((plain - exact).abs() <= bound + 1e-5).all()


@pytest.mark.parametrize("m", [1, 12, 150, 1200])
def test_int8_graphs_and_streams(cuda, m):
    """Captured calls replay on new inputs, two graphs at once on two streams."""
    from rpfq_review_b200 import ops
    k, n = 256, 384
    w, ws = ops.quantize_rows(torch.randn(n, k, device=cuda) * 0.05)
    graphs = []
    for i in range(2):
        x = torch.randn(m, k, device=cuda).half()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.linear_int8(x, w, ws)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ops.linear_int8(x, w, ws)
            z = ops.linear_int8(y, w[:, :k].contiguous(), ws) if n == k else ops.linear_int8(x, w, ws, residual=y)
        graphs.append((g, x, y, z, side))
    for step in range(3):
        for g, x, *_ in graphs:
            x.copy_(torch.randn(m, k, device=cuda).half())
        torch.cuda.synchronize()
        for g, _, _, _, side in graphs:
            with torch.cuda.stream(side):
                g.replay()
        torch.cuda.synchronize()
        for g, x, y, z, _ in graphs:
            want = ops.linear_int8(x, w, ws)
            assert torch.equal(y, want) and torch.equal(z, ops.linear_int8(x, w, ws, residual=want))
    from rpfq_review_b200 import _lib
    assert _lib.device_error() == 0


@pytest.mark.parametrize("n_c,k_c", [(96, 64), (50, 37)])
def test_packed_layer_int8(cuda, n_c, k_c):
    """PackedPhaseLinear(compute="int8"): the decoded coefficients through
    quantize_rows, the activations through linear_int8."""
    from rpfq_review_b200 import PackedPhaseLinear, ops
    from rpfq_review_b200.packing import random_packed
    layer = random_packed(n_c, k_c, seed=3, device=cuda)
    mod = PackedPhaseLinear.from_packed(layer, compute="int8", activation="gelu")
    x = torch.randn(2, 33, 2 * k_c, generator=torch.Generator().manual_seed(0)).to(cuda)
    w, ws = ops.quantize_rows(ops.prepack(layer))
    for inp in (x, x.half()):
        y = mod(inp)
        assert y.dtype == inp.dtype and y.shape == (2, 33, 2 * n_c)
        assert torch.equal(y, ops.linear_int8(inp, w, ws, layer.bias.float(), activation="gelu", out_dtype=inp.dtype))
    assert mod.dense is None and mod.codes8.dtype == torch.int8
    # near the fp16 layer: 8-bit steps of operands whose largest value is a few times their rms
    ref = PackedPhaseLinear.from_packed(layer, activation="gelu")(x).double()
    assert ((mod(x).double() - ref).norm() / ref.norm()).item() < 0.05


@pytest.mark.parametrize("m,n,k", [(1, 5, 1), (1, 1000, 768), (2, 33, 17), (3, 4097, 100), (4, 64, 4096), (5, 31, 257),
                                   (7, 1000, 1003), (8, 770, 2048), (8, 9, 12288), (8, 20, 12304), (4, 5, 24576),
                                   (4, 6, 24592), (1, 7, 98304), (1, 7, 98320)])
def test_few_rows_same_bits(cuda, m, n, k):
    """Few rows run on their own kernel (and quantize inside it); rows of a larger
    product on the tensor cores: the same bits, for codes, fp16 and fp32."""
    from rpfq_review_b200 import ops
    g = torch.Generator().manual_seed(m + n + k)
    x = torch.randn(40, k, generator=g).to(cuda)
    w, ws = ops.quantize_rows((torch.randn(n, k, generator=g) * 0.1).to(cuda))
    bias = torch.randn(n, generator=g).to(cuda)
    for src in (x, x.half()):
        xq, xs = ops.quantize_rows(src)
        for dtype in (torch.float16, torch.float32):
            res = torch.randn(40, n, generator=g).to(dtype).to(cuda)
            many = ops.gemm_int8(xq, xs, w, ws, bias, res, "gelu", out_dtype=dtype)
            few = ops.gemm_int8(xq[3:3 + m], xs[3:3 + m], w, ws, bias, res[3:3 + m], "gelu", out_dtype=dtype)
            assert torch.equal(few, many[3:3 + m])
            assert torch.equal(ops.linear_int8(src[3:3 + m], w, ws, bias, res[3:3 + m], "gelu", out_dtype=dtype), few)
            odd = torch.zeros(m, k + 3, dtype=src.dtype, device=cuda)[:, 1:1 + k]
            odd.copy_(src[3:3 + m])
            assert torch.equal(ops.linear_int8(odd, w, ws, bias, res[3:3 + m], "gelu", out_dtype=dtype), few)


@pytest.mark.parametrize("m,n,k", [(1, 40, 128), (3, 130, 1025), (9, 1000, 2048), (130, 200, 257), (200, 64, 4000), (300, 333, 900)])
def test_gemm_int8_tiles_and_splits_same_bits(cuda, m, n, k):
    """Every tile width and number of k parts (more parts than k-blocks included) gives
    the same bits: the sums are exact."""
    from rpfq_review_b200 import _lib, ops
    g = torch.Generator().manual_seed(m + n + k)
    x = torch.randn(m, k, generator=g).to(cuda)
    xq, xs = ops.quantize_rows(x)
    w, ws = ops.quantize_rows((torch.randn(n, k, generator=g) * 0.1).to(cuda))
    bias = torch.randn(n, generator=g).to(cuda)
    for dtype in (torch.float16, torch.float32):
        res = torch.randn(m, n, generator=g).to(dtype).to(cuda)
        want = ops.gemm_int8(xq, xs, w, ws, bias, res, "gelu", out_dtype=dtype)
        _check(want, _product_ref(xq, xs, w, ws, bias, "gelu", res, dtype))
        for bn, splits in [(b, s) for b in (64, 128) for s in range(1, 9)] + [(256, 0), (256, 1), (0, 3)]:
            y = ops.gemm_int8(xq, xs, w, ws, bias, res, "gelu", out_dtype=dtype, block_n=bn, split_k=splits)
            assert torch.equal(y, want), (bn, splits)
        assert torch.equal(ops.linear_int8(x, w, ws, bias, res, "gelu", out_dtype=dtype, block_n=64, split_k=2), want)
        inplace = res.clone()
        ops.gemm_int8(xq, xs, w, ws, bias, inplace, "gelu", out=inplace, split_k=4)
        assert torch.equal(inplace, want)
    torch.cuda.synchronize()
    assert _lib.device_error() == 0


def test_int8_refusals(cuda):
    from rpfq_review_b200 import ops
    xq, xs, wq, ws = _operands(cuda, 4, 6, 32)
    x = torch.randn(4, 32, device=cuda)
    bad = [
        lambda: ops.gemm_int8(x, xs, wq, ws), lambda: ops.gemm_int8(xq, xs, x, ws),
        lambda: ops.gemm_int8(xq, xs.half(), wq, ws), lambda: ops.gemm_int8(xq, xs, wq, ws.double()),
        lambda: ops.gemm_int8(xq, xs[:3], wq, ws), lambda: ops.gemm_int8(xq, xs, wq, ws[:5]),
        lambda: ops.gemm_int8(xq[:, :31], xs, wq, ws), lambda: ops.gemm_int8(xq, xs, wq[0], ws),
        lambda: ops.gemm_int8(xq, xs, wq[:, :0], ws), lambda: ops.gemm_int8(xq, xs, wq, ws, bias=ws[:5]),
        lambda: ops.gemm_int8(xq, xs, wq, ws, bias=ws.double()), lambda: ops.gemm_int8(xq, xs, wq, ws, bias=ws.cpu()),
        lambda: ops.gemm_int8(xq, xs, wq, ws, activation="relu"),
        lambda: ops.gemm_int8(xq, xs, wq, ws, out_dtype=torch.bfloat16),
        lambda: ops.gemm_int8(xq, xs, wq, ws, out=torch.empty(3, 6, device=cuda)),
        lambda: ops.gemm_int8(xq, xs, wq, ws, out=torch.empty(4, 5, device=cuda)),
        lambda: ops.gemm_int8(xq, xs, wq, ws, out=torch.empty(6, 4, device=cuda).t()),
        lambda: ops.gemm_int8(xq, xs, wq, ws, residual=torch.zeros(3, 6, device=cuda)),
        lambda: ops.gemm_int8(xq, xs, wq, ws, block_n=32), lambda: ops.gemm_int8(xq, xs, wq, ws, split_k=9),
        lambda: ops.linear_int8(xq, wq, ws), lambda: ops.linear_int8(x.double(), wq, ws),
        lambda: ops.linear_int8(x.bfloat16(), wq, ws), lambda: ops.linear_int8(x[:, :31], wq, ws),
        lambda: ops.linear_int8(x.requires_grad_(), wq, ws), lambda: ops.quantize_rows(x.detach()[:, :0]),
        lambda: ops.quantize_rows(x.detach().requires_grad_()), lambda: ops.quantize_rows(xq),
        lambda: ops.quantize_rows(torch.tensor(1.0, device=cuda))]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"case {i} was accepted")
    with pytest.raises(NotImplementedError):  # residual and output of different types
        ops.gemm_int8(xq, xs, wq, ws, residual=torch.zeros(4, 6, device=cuda))
    with torch.no_grad():
        ops.linear_int8(x, wq, ws)
    out = torch.ops.rpfq.linear_int8(x.detach(), wq, ws, None, None, 1, True)
    assert torch.equal(out, ops.linear_int8(x.detach(), wq, ws, activation="gelu", out_dtype=torch.float32))
    q, s = torch.ops.rpfq.quantize_rows(x.detach())
    assert torch.equal(torch.ops.rpfq.gemm_int8(q, s, wq, ws, None, None, 1, True), out)


def test_gelu_over_its_range(cuda):
    """The GELU of the product over all magnitudes, infinities and NaN: one code times
    w_scale gives the argument exactly."""
    from rpfq_review_b200 import ops
    v = torch.cat([torch.linspace(-12, 12, 20001), torch.logspace(-30, 30, 600), -torch.logspace(-30, 30, 600),
                   torch.tensor([float("inf"), float("-inf"), float("nan"), 0.0])])
    one = torch.ones(1, 1, dtype=torch.int8, device=cuda)
    w = torch.ones(v.numel(), 1, dtype=torch.int8, device=cuda)
    for rows in (1, 20, 40000):  # few rows, tiles, CTA pairs
        n = 21205 if rows < 40000 else 256
        vv = v[:n] if n == v.numel() else v[:: v.numel() // n][:n]
        y = ops.gemm_int8(one.expand(rows, 1), torch.ones(rows, device=cuda), w[:n], vv.to(cuda), activation="gelu",
                          out_dtype=torch.float32)[rows // 2].cpu().double()
        x = vv.double()
        ref = x * torch.special.ndtr(x)
        fin = torch.isfinite(vv)
        assert ((y - ref).abs()[fin] <= 2.0 ** -20 * x.abs()[fin] + 1e-37).all()
        if n == v.numel():
            assert y[-4] == float("inf") and y[-3] == 0 and torch.isnan(y[-2]) and y[-1] == 0


def test_int8_vectors_and_shared_buffers(cuda):
    """One-dimensional inputs, a broadcast residual, input and output columns of one
    buffer; an output over its own input is refused."""
    from rpfq_review_b200 import ops
    w, ws = ops.quantize_rows(torch.randn(48, 64, device=cuda))
    x = torch.randn(40, 64, device=cuda)
    y = ops.linear_int8(x, w, ws, out_dtype=torch.float32)
    assert torch.equal(ops.linear_int8(x[3], w, ws, out_dtype=torch.float32), y[3])
    q, s = ops.quantize_rows(x[3])
    assert q.shape == (64,) and s.shape == ()
    assert torch.equal(ops.gemm_int8(q, s, w, ws, out_dtype=torch.float32), y[3])
    assert torch.equal(ops.linear_int8(x.t().contiguous().t()[5], w, ws, out_dtype=torch.float32), y[5])
    row = torch.randn(48, device=cuda)
    assert torch.equal(ops.linear_int8(x, w, ws, residual=row.expand(40, 48), out_dtype=torch.float32),
                       ops.linear_int8(x, w, ws, residual=row.repeat(40, 1), out_dtype=torch.float32))
    for rows in (2, 40):
        both = torch.zeros(rows, 112, device=cuda)
        both[:, :64] = x[:rows]
        ops.linear_int8(both[:, :64], w, ws, out=both[:, 64:])
        assert torch.equal(both[:, 64:], y[:rows]) and torch.equal(both[:, :64], x[:rows])
        with pytest.raises(ValueError, match="overlap"):
            ops.linear_int8(both[:, :64], w, ws, out=both[:, 40:88])


def test_int8_past_31_bits(cuda):
    """Rows whose elements lie past 2^31: the last ones equal a small call's, in place too."""
    from rpfq_review_b200 import _lib, ops
    m, n, k = 530000, 4100, 32
    x, xs = ops.quantize_rows(torch.randn(m, k, device=cuda))
    w, ws = ops.quantize_rows(torch.randn(n, k, device=cuda))
    y = ops.gemm_int8(x, xs, w, ws)  # 2.17e9 elements
    assert torch.equal(y[-300:], ops.gemm_int8(x[-300:], xs[-300:], w, ws))
    ops.gemm_int8(x, xs, w, ws, residual=y, out=y)
    assert torch.equal(y[-300:], ops.gemm_int8(x[-300:], xs[-300:], w, ws, residual=ops.gemm_int8(x[-300:], xs[-300:], w, ws)))
    q, s = ops.quantize_rows(y)
    want = ops.quantize_rows(y[-3:])
    assert torch.equal(q[-3:], want[0]) and torch.equal(s[-3:], want[1])
    del q
    far = y.view(-1)[: 129 * 16_800_000].view(129, 16_800_000)[:, -64:]  # rows 33.6 MB apart: the tile kernel
    out = far[:, :40]
    ops.gemm_int8(x[:129], xs[:129], w[:40], ws[:40], out=out)
    assert torch.equal(out, ops.gemm_int8(x[:129], xs[:129], w[:40], ws[:40]))
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
