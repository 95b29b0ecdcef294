"""The 8-bit linear path and the rotary positions, measured call by call.

Three operators that serve a quantized transformer next to the packed layers:

* ``gemm_int8``: ``act(x_scale[m] w_scale[n] (xq wq^T) + bias) (+ residual)`` of
  int8 codes with one scale per token and one per output channel;
* ``linear_int8``: the same from 16- or 32-bit activations, whose rows are
  first quantized to 8 bits (per row: s = 127 / amax, q = rint(x s));
* ``rotary``: rotation of query and key heads by their positions, in both
  pair layouts, over a part of the head, along one axis or two, and its
  transpose (the gradient).

``run`` computes them in elementary torch operations where ``own`` is false
and through ``rpfq_review_b200.ops`` where it is true.
"""

import math

import torch

own = False

TINY = 1e-30  # smallest row maximum that sets a scale: rows of zeros get codes and outputs of zero

HALF, FULL = "float16", "float32"


def listed():
    product = dict(op="gemm_int8", act="none", bias="float16", residual=False, out=HALF)
    linear = dict(op="linear_int8", act="none", bias="float32", residual=False, x=HALF, out=HALF)
    rotary = dict(op="rotary", layout="half", axes=1, batch=1, shared=True, dtype=HALF, start=0, transpose=False,
                  magnitude=1.0, base=10000.0, factor=1.0)
    return [
        # the classification head on one image's class token: latency
        dict(product, name="product_one_token", m=1, k=768, n=1000, out=FULL),
        # fc1 of one image (ViT-L): exact GELU in the epilogue, weights read once
        dict(product, name="product_one_image_gelu", m=197, k=1024, n=4096, act="gelu"),
        # qkv of 32 images (ViT-B): an ordinary batch
        dict(product, name="product_batch_qkv", m=6304, k=768, n=2304, bias="float32"),
        # fc2 of 256 images (ViT-L) added to the fp32 residual stream: the largest product
        dict(product, name="product_full_batch_residual", m=50432, k=4096, n=1024, residual=True, out=FULL),
        # rows, columns and depth that fill no tile, no bias
        dict(product, name="product_ragged", m=1571, k=1003, n=1001, bias="none"),
        # one token through a projection, quantized on the way in
        dict(linear, name="linear_one_token", m=1, k=768, n=768),
        # fc1 of 256 images (ViT-L) from the LayerNorm's fp16 rows
        dict(linear, name="linear_full_batch_gelu", m=50432, k=1024, n=4096, act="gelu"),
        # odd sizes in fp32 throughout, with a residual
        dict(linear, name="linear_ragged_fp32", m=613, k=390, n=771, residual=True, x=FULL, out=FULL),
        # one new token for each of 16 sequences far into a long context, base raised for it
        dict(rotary, name="rotary_one_token", batch=16, length=1, heads=32, dim=128, rot=128, shared=False,
             start=131072, base=500000.0),
        # query and key heads of the qkv rows of 256 images (ViT-L), positions on the patch grid
        dict(rotary, name="rotary_patch_grid", batch=256, length=197, heads=32, dim=64, rot=64, axes=2, base=100.0),
        # a long sequence, neighbouring pairs, half of each head, frequencies divided for the length
        dict(rotary, name="rotary_long_interleaved", length=65531, heads=24, dim=128, rot=64, layout="interleaved",
             factor=8.0, magnitude=1.2),
        # the gradient of heads whose pairs fill no 16-byte chunk, in fp32
        dict(rotary, name="rotary_gradient_fp32", batch=8, length=1001, heads=12, dim=80, rot=40, dtype=FULL,
             transpose=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["gemm_int8", "linear_int8", "rotary"])
    if op == "rotary":
        dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
        axes = rng.choice([1, 1, 2])
        rot = rng.choice([dim, dim, dim // 2, dim // 4 * 3])
        rot -= rot % (2 * axes)
        heads = rng.randint(1, 48)
        length = _log(rng, 1, 65536)
        batch = _log(rng, 1, 256)
        dtype = rng.choice([HALF, FULL])
        most = 65531 * 24 * 128 // (2 if dtype == FULL else 1)
        while batch * length * heads * dim > most:
            batch, length, heads = max(1, batch // 2), max(1, length * 3 // 4), max(1, heads * 3 // 4)
        return dict(op=op, layout=rng.choice(["half", "interleaved"]), axes=axes, batch=batch, length=length,
                    heads=heads, dim=dim, rot=rot, shared=rng.random() < 0.5, dtype=dtype,
                    start=rng.choice([0, 0, rng.randrange(1 << 20)]), transpose=rng.random() < 0.3,
                    magnitude=rng.choice([1.0, 1.2]), base=rng.choice([100.0, 10000.0, 500000.0]),
                    factor=rng.choice([1.0, 8.0]))
    m, k, n = _log(rng, 1, 50432), _log(rng, 32, 4096), _log(rng, 8, 4096)
    while m * k * n > 50432 * 1024 * 4096:
        m = m * 3 // 4
    case = dict(op=op, m=m, k=k, n=n, act=rng.choice(["none", "gelu"]), residual=rng.random() < 0.4,
                bias=rng.choice(["none", "float16", "float32"]), out=rng.choice([HALF, FULL]))
    if op == "linear_int8":
        case["x"] = rng.choice([HALF, FULL])
    return case


def _dtype(name):
    return getattr(torch, name)


def _codes(rows, cols, g):
    """int8 codes [rows, cols] of a row-quantized normal matrix, in rows that start on 16 bytes."""
    buf = torch.zeros((rows, -(-cols // 16) * 16), dtype=torch.int8, device="cuda")
    q = torch.randn((rows, cols), generator=g, device="cuda").mul_(34.0).round_().clamp_(-127, 127)
    buf[:, :cols] = q
    return buf[:, :cols]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def rand(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    s = dict(case)
    if case["op"] == "rotary":
        B, L, H, D = case["batch"], case["length"], case["heads"], case["dim"]
        # the heads lie in a wider row, as query and key heads do in the rows of a qkv product
        s["x"] = randn(B, L, H + (H + 1) // 2, D).to(_dtype(case["dtype"]))[:, :, :H]
        at = torch.arange(L, device="cuda") + case["start"]
        if not case["shared"]:  # every sequence at its own place
            at = at + torch.randint(0, 4096, (B, 1), generator=g, device="cuda")
        if case["axes"] == 2:  # row and column of a token on the patch grid
            side = max(1, math.isqrt(L))
            at = torch.stack([at // side, at % side], -1)
        s["positions"] = at.to(torch.int32)
        per = case["rot"] // 2 // case["axes"]
        j = torch.arange(per, dtype=torch.float64, device="cuda")
        s["inv_freq"] = (case["base"] ** (-j / per) / case["factor"]).repeat(case["axes"])
        return s
    m, k, n = case["m"], case["k"], case["n"]
    s["wq"] = _codes(n, k, g)
    s["w_scale"] = (0.5 + rand(n)) * (0.1 / 127 / math.sqrt(k / 256))
    if case["op"] == "gemm_int8":
        s["xq"] = _codes(m, k, g)
        s["x_scale"] = (0.5 + rand(m)) * (4.0 / 127)
    else:
        # rows of different magnitudes, a few channels far larger than the others
        s["x"] = (randn(m, k) * (0.25 + rand(m, 1)) * torch.where(rand(k) < 0.01, 6.0, 1.0)).to(_dtype(case["x"]))
    s["bias_values"] = None if case["bias"] == "none" else (0.5 * randn(n)).to(_dtype(case["bias"]))
    s["residual_values"] = randn(m, n).to(_dtype(case["out"])) if case["residual"] else None
    return s


def _quantized(x):
    """Codes (as fp32 values) and scales of the rows of x, in fp32."""
    x = x.float()
    amax = x.abs().amax(dim=1, keepdim=True).clamp_min(TINY)
    return torch.round(x * (amax.reciprocal() * 127.0)), (amax / 127.0).squeeze(1)


def _plain_product(s):
    if s["op"] == "linear_int8":
        xq, x_scale = _quantized(s["x"])
    else:
        xq, x_scale = s["xq"].float(), s["x_scale"]
    v = (xq @ s["wq"].float().t()) * x_scale[:, None] * s["w_scale"]
    if s["bias_values"] is not None:
        v = v + s["bias_values"].float()
    if s["act"] == "gelu":
        v = 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if s["residual_values"] is not None:
        v = v + s["residual_values"].float()
    return v.to(_dtype(s["out"]))


def _angles(s):
    """positions x frequencies in 64 bits, [.., L, 1, pairs]: far positions lose their angle in 32."""
    at = s["positions"].double()
    if s["axes"] == 2:
        at = at.repeat_interleave(s["rot"] // 4, dim=-1)
    else:
        at = at.unsqueeze(-1)
    return (at * s["inv_freq"]).unsqueeze(-2)


def _plain_rotary(s):
    angle = _angles(s)
    cos = (torch.cos(angle) * s["magnitude"]).float()
    sin = (torch.sin(angle) * s["magnitude"]).float()
    if s["transpose"]:
        sin = -sin
    x = s["x"].float()
    rot, rest = x[..., : s["rot"]], x[..., s["rot"]:]
    if s["layout"] == "half":
        a, b = rot[..., : s["rot"] // 2], rot[..., s["rot"] // 2:]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    else:
        a, b = rot[..., 0::2], rot[..., 1::2]
        y = torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)
    return y.to(s["x"].dtype)


def run(state):
    if not own:
        return _plain_rotary(state) if state["op"] == "rotary" else _plain_product(state)
    from rpfq_review_b200 import ops

    if state["op"] == "rotary":
        return ops.rotary(state["x"], state["positions"], state["inv_freq"], layout=state["layout"],
                          axes=state["axes"], magnitude=state["magnitude"], transpose=state["transpose"])
    more = dict(bias=state["bias_values"], residual=state["residual_values"], activation=state["act"],
                out_dtype=_dtype(state["out"]))
    if state["op"] == "gemm_int8":
        return ops.gemm_int8(state["xq"], state["x_scale"], state["wq"], state["w_scale"], **more)
    return ops.linear_int8(state["x"], state["wq"], state["w_scale"], **more)


def work(case):
    if case["op"] == "rotary":
        tokens = case["batch"] * case["length"]
        size = 2 if case["dtype"] == HALF else 4
        at = 4 * case["axes"] * (case["length"] if case["shared"] else tokens)
        return {"bytes": 2 * tokens * case["heads"] * case["dim"] * size + at + 4 * case["rot"],
                "flops": 3 * tokens * case["heads"] * case["rot"]}
    m, k, n = case["m"], case["k"], case["n"]
    size = {HALF: 2, FULL: 4, "none": 0}
    given = m * (k + 4) if case["op"] == "gemm_int8" else m * k * size[case["x"]]
    out = m * n * size[case["out"]] * (2 if case["residual"] else 1)
    return {"bytes": given + n * (k + 4 + size[case["bias"]]) + out, "flops": 2 * m * n * k}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        x = s["x"].double()
        at = s["positions"].double().reshape(-1, case["length"], case["axes"])
        pairs = case["rot"] // 2
        axis = torch.arange(pairs, device="cuda") * case["axes"] // pairs
        turn = torch.polar(torch.full_like(at[..., axis], case["magnitude"]), at[..., axis] * s["inv_freq"])
        if case["transpose"]:
            turn = turn.conj()
        first = torch.arange(pairs, device="cuda") * (1 if case["layout"] == "half" else 2)
        second = first + (pairs if case["layout"] == "half" else 1)
        y = x.clone()
        z = torch.complex(x[..., first], x[..., second]) * turn.unsqueeze(-2)
        y[..., first], y[..., second] = z.real, z.imag
        return y
    if case["op"] == "linear_int8":
        # the codes are defined by fp32 steps: fl(fl(1 / amax) 127), fl(x s), half to even
        x = s["x"].to(torch.float32)
        amax = torch.maximum(x.max(dim=1).values, -x.min(dim=1).values)
        amax = torch.where(amax < TINY, torch.full_like(amax, TINY), amax)
        code = torch.round(x * (torch.ones_like(amax) / amax * torch.full_like(amax, 127.0)).unsqueeze(1)).double()
        x_scale = amax.double() / 127.0
    else:
        code, x_scale = s["xq"].double(), s["x_scale"].double()
    y = torch.mm(code, s["wq"].double().T)
    y *= torch.outer(x_scale, s["w_scale"].double())
    if s["bias_values"] is not None:
        y += s["bias_values"].double()
    if case["act"] == "gelu":
        y = y * torch.special.ndtr(y)
    if s["residual_values"] is not None:
        y += s["residual_values"].double()
    return y
