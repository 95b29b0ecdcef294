"""CPU test of the polynomial that the 8-bit product's GELU is made of: the coefficients in the
source, in fp32 Horner steps, against float64."""

import os
import re

import numpy as np
import torch

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rpfq_review_b200", "csrc",
                      "gemm_i8.cuh")


def _coefficients():
    text = open(SOURCE).read()
    body = text[text.index("void gelu_log_pair("):]
    body = body[:body.index("f2_unpack(q, q0, q1)")]
    return [np.float32(c) for c in re.findall(r"c2\((-?[0-9.e+-]+)f\)", body)]


def test_gelu_before_its_last_roundings():
    """max(v, 0) - a 2^Q(a), with Q in fp32 fused steps and the rest exact, is within
    0.75 x 2^-24 |v| of v Phi(v)."""
    c = _coefficients()
    assert len(c) == 9
    v = np.concatenate([np.linspace(-14, 14, 400001), -np.logspace(-6, 1.2, 100000), np.logspace(-6, 1.2, 100000)])
    v = v[v != 0].astype(np.float32)
    a = -np.maximum(-np.abs(v), np.float32(-64)).astype(np.float64)
    q = np.full_like(v, c[0])
    for ci in c[1:]:
        # products of two fp32 values are exact in fp64; the sum rounds there to 2^-53 first
        q = (-a * q.astype(np.float64) + np.float64(ci)).astype(np.float32)
    y = np.maximum(v, 0).astype(np.float64) - a * np.exp2(q.astype(np.float64))
    x = torch.from_numpy(v.astype(np.float64))
    ref = (x * torch.special.ndtr(x)).numpy()
    worst = (np.abs(y - ref) / a).max() * 2 ** 24
    assert 0.5 < worst <= 0.75, worst
