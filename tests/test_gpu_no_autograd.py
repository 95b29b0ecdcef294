"""GPU tests: the 8-bit path and the rotary positions have no autograd, and say so for every
tensor that asks for a derivative."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _calls(cuda):
    """Name -> (function of the tensors that a derivative could be asked for, those tensors)."""
    from rpfq_review_b200 import ops
    m, n, k = 5, 16, 32
    xq, xs = ops.quantize_rows(torch.randn(m, k, device=cuda))
    w, ws = ops.quantize_rows(torch.randn(n, k, device=cuda))
    x, bias, res = torch.randn(m, k, device=cuda), torch.randn(n, device=cuda), torch.randn(m, n, device=cuda)
    out = torch.empty(m, n, device=cuda)
    heads, pos, f = torch.randn(7, 2, 16, device=cuda), torch.rand(7, device=cuda), ops.rotary_frequencies(16, device=cuda)[0]
    turned = torch.empty_like(heads)
    kw = dict(out_dtype=torch.float32)
    return {
        "quantize_rows": (lambda x: ops.quantize_rows(x), dict(x=x)),
        "gemm_int8": (lambda xs, ws, bias, res, out: ops.gemm_int8(xq, xs, w, ws, bias, res, out=out, **kw),
                      dict(xs=xs, ws=ws, bias=bias, res=res, out=out)),
        "linear_int8": (lambda x, ws, bias, res, out: ops.linear_int8(x, w, ws, bias, res, out=out, **kw),
                        dict(x=x, ws=ws, bias=bias, res=res, out=out)),
        "rotary": (lambda x, pos, f, out: ops.rotary(x, pos, f, out=out), dict(x=heads, pos=pos, f=f, out=turned)),
        "op gemm_int8": (lambda xs, ws, bias, res: torch.ops.rpfq.gemm_int8(xq, xs, w, ws, bias, res, 0, True),
                         dict(xs=xs, ws=ws, bias=bias, res=res)),
        "op linear_int8": (lambda x, ws, bias, res: torch.ops.rpfq.linear_int8(x, w, ws, bias, res, 0, True),
                           dict(x=x, ws=ws, bias=bias, res=res)),
        "op rotary": (lambda x, pos, f: torch.ops.rpfq.rotary(x, pos, f), dict(x=heads, pos=pos, f=f)),
        "op quantize_rows": (lambda x: torch.ops.rpfq.quantize_rows(x), dict(x=x))}


def test_gradients_are_refused(cuda):
    for name, (call, tensors) in _calls(cuda).items():
        call(**tensors)
        for which in tensors:
            given = dict(tensors, **{which: tensors[which].clone().requires_grad_()})
            with pytest.raises(ValueError, match="no autograd"):
                call(**given)
                pytest.fail(f"{name} took {which} with a gradient")
            with torch.no_grad():
                call(**given)


def test_tangents_are_refused(cuda):
    """Forward mode: a dual tensor's tangent would be dropped."""
    import torch.autograd.forward_ad as fwd
    for name, (call, tensors) in _calls(cuda).items():
        with fwd.dual_level(), torch.no_grad():
            call(**tensors)
            for which, t in tensors.items():
                given = dict(tensors, **{which: fwd.make_dual(t.clone(), torch.ones_like(t))})
                with pytest.raises(ValueError, match="no autograd"):
                    call(**given)
                    pytest.fail(f"{name} took {which} with a tangent")


def test_written_outputs_are_seen_by_autograd(cuda):
    """A backward pass that needs the old values of a tensor given as ``out`` says so."""
    from rpfq_review_b200 import ops
    calls = _calls(cuda)
    for name in ("gemm_int8", "linear_int8", "rotary"):
        call, tensors = calls[name]
        out = tensors["out"].zero_()
        a = torch.ones_like(out).requires_grad_()
        loss = (a * out).sum()
        with torch.no_grad():
            version = out._version
            assert call(**tensors) is out and out._version > version
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()
    heads, f = torch.randn(7, 2, 16, device=cuda), ops.rotary_frequencies(16, device=cuda)[0]
    version = heads._version
    ops.rotary(heads, torch.arange(7, device=cuda), f, out=heads)
    assert heads._version > version
    rows = torch.randn(7, 64, device=cuda)
    version = rows._version
    part = rows.view(7, 4, 16)[:, :2]
    ops.rotary(part, torch.arange(7, device=cuda), f, out=part)
    assert rows._version > version
    with torch.inference_mode():
        fresh = torch.randn(7, 2, 16, device=cuda)
        ops.rotary(fresh, torch.arange(7, device=cuda), f, out=fresh)
