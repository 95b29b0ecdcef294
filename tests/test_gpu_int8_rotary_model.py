"""GPU test of the 8-bit linears and the rotary positions together, as a model
runs them: ``PackedViT(compute="int8", rotary=...)`` against the same forward
with every new operator replaced by its float64 form.

Tolerance: where the two differ by an fp16 rounding (2^-11 of a value) a code can
flip by one step. With amax about 4 rms, a step is 4 / 127 of the rms and a value
is within 2^-11 of a tie for about 2^-11 x 127 / 4 = 1.6 % of the codes, so the
flips add sqrt(0.016) x 3.1 % = 0.4 % of the rms per product; the eight products
on the way to the logits (two blocks) add up to sqrt(8) x 0.4 % = 1.1 % when
nothing is averaged out. The bar is 3 %."""

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


def _tiny():
    from rpfq_review_b200.vit import ViTConfig
    return ViTConfig("tiny", dim=192, depth=2, heads=3, mlp=384, img=64, patch=16, classes=10)


def _linear(mod, x, residual=None):
    from rpfq_review_b200 import ops
    rows = lambda t: (t.double() / (s := t.double().abs().amax(-1, keepdim=True) / 127)).round() * s  # noqa: E731
    w = ops.prepack(mod.packed())
    y = rows(x) @ rows(w).t() + mod.bias.double()
    if mod.activation == "gelu":
        y = F.gelu(y)
    return y if residual is None else y + residual


def _turn(x, pos, f, layout):
    angle = (pos.double()[:, torch.arange(f.numel()) * 2 // f.numel()] * f).unsqueeze(1)
    i = torch.arange(f.numel()) * (1 if layout == "half" else 2)
    j = i + (f.numel() if layout == "half" else 1)
    y = x.clone()
    y[..., i] = x[..., i] * angle.cos() - x[..., j] * angle.sin()
    y[..., j] = x[..., j] * angle.cos() + x[..., i] * angle.sin()
    return y


def _forward_ref(model, images, layout):
    from rpfq_review_b200 import ops
    cfg, B = model.cfg, images.shape[0]
    d, H, L = cfg.dim, cfg.heads, cfg.tokens
    patches = ops.patch_unfold(images, cfg.patch).double()
    x = (patches @ model.patch_w.double().t() + model.patch_b.double())
    x = torch.cat([model.cls_tokens.double().expand(B, -1, -1), x], 1) + model.pos_embed.double()
    norm = lambda t, w, b: F.layer_norm(t, (d,), w.double(), b.double(), cfg.eps)  # noqa: E731
    for blk in model.blocks:
        qkv = _linear(blk.qkv, norm(x, blk.norm1_w, blk.norm1_b)).view(B, L, 3, H, d // H)
        q, k = (_turn(qkv[:, :, i], *model._rotary_table(images.device), layout) for i in (0, 1))
        q, k, v = (t.transpose(1, 2) for t in (q, k, qkv[:, :, 2]))
        a = torch.softmax(q @ k.transpose(-2, -1) / 8.0, -1) @ v
        x = _linear(blk.proj, a.transpose(1, 2).reshape(B, L, d), x)
        h = norm(x, blk.norm2_w, blk.norm2_b)
        x = _linear(blk.fc2, _linear(blk.fc1, h), x)
    return _linear(model.head, norm(x[:, 0], model.norm_w, model.norm_b))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("attention", ["sdpa", "rpfq"])
def test_int8_rotary_vit(cuda, layout, attention):
    from rpfq_review_b200 import _lib
    from rpfq_review_b200.vit import PackedViT
    kw = dict(seed=1, attention=attention, compute="int8")
    model = PackedViT(_tiny(), cuda, rotary=dict(base=100.0, layout=layout), **kw)
    images = torch.randn(5, 3, 64, 64, generator=torch.Generator().manual_seed(2)).to(cuda)
    y = model(images)
    assert y.shape == (5, 10) and y.dtype == torch.float32
    ref = _forward_ref(model, images, layout)
    assert ((y.double() - ref).norm() / ref.norm()).item() < 0.03
    g = torch.cuda.CUDAGraph()
    static = images.clone()
    model(static)
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        z = model(static)
    static.copy_(images)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(z, y)
    assert not torch.equal(PackedViT(_tiny(), cuda, **kw)(images), y)
    assert _lib.device_error() == 0


def test_int8_rotary_vit_follows_its_weights(cuda):
    """Planes loaded into a model that has run, a cast and a move of the module: the codes
    are those of the planes, the angles stay in 64 bits."""
    from rpfq_review_b200.vit import PackedViT
    kw = dict(compute="int8", rotary=dict(base=100.0))
    a, b = PackedViT(_tiny(), cuda, seed=1, **kw), PackedViT(_tiny(), cuda, seed=2, **kw)
    images = torch.randn(2, 3, 64, 64, generator=torch.Generator().manual_seed(2)).to(cuda)
    ya, yb = a(images), b(images)
    assert not torch.equal(ya, yb)
    a.load_state_dict(b.state_dict())
    assert torch.equal(a(images), yb)
    a.half()
    assert torch.equal(a(images), yb)
    a.cpu()
    a.to(cuda)
    assert torch.equal(a(images), yb)
