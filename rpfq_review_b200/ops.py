"""PyTorch entry points over the C ABI (``include/rpfq_b200.h``).

Functional wrappers (:func:`prepack`, :func:`gemm`, :func:`act_quant`,
:func:`wide_linear`, the 8-bit linear path :func:`quantize_rows`,
:func:`gemm_int8`, :func:`linear_int8`, and :func:`rotary` positions) and the
``torch.ops.rpfq`` operators, registered with
``torch.library`` in the same way the reference registers its GPU op
(``Library("quant", "DEF")`` + ``define`` + ``impl``,
RPFQ-ViT-main/quant_models/kernel.py:599-605). Every op has a CUDA
implementation only: calling one on CPU tensors fails in the dispatcher, and
a missing library raises — there is no fallback path.
"""

from __future__ import annotations

import ctypes
import os
import math

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _lib
from .packing import PackedLayer

_ACT = {"none": _lib.ACT_NONE, "gelu": _lib.ACT_GELU, None: _lib.ACT_NONE,
        _lib.ACT_NONE: _lib.ACT_NONE, _lib.ACT_GELU: _lib.ACT_GELU}
_ROUND = {"rne": _lib.ROUND_NEAREST_EVEN, "ties_away": _lib.ROUND_TIES_AWAY}


def _stream(device: torch.device) -> int:
    index = device.index
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device() if index is None else index)


class LaunchTimer:
    """Optional instrumentation: a count of every kernel this library launches
    and, with ``events=True``, CUDA events around every GEMM launch. Events
    are created with ``external=True`` so that they become event-record nodes
    when the launches are captured into a CUDA graph (timings are then those
    of the last replay). Event nodes sit between the kernel nodes and so cut
    the programmatic (PDL) chaining of consecutive launches: time a graph
    captured with ``events=False`` and read GEMM times from a separate one."""

    def __init__(self, events: bool = True):
        self.gemm_events: list[tuple[torch.cuda.Event, torch.cuda.Event, int]] = []
        self.launches = 0
        self.events = events

    def gemm_ms_and_flops(self) -> tuple[float, int]:
        ms = sum(s.elapsed_time(e) for s, e, _ in self.gemm_events)
        return ms, sum(f for _, _, f in self.gemm_events)


_timer: LaunchTimer | None = None


def set_launch_timer(timer: LaunchTimer | None) -> None:
    global _timer
    _timer = timer


def _count_launch(n: int = 1) -> None:
    if _timer is not None:
        _timer.launches += n


# Largest row count of the fused decode path (``dense=None``); the C ABI
# rejects more.
FUSED_DECODE_MAX_ROWS = 256


def _p(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


# Split-K for small-M GEMMs: 0 = automatic, 1 = never, 2..8 = forced (the
# RPFQ_SPLIT_K environment variable sets the default of every call).
SPLIT_K = int(os.environ.get("RPFQ_SPLIT_K", "0"))

# One split-K workspace per (device, stream): calls on one stream run in
# order, so they can share it; calls on different streams may overlap.
_workspaces: dict[tuple[int, int], torch.Tensor] = {}


def _workspace(device: torch.device, split_k: int) -> tuple[int | None, int]:
    if split_k == 1:
        return None, 0
    key = (device.index if device.index is not None else torch.cuda.current_device(), _stream(device))
    ws = _workspaces.get(key)
    if ws is None:
        with torch.cuda.device(device):
            nbytes = int(_lib.lib().rpfq_gemm_workspace_bytes(0, 0, 0))
        # zeroed: the stream-K flag words at its end start at zero (the library
        # leaves them zero after every call)
        ws = torch.zeros(nbytes, dtype=torch.uint8, device=device)
        _workspaces[key] = ws
    return ws.data_ptr(), ws.numel()


def _require(t: torch.Tensor, name: str, dtype=torch.float16):
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (the packed phase-linear path has no CPU implementation)")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")


def _rows(x: torch.Tensor, k: int, name: str):
    """View ``x[..., k]`` as a 2-D row-major matrix with unit column stride."""
    if x.shape[-1] != k:
        raise ValueError(f"{name}: last dim {x.shape[-1]} != {k}")
    x2 = x.reshape(-1, k)
    if x2.stride(-1) != 1:
        x2 = x2.contiguous()
    ld = x2.stride(0) if x2.shape[0] > 1 else k
    return x2, ld


def layer_struct(layer: PackedLayer) -> _lib.RpfqPackedLinear:
    s = _lib.RpfqPackedLinear()
    s.n_c, s.k_c = layer.n_c, layer.k_c
    s.n_cp, s.k_cp = layer.n_cp, layer.k_cp
    s.stages, s.code_bits = layer.stages, layer.code_bits
    for i in range(layer.stages):
        for tag, arr in (("u", s.u), ("w", s.w)):
            c, gr, gi = layer.planes[f"{tag}_s{i}"]
            arr[i].codes, arr[i].gamma_real, arr[i].gamma_imag = c.data_ptr(), gr.data_ptr(), gi.data_ptr()
    return s


def prepack(layer: PackedLayer, rounding: str = "rne") -> torch.Tensor:
    """K1: packed planes -> dense fp16 ``[2 n_c, 2 k_c]`` = ``[[rr, ir], [ri, ii]]``."""
    c0 = layer.planes["u_s0"][0]
    _require(c0, "codes", torch.uint8)
    dev = c0.device
    out = torch.empty((2 * layer.n_c, 2 * layer.k_c), dtype=torch.float16, device=dev)
    s = layer_struct(layer)
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().rpfq_prepack_sm100(ctypes.byref(s), out.data_ptr(), _ROUND[rounding], _stream(dev)),
                   "rpfq_prepack_sm100")
    return out


ATTENTION_MAX_TOKENS = 256


def attention(qkv: torch.Tensor, heads: int, out: torch.Tensor | None = None) -> torch.Tensor:
    """Self-attention of the qkv GEMM output ``[B, L, 3 d]`` (fp16, head dim
    64, L <= 256) through ``rpfq_attention_sm100`` -> ``[B, L, d]`` fp16:
    softmax(q k^T / 8) v per head, heads concatenated."""
    _require(qkv, "qkv")
    if qkv.dim() != 3 or qkv.shape[-1] != 3 * 64 * heads:
        raise ValueError(f"qkv must be [B, L, 3 * heads * 64], got {tuple(qkv.shape)} for {heads} heads")
    if not qkv.is_contiguous():
        qkv = qkv.contiguous()
    B, L, _ = qkv.shape
    d = 64 * heads
    if out is None:
        out = torch.empty((B, L, d), dtype=torch.float16, device=qkv.device)
    o2, ldo = _rows(out, d, "out")
    with torch.cuda.device(qkv.device):
        _lib.check(_lib.lib().rpfq_attention_sm100(qkv.data_ptr(), B, L, heads, 64, o2.data_ptr(), ldo,
                                                   _stream(qkv.device)), "rpfq_attention_sm100")
    if B:
        _count_launch(1)
    return out


WINDOW_TOKENS = 49  # 7 x 7 Swin windows
WINDOW_HEAD_DIM = 32


def window_bias_layout(bias: torch.Tensor) -> torch.Tensor:
    """``[bm_windows, heads, 49, 49]`` additive attention bias (relative
    position bias + shift mask, natural units) -> the float32
    ``[bm_windows, heads, 16, 49, 4]`` operand of :func:`window_attention`
    (scaled by log2(e), -inf in the padding keys)."""
    n, h, L, L2 = bias.shape
    if L != WINDOW_TOKENS or L2 != WINDOW_TOKENS:
        raise ValueError("window_bias_layout: expects [bm_windows, heads, 49, 49]")
    full = torch.full((n, h, L, 64), float("-inf"), dtype=torch.float32, device=bias.device)
    full[..., :L] = bias.float() * 1.4426950408889634
    return full.view(n, h, L, 16, 4).permute(0, 1, 3, 2, 4).contiguous()


def window_attention(qkv: torch.Tensor, heads: int, bias_mask: torch.Tensor,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Swin window attention (``rpfq_window_attention_sm100``): ``qkv`` is the
    qkv GEMM output in window order, fp16 ``[windows * 49, 3 * 32 * heads]``;
    ``bias_mask`` fp32 ``[bm_windows, heads, 16, 49, 4]`` holds log2(e) times
    the relative position bias (+ shift mask) of query row i and key column j
    at ``[..., j // 4, i, j % 4]``, -inf in key columns 49..63 (window w uses
    entry ``w % bm_windows``; :func:`window_bias_layout` builds it from
    ``[bm_windows, heads, 49, 49]``). Returns fp16 ``[windows * 49, 32 * heads]``
    (or writes ``out``)."""
    _require(qkv, "qkv")
    if not bias_mask.is_cuda or bias_mask.dtype != torch.float32 or not bias_mask.is_contiguous():
        raise ValueError("window_attention: bias_mask must be a contiguous float32 CUDA tensor")
    d = WINDOW_HEAD_DIM * heads
    q2, ldq = _rows(qkv, 3 * d, "qkv")
    if ldq != 3 * d:
        raise ValueError("window_attention: qkv rows must be contiguous")
    rows = q2.shape[0]
    if rows % WINDOW_TOKENS:
        raise ValueError(f"window_attention: {rows} rows are not whole {WINDOW_TOKENS}-token windows")
    bm = bias_mask.shape
    if len(bm) != 5 or bm[1] != heads or bm[2] != 16 or bm[3] != WINDOW_TOKENS or bm[4] != 4:
        raise ValueError(f"window_attention: bias_mask must be [bm_windows, {heads}, 16, 49, 4], got {tuple(bm)}")
    if out is None:
        out = torch.empty((rows, d), dtype=torch.float16, device=qkv.device)
    o2, ldo = _rows(out, d, "out")
    with torch.cuda.device(qkv.device):
        _lib.check(_lib.lib().rpfq_window_attention_sm100(
            q2.data_ptr(), rows // WINDOW_TOKENS, heads, WINDOW_HEAD_DIM, WINDOW_TOKENS, bias_mask.data_ptr(),
            bm[0], o2.data_ptr(), ldo, _stream(qkv.device)), "rpfq_window_attention_sm100")
    if rows:
        _count_launch()
    return out


def vision_act_quant(x: torch.Tensor, salient_token_ratio: float = 0.25, background_clip_ratio: float = 0.75,
                     energy_score_weight: float = 0.5, protect_cls_token: bool = True,
                     out: torch.Tensor | None = None, return_mask: bool = False):
    """Vision-aware activation quantization (``VisionAwareActivationQuantizer``,
    quant_rpfq_vit_vision.py:26-171) of fp16 ``x`` through
    ``rpfq_vision_act_quant_sm100``. ``x`` is ``[B, T, K]`` (saliency over each
    image's T tokens when T = 1 + g*g) or ``[M, K]`` (per-token int8 scales,
    the reference's fallback for inputs that are not 3-D). ``out`` may be ``x``."""
    _require(x, "x")
    if x.dim() == 3:
        images, tokens, K = x.shape
    elif x.dim() == 2:
        images, tokens, K = x.shape[0], 1, x.shape[1]
    else:
        raise ValueError(f"x must be [B, T, K] or [M, K], got {tuple(x.shape)}")
    x2, ldx = _rows(x, K, "x")
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    y2, ldy = _rows(out, K, "out")
    mask = torch.empty(x.shape[:-1], dtype=torch.uint8, device=x.device) if return_mask else None
    L = _lib.lib()
    ws_bytes = int(L.rpfq_vision_workspace_bytes(images, tokens))
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device) if ws_bytes else None
    with torch.cuda.device(x.device):
        _lib.check(L.rpfq_vision_act_quant_sm100(
            x2.data_ptr(), ldx, y2.data_ptr(), ldy, images, tokens, K, float(salient_token_ratio),
            float(background_clip_ratio), float(energy_score_weight), int(bool(protect_cls_token)), _p(mask),
            _p(ws), ws_bytes, _stream(x.device)), "rpfq_vision_act_quant_sm100")
    if images:
        g = math.isqrt(tokens - 1) if tokens > 1 else 0
        _count_launch(3 if g and g * g == tokens - 1 else 1)
    return (out, mask.bool()) if return_mask else out


def pack_linear(weight: torch.Tensor, bias: torch.Tensor | None = None, stages: int = 2) -> PackedLayer:
    """The exporter's packing on the GPU (``save_quantized_linear``,
    export_rpfq_vit_to_mlx.py:384-423) through ``rpfq_pack_linear_sm100``:
    float ``[N, K]`` weight -> ``stages`` residual stages of 2-bit axial codes
    and fp16 gammas for U and W, bit-identical to the exporter; bias -> fp16."""
    if not weight.is_cuda:
        raise ValueError("weight must be a CUDA tensor (rpfq_pack_linear_sm100 packs on the GPU)")
    n, k = weight.shape
    if n % 2 or k % 2:
        raise ValueError(f"Complex decomposition requires even dims, got {tuple(weight.shape)}")
    from .packing import BLOCK_SIZE, round_up
    w = weight.detach().to(torch.float32)
    if w.stride(1) != 1 or w.data_ptr() % 4:
        w = w.contiguous()
    dev = w.device
    n_c, k_c = n // 2, k // 2
    n_cp, k_cp = round_up(n_c, BLOCK_SIZE), round_up(k_c, BLOCK_SIZE)
    outs = {"u": (_lib.RpfqPhasePlaneOut * stages)(), "w": (_lib.RpfqPhasePlaneOut * stages)()}
    planes = {}
    for tag in ("u", "w"):
        for i in range(stages):
            codes = torch.empty((n_cp, k_cp // 4), dtype=torch.uint8, device=dev)
            gr = torch.empty((n_cp, k_cp // BLOCK_SIZE), dtype=torch.float16, device=dev)
            gi = torch.empty_like(gr)
            outs[tag][i].codes, outs[tag][i].gamma_real, outs[tag][i].gamma_imag = (
                codes.data_ptr(), gr.data_ptr(), gi.data_ptr())
            planes[f"{tag}_s{i}"] = (codes, gr, gi)
    L = _lib.lib()
    ws_bytes = int(L.rpfq_pack_workspace_bytes(n_c, k_c))
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        _lib.check(L.rpfq_pack_linear_sm100(w.data_ptr(), w.stride(0), n_c, k_c, stages, outs["u"], outs["w"],
                                            ws.data_ptr(), ws_bytes, _stream(dev)), "rpfq_pack_linear_sm100")
    b = torch.zeros(n, device=dev) if bias is None else bias.detach()
    return PackedLayer(n_c, k_c, stages, 2, planes, b.to(device=dev, dtype=torch.float16).contiguous())


def _flags(out: torch.Tensor, residual: torch.Tensor | None, bias: torch.Tensor | None = None) -> int:
    f = 0
    if bias is not None:
        if bias.dtype == torch.float32:
            f |= _lib.GEMM_BIAS_F32
        elif bias.dtype != torch.float16:
            raise ValueError(f"bias must be float16 or float32, got {bias.dtype}")
    if out.dtype == torch.float32:
        f |= _lib.GEMM_OUT_F32
    elif out.dtype != torch.float16:
        raise ValueError(f"out must be float16 or float32, got {out.dtype}")
    if residual is not None:
        if residual.dtype == torch.float32:
            f |= _lib.GEMM_RESIDUAL_F32
        elif residual.dtype != torch.float16:
            raise ValueError(f"residual must be float16 or float32, got {residual.dtype}")
    return f


def gemm(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None,
         residual: torch.Tensor | None = None, activation="none", block_n: int = 0,
         out: torch.Tensor | None = None, out_dtype: torch.dtype = torch.float16, cta_pair: int = 0,
         split_k: int | None = None) -> torch.Tensor:
    """K2: ``act(x @ w.T + bias) + residual`` with fp16 operands, fp32
    accumulation; ``residual`` and ``out`` may be fp16 or fp32 (and may be the
    same tensor for an in-place residual add). ``split_k``: 0 automatic (small
    M splits K over a cluster of CTAs), 1 never, 2..8 forced; None = ``SPLIT_K``."""
    _require(x, "x")
    _require(w, "w")
    n, k = w.shape
    if not w.is_contiguous():
        w = w.contiguous()
    x2, ldx = _rows(x, k, "x")
    m = x2.shape[0]
    if bias is not None:
        _require(bias, "bias", bias.dtype)
        bias = bias.contiguous()
    r2, ldr = (None, 0)
    if residual is not None:
        if not residual.is_cuda:
            raise ValueError("residual must be a CUDA tensor")
        r2, ldr = _rows(residual, n, "residual")
        if r2.shape[0] != m:
            raise ValueError("residual rows do not match x")
    if out is None:
        out = torch.empty((*x.shape[:-1], n), dtype=out_dtype, device=x.device)
    y2, ldy = _rows(out, n, "out")
    if y2.data_ptr() != out.data_ptr() or y2.shape[0] != m:
        raise ValueError("out must be a row-major view with unit column stride")
    split_k = SPLIT_K if split_k is None else int(split_k)
    ws, ws_bytes = _workspace(x.device, split_k)
    a = _lib.RpfqGemmArgs(x=x2.data_ptr(), ldx=ldx, w=w.data_ptr(), bias=_p(bias), residual=_p(r2), ldr=ldr,
                          y=y2.data_ptr(), ldy=ldy, m=m, n=n, k=k, activation=_ACT[activation], block_n=block_n,
                          flags=_flags(out, r2, bias), cta_pair=cta_pair, split_k=split_k, workspace=ws,
                          workspace_bytes=ws_bytes)
    timer = _timer if _timer is not None and _timer.events else None
    with torch.cuda.device(x.device):
        if timer is not None:
            ev0 = torch.cuda.Event(enable_timing=True, external=True)
            ev1 = torch.cuda.Event(enable_timing=True, external=True)
            ev0.record()
        _lib.check(_lib.lib().rpfq_gemm_sm100(ctypes.byref(a), _stream(x.device)), "rpfq_gemm_sm100")
        if timer is not None:
            ev1.record()
            timer.gemm_events.append((ev0, ev1, 2 * m * n * k))
    if m:
        _count_launch()
    return out


def gemm_plan(m: int, n: int, k: int, *, out_dtype: torch.dtype = torch.float16, residual: bool = False,
              block_n: int = 0, cta_pair: int = 0, split_k: int | None = None,
              device: torch.device | None = None) -> dict:
    """The tile plan :func:`gemm` runs for an ``[m, k] x [n, k]`` product on
    ``device`` with the same choices (``rpfq_gemm_plan_sm100``; nothing is
    launched): tile width, CTA pairs, K splits, stream-K tail, grid units."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    split_k = SPLIT_K if split_k is None else int(split_k)
    ws, ws_bytes = _workspace(device, split_k)
    f = (_lib.GEMM_OUT_F32 if out_dtype == torch.float32 else 0)
    if residual:
        f |= _lib.GEMM_RESIDUAL_F32 if out_dtype == torch.float32 else 0
    # placeholders: only alignment and strides are validated, nothing is read
    a = _lib.RpfqGemmArgs(x=256, ldx=k, w=256, bias=None, residual=256 if residual else None, ldr=n if residual else 0,
                          y=256, ldy=n, m=m, n=n, k=k, activation=0, block_n=block_n, flags=f, cta_pair=cta_pair,
                          split_k=split_k, workspace=ws, workspace_bytes=ws_bytes)
    plan = _lib.RpfqGemmPlan()
    with torch.cuda.device(device):
        _lib.check(_lib.lib().rpfq_gemm_plan_sm100(ctypes.byref(a), ctypes.byref(plan)), "rpfq_gemm_plan_sm100")
    return {f: getattr(plan, f) for f, _ in _lib.RpfqGemmPlan._fields_}


def layernorm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, eps: float, act_bits: int = 0,
              out: torch.Tensor | None = None, rows: torch.Tensor | None = None) -> torch.Tensor:
    """LayerNorm of an fp32 ``x[..., d]`` into fp16, with the activation
    quantization of the next packed GEMM fused in when ``act_bits > 0``.
    ``rows`` (int32 CUDA tensor of the flattened row count) gathers: output
    row r is the normalized input row ``rows[r]``."""
    if not x.is_cuda or x.dtype != torch.float32:
        raise ValueError("layernorm: x must be a float32 CUDA tensor")
    _require(weight, "weight")
    _require(bias, "bias")
    d = x.shape[-1]
    x2, ldx = _rows(x, d, "x")
    if out is None:
        out = torch.empty(x.shape, dtype=torch.float16, device=x.device)
    y2, ldy = _rows(out, d, "out")
    if rows is not None:
        _require(rows, "rows", torch.int32)
        if rows.numel() != y2.shape[0]:
            raise ValueError("layernorm: rows must hold one index per output row")
    with torch.cuda.device(x.device):
        _lib.check(_lib.lib().rpfq_layernorm_rows_sm100(
            x2.data_ptr(), ldx, x2.shape[0], _p(rows), weight.data_ptr(), bias.data_ptr(), y2.data_ptr(), ldy,
            y2.shape[0], d, float(eps), int(act_bits), _stream(x.device)), "rpfq_layernorm_rows_sm100")
    if y2.shape[0]:
        _count_launch()
    return out


def layernorm_ex(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, eps: float, act_bits: int = 0, *,
                 rows: torch.Tensor | None = None, merge_side: int = 0, add: torch.Tensor | None = None,
                 add_rows: torch.Tensor | None = None, out: torch.Tensor | None = None, fp16_out: bool = True,
                 out32: torch.Tensor | None = None, out32_prenorm: bool = False):
    """The LayerNorm pass with all its row sources and outputs
    (``rpfq_layernorm_ex_sm100``); returns ``(fp16 output or None, fp32
    output or None)``.

    Row sources: ``x`` rows as they are; ``rows`` gathers (output row r is
    input row ``rows[r]``); ``merge_side`` = s > 0 is Swin's 2x2 patch merging
    of an ``x`` of ``[images * s * s, c]`` tokens into ``[images * (s/2)^2, 4c]``
    rows; ``add`` adds ``add[add_rows[r]]`` (or ``add[r]``) to row r before the
    normalization and needs ``out32`` with ``out32_prenorm=True``, which then
    receives the updated rows (``out32`` may be ``x``: in place). ``out32``
    without ``out32_prenorm`` receives the normalized rows in fp32."""
    if not x.is_cuda or x.dtype != torch.float32:
        raise ValueError("layernorm: x must be a float32 CUDA tensor")
    _require(weight, "weight")
    _require(bias, "bias")
    c = x.shape[-1]
    x2, ldx = _rows(x, c, "x")
    if merge_side:
        d, m = 4 * c, x2.shape[0] // 4
    else:
        d, m = c, (rows.numel() if rows is not None else x2.shape[0])
    if rows is not None:
        _require(rows, "rows", torch.int32)
    if fp16_out and out is None:
        out = torch.empty((m, d), dtype=torch.float16, device=x.device)
    y2, ldy = _rows(out, d, "out") if out is not None else (None, 0)
    z2, ldz = _rows(out32, d, "out32") if out32 is not None else (None, 0)
    for t in (y2, z2):
        if t is not None and t.shape[0] != m:
            raise ValueError(f"layernorm: the outputs must have {m} rows")
    a2, lda = (None, 0)
    if add is not None:
        if not add.is_cuda or add.dtype != torch.float32:
            raise ValueError("layernorm: add must be a float32 CUDA tensor")
        a2, lda = _rows(add, d, "add")
    if add_rows is not None:
        _require(add_rows, "add_rows", torch.int32)
    args = _lib.RpfqLayerNormArgs(
        x=x2.data_ptr(), ldx=ldx, x_rows=x2.shape[0], rows=_p(rows), add=_p(a2), ld_add=lda,
        add_bound=a2.shape[0] if a2 is not None else 0, add_rows=_p(add_rows), weight=weight.data_ptr(),
        bias=bias.data_ptr(), y=_p(y2), ldy=ldy, y32=_p(z2), ldy32=ldz, m=m, d=d, eps=float(eps),
        act_bits=int(act_bits), merge_side=int(merge_side), y32_prenorm=int(bool(out32_prenorm)))
    with torch.cuda.device(x.device):
        _lib.check(_lib.lib().rpfq_layernorm_ex_sm100(ctypes.byref(args), _stream(x.device)),
                   "rpfq_layernorm_ex_sm100")
    if m:
        _count_launch()
    return out, out32


def patch_unfold(images: torch.Tensor, patch: int, out: torch.Tensor | None = None) -> torch.Tensor:
    """images ``[B, C, H, W]`` (fp16 or fp32) -> fp16 patch rows ``[B, (H/P)(W/P), C P P]``
    in the CHW patch order of the reference's ``patchify_tensor``
    (``audit_rpfq_vit_ios_parity.py:125-134``), ``rpfq_patch_unfold_sm100``."""
    if not images.is_cuda or images.dtype not in (torch.float16, torch.float32) or images.dim() != 4:
        raise ValueError("patch_unfold: images must be a [B, C, H, W] float16 or float32 CUDA tensor")
    images = images.contiguous()
    B, C, H, W = images.shape
    if patch <= 0 or H % patch or W % patch:
        raise ValueError(f"patch_unfold: patch {patch} must divide the image size {H}x{W}")
    n, k = (H // patch) * (W // patch), C * patch * patch
    if out is None:
        out = torch.empty((B, n, k), dtype=torch.float16, device=images.device)
    o2, ldo = _rows(out, k, "out")
    if o2.data_ptr() != out.data_ptr() or o2.shape[0] != B * n:
        raise ValueError(f"patch_unfold: out must be a row-major view of {B * n} rows with unit column stride")
    if B == 0:
        return out
    with torch.cuda.device(images.device):
        _lib.check(_lib.lib().rpfq_patch_unfold_sm100(images.data_ptr(), int(images.dtype == torch.float32), B, C, H,
                                                      W, int(patch), o2.data_ptr(), ldo, _stream(images.device)),
                   "rpfq_patch_unfold_sm100")
    _count_launch()
    return out


def act_quant(x: torch.Tensor, num_bits: int, out: torch.Tensor | None = None) -> torch.Tensor:
    """Per-row symmetric quantization of the Re / Im halves (ActivationQuantSTE)."""
    _require(x, "x")
    k = x.shape[-1]
    x2, ldx = _rows(x, k, "x")
    if out is None:
        out = torch.empty_like(x2)
    o2, ldo = _rows(out, k, "out")
    with torch.cuda.device(x.device):
        _lib.check(_lib.lib().rpfq_act_quant_sm100(x2.data_ptr(), ldx, o2.data_ptr(), ldo, x2.shape[0], k,
                                                   int(num_bits), _stream(x.device)), "rpfq_act_quant_sm100")
    if x2.shape[0]:
        _count_launch()
    return out.reshape(x.shape)


# ---------------------------------------------------------------------------
# 8-bit linear path
# ---------------------------------------------------------------------------

GEMM_INT8_MAX_K = 131071  # 128 * 128 * k < 2^31: the int32 sums cannot overflow
_GEMM_INT8_MAX_N = 2 ** 31 - 257
_QUANTIZE_MAX_K = 2 ** 30
_ROTARY_MAX_HEADS = 2 ** 24
_ROTARY_MAX_DIM = 2 ** 31 - 1


def _too_large(name: str, what: str, value: int, limit: int):
    """What the C structures hold in 32 bits is refused here: there it would come out small."""
    return NotImplementedError(f"{name}: {what} must be at most {limit}, got {value}")


def _tensors(name: str, index: int, tensors) -> None:
    """Every tensor (None: not given) is on cuda:index, and no gradient is asked for
    through any, nor a tangent given: these operators have no autograd."""
    grad, forward = torch.is_grad_enabled(), forward_ad._current_level >= 0
    for t in tensors:
        if t is not None:
            if t.get_device() != index:
                raise ValueError(f"{name}: every tensor must be on cuda:{index}, got one on {t.device}")
            if grad and t.requires_grad:
                raise ValueError(f"{name} has no autograd: call it under torch.no_grad() or on detached tensors")
            if forward and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError(f"{name} has no autograd: it takes no tensor with a tangent")


def _float_type(t: torch.Tensor, name: str) -> bool:
    """True for float32, False for float16; anything else is refused."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype is torch.float16:
        return False
    if t.dtype is torch.float32:
        return True
    raise ValueError(f"{name} must be float16 or float32, got {t.dtype}")


def _matrix(t: torch.Tensor, k: int, name: str):
    """``t[..., k]`` as rows: (tensor to keep, rows, row stride)."""
    shape = t.shape
    if not shape or shape[-1] != k:
        raise ValueError(f"{name}: last dim of {tuple(shape)} is not {k}")
    if t.is_contiguous():
        return t, t.numel() // k, k
    if len(shape) == 2:
        ld, step = t.stride()
        if step == 1 and ld >= k:
            return t, shape[0], ld
    t2, ld = _rows(t, k, name)
    if ld < k:  # rows that overlap (expanded): one copy
        t2, ld = t2.contiguous(), k
    return t2, t2.shape[0], ld


def _code_rows(q: torch.Tensor, k: int, name: str):
    """``q[..., k]`` int8 as rows that start on 16 bytes (what the TMA loads need):
    rows of another stride or address are copied into such rows."""
    q2, rows, ld = _matrix(q, k, name)
    if rows <= 1:
        ld = (k + 15) // 16 * 16
    if ld % 16 or q2.data_ptr() % 16:
        ld = (k + 15) // 16 * 16
        buf = torch.empty((rows, ld), dtype=torch.int8, device=q.device)
        buf[:, :k] = q2.reshape(rows, k)
        q2 = buf
    return q2, rows, ld


def quantize_rows(x: torch.Tensor):
    """8-bit codes and one scale per row of fp16 or fp32 ``x[..., k]``
    (``rpfq_quantize_rows_sm100``): ``t = max(amax |x|, 1e-30)``,
    ``codes = rint(x * (1 / t * 127))`` in fp32 steps, ``scale = t / 127``.
    Returns int8 ``[..., k]`` (rows padded to a multiple of 16 bytes in memory,
    so a view when k is none) and fp32 ``[...]``. A row that holds a NaN or an
    infinity gets codes of zero and a scale of NaN. The tokens of an activation
    matrix, or the output channels of a weight ``[n, k]``."""
    f32 = _float_type(x, "x")
    index = x.get_device()
    if torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            return quantize_rows(x)
    _tensors("quantize_rows", index, (x,))
    shape = x.shape
    if not shape or shape[-1] == 0:
        raise ValueError(f"quantize_rows: x must be [..., k] with k > 0, got {tuple(shape)}")
    k, lead = shape[-1], shape[:-1]
    if k > _QUANTIZE_MAX_K:
        raise _too_large("quantize_rows", "k", k, _QUANTIZE_MAX_K)
    x2, m, ldx = _matrix(x, k, "x")
    ld = (k + 15) // 16 * 16
    q = x.new_empty((*lead, ld), dtype=torch.int8)
    scale = x.new_empty(lead, dtype=torch.float32)
    rc = _lib.lib().rpfq_quantize_rows_sm100(x2.data_ptr(), int(f32), ldx, q.data_ptr(), ld, scale.data_ptr(), m, k,
                                             torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc, "rpfq_quantize_rows_sm100")
    if _timer is not None and m:
        _count_launch()
    return (q if ld == k else q[..., :k]), scale


def _gemm_int8(name: str, index: int, x: torch.Tensor, x2: torch.Tensor, m: int, ldx: int, x_scale, x_flag: int,
               w: torch.Tensor, w_scale: torch.Tensor, bias, residual, activation, out, out_dtype, block_n,
               split_k) -> torch.Tensor:
    """What gemm_int8 and linear_int8 share: the checks of everything but x, and the launch."""
    if torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            return _gemm_int8(name, index, x, x2, m, ldx, x_scale, x_flag, w, w_scale, bias, residual, activation, out,
                              out_dtype, block_n, split_k)
    _tensors(name, index, (x, w, w_scale, bias, residual, out))
    n, k = w.shape
    if w_scale.dtype is not torch.float32 or w_scale.numel() != n:
        raise ValueError(f"{name}: w_scale must hold {n} float32 values, got {w_scale.numel()} of {w_scale.dtype}")
    act = _ACT.get(activation)
    if act is None:
        raise ValueError(f"{name}: unknown activation {activation!r}")
    flags, bias_ptr, r_ptr, ldr = x_flag, None, None, 0
    w2, _, ldw = _code_rows(w, k, "w")
    w_scale = w_scale.contiguous()
    given = out is not None
    if not given:
        out = x.new_empty((*x.shape[:-1], n), dtype=out_dtype)
        ldy = n
    else:
        y2, rows, ldy = _matrix(out, n, "out")
        out_dtype = out.dtype
        if y2.data_ptr() != out.data_ptr() or rows != m:
            raise ValueError(f"{name}: out must be a row-major view of {m} rows with unit column stride")
    if out_dtype is torch.float32:
        flags |= _lib.GEMM_OUT_F32
    elif out_dtype is not torch.float16:
        raise ValueError(f"{name}: out must be float16 or float32, got {out_dtype}")
    if bias is not None:
        if bias.numel() != n:
            raise ValueError(f"{name}: bias must hold {n} values, got {bias.numel()}")
        if bias.dtype is torch.float32:
            flags |= _lib.GEMM_BIAS_F32
        elif bias.dtype is not torch.float16:
            raise ValueError(f"{name}: bias must be float16 or float32, got {bias.dtype}")
        bias = bias.contiguous()
        bias_ptr = bias.data_ptr()
    if residual is not None:
        r2, rows, ldr = _matrix(residual, n, "residual")
        if rows != m:
            raise ValueError(f"{name}: residual rows do not match x")
        if r2.dtype is torch.float32:
            flags |= _lib.GEMM_RESIDUAL_F32
        elif r2.dtype is not torch.float16:
            raise ValueError(f"{name}: residual must be float16 or float32, got {r2.dtype}")
        r_ptr = r2.data_ptr()
    L = _lib.lib()
    scratch, scratch_ptr, need = None, None, 0
    if x_flag:
        # a few rows are quantized inside the launch; the library says which
        need = m * ((k + 15) // 16 * 16 + 4) if block_n or split_k else L.rpfq_gemm_i8_scratch_bytes(m, k)
        if need:
            scratch = x.new_empty(need, dtype=torch.uint8)
            scratch_ptr = scratch.data_ptr()
    a = _lib.RpfqGemmI8Args(x2.data_ptr(), ldx, x_scale, w2.data_ptr(), ldw, w_scale.data_ptr(), bias_ptr, r_ptr, ldr,
                            out.data_ptr(), ldy, m, n, k, act, flags, block_n, split_k, scratch_ptr, need)
    rc = L.rpfq_gemm_i8_sm100(ctypes.byref(a), torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc, "rpfq_gemm_i8_sm100")
    if given:
        increment_version(out)
    if _timer is not None and m:
        _count_launch(2 if need else 1)
    return out


def _check_codes(name: str, w: torch.Tensor) -> None:
    if w.dtype is not torch.int8 or w.dim() != 2 or w.numel() == 0:
        raise ValueError(f"{name}: w must be int8 [n, k] with n, k > 0, got {w.dtype} {tuple(w.shape)}")
    n, k = w.shape
    if k > GEMM_INT8_MAX_K:
        raise _too_large(name, "k", k, GEMM_INT8_MAX_K)
    if n > _GEMM_INT8_MAX_N:
        raise _too_large(name, "n", n, _GEMM_INT8_MAX_N)


def gemm_int8(x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
              bias: torch.Tensor | None = None, residual: torch.Tensor | None = None, activation="none",
              out: torch.Tensor | None = None, out_dtype: torch.dtype = torch.float16, block_n: int = 0,
              split_k: int = 0) -> torch.Tensor:
    """``act(x_scale[..., None] * w_scale * (x @ w.T) + bias) + residual`` of
    int8 codes ``x[..., k]`` and ``w[n, k]`` with a scale per token and per output
    channel (``rpfq_gemm_i8_sm100``): exact int32 sums on the tensor cores
    (k up to ``GEMM_INT8_MAX_K``), scaled in fp32. ``bias`` fp16 or fp32;
    ``residual`` and ``out`` fp16 or fp32 alike (and may be the same tensor for
    an in-place residual add; ``out`` must not share memory with anything else that
    the call reads). Code rows that do not start on 16 bytes are copied into rows
    that do; :func:`quantize_rows` returns such rows.
    ``block_n`` (64, 128, 256) and ``split_k`` (1..8) fix the tiles and the parts
    of k, 0 leaves them to the library; the result is the same bit for bit.

    No autograd: a tensor that asks for a gradient or carries a tangent is refused."""
    name = "gemm_int8"
    _require(x, "x", torch.int8)
    _check_codes(name, w)
    index = x.get_device()
    _tensors(name, index, (x_scale,))
    x2, m, ldx = _code_rows(x, w.shape[1], "x")
    if x_scale.dtype is not torch.float32 or x_scale.numel() != m:
        raise ValueError(f"{name}: x_scale must hold one float32 value per row ({m}), got {x_scale.numel()} of "
                         f"{x_scale.dtype}")
    x_scale = x_scale.contiguous()
    return _gemm_int8(name, index, x, x2, m, ldx, x_scale.data_ptr(), 0, w, w_scale, bias, residual, activation, out,
                      out_dtype, block_n, split_k)


def linear_int8(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: torch.Tensor | None = None,
                residual: torch.Tensor | None = None, activation="none", out: torch.Tensor | None = None,
                out_dtype: torch.dtype = torch.float16, block_n: int = 0, split_k: int = 0) -> torch.Tensor:
    """The 8-bit linear layer of fp16 or fp32 activations ``x[..., k]``: the rows
    of x as :func:`quantize_rows` codes them, then :func:`gemm_int8` with the
    weight's codes and scales (``w, w_scale = quantize_rows(weight)``), the same
    bits as the two calls. The other arguments as there."""
    name = "linear_int8"
    x_flag = _lib.GEMM_X_F32 if _float_type(x, "x") else _lib.GEMM_X_F16
    _check_codes(name, w)
    x2, m, ldx = _matrix(x, w.shape[1], "x")
    return _gemm_int8(name, x.get_device(), x, x2, m, ldx, None, x_flag, w, w_scale, bias, residual, activation, out,
                      out_dtype, block_n, split_k)


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------

_POSITION = {torch.int32: _lib.POS_I32, torch.int64: _lib.POS_I64, torch.float32: _lib.POS_F32,
             torch.float64: _lib.POS_F64}


def rotary_frequencies(rot_dim: int, base: float = 10000.0, *, axes: int = 1, scaling: str = "none",
                       factor: float = 1.0, original_length: int | None = None, low: float = 1.0, high: float = 32.0,
                       device=None):
    """The ``(inv_freq, magnitude)`` that :func:`rotary` takes for ``rot_dim``
    rotated values per head: fp64 ``[rot_dim / 2]``, ``base ** (-j / p)`` for the
    p = rot_dim / 2 / axes pairs of each axis.

    ``scaling`` stretches them for sequences ``factor`` times longer than the
    model has seen:

    * ``"linear"``: every frequency divided by ``factor`` (positions interpolated);
    * ``"base"``: base times ``factor ** (d / (d - 2))``, d = rot_dim / axes: the
      fastest pair keeps its frequency, the slowest is divided by ``factor``;
    * ``"parts"``: by how often a pair turns within ``original_length``: at
      least ``high`` turns keep the frequency, at most ``low`` divide it by
      ``factor``, linear in between; magnitude ``0.1 ln(factor) + 1``.

    The magnitude is 1 otherwise."""
    if axes not in (1, 2):
        raise ValueError(f"rotary_frequencies: axes must be 1 or 2, got {axes}")
    if rot_dim <= 0 or rot_dim % (2 * axes):
        raise ValueError(f"rotary_frequencies: rot_dim must be a positive multiple of {2 * axes}, got {rot_dim}")
    if not base > 0 or not factor >= 1:
        raise ValueError(f"rotary_frequencies: base must be positive and factor at least 1, got {base}, {factor}")
    per = rot_dim // 2 // axes
    magnitude = 1.0
    if scaling == "base":
        if per < 2:
            raise ValueError("rotary_frequencies: scaling 'base' needs at least two pairs per axis")
        base = base * factor ** (per / (per - 1))
    elif scaling not in ("none", "linear", "parts"):
        raise ValueError(f"rotary_frequencies: unknown scaling {scaling!r}")
    freq = base ** (-torch.arange(per, dtype=torch.float64) / per)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "parts":
        if not original_length or not high > low:
            raise ValueError("rotary_frequencies: scaling 'parts' needs original_length and high > low")
        turns = original_length * freq / (2.0 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        freq = freq * (keep + (1.0 - keep) / factor)
        magnitude = 0.1 * math.log(factor) + 1.0
    return freq.repeat(axes).to(device), magnitude


def rotary(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *, layout: str = "half", axes: int = 1,
           magnitude: float = 1.0, transpose: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotary positions on fp16 or fp32 heads ``x[L, H, D]`` or ``[B, L, H, D]``
    (any strides, unit stride inside a head), ``rpfq_rotary_sm100``: pair j of
    the first ``2 * inv_freq.numel()`` values of each head turns by
    ``positions * inv_freq[j]`` (fp64 angles) and is scaled by ``magnitude``; the
    other values are copied.

    ``layout``: pairs at ``(j, j + P)`` (``"half"``) or ``(2j, 2j + 1)``
    (``"interleaved"``). ``positions``: int32, int64, fp32 or fp64, ``[L]`` or
    ``[B, L]``; with ``axes=2`` a trailing dimension of two, of which the first half
    of the pairs takes the first (a patch's row) and the rest the second (its
    column). ``out`` may be ``x`` (in place), e.g. the query and key heads of a
    qkv product's rows: ``q = qkv.view(B, L, 3 * H, D)[:, :, :2 * H]``. It must
    not overlap x in any other way, nor the positions or frequencies.

    No autograd: ``transpose=True`` turns the other way, which maps the gradient
    of the output to the gradient of x."""
    name = "rotary"
    f32 = _float_type(x, "x")
    index = x.get_device()
    _tensors(name, index, (x, positions, inv_freq, out))
    four = x.dim() == 4
    if not four and x.dim() != 3:
        raise ValueError(f"{name}: x must be [L, H, D] or [B, L, H, D], got {tuple(x.shape)}")
    if layout not in ("half", "interleaved"):
        raise ValueError(f"{name}: layout must be 'half' or 'interleaved', got {layout!r}")
    if axes not in (1, 2):
        raise ValueError(f"{name}: axes must be 1 or 2, got {axes}")
    if inv_freq.dtype is not torch.float64:
        raise ValueError(f"{name}: inv_freq must be float64, got {inv_freq.dtype}")
    B, L, H, D = x.shape if four else (1, *x.shape)
    if H > _ROTARY_MAX_HEADS:
        raise _too_large(name, "heads", H, _ROTARY_MAX_HEADS)
    if D > _ROTARY_MAX_DIM:
        raise _too_large(name, "the head dim", D, _ROTARY_MAX_DIM)
    pairs = inv_freq.numel()
    if pairs == 0 or 2 * pairs > D or pairs % axes:
        raise ValueError(f"{name}: inv_freq must hold 1..{D // 2} values, a multiple of axes, got {pairs}")
    position_type = _POSITION.get(positions.dtype)
    if position_type is None:
        raise ValueError(f"{name}: positions must be int32, int64, float32 or float64, got {positions.dtype}")
    tail = (axes,) if axes > 1 else ()
    shape = positions.shape
    if shape == (L, *tail):
        per_sequence = 0
    elif four and shape == (B, L, *tail):
        per_sequence = L * axes
    else:
        raise ValueError(f"{name}: positions must be {(L, *tail)} or {(B, L, *tail)}, got {tuple(shape)}")
    if x.stride(-1) != 1 and D > 1:
        if out is x:
            raise ValueError(f"{name}: in place, a head must have unit stride")
        x = x.contiguous()
    given = out is not None
    if not given:
        out = x.new_empty(x.shape)
    elif out.shape != x.shape or out.dtype != x.dtype:
        raise ValueError(f"{name}: out must be {tuple(x.shape)} {x.dtype}, got {tuple(out.shape)} {out.dtype}")
    elif any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride())) or (D > 1 and out.stride(-1) != 1):
        raise ValueError(f"{name}: out must not be expanded and must have unit stride inside a head")
    positions, inv_freq = positions.contiguous(), inv_freq.contiguous()
    xs, ys = x.stride(), out.stride()
    a = _lib.RpfqRotaryArgs(x.data_ptr(), xs[0] if four else 0, xs[-3], xs[-2], out.data_ptr(), ys[0] if four else 0,
                            ys[-3], ys[-2], positions.data_ptr(), per_sequence, inv_freq.data_ptr(), B, L, H, D,
                            pairs, axes, position_type, f32, layout == "interleaved", bool(transpose), magnitude)
    if torch.cuda.current_device() == index:
        rc = _lib.lib().rpfq_rotary_sm100(ctypes.byref(a), torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = _lib.lib().rpfq_rotary_sm100(ctypes.byref(a), torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc, "rpfq_rotary_sm100")
    if given:
        increment_version(out)
    if _timer is not None and x.numel():
        _count_launch()
    return out



def wide_linear(x: torch.Tensor, layer: PackedLayer, dense: torch.Tensor | None, act_bits: int = 0,
                activation="none", residual: torch.Tensor | None = None,
                out: torch.Tensor | None = None, out_dtype: torch.dtype = torch.float16,
                bias: torch.Tensor | None = None, split_k: int | None = None) -> torch.Tensor:
    """Whole layer through ``rpfq_wide_linear_sm100``: optional activation
    quantization, then the GEMM over the prepacked coefficients with bias and
    epilogue. ``x`` is fp16 ``[..., 2 k_c]``; ``residual`` / ``out`` fp16 or
    fp32 (``out`` may be ``residual`` for an in-place residual add).

    ``dense=None`` selects the fused decode path (at most ``FUSED_DECODE_MAX_ROWS``
    rows, 2-bit codes, ``n_c`` and ``k_c`` multiples of 8): the packed planes
    are decoded inside the GEMM and no dense matrix exists anywhere.

    ``bias`` (optional) replaces ``layer.bias`` for this call, e.g. the same
    values widened to fp32 once, which the epilogue adds without converting.
    ``split_k`` as in :func:`gemm` (both paths: the fused decode splits K over
    a cluster of CTAs per block of output rows when those blocks alone leave
    most SMs idle)."""
    _require(x, "x")
    if dense is not None:
        _require(dense, "dense")
    if bias is None:
        bias = layer.bias
    K, N = 2 * layer.k_c, 2 * layer.n_c
    x2, ldx = _rows(x, K, "x")
    m = x2.shape[0]
    r2, ldr = (None, 0)
    if residual is not None:
        if not residual.is_cuda:
            raise ValueError("residual must be a CUDA tensor")
        r2, ldr = _rows(residual, N, "residual")
    if out is None:
        out = torch.empty((*x.shape[:-1], N), dtype=out_dtype, device=x.device)
    y2, ldy = _rows(out, N, "out")
    if y2.data_ptr() != out.data_ptr() or y2.shape[0] != m:
        raise ValueError("out must be a row-major view with unit column stride")
    scratch = torch.empty((m, K), dtype=torch.float16, device=x.device) if act_bits else None
    s = layer_struct(layer)
    split_k = SPLIT_K if split_k is None else int(split_k)
    ws, ws_bytes = _workspace(x.device, split_k)
    a = _lib.RpfqWideLinearArgs(layer=ctypes.pointer(s), dense=_p(dense), x=x2.data_ptr(), ldx=ldx,
                                bias=_p(bias), residual=_p(r2), ldr=ldr, y=y2.data_ptr(), ldy=ldy, m=m,
                                act_bits=int(act_bits), activation=_ACT[activation], scratch=_p(scratch),
                                flags=_flags(out, r2, bias), split_k=split_k, workspace=ws,
                                workspace_bytes=ws_bytes)
    timer = _timer if _timer is not None and _timer.events else None
    with torch.cuda.device(x.device):
        if timer is not None:
            # With act_bits > 0 the span also holds the quantization kernel.
            ev0 = torch.cuda.Event(enable_timing=True, external=True)
            ev1 = torch.cuda.Event(enable_timing=True, external=True)
            ev0.record()
        _lib.check(_lib.lib().rpfq_wide_linear_sm100(ctypes.byref(a), _stream(x.device)), "rpfq_wide_linear_sm100")
        if timer is not None:
            ev1.record()
            timer.gemm_events.append((ev0, ev1, 2 * m * N * K))
    if m:
        _count_launch(2 if act_bits else 1)
    return out


# ---------------------------------------------------------------------------
# torch.ops.rpfq.* (CUDA only)
# ---------------------------------------------------------------------------

_LIB = torch.library.Library("rpfq", "DEF")
_LIB.define("gemm(Tensor x, Tensor w, Tensor? bias=None, Tensor? residual=None, int activation=0) -> Tensor")
_LIB.define("act_quant(Tensor x, int num_bits) -> Tensor")
_LIB.define("prepack(Tensor[] codes, Tensor[] gamma_real, Tensor[] gamma_imag, int n_c, int k_c, "
            "int code_bits=2, int rounding=0) -> Tensor")
# The packed layer as the reference stores it: codes / gammas of the U stages
# then the W stages (export_rpfq_vit_to_mlx.py:384-423 key order), exactly the
# tensors a caller of QATLinearComplexPhase's packed form holds.
_LIB.define("wide_linear(Tensor x, Tensor[] codes, Tensor[] gamma_re, Tensor[] gamma_im, Tensor? bias, int n_c, "
            "int k_c, int act_bits=0, bool gelu=False) -> Tensor")
_LIB.define("wide_linear_dense(Tensor x, Tensor dense, Tensor? bias, int n_c, int k_c, int act_bits=0, "
            "int activation=0, Tensor? residual=None) -> Tensor")
# The 8-bit linear path and the rotary positions (the functions of the same names).
_LIB.define("quantize_rows(Tensor x) -> (Tensor, Tensor)")
_LIB.define("gemm_int8(Tensor x, Tensor x_scale, Tensor w, Tensor w_scale, Tensor? bias=None, Tensor? residual=None, "
            "int activation=0, bool out_f32=False) -> Tensor")
_LIB.define("linear_int8(Tensor x, Tensor w, Tensor w_scale, Tensor? bias=None, Tensor? residual=None, "
            "int activation=0, bool out_f32=False) -> Tensor")
_LIB.define("rotary(Tensor x, Tensor positions, Tensor inv_freq, str layout=\"half\", int axes=1, "
            "float magnitude=1.0, bool transpose=False) -> Tensor")


def _op_gemm_int8(x, x_scale, w, w_scale, bias=None, residual=None, activation=0, out_f32=False):
    return gemm_int8(x, x_scale, w, w_scale, bias, residual, int(activation),
                     out_dtype=torch.float32 if out_f32 else torch.float16)


def _op_linear_int8(x, w, w_scale, bias=None, residual=None, activation=0, out_f32=False):
    return linear_int8(x, w, w_scale, bias, residual, int(activation),
                       out_dtype=torch.float32 if out_f32 else torch.float16)


def _op_rotary(x, positions, inv_freq, layout="half", axes=1, magnitude=1.0, transpose=False):
    return rotary(x, positions, inv_freq, layout=layout, axes=int(axes), magnitude=float(magnitude),
                  transpose=bool(transpose))


def _op_gemm(x, w, bias=None, residual=None, activation=0):
    return gemm(x, w, bias, residual, int(activation))


def _op_act_quant(x, num_bits):
    return act_quant(x, int(num_bits))


def _planes_from_lists(codes, gamma_real, gamma_imag, n_c, k_c, code_bits, bias=None):
    if len(codes) % 2 or not (len(codes) == len(gamma_real) == len(gamma_imag)) or not codes:
        raise ValueError("codes / gammas must list the U stages then the W stages")
    stages = len(codes) // 2
    planes = {}
    for i in range(stages):
        planes[f"u_s{i}"] = (codes[i], gamma_real[i], gamma_imag[i])
        planes[f"w_s{i}"] = (codes[stages + i], gamma_real[stages + i], gamma_imag[stages + i])
    return PackedLayer(int(n_c), int(k_c), stages, int(code_bits), planes, bias)


def _op_prepack(codes, gamma_real, gamma_imag, n_c, k_c, code_bits=2, rounding=0):
    layer = _planes_from_lists(codes, gamma_real, gamma_imag, n_c, k_c, code_bits)
    return prepack(layer, "rne" if int(rounding) == 0 else "ties_away")


# Decoded coefficient matrices of packed layers called through the packed op
# with more rows than the fused decode path takes: keyed by the planes'
# storage and version counters (a plane written in place decodes again). An
# entry holds its plane tensors, so their storage cannot be handed to another
# layer while the entry exists; the oldest entry goes first past the limit.
_DENSE_CACHE: dict = {}
_DENSE_CACHE_MAX = 256
dense_cache_stats = {"hits": 0, "decodes": 0}


def _cached_dense(layer: PackedLayer, tensors) -> torch.Tensor:
    key = (layer.n_c, layer.k_c, layer.stages, layer.code_bits,
           tuple((t.data_ptr(), t._version, tuple(t.shape), t.dtype) for t in tensors))
    entry = _DENSE_CACHE.get(key)
    if entry is not None:
        dense_cache_stats["hits"] += 1
        return entry[1]
    while len(_DENSE_CACHE) >= _DENSE_CACHE_MAX:
        _DENSE_CACHE.pop(next(iter(_DENSE_CACHE)))
    dense = prepack(layer)
    dense_cache_stats["decodes"] += 1
    _DENSE_CACHE[key] = (list(tensors), dense)
    return dense


def _op_wide_linear(x, codes, gamma_re, gamma_im, bias, n_c, k_c, act_bits=0, gelu=False):
    """The packed layer ``y = act(Q(W) x + b)`` straight from the reference's
    packed tensors: codes uint8 ``[n_cp, k_cp * b / 8]`` and fp16 gammas
    ``[n_cp, k_cp / 256]`` per stage (U stages, then W stages; the code width
    b follows from the codes' shape), optional fp16 bias ``[2 n_c]``, fp16
    ``x[..., 2 k_c]`` -> fp16 ``[..., 2 n_c]``. ``act_bits`` > 0 quantizes x
    first (ActivationQuantSTE); ``gelu`` applies exact GELU to the output.

    Up to ``FUSED_DECODE_MAX_ROWS`` rows (2-bit codes, ``n_c``, ``k_c``
    multiples of 8) the codes are decoded inside the GEMM and no dense matrix
    exists; otherwise the planes are decoded once into the fp16 coefficient
    matrix (kept for later calls with the same planes) and the tcgen05 GEMM
    runs over it."""
    _require(x, "x")
    from .packing import BLOCK_SIZE, round_up
    n_c, k_c = int(n_c), int(k_c)
    if n_c <= 0 or k_c <= 0:
        raise ValueError(f"n_c and k_c must be positive, got {n_c}, {k_c}")
    k_cp = round_up(k_c, BLOCK_SIZE)
    if not codes or codes[0].dim() != 2 or (codes[0].shape[1] * 8) % k_cp:
        raise ValueError("codes must be [n_cp, k_cp * code_bits / 8] uint8 tensors")
    code_bits = codes[0].shape[1] * 8 // k_cp
    if bias is not None:
        _require(bias, "bias")
        if bias.numel() != 2 * n_c:
            raise ValueError(f"bias must hold {2 * n_c} values, got {bias.numel()}")
    layer = _planes_from_lists(codes, gamma_re, gamma_im, n_c, k_c, code_bits,
                               bias if bias is not None else torch.zeros(2 * n_c, dtype=torch.float16,
                                                                          device=x.device))
    m = x.numel() // x.shape[-1] if x.dim() else 0
    act = "gelu" if gelu else "none"
    fused = m <= FUSED_DECODE_MAX_ROWS and code_bits == 2 and n_c % 8 == 0 and k_c % 8 == 0
    dense = None if fused else _cached_dense(layer, [*codes, *gamma_re, *gamma_im])
    return wide_linear(x, layer, dense, int(act_bits), activation=act)


def _op_wide_linear_dense(x, dense, bias, n_c, k_c, act_bits=0, activation=0, residual=None):
    _require(x, "x")
    if tuple(dense.shape) != (2 * int(n_c), 2 * int(k_c)):
        raise ValueError(f"dense must be [{2 * int(n_c)}, {2 * int(k_c)}], got {tuple(dense.shape)}")
    if act_bits:
        x = act_quant(x, int(act_bits))
    return gemm(x, dense, bias, residual, int(activation))


_LIB.impl("gemm", _op_gemm, "CUDA")
_LIB.impl("act_quant", _op_act_quant, "CUDA")
_LIB.impl("quantize_rows", quantize_rows, "CUDA")
_LIB.impl("gemm_int8", _op_gemm_int8, "CUDA")
_LIB.impl("linear_int8", _op_linear_int8, "CUDA")
_LIB.impl("rotary", _op_rotary, "CUDA")
_LIB.impl("prepack", _op_prepack, "CUDA")
_LIB.impl("wide_linear", _op_wide_linear, "CUDA")
_LIB.impl("wide_linear_dense", _op_wide_linear_dense, "CUDA")
