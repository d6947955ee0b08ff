"""Torch-facing wrappers of the libbmx C ABI.

Three groups:

* the reference's native operator set, same names and argument meaning as
  the reference's extension functions (``norm``, ``gate``, ``split``,
  ``pack``, ``silu_mul``, ``epilogue``, ``ordered_softmax``), each raising
  ``RuntimeError`` on bad input like the reference's ``TORCH_CHECK``s;
* the fused hot-path modules (``trimul``, ``triattn``, ``pair_transition``,
  ``adaln``) that take a module with Boltz's parameter names;
* sequence operators with gradients (``qk_norm_rope``, ``relative_bias``,
  ``cross_attention``; ``residual_norm``, ``causal_conv``, ``selective_scan``)
  for an encoder / decoder beside the pair stack.

Every call launches on torch's current stream of the input's device, allocates
outputs and workspaces through torch's caching allocator and never
synchronises.  There is no fallback: without the built library every call
raises.
"""

from __future__ import annotations

import ctypes
import os
from functools import lru_cache

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _native as N

C = 128

# ---------------------------------------------------------------- helpers


# The current stream's handle by device index: what
# ``torch.cuda.current_stream(device).cuda_stream`` returns, without building a
# Stream object per call (2 us of a 20-us call).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(t: torch.Tensor) -> int:
    if _raw_stream is None:
        return torch.cuda.current_stream(t.device).cuda_stream
    return _raw_stream(t.get_device())


def _code(dtype: torch.dtype) -> int:
    if dtype == torch.float32:
        return N.F32
    if dtype == torch.bfloat16:
        return N.BF16
    raise RuntimeError(f"unsupported dtype {dtype}; expected float32 or bfloat16")


def _check(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def _cuda(*tensors: torch.Tensor) -> None:
    dev = tensors[0].get_device()
    for t in tensors:
        if not t.is_cuda:
            raise RuntimeError("expected CUDA (HIP) tensors")
        if t.get_device() != dev:
            raise RuntimeError("all tensors must be on the same device")


def _inference_only() -> None:
    _check(not torch.is_grad_enabled(), "Inference only")


def cached_value(module, name: str, sources, build):
    """``build()``: derived weights (e.g. a bf16 concatenation, or several packed
    weights at once), cached on ``module`` under ``name``.

    Reused only while every source parameter keeps its identity, version
    counter, storage and dtype (the rule of the reference's joint projection
    cache, multiplication.py:29-40, plus the storage address, which a
    ``param.data = ...`` swap changes; an address belongs to one device).
    Inference tensors (parameters made or loaded under
    ``torch.inference_mode``) carry no version counter, so an in-place update of
    one cannot be seen: with such a source the value is rebuilt on every call
    and never cached."""
    cache = module.__dict__.get("_bmx_weight_cache")
    if cache is None:
        cache = module.__dict__["_bmx_weight_cache"] = {}
    hit, key = cache.get(name), None
    # Reading a missing version counter raises, which costs 30 us; asking every source costs 0.2 us each.
    # So a cached value's sources are read at once, and others are asked first.
    if hit is not None:
        try:
            key = [(id(p), p._version, p.data_ptr(), p.dtype) for p in sources]
        except RuntimeError:
            if not any(p.is_inference() for p in sources):
                raise
            cache.pop(name, None)  # an inference tensor has taken a source's place
        else:
            if hit[0] == key:
                return hit[1]
    elif not any(p.is_inference() for p in sources):
        key = [(id(p), p._version, p.data_ptr(), p.dtype) for p in sources]
    with torch.no_grad():
        value = build()
    if key is not None:
        cache[name] = (key, value)
    return value


def cached_weight(module, name: str, sources, build):
    """One derived weight, ``build(*sources)``, cached as ``cached_value`` does."""
    return cached_value(module, name, sources, lambda: build(*sources).contiguous())


def _bf16(*ws):
    return torch.cat([w.detach() for w in ws], 0).to(torch.bfloat16)


def _f32(t):
    return t.detach().to(torch.float32).contiguous()


def _aligned(t):
    """``t``, copied where its storage offset leaves it short of 16-byte alignment."""
    return t if t.data_ptr() % 16 == 0 else t.clone()


def pack_mfma_weights(w):
    """bf16 copy of the row-major matrix ``w`` in MFMA A-operand order
    (``bmx_pack_mfma_weights``): each 32-row x 16-column operand tile becomes
    one contiguous 1 KB run."""
    _cuda(w)
    w = w.detach().to(torch.bfloat16).contiguous()
    rows, cols = w.shape
    out = torch.empty_like(w)
    N.call("bmx_pack_mfma_weights", w.data_ptr(), rows, cols, out.data_ptr(), _stream(w))
    return out


def _bf16_packed(*ws):
    return pack_mfma_weights(_bf16(*ws))


def _workspace(nbytes: int, device) -> torch.Tensor:
    return torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device=device)


# ------------------------------------------------- reference operator set


def norm(x, weight, bias, eps, channel_first=False, waves=None, rows=None, bf16_output=True):
    """LayerNorm over 128 channels (reference ``multiplication_norm``,
    kernels/multiplication_hip.cu:105-156).  ``waves``/``rows`` were gfx90a
    launch-table knobs and are accepted for signature compatibility only."""
    _cuda(x, weight, bias)
    _check(x.is_contiguous() and weight.is_contiguous() and bias.is_contiguous(), "expected contiguous tensors")
    _check(x.dim() == 2 and (x.size(0) == C if channel_first else x.size(1) == C), "expected 128 channels")
    _check(weight.numel() == C and bias.numel() == C and weight.dtype == torch.float32
           and bias.dtype == torch.float32, "expected fp32 weight/bias of 128 elements")
    _inference_only()
    _check(eps > 0, "eps must be positive")
    m = x.size(1) if channel_first else x.size(0)
    out = torch.empty((m, C), device=x.device, dtype=torch.bfloat16 if bf16_output else torch.float32)
    if m:
        N.call("bmx_layernorm128", x.data_ptr(), _code(x.dtype), int(channel_first), weight.data_ptr(),
               bias.data_ptr(), float(eps), out.data_ptr(), _code(out.dtype), m, _stream(x))
    return out


def layer_norm(x, weight, bias, eps):
    """LayerNorm over the last axis (<= 1024 channels) with optional weight/bias."""
    _cuda(x)
    _check(x.is_contiguous(), "expected a contiguous input")
    d = x.shape[-1]
    out = torch.empty_like(x)
    rows = x.numel() // d if d else 0
    w = None if weight is None else _f32(weight)
    b = None if bias is None else _f32(bias)
    if rows:
        N.call("bmx_layernorm", x.data_ptr(), None if w is None else w.data_ptr(), None if b is None else b.data_ptr(),
               float(eps), out.data_ptr(), _code(x.dtype), rows, d, _stream(x))
    return out


def gate(p, g):
    """``bf16(p * bf16(sigmoid(g)))`` (reference ``multiplication_gate``)."""
    _cuda(p, g)
    _check(p.shape == g.shape, "shape mismatch")
    _check(p.dtype == torch.bfloat16 and g.dtype == torch.bfloat16, "expected bf16 inputs")
    _inference_only()
    _check(p.is_contiguous() and g.is_contiguous(), "expected contiguous tensors")
    out = torch.empty_like(p)
    if p.numel():
        N.call("bmx_gate", p.data_ptr(), g.data_ptr(), out.data_ptr(), p.numel(), _stream(p))
    return out


def _check_projection(p, g, mask):
    _cuda(p, g, mask)
    _check(p.shape == g.shape and p.dtype == torch.bfloat16 and g.dtype == torch.bfloat16, "expected bf16 p, g")
    _inference_only()
    _check(p.dim() == 4 and p.size(0) == 1 and p.size(1) == p.size(2) and p.size(3) == 2 * C,
           "expected [1, N, N, 256] projections")
    s = p.stride()
    _check(s[3] == 1 and s[2] in (2 * C, 4 * C) and s[1] == p.size(2) * s[2] and g.stride() == s,
           "Expected dense or joint-projection rows")
    _check(mask.dtype == torch.float32 and mask.is_contiguous() and mask.numel() * 2 * C == p.numel(),
           "expected an fp32 contiguous [1, N, N] mask")
    return s[2]


def split(p, g, mask):
    """Gate and mask into channel-last a, b (reference ``multiplication_gate_split``)."""
    stride = _check_projection(p, g, mask)
    n = p.size(1)
    a = torch.empty((1, n, n, C), device=p.device, dtype=torch.bfloat16)
    b = torch.empty_like(a)
    if n:
        N.call("bmx_trimul_split", p.data_ptr(), g.data_ptr(), mask.data_ptr(), a.data_ptr(), b.data_ptr(), n * n,
               stride, _stream(p))
    return a, b


def pack(p, g, mask, outgoing, channels_per_tile=None):
    """Gate, mask and channel-major operand layout (reference ``multiplication_gate_pack``)."""
    stride = _check_projection(p, g, mask)
    n = p.size(1)
    a = torch.empty((C, n, n), device=p.device, dtype=torch.bfloat16)
    b = torch.empty_like(a)
    if n:
        N.call("bmx_trimul_pack", p.data_ptr(), g.data_ptr(), mask.data_ptr(), a.data_ptr(), b.data_ptr(), n, stride,
               int(bool(outgoing)), _stream(p))
    return a, b


def silu_mul(a, b):
    """``bf16(bf16(silu(a)) * b)`` (reference ``pair_silu_mul``)."""
    _cuda(a, b)
    _check(a.shape == b.shape, "shape mismatch")
    _check(a.dtype == torch.bfloat16 and b.dtype == torch.bfloat16 and a.is_contiguous() and b.is_contiguous(),
           "expected contiguous bf16 inputs")
    _check(not a.requires_grad and not b.requires_grad, "Inference only")
    out = torch.empty_like(a)
    if a.numel():
        N.call("bmx_silu_mul", a.data_ptr(), b.data_ptr(), out.data_ptr(), a.numel(), _stream(a))
    return out


SPLIT_TAIL = 64  # operand columns past 3 k: two ones that meet the split bias, then zeros


def split_width(k: int) -> int:
    """Columns of a split-bf16 operand row for ``k`` input channels."""
    return 3 * k + SPLIT_TAIL


def _row_stride(t) -> int:
    """Element stride between consecutive rows of ``t`` (last axis dense, the
    leading axes collapsing to one row index), e.g. a column slice of a wider
    projection; raises otherwise."""
    _check(t.dim() >= 1 and (t.shape[-1] <= 1 or t.stride(-1) == 1), "the last axis must be dense")
    lead = [(t.shape[i], t.stride(i)) for i in range(t.dim() - 1) if t.shape[i] != 1]
    if not lead:
        return max(t.shape[-1], 1)
    for (_, outer), (n, inner) in zip(lead, lead[1:]):
        _check(outer == inner * n, "the leading axes must collapse to one row index")
    return lead[-1][1]


def _split_out(x, k):
    return torch.empty(x.shape[:-1] + (split_width(k),), device=x.device, dtype=torch.bfloat16)


def split3(x):
    """Split-bf16 operand of fp32 ``x`` (``bmx_split3_bf16``): bf16 [..., 3 k + 64],
    rows [bf16(x) | bf16(x) | bf16(x - bf16(x)) | 1 1 0 ... 0].  ``x`` may be a
    column slice (rows at a stride)."""
    _cuda(x)
    _check(x.dtype == torch.float32 and x.shape[-1] % 4 == 0 and x.shape[-1] > 0,
           "expected fp32 x with a positive multiple of 4 columns")
    k = x.shape[-1]
    out = _split_out(x, k)
    rows = x.numel() // k
    if rows:
        N.call("bmx_split3_bf16", x.data_ptr(), rows, k, _row_stride(x), out.data_ptr(), _stream(x))
    return out


def layernorm_split3(x, eps):
    """Split-bf16 operand of LayerNorm-without-affine(x) (``bmx_layernorm_split3_bf16``)."""
    _cuda(x)
    _check(x.dtype == torch.float32 and 0 < x.shape[-1] <= 1024 and x.shape[-1] % 4 == 0,
           "expected fp32 x with a multiple of 4 columns, at most 1024")
    k = x.shape[-1]
    out = _split_out(x, k)
    rows = x.numel() // k
    if rows:
        N.call("bmx_layernorm_split3_bf16", x.data_ptr(), rows, k, _row_stride(x), float(eps), out.data_ptr(),
               _stream(x))
    return out


def layernorm_split3_t(x, eps):
    """``layernorm_split3`` of the rows of ``x.transpose(0, 1)`` for a square
    pair frame x [N, N, k] with dense rows, without the transposed copy
    (``bmx_layernorm_split3_t_bf16``); bf16 [N, N, 3 k + 64].  Part of the
    public operator set; no module of this package calls it any more."""
    _cuda(x)
    _check(x.dim() == 3 and x.shape[0] == x.shape[1] and x.dtype == torch.float32 and x.is_contiguous()
           and 0 < x.shape[-1] <= 1024 and x.shape[-1] % 4 == 0,
           "expected contiguous fp32 x [N, N, k] with a multiple of 4 columns, at most 1024")
    n, k = x.shape[0], x.shape[-1]
    out = _split_out(x, k)
    if n:
        N.call("bmx_layernorm_split3_t_bf16", x.data_ptr(), n, k, k, float(eps), out.data_ptr(), _stream(x))
    return out


def _same_rows(a, *mods):
    """Row stride shared by ``mods`` (column slices of one projection, or dense
    tensors of a's shape)."""
    _check(all(m.shape == a.shape and m.dtype == a.dtype and m.device == a.device for m in mods),
           "shape/dtype mismatch")
    lds = {_row_stride(m) for m in mods}
    _check(len(lds) == 1, "the modulation operands must share one row stride")
    return lds.pop()


def adaln_split3(a, scale, shift, eps):
    """Split-bf16 operand of ``sigmoid(scale) * LN_noaffine(a) + shift``
    (``bmx_adaln_split3_bf16``); scale and shift may be column slices of one
    wider fp32 projection (rows at one stride)."""
    _cuda(a, scale, shift)
    _check(a.dtype == torch.float32 and a.is_contiguous(), "expected contiguous fp32 a")
    d = a.shape[-1]
    _check(0 < d <= 1024 and d % 4 == 0, "expected a multiple of 4 channels, at most 1024")
    ld = _same_rows(a, scale, shift)
    out = _split_out(a, d)
    rows = a.numel() // d
    if rows:
        N.call("bmx_adaln_split3_bf16", a.data_ptr(), scale.data_ptr(), shift.data_ptr(), ld, rows, d, float(eps),
               out.data_ptr(), _stream(a))
    return out


def gated_residual_adaln_split3(a, gate, c, scale, shift, eps, out=None):
    """``r = c + sigmoid(gate) * a`` (fp32, into ``out``, which may be ``c``) and
    the split-bf16 operand of ``sigmoid(scale) * LN_noaffine(r) + shift`` in one
    pass (``bmx_gated_residual_adaln_split3_bf16``); gate, scale and shift may
    be column slices.  Returns (r, operand)."""
    _cuda(a, gate, c, scale, shift)
    _check(a.dtype == c.dtype == torch.float32 and a.is_contiguous() and c.is_contiguous() and a.shape == c.shape,
           "expected contiguous fp32 a and c of one shape")
    d = a.shape[-1]
    _check(0 < d <= 1024 and d % 4 == 0, "expected a multiple of 4 channels, at most 1024")
    ldg = _same_rows(a, gate)
    ldm = _same_rows(a, scale, shift)
    if out is None:
        out = torch.empty_like(a)
    _check(out.shape == a.shape and out.is_contiguous() and out.dtype == torch.float32, "bad out")
    op = _split_out(a, d)
    rows = a.numel() // d
    if rows:
        N.call("bmx_gated_residual_adaln_split3_bf16", a.data_ptr(), gate.data_ptr(), ldg, c.data_ptr(), out.data_ptr(),
               scale.data_ptr(), shift.data_ptr(), ldm, rows, d, float(eps), op.data_ptr(), _stream(a))
    return out, op


def swiglu_split3(u, cols):
    """Split-bf16 operand of ``silu(g) * x * b`` for rows [x | g | b | ...] of
    fp32 ``u`` (``cols`` values each; ``bmx_swiglu_split3_bf16``)."""
    _cuda(u)
    _check(u.dtype == torch.float32 and cols > 0 and cols % 4 == 0 and u.shape[-1] >= 3 * cols,
           "expected fp32 u with at least 3 cols columns, cols a multiple of 4")
    out = torch.empty(u.shape[:-1] + (split_width(cols),), device=u.device, dtype=torch.bfloat16)
    rows = u.numel() // u.shape[-1]
    if rows:
        N.call("bmx_swiglu_split3_bf16", u.data_ptr(), _row_stride(u), rows, cols, out.data_ptr(), _stream(u))
    return out


def gated_residual(a, gate, c, out=None):
    """``c + sigmoid(gate) * a`` (fp32, ``bmx_gated_residual``; the MODULATION
    epilogue) with ``gate`` possibly a column slice of a wider projection;
    ``out`` may be ``c``."""
    _cuda(a, gate, c)
    _check(a.dtype == gate.dtype == c.dtype == torch.float32, "expected fp32 operands")
    _check(a.is_contiguous() and c.is_contiguous() and a.shape == c.shape == gate.shape, "shape mismatch")
    if out is None:
        out = torch.empty_like(a)
    _check(out.shape == a.shape and out.is_contiguous() and out.dtype == torch.float32, "bad out")
    cols = a.shape[-1]
    rows = a.numel() // cols if cols else 0
    if rows:
        N.call("bmx_gated_residual", a.data_ptr(), gate.data_ptr(), _row_stride(gate), c.data_ptr(), out.data_ptr(),
               rows, cols, _stream(a))
    return out


def _x3_weight(w, b=None):
    """Weight rows [Wh | Wl | Wh | bh bl 0 ... 0] (Wh = bf16(W), Wl = bf16(W - Wh),
    likewise for the bias), bf16 [N, 3 K + 64], for W [N, K] and bias b [N] or None."""
    w = w.detach().float()
    hi = w.to(torch.bfloat16)
    lo = (w - hi.float()).to(torch.bfloat16)
    tail = torch.zeros(w.shape[0], SPLIT_TAIL, device=w.device, dtype=torch.bfloat16)
    if b is not None:
        b = b.detach().float()
        bh = b.to(torch.bfloat16)
        tail[:, 0] = bh
        tail[:, 1] = (b - bh.float()).to(torch.bfloat16)
    return torch.cat([hi, lo, hi, tail], dim=1)


def x3_weight(module, name, weights, biases=None):
    """Split weight of ``mm_split`` for the row concatenation of ``weights``
    ([N_i, K] each) with the biases ``biases`` (one per weight, None for none),
    cached on ``module`` under ``name``."""
    weights = tuple(weights)
    biases = tuple(biases) if biases is not None else (None,) * len(weights)
    _check(len(biases) == len(weights), "one bias (or None) per weight")
    present = tuple(b for b in biases if b is not None)

    def build(*srcs):
        ws = srcs[:len(weights)]
        b = None
        if present:
            it = iter(srcs[len(weights):])
            b = torch.cat([next(it).detach().float() if bb is not None else w.new_zeros(w.shape[0], dtype=torch.float32)
                           for bb, w in zip(biases, ws)])
        return _x3_weight(torch.cat(ws, 0), b)

    return cached_weight(module, name, weights + present, build)


def mm_split(op, w3):
    """``x @ W^T + b`` from the split operand ``op`` of x ([M, 3 K + 64] bf16)
    and ``w3 = x3_weight(..W.., ..b..)``: one hipBLASLt bf16 GEMM with fp32
    accumulation (x W + b up to about 2^-16 relative per product); fp32 [M, N]."""
    _check(op.dim() == 2 and op.shape[1] == w3.shape[1], "operand does not match the split weight")
    return torch.mm(op, w3.t(), out_dtype=torch.float32)


def mm_x3(x, w3):
    """``mm_split(split3(x), w3)`` for fp32 x [M, K]."""
    _check(x.dim() == 2 and w3.shape[1] == split_width(x.shape[1]), "x does not match the split weight")
    return mm_split(split3(x.float()), w3)


# fp32 linears run as split-bf16 GEMMs from 512 input channels up (the token
# transformer's 768 / 1536: ~1.5x faster per block), and from 128 up when
# they are tall (the atom transformer's 5 x 8192 rows at 128 / 256 channels:
# 46.5 against 65.3 us at N = 512, 53 against 89 us at N = 768, 0.23 ms per
# configs[4] step).  Short narrow ones (the Pairformer sequence stack's 1024
# rows of 384) stay on hipBLASLt's fp32 GEMM, and so do tall narrow ones with
# fewer than 512 outputs whose operand needs a split pass of its own (40 960 x
# 128: 12 us for the pass + 27 us against 29 us in fp32 at N = 128).
X3_MIN_K = 512
X3_TALL_MIN_K, X3_TALL_MIN_ROWS, X3_TALL_MIN_N = 128, 16384, 512

# Set BMX_EXACT_FP32_LINEARS=1 (or call exact_fp32_linears(True)) to run every
# fp32 linear of the diffusion blocks and of fp32-mode triangle attention as a
# true fp32 GEMM and fp32-mode attention on fp32 MFMA, as the reference does,
# instead of the split-bf16 form (about 2^-16 relative per product).
_EXACT_FP32 = [os.environ.get("BMX_EXACT_FP32_LINEARS", "0") not in ("", "0")]


def exact_fp32_linears(enabled: bool = True) -> bool:
    """Switch ``linear_fp32`` between the split-bf16 GEMM (False, default) and
    the plain fp32 GEMM (True) for the whole process; returns the previous
    setting."""
    before = _EXACT_FP32[0]
    _EXACT_FP32[0] = bool(enabled)
    return before


def use_split(k: int, rows: int = 0, n: int | None = None) -> bool:
    """Whether fp32 linears of ``k`` input channels over ``rows`` rows run as
    split-bf16 GEMMs (never in exact fp32 mode).  ``n``: the GEMM's outputs
    when its operand is split for it alone (None: a shared split operand)."""
    if _EXACT_FP32[0] or k % 4:
        return False
    return k >= X3_MIN_K or (k >= X3_TALL_MIN_K and rows >= X3_TALL_MIN_ROWS and (n is None or n >= X3_TALL_MIN_N))


def linear_fp32(x, linear):
    """``linear(x)`` for fp32 x: ``linear_x3`` where ``use_split`` says so
    (never with exact fp32 linears switched on), else the fp32 GEMM."""
    if use_split(x.shape[-1], x.numel() // max(x.shape[-1], 1), linear.weight.shape[0]):
        return linear_x3(x, linear)
    return torch.nn.functional.linear(x, linear.weight, linear.bias)


def linear_x3(x, linear):
    """``linear(x)`` for fp32 x through ``mm_x3``, the bias folded into the GEMM."""
    _cuda(x)
    k = x.shape[-1]
    _check(linear.weight.shape[1] == k, "x does not match the linear's input width")
    w = x3_weight(linear, "x3", (linear.weight,), (linear.bias,))
    y = mm_x3(x.reshape(-1, k), w)
    return y.view(x.shape[:-1] + (w.shape[0],))


def x3_pack(out, tile0, w, tile_stride=1, col_scale=None):
    """Weight rows ``w`` [N, K] (times ``col_scale`` [K] per column) into the
    packed split operand ``out`` (``bmx_x3_pack``): 32-row tile t at tile
    ``tile0 + t * tile_stride``."""
    w, rows, k = _f32(w), *w.shape
    scale = None
    if col_scale is not None:
        scale = _f32(col_scale)
        _check(scale.shape == (k,), "expected one column scale per column")
        _cuda(out, scale)
    if out.get_device() != w.get_device() or not w.is_cuda:
        _cuda(out, w)
    _check(rows % 32 == 0 and (tile0 + (rows // 32 - 1) * tile_stride + 1) * 64 * k <= out.numel(),
           "the weight's 32-row tiles do not fit the packed operand")
    N.call("bmx_x3_pack", w.data_ptr(), rows, k, k, None if scale is None else scale.data_ptr(), tile0, tile_stride,
           out.data_ptr(), _stream(w))


MODULATION, GATE, GATED_SWIGLU = 0, 1, 3


def epilogue(a, b, c, kind):
    """Diffusion epilogues (reference ``diffusion_epilogue``, op codes diffusion.py:27)."""
    _check(kind in (MODULATION, GATE, GATED_SWIGLU), "unknown epilogue kind")
    _cuda(a, b)
    _check(a.dtype == b.dtype and a.dtype in (torch.float32, torch.bfloat16), "expected fp32 or bf16 inputs")
    _check(a.is_contiguous() and b.is_contiguous(), "expected contiguous inputs")
    shape = list(a.shape)
    cols = shape[-1]
    if kind == GATED_SWIGLU:
        _check(cols % 2 == 0, "SwiGLU input needs an even last dimension")
        cols //= 2
        shape[-1] = cols
    _check(list(b.shape) == shape, "b must match the output shape")
    if kind == MODULATION:
        _check(c is not None and list(c.shape) == shape and c.dtype == a.dtype and c.is_contiguous()
               and c.device == a.device, "MODULATION needs c of the output shape")
    out = torch.empty(shape, device=a.device, dtype=a.dtype)
    n = out.numel()
    if n:
        N.call("bmx_diffusion_epilogue", kind, a.data_ptr(), b.data_ptr(), None if c is None else c.data_ptr(),
               out.data_ptr(), _code(a.dtype), n // cols, cols, _stream(a))
    return out


def ordered_softmax(scores, bias, mask, *, rows=None, waves_per_eu=None, allow_large=False):
    """``softmax(round(round(scores + mask) + bias))`` over keys
    (reference ``ordered_softmax``, kernels/triangle_softmax.py:117-161).
    scores [B,I,H,Q,K], bias [B,1,H,Q,K] (broadcast over I), mask [B,I,1,1,K]."""
    if torch.is_grad_enabled() or scores.dtype not in (torch.float32, torch.bfloat16) or scores.ndim != 5:
        raise ValueError("Expected inference-only FP32/BF16 triangle scores")
    bt, i, h, q, k = scores.shape
    if q <= 0 or k != q:
        raise ValueError("Expected nonempty square score matrices")
    _cuda(scores, bias, mask)
    if bias.dtype != scores.dtype or mask.dtype != torch.float32:
        raise ValueError("bias must match the score dtype and mask must be fp32")
    out = torch.empty(scores.shape, device=scores.device, dtype=scores.dtype)
    N.call("bmx_bias_softmax", scores.data_ptr(), bias.data_ptr(), mask.data_ptr(), out.data_ptr(),
           _code(scores.dtype), N.int64_array(scores.shape), N.int64_array(scores.stride()),
           N.int64_array(bias.stride()), N.int64_array(mask.stride()), _stream(scores))
    return out


# ----------------------------------------------------- fused hot-path ops

# out_mode: write bf16 / write fp32 / out += y (in-place residual) / out = x + y
OUT_BF16, OUT_F32, OUT_ACCUMULATE, OUT_RESIDUAL = 0, 1, 2, 3
ALL_STAGES = 7


def _out_tensor(x, out, out_mode):
    if out_mode == OUT_ACCUMULATE:
        _check(out is not None and out.dtype == torch.float32 and out.shape == x.shape and out.is_contiguous(),
               "accumulate mode needs an fp32 contiguous `out` of x's shape")
        return out
    dtype = torch.bfloat16 if out_mode == OUT_BF16 else torch.float32
    if out is None:
        return torch.empty(x.shape, device=x.device, dtype=dtype)
    _check(out.dtype == dtype and out.shape == x.shape and out.is_contiguous(), "bad `out` tensor")
    if out_mode == OUT_RESIDUAL:
        _check(out.data_ptr() != x.data_ptr(), "residual-write mode needs `out` distinct from x")
    return out


def _row_scale(row_scale, x, n):
    """Checked fp32 [n] row scale (or None) for the fused modules' output kernels."""
    if row_scale is None:
        return None
    _cuda(x, row_scale)
    _check(row_scale.dtype == torch.float32 and row_scale.numel() == n and row_scale.is_contiguous(),
           "expected a contiguous fp32 row scale of n values")
    return row_scale


def trimul(module, x, mask, outgoing, out_mode=OUT_BF16, out=None, workspace=None, stages=ALL_STAGES,
           row_scale=None):
    """Fused TriangleMultiplication{Outgoing,Incoming} for x [N, N, 128] fp32.

    ``stages`` selects the kernels (1 projection, 2 contraction, 4 output);
    separate calls must share ``workspace``.  ``row_scale`` (fp32 [N] or None)
    multiplies output row i (before the residual add): PairformerLayer's
    row-wise dropout mask."""
    _cuda(x, mask)
    _check(x.dim() == 3 and x.size(0) == x.size(1) and x.size(2) == C, "expected x of shape [N, N, 128]")
    _check(x.dtype == torch.float32 and x.is_contiguous(), "expected contiguous fp32 x")
    _check(mask.shape == x.shape[:2] and mask.dtype == torch.float32 and mask.is_contiguous(),
           "expected a contiguous fp32 [N, N] mask")
    n = x.size(0)
    ni, no = module.norm_in, module.norm_out
    srcs = (module.p_in.weight, module.g_in.weight, module.p_out.weight, module.g_out.weight, ni.weight, ni.bias,
            no.weight, no.bias)
    w_in, w_pout, w_gout, niw, nib, now, nob = cached_value(module, "trimul", srcs, lambda: (
        _bf16(*srcs[:2]), _bf16(srcs[2]), _bf16(srcs[3]), *map(_f32, srcs[4:])))
    out = _out_tensor(x, out, out_mode)
    rs = _row_scale(row_scale, x, n)
    nbytes = N.lib().bmx_trimul_workspace_bytes(n)
    ws = workspace if workspace is not None and workspace.numel() >= nbytes else _workspace(nbytes, x.device)
    if n:
        N.call("bmx_trimul_fwd", x.data_ptr(), mask.data_ptr(), n, int(bool(outgoing)), niw.data_ptr(),
               nib.data_ptr(), float(ni.eps), w_in.data_ptr(), now.data_ptr(), nob.data_ptr(), float(no.eps),
               w_pout.data_ptr(), w_gout.data_ptr(), out.data_ptr(), out_mode, None if rs is None else rs.data_ptr(),
               ws.data_ptr(), ws.numel(), stages, _stream(x))
    return out


def workspace_bytes(n: int) -> int:
    """Workspace that serves both fused triangle ops at size n."""
    lib = N.lib()
    return max(lib.bmx_trimul_workspace_bytes(n), lib.bmx_triattn_workspace_bytes(n))


def new_workspace(n: int, device) -> torch.Tensor:
    return _workspace(workspace_bytes(n), device)


def _triattn_proj_weight(wq, wk, wv, wb):
    rows = N.lib().bmx_triattn_proj_rows()
    w = torch.zeros((rows, C), dtype=torch.bfloat16, device=wq.device)
    used = torch.cat([wq, wk, wv, wb], 0)
    w[: used.shape[0]] = used.to(torch.bfloat16)
    return w


def triattn(module, x, mask, starting, out_mode=OUT_BF16, out=None, workspace=None, stages=ALL_STAGES,
            row_scale=None):
    """Fused TriangleAttention (starting or ending node) for x [N, N, 128].

    ``module`` carries Boltz's TriangleAttention parameters: ``layer_norm``,
    ``linear`` (triangle bias), ``mha.linear_{q,k,v,g,o}``, ``inf``.
    ``stages`` selects the kernels (1 projection, 2 attention core, 4 output).
    ``row_scale`` (fp32 [N] or None) multiplies the output of x's row i
    (starting) or column i (ending) before the residual add:
    PairformerLayer's dropout mask (row-wise / column-wise)."""
    _cuda(x)
    _check(x.dim() == 3 and x.size(0) == x.size(1) and x.size(2) == C, "expected x of shape [N, N, 128]")
    _check(x.dtype in (torch.float32, torch.bfloat16) and x.is_contiguous(), "expected contiguous fp32/bf16 x")
    n = x.size(0)
    if mask is not None:
        _cuda(x, mask)
        _check(mask.shape == x.shape[:2] and mask.dtype == torch.float32 and mask.is_contiguous(),
               "expected a contiguous fp32 [N, N] mask")
    mha = module.mha
    ln, lg, lo = module.layer_norm, mha.linear_g, mha.linear_o
    srcs = (mha.linear_q.weight, mha.linear_k.weight, mha.linear_v.weight, module.linear.weight, lg.weight, lo.weight,
            lg.bias, lo.bias, ln.weight, ln.bias)
    w_proj, w_g, w_o, b_g, b_o, lnw, lnb = cached_value(module, "triattn", srcs, lambda: (
        _triattn_proj_weight(*srcs[:4]), _bf16(srcs[4]), _bf16(srcs[5]), *map(_f32, srcs[6:])))
    out = _out_tensor(x, out, out_mode)
    rs = _row_scale(row_scale, x, n)
    nbytes = N.lib().bmx_triattn_workspace_bytes(n)
    ws = workspace if workspace is not None and workspace.numel() >= nbytes else _workspace(nbytes, x.device)
    if n:
        N.call("bmx_triattn_fwd", x.data_ptr(), _code(x.dtype), None if mask is None else mask.data_ptr(), n,
               int(bool(starting)), float(module.inf), lnw.data_ptr(), lnb.data_ptr(), float(ln.eps),
               w_proj.data_ptr(), w_g.data_ptr(), b_g.data_ptr(), w_o.data_ptr(), b_o.data_ptr(), out.data_ptr(),
               out_mode, None if rs is None else rs.data_ptr(), ws.data_ptr(), ws.numel(), stages, _stream(x))
    return out


def _triattn_fp32_split_weights(module):
    """fp32 mode's weights: q | k | v | g packed as a split operand, their biases
    and the triangle bias's [512 + 4], the triangle-bias rows as bf16 [high,
    low][16][128], the LayerNorm's weight and bias (or None) and linear_o's."""
    mha, ln, lo = module.mha, module.layer_norm, module.mha.linear_o
    lins = (mha.linear_q, mha.linear_k, mha.linear_v, mha.linear_g, module.linear)

    def build():
        shapes = [(C, C)] * 4 + [(4, C), (C, C)]
        _check(all(lin.weight.shape == shape and (lin.bias is None or lin.bias.shape == shape[:1])
                   for lin, shape in zip(lins + (lo,), shapes)) and lo.bias is not None,
               "expected 128 -> 128 and 128 -> 4 projections and a linear_o with a bias")
        _check(ln.weight.shape == (C,) and (ln.bias is None or ln.bias.shape == (C,)),
               "expected a LayerNorm of 128 channels")
        _cuda(*srcs)
        w = torch.empty(2 * 4 * C * C, device=lo.weight.device, dtype=torch.bfloat16)
        for i, lin in enumerate(lins[:4]):
            x3_pack(w, i * C // 32, lin.weight)
        b = torch.cat([lin.bias.detach().float() if lin.bias is not None
                       else lin.weight.new_zeros(lin.out_features, dtype=torch.float32) for lin in lins])
        rows = module.linear.weight.detach().float()
        rows = torch.cat([rows, rows.new_zeros(16 - rows.shape[0], C)])
        hi = rows.to(torch.bfloat16)
        return (w, b, torch.stack([hi, (rows - hi.float()).to(torch.bfloat16)]).contiguous(),
                *(None if t is None else _aligned(_f32(t)) for t in (ln.weight, ln.bias, lo.weight, lo.bias)))

    srcs = [t for lin in lins + (ln, lo) for t in (lin.weight, lin.bias) if t is not None]
    return cached_value(module, "fp32_proj_x3", srcs, build)


def _triattn_fp32_native(module, weights, x, mask, starting, tri_bias, stages, row0, rows, out=None, ws=None):
    """One ``bmx_triattn_fp32_fwd`` call on frame rows row0 .. row0 + rows - 1;
    ``weights``: ``_triattn_fp32_split_weights``."""
    w, b, wb, lnw, lnb = weights[:5]
    N.call("bmx_triattn_fp32_fwd", x.data_ptr(), None if mask is None else mask.data_ptr(), x.shape[0], int(starting),
           row0, rows, float(module.inf), lnw.data_ptr(), None if lnb is None else lnb.data_ptr(),
           float(module.layer_norm.eps), w.data_ptr(), b.data_ptr(), wb.data_ptr(), tri_bias.data_ptr(), stages,
           None if out is None else out.data_ptr(), None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(),
           _stream(x))


def _triattn_fp32_exact_weights(module):
    """fp32 q | k | v | g weight [512, 128] and bias (linear_g's only)."""
    mha = module.mha
    w = cached_weight(module, "qkvg_f32", (mha.linear_q.weight, mha.linear_k.weight, mha.linear_v.weight,
                                           mha.linear_g.weight), lambda *ws: torch.cat(ws, 0).float())
    b = cached_weight(module, "qkvg_bias_f32", (mha.linear_g.bias,),
                      lambda bg: torch.cat([bg.new_zeros(3 * C), bg]).float())
    return w, b


def triattn_fp32(module, x, mask, starting, block_rows=None):
    """TriangleAttention (starting or ending node) in fp32 for x [N, N, 128]
    fp32, the fp32 mode of the module (autocast off; reference
    triangle.py:38-52 accelerates it too).  One kernel normalises x, projects
    q | k | v | g and the triangle bias with split-bf16 products (about 2^-16
    relative each) and writes the attention's operands
    (``bmx_triattn_fp32_fwd``; the ending node reads x's columns in place); the
    attention, mask bias, softmax, PV product and gate run fused on split-bf16
    products, two rows sharing each fetch of the [4, N, N] triangle bias, so the
    [N, 4, N, N] scores never reach HBM; ``linear_o`` runs in place on the fp32
    matrix cores.  In exact fp32 mode the fp32
    LN128 kernel, fp32 GEMMs and the fp32-MFMA attention run instead.  Returns
    fp32 [N, N, 128].

    ``block_rows`` < N processes the rows of the frame (x's rows for the
    starting node, its columns for the ending node) in blocks of that many
    (``_triattn_fp32_blocked``): the same products, with the per-pair working
    set held for one block at a time."""
    _cuda(x)
    _check(x.dim() == 3 and x.size(0) == x.size(1) and x.size(2) == C and x.dtype == torch.float32,
           "expected fp32 x of shape [N, N, 128]")
    n = x.size(0)
    mha, heads, d = module.mha, module.no_heads, module.c_hidden
    _check(heads * d == C, "expected heads x head dim = 128")
    if block_rows is not None and 0 < block_rows < n:
        return _triattn_fp32_blocked(module, x, mask, starting, int(block_rows))
    ln = module.layer_norm
    if not _EXACT_FP32[0] and ln.weight is not None and heads == 4:
        return _triattn_fp32_split(module, x.contiguous(), mask, starting, n)
    if not starting:
        mask = None if mask is None else mask.transpose(0, 1)
        x = x.transpose(0, 1)
    x = x.contiguous()
    xn = norm(x.view(-1, C), _f32(ln.weight), _f32(ln.bias), ln.eps, bf16_output=False)
    w, b = _triattn_fp32_exact_weights(module)
    proj = torch.nn.functional.linear(xn, w, b).view(n, n, 4 * C)
    tri_bias = torch.nn.functional.linear(xn, module.linear.weight.float()).view(n, n, heads)
    tri_bias = tri_bias.permute(2, 0, 1).contiguous()  # [H, q, k], shared by every row
    m = x.new_ones(n, n) if mask is None else mask.to(torch.float32).contiguous()
    q, k, v, g = proj.split(C, dim=-1)
    o = seq_attention_batched(q, k, v, tri_bias[None], m, g, module.inf, bias_div=n, split=False)
    del q, k, v, g, proj, tri_bias  # 2.3 KB per pair, before linear_o's output is allocated
    out = torch.nn.functional.linear(o, mha.linear_o.weight.float(), mha.linear_o.bias.float())
    return out if starting else out.transpose(0, 1)


def _triattn_fp32_split(module, x, mask, starting, rows):
    """``triattn_fp32`` on split-bf16 products in blocks of ``rows`` frame rows
    (all of them in one block: one kernel writes the triangle bias, which every
    row shares, beside the rows' operands; several blocks: a first pass writes
    it for all rows)."""
    n, x, m = x.shape[0], _aligned(x), None
    if mask is not None:
        if mask.shape != x.shape[:2]:
            _check(mask.shape == ((1, n) if starting else (n, 1)),
                   "expected a mask of [N, N], or one row (starting) or column (ending) of it")
            mask = mask.expand(n, n)
        m = mask.to(torch.float32).contiguous()
    tri_bias = torch.empty(4, n, (n + 63) // 64 * 64, device=x.device, dtype=torch.float32)
    ws = _workspace(N.lib().bmx_triattn_fp32_workspace_bytes(n, rows), x.device)
    weights = _triattn_fp32_split_weights(module)
    w_o, b_o = weights[5:]
    for t in (w_o,) if m is None else (w_o, m):  # all weights are on one device
        if t.get_device() != x.get_device():
            _cuda(x, t)
    out = torch.empty(n, n, C, device=x.device, dtype=torch.float32)  # the attention's output, then linear_o's

    def linear_o(o):
        N.call("bmx_linear128_f32_fwd", o.data_ptr(), o.shape[0] * n, w_o.data_ptr(), b_o.data_ptr(), o.data_ptr(),
               _stream(x))

    if rows >= n:
        if n:
            _triattn_fp32_native(module, weights, x, m, starting, tri_bias, 3, 0, n, out, ws)
            linear_o(out)
    else:
        rows -= rows % 2 if rows > 1 else 0  # the attention pairs rows: the pairs of one pass
        _triattn_fp32_native(module, weights, x, m, starting, tri_bias, 1, 0, n)
        for i0 in range(0, n, rows):
            o = out[i0:i0 + rows]
            _triattn_fp32_native(module, weights, x, m, starting, tri_bias, 2, i0, o.shape[0], o, ws)
            linear_o(o)
    return out if starting else out.transpose(0, 1)


def _triattn_fp32_blocked(module, x, mask, starting, rows):
    """``triattn_fp32`` over blocks of ``rows`` frame rows (x's rows for the
    starting node, x's columns for the ending node).  A first pass writes the
    [H, N, N] triangle bias, which every row shares; a second pass runs each
    block's projection, the fused attention over the block's rows and
    ``linear_o`` into the output frame.  Full-frame memory: the output, the
    bias and the mask (about 532 bytes per pair); the rest is per block.  Exact
    fp32 mode copies the ending node's columns transposed one block at a time
    and computes the bias from each block's LayerNorm and only the bias rows of
    the projection weight."""
    n = x.size(0)
    mha, heads, ln = module.mha, module.no_heads, module.layer_norm
    if not _EXACT_FP32[0] and ln.weight is not None and heads == 4:
        return _triattn_fp32_split(module, x.contiguous(), mask, starting, rows)
    if mask is None:
        m = x.new_ones(n, n)
    else:
        m = (mask if starting else mask.transpose(0, 1)).to(torch.float32).contiguous()

    def features(i0, i1):  # LayerNorm of frame rows i0 .. i1 - 1: [(i1 - i0) N, 128] fp32
        xb = x[i0:i1].contiguous() if starting else x[:, i0:i1].transpose(0, 1).contiguous()
        return norm(xb.view(-1, C), _f32(ln.weight), _f32(ln.bias), ln.eps, bf16_output=False)

    w, b = _triattn_fp32_exact_weights(module)
    w_bias = module.linear.weight.float()
    blocks = [(i0, min(n, i0 + rows)) for i0 in range(0, n, rows)]
    tri_bias = torch.empty(heads, n, n, device=x.device, dtype=torch.float32)  # [H, q, k]
    for i0, i1 in blocks:
        bias = torch.nn.functional.linear(features(i0, i1), w_bias)
        tri_bias[:, i0:i1] = bias.view(i1 - i0, n, heads).permute(2, 0, 1)
        del bias
    out = torch.empty(n, n, C, device=x.device, dtype=torch.float32)  # the output frame
    w_o, b_o = mha.linear_o.weight.float(), mha.linear_o.bias.float()
    for i0, i1 in blocks:
        proj = torch.nn.functional.linear(features(i0, i1), w, b).view(i1 - i0, n, -1)
        q, k, v, g = proj.split(C, dim=-1)
        o = seq_attention_batched(q, k, v, tri_bias[None], m[i0:i1], g, module.inf, bias_div=i1 - i0, split=False)
        del q, k, v, g, proj
        torch.addmm(b_o, o.view(-1, C), w_o.t(), out=out[i0:i1].view(-1, C))
        del o
    return out if starting else out.transpose(0, 1)


def pair_transition(module, x, out_mode=OUT_BF16, out=None, pair_bias=None):
    """Fused Transition(128, 512) over the rows of x [..., 128].

    ``pair_bias=(proj_z_norm, proj_z_linear, bias_out)`` also writes the
    sequence stack's pair bias of the result (``pair_bias`` below applied to
    ``out``) into ``bias_out`` [16, rows] in the same pass; it needs an fp32
    ``out_mode``."""
    _cuda(x)
    _check(x.shape[-1] == C and x.dtype in (torch.float32, torch.bfloat16) and x.is_contiguous(),
           "expected contiguous fp32/bf16 x with 128 channels")
    fc1, fc3 = module.fc1.weight, module.fc3.weight
    _check(fc1.shape == (4 * C, C) and fc3.shape == (C, 4 * C), "expected a 128 -> 512 -> 128 transition")
    ln = module.norm
    srcs = (fc1, module.fc2.weight, fc3, ln.weight, ln.bias)
    w12, w3, lnw, lnb = cached_value(module, "transition", srcs, lambda: (
        _bf16_packed(*srcs[:2]), _bf16_packed(srcs[2]), _f32(srcs[3]), _f32(srcs[4])))
    out = _out_tensor(x, out, out_mode)
    rows = x.numel() // C
    if pair_bias is None:
        if rows:
            N.call("bmx_pair_transition_fwd", x.data_ptr(), _code(x.dtype), rows, lnw.data_ptr(), lnb.data_ptr(),
                   float(ln.eps), w12.data_ptr(), w3.data_ptr(), out.data_ptr(), out_mode, _stream(x))
        return out
    norm, lin, bias_out = pair_bias
    _check(out_mode != OUT_BF16, "the fused pair bias needs an fp32 out_mode")
    _check(lin.weight.shape == (16, C), "expected a 128 -> 16 projection")
    _check(bias_out.numel() == 16 * rows and bias_out.dtype == torch.float32 and bias_out.is_contiguous(),
           "bias_out must be a contiguous fp32 tensor of 16 x rows")
    fold = cached_weight(lin, "pair_bias_fold", (norm.weight, norm.bias, lin.weight), pair_bias_fold)
    if rows:
        N.call("bmx_pair_transition_bias_fwd", x.data_ptr(), _code(x.dtype), rows, lnw.data_ptr(), lnb.data_ptr(),
               float(ln.eps), w12.data_ptr(), w3.data_ptr(), out.data_ptr(), out_mode, fold.data_ptr(),
               float(norm.eps), bias_out.data_ptr(), _stream(x))
    return out


def pair_bias_fold(ln_w, ln_b, w):
    """Folded pair-bias weights (``bmx_pair_bias_fold``): the LayerNorm affine
    folded into the 128 -> 16 projection, in the fused epilogue's operand order."""
    _cuda(ln_w, ln_b, w)
    _check(ln_w.shape == (C,) and ln_b.shape == (C,) and w.shape == (16, C), "expected a 128 -> 16 projection")
    ln_w, ln_b, w = (_f32(t) for t in (ln_w, ln_b, w))
    out = torch.empty(N.lib().bmx_pair_bias_fold_bytes(), dtype=torch.uint8, device=w.device)
    N.call("bmx_pair_bias_fold", ln_w.data_ptr(), ln_b.data_ptr(), w.data_ptr(), 16, out.data_ptr(), _stream(w))
    return out


def pair_bias(proj_z_norm, proj_z_linear, z, out=None):
    """fp32 ``Linear(LN(z))`` for 16 heads, returned (or written into ``out``)
    head-major as [H, N, N] (the layout AttentionPairBias adds to its logits);
    z is [N, N, 128]."""
    _cuda(z)
    _check(z.dim() == 3 and z.shape[-1] == C and z.dtype in (torch.float32, torch.bfloat16) and z.is_contiguous(),
           "expected contiguous z of shape [N, N, 128]")
    heads = proj_z_linear.weight.shape[0]
    _check(heads == 16 and proj_z_linear.weight.shape[1] == C, "expected a 128 -> 16 projection")
    w = cached_weight(proj_z_linear, "w32", (proj_z_linear.weight,), _f32)
    lnw = cached_weight(proj_z_norm, "w32", (proj_z_norm.weight,), _f32)
    lnb = cached_weight(proj_z_norm, "b32", (proj_z_norm.bias,), _f32)
    shape = (heads, z.shape[0], z.shape[1])
    if out is None:
        out = torch.empty(shape, device=z.device, dtype=torch.float32)
    _check(out.shape == shape and out.dtype == torch.float32 and out.is_contiguous(),
           "out must be a contiguous fp32 [16, N, N]")
    rows = z.shape[0] * z.shape[1]
    if rows:
        N.call("bmx_pair_bias_fwd", z.data_ptr(), _code(z.dtype), rows, lnw.data_ptr(), lnb.data_ptr(),
               float(proj_z_norm.eps), w.data_ptr(), heads, out.data_ptr(), _stream(z))
    return out


def seq_attention(q, k, v, bias, mask, g, inf, out=None):
    """Pair-biased softmax attention of AttentionPairBias, fp32, for one batch
    element: q, k, v and the gate logits g are [N, H * D] (D = 24 or 48) with
    unit column stride and one common row stride (e.g. column slices of a
    fused [N, 4 H D] projection), bias [H, N, N], mask [N].  Returns (or
    writes into ``out``) ``sigmoid(g) * softmax(q k^T / sqrt(D) + bias +
    (1 - mask) * -inf) v`` as a contiguous [N, H * D]."""
    _cuda(q, k, v, bias, mask, g)
    _check(bias.dim() == 3, "expected a [H, N, N] bias")
    heads, n = bias.shape[0], q.shape[0]
    width = q.shape[1] if q.dim() == 2 else -1
    _check(width > 0 and width % heads == 0 and width // heads in (24, 48), "expected H heads of 24 or 48 dims")
    ld = q.stride(0) if n > 1 else width
    for t in (q, k, v, g):
        _check(t.shape == (n, width) and t.dtype == torch.float32 and t.stride(1) == 1
               and (n <= 1 or t.stride(0) == ld), "expected fp32 [N, H * D] q / k / v / g with one row stride")
    _check(bias.shape == (heads, n, n) and bias.dtype == torch.float32 and bias.is_contiguous(),
           "expected a contiguous fp32 [H, N, N] bias")
    _check(mask.shape == (n,) and mask.dtype == torch.float32 and mask.is_contiguous(), "expected an fp32 [N] mask")
    if out is None:
        out = torch.empty((n, width), device=q.device, dtype=torch.float32)
    _check(out.shape == (n, width) and out.dtype == torch.float32 and out.is_contiguous(),
           "out must be a contiguous fp32 [N, H * D]")
    N.call("bmx_seq_attention_fwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), bias.data_ptr(), mask.data_ptr(),
           g.data_ptr(), n, ld, heads, width // heads, float(inf), out.data_ptr(), _stream(q))
    return out


# The token transformer's attention (H * D = 768 >= X3_MIN_K, 1024 keys) runs
# its two products as split-bf16 MFMA (bmx_seq_attention_x3_batched_fwd) like
# its linears, unless exact fp32 is switched on; short key rows (the atom
# windows' 128) and the Pairformer sequence stack (H * D = 384) keep the fp32
# MFMA kernel, where the split pre-pass would cost more than it saves.
X3_ATTN_MIN_KEYS = 256


def seq_attention_split_ok(q, g, nk) -> bool:
    """Whether ``seq_attention_batched`` takes the split-bf16 kernel by default:
    not in exact fp32 mode, width >= ``X3_MIN_K``, >= ``X3_ATTN_MIN_KEYS`` keys,
    and 16-byte g rows."""
    width = q.shape[-1]
    return (not _EXACT_FP32[0] and width >= X3_MIN_K and nk >= X3_ATTN_MIN_KEYS and g.data_ptr() % 16 == 0
            and q.stride(1) % 4 == 0 and q.stride(0) % 4 == 0)


def seq_attention_batched(q, k, v, bias, mask, g, inf, bias_div=1, out=None, split=None, split_out=False):
    """``seq_attention`` for a batch in one launch (``bmx_seq_attention_batched_fwd``):
    q, g [B, NQ, H * D] and k, v [B, NK, H * D] (D = 24, 32 or 48; unit column
    stride; q and g share their strides, k and v theirs), bias
    [B / bias_div, H, NQ, NK] with dense elements (element b uses bias
    b // bias_div), mask [B or 1, NK] with unit stride.  Returns (or writes into
    ``out``) a contiguous fp32 [B, NQ, H * D].  ``split``: True for the
    split-bf16 kernel (``bmx_seq_attention_x3_batched_fwd``, about 2^-16
    relative per product), False for fp32 MFMA, None to choose as above.
    ``split_out``: return the output rows as the split-bf16 operand of the next
    linear instead ([B * NQ, 3 H D + 64] bf16, ``bmx_seq_attention_x3_batched_split_fwd``;
    split-bf16 kernel only)."""
    _cuda(q, k, v, bias, mask, g)
    _check(q.dim() == 3 and k.dim() == 3 and bias.dim() == 4 and mask.dim() == 2, "expected 3-d q/k, 4-d bias, 2-d mask")
    b, nq, width = q.shape
    nk, heads = k.shape[1], bias.shape[1]
    _check(width % heads == 0 and width // heads in (24, 32, 48), "expected H heads of 24, 32 or 48 dims")
    _check(g.shape == q.shape and g.stride() == q.stride() and k.shape == (b, nk, width) and v.shape == k.shape
           and v.stride() == k.stride(), "q / g and k / v must match in shape and strides")
    for t in (q, k, v, g):
        _check(t.dtype == torch.float32 and t.stride(2) == 1, "expected fp32 q / k / v / g with unit column stride")
    _check(bias.dtype == torch.float32 and bias.shape[1:] == (heads, nq, nk) and bias.shape[0] * bias_div == b
           and (bias.shape[0] == 0 or bias[0].is_contiguous()), "expected fp32 [B / bias_div, H, NQ, NK] dense bias")
    _check(mask.dtype == torch.float32 and mask.shape[1] == nk and mask.shape[0] in (1, b) and mask.stride(1) == 1,
           "expected an fp32 [B or 1, NK] mask")
    if split is None:
        split = seq_attention_split_ok(q, g, nk)
    if split_out:
        _check(split and out is None, "split_out needs the split-bf16 kernel and no out")
        out = torch.empty((b * nq, split_width(width)), device=q.device, dtype=torch.bfloat16)
    elif out is None:
        out = torch.empty((b, nq, width), device=q.device, dtype=torch.float32)
    else:
        _check(out.shape == (b, nq, width) and out.dtype == torch.float32 and out.is_contiguous(),
               "out must be a contiguous fp32 [B, NQ, H * D]")
    if b and nq:
        args = (q.data_ptr(), k.data_ptr(), v.data_ptr(), bias.data_ptr(), mask.data_ptr(), g.data_ptr(), b, nq, nk,
                q.stride(1), k.stride(1), q.stride(0), k.stride(0), bias.stride(0),
                mask.stride(0) if mask.shape[0] > 1 else 0, bias_div, heads, width // heads, float(inf),
                out.data_ptr())
        if split:
            nbytes = N.lib().bmx_seq_attention_x3_workspace_bytes(b, nk, heads, width // heads)
            ws = torch.empty(nbytes, device=q.device, dtype=torch.uint8)
            name = "bmx_seq_attention_x3_batched_split_fwd" if split_out else "bmx_seq_attention_x3_batched_fwd"
            N.call(name, *args, ws.data_ptr(), nbytes, _stream(q))
        else:
            N.call("bmx_seq_attention_batched_fwd", *args, _stream(q))
    return out


def seq_attention_windowed(q, k, v, bias, mask, g, inf, *, windows, key_offset, bias_group):
    """The atom transformer's windowed attention (``bmx_seq_attention_windowed_fwd``):
    q, g [E, W, H * D] query windows (E = samples x ``windows`` windows; rows
    at one stride, windows contiguous), k, v [E * W, H * D] (the projected atom
    rows, rows at one stride), mask [E * W] (the atom mask).  Window e reads
    key j from atom row e * W + key_offset + j of its sample; keys past the
    sample's ends are zero keys and values with mask 0 (upstream's zero rows of
    single_to_keys).  bias [B, windows, W, NK, H] (or [B * windows, W, NK, H])
    in any strides (one layer's heads of the atom bias, in place): window e
    uses window e % windows of structure e // bias_group.  Returns a
    contiguous fp32 [E, W, H * D]."""
    _cuda(q, k, v, bias, mask, g)
    if bias.dim() == 4:  # [Eb, W, NK, H]: structures of ``windows`` consecutive elements
        _check(bias.shape[0] % windows == 0, "bias elements must be whole structures")
        bias = bias.unflatten(0, (bias.shape[0] // windows, windows))
    _check(q.dim() == 3 and bias.dim() == 5 and k.dim() == 2 and mask.dim() == 1, "expected 3-d q, 2-d k, 5-d bias")
    e, w, width = q.shape
    nk, heads = bias.shape[3], bias.shape[4]
    _check(width % heads == 0 and width // heads in (24, 32, 48), "expected H heads of 24, 32 or 48 dims")
    _check(g.shape == q.shape and g.stride() == q.stride() and q.stride(2) == 1 and q.stride(0) == w * q.stride(1),
           "q / g must be [E, W, H * D] windows with dense rows, sharing strides")
    _check(k.shape == (e * w, width) and v.shape == k.shape and k.stride() == v.stride() and k.stride(1) == 1,
           "k / v must be [E * W, H * D] with dense rows, sharing strides")
    _check(mask.shape == (e * w,) and mask.is_contiguous() and mask.dtype == torch.float32, "mask must be fp32 [E * W]")
    _check(bias.dtype == torch.float32 and tuple(bias.shape[1:3]) == (windows, w) and bias.shape[0] * bias_group == e
           and e % windows == 0 and bias_group % windows == 0, "bias does not match the windows")
    for t in (q, k, v, g):
        _check(t.dtype == torch.float32, "expected fp32 q / k / v / g")
    out = torch.empty((e, w, width), device=q.device, dtype=torch.float32)
    if e:
        N.call("bmx_seq_attention_windowed_fwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), bias.data_ptr(),
               mask.data_ptr(), g.data_ptr(), e, w, nk, q.stride(1), k.stride(0), windows, key_offset, bias_group,
               bias.stride(0), bias.stride(1), bias.stride(4), bias.stride(2), bias.stride(3), heads, width // heads,
               float(inf), out.data_ptr(), _stream(q))
    return out


def f32_pack(rows, k, *parts):
    """Packed fp32 operand of ``rows`` x ``k`` (``bmx_f32_pack``) from ``parts`` of
    (tile0, tile stride, weight)."""
    _cuda(*(w for _, _, w in parts))
    for tile0, stride, w in parts:
        _check(w.dim() == 2 and w.shape[1] == k and w.shape[0] % 32 == 0
               and (tile0 + (w.shape[0] // 32 - 1) * stride + 1) * 32 <= rows, "a weight does not fit the packed operand")
    out = torch.empty(rows * k, device=parts[0][2].device, dtype=torch.float32)
    for tile0, stride, w in parts:
        w = _aligned(_f32(w))
        N.call("bmx_f32_pack", w.data_ptr(), w.shape[0], w.shape[1], w.stride(0), tile0, stride, out.data_ptr(),
               _stream(w))
    return out


def sequence_stack(s, params, eps_attn, eps_trans, bias, mask, heads, hidden, inf):
    """A PairformerLayer's fp32 sequence stack as one native call
    (``bmx_sequence_stack_fwd``): s [B, N, d], the 9 fp32 parameter tensors
    (None for an absent proj_q bias) in its order, bias [B, H, N, N], mask
    [B, N]; returns the new s."""
    _cuda(s, bias, mask, *(p for p in params if p is not None))
    _check(s.dim() == 3 and s.dtype == torch.float32 and s.is_contiguous(), "expected contiguous fp32 s [B, N, d]")
    b, n, d = s.shape
    _check(len(params) == 9 and all(p is None or (p.dtype == torch.float32 and p.is_contiguous()) for p in params),
           "expected 9 contiguous fp32 parameters")
    _check(bias.shape == (b, heads, n, n) and bias.dtype == torch.float32 and bias.is_contiguous(),
           "expected a contiguous fp32 [B, H, N, N] bias")
    _check(mask.shape == (b, n) and mask.dtype == torch.float32 and mask.stride(1) == 1, "expected an fp32 [B, N] mask")
    s, addresses = _aligned(s), [0 if p is None else p.data_ptr() for p in params]
    if any(address % 16 for address in addresses):
        # views at an odd storage offset (slices of one flat buffer): the call reads 16 bytes at a time
        params = [None if p is None else _aligned(p) for p in params]
        addresses = [0 if p is None else p.data_ptr() for p in params]
    out = torch.empty_like(s)
    ws = _workspace(N.lib().bmx_sequence_stack_workspace_bytes(b * n, d, hidden), s.device)
    N.call("bmx_sequence_stack_fwd", s.data_ptr(), b, n, heads, d // heads, hidden,
           (ctypes.c_void_p * 9)(*addresses), float(eps_attn),
           float(eps_trans), bias.data_ptr(), mask.data_ptr(), mask.stride(0) if b > 1 else 0, float(inf),
           out.data_ptr(), ws.data_ptr(), ws.numel(), _stream(s))
    return out


def token_stack(a, s, params, eps, eps_s, heads, inner, mask, sbias, bias_div, inf):
    """A stack of diffusion transformer layers on at most 1024 rows as one
    native call (``bmx_token_stack_fwd``): a, s [B, N, d] fp32, ``params`` the
    11 device addresses per layer and ``eps`` the 2 a_norm eps per layer in its
    order, mask [1 or B, N] with unit stride, ``sbias`` the pair bias's stride
    per structure of ``bias_div`` samples."""
    _cuda(a, s, mask)
    _check(a.shape == s.shape and a.dim() == 3 and a.dtype == s.dtype == mask.dtype == torch.float32
           and a.is_contiguous() and s.is_contiguous(), "expected contiguous fp32 a and s [B, N, d]")
    b, n, d = a.shape
    layers = len(eps) // 2
    _check(len(params) == 11 * layers and len(eps) == 2 * layers, "expected 11 addresses and 2 eps per layer")
    _check(mask.dim() == 2 and mask.shape[1] == n and mask.shape[0] in (1, b) and mask.stride(1) == 1,
           "expected an fp32 [B or 1, N] mask")
    out = torch.empty_like(a)
    nbytes = N.lib().bmx_token_stack_workspace_bytes(b, n, heads, d // heads, inner)
    ws = _workspace(nbytes, a.device)
    N.call("bmx_token_stack_fwd", a.data_ptr(), s.data_ptr(), b, n, heads, d // heads, inner, layers,
           (ctypes.c_void_p * len(params))(*params), float(eps_s), (ctypes.c_float * len(eps))(*eps), mask.data_ptr(),
           mask.stride(0) if mask.shape[0] > 1 else 0, sbias, bias_div, float(inf), out.data_ptr(), ws.data_ptr(),
           ws.numel(), _stream(a))
    return out


def adaln_modulate(a, scale, shift, eps):
    """``sigmoid(scale) * LN_noaffine(a) + shift`` in one pass; scale and shift
    may be column slices of one wider projection (rows at one stride,
    ``bmx_adaln_strided``)."""
    _cuda(a, scale, shift)
    _check(a.is_contiguous(), "expected contiguous a")
    ld = _same_rows(a, scale, shift)
    d = a.shape[-1]
    out = torch.empty_like(a)
    rows = a.numel() // d if d else 0
    if rows:
        N.call("bmx_adaln_strided", a.data_ptr(), scale.data_ptr(), shift.data_ptr(), ld, out.data_ptr(),
               _code(a.dtype), rows, d, float(eps), _stream(a))
    return out


# ------------------------------------------------------ sequence operators
#
# Differentiable (torch.autograd; one backward pass, no double backward).  A
# call that needs no gradient does not go through autograd.  Forward-mode
# derivatives and tracing are refused: neither sees a native launch, so the
# result would have no tangent, or be an empty tensor in the trace.  To capture
# a backward pass in a graph, make its leaves inside the capture
# (``t.detach().requires_grad_()``) and take the gradients with
# torch.autograd.grad.  A leaf from before it must not belong to an eager graph
# that is still alive: that graph's stream enters the capture and ends the
# process, as with torch's own operators.


def _needs_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _layout(t):
    """What a plan needs to know of a tensor."""
    return None if t is None else (t.shape, t.stride(), t.dtype)


_PROXY = torch._C._TorchDispatchModeKey.PROXY


def _same_device(first, *tensors) -> int:
    """The device index that the tensors share; raises as ``_cuda`` does, and
    where the call would be traced or carries forward-mode tangents."""
    if forward_ad._current_level >= 0:
        _check(all(t is None or forward_ad.unpack_dual(t).tangent is None for t in (first, *tensors)),
               "forward-mode derivatives are not supported")
    _check(torch._C._get_tracing_state() is None
           and (not torch._C._len_torch_dispatch_stack() or torch._C._get_dispatch_mode(_PROXY) is None),
           "tracing is not supported")
    dev = first.get_device()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            _cuda(first, t)
    if dev < 0:
        _cuda(first)
    return dev


def _launch(dev, name, *args):
    """One native call on the current stream of device ``dev``."""
    if dev == torch.cuda.current_device():
        N.call(name, *args, _raw_stream(dev) if _raw_stream is not None else torch.cuda.current_stream(dev).cuda_stream)
    else:
        with torch.cuda.device(dev):
            N.call(name, *args, torch.cuda.current_stream(dev).cuda_stream)


def _rows_ok(shape, stride, unit, most=1 << 62) -> bool:
    """[B, T, H, D] strides that a kernel reads in place: a dense last axis, the others multiples of ``unit``
    elements (a token's below ``most``); axes of one element are never stepped."""
    return stride[3] == 1 and all(n <= 1 or st % unit == 0 for n, st in zip(shape, stride[:3])) and (
        shape[1] <= 1 or stride[1] < most)


def _steps(shape, stride, axes):
    """Strides of the leading axes, 0 for those of one element."""
    return [st if n > 1 else 0 for n, st in zip(shape[:axes], stride)]


class _Plan:
    """What one layout of operands needs of a native call: checked once, kept by sizes, strides and types (never by a
    tensor's identity or address)."""


def _check_positions(pos, tokens, batch, what):
    """The batch stride of positions [tokens] or [batch, tokens]."""
    shape, _, dtype = pos
    _check(dtype in (torch.int32, torch.int64), f"expected int32 or int64 {what}")
    _check(shape in ((tokens,), (batch, tokens)), f"expected {what} of shape [tokens] or [batch, tokens]")
    return tokens if len(shape) == 2 else 0


@lru_cache(maxsize=512)
def _norm_rope_plan(q, k, q_weight, k_weight, q_pos, k_pos, inv_freq):
    _check(len(q[0]) == 4 and (k is None or len(k[0]) == 4), "expected q and k of shape [B, tokens, heads, D]")
    (b, m, h, d), dtype = q[0], q[2]
    code = _code(dtype)
    _check(8 <= d <= 256 and d % 8 == 0, "head dim must be a multiple of 8 in [8, 256]")
    _check(k is None or (k[0][0] == b and k[0][3] == d and k[2] == dtype), "k must match q's batch, head dim and dtype")
    _check(k is not None or k_weight is None, "k_weight needs k")
    for w in (q_weight, k_weight):
        _check(w is None or (w[0] == (d,) and w[2] in (torch.float32, dtype)), "expected weights of [D] in fp32 or q's dtype")
    _check(q_weight is None or k_weight is None or q_weight[2] == k_weight[2], "the weights must share a dtype")
    n, hk = k[0][1:3] if k is not None else (0, 0)
    half, freq64, pos64, sbs = 0, 0, 0, [0, 0]
    if inv_freq is not None:
        (half,), freq64 = inv_freq[0] if len(inv_freq[0]) == 1 else (0,), int(inv_freq[2] == torch.float64)
        _check(inv_freq[2] in (torch.float32, torch.float64) and half > 0 and half % 4 == 0 and 2 * half <= d,
               "expected fp32 or fp64 inv_freq, a multiple of 4 of at most D / 2 values")
        _check(q_pos is not None and (k is None or k_pos is not None), "expected int32 or int64 positions")
        sbs[0] = _check_positions(q_pos, m, b, "q_pos")
        if k is not None:
            sbs[1] = _check_positions(k_pos, n, b, "k_pos")
            _check(q_pos[2] == k_pos[2], "the positions must share a dtype")
        pos64 = int(q_pos[2] == torch.int64)
    plan = _Plan()
    plan.q_ok, plan.k_ok = _rows_ok(q[0], q[1], 4), k is None or _rows_ok(k[0], k[1], 4)
    plan.unit = 4 * (4 if code == N.F32 else 2)  # bytes
    strides = _steps(q[0], q[1], 3) + (_steps(k[0], k[1], 3) if k is not None else [0, 0, 0]) + sbs
    weight = q_weight or k_weight
    plan.code, plan.w_code = code, _code(weight[2]) if weight else code
    plan.shape, plan.strides = N.int64_array([b, m, n, h, hk, d]), N.int64_array(strides)
    plan.tail = (pos64, freq64, half)
    plan.ws = N.lib().bmx_qk_norm_rope_workspace_bytes(d)
    return plan


def _norm_rope_args(plan, q, k, q_weight, k_weight, q_pos, k_pos, inv_freq, eps, interleaved):
    pos64, freq64, half = plan.tail
    return (q.data_ptr(), _ptr(k), plan.code, plan.shape, plan.strides, _ptr(q_weight), _ptr(k_weight), plan.w_code, _ptr(q_pos),
            _ptr(k_pos), pos64, _ptr(inv_freq), freq64, half, interleaved, eps)


def _norm_rope_fwd(plan, dev, q, k, *rest):
    q_out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    k_out = torch.empty(k.shape, device=k.device, dtype=k.dtype) if k is not None else None
    _launch(dev, "bmx_qk_norm_rope_fwd", *_norm_rope_args(plan, q, k, *rest), q_out.data_ptr(), _ptr(k_out))
    return q_out, k_out


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, plan, dev, q, k, q_weight, k_weight, q_pos, k_pos, inv_freq, eps, interleaved):
        ctx.save_for_backward(q, k, q_weight, k_weight, q_pos, k_pos, inv_freq)
        ctx.rest = plan, dev, eps, interleaved
        ctx.set_materialize_grads(False)
        return _norm_rope_fwd(plan, dev, q, k, q_weight, k_weight, q_pos, k_pos, inv_freq, eps, interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        plan, dev, eps, interleaved = ctx.rest
        q, k, q_weight, k_weight, q_pos, k_pos, inv_freq = ctx.saved_tensors
        need, ws = ctx.needs_input_grad, None
        dq = dk = dqw = dkw = None  # a tensor whose result got no gradient takes no part
        if dq_out is not None:
            dq_out = _aligned(dq_out.contiguous())
            dq = torch.empty(q.shape, device=q.device, dtype=q.dtype) if need[2] else None
            dqw = torch.empty_like(q_weight) if need[4] else None
        if dk_out is not None:
            dk_out = _aligned(dk_out.contiguous())
            dk = torch.empty(k.shape, device=k.device, dtype=k.dtype) if need[3] else None
            dkw = torch.empty_like(k_weight) if need[5] else None
        if dqw is not None or dkw is not None:
            ws = _workspace(plan.ws, q.device)
        if ws is not None or dq is not None or dk is not None:
            _launch(dev, "bmx_qk_norm_rope_bwd",
                    *_norm_rope_args(plan, q, k, q_weight, k_weight, q_pos, k_pos, inv_freq, eps, interleaved),
                    _ptr(dq_out), _ptr(dk_out), _ptr(dq), _ptr(dk), _ptr(dqw), _ptr(dkw), _ptr(ws),
                    plan.ws if ws is not None else 0)
        return None, None, dq, dk, dqw, dkw, None, None, None, None, None


def qk_norm_rope(q, k, q_weight, k_weight, q_pos, k_pos, inv_freq, eps=1e-6, interleaved=False):
    """RMS norm of every query and key head and the rotation by position, one
    pass (``bmx_qk_norm_rope_fwd``): ``R(pos) (x / sqrt(mean(x^2) + eps) * weight)``.

    q [B, M, H, D] and k [B, N, Hk, D] (or None: queries alone) are fp32 or bf16
    with D a multiple of 8 in [8, 256], in any strides (column slices of one
    projection are read in place; layouts that the kernel cannot read are
    copied).  Weights are [D] fp32 or in q's type, or None.  q_pos [M] or
    [B, M] and k_pos [N] or [B, N] are int32 / int64.  inv_freq (fp32 / fp64,
    a multiple of 4 of at most D / 2 values) turns channels (i, R + i) by
    ``pos * inv_freq[i]``, R = len(inv_freq) (``interleaved``: channels
    (2 i, 2 i + 1)); channels past 2 R are only normalised.  With inv_freq None
    nothing turns and the positions may be None.  Returns dense (q', k');
    gradients reach q, k and the weights."""
    if inv_freq is None:
        q_pos = k_pos = None
    else:
        _check(isinstance(q_pos, torch.Tensor) and (k is None or isinstance(k_pos, torch.Tensor)),
               "expected int32 or int64 positions")
        _check(not inv_freq.requires_grad, "inv_freq takes no gradient")
        k_pos = None if k is None else k_pos
        q_pos, k_pos = q_pos.contiguous(), None if k_pos is None else k_pos.contiguous()
        inv_freq = inv_freq.contiguous()
    dev = _same_device(q, k, q_weight, k_weight, q_pos, k_pos, inv_freq)
    _check(eps >= 2.0 ** -126, "eps must be positive, at least 2^-126")
    plan = _norm_rope_plan(_layout(q), _layout(k), _layout(q_weight), _layout(k_weight), _layout(q_pos), _layout(k_pos),
                           _layout(inv_freq))
    if not plan.q_ok or q.data_ptr() % plan.unit or not plan.k_ok or (k is not None and k.data_ptr() % plan.unit):
        q, k = _aligned(q.contiguous()), None if k is None else _aligned(k.contiguous())
        plan = _norm_rope_plan(_layout(q), _layout(k), _layout(q_weight), _layout(k_weight), _layout(q_pos),
                               _layout(k_pos), _layout(inv_freq))
    if q_weight is not None:
        q_weight = _aligned(q_weight.contiguous())
    if k_weight is not None:
        k_weight = _aligned(k_weight.contiguous())
    args = (plan, dev, q, k, q_weight, k_weight, q_pos, k_pos, inv_freq, float(eps), int(interleaved))
    return _QkNormRope.apply(*args) if _needs_grad(q, k, q_weight, k_weight) else _norm_rope_fwd(*args)


@lru_cache(maxsize=64)
def _relative_thresholds(side, exact, max_distance):
    """Least distances of buckets 1 .. side - 1 of one direction (whole numbers,
    no logarithm): i for i <= exact, then the least n with
    ``(n / exact)^steps >= (max_distance / exact)^k``, steps = side - exact."""
    steps, edges = side - exact, list(range(1, exact + 1))
    for k in range(1, steps):
        reach = exact ** (steps - k) * max_distance ** k
        lo, hi = edges[-1], max_distance  # max_distance itself satisfies every k < steps
        while lo < hi:
            mid = (lo + hi) // 2
            lo, hi = (lo, mid) if mid ** steps >= reach else (mid + 1, hi)
        edges.append(lo)
    return (ctypes.c_int32 * len(edges))(*edges)


@lru_cache(maxsize=512)
def _relative_plan(table, q_pos, k_pos, exact, max_distance, bidirectional):
    _check(len(table[0]) == 2 and table[0][0] > 0 and table[0][1] > 0, "expected a [buckets, heads] table")
    (buckets, heads), code = table[0], _code(table[2])
    _check(buckets <= MAX_BUCKETS and heads <= 65535, "at most 256 buckets and 65535 heads")
    _check(not bidirectional or buckets % 2 == 0, "bidirectional buckets must be even in number")
    side = buckets // 2 if bidirectional else buckets
    _check(side >= 2, "expected at least two buckets a direction")
    exact = side // 2 if exact is None else exact
    _check(1 <= exact < side, "exact must be in [1, buckets of a direction)")
    if exact == side - 1:
        max_distance = side - 1  # nothing is shared by logarithm
    _check(exact == side - 1 or exact < max_distance <= 1 << 30, "max_distance must be above exact, at most 2^30")
    _check(len(q_pos[0]) in (1, 2) and len(k_pos[0]) in (1, 2), "expected positions [tokens] or [batch, tokens]")
    batch = next((p[0][0] for p in (q_pos, k_pos) if len(p[0]) == 2), None)
    m, n = q_pos[0][-1], k_pos[0][-1]
    steps = _check_positions(q_pos, m, batch, "q_pos"), _check_positions(k_pos, n, batch, "k_pos")
    _check(q_pos[2] == k_pos[2], "the positions must share a dtype")
    plan = _Plan()
    thresholds = _relative_thresholds(side, exact, max_distance)
    plan.head = code, buckets, heads
    plan.tail = (int(q_pos[2] == torch.int64), 1 if batch is None else batch, m, n, *steps, thresholds, len(thresholds),
                 int(bidirectional))
    plan.shape = (heads, m, n) if batch is None else (batch, heads, m, n)
    plan.ws = N.lib().bmx_relative_bias_workspace_bytes(code, buckets, heads, plan.tail[1], m, n)
    return plan


def _relative_bias_fwd(plan, dev, table, q_pos, k_pos):
    out = torch.empty(plan.shape, device=table.device, dtype=table.dtype)
    if out.numel():
        _launch(dev, "bmx_relative_bias_fwd", table.data_ptr(), *plan.head, q_pos.data_ptr(), k_pos.data_ptr(), *plan.tail,
                out.data_ptr())
    return out


class _RelativeBias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, plan, dev, table, q_pos, k_pos):
        ctx.save_for_backward(q_pos, k_pos)
        ctx.rest = plan, dev
        return _relative_bias_fwd(plan, dev, table, q_pos, k_pos)

    @staticmethod
    @once_differentiable
    def backward(ctx, dbias):
        q_pos, k_pos = ctx.saved_tensors
        plan, dev = ctx.rest
        dbias = dbias.contiguous()
        dtable = torch.empty(plan.head[1:], device=dbias.device, dtype=dbias.dtype)
        ws = _workspace(plan.ws, dbias.device)
        _launch(dev, "bmx_relative_bias_bwd", dbias.data_ptr(), *plan.head, q_pos.data_ptr(), k_pos.data_ptr(), *plan.tail,
                dtable.data_ptr(), ws.data_ptr(), plan.ws)
        return None, None, dtable, None, None


MAX_BUCKETS = 256


def relative_bias(table, q_pos, k_pos, exact=None, max_distance=128, bidirectional=True):
    """Learned relative-position bias (``bmx_relative_bias_fwd``):
    ``bias[h, i, j] = table[bucket(k_pos[j] - q_pos[i]), h]``, [H, M, N] (or
    [B, H, M, N] where a position tensor has a batch axis), dense, in the type
    of ``table`` [buckets, H] (fp32 or bf16): the additive bias of
    ``cross_attention`` or ``seq_attention``.

    Bidirectional, half of the buckets (``side``) hold d <= 0 and half d > 0,
    by n = |d|; otherwise all hold n = max(-d, 0).  Distances below ``exact``
    (default side // 2) have a bucket each; the others share the rest by
    logarithm, ``exact + floor(log(n / exact) / log(max_distance / exact) *
    (side - exact))``, at most the last one: it begins below ``max_distance``
    and holds everything from there on.  ``exact = side - 1``
    is the clipped form (every distance its own bucket up to side - 1).
    Positions are int32 / int64, |pos| < 2^62, in any order.  The gradient
    reaches the table (fp32 sums, the same bits on every run)."""
    q_pos, k_pos, table = q_pos.contiguous(), k_pos.contiguous(), table.contiguous()
    dev = _same_device(table, q_pos, k_pos)
    plan = _relative_plan(_layout(table), _layout(q_pos), _layout(k_pos), None if exact is None else int(exact),
                          int(max_distance), bool(bidirectional))
    args = plan, dev, table, q_pos, k_pos
    return _RelativeBias.apply(*args) if _needs_grad(table) else _relative_bias_fwd(*args)


MAX_TOKEN_STRIDE = 1 << 22  # elements, of cross_attention's operands
MAX_BIAS_STRIDE = 1 << 26


@lru_cache(maxsize=512)
def _cross_plan(q, k, v, mask, bias):
    _check(len(q[0]) == 4 and len(k[0]) == 4 and len(v[0]) == 4, "expected q, k and v of shape [B, tokens, heads, D]")
    (b, m, h, d), (n, hk), dtype = q[0], k[0][1:3], q[2]
    code = _code(dtype)
    _check(k[0] == v[0] and k[0][0] == b and k[0][3] == d and k[2] == v[2] == dtype,
           "k and v must match q's batch, head dim and dtype")
    _check(8 <= d <= 128 and d % 8 == 0, "head dim must be a multiple of 8 in [8, 128]")
    _check(h > 0 and hk > 0 and h % hk == 0, "the query heads must be a multiple of the key heads")
    _check(h * d < MAX_TOKEN_STRIDE, "expected fewer than 2^22 channels")
    plan, unit = _Plan(), 16 // (4 if code == N.F32 else 2)
    plan.ok = tuple(_rows_ok(*t[:2], unit, MAX_TOKEN_STRIDE) for t in (q, k, v))
    strides = [st for t in (q, k, v) for st in _steps(t[0], t[1], 3)] + [0, 0, 0, 0]
    plan.mask_ok = plan.bias_ok = True
    if mask is not None:
        shape, stride, kind = mask
        _check(kind == torch.bool and shape in ((b, n), (1, n), (n,)), "expected a bool mask [B, N]")
        plan.mask_ok = stride[-1] == 1 or n <= 1
        strides[9] = stride[0] if len(shape) == 2 and shape[0] > 1 else 0
    if bias is not None:
        shape, stride, kind = bias
        _check(len(shape) == 4 and kind == dtype and shape[0] in (1, b) and shape[1] in (1, h) and shape[2:] == (m, n),
               "expected a bias [B or 1, H or 1, M, N] in q's dtype")
        _check(n < MAX_BIAS_STRIDE, "a bias takes at most 2^26 - 1 keys")
        plan.bias_ok = (stride[3] == 1 or n <= 1) and (m <= 1 or stride[2] < MAX_BIAS_STRIDE)
        strides[10:] = _steps(shape, stride, 3)
        dense = [shape[1] * m * n if shape[0] > 1 else 0, m * n if shape[1] > 1 else 0, n]
        plan.dbias_strides = N.int64_array(dense)
    plan.code, plan.scale = code, d ** -0.5
    plan.shape, plan.strides = N.int64_array([b, m, n, h, hk, d]), N.int64_array(strides)
    plan.out, plan.stats, plan.empty = (b, m, h, d), (b, h, m, 2), not (b and m and n)
    plan.ws = N.lib().bmx_cross_attention_workspace_bytes(code, b, m, n, h, hk, d)
    plan.ws_bwd = N.lib().bmx_cross_attention_bwd_workspace_bytes(b, m, n, h, hk, d)
    return plan


def _cross_attention_fwd(plan, dev, q, k, v, mask, bias, scale, for_backward=False):
    """(out, what rounding out left or None, row statistics or None)."""
    out = torch.empty(plan.out, device=q.device, dtype=q.dtype)
    lo = torch.empty_like(out) if for_backward and plan.code == N.BF16 else None
    stats = torch.empty(plan.stats, device=q.device, dtype=torch.float32) if for_backward else None
    ws = _workspace(plan.ws, q.device) if plan.ws else None
    _launch(dev, "bmx_cross_attention_fwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(mask), _ptr(bias), plan.code,
            plan.shape, plan.strides, scale, out.data_ptr(), _ptr(lo), _ptr(stats), _ptr(ws), plan.ws)
    return out, lo, stats


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, plan, dev, q, k, v, mask, bias, scale):
        out, lo, stats = _cross_attention_fwd(plan, dev, q, k, v, mask, bias, scale, for_backward=True)
        ctx.save_for_backward(q, k, v, mask, bias, out, lo, stats)
        ctx.rest = plan, dev, scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, mask, bias, out, lo, stats = ctx.saved_tensors
        plan, dev, scale = ctx.rest
        make = torch.zeros if plan.empty else torch.empty  # without queries or keys nothing depends on anything
        dq, dk, dv, dbias = (make(t.shape, device=q.device, dtype=q.dtype) if need else None
                             for need, t in zip((*ctx.needs_input_grad[2:5], ctx.needs_input_grad[6]), (q, k, v, bias)))
        if not plan.empty:
            dout = _aligned(dout.contiguous())
            ws = _workspace(plan.ws_bwd, q.device)
            _launch(dev, "bmx_cross_attention_bwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(mask), _ptr(bias),
                    plan.code, plan.shape, plan.strides, scale, out.data_ptr(), _ptr(lo), stats.data_ptr(), dout.data_ptr(),
                    _ptr(dq), _ptr(dk), _ptr(dv), _ptr(dbias), None if dbias is None else plan.dbias_strides,
                    ws.data_ptr(), plan.ws_bwd)
        return None, None, dq, dk, dv, None, dbias, None


def cross_attention(q, k, v, mask=None, bias=None, scale=None):
    """Softmax attention of q [B, M, H, D] over another sequence's k and v
    [B, N, Hk, D] (``bmx_cross_attention_fwd``):
    ``softmax(scale q k^T + bias) v``, dense [B, M, H, D].

    fp32 or bf16, D a multiple of 8 up to 128, H a multiple of Hk (query head h
    reads key head ``h // (H / Hk)``), any M and N down to 0 and 1; layouts that
    the kernel cannot read in place (a strided last axis, rows off 16 bytes) are
    copied.  mask: bool [B, N] (or [1, N], [N]), True for the keys that take
    part; the others' values are never looked at, NaN or not.  bias: q's type,
    [B or 1, H or 1, M, N], added to the logits; -inf leaves a pair out.  A
    query without keys gives zeros, and zero gradients.  scale: positive
    (2^-126 to 2^127), 1 / sqrt(D) by default.  Sums are fp32; bf16 weights
    enter the products with 16 bits in decoding steps (M H / Hk <= 32), over up
    to 256 keys and where a batch element is small (H M N D <= 2^28), else with
    8, whose error is about 1.4 times that of rounding the result.  Gradients
    reach q, k, v and bias (summed over its shared axes in fp32) and are the
    same bits on every run."""
    dev = _same_device(q, k, v, mask, bias)
    plan = _cross_plan(_layout(q), _layout(k), _layout(v), _layout(mask), _layout(bias))
    scale = plan.scale if scale is None else float(scale)
    _check(2.0 ** -126 <= scale <= 2.0 ** 127, "scale must be positive and finite, in [2^-126, 2^127]")
    if not (all(plan.ok) and plan.mask_ok and plan.bias_ok) or (q.data_ptr() | k.data_ptr() | v.data_ptr()) % 16:
        q, k, v = (t if ok and t.data_ptr() % 16 == 0 else _aligned(t.contiguous()) for t, ok in zip((q, k, v), plan.ok))
        mask = mask if plan.mask_ok else mask.contiguous()
        bias = bias if plan.bias_ok else bias.contiguous()
        plan = _cross_plan(_layout(q), _layout(k), _layout(v), _layout(mask), _layout(bias))
    if _needs_grad(q, k, v, bias):
        return _CrossAttention.apply(plan, dev, q, k, v, mask, bias, scale)
    return _cross_attention_fwd(plan, dev, q, k, v, mask, bias, scale)[0]


def _rows_in_place(layout, unit) -> bool:
    """[..., C] that a kernel reads in place: a dense last axis, the others at multiples of ``unit`` elements."""
    return layout is None or (layout[1][-1] == 1
                              and all(n <= 1 or st % unit == 0 for n, st in zip(layout[0][:-1], layout[1][:-1])))


def _is_dense(layout) -> bool:
    if layout is None or 0 in layout[0]:
        return True
    step = 1
    for n, st in zip(reversed(layout[0]), reversed(layout[1])):
        if n != 1 and st != step:
            return False
        step *= n
    return True


def _bits(*tensors) -> int:
    """The addresses' bits, for a look at what all are aligned to."""
    bits = 0
    for t in tensors:
        if t is not None:
            bits |= t.data_ptr()
    return bits


def _readable(t, ok, unit=16):
    """``t``, copied where its layout (``ok``) or its address cannot be read in place."""
    return t if t is None or (ok and t.data_ptr() % unit == 0) else _aligned(t.contiguous())


def _dense(t):
    return None if t is None else _aligned(t.contiguous())


def _span(layout, size):
    """Bytes from a tensor's first element to behind its last."""
    shape, stride, _ = layout
    return 0 if 0 in shape else size * (1 + sum((n - 1) * st for n, st in zip(shape, stride)))


def _like(t):
    """A dense tensor of ``t``'s shape, to be written."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, device=t.device, dtype=t.dtype)


def _grads(needed, tensors, empty):
    """Room for the gradients that are needed; zeros where nothing is there to be computed."""
    if empty:
        return [torch.zeros(t.shape, device=t.device, dtype=t.dtype) if need else None for need, t in zip(needed, tensors)]
    return [_like(t) if need else None for need, t in zip(needed, tensors)]


@lru_cache(maxsize=512)
def _frame_plan(x, y, gate, y_weight, scale, weight, post_norm, pre_norm):
    _check(len(x[0]) == 3 and x[0] == y[0], "expected x and y of one shape [B, tokens, D]")
    (b, t, d), x_code, code = x[0], _code(x[2]), _code(y[2])
    _check(x_code == N.F32 or code == N.BF16, "fp32 y needs fp32 x")
    _check(8 <= d <= 8192 and d % 8 == 0, "D must be a multiple of 8 in [8, 8192]")
    _check(gate is None or (gate[0] in ((b, t, d), (b, 1, d)) and gate[2] == y[2]),
           "expected a gate [B, tokens, D] or [B, 1, D] in y's dtype")
    weights = [w for w in (y_weight, scale, weight) if w is not None]
    for w in weights:
        _check(w[0] == (d,) and w[2] in (torch.float32, y[2]), "expected weights of [D] in fp32 or y's dtype")
        _check(w[2] == weights[0][2], "the weights must share a dtype")
    _check(post_norm or y_weight is None, "y_weight needs post_norm")
    _check(pre_norm or weight is None, "weight needs pre_norm")
    plan = _Plan()
    plan.kind = 0 if gate is None else 2 if gate[0][1] != t else 1
    plan.codes, plan.w_code = (x_code, code), _code(weights[0][2]) if weights else N.F32
    strides = _steps(x[0], x[1], 2) + _steps(y[0], y[1], 2) + ([0, 0] if gate is None else _steps(gate[0], gate[1], 2))
    plan.shape, plan.strides, plan.rows = N.int64_array([b, t, d]), N.int64_array(strides), b * t
    plan.norms = int(post_norm), int(pre_norm)
    plan.ok = tuple(_rows_in_place(m, 8) for m in (x, y, gate)) + tuple(map(_is_dense, (y_weight, scale, weight)))
    plan.in_place = all(plan.ok)
    plan.ws = N.lib().bmx_residual_norm_workspace_bytes(b, t, d, plan.kind)
    return plan


def _frame_args(plan, x, y, gate, y_weight, scale, weight, eps):
    return (x.data_ptr(), y.data_ptr(), _ptr(gate), *plan.codes, plan.shape, plan.strides, plan.kind, _ptr(y_weight),
            _ptr(scale), _ptr(weight), plan.w_code, *plan.norms, eps)


def _residual_norm_fwd(plan, dev, x, y, *rest):
    r, h = _like(x), _like(y) if plan.norms[1] else None
    if plan.rows:
        _launch(dev, "bmx_residual_norm_fwd", *_frame_args(plan, x, y, *rest), r.data_ptr(), _ptr(h))
    return r, h


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, plan, dev, x, y, gate, y_weight, scale, weight, eps):
        ctx.save_for_backward(x, y, gate, y_weight, scale, weight)
        ctx.rest = plan, dev, eps
        ctx.set_materialize_grads(False)
        return _residual_norm_fwd(plan, dev, x, y, gate, y_weight, scale, weight, eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, dr, dh):
        plan, dev, eps = ctx.rest
        tensors = ctx.saved_tensors
        grads = _grads(ctx.needs_input_grad[2:8], tensors, not plan.rows)
        if plan.rows and any(g is not None for g in grads):
            dr, dh = _dense(dr), _dense(dh)
            ws = _workspace(plan.ws, tensors[0].device)
            _launch(dev, "bmx_residual_norm_bwd", *_frame_args(plan, *tensors, eps), _ptr(dr), _ptr(dh),
                    *map(_ptr, grads), ws.data_ptr(), plan.ws)
        return None, None, *grads, None


def residual_norm(x, y, gate=None, y_weight=None, scale=None, weight=None, eps=1e-6, post_norm=True, pre_norm=True):
    """The frame between two blocks of a sequence stack, one pass (``bmx_residual_norm_fwd``): the RMS norm of a
    block's result, its gate and residual scale, the residual add, and the next block's RMS norm:

        ``m = y / sqrt(mean(y^2) + eps) * y_weight``  (``post_norm`` False: ``m = y``)
        ``r = x + scale * sigmoid(gate) * m``
        ``h = r / sqrt(mean(r^2) + eps) * weight``

    x (the residual stream) and y (the block's result) are [B, T, D], fp32 or bf16, D a multiple of 8 up to 8192, any
    T; an fp32 stream takes blocks of either type.  gate: logits in y's type, [B, T, D] or one per batch element
    [B, 1, D], or None (no gate).  Weights and scale are [D] in fp32 or y's type, or None (1).  Any strides: layouts that
    the kernel cannot read (a strided last axis, rows off 16 bytes) are copied.  Returns dense (r in x's type, h in y's
    type, from r before its rounding), or r alone with ``pre_norm`` False.  Gradients reach every tensor (a shared gate's
    summed over its tokens); sums are fp32 and the same bits on every run."""
    dev = _same_device(x, y, gate, y_weight, scale, weight)
    _check(eps >= 2.0 ** -126, "eps must be positive, at least 2^-126")
    norms = bool(post_norm), bool(pre_norm)
    plan = _frame_plan(_layout(x), _layout(y), _layout(gate), _layout(y_weight), _layout(scale), _layout(weight), *norms)
    if not plan.in_place or _bits(x, y, gate, y_weight, scale, weight) % 16:
        x, y, gate, y_weight, scale, weight = map(_readable, (x, y, gate, y_weight, scale, weight), plan.ok)
        plan = _frame_plan(_layout(x), _layout(y), _layout(gate), _layout(y_weight), _layout(scale), _layout(weight), *norms)
    args = plan, dev, x, y, gate, y_weight, scale, weight, float(eps)
    r, h = (_ResidualNorm.apply if _needs_grad(x, y, gate, y_weight, scale, weight) else _residual_norm_fwd)(*args)
    return (r, h) if pre_norm else r


def _check_lengths(lengths, batch):
    _check(lengths is None or (lengths[0] == (batch,) and lengths[2] in (torch.int32, torch.int64)),
           "expected int32 or int64 lengths [B]")
    return int(lengths is not None and lengths[2] == torch.int64)


def _check_state_out(state_out, plan, dtype, state, inputs, grad):
    """A buffer for the last state: dense, of the state's kind, apart from everything but the state that it may replace."""
    _check(not grad, "state_out takes no gradient: use return_state")
    lo = state_out.data_ptr()
    _check(state_out.shape == plan.state and state_out.dtype == dtype and state_out.is_contiguous() and lo % 16 == 0,
           "state_out must be a dense 16-byte aligned tensor of the state's shape and dtype")
    hi = lo + plan.state_bytes
    for t, span in zip(inputs, plan.spans):
        if t is not None and span:
            at = t.data_ptr()
            _check(at >= hi or lo >= at + span, "state_out shares memory with an input")
    if state is not None:
        at = state.data_ptr()
        _check(at == lo or at >= hi or lo >= at + plan.state_bytes, "state_out shares memory with an input")


def _empty_state(shape, dtype, device, state, state_out):
    """The last state of a call without tokens: the first one."""
    out = torch.empty(shape, device=device, dtype=dtype) if state_out is None else state_out
    return out.zero_() if state is None else out if out is state else out.copy_(state)


def _written(t):
    """Tells autograd that a native call wrote into ``t``."""
    if t is not None and not t.is_inference():
        torch.autograd.graph.increment_version(t)


@lru_cache(maxsize=512)
def _conv_plan(x, weight, bias, state, lengths, silu):
    _check(len(x[0]) == 3 and len(weight[0]) == 2, "expected x of shape [B, tokens, channels] and a [channels, width] weight")
    (b, t, c), width, code = x[0], weight[0][1], _code(x[2])
    _check(c % 8 == 0 and 8 <= c < 1 << 20, "channels must be a multiple of 8 below 2^20")
    _check(weight[0][0] == c and 2 <= width <= 4, "expected a [channels, width] weight of width 2, 3 or 4")
    for w in (weight, bias):
        _check(w is None or w[2] in (torch.float32, x[2]), "expected weight and bias in fp32 or x's dtype")
    _check(bias is None or bias[0] == (c,), "expected a bias of [channels]")
    _check(state is None or (state[0] == (b, width - 1, c) and state[2] == x[2]),
           "expected a state [B, width - 1, channels] in x's dtype")
    plan = _Plan()
    lengths64 = _check_lengths(lengths, b)
    plan.head = code, N.int64_array([b, t, c, width]), N.int64_array(_steps(x[0], x[1], 2))
    plan.codes, plan.tail = (_code(weight[2]), _code(bias[2]) if bias else code), (lengths64, silu)
    plan.ok = (_rows_in_place(x, 16 // x[2].itemsize), *map(_is_dense, (weight, bias, state)))
    plan.in_place = all(plan.ok) and _is_dense(lengths)
    plan.state, plan.empty = (b, width - 1, c), not (b and t)
    plan.state_bytes = b * (width - 1) * c * x[2].itemsize
    plan.spans = [0 if w is None else _span(w, w[2].itemsize) for w in (x, weight, bias, lengths)]
    plan.ws = N.lib().bmx_causal_conv_workspace_bytes(b, t, c, width)
    return plan


def _conv_args(plan, x, weight, bias, state, lengths):
    return (x.data_ptr(), *plan.head, weight.data_ptr(), plan.codes[0], _ptr(bias), plan.codes[1], _ptr(state), _ptr(lengths),
            *plan.tail)


def _causal_conv_fwd(plan, dev, x, weight, bias, state, lengths, want_state, state_out):
    y = _like(x)
    if plan.empty:
        return y, _empty_state(plan.state, x.dtype, x.device, state, state_out) if want_state else None
    if want_state and state_out is None:
        state_out = torch.empty(plan.state, device=x.device, dtype=x.dtype)
    _launch(dev, "bmx_causal_conv_fwd", *_conv_args(plan, x, weight, bias, state, lengths), y.data_ptr(), _ptr(state_out))
    return y, state_out


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, plan, dev, x, weight, bias, state, lengths, want_state, state_out):
        ctx.save_for_backward(x, weight, bias, state, lengths)
        ctx.rest = plan, dev
        ctx.set_materialize_grads(False)
        return _causal_conv_fwd(plan, dev, x, weight, bias, state, lengths, want_state, state_out)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dnext):
        plan, dev = ctx.rest
        x, weight, bias, state, lengths = ctx.saved_tensors
        dx, dw, db, dstate = _grads(ctx.needs_input_grad[2:6], (x, weight, bias, state), plan.empty)
        if plan.empty:
            dstate = dnext if dstate is not None and dnext is not None else dstate
        elif any(g is not None for g in (dx, dw, db, dstate)):
            dy, dnext = _dense(dy), _dense(dnext)
            ws = _workspace(plan.ws, x.device) if dw is not None or db is not None else None
            _launch(dev, "bmx_causal_conv_bwd", *_conv_args(plan, x, weight, bias, state, lengths), _ptr(dy), _ptr(dnext),
                    _ptr(dx), _ptr(dw), _ptr(db), _ptr(dstate), _ptr(ws), plan.ws if ws is not None else 0)
        return None, None, dx, dw, db, dstate, None, None, None


def causal_conv(x, weight, bias=None, state=None, lengths=None, silu=True, return_state=False, state_out=None):
    """Short causal convolution of every channel on its own (``bmx_causal_conv_fwd``), with SiLU (``silu`` False:
    without): ``y[b, t, c] = silu(bias[c] + sum_j weight[c, j] x[b, t - (W - 1) + j, c])``, dense, in x's type.

    x [B, T, C] is fp32 or bf16, C a multiple of 8, in any strides (layouts that the kernel cannot read are copied).
    weight [C, W], W 2 to 4, and bias [C] are fp32 or in x's type.  state: the W - 1 inputs before the first, oldest first,
    [B, W - 1, C] in x's type (None: zeros).  lengths: int32 or int64 [B] on the device, the tokens of each sequence (taken
    into [0, T]); later rows are never read and give zeros.

    ``return_state``: (y, the W - 1 inputs before each sequence's end): the next call's state.  ``state_out``: a
    dense buffer that takes it instead of a new tensor, ``state`` itself included (a decoder's step in place); without
    gradients only.  Gradients reach x, weight, bias and state, from y and the returned state; sums are fp32 and the same
    bits on every run."""
    want, grad = return_state or state_out is not None, _needs_grad(x, weight, bias, state)
    dev = _same_device(x, weight, bias, state, lengths, state_out)
    silu = int(bool(silu))
    plan = _conv_plan(_layout(x), _layout(weight), _layout(bias), _layout(state), _layout(lengths), silu)
    if not plan.in_place or _bits(x, weight, bias, state) % 16:
        x, weight, bias, state = map(_readable, (x, weight, bias, state), plan.ok)
        lengths = None if lengths is None else lengths.contiguous()
        plan = _conv_plan(_layout(x), _layout(weight), _layout(bias), _layout(state), _layout(lengths), silu)
    if state_out is not None:
        _check_state_out(state_out, plan, x.dtype, state, (x, weight, bias, lengths), grad or _needs_grad(state_out))
    args = plan, dev, x, weight, bias, state, lengths, want, state_out
    y, last = (_CausalConv.apply if grad else _causal_conv_fwd)(*args)
    _written(state_out)
    return (y, last) if return_state else y


MAX_SCAN_STRIDE = 1 << 25  # elements, of a token of selective_scan's operands


@lru_cache(maxsize=512)
def _scan_plan(u, dt, A, B, C, D, z, dt_bias, state, lengths, softplus):
    _check(len(u[0]) == 3 and len(A[0]) == 2 and len(B[0]) == 4, "expected u [B, tokens, channels], A [channels, states] "
           "and B, C [B, tokens, groups, states]")
    (b, t, c), states, groups, code = u[0], A[0][1], B[0][2], _code(u[2])
    _check(dt[0] == u[0] and dt[2] == u[2] and (z is None or (z[0] == u[0] and z[2] == u[2])),
           "dt and z must match u's shape and dtype")
    _check(states in (8, 16, 32, 64), "states must be 8, 16, 32 or 64")
    _check(B[0] == C[0] == (b, t, groups, states) and B[2] == C[2] == u[2],
           "expected B and C [B, tokens, groups, states] in u's dtype")
    _check(groups >= 1 and 8 <= c < 1 << 20 and c % (8 * groups) == 0, "channels must be a multiple of 8 per group, below 2^20")
    _check(A[0][0] == c and A[2] == torch.float32, "expected A [channels, states] in fp32")
    for w in (D, dt_bias):
        _check(w is None or (w[0] == (c,) and w[2] == torch.float32), "expected D and dt_bias [channels] in fp32")
    _check(state is None or (state[0] == (b, c, states) and state[2] == torch.float32),
           "expected a state [B, channels, states] in fp32")
    plan = _Plan()
    plan.ok = tuple(_rows_in_place(m, 4) and (t <= 1 or m is None or m[1][1] < MAX_SCAN_STRIDE) for m in (u, dt, B, C, z))
    plan.dense = tuple(map(_is_dense, (A, D, dt_bias, state)))
    plan.in_place = all(plan.ok) and all(plan.dense) and _is_dense(lengths)
    none = [0, 0]
    strides = [st for m in (u, dt) for st in _steps(m[0], m[1], 2)] + (_steps(z[0], z[1], 2) if z else none)
    strides += _steps(B[0], B[1], 3) + _steps(C[0], C[1], 3)
    plan.codes = code, _check_lengths(lengths, b)
    plan.shape, plan.strides = N.int64_array([b, t, c, states, groups]), N.int64_array(strides)
    plan.softplus, plan.state, plan.empty = softplus, (b, c, states), not (b and t)
    plan.state_bytes = b * c * states * 4
    plan.spans = [0 if w is None else _span(w, w[2].itemsize) for w in (u, dt, A, B, C, D, z, dt_bias, lengths)]
    plan.unit = 4 * u[2].itemsize  # bytes that activations are aligned to
    plan.ws = N.lib().bmx_selective_scan_workspace_bytes(b, t, c, states, groups)
    plan.ws_bwd = N.lib().bmx_selective_scan_bwd_workspace_bytes(b, t, c, states, groups)
    plan.saved = N.lib().bmx_selective_scan_saved_bytes(b, t, c, states) // 4
    return plan


def _selective_scan_fwd(plan, dev, u, dt, A, B, C, D, z, dt_bias, state, lengths, want_state, state_out,
                        for_backward=False):
    """(out, last state or None, states at the tiles' starts, out before its gate; the latter two for the gradient)."""
    out = _like(u)
    if plan.empty:
        return out, _empty_state(plan.state, torch.float32, u.device, state, state_out) if want_state else None, None, None
    if want_state and state_out is None:
        state_out = torch.empty(plan.state, device=u.device, dtype=torch.float32)
    saved = torch.empty(plan.saved, device=u.device, dtype=torch.float32) if for_backward else None
    raw = torch.empty(u.shape, device=u.device, dtype=torch.float32) if for_backward and z is not None else None
    ws = _workspace(plan.ws, u.device) if plan.ws else None
    _launch(dev, "bmx_selective_scan_fwd", u.data_ptr(), dt.data_ptr(), A.data_ptr(), B.data_ptr(), C.data_ptr(), _ptr(D),
            _ptr(z), _ptr(dt_bias), _ptr(state), _ptr(lengths), *plan.codes, plan.shape, plan.strides, plan.softplus,
            out.data_ptr(), _ptr(state_out), _ptr(saved), _ptr(raw), _ptr(ws), plan.ws)
    return out, state_out, saved, raw


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, plan, dev, u, dt, A, B, C, D, z, dt_bias, state, lengths, want_state):
        out, last, saved, raw = _selective_scan_fwd(plan, dev, u, dt, A, B, C, D, z, dt_bias, state, lengths, want_state, None,
                                                    for_backward=True)
        # not the first state, which the gradient does not read (`saved` has it): it may move on in place before then
        ctx.save_for_backward(u, dt, A, B, C, D, z, dt_bias, lengths, saved, raw)
        ctx.rest = plan, dev
        ctx.set_materialize_grads(False)
        return out, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dlast):
        plan, dev = ctx.rest
        *tensors, lengths, saved, raw = ctx.saved_tensors
        u, dt, A, B, C, D, z, dt_bias = tensors
        grads = _grads(ctx.needs_input_grad[2:10], tensors, plan.empty)
        grads.append(torch.empty(plan.state, device=u.device, dtype=torch.float32) if ctx.needs_input_grad[10] else None)
        if plan.empty:
            if grads[8] is not None:
                grads[8] = grads[8].zero_() if dlast is None else dlast
        elif any(g is not None for g in grads):
            dout, dlast = torch.zeros_like(u, memory_format=torch.contiguous_format) if dout is None else _dense(dout), _dense(dlast)
            ws = _workspace(plan.ws_bwd, u.device)
            du, ddt, dA, dB, dC, dD, dz, dbias, dstate = map(_ptr, grads)
            _launch(dev, "bmx_selective_scan_bwd", u.data_ptr(), dt.data_ptr(), A.data_ptr(), B.data_ptr(), C.data_ptr(),
                    _ptr(D), _ptr(z), _ptr(dt_bias), _ptr(lengths), *plan.codes, plan.shape, plan.strides, plan.softplus,
                    saved.data_ptr(), _ptr(raw), dout.data_ptr(), _ptr(dlast), du, ddt, dA, dB, dC, dD, dz, dbias, dstate,
                    ws.data_ptr(), plan.ws_bwd)
        return None, None, *grads, None, None


def selective_scan(u, dt, A, B, C, D=None, z=None, dt_bias=None, state=None, lengths=None, softplus=True,
                   return_state=False, state_out=None):
    """A diagonal state space whose step and whose input and output maps depend on the token
    (``bmx_selective_scan_fwd``), token after token for every channel c (of group g) and state n:

        ``d = softplus(dt + dt_bias)``  (``softplus`` False: ``d = dt + dt_bias``)
        ``h = exp(d A[c, n]) h + d u B[g, n]``
        ``y = sum_n C[g, n] h + D u``,  ``out = y * silu(z)``  (z None: y)

    u, dt, z [B, T, C] and B, C [B, T, G, N] are fp32 or bf16, one type; C a multiple of 8 G, N 8, 16, 32 or 64, any T
    from one token on, in any strides (column slices of one projection are read in place; layouts that the kernel cannot
    read are copied).  A [C, N] (finite), D and dt_bias [C] are fp32.  state: what h starts from, [B, C, N] fp32
    (None: zeros).  lengths: int32 or int64 [B] on the device, the tokens of each sequence (taken into [0, T]); later ones
    are never read, give zeros and leave the state alone.

    Returns out, dense, in u's type; ``return_state``: (out, the last state, fp32), the next call's state.  ``state_out``:
    a dense buffer that takes it instead of a new tensor, ``state`` itself included (a decoder's step in place); without
    gradients only.  States and sums are fp32.  Gradients reach every tensor but lengths, from out and the returned state,
    and are the same bits on every run.  For them a call keeps, beside its operands but the first state, N / 4 bytes for every
    token and channel (states every 16 tokens) and with z four more (y)."""
    tensors = u, dt, A, B, C, D, z, dt_bias, state
    want, grad = return_state or state_out is not None, _needs_grad(*tensors)
    dev = _same_device(*tensors, lengths, state_out)
    softplus = int(bool(softplus))

    def plan_of(u, dt, A, B, C, D, z, dt_bias, state, lengths):
        return _scan_plan(_layout(u), _layout(dt), _layout(A), _layout(B), _layout(C), _layout(D), _layout(z), _layout(dt_bias),
                          _layout(state), _layout(lengths), softplus)

    plan = plan_of(*tensors, lengths)
    if not plan.in_place or _bits(u, dt, B, C, z) % plan.unit or _bits(A, D, dt_bias, state) % 16:
        u, dt, B, C, z = map(_readable, (u, dt, B, C, z), plan.ok, [plan.unit] * 5)
        A, D, dt_bias, state = map(_readable, (A, D, dt_bias, state), plan.dense)
        lengths = None if lengths is None else lengths.contiguous()
        plan = plan_of(u, dt, A, B, C, D, z, dt_bias, state, lengths)
    if state_out is not None:
        _check_state_out(state_out, plan, torch.float32, state, (u, dt, A, B, C, D, z, dt_bias, lengths),
                         grad or _needs_grad(state_out))
    args = plan, dev, u, dt, A, B, C, D, z, dt_bias, state, lengths, want
    out, last = _SelectiveScan.apply(*args) if grad else _selective_scan_fwd(*args, state_out)[:2]
    _written(state_out)
    return (out, last) if return_state else out
