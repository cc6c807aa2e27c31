"""Products with weights and activations in 8-bit integers (``csrc/int8_linear.cu``), for serving.

A row of activations is held as whole numbers c = rint(x / s) (halves to even) with s = max(|x|, 1e-10) / 127 in fp32, a scale for each token; a row of
weights likewise, a scale for each output channel. Codes of the caller's own may be any int8, -128 among them. Sums of products are whole numbers that 32 bits
hold up to K = 131071 (128 * 128 K < 2^31), so that a result depends on no order and not on how many tokens came with it; scales and bias are applied in fp32 and the
result is rounded once. A row with a value that is not finite gives NaN, and so does a sum of zero where a token's scale times a channel's is beyond fp32.
``engines.int8_quantize_per_token`` and ``inference.serving.INT8Inference`` hold rows the same way but for quotients next to a half, which they take from rounded
quotients; the product of the latter is of fp32.

No gradient and no tangent passes through these."""
from __future__ import annotations

import functools
import struct
from typing import NamedTuple, Optional, Union

import torch
import torch.nn.functional as F
from torch.autograd import forward_ad

from .. import _native
from . import runtime as rt
from .functional import swiglu
from .gemm import linear

_native.register_cuda_sigs({"inv_int8_rows": [_native.vp], "inv_int8_linear": [_native.vp],
                            "inv_int8_alone": [_native.i64] * 3, "inv_int8_plan": [_native.i64] * 3 + [_native.i32, _native.vp]})

# What the entries are given: x, weights, their scales, bias, result, codes, their scales, status and stream; tokens, weight rows, K; strides of x, weights,
# result and codes; whether x, the result and the bias are fp32; gated.
_CALL = struct.Struct("=9Q 11q").pack

MAX_K, LEAST = 131071, 1e-10
_int8, _fp32, _bf16 = torch.int8, torch.float32, torch.bfloat16


class Int8Rows(NamedTuple):
    """Activations. On a GPU rows start on 16-byte boundaries, as ``quantize_rows`` makes them."""
    q: torch.Tensor          # [..., K] int8
    scale: torch.Tensor      # [...] fp32

    def dequantize(self) -> torch.Tensor:
        return self.q.float() * self.scale.unsqueeze(-1)


class Int8Weight(NamedTuple):
    """A weight [N, K], or a stack of them [experts, N, K]. On a GPU rows start on 16-byte boundaries, as ``quantize`` makes them."""
    q: torch.Tensor          # [..., N, K] int8
    scale: torch.Tensor      # [..., N] fp32

    @staticmethod
    def quantize(w: torch.Tensor) -> "Int8Weight":
        """w [..., N, K] in bf16 or fp32. Nothing of the weight's size is held beside the result, unless w's rows have no even distance or no unit stride: then a copy."""
        return Int8Weight(*quantize_rows(w.detach()))

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values that the codes stand for: products in fp32, rounded once to ``dtype``."""
        s = self.scale.unsqueeze(-1)
        if dtype is _fp32 or s.requires_grad:
            return (self.q * s).to(dtype)
        return torch.mul(self.q, s, out=torch.empty(self.q.shape, dtype=dtype, device=self.q.device))      # nothing of fp32 held on the way


def refuse_gradients(what, *tensors):
    grad = forward_ad._current_level >= 0
    if torch.is_grad_enabled():
        for t in tensors:
            grad = grad or (t is not None and t.requires_grad)
    if grad:
        raise RuntimeError(f"{what} serves: no gradient and no tangent passes through it (call it under torch.no_grad())")


def _empty_rows(shape, device):
    """int8 [..., K] whose rows start on 16-byte boundaries."""
    k = shape[-1]
    return torch.empty(*shape[:-1], (k + 15) // 16 * 16, dtype=_int8, device=device)[..., :k]


def _rows_of(x):
    """x [..., K] as rows [T, K] with unit stride, and how far apart they are."""
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    if x.stride(1) != 1 and x.shape[1] > 1:
        x = x.contiguous()
    return x, x.stride(0) if x.shape[0] > 1 else x.shape[1]


def quantize_rows(x: torch.Tensor) -> Int8Rows:
    """x [..., K] in bf16 or fp32 -> whole numbers and a scale for each row, to be given to several products."""
    refuse_gradients("quantize_rows", x)
    if x.dim() < 1 or x.dtype not in (_bf16, _fp32):
        raise TypeError(f"rows of bf16 or fp32, not {x.dtype} {tuple(x.shape)}")
    K = x.shape[-1]
    if not x.is_cuda:
        s = x.float().abs().amax(-1).clamp(min=LEAST).div(torch.tensor(127.0)) if K else torch.full(x.shape[:-1], LEAST / 127)
        s = torch.where(torch.isfinite(s), s, torch.nan)
        q = torch.nan_to_num((x.double() / s.double().unsqueeze(-1)).round(), nan=0.0).to(_int8)
        return Int8Rows(q, s)
    q, s = _empty_rows(x.shape, x.device), torch.empty(x.shape[:-1], dtype=_fp32, device=x.device)
    if x.numel():
        with rt.device_of(x):
            rows, ld = _rows_of(x)
            rt.check(rt.lib().inv_int8_rows(_CALL(rows.data_ptr(), 0, 0, 0, 0, q.data_ptr(), s.data_ptr(), 0, rt.stream_ptr(), rows.shape[0], 0, K, ld, 0, 0,
                                                  q.stride(-2) if x.dim() > 1 else 0, x.dtype is _fp32, 0, 0, 0)), "inv_int8_rows")
    else:
        s.fill_(LEAST / 127)
    return Int8Rows(q, s)


def check_weight(w: Int8Weight, dims: int):
    q, s = w
    if q.dim() != dims or q.dtype != _int8 or s.shape != q.shape[:-1] or s.dtype != _fp32 or not s.is_contiguous() or s.device != q.device:
        raise ValueError(f"weight of {q.dtype} {tuple(q.shape)} with scales of {s.dtype} {tuple(s.shape)} on {s.device}: int8 {'[experts, N, K]' if dims == 3 else '[N, K]'} "
                         f"and contiguous fp32 for its rows on {q.device}")
    if q.shape[-1] > MAX_K:
        raise ValueError(f"K of {q.shape[-1]}: sums of more than {MAX_K} products do not fit in 32 bits")
    if q.is_cuda and (q.data_ptr() % 16 or q.stride(-1) != 1 or any(d % 16 for d in q.stride()[:-1]) or q.stride(-2) < q.shape[-1]):
        raise ValueError(f"weight rows with strides {q.stride()}: unit stride, 16-byte boundaries and no overlap on a GPU (Int8Weight.quantize makes them so)")


@functools.lru_cache(maxsize=1024)
def _alone(T, N, K):
    return rt.lib().inv_int8_alone(T, N, K) != 0


def int8_linear(x: Union[torch.Tensor, Int8Rows], w: Int8Weight, bias: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                gated: bool = False) -> torch.Tensor:
    """x [..., K], in bf16 or fp32 or as ``quantize_rows`` gives it, times w [N, K] -> [..., N] in ``out_dtype`` (bf16 or fp32; that of x if not given, bf16
    for ``Int8Rows``). ``bias`` [N] in bf16 or fp32. ``gated``: w holds gate rows [0, N / 2) and up rows behind them, the result is silu(gate) * up
    [..., N / 2]."""
    codes = None
    if isinstance(x, Int8Rows):
        codes, x = x, x.q
    q, sw = w
    dtype, shape, dev = x.dtype, x.shape, x.get_device()
    out_dtype = out_dtype or (_bf16 if codes is not None else dtype)
    N, K = q.shape if q.dim() == 2 else (0, -1)
    ldw = K if K % 16 == 0 and q.is_contiguous() else q.stride(0) if K >= 0 and q.stride(1) == 1 else -1
    if not (shape and shape[-1] == K <= MAX_K and q.dtype is _int8 and sw.dtype is _fp32 and sw.shape == (N,) and sw.is_contiguous()
            and dev == q.get_device() == sw.get_device() and (codes is not None or dtype is _bf16 or dtype is _fp32) and (out_dtype is _bf16 or out_dtype is _fp32)
            and (bias is None or bias.shape == (N,) and (bias.dtype is _bf16 or bias.dtype is _fp32) and bias.get_device() == dev)
            and (codes is None or dtype is _int8 and codes.scale.shape == shape[:-1] and codes.scale.dtype is _fp32 and codes.scale.get_device() == dev)
            and (dev < 0 or ldw % 16 == 0 and ldw >= K and q.data_ptr() % 16 == 0)) or gated and N % 2:
        _refuse(x, codes, w, bias, out_dtype, gated)
    refuse_gradients("int8_linear", x, bias, sw, None if codes is None else codes.scale)
    cols = N // 2 if gated else N
    if dev < 0:
        codes = quantize_rows(x) if codes is None else codes
        y = F.linear(codes.q.double(), q.double()).float() * (codes.scale.unsqueeze(-1) * sw)      # in this order: sums times a large scale alone may not fit
        y = y if bias is None else y + bias.float()
        return (F.silu(y[..., :cols]) * y[..., cols:] if gated else y).to(out_dtype)
    out = x.new_empty((*shape[:-1], cols), dtype=out_dtype)
    if cols == 0 or K == 0 or x.numel() == 0:
        return _without_products(out, bias, cols, gated)
    rows, ld = (x, K) if len(shape) == 2 and x.is_contiguous() else _rows_of(x)
    T = rows.shape[0]
    with rt.device_of(x):
        alone = codes is None and T <= 4 and _alone(T, N, K)
        if alone:
            from_x, from_codes, from_scale, ld_codes = rows.data_ptr(), 0, 0, 0
        elif codes is None:
            wide = (K + 15) // 16 * 16
            work = x.new_empty(T * (wide + 4), dtype=torch.uint8)
            at = work.data_ptr()
            from_x, from_codes, from_scale, ld_codes = rows.data_ptr(), at, at + T * wide, wide
        else:
            if rows.data_ptr() % 16 or ld % 16 or ld < K:
                aligned = _empty_rows(rows.shape, x.device)
                rows, ld = aligned.copy_(rows), aligned.stride(0)
            scale = codes.scale.contiguous()
            from_x, from_codes, from_scale, ld_codes = 0, rows.data_ptr(), scale.data_ptr(), ld
        bias = bias if bias is None else bias.contiguous()
        rt.check(rt.lib().inv_int8_linear(_CALL(from_x, q.data_ptr(), sw.data_ptr(), rt.ptr(bias), out.data_ptr(), from_codes, from_scale, rt.status_ptr(x),
                                                rt.stream_ptr(), T, N, K, ld, ldw, cols, ld_codes, dtype is _fp32, out_dtype is _fp32,
                                                bias is not None and bias.dtype is _fp32, gated)), "inv_int8_linear")
        if codes is None and not alone:
            rt.count_launches(1)
    return out


class Int8Linears:
    """A ``linear_fn`` of ``inference.Generator``: projections with their weights in 8-bit integers, laid out once; others as they are. The modules keep their
    own weights beside them, which later changes of them do not reach."""

    def __init__(self, linears):
        with torch.no_grad():
            self.weights = {lin: Int8Weight.quantize(lin.weight) for lin in linears}

    def __call__(self, x, lin):
        w = self.weights.get(lin)
        return linear(x, lin.weight, lin.bias) if w is None else int8_linear(x, w, lin.bias)

    def gated(self, x, lin):
        """silu(gate) * up of a projection that holds both."""
        w = self.weights.get(lin)
        return swiglu(linear(x, lin.weight, lin.bias)) if w is None else int8_linear(x, w, lin.bias, gated=True)


def _without_products(out, bias, cols, gated):
    y = torch.zeros(2 * cols if gated else cols, device=out.device) if bias is None else bias.float()
    return out.copy_(F.silu(y[:cols]) * y[cols:] if gated else y)


def _refuse(x, codes, w, bias, out_dtype, gated):
    check_weight(w, 2)
    q = w.q
    if codes is not None and (x.dtype != _int8 or codes.scale.shape != x.shape[:-1] or codes.scale.dtype != _fp32 or codes.scale.device != x.device):
        raise ValueError(f"rows of {x.dtype} {tuple(x.shape)} with scales of {codes.scale.dtype} {tuple(codes.scale.shape)}: int8 [..., K] and fp32 [...]")
    if x.dim() == 0 or x.shape[-1] != q.shape[1]:
        raise ValueError(f"x of {tuple(x.shape)} for a weight of {tuple(q.shape)}")
    if x.device != q.device:
        raise ValueError(f"x on {x.device}, weight on {q.device}")
    if codes is None and x.dtype not in (_bf16, _fp32):
        raise TypeError(f"x in bf16 or fp32, not {x.dtype}")
    if out_dtype not in (_bf16, _fp32):
        raise TypeError(f"a result in bf16 or fp32, not {out_dtype}")
    if bias is not None and (bias.shape != w.scale.shape or bias.dtype not in (_bf16, _fp32) or bias.device != q.device):
        raise ValueError(f"bias of {bias.dtype} {tuple(bias.shape)} on {bias.device}: bf16 or fp32 [{q.shape[0]}] on {q.device}")
    raise ValueError(f"gated: {q.shape[0]} rows do not come in pairs")
