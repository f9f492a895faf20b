"""RMS norm, with the residual add in front of it and 8-bit rows behind it, in one pass.

``s = x + delta`` (rounded to bf16 as the residual stream is stored), ``y = s * rsqrt(mean(s^2) + eps) * w``, and ``y``
rounded once to 8 bits, in one of the two layouts that a product here reads:

* ``"int8"``: int8 rows with one fp32 scale each (``max|y| / 127``), for ``gemm_int8``;
* ``"e4m3_1x128"``: e4m3 with one fp32 scale per row and 128 columns (``max|y| / 448``), for ``grouped_gemm_fp8``.

The bf16 form with a gradient is ``add_rmsnorm``; these have none and say so when one is asked for.  A row (block) of
zeros has scale 1; one that holds a NaN or an infinity has scale NaN.
"""
from __future__ import annotations

import torch

from . import native
from .fp8 import E4M3_MAX
from .fused import rmsnorm_reference
from .gemm import count_launch
from .int8 import MAX_ROW, _no_gradient, pitched_int8, pitched_like, quantize_rows_int8_reference

FORMATS = ("int8", "e4m3_1x128")


def _quantized_e4m3(y: torch.Tensor):
    rows, H = y.shape
    b = y.view(rows, H // 128, 128)
    top = b.abs().amax(dim=-1)
    some = top >= 6e-36
    scale = torch.where(some, top / E4M3_MAX, 1.0)
    q = torch.where(some.unsqueeze(-1), b / scale.unsqueeze(-1), 0.0).clamp(-E4M3_MAX, E4M3_MAX)
    return q.to(torch.float8_e4m3fn).view(rows, H), torch.where(torch.isfinite(top), scale, float("nan"))


def _statement(s, weight, eps, zero_centered, fmt):
    y = rmsnorm_reference(s.float(), weight, eps, zero_centered)
    if fmt == "int8":
        q, scale = quantize_rows_int8_reference(y)
        return pitched_like(q), scale
    return _quantized_e4m3(y)


def _run(x, delta, weight, eps, zero_centered, fmt, what):
    if fmt not in FORMATS:
        raise ValueError(f"{what}: fmt is one of {FORMATS}, got {fmt!r}")
    if x.dim() < 1 or weight.shape != x.shape[-1:] or x.shape[-1] < 1:
        raise ValueError(f"{what}: weight {tuple(weight.shape)} does not fit rows of {tuple(x.shape)}")
    if delta is not None and delta.shape != x.shape:
        raise ValueError(f"{what}: x {tuple(x.shape)} and delta {tuple(delta.shape)} differ")
    index = x.get_device()              # -1 on the CPU
    if weight.get_device() != index or (delta is not None and delta.get_device() != index):
        raise ValueError(f"{what}: operands on different devices")
    H = x.shape[-1]
    if fmt == "e4m3_1x128" and H % 128:
        raise ValueError(f"{what}: e4m3 blocks need a multiple of 128 columns, got {H}")
    _no_gradient(what, x, delta, weight)
    flat = x.dim() == 2
    x2 = x if flat else x.reshape(-1, H)
    d2 = delta if flat or delta is None else delta.reshape(-1, H)
    rows = x2.shape[0]
    if index < 0:
        s = x2 if d2 is None else (x2.float() + d2.float()).to(x.dtype)
        q, scale = _statement(s, weight, eps, zero_centered, fmt)
        return s, q, scale
    bf16 = torch.bfloat16
    if x.dtype != bf16 or weight.dtype != bf16 or (delta is not None and delta.dtype != bf16):
        raise TypeError(f"{what}: x, delta and weight are bf16 on the GPU")
    if H > MAX_ROW:
        raise ValueError(f"{what}: at most {MAX_ROW} columns, got {H}")
    if x2.stride(1) != 1:
        x2 = x2.contiguous()
    s, sp, dp, ldd = None, None, None, 0
    if d2 is not None:
        if d2.stride(1) != 1:
            d2 = d2.contiguous()
        s = x2.new_empty((rows, H))
        sp, dp, ldd = s.data_ptr(), d2.data_ptr(), d2.stride(0)
    if weight.stride(0) != 1:
        weight = weight.contiguous()
    if fmt == "int8":
        q = pitched_int8(rows, H, x2)
        scale = x2.new_empty(rows, dtype=torch.float32)
    else:
        q = x2.new_empty((rows, H), dtype=torch.float8_e4m3fn)
        scale = x2.new_empty((rows, H // 128), dtype=torch.float32)
    if rows:
        rc = native.launch(native.load().stb_norm_quant, index, x2.data_ptr(), dp, weight.data_ptr(), sp, q.data_ptr(),
                           scale.data_ptr(), rows, H, x2.stride(0), ldd, H, q.stride(0), eps, int(zero_centered),
                           int(fmt != "int8"))
        if rc:
            native.check(rc, f"{what} rows={rows} H={H} {fmt}")
        count_launch()
    return s, q, scale


def rmsnorm_quant(x, weight, eps: float = 1e-6, zero_centered: bool = False, fmt: str = "int8"):
    """``rmsnorm(x)`` in 8 bits: ``(q [rows, H], scales)`` for bf16 ``x [..., H]``, leading dimensions flattened."""
    _, q, scale = _run(x, None, weight, eps, zero_centered, fmt, "rmsnorm_quant")
    return q, scale


def add_rmsnorm_quant(x, delta, weight, eps: float = 1e-6, zero_centered: bool = False, fmt: str = "int8"):
    """``(x + delta, q, scales)``: the residual stream and ``rmsnorm`` of it in 8 bits (``q [rows, H]``)."""
    s, q, scale = _run(x, delta, weight, eps, zero_centered, fmt, "add_rmsnorm_quant")
    return s if x.dim() == 2 else s.view(x.shape), q, scale
