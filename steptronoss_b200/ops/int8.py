"""Products of frozen weights in 8-bit integers: one scale per token, one per output channel.

``Y[m, n] = sx[m] * sw[n] * sum_k xq[m, k] * wq[n, k]`` with exact int32 sums (``csrc/gemm_int8_sm100.cu``), rounded
once to bf16 (or fp32).  A frozen model (a distillation teacher, the reference policy of a PPO run) lays its weights
out once with ``quantize_rows_int8`` and runs its projections with ``linear_int8``, or with ``gemm_int8`` behind
``add_rmsnorm_quant``, which already leaves int8 rows.  These operators carry no gradient and say so when one is asked
for.  The reference runs such models in bf16.

Rows of an 8-bit operand start on 16-byte boundaries (the tensor-map copies of the kernel need that):
``quantize_rows_int8`` returns a view with such a pitch whatever the width, on 128-byte boundaries where rows are long.
"""
from __future__ import annotations

import torch

from . import native
from .gemm import count_launch

INT8_MAX = 127.0
MAX_K = 131071            # int32 sums of 128 * 128 stay below 2^31
MAX_ROWS = 1 << 30        # tokens or channels of a product; its C entry point takes 32-bit numbers
MAX_ROW = 32768           # widest row of the quantisation kernels
P, I, L, F = native.P, native.I, native.L, native.F
native.register_signature("stb_gemm_int8", [P, P, P, P, P, I, I, I, L, L, L, I, P, P])
native.register_signature("stb_norm_quant", [P, P, P, P, P, P, L, I, L, L, L, L, F, I, I, P])


def _no_gradient(what: str, *tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{what} has no gradient: run frozen models under torch.no_grad() or detach the operands")


def pitched_int8(rows: int, width: int, like: torch.Tensor) -> torch.Tensor:
    """An uninitialised int8 ``[rows, width]`` on the device of ``like`` whose rows start on 128-byte boundaries (on 16-byte
    boundaries where they are shorter than that): the product takes multiples of 16 bytes, and loads whole lines
    faster (515 x 2048 x 1990: 11.6 us with a pitch of 2000 bytes on both sides, 9.3 us for rows of 2048)."""
    unit = 128 if width > 128 else 16
    pitch = (width + unit - 1) // unit * unit
    q = like.new_empty((rows, pitch), dtype=torch.int8)
    return q if width == pitch else q[:, :width]


def pitched_like(q: torch.Tensor) -> torch.Tensor:
    """A copy of int8 rows with a pitch that the product takes."""
    out = pitched_int8(q.shape[0], q.shape[1], q)
    out.copy_(q)
    return out


# ----------------------------------------------------------------------------------------------- quantisation
def quantize_rows_int8_reference(x: torch.Tensor):
    """``x [M, K]`` -> ``(q [M, K] int8, scales [M] fp32)``, ``scale = max|x| / 127`` per row, rounded to nearest even.

    A row of zeros has scale 1; a row with a NaN or an infinity has scale NaN and values 0."""
    xf = x.float()
    top = xf.abs().amax(dim=-1) if x.shape[-1] else xf.new_zeros(x.shape[:-1])
    some, finite = top >= 6e-36, torch.isfinite(top)
    scale = torch.where(some, top / INT8_MAX, 1.0)
    q = torch.where((some & finite).unsqueeze(-1), torch.round(xf / scale.unsqueeze(-1)), 0.0).to(torch.int8)
    return q, torch.where(finite, scale, float("nan"))


def quantize_rows_int8(x: torch.Tensor):
    """bf16 rows ``[M, K]`` to int8 with one scale each: tokens of an activation, or output channels of a weight."""
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"quantize_rows_int8 takes [M, K], got {tuple(x.shape)}")
    _no_gradient("quantize_rows_int8", x)
    M, K = x.shape
    if M > MAX_ROWS:
        raise ValueError(f"quantize_rows_int8 takes at most {MAX_ROWS} rows, got {M}")
    if not x.is_cuda:
        q, s = quantize_rows_int8_reference(x)
        return pitched_like(q), s
    if x.dtype != torch.bfloat16:
        raise TypeError(f"quantize_rows_int8 takes bf16 on the GPU, got {x.dtype}")
    if K > MAX_ROW:
        raise ValueError(f"quantize_rows_int8 takes rows of at most {MAX_ROW} columns, got {K}")
    if x.stride(1) != 1 and K > 1:
        x = x.contiguous()
    q = pitched_int8(M, K, x)
    s = x.new_empty(M, dtype=torch.float32)
    if M:
        rc = native.launch(native.load().stb_norm_quant, x.get_device(), x.data_ptr(), None, None, None, q.data_ptr(),
                           s.data_ptr(), M, K, x.stride(0), 0, 0, q.stride(0), 0.0, 0, 0)
        if rc:
            native.check(rc, f"quantize_rows_int8 M={M} K={K}")
        count_launch()
    return q, s


def dequantize_rows_int8(q: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    return q.float() * s.unsqueeze(-1)


# ----------------------------------------------------------------------------------------------- products
def gemm_int8_reference(xq, sx, wq, sw, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The sums in fp64, where every int8 product sum is exact."""
    dot = xq.double() @ wq.double().t()
    return (dot.float() * sx.unsqueeze(-1) * sw.unsqueeze(0)).to(out_dtype)


def _pitch(t: torch.Tensor) -> int:
    """Bytes from row to row if the kernel takes these rows, else 0 (a single row has any pitch)."""
    pitch, step = t.stride()
    rows, width = t.shape
    if rows <= 1:
        pitch = (width + 15) // 16 * 16
    ok = t.data_ptr() % 16 == 0 and pitch % 16 == 0 and pitch >= width and (step == 1 or width == 1)
    return pitch if ok or rows == 0 else 0


def gemm_int8(xq: torch.Tensor, sx: torch.Tensor, wq: torch.Tensor, sw: torch.Tensor,
              out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """``xq [M, K]`` (scales ``sx [M]``) times ``wq [N, K]`` transposed (scales ``sw [N]``) -> ``[M, N]``.

    ``out`` (bf16 or fp32, last dimension contiguous, any row stride) takes the result instead of a new tensor."""
    if xq.dim() != 2 or wq.dim() != 2 or xq.shape[1] != wq.shape[1]:
        raise ValueError(f"gemm_int8 takes [M, K] and [N, K], got {tuple(xq.shape)} and {tuple(wq.shape)}")
    M, K = xq.shape
    N = wq.shape[0]
    if xq.dtype != torch.int8 or wq.dtype != torch.int8:
        raise TypeError(f"gemm_int8 takes int8 operands, got {xq.dtype} and {wq.dtype}")
    if sx.dtype != torch.float32 or sw.dtype != torch.float32 or sx.shape != (M,) or sw.shape != (N,):
        raise ValueError(f"gemm_int8 takes fp32 scales [{M}] and [{N}], got {sx.dtype} {tuple(sx.shape)} and "
                         f"{sw.dtype} {tuple(sw.shape)}")
    if M > MAX_ROWS or N > MAX_ROWS:
        raise ValueError(f"gemm_int8 takes at most {MAX_ROWS} tokens and channels, got {M} and {N}")
    index = xq.get_device()              # -1 on the CPU
    if wq.get_device() != index or sx.get_device() != index or sw.get_device() != index:
        raise ValueError("gemm_int8: operands on different devices")
    if not 1 <= K <= MAX_K:
        raise ValueError(f"gemm_int8 takes 1 <= K <= {MAX_K}, got {K}")
    if out is not None:
        out_dtype = out.dtype
        if out.shape != (M, N) or out.get_device() != index or (N > 1 and out.stride(1) != 1) or (
                M > 1 and out.stride(0) < N):
            raise ValueError(f"gemm_int8: out must be [{M}, {N}] on {xq.device} with separate rows and a contiguous last "
                             f"dimension, got {tuple(out.shape)} with strides {out.stride()} on {out.device}")
    if out_dtype != torch.bfloat16 and out_dtype != torch.float32:
        raise TypeError(f"gemm_int8 writes bf16 or fp32, not {out_dtype}")
    _no_gradient("gemm_int8", sx, sw, out)
    if index < 0:
        res = gemm_int8_reference(xq, sx, wq, sw, out_dtype)
        return res if out is None else out.copy_(res)
    ldx, ldw = _pitch(xq), _pitch(wq)
    if not ldx or not ldw:
        raise ValueError(f"gemm_int8: the rows of xq and wq must be contiguous and start on 16-byte boundaries, got "
                         f"strides {xq.stride()} and {wq.stride()} (quantize_rows_int8 returns such rows, pitched_like "
                         "makes them)")
    given = out
    if out is None:
        out = xq.new_empty((M, N), dtype=out_dtype)
    if M and N:
        if not sx.is_contiguous():
            sx = sx.contiguous()
        if not sw.is_contiguous():
            sw = sw.contiguous()
        rc = native.launch(native.load().stb_gemm_int8, index, xq.data_ptr(), sx.data_ptr(), wq.data_ptr(), sw.data_ptr(),
                           out.data_ptr(), M, N, K, ldx, ldw, out.stride(0) if M > 1 else N,
                           int(out_dtype == torch.float32), native.status_ptr(index))
        if rc:
            native.check(rc, f"gemm_int8 M={M} N={N} K={K}")
        count_launch()
        if given is not None:
            torch.autograd.graph.increment_version(out)
    return out


def linear_int8(x: torch.Tensor, wq: torch.Tensor, sw: torch.Tensor, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x @ dequantised(w).T`` for bf16 ``x [..., K]``: its rows are quantised on the fly."""
    _no_gradient("linear_int8", x, sw)
    if x.dim() < 1 or wq.dim() != 2 or x.shape[-1] != wq.shape[1]:
        raise ValueError(f"linear_int8 takes [..., K] and [N, K], got {tuple(x.shape)} and {tuple(wq.shape)}")
    q, s = quantize_rows_int8(x if x.dim() == 2 else x.reshape(-1, x.shape[-1]))
    y = gemm_int8(q, s, wq, sw, out_dtype=out_dtype or torch.bfloat16)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], wq.shape[0])
