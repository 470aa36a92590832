"""Device-tensor front ends of the matrix-vector product, transpose, cast and row-norm entry points of the C ABI
(used by the tests and the benchmark; torch only owns memory and the stream).

Reference semantics: the Vector overloads of ``de::blas::cuda::GEMM`` (srcs/modules/BLAS/GEMM/CUDA/VMM.cu:142-184),
``de::cuda::Transpose`` (srcs/modules/BLAS/Basic_process/transpose/transpose.cu:50-101) and ``de::cuda::TypeCast``
(srcs/modules/BLAS/Basic_process/type_cast/GPU_Matrix_type_cast.cu:38-85).
"""
import ctypes

import torch

from . import capi
from .gemm import _ld

_OUT = {(capi.FP32, 0): torch.float32, (capi.FP16, capi.ACCU_L1): torch.float32,
        (capi.FP16, capi.ACCU_L2): torch.float16, (capi.FP16, capi.ACCU_L3): torch.float16}


def gemv(A, x, trans=False, fp16_accu=capi.ACCU_L1, out=None, workspace=None):
    """``y = A @ x`` (trans=False, x has A.shape[1] entries) or ``y = x @ A`` (trans=True, x has A.shape[0]).

    float32: fp32 result.  float16: ``fp16_accu`` 0 = fp32 arithmetic and an fp32 result, 1 = fp32 arithmetic and
    an fp16 result, 2 = fp16 arithmetic and an fp16 result.  Launches on torch's current stream."""
    if not A.is_cuda:
        raise RuntimeError("decx_b200.blas works on CUDA tensors only (no CPU fallback)")
    dt = {torch.float32: capi.FP32, torch.float16: capi.FP16}.get(A.dtype)
    if dt is None or x.dtype != A.dtype:
        raise TypeError("A and x must both be float32 or both float16")
    rows, cols = A.shape
    if x.numel() != (rows if trans else cols) or not x.is_contiguous():
        raise ValueError("x must be a contiguous vector matching A")
    accu = fp16_accu if dt == capi.FP16 else 0
    n = cols if trans else rows
    if out is None:
        out = torch.empty(n, dtype=_OUT[(dt, accu)], device=A.device)
    need = int(capi.lib.decxb200_gemv_workspace_bytes(dt, accu, int(trans), rows, cols))
    if need and (workspace is None or workspace.numel() < need):
        workspace = torch.empty(need, dtype=torch.uint8, device=A.device)
    with torch.cuda.device(A.device):
        capi.check(capi.lib.decxb200_gemv(dt, accu, int(trans), torch.cuda.current_stream().cuda_stream, rows, cols,
                                          A.data_ptr(), _ld(A), x.data_ptr(), out.data_ptr(),
                                          workspace.data_ptr() if need else None, need))
    return out


def transpose(src, out=None):
    """``out[c, r] = src[r, c]`` for a pitched 2-D tensor of 1-, 2-, 4-, 8- or 16-byte elements."""
    if not src.is_cuda:
        raise RuntimeError("decx_b200.blas works on CUDA tensors only (no CPU fallback)")
    rows, cols = src.shape
    if out is None:
        out = torch.empty((cols, rows), dtype=src.dtype, device=src.device)
    with torch.cuda.device(src.device):
        capi.check(capi.lib.decxb200_transpose(src.element_size(), torch.cuda.current_stream().cuda_stream, rows, cols,
                                               src.data_ptr(), _ld(src), out.data_ptr(), _ld(out)))
    return out


_CASTS = {(torch.float32, torch.float16): capi.CAST_F32_F16, (torch.float16, torch.float32): capi.CAST_F16_F32,
          (torch.float32, torch.float64): capi.CAST_F32_F64, (torch.float64, torch.float32): capi.CAST_F64_F32,
          (torch.int32, torch.float32): capi.CAST_I32_F32, (torch.float32, torch.int32): capi.CAST_F32_I32}


def cast(src, dtype, out=None):
    """Element type cast of a pitched 2-D tensor (fp32<->fp16, fp32<->fp64, int32<->fp32)."""
    if not src.is_cuda:
        raise RuntimeError("decx_b200.blas works on CUDA tensors only (no CPU fallback)")
    kind = _CASTS.get((src.dtype, dtype))
    if kind is None:
        raise TypeError(f"no device cast from {src.dtype} to {dtype}")
    rows, cols = src.shape
    if out is None:
        out = torch.empty((rows, cols), dtype=dtype, device=src.device)
    with torch.cuda.device(src.device):
        capi.check(capi.lib.decxb200_cast2d(kind, torch.cuda.current_stream().cuda_stream, rows, cols, src.data_ptr(),
                                            _ld(src), out.data_ptr(), _ld(out)))
    return out


def new_q8(rows, cols, device):
    """An empty 8-bit operand: a rows x cols float8_e4m3fn view whose rows start a multiple of 128 bytes apart
    (the layout ``gemm.gemm_q8`` takes), and its rows' float32 scales."""
    buf = torch.empty((rows, -(-cols // 128) * 128), dtype=torch.float8_e4m3fn, device=device)
    return buf[:, :cols], torch.empty(rows, dtype=torch.float32, device=device)


def _q8_out(src, out, scales):
    rows, cols = src.shape
    q, s = new_q8(rows, cols, src.device)
    return (q if out is None else out), (s if scales is None else scales)


def cast_q8(src, out=None, scales=None):
    """``src`` (rows x cols, float16 or float32, pitched) as an 8-bit operand: returns ``(q, scales)`` with
    ``scales[r] = max|src[r]| / 448`` and ``q = e4m3(src / scales[:, None])``.  Launches on torch's current stream."""
    if out is None or scales is None:
        out, scales = _q8_out(src, out, scales)
    code = capi.front.cast_q8(src, out, scales)
    if code:
        capi.check(code)
    return out, scales


def rmsnorm_q8(x, weight, residual=None, eps=1e-6, out=None, scales=None, sum_out=None):
    """Root-mean-square norm of the rows of ``x + residual`` as an 8-bit operand: returns ``(q, scales, sum)``.

    ``h = x + residual``, ``sum = h`` rounded to x's type (None without a residual), ``y = h / sqrt(mean(h^2) + eps) *
    weight``, ``scales[r] = max|y[r]| / 448``, ``q = e4m3(y / scales[:, None])``.  float16 or float32, pitched rows;
    ``sum_out`` may be ``x`` or ``residual`` themselves.  Launches on torch's current stream."""
    if out is None or scales is None:
        out, scales = _q8_out(x, out, scales)
    if sum_out is None and residual is not None:
        sum_out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    code = capi.front.rmsnorm_q8(x, weight, residual, eps, out, scales, sum_out)
    if code:
        capi.check(code)
    return out, scales, sum_out


def pack_q4(q):
    """Values 0..15 (rows x cols, any integer type) in the layout ``gemv_q4`` takes: two per byte, the even column in the
    low nibble, rows 16 bytes apart or a multiple.  Meant for laying weights out once."""
    rows, cols = q.shape
    buf = torch.zeros((rows, -(-cols // 32) * 16), dtype=torch.uint8, device=q.device)
    nibbles = q.to(torch.uint8) & 15
    buf[:, :(cols + 1) // 2] = nibbles[:, 0::2]
    buf[:, :cols // 2] |= nibbles[:, 1::2] << 4
    return buf[:, :(cols + 1) // 2]


def gemv_q4(W, scales, x, group, zeros=None, x_scales=None, out_dtype=torch.float32, out=None):
    """``y = W4 @ x`` for one vector (x of shape (cols,)) or 1 to 16 of them (x of shape (n, cols), y of shape (n, rows)).

    ``W``: uint8, rows x ceil(cols / 2), two weights per byte (``pack_q4``); weight k of row r stands for
    ``(q - zeros[r, k // group]) * scales[r, k // group]``, with 8 for the zero when ``zeros`` is None.  ``scales``:
    float16; ``zeros``: uint8; ``group``: 32, 64 or 128.  ``x``: float16, or float8_e4m3fn whose rows stand for
    ``x * x_scales[:, None]``.  Sums are float32.  Launches on torch's current stream."""
    if out is None:
        rows = W.shape[0]
        out = torch.empty(rows if x.dim() == 1 else (x.shape[0], rows), dtype=out_dtype, device=W.device)
    code = capi.front.gemv_q4(W, scales, x, group, zeros, x_scales, out)
    if code:
        capi.check(code)
    return out


def conv2d(src, kernels, strides=(1, 1), extend=0, out=None, workspace=None, status=None):
    """fp32 cross-correlation ``out[y, x, t] = sum src[y*sy+i-py, x*sx+j-px, c] * kernels[t, i, j, c]`` of an
    H x W x C tensor with n kernels of kh x kw x C (``de::nn::cuda::Conv2D``); ``extend`` 0 = no border,
    2 = zero border.  Tensors are channels-innermost and may be pitched views.  Launches on the current stream."""
    if not src.is_cuda or src.dtype != torch.float32 or kernels.dtype != torch.float32:
        raise TypeError("conv2d takes float32 CUDA tensors")
    H, W, C = src.shape
    n, kh, kw, C2 = kernels.shape
    if C2 != C or src.stride(2) != 1 or kernels.stride(3) != 1:
        raise ValueError("src is H x W x C, kernels n x kh x kw x C, channels innermost")
    sx, sy = strides
    oh, ow = ctypes.c_uint32(), ctypes.c_uint32()
    capi.check(capi.lib.decxb200_conv2d_fp32_out_dims(H, W, kh, kw, sx, sy, extend, ctypes.byref(oh), ctypes.byref(ow)))
    if out is None:
        out = torch.empty((oh.value, ow.value, n), dtype=torch.float32, device=src.device)
    src_dp, src_wp = src.stride(1), src.stride(0) // src.stride(1)
    k_dp, k_wp = kernels.stride(2), kernels.stride(1) // kernels.stride(2)
    dst_dp, dst_wp = out.stride(1), out.stride(0) // out.stride(1)
    # an odd pitch in the query selects the form that works for every destination
    need = int(capi.lib.decxb200_conv2d_fp32_workspace_bytes(H, W, C, kh, kw, n, sx, sy, extend, dst_wp,
                                                             dst_dp if out.data_ptr() % 16 == 0 else 1))
    if workspace is None or workspace.numel() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=src.device)
    with torch.cuda.device(src.device):
        capi.check(capi.lib.decxb200_conv2d_fp32(
            torch.cuda.current_stream().cuda_stream, src.data_ptr(), H, W, C, src_wp, src_dp, kernels.data_ptr(), kh, kw, n,
            k_wp, k_dp, kernels.stride(0), out.data_ptr(), dst_wp, dst_dp, sx, sy, extend, workspace.data_ptr(), need,
            status.data_ptr() if status is not None else None))
    return out
