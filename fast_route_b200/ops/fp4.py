"""Microscaled 4-bit floating point: E2M1 codes with a scale per block of 16 or 32 elements of a row.

``block=16``: E4M3 block scales and one fp32 scale per matrix (``value = code * (scale * global)``);
``block=32``: E8M0 block scales (powers of two, ``value = code * scale``).  Codes are packed two per byte, the even
element in the low half.  The type of the scale tensor (``float8_e4m3fn`` / ``float8_e8m0fnu``) tells the two apart.
The reference has no such format; its 4-bit weights are GPTQ integers (``ops/splitk_gemm.py``).
"""

from __future__ import annotations

import torch

from .. import _lib

_SMALL = 32768      # elements of a matrix up to which one CTA quantises it, without a workspace
_SCALE_DTYPE = {16: torch.float8_e4m3fn, 32: torch.float8_e8m0fnu}


_BLOCK = {v: k for k, v in _SCALE_DTYPE.items()}


def block_of(q: torch.Tensor, scale: torch.Tensor, what: str = "scale") -> int:
    """The block size of a quantised matrix, after checking that codes and scales belong together."""
    assert q.dtype == torch.uint8, "codes are packed in uint8"
    block = _BLOCK.get(scale.dtype)
    assert block is not None, f"{what} must be float8_e4m3fn or float8_e8m0fnu"
    assert q.is_contiguous() and scale.is_contiguous(), f"codes and {what} must be contiguous"
    a, b = q.shape, scale.shape
    assert a[:-1] == b[:-1] and b[-1] * block == a[-1] * 2, f"{what} does not match the codes"
    return block


def check_global(g: torch.Tensor, mats: int, block: int, what: str = "global_scale") -> None:
    if g is None:
        return
    assert block == 16, f"{what} goes with block 16 only"
    assert g.dtype == torch.float32 and g.numel() == mats and g.is_contiguous(), f"{what}: one fp32 number per matrix"


def quantize_fp4(x: torch.Tensor, block: int = 16, global_scale: torch.Tensor = None):
    """``x[rows, cols]`` or ``x[mats, rows, cols]`` (fp16, bf16 or fp32; any strides with adjacent elements in a row)
    -> ``(q[..., cols/2] uint8, scale[..., cols/block], global_scale)``.

    ``block=16``: ``global_scale`` (fp32, one per matrix) is computed from the largest magnitude, or taken from the
    caller (a calibrated positive value: one pass over ``x`` less) and returned as given.  ``block=32`` has none (``None``).
    A block holding an infinity or a NaN gets a NaN scale; such blocks do not enter the computed ``global_scale``.
    """
    _lib.require_cuda(x, global_scale)
    assert block in _SCALE_DTYPE, "block is 16 or 32"
    shape, dev = x.shape, x.device
    dims = len(shape)
    assert dims == 2 or dims == 3, "x is [rows, cols] or [mats, rows, cols]"
    rows, cols = shape[-2], shape[-1]
    mats = shape[0] if dims == 3 else 1
    strides = x.stride()
    assert cols > 0 and cols % block == 0, f"the row length must be a multiple of {block}"
    assert strides[-1] == 1, "the elements of a row must be adjacent"
    assert block == 16 or global_scale is None, "block 32 has no global scale"
    if global_scale is not None:
        check_global(global_scale, mats, block)
        _lib.require_device(dev, global_scale)
    if _lib.elsewhere(dev):
        with torch.cuda.device(dev):
            return quantize_fp4(x, block, global_scale)
    lead = shape[:-1]
    q = torch.empty((*lead, cols // 2), dtype=torch.uint8, device=dev)
    scale = torch.empty((*lead, cols // block), dtype=_SCALE_DTYPE[block], device=dev)
    own = block == 16 and global_scale is None
    if own:
        global_scale = (torch.empty if rows else torch.ones)(mats, dtype=torch.float32, device=dev)
    if mats == 0 or rows == 0:
        return q, scale, global_scale
    lib = _lib.load()
    ws, nbytes = None, 0
    if own and rows * cols > _SMALL:        # two launches: memory of this call's own, held until both are enqueued
        nbytes = lib.fr_fp4_quantize_workspace_bytes(mats, rows, cols)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    rc = lib.fr_fp4_quantize(x.data_ptr(), _lib.dtype_code(x.dtype), mats, rows, cols, strides[0] if dims == 3 else 0,
                             strides[-2] if rows > 1 else cols, block,
                             None if global_scale is None else global_scale.data_ptr(), 1 if own else 0, q.data_ptr(),
                             scale.data_ptr(), _lib.ptr(ws), nbytes, _lib.stream_ptr(dev))
    if rc:
        _lib.check(rc, "fr_fp4_quantize")
    return q, scale, global_scale


def dequantize_fp4(q: torch.Tensor, scale: torch.Tensor, global_scale: torch.Tensor = None,
                   dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The numbers that codes and scales stand for, in ``dtype`` (fp16, bf16 or fp32).  Block 16: scale * global is rounded to
    fp32, then code times that, then the result to ``dtype``."""
    _lib.require_cuda(q, scale, global_scale)
    shape, dev = q.shape, q.device
    dims = len(shape)
    assert dims == 2 or dims == 3, "codes are [rows, cols/2] or [mats, rows, cols/2]"
    block = block_of(q, scale)
    rows, cols = shape[-2], shape[-1] * 2
    mats = shape[0] if dims == 3 else 1
    _lib.require_device(dev, scale)
    if global_scale is not None:
        check_global(global_scale, mats, block)
        _lib.require_device(dev, global_scale)
    code = _lib.dtype_code(dtype)
    if _lib.elsewhere(dev):
        with torch.cuda.device(dev):
            return dequantize_fp4(q, scale, global_scale, dtype)
    out = torch.empty((*shape[:-1], cols), dtype=dtype, device=dev)
    if mats * rows * cols == 0:
        return out
    rc = _lib.load().fr_fp4_dequantize(q.data_ptr(), scale.data_ptr(), None if global_scale is None else global_scale.data_ptr(),
                                       mats, rows, cols, block, code, out.data_ptr(), _lib.stream_ptr(dev))
    if rc:
        _lib.check(rc, "fr_fp4_dequantize")
    return out


def matmul_fp4(a_q: torch.Tensor, a_scale: torch.Tensor, b_q: torch.Tensor, b_scale: torch.Tensor,
               a_global: torch.Tensor = None, b_global: torch.Tensor = None, dtype: torch.dtype = torch.bfloat16,
               out: torch.Tensor = None) -> torch.Tensor:
    """``c[m,n] = a[m,k] . b[n,k]^T`` of two quantised matrices of the same block size (``k`` a multiple of 32) on the
    block-scaled tensor-core instructions: sums in fp32, times the product of the global scales (two fp32 roundings), then
    rounded to ``dtype`` (fp16 or bf16).  ``out`` (of either type; ``dtype`` is then not looked at) may have any row pitch."""
    _lib.require_cuda(a_q, a_scale, b_q, b_scale, a_global, b_global, out)
    assert a_q.dim() == 2 and b_q.dim() == 2, "codes are [rows, k/2]"
    block = block_of(a_q, a_scale, "a_scale")
    assert block_of(b_q, b_scale, "b_scale") == block, "both matrices take the same block size"
    m, n, k = a_q.shape[0], b_q.shape[0], a_q.shape[1] * 2
    assert b_q.shape[1] * 2 == k, "Incompatible dimensions"
    assert k > 0 and k % 32 == 0, "k must be a multiple of 32"
    if a_global is not None:
        check_global(a_global, 1, block, "a_global")
    if b_global is not None:
        check_global(b_global, 1, block, "b_global")
    dev = a_q.device
    _lib.require_device(dev, a_scale, b_q, b_scale, a_global, b_global, out)
    if out is not None:
        assert out.shape == (m, n) and out.dtype in (torch.float16, torch.bfloat16), "out is [m, n] in fp16 or bf16"
        assert out.stride(1) == 1 or n == 1, "the elements of a row of out must be adjacent"
        assert m <= 1 or out.stride(0) >= n, "rows of out must not overlap"
    if _lib.elsewhere(dev):
        with torch.cuda.device(dev):
            return matmul_fp4(a_q, a_scale, b_q, b_scale, a_global, b_global, dtype, out)
    if out is None:
        assert dtype in (torch.float16, torch.bfloat16), f"unsupported dtype {dtype}"
        out = torch.empty((m, n), dtype=dtype, device=dev)
    if m == 0 or n == 0:
        return out
    lib = _lib.load()
    ws, nbytes = None, 0
    if m > 128:                 # the scales are laid out first: memory of this call's own, held until both are enqueued
        nbytes = lib.fr_fp4_gemm_workspace_bytes(m, n, k, block)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    rc = lib.fr_fp4_gemm(a_q.data_ptr(), a_scale.data_ptr(), _lib.ptr(a_global), b_q.data_ptr(), b_scale.data_ptr(),
                         _lib.ptr(b_global), block, m, n, k, _lib.dtype_code(out.dtype), out.data_ptr(),
                         out.stride(0) if m > 1 else n, _lib.ptr(ws), nbytes, _lib.stream_ptr(dev))
    if rc:
        _lib.check(rc, "fr_fp4_gemm")
    return out


__all__ = ["quantize_fp4", "dequantize_fp4", "matmul_fp4"]
