"""The MoE layer for a handful of tokens (single-token generation): one cooperative kernel for the whole layer.

``fused_moe_decode`` has the contract of ``fused_moe``; ``fused_moe_decode_fp4`` takes experts in the 4-bit format of
``ops/fp4.py`` and keeps the activations in 16 bits.  ``quantize_experts_fp4`` makes such experts.
"""

from __future__ import annotations

import torch

from .. import _lib
from ..ops.fp4 import block_of, check_global, quantize_fp4

MAX_TOKENS = 16


def _run(hidden_states, gate, w1, w2, dims, topk, renormalize, inplace, return_routing, block=0, s1=None, g1=None, s2=None,
         g2=None):
    M, H, I, E = dims
    assert 0 < topk <= E
    assert E <= 256, f"{E} experts: at most 256 are supported"
    assert M <= MAX_TOKENS, f"{M} tokens: at most {MAX_TOKENS}; use fused_moe for larger batches"
    dev = hidden_states.device
    _lib.require_device(dev, gate, w1, w2, s1, g1, s2, g2)
    if _lib.elsewhere(dev):
        with torch.cuda.device(dev):
            return _run(hidden_states, gate, w1, w2, dims, topk, renormalize, inplace, return_routing, block, s1, g1, s2, g2)
    out = hidden_states if inplace else torch.empty_like(hidden_states)
    tw = ti = None
    if return_routing:
        tw = torch.empty((M, topk), dtype=torch.float32, device=dev)
        ti = torch.empty((M, topk), dtype=torch.int32, device=dev)
    if M == 0:
        return (out, tw, ti) if return_routing else out
    lib = _lib.load()
    nbytes = lib.fr_moe_decode_workspace_bytes(M, H, I, E, topk)
    ws = _lib.call_workspace(nbytes, dev, "decode", lib.fr_moe_decode_state_bytes)
    rc = lib.fr_moe_decode(hidden_states.data_ptr(), gate.data_ptr(), gate.stride(0), gate.stride(1), w1.data_ptr(),
                           _lib.ptr(s1), _lib.ptr(g1), w2.data_ptr(), _lib.ptr(s2), _lib.ptr(g2),
                           _lib.dtype_code(hidden_states.dtype), block, M, H, I, E, topk, 1 if renormalize else 0,
                           out.data_ptr(), _lib.ptr(tw), _lib.ptr(ti), ws.data_ptr(), nbytes, _lib.stream_ptr(dev))
    if rc:
        _lib.check(rc, "fr_moe_decode")
    return (out, tw, ti) if return_routing else out


def fused_moe_decode(hidden_states: torch.Tensor, gate: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor, topk: int,
                     renormalize: bool = True, inplace: bool = False, return_routing: bool = False):
    """``fused_moe`` for at most 16 tokens in one kernel: same arguments, layouts and tie rule.  The activations between the
    two products are rounded to the input type, as there, and the output once (``fused_moe`` may also round every expert's
    share); the order of summation is another.  Faster than ``fused_moe`` up to 8 tokens, level with it for 9 to 16
    tokens of few large experts."""
    assert hidden_states.dim() == 2 and gate.dim() == 2 and w1.dim() == 3 and w2.dim() == 3
    assert hidden_states.shape[1] == w1.shape[2], "Incompatible dimensions"
    assert hidden_states.is_contiguous(), "Hidden_states must be contiguous"
    assert w1.is_contiguous(), "Expert weights1 must be contiguous"
    assert w2.is_contiguous(), "Expert weights2 must be contiguous"
    assert hidden_states.dtype in [torch.float16, torch.bfloat16]
    assert w1.dtype == hidden_states.dtype and w2.dtype == hidden_states.dtype and gate.dtype == hidden_states.dtype
    _lib.require_cuda(hidden_states, gate, w1, w2)
    M, H = hidden_states.shape
    E, N, _ = w1.shape
    I = N // 2
    assert N == 2 * I and w2.shape == (E, H, I) and gate.shape == (H, E)
    return _run(hidden_states, gate, w1, w2, (M, H, I, E), topk, renormalize, inplace, return_routing)


def fused_moe_decode_fp4(hidden_states: torch.Tensor, gate: torch.Tensor, w1_q: torch.Tensor, w1_scale: torch.Tensor,
                         w2_q: torch.Tensor, w2_scale: torch.Tensor, topk: int, w1_global: torch.Tensor = None,
                         w2_global: torch.Tensor = None, renormalize: bool = True, inplace: bool = False,
                         return_routing: bool = False):
    """The same with 4-bit experts: ``w1_q[E,2I,H/2]``, ``w2_q[E,H,I/2]`` and their block scales as ``quantize_fp4`` returns
    them for ``w1[E,2I,H]`` / ``w2[E,H,I]``; ``w1_global`` / ``w2_global`` hold one fp32 scale per expert (block 16;
    ``None`` = 1).  The expanded weights are exact 16-bit numbers.  Block 32 (E8M0) needs bf16 activations; block scales
    above 2^6 (weights of 512 and more) are right but slow, and weights of 2^128 and more are infinite, as
    ``dequantize_fp4`` gives them.  ``H`` and ``I`` are multiples of 32."""
    assert hidden_states.dim() == 2 and gate.dim() == 2 and w1_q.dim() == 3 and w2_q.dim() == 3
    assert hidden_states.is_contiguous(), "Hidden_states must be contiguous"
    assert hidden_states.dtype in [torch.float16, torch.bfloat16] and gate.dtype == hidden_states.dtype
    _lib.require_cuda(hidden_states, gate, w1_q, w1_scale, w2_q, w2_scale, w1_global, w2_global)
    block = block_of(w1_q, w1_scale, "w1_scale")
    assert block_of(w2_q, w2_scale, "w2_scale") == block, "both products take the same block size"
    M, H = hidden_states.shape
    E, N, _ = w1_q.shape
    I = N // 2
    assert w1_q.shape == (E, 2 * I, H // 2) and w2_q.shape == (E, H, I // 2) and gate.shape == (H, E), "Incompatible dimensions"
    assert H % 32 == 0 and I % 32 == 0, "4-bit experts need H and I to be multiples of 32"
    assert block == 16 or hidden_states.dtype == torch.bfloat16, "E8M0 block scales need bf16 activations"
    check_global(w1_global, E, block, "w1_global")
    check_global(w2_global, E, block, "w2_global")
    return _run(hidden_states, gate, w1_q, w2_q, (M, H, I, E), topk, renormalize, inplace, return_routing, block, w1_scale,
                w1_global, w2_scale, w2_global)


def quantize_experts_fp4(w1: torch.Tensor, w2: torch.Tensor, block: int = 16):
    """``(w1_q, w1_scale, w1_global, w2_q, w2_scale, w2_global)`` of ``w1[E,2I,H]`` and ``w2[E,H,I]`` for
    ``fused_moe_decode_fp4``: one global scale per expert (``None`` for block 32)."""
    assert w1.dim() == 3 and w2.dim() == 3 and w1.shape[0] == w2.shape[0]
    return (*quantize_fp4(w1, block), *quantize_fp4(w2, block))


__all__ = ["fused_moe_decode", "fused_moe_decode_fp4", "quantize_experts_fp4"]
