"""The norms before and after a block, fused with the block's gate and the residual sum, and their gradients.

    z, h = rms_norm(h0, w_in), h0                          # before the first block
    y = fused_moe(z, ...)                                  # the block
    h, z = block_norm(y, h, w_post, gate, w_pre)           # behind it, with the norm in front of the next one

No counterpart in the reference; the element-wise side of a layer, beside silu_and_mul and combine_topk. The work runs in the
HIP kernels behind include/moe_gg.h (csrc/block_norm.hip); torch only provides the buffers."""
from typing import Optional, Tuple

import torch

from . import _lib
from . import ops as _ops

_DTYPE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}  # MOE_GG_DTYPE_BF16 / _FP16 / _FP32
_NONE, _CHANNEL, _ROW = 0, 1, 2                                    # MOE_GG_GATE_*
_TYPES = (torch.bfloat16, torch.float16)


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _check(y, stream, post_weight, gate, pre_weight, extra=()):
    """(device, T, d, gate kind, weights' type) of a call on y (or None) and the residual stream, both [T, d]."""
    if stream.dim() != 2:
        raise ValueError("the residual stream must be [T, d]")
    T, d = shape = stream.shape
    tensors = [stream]
    if y is not None:
        dtype = y.dtype
        if y.shape != shape or dtype not in _TYPES:
            raise ValueError("the block's output must be bf16 or fp16 of the residual stream's shape")
        if stream.dtype != dtype and stream.dtype != torch.float32:
            raise ValueError("the residual stream must have the block output's type or be fp32")
        tensors.append(y)
    kind, wt = _NONE, None
    if gate is not None:
        kind = _CHANNEL if gate.shape == (d,) else _ROW if gate.shape == (T, 1) else -1
        if kind < 0:
            raise ValueError(f"the gate must be [{d}] (per channel) or [{T}, 1] (per row)")
        wt = gate.dtype
        tensors.append(gate)
        if not gate.is_contiguous():
            raise ValueError("the gate must be contiguous")
    for t in (post_weight, pre_weight):
        if t is not None:
            if t.shape != (d,) or not t.is_contiguous():
                raise ValueError(f"a norm's weight must be contiguous [{d}]")
            if wt is not None and t.dtype != wt:
                raise ValueError("the norms' weights and the gate must be of one type")
            wt = t.dtype
            tensors.append(t)
    for t in extra:
        if t is not None:
            tensors.append(t)
    return _ops._require_cuda(*tensors), T, d, kind, wt


def block_norm(y: torch.Tensor, residual: torch.Tensor, post_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
               pre_weight: Optional[torch.Tensor] = None, residual_scale: float = 1.0, block_scale: float = 1.0,
               eps: float = 1e-6) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(h, z) behind a block with output y [T, d] and the residual stream in front of it:

        h = residual_scale * residual + block_scale * gate * rms(y) * post_weight       (no post_weight: y as it is)
        z = rms(h) * pre_weight                                                         (no pre_weight: None)

    rms(v) = v / sqrt(mean(v^2) + eps). y bf16 or fp16; residual and h in y's type or fp32; gate [d] or [T, 1]; weights and gate
    in y's type or fp32, all alike; z in y's type. z is computed from h before its rounding. d <= 16384."""
    dev, T, d, kind, wt = _check(y, residual, post_weight, gate, pre_weight)
    dtype = y.dtype
    if wt is not None and wt != dtype and wt != torch.float32:
        raise ValueError("weights and gate must have the block output's type or be fp32")
    (y, ldy), (residual, ldr) = _ops._row_major(y), _ops._row_major(residual)
    h = _ops._empty_like(residual)
    z = _ops._empty_like(y) if pre_weight is not None else None
    with _ops._on_device(dev):
        rc = _lib.lib().moe_gg_block_norm(y.data_ptr(), ldy, residual.data_ptr(), ldr, _ptr(post_weight), _ptr(gate), kind, _ptr(pre_weight),
                                          residual_scale, block_scale, eps, h.data_ptr(), _ptr(z), T, d, _DTYPE[dtype], _DTYPE[residual.dtype],
                                          _DTYPE[wt or dtype], _ops._stream_ptr(dev))
    if rc:
        _lib.check(rc, "moe_gg_block_norm")
    return h, z


def block_norm_backward(grad_h: Optional[torch.Tensor], grad_z: Optional[torch.Tensor], y: torch.Tensor, h: torch.Tensor,
                        post_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                        pre_weight: Optional[torch.Tensor] = None, residual_scale: float = 1.0, block_scale: float = 1.0, eps: float = 1e-6):
    """Gradients of block_norm: (grad_y, grad_residual, grad_post_weight, grad_gate, grad_pre_weight), None for what was not
    given. y and the arguments behind it are block_norm's, h its first result; grad_h (None: zeros) and grad_z (needed with
    pre_weight) are the gradients of its results, in their types. Gradients have the types of what they belong to."""
    return _backward(grad_h, grad_z, y, h, post_weight, gate, pre_weight, residual_scale, block_scale, eps)


def _backward(grad_h, grad_z, y, h, post_weight, gate, pre_weight, residual_scale, block_scale, eps):
    dev, T, d, kind, wt = _check(y, h, post_weight, gate, pre_weight, (grad_h, grad_z))
    if (pre_weight is None) != (grad_z is None):
        raise ValueError("grad_z goes with pre_weight: give both or neither")
    dtype = y.dtype if y is not None else grad_z.dtype
    if dtype not in _TYPES or h.dtype not in (dtype, torch.float32):
        raise ValueError("rows must be bf16 or fp16, the residual stream in that type or fp32")
    if wt is not None and wt not in (dtype, torch.float32):
        raise ValueError("weights and gate must have the block output's type or be fp32")
    if grad_z is not None and (grad_z.shape != h.shape or grad_z.dtype != dtype):
        raise ValueError(f"grad_z must be {dtype} {tuple(h.shape)}")
    if grad_h is not None and (grad_h.shape != h.shape or grad_h.dtype != h.dtype):
        raise ValueError(f"grad_h must be {h.dtype} {tuple(h.shape)}")
    (y, ldy), (h, ldh), (grad_h, ldgh), (grad_z, ldgz) = ((None, 0) if t is None else _ops._row_major(t) for t in (y, h, grad_h, grad_z))
    grad_y = None if y is None else _ops._empty_like(y)
    grad_residual = _ops._empty_like(h)
    grad_post, grad_gate, grad_pre = (None if t is None else torch.empty_like(t) for t in (post_weight, gate, pre_weight))
    lib = _lib.lib()
    nbytes = lib.moe_gg_block_norm_backward_workspace(T, d)
    with _ops._on_device(dev):
        workspace = h.new_empty((max(nbytes, 256),), dtype=torch.uint8)
        rc = lib.moe_gg_block_norm_backward(_ptr(grad_h), ldgh, _ptr(grad_z), ldgz, _ptr(y), ldy, h.data_ptr(), ldh, _ptr(post_weight), _ptr(gate), kind,
                                            _ptr(pre_weight), residual_scale, block_scale, eps, _ptr(grad_y), grad_residual.data_ptr(),
                                            _ptr(grad_post), _ptr(grad_gate), _ptr(grad_pre), T, d, _DTYPE[dtype], _DTYPE[h.dtype],
                                            _DTYPE[wt or dtype], workspace.data_ptr(), workspace.numel(), _ops._stream_ptr(dev))
    if rc:
        _lib.check(rc, "moe_gg_block_norm_backward")
    return grad_y, grad_residual, grad_post, grad_gate, grad_pre


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x / sqrt(mean(x^2) + eps) * weight: the norm in front of a block on its own. x [T, d] bf16, fp16 or fp32; weight [d] in
    the result's type or fp32. The result has x's type, or dtype (bf16 or fp16, needed for fp32 x)."""
    dtype = dtype or x.dtype
    dev, T, d, _, wt = _check(None, x, None, None, weight)
    if dtype not in (torch.bfloat16, torch.float16) or x.dtype not in (dtype, torch.float32):
        raise ValueError("the result must be bf16 or fp16, x of that type or fp32")
    if wt not in (dtype, torch.float32):
        raise ValueError("the weight must have the result's type or be fp32")
    x, ldx = _ops._row_major(x)
    z = x.new_empty((T, d), dtype=dtype)
    with _ops._on_device(dev):
        rc = _lib.lib().moe_gg_block_norm(None, 0, x.data_ptr(), ldx, None, None, _NONE, weight.data_ptr(), 1.0, 1.0, eps, None, z.data_ptr(), T, d,
                                          _DTYPE[dtype], _DTYPE[x.dtype], _DTYPE[wt], _ops._stream_ptr(dev))
    if rc:
        _lib.check(rc, "moe_gg_block_norm")
    return z


def rms_norm_backward(grad_z: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
                      grad_x: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Gradients of rms_norm: (grad_x, grad_weight). grad_x, if given, is another part of x's gradient (the residual's, in
    x's type) that is added."""
    out = _backward(grad_x, grad_z, None, x, None, None, weight, 1.0, 1.0, eps)
    return out[1], out[4]
