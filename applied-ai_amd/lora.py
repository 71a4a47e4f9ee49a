"""Low-rank adapters of many requests at once beside a shared projection, and their gradients.

A batch whose rows belong to different fine-tuned variants of one model runs the shared projections once (grouped_gemm,
matmul_split_k, a library GEMM) and adds every row's own correction to the result:

    plan = lora_plan(adapter_ids, num_adapters)         # once per batch, for all projections
    y = ...                                             # the shared projection of x
    y = lora_add(y, x, a, b, plan, scales, out=y)

No counterpart in the reference; products grouped by an id per row, like its grouped GEMM. The work runs in the HIP kernels
behind include/moe_gg.h (csrc/lora.hip); torch only provides the buffers. The plan stays on the device: nothing synchronises, and
every call can be captured into a graph."""
from typing import NamedTuple, Optional

import torch

from . import _lib
from . import ops as _ops


_TYPES = (torch.bfloat16, torch.float16)


class LoraPlan(NamedTuple):
    """The rows of a batch grouped by adapter: perm [T] int32 holds the rows of adapter 0, 1, ... in their order and then
    the rows without an adapter, offsets [L + 2] int32 where each group begins (the last entry is T)."""
    perm: torch.Tensor
    offsets: torch.Tensor


def lora_plan(adapter_ids: torch.Tensor, num_adapters: int) -> LoraPlan:
    """Groups the rows of a batch by adapter_ids [T] int32; an id outside [0, num_adapters) means no adapter."""
    if adapter_ids.dim() != 1 or adapter_ids.dtype != torch.int32:
        raise ValueError("adapter_ids must be int32 [T]")
    if num_adapters < 0:
        raise ValueError("num_adapters must not be negative")
    dev = _ops._require_cuda(adapter_ids)
    ids = adapter_ids.contiguous()
    T = ids.shape[0]
    perm = torch.empty((T,), dtype=torch.int32, device=dev)
    offsets = torch.empty((num_adapters + 2,), dtype=torch.int32, device=dev)
    scratch = torch.empty((T + num_adapters + 1,), dtype=torch.int32, device=dev)
    with _ops._on_device(dev):
        rc = _lib.lib().moe_gg_lora_plan(ids.data_ptr(), T, num_adapters, perm.data_ptr(), offsets.data_ptr(), scratch.data_ptr(), _ops._stream_ptr(dev))
    _lib.check(rc, "moe_gg_lora_plan")
    return LoraPlan(perm, offsets)


def _check(rows: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, plan: LoraPlan, scales: Optional[torch.Tensor], what: str):
    """(device, L, T, K, N, R) of a call whose [T, N] operand is `rows`."""
    if x.dim() != 2 or rows.dim() != 2 or a.dim() != 3 or b.dim() != 3:
        raise ValueError(f"{what} and x must be [T, N] and [T, K], a [L, R, K], b [L, N, R]")
    T, K = x.shape
    L, R, k = a.shape
    l, N, r = b.shape
    if k != K or l != L or r != R or rows.shape != (T, N):
        raise ValueError(f"shapes do not match: {what} {tuple(rows.shape)}, x {tuple(x.shape)}, a {tuple(a.shape)}, b {tuple(b.shape)}")
    dtype = x.dtype
    if dtype not in _TYPES or rows.dtype != dtype or a.dtype != dtype or b.dtype != dtype:
        raise ValueError(f"{what}, x, a and b must all be bf16 or all be fp16")
    perm, offsets = plan
    if perm.shape != (T,) or offsets.shape != (L + 2,) or perm.dtype != torch.int32 or offsets.dtype != torch.int32:
        raise ValueError(f"the plan is not one of {T} rows and {L} adapters")
    if not (a.is_contiguous() and b.is_contiguous() and perm.is_contiguous() and offsets.is_contiguous()):
        raise ValueError("a, b and the plan must be contiguous")
    if scales is None:
        return _ops._require_cuda(rows, x, a, b, perm, offsets), L, T, K, N, R
    if scales.shape != (L,) or scales.dtype != torch.float32 or not scales.is_contiguous():
        raise ValueError(f"scales must be contiguous fp32 [{L}]")
    return _ops._require_cuda(rows, x, a, b, perm, offsets, scales), L, T, K, N, R


def _result(out: Optional[torch.Tensor], like: torch.Tensor, name: str):
    """(out or a new tensor like `like`, its elements from row to row)."""
    if out is None:
        return _ops._empty_like(like), like.shape[1]
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device or _ops._row_major(out)[0] is not out:
        raise ValueError(f"{name} must be a row-major tensor of shape {tuple(like.shape)} and {like.dtype} on the inputs' device")
    return out, _ops._row_major(out)[1]


def _disjoint(out: torch.Tensor, ld: int, others, name: str) -> None:
    """others: (tensor or None, bytes from its first element to behind its last one), none of which may share memory with out."""
    lo = out.data_ptr()
    hi = lo + 2 * ((out.shape[0] - 1) * ld + out.shape[1])
    for t, n in others:
        if t is not None:
            p = t.data_ptr()
            if p < hi and lo < p + n and _ops._overlap(out, t):
                raise ValueError(f"{name} shares memory with an input that other rows of it are computed from")


def lora_add(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, plan: LoraPlan, scales: Optional[torch.Tensor] = None,
             out: Optional[torch.Tensor] = None, return_h: bool = False):
    """out[t] = y[t] + scales[e] * b[e] @ (a[e] @ x[t]) with e the row's adapter; rows without one get y[t].

    y [T, N], x [T, K] (rows may lie apart), a [L, R, K], b [L, N, R], all bf16 or all fp16, R <= 128; scales fp32 [L] (default 1).
    out may be y itself, but must not share memory with another part of y or with another argument. return_h=True returns
    (out, h) with h = a[e] @ x[t] in fp32 [T, R] (zeros without an adapter), which lora_backward takes. fp32 accumulation, one
    rounding of the result."""
    dev, L, T, K, N, R = _check(y, x, a, b, plan, scales, "y")
    x, ldx = _ops._row_major(x)
    given = out
    out, ldo = _result(out, y, "out")
    y, ldy = _ops._row_major(y)  # (y itself where out is y: out is row-major)
    if given is not None:
        same = out is y or (ldo == ldy and out.data_ptr() == y.data_ptr())
        _disjoint(out, ldo, ((None if same else y, 2 * T * ldy), (x, 2 * T * ldx), (a, 2 * L * R * K), (b, 2 * L * N * R), (scales, 4 * L), (plan.perm, 4 * T),
                             (plan.offsets, 4 * L + 8)), "out")
    h = x.new_empty((T, R), dtype=torch.float32) if return_h else None
    lib = _lib.lib()
    nbytes = lib.moe_gg_lora_add_workspace(T, L, K, N, R)
    with _ops._on_device(dev):
        workspace = x.new_empty((nbytes,), dtype=torch.uint8) if nbytes else None
        rc = lib.moe_gg_lora_add(y.data_ptr(), ldy, x.data_ptr(), ldx, a.data_ptr(), b.data_ptr(), None if scales is None else scales.data_ptr(),
                                 plan.perm.data_ptr(), plan.offsets.data_ptr(), L, T, K, N, R, out.data_ptr(), ldo,
                                 h.data_ptr() if return_h else None, 1 if x.dtype == torch.float16 else 0, workspace.data_ptr() if nbytes else None,
                                 nbytes, _ops._stream_ptr(dev))
    if rc:
        _lib.check(rc, "moe_gg_lora_add")
    return (out, h) if return_h else out


def lora_backward(grad_out: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, plan: LoraPlan, scales: Optional[torch.Tensor] = None,
                  h: Optional[torch.Tensor] = None, grad_x: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None):
    """Gradients of lora_add: returns (grad_x [T, K], grad_a [L, R, K], grad_b [L, N, R]) in the tensors' type.

    grad_out [T, N] is the gradient of lora_add's result (and of y as it is). h is what the forward pass returned
    (return_h=True); without it a[e] @ x[t] is computed again. grad_x is the shared projection's part of x's gradient, to
    which the adapters' is added (default: none); out takes the sum and may be grad_x itself, but must not share memory with
    another part of grad_x, a, scales or the plan. An adapter without rows gets zeros. Sums over rows are taken in a fixed
    order."""
    dev, L, T, K, N, R = _check(grad_out, x, a, b, plan, scales, "grad_out")
    if h is not None and (h.shape != (T, R) or h.dtype != torch.float32 or not h.is_contiguous() or h.device != dev):
        raise ValueError(f"h must be contiguous fp32 [{T}, {R}] on the inputs' device")
    if grad_x is not None and (grad_x.shape != x.shape or grad_x.dtype != x.dtype or grad_x.device != dev):
        raise ValueError(f"grad_x must be a {x.dtype} tensor of shape {tuple(x.shape)} on the inputs' device")
    if T == 0:
        h = None
    given = out
    out, ldo = _result(out, x, "out")
    (x, ldx), (grad_out, ldg) = _ops._row_major(x), _ops._row_major(grad_out)
    grad_x, ld_in = (None, 0) if grad_x is None else _ops._row_major(grad_x)
    if given is not None:  # (x, grad_out, b and h have been read when out is written)
        same = grad_x is None or grad_x is out or (ldo == ld_in and out.data_ptr() == grad_x.data_ptr())
        _disjoint(out, ldo, ((None if same else grad_x, 2 * T * ld_in), (a, 2 * L * R * K), (scales, 4 * L), (plan.perm, 4 * T), (plan.offsets, 4 * L + 8)), "out")
    grad_a, grad_b = torch.empty_like(a), torch.empty_like(b)
    lib = _lib.lib()
    nbytes = lib.moe_gg_lora_backward_workspace(T, L, K, N, R, 0 if h is None else 1)
    with _ops._on_device(dev):
        workspace = x.new_empty((max(nbytes, 256),), dtype=torch.uint8)
        rc = lib.moe_gg_lora_backward(grad_out.data_ptr(), ldg, x.data_ptr(), ldx, a.data_ptr(), b.data_ptr(),
                                      None if scales is None else scales.data_ptr(), plan.perm.data_ptr(), plan.offsets.data_ptr(), L, T, K, N, R,
                                      None if h is None else h.data_ptr(), None if grad_x is None else grad_x.data_ptr(),
                                      ld_in, out.data_ptr(), ldo, grad_a.data_ptr(), grad_b.data_ptr(),
                                      1 if x.dtype == torch.float16 else 0, workspace.data_ptr(), workspace.numel(), _ops._stream_ptr(dev))
    if rc:
        _lib.check(rc, "moe_gg_lora_backward")
    return out, grad_a, grad_b
