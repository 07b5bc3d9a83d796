"""Matrix products grouped by adapter copy, with ragged rows (no reference counterpart).

A scoring batch holds the rollouts of perturbed copies one behind the other: rows sorted by copy,
a device vector of row offsets, and one factor matrix a copy (an AdapterSet's K + copies lie in one
arena and its K - copies in another: a call for each). ``grouped_matmul`` multiplies every group of rows by its own matrix, ``grouped_weight_grad``
forms the gradient of every matrix, and ``adapter_forward`` / ``adapter_backward`` combine them
to the rank-r product of an adapter and its gradients. One launch for all groups; bf16
operands, fp32 sums on the tensor cores. The same entry points serve any set of experts.

A kernel whose barriers do not complete within a limit (``set_wait_limit``, 1 s at first: a
preempted device, a defect) returns all the same: the parts of its output that it did not produce
are NaN, and ``device_error`` (or ``AdapterSet.device_error``) tells of it. Later calls run as usual.

Nothing here records an autograd graph. A forward product of tensors that require grad, with grad
mode on, is refused, since its result would silently drop out of the graph: call it under
``torch.no_grad()`` and take the gradients from ``grouped_matmul`` of the other layout and
``grouped_weight_grad``, for instance in the backward of a ``torch.autograd.Function``.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from ._lib import DSMZ_BF16, DSMZ_F32, GROUPED_ACCUMULATE, GROUPED_ZERO_REST, MAX_GROUPS, check, launch, lib

__all__ = ["grouped_matmul", "grouped_weight_grad", "adapter_forward", "adapter_backward", "device_error",
           "set_wait_limit"]

_DT = {torch.float32: DSMZ_F32, torch.bfloat16: DSMZ_BF16}


def _rows(t: torch.Tensor, what: str) -> torch.Tensor:
    """t (rows x width, bf16) as the kernels read it: unit column stride, 16-byte aligned rows.
    Any other layout is copied to one."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise ValueError(f"{what}: CUDA tensors only (no CPU fallback)")
    if t.dim() != 2 or t.dtype != torch.bfloat16:
        raise ValueError(f"{what}: operands are 2-D bfloat16 tensors")
    width = t.shape[1]
    if width < 1:
        raise ValueError(f"{what}: an operand has no columns")
    pitch, unit = t.stride()
    if unit == 1 and pitch % 8 == 0 and pitch >= width and t.data_ptr() % 16 == 0:
        return t
    return t.new_empty(t.shape[0], (width + 7) // 8 * 8)[:, :width].copy_(t)


def _weights(w: torch.Tensor, what: str) -> Tuple[torch.Tensor, int, int, int]:
    """(tensor, group stride, row pitch, whether N is the contiguous dimension) of w: G x K x N."""
    G, K, N = w.shape
    gs, sk, sn = w.stride()
    if (G == 1 or (gs % 8 == 0 and gs > 0)) and w.data_ptr() % 16 == 0:
        if sk == 1 and sn % 8 == 0 and sn >= K:
            return w, gs, sn, 0
        if sn == 1 and sk % 8 == 0 and sk >= N:
            return w, gs, sk, 1
    nc = 0 if sk < sn else 1                                       # keep the faster dimension
    inner = K if nc == 0 else N
    pad = (inner + 7) // 8 * 8
    c = w.new_empty(G, N if nc == 0 else K, pad)[:, :, :inner]
    c = c.transpose(1, 2) if nc == 0 else c
    return c.copy_(w), c.stride(0), pad, nc


def _offsets(row_offsets: torch.Tensor, G: int, device, what: str) -> torch.Tensor:
    if not 1 <= G <= MAX_GROUPS:
        raise ValueError(f"{what}: 1 to {MAX_GROUPS} groups")
    if row_offsets.dtype != torch.int32 or row_offsets.dim() != 1 or row_offsets.numel() != G + 1 or \
            row_offsets.device != device or not row_offsets.is_contiguous():
        raise ValueError(f"{what}: row_offsets must be a contiguous int32 vector of groups + 1 on the operands' device")
    return row_offsets


def grouped_matmul(x: torch.Tensor, w: torch.Tensor, row_offsets: torch.Tensor, *, out: Optional[torch.Tensor] = None,
                   out_dtype: torch.dtype = torch.bfloat16, alpha: float = 1.0, accumulate: bool = False) -> torch.Tensor:
    """y[i] = alpha * x[i] @ w[g] for every row i of group g, rows [row_offsets[g], row_offsets[g+1]).

    x: M x K bf16. w: G x K x N bf16 with either of its last two dimensions contiguous (a stack
    of nn.Linear weights as ``weight.transpose(1, 2)``; the same stack untransposed gives the
    input gradient). row_offsets: G + 1 int32 on the device, ascending; values beyond [0, M]
    or below an earlier one are clamped. out: M x N, bf16 or fp32, any row pitch; rows outside
    every group stay as they are. Without out a new tensor of ``out_dtype`` is returned whose
    rows outside every group are zero. accumulate: add to out (fp32 sum, rounded once). NaN
    where a wait of the kernel ran out of time: ``device_error`` tells."""
    me = "grouped_matmul"
    x = _rows(x, me)
    if not isinstance(w, torch.Tensor) or w.dim() != 3 or w.dtype != torch.bfloat16 or w.device != x.device:
        raise ValueError(f"{me}: w must be a G x K x N bfloat16 tensor on x's device")
    M, K = x.shape
    G, Kw, N = w.shape
    if Kw != K or N < 1:
        raise ValueError(f"{me}: x is M x K and w is G x K x N")
    row_offsets = _offsets(row_offsets, G, x.device, me)
    flags = GROUPED_ACCUMULATE if accumulate else 0
    if out is None:
        if accumulate:
            raise ValueError(f"{me}: accumulate needs out")
        if out_dtype not in _DT:
            raise TypeError(f"{me}: out_dtype must be float32 or bfloat16")
        out = torch.empty(M, N, dtype=out_dtype, device=x.device)
        flags |= GROUPED_ZERO_REST
    elif tuple(out.shape) != (M, N) or out.dtype not in _DT or out.device != x.device or \
            (N > 1 and out.stride(1) != 1) or (M > 1 and out.stride(0) < N):
        raise ValueError(f"{me}: out must be M x N float32 or bfloat16 with unit column stride, on x's device")
    if (x.requires_grad or w.requires_grad or out.requires_grad) and torch.is_grad_enabled():
        raise RuntimeError(f"{me} records no autograd graph: call it under torch.no_grad(), or in the forward of a "
                           "torch.autograd.Function whose backward calls grouped_matmul and grouped_weight_grad")
    if M == 0:
        return out
    w, gs, ld, nc = _weights(w, me)
    launch(me, x.device, lib().dsmz_grouped_matmul, x.data_ptr(), M, K, x.stride(0) if M > 1 else (K + 7) // 8 * 8,
           w.data_ptr(), G, N, gs, ld, nc, row_offsets.data_ptr(), _DT[out.dtype], out.data_ptr(),
           out.stride(0) if M > 1 else N, float(alpha), flags)
    return out


def grouped_weight_grad(x: torch.Tensor, dy: torch.Tensor, row_offsets: torch.Tensor, *,
                        out: Optional[torch.Tensor] = None, alpha: float = 1.0, accumulate: bool = False) -> torch.Tensor:
    """dw[g] = alpha * x[rows of g].T @ dy[rows of g]: the gradient of ``grouped_matmul`` in w.

    x: M x K and dy: M x N, bf16. out: G x K x N contiguous fp32 (new unless given); a group
    without rows gives zeros. accumulate: add to out. NaN where a wait of the kernel ran out of
    time: ``device_error`` tells."""
    me = "grouped_weight_grad"
    x, dy = _rows(x, me), _rows(dy, me)
    M, K = x.shape
    N = dy.shape[1]
    if dy.shape[0] != M or dy.device != x.device:
        raise ValueError(f"{me}: x is M x K and dy is M x N, on one device")
    G = row_offsets.numel() - 1
    row_offsets = _offsets(row_offsets, G, x.device, me)
    if out is None:
        if accumulate:
            raise ValueError(f"{me}: accumulate needs out")
        out = torch.empty(G, K, N, dtype=torch.float32, device=x.device)
    elif tuple(out.shape) != (G, K, N) or out.dtype != torch.float32 or out.device != x.device or not out.is_contiguous():
        raise ValueError(f"{me}: out must be a contiguous G x K x N float32 tensor on the operands' device")
    launch(me, x.device, lib().dsmz_grouped_weight_grad, x.data_ptr(), M, K, x.stride(0) if M > 1 else (K + 7) // 8 * 8,
           dy.data_ptr(), N, dy.stride(0) if M > 1 else (N + 7) // 8 * 8, G, row_offsets.data_ptr(), out.data_ptr(),
           float(alpha), GROUPED_ACCUMULATE if accumulate else 0)
    return out


def adapter_forward(x: torch.Tensor, A: torch.Tensor, B: torch.Tensor, row_offsets: torch.Tensor, *,
                    out: Optional[torch.Tensor] = None, alpha: float = 1.0,
                    accumulate: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """The adapters' share of a module's output: y[i] = alpha * (x[i] @ B[g].T) @ A[g].T.

    x: M x d_in; A: G x d_out x r and B: G x r x d_in (one copy a group), all bf16. Returns
    (y, t) with t = x @ B[g].T in bf16, which ``adapter_backward`` takes. out / accumulate: add
    the share to a base output in place. Rows outside every group as for ``grouped_matmul``."""
    t = grouped_matmul(x, B.transpose(1, 2), row_offsets)
    y = grouped_matmul(t, A.transpose(1, 2), row_offsets, out=out, alpha=alpha, accumulate=accumulate)
    return y, t


def adapter_backward(dy: torch.Tensor, x: torch.Tensor, t: torch.Tensor, A: torch.Tensor, B: torch.Tensor,
                     row_offsets: torch.Tensor, *, alpha: float = 1.0, dA: Optional[torch.Tensor] = None,
                     dB: Optional[torch.Tensor] = None, accumulate: bool = False, need_dx: bool = True):
    """Gradients of ``adapter_forward``: (dx, dA, dB) with dx bf16 (None without need_dx), dA
    G x d_out x r and dB G x r x d_in fp32 (into the tensors given; accumulate adds to them).
    The gradient in t is rounded to bf16, as t is."""
    dt = grouped_matmul(dy, A, row_offsets, alpha=alpha)
    dx = grouped_matmul(dt, B, row_offsets) if need_dx else None
    dA = grouped_weight_grad(dy, t, row_offsets, out=dA, alpha=alpha, accumulate=accumulate)
    dB = grouped_weight_grad(dt, x, row_offsets, out=dB, accumulate=accumulate)
    return dx, dA, dB


def device_error(device=None) -> int:
    """Reads and clears the device's error word of the grouped products (synchronises the
    current stream): nonzero when a kernel's barrier wait has run out of time since the last
    reading. Its output holds NaN where it was not produced."""
    with torch.cuda.device(device):
        return int(lib().dsmz_first_order_device_error(torch.cuda.current_stream().cuda_stream))


def set_wait_limit(seconds: float) -> None:
    """Limit of the barrier waits inside the grouped products, for the calls (and captures) that
    follow in this process: 0 to 60 s, 1 s at first. It counts wall time, so a device that other
    processes preempt for longer needs more. At 0 the kernels load nothing, so that their waits
    run out: how a program tries what it does about ``device_error``."""
    check(lib().dsmz_first_order_set_wait_limit(round(float(seconds) * 1e9)), "set_wait_limit")
