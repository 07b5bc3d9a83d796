"""AdamW over many tensors, up to 256 in one launch, with fp32 or 8-bit states (first-order
counterpart of the ZO-Muon update; the reference has none).

``AdamW`` binds a list of parameters, their states and optionally fixed gradient buffers, as a
plan binds an adapter set, and steps them all in one call (``dsmz_adamw_step``). An
``AdapterSet`` goes in as one flat arena (``AdamW.for_adapters``): fp32 masters updated in
place and the bf16 shadow that the rollout loads rewritten in the same pass, as the
zeroth-order update does.
"""
from __future__ import annotations

import bisect
import ctypes
from dataclasses import dataclass
from typing import Optional, Sequence

import numpy as np
import torch

from . import _lib
from ._lib import ADAMW_BLOCK, DSMZ_BF16, DSMZ_F32, AdamWDesc, AdamWTensor, lib

__all__ = ["AdamW", "AdamWState"]

_DT = {torch.float32: DSMZ_F32, torch.bfloat16: DSMZ_BF16}


@dataclass(frozen=True)
class AdamWState:
    """Mean and second moment of one parameter: fp32 tensors of its size, or int8 / uint8 codes
    with one fp32 scale for every 256 elements (m = sign q^2 scale, sqrt(v) = q^2 scale). The
    tensors stay: a saved state is copied into them."""
    m: torch.Tensor
    v: torch.Tensor
    m_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None

    @classmethod
    def zeros(cls, param: torch.Tensor, bits: int = 32) -> "AdamWState":
        """The state before the first step."""
        if bits == 32:
            return cls(*(torch.zeros(param.numel(), dtype=torch.float32, device=param.device) for _ in range(2)))
        if bits != 8:
            raise ValueError("AdamWState: bits must be 32 or 8")
        nb = -(-param.numel() // ADAMW_BLOCK)
        return cls(torch.zeros(param.numel(), dtype=torch.int8, device=param.device),
                   torch.zeros(param.numel(), dtype=torch.uint8, device=param.device),
                   *(torch.zeros(nb, dtype=torch.float32, device=param.device) for _ in range(2)))

    @property
    def bits(self) -> int:
        return 32 if self.m.dtype == torch.float32 else 8


def _addresses(tensors: Sequence[torch.Tensor]) -> list:
    return list(map(torch.Tensor.data_ptr, tensors))     # 60 ns a tensor


def _span(t: torch.Tensor):
    return t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()


class AdamW:
    """Steps ``params`` (contiguous CUDA tensors, all fp32 or all bf16, on one device).

    grads: gradient buffers bound once, or given to each ``step``; fp32 or bf16, one type.
    states: one ``AdamWState`` a parameter (default: zeros of ``state_bits`` bits).
    shadows: bf16 tensors that receive the updated fp32 parameters, rounded once (an entry may
    be None). step: steps already taken. capturable: keep the step count in a device counter,
    which a captured ``step`` advances at every replay; without it the count is the host's,
    and capturing a step is refused, since its replays would repeat one step number.

    The tensors are bound once (``params``, ``states``, ``shadows``, ``grads`` and
    ``step_counter`` are read-only; what they hold may be written). A step that finds the memory
    of one exchanged (``tensor.data = ...``) is refused: that of a parameter or gradient at once,
    that of a state or shadow when its turn comes (each step looks at sixteen of these; until
    then it works on the old memory, which stays allocated). A captured step cannot look.
    ``lr``, ``betas``, ``eps``,
    ``weight_decay`` and ``step_count`` may be set between steps.
    """

    def __init__(self, params: Sequence[torch.Tensor], lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, grads: Optional[Sequence[torch.Tensor]] = None,
                 states: Optional[Sequence[AdamWState]] = None, state_bits: int = 32,
                 shadows: Optional[Sequence[Optional[torch.Tensor]]] = None, step: int = 0, capturable: bool = False):
        self._params = tuple(params)
        if not self.params:
            raise ValueError("AdamW: no parameters")
        p0 = self.params[0]
        for p in self.params:
            if not (isinstance(p, torch.Tensor) and p.is_cuda):
                raise ValueError("AdamW takes CUDA tensors only (no CPU fallback)")
            if p.dtype not in _DT or p.dtype != p0.dtype or p.device != p0.device:
                raise ValueError("AdamW: parameters must be all float32 or all bfloat16, on one device")
            if not p.is_contiguous():
                raise ValueError("AdamW: parameters must be contiguous")
        b1, b2 = (float(b) for b in betas)
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and float(eps) >= 0.0 and float(weight_decay) >= 0.0):
            raise ValueError("AdamW: need 0 <= beta < 1, eps >= 0 and weight_decay >= 0")
        if int(step) < 0:
            raise ValueError("AdamW: step counts from 0")
        n = len(self.params)
        self._numels = [p.numel() for p in self.params]
        self.device, self.lr, self.betas = p0.device, float(lr), (b1, b2)
        self.eps, self.weight_decay = float(eps), float(weight_decay)
        self._states = tuple(AdamWState.zeros(p, state_bits) for p in self.params) if states is None else tuple(states)
        if len(self.states) != n:
            raise ValueError("AdamW: one state a parameter")
        self.state_bits = self.states[0].bits
        if self.state_bits == 8 and self.eps < 1e-12:
            raise ValueError("AdamW: 8-bit states need eps >= 1e-12")
        for p, s in zip(self.params, self.states):
            self._check_state(p, s)
        self._shadows = (None,) * n if shadows is None else tuple(shadows)
        if len(self.shadows) != n:
            raise ValueError("AdamW: one shadow (or None) a parameter")
        for p, s in zip(self.params, self.shadows):
            if s is not None and (p.dtype != torch.float32 or s.dtype != torch.bfloat16 or s.numel() != p.numel() or
                                  s.device != p.device or not s.is_contiguous()):
                raise ValueError("AdamW: a shadow is a contiguous bfloat16 tensor of its fp32 parameter's size")
        written = [_span(t) for p, s, sh in zip(self.params, self.states, self.shadows)
                   for t in (p, s.m, s.v, s.m_scale, s.v_scale, sh) if t is not None and t.numel() > 0]
        written.sort()
        if any(a[1] > b[0] for a, b in zip(written, written[1:])):
            raise ValueError("AdamW: parameters, states and shadows must not overlap")
        self._written, self._starts = written, [a for a, _ in written]
        self._table = (AdamWTensor * n)()
        for e, p, s, sh in zip(self._table, self.params, self.states, self.shadows):
            e.param, e.m, e.v, e.n = p.data_ptr(), s.m.data_ptr(), s.v.data_ptr(), p.numel()
            if self.state_bits == 8:
                e.m_scale, e.v_scale = s.m_scale.data_ptr(), s.v_scale.data_ptr()
            if sh is not None:
                e.shadow = sh.data_ptr()
        self._desc = AdamWDesc(param_dtype=_DT[p0.dtype], state_bits=self.state_bits)
        # what the table holds the addresses of: a tensor's memory may be exchanged under it
        self._pointers = _addresses(self.params)
        self._others = tuple(t for s, sh in zip(self.states, self.shadows)
                             for t in (s.m, s.v, s.m_scale, s.v_scale, sh) if t is not None)
        self._other_pointers, self._look = _addresses(self._others), 0
        self._kept = tuple(map(torch.Tensor.untyped_storage, self._others))
        self.step_count = int(step)              # steps taken (host count; not moved when capturable)
        self._counter = torch.full((1,), int(step), dtype=torch.int64, device=self.device) if capturable else None
        self._grads = None
        if grads is not None:
            self._grads = tuple(grads)
            self._check_grads(self._grads)
            self._put_grads(self._grads)
            self._grad_pointers = _addresses(self._grads)

    # The C table holds their addresses, so what they refer to is not exchanged.
    params = property(lambda self: self._params)
    states = property(lambda self: self._states)
    shadows = property(lambda self: self._shadows)
    grads = property(lambda self: self._grads)
    step_counter = property(lambda self: self._counter)

    @classmethod
    def for_adapters(cls, adapter_set, grad: torch.Tensor, **kw) -> "AdamW":
        """AdamW over an AdapterSet's fp32 masters as one flat tensor, rewriting its bf16 shadow;
        ``grad``: a flat gradient arena laid out as the masters (``AdapterSet.grad_arena()``)."""
        n = adapter_set.numel
        shadow = None if adapter_set.shadow is None else [adapter_set.shadow[:n]]
        return cls([adapter_set.factors[:n]], grads=[grad], shadows=shadow, **kw)

    def _check_state(self, p: torch.Tensor, s: AdamWState) -> None:
        n, nb = p.numel(), -(-p.numel() // ADAMW_BLOCK)
        if s.bits == 32:
            want = ((s.m, torch.float32, n), (s.v, torch.float32, n))
        else:
            want = ((s.m, torch.int8, n), (s.v, torch.uint8, n), (s.m_scale, torch.float32, nb),
                    (s.v_scale, torch.float32, nb))
        for t, dt, k in want:
            if t is None or t.dtype != dt or t.numel() != k or t.device != p.device or not t.is_contiguous():
                raise ValueError("AdamW: a state is fp32 (m, v) of the parameter's size, or int8 m and uint8 v codes "
                                 "with one fp32 scale each for every 256 elements; contiguous, on its device")
        if s.bits != self.state_bits:
            raise ValueError("AdamW: states must be all fp32 or all 8-bit")

    def _check_grads(self, grads: Sequence[torch.Tensor]) -> None:
        if len(grads) != len(self.params):
            raise ValueError("AdamW: one gradient a parameter")
        dt = grads[0].dtype
        for p, g in zip(self._params, grads):
            if g.dtype != dt or dt not in _DT or g.numel() != p.numel() or g.device != p.device or not g.is_contiguous():
                raise ValueError("AdamW: gradients must be contiguous, all float32 or all bfloat16, of their "
                                 "parameters' sizes and device")
            lo, hi = _span(g)
            k = bisect.bisect_left(self._starts, hi)       # the last written range that starts before g ends
            if lo < hi and k > 0 and self._written[k - 1][1] > lo:
                raise ValueError("AdamW: a gradient overlaps a parameter, state or shadow")

    def _put_grads(self, grads: Sequence[torch.Tensor]) -> None:
        """Into the C table."""
        for e, g in zip(self._table, grads):
            e.grad = g.data_ptr()
        self._desc.grad_dtype = _DT[grads[0].dtype]

    def _scalar(self, t: Optional[torch.Tensor], what: str) -> Optional[int]:
        if t is None:
            return None
        if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.numel() != 1 or t.device != self.device:
            raise ValueError(f"AdamW: {what} must be a one-element float32 tensor on the parameters' device")
        return t.data_ptr()

    def step(self, grads: Optional[Sequence[torch.Tensor]] = None, *, lr=None,
             grad_scale: Optional[torch.Tensor] = None) -> None:
        """One step on the current stream. lr: a float (default: the constructor's) or a
        one-element fp32 device tensor; grad_scale: one-element fp32 device tensor that
        multiplies every gradient (a clipping or loss-scale factor)."""
        if grads is not None:
            grads = tuple(grads)
            self._check_grads(grads)
        elif self._grads is None:
            raise ValueError("AdamW: no gradients bound; give them to step()")
        elif _addresses(self._grads) != self._grad_pointers:
            raise RuntimeError("AdamW: a gradient's memory has been replaced since it was bound")
        if _addresses(self._params) != self._pointers:
            raise RuntimeError("AdamW: a parameter's memory has been replaced since it was bound")
        a, b = self._look, self._look + 16       # all of them would double the host's time for many small tensors
        if _addresses(self._others[a:b]) != self._other_pointers[a:b]:
            raise RuntimeError("AdamW: the memory of a state or shadow has been replaced since it was bound")
        d = self._desc
        if self._counter is None and _lib.capturing(self.device):
            raise RuntimeError("AdamW: a captured step would repeat one step number at every replay; "
                               "construct with capturable=True")
        d.lr_device = self._scalar(lr, "lr") if isinstance(lr, torch.Tensor) else None
        d.lr = self.lr if lr is None or d.lr_device else float(lr)
        d.grad_scale = self._scalar(grad_scale, "grad_scale")
        d.beta1, d.beta2 = self.betas
        d.eps, d.weight_decay = self.eps, self.weight_decay
        d.step = self.step_count + 1
        d.step_counter = None if self._counter is None else self._counter.data_ptr()
        ws, nbytes = None, 0
        if d.step_counter or d.lr_device:
            ws = torch.empty(_lib.ADAMW_WORKSPACE_BYTES, dtype=torch.uint8, device=self.device)
            nbytes = ws.numel()
        if grads is not None:
            self._put_grads(grads)
        try:
            _lib.launch("adamw_step", self.device, lib().dsmz_adamw_step, ctypes.byref(d), self._table,
                        len(self.params), None if ws is None else ws.data_ptr(), nbytes)
        except BaseException:
            if grads is not None and self._grads is not None:
                self._put_grads(self._grads)     # a refused step changes nothing
            raise
        self._look = b if b < len(self._others) else 0
        if grads is not None:
            self._grads = None                   # a later step() must be given its own again
        if self._counter is None:
            self.step_count += 1

    def state_values(self, m_out: Sequence[torch.Tensor], v_out: Sequence[torch.Tensor]) -> None:
        """Writes the fp32 values of 8-bit states (a checkpoint in plain fp32, a diagnostic) to
        tensors apart from the optimizer's own."""
        if self.state_bits != 8:
            raise ValueError("AdamW: fp32 states are their own values")
        n = len(self.params)
        if len(m_out) != n or len(v_out) != n:
            raise ValueError("AdamW: one output a parameter")
        at, T = [self.device.index] * n, torch.Tensor
        for outs in (m_out, v_out):
            if list(map(T.numel, outs)) != self._numels or list(map(T.get_device, outs)) != at or \
                    {t.dtype for t in outs} != {torch.float32} or not all(map(T.is_contiguous, outs)):
                raise ValueError("AdamW: state values go to contiguous float32 tensors of the parameters' sizes")
        table = type(self._table).from_buffer_copy(self._table)
        words = np.frombuffer(table, dtype=np.int64).reshape(n, -1)       # rows of 64-bit words: no loop over tensors
        words[:, AdamWTensor.param.offset // 8] = [t.data_ptr() for t in m_out]
        words[:, AdamWTensor.shadow.offset // 8] = [t.data_ptr() for t in v_out]
        _lib.launch("adamw_state_values", self.device, lib().dsmz_adamw_state_values, table, n)
