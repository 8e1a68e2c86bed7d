"""Fused Adam for the Gaussian parameters (include/gsr_optim.h).

`FusedAdam` is a drop-in for the optimizer GaussianModel.training_setup creates
(`torch.optim.Adam(param_groups, lr=0.0, eps=1e-15)`, scene/gaussian_model.py:217-271): it IS a
torch.optim.Adam (same constructor, param groups, state dict with exp_avg / exp_avg_sq / step), so
the reference's learning-rate schedule (`update_learning_rate`, :277) and its densification code,
which edits `optimizer.state` and `group["params"]` directly (:400-470), work unchanged.  Only
`step()` differs: every tensor of every group is updated by ONE HIP launch (one streaming pass,
28 B per element) instead of PyTorch's per-group foreach passes.  There is no CPU path.

Failed forwards (include/gsr_optim.h): the step is skipped ON THE DEVICE when the step's guard
slot is set -- the device's forward fault word snapshot, or, with a multi-GPU reducer, that
snapshot summed over the ranks (``step(skip=reducer.skip_flag())``), so every rank skips together
when any rank's forward failed.  The launch also reports the decision into a pinned host word; the
next step() reads it (no synchronisation in the normal case) and, for a skipped step, takes back
the step counts it had advanced (state["step"]: a skipped step leaves parameters, moments AND
counts as they were) and raises, unless reset_forward_faults() ran since the skipped step -- a
caller that swallows one error does not silently stall.

Gradient clipping: `grad_norm` and `clip_grad_norm_` (torch.nn.utils' total norm and in-place
scaling, one streaming pass each over any number of tensors of mixed types), and
``FusedAdam(..., max_grad_norm=)``, which applies the same factor inside the Adam launch.
"""
from __future__ import annotations

import ctypes
import math
import operator

import torch

from . import _lib

MAX_TENSORS = 16  # GSR_ADAM_MAX_TENSORS

_NORMS = {math.inf: 0, 1.0: 1, 2.0: 2}  # GSR_NORM_INF / 1 / 2
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # GSR_F32 / F16 / BF16
_SIZES = {torch.float32: 4, torch.float16: 2, torch.bfloat16: 2}


def _dense(t):
    """Whether t's elements fill its memory without gaps or repeats, in any order of dimensions
    (then the kernels take them in the order they lie)."""
    if t.is_contiguous():
        return True
    want = 1
    for size, stride in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n != 1),
                               key=lambda d: d[1]):
        if stride != want:
            return False
        want *= size
    return True


def _without_gaps(t):
    if t.layout is not torch.strided:
        raise RuntimeError("gradient norm: sparse gradients are not supported")
    return t if _dense(t) else t.contiguous()


def _norm_code(norm_type):
    if isinstance(norm_type, str) or float(norm_type) not in _NORMS:
        raise ValueError(f"norm_type must be 1, 2 or inf, not {norm_type!r}")
    return _NORMS[float(norm_type)]


def _limit(max_norm, name):
    max_norm = float(max_norm)
    if not max_norm >= 0.0:  # NaN is refused too
        raise ValueError(f"{name} must be at least 0, not {max_norm}")
    return max_norm


class _CTensors:
    """The tensors that hold elements, checked, as the C entries take them; one with gaps between
    its elements as a copy.  (Each attribute of each tensor is asked for once: a head has many.)"""

    def __init__(self, tensors):
        kinds = [t.dtype for t in tensors]
        for kind in set(kinds):
            if kind not in _DTYPES:
                raise ValueError(f"gradient norm: float32, float16 or bfloat16 expected, not {kind}")
        devices = {t.get_device() for t in tensors}
        if len(devices) > 1:
            raise ValueError("gradient norm: every gradient must be on one device")
        if -1 in devices:
            raise RuntimeError("gradient norm: HIP tensors only (no CPU path)")
        numel = [t.numel() for t in tensors]
        if 0 in numel:
            keep = [i for i, m in enumerate(numel) if m]
            tensors, kinds, numel = ([v[i] for i in keep] for v in (tensors, kinds, numel))
        self.given = tensors
        self.n = n = len(tensors)
        if not n:
            return
        self.tensors = [t if t.is_contiguous() else _without_gaps(t) for t in tensors]
        self.pointers = [t.data_ptr() for t in self.tensors]
        self.ends = [p + m * _SIZES[k] for p, m, k in zip(self.pointers, numel, kinds)]
        self.args = ((ctypes.c_void_p * n)(*self.pointers), (ctypes.c_int64 * n)(*numel),
                     (ctypes.c_int * n)(*[_DTYPES[k] for k in kinds]))
        self.device = tensors[0].device
        self.scratch = torch.empty(_lib.load().gsr_grad_norm_scratch_bytes(n), dtype=torch.uint8,
                                   device=self.device)
        self.norm = torch.empty((), dtype=torch.float32, device=self.device)


def _norm_and_scale(c, norm_code, max_norm, scale=None):
    """gsr_grad_norm on the current stream: the norm (and `scale`, a one-float tensor)."""
    with _lib.on_device(c.device):
        rc = _lib.load().gsr_grad_norm(c.n, *c.args, norm_code, float(max_norm), c.norm.data_ptr(),
                                       None if scale is None else scale.data_ptr(),
                                       c.scratch.data_ptr(), _lib.raw_stream(c.device))
    if rc != 0:
        raise RuntimeError(f"gsr_grad_norm failed with status {rc}")
    return c.norm


@torch.no_grad()
def grad_norm(tensors, norm_type=2.0):
    """The norm (1, 2 or inf) of all elements of `tensors` together, as a float32 scalar on their
    device (not synchronised).  Any number of tensors, of mixed types, strides and sizes; sums in
    64 bits, the same tensors give the same bits.  No tensors (or only empty ones): 0."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    code, c = _norm_code(norm_type), _CTensors(tensors)
    if not c.n:
        return torch.zeros((), device=tensors[0].device if tensors else "cpu")
    return _norm_and_scale(c, code, math.inf)


def _refuse_overlap(c):
    """Two workgroups may not scale the same memory.  Gradients with gaps are scaled in copies and may
    lie between each other (columns of one buffer); refused are one that lies over a gradient that is
    scaled in place, and two that begin at the same element."""
    if all(map(operator.is_, c.given, c.tensors)):
        spans = sorted(zip(c.pointers, c.ends))
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("clip_grad_norm_: two gradients share memory (the same one twice?)")
        return
    spans = []
    for t, own, start, end in zip(c.given, c.tensors, c.pointers, c.ends):
        if t is not own:
            if 0 in [s for n, s in zip(t.shape, t.stride()) if n > 1]:
                raise ValueError("clip_grad_norm_: an expanded gradient cannot be scaled in place")
            last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
            start, end = t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()
        spans.append((start, end, t is own))
    spans.sort()
    end_dense = end_any = last = 0
    for start, end, dense in spans:
        if start < (end_any if dense else end_dense) or start == last:
            raise ValueError("clip_grad_norm_: two gradients share memory (the same one twice?)")
        last = start
        if end > end_any:
            end_any = end
        if dense and end > end_dense:
            end_dense = end


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """torch.nn.utils.clip_grad_norm_: scale every parameter's .grad in place by
    min(1, max_norm / (norm + 1e-6)), norm = grad_norm of all of them; returns the norm.  As there,
    a norm that is NaN makes every gradient NaN, unless error_if_nonfinite (which waits for the
    norm) raises first.  Gradients must not share memory with each other."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    max_norm = _limit(max_norm, "max_norm")
    code = _norm_code(norm_type)
    grads = [g for g in [p.grad for p in parameters] if g is not None]
    c = _CTensors(grads)
    if not c.n:
        return torch.zeros((), device=grads[0].device if grads else "cpu")
    _refuse_overlap(c)
    if error_if_nonfinite and not bool(torch.isfinite(_norm_and_scale(c, code, math.inf))):
        raise RuntimeError(f"The total norm of order {norm_type} is non-finite, so it cannot "
                           "be clipped")
    with _lib.on_device(c.device):
        rc = _lib.load().gsr_clip_grads(c.n, *c.args, code, max_norm, c.norm.data_ptr(),
                                        c.scratch.data_ptr(), _lib.raw_stream(c.device))
    if rc != 0:
        raise RuntimeError(f"gsr_clip_grads failed with status {rc}")
    for t, own in zip(c.given, c.tensors):
        if t is not own:  # a gradient with gaps: its scaled copy goes back
            t.copy_(own)
    return c.norm


class FusedAdam(torch.optim.Adam):
    """max_grad_norm: clip by the global 2-norm of every parameter's gradient in each step, as
    clip_grad_norm_(parameters, max_grad_norm) before it would, but inside the Adam launch: .grad
    keeps its unclipped values.  `grad_norm` is the last step's norm (a device scalar, not
    synchronised; None before the first step and after one without clipping).  A step in row slices
    (begin_rows) takes the norm when it begins, so every gradient must be final by then.  All
    gradients of a clipped step are on one device."""

    max_grad_norm = grad_norm = None  # of optimizers pickled before there were these

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0,
                 amsgrad=False, *, maximize=False, max_grad_norm=None):
        if amsgrad or maximize:
            raise ValueError("FusedAdam implements Adam without amsgrad / maximize")
        if max_grad_norm is not None:
            _limit(max_grad_norm, "max_grad_norm")
        super().__init__(params, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                         amsgrad=False, foreach=False)
        self._mailbox = {}     # device -> pinned int32 [1]: 1 = the step's launches skipped it
        self._guard = {}       # device -> float32 [1] device slot: the step's one fault snapshot
        self._pending = None   # (events, mailboxes, stepped states, fault-reset count)
        self.skipped_steps = 0
        self.max_grad_norm = max_grad_norm
        self.grad_norm = None

    def _resolve_pending(self):
        """The previous step's device decision: undo its step counts if it was skipped."""
        pend, self._pending = self._pending, None
        if pend is None:
            return
        events, boxes, states, resets = pend
        for ev in events:
            if not ev.query():
                ev.synchronize()  # rare: the previous step's launch has not finished yet
        if not any(int(b[0]) for b in boxes):
            return
        for st in states:
            st["step"] -= 1
        self.skipped_steps += 1
        if _lib.fault_resets() == resets:
            raise RuntimeError(
                "FusedAdam: the previous step was skipped on the device because a rasterizer "
                "forward of that step failed (on this or another rank); parameters, moments and "
                "step counts are unchanged.  Handle the failure and call "
                "gsr_amd._lib.reset_forward_faults() before stepping again.")

    @torch.no_grad()
    def step(self, closure=None, *, skip=None):
        """One Adam step of every parameter with a gradient.  skip: a one-float device tensor
        whose non-zero value skips the step (GradAllReducer.skip_flag(): the ranks' summed fault
        snapshots); None = this device's own fault word."""
        self._resolve_pending()
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        h = self.begin_rows(skip=skip)
        self.step_rows(h, 0, None)
        self.end_rows(h)
        return loss

    # -- the step in row slices (multi-GPU: Adam on the rows whose all-reduce is done while the
    # next slice's collective runs, gsr_amd.trainer.train_step_views) ---------------------------
    @torch.no_grad()
    def begin_rows(self, *, skip=None):
        """Start a step applied in row ranges: the step counts advance once here and the
        (betas, eps) batches are fixed; step_rows(h, a, b) then updates rows [a, b) of every
        parameter (dim 0), end_rows(h) finishes.  The row ranges must cover every row exactly
        once; the result is bitwise the one of step() (the update is elementwise)."""
        self._resolve_pending()
        grads = None
        if self.max_grad_norm is not None:  # refused before any step count advances
            limit = _limit(self.max_grad_norm, "max_grad_norm")  # it may have been set since __init__
            grads = _CTensors([p.grad for group in self.param_groups for p in group["params"]
                               if p.grad is not None])
        batches = {}
        for group in self.param_groups:
            beta1, beta2 = group["betas"]
            for p in group["params"]:
                if p.grad is None:
                    continue
                g = p.grad
                if g.is_sparse:
                    raise RuntimeError("FusedAdam does not support sparse gradients")
                if not p.is_cuda:
                    raise RuntimeError("FusedAdam updates HIP tensors only (no CPU path)")
                if p.dtype != torch.float32 or g.dtype != torch.float32:
                    raise RuntimeError("FusedAdam expects float32 parameters and gradients")
                state = self.state[p]
                if len(state) == 0:  # torch.optim.Adam._init_group layout
                    state["step"] = torch.tensor(0.0, dtype=torch.float32)
                    state["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                    state["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                state["step"] += 1
                m, v = state["exp_avg"], state["exp_avg_sq"]
                for t, name in ((p, "param"), (g, "grad"), (m, "exp_avg"), (v, "exp_avg_sq")):
                    if not t.is_contiguous() or t.numel() != p.numel() or t.device != p.device:
                        raise RuntimeError(f"FusedAdam: {name} must be contiguous, on the "
                                           "parameter's device, with the parameter's size")
                key = (p.device, float(beta1), float(beta2), float(group["eps"]))
                batches.setdefault(key, []).append(
                    (p, g, m, v, float(group["lr"]), float(group["weight_decay"]),
                     float(state["step"])))
        skips = {}
        for (dev, _, _, _) in batches:
            if dev in skips:
                continue
            box = self._mailbox.get(dev)
            if box is None:
                box = torch.zeros(1, dtype=torch.int32, pin_memory=True)
                self._mailbox[dev] = box
            box[0] = 0
            if skip is not None and (skip.device != dev or skip.dtype != torch.float32):
                raise ValueError("FusedAdam.step: skip must be a float32 tensor on the parameters' device")
            if skip is None:
                # ONE snapshot of the device's fault word for every launch of the step (chunks of
                # MAX_TENSORS, (betas, eps) batches, row slices): a fault published between two
                # launches cannot leave some rows updated and others not
                slot = self._guard.get(dev)
                if slot is None:
                    slot = torch.zeros(1, dtype=torch.float32, device=dev)
                    self._guard[dev] = slot
                with _lib.on_device(dev):
                    _lib.step_guard(slot)
                skips[dev] = (slot.data_ptr(), box)
            else:
                skips[dev] = (skip.data_ptr(), box)
        states = [self.state[it[0]] for its in batches.values() for it in its]
        scale = self.grad_norm = None  # a step that is not clipped has no norm
        if grads is not None and not grads.n:
            self.grad_norm = torch.zeros((), device=self.param_groups[0]["params"][0].device)
        elif grads is not None:
            scale = torch.empty(1, dtype=torch.float32, device=grads.device)
            self.grad_norm = _norm_and_scale(grads, _NORMS[2.0], limit, scale)
        return {"batches": batches, "skips": skips, "states": states, "issued": False,
                "scale": scale}

    def abort_rows(self, h):
        """Give back the step counts begin_rows advanced when the step is abandoned before any
        step_rows launch was issued (a forward or backward between them raised): the next step's
        bias corrections then see the counts of the updates actually applied.  Once a
        slice was issued the rows it updated used the advanced counts, so they are kept."""
        if h is None or h["issued"]:
            return
        for st in h["states"]:
            st["step"] -= 1
        h["issued"] = True  # idempotent

    @torch.no_grad()
    def step_rows(self, h, a: int, b):
        """Rows [a, b) of every parameter of the step begun by begin_rows (b None: to the end).
        Issued on the current stream of each parameter's device."""
        L = _lib.load()
        h["issued"] = True
        scale = None
        if h["scale"] is not None:
            scale = h["scale"].data_ptr()
            h["scale"].record_stream(torch.cuda.current_stream(h["scale"].device))
        for (dev, beta1, beta2, eps), items in h["batches"].items():
            stream = _lib.raw_stream(dev)
            skip_ptr, box = h["skips"][dev]
            sel = []
            for it in items:
                rows = it[0].shape[0] if it[0].dim() else 1
                row = it[0].numel() // max(1, rows)
                lo, hi = a, rows if b is None else min(b, rows)
                if hi > lo:
                    sel.append((it, lo * row * 4, (hi - lo) * row))
            for c in range(0, len(sel), MAX_TENSORS):
                chunk = sel[c:c + MAX_TENSORS]
                n = len(chunk)
                ptrs = [(ctypes.c_void_p * n)(*[s[0][k].data_ptr() + s[1] for s in chunk])
                        for k in range(4)]
                numel = (ctypes.c_int64 * n)(*[s[2] for s in chunk])
                lr = (ctypes.c_double * n)(*[s[0][4] for s in chunk])
                wd = (ctypes.c_double * n)(*[s[0][5] for s in chunk])
                steps = (ctypes.c_double * n)(*[s[0][6] for s in chunk])
                with _lib.on_device(dev):
                    rc = L.gsr_adam_step_scaled(n, ptrs[0], ptrs[1], ptrs[2], ptrs[3], numel, lr,
                                                wd, steps, beta1, beta2, eps, skip_ptr,
                                                box.data_ptr(), scale, stream)
                if rc != 0:
                    raise RuntimeError(f"gsr_adam_step failed with status {rc}")

    def end_rows(self, h):
        """Finish a step begun by begin_rows: its skip decision is read back by the next step."""
        events, boxes = [], []
        for dev, (_, box) in h["skips"].items():
            with _lib.on_device(dev):
                ev = torch.cuda.Event()
                ev.record(torch.cuda.current_stream(dev))
            events.append(ev)
            boxes.append(box)
        if events:
            self._pending = (events, boxes, h["states"], _lib.fault_resets())
