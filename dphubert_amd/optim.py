"""Fused AdamW + global-norm clipping on the GPU (torch.optim.AdamW semantics).

Drop-in for the optimizer built in lightning.py:200-228 (three param groups:
main / log_alpha / lambda with negative lr) plus Lightning's
``gradient_clip_val`` (distill.py:48).  One ``dph_grad_sumsq`` + one
``dph_adamw_step`` launch update every parameter; the clip coefficient never
leaves the device.
"""

import math
from typing import Iterable, List, Optional

import torch
from torch.autograd.graph import increment_version

from . import _lib
from ._lib import DphAdamGroup, DphMuonSlot, DphTensorSlot, call, ptr

CHUNK = 8192   # must match optim.hip
SUMSQ_FLOATS = 1025   # DPH_SUMSQ_FLOATS (include/dphubert_hip.h)


class FusedAdamW(torch.optim.Optimizer):
    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                 max_grad_norm: Optional[float] = None):
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay)
        super().__init__(params, defaults)
        self.max_grad_norm = max_grad_norm
        self._chunk_key = None
        self._pinned = None
        self._slots_dev = None
        self._event = None
        self._slot_key = None
        self._step = 0
        self._step_t = torch.zeros((), dtype=torch.float32)   # one counter shared by every param's state
        self.dyn_ptr = None          # device DphAdamDyn (stepstate.StepScalars) -> dph_adamw_step_dev
        self._captured = False       # a launch was captured: the graph reads the device tables by address
        self._kept = []              # the tables that such a graph may read and that others have taken the place of

    def add_param_group(self, group):
        if len(self.param_groups) == 4:      # (what a DphAdamDyn holds)
            raise ValueError(f"{type(self).__name__} supports at most 4 param groups")
        super().add_param_group(group)

    def _params(self):
        out = []
        for gi, g in enumerate(self.param_groups):
            for p in g["params"]:
                out.append((gi, p))
        return out

    def _replace(self, *tables):
        """Other tables take the place of these: a graph that reads them goes on doing so."""
        if self._captured:
            self._kept.append(tables)

    def _ensure_chunks(self, plist):
        dev = plist[0][1].device
        key = (dev,) + tuple(p.numel() for _, p in plist)     # (moved pointers are written into the same slots)
        if key == self._chunk_key:
            return
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"{type(self).__name__}: the parameter list changed inside a HIP graph capture")
        if self._chunk_key is not None:
            self._replace(self._cslot, self._cstart, self._slots_dev, self._sumsq)
        self._slot_key = None
        cslot, cstart = [], []
        for si, (_, p) in enumerate(plist):
            n = p.numel()
            for s in range(0, n, CHUNK):
                cslot.append(si)
                cstart.append(s)
        self._cslot = torch.tensor(cslot, dtype=torch.int64, device=dev)
        self._cstart = torch.tensor(cstart, dtype=torch.int64, device=dev)
        self._nchunks = len(cslot)
        nbytes = len(plist) * C_SIZEOF_SLOT
        self._pinned = torch.empty(nbytes, dtype=torch.uint8, pin_memory=True)
        self._slots_dev = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        self._sumsq = torch.zeros(SUMSQ_FLOATS, dtype=torch.float32, device=dev)   # [0] = ||g||^2, [1:] partials
        self._chunk_key = key

    def _state_keys(self, gi):
        """The state tensors of a parameter of group ``gi``."""
        return ("exp_avg", "exp_avg_sq")

    def _slot_table(self, plist):
        """Upload the (param, grad, exp_avg, exp_avg_sq) pointer table when any pointer changed.
        With a GradReducer the gradients are fixed bucket views, so this runs once."""
        capturing = torch.cuda.is_current_stream_capturing()
        self._captured |= capturing
        key = []
        for gi, p in plist:
            st = self.state[p]
            if len(st) == 0:
                for k in self._state_keys(gi):
                    st[k] = torch.zeros_like(p, memory_format=torch.preserve_format)
                st["step"] = self._step_t
            elif st.get("step") is not self._step_t:
                # loaded state (load_state_dict): adopt its step count, then share one counter
                self._step = max(self._step, int(st["step"]))
                self._step_t.fill_(self._step)
                st["step"] = self._step_t
            if p.grad is not None and not p.grad.is_contiguous():
                p.grad = p.grad.contiguous()
            if p.grad is not None and p.grad.dtype != torch.float32:
                raise TypeError("FusedAdamW expects fp32 gradients")
            ma, va = [st[k].data_ptr() for k in self._state_keys(gi)] + [0] * (2 - len(self._state_keys(gi)))
            key.append((p.data_ptr(), p.grad.data_ptr() if p.grad is not None else 0, ma, va, p.numel(), gi))
        key = tuple(key)
        if key == self._slot_key:
            return
        if capturing:
            raise RuntimeError("FusedAdamW: parameter/gradient storage changed inside a HIP graph capture")
        if self._event is not None:
            self._event.synchronize()     # previous H2D copy of the pinned table is done
        slots = (DphTensorSlot * len(plist)).from_address(self._pinned.data_ptr())
        for i, (pp, gp, ma, va, n, gi) in enumerate(key):
            slots[i].param, slots[i].grad, slots[i].exp_avg, slots[i].exp_avg_sq = pp, gp, ma, va
            slots[i].n = n
            slots[i].group = gi
        self._slots_dev.copy_(self._pinned, non_blocking=True)
        self._event = torch.cuda.Event()
        self._event.record()
        self._slot_key = key

    def begin_step(self) -> int:
        """Host half of a step: advance the step counter; returns the 1-based AdamW step that a
        device-resident DphAdamDyn must carry together with the current ``param_groups`` values."""
        self._step += 1
        self._step_t.fill_(self._step)
        self._opt_called = True       # what torch's LRScheduler checks for "optimizer.step() ran first"
        return self._step

    @torch.no_grad()
    def launch(self):
        """Device half of a step: clip + AdamW over every parameter (2 launches), stream-ordered and
        capturable.  Reads lr / step from ``self.dyn_ptr`` (a DphAdamDyn in device memory) when set,
        else from ``param_groups`` at launch time."""
        plist = self._params()
        if not plist:
            return
        self._ensure_chunks(plist)
        self._slot_table(plist)
        s = _lib.stream_ptr()
        clip = self.max_grad_norm is not None and self.max_grad_norm > 0
        if clip:
            call("dph_grad_sumsq", ptr(self._slots_dev), len(plist), ptr(self._cslot), ptr(self._cstart),
                 self._nchunks, ptr(self._sumsq), s)
        from . import ops
        ids = {id(p) for _, p in plist}
        # the bf16 GEMM images of the updated weights are written by the AdamW kernel itself (one pass over the
        # masters instead of a second cast launch re-reading all of them)
        dst, cast_done = ops.image_targets(ids)
        img = ops._table([(dst.get(id(p), 0),) for _, p in plist])
        groups = (DphAdamGroup * 4)()
        if self.dyn_ptr is None:
            for gi, g in enumerate(self.param_groups):
                groups[gi].lr = g["lr"]
                groups[gi].weight_decay = g["weight_decay"]
                groups[gi].beta1 = g["betas"][0]
                groups[gi].beta2 = g["betas"][1]
                groups[gi].eps = g["eps"]
        from .kernels import SPAN_HINT
        SPAN_HINT["adamw_params"] = sum(p.numel() for _, p in plist)   # bench.py's kernel table (bytes per launch)
        self._update(plist, dst, img, groups, clip, s)
        # the kernel wrote the masters behind autograd's back: bump their version counters so every
        # cached bf16 GEMM image of them (ops.bf16_image & co.) is rebuilt before its next use
        increment_version([p for _, p in plist])
        # cast the images the kernel did not cover, re-transpose the W^T images, and move the cache keys to the
        # new versions
        ops.refresh_images(ids, cast_done)

    def _update(self, plist, dst, img, groups, clip, s):
        """The update's launches, every parameter's bf16 image (``dst``) with it."""
        call("dph_adamw_step_img", ptr(self._slots_dev), len(plist), ptr(self._cslot), ptr(self._cstart),
             self._nchunks, self.dyn_ptr, groups, len(self.param_groups), self._step,
             ptr(self._sumsq) if clip else None, float(self.max_grad_norm or 0.0), ptr(img), s)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if not self._params():
            return loss
        self.begin_step()
        self.launch()
        return loss


import ctypes as _C  # noqa: E402

C_SIZEOF_SLOT = _C.sizeof(DphTensorSlot)


class FusedMuon(FusedAdamW):
    """FusedAdamW whose groups marked ``muon=True`` take the Muon step instead: matrices (parameters of two dimensions, or
    more taken as [first, rest]) move along the orthogonal factor of their momentum (kernels.newton_schulz),

        m <- m + (g - m) (1 - beta),   u = g + (m - g) beta   (``nesterov``; else u = m)
        p <- p (1 - lr weight_decay) - lr 0.2 sqrt(max(rows, columns)) orth(u)

    with beta the group's ``momentum``.  orth(u)'s entries have the root mean square 1 / sqrt(max(rows, columns)), so a
    step has 0.2 lr, about AdamW's, and AdamW's learning rates and weight decay carry over (Jordan et al., 2024; the factor
    0.2 sqrt(max) and the decay: Liu et al., 2025).  A group's ``momentum`` may change between steps.  The gradient norm that
    ``max_grad_norm`` clips is that of all groups.  State: ``momentum_buffer``; a parameter without a gradient is left
    alone.  Captured in a HIP graph like FusedAdamW: a replay steps with the gradients, states and images that the last
    step outside it found (they have to live as long), and a graph captured before a group was added steps the groups it
    knew.  The updates, their factors and the iteration's workspace are the optimiser's own."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                 max_grad_norm: Optional[float] = None, momentum: float = 0.95, nesterov: bool = True,
                 ns_steps: int = 5, ns_coeffs=None, ns_eps: float = 1e-7):
        if not 0.0 <= momentum < 1.0:
            raise ValueError(f"momentum must be in [0, 1), got {momentum}")
        if not 1 <= int(ns_steps) <= 64:
            raise ValueError(f"ns_steps must be 1 to 64, got {ns_steps}")
        self._momentum = momentum
        super().__init__(params, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, max_grad_norm=max_grad_norm)
        self.nesterov = bool(nesterov)
        self._ns = dict(steps=int(ns_steps), eps=float(ns_eps))
        if ns_coeffs is not None:
            self._ns["coeffs"] = tuple(ns_coeffs)
        self._muon_key = self._muon_shapes = self._plan = None

    def add_param_group(self, group):
        super().add_param_group(group)
        g = self.param_groups[-1]
        if not g.get("muon", False):
            return
        try:
            for p in g["params"]:
                if p.dim() < 2 or p.numel() == 0:
                    raise ValueError(f"muon group: parameters of two or more dimensions, got {tuple(p.shape)}")
                if p.dtype != torch.float32 or not p.is_contiguous():
                    raise ValueError("muon group: contiguous fp32 parameters")
            g["momentum"] = g.get("momentum", self._momentum)
            if not 0.0 <= g["momentum"] < 1.0:
                raise ValueError(f"momentum must be in [0, 1), got {g['momentum']}")
        except ValueError:
            self.param_groups.pop()
            raise
        g["betas"] = (g["momentum"], 0.0)

    def _read_momentum(self):
        """A group's momentum as it is now goes where the kernels' beta1 comes from (the uploaded scalars or the launch)."""
        for g in self.param_groups:
            if g.get("muon", False):
                if not 0.0 <= g["momentum"] < 1.0:
                    raise ValueError(f"momentum must be in [0, 1), got {g['momentum']}")
                g["betas"] = (g["momentum"], 0.0)

    def begin_step(self) -> int:
        self._read_momentum()
        return super().begin_step()

    def launch(self):
        self._read_momentum()
        super().launch()

    def _is_muon(self, gi):
        return bool(self.param_groups[gi].get("muon", False))

    def _state_keys(self, gi):
        return ("momentum_buffer",) if self._is_muon(gi) else super()._state_keys(gi)

    def _muon_tables(self, plist, dst):
        """Slots, chunks, update buffers and the iteration's plan.  Like FusedAdamW's slots these are written in place when a
        pointer moves, since a captured step reads them by address; other lists have their own."""
        at = [(i, gi, p) for i, (gi, p) in enumerate(plist) if self._is_muon(gi)]
        key = tuple((p.data_ptr(), p.grad.data_ptr() if p.grad is not None else 0,
                     self.state[p]["momentum_buffer"].data_ptr(), dst.get(id(p), 0), p.numel(), gi) for _, gi, p in at)
        # (the others' sizes too: their chunks are laid out here)
        shapes = tuple((i, tuple(p.shape), p.device) for i, _, p in at) + tuple(p.numel() for _, p in plist)
        if key == self._muon_key and shapes == self._muon_shapes:
            return
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("FusedMuon: parameter/gradient storage changed inside a HIP graph capture")
        from . import kernels as K
        if at and shapes != self._muon_shapes:
            dev = at[0][2].device
            if self._plan is not None:
                self._replace(self._plan, self._m_slots, self._m_cslot, self._m_cstart, self._a_cslot, self._a_cstart)
            pad = lambda n: (n + 3) & ~3  # noqa: E731
            flat = torch.zeros(sum(pad(p.numel()) for _, _, p in at), dtype=torch.float32, device=dev)
            ups, o = [], 0
            for _, _, p in at:
                ups.append(flat[o:o + p.numel()].view(p.shape[0], -1))
                o += pad(p.numel())
            self._plan = K.NewtonSchulzPlan(ups, **self._ns)
            cslot = [k for k, (_, _, p) in enumerate(at) for _ in range(0, p.numel(), CHUNK)]
            cstart = [c for _, _, p in at for c in range(0, p.numel(), CHUNK)]
            self._m_cslot = torch.tensor(cslot, dtype=torch.int64, device=dev)
            self._m_cstart = torch.tensor(cstart, dtype=torch.int64, device=dev)
            rest = [(i, c) for i, (gi, p) in enumerate(plist) if not self._is_muon(gi)
                    for c in range(0, p.numel(), CHUNK)]
            self._a_cslot = torch.tensor([i for i, _ in rest], dtype=torch.int64, device=dev)
            self._a_cstart = torch.tensor([c for _, c in rest], dtype=torch.int64, device=dev)
            self._m_slots = torch.empty(len(at) * _C.sizeof(DphMuonSlot), dtype=torch.uint8, device=dev)
        self._muon_shapes = shapes
        if at:
            slots = (DphMuonSlot * len(at))()
            for s, k, u, o, (_, _, p) in zip(slots, key, self._plan.mats, self._plan.out, at):
                s.param, s.grad, s.momentum, s.img, s.n, s.group = k
                s.update, s.dir = u.data_ptr(), o.data_ptr()
                s.scale = 0.2 * math.sqrt(max(u.shape))
            # (a synchronous copy: pointers move when buffers are first laid out, not from step to step)
            self._m_slots.copy_(torch.frombuffer(bytearray(bytes(slots)), dtype=torch.uint8))
        self._muon_key = key

    def _update(self, plist, dst, img, groups, clip, s):
        self._muon_tables(plist, dst)
        if not self._muon_key:
            return super()._update(plist, dst, img, groups, clip, s)
        ng, sumsq, mx = len(self.param_groups), ptr(self._sumsq) if clip else None, float(self.max_grad_norm or 0.0)
        if self._a_cslot.numel():
            call("dph_adamw_step_img", ptr(self._slots_dev), len(plist), ptr(self._a_cslot), ptr(self._a_cstart),
                 self._a_cslot.numel(), self.dyn_ptr, groups, ng, self._step, sumsq, mx, ptr(img), s)
        m = (ptr(self._m_slots), len(self._muon_key), ptr(self._m_cslot), ptr(self._m_cstart), self._m_cslot.numel(),
             self.dyn_ptr, groups, ng)
        call("dph_muon_momentum", *m, int(self.nesterov), sumsq, mx, s)
        self._plan.run()
        call("dph_muon_apply", *m, s)


class LinearDecayLRScheduler(torch.optim.lr_scheduler.LRScheduler):
    """Linear warmup then linear decay (formula of lightning.py:37-44; the reference class itself
    passes a `verbose` kwarg that torch 2.10 removed)."""

    def __init__(self, optimizer, warmup_updates: int, max_updates: int, last_epoch: int = -1):
        self.warmup_updates = warmup_updates
        self.max_updates = max_updates
        super().__init__(optimizer, last_epoch=last_epoch)

    def get_lr(self):
        if self._step_count <= self.warmup_updates:
            return [self._step_count / self.warmup_updates * base_lr for base_lr in self.base_lrs]
        elif self._step_count >= self.max_updates:
            return [0.0 for _ in self.base_lrs]
        pct_remaining = (self.max_updates - self._step_count) / (self.max_updates - self.warmup_updates)
        return [base_lr * pct_remaining for base_lr in self.base_lrs]
