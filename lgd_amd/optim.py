"""Gradient norms and clipping over many tensors, and gradient clipping + the two SGD updates of the distillation step as ONE HIP launch
(csrc/grad_norm.hip, csrc/optim.hip).

[ref: train.py:200-204 -- `stu_optimizer.step(); tea_optimizer.step()`; utils/build.py:494-529 -- torch.optim.SGD with momentum and
weight decay, wrapped by detectron2's per-parameter gradient clipping (CLIP_TYPE "value").]

The torch.optim.SGD objects stay the owners of the state (momentum buffers under the reference's keys, param groups, the LR
schedulers drive their `lr`), so checkpoints and `Trainer.state_dict()` are unchanged; only the arithmetic of `step()` moves into
`lgd_sgd_clip_step`.  torch's multi-tensor path costs ~1.7 ms of Python per step (grouping ~330-530 tensors for each of six foreach
ops and two optimizers) and ~40 launches over 13 tensor transfers per element; at 2 images per GPU the GPU ran dry for 0.7 ms at the
optimizer entry.  Here the host builds one table (three pointers, length, lr / wd / mu per tensor) in pinned memory and launches once.
"""
import ctypes

import numpy as np
import torch

from . import hip

_TENSOR_DT = np.dtype([("p", "<u8"), ("g", "<u8"), ("m", "<u8"), ("n", "<i8"), ("lr", "<f4"), ("wd", "<f4"), ("mu", "<f4"),
                       ("reserved", "<i4")])  # mirror of lgd_sgd_tensor (include/lgd_hip.h), 48 bytes
assert _TENSOR_DT.itemsize == 48

_NORMS = {2.0: 0, 1.0: 1, float("inf"): 2}   # LGD_NORM_*


def _norm_code(norm_type):
    code = _NORMS.get(float(norm_type))
    if code is None:
        raise hip.LgdHipError("norm_type %r: one of 1, 2, inf" % (norm_type,))
    return code


def grad_norm(tensors, norm_type=2.0):
    """norm over every element of every tensor (fp32 / bf16 / fp16, mixed) as ONE vector -> 0-dim fp32 tensor on their device, no host sync:
    norm_type 2, 1 or inf.  Sums are 64-bit and run in a fixed order.  A NaN anywhere gives NaN.  No tensors: 0 on the CPU."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    return _norm(hip.host().norm(tensors, False, _norm_code(norm_type), None), tensors)


def clip_grad_norm_(parameters, max_norm, norm_type=2.0):
    """clip the gradients of `parameters` (a tensor or an iterable; those without a gradient are skipped) IN PLACE by the norm of all of them
    taken together, torch.nn.utils.clip_grad_norm_'s arithmetic: g *= min(1, max_norm / (norm + 1e-6)).  -> the norm before clipping (0-dim
    fp32 on the device).  No host sync, two launches over all the tensors; nothing is written where nothing has to be clipped.  A norm that is
    not finite reaches the gradients as it does in torch (NaN everywhere, or 0 and NaN).  The gradients must not share memory."""
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise hip.LgdHipError("max_norm must not be negative, got %r" % max_norm)
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    return _norm(hip.host().norm(parameters, True, _norm_code(norm_type), max_norm), parameters)


def _norm(got, tensors):
    """csrc/host.cpp's answer: a tensor, None (there were no tensors) or False (they are not on a GPU)"""
    if got is None:
        return torch.tensor(0.0)
    if got is False:
        hip.require_gpu(*tensors)
        raise hip.LgdHipError("gradients are not on a GPU")
    return got


def supported(optimizers, clip):
    """the fused step covers what the reference's configs use: SGD (dampening 0, no Nesterov, not maximize) on fp32 CUDA parameters,
    gradient clipping off, CLIP_TYPE 'value', or 'full_model' (by the norm of each optimizer's whole gradient; NORM_TYPE 1, 2 or inf); anything
    else stays on torch's own multi-tensor path."""
    if clip.ENABLED and clip.CLIP_TYPE not in ("value", "full_model"):
        return False
    if clip.ENABLED and clip.CLIP_TYPE == "full_model" and float(clip.NORM_TYPE) not in _NORMS:
        return False
    for o in optimizers:
        if type(o) is not torch.optim.SGD:
            return False
        for g in o.param_groups:
            if g.get("dampening", 0) != 0 or g.get("nesterov", False) or g.get("maximize", False):
                return False
            for p in g["params"]:
                if not p.is_cuda or p.dtype != torch.float32 or not p.is_contiguous():
                    return False
    return True


class FusedClipSGD:
    """step() = clip + update of every parameter that has a gradient, over all the given torch.optim.SGD objects.
    clip_value: element-wise clamp.  clip_norm: the gradients of EACH optimizer are scaled by min(1, clip_norm / (norm + 1e-6)) of their own
    norm (norm_type 2, 1 or inf) -- torch.nn.utils.clip_grad_norm_ per optimizer, then its step(); `total_norms` then holds the norms
    before clipping of the last step (one fp32 per optimizer, on the device).  Neither: no clipping.  The clipped gradients are written back."""
    SLOTS = 8  # pinned staging tables in flight (a slot is reused SLOTS steps later, after its upload event has completed)

    def __init__(self, optimizers, clip_value=None, clip_norm=None, norm_type=2.0):
        self.optimizers = list(optimizers)
        if clip_value is not None and clip_norm is not None:
            raise hip.LgdHipError("clip by value or by norm, not both")
        self.clip_value = float("inf") if clip_value is None else float(clip_value)
        self.clip_norm, self.norm_type, self.total_norms = clip_norm, norm_type, None
        self.params, self.owner = [], []
        for k, o in enumerate(self.optimizers):
            for gi, g in enumerate(o.param_groups):
                for p in g["params"]:
                    self.params.append(p)
                    self.owner.append((k, gi))
        n = len(self.params)
        if clip_norm is not None:
            _norm_code(norm_type)
            if len({id(p) for p in self.params}) != n or not 1 <= len(self.optimizers) <= 16:
                raise hip.LgdHipError("clipping by norm takes 1 to 16 optimizers (LGD_MAX_SGD_GROUPS) that share no parameter")
        self._numel = np.array([p.numel() for p in self.params], dtype=np.int64)
        self._m_ptr = np.zeros(n, dtype=np.uint64)
        self._m_ref = [None] * n   # the buffer each cached pointer belongs to
        self._state_ids = None     # Optimizer.load_state_dict installs a new state dict: the cached buffers are then stale
        self._grp = np.array([k * 4096 + gi for k, gi in self.owner], dtype=np.int64)
        self.chunk = None
        self._checked_idx = self._plan = None
        rec = 48 * n + 4 * (n + 1)
        self._slot_bytes = (rec + 255) // 256 * 256
        self._pinned = None
        self._events = [None] * self.SLOTS
        self._slot = 0

    def zero_grad(self):
        """`optimizer.zero_grad(set_to_none=True)` of all the optimizers (plain loop: no per-optimizer bookkeeping)."""
        for p in self.params:
            p.grad = None

    def _buffers(self, idx):
        """momentum buffers of the parameters `idx` (created zero-filled on first use: torch's first step sets buf = d_p, which
        is what mu * 0 + d_p gives); the cache is dropped when an optimizer's state dict has been replaced (load_state_dict)."""
        ids = [id(o.state) for o in self.optimizers]
        if ids != self._state_ids:
            self._state_ids = ids
            self._m_ref = [None] * len(self.params)
        for i in idx:
            if self._m_ref[i] is not None:
                continue
            p = self.params[i]
            st = self.optimizers[self.owner[i][0]].state[p]
            m = st.get("momentum_buffer")
            if m is None:
                m = st["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
            if not (m.is_cuda and m.dtype == torch.float32 and m.is_contiguous() and m.numel() == p.numel()):
                raise hip.LgdHipError("momentum buffer of a fused-SGD parameter must be a dense fp32 device tensor")
            self._m_ref[i] = m
            self._m_ptr[i] = m.data_ptr()

    @torch.no_grad()
    def step(self):
        lib = hip.load()
        if self.chunk is None:
            self.chunk = int(lib.lgd_sgd_chunk_elems())
        grads = [p.grad for p in self.params]
        idx = [i for i, g in enumerate(grads) if g is not None]
        by_norm = self.clip_norm is not None
        if by_norm and not float(self.clip_norm) >= 0:
            raise hip.LgdHipError("clip_norm must not be negative, got %r" % (self.clip_norm,))
        if not idx:
            if by_norm:
                self.total_norms = torch.zeros(len(self.optimizers), device=self.params[0].device if self.params else None)
            return
        hip.require_gpu(grads[idx[0]])
        if by_norm and torch.cuda.is_current_stream_capturing():
            raise hip.LgdHipError("the fused step uploads its table from host memory that later steps reuse: it cannot be captured into a graph")
        params = [self.params[i] for i in idx]
        grads = [grads[i] for i in idx]
        k = len(idx)
        if idx != self._checked_idx:   # once per set of parameters that receive gradients: layout checks (autograd hands out the same kind of
            for g in grads:            # tensor every step) and what the table's other columns follow from
                if g.dtype != torch.float32 or not g.is_contiguous() or g.is_sparse:
                    raise hip.LgdHipError("fused SGD needs dense contiguous fp32 gradients")
            ii = np.asarray(idx, dtype=np.int64)
            tab, blk = np.zeros(k, dtype=_TENSOR_DT), np.zeros(k + 1, dtype=np.int32)
            tab["n"] = self._numel[ii]
            blk[1:] = np.cumsum((self._numel[ii] + self.chunk - 1) // self.chunk)
            keys, which = np.unique(self._grp[ii], return_inverse=True)
            owner = self._grp[ii] // 4096
            if by_norm:
                tab["reserved"] = owner
            border = np.searchsorted(owner, np.arange(len(self.optimizers) + 1)).astype(np.int32)   # the table is ordered by optimizer
            self._plan = (ii, tab, blk, [divmod(key, 4096) for key in keys.tolist()], which, border, blk[border])
            self._checked_idx = idx
        elif not all(map(torch.Tensor.is_contiguous, grads)):
            raise hip.LgdHipError("fused SGD needs dense contiguous fp32 gradients")
        self._buffers(idx)
        ii, tab, blk, keys, which, border, border_blk = self._plan
        ptr_of = torch.Tensor.data_ptr
        gp = list(map(ptr_of, grads))
        if by_norm and len(set(gp)) < k and len({q for q, g in zip(gp, grads) if g.numel()}) < sum(g.numel() > 0 for g in grads):
            raise hip.LgdHipError("two of the gradients share memory: each element can be clipped once")
        tab["p"] = list(map(ptr_of, params))
        tab["g"] = gp
        tab["m"] = self._m_ptr[ii]
        hy = np.array([[g["lr"], g["weight_decay"], g["momentum"]] for g in (self.optimizers[o].param_groups[j] for o, j in keys)], dtype=np.float32)[which]
        tab["lr"], tab["wd"], tab["mu"] = hy[:, 0], hy[:, 1], hy[:, 2]
        device = grads[0].device
        if self._pinned is None:
            self._pinned = torch.empty(self.SLOTS * self._slot_bytes, dtype=torch.uint8).pin_memory()
        s = self._slot
        self._slot = (s + 1) % self.SLOTS
        if self._events[s] is not None:
            self._events[s].synchronize()   # SLOTS steps old: long complete unless the host ran that far ahead
        nbytes = 48 * k + 4 * (k + 1)
        host = self._pinned[s * self._slot_bytes:s * self._slot_bytes + nbytes]
        raw = host.numpy()
        raw[:48 * k] = tab.view(np.uint8)
        raw[48 * k:] = blk.view(np.uint8)
        n_blocks = int(blk[k])
        dev = torch.empty(nbytes, dtype=torch.uint8, device=device)
        dev.copy_(host, non_blocking=True)
        ev = self._events[s]
        if ev is None:
            ev = self._events[s] = torch.cuda.Event()
        ev.record()
        base = dev.data_ptr()
        if by_norm:
            ng = len(self.optimizers)
            norms = torch.empty(ng, dtype=torch.float32, device=device)
            ws = torch.empty(lib.lgd_sgd_norm_ws_bytes(ng), dtype=torch.uint8, device=device)
            hip.check(lib.lgd_sgd_norm_step(base, base + 48 * k, k, n_blocks, border.ctypes.data, border_blk.ctypes.data, ng, _norm_code(self.norm_type),
                                            float(self.clip_norm), ws.data_ptr(), norms.data_ptr(), hip.stream_ptr()), "lgd_sgd_norm_step")
            self.total_norms = norms
        else:
            hip.check(lib.lgd_sgd_clip_step(base, base + 48 * k, k, n_blocks, self.clip_value, hip.stream_ptr()), "lgd_sgd_clip_step")
        # the kernel wrote p, g and the momentum buffers through raw pointers: tell autograd's version counters, which the fold
        # caches (ConvBN._frozen_fold, FrozenBatchNorm2d.scale_shift) key on and the saved-tensor check reads
        torch.autograd.graph.increment_version(params + grads + [self._m_ref[i] for i in idx])
        for o in self.optimizers:
            o._opt_called = True   # what the LR schedulers' "scheduler.step() before optimizer.step()" check looks at
