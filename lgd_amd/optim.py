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
import numpy as np
import torch

from . import hip

_TENSOR_DT = np.dtype([("p", "<u8"), ("g", "<u8"), ("m", "<u8"), ("n", "<i8"), ("lr", "<f4"), ("wd", "<f4"), ("mu", "<f4"),
                       ("reserved", "<i4")])  # mirror of lgd_sgd_tensor (include/lgd_hip.h), 48 bytes
assert _TENSOR_DT.itemsize == 48

MAX_GROUPS = 16   # LGD_MAX_SGD_GROUPS
_NORMS = {2.0: 0, 1.0: 1, float("inf"): 2}   # LGD_NORM_*


def has_norm(norm_type):
    return float(norm_type) in _NORMS


def _norm_code(norm_type):
    code = _NORMS.get(float(norm_type))
    if code is None:
        raise hip.LgdHipError("norm_type %r: one of 1, 2, inf" % (norm_type,))
    return code


def grad_norm(tensors, norm_type=2.0):
    """norm over every element of every tensor (fp32 / bf16 / fp16, mixed) as ONE vector -> 0-dim fp32 tensor on their device, no host sync:
    norm_type 2, 1 or inf.  Sums are 64-bit and run in a fixed order.  A NaN anywhere gives NaN.  No tensors: 0 on the CPU.
    It has no derivative: differentiating the norm of tensors that are part of a graph raises."""
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
    gradient clipping off, CLIP_TYPE 'value', or 'full_model' (by the norm of each optimizer's whole gradient; NORM_TYPE 1, 2 or inf; at most 16
    optimizers that share no parameter); anything else stays on torch's own multi-tensor path."""
    if clip.ENABLED and clip.CLIP_TYPE not in ("value", "full_model"):
        return False
    if clip.ENABLED and clip.CLIP_TYPE == "full_model":
        ids = [id(p) for o in optimizers for g in o.param_groups for p in g["params"]]
        if not has_norm(clip.NORM_TYPE) or len(optimizers) > MAX_GROUPS or len(set(ids)) != len(ids):
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
    before clipping of the last step (one fp32 per optimizer, on the device).  Neither: no clipping.  The clipped gradients are written back.
    A step cannot be captured into a graph (refused): its table of addresses and learning rates is the host's of that call."""

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
            if len({id(p) for p in self.params}) != n or not 1 <= len(self.optimizers) <= MAX_GROUPS:
                raise hip.LgdHipError("clipping by norm takes 1 to 16 optimizers (LGD_MAX_SGD_GROUPS) that share no parameter")
        self._numel = np.array([p.numel() for p in self.params], dtype=np.int64)
        self._m_ref = [None] * n   # momentum buffers
        self._grp = np.array([k * 4096 + gi for k, gi in self.owner], dtype=np.int64)
        self._plan = None

    def zero_grad(self):
        """`optimizer.zero_grad(set_to_none=True)` of all the optimizers (plain loop: no per-optimizer bookkeeping)."""
        for p in self.params:
            p.grad = None

    def _buffers(self, idx):
        """momentum buffers of the parameters `idx` as the optimizers hold them now (created zero-filled on first use: torch's first
        step sets buf = d_p, which is what mu * 0 + d_p gives)."""
        for i in idx:
            p = self.params[i]
            st = self.optimizers[self.owner[i][0]].state[p]
            m = st.get("momentum_buffer")
            if m is None:
                m = st["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
            elif m is self._m_ref[i]:
                continue
            if not (m.is_cuda and m.dtype == torch.float32 and m.is_contiguous() and m.numel() == p.numel()):
                raise hip.LgdHipError("momentum buffer of a fused-SGD parameter must be a dense fp32 device tensor")
            self._m_ref[i] = m

    def _make_plan(self):
        """(parameter groups whose hyper-parameters the table needs, the columns of csrc/host.cpp's SgdPlan, what the optimizers' states held):
        what follows from the set of parameters that have a gradient; None where none has.  The states' entries (parameter, its state, its
        momentum buffer) are kept as objects, so that none of their addresses can come back as another's while the plan lives: a state dict that
        load_state_dict put in, a buffer that was replaced or an entry that was dropped is seen at the next step"""
        idx = [i for i, p in enumerate(self.params) if p.grad is not None]
        if not idx:
            return None
        hip.require_gpu(self.params[idx[0]].grad)
        if torch.cuda.is_current_stream_capturing():   # (a first step's momentum buffers would come out of the graph's pool, and their zeros with it)
            raise hip.LgdHipError("the fused step's table (addresses, learning rates) is the host's of this call: it cannot be captured into a graph")
        self._buffers(idx)
        chunk = int(hip.load().lgd_sgd_chunk_elems())
        ii = np.asarray(idx, dtype=np.int64)
        tab, blk = np.zeros(len(idx), dtype=_TENSOR_DT), np.zeros(len(idx) + 1, dtype=np.int32)
        tab["n"] = self._numel[ii]
        blk[1:] = np.cumsum((self._numel[ii] + chunk - 1) // chunk)
        keys, which = np.unique(self._grp[ii], return_inverse=True)
        tab["reserved"] = owner = self._grp[ii] // 4096   # clipping by norm: the row's optimizer
        border = np.searchsorted(owner, np.arange(len(self.optimizers) + 1))   # the table is ordered by optimizer
        columns = (ii.astype(np.int32), tab, blk, which.astype(np.int32), border.astype(np.int32), blk[border])
        held = [x for o in self.optimizers for p, st in o.state.items() for x in (p, st, st.get("momentum_buffer"))]
        return [divmod(key, 4096) for key in keys.tolist()], tuple(c.tobytes() for c in columns), held

    @torch.no_grad()
    def step(self):
        by_norm = self.clip_norm is not None
        if by_norm and not float(self.clip_norm) >= 0:
            raise hip.LgdHipError("clip_norm must not be negative, got %r" % (self.clip_norm,))
        code, clip = (_norm_code(self.norm_type), float(self.clip_norm)) if by_norm else (None, self.clip_value)
        got = None
        while got is None:   # a plan serves until another set of parameters has gradients or a state holds something else
            if self._plan is None:
                self._plan = self._make_plan()
                if self._plan is None:
                    if by_norm:
                        self.total_norms = torch.zeros(len(self.optimizers), device=self.params[0].device if self.params else None)
                    return
            keys, columns, held = self._plan
            groups = [self.optimizers[o].param_groups[j] for o, j in keys]
            hyper = [float(g[name]) for g in groups for name in ("lr", "weight_decay", "momentum")]
            got = hip.host().sgd_step(self.params, self._m_ref, columns, hyper, code, clip, [o.state for o in self.optimizers], held)
            if got is None:
                self._plan = None
        if got is False:
            hip.require_gpu(*[p.grad for p in self.params if p.grad is not None])
            raise hip.LgdHipError("gradients are not on a GPU")
        if by_norm:
            self.total_norms = got
        for o in self.optimizers:
            o._opt_called = True   # what the LR schedulers' "scheduler.step() before optimizer.step()" check looks at
