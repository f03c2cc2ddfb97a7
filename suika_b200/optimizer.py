"""Gradient norm, clipping and the AdamW update on a rank's shards, on B200.

The state that migrates ({name: {sub_field: tensor}}: param, step, master, exp_avg, exp_avg_sq, as
merge_model_and_optimizer_state_dict builds it, Suika/migration.py:675-746) is stepped where it
lies. The reference's worker steps it with torch.optim.AdamW (tasks/task.py:72-73); here one
launch walks all tensors, with the moments and masters of every shard updated in place:
  - grad_sumsq / clip_grads: the global norm over many tensors and clipping, torch.nn.utils.
    clip_grad_norm_'s arithmetic. counted_spans picks what this rank counts, so that a tensor
    held by several ranks (a norm weight on every TP rank, a DP replica, a replicated KV head)
    counts once in the sum over all ranks;
  - ShardAdamW: norm, clipping and torch.optim.AdamW's update of every sub-field, without a host
    synchronisation. The clip factor is applied as the gradient is read; gradients are not
    written.
Every call is stream-ordered on the current stream of the tensors' device and can be captured.
There is no CPU path.
"""
from __future__ import annotations

from typing import Dict, Iterable, List, Optional, Sequence, Tuple, Union

import numpy as np
import torch
import torch.distributed as dist

from . import _lib as L
from .layouts import actual_shape, shard_spans

DTYPE_CODES = {torch.float32: L.RS_F32, torch.bfloat16: L.RS_BF16, torch.float16: L.RS_F16}
Grads = Union[Dict[str, torch.Tensor], Sequence[torch.Tensor]]
Counted = Dict[str, List[Tuple[int, int]]]


def counted_spans(layout, rank: int) -> Counted:
    """name -> [(offset, numel)]: the elements of `rank`'s shards that count in a sum over all ranks
    of a ParamLayout. Of the ranks that hold the same piece the first in the layout counts it. A
    name whose holders split it to different TP degrees is counted by those of its first holder's
    degree."""
    out: Counted = {}
    for name, m in layout.layout[rank].items():
        shape = actual_shape(m)
        numel = int(np.prod(shape, dtype=np.int64)) if len(shape) else 1
        holders = [(r, metas[name].tp_meta) for r, metas in layout.layout.items() if name in metas]
        deg = holders[0][1][2] if holders[0][1] is not None else 1
        mine = m.tp_meta
        if (mine[2] if mine is not None else 1) != deg:
            out[name] = []
            continue
        same = [r for r, t in holders if (t[2] if t is not None else 1) == deg and (t[1] if t is not None else 0) == (mine[1] if mine is not None else 0)]
        if same[0] != rank:
            out[name] = []
            continue
        rule = getattr(m, "tp_rule", None)
        if mine is None or not rule:
            out[name] = [(0, numel)]
            continue
        # a slice rule may give several TP indices the same units (replicated KV heads): the lowest counts
        spans = shard_spans(m.shape, mine, rule)
        earlier = {s for i in range(mine[1]) for s in shard_spans(m.shape, (mine[0], i, mine[2]), rule)}
        kept = [s not in earlier for s in spans]
        if all(kept):
            out[name] = [(0, numel)]
            continue
        if mine[0] % len(shape) != 0:
            raise ValueError(f"{name}: replicated units along dim {mine[0]} are not contiguous; only dim 0 can be counted by units")
        row = numel // shape[0]
        at, picked = 0, []
        for (lo, hi), keep in zip(spans, kept):
            if keep:
                picked.append((at * row, (hi - lo) * row))
            at += hi - lo
        out[name] = picked
    return out


def _listed(grads: Grads) -> List[Optional[torch.Tensor]]:
    return list(grads.values()) if hasattr(grads, "values") else list(grads)


def _counted_parts(grads: Grads, counted: Counted) -> List[torch.Tensor]:
    if not hasattr(grads, "items"):
        raise ValueError("counted spans go by name: give the gradients as {name: tensor}")
    parts = []
    for name, t in grads.items():
        if t is None:
            continue
        if name not in counted:
            raise AssertionError(f"no counted spans for {name}")
        if not t.is_contiguous():
            raise ValueError("gradients must be contiguous")
        flat = t.detach().view(-1)
        for off, n in counted[name]:
            if off < 0 or n < 0 or off + n > t.numel():
                raise AssertionError(f"{name}: counted span [{off}, {off + n}) leaves a gradient of {t.numel()} elements")
            parts.append(flat[off:off + n])
    return parts


def grad_sumsq(grads: Grads, counted: Optional[Counted] = None) -> torch.Tensor:
    """Sum of squares of the gradients ({name: tensor} or a sequence; None entries are left out), a
    float64 tensor of one element on their device, summed in 64 bits. `counted` (counted_spans):
    only what this rank counts; then an all-reduce over the ranks gives the global sum."""
    if counted is None:
        return L.extension().grad_sumsq(_listed(grads), None)
    like = next((g for g in _listed(grads) if g is not None), None)
    return L.extension().grad_sumsq(_counted_parts(grads, counted), like)


def _group_sumsq(grads: Grads, counted: Optional[Counted], group: Optional[dist.ProcessGroup], device: Optional[torch.device]) -> torch.Tensor:
    """grad_sumsq summed over `group`; a rank without gradients brings 0 (on `device`), so that no other waits for it."""
    if group is None:
        return grad_sumsq(grads, counted)
    if all(g is None for g in _listed(grads)):
        sumsq = torch.zeros(1, dtype=torch.float64, device=device or torch.device("cuda", torch.cuda.current_device()))
    else:
        sumsq = grad_sumsq(grads, counted)
    dist.all_reduce(sumsq, group=group)
    return sumsq


def _norm_of(sumsq: torch.Tensor) -> torch.Tensor:
    return sumsq.sqrt().float().reshape(())


def clip_grads(grads: Grads, max_norm: float, *, sumsq: Optional[torch.Tensor] = None, counted: Optional[Counted] = None,
               group: Optional[dist.ProcessGroup] = None) -> torch.Tensor:
    """Scale the gradients in place by min(1, max_norm / (norm + 1e-6)) and return the norm (float32, on
    the device; nothing is synchronised). The norm is that of grad_sumsq(grads, counted), summed over
    `group` if one is given, or sqrt(sumsq) if the caller has the global sum of squares already. All
    of every gradient is scaled, whether counted here or by another rank; gradients that share memory
    are refused. A norm that is not finite reaches the gradients, as in torch.nn.utils.clip_grad_norm_.
    With `group` a rank may have no gradients (a frozen stage): it takes part in the sum, on the current device,
    and gets the norm."""
    if not max_norm > 0:
        raise ValueError("max_norm must be positive")
    if sumsq is None and (counted is not None or group is not None):
        sumsq = _group_sumsq(grads, counted, group, None)
    if group is not None and all(g is None for g in _listed(grads)):
        return _norm_of(sumsq)
    return L.extension().grad_clip(_listed(grads), max_norm, sumsq)


class ShardAdamW:
    """AdamW over a rank's state, in place.

    state: {name: {sub_field: tensor}} as schedule_and_execute_param_transfer returns it. Sub-fields:
    `param` (float32, bfloat16 or float16), `exp_avg` and `exp_avg_sq` (both float32 or both
    bfloat16), `step` (one element) and, optionally, `master` (float32): with a master the update
    runs on it and param receives it rounded to nearest; without one it runs on param. A step that
    is not a float32 on the device is replaced in `state` by one that is, so the state can migrate
    again with its count. Arithmetic is in 32 bits whatever the types (bias corrections in 64), one
    rounding per stored value.

    The tensors that `state` holds when the optimizer is made are the ones it updates; states that view
    one source (reshard_local with views=True) must not each be stepped. no_decay: names
    whose weight decay is 0. max_norm: clip by the global norm; `counted` and `group` as in
    clip_grads. lr, weight_decay and max_norm may be assigned between steps; a captured step keeps
    those of its capture (the step counts live on the device and advance on replay).
    """

    def __init__(self, state: Dict[str, Dict[str, torch.Tensor]], lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 1e-2, no_decay: Iterable[str] = (), max_norm: Optional[float] = None,
                 counted: Optional[Counted] = None, group: Optional[dist.ProcessGroup] = None):
        if not state:
            raise ValueError("no state to step")
        if not (lr >= 0 and eps >= 0 and 0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError("lr, betas or eps out of range")
        if max_norm is not None and not max_norm > 0:
            raise ValueError("max_norm must be positive")
        self.state, self.lr, self.betas, self.eps, self.weight_decay, self.max_norm = state, lr, tuple(betas), eps, weight_decay, max_norm
        self.counted, self.group = counted, group
        self.names = list(state)
        no_decay = set(no_decay)
        unknown = no_decay - set(self.names)
        if unknown:
            raise ValueError(f"no_decay names that the state does not hold: {sorted(unknown)}")
        self.device = next(iter(state.values()))["param"].device if "param" in next(iter(state.values())) else None
        self._fields = [[], [], [], [], []]  # param, master or None, exp_avg, exp_avg_sq, step of each name
        self._decays = [0.0 if n in no_decay else 1.0 for n in self.names]
        for name in self.names:
            ent = state[name]
            for s in ("param", "exp_avg", "exp_avg_sq", "step"):
                if s not in ent:
                    raise AssertionError(f"expected sub-fields mismatch: {name} has no {s}")
            p, m, v, w = ent["param"], ent["exp_avg"], ent["exp_avg_sq"], ent.get("master")
            body = [t for t in (p, m, v, w) if t is not None]
            if self.device is None or self.device.type != "cuda":
                raise ValueError(f"{name}'s sub-fields must be CUDA tensors")
            if any(t.device != self.device for t in body):
                raise ValueError(f"{name}'s sub-fields must share one device")
            if not all(t.is_contiguous() for t in body):
                raise ValueError(f"{name}'s sub-fields must be contiguous")
            if p.dtype not in DTYPE_CODES:
                raise ValueError(f"{name}'s param of {p.dtype}: float32, bfloat16 and float16 are taken")
            if any(t.shape != p.shape for t in body):
                raise AssertionError(f"{name}'s sub-fields differ in shape")
            if m.dtype != v.dtype or m.dtype not in (torch.float32, torch.bfloat16):
                raise ValueError(f"{name}: moments of {m.dtype} and {v.dtype}: both float32 or both bfloat16 are taken")
            if w is not None and w.dtype != torch.float32:
                raise ValueError(f"{name}: a master of {w.dtype}: float32 is taken")
            step = ent["step"]
            if step.numel() != 1:
                raise AssertionError(f"{name}: a step of {step.numel()} elements")
            if step.dtype != torch.float32 or step.device != self.device:
                step = ent["step"] = step.to(device=self.device, dtype=torch.float32)
            for kept, t in zip(self._fields, (p, w, m, v, step)):
                kept.append(t)
        self._check_disjoint()

    def _check_disjoint(self) -> None:
        tensors = [t for kept in self._fields for t in kept if t is not None and t.numel()]
        b = np.array([t.data_ptr() for t in tensors], np.uint64)
        n = np.array([t.numel() * t.element_size() for t in tensors], np.uint64)
        order = np.argsort(b)
        if ((b + n)[order][:-1] > b[order][1:]).any():
            raise ValueError("sub-fields of the state share memory")

    def step(self, grads: Dict[str, torch.Tensor], *, sumsq: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """One update from {name: gradient}; names without a gradient (missing or None) stay as they are, and
        gradients share no memory with the state.
        Returns the norm before clipping (float32, on the device), or None without max_norm. `sumsq`:
        the global sum of squares, if the caller has it already. With a group, or a given sumsq, there may be
        no gradient at all: the rank takes part in the sum and nothing is updated."""
        gs = [grads.get(n) for n in self.names]
        if len(grads) > len(gs) or any(g is None for g in gs):
            extra = [n for n, g in grads.items() if g is not None and n not in self.state]
            if extra:
                raise AssertionError(f"gradients of names that the state does not hold: {extra[:3]}")
        if self.max_norm is not None and sumsq is None and (self.counted is not None or self.group is not None):
            sumsq = _group_sumsq(dict(zip(self.names, gs)), self.counted, self.group, self.device)
        if (self.group is not None or sumsq is not None) and all(g is None for g in gs):
            return _norm_of(sumsq) if self.max_norm is not None else None
        return L.extension().adamw_step(*self._fields, self._decays, gs, self.lr, *self.betas, self.eps, self.weight_decay, self.max_norm, sumsq)
