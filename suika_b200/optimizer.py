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

import ctypes as C
from typing import Dict, Iterable, List, Optional, Sequence, Tuple, Union

import numpy as np
import torch
import torch.distributed as dist

from . import _lib as L
from .layouts import actual_shape, shard_spans

DTYPE_CODES = {torch.float32: L.RS_F32, torch.bfloat16: L.RS_BF16, torch.float16: L.RS_F16}
Grads = Union[Dict[str, torch.Tensor], Sequence[torch.Tensor]]
Counted = Dict[str, List[Tuple[int, int]]]


def raw_stream(device_index: int) -> int:
    """The current stream's handle (torch.cuda.current_stream builds an object around it, which
    costs as much as a small launch)."""
    return torch._C._cuda_getCurrentRawStream(device_index)


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


def _refuse(t: torch.Tensor, index: int, what: str) -> None:
    """Raise for a tensor that the kernels do not take."""
    if t.device.type != "cuda":
        raise ValueError(f"{what} must be CUDA tensors")
    if t.get_device() != index:
        raise ValueError(f"{what} must share one device")
    if not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous")
    raise ValueError(f"{what} of {t.dtype}: float32, bfloat16 and float16 are taken")


def _named(grads: Grads) -> Tuple[Optional[List[str]], List[torch.Tensor]]:
    """(names or None, tensors); entries of None (a parameter without a gradient) are left out."""
    if hasattr(grads, "items"):
        kept = [(n, g) for n, g in grads.items() if g is not None]
        names, tensors = [n for n, _ in kept], [g for _, g in kept]
    else:
        names, tensors = None, [g for g in grads if g is not None]
    if not tensors:
        raise ValueError("no gradients")
    if tensors[0].device.type != "cuda":
        raise ValueError("gradients must be CUDA tensors")
    return names, tensors


def _spans(tensors: List[torch.Tensor], what: str = "gradients"):
    """(rs_grad_span array, its length) of whole tensors: one device, contiguous, a type the kernels take.
    (A span is three 64-bit words, the type in the low half of the last.)"""
    index = tensors[0].get_device()
    words: List[int] = []
    for t in tensors:
        code = DTYPE_CODES.get(t.dtype)
        if code is None or t.get_device() != index or not t.is_contiguous():
            _refuse(t, index, what)
        words += (t.data_ptr(), t.numel(), code)
    return (C.c_uint64 * len(words))(*words), len(tensors)


def _counted_spans(names: Optional[List[str]], tensors: List[torch.Tensor], counted: Counted):
    if names is None:
        raise ValueError("counted spans go by name: give the gradients as {name: tensor}")
    _spans(tensors)  # the checks
    words: List[int] = []
    for name, t in zip(names, tensors):
        if name not in counted:
            raise AssertionError(f"no counted spans for {name}")
        for off, n in counted[name]:
            if off < 0 or n < 0 or off + n > t.numel():
                raise AssertionError(f"{name}: counted span [{off}, {off + n}) leaves a gradient of {t.numel()} elements")
            words += (t.data_ptr() + off * t.element_size(), n, DTYPE_CODES[t.dtype])
    return (C.c_uint64 * len(words))(*words), len(words) // 3


def _sumsq(spans, n: int, dev: torch.device) -> torch.Tensor:
    lib = L.load()
    nb = C.c_uint64()
    L.check(lib.rs_grad_sumsq_workspace_bytes(n, C.byref(nb)))
    workspace = torch.empty(nb.value, dtype=torch.uint8, device=dev)
    out = torch.empty(1, dtype=torch.float64, device=dev)
    L.check(lib.rs_grad_sumsq(spans, n, workspace.data_ptr(), nb.value, out.data_ptr(), dev.index, raw_stream(dev.index)))
    return out


def grad_sumsq(grads: Grads, counted: Optional[Counted] = None) -> torch.Tensor:
    """Sum of squares of the gradients ({name: tensor} or a sequence; None entries are left out), a
    float64 tensor of one element on their device, summed in 64 bits. `counted` (counted_spans):
    only what this rank counts; then an all-reduce over the ranks gives the global sum."""
    names, tensors = _named(grads)
    spans, n = _spans(tensors) if counted is None else _counted_spans(names, tensors, counted)
    return _sumsq(spans, n, tensors[0].device)


def _check_sumsq(sumsq: torch.Tensor, dev: torch.device) -> None:
    if sumsq.dtype != torch.float64 or sumsq.numel() != 1 or sumsq.device != dev:
        raise ValueError("sumsq must be one float64 on the gradients' device")


def clip_grads(grads: Grads, max_norm: float, *, sumsq: Optional[torch.Tensor] = None, counted: Optional[Counted] = None,
               group: Optional[dist.ProcessGroup] = None) -> torch.Tensor:
    """Scale the gradients in place by min(1, max_norm / (norm + 1e-6)) and return the norm (float32, on
    the device; nothing is synchronised). The norm is that of grad_sumsq(grads, counted), summed over
    `group` if one is given, or sqrt(sumsq) if the caller has the global sum of squares already. All
    of every gradient is scaled, whether counted here or by another rank; gradients that share memory
    are refused. A norm that is not finite reaches the gradients, as in torch.nn.utils.clip_grad_norm_."""
    if not max_norm > 0:
        raise ValueError("max_norm must be positive")
    names, tensors = _named(grads)
    dev = tensors[0].device
    spans, n = _spans(tensors)
    if sumsq is None:
        sumsq = _sumsq(*((spans, n) if counted is None else _counted_spans(names, tensors, counted)), dev)
        if group is not None:
            dist.all_reduce(sumsq, group=group)
    else:
        _check_sumsq(sumsq, dev)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    L.check(L.load().rs_grad_clip(spans, n, sumsq.data_ptr(), max_norm, norm.data_ptr(), dev.index, raw_stream(dev.index)))
    return norm


class ShardAdamW:
    """AdamW over a rank's state, in place.

    state: {name: {sub_field: tensor}} as schedule_and_execute_param_transfer returns it. Sub-fields:
    `param` (float32, bfloat16 or float16), `exp_avg` and `exp_avg_sq` (both float32 or both
    bfloat16), `step` (one element) and, optionally, `master` (float32): with a master the update
    runs on it and param receives it rounded to nearest; without one it runs on param. A step that
    is not a float32 on the device is replaced in `state` by one that is, so the state can migrate
    again with its count. Arithmetic is in 32 bits whatever the types (bias corrections in 64), one
    rounding per stored value.

    no_decay: names whose weight decay is 0. max_norm: clip by the global norm; `counted` and `group`
    as in clip_grads. lr, weight_decay and max_norm may be assigned between steps; a captured step
    keeps those of its capture (the step counts live on the device and advance on replay).
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
        table = np.zeros(len(self.names), dtype=L.ADAMW_TENSOR_DTYPE)
        self._decays = np.ones(len(self.names), dtype=np.float32)
        self._shapes = []
        for i, name in enumerate(self.names):
            ent = state[name]
            for s in ("param", "exp_avg", "exp_avg_sq", "step"):
                if s not in ent:
                    raise AssertionError(f"expected sub-fields mismatch: {name} has no {s}")
            p, m, v, w = ent["param"], ent["exp_avg"], ent["exp_avg_sq"], ent.get("master")
            body = [t for t in (p, m, v, w) if t is not None]
            if self.device is None or self.device.type != "cuda":
                raise ValueError(f"{name}'s sub-fields must be CUDA tensors")
            for t in body:
                if t.device != self.device or not t.is_contiguous() or t.dtype not in DTYPE_CODES:
                    _refuse(t, self.device.index, f"{name}'s sub-fields")
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
            table[i] = (0, p.data_ptr(), 0 if w is None else w.data_ptr(), m.data_ptr(), v.data_ptr(), step.data_ptr(), p.numel(), 0, 0,
                        DTYPE_CODES[p.dtype], DTYPE_CODES[m.dtype])
            self._shapes.append(p.shape)
            if name in no_decay:
                self._decays[i] = 0
        self._table = table
        self._check_disjoint()

    def _check_disjoint(self) -> None:
        begin, size = [], []
        for name in self.names:
            for s, t in self.state[name].items():
                if s in ("param", "master", "exp_avg", "exp_avg_sq", "step") and t is not None and t.numel():
                    begin.append(t.data_ptr())
                    size.append(t.numel() * t.element_size())
        b, n = np.array(begin, np.uint64), np.array(size, np.uint64)
        order = np.argsort(b)
        if ((b + n)[order][:-1] > b[order][1:]).any():
            raise ValueError("sub-fields of the state share memory")

    def step(self, grads: Dict[str, torch.Tensor], *, sumsq: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """One update from {name: gradient}; names without a gradient (missing or None) stay as they are.
        Returns the norm before clipping (float32, on the device), or None without max_norm. `sumsq`:
        the global sum of squares, if the caller has it already."""
        names, shapes, table, decays = self.names, self._shapes, self._table, self._decays
        gs = [grads.get(n) for n in names]
        if any(g is None for g in gs):
            given = [g is not None for g in gs]
            if not any(given):
                raise ValueError("no gradients")
            names, gs, shapes = ([x for x, k in zip(xs, given) if k] for xs in (names, gs, shapes))
            table, decays = table[given], decays[given]
        if len(grads) > len(gs):
            extra = [n for n, g in grads.items() if g is not None and n not in self.state]
            if extra:
                raise AssertionError(f"gradients of names that the state does not hold: {extra[:3]}")
        dev = self.device
        index = dev.index
        at: List[int] = []
        codes: List[int] = []
        for n, g, shape in zip(names, gs, shapes):
            code = DTYPE_CODES.get(g.dtype)
            if code is None or g.get_device() != index or not g.is_contiguous():
                _refuse(g, index, "gradients")
            if g.shape != shape:
                raise AssertionError(f"{n}: a gradient of another shape")
            at.append(g.data_ptr())
            codes.append(code)
        lib = L.load()
        norm = None
        if self.max_norm is not None:
            if sumsq is None:
                sumsq = _sumsq(*(_spans(gs) if self.counted is None else _counted_spans(names, gs, self.counted)), dev)
                if self.group is not None:
                    dist.all_reduce(sumsq, group=self.group)
            else:
                _check_sumsq(sumsq, dev)
            norm = torch.empty((), dtype=torch.float32, device=dev)
        table["grad_dev"] = at
        table["grad_dtype"] = codes
        table["weight_decay"] = decays * np.float32(self.weight_decay)
        opts = L.RsAdamwOpts(self.lr, self.betas[0], self.betas[1], self.eps, self.max_norm or 0.0)
        nb = C.c_uint64()
        L.check(lib.rs_adamw_workspace_bytes(len(table), C.byref(nb)))
        workspace = torch.empty(nb.value, dtype=torch.uint8, device=dev)
        L.check(lib.rs_adamw_step(table.ctypes.data, len(table), C.byref(opts), None if norm is None else sumsq.data_ptr(),
                                  None if norm is None else norm.data_ptr(), workspace.data_ptr(), nb.value, index, raw_stream(index)))
        return norm
