"""The two ends of a model that its layouts slice by vocabulary, on B200: the embedding (wte) and the
logits of the lm_head.

The reference replicates wte and gathers whole logits for torch's cross entropy (lm_head is column
parallel, Suika/tensor_parallel.py:200-261; Suika/models/llama_model.py:126-157). Here each rank works
on the vocabulary rows [lo, lo + rows) that its TensorMeta gives it (shard_range):
  - embedding / embedding_grad: scaled lookup, zeros for tokens of other shards, so the sum over the
    shards is the whole lookup; the gradient by sorted tokens, without float atomics;
  - token_logprobs / token_logprobs_grad: log probability of given tokens, entropy, log-sum-exp and
    top alternatives from one pass over the logits; over several shards (`group`) each rank sends a
    record of 4 + 2 top floats per row, not its logits.
embedding and token_logprobs are differentiable (torch.autograd, reverse mode). Every call is
stream-ordered on the current stream of the tensors' device and can be captured into a CUDA graph. To
capture a backward pass, call embedding_grad and token_logprobs_grad: torch's autograd engine cannot be captured while
an eager graph of the same leaves lives. There is no CPU path.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Sequence, Tuple

import numpy as np
import torch
import torch.distributed as dist
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib as L
from .layouts import shard_spans

_MAX_SORTED = 65536  # tokens that one cluster sorts; longer batches are taken in parts


def shard_range(meta) -> Tuple[int, int]:
    """[lo, hi): the rows that a TensorMeta (sliced on dim 0, or whole) holds of its full tensor."""
    if meta.tp_meta is None:
        return 0, int(meta.shape[0])
    if meta.tp_meta[0] % len(meta.shape) != 0 or getattr(meta, "tp_rule", None):
        raise ValueError(f"{meta.name}: not one contiguous range of rows")
    return shard_spans(meta.shape, meta.tp_meta)[0]


# ---------------------------------------------------------------------------------------------
# Embedding
# ---------------------------------------------------------------------------------------------
def _lookup(ids: torch.Tensor, weight: torch.Tensor, scale: float, lo: int, group) -> torch.Tensor:
    out = L.extension().embed_lookup(ids, weight, scale, lo)
    if group is not None:
        dist.all_reduce(out, group=group)  # one shard holds each token, the others give zeros: the sum is exact
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, lo, group):
        ctx.save_for_backward(ids)
        ctx.args = (weight.shape[0], scale, lo, weight.dtype)
        return _lookup(ids, weight, scale, lo, group)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        rows, scale, lo, dtype = ctx.args
        return None, embedding_grad(grad_out, ctx.saved_tensors[0], rows, scale=scale, lo=lo, dtype=dtype), None, None, None


def embedding(ids: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0, lo: int = 0,
              group: Optional[dist.ProcessGroup] = None) -> torch.Tensor:
    """scale * weight[ids - lo], of shape [*ids.shape, hidden] and weight's type, rounded once from 32
    bits; zeros for an id outside [lo, lo + rows): another shard's token, or padding (-1). weight
    (rows of any stride, contiguous within) is the shard that starts at vocabulary row `lo`. With
    `group`, the ranks of a TP group that hold the other shards, the shards' outputs are summed."""
    if weight.requires_grad and torch.is_grad_enabled():
        return _Embedding.apply(ids, weight, scale, lo, group)
    return _lookup(ids, weight, scale, lo, group)


def _touches(g: torch.Tensor, out: torch.Tensor) -> bool:
    """Whether the contiguous `out` shares memory with a row of g, [n, hidden] with contiguous rows."""
    size = g.element_size()
    pitch, width = g.stride(0) * size, g.shape[1] * size
    lo, hi = out.data_ptr() - g.data_ptr(), out.data_ptr() - g.data_ptr() + out.numel() * out.element_size()
    if not g.numel() or not out.numel() or (pitch == 0 and lo >= width):
        return False
    i = max(0, (lo - width) // pitch + 1) if lo >= width else 0  # the first row that ends past lo
    return i < g.shape[0] and i * pitch < hi


def embedding_grad(grad_out: torch.Tensor, ids: torch.Tensor, rows: int, *, scale: float = 1.0, lo: int = 0,
                   dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None, accumulate: bool = False) -> torch.Tensor:
    """The gradient of embedding()'s weight, [rows, hidden]: row r is scale * the sum of grad_out over
    the tokens with id lo + r, summed in 32 bits in an order that the ids alone fix, and rounded
    once to `dtype` (default: grad_out's, or out's). `out` (contiguous, sharing no memory with
    grad_out) receives it; with accumulate=True it is added to what `out` holds. Rows without a token
    are 0 (left alone when accumulating).

    More than 65536 tokens are taken in parts of that many; for a 16-bit gradient the parts meet in a
    float32 one, so that it is rounded once all the same."""
    if ids.numel() <= _MAX_SORTED:
        return L.extension().embed_grad(grad_out, ids, rows, scale, lo, dtype, out, accumulate)
    # the checks of a call, and the gradient to start from
    n, hidden = ids.numel(), grad_out.shape[-1]
    if tuple(grad_out.shape[:-1]) != tuple(ids.shape):
        raise AssertionError(f"grad_out has shape {list(grad_out.shape)}, ids {list(ids.shape)}")
    g, flat = grad_out.reshape(n, hidden), ids.reshape(-1)
    if hidden > 1 and g.stride(1) != 1:
        g = g.contiguous()
    if out is not None and _touches(g, out):
        raise L.ReshardError(L.RS_ERR_ARG, "embedding_grad: the gradient overlaps the output's gradient")
    out = L.extension().embed_grad(g[:0], flat[:0], rows, scale, lo, dtype, out, accumulate)
    wide = out if out.dtype == torch.float32 else torch.zeros(out.shape, dtype=torch.float32, device=out.device)
    for at in range(0, n, _MAX_SORTED):
        L.extension().embed_grad(g[at:at + _MAX_SORTED], flat[at:at + _MAX_SORTED], rows, scale, lo, None, wide, True)
    return out if wide is out else out.copy_(wide.add_(out))


# ---------------------------------------------------------------------------------------------
# Token log probabilities
# ---------------------------------------------------------------------------------------------
class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor                  # float32, targets' shape
    entropy: torch.Tensor
    lse: torch.Tensor                      # log-sum-exp of the row
    top_logprob: Optional[torch.Tensor]    # [*targets.shape, top], largest first
    top_index: Optional[torch.Tensor]      # int64 vocabulary indices


def token_record(logits: torch.Tensor, targets: torch.Tensor, *, top: int = 0, lo: int = 0) -> torch.Tensor:
    """One vocabulary shard's part of token_logprobs: float32 [rows, 4 + 2 top], for merge_token_records."""
    return L.extension().token_record(logits, targets, top, lo, 0)


def merge_token_records(records: torch.Tensor, starts: Sequence[int]) -> TokenLogprobs:
    """token_logprobs from all shards' records, [shards, rows, 4 + 2 top]; starts[s] is the first
    vocabulary index of shard s, ascending (at most 64 shards)."""
    dev = records.device
    if dev.type != "cuda":
        raise ValueError("records must be a CUDA tensor")
    if forward_ad.unpack_dual(records).tangent is not None:
        raise ValueError("records with a forward-mode tangent: reverse mode alone is there")
    if records.dim() != 3 or records.dtype != torch.float32 or not records.is_contiguous() or records.shape[2] < 4 or records.shape[2] % 2:
        raise ValueError("records must be a contiguous float32 [shards, rows, 4 + 2 top]")
    shards, n, words = records.shape
    if len(starts) != shards:
        raise AssertionError(f"{len(starts)} starts for {shards} shards")
    top = (words - 4) // 2
    out = [torch.empty(n, dtype=torch.float32, device=dev) for _ in range(3)]
    out += [torch.empty((n, top), dtype=t, device=dev) if top else None for t in (torch.float32, torch.int64)]
    at = np.array([int(s) for s in starts], dtype=np.int64)
    L.check(L.load().rs_token_merge(records.data_ptr(), at.ctypes.data, shards, n, top, *(None if t is None else t.data_ptr() for t in out),
                                    dev.index, torch.cuda.current_stream(dev).cuda_stream))
    return TokenLogprobs(*out)


def _forward(logits, targets, top, lo, group, starts):
    """token_logprobs' five outputs and, over a group, the records of all shards."""
    if group is None:
        return L.extension().token_logprobs(logits, targets, top, lo), None
    world = dist.get_world_size(group)
    # without starts a rank knows its own place alone: its record holds indices of the whole vocabulary
    mine = L.extension().token_record(logits, targets, top, lo, lo if starts is None else 0)
    everyone = torch.empty((world * mine.shape[0], mine.shape[1]), dtype=mine.dtype, device=mine.device)
    dist.all_gather_into_tensor(everyone, mine, group=group)
    everyone = everyone.view(world, *mine.shape)
    r = merge_token_records(everyone, [0] * world if starts is None else starts)
    return tuple(None if t is None else t.reshape(*targets.shape, *t.shape[1:]) for t in r), everyone


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top, lo, group, starts):
        out, records = _forward(logits, targets, top, lo, group, starts)
        if records is not None:  # a target that no shard holds has no gradient on any
            targets = targets.masked_fill((records[:, :, 3] == math.inf).all(0).view(targets.shape), -1)
        ctx.save_for_backward(logits, targets, out[2], out[1])
        ctx.lo, ctx.sharded = lo, group is not None
        if top:
            ctx.mark_non_differentiable(out[3], out[4])
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logprob, g_entropy, g_lse, *_):
        logits, targets, lse, entropy = ctx.saved_tensors
        if not ctx.needs_input_grad[0]:
            return None, None, None, None, None, None
        return (token_logprobs_grad(logits, targets, lse, entropy, g_logprob, g_entropy, grad_lse=g_lse, lo=ctx.lo, sharded=ctx.sharded),
                None, None, None, None, None)


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, *, top: int = 0, lo: int = 0,
                   group: Optional[dist.ProcessGroup] = None, starts: Optional[Sequence[int]] = None) -> TokenLogprobs:
    """Log probability of targets[i] under softmax(logits[i]), the entropy, the log-sum-exp, and the `top`
    (0..32) most probable tokens, largest first, ties to the lowest index; float32, summed in 32 bits.

    logits: [*targets.shape, cols], rows of any stride; column j is vocabulary index lo + j. A target
    outside the vocabulary (-1, -100) is none: its log probability is 0 and has no gradient. A
    vocabulary of fewer than `top` tokens fills up with index -1 and -inf. Logits of -inf (a mask)
    have probability 0; a row of nothing else has lse and log probabilities -inf, entropy 0 and gradient 0.

    With `group`, the ranks of a TP group that hold the vocabulary's shards in rank order (of any sizes), the
    result is that of the whole vocabulary on every rank; `starts`: the shards' first indices, needed only past
    31 bits. logprob, entropy and lse are differentiable with respect to logits."""
    if logits.requires_grad and torch.is_grad_enabled():
        return TokenLogprobs(*_TokenLogprobs.apply(logits, targets, top, lo, group, starts))
    return TokenLogprobs(*_forward(logits, targets, top, lo, group, starts)[0])


def token_logprobs_grad(logits: torch.Tensor, targets: torch.Tensor, lse: torch.Tensor, entropy: Optional[torch.Tensor],
                        grad_logprob: torch.Tensor, grad_entropy: Optional[torch.Tensor] = None, *,
                        grad_lse: Optional[torch.Tensor] = None, lo: int = 0, sharded: bool = False,
                        vocab: Optional[Tuple[int, int]] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gradient of token_logprobs' logits, in their shape and type, from the gradients of logprob,
    entropy and lse (float32). lse and entropy are token_logprobs' own. `out` may be the logits themselves.
    sharded=True: the logits are one of several shards; probabilities then come from lse alone, whose 32
    bits leave them off by |lse| 2^-24 (a whole row with |lse| over 1024 has its maximum and sum taken
    again). A target outside this shard is another's if it lies in `vocab`, the whole vocabulary's [first, end),
    and none otherwise. Without `vocab` negative targets alone are none: give it where others may
    lie outside the vocabulary (autograd through token_logprobs needs no telling)."""
    if vocab is not None and not sharded:
        raise ValueError("vocab is given with sharded=True")
    first, end = vocab if vocab is not None else (None, None)
    return L.extension().token_logprobs_grad(logits, targets, lse, entropy, grad_logprob, grad_entropy, grad_lse, lo, sharded, out, first, end)
