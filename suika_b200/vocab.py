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
embedding and token_logprobs are differentiable (torch.autograd). Every call is stream-ordered on the
current stream of the tensors' device and can be captured. There is no CPU path.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional, Sequence, Tuple

import numpy as np
import torch
import torch.distributed as dist
from torch.autograd.function import once_differentiable

from . import _lib as L
from .layouts import shard_spans
from .optimizer import DTYPE_CODES, raw_stream

MAX_TOP = 32
_MAX_SORTED = 65536  # tokens that one cluster sorts; longer batches are taken in parts


def shard_range(meta) -> Tuple[int, int]:
    """[lo, hi): the rows that a TensorMeta (sliced on dim 0, or whole) holds of its full tensor."""
    if meta.tp_meta is None:
        return 0, int(meta.shape[0])
    if meta.tp_meta[0] % len(meta.shape) != 0 or getattr(meta, "tp_rule", None):
        raise ValueError(f"{meta.name}: not one contiguous range of rows")
    return shard_spans(meta.shape, meta.tp_meta)[0]


def _dtype_code(t: torch.Tensor, what: str) -> int:
    code = DTYPE_CODES.get(t.dtype)
    if code is None:
        raise ValueError(f"{what} of {t.dtype}: float32, bfloat16 and float16 are taken")
    return code


def _check_index(t: torch.Tensor, dev: torch.device, what: str) -> torch.Tensor:
    if t.dtype != torch.int64 and t.dtype != torch.int32:
        raise ValueError(f"{what} of {t.dtype}: int64 and int32 are taken")
    if t.device != dev:
        raise ValueError(f"{what} must be on the device of the other tensors")
    return t if t.is_contiguous() else t.contiguous()


def _check_cuda(t: torch.Tensor, what: str) -> torch.device:
    dev = t.device
    if dev.type != "cuda":
        raise ValueError(f"{what} must be a CUDA tensor")
    return dev


# ---------------------------------------------------------------------------------------------
# Embedding
# ---------------------------------------------------------------------------------------------
def _lookup(ids: torch.Tensor, weight: torch.Tensor, scale: float, lo: int, group) -> torch.Tensor:
    dev = _check_cuda(weight, "weight")
    if weight.dim() != 2:
        raise ValueError("weight must be [rows, hidden]")
    rows, hidden = weight.shape
    code = _dtype_code(weight, "weight")
    stride = weight.stride()
    if stride[1] != 1 and hidden > 1:
        raise ValueError("weight must have contiguous rows")
    ids = _check_index(ids, dev, "ids")
    out = torch.empty((*ids.shape, hidden), dtype=weight.dtype, device=dev)
    opts = L.RsEmbedOpts(ids.numel(), rows, hidden, lo, stride[0], 0, scale, code, code, ids.dtype == torch.int64, 0, 0)
    L.check(L.load().rs_embed_lookup(C.byref(opts), ids.data_ptr(), weight.data_ptr(), out.data_ptr(), dev.index, raw_stream(dev.index)))
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


def embedding_grad(grad_out: torch.Tensor, ids: torch.Tensor, rows: int, *, scale: float = 1.0, lo: int = 0,
                   dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None, accumulate: bool = False) -> torch.Tensor:
    """The gradient of embedding()'s weight, [rows, hidden]: row r is scale * the sum of grad_out over
    the tokens with id lo + r, summed in 32 bits in an order that the ids alone fix, and rounded
    once to `dtype` (default: grad_out's, or out's). `out` (contiguous) receives it; with accumulate=True it is
    added to what `out` holds. Rows without a token are 0 (left alone when accumulating).

    More than 65536 tokens are taken in parts of that many; for a 16-bit gradient the parts meet in a
    float32 one, so that it is rounded once all the same."""
    dev = _check_cuda(grad_out, "grad_out")
    hidden = grad_out.shape[-1]
    code = _dtype_code(grad_out, "grad_out")
    ids = _check_index(ids, dev, "ids")
    n = ids.numel()
    if tuple(grad_out.shape[:-1]) != tuple(ids.shape):
        raise AssertionError(f"grad_out has shape {list(grad_out.shape)}, ids {list(ids.shape)}")
    if out is None:
        if accumulate:
            raise ValueError("accumulate=True adds to `out`: give one")
        out = torch.empty((rows, hidden), dtype=dtype or grad_out.dtype, device=dev)
    else:
        if out.device != dev or not out.is_contiguous():
            raise ValueError("out must be contiguous and on grad_out's device")
        if tuple(out.shape) != (rows, hidden):
            raise AssertionError(f"out has shape {list(out.shape)}, expected {[rows, hidden]}")
        if dtype is not None and out.dtype != dtype:
            raise ValueError(f"out of {out.dtype}, but a gradient of {dtype} is asked for")
    out_code = _dtype_code(out, "the gradient")
    g = grad_out if grad_out.dim() == 2 else grad_out.reshape(-1, hidden)
    if g.stride(1) != 1 and hidden > 1:
        g = g.contiguous()
    if n > _MAX_SORTED:
        return _grad_in_parts(g, ids.reshape(-1), rows, scale, lo, out, accumulate)
    lib, stream = L.load(), raw_stream(dev.index)
    opts = L.RsEmbedOpts(n, rows, hidden, lo, 0, g.stride(0), scale, code, out_code, ids.dtype == torch.int64, accumulate, 0)
    nb = C.c_uint64()
    L.check(lib.rs_embed_grad_workspace_bytes(C.byref(opts), dev.index, C.byref(nb)))
    workspace = torch.empty(nb.value, dtype=torch.uint8, device=dev)
    L.check(lib.rs_embed_grad(C.byref(opts), ids.data_ptr(), g.data_ptr(), out.data_ptr(), workspace.data_ptr(), nb.value, dev.index, stream))
    return out


def _grad_in_parts(g: torch.Tensor, ids: torch.Tensor, rows: int, scale: float, lo: int, out: torch.Tensor, accumulate: bool) -> torch.Tensor:
    wide = out if out.dtype == torch.float32 else torch.empty(out.shape, dtype=torch.float32, device=out.device)
    for at in range(0, ids.numel(), _MAX_SORTED):
        embedding_grad(g[at:at + _MAX_SORTED], ids[at:at + _MAX_SORTED], rows, scale=scale, lo=lo, out=wide,
                       accumulate=at > 0 or (accumulate and wide is out))
    if wide is not out:
        out.copy_(wide.add_(out) if accumulate else wide)
    return out


# ---------------------------------------------------------------------------------------------
# Token log probabilities
# ---------------------------------------------------------------------------------------------
class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor                  # float32, targets' shape
    entropy: torch.Tensor
    lse: torch.Tensor                      # log-sum-exp of the row
    top_logprob: Optional[torch.Tensor]    # [*targets.shape, top], largest first
    top_index: Optional[torch.Tensor]      # int64 vocabulary indices


def _rows(logits: torch.Tensor, targets: torch.Tensor):
    dev = _check_cuda(logits, "logits")
    code = _dtype_code(logits, "logits")
    targets = _check_index(targets, dev, "targets")
    if logits.shape[:-1] != targets.shape:
        raise AssertionError(f"logits have shape {list(logits.shape)}, targets {list(targets.shape)}")
    cols = logits.shape[-1]
    if cols == 0:
        raise ValueError("logits of no columns")
    z = logits if logits.dim() == 2 else logits.reshape(-1, cols)
    if z.stride(1) != 1 and cols > 1:
        z = z.contiguous()
    return z, targets, dev, code


def _opts(z: torch.Tensor, targets: torch.Tensor, code: int, lo: int, top: int, sharded: bool) -> L.RsLogprobOpts:
    return L.RsLogprobOpts(z.shape[0], z.shape[1], z.stride(0), lo, code, targets.dtype == torch.int64, top, sharded)


def _outputs(shape, n: int, top: int, dev: torch.device):
    logprob, entropy, lse = torch.empty((3, *shape), dtype=torch.float32, device=dev).unbind(0)
    if not top:
        return logprob, entropy, lse, None, None
    return (logprob, entropy, lse, torch.empty((*shape, top), dtype=torch.float32, device=dev),
            torch.empty((*shape, top), dtype=torch.int64, device=dev))


def _check_top(top: int) -> None:
    if not 0 <= top <= MAX_TOP:
        raise ValueError(f"top must be in 0..{MAX_TOP}")


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def token_record(logits: torch.Tensor, targets: torch.Tensor, *, top: int = 0, lo: int = 0) -> torch.Tensor:
    """One vocabulary shard's part of token_logprobs: float32 [rows, 4 + 2 top], for merge_token_records."""
    _check_top(top)
    z, targets, dev, code = _rows(logits, targets)
    opts = _opts(z, targets, code, lo, top, True)
    out = torch.empty((z.shape[0], 4 + 2 * top), dtype=torch.float32, device=dev)
    L.check(L.load().rs_token_record(C.byref(opts), z.data_ptr(), targets.data_ptr(), out.data_ptr(), dev.index, raw_stream(dev.index)))
    return out


def merge_token_records(records: torch.Tensor, starts: Sequence[int]) -> TokenLogprobs:
    """token_logprobs from all shards' records, [shards, rows, 4 + 2 top]; starts[s] is the first
    vocabulary index of shard s, ascending (at most 64 shards)."""
    dev = _check_cuda(records, "records")
    if records.dim() != 3 or records.dtype != torch.float32 or not records.is_contiguous() or records.shape[2] < 4 or records.shape[2] % 2:
        raise ValueError("records must be a contiguous float32 [shards, rows, 4 + 2 top]")
    shards, n, words = records.shape
    if len(starts) != shards:
        raise AssertionError(f"{len(starts)} starts for {shards} shards")
    top = (words - 4) // 2
    out = _outputs((n,), n, top, dev)
    at = np.array([int(s) for s in starts], dtype=np.int64)
    L.check(L.load().rs_token_merge(records.data_ptr(), at.ctypes.data, shards, n, top, *map(_ptr, out), dev.index, raw_stream(dev.index)))
    return TokenLogprobs(*out)


def _forward(logits, targets, top, lo, group, starts):
    _check_top(top)
    z, targets, dev, code = _rows(logits, targets)
    if group is not None:
        world = dist.get_world_size(group)
        if starts is None:  # equal shards in rank order
            starts = [lo + (r - dist.get_rank(group)) * z.shape[1] for r in range(world)]
        mine = token_record(z, targets.reshape(-1), top=top, lo=lo)
        everyone = torch.empty((world, *mine.shape), dtype=mine.dtype, device=dev)
        dist.all_gather_into_tensor(everyone, mine, group=group)
        r = merge_token_records(everyone, starts)
        return tuple(None if t is None else t.reshape(*targets.shape, *t.shape[1:]) for t in r)
    out = _outputs(targets.shape, z.shape[0], top, dev)
    opts = _opts(z, targets, code, lo, top, False)
    L.check(L.load().rs_token_logprobs(C.byref(opts), z.data_ptr(), targets.data_ptr(), *map(_ptr, out), dev.index, raw_stream(dev.index)))
    return out


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top, lo, group, starts):
        out = _forward(logits, targets, top, lo, group, starts)
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

    With `group`, the ranks of a TP group that hold the vocabulary's shards in rank order, the result is
    that of the whole vocabulary on every rank; `starts`: the shards' first indices (default: equal
    shards). logprob, entropy and lse are differentiable with respect to logits."""
    if logits.requires_grad and torch.is_grad_enabled():
        return TokenLogprobs(*_TokenLogprobs.apply(logits, targets, top, lo, group, starts))
    return TokenLogprobs(*_forward(logits, targets, top, lo, group, starts))


def _row_values(t: Optional[torch.Tensor], shape, dev: torch.device, what: str) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.shape != shape or t.dtype != torch.float32 or t.device != dev:
        raise ValueError(f"{what} must be float32, of targets' shape and on their device")
    return t if t.is_contiguous() else t.contiguous()


def token_logprobs_grad(logits: torch.Tensor, targets: torch.Tensor, lse: torch.Tensor, entropy: Optional[torch.Tensor],
                        grad_logprob: torch.Tensor, grad_entropy: Optional[torch.Tensor] = None, *,
                        grad_lse: Optional[torch.Tensor] = None, lo: int = 0, sharded: bool = False,
                        out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gradient of token_logprobs' logits, in their shape and type, from the gradients of logprob,
    entropy and lse (float32). lse and entropy are token_logprobs' own. sharded=True: the logits are
    one of several shards, and a target outside it is another's. `out` may be the logits themselves."""
    z, targets, dev, code = _rows(logits, targets)
    if grad_entropy is not None and entropy is None:
        raise ValueError("a gradient of the entropy needs the entropy")
    rows = [_row_values(t, targets.shape, dev, w) for t, w in
            ((lse, "lse"), (entropy, "entropy"), (grad_logprob, "grad_logprob"), (grad_entropy, "grad_entropy"), (grad_lse, "grad_lse"))]
    if rows[0] is None or rows[2] is None:
        raise ValueError("lse and grad_logprob are needed")
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
    elif out.shape != logits.shape or out.dtype != logits.dtype or out.device != dev:
        raise ValueError("out must have the logits' shape, type and device")
    o = out if out.dim() == 2 else out.view(-1, z.shape[1])
    if o.stride(1) != 1 and z.shape[1] > 1:
        raise ValueError("out must have contiguous rows")
    opts = _opts(z, targets, code, lo, 0, sharded)
    L.check(L.load().rs_token_logprobs_grad(C.byref(opts), z.data_ptr(), targets.data_ptr(), *map(_ptr, rows), o.data_ptr(),
                                            max(o.stride(0), o.shape[1]), dev.index, raw_stream(dev.index)))
    return out
