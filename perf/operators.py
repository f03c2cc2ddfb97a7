"""The operators of a training step around the transformer blocks: plain forms, cases and calls.

  clip      global gradient norm over many tensors and clipping in place
  adamw     gradient norm, clipping and the AdamW update of a rank's state sub-fields
  embed     scaled lookup in a vocabulary shard of the embedding, and its gradient
  logprobs  log probabilities of given tokens, entropy and top alternatives of a vocabulary
            shard's logits, and their gradient

run() computes them in elementary torch operations (own = False) or calls the package (own = True).
"""
import math

import torch

own = False

DEV = "cuda"
LR, BETA1, BETA2, EPS, DECAY = 3e-4, 0.9, 0.95, 1e-8, 0.1


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # clipping in a debugging run: one small Llama layer's bf16 gradients on one of 8 TP ranks
        {"name": "clip_one_layer", "op": "clip", "layers": 1, "hidden": 1024, "ffn": 2816, "tp": 8, "vocab": 0,
         "grad": "bfloat16", "max_norm": 1.0},
        # fp32 accumulated gradients of a 7B Llama on one of 8 TP ranks, embeddings included
        {"name": "clip_7b_rank", "op": "clip", "layers": 32, "hidden": 4096, "ffn": 11008, "tp": 8, "vocab": 32000,
         "grad": "float32", "max_norm": 1.0},
        # the update of a toy model with odd sizes: the step is all launch latency
        {"name": "adamw_odd_small", "op": "adamw", "layers": 2, "hidden": 205, "ffn": 611, "tp": 1, "vocab": 1003,
         "grad": "bfloat16", "param": "bfloat16", "moments": "float32", "master": True, "max_norm": 1.0},
        # bf16 parameters and bf16 moments without a master copy: what the reference's worker keeps
        {"name": "adamw_bf16_state", "op": "adamw", "layers": 8, "hidden": 1024, "ffn": 2816, "tp": 1, "vocab": 32000,
         "grad": "bfloat16", "param": "bfloat16", "moments": "bfloat16", "master": False, "max_norm": 0.0},
        # mixed-precision state of a 7B Llama on one of 8 ranks, fp32 gradients, clipped
        {"name": "adamw_7b_rank", "op": "adamw", "layers": 32, "hidden": 4096, "ffn": 11008, "tp": 8, "vocab": 32000,
         "grad": "float32", "param": "bfloat16", "moments": "float32", "master": True, "max_norm": 1.0},
        # one decoding step of a few sequences: lookup only, latency bound
        {"name": "embed_decode", "op": "embed", "tokens": 5, "vocab": 152064, "lo": 0, "rows": 152064, "hidden": 3584,
         "weight": "bfloat16", "grad": "none", "accumulate": False, "scale": 1.0, "pad": 0.0},
        # a training micro-batch on one of 2 vocabulary shards, bf16 gradient written whole
        {"name": "embed_train_shard", "op": "embed", "tokens": 8192, "vocab": 32000, "lo": 16000, "rows": 16000, "hidden": 4096,
         "weight": "bfloat16", "grad": "bfloat16", "accumulate": False, "scale": 64.0, "pad": 0.0},
        # a long padded batch on a whole large vocabulary, added to an fp32 gradient that is there
        {"name": "embed_accumulate", "op": "embed", "tokens": 30011, "vocab": 152064, "lo": 0, "rows": 152064, "hidden": 3584,
         "weight": "bfloat16", "grad": "float32", "accumulate": True, "scale": 1.0, "pad": 0.25},
        # sampling diagnostics of one decoding step: few rows, a large vocabulary, 20 alternatives
        {"name": "logprobs_decode", "op": "logprobs", "tokens": 3, "vocab": 152064, "lo": 0, "cols": 152064, "logits": "bfloat16",
         "top": 20, "grad": False, "masked": 0.0, "ignored": 0.0},
        # scoring given continuations with constrained (masked) vocabularies, fp32 logits
        {"name": "logprobs_score", "op": "logprobs", "tokens": 2047, "vocab": 50257, "lo": 0, "cols": 50257, "logits": "float32",
         "top": 5, "grad": False, "masked": 0.3, "ignored": 0.0},
        # a short training sequence, loss and its gradient
        {"name": "logprobs_train_short", "op": "logprobs", "tokens": 129, "vocab": 32000, "lo": 0, "cols": 32000, "logits": "float16",
         "top": 0, "grad": True, "masked": 0.0, "ignored": 0.1},
        # a training micro-batch over a large vocabulary, loss, entropy term and their gradient
        {"name": "logprobs_train", "op": "logprobs", "tokens": 4096, "vocab": 152064, "lo": 0, "cols": 152064, "logits": "bfloat16",
         "top": 0, "grad": True, "masked": 0.0, "ignored": 0.2},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["clip", "adamw", "embed", "logprobs"])
    if op in ("clip", "adamw"):
        hidden = _log_int(rng, 64, 4096)
        case = {"op": op, "layers": _log_int(rng, 1, 24), "hidden": hidden, "ffn": int(hidden * rng.uniform(2.0, 3.0)),
                "tp": rng.choice([1, 2, 4, 8]) if hidden <= 2048 else 8, "vocab": rng.choice([0, _log_int(rng, 100, 32000)]),
                "grad": rng.choice(["bfloat16", "float16", "float32"]), "max_norm": rng.choice([0.5, 1.0, 20.0])}
        if op == "adamw":
            case["master"] = rng.choice([True, True, False])
            case["param"] = rng.choice(["bfloat16", "float16"]) if case["master"] else rng.choice(["bfloat16", "float32"])
            case["moments"] = "float32" if case["master"] else rng.choice(["bfloat16", "float32"])
            case["max_norm"] = rng.choice([0.0, case["max_norm"]])
        return case
    if op == "embed":
        vocab = _log_int(rng, 500, 152064)
        rows = vocab if rng.random() < 0.5 else max(1, vocab // rng.choice([2, 4, 8]))
        lo = rng.randrange(0, vocab - rows + 1)
        weight = rng.choice(["bfloat16", "float16", "float32"])
        grad = rng.choice(["none", weight, "float32"])
        return {"op": op, "tokens": _log_int(rng, 1, 30000), "vocab": vocab, "lo": lo, "rows": rows, "hidden": _log_int(rng, 33, 3584),
                "weight": weight, "grad": grad, "accumulate": grad != "none" and rng.random() < 0.4, "scale": rng.choice([1.0, 0.5, 45.3]),
                "pad": rng.choice([0.0, 0.0, 0.3, 0.9])}
    vocab = _log_int(rng, 100, 152064)
    cols = vocab if rng.random() < 0.7 else max(32, vocab // rng.choice([2, 4]))
    grad = rng.random() < 0.5
    logits = rng.choice(["bfloat16", "float16", "float32"])
    most = max(2, min(8192, (300_000_000 if logits == "float32" else 600_000_000) // cols))
    return {"op": op, "tokens": _log_int(rng, 1, most), "vocab": vocab, "lo": rng.randrange(0, vocab - cols + 1), "cols": cols,
            "logits": logits, "top": rng.choice([0, 1, 5, 20, 32]), "grad": grad, "masked": rng.choice([0.0, 0.0, 0.5, 0.95]),
            "ignored": rng.choice([0.0, 0.3])}


def _shapes(case):
    """Shard shapes of a Llama rank: the order and slicing of its decoder layers, then wte, lm_head and the last norm."""
    h, f, tp = case["hidden"], max(case["tp"], case["ffn"] // case["tp"] * case["tp"]), case["tp"]
    hs, fs = max(1, h // tp), f // tp
    out = [(hs, h), (hs, h), (hs, h), (h, hs), (fs, h), (fs, h), (h, fs), (h,), (h,)] * case["layers"]
    if case["vocab"]:
        out = out + [(case["vocab"], h), (max(1, case["vocab"] // tp), h), (h,)]
    return out


def _spans(case):
    """[(offset, numel, shape)] of each tensor in an arena with 64-element aligned slots, and the arena's length."""
    at, out = 0, []
    for s in _shapes(case):
        n = math.prod(s)
        out.append((at, n, s))
        at = (at + n + 63) // 64 * 64
    return out, at


def _itemsize(name):
    return getattr(torch, name).itemsize


def work(case):
    if case["op"] in ("clip", "adamw"):
        n = sum(m for _, m, _ in _spans(case)[0])
        g = _itemsize(case["grad"])
        if case["op"] == "clip":
            return {"bytes": 2 * g * n, "flops": 3 * n}
        p, m = _itemsize(case["param"]), _itemsize(case["moments"])
        return {"bytes": n * (g + 4 * m + (8 + p if case["master"] else 2 * p)), "flops": 17 * n}
    if case["op"] == "embed":
        n, h, w = case["tokens"], case["hidden"], _itemsize(case["weight"])
        rows = min(n, case["rows"])
        bytes_, flops = 8 * n + (rows + n) * h * w, n * h
        if case["grad"] != "none":
            g = _itemsize(case["grad"])
            bytes_ += n * h * w + (2 * rows if case["accumulate"] else case["rows"]) * h * g
            flops += n * h
        return {"bytes": bytes_, "flops": flops}
    n, b = case["tokens"] * case["cols"], _itemsize(case["logits"])
    return {"bytes": n * b * (2 if case["grad"] else 1) + 40 * case["tokens"], "flops": n * (14 if case["grad"] else 6)}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _names(case):
    return ["t%d.weight" % i for i in range(len(_spans(case)[0]))]


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    s = {"case": dict(case)}
    if case["op"] in ("clip", "adamw"):
        spans, total = _spans(case)
        s["spans"] = spans
        grad = torch.zeros(total, dtype=getattr(torch, case["grad"]), device=DEV)
        views = [grad[o:o + n].view(shape) for o, n, shape in spans]
        for v in views:  # the padding between tensors stays zero
            v.copy_(torch.randn(v.shape, generator=g, device=DEV).mul_(1e-3))
        s["grad"] = grad
        s["grads"] = dict(zip(_names(case), views))
        # the other ranks' share of the sum of squares, as an all-reduce brings it: a little over the limit,
        # so that every pass on the same gradients clips
        s["others"] = torch.full((1,), case["max_norm"] ** 2 * (1 + 1e-4), dtype=torch.float64, device=DEV)
        if case["op"] == "adamw":
            kinds = [("param", case["param"]), ("exp_avg", case["moments"]), ("exp_avg_sq", case["moments"])]
            if case["master"]:
                kinds.insert(1, ("master", "float32"))
            arenas = {k: torch.zeros(total, dtype=getattr(torch, t), device=DEV) for k, t in kinds}
            for o, n, shape in spans:
                w = torch.randn(n, generator=g, device=DEV).mul_(0.02)
                arenas["param"][o:o + n] = w.to(arenas["param"].dtype)
                if case["master"]:
                    arenas["master"][o:o + n] = w
                arenas["exp_avg"][o:o + n] = torch.randn(n, generator=g, device=DEV).mul_(1e-3).to(arenas["exp_avg"].dtype)
                arenas["exp_avg_sq"][o:o + n] = torch.randn(n, generator=g, device=DEV).square_().mul_(1e-6).to(arenas["exp_avg_sq"].dtype)
            step = torch.full((len(spans),), float(1 + int(seed) % 50), device=DEV)
            s.update(arenas=arenas, step=step)
            if own:
                from suika_b200.optimizer import ShardAdamW
                state = {}
                for i, (name, (o, n, shape)) in enumerate(zip(_names(case), spans)):
                    state[name] = {k: a[o:o + n].view(shape) for k, a in arenas.items()}
                    state[name]["step"] = step[i]
                s["optimizer"] = ShardAdamW(state, lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY,
                                            max_norm=case["max_norm"] or None)
        return s
    if case["op"] == "embed":
        n, h, w = case["tokens"], case["hidden"], getattr(torch, case["weight"])
        # token frequencies fall with the id, as in text sorted by frequency; shards start further down
        u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
        ids = (torch.pow(float(case["vocab"]), u) - 1).long().clamp_(0, case["vocab"] - 1)
        if case["lo"]:
            ids = (ids * 7919 + int(seed) % 1000) % case["vocab"]
        ids = torch.where(torch.rand(n, generator=g, device=DEV) < case["pad"], torch.full_like(ids, -1), ids)
        s["ids"] = ids
        s["weight"] = torch.empty(case["rows"], h, dtype=w, device=DEV).normal_(0, 0.02, generator=g)
        if case["grad"] != "none":
            s["grad_out"] = torch.empty(n, h, dtype=w, device=DEV).normal_(0, 1e-2, generator=g)
            if case["accumulate"]:
                s["acc"] = torch.empty(case["rows"], h, dtype=getattr(torch, case["grad"]), device=DEV).normal_(0, 1e-2, generator=g)
        return s
    n, v = case["tokens"], case["cols"]
    z = torch.empty(n, v, dtype=torch.float32, device=DEV).normal_(0, 2.5, generator=g)
    if case["masked"]:
        z.masked_fill_(torch.rand(n, v, generator=g, device=DEV) < case["masked"], -math.inf)
        z[:, 0] = 0.25  # a constrained vocabulary leaves something
    t = torch.randint(case["lo"], case["lo"] + v, (n,), generator=g, device=DEV)
    z.scatter_add_(1, (t - case["lo"]).unsqueeze(1), torch.full((n, 1), 6.0, device=DEV))
    t = torch.where(torch.isinf(z.gather(1, (t - case["lo"]).unsqueeze(1)).squeeze(1)), torch.full_like(t, case["lo"]), t)
    t = torch.where(torch.rand(n, generator=g, device=DEV) < case["ignored"], torch.full_like(t, -1), t)
    s["logits"], s["targets"] = z.to(getattr(torch, case["logits"])), t
    if case["grad"]:
        s["grad_logprob"] = torch.empty(n, device=DEV).normal_(-1.0, 0.2, generator=g)
        s["grad_entropy"] = torch.empty(n, device=DEV).normal_(0.0, 0.1, generator=g)
    return s


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    return {"clip": _clip, "adamw": _adamw, "embed": _embed, "logprobs": _logprobs}[case["op"]](case, state)


def _clip(case, s):
    if own:
        from suika_b200.optimizer import clip_grads, grad_sumsq
        norm = clip_grads(s["grads"], case["max_norm"], sumsq=grad_sumsq(s["grads"]).add_(s["others"]))
        return {"norm": norm.reshape(1), "grad": s["grad"]}
    g = s["grad"]
    norm = (g.float().square().sum(dtype=torch.float64) + s["others"]).sqrt().float()
    c = (case["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    g.copy_(g.float() * c)
    return {"norm": norm, "grad": g}


def _adamw(case, s):
    a, step = s["arenas"], s["step"]
    if own:
        norm = s["optimizer"].step(s["grads"])
        out = {"step": step, **a}
        return {"norm": norm, **out} if case["max_norm"] else out
    g = s["grad"].float()
    out = {}
    if case["max_norm"]:
        out["norm"] = g.square().sum(dtype=torch.float64).sqrt().float()
        g = g * (case["max_norm"] / (out["norm"] + 1e-6)).clamp(max=1.0)
    step += 1
    t = step[0].double()  # every tensor of the state is at the same step
    bc1, bc2 = (1 - BETA1 ** t).float(), (1 - BETA2 ** t).float()
    w = a["master"] if case["master"] else a["param"].float()
    m, v = a["exp_avg"].float(), a["exp_avg_sq"].float()
    w = w * (1 - LR * DECAY)
    m = m + (g - m) * (1 - BETA1)
    v = v * BETA2 + g * g * (1 - BETA2)
    w = w - (LR / bc1) * m / (v.sqrt() / bc2.sqrt() + EPS)
    if case["master"]:
        a["master"].copy_(w)
    a["param"].copy_(w)
    a["exp_avg"].copy_(m)
    a["exp_avg_sq"].copy_(v)
    return {**out, "step": step, **a}


def _embed(case, s):
    ids, lo, rows, scale = s["ids"], case["lo"], case["rows"], case["scale"]
    if own:
        from suika_b200.vocab import embedding, embedding_grad
        out = {"out": embedding(ids, s["weight"], scale=scale, lo=lo)}
        if case["grad"] != "none":
            out["grad"] = embedding_grad(s["grad_out"], ids, rows, scale=scale, lo=lo, dtype=getattr(torch, case["grad"]),
                                         out=s.get("acc"), accumulate=case["accumulate"])
        return out
    held = (ids >= lo) & (ids < lo + rows)
    at = torch.where(held, ids - lo, torch.zeros_like(ids))
    x = s["weight"][at].float() * scale
    out = {"out": torch.where(held.unsqueeze(1), x, torch.zeros_like(x)).to(s["weight"].dtype)}
    if case["grad"] != "none":
        dy = torch.where(held.unsqueeze(1), s["grad_out"].float(), torch.zeros_like(x)) * scale
        dw = torch.zeros(rows, case["hidden"], dtype=torch.float32, device=ids.device).index_add_(0, at, dy)
        out["grad"] = s["acc"].copy_(s["acc"].float() + dw) if case["accumulate"] else dw.to(getattr(torch, case["grad"]))
    return out


def _logprobs(case, s):
    z, t, lo, k = s["logits"], s["targets"], case["lo"], case["top"]
    if own:
        from suika_b200.vocab import token_logprobs, token_logprobs_grad
        r = token_logprobs(z, t, top=k, lo=lo)
        out = {"logprob": r.logprob, "entropy": r.entropy, "lse": r.lse}
        if k:
            out.update(top_logprob=r.top_logprob, top_index=r.top_index)
        if case["grad"]:
            out["grad"] = token_logprobs_grad(z, t, r.lse, r.entropy, s["grad_logprob"], s["grad_entropy"], lo=lo)
        return out
    x = z.float()
    m = x.amax(1, keepdim=True)
    e = (x - m).exp()
    total = e.sum(1, keepdim=True)
    lse = m + total.log()
    p = e / total
    log_p = x - lse
    entropy = -torch.where(p > 0, p * log_p, torch.zeros_like(p)).sum(1)
    known = (t >= lo) & (t < lo + case["cols"])
    at = torch.where(known, t - lo, torch.zeros_like(t)).unsqueeze(1)
    logprob = log_p.gather(1, at).squeeze(1)
    out = {"logprob": torch.where(known, logprob, torch.zeros_like(logprob)), "entropy": entropy, "lse": lse.squeeze(1)}
    if k:
        best, index = x.sort(dim=1, descending=True, stable=True)
        out.update(top_logprob=best[:, :k] - lse, top_index=index[:, :k] + lo)
    if case["grad"]:
        gl = torch.where(known, s["grad_logprob"], torch.zeros_like(s["grad_logprob"])).unsqueeze(1)
        grad = -gl * p - s["grad_entropy"].unsqueeze(1) * torch.where(p > 0, p * (log_p + entropy.unsqueeze(1)), torch.zeros_like(p))
        out["grad"] = grad.scatter_add_(1, at, gl).to(z.dtype)
    return out


# ---------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embed":
        return _exact_embed(case, s)
    if case["op"] == "logprobs":
        return _exact_logprobs(case, s)
    grad = s["grad"].double()
    norm = torch.linalg.vector_norm(grad)
    if case["op"] == "clip":
        norm = (norm ** 2 + s["others"]) ** 0.5
    if case["max_norm"]:
        grad = grad * min(1.0, case["max_norm"] / (float(norm) + 1e-6))
    if case["op"] == "clip":
        return {"norm": norm, "grad": grad}
    a, t = s["arenas"], float(s["step"][0]) + 1
    m = BETA1 * a["exp_avg"].double() + (1 - BETA1) * grad
    v = BETA2 * a["exp_avg_sq"].double() + (1 - BETA2) * grad ** 2
    del grad
    w = a["master" if case["master"] else "param"].double()
    w = w - LR * DECAY * w - LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)) ** 0.5 + EPS)
    out = {"step": s["step"].double() + 1, "param": w, "exp_avg": m, "exp_avg_sq": v}
    if case["master"]:
        out["master"] = w
    if case["max_norm"]:
        out["norm"] = norm
    return out


def _exact_embed(case, s):
    ids = s["ids"] - case["lo"]
    mine = ((ids >= 0) & (ids < case["rows"])).nonzero().squeeze(1)
    x = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device=ids.device)
    x[mine] = s["weight"].double()[ids[mine]] * case["scale"]
    out = {"out": x}
    if case["grad"] != "none":
        dw = s["acc"].double() if case["accumulate"] else torch.zeros(case["rows"], case["hidden"], dtype=torch.float64, device=ids.device)
        out["grad"] = dw.index_put_((ids[mine],), s["grad_out"][mine].double() * case["scale"], accumulate=True)
    return out


def _exact_logprobs(case, s):
    z, k = s["logits"].double(), case["top"]
    lse = torch.logsumexp(z, 1)
    lp = z - lse.unsqueeze(1)
    p = lp.exp()
    plp = torch.nan_to_num(p * lp, nan=0.0)  # 0 * -inf
    entropy = -plp.sum(1)
    t = s["targets"] - case["lo"]
    hot = torch.arange(case["cols"], device=z.device).unsqueeze(0) == t.unsqueeze(1)
    out = {"logprob": torch.where(hot, lp, torch.zeros((), dtype=lp.dtype, device=lp.device)).sum(1), "entropy": entropy, "lse": lse}
    if k:  # the largest that is left, at its first place, k times
        left = z.clone()
        column = torch.arange(case["cols"], device=z.device).unsqueeze(0)
        taken = torch.zeros_like(hot)
        values, places = [], []
        for _ in range(k):
            best = torch.where(taken, -math.inf, left).amax(1, keepdim=True)
            place = torch.where(~taken & (left == best), column, case["cols"]).amin(1, keepdim=True)
            values.append(best - lse.unsqueeze(1))
            places.append(place + case["lo"])
            taken = taken.scatter(1, place, True)
        out.update(top_logprob=torch.cat(values, 1), top_index=torch.cat(places, 1))
    if case["grad"]:
        gl = torch.where((t >= 0) & (t < case["cols"]), s["grad_logprob"].double(), 0.0).unsqueeze(1)
        out["grad"] = gl * (hot.double() - p) - s["grad_entropy"].double().unsqueeze(1) * (plp + p * entropy.unsqueeze(1))
    return out
