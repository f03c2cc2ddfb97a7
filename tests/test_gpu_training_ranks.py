"""The training-step operators on a migrated state and over a group of ranks.

test_next_step_from_the_reference: the reference's own next training step (tests/golden/next_step_losses.json) on the
state that the reshard moved, with the embedding, the cross entropy and AdamW of both target ranks done by the
operators on the ranks' shards (the transformer blocks by torch).
test_operators_over_a_group: one process per rank; with fewer GPUs than ranks both share cuda:0 (gloo). No kernel
waits on another rank.
"""
import datetime
import json
import os
import tempfile
import traceback

import numpy as np
import pytest
import torch

from suika_b200 import migration as M
from suika_b200 import optimizer as OPT
from suika_b200 import synthetic as S
from suika_b200 import vocab as V
from tests import next_step as NS
from tests.golden.cases import CASES
from tests.helpers import GOLDEN_DIR, SUBS, load_golden

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def test_next_step_from_the_reference():
    with open(os.path.join(GOLDEN_DIR, "next_step_losses.json")) as f:
        gold = json.load(f)["reference_order"]
    g, cfg = load_golden("next_step"), CASES["next_step"]["config"]
    spl, tpl = cfg.layouts()
    kinds = dict(SUBS)
    src = {r: {n: {s: S.to_torch(a, kinds[s], DEV if kinds[s] != "meta" else None) for s, a in e.items()} for n, e in st.items()}
           for r, st in S.host_states(spl, SUBS, seed=g["seed"], distinct_steps=True).items()}
    states = M.reshard_local(spl, tpl, src, S.expected_sub_fields(), DEV, order="reference", minimum_est_peers=g["minimum_est_peers"])
    ranks = sorted(states)
    ids = NS.tokens(cfg.spec).to(DEV)
    model = NS.LlamaStage(NS.llama_config(cfg.spec)).float().to(DEV)
    metas = tpl.layout

    def whole(name):
        m = metas[0][name]
        parts = [states[r][name]["param"].float() for r in ranks]
        return parts[0] if m.tp_meta is None else torch.cat(parts, m.tp_meta[0])

    def load():
        with torch.no_grad():
            model.load_state_dict({n: whole(n) for n in metas[0]}, strict=True)
        model.zero_grad(set_to_none=True)

    def forward():
        """(loss, per-rank logits, log probabilities, embedding output): the ends on the ranks' shards."""
        wte = states[0]["wte.weight"]["param"].float()  # replicated in this layout: every rank has it all
        x = V.embedding(ids, wte).requires_grad_()
        rope = model.rotary_emb(x, torch.arange(ids.shape[1], device=DEV).unsqueeze(0))
        h = x
        for block in model.h:
            h = block(h, attention_mask=None, position_embeddings=rope)
        h = model.norm(h)[:, :-1].reshape(-1, cfg.spec.hidden)
        heads = [states[r]["lm_head.weight"]["param"].float().requires_grad_() for r in ranks]
        z = [h @ w.t() for w in heads]
        starts = [V.shard_range(metas[r]["lm_head.weight"])[0] for r in ranks]
        t = ids[:, 1:].reshape(-1)
        recs = torch.stack([V.token_record(zr.detach(), t, lo=lo) for zr, lo in zip(z, starts)])
        lp = V.merge_token_records(recs, starts)
        return -lp.logprob.mean(), z, lp, starts, t, heads, x

    load()
    loss, z, lp, starts, t, heads, x = forward()
    # sums of at most 256 products in 32 bits on both sides, a few hundred roundings on each path: 2e-5 of the value
    want, after = float.fromhex(gold["loss"]), float.fromhex(gold["loss_after"])
    assert abs(float(loss) - want) <= 2e-5 * want
    gl = torch.full_like(lp.logprob, -1.0 / t.numel())
    torch.autograd.backward(z, [V.token_logprobs_grad(zr.detach(), t, lp.lse, lp.entropy, gl, lo=lo, sharded=True) for zr, lo in zip(z, starts)])
    full = {n: p.grad for n, p in model.named_parameters() if p.grad is not None}
    full["wte.weight"] = V.embedding_grad(x.grad, ids, cfg.spec.vocab)
    for i, r in enumerate(ranks):
        grads = {}
        for n, m in metas[r].items():
            if n == "lm_head.weight":
                grads[n] = heads[i].grad
            elif m.tp_meta is None:
                grads[n] = full[n]
            else:
                grads[n] = full[n].chunk(m.tp_meta[2], dim=m.tp_meta[0])[m.tp_meta[1]].contiguous()
        OPT.ShardAdamW(states[r], lr=NS.LR, betas=NS.BETAS, eps=NS.EPS, weight_decay=NS.WEIGHT_DECAY).step(grads)
    load()
    # as above, and a handful of bf16 weights that round to the other side
    assert abs(float(forward()[0]) - after) <= 5e-5 * after


def _worker(rank, world, port, outdir):
    res = {}
    try:
        os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), NCCL_NVLS_ENABLE="0")
        import torch.distributed as dist
        from tests.helpers import rank_device
        dev, backend = rank_device(rank, world)
        torch.cuda.set_device(dev)
        dist.init_process_group(backend, rank=rank, world_size=world, timeout=datetime.timedelta(seconds=300))
        group = dist.group.WORLD
        gen = torch.Generator().manual_seed(5)  # the same whole tensors on every rank
        rows, hidden, n = 60, 24, 33
        w = torch.randn(rows, hidden, generator=gen).to(dev, torch.bfloat16)
        ids = torch.randint(-1, rows, (n,), generator=gen).to(dev)
        z = (torch.randn(n, rows, generator=gen) * 2).to(dev)
        t = torch.randint(-1, rows, (n,), generator=gen).to(dev)
        gl, gh = torch.randn(n, generator=gen).to(dev), torch.randn(n, generator=gen).to(dev)
        per = rows // world
        lo = rank * per
        mine = w[lo:lo + per].clone().requires_grad_()
        out = V.embedding(ids, mine, lo=lo, group=group)
        res["embedding"] = bool(torch.equal(out, V.embedding(ids, w)))
        out.float().sum().backward()
        res["embedding_grad"] = bool(torch.equal(mine.grad, V.embedding_grad(torch.ones_like(out), ids, rows)[lo:lo + per]))
        part = z[:, lo:lo + per].clone().requires_grad_()
        r = V.token_logprobs(part, t, top=7, lo=lo, group=group)
        whole = V.token_logprobs(z, t, top=7)
        res["index"] = bool(torch.equal(r.top_index, whole.top_index))
        res["off"] = [float((a - b).detach().abs().max()) for a, b in zip(r[:4], whole[:4])]
        ((r.logprob * gl).sum() + (r.entropy * gh).sum()).backward()
        ref = V.token_logprobs_grad(z, t, whole.lse, whole.entropy, gl, gh)[:, lo:lo + per]
        res["off"].append(float((part.grad - ref).abs().max()))
        shared, own = torch.randn(50, generator=gen).to(dev), torch.randn(40, generator=gen).to(dev) + rank
        counted = {"own": [(0, 40)], "shared": [(0, 50)] if rank == 0 else []}
        grads = {"own": own.clone(), "shared": shared.clone()}
        norm = OPT.clip_grads(grads, 1.0, counted=counted, group=group)
        base = own - rank
        total = float(shared.double().square().sum()) + sum(float((base.double() + k).square().sum()) for k in range(world))
        res["norm"] = [float(norm), total ** 0.5]
        res["clipped"] = float((grads["shared"] - shared / (total ** 0.5 + 1e-6)).abs().max())
        state = {n: {"param": torch.zeros_like(g), "exp_avg": torch.zeros_like(g), "exp_avg_sq": torch.zeros_like(g), "step": torch.tensor(0.0)}
                 for n, g in (("own", own), ("shared", shared))}
        res["step_norm"] = float(OPT.ShardAdamW(state, max_norm=1.0, counted=counted, group=group).step({"own": own, "shared": shared}))
        res["state"] = float(state["own"]["step"])
        dist.barrier()
        dist.destroy_process_group()
    except Exception:
        res["error"] = traceback.format_exc()
    with open(os.path.join(outdir, f"rank{rank}.json"), "w") as f:
        json.dump(res, f)


@pytest.mark.parametrize("world", [2, 3])
def test_operators_over_a_group(world):
    import torch.multiprocessing as mp
    with tempfile.TemporaryDirectory() as d:
        mp.spawn(_worker, args=(world, 29760 + world, d), nprocs=world, join=True)
        results = [json.load(open(os.path.join(d, f"rank{r}.json"))) for r in range(world)]
    for r in results:
        assert "error" not in r, r.get("error")
        assert r["embedding"] and r["embedding_grad"] and r["index"]
        # the sums of 60 exponentials are taken in another order: 100 roundings of values of at most 12
        assert max(r["off"]) <= 100 * 2.0 ** -24 * 12, r["off"]
        assert abs(r["norm"][0] - r["norm"][1]) <= 18 * 2.0 ** -24 * r["norm"][1] and r["step_norm"] == r["norm"][0]
        assert r["clipped"] <= 25 * 2.0 ** -24 and r["state"] == 1.0
