"""The training-step operators at the edges of what their documentation allows, on a B200, against a plain
computation in 64 bits where numbers are compared."""
import ctypes
import datetime
import json
import math
import os
import tempfile
import threading
import time
import traceback

import pytest
import torch

from suika_b200 import _lib as L
from suika_b200 import optimizer as OPT
from suika_b200 import vocab as V
from tests.test_gpu_training import (BF16, DEV, F32, HYPER, TYPES, U, assert_close, clone_state, gen, grads_of, half, make_state, randn,
                                     ref_grad, ref_log_p, stat_rel, tiny)

pytestmark = pytest.mark.gpu


# ---- gradient of masked rows under large factors ------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [9, 33, 3001, 50257])
@pytest.mark.parametrize("factor", [1e2, 1e4, 65536.0, 1e30])
def test_masked_logits_have_no_gradient_whatever_the_entropys(dtype, cols, factor):
    """p = 0 gives 0 for every finite gradient of the entropy; the rest is the formula's, where the type holds it."""
    low, n = torch.finfo(dtype).min, 7
    z = randn(n, cols, dtype=dtype, scale=2.0, seed=cols)
    z[0, ::2] = -math.inf
    z[1, 5:] = low
    z[2, :3], z[2, -3:] = low, -math.inf
    z[3, 1:] = -math.inf
    z[4, 1::2] = low
    z[5, 2:] = -math.inf
    masked = (z == -math.inf) | (z == low)
    t = torch.tensor([1, 4, cols - 1, 0, 0, -1, 2], device=DEV)
    gl, gh, gz = grads_of(n, 3)
    gh = gh.sign() * (gh.abs() + 0.1) * factor
    r = V.token_logprobs(z, t)
    ref, size = ref_grad(z, t, 0, gl, gh, gz)
    hot = (torch.arange(cols, device=DEV).unsqueeze(0) == t.unsqueeze(1)) & masked  # a target that is masked has its own gradient
    lp, lse, _ = ref_log_p(z)
    # as for small factors: S's error and that of the exponent's argument, linear in the factor
    rel = 4 * stat_rel(z) + U * (6 + 4 * lp.abs().nan_to_num(0, 0, 0).clamp(max=120) + 4 * lse.abs().clamp(max=1024).unsqueeze(1))
    bound = rel * size + half(dtype) * ref.abs() + tiny(dtype) + 2.0 ** -126
    fits = ref.abs() + bound < torch.finfo(dtype).max
    wide = torch.zeros(n, cols + 9, dtype=dtype, device=DEV)
    own = z.clone()
    for out in (None, wide[:, 1:1 + cols], wide[:, 8:8 + cols], own):  # whole vectors, one logit at a time, both, in place
        src = own if out is own else z
        got = V.token_logprobs_grad(src, t, r.lse, r.entropy, gl, gh, grad_lse=gz, out=out)
        assert not got.isnan().any()
        assert (got[masked & ~hot] == 0).all()
        assert_close(torch.where(fits, got, 0), torch.where(fits, ref, 0), torch.where(fits, bound, 0))


# ---- targets that no shard holds --------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cuts", [[0, 500], [0, 1, 30, 500], [0, 100, 200, 300, 400, 500]])
def test_targets_outside_the_vocabulary_have_no_gradient_on_shards(dtype, cuts):
    n, lo, end = 8, 1000, 1500
    z = randn(n, 500, dtype=dtype, scale=2.0, seed=6)
    t = torch.tensor([end, end + 7, lo - 1, 0, -1, -100, end - 1, lo], device=DEV)
    gl, gh, gz = grads_of(n, 5)
    recs = torch.stack([V.token_record(z[:, a:b], t, lo=lo + a) for a, b in zip(cuts, cuts[1:])])
    r = V.merge_token_records(recs, [lo + a for a in cuts[:-1]])
    assert not r.logprob[:6].any() and r.logprob[6:].all()
    for tt in (t, t.int()):
        for h, g in ((gh, gz), (None, None)):
            ref, size = ref_grad(z, t, lo, gl, torch.zeros_like(gl) if h is None else h, torch.zeros_like(gl) if g is None else g)
            got = torch.cat([V.token_logprobs_grad(z[:, a:b], tt, r.lse, r.entropy, gl, h, grad_lse=g, lo=lo + a, sharded=True, vocab=(lo, end))
                             for a, b in zip(cuts, cuts[1:])], 1)
            assert_close(got, ref, 400 * U * size + half(dtype) * ref.abs() + tiny(dtype))
            if h is None:
                assert not got[:6].any()


def test_a_vocabulary_is_given_with_shards_only():
    z, t, f = torch.zeros(3, 8, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV), torch.zeros(3, device=DEV)
    with pytest.raises(ValueError, match="sharded"):
        V.token_logprobs_grad(z, t, f, f, f, vocab=(0, 8))
    for bad in ((4, 8), (0, 7), (8, 0)):
        with pytest.raises(RuntimeError, match="vocabulary"):
            V.token_logprobs_grad(z, t, f, f, f, sharded=True, vocab=bad)


class Ranks:
    """The collectives of suika_b200.vocab among ranks that run one after the other in this process."""

    def __init__(self, monkeypatch):
        monkeypatch.setattr(V, "dist", self)
        self.rank, self.parts = 0, []

    def get_world_size(self, group):
        return self.world

    def get_rank(self, group):
        return self.rank

    def all_gather_into_tensor(self, out, mine, group=None):
        if len(self.parts) < self.world:
            self.parts.append(mine.clone())
            raise StopIteration
        out.copy_(torch.cat(self.parts))

    def run(self, world, call):
        self.world, self.parts, done = world, [], []
        for self.rank in range(world):
            with pytest.raises(StopIteration):
                call(self.rank)
        for self.rank in range(world):
            done.append(call(self.rank))
        return done


@pytest.mark.parametrize("cuts", [[0, 250, 500], [0, 100, 200, 300, 400, 500]])
def test_targets_outside_the_vocabulary_over_a_group(monkeypatch, cuts):
    ranks, n = Ranks(monkeypatch), 8
    z = randn(n, 500, scale=2.0, seed=6)
    t = torch.tensor([500, 507, 1 << 40, 499, -1, -100, 250, 0], device=DEV)
    gl, gh, gz = grads_of(n, 5)
    leaves = [z[:, a:b].clone().requires_grad_() for a, b in zip(cuts, cuts[1:])]
    out = ranks.run(len(leaves), lambda r: V.token_logprobs(leaves[r], t, lo=cuts[r], group="ranks"))
    for r in out:
        ((r.logprob * gl).sum() + (r.entropy * gh).sum() + (r.lse * gz).sum()).backward()
    ref, size = ref_grad(z, t, 0, gl, gh, gz)
    assert_close(torch.cat([x.grad for x in leaves], 1), ref, 400 * U * size + 2.0 ** -126)


@pytest.mark.parametrize("dtype", TYPES)
def test_targets_that_are_none_on_rows_of_nan_and_infinity(dtype):
    """No target: log probability 0 and no gradient from it, whatever the row holds (the logits of padding are often NaN)."""
    n, cols = 6, 700
    z = randn(n, cols, dtype=dtype, seed=1)
    z[0, 3], z[1, 4], z[2], z[3, 600], z[4, 699] = math.nan, math.inf, math.nan, math.inf, math.inf
    none = torch.tensor([-1, -100, cols, 1 << 40, -1, -1], device=DEV)
    r = V.token_logprobs(z, none)
    assert (r.logprob == 0).all()
    held = torch.tensor([5, 4, 5, 600, 5, 5], device=DEV)  # two of them the infinite logit itself
    whole = V.token_logprobs(z, held)
    assert whole.logprob[:5].isnan().all() and whole.logprob[5].isfinite()
    gl = torch.ones(n, device=DEV)
    assert not V.token_logprobs_grad(z, none, r.lse, r.entropy, gl).any()
    cuts = [0, 100, 650, 700]
    for t, want in ((none, r.logprob), (held, whole.logprob)):
        recs = torch.stack([V.token_record(z[:, a:b], t, lo=a) for a, b in zip(cuts, cuts[1:])])
        got = V.merge_token_records(recs, cuts[:-1])
        assert torch.equal(got.logprob.isnan(), want.isnan())
        assert_close(got.logprob, want, 700 * U * 12)


# ---- a rank without gradients -----------------------------------------------------------------
def test_a_rank_without_gradients_takes_part_in_the_sum(monkeypatch):
    sums = []

    class Dist:
        @staticmethod
        def all_reduce(t, group=None):
            sums.append((t.clone(), group))
            t.add_(9.0)
    monkeypatch.setattr(OPT, "dist", Dist)
    for grads in ({}, {"a": None}, []):
        norm = OPT.clip_grads(grads, 1.0, group="ranks")
        assert norm.shape == () and norm.dtype == F32 and float(norm) == 3.0
    assert float(OPT.clip_grads({"a": None}, 1.0, counted={"a": [(0, 4)]}, group="ranks")) == 3.0
    state = make_state([10], BF16, F32, True)
    old = clone_state(state)
    opt = OPT.ShardAdamW(state, max_norm=1.0, group="ranks", **HYPER)
    for grads in ({}, {"t0": None}):
        norm = opt.step(grads)
        assert norm.shape == () and norm.dtype == F32 and float(norm) == 3.0
    assert len(sums) == 6 and all(float(s) == 0.0 and s.dtype == torch.float64 and s.is_cuda and g == "ranks" for s, g in sums)
    given = torch.full((1,), 16.0, dtype=torch.float64, device=DEV)
    assert float(opt.step({}, sumsq=given)) == 4.0 and float(OPT.clip_grads([], 1.0, sumsq=given, group="ranks")) == 4.0 and len(sums) == 6
    assert OPT.ShardAdamW(state, group="ranks", **HYPER).step({}) is None
    assert all(torch.equal(state[n][s], old[n][s]) for n in old for s in old[n])
    with pytest.raises(ValueError, match="no gradients"):  # alone there is nothing to take part in
        OPT.clip_grads({"a": None}, 1.0)
    with pytest.raises(ValueError, match="no gradients"):
        OPT.ShardAdamW(state, max_norm=1.0, **HYPER).step({})


def _empty_rank_worker(rank, world, port, outdir):
    res = {}
    try:
        os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), NCCL_NVLS_ENABLE="0")
        import torch.distributed as dist
        from tests.helpers import rank_device
        dev, backend = rank_device(rank, world)
        torch.cuda.set_device(dev)
        dist.init_process_group(backend, rank=rank, world_size=world, timeout=datetime.timedelta(seconds=60))
        grads = {"a": torch.full((4,), 2.0, device=dev)} if rank == 0 else {"a": None}
        res["clip"] = float(OPT.clip_grads(grads, 1.0, group=dist.group.WORLD))
        state = {"a": {"param": torch.ones(4, device=dev), "exp_avg": torch.zeros(4, device=dev), "exp_avg_sq": torch.zeros(4, device=dev),
                       "step": torch.tensor(0.0, device=dev)}}
        opt = OPT.ShardAdamW(state, max_norm=1.0, group=dist.group.WORLD)
        res["norm"] = float(opt.step({"a": torch.full((4,), 3.0, device=dev)} if rank == 0 else {}))
        res["step"] = float(state["a"]["step"])
        dist.barrier()
        dist.destroy_process_group()
    except Exception:
        res["error"] = traceback.format_exc()
    with open(os.path.join(outdir, f"rank{rank}.json"), "w") as f:
        json.dump(res, f)


def test_two_ranks_one_of_them_without_gradients():
    """One process per rank (gloo where they share a GPU); no kernel waits on the other rank."""
    import torch.multiprocessing as mp
    with tempfile.TemporaryDirectory() as d:
        mp.spawn(_empty_rank_worker, args=(2, 29790, d), nprocs=2, join=True)
        results = [json.load(open(os.path.join(d, f"rank{r}.json"))) for r in range(2)]
    for rank, r in enumerate(results):
        assert "error" not in r, r.get("error")
        assert r == {"clip": 4.0, "norm": 6.0, "step": 1.0 - rank}


# ---- shards of unequal size -------------------------------------------------------------------
@pytest.mark.parametrize("cuts", [[0, 1, 30, 500], [0, 300, 500], [7, 207, 407, 500], [0, 250, 500]])
@pytest.mark.parametrize("top", [0, 1, 32])
def test_unequal_shards_over_a_group_find_their_places(monkeypatch, cuts, top):
    ranks, n, z = Ranks(monkeypatch), 9, randn(9, 500, dtype=BF16, scale=2.0, seed=2)
    z[1], z[2, 40:] = 1.0, -math.inf
    z = z[:, :cuts[-1] - cuts[0]]
    t = cuts[0] + torch.randint(0, z.shape[1], (n,), generator=gen(1), device=DEV)
    whole = V.token_logprobs(z, t, top=top, lo=cuts[0])
    parts = [z[:, a - cuts[0]:b - cuts[0]] for a, b in zip(cuts, cuts[1:])]
    for starts in (None, cuts[:-1]):
        for r in ranks.run(len(parts), lambda i: V.token_logprobs(parts[i], t, top=top, lo=cuts[i], group="ranks", starts=starts)):
            assert_close(r.logprob, whole.logprob, 500 * U * 12)
            if top:
                assert torch.equal(r.top_index, whole.top_index)


def test_update_entry_without_tensors_gives_the_norm():
    lib, norm, ws = L.load(), torch.full((2,), 7.0, device=DEV), torch.zeros(1 << 20, dtype=torch.uint8, device=DEV)
    sumsq = torch.full((1,), 25.0, dtype=torch.float64, device=DEV)
    stream = torch.cuda.current_stream().cuda_stream
    for given, want in ((sumsq.data_ptr(), 5.0), (None, 0.0)):
        o = L.RsAdamwOpts(1e-3, 0.9, 0.99, 1e-8, 1.0)
        L.check(lib.rs_adamw_step(None, 0, ctypes.byref(o), given, norm.data_ptr(), ws.data_ptr(), ws.numel(), 0, stream))
        assert norm.tolist() == [want, 7.0]
    o = L.RsAdamwOpts(1e-3, 0.9, 0.99, 1e-8, 0.0)
    L.check(lib.rs_adamw_step(None, 0, ctypes.byref(o), None, norm.data_ptr(), None, 0, 0, stream))  # no clipping, no norm


# ---- tensors that autograd follows --------------------------------------------------------------
def test_what_is_written_in_place_counts_as_written():
    state = make_state([100, 7], BF16, F32, True)
    grads = {n: randn(e["param"].numel(), dtype=BF16, seed=1) for n, e in state.items()}
    before = {n: {s: t._version for s, t in e.items()} for n, e in state.items()}
    opt = OPT.ShardAdamW(state, max_norm=1.0, **HYPER)
    opt.step({"t0": grads["t0"]})
    assert all(t._version > before["t0"][s] for s, t in state["t0"].items())
    assert all(t._version == before["t1"][s] for s, t in state["t1"].items())
    v = grads["t0"]._version
    OPT.clip_grads(grads, 1e-3)
    assert grads["t0"]._version > v
    ids, g = torch.arange(3, device=DEV), randn(3, 6, seed=2)
    out = torch.zeros(4, 6, device=DEV)
    v = out._version
    V.embedding_grad(g, ids, 4, out=out)
    assert out._version > v
    z, t = randn(3, 8, seed=1), torch.zeros(3, dtype=torch.int64, device=DEV)
    r = V.token_logprobs(z, t)
    v = z._version
    V.token_logprobs_grad(z, t, r.lse, r.entropy, r.lse, out=z)
    assert z._version > v


def test_a_refused_call_counts_as_nothing_written():
    x = torch.zeros(100, device=DEV)
    v = x._version
    with pytest.raises(RuntimeError, match="share memory"):
        OPT.clip_grads([x[:60], x[50:]], 1.0)
    state = make_state([100, 7], BF16, F32, True)
    before = {n: {s: t._version for s, t in e.items()} for n, e in state.items()}
    opt = OPT.ShardAdamW(state, **HYPER)
    for grads in ({"t0": torch.zeros(100, device=DEV), "t1": torch.zeros(8, device=DEV)}, {"t0": torch.zeros(200, device=DEV)[::2]}):
        with pytest.raises((AssertionError, ValueError)):
            opt.step(grads)
    opt.lr = -1.0
    with pytest.raises(RuntimeError, match="out of range"):
        opt.step({"t0": torch.zeros(100, device=DEV)})
    assert x._version == v and before == {n: {s: t._version for s, t in e.items()} for n, e in state.items()}


def test_a_backward_pass_over_what_was_written_is_an_error():
    state = make_state([12], F32, F32, False)
    w = state["t0"]["param"].requires_grad_()
    y = (w * w).sum()
    OPT.ShardAdamW(state, **HYPER).step({"t0": randn(12, seed=1)})
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()
    z = randn(3, 8, seed=1).requires_grad_()
    t = torch.zeros(3, dtype=torch.int64, device=DEV)
    r = V.token_logprobs(z, t)
    V.token_logprobs_grad(z.detach(), t, r.lse.detach(), r.entropy.detach(), r.lse.detach(), out=z.detach())
    with pytest.raises(RuntimeError, match="inplace"):
        r.logprob.sum().backward()
    with torch.inference_mode():  # no versions are kept there
        s = make_state([12], F32, F32, False)
        g = {"t0": randn(12, seed=1)}
    OPT.ShardAdamW(s, max_norm=1.0, **HYPER).step(g)
    OPT.clip_grads(g, 1.0)


def test_forward_mode_tangents_are_refused():
    import torch.autograd.forward_ad as fwad
    w, z = randn(5, 6, seed=1), randn(3, 8, seed=2)
    ids, t, f = torch.arange(3, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV), torch.zeros(3, device=DEV)
    with fwad.dual_level():
        dw, dz = fwad.make_dual(w, torch.ones_like(w)), fwad.make_dual(z, torch.ones_like(z))
        rec = fwad.make_dual(torch.zeros(1, 3, 4, device=DEV), torch.ones(1, 3, 4, device=DEV))
        for call in (lambda: V.embedding(ids, dw), lambda: V.embedding_grad(dw[:3], ids, 5), lambda: V.token_logprobs(dz, t, top=2),
                     lambda: V.token_record(dz, t), lambda: V.token_logprobs_grad(dz, t, f, f, f), lambda: OPT.grad_sumsq([dw]),
                     lambda: OPT.clip_grads([dw], 1.0), lambda: V.merge_token_records(rec, [0])):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
        V.embedding(ids, w), V.token_logprobs(z, t)  # tensors without a tangent


# ---- memory used twice, and sizes of nothing ------------------------------------------------------
@pytest.mark.parametrize("n", [100, 70000])
def test_a_gradient_over_its_own_input_is_refused(n):
    """The output is cleared and written while grad_out is read."""
    for dtype in (F32, BF16):
        buf = randn(n + 64, 16, dtype=dtype, seed=1)
        ids = torch.randint(0, 64, (n,), generator=gen(1), device=DEV)
        kept = buf.clone()
        for g, out in ((buf[:n], buf[:64]), (buf[:n], buf[n - 64:n]), (buf[:n], buf[n - 1:n + 63]), (buf[:n, :8], buf.view(-1)[:512].view(64, 8)),
                       (buf[:1].expand(n, 16), buf[:64])):
            for acc in (False, True):
                with pytest.raises(RuntimeError, match="overlaps"):
                    V.embedding_grad(g, ids, 64, out=out, accumulate=acc)
        assert torch.equal(buf, kept)
        out = buf[n:]  # beside it
        assert torch.equal(V.embedding_grad(buf[:n], ids, 64, out=out), V.embedding_grad(kept[:n], ids, 64, dtype=dtype))
        one = torch.where(ids == 3, 0, -1)  # between two of its rows
        wide = kept.clone()
        got = V.embedding_grad(wide[:n, :8], one, 1, out=wide[5:6, 8:])
        assert torch.equal(got, V.embedding_grad(kept[:n, :8].contiguous(), one, 1))


def test_gradient_of_no_columns():
    for n in (3, 70000):
        ids = torch.zeros(2, n, dtype=torch.int64, device=DEV)
        assert V.embedding_grad(torch.zeros(2, n, 0, device=DEV), ids, 5).shape == (5, 0)
        assert V.embedding(ids, torch.zeros(5, 0, device=DEV)).shape == (2, n, 0)


# ---- errors of the allocator --------------------------------------------------------------------
def test_out_of_memory_is_torchs_own_error():
    """A call that finds no memory raises what torch's operators raise, without the library's stack."""
    ids, w = torch.zeros(1 << 18, dtype=torch.int64, device=DEV), torch.zeros(1, 1 << 22, dtype=BF16, device=DEV)  # 2 TB
    with pytest.raises(torch.OutOfMemoryError) as e:
        V.embedding(ids, w)
    assert "c10::" not in str(e.value)
    assert torch.equal(V.embedding(ids[:2], w), w.expand(2, -1))


# ---- other threads ------------------------------------------------------------------------------
def test_other_threads_run_while_a_call_waits_for_the_launch_queue():
    """A call that finds the launch queue full waits in the driver; Python goes on meanwhile."""
    w, ids = randn(50, 64, seed=1), torch.arange(8, device=DEV)
    V.embedding(ids, w)
    torch.cuda.synchronize()
    gaps, stop = [0.0], threading.Event()

    def count():
        last = time.perf_counter()
        while not stop.is_set():
            now = time.perf_counter()
            gaps[0] = max(gaps[0], now - last)
            last = now
            time.sleep(0.001)
    other = threading.Thread(target=count)
    other.start()
    torch.cuda._sleep(1_500_000_000)  # about 0.8 s of a kernel that does nothing
    longest = 0.0
    for _ in range(6000):
        t0 = time.perf_counter()
        V.embedding(ids, w)
        longest = max(longest, time.perf_counter() - t0)
    stop.set()
    other.join()
    torch.cuda.synchronize()
    print(f"longest call {longest:.3f} s, the other thread's longest wait {gaps[0]:.3f} s")
    if longest < 0.2:
        pytest.skip("the launch queue did not fill")
    assert gaps[0] < longest / 2
