"""Gradient norm, clipping and AdamW, the embedding and the token log probabilities on a B200, each against
a plain computation in 64 bits.

Tolerances count roundings: half a step, eps / 2 relative (u = 2^-24 in 32 bits), for each of the roundings that
lie between an input and a value, and eps / 2 of the stored type once. They are written at each test.
"""
import math

import numpy as np
import pytest
import torch

from suika_b200 import migration as M
from suika_b200 import optimizer as OPT
from suika_b200 import synthetic as S
from suika_b200 import vocab as V
from suika_b200.layouts import SPECS, ReshardConfig, mesh_layout, scaled_spec

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    """Half of the smallest subnormal step: a value below the normal range is off by at most this."""
    return torch.finfo(t).tiny * torch.finfo(t).eps / 2


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(*shape, dtype=F32, scale=1.0, seed=0, offset=0):
    """A tensor whose first element lies `offset` elements past an aligned address."""
    n = math.prod(shape)
    x = torch.empty(n + offset, dtype=dtype, device=DEV)
    x.copy_(torch.randn(n + offset, generator=gen(seed), device=DEV) * scale)
    return x[offset:offset + n].view(*shape)


def assert_close(got, ref, bound, what=""):
    got, ref = got.double(), ref.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    same = (got == ref) | (got.isnan() & ref.isnan())
    off = torch.where(same, torch.zeros_like(ref), (got - ref).abs())
    bad = ~(off <= bound)
    assert not bad.any().item(), (what, int(bad.sum()), float(off.nan_to_num(nan=math.inf).max()), got[bad][:4].tolist(), ref[bad][:4].tolist())


# ---- norm and clipping ----------------------------------------------------------------------
# Squares and the sum of at most 32 of them round in 32 bits (33 roundings of values that do not cancel), the rest in 64.
SUMSQ_REL = 34 * U


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [0, 1, 3, 7])
def test_sumsq_sizes_and_alignment(dtype, offset):
    sizes = [0, 1, 2, 7, 8, 9, 31, 1023, 1024, 1025, 4097, 70001]
    gs = {f"t{i}": randn(n, dtype=dtype, seed=i, offset=offset) for i, n in enumerate(sizes)}
    got = OPT.grad_sumsq(gs)
    ref = sum(float(g.double().square().sum()) for g in gs.values())
    assert abs(float(got) - ref) <= SUMSQ_REL * ref
    assert torch.equal(got, OPT.grad_sumsq(list(gs.values())))  # a sequence; and the same bits again


def test_sumsq_of_many_tensors_and_types():
    gs = {f"t{i}": randn(1 + i % 37, dtype=TYPES[i % 3], seed=i) for i in range(2600)}  # three launches' tables
    ref = sum(float(g.double().square().sum()) for g in gs.values())
    assert abs(float(OPT.grad_sumsq(gs)) - ref) <= SUMSQ_REL * ref


@pytest.mark.parametrize("scale", [1e-40, 1e-25, 1e-12, 1e15, 1e25, 3e37])
def test_sumsq_beyond_the_range_of_squares(scale):
    g = randn(5000, seed=1).clamp(-10, 10).mul_(scale)
    g[3], g[4000] = 1.0 * scale, 0.0
    ref = float(g.double().square().sum())
    assert abs(float(OPT.grad_sumsq([g])) - ref) <= SUMSQ_REL * ref


def test_sumsq_of_zeros_infinities_and_nan():
    assert float(OPT.grad_sumsq([torch.zeros(5000, device=DEV)])) == 0.0
    assert float(OPT.grad_sumsq([torch.zeros(0, device=DEV)])) == 0.0
    for bad in (math.inf, -math.inf, math.nan):
        for at in (0, 17, 4999):
            g = torch.ones(5000, device=DEV, dtype=BF16)
            g[at] = bad
            s = float(OPT.grad_sumsq([g]))
            assert math.isnan(s) if math.isnan(bad) else s == math.inf


def test_sumsq_of_a_long_tensor():
    n = (1 << 31) + 12345  # offsets past 32 bits
    g = torch.full((n,), 0.5, dtype=BF16, device=DEV)
    g[-1] = 3.0
    ref = 0.25 * (n - 1) + 9.0
    assert abs(float(OPT.grad_sumsq([g])) - ref) <= SUMSQ_REL * ref


# c = max_norm / (norm + 1e-6): the norm is off by half of SUMSQ_REL and one rounding, then a sum, a quotient and the product.
CLIP_REL = SUMSQ_REL / 2 + 4 * U


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [0, 1, 5])
def test_clip(dtype, offset):
    gs = {f"t{i}": randn(n, dtype=dtype, scale=0.1, seed=i, offset=offset) for i, n in enumerate([1, 9, 2048, 100003])}
    old = {n: g.clone() for n, g in gs.items()}
    norm = OPT.clip_grads(gs, 0.75)
    ref = math.sqrt(sum(float(g.double().square().sum()) for g in old.values()))
    assert norm.shape == () and abs(float(norm) - ref) <= (SUMSQ_REL / 2 + U) * ref
    for n, g in gs.items():
        want = old[n].double() * (0.75 / (ref + 1e-6))
        assert_close(g, want, want.abs() * (half(dtype) * (1 + CLIP_REL) + CLIP_REL) + tiny(dtype), n)


def test_clip_leaves_gradients_within_the_limit_alone():
    g = randn(1000, dtype=BF16, seed=3)
    old = g.clone()
    norm = OPT.clip_grads([g], 1e3)
    assert torch.equal(g, old) and float(norm) > 1
    z = torch.zeros(7, device=DEV)
    assert float(OPT.clip_grads([z], 1.0)) == 0 and not z.any()


def test_clip_with_a_given_sum():
    g = randn(1000, seed=3)
    old = g.clone()
    total = OPT.grad_sumsq([g]) + 1e6  # as if other ranks held the rest
    norm = OPT.clip_grads([g], 2.0, sumsq=total)
    want = old.double() * (2.0 / (math.sqrt(float(total)) + 1e-6))
    assert abs(float(norm) - math.sqrt(float(total))) <= U * float(norm)
    assert_close(g, want, want.abs() * (5 * U))


def test_clip_of_norms_that_are_not_finite():
    for bad, want in ((math.inf, 0.0), (math.nan, math.nan)):  # torch's clip_grad_norm_: c = 0, or NaN
        g = torch.ones(100, device=DEV)
        g[7] = bad
        OPT.clip_grads([g], 1.0)
        assert math.isnan(float(g[7])) and (torch.isnan(g[0]) if math.isnan(want) else g[0] == want)


def test_clip_refuses_what_it_cannot_scale_once():
    x = torch.zeros(100, device=DEV)
    with pytest.raises(RuntimeError, match="share memory"):
        OPT.clip_grads([x, x], 1.0)
    with pytest.raises(RuntimeError, match="share memory"):
        OPT.clip_grads([x[:60], x[50:]], 1.0)
    with pytest.raises(ValueError, match="contiguous"):
        OPT.clip_grads([torch.zeros(4, 6, device=DEV).t()], 1.0)
    with pytest.raises(ValueError, match="bfloat16"):
        OPT.clip_grads([torch.zeros(4, device=DEV, dtype=torch.int32)], 1.0)
    with pytest.raises(ValueError, match="sumsq"):
        OPT.clip_grads([x], 1.0, sumsq=torch.zeros(1, device=DEV))
    with pytest.raises(ValueError, match="by name"):
        OPT.grad_sumsq([x], counted={"x": [(0, 100)]})
    with pytest.raises(AssertionError, match="leaves a gradient"):
        OPT.grad_sumsq({"x": x}, counted={"x": [(1, 100)]})


@pytest.mark.parametrize("fused", [False, True])
def test_ranks_sums_add_up_to_the_whole_models(fused):
    spec = scaled_spec(SPECS["qwen2-7b"], name="m", hidden=32, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=8, ffn=48, vocab=40,
                       fused_qkv=fused, vocab_parallel_wte=True)
    whole = S.host_states(mesh_layout(spec, [[[0]]]), [("exp_avg", "f32")], seed=1)[0]
    ref = sum(float(np.square(e["exp_avg"].astype(np.float64)).sum()) for e in whole.values())
    layout = mesh_layout(spec, [[[0, 1, 2, 3], [4, 5, 6, 7]]])  # TP4 x DP2; KV heads replicated by pairs when fused
    total = 0.0
    for rank, st in S.host_states(layout, [("exp_avg", "f32")], seed=1).items():
        grads = {n: torch.from_numpy(e["exp_avg"]).to(DEV) for n, e in st.items()}
        total += float(OPT.grad_sumsq(grads, counted=OPT.counted_spans(layout, rank)))
    assert abs(total - ref) <= SUMSQ_REL * ref


# ---- AdamW ----------------------------------------------------------------------------------
def make_state(sizes, param, moments, master, offset=0, seed=0, step=None):
    state = {}
    for i, n in enumerate(sizes):
        w = randn(n, scale=0.05, seed=seed + 10 * i)
        ent = {"param": torch.empty(n + offset, dtype=param, device=DEV)[offset:], "step": torch.tensor(float(i % 5 if step is None else step), device=DEV)}
        ent["param"].copy_(w)
        if master:
            ent["master"] = torch.empty(n + offset, device=DEV)[offset:]
            ent["master"].copy_(w)
        ent["exp_avg"] = randn(n, dtype=moments, scale=1e-3, seed=seed + 10 * i + 1, offset=offset)
        ent["exp_avg_sq"] = randn(n, dtype=moments, scale=1e-3, seed=seed + 10 * i + 2, offset=offset).square_()
        state[f"t{i}"] = ent
    return state


def clone_state(state):
    return {n: {s: t.clone() for s, t in e.items()} for n, e in state.items()}


HYPER = dict(lr=3e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)


def check_adam(old, new, grads, factor=1.0, factor_rel=0.0, decay=lambda n: 0.1, lr=3e-3):
    """One step against torch.optim.AdamW in 64 bits. Roundings in 32 bits: the gradient factor_rel and one; m: the
    difference, the product and the sum (3, of terms no larger than |m| + |g|); v: two products of the gradient, its
    own twice, and the sum (6); then sqrt, product, sum, quotient, two products and the difference (8)."""
    b1, b2 = HYPER["betas"]
    for n, e in old.items():
        g = grads[n].double() * factor
        wide = e["master"] if "master" in e else e["param"]
        p = torch.nn.Parameter(wide.double())
        p.grad = g
        opt = torch.optim.AdamW([p], lr=lr, betas=(b1, b2), eps=HYPER["eps"], weight_decay=decay(n), foreach=False, fused=False)
        opt.state[p] = {"step": e["step"].double().cpu().reshape(()), "exp_avg": e["exp_avg"].double(), "exp_avg_sq": e["exp_avg_sq"].double()}
        opt.step()
        st, w = opt.state[p], p.detach()
        got, mt = new[n], e["exp_avg"].dtype
        t = float(e["step"]) + 1
        assert float(got["step"]) == t, n
        rg = factor_rel + U
        dm = 3 * U * (e["exp_avg"].double().abs() + g.abs()) + 0.1 * rg * g.abs()
        dv = (6 * U + 2 * rg) * st["exp_avg_sq"] + torch.finfo(F32).tiny * 2 ** -23
        assert_close(got["exp_avg"], st["exp_avg"], dm + half(mt) * st["exp_avg"].abs() * (1 + 4 * U) + tiny(mt), n + " exp_avg")
        assert_close(got["exp_avg_sq"], st["exp_avg_sq"], dv + half(mt) * st["exp_avg_sq"] * (1 + 4 * U) + tiny(mt), n + " exp_avg_sq")
        denom = (st["exp_avg_sq"] / (1 - b2 ** t)).sqrt() + HYPER["eps"]
        update = lr / (1 - b1 ** t) * st["exp_avg"].abs() / denom
        # a v below 32 bits' normal range leaves sqrt(v) off by more than its share: those values stand aside in eps' shadow
        dw = lr / (1 - b1 ** t) * dm / denom + update * (8 * U + (6 * U + 2 * rg) / 2) + 3 * U * (wide.double().abs() + update)
        if "master" in e:
            assert_close(got["master"], w, dw, n + " master")
            pt = got["param"].dtype
            assert torch.equal(got["param"], got["master"].to(pt)), n  # the master rounded to nearest
        else:
            pt = got["param"].dtype
            assert_close(got["param"], w, dw + half(pt) * w.abs() * (1 + 4 * U) + tiny(pt), n + " param")


ADAM_KINDS = [(BF16, F32, True), (F16, F32, True), (F32, F32, True), (BF16, BF16, True), (BF16, BF16, False), (F32, F32, False),
              (F16, F32, False), (BF16, F32, False)]


@pytest.mark.parametrize("param,moments,master", ADAM_KINDS)
@pytest.mark.parametrize("grad", TYPES)
@pytest.mark.parametrize("offset", [0, 1])
def test_adamw_step(param, moments, master, grad, offset):
    state = make_state([1, 7, 8, 9, 1023, 5000, 40001], param, moments, master, offset)
    grads = {n: randn(e["param"].numel(), dtype=grad, scale=1e-2, seed=77 + i, offset=offset) for i, (n, e) in enumerate(state.items())}
    kept = {n: g.clone() for n, g in grads.items()}
    old = clone_state(state)
    opt = OPT.ShardAdamW(state, no_decay=["t2"], **HYPER)
    assert opt.step(grads) is None
    check_adam(old, state, grads, decay=lambda n: 0.0 if n == "t2" else 0.1)
    assert all(torch.equal(g, kept[n]) for n, g in grads.items())
    second = clone_state(state)
    opt.lr = 1e-3
    opt.step(grads)
    check_adam(second, state, grads, decay=lambda n: 0.0 if n == "t2" else 0.1, lr=1e-3)


def test_adamw_clips_and_returns_the_norm():
    state = make_state([100, 5000, 333], BF16, F32, True)
    grads = {n: randn(e["param"].numel(), dtype=BF16, scale=0.5, seed=i) for i, (n, e) in enumerate(state.items())}
    old = clone_state(state)
    norm = OPT.ShardAdamW(state, max_norm=1.0, **HYPER).step(grads)
    ref = math.sqrt(sum(float(g.double().square().sum()) for g in grads.values()))
    assert abs(float(norm) - ref) <= (SUMSQ_REL / 2 + U) * ref
    check_adam(old, state, grads, 1.0 / (ref + 1e-6), CLIP_REL)


def test_adamw_of_many_small_tensors():
    state = make_state([1 + i % 19 for i in range(1200)], BF16, F32, True)  # three launches' tables
    grads = {n: randn(e["param"].numel(), dtype=F32, scale=1e-2, seed=i) for i, (n, e) in enumerate(state.items())}
    old = clone_state(state)
    OPT.ShardAdamW(state, max_norm=1e9, **HYPER).step(grads)
    check_adam(old, state, grads, 1.0, 0.0)


def test_adamw_without_some_gradients_and_with_host_steps():
    state = make_state([50, 60, 70], BF16, F32, True)
    for e in state.values():
        e["step"] = torch.tensor(2.0)  # where torch.optim.AdamW keeps it
    old = clone_state(state)
    grads = {"t0": randn(50, seed=1), "t1": None}
    OPT.ShardAdamW(state, **HYPER).step(grads)
    assert all(e["step"].is_cuda for e in state.values())
    check_adam({"t0": old["t0"]}, state, grads)
    for n in ("t1", "t2"):
        assert all(torch.equal(state[n][s].cpu(), old[n][s].cpu()) for s in old[n]), n


def test_adamw_mixed_types_and_empty_tensors():
    state = make_state([300, 0, 400], BF16, F32, True)
    state["t2"] = make_state([400], F32, BF16, False, seed=9)["t0"]
    grads = {"t0": randn(300, dtype=BF16, seed=1), "t1": randn(0, seed=2), "t2": randn(400, dtype=F16, seed=3)}
    old = clone_state(state)
    OPT.ShardAdamW(state, **HYPER).step(grads)
    check_adam(old, state, grads)


def test_adamw_refuses_what_it_cannot_step():
    mk = lambda: make_state([10], BF16, F32, True)  # noqa: E731
    for sub, value, exc, word in (("exp_avg", torch.zeros(10, dtype=F16, device=DEV), ValueError, "moments"),
                                  ("exp_avg_sq", torch.zeros(10, dtype=BF16, device=DEV), ValueError, "moments"),
                                  ("master", torch.zeros(10, dtype=BF16, device=DEV), ValueError, "master"),
                                  ("exp_avg", torch.zeros(9, device=DEV), AssertionError, "shape"),
                                  ("step", torch.zeros(2, device=DEV), AssertionError, "step"),
                                  ("param", torch.zeros(20, device=DEV, dtype=BF16)[::2], ValueError, "contiguous")):
        s = mk()
        s["t0"][sub] = value
        with pytest.raises(exc, match=word):
            OPT.ShardAdamW(s, **HYPER)
    s = mk()
    s["t1"] = dict(s["t0"])
    with pytest.raises(ValueError, match="share memory"):
        OPT.ShardAdamW(s, **HYPER)
    opt = OPT.ShardAdamW(mk(), **HYPER)
    with pytest.raises(AssertionError, match="shape"):
        opt.step({"t0": torch.zeros(9, device=DEV)})
    with pytest.raises(AssertionError, match="does not hold"):
        opt.step({"t0": torch.zeros(10, device=DEV), "x": torch.zeros(1, device=DEV)})
    with pytest.raises(ValueError, match="contiguous"):
        opt.step({"t0": torch.zeros(20, device=DEV)[::2]})
    with pytest.raises(ValueError, match="no gradients"):
        opt.step({})


# ---- embedding ------------------------------------------------------------------------------
def ref_lookup(ids, w, scale, lo):
    held = (ids >= lo) & (ids < lo + w.shape[0])
    x = w.double()[torch.where(held, ids - lo, 0)] * float(np.float32(scale))
    return torch.where(held.unsqueeze(-1), x, 0.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hidden", [1, 3, 8, 33, 130, 2048, 4104])
@pytest.mark.parametrize("scale", [1.0, 11.3])
def test_lookup(dtype, hidden, scale):
    w = randn(50, hidden, dtype=dtype, seed=hidden)
    for shape in ((1,), (7,), (3, 41), (0,)):
        ids = torch.randint(90, 170, shape, generator=gen(1), device=DEV)
        if ids.numel() > 3:
            ids.view(-1)[:4] = torch.tensor([-1, 1 << 40, -(1 << 40), 149], device=DEV)
        got = V.embedding(ids, w, scale=scale, lo=100)
        ref = ref_lookup(ids, w, scale, 100)
        if scale == 1.0:
            assert torch.equal(got.double(), ref)
        else:  # the product in 32 bits, then the type
            assert_close(got, ref, ref.abs() * (half(dtype) * (1 + U) + U) + tiny(dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_lookup_strides_offsets_and_id_types(dtype):
    big = randn(60, 200, dtype=dtype, seed=4)
    for w in (big[:, :64], big[:, 1:66], big[::2, 8:72], big[3:4], randn(20, 24, dtype=dtype, seed=5, offset=3), big[:1].expand(60, 200)):
        for idt in (torch.int32, torch.int64):
            ids = torch.randint(0, w.shape[0], (40, 2), generator=gen(2), device=DEV).to(idt)[:, 1]  # not contiguous
            assert torch.equal(V.embedding(ids, w), w[ids.long()])


def test_lookup_offsets_past_32_bits():
    rows, hidden = (1 << 31) // 512 + 8, 1024  # 2^32 elements and more
    w = torch.zeros(rows, hidden, dtype=BF16, device=DEV)
    w[-3:] = randn(3, hidden, dtype=BF16, seed=1)
    ids = torch.tensor([rows - 1, 0, rows - 3], device=DEV)
    assert torch.equal(V.embedding(ids, w), w[ids])
    g = randn(3, hidden, dtype=BF16, seed=2)
    dw = V.embedding_grad(g, ids, rows)
    assert torch.equal(dw[ids], g)
    dw[ids] = 0
    assert not dw.any()


def spread(kind, n, rows, lo, seed=0):
    if kind == "same":
        return torch.full((n,), lo + rows // 2, device=DEV)
    if kind == "none":
        return torch.full((n,), -1, device=DEV)
    if kind == "distinct":
        return (torch.arange(n, device=DEV).flip(0) % rows) + lo
    u = torch.rand(n, generator=gen(seed), device=DEV, dtype=torch.float64)  # a few rows take most tokens, some are not held
    return (torch.pow(float(rows * 2), u).long() - 1) + lo - 1


def check_grad(g, ids, rows, lo=0, scale=1.0, dtype=None, acc=None):
    """A sum of c terms in 32 bits is off by at most c U of the sum of their sizes; the scale, the addition and the type round once."""
    held = (ids >= lo) & (ids < lo + rows)
    at, gd = (ids - lo)[held].long().reshape(-1), g.double()[held].reshape(-1, g.shape[-1])
    z = lambda: torch.zeros(rows, g.shape[-1], dtype=torch.float64, device=DEV)  # noqa: E731
    s = float(np.float32(scale))
    ref, size = z().index_add_(0, at, gd) * s, z().index_add_(0, at, gd.abs()) * s
    count = torch.zeros(rows, dtype=torch.float64, device=DEV).index_add_(0, at, torch.ones_like(at, dtype=torch.float64)).unsqueeze(1)
    out = None
    if acc is not None:
        out, ref = acc.clone(), ref + acc.double()
    got = V.embedding_grad(g, ids, rows, scale=scale, lo=lo, dtype=dtype, out=out, accumulate=acc is not None)
    assert out is None or got is out
    t = got.dtype
    bound = (count + 2) * U * size + ref.abs() * (half(t) * (1 + U) + U) + tiny(t)
    assert_close(got, ref, torch.where(count > 0, bound, torch.zeros_like(bound)))
    again = V.embedding_grad(g, ids, rows, scale=scale, lo=lo, dtype=dtype, out=None if acc is None else acc.clone(), accumulate=acc is not None)
    assert torch.equal(got, again)  # no sum's order changes
    return got


@pytest.mark.parametrize("n", [0, 1, 2, 7, 8, 9, 17, 64, 65, 200, 1000, 1025, 2049, 5000])
@pytest.mark.parametrize("kind", ["same", "none", "distinct", "skewed"])
def test_embedding_grad_lengths(n, kind):
    rows, lo = 300, 1000
    check_grad(randn(n, 40, dtype=BF16, seed=n), spread(kind, n, rows, lo), rows, lo, scale=2.5)


@pytest.mark.parametrize("n", [8193, 20000, 40001, 65536, 70001, 131073])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_embedding_grad_long(n, dtype):
    for kind in ("skewed", "same"):
        check_grad(randn(n, 24, dtype=BF16, seed=n), spread(kind, n, 70000, 0), 70000, dtype=dtype)
    check_grad(randn(n, 24, dtype=BF16, seed=n), spread("skewed", n, 500, 7), 500, 7, dtype=dtype, acc=randn(500, 24, dtype=dtype, seed=2))


@pytest.mark.parametrize("gt", TYPES)
@pytest.mark.parametrize("wt", TYPES)
@pytest.mark.parametrize("hidden", [1, 2, 36, 257, 2056, 4100])
def test_embedding_grad_types_and_widths(gt, wt, hidden):
    ids = spread("skewed", 333, 60, 0)
    g = randn(333, hidden, dtype=gt, seed=hidden)
    check_grad(g, ids, 60, scale=0.3, dtype=wt)
    check_grad(g, ids, 60, scale=0.3, dtype=wt, acc=randn(60, hidden, dtype=wt, seed=1))


@pytest.mark.parametrize("rows", [1, 2, 255, 256, 257, 511, 512, 65535, 65536, 262143, 262144, 1 << 20])
def test_embedding_grad_key_widths(rows):
    check_grad(randn(3000, 16, seed=rows), spread("skewed", 3000, rows, 0), rows)
    check_grad(randn(1500, 16, seed=rows), spread("distinct", 1500, rows, 0).int(), rows)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,rows,hidden", [(1, 70001, 1024), (9, 9001, 8192), (3000, 40003, 2048), (9000, 300000, 256), (64, 17, 4 << 20), (5, 20000, 4100)])
def test_embedding_grad_of_large_tables(n, rows, hidden, dtype):
    """Outputs much larger than what the tokens touch: every other row is cleared, and the last row is written."""
    g = randn(n, hidden, dtype=BF16, seed=n)
    for kind in ("skewed", "distinct"):
        ids = spread(kind, n, rows, 0)
        ids[0] = rows - 1
        out = torch.full((rows, hidden), 7.0, dtype=dtype, device=DEV)
        held = (ids >= 0) & (ids < rows)
        V.embedding_grad(g, ids, rows, out=out)
        at = ids[held].unique()
        few = torch.searchsorted(at, ids)  # the same sums on a table of the touched rows alone
        few = torch.where(held, few, -1)
        assert torch.equal(out[at], V.embedding_grad(g, few, len(at), dtype=dtype))
        out[at] = 0
        assert not out.any()


def test_embedding_grad_strides():
    ids = torch.randint(0, 30, (50, 4), generator=gen(3), device=DEV)
    big = randn(200, 300, dtype=BF16, seed=3)
    check_grad(big[:, 8:136], ids.reshape(-1), 30)      # rows 16-byte aligned, strided
    check_grad(big[:, 1:130], ids.reshape(-1), 30)      # rows at odd addresses
    check_grad(big[:1, :64].expand(200, 64), ids.reshape(-1), 30)
    check_grad(torch.ones((), device=DEV).expand(200, 33), ids.reshape(-1), 30)  # the gradient of a sum
    check_grad(randn(50, 4, 20, seed=5), ids, 30)
    check_grad(randn(4, 50, 20, seed=5).transpose(0, 1), ids, 30)
    odd = torch.empty(30 * 24 + 1, dtype=BF16, device=DEV)[1:].view(30, 24)  # an output at an odd address
    g = randn(200, 24, dtype=BF16, seed=6)
    assert torch.equal(V.embedding_grad(g, ids.reshape(-1), 30, out=odd), V.embedding_grad(g, ids.reshape(-1), 30))


def test_embedding_refusals():
    w, ids = torch.zeros(4, 6, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    g = torch.zeros(3, 6, device=DEV)
    for call, exc in ((lambda: V.embedding(ids, w.t()), ValueError), (lambda: V.embedding(ids.float(), w), ValueError),
                      (lambda: V.embedding(ids.cpu(), w), ValueError), (lambda: V.embedding(ids, w.int()), ValueError),
                      (lambda: V.embedding(ids, w[0]), ValueError), (lambda: V.embedding_grad(g[:2], ids, 4), AssertionError),
                      (lambda: V.embedding_grad(g, ids, 4, accumulate=True), ValueError),
                      (lambda: V.embedding_grad(g, ids, 4, out=torch.zeros(5, 6, device=DEV)), AssertionError),
                      (lambda: V.embedding_grad(g, ids, 4, out=torch.zeros(6, 4, device=DEV).t()), ValueError),
                      (lambda: V.embedding_grad(g, ids, 4, out=w, dtype=BF16), ValueError)):
        with pytest.raises(exc):
            call()


def test_embedding_autograd():
    w = randn(40, 24, seed=1).requires_grad_()
    ids = torch.randint(0, 60, (5, 9), generator=gen(4), device=DEV)
    c = randn(5, 9, 24, seed=2)
    (V.embedding(ids, w, scale=3.0, lo=10) * c).sum().backward()
    assert torch.equal(w.grad, V.embedding_grad(c, ids, 40, scale=3.0, lo=10))
    V.embedding(ids, w, scale=3.0, lo=10).sum().backward()  # the gradient of a broadcast input: ones, expanded
    assert torch.isfinite(w.grad).all()
    with torch.no_grad():
        assert not V.embedding(ids, w).requires_grad


# ---- token log probabilities -----------------------------------------------------------------
def ref_log_p(z):
    """(log p, lse, rows of -inf alone) in 64 bits. log p = (z - m) - log S, as m + log S loses log S where m is the type's lowest value."""
    z = z.double()
    m = z.amax(1, keepdim=True)
    empty = (m == -math.inf).squeeze(1)
    log_s = (z - m).exp().sum(1, keepdim=True).log()
    lse = torch.where(empty, -math.inf, (m + log_s).squeeze(1))
    lp = torch.where(empty.unsqueeze(1), -math.inf, (z - m) - log_s)
    return torch.where(lp < torch.finfo(F32).min, -math.inf, lp), lse, empty  # what 32 bits hold of it


def ref_logprobs(z, t, lo=0, top=0):
    lp, lse, empty = ref_log_p(z)
    z = z.double()
    m = z.amax(1, keepdim=True)
    p = lp.exp()
    h = -torch.where(p > 0, p * lp, 0.0).sum(1)
    h = torch.where(z.isnan().any(1) | (m.squeeze(1) == math.inf), math.nan, torch.where(empty, 0.0, h))
    known = (t >= lo) & (t < lo + z.shape[1])
    got = lp.gather(1, torch.where(known, t - lo, 0).long().unsqueeze(1)).squeeze(1)
    out = [torch.where(known, got, 0.0), h, lse]
    if top:
        v, i = z.sort(dim=1, descending=True, stable=True)
        fill = top - z.shape[1]
        v, i = lp.gather(1, i)[:, :top], (i + lo)[:, :top]
        if fill > 0:
            v = torch.cat([v, torch.full((len(v), fill), -math.inf, device=DEV)], 1)
            i = torch.cat([i, torch.full((len(i), fill), -1, device=DEV)], 1)
        out += [v, i]
    return out


def stat_rel(z):
    """Relative error of S = sum e^(z - m): the exponent's argument two roundings of |t| (weighted with p, E|t| <= 40 here),
    the exponential 2^-22, rescaling at each of the thread's batches (at most 12 U), cols / 256 additions and 13 joins."""
    return (z.shape[1] / 256 + 13 + 12 + 80) * U + 2.0 ** -22


def check_logprobs(z, t, lo=0, top=0, got=None):
    r = got or V.token_logprobs(z, t, lo=lo, top=top)
    ref = ref_logprobs(z, t, lo, top)
    s = stat_rel(z)
    # lse = m + log S: S's error, the logarithm's and the sum's; a log probability likewise; the entropy is
    # log S - A / S with A of the same error relative to its size |A / S| <= H + log S
    finite = lambda x: torch.where(x.isfinite(), x.abs(), 0.0)  # noqa: E731
    span = finite(ref[1]) + math.log(z.shape[1]) + 1
    assert_close(r.lse, ref[2], s + 3 * U * (finite(ref[2]) + span + finite(z.double().amax(1))), "lse")
    assert_close(r.logprob, ref[0], s + 4 * U * (finite(ref[0]) + span), "logprob")
    assert_close(r.entropy, ref[1], 3 * s * span, "entropy")
    if top:
        assert torch.equal(r.top_index, ref[4]), "indices"
        assert_close(r.top_logprob, ref[3], (s + 4 * U * span).unsqueeze(1) + 4 * U * finite(ref[3]), "top")
    else:
        assert r.top_index is None and r.top_logprob is None
    return r


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [1, 2, 7, 8, 9, 33, 255, 1000, 4099, 32000, 50257])
def test_logprobs_sizes(dtype, cols):
    for n, top in ((1, 1), (3, 20), (40, 5), (400, 0), (2, 32)):
        z = randn(n, cols, dtype=dtype, scale=3.0, seed=cols + n)
        t = torch.randint(0, cols, (n,), generator=gen(n), device=DEV)
        if n > 2:
            t[0], t[1] = -1, -100
        r = check_logprobs(z, t, 0, top)
        assert all(torch.equal(a, b) for a, b in zip(r, V.token_logprobs(z, t, top=top)) if a is not None)  # the same bits again


@pytest.mark.parametrize("dtype", TYPES)
def test_logprobs_of_a_large_vocabulary(dtype):
    z = randn(5, 152064, dtype=dtype, scale=2.0, seed=9)
    t = torch.randint(0, 152064, (5,), generator=gen(9), device=DEV).int()
    check_logprobs(z, t, 0, 20)
    check_logprobs(z[:1], t[:1], 0, 32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [40, 3001, 33000])
def test_logprobs_masks_and_ties(dtype, cols):
    low = torch.finfo(dtype).min
    z = randn(12, cols, dtype=dtype, scale=2.0, seed=5)
    z[0, 1:] = -math.inf               # one token is left
    z[1] = -math.inf                   # none is
    z[2, ::2] = -math.inf
    z[3] = low                         # masked with the lowest value, all alike
    z[4, 5:] = low
    z[5] = 0.0                         # all tie
    z[6] = z[6].round()                # many ties
    z[7, : cols // 2] = 7.0
    z[8, -1] = 30.0 if dtype != F16 else 20.0
    z[9] = torch.finfo(dtype).max      # all at the largest value
    z[10, :10], z[10, 10:] = torch.finfo(dtype).max, low
    z[11, cols - 3:], z[11, : cols - 3] = 1.0, -math.inf
    t = torch.tensor([0, 3, 1, 2, 7, cols - 1, 0, cols - 1, cols - 1, 5, 3, cols - 1], device=DEV)
    for top in (0, 1, 7, 32):
        check_logprobs(z, t, 0, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [3001, 40000, 152064])
def test_top_of_rows_with_few_distinct_logits(dtype, cols):
    """Masks that leave fewer tokens than asked for, ties at the last place in the first and last columns, and large
    logits at periods that meet the kernel's groups of threads."""
    low, g = torch.finfo(dtype).min, gen(2)
    for n in (3, 40):
        z = torch.full((n, cols), -math.inf, dtype=dtype, device=DEV)
        for i in range(n):
            kind = i % 8
            if kind < 3:  # 0 to 24 tokens are left, masked by -inf, -1e4 or the lowest value
                z[i] = (-math.inf, -1e4, low)[kind]
                left = torch.randint(0, cols, (1 + (i * 5) % 24,), generator=g, device=DEV)
                z[i, left] = torch.randn(len(left), generator=g, device=DEV).to(dtype)
            elif kind == 3:
                z[i] = 0.5
                z[i, -40:] = 0.75  # the ties of the top are in the last columns
            elif kind == 4:
                z[i] = torch.randint(0, 3, (cols,), generator=g, device=DEV).to(dtype)
            elif kind == 5:
                z[i] = torch.randn(cols, generator=g, device=DEV).to(dtype)
                z[i, 5::512] += 20  # one vector position of one group
            elif kind == 6:
                z[i] = 0
                z[i, 8::1024], z[i, 9::1024] = 3, 4
            else:
                z[i, :] = 1
                z[i, 1::2] = -math.inf
        t = torch.zeros(n, dtype=torch.int64, device=DEV)
        for top in (1, 5, 32):
            check_logprobs(z, t, 0, top)
            check_logprobs(z[:, 1:], t, 0, top)


@pytest.mark.parametrize("dtype", TYPES)
def test_logprobs_and_gradient_of_minus_infinity_beside_very_low_logits(dtype):
    """-inf has probability 0 even where the largest logit is the type's lowest value or not far from it."""
    low = torch.finfo(dtype).min
    tops = [low, low / 2, -1e4, -1e36, -1e37, -2e37, 1e36, 2e37, 1e38] if dtype != F16 else [low, -65000.0, -60032.0, -59000.0, 60000.0, 65000.0]
    z = torch.full((len(tops), 4001), -math.inf, dtype=dtype, device=DEV)
    for i, v in enumerate(tops):
        z[i, i::7] = v
    t = torch.arange(len(tops), device=DEV)
    check_logprobs(z, t, 0, 3)
    check_logprob_grad(z, t, 0, *grads_of(len(tops), 1))


@pytest.mark.parametrize("dtype", TYPES)
def test_logprobs_of_nan_and_infinity(dtype):
    z = randn(4, 500, dtype=dtype, seed=1)
    z[0, 3], z[1, 4], z[2] = math.nan, math.inf, math.nan
    t = torch.tensor([5, 5, 5, 5], device=DEV)
    r = V.token_logprobs(z, t, top=4)
    for x in (r.logprob, r.entropy, r.lse):
        assert x[:3].isnan().logical_or(x[:3] == math.inf).all() and x[3].isfinite()
    assert ((r.top_index >= -1) & (r.top_index < 500)).all()
    check_logprobs(z[3:], t[3:], 0, 4)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_logprobs_strides_shapes_and_offsets(dtype):
    big = randn(24, 1100, dtype=dtype, scale=2.0, seed=2)
    t = torch.randint(100, 160, (24,), generator=gen(1), device=DEV)
    for z in (big[:, :1000], big[:, 1:1000], big[:, 3:1100], big[::2, 5:900], big[:1].expand(24, 1100), big.t()[:24, :24]):
        tt = t[: z.shape[0]]
        check_logprobs(z, torch.where(tt < 100 + z.shape[1], tt, 100), 100, 5)
    z3 = big[:, :900].reshape(4, 6, 900)[:, :-1]  # a slice of the sequence
    r = V.token_logprobs(z3, t.view(4, 6)[:, 1:], lo=100, top=3)
    assert r.logprob.shape == (4, 5) and r.top_index.shape == (4, 5, 3)
    flat = V.TokenLogprobs(*(x.reshape(20, *x.shape[2:]) for x in r))
    check_logprobs(z3.reshape(20, 900), t.view(4, 6)[:, 1:].reshape(20), 100, 3, flat)
    empty = V.token_logprobs(big[:0], t[:0], top=2)
    assert empty.logprob.shape == (0,) and empty.top_index.shape == (0, 2)


def ref_grad(z, t, lo, gl, gh, gz):
    lp, lse, empty = ref_log_p(z)
    h = ref_logprobs(z, t, lo)[1].unsqueeze(1)
    p = lp.exp()
    known = (t >= lo) & (t < lo + z.shape[1])
    gl = torch.where(known, gl.double(), 0.0).unsqueeze(1)
    gh, gz = gh.double().unsqueeze(1), gz.double().unsqueeze(1)
    hot = torch.arange(z.shape[1], device=DEV).unsqueeze(0) == (t - lo).unsqueeze(1)
    plp = torch.where(p > 0, p * lp, 0.0)
    g = gl * (hot.double() - p) - gh * (plp + p * h) + gz * p
    size = gl.abs() * (hot.double() + p) + gh.abs() * (plp.abs() + p * h.abs()) + gz.abs() * p
    none = empty.unsqueeze(1).expand_as(g)
    return torch.where(none, 0.0, g), torch.where(none, 0.0, size)


def grads_of(n, seed):
    return randn(n, seed=seed), randn(n, scale=0.3, seed=seed + 1), randn(n, scale=0.1, seed=seed + 2)


def check_logprob_grad(z, t, lo, gl, gh, gz, out=None, **kw):
    """p is off by S's error and that of its argument (|lp| weighted); its factors by a few roundings; the type rounds once."""
    r = V.token_logprobs(z, t, lo=lo)
    ref, size = ref_grad(z, t, lo, gl, torch.zeros_like(gl) if gh is None else gh, torch.zeros_like(gl) if gz is None else gz)
    got = V.token_logprobs_grad(z, t, r.lse, r.entropy, gl, gh, grad_lse=gz, lo=lo, out=out, **kw)
    lp, lse, _ = ref_log_p(z)
    # e is 0 below e^-120; the 32 bits of lse count up to 1024, beyond which the kernel does not use them
    rel = 4 * stat_rel(z) + U * (6 + 4 * lp.abs().nan_to_num(0, 0, 0).clamp(max=120) + 4 * lse.abs().clamp(max=1024).unsqueeze(1))
    assert_close(got, ref, rel * size + half(z.dtype) * ref.abs() + tiny(z.dtype) + 2.0 ** -126)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [1, 2, 9, 255, 4099, 32000])
def test_logprob_grad(dtype, cols):
    n = 37
    z = randn(n, cols, dtype=dtype, scale=3.0, seed=cols)
    t = torch.randint(0, cols, (n,), generator=gen(n), device=DEV)
    t[0], t[5] = -1, cols  # no targets
    gl, gh, gz = grads_of(n, 7)
    gl[3] = gh[3] = gz[3] = 0.0
    check_logprob_grad(z, t, 0, gl, gh, gz)
    check_logprob_grad(z, t, 0, gl, None, None)
    got = check_logprob_grad(z[3:4], t[3:4], 0, gl[3:4], None, None)
    assert not got.any()


@pytest.mark.parametrize("dtype", TYPES)
def test_logprob_grad_masks(dtype):
    z = randn(10, 3001, dtype=dtype, scale=2.0, seed=3)
    z[0] = -math.inf
    z[1, ::2] = -math.inf
    z[2, 5:] = torch.finfo(dtype).min
    z[3] = 1.0
    z[4, 1:] = -math.inf
    z[6] = torch.finfo(dtype).min  # a row masked with the lowest value throughout
    z[7] = torch.finfo(dtype).max
    z[8] += 3000                   # logits far from 0
    z[9, ::3] = torch.finfo(dtype).max
    t = torch.tensor([1, 7, 2, 3, 0, -1, 5, 6, 7, 8], device=DEV)
    got = check_logprob_grad(z, t, 0, *grads_of(10, 1))
    assert got.isfinite().all() and not got[0].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_logprob_grad_strides_and_in_place(dtype):
    big = randn(20, 1100, dtype=dtype, scale=2.0, seed=2)
    t = torch.randint(100, 1000, (20,), generator=gen(1), device=DEV)
    gl, gh, gz = grads_of(20, 4)
    for z in (big[:, :1000], big[:, 1:1000], big[::2, 5:1005]):
        k = z.shape[0]
        check_logprob_grad(z, t[:k], 100, gl[:k], gh[:k], gz[:k])
        b = z.clone()
        a = check_logprob_grad(b, t[:k], 100, gl[:k], gh[:k], gz[:k])
        r = V.token_logprobs(b, t[:k], lo=100)
        c = V.token_logprobs_grad(b, t[:k], r.lse, r.entropy, gl[:k], gh[:k], grad_lse=gz[:k], lo=100, out=b)
        assert c is b and torch.equal(a, b)
        wide = torch.full((k, z.shape[1] + 9), 5.0, dtype=dtype, device=DEV)
        check_logprob_grad(z, t[:k], 100, gl[:k], gh[:k], gz[:k], out=wide[:, 2:2 + z.shape[1]])
        assert (wide[:, :2] == 5).all() and (wide[:, 2 + z.shape[1]:] == 5).all()  # beside the rows nothing is written


@pytest.mark.parametrize("dtype", TYPES)
def test_logprob_grad_in_place_of_far_rows(dtype):
    """Rows beyond what lse holds are read again before they are overwritten, at any number of pieces of a row."""
    z = randn(5, 40001, dtype=dtype, scale=2.0, seed=3)
    z[1] = torch.finfo(dtype).min
    z[2] += 3000
    z[3] = torch.finfo(dtype).max
    t = torch.tensor([1, 40000, 2, 3, 0], device=DEV)
    gl, gh, gz = grads_of(5, 1)
    want = check_logprob_grad(z, t, 0, gl, gh, gz)
    r = V.token_logprobs(z, t)
    V.token_logprobs_grad(z, t, r.lse, r.entropy, gl, gh, grad_lse=gz, out=z)
    assert torch.equal(z, want)


def test_logprob_grad_beside_the_logits():
    big = randn(6, 640, seed=3)
    z, out = big[:, :300], big[:, 320:620]
    t = torch.randint(0, 300, (6,), generator=gen(1), device=DEV)
    gl, gh, gz = grads_of(6, 1)
    want = check_logprob_grad(z, t, 0, gl, gh, gz)
    r = V.token_logprobs(z, t)
    assert torch.equal(V.token_logprobs_grad(z, t, r.lse, r.entropy, gl, gh, grad_lse=gz, out=out), want)
    for bad in (big[:, 8:308], big[:, 290:590], big.view(-1)[:1800].view(6, 300)):
        with pytest.raises(RuntimeError, match="overlaps"):
            V.token_logprobs_grad(z, t, r.lse, r.entropy, gl, gh, out=bad)


def test_logprob_grad_against_differences():
    n, cols = 3, 41
    z = randn(n, cols, scale=1.5, seed=8)
    t = torch.tensor([3, 40, -1], device=DEV)
    gl, gh, gz = grads_of(n, 2)
    got = V.token_logprobs_grad(z, t, *(lambda r: (r.lse, r.entropy))(V.token_logprobs(z, t)), gl, gh, grad_lse=gz)

    def f(x):
        lp, h, lse = ref_logprobs(x, t)[:3]
        return (lp * gl.double()).sum() + (h * gh.double()).sum() + (lse * gz.double()).sum()
    step = 1e-5  # in 64 bits: the difference is off by about step^2 and 1e-16 * 100 / step
    for i in range(n):
        for j in range(cols):
            a, b = z.double().clone(), z.double().clone()
            a[i, j] += step
            b[i, j] -= step
            d = float(f(a) - f(b)) / (2 * step)
            assert abs(float(got[i, j]) - d) <= 1e-8 + 200 * U * (1 + abs(d))


def test_logprobs_autograd():
    z = randn(6, 300, dtype=F32, scale=2.0, seed=1).requires_grad_()
    t = torch.randint(0, 300, (6,), generator=gen(1), device=DEV)
    r = V.token_logprobs(z, t, top=3)
    assert not r.top_logprob.requires_grad and not r.top_index.requires_grad
    gl, gh, gz = grads_of(6, 3)
    ((r.logprob * gl).sum() + (r.entropy * gh).sum() + (r.lse * gz).sum()).backward()
    assert torch.equal(z.grad, V.token_logprobs_grad(z.detach(), t, r.lse.detach(), r.entropy.detach(), gl, gh, grad_lse=gz))
    z.grad = None
    (-V.token_logprobs(z, t).logprob.mean()).backward()  # an expanded gradient
    ref = torch.autograd.grad(torch.nn.functional.cross_entropy(z.double(), t), z)[0]
    assert_close(z.grad, ref, 300 * U * ref.abs() + 1e-9)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cuts", [[0, 500], [0, 1, 30, 500], [0, 100, 200, 300, 400, 500]])
def test_shards_give_the_whole(dtype, cuts):
    n, lo = 9, 1000
    z = randn(n, 500, dtype=dtype, scale=2.0, seed=6)
    z[3, 100:] = -math.inf
    z[4] = -math.inf
    z[5] = 2.0
    t = lo + torch.randint(0, 500, (n,), generator=gen(2), device=DEV)
    t[3], t[7] = lo + 5, -1
    for top in (0, 5, 32):
        recs = torch.stack([V.token_record(z[:, a:b], t, top=top, lo=lo + a) for a, b in zip(cuts, cuts[1:])])
        r = check_logprobs(z, t, lo, top, V.merge_token_records(recs, [lo + a for a in cuts[:-1]]))
    gl, gh, gz = grads_of(n, 5)
    ref, size = ref_grad(z, t, lo, gl, gh, gz)
    got = torch.cat([V.token_logprobs_grad(z[:, a:b], t, r.lse, r.entropy, gl, gh, grad_lse=gz, lo=lo + a, sharded=True)
                     for a, b in zip(cuts, cuts[1:])], 1)
    assert_close(got, ref, 400 * U * size + half(dtype) * ref.abs() + tiny(dtype))


def test_logprob_refusals():
    z, t = torch.zeros(3, 8, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    f = torch.zeros(3, device=DEV)
    recs = torch.zeros(2, 3, 4, device=DEV)
    for call, exc in ((lambda: V.token_logprobs(z, t[:2]), AssertionError), (lambda: V.token_logprobs(z, t.float()), ValueError),
                      (lambda: V.token_logprobs(z.int(), t), ValueError), (lambda: V.token_logprobs(z[:, :0], t), ValueError),
                      (lambda: V.token_logprobs(z, t.cpu()), ValueError), (lambda: V.token_logprobs_grad(z, t, f, None, f, f), ValueError),
                      (lambda: V.token_logprobs_grad(z, t, f, f, f.double()), ValueError), (lambda: V.token_logprobs_grad(z, t, f, f, f[:2]), ValueError),
                      (lambda: V.token_logprobs_grad(z, t, f, f, f, out=z.half()), ValueError),
                      (lambda: V.token_logprobs_grad(z, t, f, f, f, out=torch.zeros(8, 3, device=DEV).t()), ValueError),
                      (lambda: V.merge_token_records(recs, [0]), AssertionError), (lambda: V.merge_token_records(recs, [8, 0]), RuntimeError),
                      (lambda: V.merge_token_records(recs[:, :, :3], [0, 8]), ValueError)):
        with pytest.raises(exc):
            call()


# ---- streams and graphs ------------------------------------------------------------------------
def everything(seed):
    """A pass through every operator on inputs of its own: (run, inputs that a replay reads)."""
    state = make_state([33, 5000, 800], BF16, F32, True, seed=seed)
    grads = {n: randn(e["param"].numel(), dtype=BF16, scale=0.5, seed=seed + i) for i, (n, e) in enumerate(state.items())}
    opt = OPT.ShardAdamW(state, max_norm=1.0, **HYPER)
    w, ids = randn(3000, 64, dtype=BF16, seed=seed), spread("skewed", 3000, 3000, 0, seed)
    z, t = randn(70, 5000, dtype=BF16, scale=2.0, seed=seed), torch.randint(0, 5000, (70,), generator=gen(seed), device=DEV)
    gl, gh, _ = grads_of(70, seed)
    clipped = randn(4000, seed=seed)

    def run():
        x = V.embedding(ids, w, scale=2.0)
        dw = V.embedding_grad(x, ids, 3000, scale=2.0, dtype=F32)
        r = V.token_logprobs(z, t, top=8)
        few = V.token_logprobs(z[:2], t[:2], top=8)
        dz = V.token_logprobs_grad(z, t, r.lse, r.entropy, gl, gh)
        norm = opt.step(grads)
        c = clipped.clone()
        OPT.clip_grads([c], 1.0)
        return [x, dw, *r, *few, dz, norm, c]
    return run, state, (w, z, clipped)


def test_side_streams_and_graph_replays():
    run, state, inputs = everything(1)
    start = clone_state(state)

    def reset():
        for n, e in state.items():
            for s, v in e.items():
                v.copy_(start[n][s])
    eager = [x.clone() for x in run()]
    once = clone_state(state)
    reset()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, got))
    reset()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = run()
    assert all(torch.equal(state[n][s], start[n][s]) for n in state for s in state[n])  # capturing runs nothing
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, held))
    assert all(torch.equal(state[n][s], once[n][s]) for n in state for s in state[n])
    g.replay()  # the step counts advance on the device
    torch.cuda.synchronize()
    assert all(float(state[n]["step"]) == float(start[n]["step"]) + 2 for n in state)
    w, z, clipped = inputs  # new values at the same addresses
    w.mul_(0.5)
    z.mul_(0.5)
    clipped.add_(1.0)
    reset()
    g.replay()
    torch.cuda.synchronize()
    new = [x.clone() for x in held]
    reset()
    assert all(torch.equal(a, b) for a, b in zip(new, run()))


def test_two_graphs_replayed_at_once():
    runs = [everything(s) for s in (3, 4)]
    starts = [clone_state(r[1]) for r in runs]

    def reset():
        for (_, state, _), start in zip(runs, starts):
            for n, e in state.items():
                for s, v in e.items():
                    v.copy_(start[n][s])
    eager = [[x.clone() for x in r[0]()] for r in runs]
    graphs, held = [], []
    for r in runs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(r[0]())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in runs]
    for _ in range(5):
        reset()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for e, h in zip(eager, held):
            assert all(torch.equal(a, b) for a, b in zip(e, h))


@pytest.mark.multigpu
def test_tensors_on_another_device_than_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    dev = torch.device("cuda", 1)
    assert torch.cuda.current_device() == 0
    w, ids = torch.randn(20, 16, device=dev), torch.tensor([3, 19], device=dev)
    assert torch.equal(V.embedding(ids, w), w[ids]) and torch.cuda.current_device() == 0
    g = torch.ones(10, device=dev)
    assert abs(float(OPT.clip_grads([g], 1.0)) - math.sqrt(10)) < 1e-5 and torch.cuda.current_device() == 0


# ---- the operators together, on a migrated state -------------------------------------------------
def test_a_training_step_on_a_resharded_state():
    """TP4 -> TP2 with a vocabulary-parallel wte, then one step of a one-layer model (embedding, one gated
    block, lm_head, cross entropy) on both target ranks' shards, against the whole model in 64 bits."""
    spec = scaled_spec(SPECS["llama2-7b"], name="m", hidden=32, n_layers=1, n_heads=4, ffn=48, vocab=80, vocab_parallel_wte=True)
    cfg = ReshardConfig("step", spec, [[[0, 1, 2, 3]]], [[[0, 1]]])
    spl, tpl = cfg.layouts()
    kinds = dict(S.SUBFIELDS)
    src = {r: {n: {s: S.to_torch(a, kinds[s], DEV if kinds[s] != "meta" else None) for s, a in e.items()} for n, e in st.items()}
           for r, st in S.host_states(spl, S.SUBFIELDS, seed=3, distinct_steps=True).items()}
    states = M.reshard_local(spl, tpl, src, S.expected_sub_fields(), DEV, order="semantic", minimum_est_peers=1)
    whole = S.host_states(mesh_layout(spec, [[[0]]]), S.SUBFIELDS, seed=3, distinct_steps=True)[0]
    ids = torch.randint(0, spec.vocab, (3, 17), generator=gen(1), device=DEV)
    x_ids, targets = ids[:, :-1], ids[:, 1:].clone()
    targets[0, :4] = -1
    count = int((targets >= 0).sum())
    used = ["wte.weight", "h.0.mlp.gate_proj.weight", "h.0.mlp.up_proj.weight", "h.0.mlp.down_proj.weight", "lm_head.weight"]

    # the whole model, 64 bits, from the bf16 parameters
    full = {n: torch.from_numpy(S.bf16_to_f32(whole[n]["param"])).double().to(DEV).requires_grad_() for n in used}

    def block(x, gate, up, down):
        return (torch.nn.functional.silu(x @ gate.t()) * (x @ up.t())) @ down.t()
    e = full["wte.weight"][x_ids] * 4.0
    y = e + block(e, *(full[f"h.0.mlp.{k}_proj.weight"] for k in ("gate", "up", "down")))
    logits = y @ full["lm_head.weight"].t()
    loss = torch.nn.functional.cross_entropy(logits.reshape(-1, spec.vocab), targets.reshape(-1), ignore_index=-1)
    loss.backward()
    ref_norm = math.sqrt(sum(float(p.grad.square().sum()) for p in full.values()))

    # the two ranks, one after the other on one device; sums over ranks are written out
    leaf = {r: {n: states[r][n]["param"].float().requires_grad_() for n in used} for r in (0, 1)}
    ranges = {r: {n: V.shard_range(tpl.layout[r][n]) for n in ("wte.weight", "lm_head.weight")} for r in (0, 1)}
    x = sum(V.embedding(x_ids, leaf[r]["wte.weight"], scale=4.0, lo=ranges[r]["wte.weight"][0]) for r in (0, 1))
    h = x + sum(block(x, *(leaf[r][f"h.0.mlp.{k}_proj.weight"] for k in ("gate", "up", "down"))) for r in (0, 1))
    z = {r: h @ leaf[r]["lm_head.weight"].t() for r in (0, 1)}
    flat = targets.reshape(-1)
    recs = torch.stack([V.token_record(z[r].detach().reshape(-1, z[r].shape[-1]), flat, lo=ranges[r]["lm_head.weight"][0]) for r in (0, 1)])
    lp = V.merge_token_records(recs, [ranges[r]["lm_head.weight"][0] for r in (0, 1)])
    got_loss = -lp.logprob.sum() / count
    # tens of products and sums of length <= 80 in 32 bits on each path to the loss
    rel = 2e-5
    assert abs(float(got_loss) - float(loss.detach())) <= rel * float(loss.detach())
    gl = torch.full_like(lp.logprob, -1.0 / count)
    dz = {r: V.token_logprobs_grad(z[r].detach().reshape(-1, z[r].shape[-1]), flat, lp.lse, lp.entropy, gl, lo=ranges[r]["lm_head.weight"][0],
                                   sharded=True).view_as(z[r]) for r in (0, 1)}
    torch.autograd.backward([z[0], z[1]], [dz[0], dz[1]])
    total = torch.zeros(1, dtype=torch.float64, device=DEV)
    counted = {r: OPT.counted_spans(tpl, r) for r in (0, 1)}
    for r in (0, 1):
        total += OPT.grad_sumsq({n: leaf[r][n].grad for n in used}, counted=counted[r])
    assert abs(math.sqrt(float(total)) - ref_norm) <= 1e-4 * ref_norm
    for r in (0, 1):
        for n in used:
            m = tpl.layout[r][n]
            d, i, g = m.tp_meta
            want = full[n].grad.chunk(g, dim=d)[i]
            assert_close(leaf[r][n].grad, want, 1e-4 * float(want.abs().max()), n)
        old = {n: {s: t.clone() for s, t in states[r][n].items()} for n in states[r]}
        opt = OPT.ShardAdamW(states[r], max_norm=0.5 * ref_norm, counted=counted[r], **HYPER)
        norm = opt.step({n: leaf[r][n].grad for n in used}, sumsq=total)
        assert abs(float(norm) - ref_norm) <= 1e-4 * ref_norm
        grads = {n: leaf[r][n].grad for n in used}
        check_adam({n: old[n] for n in used}, states[r], grads, 0.5 * ref_norm / (float(norm) + 1e-6), CLIP_REL)
        for n in states[r]:
            if n not in used:
                assert all(torch.equal(states[r][n][s].reshape(-1), old[n][s].reshape(-1)) for s in old[n])


def test_offsets_past_32_bits_in_logits():
    n, cols = 14200, 152064  # 2.16e9 logits
    z = torch.zeros(n, cols, dtype=BF16, device=DEV)
    z[-2:] = randn(2, cols, dtype=BF16, scale=2.0, seed=1)
    t = torch.randint(0, cols, (n,), generator=gen(1), device=DEV)
    r = V.token_logprobs(z, t, top=5)
    check_logprobs(z[-2:], t[-2:], 0, 5, V.TokenLogprobs(*(x[-2:] for x in r)))
    gl, gh, _ = grads_of(n, 1)
    g = V.token_logprobs_grad(z, t, r.lse, r.entropy, gl, gh)
    ref, size = ref_grad(z[-2:], t[-2:], 0, gl[-2:], gh[-2:], torch.zeros_like(gl[-2:]))
    assert_close(g[-2:], ref, 400 * U * size + half(BF16) * ref.abs() + tiny(BF16))


def test_steps_of_one_tensor_past_32_bits():
    n = (1 << 32) + 4096 + 7  # elements: a bf16 state without a master
    state = {"w": {"param": torch.zeros(n, dtype=BF16, device=DEV), "exp_avg": torch.zeros(n, dtype=BF16, device=DEV),
                   "exp_avg_sq": torch.zeros(n, dtype=BF16, device=DEV), "step": torch.tensor(0.0, device=DEV)}}
    g = torch.zeros(n, dtype=BF16, device=DEV)
    at = torch.tensor([0, 4095, 1 << 31, (1 << 32) + 1, n - 1], device=DEV)
    g[at] = torch.tensor([1.0, -2.0, 0.5, 3.0, -1.0], dtype=BF16, device=DEV)
    norm = OPT.ShardAdamW(state, max_norm=1e3, **HYPER).step({"w": g})
    ref = math.sqrt(1 + 4 + 0.25 + 9 + 1)
    assert abs(float(norm) - ref) <= (SUMSQ_REL / 2 + U) * ref
    small = {"w": {s: (t.clone() if s == "step" else torch.zeros(5, dtype=BF16, device=DEV)) for s, t in state["w"].items()}}
    small["w"]["step"] = torch.tensor(0.0, device=DEV)
    OPT.ShardAdamW(small, max_norm=1e3, **HYPER).step({"w": g[at]})
    for s in ("param", "exp_avg", "exp_avg_sq"):
        assert torch.equal(state["w"][s][at], small["w"][s]), s
        state["w"][s][at] = 0
        assert not state["w"][s].any()


def test_lists_of_the_module_are_checked():
    from suika_b200 import _lib
    ext = _lib.extension()
    x = torch.zeros(4, device=DEV)
    for call in (lambda: ext.grad_sumsq((x,), None), lambda: ext.grad_clip([x, 1], 1.0, None), lambda: ext.embed_lookup(x, x), lambda: ext.embed_lookup(1, 2, 3, 4),
                 lambda: ext.adamw_step([x], [], [x], [x], [x], [1.0], [x], 1e-3, 0.9, 0.9, 1e-8, 0.0, None, None)):
        with pytest.raises(TypeError):
            call()
    state = make_state([10], BF16, F32, True)
    opt = OPT.ShardAdamW(state, **HYPER)
    state["t0"]["exp_avg"].untyped_storage().resize_(0)  # released, as the shrink path of a migration does
    with pytest.raises(RuntimeError):
        opt.step({"t0": torch.zeros(10, device=DEV)})
