"""The training-step operators without a GPU: what a rank counts of its gradients, argument checks of the
C entries (made before any CUDA call) and of the Python ones, and the binding's structures."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest
import torch

from suika_b200 import _lib as L
from suika_b200 import optimizer as OPT
from suika_b200 import vocab as V
from suika_b200.layouts import CONFIGS, SPECS, actual_shape, mesh_layout, scaled_spec, shard_spans
from suika_b200.migration import ParamLayout, TensorMeta
from tests.golden.cases import CASES

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = 1 << 20  # an address that no check dereferences


# ---- counted spans --------------------------------------------------------------------------
def _count(layout):
    """How often each element of each full tensor is counted over the ranks."""
    seen = {}
    for rank, metas in layout.layout.items():
        for name, spans in OPT.counted_spans(layout, rank).items():
            m = metas[name]
            full = tuple(int(s) for s in m.shape)
            got = seen.setdefault(name, np.zeros(full, np.int32))
            shard = np.zeros(actual_shape(m), np.int32)
            for off, n in spans:
                shard.reshape(-1)[off:off + n] += 1
            if m.tp_meta is None:
                got += shard
                continue
            d = m.tp_meta[0] % len(full)
            at = 0
            for lo, hi in shard_spans(full, m.tp_meta, getattr(m, "tp_rule", None)):
                dst = [slice(None)] * len(full)
                src = [slice(None)] * len(full)
                dst[d], src[d] = slice(lo, hi), slice(at, at + hi - lo)
                got[tuple(dst)] += shard[tuple(src)]
                at += hi - lo
    return seen


MESHES = [[[[0]]], [[[0, 1]]], [[[0, 1], [2, 3]]], [[[0, 1]], [[2, 3]]], [[[2, 3], [0, 1]]], [[[0, 1, 2, 3], [4, 5, 6, 7]]]]


@pytest.mark.parametrize("mesh", MESHES)
@pytest.mark.parametrize("fused", [False, True])
def test_every_element_counts_once(mesh, fused):
    spec = scaled_spec(SPECS["qwen2-7b"], name="m", hidden=16, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=4, ffn=24, vocab=40,
                       fused_qkv=fused, vocab_parallel_wte=True)
    seen = _count(mesh_layout(spec, mesh))
    assert seen and all((c == 1).all() for c in seen.values())


@pytest.mark.parametrize("case", sorted(CASES))
def test_every_element_counts_once_in_the_golden_layouts(case):
    for layout in CASES[case]["config"].layouts():
        assert all((c == 1).all() for c in _count(layout).values())


def test_groups_of_different_degree_count_once():
    lay = ParamLayout()
    full = (8, 6)
    lay.layout = {0: {"w": TensorMeta(name="w", dtype=torch.float32, shape=full, tp_meta=(0, 0, 2))},
                  1: {"w": TensorMeta(name="w", dtype=torch.float32, shape=full, tp_meta=(0, 1, 2))},
                  2: {"w": TensorMeta(name="w", dtype=torch.float32, shape=full, tp_meta=(0, 0, 1))},
                  3: {"b": TensorMeta(name="b", dtype=torch.float32, shape=(3,))},
                  4: {"b": TensorMeta(name="b", dtype=torch.float32, shape=(3,)), "s": TensorMeta(name="s", dtype=torch.float32, shape=())}}
    seen = _count(lay)
    assert (seen["w"] == 1).all() and (seen["b"] == 1).all() and seen["s"] == 1
    assert OPT.counted_spans(lay, 2) == {"w": []} and OPT.counted_spans(lay, 4)["b"] == []


def test_shard_range():
    spec = scaled_spec(SPECS["llama2-7b"], name="m", hidden=8, n_layers=1, n_heads=2, ffn=8, vocab=64, vocab_parallel_wte=True)
    lay = mesh_layout(spec, [[[0, 1, 2, 3]]])
    assert [V.shard_range(lay.layout[r]["wte.weight"]) for r in range(4)] == [(0, 16), (16, 32), (32, 48), (48, 64)]
    assert V.shard_range(TensorMeta(name="w", dtype=torch.float32, shape=(5, 2))) == (0, 5)
    with pytest.raises(ValueError, match="contiguous range"):
        V.shard_range(lay.layout[0]["h.0.mlp.down_proj.weight"])


# ---- refusals -------------------------------------------------------------------------------
def test_host_tensors_are_refused():
    x = torch.zeros(4)
    with pytest.raises(ValueError, match="CUDA"):
        OPT.grad_sumsq({"x": x})
    with pytest.raises(ValueError, match="CUDA"):
        OPT.clip_grads([x], 1.0)
    with pytest.raises(ValueError, match="CUDA"):
        OPT.ShardAdamW({"x": {s: torch.zeros(4) for s in ("param", "exp_avg", "exp_avg_sq", "step")}})
    with pytest.raises(ValueError, match="CUDA"):
        V.embedding(torch.zeros(1, dtype=torch.int64), torch.zeros(2, 2))
    with pytest.raises(ValueError, match="CUDA"):
        V.embedding_grad(torch.zeros(1, 2), torch.zeros(1, dtype=torch.int64), 2)
    with pytest.raises(ValueError, match="CUDA"):
        V.token_logprobs(torch.zeros(1, 2), torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        V.token_logprobs_grad(torch.zeros(1, 2), torch.zeros(1, dtype=torch.int64), x, x, x)
    with pytest.raises(ValueError, match="CUDA"):
        V.merge_token_records(torch.zeros(1, 1, 4), [0])


def test_values_are_checked_first():
    with pytest.raises(ValueError, match="max_norm"):
        OPT.clip_grads([torch.zeros(1)], 0.0)
    with pytest.raises(ValueError, match="no gradients"):
        OPT.grad_sumsq({"x": None})
    with pytest.raises(ValueError, match="out of range"):
        OPT.ShardAdamW({"x": {}}, betas=(1.0, 0.9))
    with pytest.raises(ValueError, match="no_decay"):
        OPT.ShardAdamW({"x": {}}, no_decay=["y"])
    with pytest.raises(AssertionError, match="has no param"):
        OPT.ShardAdamW({"x": {}})
    for top in (-1, 33):
        with pytest.raises(ValueError, match="top"):
            V.token_logprobs(torch.zeros(1, 2), torch.zeros(1, dtype=torch.int64), top=top)
        with pytest.raises(ValueError, match="top"):
            V.token_record(torch.zeros(1, 2), torch.zeros(1, dtype=torch.int64), top=top)


def _spans(rows):
    return np.array(rows, dtype=L.GRAD_SPAN_DTYPE)


def test_norm_and_clip_entries_check_their_arguments():
    lib = L.load()
    for rows, word in (([(0, 4, 0, 0)], b"NULL"), ([(FAKE, 4, 7, 0)], b"dtype"), ([(FAKE + 2, 4, L.RS_F32, 0)], b"aligned")):
        t = _spans(rows)
        assert lib.rs_grad_sumsq(t.ctypes.data, 1, FAKE, 1 << 20, FAKE, 0, None) == L.RS_ERR_ARG and word in lib.rs_last_error()
        assert lib.rs_grad_clip(t.ctypes.data, 1, FAKE, 1.0, FAKE, 0, None) == L.RS_ERR_ARG
    t = _spans([(FAKE, 4, 0, 0)])
    assert lib.rs_grad_sumsq(t.ctypes.data, 1, FAKE, 8, FAKE, 0, None) == L.RS_ERR_CAPACITY
    assert lib.rs_grad_sumsq(t.ctypes.data, 1, FAKE, 1 << 20, None, 0, None) == L.RS_ERR_ARG
    assert lib.rs_grad_sumsq(None, 1, FAKE, 1 << 20, FAKE, 0, None) == L.RS_ERR_ARG
    for bad in (0.0, -1.0, float("nan")):
        assert lib.rs_grad_clip(t.ctypes.data, 1, FAKE, bad, FAKE, 0, None) == L.RS_ERR_ARG and b"max_norm" in lib.rs_last_error()


def test_adamw_entry_checks_its_arguments():
    lib = L.load()
    ok = (FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 4, 0.0, 0, 0, 0)

    def call(changes=(), opts=(1e-3, 0.9, 0.99, 1e-8, 1.0), sumsq=None, ws=FAKE, nb=1 << 20):
        row = list(ok)
        for i, v in changes:
            row[i] = v
        t = np.array([tuple(row)], dtype=L.ADAMW_TENSOR_DTYPE)
        return lib.rs_adamw_step(t.ctypes.data, 1, ctypes.byref(L.RsAdamwOpts(*opts)), sumsq, None, ws, nb, 0, None)
    for i in (0, 1, 3, 4, 5):
        assert call([(i, 0)]) == L.RS_ERR_ARG, i
    for i in (0, 1, 2, 3, 4, 5):
        assert call([(i, FAKE + 1)]) == L.RS_ERR_ARG, i
    for i in (8, 9, 10):
        assert call([(i, 3)]) == L.RS_ERR_ARG, i
    assert call([(10, L.RS_F16)]) == L.RS_ERR_ARG
    for opts in ((-1, 0.9, 0.99, 1e-8, 1), (1e-3, 1.0, 0.99, 1e-8, 1), (1e-3, 0.9, 1.0, 1e-8, 1), (1e-3, 0.9, 0.99, -1, 1), (float("nan"), 0.9, 0.99, 1e-8, 1)):
        assert call(opts=opts) == L.RS_ERR_ARG
    assert call(opts=(1e-3, 0.9, 0.99, 1e-8, 0.0), sumsq=FAKE) == L.RS_ERR_ARG
    assert call(nb=8) == L.RS_ERR_CAPACITY and call(ws=None) == L.RS_ERR_CAPACITY and call(ws=FAKE + 8) == L.RS_ERR_CAPACITY


def test_embedding_entries_check_their_arguments():
    lib = L.load()

    def opts(**kw):
        o = L.RsEmbedOpts(4, 8, 8, 0, 8, 8, 1.0, 0, 0, 1, 0, 0)
        for k, v in kw.items():
            setattr(o, k, v)
        return ctypes.byref(o)
    for kw in ({"n_tokens": -1}, {"rows": -1}, {"hidden": -1}, {"weight_stride": -1}, {"dtype": 3}, {"grad_dtype": 9}):
        assert lib.rs_embed_lookup(opts(**kw), FAKE, FAKE, FAKE, 0, None) == L.RS_ERR_ARG, kw
        assert lib.rs_embed_grad(opts(**kw), FAKE, FAKE, FAKE, FAKE, 1 << 30, 0, None) == L.RS_ERR_ARG, kw
    assert lib.rs_embed_lookup(opts(rows=1 << 31), FAKE, FAKE, FAKE, 0, None) == L.RS_ERR_CAPACITY
    assert lib.rs_embed_grad(opts(n_tokens=65537), FAKE, FAKE, FAKE, FAKE, 1 << 30, 0, None) == L.RS_ERR_CAPACITY
    for a in ((None, FAKE, FAKE), (FAKE, None, FAKE), (FAKE, FAKE, None), (FAKE + 4, FAKE, FAKE), (FAKE, FAKE + 2, FAKE), (FAKE, FAKE, FAKE + 2)):
        assert lib.rs_embed_lookup(opts(), *a, 0, None) == L.RS_ERR_ARG, a
    assert lib.rs_embed_grad(opts(), FAKE, FAKE, None, FAKE, 1 << 30, 0, None) == L.RS_ERR_ARG
    assert lib.rs_embed_lookup(opts(n_tokens=0), None, None, None, 0, None) == L.RS_OK
    assert lib.rs_embed_grad(opts(rows=0), None, None, None, None, 0, 0, None) == L.RS_OK


def test_logprob_entries_check_their_arguments():
    lib = L.load()

    def opts(**kw):
        o = L.RsLogprobOpts(4, 8, 8, 0, 0, 1, 0, 0)
        for k, v in kw.items():
            setattr(o, k, v)
        return ctypes.byref(o)
    outs = (FAKE, FAKE, FAKE, FAKE, FAKE)
    for kw in ({"n_rows": -1}, {"cols": 0}, {"stride": -1}, {"top": -1}, {"top": 33}, {"dtype": 5}):
        assert lib.rs_token_logprobs(opts(**kw), FAKE, FAKE, *outs, 0, None) == L.RS_ERR_ARG, kw
        assert lib.rs_token_record(opts(**kw), FAKE, FAKE, FAKE, 0, None) == L.RS_ERR_ARG, kw
        assert lib.rs_token_logprobs_grad(opts(**kw), FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None, FAKE, 8, 0, None) == L.RS_ERR_ARG, kw
    assert lib.rs_token_logprobs(opts(cols=1 << 31), FAKE, FAKE, *outs, 0, None) == L.RS_ERR_CAPACITY
    assert lib.rs_token_logprobs(opts(top=2), FAKE, FAKE, FAKE, FAKE, FAKE, None, FAKE, 0, None) == L.RS_ERR_ARG
    assert lib.rs_token_logprobs(opts(), FAKE + 2, FAKE, *outs, 0, None) == L.RS_ERR_ARG
    assert lib.rs_token_record(opts(), FAKE, FAKE, None, 0, None) == L.RS_ERR_ARG
    assert lib.rs_token_logprobs_grad(opts(), FAKE, FAKE, FAKE, FAKE, FAKE, None, None, FAKE, 7, 0, None) == L.RS_ERR_ARG
    assert lib.rs_token_logprobs_grad(opts(), FAKE, FAKE, FAKE, None, FAKE, FAKE, None, FAKE, 8, 0, None) == L.RS_ERR_ARG
    starts = np.array([0, 8], np.int64)
    for g, n, top in ((0, 1, 0), (65, 1, 0), (1, -1, 0), (1, 1, 33)):
        assert lib.rs_token_merge(FAKE, starts.ctypes.data, g, n, top, *outs, 0, None) == L.RS_ERR_ARG
    assert lib.rs_token_logprobs(opts(n_rows=0), None, None, None, None, None, None, None, 0, None) == L.RS_OK


def test_structures_match_the_header(tmp_path):
    if not shutil.which("gcc"):
        pytest.skip("gcc not found")
    pairs = {"rs_grad_span": L.RsGradSpan, "rs_adamw_tensor": L.RsAdamwTensor, "rs_adamw_opts": L.RsAdamwOpts,
             "rs_embed_opts": L.RsEmbedOpts, "rs_logprob_opts": L.RsLogprobOpts}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{os.path.join(REPO, "include", "suika_reshard.h")}"', "int main(void) {"]
    for cname, cls in pairs.items():
        lines.append(f'  printf("{cname} (sizeof) %zu\\n", sizeof({cname}));')
        lines += [f'  printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-std=c99", str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        cname, field, value = line.split()
        want = ctypes.sizeof(pairs[cname]) if field == "(sizeof)" else getattr(pairs[cname], field).offset
        assert int(value) == want, line
    for dt, cls in ((L.GRAD_SPAN_DTYPE, L.RsGradSpan), (L.ADAMW_TENSOR_DTYPE, L.RsAdamwTensor)):
        assert dt.itemsize == ctypes.sizeof(cls)
        assert all(dt.fields[f][1] == getattr(cls, f).offset for f, _ in cls._fields_)
