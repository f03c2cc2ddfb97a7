"""The training-step operators at the edges of what their documentation allows, on a B200, against a plain
computation in 64 bits where numbers are compared."""
import math

import pytest
import torch

from suika_b200 import vocab as V
from tests.test_gpu_training import (DEV, TYPES, U, assert_close, grads_of, half, randn, ref_grad, ref_log_p, stat_rel, tiny)

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
