"""The language-model operators at the edges of what they accept, against the same 64-bit references and derived bounds as
test_gpu_language_model.py."""
import math

import pytest

torch = pytest.importorskip("torch")

import cascade_amd  # noqa: E402
from test_gpu_language_model import U, check_attention, gen, randn, reference_attention, spans_for, within  # noqa: E402,F401

pytestmark = pytest.mark.gpu


# ---- caps ----


@pytest.mark.parametrize("cap", [100.0, 1e4, 1e6, 1e8, 1e20, 2.9e38])
@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.float16, 96), (torch.bfloat16, 128)])
def test_large_caps_leave_the_scores(cap, dtype, dim):
    check_attention(210, 4, 2, dim, dtype, "random", cap=cap, seed=31)
    check_attention(190, 2, 2, dim, dtype, "causal", cap=cap, slopes=True, seed=32)


@pytest.mark.parametrize("cap,scale", [(20.0, 4.0), (1e-3, None), (1e-30, None), (3.0, 40.0)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scores_on_both_sides_of_the_cap(cap, scale, dtype):
    check_attention(230, 4, 2, 64, dtype, "causal", cap=cap, scale=scale, seed=33)
    check_attention(1100, 1, 1, 96, dtype, "window", cap=cap, scale=scale, slopes=True, seed=34)


@pytest.mark.parametrize("cap", [1e-40, 1e-38, 1e-3])
def test_products_of_zero_under_a_small_cap(cap):
    """Scores of 0 stay 0 whatever the cap is: rows are the mean of their values, and lse the logarithm of their number."""
    g, n, u = gen(35), 100, U[torch.bfloat16]
    v = randn(g, n, 1, 64, dtype=torch.bfloat16)
    out, lse = cascade_amd.span_attention(torch.zeros_like(v), v, v, cap=cap, scale=2.0)
    count = torch.arange(1, n + 1, device="cuda").double()[:, None]
    want, size = v[:, 0].double().cumsum(0) / count, v[:, 0].double().abs().cumsum(0) / count
    within(out[:, 0], want, 1.1 * u * (size + want.abs()), "out")
    within(lse[0], count[:, 0].log(), 2e-5 * (1 + count[:, 0].log()), "lse")
