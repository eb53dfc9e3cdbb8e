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


# ---- half precision ----


@pytest.mark.parametrize("n,heads,kv_heads,dim", [(400, 2, 2, 64), (400, 4, 2, 128), (1300, 2, 1, 96)])
@pytest.mark.parametrize("what", ["padding", "documents", "heads", "rows"])
def test_large_gradients_elsewhere_take_no_bits_in_half_precision(n, heads, kv_heads, dim, what):
    """Every gradient is as exact as its own terms allow, whatever finite values stand in padding, in another document, in other heads or in later rows."""
    g, dtype, u = gen(41), torch.float16, U[torch.float16]
    q, k, v, d_out = (randn(g, n, h, dim, dtype=dtype) for h in (heads, kv_heads, kv_heads, heads))
    at = torch.arange(n, device="cuda")
    ends = torch.tensor([0, n // 3, n - 60], device="cuda")
    lo, hi = ends[torch.searchsorted(ends, at, right=True) - 1].int(), (at + 1).int()
    size = torch.full((n, heads, 1), 1e-3, device="cuda")
    if what == "padding":
        lo[n - 60:], hi[n - 60:] = 0, 0
    elif what == "documents":
        size[:n // 3] = 1e3
    elif what == "heads":
        size[:, 0] = 1e3
    else:
        size[n // 2::50] = 1e3
    d_out = (d_out * size).half()
    if what == "padding":
        for x in (q, k, v, d_out):
            x[n - 60:] = torch.where(x[n - 60:] > 0, 6e4, -6e4).half()
    out, lse = cascade_amd.span_attention(q, k, v, lo, hi)
    got = cascade_amd.span_attention_backward(d_out, q, k, v, out, lse, lo, hi)
    want, sums = reference_attention(q, k, v, lo, hi, dim ** -0.5, 0.0, None, d_out, u)
    for x, name in zip(got, ("d_q", "d_k", "d_v")):
        # two roundings, and 32-bit sums of what is computed from 32-bit scores: 1e-6 of the terms, whose size `sums` / u bounds; half precision's last step
        within(x, want[name], 1.1 * (sums[name] + u * want[name].abs()) + 2.0 ** -24, name)
