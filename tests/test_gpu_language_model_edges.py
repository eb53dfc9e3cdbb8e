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


# ---- infinities and NaN ----


@pytest.mark.parametrize("which", ["q", "k", "v", "d_out"])
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("mask,n,heads,kv_heads,dim,dtype", [("window", 700, 2, 1, 64, torch.bfloat16), ("documents", 900, 2, 2, 128, torch.float16),
                                                             ("causal", 600, 4, 2, 96, torch.bfloat16), ("window", 1700, 1, 1, 128, torch.float16)])
def test_a_bad_token_reaches_what_sees_it_and_nothing_else(which, value, mask, n, heads, kv_heads, dim, dtype):
    g = gen(51)
    x = {"q": randn(g, n, heads, dim, dtype=dtype), "k": randn(g, n, kv_heads, dim, dtype=dtype), "v": randn(g, n, kv_heads, dim, dtype=dtype),
         "d_out": randn(g, n, heads, dim, dtype=dtype)}
    lo, hi = spans_for(mask, n, g)
    at = torch.arange(n, device="cuda")
    low = torch.zeros_like(at) if lo is None else lo
    high = at + 1 if hi is None else hi
    seen = (at >= low[:, None]) & (at < high[:, None])

    def once(how):
        q, k, v, d_out = (x[name] for name in ("q", "k", "v", "d_out"))
        out, lse = cascade_amd.span_attention(q, k, v, lo, hi, **how)
        return out, lse.T[..., None], *cascade_amd.span_attention_backward(d_out, q, k, v, out, lse, lo, hi, **how)
    for how in ({}, {"cap": 20.0, "slopes": torch.linspace(0.01, 0.1, heads, device="cuda")}, {"cap": 1e3}):
        clean = once(how)
        good = x[which].clone()
        bad = torch.zeros(n, dtype=torch.bool, device="cuda")
        bad[n // 2], bad[n // 2 + 70] = True, True
        x[which][bad, 0, 5] = value
        got = once(how)
        x[which] = good
        # rows that are bad or see a bad key, and keys that are bad or that such a row sees
        rows = bad if which in ("q", "d_out") else (seen & bad).any(1)
        keys = (seen & rows[:, None]).any(0) | (bad if which in ("k", "v") else torch.zeros_like(bad))
        for name, a, b in zip(("out", "lse", "d_q", "d_k", "d_v"), got, clean):
            reached = keys if name in ("d_k", "d_v") else rows if which != "d_out" or name == "d_q" else torch.zeros_like(rows)
            # the rest is the same but for the moments at which a running maximum was raised, that is two roundings of the type at most, of the largest terms
            assert torch.isfinite(a[~reached]).all(), name
            assert ((a - b)[~reached].abs() <= (4 * U[dtype] if name != "lse" else 2e-5) * b.abs().max()).all(), name
            if math.isnan(value) and (name != "lse" or which != "v") and (name != "d_v" or which != "v"):
                first = a[:, :1] if name in ("d_k", "d_v") or which in ("q", "d_out") else a
                assert (~torch.isfinite(first[reached])).any(-1).any(-1).all(), name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bad", ["one row of d_out", "one key", "everything"])
def test_a_step_that_has_overflowed_takes_no_longer_than_a_few(dtype, bad):
    """By the tiles that are gone through twice it takes up to three times as long as any other; ten times leave room for a busy machine."""
    g, n = gen(52), 4096
    q, k, v, d_out = (randn(g, n, h, 128, dtype=dtype) for h in (8, 2, 2, 8))

    def step():
        out, lse = cascade_amd.span_attention(q, k, v)
        return (out, *cascade_amd.span_attention_backward(d_out, q, k, v, out, lse))

    def fastest():
        times = []
        for _ in range(4):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            step()
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)
    usual = fastest()
    if bad == "one row of d_out":
        d_out[n - 5] = math.inf
    elif bad == "one key":
        k[3], v[3] = math.nan, math.inf
    else:
        for x in (q, k, v, d_out):
            x.fill_(math.nan)
    overflowed = fastest()
    print(f"{bad}: {1000 * usual:.0f} us, {1000 * overflowed:.0f} us")
    assert not all(torch.isfinite(x).all() for x in step())
    assert overflowed <= 10 * usual


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_a_token_whose_loss_has_overflowed_takes_no_bits_from_the_others(dtype, value):
    g, n, dim, vocab = gen(53), 300, 128, 3000
    hidden, weight = randn(g, n, dim, dtype=dtype), randn(g, vocab, dim, dtype=dtype, scale=2 * dim ** -0.5)
    target = torch.randint(0, vocab, (n,), generator=g, device="cuda", dtype=torch.int32)
    d_loss = torch.full((n,), 3e-3, device="cuda")
    lse = cascade_amd.linear_cross_entropy(hidden, weight, target)[1]
    clean = cascade_amd.linear_cross_entropy_backward(d_loss, hidden, weight, target, lse)[0]
    d_loss[77] = value
    d_hidden, d_weight = cascade_amd.linear_cross_entropy_backward(d_loss, hidden, weight, target, lse)
    rest = torch.arange(n, device="cuda") != 77
    assert torch.equal(d_hidden[rest], clean[rest])
    assert not torch.isfinite(d_hidden[77]).any() and not torch.isfinite(d_weight).any()


# ---- clipping ----


@pytest.mark.parametrize("value,count,finite", [(3e38, 2, False), (3.4e38, 1, True), (1e38, 1000, False), (1e37, 1000, True)])
def test_values_stay_exactly_where_the_norm_is_not_finite(value, count, finite):
    """The norm of 32 bits says whether the values were scaled, also where 64 bits hold a larger one."""
    x = torch.full((count,), value, device="cuda")
    want = x[0].item() * math.sqrt(count)
    out = [torch.zeros_like(x)]
    norm = cascade_amd.clip_gradients([x], 1.0, out=out).item()
    assert math.isfinite(norm) == finite and (not finite or abs(norm - want) <= 2.0 ** -23 * want)
    if finite:
        assert torch.allclose(out[0], torch.full_like(x, count ** -0.5), rtol=1e-5)
    else:
        assert torch.equal(out[0], x)


def test_autograd_notices_that_clipping_has_changed_a_tensor():
    for in_place in (True, False):
        g = torch.full((10,), 3.0, device="cuda")
        scaled = g if in_place else torch.zeros_like(g)
        x = torch.ones(10, device="cuda", requires_grad=True)
        y = (x * scaled).sum()  # keeps `scaled` for its gradient
        before = g._version, scaled._version
        cascade_amd.clip_gradients([g], 1.0, out=None if in_place else [scaled])
        assert scaled._version == before[1] + 1 and (in_place or g._version == before[0])
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():  # tensors without versions
        g = torch.full((10,), 3.0, device="cuda")
        assert cascade_amd.clip_gradients([g], 1.0).item() == pytest.approx(3 * 10 ** 0.5)


# ---- torch.autograd ----


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("wanted", ["qkv", "q", "kv", "v"])
def test_attend_gives_autograd_the_gradients(dtype, wanted):
    g, n, u = gen(61), 260, U[dtype]
    q, k, v = (randn(g, n, h, 64, dtype=dtype) for h in (4, 2, 2))
    lo, hi = spans_for("documents", n, g)
    slopes = torch.linspace(0.01, 0.1, 4, device="cuda")
    for name, x in zip("qkv", (q, k, v)):
        x.requires_grad_(name in wanted)
    way = randn(g, 64, dtype=dtype)  # the gradient of the outputs comes expanded, with strides of 0
    out = cascade_amd.attend(q, k, v, lo, hi, cap=10.0, slopes=slopes)
    (out * way).sum(dtype=torch.float32).backward()
    d_out = way.expand(n, 4, 64)
    want, sums = reference_attention(q.detach(), k.detach(), v.detach(), lo, hi, 0.125, 10.0, slopes, d_out, u)
    within(out.detach(), want["out"], 1.1 * u * (sums["out"] + want["out"].abs()) + 2.0 ** -24, "out")
    for name, x in zip("qkv", (q, k, v)):
        if name not in wanted:
            assert x.grad is None
            continue
        small = 1e-5 * sums["d_" + name].abs().max().item() / u
        within(x.grad, want["d_" + name], 1.1 * (sums["d_" + name] + u * want["d_" + name].abs()) + small + 2.0 ** -24, name)
    with torch.no_grad():
        assert not cascade_amd.attend(q, k, v, lo, hi).requires_grad


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("wanted", ["both", "hidden", "weight"])
def test_next_token_loss_gives_autograd_the_gradients(dtype, wanted):
    g, n, dim, vocab, u = gen(62), 200, 96, 1500, U[dtype]
    hidden, weight = randn(g, n, dim, dtype=dtype), randn(g, vocab, dim, dtype=dtype, scale=0.2)
    target = torch.randint(-1, vocab, (n,), generator=g, device="cuda", dtype=torch.int32)
    target[::7] = -1
    hidden.requires_grad_(wanted != "weight")
    weight.requires_grad_(wanted != "hidden")
    loss = cascade_amd.next_token_loss(hidden, weight, target)
    (loss.sum() * 3.0).backward()  # an expanded gradient
    h, w, there = hidden.detach().double(), weight.detach().double(), target >= 0
    logits = h @ w.T
    at = target.long().clamp(min=0)[:, None]
    size = 1 + (h.abs() @ w.abs().T).max(1).values
    within(loss.detach(), torch.where(there, torch.logsumexp(logits, 1) - logits.gather(1, at)[:, 0], 0.0), 4e-6 * size, "loss")
    p = torch.softmax(logits, 1).scatter_add_(1, at, torch.full((n, 1), -1.0, dtype=torch.float64, device="cuda")) * there[:, None] * 3.0
    off = (u + 1e-5) * p.abs()
    for name, x, want, terms in (("hidden", hidden, p @ w, off @ w.abs()), ("weight", weight, p.T @ h, off.T @ h.abs())):
        if wanted not in ("both", name):
            assert x.grad is None
            continue
        within(x.grad, want, 1.1 * (terms + u * want.abs()) + 4e-6 * p.abs().max() + 2.0 ** -24, name)


def test_gradients_that_are_not_wanted_are_none_and_leave_the_others():
    g = gen(63)
    hidden, weight = randn(g, 150, 64, dtype=torch.bfloat16), randn(g, 700, 64, dtype=torch.bfloat16)
    target = torch.randint(0, 700, (150,), generator=g, device="cuda", dtype=torch.int32)
    d_loss = torch.rand(150, generator=g, device="cuda")
    lse = cascade_amd.linear_cross_entropy(hidden, weight, target)[1]
    both = cascade_amd.linear_cross_entropy_backward(d_loss, hidden, weight, target, lse)
    one = cascade_amd.linear_cross_entropy_backward(d_loss, hidden, weight, target, lse, want_weight=False)
    other = cascade_amd.linear_cross_entropy_backward(d_loss, hidden, weight, target, lse, want_hidden=False)
    assert one[1] is None and other[0] is None and torch.equal(one[0], both[0]) and torch.equal(other[1], both[1])
    assert cascade_amd.linear_cross_entropy_backward(d_loss, hidden, weight, target, lse, False, False) == (None, None)
