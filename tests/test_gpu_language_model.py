"""The language-model operators against plain implementations in 64 bits, written from the formulas.

Bounds are derived, element by element. u is half a unit of the type's last place (2^-8 for bfloat16, 2^-11 for float16,
relative). A result rounded once is off by u |x|; the factors that a kernel rounds to 16 bits before a product (probabilities, score
gradients, loss gradients) bring u times the sum of the absolute terms. What 32-bit sums and exponentials add is far below u and
covered by a tenth of the same sums' u. Nothing here is tuned to what the kernels return."""
import math

import pytest

torch = pytest.importorskip("torch")

import cascade_amd  # noqa: E402
from cascade_amd import language_model as lm  # noqa: E402
from cascade_amd._native import CascadeError  # noqa: E402

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -24}  # half precision's smallest step


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def within(got, want, bound, what):
    got = got.double()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), what
    over = ((got - want).abs() - bound).max().item() if got.numel() else 0.0
    assert over <= 0, f"{what}: {over:.3g} over its bound, error {(got - want).abs().max().item():.3g}"


# ---- spans ----


def spans_of(text, separator):
    lo, target, last = [], [], 0
    for i, t in enumerate(text):
        last = i if t == separator else last
        lo.append(last)
        target.append(text[i + 1] if i + 1 < len(text) and text[i + 1] != separator else -1)
    return lo, list(range(1, len(text) + 1)), target


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 255, 4095, 4096, 4097, 8192, 20011])
@pytest.mark.parametrize("every", [1, 7, 900, 10 ** 9])
def test_spans(n, every):
    g = gen(n)
    text = torch.randint(0, 50257, (n,), generator=g, device="cuda")
    text[torch.randint(0, every, (n,), generator=g, device="cuda") == 0] = 0xFFFF
    want = spans_of(text.tolist(), 0xFFFF)
    got = cascade_amd.token_spans(text.to(torch.int16))
    for a, b, name in zip(got, want, ("lo", "hi", "target")):
        assert a.tolist() == b, name


def test_spans_of_a_slice_and_another_separator():
    text = torch.randint(0, 3, (10001,), generator=gen(3), device="cuda").to(torch.int16)
    part = text[1:]  # not aligned to 16 bytes
    want = spans_of(part.tolist(), 2)
    assert [x.tolist() for x in cascade_amd.token_spans(part, separator=2)] == list(want)
    empty = cascade_amd.token_spans(text[:0])
    assert [x.numel() for x in empty] == [0, 0, 0]


def test_spans_of_a_long_text_look_back_over_tiles_without_separators():
    n = 4096 * 4096 + 4096 * 3 + 5  # tiles of two turns
    text = torch.zeros(n, dtype=torch.int16, device="cuda")
    seps = torch.tensor([5, 4096, 9 * 8192 - 1, n - 20], device="cuda")
    text[seps] = -1
    lo, hi, target = cascade_amd.token_spans(text)
    at = torch.arange(n, device="cuda")
    which = torch.searchsorted(seps, at, right=True)
    want = torch.where(which > 0, seps[(which - 1).clamp(min=0)], 0)
    assert torch.equal(lo.long(), want) and torch.equal(hi.long(), at + 1)
    assert torch.equal((target == -1).nonzero()[:, 0], torch.cat([seps - 1, at[-1:]]))


# ---- attention ----


def reference_attention(q, k, v, lo, hi, scale, cap, slopes, d_out=None, u=0.0):
    """out, lse and the gradients in 64 bits, with the sums that the bounds are made of."""
    q, k, v = q.double(), k.double(), v.double()
    n, heads, dim = q.shape
    group = heads // k.shape[1]
    at = torch.arange(n, device=q.device)
    seen = (at[None] >= lo[:, None]) & (at[None] < hi[:, None])
    got = {"out": torch.zeros_like(q), "lse": torch.zeros(heads, n, dtype=torch.float64, device=q.device)}
    sums = {"out": torch.zeros_like(q)}
    if d_out is not None:
        d_out = d_out.double()
        for name, x in (("d_q", q), ("d_k", k), ("d_v", v)):
            got[name], sums[name] = torch.zeros_like(x), torch.zeros_like(x)
    for h in range(heads):
        c = h // group
        y = scale * (q[:, h] @ k[:, c].T)
        z = cap * torch.tanh(y / cap) if cap else y
        bent = 1 - torch.tanh(y / cap) ** 2 if cap else torch.ones_like(y)
        if slopes is not None:
            z = z - slopes[h].double() * (at[:, None] - at[None]).abs()
        z = z.masked_fill(~seen, -math.inf)
        lse = torch.logsumexp(z, 1)
        p = torch.exp(z - lse.masked_fill(torch.isinf(lse), 0.0)[:, None])
        out = p @ v[:, c]
        got["out"][:, h], got["lse"][h], sums["out"][:, h] = out, lse, p @ v[:, c].abs()
        if d_out is None:
            continue
        go = d_out[:, h]
        ds = p * (go @ v[:, c].T - (go * out).sum(1, keepdim=True)) * bent
        got["d_q"][:, h] = scale * (ds @ k[:, c])
        got["d_k"][:, c] += scale * (ds.T @ q[:, h])
        got["d_v"][:, c] += p.T @ go
        # D is taken from the rounded out, which is off by u (sum p |v| + |out|) an element
        off = (go.abs() * u * (sums["out"][:, h] + out.abs())).sum(1, keepdim=True)
        ds_off = u * ds.abs() + 1.1 * p * off
        sums["d_q"][:, h] = scale * (ds_off @ k[:, c].abs())
        sums["d_k"][:, c] += scale * (ds_off.T @ q[:, h].abs())
        sums["d_v"][:, c] += u * (p.T @ go.abs())
    return got, sums


def spans_for(mask, n, g):
    at = torch.arange(n, device="cuda")
    if mask == "causal":
        return None, None
    if mask == "all":
        return torch.zeros_like(at).int(), torch.full_like(at, n).int()
    if mask == "documents":
        starts = torch.rand(n, generator=g, device="cuda") < 0.03
        return torch.where(starts, at, 0).cummax(0).values.int(), (at + 1).int()
    if mask == "window":
        return (at - 37).int(), (at + 30).int()  # past both ends, too
    if mask == "random":  # any spans, empty and backward ones among them
        lo, hi = (torch.randint(-5, n + 5, (n,), generator=g, device="cuda").int() for _ in range(2))
        return lo, hi
    assert mask == "none"
    return torch.zeros_like(at).int(), torch.zeros_like(at).int()


def check_attention(n, heads, kv_heads, dim, dtype, mask, cap=0.0, slopes=False, scale=None, layout="dense", seed=0):
    g = gen(seed)
    if layout == "packed":
        qkv = randn(g, n, heads + 2 * kv_heads, dim, dtype=dtype)
        q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    elif layout == "heads first":
        q, k, v = (randn(g, h, n, dim, dtype=dtype).transpose(0, 1) for h in (heads, kv_heads, kv_heads))
    elif layout == "odd":  # neither aligned nor in steps of eight
        q, k, v = (randn(g, n, h, dim + 3, dtype=dtype)[:, :, 1:1 + dim] for h in (heads, kv_heads, kv_heads))
    else:
        q, k, v = (randn(g, n, h, dim, dtype=dtype) for h in (heads, kv_heads, kv_heads))
    d_out = randn(g, n, heads, dim, dtype=dtype)
    lo, hi = spans_for(mask, n, g)
    slope = torch.linspace(0.01, 0.5, heads, device="cuda") if slopes else None
    how = dict(lo=lo, hi=hi, scale=scale, cap=cap, slopes=slope)
    out, lse = cascade_amd.span_attention(q, k, v, **how)
    d_q, d_k, d_v = cascade_amd.span_attention_backward(d_out, q, k, v, out, lse, **how)
    u, tiny = U[dtype], TINY[dtype]
    at = torch.arange(n, device="cuda")
    a = torch.zeros_like(at) if lo is None else lo.long().clamp(min=0)
    b = at + 1 if hi is None else hi.long().clamp(max=n)
    want, sums = reference_attention(q, k, v, a, b, dim ** -0.5 if scale is None else scale, cap, slope, d_out, u)
    empty = a >= b
    assert torch.equal(torch.isinf(lse), empty.expand(heads, n)) and not (lse == math.inf).any()
    there = ~empty
    within(lse[:, there], want["lse"][:, there], 2e-5 * (1 + want["lse"][:, there].abs()), "lse")
    within(out, want["out"], 1.1 * u * (sums["out"] + want["out"].abs()) + tiny, "out")
    for name, x in (("d_q", d_q), ("d_k", d_k), ("d_v", d_v)):
        # 1e-5 of the largest entry: gradients that cancel down to what 32-bit sums leave
        small = 1e-5 * sums[name].abs().max().item() / u
        within(x, want[name], 1.1 * (sums[name] + u * want[name].abs()) + small + tiny, name)
    assert (out[empty] == 0).all() and (d_q[empty] == 0).all()
    return q, k, v, out, lse, d_q, d_k, d_v


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 320, 515])
def test_attention_lengths(n, dtype):
    check_attention(n, 2, 1, 64, dtype, "causal", seed=n)


@pytest.mark.parametrize("mask", ["causal", "all", "documents", "window", "random", "none"])
@pytest.mark.parametrize("dim,dtype", [(64, torch.bfloat16), (80, torch.float16), (128, torch.bfloat16), (128, torch.float16)])
def test_attention_spans(mask, dim, dtype):
    check_attention(333, 4, 2, dim, dtype, mask, seed=dim)


@pytest.mark.parametrize("dim", [8, 16, 24, 40, 56, 72, 88, 96, 104, 120])
def test_attention_head_sizes(dim):
    check_attention(150, 3, 1, dim, torch.bfloat16, "causal", seed=dim)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (8, 2), (6, 1), (16, 4), (5, 5)])
def test_attention_shared_heads(heads, kv_heads):
    check_attention(190, heads, kv_heads, 64, torch.bfloat16, "documents", seed=heads)


@pytest.mark.parametrize("layout", ["packed", "heads first", "odd"])
@pytest.mark.parametrize("dim", [64, 80])
def test_attention_layouts(layout, dim):
    check_attention(140, 4, 2, dim, torch.bfloat16, "causal", layout=layout, seed=7)


@pytest.mark.parametrize("cap,slopes", [(30.0, False), (2.0, False), (0.0, True), (5.0, True)])
@pytest.mark.parametrize("mask", ["causal", "all", "random"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_caps_and_distances(cap, slopes, mask, dtype):
    check_attention(210, 4, 2, 64, dtype, mask, cap=cap, slopes=slopes, seed=11)


def test_attention_of_a_long_text():
    check_attention(3001, 2, 1, 128, torch.bfloat16, "causal", seed=5)
    check_attention(2800, 2, 2, 96, torch.float16, "documents", seed=6)
    check_attention(4200, 16, 16, 8, torch.bfloat16, "random", seed=9)  # tiles in the order of their work
    check_attention(2111, 32, 2, 16, torch.float16, "documents", seed=10)  # shared heads in that order, too


@pytest.mark.parametrize("n", [8193, 9001])
@pytest.mark.parametrize("mask", ["whole", "random"])
def test_the_order_of_tiles_changes_no_result(n, mask):
    g = gen(n)
    q, k, v, d_out = (randn(g, n, h, 64, dtype=torch.bfloat16) for h in (8, 2, 2, 8))
    lo, hi = spans_for("random", n, g)
    if mask == "whole":  # as without spans, where no order is made
        lo, hi = torch.zeros_like(lo), torch.arange(1, n + 1, device="cuda", dtype=torch.int32)
    aside = [torch.cat([x[:1], x])[1:] for x in (lo, hi)]  # four bytes off the alignment of wide loads
    assert aside[0].data_ptr() % 16 == 4
    found = []
    for spans in [(lo, hi), aside] + [(None, None)] * (mask == "whole"):
        out, lse = cascade_amd.span_attention(q, k, v, *spans)
        found.append((out, lse, *cascade_amd.span_attention_backward(d_out, q, k, v, out, lse, *spans)))
    for other in found[1:]:
        assert all(torch.equal(a, b) for a, b in zip(found[0], other))


@pytest.mark.parametrize("mask", ["causal", "all", "window", "random", "none"])
def test_attention_of_few_heads_shares_out_keys(mask):
    check_attention(1301, 2, 1, 64, torch.bfloat16, mask, seed=21)
    check_attention(1100, 1, 1, 96, torch.float16, mask, cap=5.0, slopes=True, seed=22)


def test_attention_of_large_scores():
    check_attention(300, 2, 2, 64, torch.bfloat16, "causal", scale=4.0, seed=8)  # a softmax of one or two keys a row


def test_half_precision_keeps_small_gradients():
    """Gradients of 1e-4 times smaller d_out than usual are as exact as others, down to what the type holds."""
    g = gen(9)
    q, k, v = (randn(g, 400, 2, 64, dtype=torch.float16) for _ in range(3))
    d_out = randn(g, 400, 2, 64, dtype=torch.float16, scale=1e-3)
    lo, hi = spans_for("all", 400, g)
    out, lse = cascade_amd.span_attention(q, k, v, lo=lo, hi=hi)
    got = cascade_amd.span_attention_backward(d_out, q, k, v, out, lse, lo=lo, hi=hi)
    want, sums = reference_attention(q, k, v, lo, hi, 0.125, 0.0, None, d_out, U[torch.float16])
    for x, name in zip(got, ("d_q", "d_k", "d_v")):
        within(x, want[name], 1.1 * (sums[name] + U[torch.float16] * want[name].abs()) + 2.0 ** -24, name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv_heads,dim,n", [(2, 2, 64, 500), (4, 1, 128, 500), (3, 3, 88, 500), (2, 1, 64, 1700), (2, 2, 80, 1700)])
def test_what_a_row_may_not_see_may_hold_anything(dtype, heads, kv_heads, dim, n):
    """Infinities and NaN in padding, and in one document of three, change nothing elsewhere, forwards and backwards."""
    g = gen(13)
    text = n - 30  # padding behind it
    at = torch.arange(n, device="cuda")
    ends = torch.tensor([0, n - 350, n - 199, text], device="cuda")
    lo = ends[torch.searchsorted(ends, at, right=True) - 1].int()
    hi = (at + 1).int()
    lo[text:], hi[text:] = 0, 0
    q, d_out = (randn(g, n, heads, dim, dtype=dtype) for _ in range(2))
    k, v = (randn(g, n, kv_heads, dim, dtype=dtype) for _ in range(2))

    def once(q, k, v, d_out, **how):
        out, lse = cascade_amd.span_attention(q, k, v, lo, hi, **how)
        return out, lse.T, *cascade_amd.span_attention_backward(d_out, q, k, v, out, lse, lo, hi, **how)
    for how in ({}, {"cap": 10.0, "slopes": torch.linspace(0.01, 0.1, heads, device="cuda")}):
        clean = once(q, k, v, d_out, **how)
        for where in (slice(text, n), slice(n - 350, n - 199)):
            spoilt = [x.clone() for x in (q, k, v, d_out)]
            for i, x in enumerate(spoilt):
                x[where][i % 2::2] = math.nan
                x[where][(i + 1) % 2::3] = math.inf
            got = once(*spoilt, **how)
            rest = torch.ones(n, dtype=torch.bool, device="cuda")
            rest[where] = False
            for a, b, name in zip(got, clean, ("out", "lse", "d_q", "d_k", "d_v")):
                # sums that were done again one by one are rounded elsewhere: by two roundings of the type at most, of the largest terms
                a, b = a[rest].double(), b[rest].double()
                fine = torch.isfinite(b)
                assert torch.equal(torch.isfinite(a), fine) and torch.equal(a[~fine], b[~fine]), name
                assert ((a - b)[fine].abs() <= 4 * U[dtype] * b[fine].abs().max()).all(), name
            if where.start == text:
                assert all((x[text:] == 0).all() for x in (got[0], got[2], got[3], got[4]))


def test_attention_gradients_agree_with_differences():
    g = gen(10)
    n, h, d = 70, 2, 64
    q, k, v = (randn(g, n, h, d, dtype=torch.bfloat16) for _ in range(3))
    d_out = randn(g, n, h, d, dtype=torch.bfloat16)
    lo, hi = spans_for("documents", n, g)
    how = dict(lo=lo, hi=hi, cap=8.0)
    out, lse = cascade_amd.span_attention(q, k, v, **how)
    grads = cascade_amd.span_attention_backward(d_out, q, k, v, out, lse, **how)
    at = torch.arange(n, device="cuda")
    for which, grad in enumerate(grads):
        way = randn(g, n, h, d).double()
        values = []
        for step in (1e-4, -1e-4):
            x = [t.double() for t in (q, k, v)]
            x[which] = x[which] + step * way
            got, _ = reference_attention(*x, lo.long(), hi.long(), d ** -0.5, 8.0, None)
            values.append((got["out"] * d_out.double()).sum().item())
        slope = (values[0] - values[1]) / 2e-4
        # each entry is off by at most about 2^-7 of its size, at random: the sum of n entries by 2^-7 of the norm, four times over
        assert abs((grad.double() * way).sum().item() - slope) <= 4 * 2.0 ** -7 * (grad.double() * way).norm().item()


def test_attention_is_the_same_every_time_and_on_any_stream():
    g = gen(12)
    q, k, v, d_out = (randn(g, 700, 4, 64, dtype=torch.float16) for _ in range(4))
    lo, hi = spans_for("documents", 700, g)

    def once():
        out, lse = cascade_amd.span_attention(q, k, v, lo, hi)
        return (out, lse, *cascade_amd.span_attention_backward(d_out, q, k, v, out, lse, lo, hi))
    first = once()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        second = once()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))


# ---- cross entropy ----


def check_entropy(n, dim, vocab, dtype, ignored=0.1, scale=1.0, layout="dense", seed=0, weights=None):
    g = gen(seed)
    if layout == "odd":
        hidden, weight = (randn(g, r, dim + 5, dtype=dtype)[:, 1:1 + dim] for r in (n, vocab))
    elif layout == "strided":
        hidden, weight = (randn(g, r, dim + 16, dtype=dtype)[:, 8:8 + dim] for r in (n, vocab))
    else:
        hidden, weight = (randn(g, r, dim, dtype=dtype) for r in (n, vocab))
    weight = weight.mul_(2 * dim ** -0.5)
    target = torch.randint(0, vocab, (n,), generator=g, device="cuda", dtype=torch.int32)
    target[torch.rand(n, generator=g, device="cuda") < ignored] = -1
    if n > 3:
        target[1], target[2] = vocab - 1, vocab + 5  # the last word; none
    d_loss = randn(g, n, scale=scale) if weights is None else weights
    loss, lse = cascade_amd.linear_cross_entropy(hidden, weight, target)
    d_hidden, d_weight = cascade_amd.linear_cross_entropy_backward(d_loss, hidden, weight, target, lse)
    h, w = hidden.double(), weight.double()
    logits = h @ w.T
    want_lse = torch.logsumexp(logits, 1)
    there = (target >= 0) & (target < vocab)
    at = target.long().clamp(0, vocab - 1)[:, None]
    size = 1 + (h.abs() @ w.abs().T).max(1).values  # what the sums of a row's logits run over
    within(lse, want_lse, 2e-6 * size, "lse")
    within(loss, torch.where(there, want_lse - logits.gather(1, at)[:, 0], 0.0), 4e-6 * size, "loss")
    p = torch.exp(logits - want_lse[:, None])
    p.scatter_add_(1, at, torch.full_like(p[:, :1], -1.0))
    p *= torch.where(there, d_loss.double(), 0.0)[:, None]
    u = U[dtype]
    off = u * p.abs() + 1e-5 * d_loss.double().abs()[:, None] * (p != 0) * (p.abs() / d_loss.double().abs()[:, None].clamp(min=1e-30))
    floor = 2.0 ** -24 if dtype == torch.float16 else 0.0
    within(d_hidden, p @ w, 1.1 * (off @ w.abs() + u * (p @ w).abs()) + 1e-6 * p.abs().max() * 4 + floor, "d_hidden")
    within(d_weight, p.T @ h, 1.1 * (off.T @ h.abs() + u * (p.T @ h).abs()) + 1e-6 * p.abs().max() * 4 + floor, "d_weight")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,dim,vocab", [(1, 8, 1), (1, 64, 300), (3, 72, 257), (61, 512, 5000), (64, 128, 256), (65, 200, 1025), (257, 320, 3000),
                                         (513, 136, 511), (700, 256, 2049), (1025, 1024, 777)])
def test_cross_entropy_sizes(n, dim, vocab, dtype):
    check_entropy(n, dim, vocab, dtype, seed=n)


@pytest.mark.parametrize("dim", [1, 5, 63, 100])
@pytest.mark.parametrize("layout", ["dense", "odd", "strided"])
def test_cross_entropy_layouts(dim, layout):
    check_entropy(70, dim, 333, torch.bfloat16, layout=layout, seed=dim)


def test_cross_entropy_over_the_corpus_vocabulary():
    check_entropy(600, 256, 50257, torch.bfloat16, seed=3)
    check_entropy(40, 256, 65535, torch.float16, seed=4)


def test_cross_entropy_in_pieces_of_the_vocabulary():
    """More than one piece of the vocabulary, and shares of d_hidden, in both tile widths."""
    check_entropy(6000, 64, 50257, torch.bfloat16, seed=5)


def test_cross_entropy_small_and_uneven_weights():
    w = torch.logspace(-6, 0, 300, device="cuda")
    check_entropy(300, 128, 1000, torch.float16, weights=w, seed=6)
    check_entropy(300, 128, 1000, torch.bfloat16, weights=w, seed=6)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_equal_weights_of_tokens_leave_no_common_error(dtype):
    """A mean's weight of 1 / n is no number of 16 bits; its rounding, the same for every token, would stay in every sum. The 2-norm of the error is held to
    that of two independent roundings, of the result and of the terms: each is u / sqrt(3) of a value at most, and u / 2 on average over a binade."""
    g = gen(14)
    n, dim, vocab = 700, 256, 3000
    hidden, weight = randn(g, n, dim, dtype=dtype), randn(g, vocab, dim, dtype=dtype, scale=2 * dim ** -0.5)
    target = torch.randint(0, vocab, (n,), generator=g, device="cuda", dtype=torch.int32)
    lse = cascade_amd.linear_cross_entropy(hidden, weight, target)[1]
    h, w = hidden.double(), weight.double()
    p = torch.softmax(h @ w.T, 1)
    p[torch.arange(n, device="cuda"), target.long()] -= 1
    for x in (1.00390625 - 2.0 ** -10, 1.001953, 1.2539, 1.9941):  # far from 8-bit and from 11-bit numbers
        d_loss = torch.full((n,), x, device="cuda")
        d_hidden, d_weight = cascade_amd.linear_cross_entropy_backward(d_loss, hidden, weight, target, lse)
        for got, want in ((d_hidden, x * (p @ w)), (d_weight, x * (p.T @ h))):
            assert (got.double() - want).norm() <= math.sqrt(2) * 0.5 * U[dtype] * want.norm()


def test_tokens_without_a_target_may_hold_anything():
    g = gen(7)
    for n in (50, 600):
        hidden, weight = randn(g, n, 64, dtype=torch.bfloat16), randn(g, 500, 64, dtype=torch.bfloat16)
        target = torch.randint(0, 500, (n,), generator=g, device="cuda", dtype=torch.int32)
        target[::3] = -1
        d_loss = torch.ones(n, device="cuda")
        want = cascade_amd.linear_cross_entropy_backward(d_loss, hidden, weight, target, cascade_amd.linear_cross_entropy(hidden, weight, target)[1])
        spoilt, odd = hidden.clone(), d_loss.clone()
        spoilt[::6], spoilt[3::6] = math.nan, math.inf
        odd[::3] = math.nan
        loss, lse = cascade_amd.linear_cross_entropy(spoilt, weight, target)
        assert (loss[::3] == 0).all() and torch.isfinite(loss).all()
        got = cascade_amd.linear_cross_entropy_backward(odd, spoilt, weight, target, lse)
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and (got[0][::3] == 0).all()


def test_cross_entropy_of_no_tokens():
    hidden, weight = torch.empty(0, 33, dtype=torch.bfloat16, device="cuda"), torch.ones(50, 33, dtype=torch.bfloat16, device="cuda")
    none = torch.empty(0, device="cuda")
    loss, lse = cascade_amd.linear_cross_entropy(hidden, weight, none.int())
    assert loss.numel() == lse.numel() == 0
    d_hidden, d_weight = cascade_amd.linear_cross_entropy_backward(none, hidden, weight, none.int(), none)
    assert d_hidden.shape == (0, 33) and (d_weight == 0).all()


def test_cross_entropy_gradients_agree_with_differences():
    g = gen(8)
    hidden, weight = randn(g, 40, 64, dtype=torch.bfloat16), randn(g, 300, 64, dtype=torch.bfloat16, scale=0.2)
    target = torch.randint(0, 300, (40,), generator=g, device="cuda", dtype=torch.int32)
    d_loss = torch.rand(40, generator=g, device="cuda")
    grads = cascade_amd.linear_cross_entropy_backward(d_loss, hidden, weight, target, cascade_amd.linear_cross_entropy(hidden, weight, target)[1])
    for which, grad in enumerate(grads):
        way = randn(g, *grad.shape).double()
        values = []
        for step in (1e-4, -1e-4):
            x = [hidden.double(), weight.double()]
            x[which] = x[which] + step * way
            logits = x[0] @ x[1].T
            loss = torch.logsumexp(logits, 1) - logits.gather(1, target.long()[:, None])[:, 0]
            values.append((loss * d_loss.double()).sum().item())
        slope = (values[0] - values[1]) / 2e-4
        assert abs((grad.double() * way).sum().item() - slope) <= 4 * 2.0 ** -7 * (grad.double() * way).norm().item()


# ---- clipping ----


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes", [[1], [7, 1, 4096], [16384, 16385, 3, 100001], [5] * 130])
@pytest.mark.parametrize("shrink", [True, False])
def test_clip(dtype, sizes, shrink):
    g = gen(len(sizes))
    grads = [randn(g, s, dtype=dtype) for s in sizes]
    norm = math.sqrt(sum(x.double().square().sum().item() for x in grads))
    most = norm / 2 if shrink else 2 * norm
    want = [x.double() * min(1.0, most / norm) for x in grads]
    out = [torch.full_like(x, 7) for x in grads]
    before = [x.clone() for x in grads]
    got = cascade_amd.clip_gradients(grads, most, out=out)
    assert got.shape == () and abs(got.item() - norm) <= 2.0 ** -23 * norm
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    got = cascade_amd.clip_gradients(grads, most)
    u = {torch.float32: 2.0 ** -22, **U}[dtype]
    for a, b, w in zip(grads, out, want):
        assert torch.equal(a, b)
        within(a, w, u * w.abs() + TINY.get(dtype, 0.0), "clipped")
    if not shrink:
        assert all(torch.equal(a, b) for a, b in zip(grads, before))


def test_clip_of_unaligned_mixed_and_empty_tensors():
    g = gen(1)
    base = [randn(g, 5003, dtype=d) for d in (torch.float32, torch.bfloat16, torch.float16)]
    grads = [b[1:] for b in base] + [torch.empty(0, device="cuda"), randn(g, 30, 40)]
    want = [x.double() for x in grads]
    norm = math.sqrt(sum(x.square().sum().item() for x in want))
    got = cascade_amd.clip_gradients(grads, 1.0)
    assert abs(got.item() - norm) <= 2.0 ** -23 * norm
    for a, w in zip(grads, want):
        within(a, w / norm, {torch.float32: 2.0 ** -22, **U}[a.dtype] * (w / norm).abs() + 2.0 ** -24, "clipped")
    assert all(b[0] == x for b, x in zip(base, [b[0].item() for b in base]))


def test_clip_does_not_overflow_and_leaves_what_has_no_norm():
    big = torch.full((1000,), 1e30, device="cuda")
    assert cascade_amd.clip_gradients([big], 1.0).item() == pytest.approx(1e30 * math.sqrt(1000), rel=1e-6)
    assert torch.allclose(big, torch.full_like(big, 1000 ** -0.5), rtol=1e-6)
    for bad in (math.nan, math.inf):
        x = torch.tensor([1.0, bad, 3.0], device="cuda")
        norm = cascade_amd.clip_gradients([x], 1.0).item()
        assert not math.isfinite(norm) and x[0] == 1 and x[2] == 3
    zero = torch.zeros(10, device="cuda")
    assert cascade_amd.clip_gradients([zero], 1.0).item() == 0 and (zero == 0).all()


# ---- graphs ----


def test_calls_recorded_into_a_graph_give_the_same_in_every_replay():
    g = gen(15)
    n, heads, dim, vocab = 1100, 4, 64, 2000
    text = torch.randint(0, vocab, (n,), generator=g, device="cuda").to(torch.int16)
    text[torch.randint(0, n, (9,), generator=g, device="cuda")] = -1
    q, d_out = (randn(g, n, heads, dim, dtype=torch.float16) for _ in range(2))
    k, v = (randn(g, n, 2, dim, dtype=torch.float16) for _ in range(2))
    words, d_loss = randn(g, vocab, heads * dim, dtype=torch.float16, scale=0.1), torch.rand(n, generator=g, device="cuda")

    def step():
        lo, hi, target = cascade_amd.token_spans(text)
        out, lse = cascade_amd.span_attention(q, k, v, lo, hi, cap=20.0)
        grads = cascade_amd.span_attention_backward(d_out, q, k, v, out, lse, lo, hi, cap=20.0)
        hidden = out.view(n, -1)
        loss, sums = cascade_amd.linear_cross_entropy(hidden, words, target)
        grads = [*grads, *cascade_amd.linear_cross_entropy_backward(d_loss, hidden, words, target, sums)]
        norm = cascade_amd.clip_gradients(grads, 0.5)
        return [lo, hi, target, out, lse, loss, sums, norm, *grads]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = step()
    for turn in range(4):
        for x in (q, k, v, d_out):
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        text.copy_(torch.where(text == -1, text, (text + turn) % vocab))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(recorded, want)):
            assert torch.equal(a, b), f"value {i} of replay {turn}"


# ---- refusals ----


def test_refusals():
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        cascade_amd.span_attention(q, q[:, :, :32], q[:, :, :32])
    with pytest.raises(ValueError):
        cascade_amd.span_attention(q[:, :1], q, q)  # fewer heads than keys have
    with pytest.raises(ValueError):
        cascade_amd.span_attention(q, q, q, scale=-1.0)
    with pytest.raises(ValueError):
        cascade_amd.span_attention(q, q, q, cap=-1.0)
    with pytest.raises(ValueError):
        cascade_amd.span_attention(q, q, q, lo=torch.zeros(4, device="cuda"))
    with pytest.raises(ValueError):
        cascade_amd.span_attention(q.cpu(), q.cpu(), q.cpu())
    with pytest.raises(TypeError):
        cascade_amd.span_attention(q.float(), q.float(), q.float())
    for dim in (4, 65, 136):
        x = torch.zeros(4, 2, dim, dtype=torch.bfloat16, device="cuda")
        with pytest.raises(ValueError):
            cascade_amd.span_attention(x, x, x)
    w = torch.zeros(10, 64, dtype=torch.bfloat16, device="cuda")
    t = torch.zeros(4, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        cascade_amd.linear_cross_entropy(w[:4, :32], w, t)
    with pytest.raises(ValueError):
        cascade_amd.linear_cross_entropy(w[:4], w, t.long())
    with pytest.raises(TypeError):
        cascade_amd.linear_cross_entropy(w[:4].float(), w.float(), t)
    with pytest.raises(ValueError):
        cascade_amd.clip_gradients([w], -1.0)
    with pytest.raises(ValueError):
        cascade_amd.clip_gradients([w.t()], 1.0)
    with pytest.raises(TypeError):
        cascade_amd.clip_gradients([w.double()], 1.0)
    with pytest.raises(ValueError):
        cascade_amd.token_spans(torch.zeros(4, device="cuda"))


def test_slopes_that_want_a_gradient_are_refused():
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    slopes = torch.ones(2, device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="slopes"):
        cascade_amd.attend(q, q, q, slopes=slopes)
    assert cascade_amd.attend(q, q, q, slopes=slopes.detach()).shape == q.shape


def test_the_library_refuses_what_the_kernels_cannot_read():
    import ctypes as C
    native = lm.native
    lib = native.load()
    x = torch.zeros(64, 2, 64, dtype=torch.bfloat16, device="cuda")
    lse = torch.zeros(2, 64, device="cuda")
    work = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    heads = native.CsaLmHeads(x.data_ptr(), 128, 64)

    def call(**change):
        a = dict(type=0, q_heads=2, kv_heads=2, head_dim=64, tokens=64, d_lo=None, d_hi=None, d_slope=None, scale=1.0, cap=0.0, q=heads, k=heads, v=heads)
        a.update(change)
        return lib.csa_lm_attention_forward_dev(C.byref(native.CsaLmAttention(**a)), heads, lse.data_ptr(), work.data_ptr(), work.numel(), None)
    odd = native.CsaLmHeads(x.data_ptr() + 2, 128, 64)
    for change in (dict(type=2), dict(q_heads=3), dict(kv_heads=0), dict(head_dim=60), dict(head_dim=136), dict(scale=0.0), dict(scale=math.nan), dict(cap=-1.0),
                   dict(q=odd), dict(k=native.CsaLmHeads(None, 128, 64)), dict(v=native.CsaLmHeads(x.data_ptr(), 100, 64)),
                   dict(v=native.CsaLmHeads(x.data_ptr(), 56, 64))):
        with pytest.raises(CascadeError):
            native.check(call(**change))
    assert call(tokens=(1 << 30) + 1) == -2
    a = native.CsaLmAttention(0, 2, 2, 64, 64, None, None, None, 1.0, 0.0, heads, heads, heads)
    need = lib.csa_lm_attention_workspace(64, 2, 2, 64, native.CSA_LM_BACKWARD)
    assert lib.csa_lm_attention_backward_dev(C.byref(a), heads, lse.data_ptr(), heads, heads, heads, heads, work.data_ptr(), need - 1, None) == -1
    assert b"workspace" in lib.csa_lm_last_error()
