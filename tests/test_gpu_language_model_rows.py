"""Embeddings and norms of residual streams against plain implementations in 64 bits, written from the formulas.

Bounds are derived, element by element. u is half a unit of the type's last place, and E that of 32 bits, in which everything is computed: a result is
off by u of itself, by E of it for every operation that makes it, and by E times the sum of its absolute terms for every addition that a term goes through."""
import math

import pytest

torch = pytest.importorskip("torch")

import cascade_amd  # noqa: E402
from test_gpu_language_model import gen, randn, within  # noqa: E402

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: E}  # of what is rounded to the type
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -24, torch.float32: 0.0}  # half precision's smallest step
TYPES = [torch.bfloat16, torch.float16, torch.float32]


# ---- embeddings ----


def words_of(tokens, rows):
    w = tokens.long()
    if tokens.element_size() == 2:
        w = w & 0xFFFF
    return torch.where((w >= 0) & (w < rows), w, -1)


def sums_of_words(word, x, rows):
    """The sum of the rows of x of every word, in 64 bits: what a running sum over the places in the order of their words gains over a word's places."""
    word, order = torch.sort(word)
    words, counts = torch.unique_consecutive(word, return_counts=True)
    upto = x[order].double().cumsum(0)[counts.cumsum(0) - 1]
    sums = torch.zeros(rows, x.shape[1], dtype=torch.float64, device="cuda")
    if words.numel():
        sums[words] = upto.diff(dim=0, prepend=torch.zeros_like(upto[:1]))
    return sums


def check_embed(tokens, rows, dim, dtype, scale=1.0, layout="dense", seed=0):
    g = gen(seed)
    n = tokens.numel()
    if layout == "odd":  # rows that begin anywhere
        weight, d_out = (randn(g, r, dim + 5, dtype=dtype)[:, 3:3 + dim] for r in (rows, n))
    else:
        weight, d_out = randn(g, rows, dim, dtype=dtype), randn(g, n, dim, dtype=dtype)
    word = words_of(tokens, rows)
    there = word >= 0
    u, tiny = U[dtype], TINY[dtype]
    out = cascade_amd.embed_tokens(tokens, weight, scale)
    want = torch.where(there[:, None], weight[word.clamp(min=0)].double() * scale, 0.0)
    within(out, want, (u + E) * want.abs() + tiny, "out")
    got = cascade_amd.embed_tokens_backward(d_out, tokens, rows, scale)
    want, size = (sums_of_words(word[there], x[there], rows) * scale for x in (d_out, d_out.abs()))
    count = torch.bincount(word[there], minlength=rows)[:, None]
    # a sum over a run of at most 64 entries, joined over at most 1 + count / 8 runs by additions one after the other in the worst case
    within(got, want, (u + E) * want.abs() + E * (count.clamp(max=64) + count / 8 + 1) * size.abs() + 1e-12 * n * abs(scale) + tiny, "d_weight")
    assert (got[count[:, 0] == 0] == 0).all()
    assert torch.equal(got, cascade_amd.embed_tokens_backward(d_out, tokens, rows, scale))
    return out, got


def text(n, rows, spread, g, bits=32):
    if spread == "zipf":
        t = torch.exp(torch.rand(n, generator=g, device="cuda") * math.log(rows + 1)).long() - 1
    elif spread == "one":
        t = torch.full((n,), rows // 2, device="cuda")
    else:
        t = torch.randint(0, rows, (n,), generator=g, device="cuda")
    t = t.clamp(0, rows - 1)
    if bits == 16:
        t = torch.where(torch.rand(n, generator=g, device="cuda") < 0.05, 0xFFFF, t & 0xFFFF)
        return torch.where(t >= 1 << 15, t - (1 << 16), t).to(torch.int16)
    return torch.where(torch.rand(n, generator=g, device="cuda") < 0.05, torch.randint(-5, 2, (n,), generator=g, device="cuda") * rows - 1, t).to(torch.int32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 63, 64, 65, 127, 1023, 1025, 4097])
@pytest.mark.parametrize("spread", ["zipf", "even", "one"])
def test_embed_lengths(n, spread, dtype):
    check_embed(text(n, 300, spread, gen(n)), 300, 72, dtype, scale=8.5, seed=n)


@pytest.mark.parametrize("dim", [8, 9, 15, 16, 17, 63, 65, 100, 127, 256, 333, 511, 513, 1030, 4099])
@pytest.mark.parametrize("layout", ["dense", "odd"])
def test_embed_row_lengths(dim, layout):
    for dtype in TYPES:
        check_embed(text(150, 40, "zipf", gen(dim)), 40, dim, dtype, layout=layout, seed=dim)


@pytest.mark.parametrize("rows", [1, 2, 3, 255, 256, 511, 512, 513, 1 << 15, 50257, 65535, 65536, 200001])
@pytest.mark.parametrize("bits", [16, 32])
def test_embed_vocabularies(rows, bits):
    check_embed(text(700, rows, "zipf", gen(rows), bits), rows, 16, torch.bfloat16, scale=-3.0, seed=rows)


@pytest.mark.parametrize("n", [8192, 8193, 20011, 70001, 262144 + 5])  # from where on places are sorted by digits
@pytest.mark.parametrize("rows,bits", [(1, 16), (300, 16), (511, 32), (512, 32), (50257, 16), (65535, 16), (65536, 32), (300007, 32)])
def test_embed_of_long_texts(n, rows, bits):
    for spread in ("zipf", "even", "one"):
        check_embed(text(n, rows, spread, gen(n), bits), rows, 24, torch.float16 if bits == 16 else torch.float32, seed=n)


@pytest.mark.parametrize("n", [100, 5000, 8192, 8193, 70001, 262144 + 5])
@pytest.mark.parametrize("dim", [24, 56, 120, 250, 600])  # teams of 8, 16, 32 and 64 lanes, one slice of a row and several
@pytest.mark.parametrize("spread", ["zipf", "even", "one"])
def test_embed_gradients_of_whole_numbers_are_exact(spread, dim, n):
    """Small whole numbers add up without rounding in 32 bits, whatever the order: every sum has to be that of 64-bit integers. A lost, doubled or swapped row changes it."""
    g = gen(n + dim)
    rows = 3000
    tokens = text(n, rows, spread, g)
    d_out = torch.randint(-8, 9, (n, dim), generator=g, device="cuda")  # 8 n < 2^24
    word = words_of(tokens, rows)
    want = torch.zeros(rows, dim, dtype=torch.int64, device="cuda").index_add_(0, word[word >= 0], d_out[word >= 0])
    for dtype in TYPES:
        got = cascade_amd.embed_tokens_backward(d_out.to(dtype), tokens, rows)
        assert torch.equal(got, want.float().to(dtype))  # rounded to the type once


def test_embed_of_a_very_long_text():
    """More tokens than there are segments of the smallest size, and offsets past 2^32 bytes in d_out."""
    n, rows = 4300000, 70001
    check_embed(text(n, rows, "zipf", gen(1)), rows, 8, torch.bfloat16, seed=1)
    n = 1100000
    tokens = text(n, 50, "even", gen(2))
    d_out = torch.ones(n, 2048, dtype=torch.bfloat16, device="cuda")  # 4.5 GB
    got = cascade_amd.embed_tokens_backward(d_out, tokens, 50)
    counts = torch.bincount(words_of(tokens, 50) + 1, minlength=51)[1:].double()[:, None]
    within(got, counts.expand(50, 2048), 2.0 ** -8 * counts.expand(50, 2048), "counts")
    del d_out
    weight = randn(gen(3), 50, 2048, dtype=torch.bfloat16)
    out, word = cascade_amd.embed_tokens(tokens, weight), words_of(tokens, 50)
    for part in (slice(0, 5000), slice(n - 5000, n)):
        assert torch.equal(out[part], torch.where(word[part, None] >= 0, weight[word[part].clamp(min=0)], 0.0))


def test_norm_of_a_very_long_text():
    """Offsets past 2^32 bytes, and results that go past the caches."""
    n, dim = 300000, 4096
    g = gen(4)
    few = randn(g, 1000, dim, dtype=torch.bfloat16)
    x = few.repeat(n // 1000, 1)  # 2.5 GB
    out, total, rstd = cascade_amd.residual_norm(x, x)
    want = cascade_amd.residual_norm(few, few)
    for a, b in zip((out, total, rstd), want):
        assert torch.equal(a.view(n // 1000, *b.shape), b.expand(n // 1000, *b.shape))
    gain = torch.ones(dim, dtype=torch.bfloat16, device="cuda")
    d_x, _, d_gain = cascade_amd.residual_norm_backward(x, total, rstd, gain, total)
    d_few, _, d_few_gain = cascade_amd.residual_norm_backward(few, want[1], want[2], gain, want[1])
    assert torch.equal(d_x.view(n // 1000, 1000, dim), d_few.expand(n // 1000, 1000, dim))
    # sums of the same 1000 rows, 300 times: off by the rounding of both results, and by 32-bit sums of 300000 terms over 512 workgroups, joined by 16 runs
    terms = (few.double() * want[1].double() * want[2].double()[:, None]).abs().sum(0)
    assert ((d_gain.double() - 300 * d_few_gain.double()).abs() <= 300 * (2.1 * 2.0 ** -8 * d_few_gain.double().abs() + E * (300000 / 512 + 60) * terms)).all()


def test_tokens_of_any_16_bit_type_and_place():
    g = gen(5)
    tokens = torch.randint(0, 60000, (901,), generator=g, device="cuda")
    weight = randn(g, 60000, 24, dtype=torch.float16)
    want = cascade_amd.embed_tokens(tokens[1:].int(), weight)
    short = torch.where(tokens >= 1 << 15, tokens - (1 << 16), tokens).to(torch.int16)
    assert torch.equal(cascade_amd.embed_tokens(short[1:], weight), want) and torch.equal(cascade_amd.embed_tokens(short.view(torch.uint16)[1:], weight), want)
    d_out = randn(g, 900, 24, dtype=torch.float16)
    grads = [cascade_amd.embed_tokens_backward(d_out, t, 60000) for t in (tokens[1:].int(), short[1:], short.view(torch.uint16)[1:])]
    assert torch.equal(grads[0], grads[1]) and torch.equal(grads[0], grads[2])


def test_two_calls_at_once_share_nothing():
    g = gen(6)
    streams = [torch.cuda.Stream() for _ in range(2)]
    inputs = [(text(20000, 3000, "zipf", g), randn(g, 20000, 64, dtype=torch.bfloat16)) for _ in range(2)]
    want = [cascade_amd.embed_tokens_backward(d, t, 3000) for t, d in inputs]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s, (t, d) in zip(streams, inputs):
            with torch.cuda.stream(s):
                got.append(cascade_amd.embed_tokens_backward(d, t, 3000))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want[i % 2]) for i, a in enumerate(got))


def test_embed_of_nothing():
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    weight = torch.ones(30, 40, device="cuda")
    assert cascade_amd.embed_tokens(none, weight).shape == (0, 40)
    got = cascade_amd.embed_tokens_backward(weight[:0], none, 30)
    assert got.shape == (30, 40) and (got == 0).all()


@pytest.mark.parametrize("n", [100, 30000])
def test_gradients_of_tokens_that_are_no_row_may_hold_anything(n):
    g = gen(4)
    tokens = text(n, 500, "zipf", g)
    d_out = randn(g, n, 64, dtype=torch.bfloat16)
    want = cascade_amd.embed_tokens_backward(d_out, tokens, 500)
    bad = words_of(tokens, 500) < 0
    d_out[bad] = math.nan
    assert bad.any() and torch.equal(cascade_amd.embed_tokens_backward(d_out, tokens, 500), want)
    # and one bad row reaches its own word only
    at = int((~bad).nonzero()[3])
    d_out[at, 7] = math.inf
    got = cascade_amd.embed_tokens_backward(d_out, tokens, 500)
    word = int(tokens[at])
    assert got[word, 7] == math.inf
    got[word, 7] = want[word, 7]
    assert torch.equal(got, want)


def test_large_gradients_of_half_precision_are_summed_in_32_bits():
    tokens = torch.zeros(64, dtype=torch.int32, device="cuda")
    d_out = torch.full((64, 8), 6e4, dtype=torch.float16, device="cuda")
    d_out[::2] *= -1
    d_out[0] = -5.9e4
    got = cascade_amd.embed_tokens_backward(d_out, tokens, 1)
    want = d_out.double().sum(0)
    within(got[0], want, 2.0 ** -11 * want.abs(), "sum")


# ---- norms ----


EPS = 1e-6


def check_norm(n, dim, dtype, stream=None, residual=True, gain=True, flow=True, layout="dense", size=1.0, eps=EPS, seed=0):
    g = gen(seed)
    stream = dtype if stream is None else stream

    def make(rows, dtype, scale=1.0):
        if layout == "odd":
            return randn(g, rows, dim + 3, dtype=dtype, scale=scale)[:, 1:1 + dim]
        if layout == "turned":  # values of a row far apart: copied first
            return randn(g, dim, rows, dtype=dtype, scale=scale).t()
        return randn(g, rows, dim, dtype=dtype, scale=scale)
    x = make(n, dtype, size)
    r = make(n, stream, 2 * size) if residual else None
    a = (1 + randn(g, dim, scale=0.5)).to(dtype) if gain else None
    out, total, rstd = cascade_amd.residual_norm(x, r, a, eps)
    u, us, tiny = U[dtype], U[stream], TINY[dtype]
    if residual:
        want = x.double() + r.double()
        within(total, want, (us + E) * want.abs() + TINY[stream], "total")
    else:
        assert total is x
    t = total.double()
    root = (t.square().mean(1) + eps).rsqrt()
    within(rstd, root, 2 * E * root + 2.0 ** -149, "rstd")
    v = t * root[:, None]
    b = torch.ones(dim, dtype=torch.float64, device="cuda") if a is None else a.double()
    within(out, v * b, (u + 4 * E) * (v * b).abs() + tiny, "out")
    d_out = make(n, dtype)
    d_total = make(n, stream) if flow else None
    d_x, d_residual, d_gain = cascade_amd.residual_norm_backward(d_out, total, rstd, a, d_total)
    h = d_out.double() * b
    c = (h * v).mean(1, keepdim=True)
    more = d_total.double() if flow else torch.zeros_like(h)
    want = root[:, None] * (h - v * c) + more
    # of the mean, a term goes through at most 64 additions of a lane, 6 of a wave and 2 of a workgroup
    off = E * (8 * (root[:, None] * (h.abs() + (v * c).abs()) + more.abs()) + 74 * root[:, None] * v.abs() * (h * v).abs().mean(1, keepdim=True))
    within(d_x, want, u * want.abs() + off + tiny, "d_x")
    within(d_residual, want, us * want.abs() + off + TINY[stream], "d_residual")
    assert (d_x is d_residual) == (dtype == stream)
    if gain:
        want, terms = (d_out.double() * v).sum(0), (d_out.double() * v).abs().sum(0)
        # a term goes through at most as many additions as a workgroup has rows, four waves, and the workgroups' sums by 16 runs
        within(d_gain, want, u * want.abs() + E * (4 + n / 512 + 4 + 512 / 16 + 16) * terms + tiny, "d_gain")
    else:
        assert d_gain is None
    again = cascade_amd.residual_norm_backward(d_out, total, rstd, a, d_total)
    assert all(p is q is None or torch.equal(p, q) for p, q in zip((d_x, d_residual, d_gain), again))


KINDS = [(torch.bfloat16, None), (torch.float16, None), (torch.float32, None), (torch.bfloat16, torch.float32), (torch.float16, torch.float32)]


@pytest.mark.parametrize("dtype,stream", KINDS)
@pytest.mark.parametrize("dim", [8, 9, 12, 15, 16, 64, 100, 505, 511, 512, 513, 520, 765, 768, 769, 1023, 1024, 1025, 1536, 1537, 2047, 2048, 2049, 2880, 4095, 4096, 4097, 5120, 6144, 6145, 8191, 8192,
                                 8193, 12000, 12288, 12289, 16383, 16384])
def test_norm_row_lengths(dim, dtype, stream):
    check_norm(5, dim, dtype, stream, seed=dim)


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 511, 512, 513, 2047, 2049, 5000])
@pytest.mark.parametrize("dim", [40, 1000, 1100])
def test_norm_tokens(n, dim):
    check_norm(n, dim, torch.bfloat16, seed=n)
    check_norm(n, dim, torch.float16, torch.float32, seed=n)


@pytest.mark.parametrize("residual,gain,flow", [(True, True, False), (True, False, True), (False, True, False), (False, False, False), (False, True, True)])
@pytest.mark.parametrize("dim", [72, 1000, 3000])
def test_norm_without_what_may_be_left_out(residual, gain, flow, dim):
    for dtype in TYPES:
        check_norm(33, dim, dtype, residual=residual, gain=gain, flow=flow, seed=3)


@pytest.mark.parametrize("layout", ["odd", "turned"])
@pytest.mark.parametrize("dim", [8, 63, 515, 1025, 2052])
def test_norm_layouts(layout, dim):
    for dtype, stream in KINDS:
        check_norm(9, dim, dtype, stream, layout=layout, seed=dim)


@pytest.mark.parametrize("dtype,size", [(torch.bfloat16, 1e30), (torch.bfloat16, 1e-30), (torch.float32, 1e25), (torch.float32, 1e-25), (torch.float16, 5e3)])
def test_norm_of_values_whose_squares_leave_32_bits(dtype, size):
    check_norm(7, 300, dtype, flow=False, size=size, eps=1e-38 if size < 1 else EPS, seed=5)
    check_norm(7, 2100, dtype, gain=False, flow=False, size=size, eps=1e-38 if size < 1 else EPS, seed=6)


def test_norm_of_zeros_and_of_no_tokens():
    zero = torch.zeros(3, 50, dtype=torch.bfloat16, device="cuda")
    out, total, rstd = cascade_amd.residual_norm(zero, zero)
    assert (out == 0).all() and (total == 0).all() and torch.allclose(rstd, torch.full_like(rstd, 1e3))
    gain = torch.ones(50, dtype=torch.bfloat16, device="cuda")
    out, total, rstd = cascade_amd.residual_norm(zero[:0], zero[:0], gain)
    assert out.shape == total.shape == (0, 50) and rstd.shape == (0,)
    d_x, d_residual, d_gain = cascade_amd.residual_norm_backward(out, total, rstd, gain, total)
    assert d_x.shape == (0, 50) and (d_gain == 0).all()


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("dim", [70, 1030])
def test_a_bad_token_stays_in_its_row(value, dim):
    g = gen(8)
    x, r, d_out = (randn(g, 9, dim, dtype=torch.bfloat16) for _ in range(3))
    clean = cascade_amd.residual_norm(x, r)
    grads = cascade_amd.residual_norm_backward(d_out, clean[1], clean[2])
    x[4, 3] = value
    got = cascade_amd.residual_norm(x, r)
    rest = torch.arange(9, device="cuda") != 4
    for a, b in zip((*got, *cascade_amd.residual_norm_backward(d_out, got[1], got[2])[:2]), (*clean, *grads[:2])):
        assert torch.equal(a[rest], b[rest])
    assert got[0][4].isnan().any()


@pytest.mark.parametrize("dim", [70, 700, 1030, 9000])
def test_padding_without_gradient_takes_nothing_from_the_gain(dim):
    g = gen(18)
    x, r, d_out = (randn(g, 30, dim, dtype=torch.bfloat16) for _ in range(3))
    gain = (1 + randn(g, dim, scale=0.2)).bfloat16()
    d_out[20:] = 0
    _, total, rstd = cascade_amd.residual_norm(x, r, gain)
    want = cascade_amd.residual_norm_backward(d_out, total, rstd, gain)
    x[20:25], r[25:] = math.nan, math.inf
    _, total, rstd = cascade_amd.residual_norm(x, r, gain)
    got = cascade_amd.residual_norm_backward(d_out, total, rstd, gain)
    assert torch.equal(got[2], want[2]) and torch.equal(got[0][:20], want[0][:20])


# ---- gradients by torch.autograd, and against differences ----


def test_norm_gradients_agree_with_differences():
    g = gen(9)
    n, dim = 6, 40
    x, r, d_out, d_total = (randn(g, n, dim) for _ in range(4))
    gain = 1 + randn(g, dim, scale=0.3)
    out, total, rstd = cascade_amd.residual_norm(x, r, gain)
    d_x, d_residual, d_gain = cascade_amd.residual_norm_backward(d_out, total, rstd, gain, d_total)

    def value(x, r, gain):
        t = x + r
        return (t * (t.square().mean(1, keepdim=True) + EPS).rsqrt() * gain * d_out.double() + t * d_total.double()).sum().item()
    for which, grad in enumerate((d_x, d_residual, d_gain)):
        way = randn(g, *grad.shape).double()
        values = []
        for step in (1e-5, -1e-5):
            at = [t.double() for t in (x, r, gain)]
            at[which] = at[which] + step * way
            values.append(value(*at))
        # differences of 64 bits are off by the square of the step, gradients by some E of their terms
        assert abs((grad.double() * way).sum().item() - (values[0] - values[1]) / 2e-5) <= 1e-5 * (grad.double() * way).abs().sum().item()


def test_autograd_of_embed_and_add_norm():
    g = gen(10)
    n, rows, dim = 50, 30, 48
    tokens = text(n, rows, "zipf", g)
    weight = randn(g, rows, dim, dtype=torch.bfloat16).requires_grad_()
    gain = (1 + randn(g, dim, scale=0.2)).bfloat16().requires_grad_()
    other = randn(g, n, dim, dtype=torch.bfloat16).requires_grad_()
    go, gt = randn(g, n, dim, dtype=torch.bfloat16), randn(g, n, dim, dtype=torch.bfloat16)
    x = cascade_amd.embed(tokens, weight, 2.0)
    out, total = cascade_amd.add_norm(other, x, gain)
    grads = torch.autograd.grad((out, total), (weight, other, gain), (go, gt))
    _, t, rstd = cascade_amd.residual_norm(other.detach(), x.detach(), gain.detach())
    d_x, _, d_gain = cascade_amd.residual_norm_backward(go, t, rstd, gain.detach(), gt)
    for a, b in zip(grads, (cascade_amd.embed_tokens_backward(d_x, tokens, rows, 2.0), d_x, d_gain)):
        assert torch.equal(a, b)
    # out alone, total alone, no gain, no residual
    out, total = cascade_amd.add_norm(other, x.detach(), gain)
    assert torch.equal(torch.autograd.grad(out, other, go)[0], cascade_amd.residual_norm_backward(go, t, rstd, gain.detach())[0])
    out, total = cascade_amd.add_norm(other, x.detach(), gain)
    d_other, d_gain = torch.autograd.grad(total, (other, gain), gt, allow_unused=True)
    assert torch.equal(d_other, gt) and d_gain is None
    out, total = cascade_amd.add_norm(other)
    assert total is other
    _, t, rstd = cascade_amd.residual_norm(other.detach())
    assert torch.equal(torch.autograd.grad(out, other, go)[0], cascade_amd.residual_norm_backward(go, t, rstd)[0])
    # an expanded gradient
    out, total = cascade_amd.add_norm(other)
    d_other = torch.autograd.grad(out.sum(), other)[0]
    assert torch.equal(d_other, cascade_amd.residual_norm_backward(torch.ones_like(go), t, rstd)[0])


def test_autograd_of_a_stream_of_32_bits():
    g = gen(11)
    x = randn(g, 20, 64, dtype=torch.bfloat16).requires_grad_()
    stream = randn(g, 20, 64).requires_grad_()
    out, total = cascade_amd.add_norm(x, stream)
    assert out.dtype == torch.bfloat16 and total.dtype == torch.float32
    d_x, d_stream = torch.autograd.grad((out.float() * 3 + total).sum(), (x, stream))
    _, t, rstd = cascade_amd.residual_norm(x.detach(), stream.detach())
    want = cascade_amd.residual_norm_backward(torch.full_like(x, 3).detach(), t, rstd, None, torch.ones_like(t))
    assert torch.equal(d_x, want[0]) and torch.equal(d_stream, want[1])
    out, total = cascade_amd.add_norm(x, stream)
    d_x, d_stream = torch.autograd.grad(total.sum(), (x, stream))
    assert d_x.dtype == torch.bfloat16 and (d_x == 1).all() and (d_stream == 1).all()


# ---- streams and graphs ----


@pytest.mark.parametrize("n", [500, 17000])
def test_calls_on_another_stream_and_in_a_graph_give_the_same(n):
    g = gen(12)
    rows, dim = 700, 96
    tokens = text(n, rows, "zipf", g)
    weight, d_out, other = randn(g, rows, dim, dtype=torch.bfloat16), randn(g, n, dim, dtype=torch.bfloat16), randn(g, n, dim)
    gain = randn(g, dim, dtype=torch.bfloat16)

    def step():
        x = cascade_amd.embed_tokens(tokens, weight, 1.5)
        out, total, rstd = cascade_amd.residual_norm(x, other, gain)
        grads = cascade_amd.residual_norm_backward(d_out, total, rstd, gain, other)
        return [x, out, total, rstd, *grads, cascade_amd.embed_tokens_backward(grads[0], tokens, rows, 1.5)]
    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = step()
    for turn in range(4):
        tokens.copy_((tokens + turn) % rows)
        for x in (weight, d_out, other):
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(recorded, want)):
            assert torch.equal(a, b), f"value {i} of replay {turn}"


# ---- refusals ----


def test_refusals():
    w = torch.zeros(10, 64, dtype=torch.bfloat16, device="cuda")
    t = torch.zeros(4, dtype=torch.int32, device="cuda")
    for bad in (t.float(), t.long(), t.view(2, 2), t[::2], t.cpu()):
        with pytest.raises(ValueError):
            cascade_amd.embed_tokens(bad, w)
        with pytest.raises(ValueError):
            cascade_amd.embed_tokens_backward(w[:bad.numel()], bad, 10)
    with pytest.raises(TypeError):
        cascade_amd.embed_tokens(t, w.double())
    with pytest.raises(ValueError):
        cascade_amd.embed_tokens(t, w[0])
    for bad in (math.nan, math.inf):
        with pytest.raises(cascade_amd._native.CascadeError):
            cascade_amd.embed_tokens(t, w, bad)
    with pytest.raises(cascade_amd._native.CascadeError):
        cascade_amd.embed_tokens(t, w[:, :7])
    with pytest.raises(ValueError):
        cascade_amd.embed_tokens_backward(w, t, 10)  # a row for each token
    with pytest.raises(ValueError):
        cascade_amd.residual_norm(w[0])
    with pytest.raises(ValueError):
        cascade_amd.residual_norm(w, w[:5])
    with pytest.raises(ValueError):
        cascade_amd.residual_norm(w, w.half())
    with pytest.raises(ValueError):
        cascade_amd.residual_norm(w.float(), w)  # no stream of fewer bits
    with pytest.raises(ValueError):
        cascade_amd.residual_norm(w, gain=torch.ones(64, device="cuda"))
    with pytest.raises(ValueError):
        cascade_amd.residual_norm(w, w.cpu())
    with pytest.raises(TypeError):
        cascade_amd.residual_norm(w.double())
    for eps in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(cascade_amd._native.CascadeError):
            cascade_amd.residual_norm(w, eps=eps)
    for dim in (7, 16385):
        with pytest.raises(cascade_amd._native.CascadeError):
            cascade_amd.residual_norm(torch.zeros(2, dim, device="cuda"))
    out, total, rstd = cascade_amd.residual_norm(w, w)
    for bad in (rstd.double(), rstd[:3], rstd.view(2, 5), rstd.cpu()):
        with pytest.raises(ValueError):
            cascade_amd.residual_norm_backward(out, total, bad)
    with pytest.raises(ValueError):
        cascade_amd.residual_norm_backward(out, total, rstd, d_total=total.float())
    with pytest.raises(ValueError):
        cascade_amd.residual_norm_backward(out, total[:, :32], rstd)
