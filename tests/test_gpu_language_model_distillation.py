"""Distillation from a teacher's top logits against a plain implementation in 64 bits, written from the formulas.

Bounds are derived, element by element. u is half a unit of the type's last place: a result rounded once is off by u |x|, and the gradients of the logits, rounded to 16
bits before the products, bring u times the sum of the absolute terms. Sums and exponentials of 32 bits are far below u in the gradients; in losses they are all there is: E, half a unit of
32 bits' last place, for every term of a logit's sum and of the others."""
import math

import pytest

torch = pytest.importorskip("torch")

import cascade_amd  # noqa: E402
from test_gpu_language_model import U, gen, randn, within  # noqa: E402

pytestmark = pytest.mark.gpu


def reference(hidden, weight, ids, logits, temperature):
    """(loss, lse, p, q): of every token, p and q over the whole vocabulary, in 64 bits."""
    z = hidden.double() @ weight.double().T / temperature
    n, vocab = z.shape
    lse = torch.logsumexp(z, 1)
    there = (ids >= 0) & (ids < vocab) & (logits != -math.inf)
    told = (logits.double() / temperature).masked_fill(~there, -math.inf)
    counts = there.any(1)
    log_q = told - torch.where(counts, torch.logsumexp(told, 1), 0.0)[:, None]
    q = torch.where(there, log_q.exp(), 0.0)
    at = torch.where(there, ids, 0).long()
    log_p = torch.where(there, z.gather(1, at) - lse[:, None], 0.0)
    loss = torch.where(there, q * (torch.where(there, log_q, 0.0) - log_p), 0.0).sum(1)
    return loss, lse, torch.exp(z - lse[:, None]), torch.zeros_like(z).scatter_add_(1, at, q), counts


def teacher(g, n, kept, vocab, spread="zipf", ignored=0.1):
    """Entries with some missing, some told nothing about, some listed twice; tokens without any."""
    if spread == "zipf":
        ids = (torch.exp(torch.rand(n, kept, generator=g, device="cuda") * math.log(vocab + 1.0)) - 1).long().clamp(max=vocab - 1)
    elif spread == "last":  # the end of the vocabulary
        ids = vocab - 1 - torch.randint(0, min(vocab, kept + 3), (n, kept), generator=g, device="cuda")
    else:
        ids = torch.randint(0, vocab, (n, kept), generator=g, device="cuda")
    ids = torch.where(torch.rand(n, kept, generator=g, device="cuda") < 0.1, torch.randint(0, 2, (n, kept), generator=g, device="cuda") * (vocab + 3) - 2, ids)
    ids[torch.rand(n, generator=g, device="cuda") < ignored] = -1
    logits = randn(g, n, kept, scale=3.0) + 5
    logits[torch.rand(n, kept, generator=g, device="cuda") < 0.05] = -math.inf
    logits[(ids < 0) | (ids >= vocab)] = math.nan
    return ids.int().contiguous(), logits


def check_distillation(n, dim, vocab, kept, dtype, temperature=1.0, layout="dense", spread="zipf", weights=None, seed=0, told=None, ignored=0.1):
    g = gen(seed)
    if layout == "odd":
        hidden, weight = (randn(g, r, dim + 5, dtype=dtype)[:, 1:1 + dim] for r in (n, vocab))
    elif layout == "strided":
        hidden, weight = (randn(g, r, dim + 16, dtype=dtype)[:, 8:8 + dim] for r in (n, vocab))
    else:
        hidden, weight = (randn(g, r, dim, dtype=dtype) for r in (n, vocab))
    weight = weight.mul_(2 * dim ** -0.5)
    ids, logits = teacher(g, n, kept, vocab, spread, ignored) if told is None else told
    d_loss = randn(g, n) if weights is None else weights
    loss, lse = cascade_amd.linear_distillation(hidden, weight, ids, logits, temperature)
    want_loss, want_lse, p, q, counts = reference(hidden, weight, ids, logits, temperature)
    # a logit's sum runs over terms of this size; the teacher's logits are divided and exponentiated with the error of their own size
    size = 1 + (hidden.double().abs() @ weight.double().abs().T).max(1).values / temperature
    told_size = torch.where(torch.isfinite(logits), logits.abs(), 0.0).amax(1).double() / temperature
    within(lse, want_lse, 2e-6 * size, "lse")
    within(loss, want_loss, 4e-6 * (size + told_size), "loss")
    assert (loss[~counts] == 0).all()
    got = cascade_amd.linear_distillation_backward(d_loss, hidden, weight, ids, logits, lse, temperature)
    w = torch.where(counts, d_loss.double() / temperature, 0.0)[:, None]
    p, q = torch.where(counts[:, None], p, 0.0), torch.where(counts[:, None], q, 0.0)
    d_z = w * (p - q)
    u = U[dtype]
    # rounded once, relative to itself; p and q come with 32-bit errors of the size of their exponents
    off = u * d_z.abs() + w.abs() * (p + q) * (2e-6 * (size + told_size))[:, None]
    floor = 2.0 ** -24 if dtype == torch.float16 else 0.0
    # half precision holds P in steps of 2^-24 of 2^14 for the largest weight
    step = w.abs().max() * 2.0 ** -38 if dtype == torch.float16 else 0.0
    off = off + step * (w != 0)
    small = 1e-6 * d_z.abs().max() * 4  # sums of 32 bits
    h, wt = hidden.double(), weight.double()
    within(got[0], d_z @ wt, 1.1 * (off @ wt.abs() + u * (d_z @ wt).abs()) + small + floor, "d_hidden")
    within(got[1], d_z.T @ h, 1.1 * (off.T @ h.abs() + u * (d_z.T @ h).abs()) + small + floor, "d_weight")
    assert (got[0][~counts] == 0).all()
    again = cascade_amd.linear_distillation_backward(d_loss, hidden, weight, ids, logits, lse, temperature)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    return hidden, weight, ids, logits, loss, lse, got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,dim,vocab", [(1, 8, 1), (1, 64, 300), (3, 72, 257), (61, 512, 5000), (64, 128, 256), (65, 200, 1025), (257, 320, 3000),
                                         (513, 136, 511), (700, 256, 2049), (1025, 1024, 777)])
def test_distillation_sizes(n, dim, vocab, dtype):
    check_distillation(n, dim, vocab, 8, dtype, seed=n)


@pytest.mark.parametrize("kept", [1, 2, 3, 31, 32, 33, 63, 64, 65, 128, 129, 255, 256, 257, 500, 1024])
@pytest.mark.parametrize("spread", ["zipf", "even", "last"])
def test_distillation_from_any_number_of_logits(kept, spread):
    check_distillation(90, 64, 1500, kept, torch.bfloat16, spread=spread, seed=kept)
    check_distillation(300, 64, 700, kept, torch.float16, spread=spread, temperature=2.0, seed=kept + 1)


@pytest.mark.parametrize("dim", [1, 5, 63, 100])
@pytest.mark.parametrize("layout", ["dense", "odd", "strided"])
def test_distillation_layouts(dim, layout):
    check_distillation(70, dim, 333, 10, torch.bfloat16, layout=layout, seed=dim)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65])  # up to 64, whose products have kernels of their own
def test_distillation_of_few_tokens(n, dtype):
    for dim, vocab in ((8, 33), (120, 63), (128, 64), (136, 65), (264, 1000), (512, 16384 + 7)):
        check_distillation(n, dim, vocab, 5, dtype, seed=n + dim)
    check_distillation(n, 4100, 300, 5, dtype, layout="odd", seed=n)


@pytest.mark.parametrize("temperature", [0.05, 0.5, 1.0, 3.0, 20.0, 1000.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_distillation_temperatures(temperature, dtype):
    check_distillation(200, 128, 1000, 20, dtype, temperature=temperature, seed=4)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 5, 32])
def test_gradients_of_few_tokens_are_rounded_once(n, dtype):
    """Up to 32 tokens the gradients of the logits have twice the bits, that is errors of u^2: what is left is the rounding of the results, which those of the formula have, too, and sums of 32
    bits, below a twentieth of it. (The average of a rounding off by up to u of a value, evenly, is u / sqrt(3), not u / sqrt(12), as was first written here.)"""
    g = gen(n)
    dim, vocab = 200, 4000
    hidden, weight = randn(g, n, dim, dtype=dtype), randn(g, vocab, dim, dtype=dtype, scale=2 * dim ** -0.5)
    ids, logits = teacher(g, n, 10, vocab, ignored=0.0)
    ids[:, 0], logits[:, 0] = 3, 9.0  # no token without entries
    d_loss = torch.full((n,), 1.00390625 - 2.0 ** -10, device="cuda")
    lse = cascade_amd.linear_distillation(hidden, weight, ids, logits, 2.0)[1]
    got = cascade_amd.linear_distillation_backward(d_loss, hidden, weight, ids, logits, lse, 2.0)
    _, _, p, q, _ = reference(hidden, weight, ids, logits, 2.0)
    d_z = (p - q) * d_loss.double()[:, None] / 2.0
    for a, b in zip(got, (d_z @ weight.double(), d_z.T @ hidden.double())):
        assert (a.double() - b).norm() <= 1.05 * (b.to(dtype).double() - b).norm()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [33, 50, 64])
def test_heavy_gradients_of_33_to_64_tokens_are_rounded_once(n, dtype):
    """There the gradients of the logits have twice the bits in blocks of 64 words with an entry above an eighth of the largest weight. What is below that may be rounded twice: off by up to u of
    each product that it is part of; the rest as above."""
    g = gen(n)
    dim, vocab = 200, 4000
    hidden, weight = randn(g, n, dim, dtype=dtype), randn(g, vocab, dim, dtype=dtype, scale=2 * dim ** -0.5)
    ids, logits = teacher(g, n, 10, vocab, ignored=0.0)
    ids[:, 0], logits[:, 0] = torch.randint(0, vocab, (n,), generator=g, device="cuda").int() // 9 * 9, 9.0  # (not relative to the other logits, as was first written here: what stands beside ids that are none is NaN, in the oracle as well)
    d_loss = torch.full((n,), 1.00390625 - 2.0 ** -10, device="cuda")
    lse = cascade_amd.linear_distillation(hidden, weight, ids, logits, 1.5)[1]
    got = cascade_amd.linear_distillation_backward(d_loss, hidden, weight, ids, logits, lse, 1.5)
    _, _, p, q, _ = reference(hidden, weight, ids, logits, 1.5)
    d_z, u = (p - q) * d_loss.double()[:, None] / 1.5, torch.finfo(dtype).eps / 2
    light = torch.where((p - q).abs() <= 1 / 8, d_z, 0).abs()
    for a, b, more in zip(got, (d_z @ weight.double(), d_z.T @ hidden.double()), (light @ weight.double().abs(), light.T @ hidden.double().abs())):
        assert (a.double() - b).norm() <= 1.05 * (b.to(dtype).double() - b).norm() + u * more.norm()


def check_rows_of_33_to_64_tokens(n, d_loss, dtype):
    """Both gradients row by row, where each token has one word, in a block of 64 words of its own, that it finds unlikely: an entry of -d_loss nearly, and small ones. A row is off by the rounding of
    the result, by a twentieth of that for sums of 32 bits, and by what a single rounding makes of its small entries: u of each, one sign as likely as the other, so that their squares add up (to a
    tenth more: the rows that they are multiplied with are nearly at right angles), and in half precision half a step of 2^-24 of the largest weight over 2^14. That is up to 1.13 times the rounding in
    d_hidden. With an entry of -d_loss that is rounded once as well it is 2, which is shown on the formula's values."""
    g = gen(n)
    dim, blocks = 200, 70
    hidden, weight = randn(g, n, dim, dtype=dtype), randn(g, 64 * blocks, dim, dtype=dtype, scale=dim ** -0.5)
    h, w = hidden.double(), weight.double()
    at = torch.arange(n, device="cuda")
    block = torch.randperm(blocks, generator=g, device="cuda")[:n]
    words = (h @ w.T).view(n, blocks, 64)[at, block].argmin(1) + 64 * block
    ids, logits = words[:, None].int(), torch.zeros(n, 1, device="cuda")
    lse = cascade_amd.linear_distillation(hidden, weight, ids, logits)[1]
    got = cascade_amd.linear_distillation_backward(d_loss, hidden, weight, ids, logits, lse)
    _, _, p, q, _ = reference(hidden, weight, ids, logits, 1.0)
    d_z, u, top, full = (p - q) * d_loss.double()[:, None], U[dtype], d_loss.max().double(), 16384.0 if dtype == torch.float16 else 1.0
    off = (u * torch.where((p - q).abs() > 1 / 8, 0.0, d_z)) ** 2 + (top * 2.0 ** -25 / full if dtype == torch.float16 else 0.0) ** 2
    once = (d_z * (full / top)).to(dtype).double() * (top / full)
    for name, a, want, more, worse in (("d_hidden", got[0], d_z @ w, off @ w.square(), once @ w),
                                       ("d_weight", got[1][words], (d_z.T @ h)[words], (off.T @ h.square())[words], (once.T @ h)[words])):
        bound = 1.05 * (want.to(dtype).double() - want).norm(dim=1) + 1.1 * more.sum(1).sqrt()
        # all rows but those whose weight happens to need few bits
        assert ((worse.to(dtype).double() - want).norm(dim=1) > bound).sum() >= n - 5, name
        ratio = (a.double() - want).norm(dim=1) / bound
        assert (ratio <= 1).all(), f"{name}: {int((ratio > 1).sum())} of {n} rows are off by up to {ratio.max().item():.2f} of the bound"


def weights_that_need_bits(n, far, dtype):
    """One token's weight is 2, by which all are held; the others lie three quarters of the way to where rounding changes sides, over powers of two from 1 to 2^-far."""
    w = (1 + 0.75 * U[dtype]) * torch.exp2(-(torch.arange(n, device="cuda") % (far + 1)).float())
    w[0] = 2.0
    return w


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [33, 50, 64])
def test_rows_of_33_to_64_tokens_of_even_weights(n, dtype):
    check_rows_of_33_to_64_tokens(n, weights_that_need_bits(n, 0, dtype), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [33, 50, 64])
@pytest.mark.parametrize("far", [3, 8])
def test_rows_of_33_to_64_tokens_of_uneven_weights(far, n, dtype):
    """How exact a token's gradient is does not depend on how much the others weigh."""
    check_rows_of_33_to_64_tokens(n, weights_that_need_bits(n, far, dtype), dtype)


@pytest.mark.parametrize("n", [40, 90, 1100])  # four waves a token, and one
@pytest.mark.parametrize("kept", [5, 100, 300])
@pytest.mark.parametrize("temperature", [0.25, 1.0, 3.0])
def test_only_minus_infinity_is_no_entry(temperature, kept, n):
    """Finite logits are entries, however low or high, and a softmax is that of the logits less their largest one: less 1000 is nothing at these temperatures."""
    g = gen(n + kept)
    dim, vocab = 64, 500
    lowest, highest = torch.finfo(torch.float32).min, torch.finfo(torch.float32).max
    ids = torch.randint(0, vocab, (n, kept), generator=g, device="cuda", dtype=torch.int32)
    logits = randn(g, n, kept, scale=3.0)
    logits[0] = lowest
    logits[1] = highest
    logits[2, 1:] = lowest
    logits[3, :2] = lowest
    logits[3, 2:] = -math.inf
    logits[4, 1:] = lowest
    logits[4, 0] = highest
    logits[5] = -math.inf
    logits[6, 1:] = -2e38
    logits[6, 0] = lowest
    logits[7] += 1e30
    told = logits - logits.amax(1, keepdim=True)  # -infinity less itself is NaN: token 5 stays without entries
    told = torch.where(torch.isnan(told), -math.inf, torch.where(torch.isinf(logits), -math.inf, told.clamp(min=-1000.0)))
    hidden, weight, _, _, loss, lse, grads = check_distillation(n, dim, vocab, kept, torch.bfloat16, temperature, told=(ids, told), weights=torch.ones(n, device="cuda"), seed=n)
    got = cascade_amd.linear_distillation(hidden, weight, ids, logits, temperature)
    assert torch.equal(got[0], loss) and torch.equal(got[1], lse)
    found = cascade_amd.linear_distillation_backward(torch.ones(n, device="cuda"), hidden, weight, ids, logits, lse, temperature)
    assert all(torch.equal(a, b) for a, b in zip(found, grads))
    assert loss[0] > 0 and loss[5] == 0


def test_distillation_over_the_corpus_vocabulary():
    check_distillation(600, 256, 50257, 50, torch.bfloat16, seed=3)
    check_distillation(40, 256, 65535, 100, torch.float16, seed=4)


def test_distillation_in_pieces_of_the_vocabulary():
    """More than one piece of the vocabulary, and shares of d_hidden, in both tile widths."""
    check_distillation(6000, 64, 50257, 16, torch.bfloat16, seed=5)
    check_distillation(1500, 64, 3000, 100, torch.float16, seed=6)


def test_distillation_of_uneven_weights():
    w = torch.logspace(-6, 0, 300, device="cuda")
    check_distillation(300, 128, 1000, 12, torch.float16, weights=w, seed=6)
    check_distillation(300, 128, 1000, 12, torch.bfloat16, weights=w, seed=6)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_student_that_has_learnt_has_exact_small_gradients(dtype):
    """A teacher that keeps all words and agrees with the student but for little: p - q is a thousandth of p, and still off by its own rounding only (and by
    what 32 bits make of p and q, a part in 10^6 of them)."""
    g = gen(7)
    n, dim, vocab = 150, 64, 256
    hidden, weight = randn(g, n, dim, dtype=dtype), randn(g, vocab, dim, dtype=dtype).mul_(2 * dim ** -0.5)
    logits = (hidden.double() @ weight.double().T + 1e-3 * torch.randn(n, vocab, generator=g, device="cuda")).float()
    order = torch.rand(n, vocab, generator=g, device="cuda").argsort(1)
    told = (order.int(), logits.gather(1, order))
    check_distillation(n, dim, vocab, vocab, dtype, told=told, seed=7, weights=torch.ones(n, device="cuda"))


def test_one_entry_is_a_cross_entropy():
    """A teacher with one word: q is 1, and losses and gradients are those of that target."""
    g = gen(8)
    n, dim, vocab = 300, 128, 2000
    hidden, weight = randn(g, n, dim, dtype=torch.bfloat16), randn(g, vocab, dim, dtype=torch.bfloat16, scale=2 * dim ** -0.5)
    target = torch.randint(-1, vocab, (n,), generator=g, device="cuda", dtype=torch.int32)
    d_loss = randn(g, n)
    loss, lse = cascade_amd.linear_cross_entropy(hidden, weight, target)
    got, sums = cascade_amd.linear_distillation(hidden, weight, target[:, None].contiguous(), randn(g, n, 1))
    assert torch.allclose(got, loss, rtol=0, atol=1e-5) and torch.allclose(sums, lse, rtol=0, atol=1e-5)
    want = cascade_amd.linear_cross_entropy_backward(d_loss, hidden, weight, target, lse)
    found = cascade_amd.linear_distillation_backward(d_loss, hidden, weight, target[:, None].contiguous(), randn(g, n, 1), lse)
    for a, b in zip(found, want):
        assert (a.double() - b.double()).norm() <= 2 * 2.0 ** -8 * b.double().norm()


def test_the_order_of_entries_and_absent_ones_change_little():
    g = gen(9)
    n, dim, vocab, kept = 200, 64, 900, 30
    hidden, weight = randn(g, n, dim, dtype=torch.bfloat16), randn(g, vocab, dim, dtype=torch.bfloat16, scale=2 * dim ** -0.5)
    ids, logits = teacher(g, n, kept, vocab)
    order = torch.rand(n, kept, generator=g, device="cuda").argsort(1)
    loss = cascade_amd.linear_distillation(hidden, weight, ids, logits)[0]
    other = cascade_amd.linear_distillation(hidden, weight, ids.gather(1, order), logits.gather(1, order))[0]
    wider = cascade_amd.linear_distillation(hidden, weight, torch.cat([ids, torch.full_like(ids, -1)], 1), torch.cat([logits, torch.full_like(logits, math.nan)], 1))[0]
    assert torch.allclose(loss, other, rtol=0, atol=1e-5) and torch.allclose(loss, wider, rtol=0, atol=1e-5)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
def test_logits_of_16_bits(kind):
    g = gen(10)
    hidden, weight = randn(g, 50, 64, dtype=torch.float16), randn(g, 400, 64, dtype=torch.float16, scale=0.2)
    ids, logits = teacher(g, 50, 12, 400)
    a = cascade_amd.linear_distillation(hidden, weight, ids, logits.to(kind))
    b = cascade_amd.linear_distillation(hidden, weight, ids, logits.to(kind).float())
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("n", [50, 600])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_a_bad_weight_of_a_token_reaches_its_own_gradient_only(n, value):
    """In d_hidden; every word's gradient is a sum over all tokens."""
    g = gen(17)
    hidden, weight = randn(g, n, 64, dtype=torch.float16), randn(g, 900, 64, dtype=torch.float16, scale=0.2)
    ids, logits = teacher(g, n, 9, 900, ignored=0.0)
    ids[5] = torch.arange(9)
    d_loss = torch.rand(n, generator=g, device="cuda")
    lse = cascade_amd.linear_distillation(hidden, weight, ids, logits)[1]
    d_loss[5] = 0.5 * d_loss.max()  # not the largest one, by which all are held
    clean = cascade_amd.linear_distillation_backward(d_loss, hidden, weight, ids, logits, lse, want_weight=False)[0]
    d_loss[5] = value
    got = cascade_amd.linear_distillation_backward(d_loss, hidden, weight, ids, logits, lse, want_weight=False)[0]
    rest = torch.arange(n, device="cuda") != 5
    assert torch.equal(got[rest], clean[rest]) and not torch.isfinite(got[5]).any()


@pytest.mark.parametrize("n", [50, 600])
def test_tokens_without_entries_may_hold_anything(n):
    g = gen(11)
    hidden, weight = randn(g, n, 64, dtype=torch.bfloat16), randn(g, 500, 64, dtype=torch.bfloat16)
    ids, logits = teacher(g, n, 9, 500, ignored=0.0)
    ids[::3] = -1
    d_loss = torch.ones(n, device="cuda")
    want = cascade_amd.linear_distillation_backward(d_loss, hidden, weight, ids, logits, cascade_amd.linear_distillation(hidden, weight, ids, logits)[1])
    spoilt, odd = hidden.clone(), d_loss.clone()
    spoilt[::6], spoilt[3::6] = math.nan, math.inf
    odd[::3] = math.nan
    logits[::3] = math.inf
    loss, lse = cascade_amd.linear_distillation(spoilt, weight, ids, logits)
    assert (loss[::3] == 0).all() and torch.isfinite(loss).all()
    got = cascade_amd.linear_distillation_backward(odd, spoilt, weight, ids, logits, lse)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and (got[0][::3] == 0).all()


@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_a_bad_entry_reaches_its_token_only(value):
    g = gen(12)
    n = 90
    hidden, weight = randn(g, n, 64, dtype=torch.bfloat16), randn(g, 500, 64, dtype=torch.bfloat16)
    ids, logits = teacher(g, n, 9, 500, ignored=0.0)
    ids[7], logits[7] = torch.arange(9), 1.0
    clean = cascade_amd.linear_distillation(hidden, weight, ids, logits)[0]
    logits[7, 4] = value
    got, lse = cascade_amd.linear_distillation(hidden, weight, ids, logits)
    rest = torch.arange(n, device="cuda") != 7
    assert torch.equal(got[rest], clean[rest]) and not torch.isfinite(got[7])
    d_hidden, _ = cascade_amd.linear_distillation_backward(torch.ones(n, device="cuda"), hidden, weight, ids, logits, lse)
    assert torch.isfinite(d_hidden[rest]).all() and not torch.isfinite(d_hidden[7]).any()


def test_distillation_of_no_tokens():
    hidden, weight = torch.empty(0, 33, dtype=torch.bfloat16, device="cuda"), torch.ones(50, 33, dtype=torch.bfloat16, device="cuda")
    none = torch.empty(0, device="cuda")
    ids, logits = torch.empty(0, 5, dtype=torch.int32, device="cuda"), torch.empty(0, 5, device="cuda")
    loss, lse = cascade_amd.linear_distillation(hidden, weight, ids, logits)
    assert loss.numel() == lse.numel() == 0
    d_hidden, d_weight = cascade_amd.linear_distillation_backward(none, hidden, weight, ids, logits, none)
    assert d_hidden.shape == (0, 33) and (d_weight == 0).all()


def test_distillation_gradients_agree_with_differences():
    g = gen(13)
    hidden, weight = randn(g, 40, 64, dtype=torch.bfloat16), randn(g, 300, 64, dtype=torch.bfloat16, scale=0.2)
    ids, logits = teacher(g, 40, 12, 300)
    d_loss = torch.rand(40, generator=g, device="cuda")
    lse = cascade_amd.linear_distillation(hidden, weight, ids, logits, 1.5)[1]
    grads = cascade_amd.linear_distillation_backward(d_loss, hidden, weight, ids, logits, lse, 1.5)
    for which, grad in enumerate(grads):
        way = randn(g, *grad.shape).double()
        values = []
        for step in (1e-4, -1e-4):
            x = [hidden.double(), weight.double()]
            x[which] = x[which] + step * way
            values.append((reference(*x, ids, logits, 1.5)[0] * d_loss.double()).sum().item())
        slope = (values[0] - values[1]) / 2e-4
        assert abs((grad.double() * way).sum().item() - slope) <= 4 * 2.0 ** -7 * (grad.double() * way).norm().item()


def test_autograd_of_distillation():
    g = gen(14)
    hidden = randn(g, 100, 72, dtype=torch.float16).requires_grad_()
    weight = randn(g, 500, 72, dtype=torch.float16, scale=0.2).requires_grad_()
    ids, logits = teacher(g, 100, 12, 500)
    loss = cascade_amd.distillation_loss(hidden, weight, ids, logits, temperature=2.0)
    got = torch.autograd.grad(loss.sum(), (hidden, weight))  # an expanded gradient
    _, lse = cascade_amd.linear_distillation(hidden.detach(), weight.detach(), ids, logits, 2.0)
    want = cascade_amd.linear_distillation_backward(torch.ones_like(lse), hidden.detach(), weight.detach(), ids, logits, lse, 2.0)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    loss = cascade_amd.distillation_loss(hidden, weight.detach(), ids, logits, temperature=2.0)
    assert torch.equal(torch.autograd.grad(loss.sum(), hidden)[0], want[0])
    loss = cascade_amd.distillation_loss(hidden.detach(), weight, ids, logits, temperature=2.0)
    assert torch.equal(torch.autograd.grad(loss.sum(), weight)[0], want[1])
    with pytest.raises(ValueError, match="teacher"):
        cascade_amd.distillation_loss(hidden, weight, ids, logits.requires_grad_())


@pytest.mark.parametrize("n", [1, 40, 64, 65, 400])
def test_a_gradient_that_is_not_wanted_changes_nothing(n):
    g = gen(16)
    hidden, weight = randn(g, n, 72, dtype=torch.bfloat16), randn(g, 700, 72, dtype=torch.bfloat16, scale=0.2)
    ids, logits = teacher(g, n, 6, 700)
    d_loss = torch.rand(n, generator=g, device="cuda")
    how = (d_loss, hidden, weight, ids, logits, cascade_amd.linear_distillation(hidden, weight, ids, logits)[1])
    both = cascade_amd.linear_distillation_backward(*how)
    first = cascade_amd.linear_distillation_backward(*how, want_weight=False)
    second = cascade_amd.linear_distillation_backward(*how, want_hidden=False)
    assert torch.equal(first[0], both[0]) and first[1] is None and second[0] is None and torch.equal(second[1], both[1])


@pytest.mark.parametrize("n,vocab", [(40, 3000), (1100, 2000)])
def test_distillation_on_another_stream_and_in_a_graph_gives_the_same(n, vocab):
    g = gen(15)
    hidden, weight = randn(g, n, 128, dtype=torch.float16), randn(g, vocab, 128, dtype=torch.float16, scale=0.2)
    ids, logits = teacher(g, n, 20, vocab)
    d_loss = torch.rand(n, generator=g, device="cuda")

    def step():
        loss, lse = cascade_amd.linear_distillation(hidden, weight, ids, logits, 2.0)
        return [loss, lse, *cascade_amd.linear_distillation_backward(d_loss, hidden, weight, ids, logits, lse, 2.0)]
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
        hidden.copy_(torch.randn(hidden.shape, generator=g, device="cuda"))
        for x, y in zip((ids, logits), teacher(g, n, 20, vocab)):
            x.copy_(y)
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(recorded, want)):
            assert torch.equal(a, b), f"value {i} of replay {turn}"


def test_refusals():
    w = torch.zeros(10, 64, dtype=torch.bfloat16, device="cuda")
    ids, logits = torch.zeros(4, 3, dtype=torch.int32, device="cuda"), torch.zeros(4, 3, device="cuda")
    assert cascade_amd.linear_distillation(w[:4], w, ids, logits)[0].shape == (4,)
    for bad in (ids.long(), ids[0], ids[:3], ids.t().contiguous().t(), ids.cpu()):
        with pytest.raises(ValueError):
            cascade_amd.linear_distillation(w[:4], w, bad, logits)
    for bad in (logits[:, :2], logits.cpu(), logits.t().contiguous().t()):
        with pytest.raises(ValueError):
            cascade_amd.linear_distillation(w[:4], w, ids, bad)
    with pytest.raises(ValueError):
        cascade_amd.linear_distillation(w[:4, :32], w, ids, logits)
    for bad in (logits.double(), logits.int()):
        with pytest.raises(TypeError):
            cascade_amd.linear_distillation(w[:4], w, ids, bad)
    with pytest.raises(TypeError):
        cascade_amd.linear_distillation(w[:4].float(), w.float(), ids, logits)
    for temperature in (0.0, -1.0, math.nan, math.inf, 1e-5, 1e5):
        with pytest.raises(cascade_amd._native.CascadeError):
            cascade_amd.linear_distillation(w[:4], w, ids, logits, temperature)
    for kept in (0, 1025):
        with pytest.raises(cascade_amd._native.CascadeError):
            cascade_amd.linear_distillation(w[:4], w, torch.zeros(4, kept, dtype=torch.int32, device="cuda"), torch.zeros(4, kept, device="cuda"))
    lse = torch.zeros(4, device="cuda")
    for bad in (lse.double(), lse[:3], lse[None], lse.cpu()):
        with pytest.raises(ValueError):
            cascade_amd.linear_distillation_backward(bad, w[:4], w, ids, logits, lse)
        with pytest.raises(ValueError):
            cascade_amd.linear_distillation_backward(lse, w[:4], w, ids, logits, bad)
