"""The operators as a model uses them: embedding, norms of the residual stream, attention inside documents, and both losses, forwards and backwards through
torch.autograd, against the same model in 64 bits, written from the formulas."""
import importlib.util
import math
import os

import pytest

torch = pytest.importorskip("torch")

import cascade_amd  # noqa: E402
from test_gpu_language_model import U, gen, randn  # noqa: E402
from test_gpu_language_model_distillation import teacher  # noqa: E402

pytestmark = pytest.mark.gpu

EPS = 1e-6


class Plain:
    """The operators from their definitions, in 64 bits."""

    @staticmethod
    def embed(tokens, weight, scale):
        there = (tokens >= 0) & (tokens < weight.shape[0])
        return torch.where(there[:, None], scale * weight[torch.where(there, tokens, 0).long()], 0.0)

    @staticmethod
    def add_norm(x, residual, gain):
        total = x if residual is None else x + residual
        out = total / (total.square().mean(1, keepdim=True) + EPS).sqrt()
        return out if gain is None else out * gain, total

    @staticmethod
    def attend(q, k, v, lo, hi):
        n, heads, dim = q.shape
        at = torch.arange(n, device=q.device)
        seen = (at[None] >= lo[:, None]) & (at[None] < hi[:, None])
        out = []
        for h in range(heads):
            g = h // (heads // k.shape[1])
            z = (q[:, h] @ k[:, g].T * dim ** -0.5).masked_fill(~seen, -1e300)
            out.append(torch.where(seen.any(1)[:, None], torch.softmax(z, 1) @ v[:, g], 0.0))
        return torch.stack(out, 1)

    @staticmethod
    def next_token_loss(hidden, weight, target):
        log_p = torch.log_softmax(hidden @ weight.T, 1)
        there = target >= 0
        return torch.where(there, -log_p.gather(1, torch.where(there, target, 0).long()[:, None])[:, 0], 0.0)

    @staticmethod
    def distillation_loss(hidden, weight, ids, logits, temperature):
        log_p = torch.log_softmax(hidden @ weight.T / temperature, 1)
        there = (ids >= 0) & (ids < weight.shape[0]) & (logits != -math.inf)
        told = torch.where(there, logits.double() / temperature, -1e300)
        log_q = torch.where(there, torch.log_softmax(told, 1), 0.0)
        q = torch.where(there, log_q.exp(), 0.0)
        return (q * (log_q - log_p.gather(1, torch.where(there, ids, 0).long()))).sum(1)


def model(ops, w, text, lo, hi, target, ids, logits, heads, kv_heads):
    """The losses of a block between an embedding and a vocabulary."""
    x = ops.embed(text, w["embedding"], 4.0)
    y, x = ops.add_norm(x, None, w["gain"])
    q, k, v = (y @ w["qkv"].T).view(x.shape[0], heads + 2 * kv_heads, -1).split([heads, kv_heads, kv_heads], 1)
    y, x = ops.add_norm(ops.attend(q, k, v, lo, hi).flatten(1) @ w["out"].T, x, w["gain2"])
    y, x = ops.add_norm(torch.tanh(y @ w["up"].T) @ w["down"].T, x, None)
    return ops.next_token_loss(y, w["words"], target), ops.distillation_loss(y, w["words"], ids, logits, 2.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,dim,heads,kv_heads,vocab", [(300, 64, 2, 1, 500), (1000, 136, 4, 2, 3000)])
def test_a_model_of_all_operators(n, dim, heads, kv_heads, vocab, dtype):
    g = gen(n)
    width = dim // heads // 8 * 8
    shapes = {"embedding": (vocab, dim), "qkv": ((heads + 2 * kv_heads) * width, dim), "out": (dim, heads * width), "up": (2 * dim, dim), "down": (dim, 2 * dim), "words": (vocab, dim)}
    w = {name: randn(g, *shape, scale=shape[1] ** -0.5).to(dtype) for name, shape in shapes.items()}
    w["gain"], w["gain2"] = ((1 + randn(g, dim, scale=0.2)).to(dtype) for _ in range(2))
    text = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    text[torch.rand(n, generator=g, device="cuda") < 0.01] = 0xFFFF
    text16 = torch.where(text >= 1 << 15, text - (1 << 16), text).to(torch.int16)
    lo, hi, target = cascade_amd.token_spans(text16)
    # In bfloat16 separators have no row, and begin at zero. The norm of zeros has a slope of eps^-1/2 = 1000, and the first token of a document sees nothing but itself: two norms
    # behind each other make 10^6 of a gradient of 1024 / n there, which half precision, up to 65504, does not hold. There, they are words.
    tokens16 = text16 if dtype == torch.bfloat16 else torch.where(text16 == -1, 7, text16)
    text = torch.where(tokens16 == -1, 0xFFFF, tokens16.long())
    ids, logits = teacher(g, n, 10, vocab)
    weights = torch.rand(n, generator=g, device="cuda") / n
    results = []
    for ops, kind, tokens in ((cascade_amd, dtype, tokens16), (Plain, torch.float64, text)):
        at = {name: x.to(kind).requires_grad_() for name, x in w.items()}
        first, second = model(ops, at, tokens, lo, hi, target, ids, logits, heads, kv_heads)
        total = ((first.double() + second.double()) * weights.double()).sum() * (1024.0 if dtype == torch.float16 else 1.0)  # half precision's gradients are scaled up
        results.append((first, second, torch.autograd.grad(total, list(at.values()))))
    # Values that are rounded to 16 bits between the text and the losses: x, y, qkv, the probabilities, out, its product, x, y, two products and a tanh, their product, x, y: 14, each
    # of which moves a loss or a gradient by u of it at most, and as many gradients on the way back, with those of the logits and scores; twice over for what
    # the products and norms make of a change.
    many = 2 * 14 * U[dtype]
    for i in range(2):
        assert (results[0][i].double() - results[1][i]).norm() <= many * results[1][i].norm()
    for name, a, b in zip(w, results[0][2], results[1][2]):
        assert a.dtype == dtype and (a.double() - b).norm() <= 2 * many * b.norm(), name


def test_the_example_teaches_a_student():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_on_documents.py")
    spec = importlib.util.spec_from_file_location("train_on_documents", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    kept, lines = [], []
    example.train(tokens=20000, steps=3, length=1024, say=lines.append, keep=kept)
    losses, student = example.distil(*kept, steps=3, length=1024, say=lines.append)
    assert len(losses) == 3 and len(lines) == 7 and all(math.isfinite(x) and x > 0 for x in losses)
    # the student's gradients at the last stretch, against those of a plain loss of the same hidden values in 64 bits
    text, seen_before, model_ = kept
    _, words, lo, hi, target = example.stretch(text, 0, 1024)
    ids, logits = example.top_logits(model_, words, lo, hi, 16)
    hidden = student.hidden(words, lo, hi).detach()
    got, want = [], []
    for ops, kind, out in ((cascade_amd, torch.bfloat16, got), (Plain, torch.float64, want)):
        at = [x.detach().to(kind).requires_grad_() for x in (hidden, student.words)]
        out += torch.autograd.grad(ops.distillation_loss(*at, ids, logits, 1.0).sum(), at)
    for a, b in zip(got, want):
        assert (a.double() - b).norm() <= 2 * U[torch.bfloat16] * b.norm()
