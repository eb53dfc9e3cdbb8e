"""Trains a small language model on a corpus of documents, from the suffix sort to the clipped step.

The corpus is the benchmark's token text (uint16, 0xFFFF in front of every document, some documents copies of others). Its suffixes are
sorted on the GPU; neighbours in the suffix array that begin with the same tokens are repeated passages, and a position
whose passage also stands earlier in the corpus is left out of the loss. The training step then packs a stretch of the corpus as it
lies, without padding: spans keep attention inside documents, the loss runs over the whole vocabulary without keeping its logits, and the
gradients are clipped by their global norm.

    python examples/train_on_documents.py [--tokens 200000] [--steps 20] [--length 4096]
"""
import argparse
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

import cascade_amd  # noqa: E402
from cascade_amd import workloads  # noqa: E402

SEPARATOR = 0xFFFF
VOCAB = 50257


def repeated(text, passage):
    """Truth values of every position of text (a uint16 tensor on the GPU, viewed as int16): does the passage of `passage` tokens that begins there
    begin somewhere before it, too?"""
    n = text.numel()
    with cascade_amd.PartitionSorter(n) as sorter:
        lanes = sorter.sort(text).view(n, 5).long()
    suffixes = (lanes << torch.arange(0, 40, 8, device=text.device)).sum(1)
    padded = torch.cat([text.int(), torch.arange(-(1 << 20), -(1 << 20) + passage, device=text.device, dtype=torch.int32)])  # no two ends alike
    same = torch.ones(n - 1, dtype=torch.bool, device=text.device)  # does a suffix begin as the one before it in the suffix array does?
    for k in range(passage):
        token = padded[suffixes + k]
        same &= token[1:] == token[:-1]
    run = torch.cat([same.new_zeros(1), ~same]).cumsum(0)  # suffixes with one beginning stand in one run
    first = torch.full((n,), n, device=text.device).scatter_reduce_(0, run, suffixes, "amin")
    found = torch.empty(n, dtype=torch.bool, device=text.device)
    found[suffixes] = first[run] < suffixes
    return found


class Model(torch.nn.Module):
    """Embedding, blocks of attention over spans (heads of q share those of k and v) and a two-layer network, and a vocabulary's weight. A separator is a
    word of its own in the embedding, and no target."""

    def __init__(self, dim=256, heads=4, kv_heads=2, blocks=2):
        super().__init__()
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, dim // heads
        make = lambda *shape: torch.nn.Parameter((torch.randn(*shape) * shape[-1] ** -0.5).to(torch.bfloat16))  # noqa: E731
        self.embedding = make(VOCAB + 1, dim)
        self.qkv = torch.nn.ParameterList(make((heads + 2 * kv_heads) * self.head_dim, dim) for _ in range(blocks))
        self.out = torch.nn.ParameterList(make(dim, dim) for _ in range(blocks))
        self.up = torch.nn.ParameterList(make(4 * dim, dim) for _ in range(blocks))
        self.down = torch.nn.ParameterList(make(dim, 4 * dim) for _ in range(blocks))
        self.words = make(VOCAB, dim)
        # the further away a key is, the less it counts: a different rate for each head, in place of positions
        self.register_buffer("slopes", torch.exp2(-8.0 * torch.arange(1, heads + 1) / heads))

    @staticmethod
    def norm(x):
        return (x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6)).to(x.dtype)

    def forward(self, tokens, lo, hi, target):
        """The loss of every token's target."""
        x = self.embedding[tokens]
        for qkv, out, up, down in zip(self.qkv, self.out, self.up, self.down):
            y = (self.norm(x) @ qkv.T).view(-1, self.heads + 2 * self.kv_heads, self.head_dim)
            q, k, v = y.split([self.heads, self.kv_heads, self.kv_heads], 1)
            x = x + cascade_amd.attend(q, k, v, lo, hi, slopes=self.slopes).flatten(1) @ out.T
            x = x + torch.nn.functional.silu(self.norm(x) @ up.T) @ down.T
        return cascade_amd.next_token_loss(self.norm(x), self.words, target)


def train(tokens=200000, steps=20, length=4096, passage=32, rate=0.5, max_norm=1.0, seed=0, say=print):
    """Losses of the steps, and how much of the corpus was left out as repeated."""
    torch.manual_seed(seed)
    text = torch.from_numpy(workloads.generate(3, tokens).view("int16")).cuda()
    seen_before = repeated(text, passage)
    share = seen_before.float().mean().item()
    say(f"{tokens} tokens sorted: {100 * share:.1f} % of the positions begin a passage of {passage} tokens that stands earlier, too")
    model = Model().cuda()
    weights = list(model.parameters())
    losses = []
    for step in range(steps):
        begin = step * length % max(1, tokens - length + 1)
        part = text[begin:begin + length]
        lo, hi, target = cascade_amd.token_spans(part, separator=SEPARATOR)
        counts = (target >= 0) & ~seen_before[begin:begin + length]
        words = part.int() & 0xFFFF
        loss = model(torch.where(words == SEPARATOR, VOCAB, words).long(), lo, hi, torch.where(counts, target, -1))
        loss = loss.sum() / counts.sum().clamp(min=1)
        loss.backward()
        norm = cascade_amd.clip_gradients([w.grad for w in weights], max_norm)
        with torch.no_grad():
            for w in weights:
                w.sub_(w.grad, alpha=rate)
                w.grad = None
        losses.append(loss.item())
        say(f"step {step}: loss {losses[-1]:.4f}, gradient norm {norm.item():.3f}")
    return losses, share


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=200000)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--length", type=int, default=4096)
    a = ap.parse_args()
    train(a.tokens, a.steps, a.length)
