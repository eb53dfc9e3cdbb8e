"""What distillation's entry points refuse before anything is launched, and the sizes of their workspaces. No GPU needed: what is accepted here ends at the
workspace, which is too small."""
import math

import pytest

from cascade_amd import _native_lm as native

BAD, LARGE, FINE = -1, -2, 0
X = 1 << 20  # an address that nothing reads


def forward(**change):
    a = dict(type=0, hidden=X, hs=64, weight=X, ws=64, ids=X, logits=X, kept=8, temperature=1.0, tokens=5, dim=64, vocab=300, loss=X, lse=X, work=X, size=0)
    a.update(change)
    return native.load().csa_lm_distill_forward_dev(*a.values(), None)


def backward(**change):
    a = dict(type=0, hidden=X, hs=64, weight=X, ws=64, ids=X, logits=X, kept=8, temperature=1.0, lse=X, d_loss=X, tokens=5, dim=64, vocab=300, d_hidden=X, dhs=64,
             d_weight=X, dws=64, work=X, size=0)
    a.update(change)
    return native.load().csa_lm_distill_backward_dev(*a.values(), None)


def message():
    return native.load().csa_lm_last_error()


@pytest.mark.parametrize("change", [dict(type=2), dict(type=7), dict(kept=0), dict(kept=1025), dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=math.nan),
                                    dict(temperature=math.inf), dict(temperature=9e-5), dict(temperature=2e4), dict(ids=None), dict(ids=X + 2), dict(logits=None), dict(logits=X + 2),
                                    dict(hidden=None), dict(hidden=X + 1), dict(weight=None), dict(dim=0), dict(vocab=0), dict(hs=63), dict(ws=1 << 22), dict(lse=None),
                                    dict(lse=X + 2)])
def test_arguments(change):
    assert forward(**change) == BAD and b"workspace" not in message()
    assert backward(**change) == BAD and b"workspace" not in message()


def test_results_and_workspaces():
    assert forward(loss=None) == BAD and b"workspace" not in message()
    for change in (dict(d_loss=None), dict(d_loss=X + 2), dict(d_hidden=X + 1), dict(dhs=60), dict(d_weight=X + 1), dict(dws=60)):
        assert backward(**change) == BAD and b"workspace" not in message()
    size = native.load().csa_lm_distill_workspace
    for call, flags in ((forward, 0), (backward, native.CSA_LM_BACKWARD)):
        need = size(5, 64, 300, 8, flags)
        assert need > 0
        assert call() == BAD and b"workspace" in message()
        assert call(size=need - 1) == BAD and b"workspace" in message()
        assert call(work=X + 128, size=need) == BAD and b"workspace" in message()
    assert forward(tokens=0) == FINE


@pytest.mark.parametrize("tokens,dim,vocab", [(1 << 24, 8, 300), (1 << 23, 64, 65536), (100, 4096, 1 << 31), (100, 1 << 22, 300)])
def test_more_than_a_launch_holds(tokens, dim, vocab):
    stride = min(dim, (1 << 22) - 8)
    assert forward(tokens=tokens, dim=dim, vocab=vocab, hs=stride, ws=stride) == LARGE
    assert native.load().csa_lm_distill_workspace(tokens, dim, vocab, 8, 0) == 0


def test_workspaces_hold_the_entries_and_no_logits():
    """Beside the cross entropy's: ids and q, the first entry of each block of at least 64 words in 16 bits, a few numbers of every token, and forwards a number for
    each part of the vocabulary that a wave sums. Up to 64 tokens, backwards, also twice 32 or 64 values of 16 bits for every word, what the rounding leaves of the gradients of the logits,
    a number for each block of 64 words, and a sum of d_hidden for every workgroup of 128 values, one a compute unit."""
    lib = native.load()
    for tokens in (1, 32, 33, 61, 64, 65, 4099, 8192):
        for kept in (1, 64, 1024):
            for flags in (0, native.CSA_LM_BACKWARD):
                more = lib.csa_lm_distill_workspace(tokens, 1024, 50257, kept, flags) - lib.csa_lm_cross_entropy_workspace(tokens, 1024, 50257, flags)
                few = 50304 * 2 * tokens + 50257 * (128 if tokens <= 32 else 256) + 786 * 4 + 256 * 128 * 4 * tokens if flags and tokens <= 64 else 0
                assert tokens * kept * 8 <= more <= tokens * (kept * 8 + 2 * 787 + 8 + (0 if flags else 4 * 788)) + few + 8 * 256
    assert lib.csa_lm_distill_workspace(5, 64, 300, 0, 0) == lib.csa_lm_distill_workspace(5, 64, 300, 1025, 0) == 0
