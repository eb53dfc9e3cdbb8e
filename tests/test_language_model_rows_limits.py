"""What the embeddings' and norms' entry points refuse before anything is launched, and the sizes of their workspaces. No GPU needed: what is accepted here
ends at the workspace, which is too small, or has nothing to do."""
import math

import pytest

from cascade_amd import _native_lm as native

BAD, LARGE, FINE = -1, -2, 0
X = 1 << 20  # an address that nothing reads


def embed(**change):
    a = dict(type=0, tokens=X, token_bytes=4, n=0, weight=X, stride=64, rows=100, dim=64, scale=1.0, out=X)
    a.update(change)
    return native.load().csa_lm_embed_forward_dev(*a.values(), None)


def embed_backward(**change):
    a = dict(type=0, tokens=X, token_bytes=4, n=5, d_out=X, stride=64, rows=100, dim=64, scale=1.0, d_weight=X, work=X, size=0)
    a.update(change)
    return native.load().csa_lm_embed_backward_dev(*a.values(), None)


def norm(**change):
    a = dict(type=0, stream=0, x=X, xs=64, residual=X, rs=64, gain=X, eps=1e-6, tokens=0, dim=64, out=X, total=X, rstd=X)
    a.update(change)
    return native.load().csa_lm_norm_forward_dev(*a.values(), None)


def norm_backward(**change):
    a = dict(type=0, stream=0, d_out=X, gs=64, total=X, ts=64, rstd=X, gain=X, d_total=X, ds=64, tokens=5, dim=64, d_x=X, d_residual=X, d_gain=X, work=X, size=0)
    a.update(change)
    return native.load().csa_lm_norm_backward_dev(*a.values(), None)


@pytest.mark.parametrize("change", [dict(type=3), dict(type=-1), dict(token_bytes=8), dict(token_bytes=1), dict(rows=0), dict(dim=7), dict(scale=math.nan),
                                    dict(scale=math.inf), dict(n=5, tokens=None), dict(n=5, tokens=X + 2), dict(stride=63), dict(stride=1 << 22)])
def test_embed_arguments(change):
    assert embed() == FINE and embed(**change) == BAD
    assert embed_backward(**change) == BAD and b"workspace" not in native.load().csa_lm_last_error()


def test_embed_addresses():
    assert embed(weight=None) == embed(weight=X + 1) == embed(n=5, out=None) == embed(n=5, out=X + 1) == embed(type=2, weight=X + 2) == BAD
    for change in (dict(d_out=None), dict(d_out=X + 1), dict(d_weight=None), dict(d_weight=X + 1), dict(type=2, d_out=X + 2)):
        assert embed_backward(**change) == BAD and b"workspace" not in native.load().csa_lm_last_error()
    assert embed_backward() == BAD and b"workspace" in native.load().csa_lm_last_error()
    assert embed_backward(work=X + 8, size=1 << 20) == BAD and b"workspace" in native.load().csa_lm_last_error()


@pytest.mark.parametrize("change", [dict(n=1 << 31), dict(rows=1 << 31), dict(dim=1 << 22, stride=1 << 22), dict(n=(1 << 31) - 1, dim=128, stride=128)])
def test_embed_of_more_than_a_launch_holds(change):
    assert embed(**change) == LARGE and embed_backward(**change) == LARGE


def test_embed_gradients_of_more_than_a_launch_holds():
    size = native.load().csa_lm_embed_backward_workspace
    assert size(0, 1 << 31, 10, 64) == size(0, 5, 1 << 31, 64) == size(0, 5, 0, 64) == size(0, 5, 10, 7) == size(0, 5, 10, 1 << 22) == size(3, 5, 10, 64) == 0
    big = dict(n=5, rows=(1 << 31) - 1, dim=8192, stride=8192)
    assert embed_backward(**big) == LARGE and size(0, 5, big["rows"], 8192) == 0


def test_embed_workspaces():
    """Words and places of every token twice at most, counts of digits, and two sums of 32 bits for every run of at least eight tokens."""
    size = native.load().csa_lm_embed_backward_workspace
    for n in (1, 8, 9, 4096, 8192, 8193, 300000, 1 << 24):
        for rows in (1, 50257, 65536, 1 << 20):
            for dim in (8, 100, 4096):
                assert 0 < size(0, n, rows, dim) <= 16 * n + (4097 * 512 * 4 if n > 8192 else 0) + -(-n // 8) * 8 * dim + 2048
    assert size(0, 1 << 20, 50257, 4096) <= 16 * (1 << 20) + 4097 * 1024 + (1 << 20) // 64 * 8 * 4096 + 2048  # runs of 64 where there are many


@pytest.mark.parametrize("change", [dict(type=3), dict(stream=1), dict(type=2, stream=0), dict(dim=7), dict(dim=16385), dict(eps=0.0), dict(eps=-1.0), dict(eps=math.nan),
                                    dict(eps=math.inf), dict(residual=None, stream=2), dict(gain=X + 1)])
def test_norm_arguments(change):
    assert norm() == norm(stream=2) == norm(residual=None) == norm(gain=None) == FINE and norm(**change) == BAD


@pytest.mark.parametrize("change", [dict(x=None), dict(x=X + 1), dict(xs=63), dict(xs=1 << 22), dict(residual=X + 1), dict(rs=60), dict(total=None), dict(total=X + 1),
                                    dict(stream=2, total=X + 2), dict(stream=2, residual=X + 2), dict(out=None), dict(out=X + 1), dict(rstd=None), dict(rstd=X + 2)])
def test_norm_addresses(change):
    assert norm(tokens=5, **change) == BAD


@pytest.mark.parametrize("change", [dict(type=3), dict(stream=1), dict(dim=7), dict(dim=16385), dict(d_out=None), dict(d_out=X + 1), dict(gs=60), dict(total=None), dict(ts=60),
                                    dict(rstd=None), dict(rstd=X + 2), dict(d_total=X + 1), dict(ds=60), dict(d_x=X + 1), dict(d_residual=X + 1), dict(d_gain=X + 1),
                                    dict(gain=X + 1), dict(stream=2, d_residual=X + 2)])
def test_norm_gradient_arguments(change):
    assert norm_backward(**change) == BAD and b"workspace" not in native.load().csa_lm_last_error()
    assert norm_backward() == BAD and b"workspace" in native.load().csa_lm_last_error()


def test_norm_of_more_than_a_launch_holds():
    assert norm(tokens=1 << 24) == norm_backward(tokens=1 << 24) == LARGE
    assert norm(tokens=1 << 22, dim=2049, xs=2049, rs=2049) == norm_backward(tokens=1 << 22, dim=2049, gs=2049, ts=2049, ds=2049) == LARGE
    for fine in (dict(tokens=(1 << 24) - 1), dict(tokens=(1 << 22) - 1, dim=2049, gs=2049, ts=2049, ds=2049)):
        assert norm_backward(**fine) == BAD and b"workspace" in native.load().csa_lm_last_error()
    size = native.load().csa_lm_norm_backward_workspace
    assert size(5, 7) == size(5, 16385) == 0
    assert size(1, 64) == 256 and all(size(1 << 20, dim) <= 4096 * 4 * dim + 256 for dim in (8, 1024, 16384))


def test_norm_workspaces_hold_a_row_of_sums_for_every_workgroup():
    """Of as many workgroups as there are tokens, 768 at most: no row less, which a workgroup would write past the end, and none more."""
    size = native.load().csa_lm_norm_backward_workspace
    for tokens in (0, 1, 2, 255, 256, 257, 511, 512, 513, 767, 768, 769, 1 << 20, (1 << 24) - 1):
        for dim in (8, 9, 63, 64, 1000, 4096, 16383, 16384):
            assert size(tokens, dim) == -(-min(tokens, 768) * dim * 4 // 256) * 256
            if tokens:
                need = size(tokens, dim)
                strides = dict(gs=dim, ts=dim, ds=dim, dim=dim, tokens=min(tokens, (1 << 22) - 1))
                assert norm_backward(size=need - 1, **strides) == BAD and str(need).encode() in native.load().csa_lm_last_error()
