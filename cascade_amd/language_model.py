"""Operators of a language model over the texts that this package sorts: uint16 tokens, a separator in front of every document.

  token_spans                        the keys that each position of a text may see, and the token it has to predict
  span_attention (+ _backward)       attention of every position over its span of keys
  linear_cross_entropy (+ _backward) the loss of every target over the whole vocabulary, without keeping the logits
  clip_gradients                     the global norm of many gradients, and their clipping
  attend, next_token_loss            the middle two for torch.autograd

All take torch tensors on the GPU, enqueue kernels on the current stream of the tensors' device and return without waiting
(include/cascade_lm.h; there is no CPU form). Scratch memory comes from torch's allocator and belongs to the stream.
"""
import ctypes as C
import math

from . import _native_lm as native

SEPARATOR = 0xFFFF


def _type(dtype):
    import torch
    kinds = {torch.bfloat16: native.CSA_LM_BF16, torch.float16: native.CSA_LM_F16, torch.float32: native.CSA_LM_F32}
    if dtype not in kinds:
        raise TypeError(f"{dtype} is none of bfloat16, float16 and float32")
    return kinds[dtype]


def _matrix_type(dtype):
    kind = _type(dtype)
    if kind == native.CSA_LM_F32:
        raise TypeError("the matrix products take bfloat16 or float16")
    return kind


def _check(condition, message):
    if not condition:
        raise ValueError(message)


def _on_gpu(tensors):
    """The device that all of them lie on, which has to be a GPU."""
    device = tensors[0].device
    for t in tensors:
        _check(t.is_cuda and t.device == device, "all tensors have to lie on one GPU")
    return device


class _Call:
    """The device's current stream, with the device made current for the launches."""

    def __init__(self, device):
        import torch
        self._guard = torch.cuda.device(device)
        self._device = device

    def __enter__(self):
        import torch
        self._guard.__enter__()
        return torch.cuda.current_stream(self._device).cuda_stream or None

    def __exit__(self, *exc):
        return self._guard.__exit__(*exc)


def _work(size, device):
    import torch
    return torch.empty(max(int(size), 1), dtype=torch.uint8, device=device)


def token_spans(text, separator=SEPARATOR):
    """text: n uint16 tokens (viewed as int16 is fine), one stretch of a corpus. Returns int32 tensors (lo, hi, target) of n values:
    position i may see the keys [lo[i], hi[i]), which begin at the last separator at or before i and end with i itself, and has to
    predict target[i], the token behind it, or nothing (-1) at the end and in front of a separator (csa_lm_spans_u16_dev)."""
    import torch
    device = _on_gpu([text])
    _check(text.dim() == 1 and text.element_size() == 2 and not text.is_floating_point() and text.is_contiguous(), "text: a dense vector of 16-bit tokens")
    _check(0 <= separator <= 0xFFFF, "separator: a 16-bit token")
    lib, n = native.load(), text.numel()
    lo, hi, target = (torch.empty(n, dtype=torch.int32, device=device) for _ in range(3))
    size = lib.csa_lm_spans_workspace(n)
    work = _work(size, device) if size else None
    with _Call(device) as stream:
        native.check(lib.csa_lm_spans_u16_dev(text.data_ptr() or None, n, int(separator), lo.data_ptr() or None, hi.data_ptr() or None,
                                              target.data_ptr() or None, work.data_ptr() if size else None, size, stream))
    return lo, hi, target


# ---- attention ----


def _walkable(x):
    """x (tokens, heads, dim) as the kernels can read it: itself, or a copy where its strides or its address do not allow 16-byte loads."""
    fine = (x.stride(2) == 1 or x.shape[2] == 1) and x.data_ptr() % 16 == 0
    for size, stride in ((x.shape[0], x.stride(0)), (x.shape[1], x.stride(1))):
        fine = fine and (size <= 1 or stride % 8 == 0)
    if x.shape[0] > 1:
        fine = fine and x.shape[2] <= x.stride(0) < 1 << 22
    import torch
    return x if fine else x.clone(memory_format=torch.contiguous_format)


def _heads(x):
    """Strides of axes of length one mean nothing, and are named as a dense array's."""
    token = x.stride(0) if x.shape[0] > 1 else x.shape[1] * x.shape[2]
    head = x.stride(1) if x.shape[1] > 1 else x.shape[2]
    return native.CsaLmHeads(x.data_ptr() or None, max(token, x.shape[2]), head)


def _describe(q, k, v, lo, hi, scale, cap, slopes):
    import torch
    _check(q.dim() == 3 and k.dim() == 3 and v.dim() == 3, "q, k, v: (tokens, heads, head_dim)")
    _check(q.dtype == k.dtype == v.dtype, "q, k and v have to be of one type")
    _check(k.shape == v.shape, "k and v have to be of one shape")
    tokens, heads, dim = q.shape
    _check(k.shape[0] == tokens and k.shape[2] == dim, "q and k have to agree in tokens and head_dim")
    _check(k.shape[1] > 0 and heads > 0 and heads % k.shape[1] == 0, "the heads of q have to be a multiple of those of k and v")
    _check(8 <= dim <= 128 and dim % 8 == 0, "head_dim has to be a multiple of 8 from 8 to 128")
    for name, span in (("lo", lo), ("hi", hi)):
        _check(span is None or (span.dtype == torch.int32 and span.shape == (tokens,) and span.is_contiguous()), f"{name}: one int32 a token")
    _check(slopes is None or (slopes.dtype == torch.float32 and slopes.shape == (heads,) and slopes.is_contiguous()), "slopes: one float32 a head of q")
    scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    _check(0 < scale < 3e38 and 0 <= cap < 3e38, "scale has to be positive and finite, cap positive or 0")
    q, k, v = _walkable(q), _walkable(k), _walkable(v)
    pointer = lambda t: t.data_ptr() or None if t is not None else None  # noqa: E731
    a = native.CsaLmAttention(_matrix_type(q.dtype), heads, k.shape[1], dim, tokens, pointer(lo), pointer(hi), pointer(slopes), scale, float(cap),
                              _heads(q), _heads(k), _heads(v))
    device = _on_gpu([t for t in (q, k, v, lo, hi, slopes) if t is not None])
    return a, device, (q, k, v)


def span_attention(q, k, v, lo=None, hi=None, scale=None, cap=0.0, slopes=None):
    """Softmax attention of every token over its own span of keys.

    q: (tokens, heads, head_dim), k and v: (tokens, kv_heads, head_dim), bfloat16 or float16, in any strides (copied first where
    16-byte loads cannot walk them); heads is a multiple of kv_heads, and consecutive heads share one of k and v.
    lo, hi: int32, row i sees the keys [lo[i], hi[i]) (None: 0 and i + 1); a row may see none. scale: of the products
    (None: 1 / sqrt(head_dim)); cap: scores become cap * tanh(score / cap) (0: they stay); slopes: float32 of each head, slopes[h] * |i - j|
    is taken off the score of row i and key j.
    Returns (out of q's shape, lse float32 (heads, tokens)); rows that see nothing are zeros with lse -inf (csa_lm_attention_forward_dev)."""
    import torch
    a, device, keep = _describe(q, k, v, lo, hi, scale, cap, slopes)
    out = torch.empty(q.shape, dtype=q.dtype, device=device)
    lse = torch.empty((q.shape[1], q.shape[0]), dtype=torch.float32, device=device)
    if q.shape[0]:
        lib = native.load()
        size = lib.csa_lm_attention_workspace(q.shape[0], q.shape[1], k.shape[1], q.shape[2], 0)
        work = _work(size, device)
        with _Call(device) as stream:
            native.check(lib.csa_lm_attention_forward_dev(C.byref(a), _heads(out), lse.data_ptr(), work.data_ptr(), size, stream))
    return out, lse


def span_attention_backward(d_out, q, k, v, out, lse, lo=None, hi=None, scale=None, cap=0.0, slopes=None):
    """Gradients (d_q, d_k, d_v) for the gradient d_out of out; out and lse as span_attention returned them, the rest as it was given
    (csa_lm_attention_backward_dev). Sums run in a fixed order: the same inputs give the same bits."""
    import torch
    a, device, keep = _describe(q, k, v, lo, hi, scale, cap, slopes)
    _check(out.shape == q.shape and d_out.shape == q.shape and out.dtype == q.dtype and d_out.dtype == q.dtype, "out and d_out have to be like q")
    _check(lse.shape == (q.shape[1], q.shape[0]) and lse.dtype == torch.float32 and lse.is_contiguous(), "lse: float32 (heads, tokens)")
    _on_gpu([q, out, d_out, lse])
    out, d_out = _walkable(out), _walkable(d_out)
    d_q, d_k, d_v = (torch.empty(x.shape, dtype=q.dtype, device=device) for x in (q, k, v))
    if q.shape[0]:
        lib = native.load()
        size = lib.csa_lm_attention_workspace(q.shape[0], q.shape[1], k.shape[1], q.shape[2], native.CSA_LM_BACKWARD)
        work = _work(size, device)
        with _Call(device) as stream:
            native.check(lib.csa_lm_attention_backward_dev(C.byref(a), _heads(out), lse.data_ptr(), _heads(d_out), _heads(d_q), _heads(d_k), _heads(d_v),
                                                           work.data_ptr(), size, stream))
    return d_q, d_k, d_v


# ---- cross entropy ----


def _rows(x):
    """x (rows, dim) with its values side by side, and the distance of its rows."""
    if not ((x.stride(1) == 1 or x.shape[1] == 1) and (x.shape[0] <= 1 or x.shape[1] <= x.stride(0) < 1 << 22)):
        x = x.contiguous()
    return x, x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _entropy_work(lib, device, hidden, hs, weight, ws, flags):
    if hidden.data_ptr() % 16 or weight.data_ptr() % 16 or hs % 8 or ws % 8:
        flags |= native.CSA_LM_COPY_ROWS
    size = lib.csa_lm_cross_entropy_workspace(hidden.shape[0], hidden.shape[1], weight.shape[0], flags)
    return _work(size, device), size


def _check_entropy(hidden, weight, target):
    import torch
    _check(hidden.dim() == 2 and weight.dim() == 2 and hidden.shape[1] == weight.shape[1], "hidden: (tokens, dim), weight: (vocabulary, dim)")
    _check(hidden.dtype == weight.dtype, "hidden and weight have to be of one type")
    _check(weight.shape[0] > 0 and weight.shape[1] > 0, "weight has to hold something")
    _check(target.shape == (hidden.shape[0],) and target.dtype == torch.int32 and target.is_contiguous(), "target: one int32 a token")
    return _matrix_type(hidden.dtype)


def linear_cross_entropy(hidden, weight, target):
    """The cross entropy of softmax(hidden @ weight.T) and the targets, without keeping the logits.

    hidden: (tokens, dim), weight: (vocabulary, dim), bfloat16 or float16; target: int32, a token outside [0, vocabulary) has no loss.
    Returns float32 (loss, lse) of each token: lse is the logarithm of the sum of exponentials of its logits
    (csa_lm_cross_entropy_forward_dev)."""
    import torch
    kind = _check_entropy(hidden, weight, target)
    device = _on_gpu([hidden, weight, target])
    n, dim = hidden.shape
    loss, lse = (torch.empty(n, dtype=torch.float32, device=device) for _ in range(2))
    if n:
        lib = native.load()
        (hidden, hs), (weight, ws) = _rows(hidden), _rows(weight)
        work, size = _entropy_work(lib, device, hidden, hs, weight, ws, 0)
        with _Call(device) as stream:
            native.check(lib.csa_lm_cross_entropy_forward_dev(kind, hidden.data_ptr(), hs, weight.data_ptr(), ws, target.data_ptr(), n, dim, weight.shape[0],
                                                              loss.data_ptr(), lse.data_ptr(), work.data_ptr(), size, stream))
    return loss, lse


def linear_cross_entropy_backward(d_loss, hidden, weight, target, lse, want_hidden=True, want_weight=True):
    """Gradients (d_hidden, d_weight), of hidden's type, for the gradient d_loss (float32, one a token) of the losses; lse as
    linear_cross_entropy returned it (csa_lm_cross_entropy_backward_dev). A gradient that is not wanted is None."""
    import torch
    kind = _check_entropy(hidden, weight, target)
    device = _on_gpu([hidden, weight, target, d_loss, lse])
    n, dim = hidden.shape
    for name, x in (("d_loss", d_loss), ("lse", lse)):
        _check(x.shape == (n,) and x.dtype == torch.float32 and x.is_contiguous(), f"{name}: one float32 a token")
    d_hidden = torch.empty((n, dim), dtype=hidden.dtype, device=device) if want_hidden else None
    d_weight = torch.empty(weight.shape, dtype=weight.dtype, device=device) if want_weight else None
    lib = native.load()
    (hidden, hs), (weight, ws) = _rows(hidden), _rows(weight)
    work, size = _entropy_work(lib, device, hidden, hs, weight, ws, native.CSA_LM_BACKWARD)
    with _Call(device) as stream:
        native.check(lib.csa_lm_cross_entropy_backward_dev(kind, hidden.data_ptr() or None, hs, weight.data_ptr(), ws, target.data_ptr() or None,
                                                           lse.data_ptr() or None, d_loss.data_ptr() or None, n, dim, weight.shape[0],
                                                           (d_hidden.data_ptr() or None) if want_hidden else None, dim,
                                                           d_weight.data_ptr() if want_weight else None, dim, work.data_ptr(), size, stream))
    return d_hidden, d_weight


# ---- clipping ----


def clip_gradients(grads, max_norm, out=None):
    """Scales the gradients (a list of dense tensors, float32, bfloat16 or float16, mixed as they come) by min(1, max_norm / norm), where norm is the
    square root of the sum of all their squares, in place or into `out`, a list of tensors like them. Returns norm, a float32 tensor
    of no dimensions; where it is not finite the values stay as they are (csa_lm_clip_dev)."""
    import torch
    grads = list(grads)
    out = grads if out is None else list(out)
    _check(len(grads) > 0, "no gradients")
    _check(len(out) == len(grads), "out: a tensor for each gradient")
    _check(max_norm >= 0, "max_norm is negative or no number")
    for g, o in zip(grads, out):
        _check(g.is_contiguous() and o.is_contiguous() and g.shape == o.shape and g.dtype == o.dtype, "gradients and out: dense tensors, alike one by one")
    device = _on_gpu(grads + (out if out is not grads else []))
    lib = native.load()
    items = (native.CsaLmValues * len(grads))()
    for item, g, o in zip(items, grads, out):
        item.inp, item.out, item.n, item.type = g.data_ptr() or None, o.data_ptr() or None, g.numel(), _type(g.dtype)
    norm = torch.empty((), dtype=torch.float32, device=device)
    size = lib.csa_lm_clip_workspace(len(grads))
    work = _work(size, device)
    with _Call(device) as stream:
        native.check(lib.csa_lm_clip_dev(items, len(grads), float(max_norm), norm.data_ptr(), work.data_ptr(), size, stream))
    return norm


# ---- for torch.autograd ----


def attend(q, k, v, lo=None, hi=None, scale=None, cap=0.0, slopes=None):
    """span_attention's out, differentiable in q, k and v."""
    return _functions()[0].apply(q, k, v, lo, hi, scale, cap, slopes)


def next_token_loss(hidden, weight, target):
    """linear_cross_entropy's loss of every token, differentiable in hidden and weight."""
    return _functions()[1].apply(hidden, weight, target)


_made = None


def _functions():
    """The two torch.autograd functions, made when first asked for: this package imports torch only where it is used."""
    global _made
    if _made is not None:
        return _made
    import torch

    class Attend(torch.autograd.Function):
        @staticmethod
        def forward(ctx, q, k, v, lo, hi, scale, cap, slopes):
            out, lse = span_attention(q, k, v, lo, hi, scale, cap, slopes)
            ctx.save_for_backward(q, k, v, lo, hi, slopes, out, lse)
            ctx.how = (scale, cap)
            return out

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, d_out):
            q, k, v, lo, hi, slopes, out, lse = ctx.saved_tensors
            scale, cap = ctx.how
            return (*span_attention_backward(d_out, q, k, v, out, lse, lo, hi, scale, cap, slopes), None, None, None, None, None)

    class NextTokenLoss(torch.autograd.Function):
        @staticmethod
        def forward(ctx, hidden, weight, target):
            loss, lse = linear_cross_entropy(hidden, weight, target)
            ctx.save_for_backward(hidden, weight, target, lse)
            return loss

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, d_loss):
            hidden, weight, target, lse = ctx.saved_tensors
            want = ctx.needs_input_grad
            d_hidden, d_weight = linear_cross_entropy_backward(d_loss.contiguous(), hidden, weight, target, lse, want[0], want[1])
            return d_hidden, d_weight, None

    _made = (Attend, NextTokenLoss)
    return _made
