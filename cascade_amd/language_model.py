"""Operators of a language model over the texts that this package sorts: uint16 tokens, a separator in front of every document.

  token_spans                        the keys that each position of a text may see, and the token it has to predict
  span_attention (+ _backward)       attention of every position over its span of keys
  linear_cross_entropy (+ _backward) the loss of every target over the whole vocabulary, without keeping the logits
  clip_gradients                     the global norm of many gradients, and their clipping
  attend, next_token_loss            the middle two for torch.autograd

All take torch tensors on the GPU, enqueue kernels on the current stream of the tensors' device and return without waiting
(include/cascade_lm.h; there is no CPU form). Scratch memory comes from torch's allocator and belongs to the stream.
Only attend and next_token_loss are recorded by torch.autograd: the results of the others carry no graph, whatever their inputs want.
Probabilities and the gradients of scores and logits are rounded to 16 bits on their way into the second products (include/cascade_lm.h has the errors).
"""
import array
import ctypes as C
import math

from . import _native_lm as native

SEPARATOR = 0xFFFF


_kinds = None  # the library's number of every dtype; made when first asked for: this package imports torch only where it is used


def _type(dtype):
    global _kinds
    if _kinds is None:
        import torch
        _kinds = {torch.bfloat16: native.CSA_LM_BF16, torch.float16: native.CSA_LM_F16, torch.float32: native.CSA_LM_F32}
    kind = _kinds.get(dtype)
    if kind is None:
        raise TypeError(f"{dtype} is none of bfloat16, float16 and float32")
    return kind


def _matrix_type(dtype):
    kind = _type(dtype)
    if kind == native.CSA_LM_F32:
        raise TypeError("the matrix products take bfloat16 or float16")
    return kind


def _check(condition, message):
    if not condition:
        raise ValueError(message)


def _on_gpu(*tensors):
    """The number of the device that all of them (None aside) lie on, which has to be a GPU."""
    device = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != device:
            device = -1
    _check(device >= 0, "all tensors have to lie on one GPU")
    return device


def _enqueue(device, call, *args):
    """call(*args, stream) with the device's current stream, and the device made current for the launches. (The stream's address without
    the object that torch.cuda.current_stream makes around it: 0.1 us instead of 1.2, of the 11 that a small call takes.)"""
    import torch
    stream = torch._C._cuda_getCurrentRawStream(device) or None
    if device == torch.cuda.current_device():
        native.check(call(*args, stream))
    else:
        with torch.cuda.device(device):
            native.check(call(*args, stream))


def _work(size, like):
    """`size` bytes of scratch memory beside the tensor `like`, and their address; none where size is 0."""
    if not size:
        return None, None
    import torch
    work = like.new_empty(size, dtype=torch.uint8)
    return work, work.data_ptr()


def _address(x):
    return (x.data_ptr() or None) if x is not None else None


def token_spans(text, separator=SEPARATOR):
    """text: n uint16 tokens (viewed as int16 is fine), one stretch of a corpus. Returns int32 tensors (lo, hi, target) of n values:
    position i may see the keys [lo[i], hi[i]), which begin at the last separator at or before i and end with i itself, and has to
    predict target[i], the token behind it, or nothing (-1) at the end and in front of a separator (csa_lm_spans_u16_dev)."""
    import torch
    device = _on_gpu(text)
    _check(text.dim() == 1 and text.element_size() == 2 and not text.is_floating_point() and text.is_contiguous(), "text: a dense vector of 16-bit tokens")
    _check(0 <= separator <= 0xFFFF, "separator: a 16-bit token")
    lib, n = native.load(), text.numel()
    lo, hi, target = (text.new_empty(n, dtype=torch.int32) for _ in range(3))
    size = lib.csa_lm_spans_workspace(n)
    keep, work = _work(size, text)
    _enqueue(device, lib.csa_lm_spans_u16_dev, _address(text), n, int(separator), _address(lo), _address(hi), _address(target), work, size)
    return lo, hi, target


# ---- attention ----


def _walkable(x):
    """x (tokens, heads, dim) as the kernels can read it, and its address and strides: itself, or a copy where its strides or its address do not
    allow 16-byte loads. Strides of axes of length one mean nothing, and are named as a dense array's."""
    tokens, heads, dim = x.shape
    token, head, one = x.stride()
    token, head = token if tokens > 1 else heads * dim, head if heads > 1 else dim
    if one != 1 or token % 8 or head % 8 or not dim <= token < 1 << 22 or head < 0 or x.data_ptr() % 16:
        import torch
        x = x.clone(memory_format=torch.contiguous_format)
        token, head = heads * dim, dim
    return x, native.CsaLmHeads(x.data_ptr() or None, token, head)


def _describe(q, k, v, lo, hi, scale, cap, slopes):
    """The call's description, the device, and what has to live until it is enqueued."""
    import torch
    _check(q.dim() == 3 and k.dim() == 3 and v.dim() == 3, "q, k, v: (tokens, heads, head_dim)")
    _check(q.dtype == k.dtype == v.dtype, "q, k and v have to be of one type")
    tokens, heads, dim = q.shape
    kv_heads = k.shape[1]
    _check(k.shape == v.shape, "k and v have to be of one shape")
    _check(k.shape[0] == tokens and k.shape[2] == dim, "q and k have to agree in tokens and head_dim")
    _check(kv_heads > 0 and heads > 0 and heads % kv_heads == 0, "the heads of q have to be a multiple of those of k and v")
    _check(8 <= dim <= 128 and dim % 8 == 0, "head_dim has to be a multiple of 8 from 8 to 128")
    for span in (lo, hi):
        if span is not None:
            _check(span.dtype == torch.int32 and span.dim() == 1 and span.numel() == tokens and span.is_contiguous(), "lo, hi: one int32 a token")
    if slopes is not None:
        _check(slopes.dtype == torch.float32 and slopes.dim() == 1 and slopes.numel() == heads and slopes.is_contiguous(), "slopes: one float32 a head of q")
    scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    _check(0 < scale < 3e38 and 0 <= cap < 3e38, "scale has to be positive and finite, cap positive or 0")
    kind = _matrix_type(q.dtype)
    device = _on_gpu(q, k, v, lo, hi, slopes)
    (q, qh), (k, kh), (v, vh) = _walkable(q), _walkable(k), _walkable(v)
    a = native.CsaLmAttention(kind, heads, kv_heads, dim, tokens, _address(lo), _address(hi), _address(slopes), scale, float(cap), qh, kh, vh)
    return a, device, (q, k, v)


def span_attention(q, k, v, lo=None, hi=None, scale=None, cap=0.0, slopes=None):
    """Softmax attention of every token over its own span of keys.

    q: (tokens, heads, head_dim), k and v: (tokens, kv_heads, head_dim), bfloat16 or float16, in any strides (copied first where
    16-byte loads cannot walk them); heads is a multiple of kv_heads, and consecutive heads share one of k and v.
    lo, hi: int32, row i sees the keys [lo[i], hi[i]) (None: 0 and i + 1); a row may see none. scale: of the products
    (None: 1 / sqrt(head_dim)); cap: scores become cap * tanh(score / cap) (0: they stay); slopes: float32 of each head, slopes[h] * |i - j|
    is taken off the score of row i and key j.
    Returns (out of q's shape, lse float32 (heads, tokens)); rows that see nothing are zeros with lse -inf. What a row may not see may hold anything,
    infinities and NaN too; what sees those may become infinite or NaN throughout (csa_lm_attention_forward_dev). Without a graph: attend is the one for torch.autograd."""
    import torch
    a, device, keep = _describe(q, k, v, lo, hi, scale, cap, slopes)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = q.new_empty((a.q_heads, a.tokens), dtype=torch.float32)
    if a.tokens:
        lib = native.load()
        size = lib.csa_lm_attention_workspace(a.tokens, a.q_heads, a.kv_heads, a.head_dim, 0)
        scratch, work = _work(size, q)
        _enqueue(device, lib.csa_lm_attention_forward_dev, C.byref(a), _walkable(out)[1], lse.data_ptr(), work, size)
    return out, lse


def span_attention_backward(d_out, q, k, v, out, lse, lo=None, hi=None, scale=None, cap=0.0, slopes=None):
    """Gradients (d_q, d_k, d_v) for the gradient d_out of out; out and lse as span_attention returned them, the rest as it was given
    (csa_lm_attention_backward_dev). Sums run in a fixed order: the same inputs give the same bits."""
    import torch
    a, device, keep = _describe(q, k, v, lo, hi, scale, cap, slopes)
    _check(out.shape == q.shape and d_out.shape == q.shape and out.dtype == q.dtype and d_out.dtype == q.dtype, "out and d_out have to be like q")
    _check(lse.shape == (a.q_heads, a.tokens) and lse.dtype == torch.float32 and lse.is_contiguous(), "lse: float32 (heads, tokens)")
    _on_gpu(q, out, d_out, lse)
    (out, oh), (d_out, gh) = _walkable(out), _walkable(d_out)
    d_q, d_k, d_v = (torch.empty_like(x, memory_format=torch.contiguous_format) for x in (q, k, v))
    if a.tokens:
        lib = native.load()
        size = lib.csa_lm_attention_workspace(a.tokens, a.q_heads, a.kv_heads, a.head_dim, native.CSA_LM_BACKWARD)
        scratch, work = _work(size, q)
        _enqueue(device, lib.csa_lm_attention_backward_dev, C.byref(a), oh, lse.data_ptr(), gh, _walkable(d_q)[1], _walkable(d_k)[1], _walkable(d_v)[1], work, size)
    return d_q, d_k, d_v


# ---- cross entropy ----


def _rows(x):
    """x (rows, dim) with its values side by side, and the distance of its rows."""
    if not ((x.stride(1) == 1 or x.shape[1] == 1) and (x.shape[0] <= 1 or x.shape[1] <= x.stride(0) < 1 << 22)):
        x = x.contiguous()
    return x, x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _entropy_work(lib, hidden, hs, weight, ws, flags):
    if hidden.data_ptr() % 16 or weight.data_ptr() % 16 or hs % 8 or ws % 8:
        flags |= native.CSA_LM_COPY_ROWS
    size = lib.csa_lm_cross_entropy_workspace(hidden.shape[0], hidden.shape[1], weight.shape[0], flags)
    return (size, *_work(size, hidden))


def _check_entropy(hidden, weight, target):
    import torch
    _check(hidden.dim() == 2 and weight.dim() == 2 and hidden.shape[1] == weight.shape[1], "hidden: (tokens, dim), weight: (vocabulary, dim)")
    _check(hidden.dtype == weight.dtype, "hidden and weight have to be of one type")
    _check(weight.numel() > 0, "weight has to hold something")
    _check(target.dim() == 1 and target.numel() == hidden.shape[0] and target.dtype == torch.int32 and target.is_contiguous(), "target: one int32 a token")
    return _matrix_type(hidden.dtype)


def linear_cross_entropy(hidden, weight, target):
    """The cross entropy of softmax(hidden @ weight.T) and the targets, without keeping the logits.

    hidden: (tokens, dim), weight: (vocabulary, dim), bfloat16 or float16; target: int32, a token outside [0, vocabulary) has no loss.
    Returns float32 (loss, lse) of each token: lse is the logarithm of the sum of exponentials of its logits
    (csa_lm_cross_entropy_forward_dev). Without a graph: next_token_loss is the one for torch.autograd."""
    import torch
    kind = _check_entropy(hidden, weight, target)
    device = _on_gpu(hidden, weight, target)
    n, dim = hidden.shape
    loss, lse = hidden.new_empty(n, dtype=torch.float32), hidden.new_empty(n, dtype=torch.float32)
    if n:
        lib = native.load()
        (hidden, hs), (weight, ws) = _rows(hidden), _rows(weight)
        size, scratch, work = _entropy_work(lib, hidden, hs, weight, ws, 0)
        _enqueue(device, lib.csa_lm_cross_entropy_forward_dev, kind, hidden.data_ptr(), hs, weight.data_ptr(), ws, target.data_ptr(), n, dim, weight.shape[0],
                 loss.data_ptr(), lse.data_ptr(), work, size)
    return loss, lse


def linear_cross_entropy_backward(d_loss, hidden, weight, target, lse, want_hidden=True, want_weight=True):
    """Gradients (d_hidden, d_weight), of hidden's type, for the gradient d_loss (float32, one a token) of the losses; lse as
    linear_cross_entropy returned it (csa_lm_cross_entropy_backward_dev). A gradient that is not wanted is None."""
    import torch
    kind = _check_entropy(hidden, weight, target)
    device = _on_gpu(hidden, weight, target, d_loss, lse)
    n, dim = hidden.shape
    for x in (d_loss, lse):
        _check(x.dim() == 1 and x.numel() == n and x.dtype == torch.float32 and x.is_contiguous(), "d_loss, lse: one float32 a token")
    d_hidden = hidden.new_empty((n, dim)) if want_hidden else None
    d_weight = weight.new_empty(weight.shape) if want_weight else None
    lib = native.load()
    (hidden, hs), (weight, ws) = _rows(hidden), _rows(weight)
    size, scratch, work = _entropy_work(lib, hidden, hs, weight, ws, native.CSA_LM_BACKWARD)
    _enqueue(device, lib.csa_lm_cross_entropy_backward_dev, kind, _address(hidden), hs, weight.data_ptr(), ws, _address(target), _address(lse), _address(d_loss), n,
             dim, weight.shape[0], _address(d_hidden), dim, _address(d_weight), dim, work, size)
    return d_hidden, d_weight


# ---- clipping ----


def clip_gradients(grads, max_norm, out=None):
    """Scales the gradients (a list of contiguous tensors, at least one, float32, bfloat16 or float16, mixed as they come) by min(1, max_norm / norm), where norm
    is the square root of the sum of all their squares, in place or into `out`, a list of tensors like them. No tensor may be written twice, or where another one is
    read. Returns norm, a float32 tensor of no dimensions; where it is not finite the values stay as they are (csa_lm_clip_dev)."""
    import torch
    grads = list(grads)
    out = grads if out is None else list(out)
    _check(len(grads) > 0, "no gradients")
    _check(len(out) == len(grads), "out: a tensor for each gradient")
    _check(max_norm >= 0, "max_norm is negative or no number")
    device = grads[0].get_device()
    _check(device >= 0, "the gradients have to lie on a GPU")
    items = []  # csa_lm_values as four 64-bit words each
    for g, o in zip(grads, out):
        if not g.is_contiguous() or g.get_device() != device:
            raise ValueError("gradients: contiguous tensors on one GPU")
        if o is not g and (o.dtype != g.dtype or o.shape != g.shape or not o.is_contiguous() or o.get_device() != device):
            raise ValueError("out: tensors like the gradients, one by one")
        items += (g.data_ptr(), o.data_ptr(), g.numel(), _type(g.dtype))
    items = array.array("Q", items)
    lib = native.load()
    norm = grads[0].new_empty((), dtype=torch.float32)
    size = lib.csa_lm_clip_workspace(len(grads))
    scratch, work = _work(size, norm)
    _enqueue(device, lib.csa_lm_clip_dev, items.buffer_info()[0], len(grads), float(max_norm), norm.data_ptr(), work, size)
    torch.autograd.graph.increment_version(out)  # they have changed: what autograd has saved of them is stale
    return norm


# ---- for torch.autograd ----


def attend(q, k, v, lo=None, hi=None, scale=None, cap=0.0, slopes=None):
    """span_attention's out, differentiable in q, k and v (slopes are constants: ones that want a gradient are refused)."""
    _check(slopes is None or not slopes.requires_grad, "slopes have no gradient here: detach them")
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
