"""Operators of a language model over the texts that this package sorts: uint16 tokens, a separator in front of every document.

  token_spans                        the keys that each position of a text may see, and the token it has to predict
  embed_tokens (+ _backward)         the rows of a weight for the tokens of a text, and the gradient of the weight
  residual_norm (+ _backward)        the addition of a residual and the root-mean-square norm of the sum
  span_attention (+ _backward)       attention of every position over its span of keys
  linear_cross_entropy (+ _backward) the loss of every target over the whole vocabulary, without keeping the logits
  linear_distillation (+ _backward)  the divergence of that softmax from a teacher's over the logits that it kept
  clip_gradients                     the global norm of many gradients, and their clipping
  embed, add_norm, attend, next_token_loss, distillation_loss   the middle ones for torch.autograd

All take torch tensors on the GPU, enqueue kernels on the current stream of the tensors' device and return without waiting
(include/cascade_lm.h; there is no CPU form). Scratch memory comes from torch's allocator and belongs to the stream.
Only the latter are recorded by torch.autograd: the results of the others carry no graph, whatever their inputs want.
Probabilities and the gradients of scores and logits are rounded to 16 bits on their way into the second products (include/cascade_lm.h has the errors).
"""
import array
import ctypes as C
import math

from . import _native_lm as native

SEPARATOR = 0xFFFF


# What the calls need of torch, looked up when the first tensor comes: this package imports torch only where it is used, and looking it up in every call costs a small one
# 0.5 us of 8.
_kinds = None  # the library's number of every dtype
_float32 = _int32 = _raw_stream = _current_device = None


def _look_up():
    global _kinds, _float32, _int32, _raw_stream, _current_device
    import torch
    _float32, _int32 = torch.float32, torch.int32
    _raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice  # a stream's address, without the object around it
    _kinds = {torch.bfloat16: native.CSA_LM_BF16, torch.float16: native.CSA_LM_F16, torch.float32: native.CSA_LM_F32}


def _type(dtype):
    if _kinds is None:
        _look_up()
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
    """call(*args, stream) with the device's current stream, and the device made current for the launches."""
    if _kinds is None:
        _look_up()
    stream = _raw_stream(device) or None
    if device == _current_device():
        status = call(*args, stream)
    else:
        import torch
        with torch.cuda.device(device):
            status = call(*args, stream)
    if status:
        native.check(status)


def _work(size, like):
    """`size` bytes of scratch memory beside the tensor `like`, and their address; none where size is 0."""
    if not size:
        return None, None
    import torch
    work = like.new_empty(size, dtype=torch.uint8)
    return work, work.data_ptr()


def _address(x):
    return (x.data_ptr() or None) if x is not None else None


def _rows(x):
    """x (rows, dim) with its values side by side, and the distance of its rows."""
    if not ((x.stride(1) == 1 or x.shape[1] == 1) and (x.shape[0] <= 1 or x.shape[1] <= x.stride(0) < 1 << 22)):
        x = x.contiguous()
    return x, x.stride(0) if x.shape[0] > 1 else x.shape[1]


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


# ---- embeddings ----


def _check_tokens(tokens):
    """The bytes of a token."""
    if _kinds is None:
        _look_up()
    size = tokens.element_size()
    _check(tokens.dim() == 1 and tokens.is_contiguous() and (tokens.dtype == _int32 or (size == 2 and not tokens.is_floating_point())),
           "tokens: a dense vector of int32 or 16-bit tokens")
    return size


def embed_tokens(tokens, weight, scale=1.0):
    """scale * weight[tokens], rounded once: (n, dim) of weight's type. tokens: n int32, or 16-bit tokens as token_spans takes them (viewed as int16 is fine: they count as
    unsigned); weight: (rows, dim), float32, bfloat16 or float16, dim at least 8. A token outside [0, rows) gives zeros (csa_lm_embed_forward_dev).
    Without a graph: embed is the one for torch.autograd."""
    size = _check_tokens(tokens)
    _check(weight.dim() == 2, "weight: (rows, dim)")
    kind, device = _type(weight.dtype), _on_gpu(tokens, weight)
    n, (rows, dim) = tokens.numel(), weight.shape
    weight, stride = _rows(weight)
    out = weight.new_empty((n, dim))
    lib = native.load()
    _enqueue(device, lib.csa_lm_embed_forward_dev, kind, _address(tokens), size, n, _address(weight), stride, rows, dim, float(scale), _address(out))
    return out


def embed_tokens_backward(d_out, tokens, rows, scale=1.0):
    """The gradient of the weight, (rows, dim) of d_out's type, for the gradient d_out (n, dim) of embed_tokens' result: the rows of d_out that belong to each word, added up in 32
    bits in a fixed order, times scale; zeros for words that are not there (csa_lm_embed_backward_dev)."""
    token_size = _check_tokens(tokens)
    _check(d_out.dim() == 2 and d_out.shape[0] == tokens.numel(), "d_out: (tokens, dim)")
    kind, device = _type(d_out.dtype), _on_gpu(d_out, tokens)
    n, dim = d_out.shape
    d_out, stride = _rows(d_out)
    d_weight = d_out.new_empty((rows, dim))
    lib = native.load()
    size = lib.csa_lm_embed_backward_workspace(kind, n, rows, dim)
    scratch, work = _work(size, d_out)
    _enqueue(device, lib.csa_lm_embed_backward_dev, kind, _address(tokens), token_size, n, _address(d_out), stride, rows, dim, float(scale),
             _address(d_weight), work, size)
    return d_weight


# ---- norms ----


def _check_norm(x, gain):
    """The type, and the numbers of rows and of their values."""
    _check(x.dim() == 2, "rows: (tokens, dim)")
    dtype, (n, dim) = x.dtype, x.shape
    _check(gain is None or (gain.dtype == dtype and gain.dim() == 1 and gain.numel() == dim and gain.is_contiguous()), "gain: a value of x's type for each of a row")
    return _type(dtype), n, dim


def _check_stream(x, like, message):
    _check(x.shape == like.shape and (x.dtype == like.dtype or x.dtype == _float32), message)
    return _type(x.dtype)


def residual_norm(x, residual=None, gain=None, eps=1e-6):
    """The root-mean-square norm of x + residual.

    x: (tokens, dim), float32, bfloat16 or float16, dim from 8 to 16384; residual: like x, or a stream of 32 bits beside an x of 16; gain: dim values of x's type (None: ones).
    Returns (out, total, rstd): total = x + residual in the residual's type (x itself without one), rstd = 1 / sqrt(mean of total^2 + eps) float32 of every token, and out =
    total * rstd * gain in x's type, from the rounded total (csa_lm_norm_forward_dev). Without a graph: add_norm is the one for torch.autograd."""
    kind, n, dim = _check_norm(x, gain)
    stream = kind if residual is None else _check_stream(residual, x, "residual: like x, or in float32")
    device = _on_gpu(x, residual, gain)
    out, rstd = x.new_empty((n, dim)), x.new_empty(n, dtype=_float32)
    total = x if residual is None else residual.new_empty((n, dim))
    x, xs = _rows(x)
    residual, rs = (None, 0) if residual is None else _rows(residual)
    lib = native.load()
    _enqueue(device, lib.csa_lm_norm_forward_dev, kind, stream, _address(x), xs, _address(residual), rs, _address(gain), float(eps), n, dim, _address(out),
             None if residual is None else _address(total), _address(rstd))
    return out, total, rstd


def residual_norm_backward(d_out, total, rstd, gain=None, d_total=None, want_gain=True):
    """Gradients (d_x, d_residual, d_gain) for the gradients d_out of out and d_total of total (None: total is used nowhere else); total and rstd as residual_norm returned them.
    d_x is of d_out's type and d_residual of total's: one tensor where these are the same. d_gain is None without a gain, or if it is not wanted (csa_lm_norm_backward_dev)."""
    kind, n, dim = _check_norm(d_out, gain)
    stream = _check_stream(total, d_out, "total: like d_out, or in float32")
    _check(d_total is None or (d_total.shape == total.shape and d_total.dtype == total.dtype), "d_total: like total")
    device = _on_gpu(d_out, total, rstd, gain, d_total)
    _check(rstd.dim() == 1 and rstd.numel() == n and rstd.dtype == _float32 and rstd.is_contiguous(), "rstd: one float32 a token")
    d_residual = total.new_empty((n, dim))
    d_x = d_residual if stream == kind else d_out.new_empty((n, dim))
    d_gain = gain.new_empty(dim) if gain is not None and want_gain else None
    (d_out, gs), (total, ts) = _rows(d_out), _rows(total)
    d_total, ds = (None, 0) if d_total is None else _rows(d_total)
    lib = native.load()
    size = lib.csa_lm_norm_backward_workspace(n, dim) if d_gain is not None else 0
    scratch, work = _work(size, d_out)
    _enqueue(device, lib.csa_lm_norm_backward_dev, kind, stream, _address(d_out), gs, _address(total), ts, _address(rstd), _address(gain), _address(d_total), ds, n, dim,
             None if stream == kind else _address(d_x), _address(d_residual), _address(d_gain), work, size)
    return d_x, d_residual, d_gain


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


def _entropy_work(lib, hidden, hs, weight, ws, flags, kept=None):
    """The workspace of the cross entropy, or of the distillation from `kept` logits a token."""
    if hidden.data_ptr() % 16 or weight.data_ptr() % 16 or hs % 8 or ws % 8:
        flags |= native.CSA_LM_COPY_ROWS
    n, dim, vocab = *hidden.shape, weight.shape[0]
    size = lib.csa_lm_cross_entropy_workspace(n, dim, vocab, flags) if kept is None else lib.csa_lm_distill_workspace(n, dim, vocab, kept, flags)
    return (size, *_work(size, hidden))


def _check_linear(hidden, weight):
    _check(hidden.dim() == 2 and weight.dim() == 2 and hidden.shape[1] == weight.shape[1], "hidden: (tokens, dim), weight: (vocabulary, dim)")
    _check(hidden.dtype == weight.dtype, "hidden and weight have to be of one type")
    _check(weight.numel() > 0, "weight has to hold something")
    return _matrix_type(hidden.dtype)


def _check_entropy(hidden, weight, target):
    import torch
    kind = _check_linear(hidden, weight)
    _check(target.dim() == 1 and target.numel() == hidden.shape[0] and target.dtype == torch.int32 and target.is_contiguous(), "target: one int32 a token")
    return kind


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


# ---- distillation ----


def _check_teacher(hidden, ids, logits):
    """The number of logits kept of a token, and the logits in 32 bits."""
    import torch
    _check(ids.dim() == 2 and ids.shape[0] == hidden.shape[0] and ids.dtype == torch.int32 and ids.is_contiguous(), "ids: int32 (tokens, kept)")
    _check(logits.shape == ids.shape and logits.is_contiguous(), "logits: as many as ids")
    _type(logits.dtype)
    return ids.shape[1], logits.float()


def linear_distillation(hidden, weight, ids, logits, temperature=1.0):
    """The divergence of softmax(hidden @ weight.T / temperature) from a teacher's softmax over the logits that it kept of every token, without keeping the student's logits.

    hidden: (tokens, dim), weight: (vocabulary, dim), bfloat16 or float16; ids: int32 (tokens, kept), words in any order; logits: the teacher's, as many, float32, bfloat16 or
    float16. An id outside [0, vocabulary) or a logit of -infinity is no entry; a token without entries has no loss. With q the softmax of a token's logits / temperature over its entries
    and z its own, the loss is the sum of q (ln q - ln softmax(z)): what an entire teacher would leave out is not counted. (A loss that is to weigh like a cross entropy is taken
    times temperature squared.) Returns float32 (loss, lse) of each token: lse is the logarithm of the sum of exponentials of z (csa_lm_distill_forward_dev). Without a
    graph: distillation_loss is the one for torch.autograd."""
    import torch
    kind = _check_linear(hidden, weight)
    kept, logits = _check_teacher(hidden, ids, logits)
    device = _on_gpu(hidden, weight, ids, logits)
    n, dim = hidden.shape
    loss, lse = hidden.new_empty(n, dtype=torch.float32), hidden.new_empty(n, dtype=torch.float32)
    lib = native.load()
    (hidden, hs), (weight, ws) = _rows(hidden), _rows(weight)
    size, scratch, work = _entropy_work(lib, hidden, hs, weight, ws, 0, kept)
    _enqueue(device, lib.csa_lm_distill_forward_dev, kind, _address(hidden), hs, weight.data_ptr(), ws, _address(ids), _address(logits), kept, float(temperature), n, dim,
             weight.shape[0], _address(loss), _address(lse), work, size)
    return loss, lse


def linear_distillation_backward(d_loss, hidden, weight, ids, logits, lse, temperature=1.0, want_hidden=True, want_weight=True):
    """Gradients (d_hidden, d_weight), of hidden's type, for the gradient d_loss (float32, one a token) of the losses; lse as linear_distillation returned it
    (csa_lm_distill_backward_dev). A gradient that is not wanted is None; the teacher's logits have none. Gradients of logits are operands of the matrix units, which take 16 bits: calls of more than 64
    tokens come out with about 1.4 times the error of the result's own rounding, those of up to 32 tokens with that alone."""
    import torch
    kind = _check_linear(hidden, weight)
    kept, logits = _check_teacher(hidden, ids, logits)
    device = _on_gpu(hidden, weight, ids, logits, d_loss, lse)
    n, dim = hidden.shape
    for x in (d_loss, lse):
        _check(x.dim() == 1 and x.numel() == n and x.dtype == torch.float32 and x.is_contiguous(), "d_loss, lse: one float32 a token")
    d_hidden = hidden.new_empty((n, dim)) if want_hidden else None
    d_weight = weight.new_empty(weight.shape) if want_weight else None
    lib = native.load()
    (hidden, hs), (weight, ws) = _rows(hidden), _rows(weight)
    size, scratch, work = _entropy_work(lib, hidden, hs, weight, ws, native.CSA_LM_BACKWARD, kept)
    _enqueue(device, lib.csa_lm_distill_backward_dev, kind, _address(hidden), hs, weight.data_ptr(), ws, _address(ids), _address(logits), kept, float(temperature),
             _address(lse), _address(d_loss), n, dim, weight.shape[0], _address(d_hidden), dim, _address(d_weight), dim, work, size)
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


def embed(tokens, weight, scale=1.0):
    """embed_tokens, differentiable in weight."""
    return _functions()[2].apply(tokens, weight, scale)


def add_norm(x, residual=None, gain=None, eps=1e-6):
    """residual_norm's (out, total), differentiable in x, residual and gain. Without a residual total is x."""
    if residual is None:
        return _functions()[3].apply(x, None, gain, eps), x
    return _functions()[3].apply(x, residual, gain, eps)


def attend(q, k, v, lo=None, hi=None, scale=None, cap=0.0, slopes=None):
    """span_attention's out, differentiable in q, k and v (slopes are constants: ones that want a gradient are refused)."""
    _check(slopes is None or not slopes.requires_grad, "slopes have no gradient here: detach them")
    return _functions()[0].apply(q, k, v, lo, hi, scale, cap, slopes)


def next_token_loss(hidden, weight, target):
    """linear_cross_entropy's loss of every token, differentiable in hidden and weight."""
    return _functions()[1].apply(hidden, weight, target)


def distillation_loss(hidden, weight, ids, logits, temperature=1.0):
    """linear_distillation's loss of every token, differentiable in hidden and weight (the teacher is a constant: logits that want a gradient are refused)."""
    _check(not logits.requires_grad, "the teacher's logits have no gradient here: detach them")
    return _functions()[4].apply(hidden, weight, ids, logits, temperature)


_made = None


def _functions():
    """The torch.autograd functions, made when first asked for: this package imports torch only where it is used."""
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

    class Embed(torch.autograd.Function):
        @staticmethod
        def forward(ctx, tokens, weight, scale):
            ctx.save_for_backward(tokens)
            ctx.how = (weight.shape[0], scale)
            return embed_tokens(tokens, weight, scale)

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, d_out):
            rows, scale = ctx.how
            return None, embed_tokens_backward(d_out, *ctx.saved_tensors, rows, scale), None

    class AddNorm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, residual, gain, eps):
            out, total, rstd = residual_norm(x, residual, gain, eps)
            ctx.set_materialize_grads(False)
            ctx.save_for_backward(total, rstd, gain)
            ctx.x_type = x.dtype
            return out if residual is None else (out, total)

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, d_out, d_total=None):
            total, rstd, gain = ctx.saved_tensors
            if d_out is None and d_total is None:
                return None, None, None, None
            want_x, want_residual, want_gain, _ = ctx.needs_input_grad
            if d_out is None:  # only total is used
                d_x, d_residual, d_gain = d_total.to(ctx.x_type), d_total, None
            else:
                d_x, d_residual, d_gain = residual_norm_backward(d_out, total, rstd, gain, d_total, want_gain)
            return d_x if want_x else None, d_residual if want_residual else None, d_gain, None

    class Distillation(torch.autograd.Function):
        @staticmethod
        def forward(ctx, hidden, weight, ids, logits, temperature):
            loss, lse = linear_distillation(hidden, weight, ids, logits, temperature)
            ctx.save_for_backward(hidden, weight, ids, logits, lse)
            ctx.temperature = temperature
            return loss

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, d_loss):
            want = ctx.needs_input_grad
            d_hidden, d_weight = linear_distillation_backward(d_loss.contiguous(), *ctx.saved_tensors, ctx.temperature, want[0], want[1])
            return d_hidden, d_weight, None, None, None

    _made = (Attend, NextTokenLoss, Embed, AddNorm, Distillation)
    return _made
