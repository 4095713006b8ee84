"""Attention over batches of images and clips: what a model does with a batch once its patches are projected.

* ``rotary``: positions with several axes (time, row, column) turn queries and keys.
* ``qk_norm_rotary``: RMS norm of every head of queries and keys, and the rotation, in one pass.
* ``cross_attention``: queries read the states of images or clips, padding masked out.
* ``window_attention``: a text reads itself, every token those before it, or a window of them and a few first ones.
* ``append_rotary`` and ``cached_attention``: the same in generation, over keys and values in the pages of a cache.

All take torch tensors in GPU memory, ``[batch, tokens, heads, head_dim]`` (views of a joint projection too), and queue
their work on torch's current stream of the tensors' device; results are new contiguous tensors.  They work under
``torch.autograd`` (reverse mode, once; forward mode raises); the functions ``*_backward`` are the same gradients for programs
that do without it.  Sums are held in float32 and results rounded once to the tensors' type.  ``cross_attention`` also rounds what its
products on the tensor cores take, the weights P and in the backward pass dS = P (dP - delta), to the tensors' type, with delta from the
rounded result where keys are more than 128: errors of 1.4 to 1.6 roundings instead of one.  In float16 a dS beyond 65504 is infinite,
as a loss scaler expects of a scale that is too high.  ``cached_attention`` and ``window_attention`` round alike, the latter with delta from
the rounded result where the 128 rows of a tile (tokens times the query heads of a key head) read more than two tiles of 128 keys.  The
same call gives the same bits again.  Wrong arguments raise ``ValueError``; there is no CPU path.
"""
import importlib

__all__ = ["rotary", "qk_norm_rotary", "qk_norm_rotary_backward", "cross_attention", "cross_attention_backward", "window_attention",
           "window_attention_backward", "append_rotary", "cached_attention"]



class _Operators:
    """The compiled module, loaded on first use: importing the package does not import torch."""

    def __getattr__(self, name):
        global _ops
        importlib.import_module("torch")
        try:
            _ops = importlib.import_module("._attention", __package__)
        except ModuleNotFoundError as e:
            raise ImportError("the attention operators are missing: the package was built without torch; build it again") from e
        return getattr(_ops, name)


_ops = _Operators()
_functions = None


def _autograd():
    """The autograd functions, made on first use."""
    global _functions
    if _functions is None:
        import torch

        class Rotary(torch.autograd.Function):
            @staticmethod
            def forward(ctx, q, k, positions, frequencies, sections, inverse, adjacent, interleaved):
                out = _ops.rotary(q, k, positions, frequencies, sections, inverse, adjacent, interleaved)
                ctx.save_for_backward(positions, frequencies)
                ctx.how = (tuple(sections), not inverse, adjacent, interleaved)
                return out

            @staticmethod
            @torch.autograd.function.once_differentiable
            def backward(ctx, dq, dk):
                return (*_ops.rotary(dq, dk, *ctx.saved_tensors, *ctx.how), None, None, None, None, None, None)

        class QkNormRotary(torch.autograd.Function):
            @staticmethod
            def forward(ctx, q, k, positions, frequencies, sections, q_weight, k_weight, eps, adjacent, interleaved):
                out = _ops.qk_norm_rotary(q, k, positions, frequencies, sections, q_weight, k_weight, eps, adjacent, interleaved)
                ctx.save_for_backward(q, k, positions, frequencies, q_weight, k_weight)
                ctx.how = (tuple(sections), float(eps), adjacent, interleaved)
                return out

            @staticmethod
            @torch.autograd.function.once_differentiable
            def backward(ctx, dq, dk):
                q, k, positions, frequencies, q_weight, k_weight = ctx.saved_tensors
                sections, eps, adjacent, interleaved = ctx.how
                dq, dk, dwq, dwk = _ops.qk_norm_rotary_backward(
                    dq, dk, q, k, positions, frequencies, sections, q_weight, k_weight, eps, adjacent, interleaved)
                return dq, dk, None, None, None, dwq, dwk, None, None, None

        class CrossAttention(torch.autograd.Function):
            @staticmethod
            def forward(ctx, q, k, v, lengths, key_mask, scale):
                out, lse = _ops.cross_attention(q, k, v, lengths, key_mask, scale, True)
                ctx.save_for_backward(q, k, v, out, lse, lengths, key_mask)
                ctx.scale = None if scale is None else float(scale)
                ctx.set_materialize_grads(False)
                return out, lse

            @staticmethod
            @torch.autograd.function.once_differentiable
            def backward(ctx, dout, dlse):
                q, k, v, out, lse, lengths, key_mask = ctx.saved_tensors
                if dout is None:
                    dout = torch.zeros_like(out)
                return (*_ops.cross_attention_backward(dout, q, k, v, out, lse, lengths, key_mask, ctx.scale, dlse), None, None, None)

        class WindowAttention(torch.autograd.Function):
            @staticmethod
            def forward(ctx, q, k, v, window, sinks, lengths, scale):
                out, lse = _ops.window_attention(q, k, v, window, sinks, lengths, scale, True)
                ctx.save_for_backward(q, k, v, out, lse, lengths)
                ctx.how = (None if window is None else int(window), int(sinks), None if scale is None else float(scale))
                ctx.set_materialize_grads(False)
                return out, lse

            @staticmethod
            @torch.autograd.function.once_differentiable
            def backward(ctx, dout, dlse):
                q, k, v, out, lse, lengths = ctx.saved_tensors
                window, sinks, scale = ctx.how
                if dout is None:
                    dout = torch.zeros_like(out)
                return (*_ops.window_attention_backward(dout, q, k, v, out, lse, window, sinks, lengths, scale, dlse), None, None, None, None)

        _functions = Rotary, QkNormRotary, CrossAttention, WindowAttention
    return _functions


def _wants_gradient(*tensors):
    for t in tensors:
        if getattr(t, "requires_grad", False):
            return importlib.import_module("torch").is_grad_enabled()
    return False


def _constants(op, **tensors):
    """Refuses a gradient that would not be worked out, ahead of the autograd functions (the compiled module does so elsewhere)."""
    for name, t in tensors.items():
        if _wants_gradient(t):
            raise ValueError("%s: %s has no gradient here but requires one; pass %s.detach()" % (op, name, name))


def rotary(q, k, positions, frequencies, sections, *, inverse=False, adjacent=False, interleaved=False):
    """Turn queries and keys by positions on several axes; returns ``(q, k)`` turned.

    ``q`` [batch, tokens, q_heads, head_dim], ``k`` the same with its own number of heads, or None; float32, bfloat16 or
    float16; head_dim even, up to 256.  [tokens, heads, head_dim] is taken too.
    ``positions`` [axes, batch, tokens] int32, int64 or float32, one to four axes.
    ``frequencies`` [pairs] float32; ``sections`` the number of pairs of each axis.  Pairs go to the axes in order, or one
    to each axis in turn (``interleaved``).  Pair i turns by float32(position) * frequencies[i], the product rounded to float32.
    Pairs are elements (i, i + pairs), or (2 i, 2 i + 1) (``adjacent``); elements from 2 * pairs on stay as they are.
    ``inverse`` turns back, which is also the gradient.  Positions and frequencies have no gradient; ones that require it are
    refused.
    """
    if _wants_gradient(q, k):
        _constants("rotary", positions=positions, frequencies=frequencies)
        return _autograd()[0].apply(q, k, positions, frequencies, sections, inverse, adjacent, interleaved)
    return _ops.rotary(q, k, positions, frequencies, sections, inverse, adjacent, interleaved)


def qk_norm_rotary(q, k, positions, frequencies, sections, q_weight=None, k_weight=None, eps=1e-6, *, adjacent=False,
                   interleaved=False):
    """x / sqrt(mean(x^2) + eps) * weight for every head of queries and keys, then ``rotary``; returns ``(q, k)``.

    ``q_weight`` and ``k_weight`` [head_dim] of one type, float32, bfloat16 or float16; None stands for ones.  ``eps`` is a number,
    without a gradient.
    """
    if _wants_gradient(q, k, q_weight, k_weight):
        _constants("qk_norm_rotary", positions=positions, frequencies=frequencies, eps=eps)
        return _autograd()[1].apply(q, k, positions, frequencies, sections, q_weight, k_weight, eps, adjacent, interleaved)
    return _ops.qk_norm_rotary(q, k, positions, frequencies, sections, q_weight, k_weight, eps, adjacent, interleaved)


def qk_norm_rotary_backward(q_grad, k_grad, q, k, positions, frequencies, sections, q_weight=None, k_weight=None, eps=1e-6, *,
                            adjacent=False, interleaved=False):
    """Gradients of ``qk_norm_rotary``: those of its results come in, ``(dq, dk, dq_weight, dk_weight)`` go out (None where
    there is no k or no weight).  ``q`` and ``k`` are the inputs of the forward pass, which keeps nothing else."""
    return _ops.qk_norm_rotary_backward(q_grad, k_grad, q, k, positions, frequencies, sections, q_weight, k_weight, eps, adjacent,
                                        interleaved)


def cross_attention(q, k, v, *, lengths=None, key_mask=None, scale=None, return_lse=False):
    """softmax(scale * q k^T) v over keys of another length.

    ``q`` [batch, tokens, q_heads, head_dim]; ``k``, ``v`` [batch, keys, kv_heads, head_dim], bfloat16 or float16; q_heads a
    multiple of kv_heads (query head h reads key head h // (q_heads // kv_heads)); head_dim a multiple of 8, up to 128.
    ``scale`` is 1 / sqrt(head_dim) unless given; a number, without a gradient.
    ``lengths`` [batch] int32 or int64: the first so many keys of a sample are read.  ``key_mask`` [batch, keys] bool: keys
    that are False are not read (padding inside a batch of images).  Both may be given.  Whatever lies in k and v where
    nothing is read has no effect.  A sample without a key to read gets zeros, as does a row whose scores are all -infinity.
    Returns the result, or with ``return_lse`` also the logarithm of each row's sum of exponentials, float32
    [batch, q_heads, tokens], which ``cross_attention_backward`` takes; it has a gradient like the result.
    """
    if _wants_gradient(q, k, v):
        _constants("cross_attention", scale=scale)
        out, lse = _autograd()[2].apply(q, k, v, lengths, key_mask, scale)
        return (out, lse) if return_lse else out
    return _ops.cross_attention(q, k, v, lengths, key_mask, scale, return_lse)


def cross_attention_backward(dout, q, k, v, out, lse, *, lengths=None, key_mask=None, scale=None, lse_grad=None):
    """Gradients ``(dq, dk, dv)`` of ``cross_attention``: ``out`` and ``lse`` as it returned them, the other arguments as it
    was given.  ``lse_grad`` is the gradient of lse, where it has one.  Keys that are not read get zeros."""
    return _ops.cross_attention_backward(dout, q, k, v, out, lse, lengths, key_mask, scale, lse_grad)


def window_attention(q, k, v, *, window=None, sinks=0, lengths=None, scale=None, return_lse=False):
    """Causal attention of sequences to themselves: token i reads the tokens j <= i with i - j < window, or j < sinks.

    ``q`` [batch, tokens, q_heads, head_dim]; ``k``, ``v`` [batch, tokens, kv_heads, head_dim]; types, heads, head_dim, ``scale`` and
    ``return_lse`` as in ``cross_attention``.  ``window`` a whole number from 1 on, None: every token before; ``sinks`` first tokens that
    stay visible.  ``lengths`` [batch] int32 or int64: the first so many tokens of a sample are its sequence; what lies behind them in any
    tensor has no effect, and results and gradients there are zeros.  An infinity or NaN in a value may reach tokens of its
    sequence and head that do not read it.
    """
    if _wants_gradient(q, k, v):
        _constants("window_attention", window=window, sinks=sinks, scale=scale)
        out, lse = _autograd()[3].apply(q, k, v, window, sinks, lengths, scale)
        return (out, lse) if return_lse else out
    return _ops.window_attention(q, k, v, window, sinks, lengths, scale, return_lse)


def window_attention_backward(dout, q, k, v, out, lse, *, window=None, sinks=0, lengths=None, scale=None, lse_grad=None):
    """Gradients ``(dq, dk, dv)`` of ``window_attention``: ``out`` and ``lse`` as it returned them, the other arguments as it was
    given.  ``lse_grad`` is the gradient of lse, where it has one."""
    return _ops.window_attention_backward(dout, q, k, v, out, lse, window, sinks, lengths, scale, lse_grad)


def append_rotary(q, k, v, positions, frequencies, sections, k_pages, v_pages, page_table, lengths, *, counts=None, adjacent=False,
                  interleaved=False):
    """New tokens join a cache: keys are turned as by ``rotary`` and written with the values; returns ``q`` turned.

    ``q`` [batch, tokens, q_heads, head_dim] or None, ``k``, ``v`` [batch, tokens, kv_heads, head_dim], ``positions`` [axes, batch,
    tokens], ``frequencies``, ``sections``, ``adjacent`` and ``interleaved`` as in ``rotary``; ``positions`` None: a token's place in its
    sequence, on every axis.
    ``k_pages``, ``v_pages`` [pages, page_size, kv_heads, head_dim] of k's type, written in place; page_size a power of two from 8 on.  Pools
    of float32, and of heads of more than 128 or not a multiple of 8, are for readers of one's own: ``cached_attention`` does not take them.
    ``page_table`` [batch, pages of a sample] int32 or int64: place s of sample b lies in row s % page_size of page
    page_table[b, s // page_size]; an entry that is no page (-1) has no room.  ``lengths`` [batch] int32 or int64: the tokens that the
    cache holds; the new ones go to the places behind them.  ``counts`` [batch] int32 or int64: of a padded batch, how many of a
    sample's tokens are new ones; None: all.  Tokens behind these, and those that have no page, are not written; all queries are
    turned.  Two tokens must not go to one row, and the pools must not overlap the inputs.  There is no gradient: inputs that require one
    are refused.
    """
    return _ops.append_rotary(q, k, v, positions, frequencies, sections, k_pages, v_pages, page_table, lengths, counts, adjacent, interleaved)


def cached_attention(q, k_pages, v_pages, page_table, lengths, *, counts=None, tree=None, window=None, sinks=0, scale=None, return_lse=False):
    """Attention of new tokens over a cache that ``append_rotary`` has put them into, with the same ``lengths`` and ``counts``.

    ``q`` [batch, tokens, q_heads, head_dim], bfloat16 or float16, one token or many; head_dim a multiple of 8, up to 128; q_heads a multiple of
    kv_heads.  Token i of sample b has the place lengths[b] + i and reads the keys j up to its own place with place - j < window
    (None: all) or j < sinks.
    ``tree`` bool [batch, tokens, tokens] or [tokens, tokens], for drafted tokens: token i reads the new token j where tree[i, j], and
    of the tokens before them what the window leaves, counted from the place lengths[b] + the number of new tokens other than itself that
    it reads.  New tokens are read by the tree alone, whatever the window: of a branch longer than the window a caller takes the tokens that
    lie a window or more behind out of a row (but first tokens that stay visible) to get what ``window_attention`` would read.  Keys that
    have no page are not read.  What lies where no token of a sample reads has no effect; an infinity or NaN in a
    value that some read, or under a tree in that of any new token, may reach the sample's other tokens.  Tokens that read nothing, those behind counts[b] among them, get
    zeros.  Returns the result, or with ``return_lse`` also the logarithm of each row's sum of exponentials, float32 [batch,
    q_heads, tokens].  There is no gradient: inputs that require one are refused.
    """
    return _ops.cached_attention(q, k_pages, v_pages, page_table, lengths, counts, tree, window, sinks, scale, return_lse)
