"""Attention over batches of images and clips: what a model does with a batch once its patches are projected.

* ``rotary``: positions with several axes (time, row, column) turn queries and keys.
* ``qk_norm_rotary``: RMS norm of every head of queries and keys, and the rotation, in one pass.
* ``cross_attention``: queries read the states of images or clips, padding masked out.

All take torch tensors in GPU memory, ``[batch, tokens, heads, head_dim]`` (views of a joint projection too), and queue
their work on torch's current stream of the tensors' device; results are new contiguous tensors.  They work under
``torch.autograd`` (reverse mode, once; forward mode raises); the functions ``*_backward`` are the same gradients for programs
that do without it.  Sums are held in float32 and results rounded once to the tensors' type.  ``cross_attention`` also rounds what its
products on the tensor cores take, the weights P and in the backward pass dS = P (dP - delta), to the tensors' type, with delta from the
rounded result where keys are more than 128: errors of 1.4 to 1.6 roundings instead of one.  In float16 a dS beyond 65504 is infinite,
as a loss scaler expects of a scale that is too high.  The same call gives the same bits again.  Wrong arguments raise ``ValueError``;
there is no CPU path.
"""
import importlib

__all__ = ["rotary", "qk_norm_rotary", "qk_norm_rotary_backward", "cross_attention", "cross_attention_backward"]



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

        _functions = Rotary, QkNormRotary, CrossAttention
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
