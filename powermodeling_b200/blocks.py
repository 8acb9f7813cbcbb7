"""Operators of a transformer block on torch tensors (include/pmb200_blocks.h).

What a decode layer runs beside the complete nonlinear functions of the
powerbench arms, each one native call on the current stream:

* ``block_norm`` / ``block_norm_backward`` - the norms after and before a
  block, fused with the block's gate and residual scale; ``block_norm`` also
  records itself for autograd when an input asks for gradients;
* ``matvec_w4`` - a few tokens times a matrix of 4-bit weights with a scale
  (and zero point) per group;
* ``paged_attention`` - one new token per sequence attending over a paged
  key-value cache, its own key and value appended in the same call.

Arguments are checked (csrc/python/blocks.cpp, and again in the native
entries): a wrong type, shape or stride raises ``ValueError``, a failed native
call ``_native.NativeError``.  Tensors live on one CUDA device, which need not
be the current one; work goes to that device's current stream.  Outputs are
new tensors.  Nothing synchronizes, so every call can be captured into a graph.
"""
from __future__ import annotations

import torch

from . import _native as N

try:
    from . import _blocksnative as _ops
except ImportError as exc:
    raise N.NativeError("the block operators' extension (_blocksnative) is not built; run python -m powermodeling_b200.build") from exc


class _BlockNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, block, pre_weight, post_weight, gate, scale, eps, captured):
        hidden, normed, stats = _ops.block_norm(residual, block, pre_weight, post_weight, gate, scale, eps, True)
        ctx.save_for_backward(residual, block, pre_weight, post_weight, gate, stats)
        ctx.scale = scale
        ctx.captured = captured
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(stats)
        return hidden, normed, stats

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_hidden, grad_normed, _grad_stats):
        capturing = torch.cuda.is_current_stream_capturing()
        if capturing and not getattr(ctx, "captured", False):
            # the graph of an eager forward brings its own stream into the capture
            raise RuntimeError("block_norm: the forward pass was not captured: capture both, or capture block_norm_backward itself")
        residual, block, pre_weight, post_weight, gate, stats = ctx.saved_tensors
        held = _ops.held_outside_capture(residual, block, pre_weight, post_weight, gate) if capturing else -1
        if held >= 0:
            name = ("residual", "block", "pre_weight", "post_weight", "gate")[held]
            raise RuntimeError(f"block_norm: a graph recorded on the default stream still holds {name}, and its gradient's way "
                               "out of this capture would wait for that stream: drop that graph first, or record it on another")
        if grad_hidden is None and grad_normed is None:
            return (None,) * 8
        need = ctx.needs_input_grad
        grads = block_norm_backward(
            None if grad_hidden is None else grad_hidden.contiguous(),
            None if grad_normed is None else grad_normed.contiguous(), residual, block, pre_weight, stats,
            post_weight=post_weight, gate=gate, scale=ctx.scale, weight_grads=need[2] or need[3], gate_grad=need[4])
        return tuple(g if n else None for g, n in zip(grads, need)) + (None, None, None)


def block_norm(residual, block, pre_weight, *, post_weight=None, gate=None, scale=1.0, eps=1e-5, return_stats=False):
    """The boundary between two blocks: ``(hidden, normed)`` with

        p      = block * rsqrt(mean(block**2) + eps) * post_weight     (p = block without a post_weight)
        hidden = residual + scale * gate * p                           (no gate: scale * p)
        normed = hidden * rsqrt(mean(hidden**2) + eps) * pre_weight    (of the unrounded hidden)

    ``residual`` and ``block`` are [rows, width] of float32, bfloat16 or
    float16 (any row stride); weights are [width], the gate [width] or
    [s, width] with s dividing rows (gate row i serves the i-th run of rows / s
    rows; s = rows gates every element), each of that type or float32.  With
    ``return_stats`` a third value, [rows, 2] float32, is returned for
    ``block_norm_backward``.  A training step is captured with its forward and
    backward together, or by ``block_norm_backward``; a captured backward to a
    leaf that a living graph of the default stream holds is refused
    (``RuntimeError``).
    """
    try:
        recorded = torch.is_grad_enabled() and (residual.requires_grad or block.requires_grad or pre_weight.requires_grad
                                                or (post_weight is not None and post_weight.requires_grad)
                                                or (gate is not None and gate.requires_grad))
    except AttributeError:                       # no tensor: the native call says which
        recorded = False
    if recorded:
        out = _BlockNormFunction.apply(residual, block, pre_weight, post_weight, gate, scale, eps, _ops.captured(residual))
        return out if return_stats else out[:2]
    return _ops.block_norm(residual, block, pre_weight, post_weight, gate, scale, eps, return_stats)


def block_norm_backward(grad_hidden, grad_normed, residual, block, pre_weight, stats, *, post_weight=None, gate=None,
                        scale=1.0, weight_grads=True, gate_grad=True):
    """Gradients of ``block_norm``: (residual, block, pre_weight, post_weight, gate), None where there is none.

    Takes the forward call's inputs and its ``stats``; either incoming gradient
    may be None.  ``weight_grads`` and ``gate_grad`` say whether those are
    wanted.  Sums over rows run in a fixed order.
    """
    return _ops.block_norm_backward(residual, block, pre_weight, post_weight, gate, scale, grad_hidden, grad_normed, stats,
                                    weight_grads, gate_grad)


def matvec_w4(x, weight, scales, zeros=None, *, group_size=128):
    """``x`` [tokens, k] (bfloat16 or float16, any row stride) times the 4-bit ``weight``: [tokens, n].

    ``weight`` is [n, ceil(k / 2)] uint8 (any row stride up to 2^23), the even k
    in the low half of a byte; ``scales`` [n, ceil(k / group_size)] of x's type or
    float32; ``zeros`` the same shape in uint8 (0..15), or None for 8 everywhere.
    Meant for single tokens and small batches: the weights are read once for
    every 16 tokens.  There is no backward.
    """
    return _ops.matvec_w4(x, weight, scales, zeros, group_size)


def paged_attention(q, k_cache, v_cache, page_table, lengths, *, new_k=None, new_v=None, scale=None, window=0,
                    layout="NHD", return_lse=False):
    """One new token per sequence attends over its pages of the cache: [batch, q_heads, head_dim].

    ``q`` is [batch, q_heads, head_dim] (bfloat16 or float16); the caches
    [pages, page_size, kv_heads, head_dim] (layout "NHD") or [pages, kv_heads,
    page_size, head_dim] ("HND"), kv_heads dividing q_heads and head_dim a
    multiple of 8 up to 256; ``page_table`` [batch, columns] int32; ``lengths``
    [batch] int32, the new token counted.  Position j of a sequence is entry
    j % page_size of page page_table[b, j // page_size]; a page index outside
    the cache marks an absent page, whose positions are skipped.  ``window``
    keeps the last so many positions (0: all).  ``scale`` defaults to
    head_dim ** -0.5.  With ``new_k`` and ``new_v`` [batch, kv_heads, head_dim]
    the token's own key and value are first written to position length - 1 of
    the caches, in the same call; no other position of any sequence may be found
    at that entry.  A sequence of length 0 gives zeros.  ``return_lse`` adds the logarithm of
    each row's sum of exponentials, [batch, q_heads] float32.  There is no
    backward.
    """
    return _ops.paged_attention(q, k_cache, v_cache, page_table, lengths, new_k, new_v, scale, window, layout, return_lse)
