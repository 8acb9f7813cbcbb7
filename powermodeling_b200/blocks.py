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

Arguments are checked here and in the native entry points: a wrong type,
shape or stride raises ``ValueError``, a failed native call
``_native.NativeError``.  Tensors live on one CUDA device, which need not be
the current one; work goes to that device's current stream.  Outputs are new
tensors.  Nothing synchronizes, so every call can be captured into a graph.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _native as N

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_HEAD_DIM = 256
_p = C.c_void_p


class _BlockNorm(C.Structure):
    _fields_ = [("rows", C.c_int64), ("gate_rows", C.c_int64), ("residual_stride", C.c_int64),
                ("block_stride", C.c_int64), ("width", C.c_int32), ("dtype", C.c_int32), ("pre_dtype", C.c_int32),
                ("post_dtype", C.c_int32), ("gate_dtype", C.c_int32), ("scale", C.c_float), ("eps", C.c_float),
                ("residual", _p), ("block", _p), ("pre_weight", _p), ("post_weight", _p), ("gate", _p),
                ("hidden", _p), ("normed", _p), ("stats", _p)]


class _BlockNormGrads(C.Structure):
    _fields_ = [("grad_hidden_stride", C.c_int64), ("grad_normed_stride", C.c_int64), ("grad_hidden", _p),
                ("grad_normed", _p), ("grad_residual", _p), ("grad_block", _p), ("grad_pre", _p), ("grad_post", _p),
                ("grad_gate", _p)]


class _MatvecW4(C.Structure):
    _fields_ = [("tokens", C.c_int32), ("n", C.c_int32), ("k", C.c_int32), ("group", C.c_int32), ("dtype", C.c_int32),
                ("scales_dtype", C.c_int32), ("x_stride", C.c_int64), ("weight_stride", C.c_int64), ("x", _p),
                ("weight", _p), ("scales", _p), ("zeros", _p), ("y", _p)]


class _PagedAttention(C.Structure):
    _fields_ = [("batch", C.c_int32), ("q_heads", C.c_int32), ("kv_heads", C.c_int32), ("head_dim", C.c_int32),
                ("page_size", C.c_int32), ("n_pages", C.c_int32), ("table_columns", C.c_int32), ("dtype", C.c_int32),
                ("window", C.c_int32), ("scale", C.c_float), ("q_stride", C.c_int64), ("q_head_stride", C.c_int64),
                ("k_page_stride", C.c_int64), ("k_token_stride", C.c_int64), ("k_head_stride", C.c_int64),
                ("v_page_stride", C.c_int64), ("v_token_stride", C.c_int64), ("v_head_stride", C.c_int64),
                ("new_k_stride", C.c_int64), ("new_k_head_stride", C.c_int64), ("new_v_stride", C.c_int64),
                ("new_v_head_stride", C.c_int64), ("table_stride", C.c_int64), ("q", _p), ("k_cache", _p),
                ("v_cache", _p), ("table", _p), ("lengths", _p), ("new_k", _p), ("new_v", _p), ("out", _p), ("lse", _p)]


_bound = None


def _lib():
    global _bound
    if _bound is None:
        lib = N.library()
        lib.pm_block_norm_device.argtypes = [_p, _p]
        lib.pm_block_norm_backward_scratch_bytes.argtypes = [C.c_int64, C.c_int64, C.c_int32]
        lib.pm_block_norm_backward_scratch_bytes.restype = C.c_size_t
        lib.pm_block_norm_backward_device.argtypes = [_p, _p, _p, C.c_size_t, _p]
        lib.pm_matvec_w4_device.argtypes = [_p, _p]
        lib.pm_paged_attention_scratch_bytes.argtypes = [C.c_int32] * 4
        lib.pm_paged_attention_scratch_bytes.restype = C.c_size_t
        lib.pm_paged_attention_device.argtypes = [_p, _p, C.c_size_t, _p]
        _bound = lib
    return _bound


def _place(name, *tensors):
    """The one CUDA device of the tensors, as an ordinal."""
    device = tensors[0].device
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"{name}: tensors are on {device} and {t.device}")
    if device.type != "cuda":
        raise ValueError(f"{name}: tensors must be on a CUDA device")
    return device.index


def _call(entry, device, what, *args):
    """The native call on the device's current stream."""
    if device == torch.cuda.current_device():
        rc = entry(*args, torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            rc = entry(*args, torch.cuda.current_stream(device).cuda_stream)
    if rc != 0:
        raise N.NativeError(f"{what} failed ({rc}): {N.last_error()}")


def _rows(name, t, shape=None):
    """Row stride of a 2-D tensor with a unit inner stride (of `shape`, if given)."""
    if t.dim() != 2 or (shape is not None and t.shape != shape):
        raise ValueError(f"{name} must be {'two-dimensional' if shape is None else list(shape)}, got {list(t.shape)}")
    if t.stride(1) != 1 and t.shape[1] > 1:
        raise ValueError(f"{name}: elements of a row must be contiguous")
    stride = t.stride(0)
    if stride < t.shape[1]:
        if t.shape[0] > 1:
            raise ValueError(f"{name}: rows overlap")
        stride = t.shape[1]
    return stride


def _norm_job(residual, block, pre_weight, post_weight, gate, scale, eps):
    if residual.dtype not in _TYPES or block.dtype != residual.dtype:
        raise ValueError("block_norm: residual and block must share one of float32, bfloat16, float16")
    residual_stride = _rows("residual", residual)
    block_stride = _rows("block", block, residual.shape)
    rows, width = residual.shape
    for name, w in (("pre_weight", pre_weight), ("post_weight", post_weight)):
        if w is None and name == "post_weight":
            continue
        if w.shape != (width,) or not w.is_contiguous() or w.dtype not in (residual.dtype, torch.float32):
            raise ValueError(f"block_norm: {name} must be a contiguous [{width}] of {residual.dtype} or float32")
    gate_rows = 0
    if gate is not None:
        if gate.dim() == 1:
            gate = gate[None]
        gate_rows = gate.shape[0]
        if (gate.dim() != 2 or gate.shape[1] != width or not gate.is_contiguous() or gate_rows < 1 or rows % gate_rows
                or gate.dtype not in (residual.dtype, torch.float32)):
            raise ValueError(f"block_norm: gate must be a contiguous [s, {width}] (s dividing {rows}) of "
                             f"{residual.dtype} or float32")
    if not width:
        raise ValueError("block_norm: rows must not be empty")
    if not (math.isfinite(scale) and math.isfinite(eps) and eps >= 0):
        raise ValueError("block_norm: scale must be finite and eps >= 0")
    device = _place("block_norm", residual, block, pre_weight, post_weight, gate)
    job = _BlockNorm(rows, gate_rows, residual_stride, block_stride, width, _TYPES[residual.dtype],
                     _TYPES[pre_weight.dtype], 0 if post_weight is None else _TYPES[post_weight.dtype],
                     0 if gate is None else _TYPES[gate.dtype], scale, eps, residual.data_ptr(), block.data_ptr(),
                     pre_weight.data_ptr(), None if post_weight is None else post_weight.data_ptr(),
                     None if gate is None else gate.data_ptr(), None, None, None)
    return job, device


def _norm_forward(residual, block, pre_weight, post_weight, gate, scale, eps, want_stats):
    job, device = _norm_job(residual, block, pre_weight, post_weight, gate, scale, eps)
    hidden = residual.new_empty(residual.shape)
    normed = residual.new_empty(residual.shape)
    stats = residual.new_empty((residual.shape[0], 2), dtype=torch.float32) if want_stats else None
    if hidden.numel():
        job.hidden, job.normed = hidden.data_ptr(), normed.data_ptr()
        job.stats = stats.data_ptr() if want_stats else None
        _call(_lib().pm_block_norm_device, device, "pm_block_norm_device", C.byref(job))
    return hidden, normed, stats


class _BlockNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, block, pre_weight, post_weight, gate, scale, eps):
        hidden, normed, stats = _norm_forward(residual, block, pre_weight, post_weight, gate, scale, eps, True)
        ctx.save_for_backward(residual, block, pre_weight, post_weight, gate, stats)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(stats)
        return hidden, normed, stats

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_hidden, grad_normed, _grad_stats):
        if torch.cuda.is_current_stream_capturing():
            # an eager graph of the same leaves would pull its own stream into the capture and end it
            raise RuntimeError("block_norm: capture block_norm_backward itself, not the autograd engine's call of it")
        residual, block, pre_weight, post_weight, gate, stats = ctx.saved_tensors
        if grad_hidden is None and grad_normed is None:
            return (None,) * 7
        need = ctx.needs_input_grad
        grads = block_norm_backward(
            None if grad_hidden is None else grad_hidden.contiguous(),
            None if grad_normed is None else grad_normed.contiguous(), residual, block, pre_weight, stats,
            post_weight=post_weight, gate=gate, scale=ctx.scale, weight_grads=need[2] or need[3], gate_grad=need[4])
        return tuple(g if n else None for g, n in zip(grads, need)) + (None, None)


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
    ``block_norm_backward``.
    """
    if torch.is_grad_enabled() and (residual.requires_grad or block.requires_grad or pre_weight.requires_grad
                                    or (post_weight is not None and post_weight.requires_grad)
                                    or (gate is not None and gate.requires_grad)):
        out = _BlockNormFunction.apply(residual, block, pre_weight, post_weight, gate, scale, eps)
        return out if return_stats else out[:2]
    hidden, normed, stats = _norm_forward(residual, block, pre_weight, post_weight, gate, scale, eps, return_stats)
    return (hidden, normed, stats) if return_stats else (hidden, normed)


@torch.no_grad()
def block_norm_backward(grad_hidden, grad_normed, residual, block, pre_weight, stats, *, post_weight=None, gate=None,
                        scale=1.0, weight_grads=True, gate_grad=True):
    """Gradients of ``block_norm``: (residual, block, pre_weight, post_weight, gate), None where there is none.

    Takes the forward call's inputs and its ``stats``; either incoming gradient
    may be None.  ``weight_grads`` and ``gate_grad`` say whether those are
    wanted.  Sums over rows run in a fixed order.
    """
    job, device = _norm_job(residual, block, pre_weight, post_weight, gate, scale, 0.0)
    rows, width = residual.shape
    if stats.shape != (rows, 2) or stats.dtype != torch.float32 or not stats.is_contiguous():
        raise ValueError(f"block_norm_backward: stats must be the forward call's [{rows}, 2] float32")
    if grad_hidden is None and grad_normed is None:
        raise ValueError("block_norm_backward: no incoming gradient")
    grads = _BlockNormGrads()
    for name, g in (("grad_hidden", grad_hidden), ("grad_normed", grad_normed)):
        if g is not None:
            if g.dtype != residual.dtype:
                raise ValueError(f"block_norm_backward: {name} must be of {residual.dtype}")
            setattr(grads, name + "_stride", _rows(name, g, residual.shape))
            setattr(grads, name, g.data_ptr())
    _place("block_norm_backward", residual, grad_hidden, grad_normed, stats)
    grad_residual, grad_block = residual.new_empty(residual.shape), residual.new_empty(residual.shape)
    grad_pre = torch.empty_like(pre_weight) if weight_grads else None
    grad_post = torch.empty_like(post_weight) if weight_grads and post_weight is not None else None
    grad_gate = torch.empty_like(gate) if gate_grad and gate is not None else None
    lib = _lib()
    need = lib.pm_block_norm_backward_scratch_bytes(rows, job.gate_rows, width)
    scratch = torch.empty(need, dtype=torch.uint8, device=residual.device)
    job.stats = stats.data_ptr()
    grads.grad_residual, grads.grad_block = grad_residual.data_ptr(), grad_block.data_ptr()
    for name, g in (("grad_pre", grad_pre), ("grad_post", grad_post), ("grad_gate", grad_gate)):
        if g is not None:
            setattr(grads, name, g.data_ptr())
    _call(lib.pm_block_norm_backward_device, device, "pm_block_norm_backward_device", C.byref(job), C.byref(grads),
          scratch.data_ptr(), need)
    return grad_residual, grad_block, grad_pre, grad_post, grad_gate


def matvec_w4(x, weight, scales, zeros=None, *, group_size=128):
    """``x`` [tokens, k] (bfloat16 or float16, any row stride) times the 4-bit ``weight``: [tokens, n].

    ``weight`` is [n, ceil(k / 2)] uint8 (any row stride), the even k in the
    low half of a byte; ``scales`` [n, ceil(k / group_size)] of x's type or
    float32; ``zeros`` the same shape in uint8 (0..15), or None for 8 everywhere.
    Meant for single tokens and small batches: the weights are read once for
    every 16 tokens.
    """
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("matvec_w4: x must be bfloat16 or float16")
    x_stride = _rows("x", x)
    tokens, k = x.shape
    if weight.dtype != torch.uint8 or weight.dim() != 2 or not k or weight.shape[1] != (k + 1) // 2:
        raise ValueError(f"matvec_w4: weight must be uint8 [n, {(k + 1) // 2}]")
    weight_stride = _rows("weight", weight)
    n = weight.shape[0]
    if group_size < 32 or group_size % 32:
        raise ValueError("matvec_w4: group_size must be a multiple of 32")
    shape = (n, -(-k // group_size))
    if scales.shape != shape or not scales.is_contiguous() or scales.dtype not in (x.dtype, torch.float32):
        raise ValueError(f"matvec_w4: scales must be a contiguous {list(shape)} of {x.dtype} or float32")
    if zeros is not None and (zeros.shape != shape or not zeros.is_contiguous() or zeros.dtype != torch.uint8):
        raise ValueError(f"matvec_w4: zeros must be a contiguous {list(shape)} of uint8")
    device = _place("matvec_w4", x, weight, scales, zeros)
    y = x.new_empty((tokens, n))
    if y.numel():
        job = _MatvecW4(tokens, n, k, group_size, _TYPES[x.dtype], _TYPES[scales.dtype], x_stride, weight_stride,
                        x.data_ptr(), weight.data_ptr(), scales.data_ptr(), None if zeros is None else zeros.data_ptr(),
                        y.data_ptr())
        _call(_lib().pm_matvec_w4_device, device, "pm_matvec_w4_device", C.byref(job))
    return y


def _heads(name, t, shape, dtype):
    if t.shape != shape or t.dtype != dtype:
        raise ValueError(f"paged_attention: {name} must be {list(shape)} of {dtype}")
    if t.stride(-1) != 1:
        raise ValueError(f"paged_attention: {name}: the head's elements must be contiguous")
    # an axis of one entry has no stride that matters
    strides = tuple(s if n > 1 else 0 for s, n in zip(t.stride()[:-1], t.shape))
    if t.data_ptr() % 16 or any(s % 8 for s in strides):
        raise ValueError(f"paged_attention: {name} must be 16-byte aligned with strides in multiples of 8 elements")
    return strides


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
    the caches, in the same call; no two sequences may share that entry.  A
    sequence of length 0 gives zeros.  ``return_lse`` adds the logarithm of
    each row's sum of exponentials, [batch, q_heads] float32.
    """
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("paged_attention: q must be bfloat16 or float16")
    if q.dim() != 3 or k_cache.dim() != 4 or layout not in ("NHD", "HND"):
        raise ValueError("paged_attention: q is [batch, q_heads, head_dim], a cache four-dimensional in layout NHD or HND")
    batch, q_heads, head_dim = q.shape
    token, head = (1, 2) if layout == "NHD" else (2, 1)
    page_size, kv_heads = k_cache.shape[token], k_cache.shape[head]
    if not kv_heads or not q_heads or q_heads % kv_heads:
        raise ValueError(f"paged_attention: {kv_heads} key heads do not divide {q_heads} query heads")
    if head_dim % 8 or not 8 <= head_dim <= MAX_HEAD_DIM:
        raise ValueError(f"paged_attention: head_dim must be a multiple of 8 up to {MAX_HEAD_DIM}")
    if not 1 <= page_size <= 65536 or window < 0:
        raise ValueError("paged_attention: page_size must be in 1..65536 and window >= 0")
    if k_cache.shape[3] != head_dim:
        raise ValueError(f"paged_attention: k_cache holds heads of {k_cache.shape[3]} elements, q of {head_dim}")
    dtype = q.dtype
    qs = _heads("q", q, q.shape, dtype)
    ks, vs = _heads("k_cache", k_cache, k_cache.shape, dtype), _heads("v_cache", v_cache, k_cache.shape, dtype)
    if (new_k is None) != (new_v is None):
        raise ValueError("paged_attention: new_k and new_v come together")
    nks = nvs = (0, 0)
    if new_k is not None:
        nks = _heads("new_k", new_k, (batch, kv_heads, head_dim), dtype)
        nvs = _heads("new_v", new_v, (batch, kv_heads, head_dim), dtype)
    if page_table.dim() != 2 or page_table.shape[0] != batch or page_table.dtype != torch.int32 or \
            (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise ValueError(f"paged_attention: page_table must be int32 [{batch}, columns] with contiguous rows")
    if lengths.shape != (batch,) or lengths.dtype != torch.int32 or not lengths.is_contiguous():
        raise ValueError(f"paged_attention: lengths must be a contiguous int32 [{batch}]")
    if scale is None:
        scale = head_dim ** -0.5
    if not math.isfinite(scale):
        raise ValueError("paged_attention: scale must be finite")
    device = _place("paged_attention", q, k_cache, v_cache, page_table, lengths, new_k, new_v)
    out = q.new_empty((batch, q_heads, head_dim))
    lse = q.new_empty((batch, q_heads), dtype=torch.float32) if return_lse else None
    if batch:
        lib = _lib()
        need = lib.pm_paged_attention_scratch_bytes(batch, q_heads, kv_heads, head_dim)
        scratch = torch.empty(need, dtype=torch.uint8, device=q.device)
        job = _PagedAttention(
            batch, q_heads, kv_heads, head_dim, page_size, k_cache.shape[0], page_table.shape[1], _TYPES[dtype], window,
            scale, qs[0], qs[1], ks[0], ks[token], ks[head], vs[0], vs[token], vs[head], nks[0], nks[1], nvs[0], nvs[1],
            page_table.stride(0), q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), page_table.data_ptr(),
            lengths.data_ptr(), None if new_k is None else new_k.data_ptr(), None if new_v is None else new_v.data_ptr(),
            out.data_ptr(), None if lse is None else lse.data_ptr())
        _call(lib.pm_paged_attention_device, device, "pm_paged_attention_device", C.byref(job), scratch.data_ptr(), need)
    return (out, lse) if return_lse else out
