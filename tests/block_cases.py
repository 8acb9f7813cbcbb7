"""Plain 64-bit statements of the block operators, with the magnitudes their rounding errors scale with.

Every function returns (value, magnitude) pairs: `magnitude` is the same
formula with every term taken absolute, so a result computed in 32 bits is
within (number of roundings) x 2^-24 x magnitude of the value.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from powermodeling_b200 import _native as N

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# the smallest half step: below it a rounding is off by an absolute amount
FLOOR = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}


def within(got, want, magnitude, steps):
    """Largest excess of |got - want| over half a step of got's type plus `steps` 32-bit roundings of `magnitude`."""
    allowed = HALF[got.dtype] * want.abs() + FLOOR[got.dtype] + steps * 2.0 ** -24 * magnitude
    # the output's own rounding applies to the 32-bit value, which is off by the second term already
    allowed = allowed * (1 + HALF[got.dtype])
    off = (got.double() - want).abs()
    bad = ~(off <= allowed)
    return int(bad.sum()), float((off / allowed.clamp(min=1e-300)).max()) if off.numel() else 0.0


def norm(residual, block, pre, post, gate, scale, eps):
    r, b, w = residual.double(), block.double(), pre.double()
    n, d = r.shape
    r1 = torch.ones(n, 1, dtype=torch.float64, device=r.device)
    p = b
    if post is not None:
        r1 = 1 / (b.square().mean(1, keepdim=True) + eps).sqrt()
        p = b * r1 * post.double()
    g = torch.ones(1, 1, dtype=torch.float64, device=r.device)
    if gate is not None:
        gate = gate.reshape(-1, d)
        g = gate.double().repeat_interleave(n // gate.shape[0], 0)
    h = r + scale * g * p
    H = r.abs() + (scale * g * p).abs()
    r2 = 1 / (h.square().mean(1, keepdim=True) + eps).sqrt()
    # the mean of h^2 is off by roundings of the mean of H^2, and r2 by half of that relative
    R = r2 * (1 + (H.square().mean(1, keepdim=True)) * r2.square())
    return dict(hidden=(h, H), normed=(h * r2 * w, H * R * w.abs()), r1=r1, r2=r2, R=R, p=p, g=g, h=h, H=H)


def norm_grads(gh, gy, residual, block, pre, post, gate, scale, eps):
    f = norm(residual, block, pre, post, gate, scale, eps)
    b, w, r1, r2, g, p = block.double(), pre.double(), f["r1"], f["r2"], f["g"], f["p"]
    n, d = b.shape
    zero = torch.zeros_like(b)
    gh = zero if gh is None else gh.double()
    gy = zero if gy is None else gy.double()
    u, U = f["h"] * r2, f["H"] * f["R"]
    t, T = gy * w, (gy * w).abs()
    dh = gh + r2 * (t - u * (t * u).mean(1, keepdim=True))
    DH = gh.abs() + f["R"] * (T + U * (T * U).mean(1, keepdim=True))
    out = dict(residual=(dh, DH), pre=((gy * u).sum(0), (gy.abs() * U).sum(0)))
    dp, DP = scale * g * dh, (scale * g).abs() * DH
    if post is not None:
        bu = b * r1
        out["post"] = ((dp * bu).sum(0), (DP * bu.abs()).sum(0))
        c, Cm = dp * post.double(), DP * post.double().abs()
        out["block"] = (r1 * (c - bu * (c * bu).mean(1, keepdim=True)),
                        r1 * (Cm + bu.abs() * (Cm * bu.abs()).mean(1, keepdim=True)))
    else:
        out["block"] = (dp, DP)
    if gate is not None:
        s = gate.reshape(-1, d).shape[0]
        out["gate"] = tuple((scale * x if i == 0 else abs(scale) * x).reshape(s, n // s, d).sum(1).reshape(gate.shape)
                            for i, x in enumerate((dh * p, DH * p.abs())))
    return out


def pack(q):
    """[n, k] integers 0..15 to [n, ceil(k / 2)] bytes, the even k low."""
    n, k = q.shape
    if k % 2:
        q = torch.cat((q, torch.full((n, 1), 15, dtype=q.dtype, device=q.device)), 1)   # the unread half is not zero
    return (q[:, 0::2] | (q[:, 1::2] << 4)).to(torch.uint8)


def matvec(x, q, scales, zeros, group):
    k = x.shape[1]
    s = scales.double().repeat_interleave(group, 1)[:, :k]
    z = zeros.double().repeat_interleave(group, 1)[:, :k] if zeros is not None else torch.full_like(s, 8.0)
    y = x.double() @ ((q.double() - z) * s).t()
    return y, x.double().abs() @ ((q.double() + z + 32.0) * s.abs()).t()


def attention(q, k_cache, v_cache, table, lengths, new_k, new_v, scale, window, layout):
    """(out, magnitude, lse, lse magnitude, caches after the append); sequence by sequence."""
    kc, vc = k_cache.clone(), v_cache.clone()
    if layout == "HND":
        kt, vt = kc.transpose(1, 2), vc.transpose(1, 2)
    else:
        kt, vt = kc, vc
    pages, page, hk, d = kt.shape
    b, heads, _ = q.shape
    share = heads // hk
    out = torch.zeros(b, heads, d, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    lse = torch.full((b, heads), -math.inf, dtype=torch.float64, device=q.device)
    lmag = torch.ones_like(lse)
    tab, lens = table.tolist(), lengths.tolist()

    def at(i, pos):
        col = pos // page
        if pos < 0 or col >= len(tab[i]) or not 0 <= tab[i][col] < pages:
            return None
        return tab[i][col], pos % page

    if new_k is not None:
        for i in range(b):
            home = at(i, lens[i] - 1)
            if home is not None:
                kt[home], vt[home] = new_k[i], new_v[i]
    for i in range(b):
        first = max(0, lens[i] - window) if window else 0
        live = [p for p in (at(i, pos) for pos in range(first, min(lens[i], len(tab[i]) * page))) if p is not None]
        if not live:
            continue
        idx = torch.tensor(live, device=q.device)
        k = kt[idx[:, 0], idx[:, 1]].double().repeat_interleave(share, 1)       # [live, heads, d]
        v = vt[idx[:, 0], idx[:, 1]].double().repeat_interleave(share, 1)
        s = (k * q[i].double()).sum(2) * scale
        S = (k.abs() * q[i].double().abs()).sum(2) * abs(scale)
        w = torch.softmax(s, 0)
        out[i] = (w[:, :, None] * v).sum(0)
        lse[i] = torch.logsumexp(s, 0)
        lmag[i] = S.amax(0) + lse[i].abs() + 1
        # every weight is off by the roundings of its score and of the largest, besides its own
        mag[i] = (w[:, :, None] * v.abs() * (1 + 2 * S.amax(0))[None, :, None]).sum(0)
    return out, mag, lse, lmag, kc, vc


# ---------------------------------------------------------------- the C entries (include/pmb200_blocks.h)
_p = C.c_void_p


class BlockNorm(C.Structure):
    _fields_ = [("rows", C.c_int64), ("gate_rows", C.c_int64), ("residual_stride", C.c_int64),
                ("block_stride", C.c_int64), ("width", C.c_int32), ("dtype", C.c_int32), ("pre_dtype", C.c_int32),
                ("post_dtype", C.c_int32), ("gate_dtype", C.c_int32), ("scale", C.c_float), ("eps", C.c_float),
                ("residual", _p), ("block", _p), ("pre_weight", _p), ("post_weight", _p), ("gate", _p),
                ("hidden", _p), ("normed", _p), ("stats", _p)]


class BlockNormGrads(C.Structure):
    _fields_ = [("grad_hidden_stride", C.c_int64), ("grad_normed_stride", C.c_int64), ("grad_hidden", _p),
                ("grad_normed", _p), ("grad_residual", _p), ("grad_block", _p), ("grad_pre", _p), ("grad_post", _p),
                ("grad_gate", _p)]


class MatvecW4(C.Structure):
    _fields_ = [("tokens", C.c_int32), ("n", C.c_int32), ("k", C.c_int32), ("group", C.c_int32), ("dtype", C.c_int32),
                ("scales_dtype", C.c_int32), ("x_stride", C.c_int64), ("weight_stride", C.c_int64), ("x", _p),
                ("weight", _p), ("scales", _p), ("zeros", _p), ("y", _p)]


class PagedAttention(C.Structure):
    _fields_ = [("batch", C.c_int32), ("q_heads", C.c_int32), ("kv_heads", C.c_int32), ("head_dim", C.c_int32),
                ("page_size", C.c_int32), ("n_pages", C.c_int32), ("table_columns", C.c_int32), ("dtype", C.c_int32),
                ("window", C.c_int32), ("scale", C.c_float), ("q_stride", C.c_int64), ("q_head_stride", C.c_int64),
                ("k_page_stride", C.c_int64), ("k_token_stride", C.c_int64), ("k_head_stride", C.c_int64),
                ("v_page_stride", C.c_int64), ("v_token_stride", C.c_int64), ("v_head_stride", C.c_int64),
                ("new_k_stride", C.c_int64), ("new_k_head_stride", C.c_int64), ("new_v_stride", C.c_int64),
                ("new_v_head_stride", C.c_int64), ("table_stride", C.c_int64), ("q", _p), ("k_cache", _p),
                ("v_cache", _p), ("table", _p), ("lengths", _p), ("new_k", _p), ("new_v", _p), ("out", _p), ("lse", _p)]


def library():
    lib = N.library()
    lib.pm_block_norm_device.argtypes = [_p, _p]
    lib.pm_block_norm_backward_scratch_bytes.argtypes = [C.c_int64, C.c_int64, C.c_int32]
    lib.pm_block_norm_backward_scratch_bytes.restype = C.c_size_t
    lib.pm_block_norm_backward_device.argtypes = [_p, _p, _p, C.c_size_t, _p]
    lib.pm_matvec_w4_scratch_bytes.argtypes = [C.c_int32] * 3
    lib.pm_matvec_w4_scratch_bytes.restype = C.c_size_t
    lib.pm_matvec_w4_device.argtypes = [_p, _p, C.c_size_t, _p]
    lib.pm_paged_attention_scratch_bytes.argtypes = [C.c_int32] * 4
    lib.pm_paged_attention_scratch_bytes.restype = C.c_size_t
    lib.pm_paged_attention_device.argtypes = [_p, _p, C.c_size_t, _p]
    return lib
