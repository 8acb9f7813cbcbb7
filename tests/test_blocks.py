"""Argument checks of the block operators, on the CPU: refused before anything reaches a device."""
from __future__ import annotations

import ctypes as C
import re

import pytest
import torch

import block_cases as K
from conftest import ROOT
from powermodeling_b200 import _native as N
from powermodeling_b200 import blocks

BF = torch.bfloat16
INVALID, LIMIT = -1, -4


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def norm(**kw):
    a = dict(residual=z(4, 32), block=z(4, 32), pre_weight=z(32))
    a.update(kw)
    return blocks.block_norm(a.pop("residual"), a.pop("block"), a.pop("pre_weight"), **a)


@pytest.mark.parametrize("kw,message", [
    (dict(residual=z(4, 32, dtype=torch.float64), block=z(4, 32, dtype=torch.float64)), "float32, bfloat16, float16"),
    (dict(block=z(4, 32, dtype=torch.float16)), "must share"),
    (dict(block=z(4, 31)), "must be"),
    (dict(residual=z(32)), "two-dimensional"),
    (dict(residual=z(32, 4).t(), block=z(4, 32)), "contiguous"),
    (dict(residual=z(1, 32).expand(4, 32)), "overlap"),
    (dict(pre_weight=z(31)), "pre_weight"),
    (dict(pre_weight=z(32, dtype=torch.float16)), "pre_weight"),
    (dict(pre_weight=z(64)[::2]), "pre_weight"),
    (dict(post_weight=z(1, 32)), "post_weight"),
    (dict(gate=z(3, 32)), "gate"),
    (dict(gate=z(0, 32)), "gate"),
    (dict(gate=z(4, 31)), "gate"),
    (dict(gate=z(1, 4, 32)), "gate"),
    (dict(scale=float("nan")), "scale"),
    (dict(eps=-1e-5), "eps"),
    (dict(residual=z(4, 0), block=z(4, 0), pre_weight=z(0)), "empty"),
    (dict(), "CUDA device"),
])
def test_block_norm_refusals(kw, message):
    with pytest.raises(ValueError, match=message):
        norm(**kw)


def test_refusals_of_what_is_no_tensor():
    for kw, message in ((dict(residual=[[1.0]]), "residual"), (dict(block=None), "block"), (dict(gate=0.5), "gate")):
        with pytest.raises(ValueError, match=message + " must be a tensor"):
            norm(**kw)


def test_refusals_of_numbers_that_ask_for_gradients():
    asks = torch.tensor(0.5, requires_grad=True)
    for call in (lambda: norm(scale=asks), lambda: norm(eps=asks), lambda: attention(scale=asks)):
        with pytest.raises(ValueError, match="no gradient goes through"):
            call()


def test_block_norm_backward_refusals():
    x, w, st = z(4, 32), z(32), z(4, 2, dtype=torch.float32)
    for args, message in (((None, None, x, x, w, st), "no incoming gradient"),
                          ((x, None, x, x, w, z(4, 2)), "stats"),
                          ((x, None, x, x, w, z(3, 2, dtype=torch.float32)), "stats"),
                          ((z(4, 32, dtype=torch.float32), None, x, x, w, st), "grad_hidden"),
                          ((None, z(4, 31), x, x, w, st), "grad_normed"),
                          ((x, x, x, z(4, 31), w, st), "must be"),
                          ((x, x, x, x, w, st), "CUDA device")):
        with pytest.raises(ValueError, match=message):
            blocks.block_norm_backward(*args)


def matvec(**kw):
    a = dict(x=z(2, 64), weight=z(8, 32, dtype=torch.uint8), scales=z(8, 1), zeros=None, group_size=64)
    a.update(kw)
    return blocks.matvec_w4(a["x"], a["weight"], a["scales"], a["zeros"], group_size=a["group_size"])


@pytest.mark.parametrize("kw,message", [
    (dict(x=z(2, 64, dtype=torch.float32)), "bfloat16 or float16"),
    (dict(x=z(64)), "two-dimensional"),
    (dict(x=z(2, 66)), "weight must be"),
    (dict(x=z(2, 0), weight=z(8, 0, dtype=torch.uint8), scales=z(8, 0)), "weight must be"),
    (dict(weight=z(8, 32, dtype=torch.int8)), "weight must be"),
    (dict(weight=z(32, 8, dtype=torch.uint8).t()), "contiguous"),
    (dict(group_size=16), "multiple of 32"),
    (dict(group_size=0), "multiple of 32"),
    (dict(group_size=48), "multiple of 32"),
    (dict(scales=z(8, 2)), "scales"),
    (dict(scales=z(8, 1, dtype=torch.float16)), "scales"),
    (dict(zeros=z(8, 1)), "zeros"),
    (dict(zeros=z(8, 2, dtype=torch.uint8)), "zeros"),
    (dict(x=z(2, 64).requires_grad_()), "no backward"),
    (dict(), "CUDA device"),
])
def test_matvec_refusals(kw, message):
    with pytest.raises(ValueError, match=message):
        matvec(**kw)


def test_matvec_refuses_rows_too_far_apart():
    far = torch.zeros((1 << 23) + 64, dtype=torch.uint8).as_strided((2, 32), ((1 << 23) + 16, 1))
    with pytest.raises(ValueError, match="2\\^23 bytes apart"):
        matvec(weight=far, scales=z(2, 1))


def attention(**kw):
    a = dict(q=z(2, 4, 64), k_cache=z(3, 16, 2, 64), v_cache=z(3, 16, 2, 64), page_table=z(2, 2, dtype=torch.int32),
             lengths=z(2, dtype=torch.int32))
    a.update(kw)
    return blocks.paged_attention(a.pop("q"), a.pop("k_cache"), a.pop("v_cache"), a.pop("page_table"), a.pop("lengths"), **a)


@pytest.mark.parametrize("kw,message", [
    (dict(q=z(2, 4, 64, dtype=torch.float32)), "bfloat16 or float16"),
    (dict(q=z(4, 64)), "batch, q_heads, head_dim"),
    (dict(layout="DHN"), "layout"),
    (dict(q=z(2, 3, 64)), "do not divide"),
    (dict(q=z(2, 0, 64)), "do not divide"),
    (dict(k_cache=z(3, 16, 0, 64), v_cache=z(3, 16, 0, 64)), "do not divide"),
    (dict(q=z(2, 4, 60), k_cache=z(3, 16, 2, 60), v_cache=z(3, 16, 2, 60)), "multiple of 8"),
    (dict(q=z(2, 4, 264), k_cache=z(3, 16, 2, 264), v_cache=z(3, 16, 2, 264)), "multiple of 8"),
    (dict(k_cache=z(3, 16, 2, 72)), "holds heads"),
    (dict(k_cache=z(3, 0, 2, 64), v_cache=z(3, 0, 2, 64)), "page_size"),
    (dict(v_cache=z(3, 16, 2, 72)), "v_cache"),
    (dict(v_cache=z(4, 16, 2, 64)), "v_cache"),
    (dict(k_cache=z(3, 16, 2, 64, dtype=torch.float16)), "k_cache"),
    (dict(q=z(2, 4, 128)[:, :, ::2]), "contiguous"),
    (dict(q=z(2, 4, 65)[:, :, :64]), "strides in multiples of 8"),
    (dict(window=-1), "window"),
    (dict(scale=float("inf")), "scale"),
    (dict(new_k=z(2, 2, 64)), "come together"),
    (dict(new_k=z(2, 2, 64), new_v=z(2, 4, 64)), "new_v"),
    (dict(page_table=z(2, 2, dtype=torch.int64)), "page_table"),
    (dict(page_table=z(3, 2, dtype=torch.int32)), "page_table"),
    (dict(page_table=z(2, 4, dtype=torch.int32)[:, ::2]), "page_table"),
    (dict(lengths=z(2, dtype=torch.int64)), "lengths"),
    (dict(lengths=z(4, dtype=torch.int32)[::2]), "lengths"),
    (dict(new_k=z(2, 2, 64).requires_grad_(), new_v=z(2, 2, 64)), "no backward"),
    (dict(q="q"), "must be a tensor"),
    (dict(), "CUDA device"),
])
def test_attention_refusals(kw, message):
    with pytest.raises(ValueError, match=message):
        attention(**kw)


def operators():
    """Each operator as a function of one activation, with operands of its own beside it."""
    w, st = z(32), z(4, 2, dtype=torch.float32)
    weight, cache, table, lengths = z(8, 16, dtype=torch.uint8), z(3, 16, 2, 32), z(4, 2, dtype=torch.int32), z(4, dtype=torch.int32)
    return {"block_norm": lambda x: blocks.block_norm(x, x, w)[1],
            "block_norm_backward": lambda x: blocks.block_norm_backward(x, x, x, x, w, st)[0],
            "matvec_w4": lambda x: blocks.matvec_w4(x, weight, z(8, 1), group_size=32),
            "paged_attention": lambda x: blocks.paged_attention(x[:, None], cache[:, :, :1], cache[:, :, :1], table, lengths)}


@pytest.mark.parametrize("name", ["block_norm", "block_norm_backward", "matvec_w4", "paged_attention"])
def test_refusals_of_forward_mode_tangents(name):
    """There is no forward-mode gradient: a tangent would be lost without an error."""
    from torch.autograd import forward_ad
    run, x = operators()[name], z(4, 32)
    with forward_ad.dual_level(), pytest.raises(ValueError, match="forward-mode tangent"):
        run(forward_ad.make_dual(x, torch.ones_like(x)))


@pytest.mark.parametrize("name", ["block_norm", "block_norm_backward", "matvec_w4", "paged_attention"])
def test_refusals_of_what_would_go_unseen(name):
    """What follows or records torch's own calls does not see these: vmap, transforms, traces, fake tensors, values that are
    negated on reading."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch._subclasses.fake_tensor import FakeTensorMode
    run, x = operators()[name], z(4, 32)
    with pytest.raises(ValueError, match="CUDA device"):
        run(x)
    with pytest.raises(ValueError, match="plain strided"):
        torch.vmap(run)(z(2, 4, 32))
    with pytest.raises(ValueError, match="plain strided"):
        torch.func.jvp(run, (x,), (x,))
    with pytest.raises(ValueError, match="plain strided"):
        run(torch._neg_view(x))
    with pytest.raises(ValueError, match="traced"):
        make_fx(run)(x)
    with FakeTensorMode(allow_non_fake_inputs=True) as mode, pytest.raises(ValueError, match="traced"):
        run(mode.from_tensor(x))
    with pytest.raises(ValueError, match="traced"):
        torch.jit.trace(run, x, check_trace=False)


def test_attention_refuses_an_append_to_shared_memory():
    new = dict(new_k=z(2, 2, 64), new_v=z(2, 2, 64))
    cache = z(3, 16, 2, 64)
    for kw in (dict(k_cache=z(1, 16, 2, 64).expand(3, -1, -1, -1), v_cache=cache),
               dict(k_cache=cache, v_cache=z(3, 1, 2, 64).expand(-1, 16, -1, -1))):
        with pytest.raises(ValueError, match="share memory"):
            attention(**kw, **new)
        with pytest.raises(ValueError, match="CUDA device"):        # to be read they may
            attention(**kw)
    with pytest.raises(ValueError, match="same memory"):
        attention(k_cache=cache, v_cache=cache, **new)
    both = z(3, 2, 16, 2, 64)
    with pytest.raises(ValueError, match="CUDA device"):
        attention(k_cache=both[:, 0], v_cache=both[:, 1], **new)


# The C entries refuse the same without touching the (made up) addresses.
A = 1 << 20


def c_norm(**kw):
    a = dict(rows=4, gate_rows=0, residual_stride=32, block_stride=32, width=32, dtype=1, pre_dtype=1, post_dtype=0,
             gate_dtype=0, scale=1.0, eps=1e-5, residual=A, block=A, pre_weight=A, post_weight=None, gate=None,
             hidden=A, normed=A, stats=None)
    a.update(kw)
    return K.BlockNorm(**a)


@pytest.mark.parametrize("kw,code", [
    (dict(rows=-1), INVALID), (dict(width=0), INVALID), (dict(width=(1 << 20) + 1), INVALID), (dict(dtype=3), INVALID),
    (dict(pre_dtype=2), INVALID), (dict(post_weight=A, post_dtype=2), INVALID), (dict(gate_rows=3, gate=A), INVALID),
    (dict(gate_rows=2), INVALID), (dict(gate=A), INVALID), (dict(gate_rows=-1, gate=A), INVALID),
    (dict(scale=float("inf")), INVALID), (dict(eps=float("nan")), INVALID), (dict(rows=1 << 36), LIMIT),
    (dict(residual_stride=31), INVALID), (dict(block_stride=-1), INVALID), (dict(residual=None), INVALID),
    (dict(hidden=None), INVALID), (dict(pre_weight=None), INVALID), (dict(block=A + 1), INVALID),
    (dict(pre_weight=A + 2, pre_dtype=0), INVALID), (dict(stats=A + 2), INVALID)])
def test_c_block_norm_refusals(kw, code):
    lib = K.library()
    assert lib.pm_block_norm_device(C.byref(c_norm(**kw)), None) == code
    assert "pm_block_norm_device" in N.last_error()


def test_c_block_norm_backward_refusals():
    lib = K.library()
    job = c_norm(stats=A, hidden=None, normed=None)
    need = lib.pm_block_norm_backward_scratch_bytes(4, 0, 32)
    assert need > 0 and lib.pm_block_norm_backward_scratch_bytes(4, 3, 32) == 0
    full = dict(grad_hidden_stride=32, grad_normed_stride=32, grad_hidden=A, grad_normed=A, grad_residual=A, grad_block=A)

    def call(job=job, scratch=A, size=need, **kw):
        return lib.pm_block_norm_backward_device(C.byref(job), C.byref(K.BlockNormGrads(**{**full, **kw})), scratch, size, None)
    assert call(job=c_norm(stats=None)) == INVALID
    assert call(grad_residual=None) == INVALID
    assert call(grad_hidden_stride=31) == INVALID
    assert call(grad_normed=A + 1) == INVALID
    assert call(scratch=None) == INVALID
    assert call(scratch=A + 16) == INVALID
    assert call(size=need - 1) == INVALID
    assert lib.pm_block_norm_backward_device(None, None, None, 0, None) == INVALID


def c_w4(**kw):
    a = dict(tokens=2, n=8, k=64, group=64, dtype=1, scales_dtype=1, x_stride=64, weight_stride=32, x=A, weight=A, scales=A,
             zeros=None, y=A)
    a.update(kw)
    return K.MatvecW4(**a)


@pytest.mark.parametrize("kw,code", [
    (dict(tokens=-1), INVALID), (dict(n=0), INVALID), (dict(k=0), INVALID), (dict(tokens=1 << 17), LIMIT),
    (dict(n=1 << 25), LIMIT), (dict(k=1 << 25), LIMIT), (dict(group=0), INVALID), (dict(group=40), INVALID),
    (dict(dtype=0), INVALID), (dict(scales_dtype=2), INVALID), (dict(x_stride=63), INVALID), (dict(weight_stride=31), INVALID), (dict(weight_stride=(1 << 23) + 16), LIMIT),
    (dict(x=None), INVALID), (dict(y=None), INVALID), (dict(scales=A + 1), INVALID), (dict(x=A + 1), INVALID)])
def test_c_matvec_refusals(kw, code):
    assert K.library().pm_matvec_w4_device(C.byref(c_w4(**kw)), None, 0, None) == code
    assert "pm_matvec_w4_device" in N.last_error()


def test_c_matvec_wait_limit():
    limit = K.library().pm_matvec_w4_wait_limit
    limit.argtypes, limit.restype = [C.c_uint64], C.c_uint64
    usual = limit(5)
    assert usual == 2 * 10 ** 9 and limit(2 ** 64 - 1) == 5
    assert 10 ** 18 < limit(0) < 2 ** 63 and limit(0) == usual       # a limit that a clock in 64 bits can be added to


def c_attention(**kw):
    a = dict(batch=2, q_heads=4, kv_heads=2, head_dim=64, page_size=16, n_pages=3, table_columns=2, dtype=1, window=0,
             scale=0.125, q_stride=256, q_head_stride=64, k_page_stride=2048, k_token_stride=128, k_head_stride=64,
             v_page_stride=2048, v_token_stride=128, v_head_stride=64, new_k_stride=0, new_k_head_stride=0, new_v_stride=0,
             new_v_head_stride=0, table_stride=2, q=A, k_cache=A, v_cache=A, table=A, lengths=A, new_k=None, new_v=None, out=A,
             lse=None)
    a.update(kw)
    return K.PagedAttention(**a)


@pytest.mark.parametrize("kw,code", [
    (dict(batch=-1), INVALID), (dict(q_heads=3), INVALID), (dict(kv_heads=0), INVALID), (dict(head_dim=60), INVALID),
    (dict(head_dim=264), INVALID), (dict(page_size=0), INVALID), (dict(page_size=65537), INVALID), (dict(n_pages=-1), INVALID),
    (dict(table_columns=-1), INVALID), (dict(window=-1), INVALID), (dict(batch=1 << 23), LIMIT), (dict(dtype=0), INVALID),
    (dict(scale=float("nan")), INVALID), (dict(new_k=A), INVALID), (dict(q=None), INVALID), (dict(table=None), INVALID),
    (dict(k_cache=A + 8), INVALID), (dict(out=A + 8), INVALID), (dict(lengths=A + 2), INVALID), (dict(k_token_stride=65), INVALID),
    (dict(q_stride=-8), INVALID), (dict(table_stride=-1), INVALID)])
def test_c_attention_refusals(kw, code):
    lib = K.library()
    need = lib.pm_paged_attention_scratch_bytes(2, 4, 2, 64)
    assert lib.pm_paged_attention_device(C.byref(c_attention(**kw)), A, need, None) == code
    assert "pm_paged_attention_device" in N.last_error()


def test_c_attention_scratch():
    lib = K.library()
    need = lib.pm_paged_attention_scratch_bytes(2, 4, 2, 64)
    for scratch, size in ((None, need), (A + 16, need), (A, need - 1)):
        assert lib.pm_paged_attention_device(C.byref(c_attention()), scratch, size, None) == INVALID


def test_empty_calls_need_no_device():
    lib = K.library()
    assert lib.pm_block_norm_device(C.byref(c_norm(rows=0)), None) == 0
    assert lib.pm_matvec_w4_device(C.byref(c_w4(tokens=0)), None, 0, None) == 0
    assert lib.pm_paged_attention_device(C.byref(c_attention(batch=0)), None, 0, None) == 0


def test_structs_follow_the_header():
    """Field names and order of every job struct are the header's."""
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "pmb200_blocks.h").read_text(), flags=re.S)
    for name, struct in (("pm_block_norm", K.BlockNorm), ("pm_block_norm_grads", K.BlockNormGrads),
                         ("pm_matvec_w4", K.MatvecW4), ("pm_paged_attention", K.PagedAttention)):
        body = re.search(r"typedef struct \{([^}]*)\} " + name + ";", text).group(1)
        fields = [f.strip().split()[-1].lstrip("*") for line in body.split(";") for f in line.split(",") if f.strip()]
        assert fields == [f for f, _ in struct._fields_], name
