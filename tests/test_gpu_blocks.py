"""The block operators on the GPU against their plain 64-bit statements (tests/block_cases.py).

Tolerances count roundings: half a step of the output's type, plus a number of
32-bit roundings of the magnitude of the terms.  A sum of w terms over t
threads carries at most w / t + 16 of them (sequential in a thread, then a
tree), a norm's square root halves its sum's, and each product adds one.
"""
from __future__ import annotations

import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import block_cases as R
from powermodeling_b200 import blocks

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def randn(gen, *shape, dtype=F32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale + shift).to(dtype)


@pytest.fixture
def gen(gpu_ready):
    return torch.Generator(device="cuda").manual_seed(20)


def check(what, got, pair, steps):
    bad, worst = R.within(got, *pair, steps)
    assert not bad, f"{what}: {bad} of {got.numel()} beyond the tolerance, worst {worst:.3g} of it"


# ---------------------------------------------------------------- norms around a block
def norm_inputs(gen, rows, width, dtype, *, post=True, gate_rows=1, weights=None, gate_dtype=None):
    w = weights or dtype
    return dict(residual=randn(gen, rows, width, dtype=dtype, scale=2.0), block=randn(gen, rows, width, dtype=dtype),
                pre=randn(gen, width, dtype=w, scale=0.1, shift=1.0),
                post=randn(gen, width, dtype=w, scale=0.1, shift=1.0) if post else None,
                gate=randn(gen, gate_rows, width, dtype=gate_dtype or w, scale=0.5, shift=0.5) if gate_rows else None)


def norm_both(t, gen, scale=0.75, eps=1e-5, use=("hidden", "normed")):
    """Forward and backward of the inputs `t`, each output checked."""
    rows, width = t["residual"].shape
    steps = width / 32 + 64                      # two norms' sums and about a dozen products
    hidden, normed, stats = blocks.block_norm(t["residual"], t["block"], t["pre"], post_weight=t["post"], gate=t["gate"],
                                              scale=scale, eps=eps, return_stats=True)
    args = (t["residual"], t["block"], t["pre"], t["post"], t["gate"], scale, eps)
    want = R.norm(*args)
    check("hidden", hidden, want["hidden"], steps)
    check("normed", normed, want["normed"], steps)
    gh = randn(gen, rows, width, dtype=hidden.dtype, scale=0.3) if "hidden" in use else None
    gy = randn(gen, rows, width, dtype=hidden.dtype) if "normed" in use else None
    grads = blocks.block_norm_backward(gh, gy, t["residual"], t["block"], t["pre"], stats, post_weight=t["post"],
                                       gate=t["gate"], scale=scale)
    want = R.norm_grads(gh, gy, *args)
    for name, got in zip(("residual", "block", "pre", "post", "gate"), grads):
        if got is None:
            assert name not in want
            continue
        # sums over rows: the rows of one CTA one after the other, then its partial sums
        more = rows + 600 if name in ("pre", "post", "gate") else 0
        check("grad " + name, got, want[name], 3 * steps + more)
    again = blocks.block_norm_backward(gh, gy, t["residual"], t["block"], t["pre"], stats, post_weight=t["post"],
                                       gate=t["gate"], scale=scale)
    for a, b in zip(grads, again):
        assert (a is None and b is None) or torch.equal(a, b)
    return hidden, normed, grads


WIDTHS = [1, 2, 7, 8, 31, 64, 100, 255, 256, 520, 1023, 1024, 1032, 2048, 4096, 5120, 8192, 8200, 12288, 16384, 20000, 33001]


@pytest.mark.parametrize("dtype", [F32, BF, FP])
@pytest.mark.parametrize("width", WIDTHS)
def test_norm_widths(gen, width, dtype):
    for rows in (1, 3, 37):
        norm_both(norm_inputs(gen, rows, width, dtype), gen)


@pytest.mark.parametrize("rows,gate_rows", [(1, 1), (6, 6), (6, 2), (6, 3), (300, 1), (300, 300), (900, 9), (1200, 400),
                                            (2048, 1), (2048, 2), (1500, 500)])
@pytest.mark.parametrize("dtype,weights,gate_dtype", [(BF, BF, BF), (BF, F32, BF), (FP, F32, F32), (F32, F32, F32)])
def test_norm_gates_and_types(gen, rows, gate_rows, dtype, weights, gate_dtype):
    for width in (96, 1000, 99):
        norm_both(norm_inputs(gen, rows, width, dtype, gate_rows=gate_rows, weights=weights, gate_dtype=gate_dtype), gen)


@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("gate_rows", [0, 1, 64])
@pytest.mark.parametrize("use", [("hidden",), ("normed",), ("hidden", "normed")])
def test_norm_parts_left_out(gen, post, gate_rows, use):
    for dtype, width in ((BF, 768), (F32, 77)):
        norm_both(norm_inputs(gen, 64, width, dtype, post=post, gate_rows=gate_rows), gen, use=use)


def test_norm_many_rows(gen):
    norm_both(norm_inputs(gen, 20011, 256, BF), gen)
    norm_both(norm_inputs(gen, 5003, 4096, BF, weights=F32), gen)
    norm_both(norm_inputs(gen, 5000, 1024, FP, gate_rows=5000), gen)


@pytest.mark.parametrize("dtype,width", [(BF, 32776), (BF, 65528), (BF, 65536), (BF, 65544), (F32, 32768), (BF, 32768), (FP, 65535),
                                         (BF, 1 << 20), (F32, (1 << 20) - 1)])
@pytest.mark.parametrize("gate_rows", [1, 5])
def test_norm_widest_rows(gen, dtype, width, gate_rows):
    """Rows that eight CTAs share, the first that nobody shares, and the widest there are."""
    norm_both(norm_inputs(gen, 5, width, dtype, gate_rows=gate_rows), gen)


def test_norm_offsets_beyond_32_bits(gen):
    """Rows that lie more than 2^31 elements apart."""
    held = torch.empty((1 << 32) + 8192, dtype=BF, device="cuda")
    far = held.as_strided((3, 4096), ((1 << 31) + 8, 1))
    far.copy_(randn(gen, 3, 4096, dtype=BF))
    t = norm_inputs(gen, 3, 4096, BF)
    for name in ("residual", "block"):
        norm_both(dict(t, **{name: far}), gen)
    st = blocks.block_norm(t["residual"], t["block"], t["pre"], post_weight=t["post"], gate=t["gate"], return_stats=True)[2]
    args = (t["residual"], t["block"], t["pre"], st)
    near = far.contiguous()
    for gh, gy in ((far, None), (None, far)):
        got = blocks.block_norm_backward(gh, gy, *args, post_weight=t["post"], gate=t["gate"])
        want = blocks.block_norm_backward(None if gh is None else near, None if gy is None else near, *args, post_weight=t["post"],
                                          gate=t["gate"])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    del held, far
    torch.cuda.empty_cache()


def test_norm_row_strides_and_alignment(gen):
    for dtype in (BF, F32):
        for width, pad in ((512, 64), (512, 3), (1024, 8), (333, 5)):
            wide = {k: randn(gen, 40, width + pad, dtype=dtype) for k in ("residual", "block", "gh", "gy")}
            for shift in (0, pad, 1):
                if shift > pad:
                    continue
                part = {k: v[:, shift:shift + width] for k, v in wide.items()}
                t = norm_inputs(gen, 40, width, dtype)
                base = norm_inputs(gen, 40, width, dtype)
                t.update(residual=part["residual"], block=part["block"])
                args = dict(post_weight=t["post"], gate=t["gate"], scale=0.75)
                h, y, st = blocks.block_norm(t["residual"], t["block"], t["pre"], return_stats=True, **args)
                want = R.norm(t["residual"], t["block"], t["pre"], t["post"], t["gate"], 0.75, 1e-5)
                check("hidden", h, want["hidden"], 200)
                check("normed", y, want["normed"], 200)
                g = blocks.block_norm_backward(part["gh"], part["gy"], t["residual"], t["block"], t["pre"], st, **args)
                gw = R.norm_grads(part["gh"], part["gy"], t["residual"], t["block"], t["pre"], t["post"], t["gate"], 0.75, 1e-5)
                for name, got in zip(("residual", "block", "pre", "post", "gate"), g):
                    check("grad " + name, got, gw[name], 900)
                # a weight that starts off a 16-byte boundary
                off = torch.cat((base["pre"][:1], base["pre"]))[1:]
                h2, y2 = blocks.block_norm(base["residual"], base["block"], off, post_weight=base["post"], gate=base["gate"])
                h3, y3 = blocks.block_norm(base["residual"], base["block"], base["pre"], post_weight=base["post"], gate=base["gate"])
                check("normed, shifted weight", y2, R.norm(base["residual"], base["block"], off, base["post"], base["gate"], 1.0, 1e-5)["normed"], 200)
                assert torch.equal(h2.isnan(), h3.isnan())


def test_norm_no_rows(gen):
    t = norm_inputs(gen, 0, 64, BF, gate_rows=1)
    h, y, st = blocks.block_norm(t["residual"], t["block"], t["pre"], post_weight=t["post"], gate=t["gate"], return_stats=True)
    assert h.shape == y.shape == (0, 64) and st.shape == (0, 2)
    g = blocks.block_norm_backward(h, y, t["residual"], t["block"], t["pre"], st, post_weight=t["post"], gate=t["gate"])
    assert g[0].shape == (0, 64) and all(not x.any() for x in g[2:])


def test_norm_zero_rows_and_extreme_values(gen):
    z = torch.zeros(5, 512, device="cuda", dtype=BF)
    one = torch.ones(512, device="cuda", dtype=BF)
    h, y = blocks.block_norm(z, z, one, post_weight=one)
    assert not h.any() and not y.any()
    # values whose squares stay within 32 bits, at both ends; a row with a NaN spoils itself alone
    t = norm_inputs(gen, 6, 512, F32)
    t["residual"][1] *= 1e15
    t["block"][1] *= 1e15
    t["block"][2] *= 1e-15
    norm_both(t, gen)
    t["block"][3, 7] = float("nan")
    t["residual"][4, 9] = float("inf")
    h, y = blocks.block_norm(t["residual"], t["block"], t["pre"], post_weight=t["post"], gate=t["gate"])
    assert y[3].isnan().all() and y[4].isnan().any()
    assert y[[0, 1, 2, 5]].isfinite().all() and h[[0, 1, 2, 5]].isfinite().all()


def test_norm_gradient_against_differences(gen):
    """The formula's gradients and central differences of the 64-bit forward agree, so the kernel's do."""
    t = norm_inputs(gen, 4, 24, F32, gate_rows=2)
    names = ("residual", "block", "pre", "post", "gate")
    gh, gy = randn(gen, 4, 24), randn(gen, 4, 24)
    _, _, stats = blocks.block_norm(t["residual"], t["block"], t["pre"], post_weight=t["post"], gate=t["gate"], scale=0.75,
                                    return_stats=True)
    grads = dict(zip(names, blocks.block_norm_backward(gh, gy, t["residual"], t["block"], t["pre"], stats,
                                                       post_weight=t["post"], gate=t["gate"], scale=0.75)))

    def loss(v):
        f = R.norm(v["residual"], v["block"], v["pre"], v["post"], v["gate"], 0.75, 1e-5)
        return float((f["hidden"][0] * gh.double()).sum() + (f["normed"][0] * gy.double()).sum())

    wide = {k: v.double() for k, v in t.items()}
    for name in names:
        direction = torch.randn(wide[name].shape, generator=gen, device="cuda", dtype=torch.float64)
        step = 1e-5
        up = loss({**wide, name: wide[name] + step * direction})
        down = loss({**wide, name: wide[name] - step * direction})
        slope = float((grads[name].double() * direction).sum())
        # a third derivative of order 100 leaves 1e-8, the loss's 64-bit rounding 1e-9, the kernel's 32 bits 1e-5
        assert math.isclose((up - down) / (2 * step), slope, rel_tol=1e-4, abs_tol=1e-3), name


def test_norm_autograd(gen):
    t = norm_inputs(gen, 60, 384, BF, gate_rows=3, weights=F32, gate_dtype=BF)
    leaves = [x.clone().requires_grad_() for x in t.values()]
    hidden, normed = blocks.block_norm(*leaves[:3], post_weight=leaves[3], gate=leaves[4], scale=0.75)
    assert hidden.requires_grad and normed.requires_grad
    gh, gy = randn(gen, 60, 384, dtype=BF), randn(gen, 60, 384, dtype=BF)
    got = torch.autograd.grad((hidden, normed), leaves, (gh, gy))
    want = R.norm_grads(gh, gy, *t.values(), 0.75, 1e-5)
    for name, g in zip(("residual", "block", "pre", "post", "gate"), got):
        check("grad " + name, g, want[name], 3 * (384 / 32 + 64) + 660)
    # one output used, an expanded incoming gradient, part of the leaves
    hidden, normed = blocks.block_norm(*leaves[:3], post_weight=leaves[3], gate=leaves[4], scale=0.75)
    (g,) = torch.autograd.grad(normed.sum(), [leaves[1]])
    want = R.norm_grads(None, torch.ones_like(normed), *t.values(), 0.75, 1e-5)
    check("grad block", g, want["block"], 3 * (384 / 32 + 64))
    with torch.no_grad():
        assert not blocks.block_norm(*leaves[:3])[0].requires_grad


def test_norm_captured_backward(gen):
    """Forward and backward in one graph, replayed on new inputs; the autograd engine's call under capture is refused."""
    t = norm_inputs(gen, 50, 1024, BF, weights=F32)
    gh, gy = randn(gen, 50, 1024, dtype=BF), randn(gen, 50, 1024, dtype=BF)

    def step():
        h, y, st = blocks.block_norm(t["residual"], t["block"], t["pre"], post_weight=t["post"], gate=t["gate"],
                                     return_stats=True)
        return (h, y) + blocks.block_norm_backward(gh, gy, t["residual"], t["block"], t["pre"], st,
                                                   post_weight=t["post"], gate=t["gate"])
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in (1, 2):
        t["block"].copy_(randn(gen, 50, 1024, dtype=BF))
        gy.copy_(randn(gen, 50, 1024, dtype=BF))
        graph.replay()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


def test_norm_autograd_of_some_inputs(gen):
    """Each input alone asks for its gradient; both outputs or one lead back to it."""
    t = norm_inputs(gen, 12, 96, F32, gate_rows=3)
    gh, gy = randn(gen, 12, 96, dtype=F32), randn(gen, 12, 96, dtype=F32)
    for use in ((True, True), (True, False), (False, True)):
        want = R.norm_grads(gh if use[0] else None, gy if use[1] else None, t["residual"], t["block"], t["pre"], t["post"],
                            t["gate"], 0.5, 1e-5)
        for name in t:
            x = {k: v.clone().requires_grad_(k == name) for k, v in t.items()}
            out = blocks.block_norm(x["residual"], x["block"], x["pre"], post_weight=x["post"], gate=x["gate"], scale=0.5)
            torch.autograd.backward([o for o, u in zip(out, use) if u], [g for g, u in zip((gh, gy), use) if u])
            assert all(x[k].grad is None for k in t if k != name)
            if name in want:
                check("grad " + name, x[name].grad, want[name], 3 * (96 / 32 + 64) + 12 + 600)
            else:
                assert x[name].grad is None or not x[name].grad.any()


def test_norm_autograd_refuses_a_capture(gen):
    """The engine's backward inside a capture is refused, and the capture goes on without it."""
    w, x = randn(gen, 64, dtype=F32).requires_grad_(), randn(gen, 4, 64, dtype=F32)
    out = blocks.block_norm(x, x, w)[1].sum()
    want = blocks.block_norm(x, x, w.detach())[1]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="capture block_norm_backward itself"):
            blocks._BlockNormFunction.backward(None, x, x, None)
        y = blocks.block_norm(x, x, w.detach())[1]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)
    out.backward()
    assert w.grad is not None


def captured_step_inputs(gen):
    t = norm_inputs(gen, 48, 640, BF, gate_rows=3, weights=F32, gate_dtype=BF)
    return t, [v.requires_grad_() for v in t.values()]


@pytest.mark.parametrize("how", ["grad", "backward", "twice"])
def test_norm_training_step_in_a_graph(gen, how):
    """Forward and the autograd engine's backward captured together after a warm-up, replayed on new inputs."""
    t, leaves = captured_step_inputs(gen)
    gh, gy = randn(gen, 48, 640, dtype=BF), randn(gen, 48, 640, dtype=BF)

    def step():
        h, y = blocks.block_norm(*leaves[:3], post_weight=leaves[3], gate=leaves[4], scale=0.75)
        if how == "twice":                       # the second boundary shares the weights
            h, y = blocks.block_norm(h, y, leaves[2], post_weight=leaves[3], gate=leaves[4], scale=0.75)
        if how == "backward":
            for x in leaves:
                x.grad = None
            torch.autograd.backward((h, y), (gh, gy))
            return [x.grad for x in leaves]
        return list(torch.autograd.grad((h, y), leaves, (gh, gy)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        with torch.no_grad():
            for x in leaves:
                x.copy_(randn(gen, *x.shape, dtype=F32, scale=0.5, shift=0.5))
        gy.copy_(randn(gen, 48, 640, dtype=BF))
        graph.replay()
        kept = [x.clone() for x in got]
        for a, b in zip(kept, step()):
            assert torch.equal(a, b)


def test_norm_in_graphed_callables(gen):
    """torch's own way of capturing a module's forward and backward."""
    class Boundary(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.pre, self.post = (torch.nn.Parameter(randn(gen, 256, scale=0.1, shift=1.0)) for _ in range(2))

        def forward(self, r, b):
            return blocks.block_norm(r, b, self.pre, post_weight=self.post)
    plain = Boundary()
    sample = tuple(randn(gen, 32, 256, dtype=BF).requires_grad_() for _ in range(2))
    graphed = torch.cuda.make_graphed_callables(Boundary(), sample)
    graphed.load_state_dict(plain.state_dict())
    for _ in range(2):
        inputs = [randn(gen, 32, 256, dtype=BF) for _ in range(2)]
        results = []
        for module in (graphed, plain):
            leaves = [x.clone().requires_grad_() for x in inputs]
            module.zero_grad()
            h, y = module(*leaves)
            (h.float().square().sum() + y.float().sum()).backward()
            results.append([h.detach().clone(), y.detach().clone()] + [x.grad.clone() for x in (*leaves, module.pre, module.post)])
        for a, b in zip(*results):
            assert torch.equal(a, b)


def test_norm_capture_refuses_leaves_held_by_an_eager_graph(gen):
    """A graph of the default stream over the same leaf: the captured backward to it is refused by name and the capture goes
    on, the forward is not; without that graph the step is captured."""
    w, x = randn(gen, 64).requires_grad_(), randn(gen, 4, 64)

    def step():
        return torch.autograd.grad(blocks.block_norm(x, x, w)[1].square().sum(), [w])[0]
    held = blocks.block_norm(x, x, w)[1].sum()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="still holds pre_weight"):
            step()
        y = blocks.block_norm(x, x, w)[1].detach()
    graph.replay()
    assert torch.equal(y, blocks.block_norm(x, x, w.detach())[1])
    held.backward()
    w.grad = None
    del held
    want = step().clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    assert torch.equal(got, want)


# ---------------------------------------------------------------- 4-bit weights
def w4_inputs(gen, tokens, n, k, dtype, group, zeros, scales=None):
    groups = -(-k // group)
    q = torch.randint(0, 16, (n, k), generator=gen, device="cuda")
    return dict(x=randn(gen, tokens, k, dtype=dtype), q=q, weight=R.pack(q),
                scales=randn(gen, n, groups, scale=0.01, shift=0.0, dtype=scales or dtype),
                zeros=torch.randint(0, 16, (n, groups), generator=gen, device="cuda").to(torch.uint8) if zeros else None)


def w4_check(t, group, got=None):
    if got is None:
        got = blocks.matvec_w4(t["x"], t["weight"], t["scales"], t["zeros"], group_size=group)
    k = t["x"].shape[1]
    # 32 products to a matrix instruction, each accumulation truncated once, a few roundings per group
    check("y", got, R.matvec(t["x"], t["q"], t["scales"], t["zeros"], group), k / 8 + 64)
    return got


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("k", [1, 2, 31, 32, 33, 64, 100, 126, 128, 256, 500, 1000, 1024, 2048 + 32, 4090, 4096, 8192, 11008, 16384 + 64])
def test_w4_depths(gen, k, dtype):
    for group in (32, 64, 128):
        for tokens, n in ((1, 48), (5, 17), (16, 130)):
            w4_check(w4_inputs(gen, tokens, n, k, dtype, group, zeros=group == 64), group)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("k", [512, 4096, 8190, 8192, 11008, 16384 + 64, 28672])
def test_w4_depths_closely(gen, k, dtype):
    """Deep rows, close enough that one weight left out or exchanged would show: the zero point is taken off exactly, so
    the magnitude is |x| |q - z| |scale|.

    Steps of 2^-24: a group's sum in matrix instructions of 16 values, each cut off (2), one for each group added, 32 for
    the sums over warps and CTAs.  At 28672 in groups of 128 they are 2^-15.9 of the magnitude, 0.2 % of a typical output,
    which a single weight makes up 0.6 % of."""
    for group in (32, 128, 96):
        for tokens, n in ((1, 160), (7, 96), (16, 64), (1, 30000)):
            t = w4_inputs(gen, tokens, n, k, dtype, group, zeros=group != 96)
            x, s = t["x"].double(), t["scales"].double().repeat_interleave(group, 1)[:, :k]
            zero = t["zeros"].double().repeat_interleave(group, 1)[:, :k] if t["zeros"] is not None else 8.0
            w = (t["q"].double() - zero) * s
            y = blocks.matvec_w4(t["x"], t["weight"], t["scales"], t["zeros"], group_size=group)
            check("y", y, (x @ w.t(), x.abs() @ w.abs().t()), 2 * group / 16 + -(-k // group) + 32)


@pytest.mark.parametrize("n", [1, 2, 8, 15, 16, 17, 63, 64, 100, 128, 1001, 4096, 20000])
@pytest.mark.parametrize("tokens", [1, 2, 7, 8, 9, 16])
def test_w4_rows_and_tokens(gen, n, tokens):
    w4_check(w4_inputs(gen, tokens, n, 512, BF, 128, zeros=True), 128)
    w4_check(w4_inputs(gen, tokens, n, 2048, FP, 64, zeros=False), 64)


@pytest.mark.parametrize("group", [32, 64, 96, 128, 160, 256, 512, 1024, 4096])
@pytest.mark.parametrize("zeros", [False, True])
def test_w4_groups_and_scale_types(gen, group, zeros):
    for k in (1024, 2600):
        for scales in (BF, F32):
            w4_check(w4_inputs(gen, 3, 200, k, BF, group, zeros, scales), group)


@pytest.mark.parametrize("tokens", [17, 33, 64])
def test_w4_more_tokens_than_one_pass(gen, tokens):
    w4_check(w4_inputs(gen, tokens, 333, 768, BF, 64, True), 64)


@pytest.mark.parametrize("tokens", [1, 2, 4, 8, 9, 16, 21])
@pytest.mark.parametrize("group", [32, 64, 128, 256, 512, 1024])
def test_w4_scales_in_whole_boxes(gen, group, tokens):
    """Groups by the sixteen, whose scales and zero points copies bring; with one group less or more they do not."""
    for groups in (8, 16, 48, 15, 17):
        for zeros in (False, True):
            w4_check(w4_inputs(gen, tokens, 97, group * groups, FP, group, zeros), group)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("tokens,n,k,group", [(1, 14336, 4096, 128), (8, 14336, 4096, 32), (16, 10001, 8192, 64), (3, 40000, 1024, 64),
                                              (16, 9000, 4064, 32), (20, 12288, 2048, 256)])
def test_w4_line_cut_into_runs(gen, tokens, n, k, group, dtype):
    """Matrices large enough that runs end within row blocks, aligned and from odd addresses."""
    t = w4_inputs(gen, tokens, n, k, dtype, group, zeros=True)
    first = w4_check(t, group)
    assert torch.equal(first, blocks.matvec_w4(t["x"], t["weight"], t["scales"], t["zeros"], group_size=group))
    held = torch.full((n, t["weight"].shape[1] + 3), 255, device="cuda", dtype=torch.uint8)
    held[:, 1:-2] = t["weight"]
    w4_check(dict(t, weight=held[:, 1:-2]), group)


@pytest.mark.parametrize("tokens", [128, 129, 300])
def test_w4_many_passes_over_the_tokens(gen, tokens):
    """Runs are cut for so many tokens only; beyond, each pass takes whole row blocks and needs no scratch."""
    w4_check(w4_inputs(gen, tokens, 8200, 16384, BF, 128, zeros=True), 128)
    need = R.library().pm_matvec_w4_scratch_bytes(tokens, 8200, 16384)
    assert (need > 0) == (tokens <= 128) and need < 64 << 20


def test_w4_scales_that_start_anywhere(gen):
    """Scales and zero points from addresses that no copy can start at."""
    t = w4_inputs(gen, 2, 64, 1024, BF, 64, True)
    scales, zeros = torch.empty(64 * 16 + 1, device="cuda", dtype=BF), torch.empty(64 * 16 + 1, device="cuda", dtype=torch.uint8)
    scales[1:], zeros[1:] = t["scales"].view(-1), t["zeros"].view(-1)
    for s in (t["scales"], scales[1:].view(64, 16)):
        for z in (t["zeros"], zeros[1:].view(64, 16)):
            w4_check(dict(t, scales=s, zeros=z), 64)


def test_w4_strides_and_alignment(gen):
    for k, pad_x, pad_w, shift in ((512, 8, 16, 0), (512, 1, 16, 0), (512, 3, 1, 1), (512, 8, 4, 4), (1000, 24, 12, 4), (1001, 5, 7, 3)):
        t = w4_inputs(gen, 6, 77, k, BF, 64, True)
        xs = torch.full((6, k + pad_x), float("nan"), device="cuda", dtype=BF)
        ws = torch.full((77, t["weight"].shape[1] + pad_w + shift), 255, device="cuda", dtype=torch.uint8)
        xs[:, min(shift, pad_x):min(shift, pad_x) + k] = t["x"]
        ws[:, shift:shift + t["weight"].shape[1]] = t["weight"]
        t["x"], t["weight"] = xs[:, min(shift, pad_x):min(shift, pad_x) + k], ws[:, shift:shift + t["weight"].shape[1]]
        w4_check(t, 64)


@pytest.mark.parametrize("tokens", [1, 6, 16])
@pytest.mark.parametrize("k", [500, 1001, 4090, 9001])
def test_w4_aligned_tokens_beside_loose_weights(gen, k, tokens):
    """Tokens from 16-byte boundaries with values that are not numbers behind them; weights from every byte."""
    t = w4_inputs(gen, tokens, 200, k, FP, 64, True)
    xs = torch.full((tokens, (k + 15) // 8 * 8), float("nan"), device="cuda", dtype=FP)
    xs[:, :k] = t["x"]
    t["x"] = xs[:, :k]
    held = torch.full((200 * ((k + 1) // 2 + 1) + 16,), 255, device="cuda", dtype=torch.uint8)
    for shift in (0, 1, 2, 7, 15):
        weight = held[shift:shift + 200 * ((k + 1) // 2 + 1)].view(200, -1)[:, :-1]
        weight.copy_(t["weight"])
        w4_check(dict(t, weight=weight), 64)


def test_w4_values_that_are_not_numbers(gen):
    """A token with an infinity or a NaN spoils its own row of the result and no other."""
    t = w4_inputs(gen, 4, 64, 300, BF, 32, False)
    t["x"][1, 299] = float("inf")
    t["x"][2, 0] = float("nan")
    y = blocks.matvec_w4(t["x"], t["weight"], t["scales"], group_size=32)
    assert y[0].isfinite().all() and y[3].isfinite().all()
    assert y[2].isnan().all() and not y[1].isfinite().any()


def test_one_row_has_no_stride(gen):
    """A single row cut from a wider tensor, however far its next one would be: as if it lay alone."""
    t = w4_inputs(gen, 1, 1, 512, BF, 64, True)
    far = torch.empty(256, device="cuda", dtype=torch.uint8).as_strided((1, 256), ((1 << 23) + 17, 1))
    far.copy_(t["weight"])
    x = torch.empty(1, 513, device="cuda", dtype=BF)[:, :512].copy_(t["x"])
    assert torch.equal(w4_check(dict(t, weight=far, x=x), 64), w4_check(t, 64))
    n = norm_inputs(gen, 1, 512, BF)
    cut = {k: torch.empty(1, 515, device="cuda", dtype=BF)[:, :512].copy_(n[k]) for k in ("residual", "block")}
    for a, b in zip(norm_both(dict(n, **cut), gen)[:2], norm_both(n, gen)[:2]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("tokens,n,k,group,loose", [(1, 1024, 1024, 64, 0), (8, 4096, 4096, 128, 0), (16, 1000, 8192, 64, 0),
                                                    (1, 28672, 8192, 128, 0), (16, 9000, 8192, 32, 0), (40, 9000, 8192, 128, 0),
                                                    (3, 1001, 4090, 128, 1), (9, 20000, 4096, 64, 1), (1, 70000, 256, 64, 0)])
def test_w4_waits_that_run_out(gen, tokens, n, k, group, loose):
    """With limits that a copy's latency passes, every output is right or NaN, whoever gave up; the calls after it are
    as before."""
    limit = R.library().pm_matvec_w4_wait_limit
    limit.argtypes, limit.restype = [R.C.c_uint64], R.C.c_uint64
    t = w4_inputs(gen, tokens, n, k, BF, group, zeros=True)
    if loose:
        held = torch.full((n, t["weight"].shape[1] + 3), 255, device="cuda", dtype=torch.uint8)
        held[:, 1:-2] = t["weight"]
        t["weight"] = held[:, 1:-2]
    args = (t["x"], t["weight"], t["scales"], t["zeros"])
    before = w4_check(t, group)
    lost = []
    try:
        for ns in (1, 200, 400, 500, 600, 700, 800, 900, 1000, 1200, 1500, 2000, 4000):
            limit(ns)
            for _ in range(10):
                y = blocks.matvec_w4(*args, group_size=group)
                fine = ~y.isnan()
                assert torch.equal(y[fine], before[fine]), ns
                lost.append(int(y.numel() - fine.sum()))
    finally:
        limit(0)
    assert lost[0] > 0
    assert torch.equal(blocks.matvec_w4(*args, group_size=group), before)


@pytest.mark.parametrize("k", [32768, 32766])
def test_w4_offsets_beyond_32_bits(gen, k):
    """Weights of more than 2^32 bytes, rows from 16-byte boundaries and from any byte."""
    n, group, tail = 290000, 128, 96
    weight = torch.empty(n, (k + 1) // 2, device="cuda", dtype=torch.uint8)
    for part in weight.split(20000):
        part.copy_(torch.randint(0, 256, part.shape, generator=gen, device="cuda", dtype=torch.uint8))
    assert weight.numel() > 1 << 32
    scales = randn(gen, n, -(-k // group), scale=0.01, dtype=BF)
    for tokens in (2, 12):
        x = randn(gen, tokens, k, dtype=BF)
        y = blocks.matvec_w4(x, weight, scales, group_size=group)
        for rows in (slice(0, tail), slice(n // 2, n // 2 + tail), slice(n - tail, n)):
            q = torch.stack((weight[rows] & 15, weight[rows] >> 4), 2).flatten(1)[:, :k].long()
            check("y", y[:, rows], R.matvec(x, q, scales[rows], None, group), 400)
    del weight
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype,scales", [(BF, BF), (FP, F32)])
@pytest.mark.parametrize("tokens,n,k,group", [(1, 70, 300, 32), (9, 70, 300, 32), (3, 40, 1000, 128), (1, 64, 4096, 32), (16, 33, 5000, 64)])
def test_w4_infinite_scales(gen, tokens, n, k, group, dtype, scales):
    """An infinite scale makes its row infinite, of its group's sum's sign, a NaN not a number; the others know nothing."""
    t = w4_inputs(gen, tokens, n, k, dtype, group, True, scales)
    s, groups = t["scales"], t["scales"].shape[1]
    s[1, groups - 1], s[2, 0], s[3, groups // 2], s[4, groups - 1] = float("inf"), float("-inf"), float("inf"), float("nan")
    zero = t["zeros"].double().repeat_interleave(group, 1)[:, :k]
    sums = torch.zeros(tokens, n, groups * group, dtype=torch.float64, device="cuda")
    sums[:, :, :k] = t["x"].double()[:, None] * (t["q"].double() - zero)
    want = (sums.view(tokens, n, groups, group).sum(3) * s.double()).sum(2)
    y = blocks.matvec_w4(t["x"], t["weight"], s, t["zeros"], group_size=group)
    assert bool(want[:, 1:4].isinf().all())
    assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.isposinf(), want.isposinf()) and torch.equal(y.isneginf(), want.isneginf())


# ---------------------------------------------------------------- paged attention
def cache(gen, lens, hk, d, page, dtype, layout="NHD", columns=None, spare=2, fill=float("nan")):
    """Caches whose pages lie in no order; everything that is not live holds `fill`."""
    b = len(lens)
    used = [-(-max(n, 0) // page) for n in lens]
    columns = max(used + [1]) if columns is None else columns
    pages = sum(used) + spare
    mix = torch.randperm(pages, generator=gen, device="cuda").tolist()
    table = torch.full((b, columns), -1, dtype=torch.int32)
    kc = torch.full((pages, page, hk, d), fill, device="cuda", dtype=dtype)
    vc = kc.clone()
    for i, n in enumerate(lens):
        for c in range(min(used[i], columns)):
            p = mix.pop()
            table[i, c] = p
            m = min(page, n - c * page)
            kc[p, :m] = randn(gen, m, hk, d, dtype=dtype)
            vc[p, :m] = randn(gen, m, hk, d, dtype=dtype)
    if layout == "HND":
        kc, vc = kc.transpose(1, 2).contiguous(), vc.transpose(1, 2).contiguous()
    return kc, vc, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")


def attend(gen, lens, hk, share, d, page, dtype, *, layout="NHD", window=0, new=True, scale=None, q=None, made=None):
    kc, vc, table, lengths = made or cache(gen, lens, hk, d, page, dtype, layout)
    b = len(lens)
    q = randn(gen, b, hk * share, d, dtype=dtype) if q is None else q
    nk, nv = (randn(gen, b, hk, d, dtype=dtype), randn(gen, b, hk, d, dtype=dtype)) if new else (None, None)
    want = R.attention(q, kc, vc, table, lengths, nk, nv, d ** -0.5 if scale is None else scale, window, layout)
    out, lse = blocks.paged_attention(q, kc, vc, table, lengths, new_k=nk, new_v=nv, scale=scale, window=window,
                                      layout=layout, return_lse=True)
    # a score's sum of d products and its scaling, twice in a weight; a weight held in two 16-bit halves is off by
    # 2^-16; the sums over the live positions and the joins
    check("out", out, want[:2], d / 8 + 600)
    empty = torch.isinf(want[2])
    assert torch.equal(torch.isinf(lse) & (lse < 0), empty) and not out[empty].any()
    off = (lse.double() - want[2])[~empty].abs()
    assert bool((off <= (d / 8 + 100) * 2.0 ** -24 * want[3][~empty]).all()), float(off.max())
    assert torch.equal(kc.view(torch.int16), want[4].view(torch.int16))
    assert torch.equal(vc.view(torch.int16), want[5].view(torch.int16))
    return out


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("d", [8, 16, 40, 64, 72, 80, 96, 112, 128, 136, 160, 192, 200, 256])
def test_attention_head_sizes(gen, d, dtype):
    attend(gen, [1, 65, 130, 0, 300], 2, 4, d, 16, dtype)
    attend(gen, [17, 1], 3, 1, d, 8, dtype, layout="HND", new=False)


@pytest.mark.parametrize("share", [1, 2, 3, 4, 5, 7, 8, 9, 12, 16, 17, 32, 40])
def test_attention_shared_heads(gen, share):
    for hk in (1, 3):
        attend(gen, [100, 1, 0, 513], hk, share, 64, 16, BF)
        attend(gen, [260], hk, share, 128, 32, FP)


@pytest.mark.parametrize("page", [1, 2, 3, 8, 16, 17, 48, 64, 100, 128, 1024])
def test_attention_pages(gen, page):
    for layout in ("NHD", "HND"):
        attend(gen, [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 0, 400], 2, 2, 64, page, BF, layout=layout)


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 64, 100, 129, 1000, 5000])
def test_attention_windows(gen, window):
    attend(gen, [1, 16, 17, 100, 130, 1001, 0, 2000], 2, 4, 64, 16, FP, window=window)
    attend(gen, [700, 64], 1, 1, 80, 32, BF, window=window, layout="HND")


def test_attention_long_and_ragged(gen):
    attend(gen, [20000], 2, 4, 128, 64, BF)
    attend(gen, [9000, 3, 0, 1, 777, 4096, 8191], 4, 8, 128, 16, FP)
    attend(gen, [0, 0, 0], 2, 4, 64, 16, BF)
    attend(gen, [1] * 300, 2, 4, 64, 16, BF)
    attend(gen, [33 * (i % 7) for i in range(200)], 8, 1, 64, 16, BF)


@pytest.mark.parametrize("batch,longest", [(1, 256), (5, 128), (18, 256), (60, 256), (130, 200), (300, 64), (700, 130)])
def test_attention_many_short_sequences(gen, batch, longest):
    """Tables of one to four tiles, with a run for each segment and with fewer; some sequences are empty."""
    lens = [0 if i % 7 == 3 else (i * 37) % longest + 1 for i in range(batch)]
    lens[-1] = longest
    attend(gen, lens, 4, 4, 64, 16, BF)
    attend(gen, lens, 4, 4, 64, 16, FP, window=50, new=False)


def test_attention_absent_pages_and_short_tables(gen):
    lens = [200, 150, 64, 100]
    kc, vc, table, lengths = cache(gen, lens, 2, 64, 16, BF)
    table[0, 3] = -1                              # a hole inside
    table[1, 0] = kc.shape[0]                     # just beyond the pool
    table[2] = -7                                 # nothing left
    table[3, 6] = 2 ** 31 - 1                     # the last page, the new token's
    attend(gen, lens, 2, 4, 64, 16, BF, made=(kc, vc, table, lengths))
    attend(gen, lens, 2, 4, 64, 16, BF, made=(kc, vc, table, lengths), window=40)
    # lengths beyond the table's columns, below zero, and as long as they get
    kc, vc, table, _ = cache(gen, lens, 2, 64, 16, BF)
    odd = torch.tensor([2 ** 31 - 1, -5, 10000, -(2 ** 31)], dtype=torch.int32, device="cuda")
    nan = torch.isnan(kc)
    kc[nan], vc[nan] = 0.5, 0.25                   # every entry of the table's pages is live now
    kc2, vc2 = kc.clone(), vc.clone()
    q = randn(gen, 4, 8, 64, dtype=BF)
    nk = randn(gen, 4, 2, 64, dtype=BF)
    out = blocks.paged_attention(q, kc, vc, table, odd, new_k=nk, new_v=nk)
    capped = torch.tensor([table.shape[1] * 16, 0, table.shape[1] * 16, 0], dtype=torch.int32, device="cuda")
    want = R.attention(q, kc2, vc2, table, capped, None, None, 64 ** -0.5, 0, "NHD")
    check("out", out, want[:2], 700)
    assert torch.equal(kc, kc2) and torch.equal(vc, vc2)       # no entry for the new token
    # a table without columns, a pool without pages
    none = torch.zeros(4, 0, dtype=torch.int32, device="cuda")
    out, lse = blocks.paged_attention(q, kc, vc, none, capped, return_lse=True)
    assert not out.any() and torch.isinf(lse).all()
    out = blocks.paged_attention(q, kc[:0], vc[:0], table, capped, new_k=nk, new_v=nk)
    assert not out.any()
    assert blocks.paged_attention(q[:0], kc, vc, table[:0], capped[:0]).shape == (0, 8, 64)


def test_attention_strides(gen):
    """Cuts of wider tensors, heads and tokens in other orders, keys and values in one tensor."""
    lens = [77, 5, 130]
    kc, vc, table, lengths = cache(gen, lens, 2, 64, 16, BF)
    both = torch.stack((kc, vc), 1)               # [pages, 2, page, heads, d]
    k, v = both[:, 0], both[:, 1]
    wide = randn(gen, 3, 3, 8, 64, dtype=BF)      # q, k and v of a fused projection
    q = wide[:, 0]
    nk, nv = wide[:, 1, :2], wide[:, 2, 3:5]
    table2 = torch.cat((table, table), 1)[:, :table.shape[1]]
    assert not table2.is_contiguous()
    want = R.attention(q, k, v, table, lengths, nk, nv, 64 ** -0.5, 0, "NHD")
    out = blocks.paged_attention(q, k, v, table2, lengths, new_k=nk, new_v=nv)
    check("out", out, want[:2], 700)
    assert torch.equal(k.contiguous().view(torch.int16), want[4].view(torch.int16))
    order = randn(gen, 8, 3, 64, dtype=BF).transpose(0, 1)
    want = R.attention(order, k, v, table, lengths, None, None, 0.2, 50, "NHD")
    check("out", blocks.paged_attention(order, k, v, table2, lengths, scale=0.2, window=50), want[:2], 700)


def test_attention_of_many_sequences(gen):
    """100000 sequences of no position or of one, whose value is the answer."""
    b = 100000
    lengths = (torch.rand(b, generator=gen, device="cuda") < 0.7).to(torch.int32)
    table = torch.randperm(b, generator=gen, device="cuda").to(torch.int32)[:, None].contiguous()
    kc, vc = randn(gen, b, 1, 2, 16, dtype=BF), randn(gen, b, 1, 2, 16, dtype=BF)
    nk, nv = randn(gen, b, 2, 16, dtype=BF), randn(gen, b, 2, 16, dtype=BF)
    old = vc.clone()
    out, lse = blocks.paged_attention(randn(gen, b, 4, 16, dtype=BF), kc, vc, table, lengths, new_k=nk, new_v=nv, return_lse=True)
    live = lengths.bool()
    assert torch.equal(out, nv.repeat_interleave(2, 1) * live[:, None, None])
    assert torch.equal(lse.isneginf(), ~live[:, None].expand(-1, 4))
    home = table[:, 0].long()
    assert torch.equal(vc[home[live], 0], nv[live]) and torch.equal(vc[home[~live]], old[home[~live]])


def test_attention_largest_pages(gen):
    attend(gen, [70000, 65536, 3], 1, 2, 16, 65536, BF)
    attend(gen, [65537], 1, 8, 64, 65536, FP, window=40000, layout="HND")


def test_attention_pages_that_are_shared(gen):
    """A prefix whose pages several sequences share, a page twice in one table, caches of one memory that are only read."""
    kc, vc = randn(gen, 12, 16, 2, 64, dtype=BF), randn(gen, 12, 16, 2, 64, dtype=BF)
    table = torch.tensor([[3, 5, 7, 1], [3, 5, 2, 2], [3, 5, 5, 0]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([50, 33, 64], dtype=torch.int32, device="cuda")
    attend(gen, [50, 33, 64], 2, 4, 64, 16, BF, made=(kc, vc, table, lengths))
    attend(gen, [50, 33, 64], 2, 4, 64, 16, BF, made=(kc, kc, table, lengths), new=False)
    attend(gen, [50, 33, 64], 2, 4, 64, 16, BF, made=(kc, vc[:1].expand(12, -1, -1, -1), table, lengths), new=False)


def test_attention_graph_of_a_growing_sequence(gen):
    """One captured call replayed token by token: lengths, tables, queries and new tokens change in place, from an empty
    cache over page and tile ends to sequences that are cut."""
    page, hk, d = 16, 2, 64
    kc, vc = torch.zeros(1200, page, hk, d, dtype=BF, device="cuda"), torch.zeros(1200, page, hk, d, dtype=BF, device="cuda")
    table = torch.full((2, 600), -1, dtype=torch.int32, device="cuda")
    lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
    q, nk, nv = randn(gen, 2, 8, d, dtype=BF), randn(gen, 2, hk, d, dtype=BF), randn(gen, 2, hk, d, dtype=BF)
    blocks.paged_attention(q, kc, vc, table, lengths, new_k=nk, new_v=nv)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = blocks.paged_attention(q, kc, vc, table, lengths, new_k=nk, new_v=nv, return_lse=True)
    for lens in ([0, 0], [1, 0], [2, 1], [16, 15], [17, 16], [64, 63], [65, 64], [66, 1000], [9000, 1001], [9600, 3]):
        for i, n in enumerate(lens):
            used = -(-n // page)
            table[i] = -1
            table[i, :used] = torch.arange(used, device="cuda", dtype=torch.int32) * 2 + i
        lengths.copy_(torch.tensor(lens, dtype=torch.int32))
        for x in (kc, vc, q, nk, nv):
            x.copy_(randn(gen, *x.shape, dtype=BF))
        want = R.attention(q, kc, vc, table, lengths, nk, nv, d ** -0.5, 0, "NHD")
        graph.replay()
        check("out", out, want[:2], 700)
        assert torch.equal(lse.isneginf(), want[2].isneginf())
        assert torch.equal(kc, want[4]) and torch.equal(vc, want[5])


def test_attention_scores_far_apart(gen):
    """Large scores: weights of one and of nothing; a large negative scale; equal scores."""
    lens = [300, 40]
    q = randn(gen, 2, 8, 64, dtype=BF, scale=30.0)
    attend(gen, lens, 2, 4, 64, 16, BF, q=q)
    attend(gen, lens, 2, 4, 64, 16, BF, q=q, scale=-0.5)
    attend(gen, lens, 2, 4, 64, 16, FP, q=torch.zeros(2, 8, 64, dtype=FP, device="cuda"))


def like_definition(out, want, magnitude, steps):
    """Infinities and NaN where the 64-bit form has them, the rest within the tolerance."""
    assert torch.equal(out.isnan(), want.isnan())
    assert torch.equal(out.isposinf(), want.isposinf()) and torch.equal(out.isneginf(), want.isneginf())
    fine = want.isfinite()
    check("out", out[fine], (want[fine], magnitude[fine]), steps)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lens,hk,share,d,page,layout", [([100, 64, 1, 300], 2, 4, 64, 16, "NHD"), ([1000, 7, 2500], 2, 12, 64, 16, "HND"),
                                                         ([40000], 2, 3, 128, 64, "NHD"), ([3000, 200], 1, 9, 192, 8, "NHD")])
def test_attention_infinite_values(gen, lens, hk, share, d, page, layout, dtype):
    """Live infinities of one sign, of both, and NaN, in whole and cut segments, at every weight there is: each spoils its
    own element of the heads that share it, with its sign."""
    kc, vc, table, lengths = cache(gen, lens, hk, d, page, dtype, layout)
    v = vc if layout == "NHD" else vc.transpose(1, 2)
    inf, nan = float("inf"), float("nan")

    def put(i, pos, head, element, value):
        v[table[i, pos // page], pos % page, head, element] = value
    for i, n in enumerate(lens):
        put(i, 0, 0, 0, inf)
        put(i, n // 2, 0, 1, -inf)
        put(i, n // 3, 0, 2, inf)
        put(i, n - n // 4 - 1, 0, 2, -inf if n > 1 else inf)
        put(i, n // 5, hk - 1, 3, nan)
        for pos in range(0, n, 7):
            put(i, pos, hk - 1, 5, -inf)
    q = randn(gen, len(lens), hk * share, d, dtype=dtype)
    nk, nv = randn(gen, len(lens), hk, d, dtype=dtype), randn(gen, len(lens), hk, d, dtype=dtype)
    nv[:, 0, 7], nv[0, 0, 4] = inf, -inf
    for window in (0, 50):
        for far in (1.0, 12.0):                   # weights down to nothing in 32 bits
            want = R.attention(q * far, kc, vc, table, lengths, nk, nv, d ** -0.5, window, layout)
            out = blocks.paged_attention(q * far, kc, vc, table, lengths, new_k=nk, new_v=nv, window=window, layout=layout)
            assert bool(want[0].isinf().any())
            like_definition(out, want[0], want[1], d / 8 + 600)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lens", [[100, 30], [30000, 4000]])
def test_attention_infinite_keys(gen, lens, dtype):
    """A score of infinity makes its row NaN, one of -infinity a weight of nothing, which times an infinity is NaN; the
    other heads know nothing of it.  Only scores of -infinity give zeros."""
    kc, vc, table, lengths = cache(gen, lens, 3, 64, 16, dtype)
    q = randn(gen, 2, 6, 64, dtype=dtype)
    kc[table[0, 1], 3, 0, 5] = float("inf")       # of the scores' own sign in each head
    q[0, 0, 5], q[0, 1, 5] = 1.0, -1.0
    kc[table[1, 0], 2, 1, 6] = float("-inf")
    q[1, 2, 6], q[1, 3, 6] = 2.0, 0.5
    vc[table[1, 0], 2, 1, 9] = float("inf")
    want = R.attention(q, kc, vc, table, lengths, None, None, 0.125, 0, "NHD")
    out, lse = blocks.paged_attention(q, kc, vc, table, lengths, return_lse=True)
    assert bool(want[0][0, 0].isnan().all() and want[0][0, 1].isfinite().all() and want[0][1, 2:4, 9].isnan().all())
    like_definition(out, want[0], want[1].nan_to_num(nan=0.0), 700)
    assert torch.equal(lse.isnan(), want[2].isnan())
    out, lse = blocks.paged_attention(torch.ones_like(q), torch.full_like(kc, float("-inf")), torch.ones_like(vc), table, lengths,
                                      return_lse=True)
    assert not out.any() and bool(lse.isneginf().all())


def test_attention_values_that_are_not_numbers(gen):
    """A live NaN spoils the rows that attend to it and no others; entries that are not live may hold anything
    (every other test's caches are NaN there)."""
    lens = [100, 100]
    kc, vc, table, lengths = cache(gen, lens, 2, 64, 16, BF)
    q = randn(gen, 2, 8, 64, dtype=BF)
    kc[table[0, 2], 3, 1] = float("nan")
    out = blocks.paged_attention(q, kc, vc, table, lengths)
    assert out[0, 4:].isnan().all() and out[0, :4].isfinite().all() and out[1].isfinite().all()


def pages_of(gen, x, page):
    """Rows [batch, length, heads, d] in pages that lie in no order, and the table that finds them."""
    b, n, hk, d = x.shape
    table = torch.randperm(b * n // page, generator=gen, device="cuda").to(torch.int32).view(b, -1)
    pool = torch.empty(b * n // page, page, hk, d, device="cuda", dtype=x.dtype)
    pool[table.view(-1).long()] = x.view(-1, page, hk, d)
    return pool, table


@pytest.mark.parametrize("dtype", [BF, FP])
def test_attention_weights_have_32_bits(gen, dtype):
    """Values that let three weights cancel to 2^-18 of one of them leave an output as small as a weight's error.

    Steps of 2^-24: 4 of the exponential, 6 of three sums in a matrix instruction, which are cut off, 3 of joining four
    warps, one of the division; the scores are below 0.1, which the magnitude counts.  Weights of 16 + 1 bits are off by
    64 steps."""
    b, n, hk, d = 16, 16, 8, 64
    q, k = torch.zeros(b, hk, d, device="cuda"), torch.zeros(b, n, hk, d, device="cuda")
    q[:, :, 0], k[:, :, :, 0] = 1.0, torch.rand(b, n, hk, generator=gen, device="cuda") * -0.1
    q, k = q.to(dtype), k.to(dtype)
    w = torch.softmax(k[..., :1].double(), 1).expand(-1, -1, -1, d)      # the scale is 1
    v = torch.zeros(b, n, hk, d, device="cuda", dtype=dtype)
    at = torch.argsort(torch.rand(b, n, hk, d, generator=gen, device="cuda"), 1)[:, :3]
    one, two, three = w.gather(1, at).unbind(1)
    second = (-one / two).to(dtype)
    third = (-(one + two * second.double()) / three).to(dtype)
    v.scatter_(1, at, torch.stack((torch.ones_like(second), second, third), 1))
    (kc, table), (vc, same) = pages_of(torch.Generator("cuda").manual_seed(7), k, 16), pages_of(torch.Generator("cuda").manual_seed(7), v, 16)
    assert torch.equal(table, same)
    lengths = torch.full((b,), n, device="cuda", dtype=torch.int32)
    want = R.attention(q, kc, vc, table, lengths, None, None, 1.0, 0, "NHD")
    assert float((want[0].abs() / want[1]).median()) < 2.0 ** -15
    check("out", blocks.paged_attention(q, kc, vc, table, lengths, scale=1.0), want[:2], 14)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_attention_small_weights_keep_their_bits(gen, dtype):
    """Two positions, the one with the values a weight of 2^-1 to 2^-24 of the other's."""
    b = 240
    q, k, v = (torch.zeros(*shape, device="cuda") for shape in ((b, 1, 64), (b, 16, 1, 64), (b, 16, 1, 64)))
    q[:, :, :8] = 1.0
    k[:, 0, :, :8] = torch.linspace(0.1, 24.0, b, device="cuda")[:, None, None] * (math.log(2) / 8)
    v[:, 1] = torch.rand(b, 1, 64, generator=gen, device="cuda") * 10000 + 50000
    q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    table = torch.arange(b, device="cuda", dtype=torch.int32)[:, None].contiguous()
    lengths = torch.full((b,), 2, device="cuda", dtype=torch.int32)
    want = R.attention(q, k, v, table, lengths, None, None, 1.0, 0, "NHD")
    check("out", blocks.paged_attention(q, k, v, table, lengths, scale=1.0), want[:2], 24)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_attention_long_sums_are_rounded(gen, dtype):
    """Sums of values that are all positive, over 590 tiles a CTA.  A rounded running sum is off by up to 2^-24 of itself
    in each of 590 slices, either way: six standard deviations are 6 sqrt(590 / 3) = 84 steps; 36 more for a weight and
    its slice.  Sums that are cut off are all off the same way, by 500 steps and more."""
    b, n, d, page = 128, 131072, 64, 64
    k = randn(gen, b, n, 1, d, dtype=dtype, scale=0.03)
    size = torch.rand(b, 1, 1, d, generator=gen, device="cuda") + 1.0      # outputs at every distance from a rounding's border
    v = ((torch.rand(b, n, 1, d, generator=gen, device="cuda") + 0.5) * size).to(dtype)
    kc, table = pages_of(torch.Generator("cuda").manual_seed(7), k, page)
    vc, _ = pages_of(torch.Generator("cuda").manual_seed(7), v, page)
    q = randn(gen, b, 1, d, dtype=dtype)
    out = blocks.paged_attention(q, kc, vc, table, torch.full((b,), n, device="cuda", dtype=torch.int32))
    del kc, vc
    for i in range(b):
        s = (k[i, :, 0].double() * q[i].double()).sum(1) * d ** -0.5
        largest = (k[i, :, 0].double() * q[i].double()).abs().sum(1).amax() * d ** -0.5
        want = (torch.softmax(s, 0)[:, None] * v[i, :, 0].double()).sum(0, keepdim=True)
        half_step = R.HALF[dtype] * 2.0 ** torch.floor(torch.log2(want))
        off = (out[i].double() - want).abs() - half_step
        assert bool((off <= 120 * 2.0 ** -24 * want * (1 + 2 * largest)).all()), i


def test_attention_offsets_beyond_32_bits(gen):
    """A pool whose last pages lie more than 2^32 elements in."""
    page, hk, d = 64, 8, 128
    pages = (1 << 32) // (page * hk * d) + 40
    kc = torch.zeros(pages, page, hk, d, dtype=BF, device="cuda")
    vc = torch.zeros(pages, page, hk, d, dtype=BF, device="cuda")
    table = torch.arange(pages - 8, pages, dtype=torch.int32, device="cuda").reshape(2, 4)
    kc[-8:], vc[-8:] = randn(gen, 8, page, hk, d, dtype=BF), randn(gen, 8, page, hk, d, dtype=BF)
    lengths = torch.tensor([256, 130], dtype=torch.int32, device="cuda")
    q, nk, nv = randn(gen, 2, 32, d, dtype=BF), randn(gen, 2, hk, d, dtype=BF), randn(gen, 2, hk, d, dtype=BF)
    small = table - (pages - 8)
    want = R.attention(q, kc[-8:].clone(), vc[-8:].clone(), small, lengths, nk, nv, d ** -0.5, 0, "NHD")
    out = blocks.paged_attention(q, kc, vc, table, lengths, new_k=nk, new_v=nv)
    check("out", out, want[:2], 700)
    assert torch.equal(kc[-8:], want[4]) and torch.equal(vc[-8:], want[5])
    del kc, vc
    torch.cuda.empty_cache()


@pytest.mark.parametrize("d", [128, 256])
def test_attention_of_the_most_query_heads(gen, d):
    """2^24 query heads of one key head: an output of 2^31 and 2^32 elements, of a sequence without and with positions."""
    heads = 1 << 24
    q = torch.zeros(1, 1, d, dtype=BF, device="cuda").expand(1, heads, d)
    kc, vc = randn(gen, 1, 16, 1, d, dtype=BF), randn(gen, 1, 16, 1, d, dtype=BF)
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    for n in (0, 5):
        lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
        held = torch.ones(1, heads, d, dtype=BF, device="cuda")          # what the output's memory held before
        del held
        out = blocks.paged_attention(q, kc, vc, table, lengths)
        want = blocks.paged_attention(q[:, :1], kc, vc, table, lengths)
        assert torch.equal(want.abs().amax() > 0, lengths[0] > 0)
        assert all(bool((part == want[:, :1]).all()) for part in out.split(1 << 21, 1))
        del out
    torch.cuda.empty_cache()


# ---------------------------------------------------------------- together, on streams, in graphs
def test_decode_layer(gen):
    """A decode layer as it is used: norm, the projections, attention over the cache with its append, norm; three
    tokens one after the other, against the same layer in 64 bits."""
    b, hk, share, d, page, group = 5, 2, 4, 64, 16, 64
    width, heads = 512, 8
    lens = [40, 1, 16, 63, 200]
    kc, vc, table, lengths = cache(gen, [n + 3 for n in lens], hk, d, page, BF)
    lengths = lengths - 3
    pre, post = randn(gen, width, scale=0.1, shift=1.0), randn(gen, width, scale=0.1, shift=1.0)
    gate = randn(gen, width, scale=0.5)
    wqkv = w4_inputs(gen, 1, (heads + 2 * hk) * d, width, BF, group, True)
    wo = w4_inputs(gen, 1, width, heads * d, BF, group, False)
    kr, vr = kc.clone(), vc.clone()

    def weights(t):
        s = t["scales"].double().repeat_interleave(group, 1)
        z = t["zeros"].double().repeat_interleave(group, 1) if t["zeros"] is not None else 8.0
        return (t["q"].double() - z) * s

    for _ in range(3):
        x, blk = randn(gen, b, width, dtype=BF), randn(gen, b, width, dtype=BF)
        lengths = lengths + 1
        h, y = blocks.block_norm(x, blk, pre, post_weight=post, gate=gate)
        qkv = blocks.matvec_w4(y, wqkv["weight"], wqkv["scales"], wqkv["zeros"], group_size=group).view(b, heads + 2 * hk, d)
        att = blocks.paged_attention(qkv[:, :heads], kc, vc, table, lengths, new_k=qkv[:, heads:heads + hk],
                                     new_v=qkv[:, heads + hk:])
        o = blocks.matvec_w4(att.view(b, -1), wo["weight"], wo["scales"], group_size=group)
        h2, y2 = blocks.block_norm(h, o, pre, post_weight=post, gate=gate)
        # in 64 bits from the same inputs, the 16-bit tensors between the operators rounded as they are
        f = R.norm(x, blk, pre, post, gate, 1.0, 1e-5)
        check("hidden", h, f["hidden"], 80)
        check("normed", y, f["normed"], 80)
        qkv64 = (y.double() @ weights(wqkv).t()).view(b, heads + 2 * hk, d)
        assert torch.allclose(qkv.double(), qkv64, rtol=2.0 ** -7, atol=2e-3)
        a64 = R.attention(qkv[:, :heads], kr, vr, table, lengths, qkv[:, heads:heads + hk], qkv[:, heads + hk:],
                          d ** -0.5, 0, "NHD")
        check("attention", att, a64[:2], 700)
        kr, vr = a64[4], a64[5]
        assert torch.equal(kc.view(torch.int16), kr.view(torch.int16)) and torch.equal(vc.view(torch.int16), vr.view(torch.int16))
        check("o", o, R.matvec(att.view(b, -1), wo["q"], wo["scales"], None, group), 128)
        f = R.norm(h, o, pre, post, gate, 1.0, 1e-5)
        check("hidden 2", h2, f["hidden"], 80)
        check("normed 2", y2, f["normed"], 80)


def layer(s):
    h, y = blocks.block_norm(s["x"], s["b"], s["pre"], gate=s["gate"])
    qkv = blocks.matvec_w4(y, s["w"]["weight"], s["w"]["scales"], group_size=64).view(-1, 12, 64)
    att = blocks.paged_attention(qkv[:, :8], s["kc"], s["vc"], s["table"], s["lengths"], new_k=qkv[:, 8:10], new_v=qkv[:, 10:])
    return h, y, qkv, att


def layer_inputs(gen, lens):
    kc, vc, table, lengths = cache(gen, lens, 2, 64, 16, BF, fill=0.0)
    b = len(lens)
    return dict(x=randn(gen, b, 512, dtype=BF), b=randn(gen, b, 512, dtype=BF), pre=randn(gen, 512, dtype=BF),
                gate=randn(gen, 512, dtype=BF), w=w4_inputs(gen, 1, 768, 512, BF, 64, False), kc=kc, vc=vc, table=table,
                lengths=lengths)


def test_graphs_streams_and_repeats(gen):
    """Two captured layers replayed in turn and on two streams at once give what eager calls give, bit for bit."""
    states = [layer_inputs(gen, [700, 3, 0, 129]), layer_inputs(gen, [5000])]
    want = [[x.clone() for x in layer(s)] for s in states]
    for s, w in zip(states, want):
        for _ in range(3):
            for a, b in zip(layer(s), w):
                assert torch.equal(a, b)
    graphs, outs = [], []
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer(s))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        for a, b in zip(o, w):
            assert torch.equal(a, b)
    # eager calls on two streams at once
    got = []
    for _ in range(5):
        for s, st in zip(states, streams):
            with torch.cuda.stream(st):
                got.append((s, layer(s)))
    torch.cuda.synchronize()
    for s, o in got:
        for a, b in zip(o, want[0 if s is states[0] else 1]):
            assert torch.equal(a, b)


def test_two_graphs_with_second_kernels(gen):
    """Two graphs whose calls all leave pieces to a second kernel, replayed on two streams at once."""
    def state(lens, rows):
        t = norm_inputs(gen, rows, 1024, BF)
        stats = blocks.block_norm(t["residual"], t["block"], t["pre"], post_weight=t["post"], gate=t["gate"], return_stats=True)[2]
        kc, vc, table, lengths = cache(gen, lens, 2, 64, 16, BF, fill=0.0)
        return dict(t=t, stats=stats, g=randn(gen, rows, 1024, dtype=BF), w=w4_inputs(gen, 16, 9000, 8192, BF, 128, True),
                    q=randn(gen, len(lens), 8, 64, dtype=BF), kc=kc, vc=vc, table=table, lengths=lengths)

    def step(s):
        t = s["t"]
        grads = blocks.block_norm_backward(s["g"], s["g"], t["residual"], t["block"], t["pre"], s["stats"], post_weight=t["post"],
                                           gate=t["gate"])
        y = blocks.matvec_w4(s["w"]["x"], s["w"]["weight"], s["w"]["scales"], s["w"]["zeros"])
        return [*grads, y, blocks.paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["lengths"])]

    states = [state([9000, 17, 0, 4000], 300), state([30000], 777)]
    want = [[x.clone() for x in step(s)] for s in states]
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in states:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(s))
    for _ in range(30):
        for x in outs[0] + outs[1]:
            x.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            for a, b in zip(o, w):
                assert torch.equal(a, b)


def test_calls_from_new_threads(gen):
    """Each operator as the first thing that a thread does on the GPU, its memory at hand already."""
    from concurrent.futures import ThreadPoolExecutor
    s = layer_inputs(gen, [700, 3, 0, 129])
    t = norm_inputs(gen, 20, 256, BF)
    st = blocks.block_norm(t["residual"], t["block"], t["pre"], return_stats=True)[2]
    calls = [lambda: blocks.block_norm(s["x"], s["b"], s["pre"]),
             lambda: blocks.block_norm_backward(t["block"], t["block"], t["residual"], t["block"], t["pre"], st)[:3],
             lambda: (blocks.matvec_w4(s["x"], s["w"]["weight"], s["w"]["scales"], group_size=64),),
             lambda: (blocks.paged_attention(s["x"].view(4, 8, 64), s["kc"], s["vc"], s["table"], s["lengths"]),)]
    for call in calls:
        want = call()
        torch.cuda.synchronize()
        with ThreadPoolExecutor(1) as pool:
            got = pool.submit(call).result()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_first_calls_of_a_process_from_many_threads(gpu_ready):
    """Eight threads make a process's first calls of one kernel at once, each with another size of shared memory."""
    script = """
import ctypes as C, sys, threading
sys.path.insert(0, "tests")
import torch
import block_cases as R
lib, n, k = R.library(), 4096, 4096
gen = torch.Generator(device="cuda").manual_seed(1)
q = torch.randint(0, 16, (n, k), generator=gen, device="cuda")
weight, scales = R.pack(q), (torch.rand(n, k // 128, generator=gen, device="cuda") * 0.01).bfloat16()
x = [torch.randn(m + 1, k, generator=gen, device="cuda").bfloat16() for m in range(8)]
y = [torch.empty(m + 1, n, device="cuda", dtype=torch.bfloat16) for m in range(8)]
scratch = [torch.empty(max(lib.pm_matvec_w4_scratch_bytes(m + 1, n, k), 256), dtype=torch.uint8, device="cuda") for m in range(8)]
streams = [torch.cuda.Stream() for m in range(8)]
torch.cuda.synchronize()
start, codes = threading.Barrier(8), [None] * 8
def call(m):
    job = R.MatvecW4(tokens=m + 1, n=n, k=k, group=128, dtype=1, scales_dtype=1, x_stride=k, weight_stride=k // 2, x=x[m].data_ptr(),
                     weight=weight.data_ptr(), scales=scales.data_ptr(), zeros=None, y=y[m].data_ptr())
    torch.cuda.current_device()
    start.wait()
    codes[m] = [lib.pm_matvec_w4_device(C.byref(job), scratch[m].data_ptr(), scratch[m].numel(), streams[m].cuda_stream) for _ in range(20)]
threads = [threading.Thread(target=call, args=(m,)) for m in range(8)]
for t in threads: t.start()
for t in threads: t.join()
torch.cuda.synchronize()
assert not any(sum(codes, [])), codes
for m in range(8):
    want, magnitude = R.matvec(x[m], q, scales, None, 128)
    assert R.within(y[m], want, magnitude, k / 8 + 64)[0] == 0, m
print("right")
"""
    done = subprocess.run([sys.executable, "-c", script], capture_output=True, text=True, timeout=300,
                          cwd=Path(__file__).resolve().parent.parent)
    assert done.returncode == 0 and done.stdout.strip() == "right", done.stdout + done.stderr


def test_first_call_of_a_process_inside_a_capture(gpu_ready):
    """Kernels are loaded, their shared memory set and the devices asked on a first call, which may be a captured one."""
    script = """
import torch
from powermodeling_b200 import blocks
gen = torch.Generator(device="cuda").manual_seed(1)
def normal(*shape): return torch.randn(*shape, generator=gen, device="cuda").bfloat16()
r, b, w = normal(64, 2048), normal(64, 2048), normal(2048)
x, q, s = normal(2, 2048), torch.randint(0, 256, (30000, 1024), generator=gen, device="cuda", dtype=torch.uint8), normal(30000, 16)
heads, kc, vc = normal(2, 8, 64), normal(40, 16, 2, 64), normal(40, 16, 2, 64)
table = torch.arange(40, device="cuda", dtype=torch.int32).view(2, 20)
lengths = torch.tensor([320, 100], device="cuda", dtype=torch.int32)
def step():
    h, y, stats = blocks.block_norm(r, b, w, return_stats=True)
    grads = blocks.block_norm_backward(h, y, r, b, w, stats)
    return [h, y, stats, *(g for g in grads if g is not None), blocks.matvec_w4(x, q, s), blocks.paged_attention(heads, kc, vc, table, lengths)]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, step()))
print("same")
"""
    done = subprocess.run([sys.executable, "-c", script], capture_output=True, text=True, timeout=300,
                          cwd=Path(__file__).resolve().parent.parent)
    assert done.returncode == 0 and done.stdout.strip() == "same", done.stdout + done.stderr
