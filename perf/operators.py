"""The operators of a transformer block, as cases that can be measured.

Three operators of one decode layer: the norms around a block with its gate and
residual scale (forward, and forward with backward as a training step runs
them), the product of a few tokens with a matrix of 4-bit weights, and the
attention of one new token per sequence over a paged key-value cache.

``run`` computes the plain form (elementary torch operations in 32 bits,
rounded once at the end) or, with ``own`` set, calls the framework.  ``exact``
states each operator again in 64 bits.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5


# ---------------------------------------------------------------- cases
def _norm(name, rows, width, dtype, *, train=False, post=True, gate="vector", weights="same"):
    return dict(name=name, op="norm", rows=rows, width=width, dtype=dtype, train=train, post=post, gate=gate,
                weights=weights)


def _matvec(name, tokens, n, k, dtype, group, *, zeros=False):
    return dict(name=name, op="matvec", tokens=tokens, n=n, k=k, dtype=dtype, group=group, zeros=zeros)


def _attention(name, batch, kv_heads, share, dim, page, longest, dtype, *, window=0, layout="NHD"):
    return dict(name=name, op="attention", batch=batch, kv_heads=kv_heads, share=share, dim=dim, page=page,
                longest=longest, dtype=dtype, window=window, layout=layout)


def listed():
    return [
        # one token of a decode step: launch latency is all there is
        _norm("norm_token", 1, 4096, "bf16"),
        # a ragged prompt, each sequence modulated by a gate of its own, weights kept in 32 bits
        _norm("norm_prompt", 3 * 613, 5120, "fp16", gate="sequence3", weights="fp32"),
        # a training step's share of one block boundary
        _norm("norm_train", 16384, 8192, "bf16", train=True, weights="fp32"),
        # training in 32 bits at a width that no vector access divides, without a post norm
        _norm("norm_train_odd", 2000, 1023, "fp32", train=True, post=False),
        # a small projection for one token
        _matvec("matvec_small", 1, 1024, 1024, "bf16", 64),
        # odd rows, and a row of weights that ends inside a group and a 16-byte word
        _matvec("matvec_odd", 3, 1001, 4090, "fp16", 128, zeros=True),
        # the widest projection of a large block, one token
        _matvec("matvec_token", 1, 28672, 8192, "bf16", 128),
        # the same matrix the other way round for a batch of sequences, small groups with zero points
        _matvec("matvec_batch", 16, 8192, 28672, "fp16", 32, zeros=True),
        # a conversation's first tokens
        _attention("attention_short", 1, 8, 4, 128, 16, 77, "bf16"),
        # one sequence with a long context: the cache's length has to be split
        _attention("attention_long", 1, 8, 8, 128, 64, 131072, "bf16"),
        # a serving batch: ragged lengths, some slots idle
        _attention("attention_batch", 64, 8, 8, 128, 16, 8192, "fp16"),
        # heads that share nothing, a sliding window, head-major pages, an odd head size
        _attention("attention_window", 16, 16, 1, 80, 32, 5000, "bf16", window=1500, layout="HND"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("norm", "matvec", "attention"))
    if op == "norm":
        width = _log(rng, 64, 16384)
        if rng.random() < 0.7:
            width = max(64, width // 8 * 8)
        rows = _log(rng, 1, max(2, min(65536, (1 << 26) // width)))
        gate = rng.choice(("none", "vector", "full", "sequence%d" % rng.randint(2, 9)))
        if gate.startswith("sequence"):
            s = int(gate[8:])
            rows = s * max(1, rows // s)
        dtype = rng.choice(("bf16", "fp16", "fp32"))
        return {k: v for k, v in _norm("", rows, width, dtype, train=rng.random() < 0.5, post=rng.random() < 0.7,
                                       gate=gate, weights=rng.choice(("same", "fp32"))).items() if k != "name"}
    if op == "matvec":
        k = _log(rng, 128, 32768)
        if rng.random() < 0.75:
            k = k // 32 * 32
        n = _log(rng, 64, min(65536, 28672 * 8192 // k))
        return {a: b for a, b in _matvec("", rng.choice((1, 1, 1, 2, 3, 4, 6, 8, 11, 16)), n, k,
                                         rng.choice(("bf16", "fp16")), rng.choice((32, 64, 128, 256)),
                                         zeros=rng.random() < 0.5).items() if a != "name"}
    kv = rng.choice((1, 2, 4, 8, 16))
    dim = rng.choice((64, 80, 96, 128, 128, 192, 256))
    batch = _log(rng, 1, 128)
    longest = _log(rng, 1, max(2, min(131072, (1 << 28) // (kv * dim * batch))))
    return {a: b for a, b in _attention("", batch, kv, rng.choice((1, 2, 4, 5, 8, 12, 16)), dim,
                                        rng.choice((8, 16, 32, 64, 128)), longest, rng.choice(("bf16", "fp16")),
                                        window=rng.choice((0, 0, _log(rng, 16, 4096))),
                                        layout=rng.choice(("NHD", "HND"))).items() if a != "name"}


def _gates(case):
    """Rows of the gate, 0 without one."""
    g = case["gate"]
    return {"none": 0, "vector": 1, "full": case["rows"]}[g] if not g.startswith("sequence") else int(g[8:])


def _lengths(case):
    """Live positions of each sequence, the new token's among them: spread over the range, the longest first,
    every sixteenth slot of a batch idle."""
    b, longest = case["batch"], case["longest"]
    lens = [max(1, int(longest * (1.0 - (i * 0.6180339887498949) % 1.0))) for i in range(b)]
    return [0 if i % 16 == 15 else n for i, n in enumerate(lens)]


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0, dtype=t):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)

    if case["op"] == "norm":
        n, d, w = case["rows"], case["width"], torch.float32 if case["weights"] == "fp32" else t
        s = _gates(case)
        state = dict(case=case, residual=normal(n, d, scale=2.0), block=normal(n, d),
                     pre=normal(d, scale=0.1, shift=1.0, dtype=w),
                     post=normal(d, scale=0.1, shift=1.0, dtype=w) if case["post"] else None,
                     # a gate per element is an activation, a gate vector a parameter
                     gate=normal(s, d, scale=0.5, shift=0.5, dtype=t if s == n else w) if s else None, alpha=0.75)
        if case["train"]:
            state |= dict(grad_hidden=normal(n, d, scale=0.1), grad_normed=normal(n, d))
        return state
    if case["op"] == "matvec":
        m, n, k, group = case["tokens"], case["n"], case["k"], case["group"]
        groups = -(-k // group)
        x = torch.randn(m, k, generator=g, device="cuda")
        x[:, :: 97] *= 8.0                                   # activations have a few loud channels
        return dict(case=case, x=x.to(t),
                    weight=torch.randint(0, 256, (n, (k + 1) // 2), generator=g, device="cuda", dtype=torch.uint8),
                    scales=(torch.rand(n, groups, generator=g, device="cuda") * 0.01 + 0.005).to(t),
                    zeros=torch.randint(5, 11, (n, groups), generator=g, device="cuda", dtype=torch.uint8)
                    if case["zeros"] else None)
    b, hk, share, d, page = case["batch"], case["kv_heads"], case["share"], case["dim"], case["page"]
    cover = -(-case["longest"] // page)
    lens = _lengths(case)
    order = torch.randperm(b, generator=g, device="cuda")
    lengths = torch.tensor(lens, dtype=torch.int32).cuda()[order]
    pages = sum(-(-n // page) for n in lens) + 3             # a pool with a few pages to spare, in no order
    mix = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    used = (lengths.long() + page - 1) // page
    first = torch.cumsum(used, 0) - used
    slot = torch.arange(cover, device="cuda")[None, :]
    table = torch.where(slot < used[:, None], mix[(first[:, None] + slot).clamp(max=pages - 1)],
                        torch.full((), -1, dtype=torch.int32, device="cuda")).contiguous()
    shape = (pages, page, hk, d) if case["layout"] == "NHD" else (pages, hk, page, d)
    return dict(case=case, q=normal(b, hk * share, d), k_cache=normal(*shape), v_cache=normal(*shape), table=table,
                lengths=lengths, new_k=normal(b, hk, d), new_v=normal(b, hk, d))


# ---------------------------------------------------------------- one pass
def run(state):
    return {"norm": _run_norm, "matvec": _run_matvec, "attention": _run_attention}[state["case"]["op"]](state)


def _run_norm(s):
    train = s["case"]["train"]
    if own:
        from powermodeling_b200 import blocks
        out = blocks.block_norm(s["residual"], s["block"], s["pre"], post_weight=s["post"], gate=s["gate"],
                                scale=s["alpha"], eps=EPS, return_stats=train)
        if not train:
            return {"hidden": out[0], "normed": out[1]}
        grads = blocks.block_norm_backward(s["grad_hidden"], s["grad_normed"], s["residual"], s["block"], s["pre"],
                                           out[2], post_weight=s["post"], gate=s["gate"], scale=s["alpha"])
        return {"hidden": out[0], "normed": out[1], "grads": grads}
    r, b, pre = s["residual"].float(), s["block"].float(), s["pre"].float()
    n, d = r.shape
    post = s["post"].float() if s["post"] is not None else None
    gates = s["gate"].shape[0] if s["gate"] is not None else 0
    gate = s["gate"].float().repeat_interleave(n // gates, 0) if gates else None
    r1 = torch.rsqrt(b.square().mean(1, keepdim=True) + EPS)
    p = b * r1 * post if post is not None else b
    h = r + s["alpha"] * (gate * p if gates else p)
    r2 = torch.rsqrt(h.square().mean(1, keepdim=True) + EPS)
    y = h * r2 * pre
    t = s["residual"].dtype
    if not train:
        return {"hidden": h.to(t), "normed": y.to(t)}
    gh, gy = s["grad_hidden"].float(), s["grad_normed"].float()
    unit = h * r2
    g = gy * pre
    dh = gh + r2 * (g - unit * (g * unit).mean(1, keepdim=True))
    dpre = (gy * unit).sum(0)
    dgate = (s["alpha"] * dh * p).view(gates, n // gates, d).sum(1) if gates else None
    dp = s["alpha"] * (dh * gate if gates else dh)
    dpost = None
    db = dp
    if post is not None:
        bu = b * r1
        dpost = (dp * bu).sum(0).to(s["post"].dtype)
        c = dp * post
        db = r1 * (c - bu * (c * bu).mean(1, keepdim=True))
    return {"hidden": h.to(t), "normed": y.to(t),
            "grads": (dh.to(t), db.to(t), dpre.to(s["pre"].dtype), dpost,
                      dgate.to(s["gate"].dtype) if gates else None)}


def _run_matvec(s):
    c = s["case"]
    if own:
        from powermodeling_b200 import blocks
        return blocks.matvec_w4(s["x"], s["weight"], s["scales"], s["zeros"], group_size=c["group"])
    w = s["weight"]
    q = torch.stack((w & 15, w >> 4), 2).view(w.shape[0], -1)[:, :c["k"]].float()
    z = s["zeros"].float().repeat_interleave(c["group"], 1)[:, :c["k"]] if s["zeros"] is not None else 8.0
    w = (q - z) * s["scales"].float().repeat_interleave(c["group"], 1)[:, :c["k"]]
    return (s["x"].float() @ w.t()).to(s["x"].dtype)


def _run_attention(s):
    c = s["case"]
    q, kc, vc, table, lengths = s["q"], s["k_cache"], s["v_cache"], s["table"], s["lengths"]
    if own:
        from powermodeling_b200 import blocks
        out = blocks.paged_attention(q, kc, vc, table, lengths, new_k=s["new_k"], new_v=s["new_v"],
                                     window=c["window"], layout=c["layout"])
        return {"out": out, "k_cache": kc, "v_cache": vc}
    b, hk, d, page = c["batch"], c["kv_heads"], c["dim"], c["page"]
    # the new token's key and value go to the last live position of each sequence that has one
    at = torch.nonzero(lengths > 0).view(-1)
    last = lengths[at].long() - 1
    home, off = table[at, last // page].long(), last % page
    if c["layout"] == "NHD":
        kc[home, off], vc[home, off] = s["new_k"][at], s["new_v"][at]
        pages = table.long().clamp(min=0)
        k = kc[pages].view(b, -1, hk, d).float()
        v = vc[pages].view(b, -1, hk, d).float()
    else:
        kc[home, :, off], vc[home, :, off] = s["new_k"][at], s["new_v"][at]
        pages = table.long().clamp(min=0)
        k = kc[pages].transpose(2, 3).reshape(b, -1, hk, d).float()
        v = vc[pages].transpose(2, 3).reshape(b, -1, hk, d).float()
    scores = torch.einsum("bhgd,blhd->bhgl", q.float().view(b, hk, -1, d), k) * (1.0 / math.sqrt(d))
    pos = torch.arange(k.shape[1], device=q.device)[None, :]
    live = pos < lengths[:, None]
    if c["window"]:
        live = live & (pos >= lengths[:, None] - c["window"])
    live = live[:, None, None, :]
    scores = scores.masked_fill(~live, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    e = torch.exp(scores - top)
    out = torch.einsum("bhgl,blhd->bhgd", e, v) / e.sum(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny)[..., :1]
    return {"out": out.reshape(b, -1, d).to(q.dtype), "k_cache": kc, "v_cache": vc}


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        n, d = case["rows"], case["width"]
        w = 4 if case["weights"] == "fp32" else e
        gates = _gates(case)
        params = d * w * (2 if case["post"] else 1) + gates * d * (e if gates == n else w)
        if case["train"]:
            return {"bytes": 8.0 * n * d * e + 2 * params, "flops": 40.0 * n * d}
        return {"bytes": 4.0 * n * d * e + params, "flops": 10.0 * n * d}
    if case["op"] == "matvec":
        m, n, k = case["tokens"], case["n"], case["k"]
        groups = -(-k // case["group"])
        return {"bytes": n * ((k + 1) // 2) + n * groups * (3 if case["zeros"] else 2) + 2.0 * m * (k + n),
                "flops": 2.0 * m * n * k}
    hk, share, d = case["kv_heads"], case["share"], case["dim"]
    lens = _lengths(case)
    seen = [min(n, case["window"]) if case["window"] else n for n in lens]
    live = sum(1 for n in lens if n)
    old = sum(seen) - live                                   # the new token's entries are inputs of their own
    byte = 2 * hk * d * 2 * (old + 2 * live) + 2 * 2 * case["batch"] * hk * share * d + 4 * case["batch"]
    return {"bytes": float(byte + 4 * sum(-(-n // case["page"]) for n in seen)),
            "flops": 4.0 * sum(seen) * hk * share * d}


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "matvec":
        m, k, group = case["tokens"], case["k"], case["group"]
        x = s["x"].double()
        y = torch.zeros(m, case["n"], dtype=torch.float64, device=x.device)
        for j in range(s["scales"].shape[1]):
            lo, hi = j * group, min(k, (j + 1) * group)
            byte = s["weight"][:, lo // 2:(hi + 1) // 2].long()
            q = torch.stack((byte % 16, byte // 16), 2).flatten(1)[:, :hi - lo].double()
            zero = s["zeros"][:, j:j + 1].double() if s["zeros"] is not None else 8.0
            y += (x[:, lo:hi] @ (q - zero).t()) * s["scales"][:, j].double()
        return y
    if case["op"] == "attention":
        q, hk, page = s["q"].double(), case["kv_heads"], case["page"]
        b, heads, d = q.shape
        out = torch.zeros_like(q)
        swap = case["layout"] == "HND"
        for i, n in enumerate(s["lengths"].tolist()):
            if n == 0:
                continue
            first = max(0, n - case["window"]) if case["window"] else 0
            lot = s["table"][i, first // page:(n - 1) // page + 1].long()
            part = []
            for cache, new in ((s["k_cache"], s["new_k"]), (s["v_cache"], s["new_v"])):
                rows = cache[lot].transpose(1, 2) if swap else cache[lot]
                rows = rows.reshape(-1, hk, d)[first % page:][:n - first].double()
                rows[-1] = new[i].double()
                part.append(rows.repeat_interleave(heads // hk, 1))
            weight = torch.softmax((part[0] * q[i]).sum(2) / math.sqrt(d), 0)
            out[i] = (weight[:, :, None] * part[1]).sum(0)
        return {"out": out, "k_cache": None, "v_cache": None}
    r, b, w = (s[x].double() for x in ("residual", "block", "pre"))
    n, d = r.shape
    leaves = [r, b, w]
    p = b
    if s["post"] is not None:
        leaves.append(s["post"].double())
    if s["gate"] is not None:
        leaves.append(s["gate"].double())
    for x in leaves:
        x.requires_grad_(case["train"])
    if s["post"] is not None:
        p = b / (b.pow(2).sum(1, keepdim=True) / d + EPS).sqrt() * leaves[3]
    if s["gate"] is not None:
        p = (p.reshape(leaves[-1].shape[0], -1, d) * leaves[-1][:, None, :]).reshape(n, d)
    h = r + s["alpha"] * p
    y = h / (h.pow(2).sum(1, keepdim=True) / d + EPS).sqrt() * w
    if not case["train"]:
        return {"hidden": h, "normed": y}
    grads = list(torch.autograd.grad((h, y), leaves, (s["grad_hidden"].double(), s["grad_normed"].double())))
    more = grads[3:]
    dpost = more.pop(0) if s["post"] is not None else None
    dgate = more.pop(0) if s["gate"] is not None else None
    return {"hidden": h.detach(), "normed": y.detach(), "grads": (*grads[:3], dpost, dgate)}
