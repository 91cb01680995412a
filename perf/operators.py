"""The operators of a dense encoder over packed bags, as a list of measurable cases.

A packed batch holds several bags (slides) of patch embeddings one behind the other, without padding.  A block of
an encoder over it needs a layer norm over its tokens, rotary positions with several axes (level, row and column of
a patch) and attention in which every token sees its own bag.  The cases cover the three operators in inference and in
training, from a few tokens to whole batches.

Every case is a dict of plain values; ``prepare`` makes on the GPU what a program holds before the call, ``run`` is one
pass: in elementary torch operations where ``own`` is false, through this package's entry points where it is true.
"""
import math

import torch

own = False


def listed():
    return [
        # Inference, last block: only the two CLS tokens of each of four slides ask, over all of their slide's patches.
        dict(name="attn_cls_pool", kind="attn", q_lens="2,2,2,2", k_lens="1021,6007,517,3001", heads=6, kv_heads=6,
             head_dim=64, causal=False, train=False),
        # One new token for each of eight sequences of very different lengths, grouped heads of the NSA configuration.
        dict(name="attn_token_gqa", kind="attn", q_lens="1,1,1,1,1,1,1,1", k_lens="4096,1,131,8191,65,2048,16384,777",
             heads=16, kv_heads=2, head_dim=128, causal=True, train=False),
        # Inference on a packed batch of five slides, from a small biopsy to a resection, 12 heads of 64.
        dict(name="attn_bags_fwd", kind="attn", q_lens="257,1021,4099,2050,8960", k_lens="", heads=12, kv_heads=12,
             head_dim=64, causal=False, train=False),
        # Causal, grouped heads of 128, four packed sequences, one of them a single token.
        dict(name="attn_causal_fwd", kind="attn", q_lens="8192,4099,1,3000", k_lens="", heads=16, kv_heads=2,
             head_dim=128, causal=True, train=False),
        # A training pass over the smallest bags: latency and launches count.
        dict(name="attn_train_small", kind="attn", q_lens="1,63,130,257,512", k_lens="", heads=6, kv_heads=6,
             head_dim=64, causal=False, train=True),
        # A training pass over three ordinary slides.
        dict(name="attn_train_bags", kind="attn", q_lens="6007,1021,1160", k_lens="", heads=12, kv_heads=12,
             head_dim=64, causal=False, train=True),
        # A training pass over one long causal sequence, grouped heads of 128.
        dict(name="attn_train_causal", kind="attn", q_lens="8192", k_lens="", heads=16, kv_heads=2, head_dim=128,
             causal=True, train=True),
        # A training pass over a biopsy's tokens, the default width.
        dict(name="norm_train_biopsy", kind="norm", rows=1023, width=384, dtype="bfloat16", train=True),
        # Inference in 32 bits on patch embeddings (1280 features).
        dict(name="norm_fwd_features", kind="norm", rows=4099, width=1280, dtype="float32", train=False),
        # A training pass over a large packed batch, the width of the 12-layer model.
        dict(name="norm_train_pack", kind="norm", rows=65536, width=768, dtype="bfloat16", train=True),
        # Eight single tokens, 16 query and 2 key heads of 128, one ladder of frequencies shared by three axes.
        dict(name="rope_token", kind="rope", tokens=8, heads=18, head_dim=128, sections="16,24,24", ladder="head",
             pairing="halves", dtype="bfloat16", integer=True, train=False),
        # A training pass, the queries and keys of a 24576-patch slide with level, row and column of every patch.
        dict(name="rope_train_pack", kind="rope", tokens=24576, heads=24, head_dim=64, sections="8,12,12", ladder="axis",
             pairing="adjacent", dtype="bfloat16", integer=False, train=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "tokens", "norm", "norm", "rope", "rope"])
    if kind == "norm":
        width = rng.choice([384, 768, 1280, _log_int(rng, 2, 8192), _log_int(rng, 2, 8192)])
        return dict(kind="norm", rows=_log_int(rng, 1, min(65536, 50_000_000 // width)), width=width,
                    dtype=rng.choice(["bfloat16", "float32", "float16"]), train=rng.random() < 0.6)
    if kind == "rope":
        pairs = rng.choice([32, 40, 48, 64])
        axes = rng.choice([1, 2, 3, 3])
        part = [pairs // axes] * axes
        part[0] += rng.choice([0, pairs - sum(part)])          # sometimes some channels stay as they are
        return dict(kind="rope", tokens=_log_int(rng, 1, 24576), heads=rng.choice([7, 12, 18, 24]), head_dim=2 * pairs,
                    sections=",".join(map(str, part)), ladder=rng.choice(["axis", "head"]),
                    pairing=rng.choice(["adjacent", "halves"]), dtype=rng.choice(["bfloat16", "float32", "float16"]),
                    integer=rng.random() < 0.5, train=rng.random() < 0.5)
    heads, kv_heads, head_dim = rng.choice([(6, 6, 64), (12, 12, 64), (16, 2, 128), (8, 8, 128), (12, 4, 96), (10, 2, 80)])
    causal = rng.random() < 0.5
    if kind == "tokens":        # few queries over many keys
        n = rng.randint(1, 16)
        ks = [_log_int(rng, 1, 16384) for _ in range(n)]
        return dict(kind="attn", q_lens=",".join(str(min(k, rng.choice([1, 1, 2, 5]))) for k in ks),
                    k_lens=",".join(map(str, ks)), heads=heads, kv_heads=kv_heads, head_dim=head_dim, causal=causal,
                    train=rng.random() < 0.3)
    train = rng.random() < 0.5
    total = _log_int(rng, 200, 8192 if train else 14000)
    cuts = sorted(rng.randint(0, total) for _ in range(rng.randint(0, 6)))
    qs = [b - a for a, b in zip([0] + cuts, cuts + [total])]    # lengths of zero among them, by chance
    return dict(kind="attn", q_lens=",".join(map(str, qs)), k_lens="", heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                causal=causal, train=train)


# ------------------------------------------------------------------ inputs
def _ints(text):
    return [int(t) for t in text.split(",")]


def _lengths(case):
    q = _ints(case["q_lens"])
    return q, _ints(case["k_lens"]) if case["k_lens"] else q


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.bfloat16, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)


def _owners(lengths):
    """The sequence of every packed token, and its place in it."""
    n = torch.tensor(lengths, device="cuda")
    seq = torch.repeat_interleave(torch.arange(len(lengths), device="cuda"), n)
    return seq, torch.arange(seq.numel(), device="cuda") - (n.cumsum(0) - n)[seq]


def _positions(case, g):
    """Level, row and column of a patch: whole numbers on the slide's grid, or pixels with an offset of their own."""
    axes = len(_ints(case["sections"]))
    high = torch.tensor([8.0, 512.0, 512.0][:axes], device="cuda")
    p = (torch.rand(case["tokens"], axes, generator=g, device="cuda") * high).floor()
    return p.to(torch.int32) if case["integer"] else p * 224.0 + torch.rand(1, axes, generator=g, device="cuda") * 224.0


def _scales(case):
    return [1.0 if case["integer"] else 1.0 / 224.0] * len(_ints(case["sections"]))


def _inputs(case, seed):
    g, kind, s = _gen(seed), case["kind"], {}
    if kind == "attn":
        ql, kl = _lengths(case)
        h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
        if case["k_lens"]:
            kv = _randn(g, sum(kl), 2 * hk, d)
            s["q"], s["k"], s["v"] = _randn(g, sum(ql), h, d), kv[:, :hk], kv[:, hk:]
        else:               # views of one projection's output
            qkv = _randn(g, sum(ql), h + 2 * hk, d)
            s["q"], s["k"], s["v"] = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
        if case["train"]:
            s["do"] = _randn(g, sum(ql), h, d)
    elif kind == "norm":
        dt, n, e = getattr(torch, case["dtype"]), case["rows"], case["width"]
        s["x"] = _randn(g, n, e, dtype=dt, scale=1.7, shift=0.4)        # a residual stream, with an offset
        s["w"] = _randn(g, e, dtype=torch.float32, scale=0.2, shift=1.0)
        s["b"] = _randn(g, e, dtype=torch.float32, scale=0.2)
        if case["train"]:
            s["dy"] = _randn(g, n, e, dtype=dt)
    else:
        dt = getattr(torch, case["dtype"])
        s["x"] = _randn(g, case["tokens"], case["heads"], case["head_dim"], dtype=dt)
        s["pos"] = _positions(case, g)
        if case["train"]:
            s["dy"] = _randn(g, case["tokens"], case["heads"], case["head_dim"], dtype=dt)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["kind"] == "attn":
        ql, kl = _lengths(case)
        s["q_seq"], s["q_at"] = _owners(ql)
        s["k_seq"], s["k_at"] = _owners(kl)
        s["ahead"] = (torch.tensor(kl, device="cuda") - torch.tensor(ql, device="cuda"))[s["q_seq"]]
    if own:
        import sparse_wsi_vit_b200 as swv
        if case["kind"] == "attn":
            s["plan"] = swv.PackedPlan(ql, kl, heads=case["heads"], kv_heads=case["kv_heads"], causal=case["causal"],
                                       device="cuda")
        elif case["kind"] == "rope":
            s["rope"] = swv.RopeAxes(case["head_dim"], _ints(case["sections"]), scales=_scales(case),
                                     ladder=case["ladder"], pairing=case["pairing"])
        if case["train"]:
            s["leaves"] = [s[n].detach().requires_grad_() for n in ("q", "k", "v", "x", "w", "b") if n in s]
    return s


# ------------------------------------------------------------------ one pass
def _run_own(s):
    import sparse_wsi_vit_b200 as swv
    case = s["case"]
    kind = case["kind"]
    if kind == "attn":
        if not case["train"]:
            o, lse = swv.packed_attention(s["q"], s["k"], s["v"], s["plan"], return_lse=True)
            return {"o": o, "lse": lse}
        o = swv.packed_attention(*s["leaves"], s["plan"])
        dq, dk, dv = torch.autograd.grad(o, s["leaves"], s["do"])
        return {"o": o, "dq": dq, "dk": dk, "dv": dv}
    if kind == "norm":
        if not case["train"]:
            return {"y": swv.layer_norm(s["x"], s["w"], s["b"])}
        y = swv.layer_norm(*s["leaves"])
        dx, dw, db = torch.autograd.grad(y, s["leaves"], s["dy"])
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    if not case["train"]:
        return {"y": swv.rope_axes(s["x"], s["pos"], s["rope"])}
    y = swv.rope_axes(s["leaves"][0], s["pos"], s["rope"])
    return {"y": y, "dx": torch.autograd.grad(y, s["leaves"][0], s["dy"])[0]}


def _attn_plain(s):
    """All pairs of the packed batch at once, (kv heads, group, queries, keys); pairs of other sequences are masked."""
    case = s["case"]
    hk, d = case["kv_heads"], case["head_dim"]
    g = case["heads"] // hk
    scale = d ** -0.5
    heads = lambda t, n: t.float().unflatten(1, (hk, n)).permute(1, 2, 0, 3)      # noqa: E731  (hk, n, tokens, d)
    q, k, v = heads(s["q"], g), heads(s["k"], 1), heads(s["v"], 1)
    see = s["q_seq"][:, None] == s["k_seq"][None]
    if case["causal"]:
        see &= s["k_at"][None] <= (s["q_at"] + s["ahead"])[:, None]
    p = (q @ k.transpose(2, 3)).mul_(scale).masked_fill_(~see, -math.inf)
    m = p.amax(3, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)                   # a row without keys: probabilities and output zero
    p = p.sub_(m).exp_()
    total = p.sum(3, keepdim=True)
    lse = (m + total.log()).squeeze(3)
    p = p.div_(torch.where(total == 0, 1.0, total))
    o = p @ v
    back = lambda t, like: t.permute(2, 0, 1, 3).flatten(1, 2).to(like.dtype)     # noqa: E731  (tokens, heads, d)
    if not case["train"]:
        return {"o": back(o, s["q"]), "lse": lse.flatten(0, 1)}
    do = heads(s["do"], g)
    dv = (p.transpose(2, 3) @ do).sum(1, keepdim=True)
    ds = do @ v.transpose(2, 3)
    ds = ds.sub_((do * o).sum(3, keepdim=True)).mul_(p).mul_(scale)
    dq = ds @ k
    dk = (ds.transpose(2, 3) @ q).sum(1, keepdim=True)
    return {"o": back(o, s["q"]), "dq": back(dq, s["q"]), "dk": back(dk, s["k"]), "dv": back(dv, s["v"])}


def _norm_plain(s):
    x, w, b = s["x"].float(), s["w"], s["b"]
    mean = x.mean(1, keepdim=True)
    xh = x - mean
    rstd = (xh.square().mean(1, keepdim=True) + 1e-5).rsqrt()
    xh = xh * rstd
    y = (xh * w + b).to(s["x"].dtype)
    if "dy" not in s:
        return {"y": y}
    dy = s["dy"].float()
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return {"y": y, "dx": dx.to(s["x"].dtype), "dw": (dy * xh).sum(0), "db": dy.sum(0)}


def _frequencies(case):
    """One row of frequencies for each axis, zero outside its section: (axes, pairs), in 64 bits."""
    sections = _ints(case["sections"])
    pairs = sum(sections)
    n = torch.tensor(sections, device="cuda")
    axis = torch.repeat_interleave(torch.arange(len(sections), device="cuda"), n)
    p = torch.arange(pairs, device="cuda")
    share = p.double() / pairs if case["ladder"] == "head" else (p - (n.cumsum(0) - n)[axis]).double() / n[axis]
    row = (10000.0 ** -share) * torch.tensor(_scales(case), device="cuda", dtype=torch.float64)[axis]
    return torch.where(axis[None] == torch.arange(len(sections), device="cuda")[:, None], row[None], 0.0)


def _rope_plain(s):
    case = s["case"]
    angle = s["pos"].double() @ _frequencies(case)            # angles of far positions: 64 bits
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    r = angle.shape[1]

    def turn(x, sin):
        f = x.float()
        if case["pairing"] == "adjacent":
            a, b = f[..., 0:2 * r:2], f[..., 1:2 * r:2]
            y = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(2)
        else:
            a, b = f[..., :r], f[..., r:2 * r]
            y = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
        return torch.cat([y, f[..., 2 * r:]], dim=-1).to(x.dtype)

    if "dy" not in s:
        return {"y": turn(s["x"], sin)}
    return {"y": turn(s["x"], sin), "dx": turn(s["dy"], -sin)}


def run(state):
    if own:
        return _run_own(state)
    return {"attn": _attn_plain, "norm": _norm_plain, "rope": _rope_plain}[state["case"]["kind"]](state)


# ------------------------------------------------------------------ what a pass cannot do without
def _pairs(case):
    """Visible (query, key) pairs of one head."""
    n = 0
    for lq, lk in zip(*_lengths(case)):
        if not case["causal"]:
            n += lq * lk
        else:               # query i sees i + lk - lq + 1 keys, the last one all
            first = max(0, lk - lq + 1)
            rows = min(lq, lk)
            n += rows * (first + lk) // 2 if lk >= lq else rows * (rows + 1) // 2
    return n


def work(case):
    if case["kind"] == "attn":
        ql, kl = _lengths(case)
        d, h = case["head_dim"], case["heads"]
        rows, keys = 2.0 * sum(ql) * h * d, 2.0 * sum(kl) * case["kv_heads"] * d
        # forward: two products; backward: five (the scores once more)
        if not case["train"]:
            return {"bytes": 2 * rows + 2 * keys + 4.0 * sum(ql) * h, "flops": 4.0 * d * h * _pairs(case)}
        return {"bytes": 4 * rows + 4 * keys, "flops": 14.0 * d * h * _pairs(case)}
    es = 4.0 if case["dtype"] == "float32" else 2.0
    if case["kind"] == "norm":
        n = float(case["rows"]) * case["width"]
        return {"bytes": (4 if case["train"] else 2) * n * es + (16 if case["train"] else 8) * case["width"],
                "flops": (22.0 if case["train"] else 8.0) * n}
    n = float(case["tokens"]) * case["heads"] * case["head_dim"]
    return {"bytes": (4 if case["train"] else 2) * n * es + 4.0 * case["tokens"] * len(_ints(case["sections"])),
            "flops": (6.0 if case["train"] else 3.0) * n}


# ------------------------------------------------------------------ the definitions in 64 bits
def _attn_exact(case, s):
    """Sequence by sequence and head by head."""
    ql, kl = _lengths(case)
    h, d = case["heads"], case["head_dim"]
    group = h // case["kv_heads"]
    q, k, v = (s[n].double() for n in "qkv")
    o, lse = torch.zeros_like(q), q.new_full((h, q.shape[0]), -math.inf)
    grads = [torch.zeros_like(t) for t in (q, k, v)]
    q0 = k0 = 0
    for lq, lk in zip(ql, kl):
        rows, cols = slice(q0, q0 + lq), slice(k0, k0 + lk)
        q0, k0 = q0 + lq, k0 + lk
        if lq == 0 or lk == 0:
            continue
        hidden = None
        if case["causal"]:
            hidden = torch.ones(lq, lk, dtype=torch.bool, device=q.device).triu(lk - lq + 1)
        for i in range(h):
            j = i // group
            logits = torch.einsum("qd,kd->qk", q[rows, i], k[cols, j]) / math.sqrt(d)
            if hidden is not None:
                logits = logits.masked_fill(hidden, -math.inf)
            z = torch.logsumexp(logits, dim=1)
            prob = torch.nan_to_num(torch.exp(logits - z[:, None]), nan=0.0)      # (rows without keys)
            lse[i, rows] = z
            o[rows, i] = torch.einsum("qk,kd->qd", prob, v[cols, j])
            if case["train"]:
                up = s["do"][rows, i].double()
                inner = torch.einsum("qd,kd->qk", up, v[cols, j])
                inner = prob * (inner - (prob * inner).sum(1, keepdim=True)) / math.sqrt(d)
                grads[0][rows, i] = torch.einsum("qk,kd->qd", inner, k[cols, j])
                grads[1][cols, j] += torch.einsum("qk,qd->kd", inner, q[rows, i])
                grads[2][cols, j] += torch.einsum("qk,qd->kd", prob, up)
    if case["train"]:
        return {"o": o, "dq": grads[0], "dk": grads[1], "dv": grads[2]}
    return {"o": o, "lse": lse}


def _norm_exact(case, s):
    x, w, b = s["x"].double(), s["w"].double(), s["b"].double()
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    sd = torch.sqrt(var + 1e-5)
    unit = (x - mean) / sd
    out = {"y": unit * w + b}
    if case["train"]:
        dy = s["dy"].double()
        inner = dy * w
        e = case["width"]
        inner = inner - inner.sum(1, keepdim=True) / e - unit * torch.einsum("ne,ne->n", inner, unit)[:, None] / e
        out.update(dx=inner / sd, dw=torch.einsum("ne,ne->e", dy, unit), db=dy.sum(0))
    return out


def _rope_exact(case, s):
    """The pairs as complex numbers, turned by exp(i angle)."""
    sections = _ints(case["sections"])
    total, angle, first = sum(sections), [], 0
    for a, n in enumerate(sections):
        for i in range(n):
            power = (first + i) / total if case["ladder"] == "head" else i / n
            angle.append(s["pos"][:, a].double() * _scales(case)[a] * math.exp(-power * math.log(10000.0)))
        first += n
    unit = torch.polar(torch.ones_like(angle[0])[:, None], torch.stack(angle, dim=1))[:, None]

    def turn(x, unit):
        x = x.double().clone()
        lo = x[..., 0:2 * total:2] if case["pairing"] == "adjacent" else x[..., :total]
        hi = x[..., 1:2 * total:2] if case["pairing"] == "adjacent" else x[..., total:2 * total]
        z = torch.complex(lo.contiguous(), hi.contiguous()) * unit
        lo.copy_(z.real)
        hi.copy_(z.imag)
        return x

    out = {"y": turn(s["x"], unit)}
    if case["train"]:
        out["dx"] = turn(s["dy"], unit.conj())
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    return {"attn": _attn_exact, "norm": _norm_exact, "rope": _rope_exact}[case["kind"]](case, s)
