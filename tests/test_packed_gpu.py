"""Packed attention, layer norm and multi-axis rotary positions against plain implementations in 64 bits.

Tolerances are worst cases, element by element, from the formulas: a rounding to bf16 is off by at most 2^-8 of the
value (fp16 2^-11, fp32 2^-24), and every place where the kernels round is counted:
  o   : P rounded for the product, o rounded              2^-8 (P |v| + |o|)
  dv  : the same                                          2^-8 (P^T |do| + |dv|)
  dS  : rounded for the product, and delta = do . o from the rounded o
                                                          e_S = 2^-8 |dS| + P (|do| . e_o)
  dq  : scale e_S |k| + 2^-8 |dq|;   dk : scale e_S^T |q| + 2^-8 |dk|
fp32 arithmetic in between is allowed 2 % of the above and 2^-16 of the sums of absolute values (an exponent of a few tens
is off by 2^-20 at most, which is what P is off by)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF = 2.0 ** -8
SLACK, F32 = 1.02, 2.0 ** -16


@pytest.fixture(scope="module")
def swv():
    import sparse_wsi_vit_b200 as m
    yield m
    m.check_status(torch.device("cuda:0"))


def _half(dt):
    return torch.finfo(dt).eps / 2


def _close(got, ref, bound, what):
    err = (got.double() - ref).abs()
    bad = ~(err <= bound)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / bound.clamp_min(1e-300)).max()):.3g} of the bound"


def _qkv(ql, kl, H, Hk, D, seed, fused=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()
    if fused and ql == kl:
        t = r(sum(ql), H + 2 * Hk, D)
        return t[:, :H], t[:, H:H + Hk], t[:, H + Hk:], r(sum(ql), H, D)
    return r(sum(ql), H, D), r(sum(kl), Hk, D), r(sum(kl), Hk, D), r(sum(ql), H, D)


def reference(q, k, v, do, ql, kl, causal, scale=None):
    """All results and their bounds, sequence by sequence, in 64 bits: {name: (value, bound)}."""
    H, Hk, D = q.shape[1], k.shape[1], q.shape[2]
    g = H // Hk
    scale = D ** -0.5 if scale is None else scale
    z = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=t.device)
    o, eo, dq, eq, dk, ek, dv, ev = z(q), z(q), z(q), z(q), z(k), z(k), z(k), z(k)
    lse = torch.full((H, q.shape[0]), -math.inf, dtype=torch.float64, device=q.device)
    el = torch.zeros_like(lse)
    i = j = 0
    for lq, lk in zip(ql, kl):
        a, b = slice(i, i + lq), slice(j, j + lk)
        i, j = i + lq, j + lk
        if not lq or not lk:
            continue
        hd = lambda t, s, rep: t[s].double().transpose(0, 1).repeat_interleave(rep, 0)
        Q, K, V, G = hd(q, a, 1), hd(k, b, g), hd(v, b, g), hd(do, a, 1)
        S = Q @ K.transpose(1, 2) * scale
        mass = Q.abs() @ K.abs().transpose(1, 2) * scale
        if causal:
            hid = torch.ones(lq, lk, dtype=torch.bool, device=q.device).triu(lk - lq + 1)
            S, mass = S.masked_fill(hid, -math.inf), mass.masked_fill(hid, 0.0)
        L = torch.logsumexp(S, 2)
        P = torch.nan_to_num(torch.exp(S - L[..., None]), nan=0.0)
        O = P @ V
        EO = BF * (P @ V.abs() + O.abs()) * SLACK + F32 * (P @ V.abs())
        dP = G @ V.transpose(1, 2)
        dS = P * (dP - (G * O).sum(2, keepdim=True))
        ES = (BF * dS.abs() + P * (G.abs() * EO).sum(2, keepdim=True)) * SLACK + F32 * P * (G.abs() @ V.abs().transpose(1, 2))
        back = lambda t: t.transpose(0, 1)
        fold = lambda t: t.unflatten(0, (Hk, g)).sum(1).transpose(0, 1)
        o[a], eo[a] = back(O), back(EO)
        lse[:, a], el[:, a] = L, mass.amax(2) * 2.0 ** -19 + 2.0 ** -19
        DQ = dS @ K * scale
        dq[a], eq[a] = back(DQ), back(scale * (ES @ K.abs()) + BF * DQ.abs() * SLACK)
        DK, DV = fold(dS.transpose(1, 2) @ Q) * scale, fold(P.transpose(1, 2) @ G)
        dk[b], ek[b] = DK, scale * fold(ES.transpose(1, 2) @ Q.abs()) + BF * DK.abs() * SLACK
        PG = fold(P.transpose(1, 2) @ G.abs())
        dv[b], ev[b] = DV, (BF * (PG + DV.abs())) * SLACK + F32 * PG
    return dict(o=(o, eo), lse=(lse, el), dq=(dq, eq), dk=(dk, ek), dv=(dv, ev))


def _check(swv, q, k, v, do, ql, kl, causal, scale=None):
    plan = swv.PackedPlan(ql, kl, heads=q.shape[1], kv_heads=k.shape[1], causal=causal)
    ref = reference(q, k, v, do, ql, kl, causal, scale)
    o, lse = swv.packed_attention(q, k, v, plan, scale=scale, return_lse=True)
    empty = torch.isinf(ref["lse"][0])
    assert torch.equal(empty, torch.isinf(lse) & (lse < 0))
    _close(torch.where(empty, 0, lse), torch.where(empty, 0, ref["lse"][0]), ref["lse"][1], "lse")
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o2 = swv.packed_attention(*leaves, plan, scale=scale)
    grads = torch.autograd.grad(o2, leaves, do)
    swv.check_status(q.device)
    assert torch.equal(o, o2)
    for name, got in zip(("o", "dq", "dk", "dv"), (o,) + grads):
        _close(got, *ref[name], name)
    return plan, o, grads


SHAPES = [
    ([1], [1], 1, 1, 64, False), ([1], [1], 1, 1, 8, True), ([5], None, 3, 3, 64, False), ([127], None, 2, 2, 64, True),
    ([128], None, 2, 1, 128, True), ([129], None, 2, 2, 128, False), ([256], None, 1, 1, 64, True), ([257], None, 6, 6, 64, False),
    ([130, 1, 0, 700, 64], None, 6, 6, 64, False), ([300, 257, 1], None, 4, 2, 128, True), ([2, 3, 2, 5], None, 8, 8, 32, True),
    ([1, 2, 5], [777, 64, 3000], 16, 2, 128, True), ([2, 2], [6007, 300], 6, 6, 64, False),     # few queries: divided keys
    ([70, 3, 128], [20, 5, 128], 10, 2, 80, True),                                             # rows that see nothing
    ([1000], [2500], 12, 4, 96, True), ([3000], [100], 2, 2, 64, False),                       # divided queries
    ([0, 0], [7, 30], 2, 2, 64, False), ([5, 9], [0, 0], 2, 1, 64, True), ([0], [0], 2, 2, 64, False),    # a side without tokens
    ([200, 30], [0, 40], 2, 2, 64, False), ([0, 10], [30, 20], 3, 1, 128, False), ([40], None, 7, 1, 72, True),
    ([9], [400], 128, 1, 64, True), ([33], [70], 128, 2, 24, False), ([500, 600], None, 16, 2, 40, True),
    ([2048], None, 2, 2, 64, True), ([1025, 1023], None, 4, 4, 128, True),
]


@pytest.mark.parametrize("ql,kl,H,Hk,D,causal", SHAPES)
def test_attention_forward_and_backward(swv, ql, kl, H, Hk, D, causal):
    kl = ql if kl is None else kl
    _check(swv, *_qkv(ql, kl, H, Hk, D, 1), ql, kl, causal)


@pytest.mark.parametrize("scale", [0.02, 1.0])
def test_attention_scale_and_peaked_rows(swv, scale):
    """scale 1 makes rows of one dominant key; keys far apart in size make the stabiliser rise on the way."""
    ql = [300, 411]
    q, k, v, do = _qkv(ql, ql, 4, 2, 64, 2)
    k = (k.float() * torch.linspace(0.2, 3.0, sum(ql), device="cuda")[:, None, None]).bfloat16()
    _check(swv, q, k, v, do, ql, ql, False, scale=scale)


def test_attention_many_sequences_and_lengths_one_and_zero(swv):
    g = torch.Generator().manual_seed(3)
    ql = [int(x) for x in torch.randint(0, 40, (300,), generator=g)] + [1] * 50
    kl = [int(x) for x in torch.randint(0, 60, (350,), generator=g)]
    _check(swv, *_qkv(ql, kl, 4, 2, 64, 3), ql, kl, False)
    _check(swv, *_qkv(ql, kl, 4, 2, 64, 3), ql, kl, True)


def test_attention_layouts(swv):
    """Views with rows on 16 bytes are read as they are, others are copied: head-major, transposed channels, an odd
    offset, an expanded head; the results are those of contiguous tensors, bit for bit."""
    ql = [100, 61]
    q, k, v, do = _qkv(ql, ql, 4, 2, 64, 4, fused=False)
    plan = swv.PackedPlan(ql, heads=4, kv_heads=2)
    want = swv.packed_attention(q, k, v, plan)
    hm = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)
    ch = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)
    def odd(t):
        b = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape)
        return b.copy_(t)
    for f in (hm, ch, odd):
        assert torch.equal(swv.packed_attention(f(q), f(k), f(v), plan), want)
    k1, v1 = k[:, :1].expand(-1, 2, -1), v[:, :1].expand(-1, 2, -1)
    leaves = [t.detach().requires_grad_() for t in (q, k[:, :1].contiguous(), v[:, :1].contiguous())]
    o = swv.packed_attention(leaves[0], leaves[1].expand(-1, 2, -1), leaves[2].expand(-1, 2, -1), plan)
    assert torch.equal(o, swv.packed_attention(q, k1.contiguous(), v1.contiguous(), plan))
    grads = torch.autograd.grad(o, leaves, hm(do))
    two = [t.detach().requires_grad_() for t in (q, k1.contiguous(), v1.contiguous())]
    g2 = torch.autograd.grad(swv.packed_attention(*two, plan), two, do)
    assert torch.equal(grads[0], g2[0])
    for a, b in zip(grads[1:], g2[1:]):                # an expanded head's gradient is the sum over its copies
        assert torch.allclose(a.float(), b.float().sum(1, keepdim=True), rtol=2 ** -7, atol=2 ** -7)


def test_attention_rows_behind_the_last_sequence(swv):
    """A padded buffer: NaN behind the sequences (and between its fields) reaches nothing; with `out` those rows stay
    as they were, without it they are zero, and so are the gradients."""
    ql = [100, 29]
    q, k, v, do = _qkv(ql, ql, 4, 2, 64, 5, fused=False)
    plan = swv.PackedPlan(ql, heads=4, kv_heads=2, causal=True)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = swv.packed_attention(*leaves, plan)
    grads = torch.autograd.grad(o, leaves, do)
    pad = lambda t: torch.cat([t, torch.full_like(t[:37], math.nan)])
    wide = [pad(t).requires_grad_() for t in (q, k, v)]
    ow = swv.packed_attention(*wide, plan)
    gw = torch.autograd.grad(ow, wide, pad(do))
    n = sum(ql)
    for a, b in zip((o,) + grads, (ow,) + gw):
        assert torch.equal(a, b[:n]) and not bool(b[n:].any())
    out = torch.full_like(wide[0], 7.0)
    with torch.no_grad():
        got, lse = swv.packed_attention(*wide, plan, out=out, return_lse=True)
    assert got.data_ptr() == out.data_ptr() and torch.equal(out[:n], o) and bool((out[n:] == 7).all())
    assert bool((lse[:, n:] == -math.inf).all())


def test_attention_nonfinite_values_stay_in_their_sequence(swv):
    """NaN and infinities in one sequence's q, k, v and upstream gradient leave the others' bits alone; a NaN key that
    no row sees (causal, more keys than seen) changes nothing."""
    ql = [70, 200, 33]
    q, k, v, do = _qkv(ql, ql, 4, 4, 64, 6, fused=False)
    plan = swv.PackedPlan(ql, heads=4, causal=True)
    def run(q, k, v, do):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = swv.packed_attention(*leaves, plan)
        return (o,) + torch.autograd.grad(o, leaves, do)
    clean = run(q, k, v, do)
    bad = [t.clone() for t in (q, k, v, do)]
    for t, x in zip(bad, (math.nan, math.inf, -math.inf, math.nan)):
        t[70:270, 1] = x
    for a, b in zip(clean, run(*bad)):
        assert torch.equal(a[:70], b[:70]) and torch.equal(a[270:], b[270:])
        assert torch.equal(a[70:270, 2], b[70:270, 2])
    assert bool(torch.isnan(run(*bad)[0][70:270, 1]).all())
    k2 = k.clone()
    k2[269] = math.nan                                  # the last key of the middle sequence: its last query alone sees it
    o = run(q, k2, v, do)[0]
    assert torch.equal(o[:269], clean[0][:269]) and bool(torch.isnan(o[269]).all())


def test_attention_infinite_logits(swv):
    """Rows as the formula has them: all scores -inf gives NaN, one +inf gives NaN."""
    q = torch.ones(2, 1, 64, device="cuda", dtype=torch.bfloat16)
    k = torch.ones(3, 1, 64, device="cuda", dtype=torch.bfloat16)
    v = torch.ones_like(k)
    plan = swv.PackedPlan([2], [3], heads=1)
    big = k.clone()
    big[:, 0, 0] = -math.inf
    assert bool(torch.isnan(swv.packed_attention(q, big, v, plan)).all())
    big = k.clone()
    big[1, 0, 0] = math.inf
    assert bool(torch.isnan(swv.packed_attention(q, big, v, plan)).all())
    big = k.clone()
    big[1, 0, 0] = -math.inf                            # probability zero
    assert bool((swv.packed_attention(q, big, v, plan) == 1).all())


def test_attention_gradient_against_differences(swv):
    """The kernels' gradients against central differences of the 64-bit definition along random directions."""
    ql, causal = [40, 90], True
    q, k, v, do = _qkv(ql, ql, 4, 2, 64, 7, fused=False)
    plan, _, grads = _check(swv, q, k, v, do, ql, ql, causal)
    ref = reference(q, k, v, do, ql, ql, causal)
    def loss(q, k, v):
        return float((reference(q, k, v, do, ql, ql, causal)["o"][0] * do.double()).sum())
    g = torch.Generator(device="cuda").manual_seed(8)
    base = [t.double() for t in (q, k, v)]
    for i, (got, name) in enumerate(zip(grads, ("dq", "dk", "dv"))):
        d = torch.randn(base[i].shape, generator=g, device="cuda", dtype=torch.float64)
        h = 1e-4
        up, down = [[t + s * h * d if j == i else t for j, t in enumerate(base)] for s in (1, -1)]
        diff = (loss(*up) - loss(*down)) / (2 * h)
        bound = float((ref[name][1] * d.abs()).sum()) + 1e-5 * abs(diff) + 1e-4      # the last: rounding over 2 h
        assert abs(float((got.double() * d).sum()) - diff) <= bound


def test_attention_same_bits_and_captured_graph(swv):
    """Forward and backward twice give the same bits; captured into a graph and replayed on new inputs they give those of the
    eager call; two graphs in turn do not share anything."""
    ql, kl = [3, 500, 130], [900, 500, 260]
    plan = swv.PackedPlan(ql, kl, heads=8, kv_heads=2, causal=True)
    def run(q, k, v, do):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = swv.packed_attention(*leaves, plan)
        return (o.detach(),) + torch.autograd.grad(o, leaves, do)
    sets = [_qkv(ql, kl, 8, 2, 64, s, fused=False) for s in (10, 11)]
    want = [run(*s) for s in sets]
    assert all(torch.equal(a, b) for a, b in zip(want[0], run(*sets[0])))
    graphs = []
    for s in sets:
        buf = [t.clone() for t in s]
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            run(*buf)
        torch.cuda.current_stream().wait_stream(st)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = run(*buf)
        graphs.append((g, buf, res))
    for other in (0, 1, 0):
        for i, (g, buf, res) in enumerate(graphs):
            for b, t in zip(buf, sets[(i + other) % 2]):
                b.copy_(t)
            g.replay()
        torch.cuda.synchronize()
        for i, (g, buf, res) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(res, want[(i + other) % 2]))
    swv.check_status(torch.device("cuda:0"))


def test_attention_two_streams_share_a_plan(swv):
    ql, kl = [2, 2], [9000, 4000]                       # divided: both calls have workspaces
    plan = swv.PackedPlan(ql, kl, heads=6)
    sets = [_qkv(ql, kl, 6, 6, 64, s) for s in (20, 21)]
    want = [swv.packed_attention(*s[:3], plan) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(swv.packed_attention(*sets[i][:3], plan))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, w) for x in g)


def test_offsets_beyond_32_bits(swv):
    """Rows 2^27 elements apart (a long cache's token stride): offsets pass 2^31 elements and 2^32 bytes."""
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB")
    ql = [20]
    q, k, v, do = _qkv(ql, ql, 4, 2, 64, 30, fused=False)
    buf = torch.empty(20, 1 << 27, dtype=torch.bfloat16, device="cuda")
    far = lambda t, c: buf[:, c:c + t[0].numel()].view(t.shape).copy_(t)
    fq, fk, fv, fo = far(q, 0), far(k, 1024), far(v, 2048), far(do, 4096)
    plan = swv.PackedPlan(ql, heads=4, kv_heads=2, causal=True)
    want = swv.packed_attention(q, k, v, plan)
    assert fq.stride(0) == 1 << 27 and torch.equal(swv.packed_attention(fq, fk, fv, plan), want)
    leaves, wide = ([t.detach().requires_grad_() for t in x] for x in ((q, k, v), (fq, fk, fv)))
    for a, b in zip(torch.autograd.grad(swv.packed_attention(*leaves, plan), leaves, do),
                    torch.autograd.grad(swv.packed_attention(*wide, plan), wide, fo)):
        assert torch.equal(a, b)
    x = buf[:, 8192:8192 + 256]
    x.copy_(torch.randn(20, 256, device="cuda"))
    assert torch.equal(swv.layer_norm(x), swv.layer_norm(x.contiguous()))
    rope, pos = swv.RopeAxes(64, (16, 16)), torch.arange(40, device="cuda").view(20, 2)
    assert torch.equal(swv.rope_axes(fq, pos, rope), swv.rope_axes(q, pos, rope))


def test_attention_plan_on_a_side_stream(swv):
    """A plan made on one stream, used on another and dropped at once: its tables are not handed to others too early."""
    ql = [3000]
    q, k, v, _ = _qkv(ql, ql, 4, 4, 64, 31)
    want = swv.packed_attention(q, k, v, swv.PackedPlan(ql, heads=4))
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    got = []
    for _ in range(10):
        plan = swv.PackedPlan(ql, heads=4)
        with torch.cuda.stream(st):
            got.append(swv.packed_attention(q, k, v, plan))
        n = plan._host.size
        del plan
        torch.zeros(n, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_out_buffers_are_checked(swv):
    """`out` shares no memory with the inputs, is in no graph, and a graph that has saved it notices."""
    E = swv._lib.SwvError
    ql = [20]
    q, k, v, _ = _qkv(ql, ql, 4, 2, 64, 32, fused=False)
    plan = swv.PackedPlan(ql, heads=4, kv_heads=2)
    for bad in (q, torch.empty_like(q).requires_grad_()):
        with pytest.raises(E):
            swv.packed_attention(q, k, v, plan, out=bad)
    rope, pos = swv.RopeAxes(64, (16, 16)), torch.zeros(20, 2, device="cuda")
    buf = torch.randn(21, 4, 64, device="cuda")
    with pytest.raises(E):
        swv.rope_axes(buf[:20], pos, rope, out=buf[1:])
    x = torch.randn(20, 4, 64, device="cuda")
    w = torch.randn(20, 4, 64, device="cuda", requires_grad=True)
    y = (w * x).sum()                                  # saves x
    swv.rope_axes(x, pos, rope, out=x)
    with pytest.raises(RuntimeError):
        y.backward()


def test_attention_refusals(swv):
    E = swv._lib.SwvError
    ql = [20]
    q, k, v, _ = _qkv(ql, ql, 4, 2, 64, 1, fused=False)
    plan = swv.PackedPlan(ql, heads=4, kv_heads=2)
    for a in ((q.float(), k, v), (q.half(), k.half(), v.half()), (q[:19], k, v), (q, k[:19], v[:19]), (q, k, v[:, :1]),
              (q[:, :2], k, v), (q[None], k, v), (q, k.cpu(), v), (q[..., :12], k[..., :12], v[..., :12])):
        with pytest.raises(E):
            swv.packed_attention(*a, plan)
    wide = torch.randn(20, 2, 136, device="cuda").bfloat16()
    with pytest.raises(E):
        swv.packed_attention(wide, wide, wide, swv.PackedPlan(ql, heads=2))
    for s in (0.0, -1.0, math.inf, math.nan, 2.0 ** -61, 2.0 ** 61):
        with pytest.raises(E):
            swv.packed_attention(q, k, v, plan, scale=s)
    with pytest.raises(E):
        swv.packed_attention(q, k, v, swv.PackedPlan(ql, heads=4, kv_heads=2, device="cpu"))
    with pytest.raises(E):
        swv.packed_attention(q.requires_grad_(), k, v, plan, out=torch.empty_like(q))
    with pytest.raises(E):
        swv.packed_attention(q.detach(), k, v, plan, out=torch.empty(20, 4, 64, device="cuda"))
    with pytest.raises(E):
        swv.packed_attention(q.detach(), k, v, None)


# --------------------------------------------------------------------------- #
# layer norm
# --------------------------------------------------------------------------- #
def norm_reference(x, w, b, dy, eps):
    """Values and bounds.  A row's sums take at most 100 additions one after the other, 2^-17 of the sum of absolute
    values, so mu is off by 2^-17 max|x| and xh by e = 2^-17 (max|x| rstd + |xh|)."""
    c = 2.0 ** -17
    X, E = x.double(), x.shape[-1]
    W = torch.ones(E, dtype=torch.float64, device=x.device) if w is None else w.double()
    Bv = torch.zeros_like(W) if b is None else b.double()
    mu = X.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((X - mu).square().mean(1, keepdim=True) + eps)
    xh = (X - mu) * rstd
    e = c * (X.abs().amax(1, keepdim=True) * rstd + xh.abs())
    y = xh * W + Bv
    ey = W.abs() * e + 2.0 ** -22 * (y.abs() + Bv.abs())
    out = dict(y=(y, ey))
    if dy is not None:
        G = dy.double() * W
        m0, m1 = G.mean(1, keepdim=True), (G * xh).mean(1, keepdim=True)
        a0, a1 = G.abs().mean(1, keepdim=True), (G * xh).abs().mean(1, keepdim=True)
        dx = rstd * (G - m0 - xh * m1)
        edx = rstd * (c * a0 + e * m1.abs() + xh.abs() * (c * a1 + (G.abs() * e).mean(1, keepdim=True)) +
                      2.0 ** -22 * (G.abs() + a0 + xh.abs() * a1)) + 2 * c * dx.abs()
        n = 2.0 ** -24 * (128 + x.shape[0] / 1000)
        d = dy.double()
        out.update(dx=(dx, edx), dw=((d * xh).sum(0), (d.abs() * e).sum(0) + n * (d * xh).abs().sum(0)),
                   db=(d.sum(0), n * d.abs().sum(0)))
    return out


NORMS = [(1, 1, "float32"), (3, 2, "bfloat16"), (5, 19, "float16"), (1, 384, "bfloat16"), (1023, 384, "bfloat16"), (77, 768, "float16"),
         (300, 768, "float32"), (9, 1000, "bfloat16"), (13, 1024, "float32"), (13, 1025, "float32"), (40, 1280, "bfloat16"),
         (6, 4096, "float16"), (5, 8192, "float32"), (5, 8191, "bfloat16"), (4, 8200, "bfloat16"), (3, 20001, "float32"),
         (5000, 64, "bfloat16"), (4097, 40, "float32"), (700, 6144, "bfloat16")]


@pytest.mark.parametrize("N,E,dt", NORMS)
@pytest.mark.parametrize("shift", [0.4, 300.0])
def test_layer_norm(swv, N, E, dt, shift):
    g = torch.Generator(device="cuda").manual_seed(N * 31 + E)
    dt = getattr(torch, dt)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, dy = (r(N, E) * 1.7 + shift).to(dt).requires_grad_(), r(N, E).to(dt)
    w, b = (1 + 0.2 * r(E)).requires_grad_(), (0.2 * r(E)).requires_grad_()
    ref = norm_reference(x.detach(), w.detach(), b.detach(), dy, 1e-5)
    y = swv.layer_norm(x, w, b)
    grads = torch.autograd.grad(y, (x, w, b), dy)
    for name, got in zip(("y", "dx", "dw", "db"), (y,) + grads):
        v, e = ref[name]
        _close(got, v, e + _half(got.dtype) * (v.abs() + e) + torch.finfo(got.dtype).smallest_normal, name)
    with torch.no_grad():
        assert torch.equal(swv.layer_norm(x, w, b), y)
    again = torch.autograd.grad(swv.layer_norm(x, w, b), (x, w, b), dy)
    assert all(torch.equal(a, c) for a, c in zip(again, grads))


@pytest.mark.parametrize("xdt,ydt,wdt", [("bfloat16", "float32", "bfloat16"), ("float16", "float32", "float32"),
                                         ("float32", "bfloat16", "float16"), ("float32", "float16", "bfloat16")])
@pytest.mark.parametrize("E", [96, 97, 2000, 9001])
def test_layer_norm_types_and_optional_parts(swv, xdt, ydt, wdt, E):
    xdt, ydt, wdt = (getattr(torch, t) for t in (xdt, ydt, wdt))
    g = torch.Generator(device="cuda").manual_seed(E)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    for has_w, has_b in ((True, True), (True, False), (False, True), (False, False)):
        x = r(2, 7, E).to(xdt).requires_grad_()
        w = r(E).to(wdt).requires_grad_() if has_w else None
        b = r(E).to(wdt).requires_grad_() if has_b else None
        dy = r(2, 7, E).to(ydt)
        y = swv.layer_norm(x, w, b, eps=1e-3, out_dtype=ydt)
        assert y.dtype == ydt and y.shape == x.shape
        leaves = [t for t in (x, w, b) if t is not None]
        grads = dict(zip([n for n, t in zip(("dx", "dw", "db"), (x, w, b)) if t is not None],
                         torch.autograd.grad(y, leaves, dy)))
        flat = lambda t: t.detach().reshape(-1, E)
        ref = norm_reference(flat(x), w, b, flat(dy), 1e-3)
        for name, got in dict(y=flat(y), **grads).items():
            v, e = ref[name]
            got = got.reshape(v.shape)
            _close(got, v.detach(), (e + _half(got.dtype) * (v.abs() + e)).detach() + torch.finfo(got.dtype).smallest_normal, name)


def test_layer_norm_layouts_and_empty(swv):
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(50, 3, 128, generator=g, device="cuda")
    w, b = torch.randn(256, generator=g, device="cuda")[::2], torch.randn(128, generator=g, device="cuda")
    want = swv.layer_norm(x, w, b)
    assert torch.equal(swv.layer_norm(x.transpose(0, 1).contiguous().transpose(0, 1), w, b), want)
    assert torch.equal(swv.layer_norm(x.transpose(1, 2).contiguous().transpose(1, 2), w, b), want)
    wide = torch.randn(50, 3, 200, generator=g, device="cuda")
    wide[..., 8:136] = x
    assert torch.equal(swv.layer_norm(wide[..., 8:136], w, b), want)
    odd = torch.empty(50 * 3 * 128 + 1, device="cuda")[1:].view(x.shape).copy_(x)      # scalar form: other order of sums
    assert torch.allclose(swv.layer_norm(odd, w, b), want, rtol=1e-5, atol=1e-5)
    e = torch.empty(0, 128, device="cuda", requires_grad=True)
    wg, bg = w.contiguous().requires_grad_(), b.clone().requires_grad_()
    y = swv.layer_norm(e, wg, bg)
    ge, gw, gb = torch.autograd.grad(y, (e, wg, bg), torch.empty(0, 128, device="cuda"))
    assert y.shape == (0, 128) and ge.shape == (0, 128) and not bool(gw.any()) and not bool(gb.any())
    xb = x.clone().requires_grad_()                    # a broadcast upstream gradient (rows of stride 0)
    g1 = torch.autograd.grad(swv.layer_norm(xb, w, b), xb, torch.ones(1, 1, 128, device="cuda").expand(50, 3, 128))[0]
    g2 = torch.autograd.grad(swv.layer_norm(xb, w, b), xb, torch.ones(50, 3, 128, device="cuda"))[0]
    assert torch.equal(g1, g2)


def test_layer_norm_nonfinite_and_constant_rows(swv):
    x = torch.randn(6, 64, device="cuda")
    clean = swv.layer_norm(x)
    x[1, 3], x[3, 5] = math.nan, math.inf
    x[4] = 7.0
    y = swv.layer_norm(x)
    assert bool(torch.isnan(y[1]).all()) and bool(torch.isnan(y[3]).all()) and not bool(y[4].any())
    assert torch.equal(y[[0, 2, 5]], clean[[0, 2, 5]])


def test_layer_norm_refusals(swv):
    E = swv._lib.SwvError
    x = torch.randn(4, 8, device="cuda")
    w = torch.randn(8, device="cuda")
    for a, kw in (((x, w[:7]), {}), ((x, w, w[:7]), {}), ((x.double(), w), {}), ((x.bfloat16(), w), dict(out_dtype=torch.float16)),
                  ((x, w.cpu()), {}), ((x, w), dict(out_dtype=torch.int32)), ((torch.empty(4, 0, device="cuda"),), {}),
                  ((torch.tensor(1.0, device="cuda"),), {}), ((x, w.double()), {})):
        with pytest.raises(E):
            swv.layer_norm(*a, **kw)


# --------------------------------------------------------------------------- #
# rotary positions
# --------------------------------------------------------------------------- #
def rope_reference(x, pos, sections, scales, ladder, pairing, theta, sign=1.0):
    """Value and bound: sine and cosine are off by 2^-21 at most (the turn is rounded to 2^-25, times 2 pi, and the
    functions by two units), each of two products and their sum by 2^-24."""
    R, hd = sum(sections), x.shape[2]
    ang = []
    for a, n in enumerate(sections):
        for i in range(n):
            p = (sum(sections[:a]) + i) / R if ladder == "head" else i / n
            ang.append(pos[:, a].double() * scales[a] * theta ** -p)
    ang = torch.stack(ang, 1)[:, None] * sign
    X = x.double()
    lo, hi = (slice(0, 2 * R, 2), slice(1, 2 * R, 2)) if pairing == "adjacent" else (slice(0, R), slice(R, 2 * R))
    a, b = X[..., lo], X[..., hi]
    y, e = X.clone(), torch.zeros_like(X)
    y[..., lo], y[..., hi] = a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()
    e[..., lo] = e[..., hi] = 2.0 ** -20 * (a.abs() + b.abs())
    return y, e


ROPES = [(1, 1, 2, (1,), "axis"), (5, 3, 64, (32,), "head"), (70, 18, 128, (16, 24, 24), "head"), (33, 6, 64, (8, 12, 12), "axis"),
         (64, 7, 80, (20, 20), "axis"), (19, 5, 96, (10, 7, 5), "head"), (300, 24, 64, (16, 16), "axis"), (11, 2, 48, (8, 0, 8), "axis"),
         (9, 4, 256, (60, 60), "axis"), (40, 3, 30, (5, 4), "axis"), (3000, 4, 64, (8, 8, 8), "axis"),
         (7, 2, 128, (8,) * 8, "head")]


@pytest.mark.parametrize("T,H,hd,sections,ladder", ROPES)
@pytest.mark.parametrize("pairing", ["adjacent", "halves"])
@pytest.mark.parametrize("dt,pdt", [("bfloat16", "int32"), ("float32", "float32"), ("float16", "int64")])
def test_rope_axes(swv, T, H, hd, sections, ladder, pairing, dt, pdt):
    g = torch.Generator(device="cuda").manual_seed(T * 7 + hd)
    dt, pdt = getattr(torch, dt), getattr(torch, pdt)
    x = torch.randn(T, H, hd, generator=g, device="cuda").to(dt).requires_grad_()
    dy = torch.randn(T, H, hd, generator=g, device="cuda").to(dt)
    pos = (torch.rand(T, len(sections), generator=g, device="cuda") * 200000 - 1000).to(pdt)      # far positions, negative ones
    scales = [1.0 + 0.25 * a for a in range(len(sections))]
    rope = swv.RopeAxes(hd, sections, theta=5000.0, scales=scales, ladder=ladder, pairing=pairing)
    y = swv.rope_axes(x, pos, rope)
    dx, = torch.autograd.grad(y, x, dy)
    for got, src, sign in ((y, x.detach(), 1.0), (dx, dy, -1.0)):
        v, e = rope_reference(src, pos, sections, scales, ladder, pairing, 5000.0, sign)
        _close(got, v, e + _half(dt) * (v.abs() + e) + torch.finfo(dt).smallest_normal, "rope")
    still = slice(2 * sum(sections), hd)
    assert torch.equal(y[..., still], x[..., still])
    z = x.detach().clone()
    assert swv.rope_axes(z, pos, rope, out=z).data_ptr() == z.data_ptr() and torch.equal(z, y)


def test_rope_axes_with_two_axes_is_rope2d(swv):
    x = torch.randn(50, 3, 64, device="cuda")
    c = torch.rand(50, 2, device="cuda") * 224
    got = swv.rope_axes(x, c, swv.RopeAxes(64, (16, 16), scales=(1 / 224, 1 / 224)))
    assert torch.allclose(got, swv.rope2d(x, c, 224.0), atol=2e-6)


def test_rope_axes_layouts_and_empty(swv):
    """The queries and keys of a fused projection as its leading heads, in place and out of place; unaligned views;
    positions with rows of their own distance; no token at all."""
    qkv = torch.randn(40, 12, 64, device="cuda").bfloat16()
    pos = torch.randint(0, 500, (40, 5), device="cuda", dtype=torch.int32)[:, 1:4]
    rope = swv.RopeAxes(64, (8, 12, 12))
    want = swv.rope_axes(qkv[:, :8].contiguous(), pos.contiguous(), rope)
    v = qkv[:, 8:].clone()
    assert torch.equal(swv.rope_axes(qkv[:, :8], pos, rope), want)
    odd = torch.empty(40 * 8 * 64 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(40, 8, 64).copy_(qkv[:, :8])
    assert torch.equal(swv.rope_axes(odd, pos, rope), want)
    assert torch.equal(swv.rope_axes(qkv[:, :8].transpose(1, 2).contiguous().transpose(1, 2), pos, rope), want)
    swv.rope_axes(qkv[:, :8], pos, rope, out=qkv[:, :8])
    assert torch.equal(qkv[:, :8], want) and torch.equal(qkv[:, 8:], v)
    assert swv.rope_axes(qkv[:0, :8], pos[:0], rope).shape == (0, 8, 64)


def test_rope_axes_refusals(swv):
    E = swv._lib.SwvError
    x, pos, rope = torch.randn(4, 2, 8, device="cuda"), torch.zeros(4, 2, device="cuda"), swv.RopeAxes(8, (2, 2))
    for a in ((x[0], pos, rope), (x[..., :6], pos, rope), (x, pos[:3], rope), (x, pos[:, :1], rope), (x, pos.double(), rope),
              (x.double(), pos, rope), (x, pos.cpu(), rope), (x[:, :0], pos, rope)):
        with pytest.raises(E):
            swv.rope_axes(*a)
    with pytest.raises(E):
        swv.rope_axes(x.requires_grad_(), pos, rope, out=torch.empty_like(x))
    with pytest.raises(E):
        swv.rope_axes(x.detach(), pos, rope, out=torch.empty(4, 2, 8, device="cuda").bfloat16())


def test_rope_axes_positions_have_no_gradient(swv):
    """Positions that ask for a gradient are refused instead of getting none; without gradients they are taken."""
    x, pos, rope = torch.randn(4, 2, 8, device="cuda"), torch.ones(4, 2, device="cuda"), swv.RopeAxes(8, (2, 2))
    want = swv.rope_axes(x, pos, rope)
    pos.requires_grad_()
    with pytest.raises(swv._lib.SwvError):
        swv.rope_axes(x, pos, rope)
    with torch.no_grad():
        assert torch.equal(swv.rope_axes(x, pos, rope), want)


def test_out_buffers_hold_every_element_once(swv):
    E = swv._lib.SwvError
    rope, pos = swv.RopeAxes(64, (16, 16)), torch.zeros(20, 2, device="cuda")
    x = torch.randn(20, 1, 64, device="cuda").expand(20, 4, 64)          # the heads share their memory
    wide = torch.empty(20, 4, 128, device="cuda")
    lapped = torch.empty(4000, device="cuda").as_strided((20, 4, 64), (64, 64, 1))
    for t, bad in ((x, x), (x, lapped)):
        with pytest.raises(E):
            swv.rope_axes(t, pos, rope, out=bad)
    assert torch.equal(swv.rope_axes(x, pos, rope, out=wide[..., :64]), swv.rope_axes(x, pos, rope))
    heads_first = torch.empty(4, 20, 64, device="cuda").transpose(0, 1)  # another order of the dimensions
    assert torch.equal(swv.rope_axes(x, pos, rope, out=heads_first), swv.rope_axes(x, pos, rope))
    q, k, v, _ = _qkv([20], [20], 4, 2, 64, 32, fused=False)
    with pytest.raises(E):
        swv.packed_attention(q, k, v, swv.PackedPlan([20], heads=4, kv_heads=2), out=lapped.bfloat16().as_strided((20, 4, 64), (64, 64, 1)))


def test_plan_inside_a_capture_is_refused(swv):
    """Before the host copy that would end the capture; the capture goes on."""
    x, w = torch.randn(8, 16, device="cuda"), torch.ones(16, device="cuda")
    want = swv.layer_norm(x, w)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = swv.layer_norm(x, w)
        with pytest.raises(swv._lib.SwvError):
            swv.PackedPlan([8], heads=1)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)


@pytest.mark.parametrize("D", [64, 128])
def test_attention_row_that_sees_no_key_is_zero_beside_nan_values(swv, D):
    """Causal, 40 queries and 30 keys: the first ten rows see nothing and are zero although the values are NaN."""
    q, k, v, _ = _qkv([40, 50], [30, 50], 4, 2, D, 33, fused=False)
    plan = swv.PackedPlan([40, 50], [30, 50], heads=4, kv_heads=2, causal=True)
    clean = swv.packed_attention(q, k, v, plan)
    bad = v.clone()
    bad[:30] = math.nan
    o, lse = swv.packed_attention(q, k, bad, plan, return_lse=True)
    assert not bool(o[:10].any()) and bool((lse[:, :10] == -math.inf).all())
    assert bool(torch.isnan(o[10:40]).all()) and torch.equal(o[40:], clean[40:])


@pytest.mark.parametrize("N,E,dt", [(2500, 1280, "bfloat16"), (700, 1288, "float16"), (300, 1536, "bfloat16"), (300, 1544, "float32"),
                                    (40, 2048, "bfloat16"), (40, 2056, "float16"), (50, 1800, "float32"), (100, 600, "float32"),
                                    (5000, 512, "bfloat16"), (3000, 520, "float16")])
def test_layer_norm_widths(swv, N, E, dt):
    """Rows on both sides of the widths at which another number of threads serves a row."""
    test_layer_norm(swv, N, E, dt, 0.4)


def test_calls_that_follow_one_another(swv):
    """Thirty training passes without a wait between them, each on inputs that the one before has just read, written into
    the same memory: the launches start early, their reads and writes do not.  The bits are those of passes run alone."""
    ql, kl, H, Hk, D, E = [40, 300, 7], [900, 20, 64], 4, 2, 64, 256
    plan, rope = swv.PackedPlan(ql, kl, heads=H, kv_heads=Hk), swv.RopeAxes(D, (16, 16))
    g = torch.Generator(device="cuda").manual_seed(40)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()
    rounds = [(r(sum(ql), E), r(sum(kl), Hk, D), r(sum(kl), Hk, D), r(sum(ql), H, D)) for _ in range(30)]
    buf = [torch.zeros_like(t) for t in rounds[0]]
    pos = torch.randint(0, 500, (sum(ql), 2), device="cuda")
    w, b = torch.randn(E, device="cuda", generator=g), torch.randn(E, device="cuda", generator=g)

    def run(data):
        for t, new in zip(buf, data):
            t.copy_(new)
        x, k, v = (t.detach().requires_grad_() for t in buf[:3])
        wl, bl = w.requires_grad_(), b.requires_grad_()
        q = swv.rope_axes(swv.layer_norm(x, wl, bl).view(-1, H, D), pos, rope)
        o = swv.packed_attention(q, k, v, plan)
        grads = torch.autograd.grad(o, (x, k, v, wl, bl), buf[3])
        with torch.no_grad():
            swv.rope_axes(buf[3], pos, rope, out=buf[3])
        return (o.detach(), buf[3].clone()) + grads

    alone = []
    for data in rounds:
        alone.append(run(data))
        torch.cuda.synchronize()
    for _ in range(3):
        chained = [run(data) for data in rounds]
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for x, y in zip(alone, chained) for a, c in zip(x, y))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = [run(data) for data in rounds[:6]]
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for x, y in zip(alone, captured) for a, c in zip(x, y))
