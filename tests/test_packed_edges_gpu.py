"""Packed operators on a B200 at the edges of what they take: scores of -inf, copies of handles, buffers inside an arena, derivatives
that the kernels do not have.  Bounds and references are those of the operators' other tests."""
import copy
import gc
import math
import pickle

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from .test_packed_gpu import _close, reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def swv():
    import sparse_wsi_vit_b200 as m
    yield m
    m.check_status(torch.device("cuda:0"))


def _inputs(lq, lk, H, Hk, D, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()
    return r(lq, H, D), r(lk, Hk, D), r(lk, Hk, D), r(lq, H, D)


@pytest.mark.parametrize("low", [-math.inf, -3e38])
@pytest.mark.parametrize("lq,lk,lead,D", [(40, 500, 128, 64), (300, 1000, 300, 128), (2, 6007, 128, 64), (2, 6007, 300, 128),
                                          (1, 9000, 4111, 64), (3, 300, 299, 64)])
def test_attention_leading_keys_of_probability_zero(swv, low, lq, lk, lead, D):
    """Whole key blocks, and whole parts of divided units, whose scores are all -inf ahead of finite ones: the result is that of
    the finite keys alone.  Channel 0 of the queries is 8, of the leading keys -inf or so low that the product passes the
    range (then every gradient exists: zero for those keys)."""
    q, k, v, do = _inputs(lq, lk, 4, 2, D, lead)
    q[:, :, 0], k[:, :, 0] = 8, 0
    k[:lead, :, 0] = low
    plan = swv.PackedPlan([lq], [lk], heads=4, kv_heads=2)
    ref = reference(q, k[lead:], v[lead:], do, [lq], [lk - lead], False)
    o, lse = swv.packed_attention(q, k, v, plan, return_lse=True)
    _close(o, *ref["o"], "o")
    _close(lse, *ref["lse"], "lse")
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    dq, dk, dv = torch.autograd.grad(swv.packed_attention(*leaves, plan), leaves, do)
    for name, got in (("dk", dk), ("dv", dv)):
        assert not bool(got[:lead].any())
        _close(got[lead:], *ref[name], name)
    if low == -math.inf:
        assert bool(torch.isnan(dq[:, :, 0]).all())               # 0 x inf, as the formula has it
    else:
        _close(dq, *ref["dq"], "dq")


def test_attention_causal_leading_keys_of_probability_zero(swv):
    """Causal rows that see the leading keys alone are NaN, the ones behind them those of the finite keys."""
    n, lead = 700, 300
    q, k, v, do = _inputs(n, n, 2, 2, 64, 5)
    q[:, :, 0], k[:, :, 0] = 8, 0
    k[:lead, :, 0] = -math.inf
    o, lse = swv.packed_attention(q, k, v, swv.PackedPlan([n], heads=2, causal=True), return_lse=True)
    ref = reference(q[lead:], k[lead:], v[lead:], do[lead:], [n - lead], [n - lead], True)
    assert bool(torch.isnan(o[:lead]).all()) and bool(torch.isnan(lse[:, :lead]).all())
    _close(o[lead:], *ref["o"], "o")
    _close(lse[:, lead:], *ref["lse"], "lse")


@pytest.mark.parametrize("lq,lk", [(2, 6007), (300, 400)])
def test_attention_rows_of_infinite_scores_alone_are_nan(swv, lq, lk):
    """Divided and undivided: all scores -inf is 0 / 0, also where the values are finite."""
    q, k, v, _ = _inputs(lq, lk, 2, 1, 64, 6)
    q[:, :, 0] = 1
    k[:, :, 0] = -math.inf
    o, lse = swv.packed_attention(q, k, v, swv.PackedPlan([lq], [lk], heads=2, kv_heads=1), return_lse=True)
    assert bool(torch.isnan(o).all()) and bool(torch.isnan(lse).all())


@pytest.mark.parametrize("make", [copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x))])
def test_copied_handles_outlive_the_original(swv, make):
    q, k, v, _ = _inputs(300, 300, 4, 2, 64, 7)
    pos = torch.randint(0, 900, (300, 3), device="cuda")
    rope, plan = swv.RopeAxes(64, (8, 12, 12)), swv.PackedPlan([100, 200], heads=4, kv_heads=2)
    want = swv.packed_attention(swv.rope_axes(q, pos, rope), k, v, plan)
    r, p = make(rope), make(plan)
    del rope, plan
    gc.collect()
    junk = [np.full(n, 7.0) for n in (4, 8, 32, 64, 1024) for _ in range(50)]
    assert torch.equal(swv.packed_attention(swv.rope_axes(q, pos, r), k, v, p), want) and len(junk) == 250


def test_dual_tensors_are_refused(swv):
    """Forward-mode derivatives do not exist: a dual input, parameter, buffer or upstream gradient is refused instead of losing its
    tangent; plain tensors are served inside a dual level as outside."""
    E = swv._lib.SwvError
    q, k, v, do = _inputs(20, 20, 4, 2, 64, 8)
    plan, rope, pos = swv.PackedPlan([20], heads=4, kv_heads=2), swv.RopeAxes(64, (16, 16)), torch.rand(20, 2, device="cuda")
    w, b = torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")
    ops = [(swv.layer_norm, (q, w, b)), (lambda x, p: swv.rope_axes(x, p, rope), (q, pos)),
           (lambda *a: swv.packed_attention(*a, plan), (q, k, v))]
    want = [f(*a) for f, a in ops]
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        for (f, a), y in zip(ops, want):
            assert torch.equal(f(*a), y)
            for i in range(len(a)):
                for grad in (False, True):
                    t = a[i].detach().requires_grad_(grad and a[i] is not pos)
                    with pytest.raises(E, match="forward-mode"):
                        f(*a[:i], dual(t), *a[i + 1:])
            x = a[0].detach().requires_grad_()
            with pytest.raises(E, match="forward-mode"):
                torch.autograd.grad(f(x, *a[1:]), x, dual(do))
        for call in (lambda o: swv.rope_axes(q, pos, rope, out=o), lambda o: swv.packed_attention(q, k, v, plan, out=o)):
            with pytest.raises(E, match="forward-mode"):
                call(dual(torch.empty_like(q)))
    assert all(torch.equal(f(*a), y) for (f, a), y in zip(ops, want))


def test_results_written_beside_the_inputs(swv):
    """Results in a buffer that holds the inputs too: behind them in an arena, and between the heads of a fused projection."""
    q, k, v, _ = _inputs(300, 300, 4, 4, 64, 9)
    plan, rope = swv.PackedPlan([100, 200], heads=4), swv.RopeAxes(64, (16, 16))
    pos = torch.randint(0, 900, (300, 2), device="cuda")
    want, turned = swv.packed_attention(q, k, v, plan), swv.rope_axes(k, pos, rope)
    qkv = torch.cat([q, k, v, torch.zeros_like(q)], 1)            # four heads each
    part = lambda i: qkv[:, 4 * i:4 * i + 4]
    swv.packed_attention(part(0), part(1), part(2), plan, out=part(3))
    assert torch.equal(part(3), want)
    swv.rope_axes(part(1), pos, rope, out=part(0))
    assert torch.equal(part(0), turned) and torch.equal(part(1), k) and torch.equal(part(2), v) and torch.equal(part(3), want)
    arena = torch.cat([t.flatten() for t in (q, k, v, torch.zeros_like(q))]).view(4, 300, 4, 64)
    swv.packed_attention(arena[0], arena[1], arena[2], plan, out=arena[3])
    assert torch.equal(arena[3], want) and torch.equal(arena[2], v)
    E = swv._lib.SwvError
    for bad in (arena[0], qkv[:, 2:6], q.flatten(), q[0]):
        with pytest.raises(E):
            swv.packed_attention(part(0), arena[0], arena[2], plan, out=bad)
    for x, bad in ((part(0), qkv[:, 1:5]), (part(0), qkv[:, 2:6]), (q, q.flatten()), (q, q[0])):
        with pytest.raises(E):
            swv.rope_axes(x, pos, rope, out=bad)


@pytest.mark.parametrize("n", [(1 << 29) + 8, (1 << 32) + 8])
def test_sizes_beyond_32_bits_are_refused(swv, n):
    """Ahead of any copy or launch: a width or a number of heads that the library would take modulo 2^32."""
    one = torch.zeros(1, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(swv._lib.SwvError):
        swv.layer_norm(one.expand(1, n))
    with pytest.raises(swv._lib.SwvError):
        swv.rope_axes(one.expand(1, n, 8), torch.zeros(1, 1, device="cuda"), swv.RopeAxes(8, (4,)))


def test_attention_backward_gets_no_gradient_of_lse(swv, monkeypatch):
    """lse has no gradient: none is made up for it (a tensor of zeros and a launch in every backward pass)."""
    from sparse_wsi_vit_b200.packed import PackedAttentionFunction as F
    seen, real = [], F.backward
    monkeypatch.setattr(F, "backward", staticmethod(lambda ctx, *g: seen.append(g) or real(ctx, *g)))
    q, k, v, do = _inputs(40, 40, 4, 2, 64, 10)
    plan = swv.PackedPlan([40], heads=4, kv_heads=2)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    for lse in (False, True):
        o = swv.packed_attention(*leaves, plan, return_lse=lse)
        grads = torch.autograd.grad(o[0] if lse else o, leaves, do)
        assert all(g is not None for g in grads)
    assert len(seen) == 2 and all(g[0] is not None and g[1] is None for g in seen)
    assert real(None, None, None) == (None,) * 5


def test_first_attention_call_inside_a_capture(swv, monkeypatch):
    """The status word exists before the capture (the plan makes it): it is zero ahead of the first replay, and a replay does not
    clear what another launch has recorded."""
    from sparse_wsi_vit_b200 import ops
    monkeypatch.setattr(ops, "_status", {})
    q, k, v, _ = _inputs(40, 40, 4, 2, 64, 11)
    plan = swv.PackedPlan([40], heads=4, kv_heads=2)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = swv.packed_attention(q, k, v, plan)
    word = ops.status_word(q.device)
    assert int(word) == 0
    word.fill_(101)
    g.replay()
    assert int(word) == 101 and torch.equal(o, swv.packed_attention(q, k, v, plan))
    word.zero_()
