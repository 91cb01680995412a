"""Host side of the packed operators, without a GPU: the work tables of a plan, the refusals of the C entry points (all
before any launch) and of the Python layer."""
import ctypes

import numpy as np
import pytest
import torch


@pytest.fixture(scope="module")
def swv():
    import __graft_entry__
    __graft_entry__.build()
    import sparse_wsi_vit_b200 as m
    return m


def _tables(plan):
    """(header dict, units and joins of the three passes) of a plan's host copy."""
    w = plan._host
    names = ["magic", "words", "n_seq", "H", "Hkv", "causal", "Tq", "Tk"]
    h = dict(zip(names, w[:8].tolist()))
    f_off, f_n, q_off, q_n, k_off, k_n = w[8:14]
    joins = [w[14 + 3 * i:17 + 3 * i] for i in range(3)]
    units = [w[o:o + 8 * n].reshape(-1, 8) for o, n in ((f_off, f_n), (q_off, q_n), (k_off, k_n))]
    joins = [(w[o:o + 4 * n].reshape(-1, 4), s) for o, n, s in joins]
    return h, units, joins


CASES = [([5], None, 1, 1, False), ([130, 1, 0, 700], None, 6, 6, False), ([300, 257], None, 4, 2, True),
         ([1, 2, 5], [777, 64, 3000], 16, 2, True), ([70, 3], [20, 5], 10, 2, True), ([0, 0], None, 2, 1, False),
         ([4], [0], 2, 2, True), ([0], [9], 2, 2, True), ([40000], None, 8, 8, False), ([3] * 500, None, 12, 4, True),
         ([1] * 3, [65536, 1, 9000], 128, 1, True)]


@pytest.mark.parametrize("ql,kl,H,Hkv,causal", CASES)
def test_plan_covers_every_visible_pair_once(swv, ql, kl, H, Hkv, causal):
    """Every unit's rows are one sequence's, the blocks of the units of a row cover what it sees without overlap, every
    row belongs to one unit (or to the parts of one divided unit), slots are used once, the longest units come first."""
    kl = ql if kl is None else kl
    plan = swv.PackedPlan(ql, kl, heads=H, kv_heads=Hkv, causal=causal, device="cpu")
    h, units, joins = _tables(plan)
    assert (h["Tq"], h["Tk"], h["H"], h["Hkv"], h["words"]) == (sum(ql), sum(kl), H, Hkv, plan._host.size)
    q0, k0 = np.concatenate([[0], np.cumsum(ql)]), np.concatenate([[0], np.cumsum(kl)])
    tok = 128 // (H // Hkv)
    for side, (table, (join, slots)) in enumerate(zip(units, joins)):
        lens, starts = (kl, k0) if side == 2 else (ql, q0)
        other, other0 = (ql, q0) if side == 2 else (kl, k0)
        block = tok if side == 2 else 128
        size = {0: 2 * tok, 1: tok, 2: 128}[side]
        seen = {}
        used = []
        for t0, n, s0, ln, off, b0, b1, slot in table.tolist():
            s = int(np.searchsorted(starts, t0, side="right") - 1)
            while lens[s] == 0 or t0 >= starts[s] + lens[s]:
                s -= 1
            assert starts[s] <= t0 and t0 + n <= starts[s] + lens[s] and 0 < n <= size
            assert s0 == other0[s] and ln == other[s] and 0 <= b0 <= b1 <= -(-ln // block)
            place = t0 - starts[s]
            if side < 2:
                assert off == (place + kl[s] - ql[s] if causal else kl[s])
            else:
                assert (off == place - (kl[s] - ql[s])) if causal else off <= -128
            seen.setdefault((t0, n, s), []).append((b0, b1, slot))
            if slot >= 0:
                used.append(slot)
        assert sorted(used) == list(range(slots))
        rows = 0
        for (t0, n, s), parts in seen.items():
            rows += n
            parts.sort()
            place = t0 - starts[s]
            if side < 2:
                last = min(other[s], place + n - 1 + kl[s] - ql[s] + 1) if causal else other[s]
                want = (0, max(0, -(-last // 128)))
                assert parts[0][0] == 0 and parts[-1][1] == want[1]
            else:
                first = max(0, place - (kl[s] - ql[s])) if causal else 0
                assert parts[0][0] <= first // tok and parts[-1][1] == -(-other[s] // tok)
            assert all(a[1] == b[0] for a, b in zip(parts, parts[1:]))
            if len(parts) > 1:
                mine = [j for j in join.tolist() if j[0] == t0]
                assert len(mine) == 1 and mine[0][1] == n and mine[0][3] == len(parts)
                assert [p[2] for p in parts] == list(range(mine[0][2], mine[0][2] + mine[0][3]))
            else:
                assert parts[0][2] == -1
        assert rows == sum(lens) and len(join) == sum(len(p) > 1 for p in seen.values())
        work = (table[:, 6] - table[:, 5]).tolist()
        assert work == sorted(work, reverse=True)


def test_plan_divides_long_units_only_where_they_are_few(swv):
    few = swv.PackedPlan([1], [65536], heads=8, kv_heads=8, device="cpu")
    many = swv.PackedPlan([65536], heads=8, device="cpu")
    assert _tables(few)[2][0][1] > 1 and all(s == 0 for _, s in _tables(many)[2])


def test_plan_refusals(swv):
    E = swv._lib.SwvError
    with pytest.raises(E):
        swv.PackedPlan([4, 4], [4], heads=2, device="cpu")
    with pytest.raises(E):
        swv.PackedPlan([4, -1], heads=2, device="cpu")
    with pytest.raises(E):
        swv.PackedPlan([4], heads=6, kv_heads=4, device="cpu")
    with pytest.raises(E):
        swv.PackedPlan([4], heads=0, device="cpu")
    with pytest.raises(E):
        swv.PackedPlan([4], heads=129, kv_heads=1, device="cpu")
    with pytest.raises(E):
        swv.PackedPlan([1 << 29, 1], heads=2, device="cpu")
    with pytest.raises(E):
        swv.PackedPlan([4.5], heads=2, device="cpu")
    assert swv.PackedPlan([], heads=2, device="cpu").q_tokens == 0
    assert swv.PackedPlan(torch.tensor([3, 4]), heads=2, device="cpu").q_tokens == 7


def test_packed_attention_entry_points_refuse(swv):
    L = swv._lib.lib
    plan = swv.PackedPlan([200, 100], heads=4, kv_heads=2, device="cpu")
    hp = plan._host.ctypes.data
    fake = ctypes.c_void_p(0x1000)                       # never dereferenced
    s3 = (ctypes.c_int64 * 3)(512, 128, 1)
    odd = (ctypes.c_int64 * 3)(511, 128, 1)
    n = ctypes.c_size_t()
    assert L.swv_packed_plan(1, None, None, 1, 1, 0, None, 0, None) == -1
    lens = np.array([7], dtype=np.int64).ctypes.data
    assert L.swv_packed_plan(1, lens, lens, 1, 1, 0, hp, 8, ctypes.byref(n)) == -5 and n.value > 8
    assert L.swv_packed_attn_bytes(hp, 64, ctypes.byref(n)) == 0
    assert L.swv_packed_attn_bytes(hp, 60, ctypes.byref(n)) == -8
    assert L.swv_packed_attn_bytes(hp, 136, ctypes.byref(n)) == -8
    assert L.swv_packed_attn_bytes(None, 64, ctypes.byref(n)) == -1
    assert L.swv_packed_attn_bytes(np.zeros(32, dtype=np.int32).ctypes.data, 64, ctypes.byref(n)) == -4
    fwd = lambda q=fake, qs=s3, Tq=300, Tk=300, D=64, scale=0.1, dev=fake, st=fake: L.swv_packed_attn_fwd(
        q, qs, fake, s3, fake, s3, fake, s3, None, hp, dev, Tq, Tk, D, scale, None, 0, st, None)
    assert fwd(q=None) == -1 and fwd(dev=None) == -1 and fwd(st=None) == -1
    assert fwd(qs=odd) == -2 and fwd(q=ctypes.c_void_p(0x1008)) == -2
    assert fwd(Tq=299) == -4 and fwd(Tk=10) == -4
    assert fwd(scale=0.0) == -4 and fwd(scale=-1.0) == -4 and fwd(scale=float("nan")) == -4 and fwd(scale=float("inf")) == -4
    assert fwd(scale=2.0 ** -61) == -4 and fwd(scale=2.0 ** 61) == -4
    assert fwd(D=12) == -8 and fwd(D=256) == -8
    assert L.swv_packed_attn_bwd_bytes(hp, 300, 64, ctypes.byref(n)) == 0 and n.value >= 4 * 300 * 8
    assert L.swv_packed_attn_bwd_bytes(hp, 200, 64, ctypes.byref(n)) == -4
    bwd = lambda ws=fake, nb=1 << 30, lse=fake, dos=s3, Tq=300: L.swv_packed_attn_bwd(
        fake, dos, fake, s3, fake, s3, fake, s3, fake, s3, lse, fake, s3, fake, s3, fake, s3, hp, fake, Tq, 300, 64, 0.1, ws,
        nb, fake, None)
    assert bwd(ws=None) == -1 and bwd(lse=None) == -1 and bwd(nb=100) == -5 and bwd(dos=odd) == -2 and bwd(Tq=5) == -4
    assert bwd(ws=ctypes.c_void_p(0x1004)) == -2


def test_layer_norm_and_rope_entry_points_refuse(swv):
    L = swv._lib.lib
    fake = ctypes.c_void_p(0x1000)
    ln = lambda x=fake, xd=0, yd=0, N=4, E=8, mean=None, rstd=None: L.swv_layer_norm_fwd(
        x, 8, xd, fake, 0, fake, 0, fake, 8, yd, mean, rstd, N, E, 1e-5, None)
    assert ln(x=None) == -1 and ln(xd=7) == -3 and ln(yd=5) == -3 and ln(E=0) == -4 and ln(N=-1) == -4
    assert ln(xd=1, yd=2) == -3 and ln(mean=fake) == -1 and ln(N=0) == 0
    n = ctypes.c_size_t()
    assert L.swv_layer_norm_bwd_bytes(100, 384, ctypes.byref(n)) == 0 and n.value % (2 * 384 * 4) == 0
    assert L.swv_layer_norm_bwd_bytes(100, 0, ctypes.byref(n)) == -4
    bwd = lambda ws, nb: L.swv_layer_norm_bwd(fake, 8, 0, fake, 8, 0, fake, 0, fake, fake, fake, 8, fake, 0, fake, 0, 4, 8, ws,
                                              nb, None)
    assert bwd(None, 0) == -1 and bwd(fake, 4) == -5
    f, a = np.ones(4), np.zeros(4, dtype=np.uint8)
    s3 = (ctypes.c_int64 * 3)(16, 8, 1)
    bad = (ctypes.c_int64 * 3)(16, 8, 2)
    rope = lambda x=fake, xs=s3, pairs=4, axes=1, hd=8, T=2, pd=0, dt=0: L.swv_rope_axes_apply(
        x, xs, fake, s3, dt, fake, pd, 1, f.ctypes.data, a.ctypes.data, pairs, axes, 0, 0, T, 2, hd, None)
    assert rope(x=None) == -1 and rope(xs=bad) == -2 and rope(pd=3) == -3 and rope(dt=9) == -3
    assert rope(pairs=5) == -4 and rope(pairs=0) == -4 and rope(hd=6) == -4 and rope(axes=0) == -4 and rope(axes=9) == -8
    assert rope(T=0) == 0
    a[2] = 1
    assert rope() == -4                                  # an axis that the positions do not have


def test_python_refusals_without_a_gpu(swv):
    E = swv._lib.SwvError
    x = torch.randn(4, 8)
    with pytest.raises(E):
        swv.layer_norm(x)                                # no CPU path
    plan = swv.PackedPlan([4], heads=1, device="cpu")
    t = torch.randn(4, 1, 8).bfloat16()
    with pytest.raises(E):
        swv.packed_attention(t, t, t, plan)
    for bad in (dict(sections=(5,)), dict(sections=()), dict(sections=(-1, 2)), dict(sections=(0, 0)),
                dict(sections=(2, 2), scales=(1.0,)), dict(sections=(2,), ladder="x"), dict(sections=(2,), pairing="x"),
                dict(sections=(2,), theta=0.0), dict(sections=(2,), theta=float("inf")), dict(sections=(2,), scales=(float("nan"),)), dict(sections=(1,) * 9)):
        with pytest.raises(E):
            swv.RopeAxes(8, **bad)
    with pytest.raises(E):
        swv.RopeAxes(512, (200,))
    with pytest.raises(E):
        swv.rope_axes(torch.randn(2, 1, 8), torch.zeros(2, 1), swv.RopeAxes(8, (4,)))


def test_plan_of_more_work_than_its_tables_address_is_refused(swv):
    """2^29 tokens in tiles of one token (128 heads share a key head) are 2^29 units and more: word offsets of 32 bits do
    not reach them.  Refused before anything is allocated, with and without a buffer for the plan."""
    with pytest.raises(swv._lib.SwvError):
        swv.PackedPlan([1 << 29], [1], heads=128, kv_heads=1, device="cpu")
    n, one, size = (ctypes.c_int64 * 1)(1 << 29), (ctypes.c_int64 * 1)(1), ctypes.c_size_t()
    lib = swv._lib.lib
    assert lib.swv_packed_plan(1, n, one, 128, 1, 0, None, 0, ctypes.byref(size)) not in (0, -5)
