"""Host side of the packed operators, without a GPU: what the kernels' launches rely on, and calls at the edges of what is
taken."""
import copy
import ctypes
import os
import pickle
import re

import numpy as np
import pytest
import torch


@pytest.fixture(scope="module")
def swv():
    import __graft_entry__
    __graft_entry__.build()
    import sparse_wsi_vit_b200 as m
    return m


def _kernels(text):
    """{name: body} of the kernels of a source file."""
    out = {}
    for m in re.finditer(r"__global__ void.*?(\w+_kernel)\(", text, re.S):
        i = text.index("{", m.end())
        depth, j = 1, i + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[j], 0)
            j += 1
        out[m.group(1)] = text[i:j]
    return out


def test_every_kernel_that_starts_early_waits_in_every_thread():
    """A kernel launched close behind another one may read what earlier kernels of the stream wrote only behind a wait of its
    own: each has the wait as a statement of its outermost block, ahead of any release of the kernel behind it."""
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sparse_wsi_vit_b200", "csrc")
    seen = 0
    for f in sorted(os.listdir(csrc)):
        text = open(os.path.join(csrc, f)).read() if f.endswith(".cu") else ""
        if "launch_after(" not in text:
            continue
        for name, body in _kernels(text).items():
            waits = [k.start() for k in re.finditer(r"^  grid_wait\(\);", body, re.M)]
            assert len(waits) == 1 and body.count("grid_wait()") == 1, f"{f}: {name}"
            assert waits[0] < body.find("grid_release()") or "grid_release()" not in body, f"{f}: {name}"
            seen += 1
    assert seen >= 10


@pytest.mark.parametrize("ql,kl,H,Hkv", [([300], [260], 1, 1), ([700, 3], [650, 900], 2, 1), ([2, 256], [4000, 400], 16, 2),
                                         ([1000], [3000], 8, 1), ([256], [384], 4, 4), ([2048], [1800], 1, 1)])
def test_every_row_of_a_divided_unit_sees_a_key(swv, ql, kl, H, Hkv):
    """The join of a divided unit takes a row without any weight for one whose scores are all -inf."""
    plan = swv.PackedPlan(ql, kl, heads=H, kv_heads=Hkv, causal=True, device="cpu")
    w = plan._host
    units = w[w[8]:w[8] + 8 * w[9]].reshape(-1, 8)
    for t0, n, s0, ln, off, b0, b1, slot in units.tolist():
        assert slot < 0 or min(ln, off + 1) > 0


COPIES = [copy.copy, copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x))]


@pytest.mark.parametrize("make", COPIES)
def test_copied_handles_hold_addresses_of_their_own(swv, make):
    """Copies of a rotary handle, of a plan and of a module that holds one pass addresses of what they own themselves, with the
    same contents: they outlive the original."""
    rope = swv.RopeAxes(64, (8, 12, 12), scales=(1.0, 0.5, 0.25), pairing="halves")
    plan = swv.PackedPlan([5, 600], [70, 900], heads=4, kv_heads=2, causal=True, device="cpu")
    net = swv.PackedViTSlideEncoder(in_features=8, embed_dim=64, num_heads=2, num_layers=1, rope_sections=(4, 4))
    r, p, n = make(rope), make(plan), make(net)
    for a, b in ((r, rope), (n.rope, net.rope)):
        assert a._call[:2] == (a._freq.ctypes.data, a._axis.ctypes.data) and a._call[2:] == b._call[2:]
        assert (a._freq == b._freq).all() and (a._axis == b._axis).all() and a._axis.dtype == b._axis.dtype
    assert p._call == (p._host.ctypes.data, p._table.data_ptr()) and torch.equal(p._table, plan._table)
    assert (p.q_tokens, p.k_tokens, p.heads, p.kv_heads, p.causal, p.device) == (605, 970, 4, 2, True, plan.device)
    assert p._workspace_bytes(64) == plan._workspace_bytes(64)
    for a, b in ((r, rope), (p, plan)):                           # no address of the original, unless its memory is shared
        assert make is copy.copy or a._call[0] != b._call[0]


def test_output_buffers_beside_the_inputs(swv):
    """A part of the inputs' buffer that holds none of their elements is taken; any shared element is refused, and so is a buffer
    of another number of dimensions."""
    from sparse_wsi_vit_b200.packed import _check_out
    E = swv._lib.SwvError
    arena = torch.zeros(4000)
    x = arena[:640].view(10, 4, 16)
    _check_out(arena[640:1280].view(10, 4, 16), x, (x,))
    _check_out(x, x, (x,), same=x)
    for bad in (arena[639:1279].view(10, 4, 16), arena[16:656].view(10, 4, 16), torch.zeros(640), torch.zeros(10, 64),
                arena[:1280].view(20, 4, 16)[::2]):
        with pytest.raises(E):
            _check_out(bad, x, (x,))
    with pytest.raises(E):
        _check_out(x, x, (x,))
    qkv = torch.zeros(10, 12, 16)
    q, k, v = qkv[:, :4], qkv[:, 4:8], qkv[:, 8:]
    for out, ins in ((q, (k, v)), (k, (q, v)), (v, (q, k))):
        _check_out(out, out, ins)
        with pytest.raises(E):
            _check_out(out, out, ins + (out,))
    with pytest.raises(E):
        _check_out(qkv[:, 2:6], q, (q,))
    with pytest.raises(E):
        _check_out(q, q, (x, qkv[:, 3:5, 5]))
    odd = torch.zeros(200 * 9 + 64).as_strided((9, 4, 16), (200, 16, 1))          # another row distance in the same memory
    with pytest.raises(E):
        _check_out(odd, odd, (odd.as_strided((9, 4, 16), (192, 16, 1), 64),))
    pos = x[:, 0, :2]                                             # in place, but over the positions
    with pytest.raises(E):
        _check_out(x, x, (x, pos), same=x)
    _check_out(torch.zeros(0, 4, 16), torch.zeros(0, 4, 16), (x,))
    version = x._version
    with pytest.raises(E):
        _check_out(x, x, (x,))
    assert x._version == version


def test_sizes_beyond_32_bits_are_refused(swv):
    """The library takes widths, heads and channels as 32-bit numbers and steps beyond them in loops."""
    L, fake, n = swv._lib.lib, ctypes.c_void_p(0x1000), ctypes.c_size_t()
    big = (1 << 29) + 1
    for E in (big, (1 << 31) - 1):
        assert L.swv_layer_norm_fwd(fake, E, 0, None, 0, None, 0, fake, E, 0, None, None, 1, E, 1e-5, None) == -8
        assert L.swv_layer_norm_bwd_bytes(1, E, ctypes.byref(n)) == -8
        assert L.swv_layer_norm_bwd(fake, E, 0, fake, E, 0, None, 0, fake, fake, fake, E, None, 0, None, 0, 1, E, None, 0, None) == -8
    f, a, s3 = np.ones(4), np.zeros(4, dtype=np.uint8), (ctypes.c_int64 * 3)(16, 8, 1)
    for H, hd in ((big, 8), (2, big), ((1 << 31) - 1, 8)):
        assert L.swv_rope_axes_apply(fake, s3, fake, s3, 0, fake, 0, 1, f.ctypes.data, a.ctypes.data, 4, 1, 0, 0, 1, H, hd, None) == -8
    for heads, kv in (((1 << 32) + 4, 4), ((1 << 32) + 4, (1 << 32) + 4), (65536, 65536)):
        with pytest.raises(swv._lib.SwvError):
            swv.PackedPlan([4], heads=heads, kv_heads=kv, device="cpu")
    assert swv.PackedPlan([4], heads=65535, device="cpu").heads == 65535


def test_rotary_frequencies_are_finite(swv):
    with pytest.raises(swv._lib.SwvError):
        swv.RopeAxes(64, (32,), theta=1e-300, scales=(1e300,))
    assert swv.RopeAxes(64, (32,), theta=1e-300)._freq[-1] > 1e280
