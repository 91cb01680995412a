"""Host side of the packed operators, without a GPU: what the kernels' launches rely on, and calls at the edges of what is
taken."""
import os
import re

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
    import sparse_wsi_vit_b200 as m
    csrc = os.path.join(os.path.dirname(m.__file__), "csrc")
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
