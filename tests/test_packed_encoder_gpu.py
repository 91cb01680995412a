"""The packed dense encoder: layer norm, rotary positions and attention of ``packed`` run together, against a plain
restatement of the same model in 64 bits, forward and backward; its training step through ``training``."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def swv():
    import sparse_wsi_vit_b200 as m
    yield m
    m.check_status(torch.device("cuda:0"))


def _encoder(swv, layers=2, axes=True, seed=0, **kw):
    torch.manual_seed(seed)
    with torch.device("cuda"):
        net = swv.PackedViTSlideEncoder(in_features=48, out_features=3, embed_dim=128, num_heads=2, num_layers=layers, num_cls=2,
                                        rope_sections=(8, 12, 12) if axes else None,
                                        rope_scales=(1.0, 1 / 64, 1 / 64) if axes else None, **kw)
        for n, p in net.named_parameters():         # no zero biases, no unit weights
            with torch.no_grad():
                p.add_(0.05 * torch.randn_like(p))
    return net


def _batch(lengths, seed, axes=3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    bags = [torch.randn(n, 48, generator=g, device="cuda") for n in lengths]
    coords = [(torch.rand(n, axes, generator=g, device="cuda") * torch.tensor([4.0, 64.0, 64.0], device="cuda")[:axes]).floor()
              for n in lengths]
    return bags, coords


def plain(net, params, bag, coord):
    """One slide in 64 bits; ``params``: {name: double tensor}."""
    P = lambda n: params[n]
    lin = lambda x, n: x @ P(n + ".weight").T + (P(n + ".bias") if n + ".bias" in params else 0)
    def norm(x, n):
        mu = x.mean(-1, keepdim=True)
        return (x - mu) / torch.sqrt((x - mu).square().mean(-1, keepdim=True) + 1e-5) * P(n + ".weight") + P(n + ".bias")
    x = torch.cat([P("cls_tokens")[0], lin(bag.double(), "input_proj")])
    T, H = x.shape[0], net.num_heads
    D = net.embed_dim // H
    C = net.num_cls
    for i in range(len(net.blocks)):
        b = f"blocks.{i}."
        q, k, v = lin(norm(x, b + "norm1"), b + "attn.qkv").view(T, 3, H, D).permute(1, 2, 0, 3)
        if net.rope is not None:
            pos = torch.cat([coord.new_zeros(C, coord.shape[1]), coord]).double()
            ang = torch.stack([pos[:, a] * net.rope._freq[p] for p, a in enumerate(net.rope._axis.tolist())], 1)
            def turn(t):
                a, c = t[..., 0:2 * net.rope.pairs:2], t[..., 1:2 * net.rope.pairs:2]
                r = torch.stack([a * ang.cos() - c * ang.sin(), c * ang.cos() + a * ang.sin()], -1).flatten(-2)
                return torch.cat([r, t[..., 2 * net.rope.pairs:]], -1)
            q, k = turn(q), turn(k)
        o = torch.softmax(q @ k.transpose(1, 2) / math.sqrt(D), -1) @ v
        x = x + lin(o.transpose(0, 1).flatten(1), b + "attn.out_proj")
        x = x + lin(torch.nn.functional.gelu(lin(norm(x, b + "norm2"), b + "mlp.0")), b + "mlp.3")
    x = norm(x[:C], "norm")
    pooled = (torch.softmax(lin(x, "cls_pool"), 0) * x).sum(0)
    return lin(pooled, "head")


# The attention's operands, probabilities and results are rounded to bf16 (2^-8 each at most): five roundings a block, seen
# through layers that neither amplify nor damp much (unit-variance activations); the rest is fp32.  In the 2-norm half of
# the worst case per rounding is ample: 5 layers 2^-9.  Gradients pass twice as many.
def _tol(layers, backward=False):
    return (2 if backward else 1) * 5 * layers * 2.0 ** -9


def _rel(a, b):
    return float((a.detach().double() - b).norm() / b.norm().clamp_min(1e-30))


@pytest.mark.parametrize("layers,axes", [(1, True), (2, True), (3, False)])
def test_encoder_forward_and_gradients(swv, layers, axes):
    lengths = [130, 1, 259, 0]                           # a slide without patches: its CLS tokens alone
    net = _encoder(swv, layers, axes)
    bags, coords = _batch(lengths, 1)
    logits = net(bags, coords if axes else None)["logits"]
    assert logits.shape == (4, 3)
    w = torch.randn(4, 3, device="cuda")
    grads = dict(zip([n for n, _ in net.named_parameters()], torch.autograd.grad((logits * w).sum(), list(net.parameters()))))
    params = {n: p.detach().double().requires_grad_() for n, p in net.named_parameters()}
    ref = torch.stack([plain(net, params, b, c) for b, c in zip(bags, coords)])
    gref = dict(zip(params, torch.autograd.grad((ref * w.double()).sum(), list(params.values()), allow_unused=True)))
    assert _rel(logits, ref.detach()) <= _tol(layers)
    top = max(float(g.norm()) for g in gref.values())
    for n, g in grads.items():
        # (a gradient that cancels, as that of a key bias, is measured against the largest)
        assert float((g.double() - gref[n]).norm()) <= _tol(layers, True) * max(float(gref[n].norm()), 2.0 ** -7 * top), n


def test_encoder_batch_is_its_slides(swv):
    """A packed batch gives what its slides give one by one, whatever lies beside them, and a shared layout the same."""
    net = _encoder(swv).eval()
    lengths = [77, 300, 5]
    bags, coords = _batch(lengths, 2)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        whole = net(bags, coords)["logits"]
        again = net(bags, coords, layout=net.pack(lengths, "cuda"))["logits"]
        one = torch.cat([net(b, c)["logits"] for b, c in zip(bags, coords)])
        bad = [bags[0], torch.full_like(bags[1], math.nan), bags[2]]
        apart = net(bad, coords)["logits"]
    assert torch.equal(whole, again)
    assert _rel(whole, one.double()) <= 2 * _tol(2) + 2 * 8 * 2 * 2.0 ** -9          # bf16 activations: eight more roundings a block
    assert torch.equal(apart[[0, 2]], whole[[0, 2]]) and bool(torch.isnan(apart[1]).all())


def test_encoder_trains_on_ragged_batches(swv):
    """slide_step hands the list over in one pass; the step runs, its gradients are finite and reach every parameter, and
    equal those of the loss written out."""
    from sparse_wsi_vit_b200.training import slide_step, train_step
    net = _encoder(swv).train()
    bags, coords = _batch([120, 33, 200], 3)
    batch = {"input": bags, "coords": coords, "label": torch.tensor([0, 2, 1], device="cuda")}
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss, preds, logits = slide_step(net, batch)
        other = torch.nn.functional.cross_entropy(net(bags, coords)["logits"], batch["label"])
    assert torch.equal(loss, other) and preds.shape == (3,)
    loss.backward()
    for n, p in net.named_parameters():
        assert p.grad is not None and bool(torch.isfinite(p.grad).all()), n
    before = [p.detach().clone() for p in net.parameters()]
    assert math.isfinite(train_step(net, torch.optim.SGD(net.parameters(), lr=0.1), batch))
    assert any(not torch.equal(a, b) for a, b in zip(before, net.parameters()))


def test_encoder_captured_inference(swv):
    """Captured with a layout made before, replayed on other slides of the same lengths."""
    net = _encoder(swv).eval()
    lengths = [150, 40]
    layout = net.pack(lengths, "cuda")
    sets = [_batch(lengths, s) for s in (4, 5)]
    def run(bags, coords):
        with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16, cache_enabled=False):
            return net(bags, coords, layout)["logits"]
    want = [run(*s) for s in sets]
    buf = [[t.clone() for t in x] for x in sets[0]]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        run(*buf)
    torch.cuda.current_stream().wait_stream(st)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run(*buf)
    for i in (1, 0):
        for dst, src in zip(buf, sets[i]):
            for d, s in zip(dst, src):
                d.copy_(s)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])


def test_encoder_refusals(swv):
    net = _encoder(swv)
    bags, coords = _batch([10, 20], 6)
    for args in ((bags,), (bags, coords[:1]), (bags, [c[:, :2] for c in coords]), (bags, [coords[1], coords[0]]), ([],)):
        with pytest.raises(ValueError):
            net(*args)
    with pytest.raises(ValueError):
        net(bags, coords, layout=net.pack([10, 21], "cuda"))
    for kw in (dict(embed_dim=130, num_heads=4), dict(embed_dim=384, num_heads=2), dict(num_cls=0), dict(embed_dim=36, num_heads=3)):
        with pytest.raises(ValueError):
            swv.PackedViTSlideEncoder(**kw)
