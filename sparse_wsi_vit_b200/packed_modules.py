"""A dense slide encoder over packed batches: the skeleton of the package's other encoders (same parameter names:
cls_tokens, input_proj, blocks.i.{norm1, attn.qkv, attn.out_proj, norm2, mlp}, norm, cls_pool, head) with full attention
inside every slide and rotary positions of any number of axes.  A batch of slides of different sizes is one pass without
padding; the reference's dense ViT-5 takes one slide at a time (src/sparse_wsi_vit/models/vit_5/models_vit5.py:72-115).

Layer norms, rotary positions and attention run on the kernels of ``packed``, forward and backward; projections and the
MLP stay PyTorch / cuBLAS.  The last block's queries are the CLS tokens alone: nothing else of it reaches the head.
"""
from __future__ import annotations

import torch
import torch.nn as nn
from torch import Tensor

from .packed import PackedPlan, RopeAxes, layer_norm, packed_attention, rope_axes


class PackedBags:
    """The layout of one packed batch: slides of ``lengths`` patches, each behind its ``num_cls`` CLS tokens, with the
    attention plans of all blocks.  Made once per batch; pass it to several calls with the same lengths."""

    def __init__(self, lengths, num_cls: int, num_heads: int, device):
        self.lengths = [int(n) for n in lengths]
        self.num_cls = num_cls
        tokens = [n + num_cls for n in self.lengths]
        self.plan = PackedPlan(tokens, heads=num_heads, device=device)
        self.cls_plan = PackedPlan([num_cls] * len(tokens), tokens, heads=num_heads, device=device)
        starts = [sum(tokens[:i]) for i in range(len(tokens))]
        self.cls_index = torch.tensor([s + c for s in starts for c in range(num_cls)], dtype=torch.int64, device=device)


class PackedAttention(nn.Module):
    """Multi-head attention of every token over its own slide; same parameters as ``StaticSparseAttention``."""

    def __init__(self, embed_dim: int, num_heads: int) -> None:
        super().__init__()
        if embed_dim % num_heads != 0:
            raise ValueError(f"embed_dim ({embed_dim}) must be divisible by num_heads ({num_heads})")
        if embed_dim // num_heads % 8 or embed_dim // num_heads > 128:
            raise ValueError(f"head dimensions are multiples of 8 up to 128, not {embed_dim // num_heads}")
        self.embed_dim, self.num_heads, self.head_dim = embed_dim, num_heads, embed_dim // num_heads
        self.qkv = nn.Linear(embed_dim, 3 * embed_dim, bias=True)
        self.out_proj = nn.Linear(embed_dim, embed_dim, bias=True)

    def forward(self, x: Tensor, bags: PackedBags, positions: Tensor | None = None, rope: RopeAxes | None = None,
                cls_only: bool = False) -> Tensor:
        """``x (T, embed_dim)``; ``positions`` (T, axes), zero for CLS tokens (no rotation).  ``cls_only``: the result of
        the CLS tokens alone, (slides * num_cls, embed_dim)."""
        T, H, D = x.shape[0], self.num_heads, self.head_dim
        if cls_only:
            E = self.embed_dim
            w, b = self.qkv.weight, self.qkv.bias
            q = nn.functional.linear(x[bags.cls_index], w[:E], b[:E]).view(-1, H, D).to(torch.bfloat16)   # CLS: angle 0
            kv = nn.functional.linear(x, w[E:], b[E:]).view(T, 2 * H, D).to(torch.bfloat16)
            k, v = kv[:, :H], kv[:, H:]
            k = k if rope is None else rope_axes(k, positions, rope)
            o = packed_attention(q, k, v, bags.cls_plan)
        else:
            qkv = self.qkv(x).view(T, 3 * H, D).to(torch.bfloat16)
            qk, v = qkv[:, :2 * H], qkv[:, 2 * H:]
            qk = qk if rope is None else rope_axes(qk, positions, rope)
            o = packed_attention(qk[:, :H], qk[:, H:], v, bags.plan)
        return self.out_proj(o.flatten(1).to(x.dtype))


class PackedViTBlock(nn.Module):
    """The pre-norm block of the other encoders around ``PackedAttention``."""

    def __init__(self, embed_dim: int, num_heads: int, expansion_factor: float = 4.0, proj_dropout: float = 0.0) -> None:
        super().__init__()
        hidden = int(embed_dim * expansion_factor)
        self.norm1 = nn.LayerNorm(embed_dim)
        self.attn = PackedAttention(embed_dim, num_heads)
        self.drop1 = nn.Dropout(proj_dropout)
        self.norm2 = nn.LayerNorm(embed_dim)
        self.mlp = nn.Sequential(nn.Linear(embed_dim, hidden), nn.GELU(), nn.Dropout(proj_dropout),
                                 nn.Linear(hidden, embed_dim), nn.Dropout(proj_dropout))

    def forward(self, x: Tensor, bags: PackedBags, positions=None, rope=None, cls_only: bool = False) -> Tensor:
        h = layer_norm(x, self.norm1.weight, self.norm1.bias, self.norm1.eps)
        a = self.drop1(self.attn(h, bags, positions, rope, cls_only))
        x = (x[bags.cls_index] if cls_only else x) + a
        return x + self.mlp(layer_norm(x, self.norm2.weight, self.norm2.bias, self.norm2.eps))


class PackedViTSlideEncoder(nn.Module):
    """Bags of patch embeddings -> slide logits, all slides of a batch in one packed pass.

    ``rope_sections``: channel pairs of each position axis (for example level, row and column), None: no rotary
    positions; ``rope_scales``: a factor for each axis (1 / the coordinate that maps to one radian).  Activations run in
    the type of the projections' results: bf16 under autocast; attention itself is always bf16."""

    packs_bags = True           # training.slide_step hands a ragged batch over whole

    def __init__(self, in_features: int = 1280, out_features: int = 1, embed_dim: int = 384, num_heads: int = 6,
                 num_layers: int = 6, num_cls: int = 2, rope_sections=None, rope_scales=None, rope_theta: float = 10000.0,
                 expansion_factor: float = 4.0, proj_dropout: float = 0.0) -> None:
        super().__init__()
        if num_cls < 1 or num_layers < 1:
            raise ValueError("the encoder needs one CLS token and one layer at least")
        self.num_cls, self.num_heads, self.embed_dim, self.out_features = num_cls, num_heads, embed_dim, out_features
        self.input_proj = nn.Linear(in_features, embed_dim)
        self.cls_tokens = nn.Parameter(torch.zeros(1, num_cls, embed_dim))
        nn.init.trunc_normal_(self.cls_tokens, std=0.02)
        self.blocks = nn.ModuleList(PackedViTBlock(embed_dim, num_heads, expansion_factor, proj_dropout)
                                    for _ in range(num_layers))
        self.rope = None if rope_sections is None else RopeAxes(embed_dim // num_heads, rope_sections, theta=rope_theta,
                                                                scales=rope_scales)
        self.norm = nn.LayerNorm(embed_dim)
        self.cls_pool = nn.Linear(embed_dim, 1, bias=False)
        self.head = nn.Linear(embed_dim, out_features)
        nn.init.xavier_uniform_(self.input_proj.weight)
        nn.init.zeros_(self.input_proj.bias)
        nn.init.zeros_(self.head.bias)

    def pack(self, lengths, device) -> PackedBags:
        """The layout of a batch of slides of these lengths, for calls that share it."""
        return PackedBags(lengths, self.num_cls, self.num_heads, device)

    def forward(self, bags, coords=None, layout: PackedBags | None = None) -> dict[str, Tensor]:
        """``bags``: a list of (N_i, in_features) tensors, one such tensor, or (B, N, in_features); ``coords``: for each bag
        (N_i, axes), used if the encoder was built with ``rope_sections``.  Returns logits (slides, out_features)."""
        if isinstance(bags, Tensor):
            bags = [bags] if bags.dim() == 2 else list(bags)
            if coords is not None and isinstance(coords, Tensor):
                coords = [coords] if coords.dim() == 2 else list(coords)
        if not bags:
            raise ValueError("an empty batch has no logits")
        lengths = [b.shape[0] for b in bags]
        dev = bags[0].device
        layout = layout or self.pack(lengths, dev)
        if layout.lengths != lengths or layout.num_cls != self.num_cls:
            raise ValueError(f"the layout is for bags of {layout.lengths} patches, not {lengths}")
        patches = self.input_proj(torch.cat(bags))
        cls = self.cls_tokens[0].to(patches.dtype)
        x = torch.cat([t for p in patches.split(lengths) for t in (cls, p)])
        positions = None
        if self.rope is not None:
            if coords is None or len(coords) != len(bags) or any(c.shape != (n, len(self.rope.sections))
                                                                 for c, n in zip(coords, lengths)):
                raise ValueError(f"the encoder's rotary positions need coords of {len(self.rope.sections)} axes for every patch")
            zero = coords[0].new_zeros((self.num_cls, coords[0].shape[1]))
            positions = torch.cat([t for c in coords for t in (zero, c)])
            positions = positions if positions.dtype in (torch.int32, torch.int64) else positions.float()
        for i, blk in enumerate(self.blocks):
            x = blk(x, layout, positions, self.rope, cls_only=i + 1 == len(self.blocks))
        x = layer_norm(x, self.norm.weight, self.norm.bias, self.norm.eps).view(len(bags), self.num_cls, self.embed_dim)
        pooled = (torch.softmax(self.cls_pool(x), dim=1) * x).sum(dim=1)
        return {"logits": self.head(pooled)}
