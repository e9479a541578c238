"""ViT-B/16, the model of the end-to-end compressed train-step workload.

The reference measures its Controller on timm's ``vit_base_patch16_224`` (Activation_Compression/
test8.ipynb cell 2). timm is not a dependency of this library, so this file defines the same
architecture with the same submodule names (``patch_embed.proj``, ``blocks.<i>.attn.qkv``,
``blocks.<i>.attn.proj``, ``blocks.<i>.mlp.fc1/act/fc2``, ``norm``, ``head``), so the Controller
selects and names the same layers: 16x16 patch convolution to 768 channels, a class token and
learned position embedding, 12 pre-norm blocks (LayerNorm eps 1e-6, 12-head attention through
F.scaled_dot_product_attention, 3072-wide GELU MLP), final LayerNorm and a linear head on the
class token. Weights are random (truncated normal, std 0.02, as timm initialises them); there is
no dropout (timm's defaults are 0).

``fused=True`` builds the same model, with the same parameter names, from the block layers of
``modules.transformer``: layer norms whose backward adds the residual's gradient, linear layers with
bias, GELU and residual in the products' epilogues, and (``drop_rate``) dropout that is added to the
residual with a mask that is never stored. It trains on the GPU in bf16 or fp16, under autocast or as it is.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F
from torch import nn

from .modules import transformer


class PatchEmbed(nn.Module):
    def __init__(self, img_size=224, patch_size=16, in_chans=3, embed_dim=768):
        super().__init__()
        self.num_patches = (img_size // patch_size) ** 2
        self.proj = nn.Conv2d(in_chans, embed_dim, kernel_size=patch_size, stride=patch_size)

    def forward(self, x):
        return self.proj(x).flatten(2).transpose(1, 2)


class Attention(nn.Module):
    def __init__(self, dim, num_heads):
        super().__init__()
        self.num_heads = num_heads
        self.head_dim = dim // num_heads
        self.qkv = nn.Linear(dim, dim * 3)
        self.proj = nn.Linear(dim, dim)

    def forward(self, x):
        B, N, C = x.shape
        qkv = self.qkv(x).reshape(B, N, 3, self.num_heads, self.head_dim).permute(2, 0, 3, 1, 4)
        q, k, v = qkv.unbind(0)
        x = F.scaled_dot_product_attention(q, k, v)
        return self.proj(x.transpose(1, 2).reshape(B, N, C))


class Mlp(nn.Module):
    def __init__(self, dim, hidden):
        super().__init__()
        self.fc1 = nn.Linear(dim, hidden)
        self.act = nn.GELU()
        self.fc2 = nn.Linear(hidden, dim)

    def forward(self, x):
        return self.fc2(self.act(self.fc1(x)))


class Block(nn.Module):
    def __init__(self, dim, num_heads, mlp_ratio=4.0):
        super().__init__()
        self.norm1 = nn.LayerNorm(dim, eps=1e-6)
        self.attn = Attention(dim, num_heads)
        self.norm2 = nn.LayerNorm(dim, eps=1e-6)
        self.mlp = Mlp(dim, int(dim * mlp_ratio))

    def forward(self, x):
        x = x + self.attn(self.norm1(x))
        return x + self.mlp(self.norm2(x))


class FusedAttention(nn.Module):
    def __init__(self, dim, num_heads, drop=0.0, rng=None):
        super().__init__()
        self.num_heads = num_heads
        self.head_dim = dim // num_heads
        self.qkv = transformer.LinearAct(dim, dim * 3)
        self.proj = transformer.LinearAct(dim, dim)
        self.drop = transformer.DropoutAdd(drop, rng) if drop else None

    def forward(self, x, residual):
        B, N, C = x.shape
        qkv = self.qkv(x).view(B, N, 3, self.num_heads, self.head_dim).permute(2, 0, 3, 1, 4)
        q, k, v = qkv.unbind(0)
        x = F.scaled_dot_product_attention(q, k, v).transpose(1, 2).reshape(B, N, C)
        if self.drop is not None and self.training:
            return self.drop(self.proj(x), residual)
        return self.proj(x, residual)


class FusedBlock(nn.Module):
    def __init__(self, dim, num_heads, mlp_ratio=4.0, drop=0.0, rng=None):
        super().__init__()
        self.norm1 = transformer.LayerNorm(dim, eps=1e-6)
        self.attn = FusedAttention(dim, num_heads, drop, rng)
        self.norm2 = transformer.LayerNorm(dim, eps=1e-6)
        self.mlp = transformer.Mlp(dim, int(dim * mlp_ratio), "gelu", drop, rng)

    def forward(self, x):
        h, x = transformer.norm_residual(self.norm1, x)
        x = self.attn(h, x)
        h, x = transformer.norm_residual(self.norm2, x)
        return self.mlp(h, x)


class VisionTransformer(nn.Module):
    def __init__(self, img_size=224, patch_size=16, in_chans=3, num_classes=1000, embed_dim=768, depth=12,
                 num_heads=12, mlp_ratio=4.0, fused=False, drop_rate=0.0, dropout_seed=None):
        super().__init__()
        if drop_rate and not fused:
            raise ValueError("drop_rate needs fused=True")
        self.patch_embed = PatchEmbed(img_size, patch_size, in_chans, embed_dim)
        self.cls_token = nn.Parameter(torch.zeros(1, 1, embed_dim))
        self.pos_embed = nn.Parameter(torch.zeros(1, self.patch_embed.num_patches + 1, embed_dim))
        self.fused = fused
        self.dropout_rng = self.drop = None
        if fused:
            if drop_rate:
                self.dropout_rng = transformer.DropoutRng(dropout_seed)
                self.drop = transformer.DropoutAdd(drop_rate, self.dropout_rng)
            self.blocks = nn.Sequential(*[FusedBlock(embed_dim, num_heads, mlp_ratio, drop_rate, self.dropout_rng)
                                          for _ in range(depth)])
            self.norm = transformer.LayerNorm(embed_dim, eps=1e-6)
            self.head = transformer.LinearAct(embed_dim, num_classes)
        else:
            self.blocks = nn.Sequential(*[Block(embed_dim, num_heads, mlp_ratio) for _ in range(depth)])
            self.norm = nn.LayerNorm(embed_dim, eps=1e-6)
            self.head = nn.Linear(embed_dim, num_classes)
        self._init_weights()

    def _init_weights(self):
        nn.init.trunc_normal_(self.pos_embed, std=0.02)
        nn.init.normal_(self.cls_token, std=1e-6)
        for m in self.modules():
            if isinstance(m, (nn.Linear, transformer.LinearAct)):
                nn.init.trunc_normal_(m.weight, std=0.02)
                nn.init.zeros_(m.bias)

    def forward(self, x):
        x = self.patch_embed(x)
        x = torch.cat([self.cls_token.expand(x.shape[0], -1, -1).to(x.dtype), x], dim=1)
        x = x + self.pos_embed.to(x.dtype)
        if self.fused:
            if self.drop is not None:
                x = self.drop(self.dropout_rng(x))
            return self.head(self.norm(self.blocks(x)[:, 0]))  # (the head reads the class token only)
        x = self.blocks(x)
        x = self.norm(x)
        return self.head(x[:, 0])


def vit_base_patch16_224(num_classes=1000, **kw) -> VisionTransformer:
    return VisionTransformer(num_classes=num_classes, **kw)


__all__ = ["VisionTransformer", "vit_base_patch16_224"]
