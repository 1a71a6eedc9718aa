"""An attention block of a serving program: norm, projections, rotary positions and attention over a paged 8-bit
cache, for prompts and for single tokens alike.

    h = x + residual ;  n = rms_norm(h) as e4m3 ;  q, k, v = n @ W_qkv^T (block-scaled fp8 product)
    q, k turned by position, k and v written to the cache ;  o = attention of q over the cache ;  y = o @ W_o^T

Five launches of this package for a step of few tokens: the norm quantises, the projection reads its result as it is,
one kernel rotates, quantises and writes, one attends, one multiplies.  Pages, positions and lengths live on the
device, so a step can be captured in a CUDA graph.
"""
from __future__ import annotations

import torch

from ..ops.gemm import gemm, gemm_fp8_mx
from ..ops.kvcache import HEAD_DIM, KVCache8
from ..ops.norm import rms_norm_quant
from ..ops.rope import RopeTable
from ..ops.tp_fp8 import MxWeight


class CachedAttention:
    """``heads`` query heads over ``kv_heads`` key/value heads of 128 elements; random weights of N(0, 0.02).

    ``window`` and ``sinks`` as in :meth:`ops.kvcache.KVCache8.attend`; ``rope`` takes the arguments of
    :class:`ops.rope.RopeTable` beside the number of positions."""

    def __init__(self, hidden: int, heads: int, kv_heads: int, num_pages: int, max_positions: int, page: int = 64,
                 window: int = 0, sinks: int = 0, rope: dict | None = None, eps: float = 1e-6, seed: int = 0,
                 device=None):
        if hidden % 128 or heads % kv_heads:
            raise ValueError("hidden must be a multiple of 128 and heads of kv_heads")
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        g = torch.Generator(device=dev).manual_seed(seed)
        self.hidden, self.heads, self.kv_heads, self.eps = hidden, heads, kv_heads, eps
        self.window, self.sinks = window, sinks
        rows = (heads + 2 * kv_heads) * HEAD_DIM
        self.norm_weight = torch.ones(hidden, dtype=torch.bfloat16, device=dev)
        self.w_qkv = (torch.randn(rows, hidden, device=dev, generator=g) * 0.02).bfloat16()
        self.w_qkv_mx = MxWeight.from_bf16(self.w_qkv)
        self.w_o = (torch.randn(hidden, heads * HEAD_DIM, device=dev, generator=g) * 0.02).bfloat16()
        self.table = RopeTable(positions=max_positions, device=dev, **{"rot": HEAD_DIM, **(rope or {})})
        self.cache = KVCache8(num_pages, kv_heads, page=page, device=dev)

    def forward(self, x, pages, start, count=None, residual=None, max_len: int | None = None):
        """``x`` [B, S, hidden] bf16: the next S tokens of every sequence, ``start[b]`` of which the cache holds
        already (``count[b]`` of the S exist).  Returns ``(y, h)``, ``h`` the sum with ``residual`` (x without)."""
        B, S, _ = x.shape
        q8, _, sf, h = rms_norm_quant(x.view(B * S, -1), self.norm_weight, eps=self.eps, pow2=True,
                                      residual=None if residual is None else residual.view(B * S, -1))
        qkv = gemm_fp8_mx(q8, sf, self.w_qkv_mx.q, self.w_qkv_mx.sf).view(B, S, -1, HEAD_DIM)
        q, k, v = qkv.split((self.heads, self.kv_heads, self.kv_heads), dim=2)
        q = self.cache.append(k, v, pages, start, count=count, rope=self.table, q=q)
        o, _ = self.cache.attend(q, pages, start, count=count, window=self.window, sinks=self.sinks, max_len=max_len)
        y = gemm(o.view(B * S, -1), self.w_o)
        return y.view(B, S, -1), (x if h is None else h.view(B, S, -1))

    def reference(self, x):
        """The block over whole sequences ``x`` [B, S, hidden] in fp32, without a cache or 8-bit numbers."""
        B, S, _ = x.shape
        f = x.float()
        n = f * torch.rsqrt(f.square().mean(dim=-1, keepdim=True) + self.eps) * self.norm_weight.float()
        qkv = (n @ self.w_qkv.float().t()).view(B, S, -1, HEAD_DIM)
        t = self.table
        c, s = t.cos[:S][None, :, None], t.sin[:S][None, :, None]

        def turn(z):
            r = t.rot
            a, b = (z[..., 0:r:2], z[..., 1:r:2]) if t.interleaved else (z[..., :r // 2], z[..., r // 2:r])
            u, w = a * c - b * s, b * c + a * s
            y = torch.stack((u, w), -1).flatten(-2) if t.interleaved else torch.cat((u, w), -1)
            return torch.cat((y, z[..., r:]), -1)

        q, k, v = qkv.split((self.heads, self.kv_heads, self.kv_heads), dim=2)
        group = self.heads // self.kv_heads
        q, k = turn(q).transpose(1, 2), turn(k).transpose(1, 2).repeat_interleave(group, dim=1)
        v = v.transpose(1, 2).repeat_interleave(group, dim=1)
        i = torch.arange(S, device=x.device)
        seen = i[None, :] <= i[:, None]
        if self.window:
            seen &= (i[None, :] > i[:, None] - self.window) | (i[None, :] < self.sinks)
        p = torch.softmax((q @ k.transpose(-1, -2) / HEAD_DIM ** 0.5).masked_fill(~seen, float("-inf")), dim=-1)
        return (p @ v).transpose(1, 2).reshape(B, S, -1) @ self.w_o.float().t()
