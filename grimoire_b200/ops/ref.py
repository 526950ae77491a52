"""Plain PyTorch fp32 references of every device op.

Two uses: (1) the oracle that the CUDA kernels are compared against in ``tests/ -m gpu`` and
(2) the CPU path of the engine (tiny-model correctness runs, gloo multi-rank tests).  The math here
follows the numerics conventions the reference pins with tests (q/k norm before RoPE, NeoX RoPE
over the first ``rot`` dims, zero-centred norm weights, int8 KV with max|x|/127 scales ...).
"""
from __future__ import annotations

import math
from typing import Optional

import torch

PAGE = 16


def rmsnorm(h: torch.Tensor, w: torch.Tensor, eps: float, offset: float) -> torch.Tensor:
    h = h.float()
    r = torch.rsqrt(h.pow(2).mean(dim=-1, keepdim=True) + eps)
    return h * r * (offset + w.float())


def linear_dequant(x: torch.Tensor, w_deq: torch.Tensor) -> torch.Tensor:
    """x [M][K] (any float dtype, rounded to bf16 like the kernel input) @ dequantized W[N][K]^T in fp32."""
    return x.bfloat16().float() @ w_deq.float().t()


def swiglu(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    return torch.nn.functional.silu(gate.float()) * up.float()


def rope_inv_freq(rot: int, theta: float) -> torch.Tensor:
    return 1.0 / (theta ** (torch.arange(0, rot, 2, dtype=torch.float32) / rot))


def apply_rope(x: torch.Tensor, pos: torch.Tensor, inv_freq: torch.Tensor, rot: int) -> torch.Tensor:
    """x [M][H][D] fp32, NeoX half-split over the first ``rot`` dims (src/ops.cpp:870-912)."""
    ang = pos.float()[:, None] * inv_freq[None, :]          # [M][rot/2]
    cos, sin = ang.cos()[:, None, :], ang.sin()[:, None, :]
    a, b = x[..., : rot // 2], x[..., rot // 2: rot]
    out = x.clone()
    out[..., : rot // 2] = a * cos - b * sin
    out[..., rot // 2: rot] = b * cos + a * sin
    return out


def head_rmsnorm(x: torch.Tensor, w: Optional[torch.Tensor], eps: float, offset: float) -> torch.Tensor:
    if w is None:
        return x
    r = torch.rsqrt(x.pow(2).mean(dim=-1, keepdim=True) + eps)
    return x * r * (offset + w.float())


def quant_i8_rows(x: torch.Tensor):
    """Per-(token, head) int8 quantisation: scale = max|x|/127 (src/kv_k8.hpp:19-59)."""
    amax = x.abs().amax(dim=-1)
    scale = torch.where(amax > 0, amax / 127.0, torch.ones_like(amax))
    q = torch.round(x / scale[..., None]).clamp(-127, 127).to(torch.int8)
    return q, scale


def attention_rows(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_pos: torch.Tensor, scale: float,
                   window: int = 0) -> torch.Tensor:
    """q [M][Hq][D]; k,v [T][Hkv][D] (dequantized); row m sees keys 0..q_pos[m] (within window)."""
    M, Hq, D = q.shape
    T, Hkv, _ = k.shape
    G = Hq // Hkv
    kk = k.float().repeat_interleave(G, dim=1)               # [T][Hq][D]
    vv = v.float().repeat_interleave(G, dim=1)
    s = torch.einsum("mhd,thd->mht", q.float(), kk) * scale
    keys = torch.arange(T)[None, None, :]
    qp = q_pos.long()[:, None, None]
    ok = keys <= qp
    if window > 0:
        ok = ok & (keys > qp - window)
    s = s.masked_fill(~ok, float("-inf"))
    p = torch.softmax(s, dim=-1)
    return torch.einsum("mht,thd->mhd", p, vv)


def argmax_lowest(logits: torch.Tensor) -> torch.Tensor:
    """arg-max with ties resolved to the lowest index."""
    mx = logits.max(dim=-1, keepdim=True).values
    idx = torch.arange(logits.shape[-1], device=logits.device).expand_as(logits)
    big = torch.full_like(idx, logits.shape[-1])
    return torch.where(logits == mx, idx, big).min(dim=-1).values.to(torch.int32)


def softmax_scale(head_dim: int) -> float:
    return 1.0 / math.sqrt(head_dim)


# ---------------------------------------------------------------------------------------------
# 4-bit KV pages (layout: csrc/kernels/kv4.cuh)
# ---------------------------------------------------------------------------------------------
def quant_kv4(x: torch.Tensor):
    """bf16 [..., D] -> (codes uint8 [..., D] in 1..15, maxima bf16 [..., D / 32]).  The group of element d is
    (d / 4) % (D / 32); a group whose maximum is zero or not finite has codes of zero (8).  The factor 7 is split so that it
    cannot overflow; numerator and denominator are exact."""
    ng = x.shape[-1] // 32
    quads = x.float().unflatten(-1, (8, ng, 4))
    amax = quads.abs().amax(dim=(-3, -1))
    ok = (amax > 0) & torch.isfinite(amax)
    div = torch.where(ok, amax, torch.ones_like(amax))[..., None, :, None]
    q = torch.where(ok[..., None, :, None], torch.round(0.875 * quads / (0.125 * div)), torch.zeros_like(quads))
    return (q + 8).to(torch.uint8).flatten(-3), amax.to(torch.bfloat16)


def kv4_views(data: torch.Tensor):
    """(codes uint8 [P][Hkv][K, V][16][D / 2], maxima bf16 [P][Hkv][16][K, V][D / 32]): views of the page records."""
    D = data.shape[-1] // 18
    return (data[..., : 16 * D].unflatten(-1, (2, PAGE, D // 2)),
            data[..., 16 * D:].view(torch.bfloat16).unflatten(-1, (PAGE, 2, D // 32)))


def kv4_rows(data: torch.Tensor, page: torch.Tensor, slot: torch.Tensor):
    """K, V of the cached tokens (page[i], slot[i]) as fp32 [n][Hkv][D]."""
    codes, amax = kv4_views(data)
    c, a = codes[page, :, :, slot], amax[page, :, slot].float()              # [n][Hkv][2][D/2], [n][Hkv][2][D/32]
    q = torch.stack((c & 15, c >> 4), dim=-1).flatten(-2).float() - 8
    x = (0.125 * q.unflatten(-1, (8, a.shape[-1], 4)) * a[..., None, :, None] / 7 * 8).flatten(-3)
    return x[:, :, 0], x[:, :, 1]


def kv4_place(block_table: torch.Tensor, slot: int, positions: torch.Tensor, pages: int):
    """(page, place in the page, mapped) of positions of one sequence; a table entry outside [0, pages) maps nothing."""
    inside = (positions >= 0) & (positions < block_table.shape[1] * PAGE)
    if not 0 <= slot < block_table.shape[0]:
        inside = torch.zeros_like(inside)
        slot = 0
    p = positions.clamp(0, block_table.shape[1] * PAGE - 1).long()
    page = block_table[slot, p // PAGE].long()
    ok = inside & (page >= 0) & (page < pages)
    return page.clamp(0, pages - 1), p % PAGE, ok


def kv4_attention(q, row_seq, row_pos, block_table, data, Hq: int, scale: float, window: int = 0):
    """Attention of independent rows over the pages: (out fp32 [M][Hq * D], weights: list of fp32 [Hq][tokens])."""
    P, Hkv, D = data.shape[0], data.shape[1], data.shape[2] // 18
    M, G = q.shape[0], Hq // Hkv
    out, weights = torch.zeros(M, Hq, D), []
    for m in range(M):
        n = max(0, min(int(row_pos[m]) + 1, block_table.shape[1] * PAGE))
        t = torch.arange(n)
        page, slot, ok = kv4_place(block_table, int(row_seq[m]), t, P)
        if window > 0:
            ok = ok & (t >= n - window)
        w = torch.zeros(Hq, n)
        if bool(ok.any()):
            k, v = kv4_rows(data, page[ok], slot[ok])
            s = torch.einsum("hgd,thd->hgt", q[m].float().reshape(Hkv, G, D), k) * scale
            p = torch.softmax(s, dim=-1)
            out[m] = torch.einsum("hgt,thd->hgd", p, v).reshape(Hq, D)
            w[:, ok] = p.reshape(Hq, -1)
        weights.append(w)
    return out.reshape(M, Hq * D), weights
