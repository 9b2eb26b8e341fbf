"""Plain 64-bit forms of the low-bit operators for the tests (not a test
module): MXFP4 blocks, the FP8 latent cache's records, sink attention."""

from __future__ import annotations

import torch

E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def mxfp4(x: torch.Tensor):
    """(element codes 0..15, scale codes, values) of x [..., K] on the CPU, by
    the definition: the nearest of the sixteen values, a tie to the even code."""
    xb = x.detach().cpu().double().unflatten(-1, (-1, 32))
    amax = xb.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(xb).all(-1, keepdim=True)
    safe = torch.where(bad | (amax == 0), torch.ones_like(amax), amax)
    e = (torch.frexp(safe).exponent - 3).clamp(-127, 127)   # frexp's mantissa is in [1/2, 1)
    e = torch.where(amax == 0, torch.full_like(e, -127), e)
    a = torch.where(bad, torch.zeros_like(xb), xb).abs() * torch.exp2(-e.double())
    d = (a.clamp(max=6.0).unsqueeze(-1) - E2M1).abs()
    near = d == d.amin(-1, keepdim=True)                    # one value, or two at a tie
    rank = torch.tensor([0, 9, 1, 10, 2, 11, 3, 12])        # even codes first
    code = torch.where(near, rank, 99).argmin(-1)
    neg = torch.signbit(xb) & ~bad
    sc = torch.where(bad, torch.full_like(e, 255), e + 127).squeeze(-1)
    val = E2M1[code] * torch.where(neg, -1.0, 1.0) * torch.exp2(e.double())
    val = torch.where(bad, torch.full_like(val, float("nan")), val)
    return (code + 8 * neg).flatten(-2), sc, val.flatten(-2)


def pack_nibbles(code: torch.Tensor) -> torch.Tensor:
    return (code[..., 0::2] | (code[..., 1::2] << 4)).to(torch.uint8)


def mxfp4_values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """fp64 values of packed codes [..., K/2] and scale codes [..., K/32]."""
    c = codes.cpu().long()
    nib = torch.stack([c & 15, c >> 4], -1).flatten(-2)
    v = E2M1[nib & 7] * (1 - 2 * (nib >> 3)).double()
    s = torch.exp2(scales.cpu().double() - 127)
    s = torch.where(scales.cpu() == 255, torch.full_like(s, float("nan")), s)
    return (v.unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)


def attention(q: torch.Tensor, kv: torch.Tensor, idx: torch.Tensor, sink: torch.Tensor, scale: float):
    """q [B,S,H,D], kv [B,N,D], idx [B,S,K], sink [H] -> (o, A, d, lse) in
    fp64: the output, A = sum_k p_k |v_k| and d = the largest sum_d |q_d k_d|
    * scale of a row's live keys (for error bounds)."""
    q, kv, sink = q.cpu().double(), kv.cpu().double(), sink.cpu().double()
    B, S, H, D = q.shape
    g = torch.stack([kv[b][idx[b].cpu().long().clamp(min=0)] for b in range(B)])       # [B,S,K,D]
    dead = (idx.cpu() < 0).unsqueeze(2)
    z = (torch.einsum("bshd,bskd->bshk", q, g) * scale).masked_fill(dead, float("-inf"))
    mag = (torch.einsum("bshd,bskd->bshk", q.abs(), g.abs()) * scale).masked_fill(dead, 0.0)
    sk = sink.view(1, 1, H, 1).expand(B, S, H, 1)
    za = torch.cat([z, sk], -1)
    lse = torch.logsumexp(za, -1)
    p = torch.exp(z - lse.unsqueeze(-1))
    d = mag.amax(-1) if mag.shape[-1] else torch.zeros(B, S, H, dtype=torch.float64)
    return torch.einsum("bshk,bskd->bshd", p, g), torch.einsum("bshk,bskd->bshd", p, g.abs()), d, lse
