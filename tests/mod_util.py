"""Plain 64-bit restatement of attention with modified scores, and the error that the kernels'
roundings allow. Used by the GPU tests of attn_flash_mod_* and attn_flash_kv4_stream."""
from __future__ import annotations

import math

import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def visible(B, Sq, lens, causal, begin=None, end=None, Sk=None, dev="cuda"):
    """Truth values [B][Sq][Sk]: which keys each query sees. lens: each sequence's keys (its key axis)."""
    Sk = Sk if Sk is not None else max(lens)
    j = torch.arange(Sk, device=dev)
    n = torch.as_tensor(lens, device=dev).view(B, 1, 1)
    i = torch.arange(Sq, device=dev).view(1, Sq, 1)
    seen = (j < n).expand(B, Sq, Sk).clone()
    if causal:
        seen &= j <= n - Sq + i
    if begin is not None:
        seen &= j >= begin.view(B, Sq, 1)
    if end is not None:
        seen &= j < end.view(B, Sq, 1)
    return seen


def attend(q, k, v, seen, lens, cap=0.0, slopes=None, p_half=2.0 ** -8, out=torch.float32, p_abs=0.0):
    """64-bit attention and a bound on each element's error. q [B][Hq][Sq][D], k and v [B][Hkv][Sk][D] (any
    float type; exact values), seen [B][Sq][Sk]. The bound counts
      - P rounded to 1 / p_half steps: p_half * A, A = sum_j p_j |v_j|
      - p_abs per key, where P's type has a smallest step (fp16: 2^-24). The 4-bit kernel rounds a weight
        w = 2^(z - m) and then w * s, s the value's scale, each to fp16: 2^-11 of itself twice (p_half
        2^-10), or half of the smallest step, 2^-25 (times s for the first). A value is q * s, |q| <= 8, and
        l >= 2^4 (m is a maximum less 4, and only ever replaced by a larger one), so a key adds at most
        2^-25 * 8 * (1 + s) / 2^4 = 2^-26 * (1 + s); s is at most a sixth of the largest |v| of its group
        (a / 7 rounded to 4 bits). A merge of partials scales an error by what it scales the partial's
        weights, and the partial with the largest m keeps l >= 2^4
      - scores: D products and D sums in 32 bits (2^-23 each on the tensor cores) of size |q||k|; scale,
        cap and bias a few roundings and the tanh fit (1e-6 relative in all); an error e of a score moves
        a weight by the factor 1 + e and the sum of weights by as much: 2 e A
      - exponential, sums, accumulators, merges of key pieces in 32 bits: 2^-17 A (thousands of terms)
      - the output's own rounding: half a step of |o|"""
    B, Hq, Sq, D = q.shape
    Hkv = k.shape[1]
    g = Hq // Hkv
    q, k, v = q.double(), k.double(), v.double()
    o = torch.zeros_like(q)
    tol = torch.zeros_like(q)
    n = torch.as_tensor(lens, device=q.device)
    j = torch.arange(k.shape[2], device=q.device)
    for b in range(B):
        pos = n[b] - Sq + torch.arange(Sq, device=q.device)
        dist = (pos[:, None] - j[None]).abs().double()
        sb = seen[b]
        some = sb.any(1)
        near = torch.where(sb, dist, torch.full_like(dist, math.inf)).amin(1, keepdim=True)
        near = torch.where(some[:, None], near, torch.zeros_like(near))
        for h in range(Hq):
            kk, vv = k[b, h // g], v[b, h // g]
            # what a masked key holds is not a number's business
            used = sb.any(0)
            kk = torch.where(used[:, None], kk, torch.zeros_like(kk))
            vv = torch.where(used[:, None], vv, torch.zeros_like(vv))
            s = q[b, h] @ kk.T / math.sqrt(D)
            size = (q[b, h].abs() @ kk.abs().T / math.sqrt(D)).amax(1, keepdim=True)
            if cap > 0:
                s = cap * torch.tanh(s / cap)
            big = s.abs()
            if slopes is not None:
                bias = slopes[h].double() * (dist - near)
                s = s - bias
                big = big + torch.where(bias < 40, bias.abs(), torch.zeros_like(bias))
            s = torch.where(sb, s, torch.full_like(s, -math.inf))
            m = s.amax(1, keepdim=True)
            p = torch.where(sb, (s - m).exp(), torch.zeros_like(s))
            p = torch.where(some[:, None], p, torch.zeros_like(p))
            l = p.sum(1, keepdim=True).clamp(min=1e-300)
            p = p / l
            o[b, h] = p @ vv
            e = D * 2.0 ** -23 * size + 1e-6 * torch.where(sb, big, torch.zeros_like(big)).amax(1, keepdim=True)
            A = p @ vv.abs()
            tol[b, h] = (p_half + 2 * e + 2.0 ** -17) * A + HALF[out] * o[b, h].abs() + 1e-30
            if p_abs:
                tol[b, h] += p_abs * (sb.double() @ (1 + vv.abs().amax(1, keepdim=True)))
    return o, tol
