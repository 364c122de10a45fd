"""64-bit restatements of the text-side operators (rotary positions; masked, capped and
biased attention; a shared prefix), from their formulas, with the terms of their error bounds.
Test infrastructure only; torch float64 on whatever device the inputs live on."""
from __future__ import annotations

import math

import torch


def rotary(x, positions, inv_freq, layout="half", magnitude=1.0, inverse=False):
    """x [B, S, H, D], positions [S] or [B, S], inv_freq fp64 [r / 2] -> float64."""
    r = 2 * inv_freq.numel()
    pos = positions if positions.dim() == 2 else positions[None]
    theta = pos.double()[..., None] * inv_freq.double()
    c, s = (magnitude * theta.cos())[:, :, None], (magnitude * theta.sin())[:, :, None]
    if inverse:
        s = -s
    y = x.double().clone()
    if layout == "half":
        ia, ib = torch.arange(0, r // 2), torch.arange(r // 2, r)
    else:
        ia, ib = torch.arange(0, r, 2), torch.arange(1, r, 2)
    ia, ib = ia.to(x.device), ib.to(x.device)
    a, b = x.double()[..., ia], x.double()[..., ib]
    y[..., ia] = a * c - b * s
    y[..., ib] = b * c + a * s
    return y


def attention(q, k, v, window=(-1, -1), prefix_lens=None, q_ids=None, k_ids=None, kv_lens=None, offsets=None,
              softcap=0.0, slopes=None, bias_table=None, sm_scale=None, prefix_k=None, prefix_v=None):
    """NHD tensors -> (out, weighted magnitude sum_j p_j |v_j|, keys seen) in float64; the
    second bounds what a relative error of the weights can move.  offsets: int per batch
    element (own tokens).  Keys that a row does not see do not enter, whatever they hold."""
    B, Sq, Hq, D = q.shape
    Skv, Hkv = k.shape[1], k.shape[2]
    P = 0 if prefix_k is None else prefix_k.shape[0]
    G = Hq // Hkv
    scale = 1 / math.sqrt(D) if sm_scale is None else sm_scale
    out = torch.zeros(B, Sq, Hq, D, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    count = torch.zeros(B, Sq, dtype=torch.int64, device=q.device)
    for b in range(B):
        n = P + (Skv if kv_lens is None else min(max(int(kv_lens[b]), 0), Skv))
        off = (Skv - Sq) if offsets is None else int(offsets[b])
        for i in range(Sq):
            t = P + off + i
            j = torch.arange(n, device=q.device)
            seen = torch.ones(n, dtype=torch.bool, device=q.device)
            if window[0] >= 0:
                seen &= j >= t - window[0]
            if window[1] >= 0:
                seen &= j <= t + window[1]
            if prefix_lens is not None:
                seen |= j < int(prefix_lens[b])
            if q_ids is not None:
                seen &= (k_ids[b, j] == q_ids[b, i]) & (q_ids[b, i] >= 0)
            j = j[seen]
            count[b, i] = j.numel()
            if j.numel() == 0:
                continue
            kk, vv = (torch.cat([prefix_k, k[b]]), torch.cat([prefix_v, v[b]])) if P else (k[b], v[b])
            kk, vv = kk[j].double(), vv[j].double()
            qq = q[b, i].double().view(Hkv, G, D)
            s = torch.einsum("hgd,nhd->hgn", qq, kk).reshape(Hq, -1) * scale
            if softcap:
                s = softcap * torch.tanh(s / torch.full_like(s, softcap))  # (a scalar goes by its reciprocal, which may overflow)
            if slopes is not None:
                s = s - slopes.double()[:, None] * (t - j).abs().double()[None]
            if bias_table is not None:
                R = bias_table.shape[1] // 2
                s = s + bias_table.double()[:, (j - t).clamp(-R, R) + R]
            p = torch.softmax(s, -1).view(Hkv, G, -1)
            out[b, i] = torch.einsum("hgn,nhd->hgd", p, vv).reshape(Hq, D)
            mag[b, i] = torch.einsum("hgn,nhd->hgd", p, vv.abs()).reshape(Hq, D)
    return out, mag, count


def attention_bound(ref, mag, keys, dtype, v_max):
    """Elementwise bound on |kernel - ref|.  u = eps / 2 of the type.
      weights rounded to the type, each by at most u:              u * mag
      scores: about three fp32 roundings of a logit below 2^6 (2^-17), the capped tanh to
      2^-22 of a cap below 2^6 twice (2^-15), exp2 to 2^-22, and fp32 sums of up to 2^13
      terms, each addition to 2^-24 (2^-11 where all errors line up):  2^-10 * mag
      the result rounded once:                                       u * |ref|
      fp16 weights below 2^-14 are multiples of 2^-24 (the greatest weight is 1 or more):
                                                                     keys * 2^-25 * max |v|"""
    u = torch.finfo(dtype).eps / 2
    tol = u * mag + 2.0 ** -10 * mag + u * ref.abs() + 1e-30
    if dtype == torch.float16:
        tol = tol + keys[:, :, None, None].double() * 2.0 ** -25 * v_max + 2.0 ** -25
    return tol
