"""Plain 64-bit forms of the 8-bit operators and of attention over a cache, for their tests."""
import math

import torch


def codes64(q, s):
    """values of e4m3 codes q [..., n] with scale bytes s [...]"""
    return q.view(torch.float8_e4m3fn).double() * torch.exp2(s.double() - 127)[..., None]


def quant64(x):
    """(codes' values, scale exponent) of the blocks x [..., block], from the definition, in float64"""
    x = x.double()
    good = torch.isfinite(x)
    top = torch.where(good, x.abs(), torch.zeros_like(x)).amax(-1)
    e = torch.ceil(torch.log2(torch.where(top > 0, top, torch.full_like(top, 448.0)) / 448)).clamp(min=-126)
    e = torch.where(top > 0, e, torch.zeros_like(e))
    y = x * torch.exp2(-e)[..., None]
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6, max=448.0))) - 3)
    y = torch.where(good, torch.round(y / step) * step, torch.full_like(y, math.nan))
    return y * torch.exp2(e)[..., None], e


def seen_keys(B, T, S, kv_len, pad=None, mask=None, n=None):
    """bool [B, T, S]: which positions each token sees"""
    p = torch.arange(S)
    ln = kv_len.cpu().long()[:, None]
    see = p[None] < ln
    if pad is not None:
        see = see & (p[None] >= pad.cpu().long()[:, None])
    see = see[:, None].expand(B, T, S).clone()
    if mask is not None:
        mask = mask.cpu().expand(B, T)
        n = torch.full((B,), T) if n is None else n.cpu().long()
        for b in range(B):
            for t in range(T):
                for j in range(int(n[b])):
                    if int(mask[b, t]) >> j & 1:
                        see[b, t, int(kv_len[b]) + j] = True
    return see


def attend64(q, k, v, see, scale):
    """q [B, T, Hq, hd], k / v [B, H, S, hd] float64, see [B, T, S] -> (out, sum of w |v|, largest |score| bound)"""
    B, T, Hq, hd = q.shape
    G = Hq // k.shape[1]
    see = see.to(q.device)
    out, mag, top = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(B, T, Hq, 1, dtype=q.dtype, device=q.device)
    for b in range(B):
        for h in range(Hq):
            for t in range(T):
                at = see[b, t].nonzero()[:, 0]
                if at.numel() == 0:
                    continue
                kk, vv = k[b, h // G, at], v[b, h // G, at]
                w = torch.softmax((kk * q[b, t, h]).sum(-1) * scale, 0)
                out[b, t, h] = (w[:, None] * vv).sum(0)
                mag[b, t, h] = (w[:, None] * vv.abs()).sum(0)
                top[b, t, h] = ((kk.abs() * q[b, t, h].abs()).sum(-1) * scale).max()
    return out, mag, top


def attn_tol(ref, mag, top, keys, hd, p_step, out_dtype):
    """A score is off by at most hd steps of its magnitude's sum (f32 accumulation, twice the half step) and the
    exponential by 2^-20; both reach numerator and denominator; P is rounded by p_step, the sums over keys by
    keys * 2^-23, the output by half a step of its type."""
    half = torch.finfo(out_dtype).eps / 2
    rel = p_step + 2 * (hd * 2.0 ** -23 * top + 2.0 ** -20) + keys * 2.0 ** -23
    return mag * rel * (1 + half) + half * ref.abs() + 1e-30
