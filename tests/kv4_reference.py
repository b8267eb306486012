"""The 4-bit cache from its definition, in plain tensor operations: rows, rotation, attention in 64 bits, and the bytes of a block."""
import math

import torch

PAGE = 64


def rotated(x, pos, base):
    """bf16 [T, heads, hd] at positions pos [T], in 64 bits."""
    hd = x.shape[-1]
    ang = pos.double()[:, None, None] * base ** (-2.0 * torch.arange(hd // 2, dtype=torch.float64, device=x.device) / hd)
    a, b = x[..., :hd // 2].double(), x[..., hd // 2:].double()
    return torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)


def quantised(x):
    """f32 [..., hd] -> nibbles 0..15 (int64), s, z (f32)."""
    x = x.float()
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    s = ((hi - lo) / 15.0).bfloat16().float()
    z = (lo + 8.0 * s).bfloat16().float()
    n = torch.where(s > 0, ((x - z) / s).round().clamp(-8, 7), torch.zeros_like(x))
    bad = ~(torch.isfinite(x).all(-1, keepdim=True) & torch.isfinite(s) & torch.isfinite(z))
    nan = torch.full_like(s, math.nan)
    n = torch.where(bad | n.isnan(), torch.zeros_like(n), n)
    return (n + 8).long(), torch.where(bad, nan, s), torch.where(bad, nan, z)


def values(x):
    n, s, z = quantised(x)
    return (n.float() - 8.0) * s + z


def block_of(kn, ks, kz, vn, vs, vz):
    """Bytes of one block from nibbles [16, hd] and factors [16, 1]: the layout spelled out one nibble at a time."""
    hd = kn.shape[1]
    nib = [0] * (32 * hd)
    main = 128 if hd == 128 else 64
    order = [0, 4, 1, 5, 2, 6, 3, 7]
    for p in range(16):
        for d in range(hd):
            word = p * main // 8 + d // 8 if d < main else 2 * main + p * ((hd - main) // 8) + (d - main) // 8
            nib[8 * word + order[d % 8]] = int(kn[p, d])
            u, w = p // 2, d // 4
            if hd == 128:
                word = 32 * u + 4 * ((w // 4) ^ (2 * (u % 4))) + w % 4
            elif w < 16:
                word = 16 * u + (w ^ (8 * (u // 2 % 2)))
            else:
                word = 128 + u * ((hd - main) // 4) + w - 16
            nib[16 * hd + 8 * word + 4 * (p % 2) + d % 4] = int(vn[p, d])
    out = [nib[2 * i] | nib[2 * i + 1] << 4 for i in range(16 * hd)]
    for s, z in ((ks, kz), (vs, vz)):
        for p in range(16):
            out += torch.stack([s[p, 0], z[p, 0]]).bfloat16().cpu().view(torch.uint8).tolist()
    return torch.tensor(out, dtype=torch.uint8)


def attention(q, k, v, cached, scale, amask=None):
    """One sequence in 64 bits: q [n, heads, hd], k / v [cached + n, kv heads, hd] -> out [n, heads, hd]; rows that see nothing are zeros."""
    n, heads, hd = q.shape
    R = heads // k.shape[1]
    q, k, v = q.double(), k.double().repeat_interleave(R, 1), v.double().repeat_interleave(R, 1)
    a = torch.einsum("nhd,lhd->hnl", q, k) * scale
    see = torch.ones(n, cached + n, dtype=torch.bool, device=q.device)
    see[:, cached:] = (torch.ones(n, n, device=q.device).tril() if amask is None else amask[:, :n]) != 0
    a = a.masked_fill(~see, -math.inf)
    top = a.amax(-1, keepdim=True)
    p = torch.where(see, (a - top.clamp(min=-1e300)).exp(), torch.zeros_like(a))
    den = p.sum(-1, keepdim=True)
    vv = torch.where(see.any(0)[:, None, None], v, torch.zeros_like(v))
    out = torch.zeros(n, heads, hd, dtype=torch.float64, device=q.device)
    for i in range(n):                                     # an unseen row may be NaN: it is not multiplied by zero but left out
        m = see[i]
        if m.any():
            out[i] = torch.einsum("hl,lhd->hd", p[:, i][:, m] / den[:, i], vv[m])
    return out
