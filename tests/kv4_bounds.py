"""How far attention over the 4-bit cache may be from its definition, from the roundings that the kernels make, each off by at most half a step and independent of the
others: the output to bf16; up to 64 query rows a kv head, probability times s to fp16 (it multiplies nibbles 0 .. 15, that is the value less the row's smallest); more rows,
keys, values and probabilities to fp16, the latter two to bf16 in pages whose values leave fp16's range. Scores and sums are fp32."""
import math

import torch

FP16, BF16 = 2.0 ** -11, 2.0 ** -8                         # half a step, relative to the value


def bounds(q, K, V, cached, scale, amask=None, many=False, wide=None):
    """One sequence in 64 bits: q [n, heads, hd], K / V [cached + n, kv heads, hd] -> (output, root of mean squares of its error ahead of the last rounding, largest error that
    does not average out), [n, heads, hd]. many: more than 64 query rows a kv head. wide bool [cached + n]: positions whose page has its values in bf16. Rows
    that see a NaN are NaN."""
    n, heads, hd = q.shape
    R, L = heads // K.shape[1], K.shape[0]
    q, k, v = q.double(), K.double().repeat_interleave(R, 1), V.double().repeat_interleave(R, 1)
    see = torch.ones(n, L, dtype=torch.bool, device=q.device)
    see[:, cached:] = (torch.ones(n, n, device=q.device).tril() if amask is None else amask[:, :n]) != 0
    none = ~(k.isfinite().all(-1) & v.isfinite().all(-1))                              # [L, heads]
    spoiled = (see[:, :, None] & none[None]).any(1)                                    # [n, heads]
    k, v = k.masked_fill(none[..., None], 0), v.masked_fill(none[..., None], 0)
    a = torch.einsum("nhd,lhd->hnl", q, k) * scale
    a = a.masked_fill(~see[None], -math.inf)
    p = (a - a.amax(-1, keepdim=True).clamp(min=-1e300)).exp().masked_fill(~see[None], 0)
    den = p.sum(-1, keepdim=True)
    p = p / torch.where(den > 0, den, torch.ones_like(den))
    mix = lambda w, x: torch.einsum("hnl,lhd->nhd", w, x)  # noqa: E731
    out = mix(p, v)
    # an error of a score, as a factor of its probability: sums in single precision over products of about the same size, and keys rounded to fp16
    size = (q.abs().sum(-1)[:, :, None] * k.abs().amax(-1).T[None] * 2.0 ** -20 * abs(scale)).transpose(0, 1)
    score = size ** 2
    if many:
        score = score + torch.einsum("nhd,lhd->hnl", q ** 2, k ** 2) * (scale * FP16) ** 2 / 3
    w = p ** 2 * score
    var = mix(w, v ** 2) - 2 * out * mix(w, v) + out ** 2 * w.sum(-1).T[..., None]
    if many:
        # probability and value, each by half a step of its type. fp16's numbers below 2^-14 are 2^-24 apart: half a step of a value there is 2^-25 = 2^-11 2^-14
        h = torch.full((L,), FP16, dtype=torch.float64, device=q.device)
        least = torch.full((L, 1, 1), 2.0 ** -14, dtype=torch.float64, device=q.device)
        if wide is not None:
            h[wide], least[wide] = BF16, 0.0
        var = var + mix(p ** 2 * (h ** 2 / 3), v ** 2 + torch.maximum(v.abs(), least * (v != 0)) ** 2)
        # ... and a probability is 2^7 times what it is there: half a step below 2^-14 is 2^-32 of the largest one
        var = var + mix(see.double().expand_as(p) * (2.0 ** -64 / 3), v ** 2)
    else:
        span = v - v.amin(-1, keepdim=True)
        most = (p.unsqueeze(-1) * span.amax(-1).T[:, None, :, None]).amax(2)            # largest p s a row, [heads, n, 1]
        var = var + mix(p ** 2, span ** 2) * FP16 ** 2 / 3 + (L * (2.0 ** -25 * most) ** 2 / 3).transpose(0, 1)
    slack = 2.0 ** -18 * mix(p, v.abs())
    if many:
        # A row whose 16 numbers lie within 16 steps of the type: rows like it round alike, whatever their signs (z is not mirrored), so these errors are not independent
        # and may add up to half a step of each: |sum p e| <= h sum p |v|.
        alike = (v.amax(-1) - v.amin(-1)) <= 32 * h[:, None] * v.abs().amax(-1)
        slack = slack + mix(p, v.abs() * (h[:, None] * alike)[..., None])
    out[spoiled] = math.nan
    return out, var.clamp(min=0).sqrt(), slack


def check(got, want, sigma, slack):
    """Every element: half a step of bf16 and six times the root of mean squares. All of them together: what the mean squares add up to (a rounding's is a third
    of half a step's square at most), a quarter more for few elements that hang together, and on top of it what does not average out (norms of a sum: at most the sum)."""
    assert torch.equal(got.isnan(), want.isnan())
    fine = ~want.isnan()
    err, o, s = (got.double() - want)[fine], want[fine], sigma[fine]
    worst = float((err.abs() / (o.abs() * BF16 + 6 * s + slack[fine]).clamp(min=1e-300)).max()) if err.numel() else 0.0
    whole = float((err.norm() - slack[fine].norm()).clamp(min=0) / ((o * BF16) ** 2 / 3 + s ** 2).sum().sqrt().clamp(min=1e-300)) if err.numel() else 0.0
    assert worst <= 1.0, worst
    assert whole <= 1.25, whole
    return worst, whole
