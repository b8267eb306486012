"""What is timed of the 4-bit K/V cache: appending to it, attending over it, compacting it after a tree was accepted.

The cache is paged: a pool of pages of 64 positions, and a table that names the pages of every sequence. A page holds one record per kv head, a
record four blocks of 16 positions. A row (one position and kv head of K or V) is `head_dim` numbers of 4 bits and a bf16 pair (s, z); it stands
for (nibble - 8) * s + z, with

    s = bf16((max - min) / 15),   z = bf16(min + 8 s),   nibble = clamp(round((x - z) / s), -8, 7) + 8        (s = 0: nibble 8)

over the rotated key or the value as they come. The plain forms below read and write that layout with elementary tensor operations.

  append   new tokens: rotate q and k (half-split pairs, angle = position * base^(-2i / head_dim)), write k and v into their slots; the
           rotated q and the rows that the cache then holds
  attend   softmax(scale * q k) v of the new tokens over what is cached ahead of them and over each other (causal, or a tree's mask)
  compact  the accepted path's rows of a token tree become contiguous, in every layer; the rows that were moved

Head layouts and base frequencies are those of the repository's model configurations.
"""
from __future__ import annotations

import math
import random
from types import SimpleNamespace

import torch

from flint_b200.tree import static_tree, tree_mask

DEV = "cuda"
PAGE = 64
own = False

# query heads, kv heads, head size, base of the rotation
HEADS = {"3b": (32, 8, 80, 1e4), "1b": (32, 8, 64, 5e5), "ref": (40, 8, 64, 1e7), "8b": (32, 8, 128, 5e5), "tiny": (8, 2, 64, 1e4)}


def listed():
    return [
        # one token of a stream: latency only
        dict(name="append-token", kind="append", heads="3b", batch=1, cached=200, new=1),
        # one token each of a ragged batch
        dict(name="append-batch", kind="append", heads="ref", batch=37, cached=3000, new=1),
        # a prompt of ordinary length, not a multiple of anything
        dict(name="append-prompt", kind="append", heads="8b", batch=1, cached=0, new=725),
        # the first tokens of an answer
        dict(name="decode-short", kind="attend", heads="3b", batch=1, cached=200, new=1, tree=False),
        # long context
        dict(name="decode-32k", kind="attend", heads="3b", batch=1, cached=32768, new=1, tree=False),
        # a batch of conversations of very different lengths, one token each
        dict(name="decode-batch", kind="attend", heads="8b", batch=24, cached=8000, new=1, tree=False),
        # chain speculation with K = 3
        dict(name="chain-4", kind="attend", heads="ref", batch=1, cached=603, new=4, tree=False),
        # the static 26-node tree over 1024 positions, and the widest one late in a conversation
        dict(name="tree-26", kind="attend", heads="3b", batch=1, cached=1024, new=26, tree=True),
        dict(name="tree-61", kind="attend", heads="8b", batch=1, cached=3001, new=61, tree=True),
        # a chunk of a long prompt behind what is cached already
        dict(name="prompt-1000", kind="attend", heads="8b", batch=1, cached=7011, new=1000, tree=False),
        # after the acceptance of a tree
        dict(name="compact-tree26", kind="compact", heads="3b", layers=40, cached=1024, new=26, path=6),
        dict(name="compact-tree61", kind="compact", heads="8b", layers=32, cached=3001, new=61, path=4),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choices(("append", "attend", "compact"), (3, 8, 1))[0]
    heads = rng.choice(("3b", "1b", "ref", "8b", "tiny"))
    if kind == "compact":
        path = rng.randint(2, 6)
        return dict(kind=kind, heads=heads, layers=rng.choice((2, 16, 32, 40)), cached=_log(rng, 1, 8000), new=rng.randint(2 * path, 64), path=path)
    shape = rng.choice(("token", "token", "batch", "chain", "tree", "prompt", "prompts"))
    if shape == "token":
        batch, cached, new = 1, _log(rng, 1, 32768), 1
    elif shape == "batch":
        batch, cached, new = _log(rng, 2, 48), _log(rng, 30, 8000), 1
    elif shape in ("chain", "tree"):
        batch, cached, new = (1, _log(rng, 1, 8000), _log(rng, 2, 64)) if shape == "tree" else (rng.choice((1, 1, 3)), _log(rng, 1, 8000), rng.randint(2, 8))
    elif shape == "prompt":
        batch, cached, new = 1, rng.choice((0, _log(rng, 1, 7000))), _log(rng, 9, 1000)
    else:
        batch, cached, new = rng.randint(2, 6), rng.choice((0, _log(rng, 1, 3000))), _log(rng, 9, 300)
    case = dict(kind=kind, heads=heads, batch=batch, cached=cached, new=new)
    if kind == "attend":
        case["tree"] = shape == "tree"
    return case


def _lengths(case):
    """Cached positions and new tokens of every sequence: the first has the most of both, the others any number up to that."""
    rng = random.Random(case["cached"] * 131 + case.get("batch", 1))
    cached, new = [case["cached"]], [case["new"]]
    for _ in range(case.get("batch", 1) - 1):
        cached.append(_log(rng, 1, case["cached"]) if case["cached"] else 0)
        new.append(rng.randint(1, case["new"]))
    return cached, new


# ---------------------------------------------------------------------------------------------------------------- the layout
def _block_bytes(hd):
    return 16 * hd + 128


def _offsets(hd, device):
    """Byte offsets inside a block: of dim d's nibble of K and V at position p (and whether it is the high nibble), [16, hd] each."""
    p, d = torch.arange(16, device=device)[:, None], torch.arange(hd, device=device)[None, :]
    slot = torch.tensor([0, 4, 1, 5, 2, 6, 3, 7], device=device)[d % 8] + 0 * p            # K: dims 8w .. 8w+7 in a word, (0, 1) (2, 3) .. 16 bits apart
    wk, wv, u = d // 8, d // 4, p // 2                                                       # V: dims 4w .. 4w+3 of an even position and of the next one
    if hd == 128:
        k = p * 64 + wk * 4
        v = u * 128 + ((wv // 4) ^ (2 * (u % 4))) * 16 + wv % 4 * 4
    else:
        k = torch.where(wk < 8, p * 32 + wk * 4, 512 + p * 8 + (wk - 8) * 4)
        v = torch.where(wv < 16, u * 64 + ((wv * 4) ^ (u // 2 % 2 * 32)), 512 + u * 16 + (wv - 16) * 4)
    nv = p % 2 * 4 + d % 4
    return k + slot // 2, slot % 2, 8 * hd + v + nv // 2, nv % 2


def _quantise(x):
    """x f32 [..., hd] -> nibble - 8, s, z (f32 holding whole numbers and bf16 values)."""
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    s = ((hi - lo) / 15).bfloat16().float()
    z = (lo + 8 * s).bfloat16().float()
    n = torch.where(s > 0, ((x - z) / s).round().clamp(-8, 7), torch.zeros_like(x))
    return n, s, z


def _pair(s, z):
    return torch.cat([s, z], -1).bfloat16().view(torch.uint8)                               # 4 bytes


def _write(pool, page, pos, hd, kq, vq):
    """Rows into the pool [pages, kv heads, record]: page [n], pos [n] inside the page, (n, s, z) of [n, kv heads, hd]."""
    rec = pool.shape[-1]
    ko, kh, vo, vh = _offsets(hd, pool.device)
    base = (page[:, None] * pool.shape[-2] + torch.arange(pool.shape[-2], device=pool.device)) * rec + (pos // 16 * _block_bytes(hd))[:, None]
    flat = pool.view(-1)
    p = pos % 16
    for (n, s, z), off, high, meta in ((kq, ko, kh, 16 * hd), (vq, vo, vh, 16 * hd + 64)):
        b = (n + 8).to(torch.uint8)
        order = torch.argsort(off[p] * 2 + high[p], dim=-1)                                 # the two nibbles of a byte side by side
        at = off[p].gather(-1, order)[:, 0::2]
        b = b.gather(-1, order[:, None].expand_as(b))
        flat[base[..., None] + at[:, None]] = b[..., 0::2] | (b[..., 1::2] << 4)
        flat[base[..., None] + (meta + p * 4)[:, None, None] + torch.arange(4, device=pool.device)] = _pair(s, z)


def _unpack(rec, hd):
    """Records u8 [..., record] -> K, V f32 [..., 64, hd]."""
    ko, kh, vo, vh = _offsets(hd, rec.device)
    blk = rec.view(*rec.shape[:-1], 4, _block_bytes(hd))
    out = []
    for off, high, meta in ((ko, kh, 16 * hd), (vo, vh, 16 * hd + 64)):
        n = (blk[..., off.reshape(-1)] >> (4 * high.reshape(-1)).to(torch.uint8)) & 15
        sz = blk[..., meta:meta + 64].contiguous().view(torch.bfloat16).float().view(*blk.shape[:-1], 16, 2)
        n = n.float().view(*blk.shape[:-1], 16, hd)
        out.append(((n - 8) * sz[..., 0:1] + sz[..., 1:2]).flatten(-3, -2))
    return out


# ---------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    nh, nkv, hd, base = HEADS[case["heads"]]
    gen = torch.Generator(device=DEV).manual_seed(seed)
    cached, new = _lengths(case)
    layers = case.get("layers", 1)
    pages = [(c + n + PAGE - 1) // PAGE for c, n in zip(cached, new)]
    n_pages = sum(pages) + 3
    T = sum(new)
    s = SimpleNamespace(case=case, kind=case["kind"], nh=nh, nkv=nkv, hd=hd, base=base, scale=hd ** -0.5, T=T)
    perm = torch.randperm(n_pages, generator=gen, device=DEV)
    table = torch.zeros(len(pages), max(pages), dtype=torch.int32)
    at, perm = 0, perm.cpu()
    for b, n in enumerate(pages):
        table[b, :n] = perm[at:at + n].int()
        at += n
    s.table = table.to(DEV)
    s.pool = torch.zeros(layers, n_pages, nkv, 4 * _block_bytes(hd), dtype=torch.uint8, device=DEV)
    s.cached_host, s.new_host = cached, new
    s.one = len(pages) == 1
    s.cached = torch.tensor(cached, dtype=torch.int32, device=DEV)
    s.start = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
    # what is in the cache: keys with a few strong channels, as they come out of a model, and values of about unit size
    gain = 0.5 + 0.5 * torch.randn(nkv, hd, generator=gen, device=DEV).abs()
    shift = torch.randn(nkv, hd, generator=gen, device=DEV) * 0.7
    for layer in s.pool:
        if case["kind"] == "append":                      # only the new rows are looked at
            break
        slots = torch.arange(n_pages * PAGE, device=DEV)
        k = torch.randn(n_pages * PAGE, nkv, hd, generator=gen, device=DEV) * gain + shift
        v = torch.randn(n_pages * PAGE, nkv, hd, generator=gen, device=DEV)
        _write(layer, slots // PAGE, slots % PAGE, hd, _quantise(k.bfloat16().float()), _quantise(v.bfloat16().float()))
    s.q = (torch.randn(T, nh, hd, generator=gen, device=DEV) * 1.5).bfloat16()
    s.k = (torch.randn(T, nkv, hd, generator=gen, device=DEV) * gain + shift).bfloat16()
    s.v = torch.randn(T, nkv, hd, generator=gen, device=DEV).bfloat16()
    s.amask = None
    if case.get("tree"):
        s.amask = torch.from_numpy(tree_mask(static_tree(case["new"])[0])).to(DEV)
    if case["kind"] == "compact":                         # a path whose rows all lie behind the places they go to
        rng = random.Random(seed)
        path = [0] + sorted(rng.sample(range(case["path"], case["new"]), case["path"] - 1))
        s.path = torch.tensor(path, device=DEV)
        s.accept = torch.tensor([len(path), 5] + path + [0] * (case["new"] - len(path)), dtype=torch.int32, device=DEV)
    if own:
        from flint_b200.kv4 import KvCache4
        s.cache = KvCache4(layers, n_pages, nkv, hd, table=s.table, pool=s.pool, rope_base=base)
    return s


# ---------------------------------------------------------------------------------------------------------------- one pass
def _where(s):
    """Sequence and place among its new tokens of every new token."""
    seq = torch.searchsorted(s.start, torch.arange(s.T, dtype=torch.int32, device=DEV), right=True) - 1
    return seq, torch.arange(s.T, device=DEV) - s.start[seq]


def _rotated(x, pos, base):
    """x [T, heads, hd] rotated in 64 bits (far positions: an angle of 32 bits is off by thousandths)."""
    half = x.shape[-1] // 2
    ang = pos.double()[:, None] * base ** (-torch.arange(half, dtype=torch.float64, device=x.device) / half)
    c, n = ang.cos()[:, None], ang.sin()[:, None]
    a, b = x[..., :half].double(), x[..., half:].double()
    return torch.cat([a * c - b * n, b * c + a * n], -1).float()


def _plain_append(s):
    seq, m = _where(s)
    slot = s.cached[seq] + m
    page = s.table[seq, slot // PAGE].long()
    kq, vq = _quantise(_rotated(s.k, slot, s.base)), _quantise(s.v.float())
    _write(s.pool[0], page, (slot % PAGE).long(), s.hd, kq, vq)
    k, v = _unpack(s.pool[0][page], s.hd)
    at = (slot % PAGE).long()[:, None, None, None].expand(-1, s.nkv, 1, s.hd)
    return _rotated(s.q, slot, s.base).bfloat16(), k.gather(2, at).squeeze(2), v.gather(2, at).squeeze(2)


def _plain_attend(s):
    B, P = s.table.shape
    n = s.case["new"]
    R, hd, nkv = s.nh // s.nkv, s.hd, s.nkv
    k, v = (x.transpose(1, 2).flatten(2, 3) for x in _unpack(s.pool[0][s.table.long()], hd))          # [B, kv heads, slots, hd]
    m = torch.arange(n, device=DEV)
    tok = s.start[:-1, None] + m
    live = tok < s.start[1:, None]                                                                    # [B, n]
    q = s.q[tok.clamp(max=s.T - 1).long()].float().view(B, n, nkv, R, hd).permute(0, 2, 1, 3, 4).reshape(B, nkv, n * R, hd)
    score = (q @ k.transpose(-1, -2)).mul_(s.scale).view(B, nkv, n, R, P * PAGE)
    j = torch.arange(P * PAGE, device=DEV) - s.cached[:, None]                                        # [B, slots]: place among the new ones
    sees = j[:, None, :] <= m[:, None] if s.amask is None else s.amask[m[:, None], j.clamp(0, n - 1)[:, None, :]].bool() & (j < n)[:, None] | (j < 0)[:, None]
    score.masked_fill_(~sees[:, None, :, None, :], -math.inf)
    top = score.amax(-1, keepdim=True).clamp_(min=-1e30)
    p = score.sub_(top).exp_()
    o = (p.view(B, nkv, n * R, -1) @ v).view(B, nkv, n, R, hd) / p.sum(-1, keepdim=True).clamp(min=1e-37)
    return o.permute(0, 2, 1, 3, 4).reshape(B, n, s.nh, hd)[live].bfloat16()


def _plain_compact(s):
    src, dst = s.cached_host[0] + s.path, s.cached_host[0] + torch.arange(len(s.path), device=DEV)
    page, to = s.table[0, src // PAGE].long(), s.table[0, dst // PAGE].long()
    L = s.pool.shape[0]
    k, v = _unpack(s.pool[:, page], s.hd)                                                             # [L, n, kv heads, 64, hd]
    at = (src % PAGE)[None, :, None, None, None]
    rows = [x.gather(3, at.expand(L, -1, s.nkv, 1, s.hd)).squeeze(3) for x in (k, v)]
    # the nibbles move as they are: bytes of K's rows, halves of V's
    ko, _, vo, _ = _offsets(s.hd, DEV)
    meta = torch.arange(4, device=DEV)
    flat, size = s.pool.view(L, -1, s.pool.shape[-1]), _block_bytes(s.hd)
    head = torch.arange(s.nkv, device=DEV)

    def bytes_of(page, slot):
        p, blk = slot % 16, slot % PAGE // 16 * size
        off = torch.cat([ko[p], vo[p], 16 * s.hd + (p * 4)[:, None] + meta, 16 * s.hd + 64 + (p * 4)[:, None] + meta], -1) + blk[:, None]
        return (page[:, None] * s.nkv + head)[..., None], off[:, None]

    (a, b), (c, d) = bytes_of(page, src), bytes_of(to, dst)
    flat[:, c, d] = flat[:, a, b]
    return rows


def run(s):
    if s.kind == "append":
        if not own:
            return _plain_append(s)
        if s.one:
            q = s.cache.append(0, s.k, s.v, s.cached_host[0], q=s.q)
            return q, *s.cache.read(0, s.T, s.cached_host[0])
        q = s.cache.append(0, s.k, s.v, s.cached, q=s.q, start=s.start)
        return q, *s.cache.read(0, s.T, s.cached, start=s.start)
    if s.kind == "attend":
        if not own:
            return _plain_attend(s)
        if s.one:
            return s.cache.attend(0, s.q, s.cached_host[0], amask=s.amask, scale=s.scale)
        return s.cache.attend(0, s.q, s.cached, start=s.start, scale=s.scale, max_new=s.case["new"], max_len=s.case["cached"] + s.case["new"])
    if not own:
        return _plain_compact(s)
    s.cache.compact(s.accept, s.cached_host[0])
    return s.cache.read(None, s.case["path"], s.cached_host[0])


def work(case):
    nh, nkv, hd, _ = HEADS[case["heads"]]
    cached, new = _lengths(case)
    T, row = sum(new), hd + 8                              # a position and kv head: K and V nibbles, two pairs of factors
    if case["kind"] == "append":
        return {"bytes": T * (2 * hd * (2 * nh + 2 * nkv) + 3 * nkv * row + 8 * nkv * hd), "flops": T * (nh + nkv) * hd * 3 + T * nkv * hd * 8}
    if case["kind"] == "compact":
        n = case["layers"] * case["path"] * nkv
        return {"bytes": n * (2 * row + 8 * hd), "flops": 4 * n * hd}
    seen = sum(n * c + n * (n + 1) // 2 for c, n in zip(cached, new))
    if case["tree"]:
        seen = T * cached[0] + int(tree_mask(static_tree(T)[0]).sum())
    return {"bytes": sum(c + n for c, n in zip(cached, new)) * nkv * row + 4 * T * nh * hd, "flops": 4 * seen * nh * hd}


# ---------------------------------------------------------------------------------------------------------------- in 64 bits
def _numbers(rec, hd):
    """What one block's bytes stand for, from its definition: rec u8 [n, block] -> K, V f64 [n, 16, hd]."""
    n = rec.shape[0]
    factor = rec[:, 16 * hd:].contiguous().view(torch.bfloat16).double().view(n, 2, 16, 2)
    k = torch.empty(n, 16, hd, dtype=torch.float64, device=rec.device)
    v = torch.empty_like(k)
    nib = torch.stack([rec[:, :16 * hd] & 15, rec[:, :16 * hd] >> 4], -1).flatten(1).double() - 8     # nibble i of a block: byte i // 2
    main = 128 if hd == 128 else 64
    for p in range(16):
        for d in range(hd):
            slot = d % 8 // 2 + 4 * (d % 2)                # K: even dims of a word of eight in its low half, odd dims in the high one
            word = p * (main // 8) + d // 8 if d < main else main * 2 + p * 2 + (d - main) // 8
            k[:, p, d] = nib[:, word * 8 + slot]
            pair, w = p // 2, d // 4
            if hd == 128:
                word = pair * 32 + (w ^ (8 * (pair % 4)))
            else:
                word = pair * 16 + (w ^ (8 * (pair // 2 % 2))) if d < 64 else 128 + pair * 4 + w - 16
            v[:, p, d] = nib[:, 16 * hd + word * 8 + p % 2 * 4 + d % 4]
    return k * factor[:, 0, :, 0:1] + factor[:, 0, :, 1:2], v * factor[:, 1, :, 0:1] + factor[:, 1, :, 1:2]


def _row_values(x):
    """The definition of a stored row, in 64 bits (s and z are bf16 numbers)."""
    low, high = x.min(-1, True).values, x.max(-1, True).values
    s = ((high - low) / 15).to(torch.bfloat16).double()
    z = (low + 8 * s).to(torch.bfloat16).double()
    n = torch.round((x - z) / torch.where(s == 0, torch.ones_like(s), s)).clamp(-8, 7)
    return torch.where(s == 0, torch.zeros_like(n), n) * s + z


def _turned(x, where, base):
    hd = x.shape[-1]
    freq = torch.tensor([base ** (-2.0 * i / hd) for i in range(hd // 2)], dtype=torch.float64, device=x.device)
    w = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), where.double()[:, None] * freq)[:, None]
    y = torch.complex(x[..., :hd // 2].double(), x[..., hd // 2:].double()) * w
    return torch.cat([y.real, y.imag], -1)


def exact(case, seed):
    s = prepare(case, seed)
    hd, nkv, R = s.hd, s.nkv, s.nh // s.nkv
    if s.kind == "append":
        where = torch.cat([torch.arange(c, c + n, device=DEV) for c, n in zip(s.cached_host, s.new_host)])
        return _turned(s.q, where, s.base), _row_values(_turned(s.k, where, s.base).float().double()), _row_values(s.v.double())
    size = _block_bytes(hd)
    if s.kind == "compact":
        rows = []
        for node in s.path.tolist():
            slot = s.cached_host[0] + node
            blk = s.pool[:, int(s.table[0, slot // PAGE]), :, slot % PAGE // 16 * size:][..., :size].reshape(-1, size)
            rows.append([x[:, slot % 16].view(-1, nkv, hd) for x in _numbers(blk, hd)])
        return [torch.stack([r[i] for r in rows], 1) for i in (0, 1)]
    out = torch.empty(s.T, s.nh, hd, dtype=torch.float64, device=DEV)
    first = 0
    for b, (c, n) in enumerate(zip(s.cached_host, s.new_host)):
        pages = s.pool[0][s.table[b, :(c + n + PAGE - 1) // PAGE].long()]
        for h in range(nkv):
            k, v = (x.reshape(-1, hd)[:c + n] for x in _numbers(pages[:, h].reshape(-1, size), hd))
            for r in range(R):
                q = s.q[first:first + n, h * R + r].double()
                a = q @ k.T * s.scale
                seen = torch.ones(n, n, device=DEV).tril() if s.amask is None else s.amask
                a[:, c:] = torch.where(seen.bool(), a[:, c:], torch.full((), -math.inf, dtype=torch.float64, device=DEV))
                out[first:first + n, h * R + r] = a.softmax(-1) @ v
        first += n
    return out
