"""GPU: the paged 4-bit K/V cache (append, attention, read-back, moves) against its definition in 64 bits."""
import ctypes
import math

import pytest
import torch

from flint_b200 import _lib
from flint_b200.kv4 import NO_SCRATCH, KvCache4, page_bytes
from tests import kv4_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def make(lens, nkv, hd, layers=1, base=1e4, spare=2, seed=0, garbage=False):
    """A cache whose sequences may hold lens[b] positions, its pages in random order; `garbage`: unwritten rows hold NaN factors."""
    g = torch.Generator().manual_seed(seed)
    need = [max(1, (n + 63) // 64) for n in lens]
    perm = torch.randperm(sum(need) + spare, generator=g).int()
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    c = KvCache4(layers, sum(need) + spare, nkv, hd, table.to(DEV), rope_base=base)
    if garbage:
        c.pool.fill_(0xFF)                                  # factors 0xFFFF: NaN
    return c


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def rows(seed, T, heads, hd, scale=1.0):
    return (torch.randn(T, heads, hd, generator=gen(seed), device=DEV) * scale).bfloat16()


def within(a, b, tol):
    return bool(((a.double() - b.double()).abs() <= tol).all())


# ---------------------------------------------------------------------------------------------------------------- append, read
@pytest.mark.parametrize("hd", [64, 80, 128])
@pytest.mark.parametrize("nkv,nh,cached,T,base", [(1, 1, 0, 1, 1e4), (2, 8, 13, 70, 1e4), (8, 40, 32700, 3, 1e7), (8, 32, 64, 129, 5e5), (3, 6, 100000, 5, None)])
def test_appended_rows_are_the_definition_bit_for_bit(hd, nkv, nh, cached, T, base):
    c = make([cached + T], nkv, hd, base=base)
    q, k, v = rows(1, T, nh, hd, 2.0), rows(2, T, nkv, hd, 3.0), rows(3, T, nkv, hd)
    before = c.pool.clone()
    got = c.append(0, k, v, cached, q=q)
    K, V = c.read(0, T, cached)
    c.check()
    pos = torch.arange(cached, cached + T, device=DEV)
    turn = (lambda x: ref.rotated(x, pos, base)) if base else (lambda x: x.double())
    assert torch.equal(V, ref.values(v.float()))
    # A rotated key comes out of double precision and is rounded to single before its row is quantised: the kernel's and this file's doubles differ by about
    # 1e-11 (far positions) and single-precision values by one step in a few of 10^4 elements, which moves a nibble only within 1e-6 of a border.
    want = ref.values(turn(k).float())
    assert (K != want).float().mean() <= 1e-4
    # bf16 rounding (half a step: 2^-8 of the value), and products of single precision
    wq = turn(q)
    assert within(got, wq, wq.abs() * 2.0 ** -8 + 2.0 ** -21 * q.double().abs().amax())
    # nothing but the tokens' pages was written
    pages = c.table[0, cached // 64:(cached + T - 1) // 64 + 1].long()
    others = torch.ones(c.n_pages, dtype=torch.bool, device=DEV)
    others[pages] = False
    assert torch.equal(c.pool[:, others], before[:, others])


@pytest.mark.parametrize("hd", [64, 80, 128])
def test_bytes_of_a_block_are_as_documented(hd):
    c = make([64], 2, hd, base=None)
    k, v = rows(4, 64, 2, hd), rows(5, 64, 2, hd)
    c.append(0, k, v, 0)
    c.check()
    rec = c.pool[0, int(c.table[0, 0])].cpu()
    size = 16 * hd + 128
    for head in range(2):
        (kn, ks, kz), (vn, vs, vz) = ref.quantised(k[:, head].float()), ref.quantised(v[:, head].float())
        for blk in (0, 3):
            at = slice(16 * blk, 16 * blk + 16)
            want = ref.block_of(kn[at].cpu(), ks[at], kz[at], vn[at].cpu(), vs[at], vz[at])
            assert torch.equal(rec[head, blk * size:(blk + 1) * size], want)


def test_a_position_is_written_without_touching_its_neighbours():
    """Two positions share words of V: appending one leaves the other's bytes as they were."""
    c = make([64], 2, 80, base=None, garbage=True)
    k, v = rows(6, 64, 2, 80), rows(7, 64, 2, 80)
    for m in torch.randperm(64, generator=torch.Generator().manual_seed(1)).tolist():
        c.append(0, k[m:m + 1], v[m:m + 1], m)
    K, V = c.read(0, 64, 0)
    c.check()
    assert torch.equal(K, ref.values(k.float())) and torch.equal(V, ref.values(v.float()))


def test_rows_that_are_flat_huge_tiny_or_not_numbers():
    hd = 64
    x = torch.randn(9, 1, hd, generator=gen(8), device=DEV)
    x[0] = 1.37                                             # flat: s = 0
    x[1] = 0.0
    x[2, 0, 5] = math.inf
    x[3, 0, 60] = math.nan
    x[4, 0, :2] = torch.tensor([3e38, -3e38])               # range overflows single precision
    x[5] *= 1e-39                                           # subnormal numbers
    x[6] *= 1e30
    x[7, 0, 0] = 1e4                                        # an outlier
    x[8, 0, 7] = -math.inf
    x = x.bfloat16()
    c = make([64], 1, hd, base=None)
    c.append(0, x, x, 3)
    K, V = c.read(0, 9, 3)
    c.check()
    want = ref.values(x.float())
    assert want[[2, 3, 4, 8]].isnan().all() and want[[0, 1, 5, 6, 7]].isfinite().all()
    for got in (K, V):
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))
    assert torch.equal(want[0], x[0].float())


def test_ragged_sequences_depths_strides_and_tokens_behind_the_last_sequence():
    nkv, nh, hd = 2, 6, 80
    lens, new = [5, 0, 100, 63, 7], [3, 0, 1, 70, 0]        # two sequences without new tokens
    T = sum(new) + 4                                        # four tokens are nobody's
    c = make([a + b for a, b in zip(lens, new)], nkv, hd, garbage=True)
    fused = torch.randn(T, (nh + 2 * nkv) * hd + 8, generator=gen(9), device=DEV).bfloat16()
    q, k, v = (fused[:, a * hd:b * hd].unflatten(1, (b - a, hd)) for a, b in ((0, nh), (nh, nh + nkv), (nh + nkv, nh + 2 * nkv)))
    start, cached = ints(0, 3, 3, 4, 74, 74), ints(*lens)
    depth = torch.randint(0, 5, (T,), generator=gen(10), device=DEV, dtype=torch.int32)
    q_out = torch.full((T, nh, hd), 7.0, dtype=torch.bfloat16, device=DEV)
    c.append(0, k, v, cached, q=q, start=start, depth=depth, q_out=q_out)
    K, V = c.read(0, T, cached, start=start)
    c.check()
    pos = torch.repeat_interleave(cached, ints(*new)).long() + depth[:-4]
    assert torch.equal(V[:-4], ref.values(v[:-4].float()))
    assert (K[:-4] != ref.values(ref.rotated(k[:-4], pos, 1e4).float())).float().mean() <= 1e-4
    want = ref.rotated(q[:-4], pos, 1e4)
    assert within(q_out[:-4], want, want.abs() * 2.0 ** -8 + 1e-5)
    assert (q_out[-4:] == 7.0).all()                        # behind the last sequence: as they were
    # the same through contiguous tensors, into the same rows
    again = make([a + b for a, b in zip(lens, new)], nkv, hd, garbage=True)
    got = again.append(0, k.contiguous(), v.contiguous(), cached, q=q.contiguous(), start=start, depth=depth)
    assert torch.equal(again.pool, c.pool) and torch.equal(got[:-4], q_out[:-4])
    # q rotated in place
    qc = q.contiguous()
    assert again.append(0, k, v, cached, q=qc, start=start, depth=depth, q_out=qc) is qc and torch.equal(qc[:-4], q_out[:-4])


# ---------------------------------------------------------------------------------------------------------------- attention
def check_attention(out, q, K, V, cached, scale, amask=None, many=False, wide=False):
    """K, V: what the cache stands for. The kernels' own roundings (each at most half a step): the output to bf16 (2^-8 of the value); sums in 32 bits. Up to 64 query rows
    a kv head: probabilities to fp16 (2^-11 of each, 2^-25 of the largest one for those below 2^-14 of it), keys and values as they are. More rows:
    keys to fp16 (2^-11 of each, 2^-25 of the largest of 128), probabilities and values to fp16 too (2^-11), or bf16 (2^-8) where rows of a page lie outside
    fp16's range (`wide`): h. Keys off by 2^-11 move a score by `d` at most (below), and a probability by the factor e^(2d).
    So |error| <= 2^-8 |o| + (2 h + 2 d + L 2^-25) max |v|."""
    want = ref.attention(q, K, V, cached, scale, amask)
    of_many = q.shape[0] * (q.shape[1] // K.shape[1]) > 64 or many
    L, h = K.shape[0], 2.0 ** -8 if of_many and wide else 2.0 ** -11
    fin = torch.where(K.isfinite(), K, torch.zeros_like(K)).double()
    # sum of |q k| h over hd independent roundings: the root of their squares, times six, is never reached
    d = 6 * 2.0 ** -11 * abs(scale) * float((q.double() ** 2).amax()) ** 0.5 * float((fin ** 2).sum(-1).amax()) ** 0.5
    vmax = float(torch.where(V.isfinite(), V, torch.zeros_like(V)).abs().amax())
    tol = want.abs() * 2.0 ** -8 + (2 * h + 2 * d + L * 2.0 ** -25) * vmax
    assert torch.equal(out.isnan(), want.isnan())
    fine = ~want.isnan()
    err = (out.double() - want).abs()[fine]
    worst, whole = float((err / tol[fine].clamp(min=1e-38)).max()), float(err.norm() / tol[fine].norm().clamp(min=1e-38))
    assert worst <= 1.0, worst
    # on the whole: a rounding is uniform, its root of mean squares 1 / sqrt(3) of half a step
    assert whole <= 0.6, whole


def filled(lens, new, nh, nkv, hd, seed=0, layers=1, qscale=1.5):
    """A cache with `lens` positions and the new tokens appended; what all rows stand for, per sequence, and the queries."""
    total = [a + b for a, b in zip(lens, new)]
    c = make(total, nkv, hd, base=None, garbage=True, seed=seed, layers=layers)
    starts = ints(0, *torch.tensor(total).cumsum(0).tolist())
    n = sum(total)
    c.append(0, rows(seed + 1, n, nkv, hd, 1.3), rows(seed + 2, n, nkv, hd), ints(*[0] * len(lens)), start=starts)
    K, V = c.read(0, n, ints(*[0] * len(lens)), start=starts)
    cut = lambda x: [x[int(starts[b]):int(starts[b + 1])] for b in range(len(lens))]  # noqa: E731
    return c, cut(K), cut(V), rows(seed + 3, sum(new), nh, hd, qscale), ints(0, *torch.tensor(new).cumsum(0).tolist())


@pytest.mark.parametrize("hd,nh,nkv", [(64, 40, 8), (80, 32, 8), (128, 32, 8), (64, 8, 2), (128, 3, 3), (80, 16, 1), (64, 9, 1), (128, 34, 2)])
@pytest.mark.parametrize("cached,new", [(0, 1), (1, 1), (30, 2), (63, 1), (64, 3), (200, 1), (1000, 4), (5000, 1)])
def test_attention_of_few_tokens(hd, nh, nkv, cached, new):
    c, K, V, q, _ = filled([cached], [new], nh, nkv, hd, seed=cached + hd)
    out = c.attend(0, q, cached)
    c.check()
    check_attention(out, q, K[0], V[0], cached, hd ** -0.5)


@pytest.mark.parametrize("hd,nh,nkv", [(64, 40, 8), (80, 32, 8), (128, 32, 8), (128, 6, 6), (64, 2, 1)])
@pytest.mark.parametrize("cached,new", [(0, 5), (0, 130), (700, 17), (64, 64), (129, 300), (1000, 61)])
def test_attention_of_prompts(hd, nh, nkv, cached, new):
    c, K, V, q, _ = filled([cached], [new], nh, nkv, hd, seed=cached + hd)
    out = c.attend(0, q, cached)
    c.check()
    check_attention(out, q, K[0], V[0], cached, hd ** -0.5)


@pytest.mark.parametrize("hd,nh,nkv", [(64, 40, 8), (80, 32, 8), (128, 32, 8), (64, 8, 2)])
@pytest.mark.parametrize("cached,new", [(0, 2), (37, 9), (1024, 26), (300, 64)])
def test_attention_under_a_mask(hd, nh, nkv, cached, new):
    """Random masks: rows that see none of the new tokens among them (with nothing cached: zeros), tokens that nobody sees holding NaN."""
    c, K, V, q, _ = filled([cached], [new], nh, nkv, hd, seed=cached + hd)
    amask = (torch.rand(new, new, generator=gen(cached), device=DEV) < 0.4).to(torch.uint8)
    amask[0] = 0
    amask[:, new // 2] = 0
    bad = torch.full((1, nkv, hd), math.nan, dtype=torch.bfloat16, device=DEV)
    c.append(0, bad, bad, cached + new // 2)
    K[0][cached + new // 2], V[0][cached + new // 2] = math.nan, math.nan
    out = c.attend(0, q, cached, amask=amask)
    c.check()
    assert out.isfinite().all()
    if cached == 0:
        assert (out[0] == 0).all()
    check_attention(out, q, K[0], V[0], cached, hd ** -0.5, amask)
    assert torch.equal(out, c.attend(0, q, cached, amask=amask.bool()))          # and a second time the same bits


@pytest.mark.parametrize("new", [1, 5, 40])
def test_numbers_that_are_none_reach_the_rows_that_see_them_alone(new):
    """A NaN row among the new tokens: later tokens are NaN, earlier ones are not."""
    hd, nh, nkv, cached = 80, 8, 2, 100
    for which in ("k", "v"):
        c, K, V, q, _ = filled([cached], [new], nh, nkv, hd, seed=3)
        at = cached + new // 2
        k, v = rows(20, 1, nkv, hd), rows(21, 1, nkv, hd)
        (k if which == "k" else v)[0, 1, 3] = math.inf
        c.append(0, k, v, at)
        K[0][at], V[0][at] = (x[0] for x in c.read(0, 1, at))
        out = c.attend(0, q, cached)
        c.check()
        check_attention(out, q, K[0], V[0], cached, hd ** -0.5)
        assert out[:new // 2].isfinite().all() and out[new // 2:, 4:].isnan().all() and out[:, :4].isfinite().all()


@pytest.mark.parametrize("hd,nh,nkv", [(64, 40, 8), (80, 32, 8), (128, 8, 2)])
@pytest.mark.parametrize("lens,new", [([5, 300, 0, 64, 1, 2000], [1, 1, 1, 1, 1, 1]), ([0, 65, 700], [30, 0, 5]), ([10, 0, 130], [200, 64, 1])])
def test_attention_of_a_ragged_batch(hd, nh, nkv, lens, new):
    c, K, V, q, start = filled(lens, new, nh, nkv, hd, seed=hd)
    cached = ints(*lens)
    out = torch.full((sum(new) + 2, nh, hd), 5.0, dtype=torch.bfloat16, device=DEV)
    qq = torch.cat([q, q[:2] if len(q) > 1 else torch.cat([q, q])])              # two tokens that no sequence has
    for hints in ({}, dict(max_new=max(new), max_len=3), dict(max_new=max(new), max_len=10 ** 6)):
        out.fill_(5.0)
        assert c.attend(0, qq, cached, start=start, out=out, **hints) is out
        c.check()
        assert (out[sum(new):] == 5.0).all()
        for b in range(len(lens)):
            a, z = int(start[b]), int(start[b + 1])
            if z > a:
                check_attention(out[a:z], q[a:z], K[b], V[b], lens[b], hd ** -0.5, many=max(new) * nh // nkv > 64 or not hints)


@pytest.mark.parametrize("hd,nh,nkv", [(64, 40, 8), (80, 32, 8), (128, 32, 8)])
def test_attention_of_a_long_cache_follows_its_largest_scores(hd, nh, nkv):
    """33000 positions, sharp scores, a few positions that take almost everything."""
    cached = 33000
    c, K, V, q, _ = filled([cached], [1], nh, nkv, hd, seed=5, qscale=4.0)
    out = c.attend(0, q, cached)
    c.check()
    check_attention(out, q, K[0], V[0], cached, hd ** -0.5)


def test_values_whose_scales_span_many_powers_of_two():
    """Rows of V from 2^-40 to 2^40 and keys of small scale: the rows' factors do not fit fp16."""
    hd, nkv, nh, n = 64, 1, 4, 600
    for flip in (False, True):
        size = torch.logspace(-40, 40, n, base=2.0, device=DEV)[:, None, None]
        v = torch.randn(n, nkv, hd, generator=gen(30), device=DEV) * (size.flip(0) if flip else size)
        k = torch.randn(n, nkv, hd, generator=gen(31), device=DEV) * 1e-4
        q = rows(32, 1, nh, hd, 1e4)
        c = make([n], nkv, hd, base=None, garbage=True)
        c.append(0, k.bfloat16(), v.bfloat16(), 0)
        K, V = c.read(0, n, 0)
        out = c.attend(0, q, n - 1)
        c.check()
        check_attention(out, q, K, V, n - 1, hd ** -0.5)
        assert out.isfinite().all()


@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("kp,vp", [(0, -30), (0, -12), (0, 16), (0, 60), (40, 0), (-40, 0), (60, 90)])
def test_keys_and_values_of_any_size(new, kp, vp):
    """Keys 2^kp and values 2^vp times the usual, queries 2^-kp times: the same probabilities, values within fp16's range and outside it."""
    hd, nkv, nh, cached = 128, 2, 8, 300
    n = cached + new
    c = make([n], nkv, hd, base=None, garbage=True)
    c.append(0, rows(51, n, nkv, hd, 2.0 ** kp), rows(52, n, nkv, hd, 2.0 ** vp), 0)
    K, V = c.read(0, n, 0)
    q = rows(53, new, nh, hd, 1.5 * 2.0 ** -kp)
    out = c.attend(0, q, cached)
    c.check()
    check_attention(out, q, K, V, cached, hd ** -0.5, wide=vp != 0)


def test_one_page_of_a_step_outside_the_range_of_the_other():
    """Pages of 64 positions whose values are 1, 2^-25, 2^17 and 0 times the usual, ends of the cache at every one of them."""
    hd, nkv, nh, new = 64, 1, 2, 64
    size = torch.tensor([1, 2.0 ** -25, 2.0 ** 17, 0, 2.0 ** -25, 1, 0, 2.0 ** 17, 1, 0], device=DEV).repeat_interleave(64)
    n = size.numel()
    for page in range(n // 64 - 1):
        c = make([n], nkv, hd, base=None, garbage=True)
        q, k, v = rows(61, new, nh, hd), rows(62, n, nkv, hd), (rows(63, n, nkv, hd).float() * size[:, None, None]).bfloat16()
        c.append(0, k, v, 0)
        out = c.attend(0, q, page * 64 + 64)      # the next page's tokens are the queries: the chain mask
        c.check()
        K, V = (x[:page * 64 + 128] for x in c.read(0, n, 0))
        check_attention(out, q, K, V, page * 64 + 64, hd ** -0.5, wide=True)


@pytest.mark.parametrize("hd", [64, 80, 128])
def test_a_none_of_a_later_step_stays_there(hd):
    """Steps of 128 positions follow one another while the softmax of earlier ones runs: a value that is none in the third is not held against the first."""
    nh, nkv, cached, new = 16, 4, 256, 64
    c, K, V, q, _ = filled([cached], [new], nh, nkv, hd, seed=5)
    bad = torch.full((1, nkv, hd), math.nan, dtype=torch.bfloat16, device=DEV)
    c.append(0, rows(21, 1, nkv, hd), bad, cached + 40)
    outs = [c.attend(0, q, cached) for _ in range(40)]
    c.check()
    for out in outs:
        assert out[:40].isfinite().all() and out[40:].isnan().all()
        assert torch.equal(out[:40], outs[0][:40])


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("at", [0, 40, 199])
def test_large_values_of_small_weight_leave_the_others_as_they_are(new, at):
    """A row of V 2^30 times the others whose probability is about 2^-80, ahead of them, among them and behind them."""
    hd, nkv, nh, cached = 64, 1, 4, 200
    n = cached + new
    k, v = rows(33, n, nkv, hd, 0.01).float(), rows(34, n, nkv, hd).float()
    q = torch.ones(new, nh, hd, dtype=torch.bfloat16, device=DEV)
    k[at] -= 55.0 / hd                                      # score -55 at scale 1
    v[at] *= 2.0 ** 30
    c = make([n], nkv, hd, base=None, garbage=True)
    c.append(0, k.bfloat16(), v.bfloat16(), 0)
    K, V = c.read(0, n, 0)
    out = c.attend(0, q, cached, scale=1.0)
    c.check()
    # what the row adds is below 2^-40: the tolerance is that of the other rows
    V2 = V.clone()
    V2[at] = 0
    check_attention(out, q, K, V2, cached, 1.0, wide=True)


def test_many_rows_in_pieces_of_every_size():
    """One to nine steps of positions, one or two tiles of rows, the last of each full or not."""
    hd, nkv = 128, 2
    for nh, new in ((8, 17), (8, 32), (8, 33), (8, 64), (8, 65), (2, 129), (10, 100)):
        for cached in (0, 100, 900):
            c, K, V, q, _ = filled([cached], [new], nh, nkv, hd, seed=new)
            out = c.attend(0, q, cached)
            c.check()
            check_attention(out, q, K[0], V[0], cached, hd ** -0.5)


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("scale", [0.0, -0.1, 1.0])
def test_scales_of_any_sign(new, scale):
    hd, nh, nkv, cached = 64, 8, 2, 150
    c, K, V, q, _ = filled([cached], [new], nh, nkv, hd, seed=6, qscale=0.5)
    out = c.attend(0, q, cached, scale=scale)
    c.check()
    check_attention(out, q, K[0], V[0], cached, scale)


def test_strided_queries_and_outputs():
    hd, nh, nkv, cached, new = 80, 8, 2, 90, 6
    c, K, V, q, _ = filled([cached], [new], nh, nkv, hd, seed=7)
    want = c.attend(0, q, cached)
    wide = torch.zeros(new, nh * hd + 16, dtype=torch.bfloat16, device=DEV)
    wide[:, 8:8 + nh * hd] = q.flatten(1)
    out = torch.full((new, nh * hd + 8), 3.0, dtype=torch.bfloat16, device=DEV)
    c.attend(0, wide[:, 8:8 + nh * hd].unflatten(1, (nh, hd)), cached, out=out[:, :nh * hd].unflatten(1, (nh, hd)))
    assert torch.equal(out[:, :nh * hd], want.flatten(1)) and (out[:, nh * hd:] == 3.0).all()
    odd = torch.zeros(new * nh * hd + 1, dtype=torch.bfloat16, device=DEV)       # not 16-byte aligned, and heads apart: copied
    odd[1:] = q.flatten()
    assert torch.equal(c.attend(0, odd[1:].view(new, nh, hd), cached), want)
    assert torch.equal(c.attend(0, q.transpose(0, 1).contiguous().transpose(0, 1), cached), want)


# ---------------------------------------------------------------------------------------------------------------- moves
@pytest.mark.parametrize("hd,nkv,layers", [(64, 8, 3), (80, 2, 4), (128, 8, 2)])
def test_compaction_and_moves_follow_the_order_of_the_list(hd, nkv, layers):
    n, pos = 300, 130
    c = make([n, n], nkv, hd, layers=layers, base=None)
    c.pool.random_(0, 120, generator=gen(1))                # any bytes with finite factors
    one = KvCache4(layers, c.n_pages, nkv, hd, c.table[1:2], pool=c.pool)
    K, V = (x.clone() for x in one.read(None, n, 0))
    K0, V0 = KvCache4(layers, c.n_pages, nkv, hd, c.table[0:1], pool=c.pool).read(None, n, 0)
    path = [0, 1, 4, 5, 9, 63]
    c.compact(ints(len(path), 17, *path, *[0] * 58), pos, seq=1)
    for i, node in enumerate(path):
        K[:, pos + i], V[:, pos + i] = K[:, pos + node].clone(), V[:, pos + node].clone()
    src, dst = [5, 6, 7, 7, 200] + list(range(100)), [6, 7, 8, 7, 5] + list(range(150, 250))     # a chain, a row on itself, more than one launch
    c.move(src, dst, seq=1)
    for a, b in zip(src, dst):
        K[:, b], V[:, b] = K[:, a].clone(), V[:, a].clone()
    got = one.read(None, n, 0)
    c.check()
    assert torch.equal(got[0], K) and torch.equal(got[1], V)
    first = KvCache4(layers, c.n_pages, nkv, hd, c.table[0:1], pool=c.pool).read(None, n, 0)
    assert torch.equal(first[0], K0) and torch.equal(first[1], V0)               # the other sequence is as it was


# ---------------------------------------------------------------------------------------------------------------- how they are called
def test_a_step_of_decoding_from_a_captured_graph():
    """Append and attention of one token, captured once; the lengths live on the GPU and grow. A second graph over another cache runs on another stream meanwhile."""
    hd, nh, nkv, n = 128, 8, 2, 130
    caches = [make([n + 1, n + 1], nkv, hd, base=5e5, garbage=True, seed=s) for s in (1, 2)]
    qkv = [[rows(40 + i + 7 * s, 2 * n, h, hd) for i, h in enumerate((nh, nkv, nkv))] for s in (0, 1)]
    start, graphs, state = ints(0, 1, 2), [], []
    for s, c in enumerate(caches):
        buf = [torch.zeros(2, h, hd, dtype=torch.bfloat16, device=DEV) for h in (nh, nkv, nkv)]
        cached, out = ints(0, 3), torch.zeros(2, nh, hd, dtype=torch.bfloat16, device=DEV)
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            c.attend(0, c.append(0, buf[1], buf[2], cached, q=buf[0], start=start), cached, start=start, out=out)
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                qr = c.append(0, buf[1], buf[2], cached, q=buf[0], start=start)
                c.attend(0, qr, cached, start=start, max_new=1, out=out)
                cached += 1
        graphs.append((graph, side))
        state.append((buf, cached, out))
        cached.copy_(ints(0, 3))
        c.append(0, *(x[-6:] for x in qkv[s][1:]), ints(0, 0), start=ints(0, 0, 6))      # what the second sequence has: three (and three behind them)
    got = [[], []]
    torch.cuda.synchronize()
    for i in range(n - 4):
        for s in (0, 1):
            graph, side = graphs[s]
            with torch.cuda.stream(side):
                for b, x in zip(state[s][0], qkv[s]):
                    b.copy_(x[2 * i:2 * i + 2])
                graph.replay()
                got[s].append(state[s][2].clone())
    torch.cuda.synchronize()
    for s, c in enumerate(caches):
        c.check()
        for b in (0, 1):
            held = n - 4 + 3 * b
            K, V = KvCache4(1, c.n_pages, nkv, hd, c.table[b:b + 1], pool=c.pool).read(0, held, 0)
            for i in (0, 1, 60, 61, n - 5):
                pos = torch.tensor([i + 3 * b], device=DEV)
                q = ref.rotated(qkv[s][0][2 * i + b:2 * i + b + 1], pos, 5e5).bfloat16()
                check_attention(got[s][i][b:b + 1], q, K[:i + 1 + 3 * b], V[:i + 1 + 3 * b], i + 3 * b, hd ** -0.5)


def test_sequences_that_share_their_first_pages():
    """A common prompt: three sequences whose tables name the same pages at first, and their own behind them."""
    hd, nkv, nh, common = 80, 2, 8, 192
    own = [5, 70, 130]
    table = torch.full((3, 6), -1, dtype=torch.int32)
    table[:, :3] = torch.tensor([4, 0, 9])
    at = iter([1, 2, 3, 5, 6, 7, 8])
    for b, n in enumerate(own):
        for i in range((n + 63) // 64):
            table[b, 3 + i] = next(at)
    c = KvCache4(1, 10, nkv, hd, table.to(DEV), rope_base=None)
    k, v = rows(1, common, nkv, hd), rows(2, common, nkv, hd)
    c.append(0, k, v, ints(0, 0, 0), start=ints(0, common, common, common))         # once, by the first
    starts = ints(0, *torch.tensor(own).cumsum(0).tolist())
    c.append(0, rows(3, sum(own), nkv, hd), rows(4, sum(own), nkv, hd), ints(*[common] * 3), start=starts)
    for new in (1, 5):
        q = rows(5, 3 * new, nh, hd)
        cached = [common + n - new for n in own]
        out = c.attend(0, q, ints(*cached), start=ints(0, new, 2 * new, 3 * new), max_new=new)
        for b in range(3):
            one = KvCache4(1, 10, nkv, hd, c.table[b:b + 1].contiguous(), pool=c.pool, rope_base=None)
            K, V = one.read(0, cached[b] + new, 0)
            check_attention(out[b * new:(b + 1) * new], q[b * new:(b + 1) * new], K, V, cached[b], hd ** -0.5)
    c.check()


@pytest.mark.parametrize("new,cached", [(1, 9000), (40, 3000), (300, 600)])
def test_calls_on_two_streams_at_once_have_their_own_scratch(new, cached):
    hd, nkv, nh = 128, 2, 8
    c, K, V, q, _ = filled([cached], [new], nh, nkv, hd, seed=9)
    q2 = rows(77, new, nh, hd)
    want = c.attend(0, q, cached), c.attend(0, q2, cached)
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    outs = [], []
    for _ in range(20):
        for i, x in enumerate((q, q2)):
            with torch.cuda.stream(streams[i]):
                outs[i].append(c.attend(0, x, cached))
    torch.cuda.synchronize()
    c.check()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])


def test_a_captured_prompt_over_lengths_on_the_gpu():
    """Two graphs, captured one after the other and replayed in turn while the lengths that they read change."""
    hd, nkv, nh, new = 64, 2, 8, 40
    c, K, V, q, _ = filled([900], [new], nh, nkv, hd, seed=12)
    cached = ints(900)
    c.attend(0, q, cached)                                       # (first use sets the kernels up)
    torch.cuda.synchronize()
    q2 = rows(78, new, nh, hd)
    graphs, outs = [], []
    for x in (q, q2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c.attend(0, x, cached))
        graphs.append(g)
    for n in (900, 0, 63, 500, 64):
        cached.fill_(n)
        for g in graphs:
            g.replay()
        for x, out in zip((q, q2), outs):
            check_attention(out, x, K[0][:n + new], V[0][:n + new], n, hd ** -0.5)
    c.check()


def test_nothing_to_do():
    c = make([64], 2, 64)
    empty = torch.empty(0, 2, 64, dtype=torch.bfloat16, device=DEV)
    q = torch.empty(0, 4, 64, dtype=torch.bfloat16, device=DEV)
    before = c.pool.clone()
    assert c.append(0, empty, empty, 5, q=q).shape == q.shape and c.attend(0, q, 5).shape == q.shape
    assert c.read(0, 0, 5)[0].shape == (0, 2, 64)
    c.compact(ints(0, 0), 5)
    c.compact(ints(1, 9, 0, 0), 5)
    c.move([], [])
    c.check()
    assert torch.equal(c.pool, before)


def test_pages_lengths_and_paths_that_cannot_be_are_reported_and_left_out():
    hd, nh, nkv = 64, 4, 2
    c, K, V, q, start = filled([100, 70], [1, 1], nh, nkv, hd, seed=9)
    cached = ints(100, 70)
    good = c.attend(0, q, cached, start=start)
    c.check()
    table, pool = c.table.clone(), c.pool.clone()

    def reported(where, seq=None):
        st = c.status()
        assert st["code"] == _lib.FB_ERR_RANGE and st["where"] == where and (seq is None or st["sequence"] == seq), st
        assert c.status()["code"] == 0
        with pytest.raises(_lib.FlintError):
            c._status[0] = 6
            c.check()

    for bad in (-1, c.n_pages, 2 ** 31 - 1):
        c.table[1, 1] = bad                                 # positions 64 .. of the second sequence
        out = c.attend(0, q, cached, start=start)
        reported(21, 1)
        assert torch.equal(out[0], good[0])
        check_attention(out[1:], q[1:], K[1][:64], V[1][:64], 63, hd ** -0.5)    # as if they were not there
        c.append(0, rows(1, 2, nkv, hd), rows(2, 2, nkv, hd), ints(100, 70), start=start)
        reported(21, 1)
        c.pool.copy_(pool)
        c.table.copy_(table)
    for lengths, begin in ((ints(100, 127), ints(0, 1, 3)), (ints(100, -1), start), (ints(100, 2 ** 31 - 1), start)):
        k = rows(1, 3, nkv, hd)
        qq = torch.cat([q, q[:1]])
        out = torch.full_like(qq, 9.0)
        c.attend(0, qq, lengths, start=begin, out=out)
        reported(22, 1)
        assert torch.equal(out[0], good[0]) and (out[1:] == 9.0).all()
        before = c.pool.clone()
        c.append(0, k, k, lengths, start=begin)
        reported(22, 1)
        assert torch.equal(c.pool[:, c.table[1].long()], before[:, c.table[1].long()])
        c.pool.copy_(pool)
    for begin in (ints(0, 1, 7), ints(0, -3, 2), ints(0, 2, 1), ints(5, 6, 7)):
        c.attend(0, q, cached, start=begin)
        c.append(0, rows(1, 2, nkv, hd), rows(2, 2, nkv, hd), cached, start=begin)
        reported(23)
        c.pool.copy_(pool)
    for accept in (ints(5, 0, 0, 1, 2), ints(-1, 0, 0), ints(2, 0, 0, 10 ** 6), ints(2, 0, 0, -50)):
        c.compact(accept, 40)
        reported(24)
        assert torch.equal(c.pool, pool)


def test_one_short_sequence_needs_no_scratch():
    lib, c = _lib.load(), make([64], 2, 64)
    for nkv in (1, 2, 8, 20, 74, 140):
        for tokens in (1, 2, 3, 16, 64, 200, 5000):
            s = c._seqs(0, 0, 0, None)
            s.n_kv_head, s.n_tokens = nkv, tokens
            for r in (1, 4, 5, 16):
                if tokens * r <= NO_SCRATCH[1]:
                    assert lib.fb_kv4_attend_bytes(ctypes.byref(s), nkv * r, tokens, NO_SCRATCH[0]) == 0


def test_refused_calls():
    c = make([64, 64], 2, 64)
    k, q, cached, start = rows(1, 2, 2, 64), rows(2, 2, 4, 64), ints(3, 3), ints(0, 1, 2)
    ok = dict(start=start)
    c.append(0, k, k, cached, **ok)
    bad = [
        lambda: c.append(1, k, k, cached, **ok), lambda: c.append(-1, k, k, cached, **ok),
        lambda: c.append(0, k, k, cached), lambda: c.append(0, k, k, cached, start=start[:2]), lambda: c.append(0, k, k, cached, start=start.long()),
        lambda: c.append(0, k, k, cached.cpu(), **ok), lambda: c.append(0, k, k, cached[:1], **ok), lambda: c.append(0, k, k, -1, **ok),
        lambda: c.append(0, k.float(), k, cached, **ok), lambda: c.append(0, k[:1], k, cached, **ok), lambda: c.append(0, k[:, :1], k, cached, **ok),
        lambda: c.append(0, k.cpu(), k, cached, **ok), lambda: c.append(0, k, k, cached, q=q[:1], **ok), lambda: c.append(0, k, k, cached, depth=start, **ok),
        lambda: c.append(0, k, k, cached, q=q, q_out=torch.empty_like(k), **ok), lambda: c.append(0, k, k, cached, q=q, q_out=q.float(), **ok),
        lambda: c.append(0, k, k, cached, q=q, q_out=q.transpose(0, 1).contiguous().transpose(0, 1), **ok),
        lambda: c.attend(0, rows(1, 2, 3, 64), cached, **ok), lambda: c.attend(0, q[..., :32], cached, **ok), lambda: c.attend(0, q, cached, max_new=0, **ok),
        lambda: c.attend(0, q, cached, amask=torch.ones(2, 2, device=DEV), **ok), lambda: c.attend(0, q, cached, amask=torch.ones(1, 2, dtype=torch.uint8, device=DEV), **ok),
        lambda: c.read(2, 1, cached, **ok), lambda: c.read(0, 1, cached),
        lambda: c.compact(start.cpu(), 0), lambda: c.compact(start[:1], 0), lambda: c.compact(start, 0, seq=2), lambda: c.move([0], [1, 2]),
        lambda: KvCache4(1, 3, 2, 96, c.table), lambda: KvCache4(1, 3, 0, 64, c.table), lambda: KvCache4(1, 3, 2, 64, c.table.long()),
        lambda: KvCache4(1, 3, 2, 64, c.table.cpu()), lambda: KvCache4(1, 3, 2, 64, c.table, pool=c.pool[0]), lambda: KvCache4(1, 0, 2, 64, c.table),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    one = KvCache4(1, c.n_pages, 2, 64, c.table[:1], pool=c.pool)
    for call in (lambda: one.append(0, k, k, 63), lambda: one.attend(0, q, 64), lambda: one.attend(0, q, 3, amask=torch.ones(2, 1, dtype=torch.uint8, device=DEV))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: one.compact(ints(1, 0, 0), 64), lambda: one.compact(ints(1, 0, 0), -1), lambda: one.move([0], [64]), lambda: one.move([-1], [0])):
        with pytest.raises(_lib.FlintError) as e:
            call()
        assert e.value.code == _lib.FB_ERR_RANGE
    c.check()
    assert page_bytes(2, 64) == 2 * 4 * (16 * 64 + 128)
