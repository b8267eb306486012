"""GPU: the 4-bit cache where its calls can go wrong: pages that the table does not have, rows that nobody sees, numbers of every size, sequences that cannot be."""
import ctypes

import pytest
import torch

from flint_b200 import _lib, packing
from flint_b200.config import ModelArgs
from flint_b200.engine import DecodeEngine
from flint_b200.kv4 import KvCache4
from tests import kv4_bounds
from tests.test_gpu_kv4 import check_attention, filled, gen, ints, make, rows

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("hd", [64, 80, 128])
@pytest.mark.parametrize("nkv", [2, 148])                   # tasks of a few steps, and of all of them
@pytest.mark.parametrize("missing", [[1], [2], [5], [7], [2, 3], [4, 7]])
def test_many_rows_leave_out_pages_that_the_table_does_not_have(hd, nkv, missing):
    """First and second pages of a step in the middle of a sequence. The places that their copies would go to hold what was there before: page 3's values, which are
    numbers but none that fp16 has, or whatever shared memory held."""
    cached, new, nh = 640, 40, 2 * nkv
    c = make([cached + new], nkv, hd, base=None, garbage=True)
    k, v = rows(1, cached + new, nkv, hd, 1.3), rows(2, cached + new, nkv, hd)
    v[192:256] *= 2.0 ** 18
    c.append(0, k, v, 0)
    K, V = c.read(0, cached + new, 0)
    q = rows(3, new, nh, hd, 1.5)
    seen = torch.ones(cached + new, dtype=torch.bool, device=DEV)
    for page in missing:
        seen[64 * page:64 * page + 64] = False
        c.table[0, page] = -1
    for _ in range(2):
        out = c.attend(0, q, cached)
        st = c.status()
        assert st["code"] == _lib.FB_ERR_RANGE and st["where"] == 21
        check_attention(out, q, K[seen], V[seen], cached - 64 * len(missing), hd ** -0.5, wide=True)


@pytest.mark.parametrize("name,M,pos,limits", [("tiny", 1, 10000, (0, 0, 3, 20, 100, 300)), ("tiny", 3, 10000, (0, 10, 100)), ("llama-8b-class", 1, 32700, (0, 0, 3, 20, 100, 300)),
                                               ("llama-8b-class", 2, 9000, (0, 20, 300))])
def test_passes_over_long_caches_that_give_up_leave_nothing_behind(name, M, pos, limits):
    """Limits of the waits from nothing on, in launches whose copying warp comes back to a stage more than once: the next clean pass gives the bits of the first."""
    cfg = ModelArgs.from_name(name)
    if name != "tiny":
        cfg.n_layer, cfg.vocab_size = 1, 512
    eng = DecodeEngine(cfg, packing.synth_packed(cfg, 0, device=DEV), max_seq=pos + 64, kv_bits=4)
    for layer in range(cfg.n_layer):
        eng.cache.append(layer, rows(2 * layer, pos, cfg.n_local_heads, cfg.head_dim), rows(2 * layer + 1, pos, cfg.n_local_heads, cfg.head_dim), 0)
    toks = torch.arange(5, 5 + M, dtype=torch.int32, device=DEV)
    run = (lambda: eng.decode(17, pos).clone()) if M == 1 else (lambda: eng.verify(toks, pos)[0])
    want = run()
    eng.check()
    for limit in limits * 2:
        eng.set_option(0, limit)
        run()
        assert eng.status()["code"] in (_lib.FB_OK, _lib.FB_ERR_TIMEOUT)
        eng.set_option(0, 4000000)
        again = run()
        eng.check()
        assert torch.equal(want, again)


def test_a_bound_cache_takes_nothing_from_the_fields_that_are_not_read():
    """The structure of some earlier call, its lengths those of that call."""
    cfg = ModelArgs.from_name("tiny")
    packed = packing.synth_packed(cfg, 0, device=DEV)
    got = []
    for cached, n_tokens in ((0, 0), (1000, 128), (-7, -9), (128, 2 ** 31 - 1)):
        eng = DecodeEngine(cfg, packed, max_seq=128, kv_bits=4)
        s = eng.cache._one(0, 0)
        s.cached, s.n_tokens, s.d_start, s.d_cached, s.d_status = cached, n_tokens, 4096, 4096, None
        _lib.check(eng.lib.fb_bind_kv4(eng._ctx, ctypes.byref(s), eng.cache.layer_bytes, eng.cache.freq.data_ptr()), "fb_bind_kv4")
        toks = torch.arange(5, 25, dtype=torch.int32, device=DEV)
        eng.prefill(toks, 0)
        eng.kv_move([3, 4, 100], [5, 3, 127])
        eng.kv_compact(ints(3, 0, 0, 2, 6), 10)
        got.append(eng.decode(17, 20).clone())
        eng.check()
        assert torch.equal(got[0], got[-1])
        for name in ("head_dim", "n_kv_head", "n_seq", "device"):
            t = eng.cache._one(0, 0)
            setattr(t, name, getattr(t, name) + 1)
            assert eng.lib.fb_bind_kv4(eng._ctx, ctypes.byref(t), eng.cache.layer_bytes, eng.cache.freq.data_ptr()) in (_lib.FB_ERR_SHAPE, _lib.FB_ERR_ARG)


# ---------------------------------------------------------------------------------------------------------------- what comes out, as near as the roundings let it
@pytest.mark.parametrize("hd,nh,nkv", [(64, 40, 8), (80, 32, 8), (128, 32, 8), (64, 9, 1), (128, 34, 2)])
@pytest.mark.parametrize("cached,new,qscale", [(0, 1, 1.5), (31, 2, 1.5), (200, 1, 1.5), (1344, 3, 1.0), (1345, 1, 1.0), (5000, 1, 1.0), (11000, 1, 0.5), (33000, 1, 0.3), (33000, 3, 3.0)])
def test_few_rows_within_their_roundings(hd, nh, nkv, cached, new, qscale):
    """One CTA a group of rows, clusters, parts that a second launch joins. Flat scores: every page weighs."""
    c, K, V, q, _ = filled([cached], [new], nh, nkv, hd, seed=cached + hd, qscale=qscale)
    out = c.attend(0, q, cached)
    c.check()
    kv4_bounds.check(out, *kv4_bounds.bounds(q, K[0], V[0], cached, hd ** -0.5))


@pytest.mark.parametrize("hd,nh,nkv", [(64, 40, 8), (80, 32, 8), (128, 32, 8), (128, 8, 2)])
@pytest.mark.parametrize("cached,new,qscale", [(0, 70, 1.5), (0, 300, 1.5), (1000, 26, 1.5), (3001, 61, 1.0), (129, 200, 1.5), (9000, 33, 0.3)])
def test_many_rows_within_their_roundings(hd, nh, nkv, cached, new, qscale):
    c, K, V, q, _ = filled([cached], [new], nh, nkv, hd, seed=cached + hd, qscale=qscale)
    out = c.attend(0, q, cached)
    c.check()
    kv4_bounds.check(out, *kv4_bounds.bounds(q, K[0], V[0], cached, hd ** -0.5, many=new * nh // nkv > 64))


@pytest.mark.parametrize("hd,nh,nkv", [(64, 40, 8), (128, 8, 2)])
@pytest.mark.parametrize("lens,new", [([5, 300, 0, 64, 1, 2000], [1, 1, 0, 1, 1, 1]), ([0, 65, 700], [3, 0, 5]), ([10, 0, 130, 900], [80, 64, 1, 30]), ([3000] * 5, [1] * 5), ([6000, 5, 6000], [2, 2, 1])])
@pytest.mark.parametrize("masked", [False, True])
def test_batches_within_their_roundings(hd, nh, nkv, lens, new, masked):
    """Ragged sequences, causal and each token with a mask of its own over its sequence's new tokens, rows that see nothing of them included."""
    c, K, V, q, start = filled(lens, new, nh, nkv, hd, seed=hd)
    amask = None
    if masked:
        amask = (torch.rand(sum(new), max(new) + 3, generator=gen(7), device=DEV) < 0.5).to(torch.uint8)
        amask[::3] = 0
    many = max(new) * nh // nkv > 64
    out = c.attend(0, q, ints(*lens), start=start, amask=amask, max_new=max(new))
    c.check()
    for b in range(len(lens)):
        a, z = int(start[b]), int(start[b + 1])
        if z > a:
            kv4_bounds.check(out[a:z], *kv4_bounds.bounds(q[a:z], K[b], V[b], lens[b], hd ** -0.5, None if amask is None else amask[a:z], many=many))


# ---------------------------------------------------------------------------------------------------------------- numbers of every size
@pytest.mark.parametrize("hd", [64, 80, 128])
@pytest.mark.parametrize("new", [9, 100])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("power", [20, 30, 60, 100, -30, -90])
def test_keys_that_a_token_does_not_see_leave_it_alone(hd, new, masked, power):
    """A new token's key 2^power times the others': tokens ahead of it, or whose masks leave it out, come out within their roundings."""
    nh, nkv, cached = 8, 2, 100
    at = new // 2
    k, v = rows(71, cached + new, nkv, hd), rows(72, cached + new, nkv, hd)
    k[cached + at] = (k[cached + at].float() * 2.0 ** power).bfloat16()
    c = make([cached + new], nkv, hd, base=None, garbage=True)
    c.append(0, k, v, 0)
    K, V = c.read(0, cached + new, 0)
    q = rows(73, new, nh, hd, 1.5)
    amask = torch.ones(new, new, dtype=torch.uint8, device=DEV).tril() if masked else None
    if masked:
        amask[:, at] = 0
    out = c.attend(0, q, cached, amask=amask)
    c.check()
    blind = slice(0, new if masked else at)
    want = kv4_bounds.bounds(q, K, V, cached, hd ** -0.5, amask, many=new * nh // nkv > 64)
    kv4_bounds.check(out[blind], *(x[blind] for x in want))


@pytest.mark.parametrize("new", [1, 40])
def test_keys_of_many_sizes_side_by_side(new):
    """Keys from 2^-60 to 2^60 of the usual size, positions in random order; a query per size, 2^-60 to 2^60 times the usual, so that some keys decide and others are as nothing."""
    hd, nkv, nh, cached = 64, 1, 4, 400
    n = cached + new
    g = gen(80)
    size = torch.randint(-60, 1, (n,), generator=g, device=DEV).double().exp2().float()
    k = (torch.randn(n, nkv, hd, generator=g, device=DEV).abs() * size[:, None, None]).bfloat16()
    q = (-torch.randn(new, nh, hd, generator=g, device=DEV).abs() * torch.tensor([1.0, 2.0 ** 20, 2.0 ** 40, 2.0 ** 60], device=DEV)[:, None]).bfloat16()
    c = make([n], nkv, hd, base=None, garbage=True)
    c.append(0, k, rows(81, n, nkv, hd), 0)
    K, V = c.read(0, n, 0)
    out = c.attend(0, q, cached)
    c.check()
    kv4_bounds.check(out, *kv4_bounds.bounds(q, K, V, cached, hd ** -0.5, many=new * nh > 64))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,cached", [(1, 0), (1, 300), (2, 9000), (1, 40000), (40, 0), (40, 300), (130, 2000)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("power", [12, 22, 25, 28, 40, 98, 108])
def test_scores_of_any_size(hd, new, cached, sign, power):
    """All keys lie along one direction, the queries too, 2^power long; one position of the first 30 is ahead of all others by a sixth of its score or more (far more than a
    rounding): it takes everything, also where all scores are far below zero. Flat keys: equal scores of that size share evenly."""
    nh, nkv, n = 8, 2, cached + new
    g = gen(90)
    u = (torch.rand(hd, generator=g, device=DEV) + 0.5).bfloat16().float()
    a = torch.rand(n, 1, 1, generator=g, device=DEV) * 0.4 + 0.6
    first = min(n, 30) // 3
    a[first] = 1.2 if sign > 0 else 0.45
    c = make([n], nkv, hd, base=None, garbage=True)
    c.append(0, (a * u).expand(n, nkv, hd).bfloat16(), rows(91, n, nkv, hd), 0)
    _, V = c.read(0, n, 0)
    q = (u * sign * 2.0 ** power).expand(new, nh, hd).bfloat16()
    out = c.attend(0, q, cached)
    c.check()
    sees = slice(max(0, first - cached), new)
    want = V[first].repeat_interleave(nh // nkv, 0).expand(new, nh, hd)
    # the output to bf16; probability or probability times s, and the value, to fp16
    tol = want.abs() * 2.0 ** -8 + 2.0 ** -10 * V.abs().amax()
    assert ((out - want).abs() <= tol)[sees].all()
    if n <= 400:
        c.append(0, torch.ones(n, nkv, hd, dtype=torch.bfloat16, device=DEV), rows(92, n, nkv, hd), 0)
        _, V = c.read(0, n, 0)
        out = c.attend(0, q, cached)
        c.check()
        want = (V.double().cumsum(0) / torch.arange(1, n + 1, device=DEV)[:, None, None]).repeat_interleave(nh // nkv, 1)[cached:]
        assert ((out - want).abs() <= want.abs() * 2.0 ** -8 + 2.0 ** -10 * V.abs().amax()).all()


# ---------------------------------------------------------------------------------------------------------------- sequences that cannot be
@pytest.mark.parametrize("T", [3, 142])
@pytest.mark.parametrize("order", ["0T0T", "0T0", "00T0T", "T0T"])
def test_starts_that_go_down_leave_out_the_whole_call(T, order):
    """Two sequences would have the same tokens: nothing is written, no row of another sequence either, and the call is reported."""
    hd, nkv, nh = 64, 2, 8
    begin = [T if x == "T" else 0 for x in order]
    n_seq = len(begin) - 1
    c = make([T + 600] * n_seq, nkv, hd, base=1e4, garbage=True)
    start, cached = ints(*begin), ints(*[600] * n_seq)
    before = c.pool.clone()
    q, k = rows(1, T, nh, hd), rows(2, T, nkv, hd)
    q_out = torch.full_like(q, 7.0)

    def reported():
        st = c.status()
        assert st["code"] == _lib.FB_ERR_RANGE and st["where"] == 23 and begin[st["sequence"] + 1] < begin[st["sequence"]], st

    c.append(0, k, k, cached, q=q, start=start, q_out=q_out)
    reported()
    assert (q_out == 7.0).all() and torch.equal(c.pool, before)
    assert all((x == 0).all() for x in c.read(0, T, cached, start=start))
    reported()
    for hints in ({}, dict(max_new=1), dict(max_len=100000)):
        c.attend(0, q, cached, start=start, out=q_out, **hints)
        reported()
        assert (q_out == 7.0).all()


# ---------------------------------------------------------------------------------------------------------------- values next to the border of fp16's range
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("largest,flat,wide", [(2.0 ** -10, False, False), (2.0 ** -11.5, False, False), (2.0 ** -12.7, False, False), (2.0 ** -12.7, True, False), (2.0 ** -14, False, True),
                                               (2.0 ** -20, False, True), (2.0 ** -30, True, True), (2.0 ** 13, False, False), (2.0 ** 15, False, True)])
def test_a_row_of_small_values_takes_no_bits_from_its_page(hd, largest, flat, wide):
    """One row of every page of V has this largest number: down to 2^-13 its page stays in fp16."""
    nh, nkv, cached, new = 8, 2, 600, 40
    n = cached + new
    v = rows(101, n, nkv, hd).float()
    at = torch.arange(7, n, 64, device=DEV)
    v[at] *= largest / v[at].abs().amax(-1, keepdim=True)
    if flat:
        v[at] = largest
    c = make([n], nkv, hd, base=None, garbage=True)
    c.append(0, rows(102, n, nkv, hd, 1.3), v.bfloat16(), 0)
    K, V = c.read(0, n, 0)
    q = rows(103, new, nh, hd)
    out = c.attend(0, q, cached)
    c.check()
    kv4_bounds.check(out, *kv4_bounds.bounds(q, K, V, cached, hd ** -0.5, many=True, wide=torch.full((n,), wide, device=DEV)))


@pytest.mark.parametrize("power", [-9.5, -11.0, -12.5])
def test_rows_of_small_values_alone(power):
    """All rows that small, close together or far apart: nothing larger hides what they lose."""
    hd, nh, nkv, cached, new = 64, 8, 2, 300, 40
    n = cached + new
    for spread in (1.0, 0.1, 0.004):
        base = torch.randn(n, nkv, 1, generator=gen(111), device=DEV).sign()
        v = (base + spread * (torch.rand(n, nkv, hd, generator=gen(112), device=DEV) * 2 - 1)) / (1 + spread) * 2.0 ** power
        c = make([n], nkv, hd, base=None, garbage=True)
        c.append(0, rows(113, n, nkv, hd, 1.3), v.bfloat16(), 0)
        K, V = c.read(0, n, 0)
        q = rows(114, new, nh, hd)
        out = c.attend(0, q, cached)
        c.check()
        # steps of these rows that fp16 does not hold (below 2^-17): their page is in bf16
        narrow = 2 * spread / (1 + spread) * 2.0 ** power / 15 < 2.0 ** -16.9 and power < -9.9
        kv4_bounds.check(out, *kv4_bounds.bounds(q, K, V, cached, hd ** -0.5, many=True, wide=torch.full((n,), narrow, device=DEV)))


@pytest.mark.parametrize("hd", [64, 80, 128])
@pytest.mark.parametrize("new", [9, 100])
@pytest.mark.parametrize("masked", [False, True])
def test_values_that_a_token_does_not_see_leave_it_alone(hd, new, masked):
    """New tokens whose keys and values are the type's largest and smallest numbers, alone, among usual ones, and among others that take a row's numbers past the largest: tokens
    ahead of them, or whose masks leave them out."""
    nh, nkv, cached = 8, 2, 100
    top, at = torch.finfo(torch.bfloat16).max, new // 2
    for which in range(5):
        k, v = rows(121, cached + new, nkv, hd), rows(122, cached + new, nkv, hd)
        for x in (k, v):
            row = x[cached + at]
            if which < 2:
                row[:] = top if which else -top
            elif which == 2:
                row[:, ::5] = -top
            elif which == 3:
                row[:] = 1.08e36
                row[:, 3] = top
            else:
                row[:] = 0.0
                row[:, 1::2] = top
        c = make([cached + new], nkv, hd, base=None, garbage=True)
        c.append(0, k, v, 0)
        K, V = c.read(0, cached + new, 0)
        q = rows(123, new, nh, hd, 1.5)
        amask = torch.ones(new, new, dtype=torch.uint8, device=DEV).tril() if masked else None
        if masked:
            amask[:, at] = 0
        out = c.attend(0, q, cached, amask=amask)
        c.check()
        blind = slice(0, new if masked else at)
        K[cached + at], V[cached + at] = 0, 0              # the bounds' matrices multiply what is not seen by zero
        wide = torch.zeros(cached + new, dtype=torch.bool, device=DEV)
        wide[(cached + at) // 64 * 64:(cached + at) // 64 * 64 + 64] = True
        kv4_bounds.check(out[blind], *(x[blind] for x in kv4_bounds.bounds(q, K, V, cached, hd ** -0.5, amask, many=new * nh // nkv > 64, wide=wide)))


def test_scratch_of_an_engine_goes_by_its_cache():
    """A short cache takes next to none; a longer one bound later has what its passes need, and a pass captured over the short one still has its own."""
    cfg = ModelArgs.from_name("tiny")
    packed = packing.synth_packed(cfg, 0, device=DEV)
    nkv, hd = cfg.n_local_heads, cfg.head_dim

    def cache(slots):
        c = KvCache4(cfg.n_layer, slots // 64, nkv, hd, torch.arange(slots // 64, dtype=torch.int32, device=DEV)[None], rope_base=cfg.rope_base)
        for layer in range(cfg.n_layer):
            c.append(layer, rows(layer, slots - 640, nkv, hd), rows(layer + 9, slots - 640, nkv, hd), 0)
        return c
    short, middle, long = cache(704), cache(8000), cache(32000)
    eng = DecodeEngine(cfg, packed, max_seq=64)
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    eng.bind_kv4(short)
    assert free - torch.cuda.mem_get_info()[0] < 12e6
    tok, out = torch.tensor([7], dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    eng.decode_chained(tok, 64, out)
    want = out.clone()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        eng.decode_chained(tok, 64, out)
    toks = torch.arange(5, 605, dtype=torch.int32, device=DEV)
    for c in (middle, long, middle):
        eng.bind_kv4(c)
        for n in (1, 40, 300, 600):
            pos = c.slots - 640
            got = eng.decode(5, pos) if n == 1 else eng.prefill(toks[:n], pos)[0]
            fresh = DecodeEngine(cfg, packed, kv_bits=4, cache=c)
            again = fresh.decode(5, pos) if n == 1 else fresh.prefill(toks[:n], pos)[0]
            fresh.check()
            assert torch.equal(got, again)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    eng.check()
    assert torch.equal(out, want)


def test_a_prompt_of_several_chunks():
    """More tokens than a pass takes: the bits of the passes one by one, and of the decode steps behind them."""
    cfg = ModelArgs.from_name("tiny")
    packed = packing.synth_packed(cfg, 0, device=DEV)
    toks = torch.randint(0, cfg.vocab_size, (2300,), generator=torch.Generator().manual_seed(1), dtype=torch.int32).to(DEV)
    whole, parts = (DecodeEngine(cfg, packed, max_seq=2400, kv_bits=4) for _ in range(2))
    got, _ = whole.prefill(toks, 0)
    cuts = [0, 766, 1533, 2300]
    want = torch.cat([parts.prefill(toks[a:b], a)[0].clone() for a, b in zip(cuts, cuts[1:])])
    assert torch.equal(got, want) and torch.equal(whole.cache.pool, parts.cache.pool)
    assert torch.equal(whole.decode(5, 2300), parts.decode(5, 2300))
    whole.check()
    parts.check()


def test_tables_whose_rows_are_apart_are_refused():
    """A length on the GPU is held against the room of a row: with rows apart it could reach into the next one, or past the table."""
    big = torch.arange(24, dtype=torch.int32, device=DEV).view(3, 8)
    for table in (big[:, :4], big[:, 4:], big[::2], big.T, big.T[:, :2]):
        with pytest.raises(ValueError):
            KvCache4(1, 24, 2, 64, table)
    c = KvCache4(1, 24, 2, 64, big[1:])
    one = KvCache4(1, 24, 2, 64, big[2:, 4:])              # a piece of one row is a table
    assert c.slots == 512 and one.slots == 256
    x = rows(1, 2, 2, 64)
    for cache, cached, start in ((c, ints(512, 511), ints(0, 1, 2)), (one, ints(255), None)):
        before = cache.pool.clone()
        cache.append(0, x, x, cached, start=start)
        assert cache.status()["where"] == 22
        written = (cache.pool != before).any(-1).any(-1).nonzero()[:, 1].tolist()
        assert written == ([23] if cache is c else [])
