"""CPU: the 4-bit cache's host side: sizes, the rotation's frequencies, and the calls that the library refuses before it touches a GPU."""
import ctypes
import math

import pytest
import torch

from flint_b200 import _lib, kv4
from tests import kv4_reference as ref


def test_page_bytes():
    for hd in (64, 80, 128):
        assert kv4.page_bytes(8, hd) == 8 * 64 * (hd + 8)        # a row: a nibble a number of K and of V, two pairs of bf16
    for nkv, hd in ((8, 96), (0, 64), (-1, 64), (8, 0)):
        with pytest.raises(ValueError):
            kv4.page_bytes(nkv, hd)


@pytest.mark.parametrize("hd,base", [(64, 1e4), (80, 1e7), (128, 5e5)])
def test_turns_give_the_angle_of_far_positions(hd, base):
    t = kv4.rope_turns(hd, base, "cpu").tolist()
    for i in (0, 1, hd // 4, hd // 2 - 1):
        for pos in (1, 4095, 131071):
            turn = (pos * t[i]) % (1 << 64) / 2.0 ** 64
            want = pos * base ** (-2.0 * i / hd) / (2 * math.pi) % 1.0
            assert abs((turn - want + 0.5) % 1.0 - 0.5) < 1e-11


def test_the_reference_quantiser_is_within_half_a_step():
    x = torch.randn(200, 80).bfloat16().float()
    n, s, z = ref.quantised(x)
    # half a step of s, and what rounding s and z to bf16 moves the ends: 15 s 2^-9 and |z| 2^-9
    assert ((ref.values(x) - x).abs() <= 0.5 * s * 1.01 + 15 * s * 2.0 ** -8 + z.abs() * 2.0 ** -8).all()


def _seqs(**kw):
    d = dict(d_pool=4096, d_table=4096, d_start=None, d_cached=None, d_status=4096, cached=0, n_pages=4, n_kv_head=2, head_dim=64, n_seq=1, table_ld=4, n_tokens=1, device=0)
    d.update(kw)
    return _lib.Kv4Seqs(*[d[n] for n, _ in _lib.Kv4Seqs._fields_])


REFUSED = [
    (dict(d_pool=None), _lib.FB_ERR_ARG), (dict(d_pool=4104), _lib.FB_ERR_ARG), (dict(d_table=None), _lib.FB_ERR_ARG), (dict(d_table=4098), _lib.FB_ERR_ARG),
    (dict(d_status=None), _lib.FB_ERR_ARG), (dict(head_dim=96), _lib.FB_ERR_SHAPE), (dict(n_kv_head=0), _lib.FB_ERR_ARG), (dict(n_pages=0), _lib.FB_ERR_ARG),
    (dict(table_ld=0), _lib.FB_ERR_ARG), (dict(n_seq=-1), _lib.FB_ERR_ARG), (dict(n_tokens=-1), _lib.FB_ERR_ARG), (dict(cached=-1), _lib.FB_ERR_RANGE),
    (dict(cached=256), _lib.FB_ERR_RANGE), (dict(table_ld=2 ** 31 - 1), _lib.FB_ERR_RANGE),
]


@pytest.mark.parametrize("kw,code", REFUSED)
def test_sequences_that_cannot_be(kw, code):
    lib = _lib.load()
    s = _seqs(**kw)
    p = ctypes.byref(s)
    assert lib.fb_kv4_append(p, None, 0, 4096, 128, 4096, 128, 4, None, None, None, 0, None) == code
    assert lib.fb_kv4_attend(p, 4096, 256, 4, 1, 1, None, 0, 1.0, 4096, 256, None, 0, None) == code
    assert lib.fb_kv4_read(p, 1, 0, 4096, 4096, None) == code


def test_rows_that_cannot_be():
    lib, A = _lib.load(), _lib.FB_ERR_ARG
    s = _seqs()
    p = ctypes.byref(s)
    append = lambda q=4096, q_ld=256, k=4096, k_ld=128, v=4096, v_ld=128, nh=4, depth=None, freq=None, o=4096, o_ld=256: lib.fb_kv4_append(  # noqa: E731
        p, q, q_ld, k, k_ld, v, v_ld, nh, depth, freq, o, o_ld, None)
    for kw in (dict(k=None), dict(v=None), dict(k=4104), dict(k_ld=120), dict(v_ld=129), dict(q=4098), dict(q_ld=248), dict(o=None), dict(o_ld=260), dict(nh=0), dict(freq=4100),
               dict(depth=4097)):
        assert append(**kw) == A, kw
    attend = lambda q=4096, q_ld=256, nh=4, most=1, length=1, mask=None, m_ld=0, o=4096, o_ld=256: lib.fb_kv4_attend(  # noqa: E731
        p, q, q_ld, nh, most, length, mask, m_ld, 1.0, o, o_ld, None, 0, None)
    for kw in (dict(q=None), dict(o=None), dict(q=4100), dict(q_ld=255), dict(o_ld=8), dict(most=0), dict(length=0), dict(mask=4096, m_ld=0)):
        assert attend(**kw) == A, kw
    assert attend(nh=3) == _lib.FB_ERR_SHAPE and attend(nh=0) == _lib.FB_ERR_SHAPE
    several = _seqs(n_seq=2)
    assert lib.fb_kv4_attend(ctypes.byref(several), 4096, 256, 4, 1, 1, None, 0, 1.0, 4096, 256, None, 0, None) == A      # whose tokens?
    for n_layer, layer in ((0, 0), (70000, 0), (1, 8), (1, -16)):
        assert lib.fb_kv4_read(p, n_layer, layer, 4096, 4096, None) == A
        assert lib.fb_kv4_compact(p, n_layer, layer, 4096, 1, None) == A
        assert lib.fb_kv4_move(p, n_layer, layer, None, None, 0, None) == A
    assert lib.fb_kv4_compact(p, 1, 0, None, 1, None) == A and lib.fb_kv4_compact(p, 1, 0, 4098, 1, None) == A
    one = (ctypes.c_int32 * 1)(256)
    zero = (ctypes.c_int32 * 1)(0)
    assert lib.fb_kv4_move(p, 1, 0, one, zero, 1, None) == _lib.FB_ERR_RANGE
    assert lib.fb_kv4_move(p, 1, 0, zero, one, 1, None) == _lib.FB_ERR_RANGE
    assert lib.fb_kv4_move(p, 1, 0, None, None, 1, None) == A


def test_a_cache_needs_a_gpu():
    with pytest.raises(ValueError):
        kv4.KvCache4(1, 4, 2, 64, torch.zeros(1, 4, dtype=torch.int32))


def test_moves_need_a_sequence():
    lib = _lib.load()
    none, one = _seqs(n_seq=0, n_tokens=0), (ctypes.c_int32 * 1)(3)
    assert lib.fb_kv4_compact(ctypes.byref(none), 1, 0, 4096, 1, None) == _lib.FB_ERR_ARG
    assert lib.fb_kv4_move(ctypes.byref(none), 1, 0, one, one, 1, None) == _lib.FB_ERR_ARG
