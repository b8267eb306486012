"""CPU: how attention over the 4-bit cache is cut (flint_b200/csrc/fb_kv4_geometry.hpp, plain C++): tasks never outnumber the grid and the scratch, and a context's
scratch is enough for every pass that its cache has room for."""
import ctypes
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flint_b200", "csrc")
SHIM = """
#include "fb_kv4_geometry.hpp"
using namespace fb;
extern "C" void geometry(int n_seq, int n_tokens, int nkv, int r, int max_new, int max_len, int sms, int cut, long long* o) {
  Kv4Geometry g = attend_geometry(n_seq, n_tokens, nkv, r, max_new, max_len, sms);
  if (!cut) g = whole(g, nkv);
  o[0] = g.rows; o[1] = g.groups; o[2] = g.ctas; o[3] = g.nsplit; o[4] = g.slots; o[5] = g.chunk; o[6] = (long long)attend_work(g, 128);
}
extern "C" size_t most(int nkv, int r, int hd, long long slots, int rows_max, int sms) { return attend_most(nkv, r, hd, slots, rows_max, sms); }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("geometry")
    (d / "g.cpp").write_text(SHIM)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", CSRC, "-o", str(d / "g.so"), str(d / "g.cpp")])
    lib = ctypes.CDLL(str(d / "g.so"))
    lib.most.restype, lib.most.argtypes = ctypes.c_size_t, [ctypes.c_int] * 3 + [ctypes.c_longlong] + [ctypes.c_int] * 2
    return lib


def geometry(lib, *args, cut=1):
    o = (ctypes.c_longlong * 7)()
    lib.geometry(*args, 148, cut, o)
    return dict(zip(("rows", "groups", "ctas", "nsplit", "slots", "chunk", "work"), o))


def tasks_of(g, lens, new, nkv, r):
    """As every CTA counts them from the lengths on the GPU."""
    unit = 128 if g["rows"] >= 128 else 32
    units = [-(-(c + n) // unit) for c, n in zip(lens, new)]
    groups = [-(-n * r // g["rows"]) for n in new]
    per = max(g["chunk"], -(-sum(a * b for a, b, n in zip(units, groups, new) if n) * nkv // g["slots"])) if g["slots"] else 2 ** 31 - 1
    return sum(q * (-(-u // per)) * nkv for u, q, n in zip(units, groups, new) if n), sum(q for q, n in zip(groups, new) if n)


def test_tasks_do_not_outnumber_the_grid(lib):
    rng = random.Random(1)
    cut = 0
    for _ in range(20000):
        n_seq = rng.choice((1, 1, 2, 3, 8, 40))
        nkv, r = rng.choice((1, 2, 4, 8, 32)), rng.choice((1, 2, 4, 5, 8, 16))
        new = [rng.choice((0, 1, 1, 1, 3, 26, 61, rng.randrange(1, 400))) for _ in range(n_seq)]
        lens = [int(10 ** rng.uniform(0, 4.6)) for _ in range(n_seq)]
        T = sum(new) + rng.choice((0, 0, 5))
        if T == 0:
            continue
        true = rng.random() < 0.6                           # else: hints that are not so
        max_new = min(T, max(new) if true and max(new) else rng.randrange(1, T + 1))
        max_len = max(lens) + max(new) if true else int(10 ** rng.uniform(0, 5))
        for c in (1, 0):
            g = geometry(lib, n_seq, T, nkv, r, max_new, max_len, cut=c)
            tasks, groups = tasks_of(g, lens, new, nkv, r)
            assert tasks <= g["ctas"] and groups <= g["groups"]
            assert g["work"] == (g["ctas"] * g["rows"] * 132 * 4 if g["slots"] else 0) and (c or g["work"] == 0)
            cut += bool(g["slots"])
    assert cut > 1000


@pytest.mark.parametrize("nkv,r", [(8, 4), (8, 5), (2, 4), (32, 1), (1, 8), (4, 8)])
def test_the_scratch_of_a_context_is_enough(lib, nkv, r):
    rng = random.Random(nkv * 100 + r)
    for slots in (64, 512, 1344, 4096, 33024, 131072):
        most = lib.most(nkv, r, 128, slots, 1024, 148)
        asked = 0
        for _ in range(4000):
            m = rng.choice((1, 3, 26, 61, rng.randrange(1, 1025)))
            if m <= slots:
                asked = max(asked, geometry(lib, 1, m, nkv, r, m, rng.choice((slots, rng.randrange(m, slots + 1))))["work"])
        assert asked <= most <= 80e6
        assert slots > 512 or most <= 8e6                  # short caches: little or nothing
