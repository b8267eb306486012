"""CPU: what a launch over the 4-bit cache that gives up waits for before it ends (flint_b200/csrc/fb_drain.hpp), run against a model of the barriers in which everything ends
as late as it can: nothing may be in flight behind it, and no wait may be one that nothing ends."""
import ctypes
import itertools
import os
import re
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flint_b200", "csrc")
SHIM = """
#include "fb_drain.hpp"
typedef void (*Wait)(uint32_t);
typedef void (*Commit)();
typedef void (*RingWait)(uint32_t, uint32_t);
extern "C" void ring(uint32_t issued, RingWait wait) { fb::drain_ring_order<3>(issued, wait); }
extern "C" void commits(uint32_t committed, Wait wait, Commit commit) { fb::drain_commit_order(committed, wait, commit); }
"""
WAIT, RING_WAIT, COMMIT = ctypes.CFUNCTYPE(None, ctypes.c_uint32), ctypes.CFUNCTYPE(None, ctypes.c_uint32, ctypes.c_uint32), ctypes.CFUNCTYPE(None)


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("drain")
    (d / "drain.cpp").write_text(SHIM)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", CSRC, "-o", str(d / "drain.so"), str(d / "drain.cpp")])
    return ctypes.CDLL(str(d / "drain.so"))


class Barrier:
    """Phases 0 .. armed-1 have been issued, 0 .. over-1 of them have ended; a parity wait passes when phase over - 1 has that parity, else the next one ends."""

    def __init__(self, armed=0, over=0):
        self.armed, self.over, self.hung = armed, over, False

    def wait(self, parity):
        while (self.over & 1) == parity:
            if self.over == self.armed:
                self.hung = True
                return
            self.over += 1

    @property
    def quiet(self):
        return self.over == self.armed and not self.hung


def ring_of(issued, under_way):
    """A ring of three stages that copies 0 .. issued-1 went to, stage after stage, those in `under_way` not over."""
    stages = [Barrier() for _ in range(3)]
    for i in range(issued):
        stages[i % 3].armed += 1
        stages[i % 3].over += i not in under_way
    return stages


@pytest.mark.parametrize("issued", range(11))
def test_every_copy_has_ended(lib, issued):
    last = range(max(0, issued - 3), issued)               # the last one of a stage may be under way, those before it are over
    for under_way in itertools.chain.from_iterable(itertools.combinations(last, n) for n in range(4)):
        stages = ring_of(issued, under_way)
        lib.ring(issued, RING_WAIT(lambda s, parity: stages[s].wait(parity)))
        assert all(b.quiet for b in stages)


def test_a_copy_that_was_not_issued_does_not_count(lib):
    """One too many: the oldest copy is passed over while it is under way, and a wait that nothing ends where it is not."""
    stages = ring_of(4, {1})
    lib.ring(5, RING_WAIT(lambda s, parity: stages[s].wait(parity)))
    assert not stages[1].quiet and not stages[1].hung
    stages = ring_of(4, set())
    lib.ring(5, RING_WAIT(lambda s, parity: stages[s].wait(parity)))
    assert stages[1].hung


@pytest.mark.parametrize("committed", range(7))
def test_every_product_has_ended(lib, committed):
    """The last commit may be under way or over; the one before it is over (a tile's next products wait for it)."""
    for over in {max(0, committed - 1), committed}:
        b = Barrier(committed, over)
        lib.commits(committed, WAIT(b.wait), COMMIT(lambda: setattr(b, "armed", b.armed + 1)))
        assert b.armed == committed + 1 and b.quiet


def test_the_model_shows_the_orders_that_do_not_do():
    """One more commit and a wait for it alone passes over the commit ahead of it; a wait for both behind it may be one that nothing ends."""
    b = Barrier(3, 2)
    b.armed += 1
    b.wait(1)
    assert not b.quiet
    b = Barrier(3, 3)
    b.armed, b.over = 4, 4
    b.wait(0)
    assert b.hung


def test_no_arrival_is_left_that_nobody_waits_for():
    """The places of K and V are waited for from the third step on, two steps behind the products that free them: products of the last two steps announce nothing, or the
    announcement could come after the CTA has ended."""
    with open(os.path.join(CSRC, "fb_kv4_tc.cuh")) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    for bar in ("k_empty", "v_empty"):
        assert re.findall(r"if \(([^;{}]*)\)\s*tc_commit\(&%s\b" % bar, code) == ["t == tiles - 1 && i + 2 < n"] and code.count("tc_commit(&" + bar) == 1
        assert re.findall(r"if \(([^;{}]*)\) ok = __all_sync\(0xffffffffu, mbar_wait\(&%s\[b\], before" % bar, code) == ["i >= 2"]
    assert "before = (uint32_t)((i >> 1) - 1) & 1u" in code
