"""What a ring's barriers are told when the warps that fill it together give up after different numbers of items
(tilus_b200/csrc/ring.cuh), compiled for the host and played through with a model of the barrier."""
import ctypes
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = """
#include "ring.cuh"
extern "C" void rest(int slot, int slots, const int* issued, const unsigned* bytes, int* item, unsigned* announce, unsigned* strike) {
  const int i[4] = {issued[0], issued[1], issued[2], issued[3]};
  const uint32_t b[4] = {bytes[0], bytes[1], bytes[2], bytes[3]};
  const b200q::RingRest r = b200q::ring_rest(slot, slots, i, b);
  *item = r.item;
  *announce = r.announce;
  *strike = r.strike;
}
"""


@pytest.fixture(scope="module")
def rest(tmp_path_factory):
    base = tmp_path_factory.mktemp("rest")
    (base / "rest.cpp").write_text(SOURCE)
    out = str(base / "rest.so")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I" + os.path.join(ROOT, "tilus_b200", "csrc"),
                           str(base / "rest.cpp"), "-o", out])
    lib = ctypes.CDLL(out)

    def call(slot, slots, issued, sizes):
        item, announce, strike = ctypes.c_int(), ctypes.c_uint(), ctypes.c_uint()
        lib.rest(slot, slots, (ctypes.c_int * 4)(*issued), (ctypes.c_uint * 4)(*sizes), ctypes.byref(item), ctypes.byref(announce), ctypes.byref(strike))
        return item.value, announce.value, strike.value

    return call


class Barrier:
    """One arrival a phase, and bytes that may land before they are announced."""

    def __init__(self):
        self.phases, self.pending, self.bytes = 0, 1, 0

    def _look(self):
        if self.pending == 0 and self.bytes == 0:
            self.phases, self.pending = self.phases + 1, 1

    def arrive(self, announced):
        assert self.pending == 1
        self.pending, self.bytes = 0, self.bytes + announced
        self._look()

    def landed(self, n):
        self.bytes -= n
        self._look()


@pytest.mark.parametrize("slots", [1, 2, 6, 8])
def test_the_phases_end_when_what_was_asked_for_has_landed(rest, slots):
    rng = random.Random(slots)
    for _ in range(400):
        sizes = [16384, rng.choice([8192, 16384])] * 2
        bars, issued, flying, through = [Barrier() for _ in range(slots)], [0] * 4, [], 0
        missing = {}
        for _ in range(rng.randrange(1, 40 * slots)):
            what = rng.random()
            i = rng.randrange(4)
            if what < 0.5 and issued[i] < through + slots:  # (the slot's last item is through)
                item = issued[i]
                if i == 0:
                    bars[item % slots].arrive(sum(sizes))
                flying.append((item, i))
                missing[item] = missing.get(item, 4)
                issued[i] += 1
            elif what < 0.8 and flying:
                item, i = flying.pop(rng.randrange(len(flying)))
                bars[item % slots].landed(sizes[i])
                missing[item] -= 1
            elif missing.get(through) == 0:
                through += 1
        for slot in range(slots):
            item, announce, strike = rest(slot, slots, issued, sizes)
            mine = [j for j in range(max(issued)) if j % slots == slot]
            assert item == (mine[-1] if mine else -1)
            if announce:
                bars[slot].arrive(announce)
            if strike:
                bars[slot].landed(strike)
        rng.shuffle(flying)
        while True:
            for slot in range(slots):
                item = rest(slot, slots, issued, sizes)[0]
                if item >= 0:  # a wait for the item's parity passes when its phase, which is the item's lap, has ended, and not before
                    assert bars[slot].phases in (item // slots, item // slots + 1)
                    assert (bars[slot].phases == item // slots + 1) == all(f[0] != item for f in flying)
            if not flying:
                break
            item, i = flying.pop()
            bars[item % slots].landed(sizes[i])
