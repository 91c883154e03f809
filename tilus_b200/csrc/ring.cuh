// A warp's ring of shared-memory slots: item i is the (i / slots)-th use of slot i % slots, one phase of the slot's mbarrier each.  Plain
// integer C++, so that a test checks it on the host.
#pragma once
#include "decode.cuh"

namespace b200q {

// The uses of a ring behind which `issued` items have been asked for: how many of them belong to the last lap, its parity, and whether
// there was one before.  (Subtractions: divisions by the run-time number of slots, on a path that only a launch that gives up takes, cost the
// kernel that keeps the activations in registers up to 2 % of every other launch.)
struct RingLaps { int last; uint32_t parity; bool earlier; };
B200Q_HD RingLaps ring_laps(int issued, int slots) {
  RingLaps r = {issued, 0u, issued > slots};
  while (r.last > slots) { r.last -= slots; r.parity ^= 1u; }
  return r;
}
// whether a slot has been asked for, and the parity that a wait for its last copy names (the use two laps back has the same
// parity, but has ended)
B200Q_HD bool ring_used(const RingLaps& r, int slot) { return slot < r.last || r.earlier; }
B200Q_HD uint32_t ring_parity(const RingLaps& r, int slot) { return slot < r.last ? r.parity : r.parity ^ 1u; }

// A ring that several warps fill, each with its part of every item, whose bytes one barrier a slot counts; the first warp arrives there and
// announces the bytes of all parts.  Where they have given up after different numbers of items: what the barrier of `slot` must be told for
// the phase under way to end when what has been asked for has landed.  (A part is asked for when the slot's last item is through, so
// that only the latest item can be incomplete.)
struct RingRest {
  int item;           // the latest that any of them has asked for in this slot, -1: none
  uint32_t announce;  // bytes to arrive with (0: the first warp has)
  uint32_t strike;    // announced bytes that will not come
};
template <int N>
B200Q_HD RingRest ring_rest(int slot, int slots, const int (&issued)[N], const uint32_t (&bytes)[N]) {
  int most = 0;
  for (int i = 0; i < N; ++i) most = issued[i] > most ? issued[i] : most;
  RingRest r = {-1, 0u, 0u};
  if (slot >= most) return r;
  r.item = slot + (most - 1 - slot) / slots * slots;
  uint32_t asked = 0, all = 0;
  for (int i = 0; i < N; ++i) {
    all += bytes[i];
    if (issued[i] > r.item) asked += bytes[i];
  }
  if (issued[0] > r.item) r.strike = all - asked;
  else r.announce = asked;
  return r;
}

}  // namespace b200q
