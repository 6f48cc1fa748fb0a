// Host check of the decode kernel's division of work (csrc/decode_parts.h):
// prints what does not hold and returns the number of such findings.
#include <cstdio>
#include <initializer_list>

#include "decode_parts.h"

using namespace moe;

static int bad = 0;
#define CHECK(c, ...)                                     \
  do {                                                    \
    if (!(c)) {                                           \
      if (bad++ < 20) std::printf(__VA_ARGS__), std::puts(" (" #c ")"); \
    }                                                     \
  } while (0)

// Both passes of one call, as decode_kernel makes them.
static void check(int T, int G, int H, int F, int nact) {
  const int kb1 = (H + 63) / 64, nt1 = (F + 127) / 128, kb2 = (F + 63) / 64, nt2 = (H + 255) / 256;
  for (int pass = 1; pass <= 2; ++pass) {
    auto make = [&](int cta) {
      return pass == 1 ? make_pass(T, G, cta, nact * nt1, kb1, kb1, nt1, ragged_rows(F))
                       : make_pass(T, G, cta, nact > 0 ? nt2 : 0, nact * kb2, kb2, nt2, false);
    };
    const Pass p = make(0);
    const int parts = p.g + p.chunks, tiles = pass == 1 ? nact * p.nt : p.nt;
    CHECK(parts <= G + max_chunks(T, pass == 1 && ragged_rows(F)), "T %d H %d F %d nact %d pass %d", T, H, F, nact, pass);
    // The shares, then the chunks, are the units in order.
    int u = 0;
    for (int c = 0; c < G; ++c) {
      const Pass q = make(c);
      if (c >= p.g) {
        CHECK(q.lo == q.hi, "T %d H %d F %d nact %d pass %d: CTA %d", T, H, F, nact, pass, c);
        continue;
      }
      CHECK(q.lo == u && q.hi > q.lo, "T %d H %d F %d nact %d pass %d: CTA %d", T, H, F, nact, pass, c);
      for (u = q.lo; u < q.hi; ++u)
        CHECK(p.part_of(u) == c, "T %d H %d F %d nact %d pass %d: unit %d", T, H, F, nact, pass, u);
    }
    CHECK(u == p.fixed && p.fixed + p.chunks * p.cz == p.units, "T %d H %d F %d nact %d pass %d", T, H, F, nact, pass);
    for (; u < p.units; ++u)
      CHECK(p.part_of(u) == p.g + (u - p.fixed) / p.cz, "T %d H %d F %d nact %d pass %d: unit %d", T, H, F, nact, pass, u);
    // Joins ask for the parts of each tile's first and last unit.
    CHECK(tiles * p.tile == p.units, "T %d H %d F %d nact %d pass %d: %d tiles", T, H, F, nact, pass, tiles);
    for (int t = 0; t < tiles; ++t) {
      const int c0 = p.part_of(t * p.tile), c1 = p.part_of(t * p.tile + p.tile - 1);
      CHECK(0 <= c0 && c0 <= c1 && c1 < parts, "T %d H %d F %d nact %d pass %d: tile %d", T, H, F, nact, pass, t);
    }
  }
}

// A role follows the taker's chunks through the ring to the end marker; a
// chunk that does not come in time is reported.
static void check_runs() {
  const int H = 4096, F = 728, nact = 64, G = 148, cta = 5;
  const Pass p = make_pass(7, G, cta, nact * ((F + 127) / 128), H / 64, H / 64, (F + 127) / 128, true);
  CHECK(p.chunks > 2 * kDecRunSlots, "%d chunks", p.chunks);
  for (int given : {p.chunks, 3, 0}) {
    for (bool end : {true, false}) {
      Runs r = {0, 0, 0, 0};
      int waits = 0, fails = 0, seen = 0;
      const auto wait = [&](int slot, uint32_t parity) {
        CHECK(slot == waits % kDecRunSlots && parity == uint32_t(waits / kDecRunSlots & 1), "wait %d", waits);
        return waits++ < given + (end ? 1 : 0);
      };
      first_run(r, p, cta);
      CHECK(r.lo == p.lo && r.hi == p.hi && r.part == cta, "first run");
      while (follow_run(r, p, wait, [&](int) { return seen < given ? seen : -1; }, [&] { ++fails; })) {
        CHECK(r.lo == p.fixed + seen * p.cz && r.part == p.part_of(r.lo) && r.part == p.part_of(r.hi - 1), "chunk %d", seen);
        ++seen;
      }
      CHECK(seen == given, "%d of %d chunks", seen, given);
      CHECK(fails == (end ? 0 : 1), "%d failures reported, end marker %d", fails, int(end));
    }
  }
}

int main() {
  check_runs();
  const int Ts[] = {1, 7, 32, 33, 64}, Hs[] = {8, 64, 1344, 7168, 32768}, Fs[] = {8, 64, 728, 1408, 14336};
  for (int T : Ts)
    for (int H : Hs)
      for (int F : Fs)
        for (int nact : {0, 1, 3, 8, 17})
          for (int G : {148, 132, 1}) check(T, G, H, F, nact);
  return bad > 100 ? 100 : bad;
}
