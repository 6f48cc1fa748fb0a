// How the decode kernel deals a pass's units out to CTAs (decode.cu): plain
// integer arithmetic, the same on the host, where it is tested.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define MOE_HD __host__ __device__ __forceinline__
#else
#define MOE_HD inline
#endif

namespace moe {

constexpr int kDecMaxChunks = 640;  // handed out as CTAs get done
constexpr int kDecRunSlots = 16;    // > stages + 2 accumulators: runs under way in a CTA

// Share of CTA c of `units`, and the CTA a unit belongs to (g CTAs, g <= units;
// units * g < 2^32).
MOE_HD int share_lo(uint32_t units, uint32_t g, uint32_t c) { return int(units * c / g); }
MOE_HD int share_owner(uint32_t units, uint32_t g, uint32_t u) { return int(((u + 1) * g - 1) / units); }

MOE_HD bool ragged_rows(int n) { return n % 64 != 0; }

// The most chunks of a pass.  Their sums grow with the tokens: above 32 only
// ragged rows are worth them, and fewer (64 tokens: all would take 100 MB of
// scratch; 7168 x 2048, 64 experts: 781 us with, 756 without; 33 tokens,
// F 1000: 128 and 142).
MOE_HD int max_chunks(int T, bool ragged) { return T <= 32 ? kDecMaxChunks : ragged ? kDecMaxChunks / 2 : 0; }

// One pass: its units in order.  The first `fixed` are shared out evenly, the
// rest lies in `chunks` chunks of `cz`; a CTA's share and every chunk is a
// part.
// Pass 1: expert by expert, its tiles of 128 features of F, each over H.
// Pass 2: tile by tile of 256 features of H, each over the experts' F.
struct Pass {
  int units;     // of all CTAs
  int tile;      // units of one tile (the units whose sums belong together)
  int kb;        // units of one expert's K
  int nt;        // tiles per expert (pass 1), tiles (pass 2)
  int g;         // CTAs that have a share
  int fixed, chunks, cz;
  int lo, hi;    // this CTA's share
  MOE_HD int part_of(int u) const {
    return u < fixed ? share_owner(uint32_t(fixed), uint32_t(g), uint32_t(u)) : g + (u - fixed) / cz;
  }
};

// A pass over `tiles` tiles of `tile` units for T tokens, as CTA `cta` of G
// sees it.
MOE_HD Pass make_pass(int T, int G, int cta, int tiles, int tile, int kb, int nt, bool ragged) {
  Pass p;
  p.units = tiles * tile;
  p.tile = tile;
  p.kb = kb;
  p.nt = p.units > 0 ? nt : 0;  // no unit: no tile, whose parts a join would ask for
  p.chunks = 0;
  p.cz = 1;
  // Shorter lists: the chunks' sums cost more than they gain.  Rows of w13
  // that are no multiple of 128 bytes set the SMs further apart (18 tokens,
  // F 728: shares of pass 1 done after 70 to 107 us), so there a third is
  // dealt out, in smaller chunks and from shorter lists on (88 us); it gains
  // nothing in pass 2, whose pieces of a row are twice as long.
  const int most = max_chunks(T, ragged);
  if (most > 0 && p.units >= (ragged ? 32 : 128) * G) {
    const int rest = p.units / (ragged ? 3 : 8), smallest = ragged ? 8 : 16, needed = (rest + most - 1) / most;
    p.cz = needed > smallest ? needed : smallest;
    p.chunks = rest / p.cz;
  }
  p.fixed = p.units - p.chunks * p.cz;
  // Short lists: a part costs the one who adds a tile's up about a fifth of
  // the time of a unit, so about sqrt(tile / 5) units a CTA at least.
  int least = 1;
  while (5 * (least + 1) * (least + 1) <= tile && least < 8) ++least;
  const int few = p.fixed / least > 0 ? p.fixed / least : p.fixed > 0 ? 1 : 0;
  p.g = few < G ? few : G;
  const bool on = cta < p.g;
  p.lo = on ? share_lo(uint32_t(p.fixed), uint32_t(p.g), uint32_t(cta)) : 0;
  p.hi = on ? share_lo(uint32_t(p.fixed), uint32_t(p.g), uint32_t(cta) + 1) : 0;
  return p;
}

// The runs of units that a CTA does in a pass: its share, then chunks until
// none is left.  One thread takes them and the other roles follow through a
// ring of kDecRunSlots; `n` counts a role's chunks over both passes.
struct Runs {
  int n;       // chunks seen by this role
  int lo, hi;  // current run
  int part;
};
MOE_HD void first_run(Runs& r, const Pass& p, int cta) {
  r.lo = p.lo;
  r.hi = p.hi;
  r.part = cta;
}
MOE_HD bool set_run(Runs& r, const Pass& p, int chunk) {  // chunk -1: the end
  r.lo = p.fixed + chunk * p.cz;
  r.hi = r.lo + p.cz;
  r.part = p.g + chunk;
  return chunk >= 0;
}
// The next run that the taker left in the ring: wait(slot, parity) waits for
// it, chunk(slot) reads it.  A wait that gives up is an error, not the end.
template <typename Wait, typename Chunk, typename Fail>
MOE_HD bool follow_run(Runs& r, const Pass& p, Wait wait, Chunk chunk, Fail fail) {
  if (p.chunks == 0) return false;
  const int slot = r.n % kDecRunSlots;
  if (!wait(slot, uint32_t(r.n / kDecRunSlots) & 1)) {
    fail();
    return false;
  }
  ++r.n;
  return set_run(r, p, chunk(slot));
}

}  // namespace moe
