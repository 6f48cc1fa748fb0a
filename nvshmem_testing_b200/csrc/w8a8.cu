// The expert layer in 8-bit integers (the reference's products are bf16 only,
// baseline.py:50): rows quantised with a scale each, weights with a scale per
// output channel,
//   out[r, n] = xs[r] * ws[e, n] * sum_k xq[r, k] * wq[e, n, k],
// rows in expert order, one weight matrix per expert.
//
// Products (w8a8_kernel).  Transposed like the bf16 layer: channels are the
// MMA's M, token rows its N, so an expert's ragged row count costs at most 31
// padded rows, not a 256-row tile.  CTA pairs, tcgen05.mma.cta_group::2
// kind::i8 (M = 256, N <= 256, K = 32) with exact 32-bit sums in TMEM; both
// operands are K-major, 128 bytes of K per stage (one swizzle atom), six
// stages of 32 KB per CTA.  The scales are applied to the sums on the way out.
// With SwiGLU a CTA's 128 channels are 64 gate and the 64 matching up
// channels (two boxes of the same matrix, no relayout); the halves sit in
// different TMEM lanes and are exchanged through shared memory, and
// silu(gate) * up is written in fp32 for the quantisation that follows.
//
// Few tiles (small row counts) leave most SMs without one, although such
// products wait for the weights' bytes alone.  Then the list of (tile, 128 of
// K) units is split evenly over the pairs at any k, the partial sums go to
// scratch and, behind a grid barrier, are added and scaled.  Integer sums do
// not depend on the split.  (The barrier is cooperative groups', under a
// cooperative launch; every other wait is bounded, and after an error a CTA
// skips work, not the barrier.)
//
// Quantisation (quant_rows_kernel).  scale = absmax * (1/127) in fp32, q = the
// exact quotient x / scale rounded half to even: the product with the
// reciprocal is corrected by its remainder, which fp32 holds exactly.  One
// read of the row, kept in registers between maximum and rounding.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "moe_ep.h"
#include "moe_ep_internal.h"
#include "ptx.cuh"

namespace moe {
namespace {

namespace cg = cooperative_groups;

constexpr int kQStages = 6;
constexpr int kQKb = 128;                          // K per stage
constexpr uint32_t kQABytes = 128 * kQKb;          // 128 channels
constexpr uint32_t kQStageBytes = 2 * kQABytes;    // + up to 128 rows
constexpr int kQTileRows = 256;
constexpr int kQEpiWarps = 8;                      // two per TMEM lane quarter
constexpr int kQEpi0 = 2;
constexpr int kQThreads = (kQEpi0 + kQEpiWarps) * 32;
constexpr int kQXFloats = 32 * 20;                 // half a chunk of a warp, padded
constexpr uint32_t kQXBytes = kQEpiWarps * (kQXFloats + 32) * 4;  // and 32 row scales
constexpr int kQRowMaps = 4;                       // boxes of 16, 32, 64, 128 rows
constexpr uint64_t kQBoundNs = 2000000000ull;      // bug guard on every pipeline wait
constexpr int kQWaves = 4;                         // fewer tiles per pair: split over K
constexpr int kQMaxK = 131056;                     // 128 * 128 * K < 2^31
constexpr size_t kQSlotInts = 2 * 128 * kQTileRows;  // one pair's sums of one tile

struct QArgs {
  int E, K, N;                 // N: channels, both halves with SwiGLU
  int64_t rows;
  int F;                       // output columns: N, or N / 2
  const int32_t* counts;       // [E], or null: one matrix for all rows
  const float* xs;
  const float* ws;
  void* out;
  int out_f32;
  int32_t* part;               // split form: [pairs][2] slots
  int32_t* status_host;
};

struct QRowMaps {
  CUtensorMap m[kQRowMaps];
};

// ---------------------------------------------------------------- quantisation of one row
// Rounds x / s half to even, exactly: |x / s| <= 127.5, inv is 1 / s within
// 2^-23.  t holds the nearest integer of x * inv (within one of the answer) in its
// low mantissa bits; the remainder x - q*s fits fp32.
constexpr float kMagic = 12582912.f;  // 1.5 * 2^23
__device__ __forceinline__ int quant_one(float x, float s, float half, float inv) {
  const float t = fmaf(x, inv, kMagic);
  int q = __float_as_int(t) - __float_as_int(kMagic);
  const float r = fmaf(-(t - kMagic), s, x);
  const bool odd = q & 1;
  if (r > half || (r == half && odd)) ++q;
  if (r < -half || (r == -half && odd)) --q;
  return max(-127, min(127, q));
}

// Values by fours and eights.  inv and the product are each off by 2^-23 of
// themselves at most, so x * inv is within 127 * 2^-22 < 4e-5 of the quotient
// and its rounding is the quotient's unless that lies nearer to a tie: only
// then (bf16 rows: about 1 value in 500, half the row's maximum among them)
// the exact form runs.  t's low byte is the integer in two's complement.
__device__ __forceinline__ uint32_t quant4(const float* x, float s, float inv, bool exact) {
  uint32_t t[4];
  float far = exact ? 1.f : 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float y = fmaf(x[i], inv, kMagic);
    far = fmaxf(far, fabsf(fmaf(x[i], inv, kMagic - y)));
    t[i] = __float_as_uint(y);
  }
  if (far > 0.49995f) {
    const float half = 0.5f * s;
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = uint32_t(quant_one(x[i], s, half, inv));
  }
  return __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
}
__device__ __forceinline__ uint2 quant8(const float (&x)[8], float s, float inv, bool exact) {
  return make_uint2(quant4(x, s, inv, exact), quant4(x + 4, s, inv, exact));
}

__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 w = *reinterpret_cast<const uint4*>(p);
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&w);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(h[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  *reinterpret_cast<float4*>(&v[0]) = *reinterpret_cast<const float4*>(p);
  *reinterpret_cast<float4*>(&v[4]) = *reinterpret_cast<const float4*>(p + 4);
}

// A row's scale and what its values are rounded with, from the largest
// magnitude's bits.  Infinities and NaN (largest as numbers): no scale holds
// the row, and a NaN scale says so in every output.  Tiny rows: the
// reciprocal would overflow (powers of two change nothing), and a scale below
// the normal numbers is coarse.
struct RowScale {
  float scale, s, inv, up;
  bool zero, tiny;
  __device__ __forceinline__ explicit RowScale(uint32_t top) {
    const bool bad = top >= 0x7f800000u;
    scale = bad ? __int_as_float(0x7fffffff) : __uint_as_float(top) * (1.f / 127.f);
    zero = bad || scale == 0.f;
    tiny = scale < 0x1p-90f;
    up = tiny ? 0x1p100f : 1.f;
    s = zero ? 1.f : scale * up;
    inv = __fdividef(1.f, s);
  }
  __device__ __forceinline__ uint2 round8(float (&w)[8]) const {
    if (zero) return make_uint2(0u, 0u);
    if (tiny) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] *= up;
    }
    return quant8(w, s, inv, tiny);
  }
};

// The largest magnitude of values as they come, NaN above infinity.
template <typename In>
struct RowTop;
template <>
struct RowTop<__nv_bfloat16> {
  __nv_bfloat162 m = __floats2bfloat162_rn(0.f, 0.f);
  __device__ __forceinline__ void add(uint32_t w) {
    m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w)));
  }
  __device__ __forceinline__ uint32_t bits() const {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(&m);
    return max(w << 16, w & 0xffff0000u);
  }
};
template <>
struct RowTop<float> {
  float m = 0.f;
  __device__ __forceinline__ void add(uint32_t w) {
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(__uint_as_float(w))));
  }
  __device__ __forceinline__ uint32_t bits() const { return __float_as_uint(m); }
};

// Eight values as they lie in memory.
template <typename In>
struct Raw8 {
  uint4 r[sizeof(In) / 2];
  __device__ __forceinline__ void load(const In* p) {
#pragma unroll
    for (int i = 0; i < int(sizeof(In) / 2); ++i) r[i] = ld_nc_v4(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void top(RowTop<In>& t) const {
#pragma unroll
    for (int i = 0; i < int(sizeof(In) / 2); ++i) {
      t.add(r[i].x);
      t.add(r[i].y);
      t.add(r[i].z);
      t.add(r[i].w);
    }
  }
  __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < int(sizeof(In) / 2); ++i) {
      const uint32_t w[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(In) == 2) {
          v[2 * j] = __uint_as_float(w[j] << 16);
          v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        } else {
          v[4 * i + j] = __uint_as_float(w[j]);
        }
      }
    }
  }
};

struct alignas(16) QSmem {
  uint64_t full[kQStages];   // leader: both CTAs' bytes
  uint64_t empty[kQStages];  // each CTA: the stage has been multiplied
  uint64_t tfull[2];         // each CTA: sums ready
  uint64_t tempty[2];        // leader: both CTAs' epilogues are done with them
  uint64_t drain;
  uint32_t fills, used;      // stages loaded, multiplied (leader)
  uint32_t tmem_base;
  int err;
};

__device__ __noinline__ bool q_wait_slow(uint64_t* bar, uint32_t parity, QSmem& sm, bool cluster) {
  uint64_t deadline = 0;
  for (uint32_t spin = 0;; ++spin) {
    if (cluster ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity)) return true;
    if ((spin & 63) == 63) {
      if (*reinterpret_cast<volatile int*>(&sm.err)) return false;
      const uint64_t now = globaltimer_ns();
      if (deadline == 0) deadline = now + kQBoundNs;
      else if (now > deadline) return false;
    }
  }
}
__device__ __forceinline__ bool q_wait(uint64_t* bar, uint32_t parity, QSmem& sm) {
  return mbar_try_wait(bar, parity) || q_wait_slow(bar, parity, sm, false);
}

// Stops both CTAs of the pair.
__device__ __noinline__ void q_fail(QSmem& sm, const QArgs& a, int detail) {
  if (atomicExch(&sm.err, 1) == 0) {
    st_shared_cluster_u32(mapa_shared(smem_u32(&sm.err), cluster_ctarank() ^ 1u), 1u);
    if (a.status_host)
      *reinterpret_cast<volatile int32_t*>(a.status_host) = int32_t(status_word(kTimeout, kSitePipe, detail));
  }
}

// Row offsets and row-tile prefix of the experts.
struct QSched {
  int* off;   // [E + 1]
  int* tpre;  // [E + 1]
  int E, FT, kb;
};

struct QTile {
  int e, f, r0, rows, n;  // expert, channel tile, first row, rows, MMA N
};

__device__ __forceinline__ QTile q_tile(const QSched& s, int t) {
  const int x = t / s.FT;
  int lo = 0, hi = s.E;  // largest e with tpre[e] <= x
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s.tpre[mid] <= x) lo = mid;
    else hi = mid;
  }
  QTile q;
  q.e = lo;
  const int nrt = s.tpre[lo + 1] - s.tpre[lo], local = t - s.tpre[lo] * s.FT;
  q.f = local / nrt;
  const int r = local - q.f * nrt, n = s.off[lo + 1] - s.off[lo];
  const int tr = ((n + nrt - 1) / nrt + 31) / 32 * 32;  // rows per tile, even among an expert's tiles
  q.r0 = s.off[lo] + r * tr;
  q.rows = min(tr, n - r * tr);
  q.n = (q.rows + 31) / 32 * 32;
  return q;
}

// The runs over K that a pair does, in order: whole tiles t0, t0 + step, ...
// or (split) the tiles of a contiguous share of units.
struct QWalk {
  bool split;
  int tile, step, tiles;  // whole tiles
  int u, hi, kb;          // split
  int k0, k1;             // current run
  __device__ __forceinline__ QWalk(const QSched& s, bool split_, int tiles_, int pair, int pairs) {
    split = split_;
    tiles = tiles_;
    kb = s.kb;
    k0 = 0;
    k1 = kb;
    u = hi = 0;
    if (split) {
      const uint32_t units = uint32_t(tiles_) * uint32_t(kb);
      const uint32_t g = min(uint32_t(pairs), units);
      u = uint32_t(pair) < g ? int(uint64_t(units) * pair / g) : 0;
      hi = uint32_t(pair) < g ? int(uint64_t(units) * (pair + 1) / g) : 0;
      set();
    } else {
      tile = pair;
      step = pairs;
    }
  }
  __device__ __forceinline__ void set() {
    tile = u / kb;
    k0 = u - tile * kb;
    k1 = min(kb, k0 + hi - u);
  }
  __device__ __forceinline__ bool more() const { return split ? u < hi : tile < tiles; }
  __device__ __forceinline__ void next() {
    if (split) {
      u += k1 - k0;
      set();
    } else {
      tile += step;
    }
  }
  __device__ __forceinline__ bool whole() const { return k0 == 0 && k1 == kb; }
};

struct QRing {
  int st;
  uint32_t ph;
  __device__ __forceinline__ void next(int n) {
    if (++st == n) {
      st = 0;
      ph ^= 1;
    }
  }
};

__device__ __forceinline__ void q_store4(const QArgs& a, int64_t row, int f, float v0, float v1, float v2, float v3) {
  const int64_t at = row * a.F + f;
  if (a.out_f32) {
    *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = make_float4(v0, v1, v2, v3);
  } else {
    __nv_bfloat162 o[2] = {__floats2bfloat162_rn(v0, v1), __floats2bfloat162_rn(v2, v3)};
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + at) = *reinterpret_cast<uint2*>(o);
  }
}

// Four neighbouring scales (they are aligned like floats only).
__device__ __forceinline__ float4 scales4(const float* p) { return make_float4(p[0], p[1], p[2], p[3]); }

// The quotient within 2 steps of 2^-24 (0 where exp(-g) overflows).  Both
// sides are taken by 8: the fast division gives 0 for every divisor above
// 2^126, gates under -87.3, whose silu a large u brings back.
__device__ __forceinline__ float silu_mul(float g, float u) {
  return __fdividef(0.125f * g, fmaf(0.125f, expf(-g), 0.125f)) * u;
}

template <bool GLU, bool SPLIT>
__global__ void __launch_bounds__(kQThreads, 1)
    w8a8_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ QRowMaps tm_x,
                const __grid_constant__ QArgs a) {
  extern __shared__ unsigned char q_dyn[];
  unsigned char* stage = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(q_dyn) + 1023) & ~uintptr_t(1023));
  float* xbuf = reinterpret_cast<float*>(stage + kQStages * kQStageBytes);
  QSmem& sm = *reinterpret_cast<QSmem*>(reinterpret_cast<unsigned char*>(xbuf) + kQXBytes);
  QSched s;
  s.off = reinterpret_cast<int*>(&sm + 1);
  s.tpre = s.off + a.E + 1;
  s.E = a.E;
  s.FT = GLU ? (a.F + 127) / 128 : (a.N + 255) / 256;
  s.kb = (a.K + kQKb - 1) / kQKb;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t crank = cluster_ctarank();
  const bool leader = crank == 0;
  const int pair = int(blockIdx.x >> 1), pairs = int(gridDim.x >> 1);

  if (threadIdx.x == 0) {
    for (int i = 0; i < kQStages; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.tfull[i], 1);
      mbar_init(&sm.tempty[i], 2 * kQEpiWarps);
    }
    mbar_init(&sm.drain, 1);
    sm.fills = sm.used = 0;
    sm.err = 0;
    fence_mbar_init();
    prefetch_tensormap(&tm_w);
  }
  // Offsets and tile prefix: counts that would pass the last row are cut.
  if (warp == 2) {
    int64_t off = 0;
    int tp = 0;
    for (int e0 = 0; e0 < a.E; e0 += 32) {
      const int e = e0 + lane;
      int64_t c = 0;
      if (e < a.E) c = a.counts ? max(a.counts[e], 0) : a.rows;
      int64_t pre = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, pre, o);
        if (lane >= o) pre += v;
      }
      const int64_t end = min(off + pre, a.rows), begin = min(off + pre - c, a.rows);
      int nt = int((end - begin + kQTileRows - 1) / kQTileRows), tpre = nt;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, tpre, o);
        if (lane >= o) tpre += v;
      }
      if (e < a.E) {
        s.off[e] = int(begin);
        s.tpre[e] = tp + tpre - nt;
        if (e == a.E - 1) {
          s.off[a.E] = int(end);
          s.tpre[a.E] = tp + tpre;
        }
      }
      off += __shfl_sync(0xffffffffu, pre, 31);
      tp += __shfl_sync(0xffffffffu, tpre, 31);
    }
  }
  cluster_sync();  // the peer's barriers exist before any remote arrive
  if (warp == 1) {
    __syncwarp();
    tmem_alloc_pair(&sm.tmem_base, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, sm.tmem_base, 0);
  const int tiles = s.tpre[a.E] * s.FT;
  // Splitting saves the last round's idle pairs and costs a barrier and the
  // parts' way through memory: about 12 stages, and one for every 8 rows of a
  // tile.  (The host launches the form with a grid barrier where the rows
  // alone leave it open; ragged experts may make enough tiles all the same.)
  bool split = false;
  if (SPLIT && tiles > 0 && tiles < kQWaves * pairs) {
    const int rounds = (tiles + pairs - 1) / pairs, mean = s.off[a.E] / s.tpre[a.E];
    split = rounds * s.kb > tiles * s.kb / pairs + 12 + mean / 8;
  }

  if (warp == 0 && lane == 0) {
    // ---- loads: each CTA its 128 channels and half of the tile's rows, all
    // onto the leader's barrier
    QRing r = {0, 0};
    uint32_t fills = 0;
    const uint32_t bar0 = mapa_shared(smem_u32(&sm.full[0]), 0);
    bool stop = false;
    for (QWalk w(s, split, tiles, pair, pairs); w.more() && !stop; w.next()) {
      const QTile t = q_tile(s, w.tile);
      const int half = t.n / 2, bm = half <= 16 ? 0 : half <= 32 ? 1 : half <= 64 ? 2 : 3;
      const uint32_t tx = 2 * (kQABytes + (16u << bm) * kQKb);
      const int row = t.r0 + int(crank) * half;
      for (int k = w.k0; k < w.k1; ++k) {
        if (!q_wait(&sm.empty[r.st], r.ph ^ 1, sm)) {
          q_fail(sm, a, 1);
          stop = true;
          break;
        }
        unsigned char* dst = stage + uint32_t(r.st) * kQStageBytes;
        const uint32_t bar = bar0 + uint32_t(r.st) * sizeof(uint64_t);
        if (leader) mbar_arrive_expect_tx(&sm.full[r.st], tx);
        if constexpr (GLU) {
          const int f = t.f * 128 + int(crank) * 64;
          tma_load_3d_pair(&tm_w, bar, dst, k * kQKb, f, t.e);
          tma_load_3d_pair(&tm_w, bar, dst + kQABytes / 2, k * kQKb, a.F + f, t.e);
        } else {
          tma_load_3d_pair(&tm_w, bar, dst, k * kQKb, t.f * 256 + int(crank) * 128, t.e);
        }
        tma_load_2d_pair(&tm_x.m[bm], bar, dst + kQABytes, k * kQKb, row);
        ++fills;
        r.next(kQStages);
      }
    }
    sm.fills = fills;
  } else if (warp == 1 && leader) {
    // ---- MMA.  The whole warp walks the list, so that what an instruction
    // needs (descriptors, sums of constants) is known to be the same in all
    // lanes and stays in uniform registers; one lane issues.
    QRing r = {0, 0}, acc = {0, 0};
    bool stop = false;
    uint32_t used = 0;  // stages multiplied
    const uint64_t desc0 = smem_desc_sw128(smem_u32(stage), 16, 1024);
    const bool issuer = elect_one();
    for (QWalk w(s, split, tiles, pair, pairs); w.more() && !stop; w.next()) {
      const QTile t = q_tile(s, w.tile);
      const uint32_t idesc = make_idesc_i8(256, uint32_t(__shfl_sync(0xffffffffu, t.n, 0)));
      bool ok = mbar_try_wait_cluster(&sm.tempty[acc.st], acc.ph ^ 1) ||
                q_wait_slow(&sm.tempty[acc.st], acc.ph ^ 1, sm, true);
      if (!__all_sync(0xffffffffu, ok)) {
        q_fail(sm, a, 2);
        break;
      }
      tc_fence_after();
      const uint32_t d = tmem + uint32_t(acc.st) * 256;
      const int n = __shfl_sync(0xffffffffu, w.k1 - w.k0, 0);
      for (int k = 0; k < n; ++k) {
        if (!__all_sync(0xffffffffu, q_wait(&sm.full[r.st], r.ph, sm))) {
          q_fail(sm, a, 3);
          stop = true;
          break;
        }
        const uint64_t da = desc0 + uint32_t(r.st) * (kQStageBytes >> 4), db = da + (kQABytes >> 4);
        if (issuer) {
#pragma unroll
          for (int kk = 0; kk < kQKb / 32; ++kk)
            tc_mma_i8_pair(d, da + kk * 2, db + kk * 2, idesc, (k != 0 || kk != 0) ? 1u : 0u);
          tc_commit_pair_mc(&sm.empty[r.st], 0x3);
        }
        __syncwarp();
        ++used;
        r.next(kQStages);
      }
      if (stop) break;
      if (issuer) tc_commit_pair_mc(&sm.tfull[acc.st], 0x3);
      __syncwarp();
      acc.next(2);
    }
    if (issuer) sm.used = used;
  } else if (warp >= kQEpi0) {
    // ---- epilogue: chunks of 32 rows, even ones by the first four warps
    QRing acc = {0, 0};
    const int quarter = warp & 3, sub = (warp - kQEpi0) >> 2;
    const uint32_t tempty0 = mapa_shared(smem_u32(&sm.tempty[0]), 0);
    float* mine = xbuf + (sub * 4 + quarter) * kQXFloats;
    const float* theirs = xbuf + (sub * 4 + (quarter ^ 2)) * kQXFloats;
    float* xrow = xbuf + kQEpiWarps * kQXFloats + (warp - kQEpi0) * 32;
    const int bar_id = 1 + sub * 2 + (quarter & 1);  // this warp and its gate or up partner
    for (QWalk w(s, split, tiles, pair, pairs); w.more(); w.next()) {
      const QTile t = q_tile(s, w.tile);
      // This lane's channel: within the CTA's 128, then of the output.
      const int fl = quarter * 32 + lane;
      const bool up = GLU && quarter >= 2;
      const int f0 = GLU ? t.f * 128 + int(crank) * 64 + (quarter & 1) * 32 : t.f * 256 + int(crank) * 128 + quarter * 32;
      const int f = f0 + lane;
      const float sw = f < a.F ? a.ws[int64_t(t.e) * a.N + (up ? a.F : 0) + f] : 0.f;
      bool ok = q_wait(&sm.tfull[acc.st], acc.ph, sm);
      if constexpr (GLU) ok = named_bar_and(bar_id, 64, ok);
      if (!ok) {
        q_fail(sm, a, 4);
        break;
      }
      tc_fence_after();
      const uint32_t d = tmem + uint32_t(acc.st) * 256 + (uint32_t(quarter * 32) << 16);
      int32_t* ps = a.part + (size_t(pair) * 2 + (w.k0 == 0 ? 1 : 0)) * kQSlotInts + crank * 128 + fl;
      const bool whole = w.whole();
      // The next chunk's sums are on their way while one is finished.
      uint32_t v[32];
      if (sub * 32 < t.rows) tmem_ld_32x32b_x32(d + uint32_t(sub * 32), v);
#pragma unroll 1
      for (int jc = sub; jc * 32 < t.rows; jc += 2) {
        const int left = t.rows - jc * 32;
        const int64_t row = t.r0 + jc * 32;
        tmem_ld_wait();
        if (!whole) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (i < left) ps[(jc * 32 + i) * 256] = int32_t(v[i]);
          if ((jc + 2) * 32 < t.rows) tmem_ld_32x32b_x32(d + uint32_t((jc + 2) * 32), v);
          continue;
        }
        __syncwarp();
        xrow[lane] = lane < left ? a.xs[row + lane] : 0.f;
        __syncwarp();
        float z[32];
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 x4 = *reinterpret_cast<const float4*>(xrow + i);
          z[i] = float(int32_t(v[i])) * x4.x * sw;
          z[i + 1] = float(int32_t(v[i + 1])) * x4.y * sw;
          z[i + 2] = float(int32_t(v[i + 2])) * x4.z * sw;
          z[i + 3] = float(int32_t(v[i + 3])) * x4.w * sw;
        }
        if ((jc + 2) * 32 < t.rows) tmem_ld_32x32b_x32(d + uint32_t((jc + 2) * 32), v);
        if constexpr (GLU) {
          // The gate warp finishes rows 0..15 of the chunk, the up warp rows
          // 16..31: each hands the other half over, 16 values a lane at a
          // stride of 20 (no bank conflicts in 16-byte accesses).
          auto finish = [&](auto is_up) {
            constexpr bool kUp = decltype(is_up)::value;
            constexpr int kMine = kUp ? 16 : 0, kTheirs = 16 - kMine;
            named_bar_sync(bar_id, 64);  // the last chunk's have been read
#pragma unroll
            for (int i = 0; i < 16; i += 4)
              *reinterpret_cast<float4*>(mine + lane * 20 + i) =
                  make_float4(z[kTheirs + i], z[kTheirs + i + 1], z[kTheirs + i + 2], z[kTheirs + i + 3]);
            named_bar_sync(bar_id, 64);
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
              const float4 o = *reinterpret_cast<const float4*>(theirs + lane * 20 + i);
              const float ov[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
              for (int j = 0; j < 4; ++j)
                z[kMine + i + j] = kUp ? silu_mul(ov[j], z[kMine + i + j]) : silu_mul(z[kMine + i + j], ov[j]);
            }
            const int64_t at = (row + kMine) * a.F + f;
            const int n = f < a.F ? left - kMine : 0;
            if (a.out_f32) {
              float* o = static_cast<float*>(a.out) + at;
#pragma unroll
              for (int i = 0; i < 16; ++i, o += a.F)
                if (i < n) *o = z[kMine + i];
            } else {
              __nv_bfloat16* o = static_cast<__nv_bfloat16*>(a.out) + at;
#pragma unroll
              for (int i = 0; i < 16; ++i, o += a.F)
                if (i < n) *o = __float2bfloat16_rn(z[kMine + i]);
            }
          };
          if (up) finish(std::true_type{});
          else finish(std::false_type{});
        } else if (a.out_f32) {
          float* o = static_cast<float*>(a.out) + row * a.F + f;
          const int n = f < a.F ? left : 0;
#pragma unroll
          for (int i = 0; i < 32; ++i, o += a.F)
            if (i < n) *o = z[i];
        } else {
          // bf16, two rows to a word, through shared memory: a lane then
          // holds eight channels of two rows, 16 bytes each.
          uint32_t* words = reinterpret_cast<uint32_t*>(mine);
#pragma unroll
          for (int p = 0; p < 16; ++p) {
            const __nv_bfloat162 b2 = __floats2bfloat162_rn(z[2 * p], z[2 * p + 1]);
            words[p * 32 + lane] = *reinterpret_cast<const uint32_t*>(&b2);
          }
          __syncwarp();
          __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out);
#pragma unroll
          for (int step = 0; step < 2; ++step) {
            const int p = (lane >> 2) + step * 8, c = (lane & 3) * 8;
            const uint4 lo = *reinterpret_cast<const uint4*>(words + p * 32 + c);
            const uint4 hi = *reinterpret_cast<const uint4*>(words + p * 32 + c + 4);
            if (f0 + c >= a.F) continue;
            __nv_bfloat16* o = out + (row + 2 * p) * a.F + f0 + c;
            if (2 * p < left)
              *reinterpret_cast<uint4*>(o) = make_uint4(__byte_perm(lo.x, lo.y, 0x5410), __byte_perm(lo.z, lo.w, 0x5410),
                                                        __byte_perm(hi.x, hi.y, 0x5410), __byte_perm(hi.z, hi.w, 0x5410));
            if (2 * p + 1 < left)
              *reinterpret_cast<uint4*>(o + a.F) =
                  make_uint4(__byte_perm(lo.x, lo.y, 0x7632), __byte_perm(lo.z, lo.w, 0x7632),
                             __byte_perm(hi.x, hi.y, 0x7632), __byte_perm(hi.z, hi.w, 0x7632));
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(tempty0 + uint32_t(acc.st) * sizeof(uint64_t));
      acc.next(2);
    }
  }
  __syncwarp();

  if constexpr (SPLIT) {
    if (split) {
      cg::this_grid().sync();
      // ---- the tile that this pair started and others went on with: four
      // channels a thread, every part's loads in flight together
      const uint32_t units = uint32_t(tiles) * uint32_t(s.kb);
      const uint32_t g = min(uint32_t(pairs), units);
      const uint32_t lo = uint64_t(units) * pair / g, hi = uint64_t(units) * (pair + 1) / g;
      const uint32_t tile = (hi - 1) / s.kb, first = tile * s.kb, end = first + s.kb;
      if (uint32_t(pair) < g && first >= lo && hi < end) {
        const int c1 = int((uint64_t(end) * g - 1) / units);
        const QTile t = q_tile(s, int(tile));
        const int4* part = reinterpret_cast<const int4*>(a.part);
        auto sum4 = [&](int at) {  // of int4 `at` of the slots
          int4 z = __ldcg(part + (size_t(pair) * 2 + 1) * (kQSlotInts / 4) + at);
#pragma unroll 4
          for (int p = pair + 1; p <= c1; ++p) {
            const int4 x = __ldcg(part + size_t(p) * 2 * (kQSlotInts / 4) + at);
            z.x += x.x, z.y += x.y, z.z += x.z, z.w += x.w;
          }
          return z;
        };
        // Channels of a row: 64 int4 (both CTAs'); with SwiGLU the first 16
        // of each CTA's 32 are gate, the others up.
        constexpr int kPer = GLU ? 32 : 64;
        const int total = t.rows * kPer;
#pragma unroll 4
        for (int i = int(crank) * kQThreads + int(threadIdx.x); i < total; i += 2 * kQThreads) {
          const int j = i / kPer, c = i % kPer;
          const float xv = a.xs[t.r0 + j];
          const float* sw = a.ws + int64_t(t.e) * a.N;
          if constexpr (GLU) {
            const int at = j * 64 + (c >> 4) * 32 + (c & 15), f = t.f * 128 + c * 4;
            const int4 g4 = sum4(at), u4 = sum4(at + 16);
            if (f < a.F) {
              const float4 sg = scales4(sw + f), su = scales4(sw + a.F + f);
              q_store4(a, t.r0 + j, f, silu_mul(float(g4.x) * xv * sg.x, float(u4.x) * xv * su.x),
                       silu_mul(float(g4.y) * xv * sg.y, float(u4.y) * xv * su.y),
                       silu_mul(float(g4.z) * xv * sg.z, float(u4.z) * xv * su.z),
                       silu_mul(float(g4.w) * xv * sg.w, float(u4.w) * xv * su.w));
            }
          } else {
            const int f = t.f * 256 + c * 4;
            const int4 z = sum4(j * 64 + c);
            if (f < a.N) {
              const float4 s4 = scales4(sw + f);
              q_store4(a, t.r0 + j, f, float(z.x) * xv * s4.x, float(z.y) * xv * s4.y, float(z.z) * xv * s4.z,
                       float(z.w) * xv * s4.w);
            }
          }
        }
      }
    }
  }

  // ---- teardown.  After an abort: time for the peer's loads onto the
  // leader's barriers, then every load and MMA still under way, all bounded.
  __syncthreads();
  const bool failed = *reinterpret_cast<volatile int*>(&sm.err) != 0;
  if (failed && threadIdx.x == 0) {
    const uint64_t until = globaltimer_ns() + 200000ull;
    while (globaltimer_ns() < until) {
    }
  }
  cluster_sync();
  if (leader && threadIdx.x == 0) {
    for (uint32_t i = sm.used; i < sm.fills; ++i) {  // loaded, never multiplied
      const uint64_t until = globaltimer_ns() + kQBoundNs;
      while (!mbar_try_wait(&sm.full[i % kQStages], (i / kQStages) & 1) && globaltimer_ns() < until) {
      }
    }
  }
  if (leader && warp == 1 && elect_one()) {  // (the lane that issued the MMAs)
    tc_commit_pair(&sm.drain);
    const uint64_t until = globaltimer_ns() + kQBoundNs;
    while (!mbar_try_wait(&sm.drain, 0) && globaltimer_ns() < until) {
    }
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc_pair(tmem, 512);
  }
  cluster_sync();  // neither CTA leaves while its peer may still address it
}

// ---------------------------------------------------------------- a handful of rows
// Up to kRwMaxRows rows (a decode step's): no tile to fill, so a warp takes a
// channel (its gate and its up channel with SwiGLU) of up to four rows of an
// expert, streams the channel's K contiguous bytes once, 16 per lane, against
// the rows in shared memory with 4-way 8-bit dot products, and adds its lanes
// up.  No partial sums, barriers or tensor maps: the launch and one pass over
// the weights (one row, 7168 x 4096: 16.4 us with the tiles above and a
// launch for the quantisation, 7.4 us).  Rows given in bf16 or fp32 are
// quantised by every CTA for itself, behind the first loads of weights, as
// far as that takes less than a launch (kRwMaxFresh values).
//
// The gated layer of a few tokens is two such launches: gate and up channels
// of every (token, expert) row, then (SUM) the down channels, a warp taking
// one of all experts and adding their rows, weighted, to y.
constexpr int kRwThreads = 512;
constexpr int kRwMaxRows = 32;
constexpr int kRwMaxFresh = 32768;          // values quantised by every CTA,
constexpr int kRwMaxFreshRows = 16;         // in rows of at least a warp each
constexpr int kRwRows = 4;                  // rows of a channel's pass
constexpr uint32_t kRwMaxSmem = 96 * 1024;  // of rows: two CTAs per SM

struct RwArgs {
  int E, K, N, F;
  int rows;               // rows in memory
  const int32_t* counts;  // [E] rows per expert, in order (null: all rows one expert's), unless ids
  const int8_t* xq;
  const float* xs;
  const void* x;          // or null: xq and xs
  int x_f32;
  const int32_t* perm;
  const int32_t* live;
  const int8_t* wq;
  const float* ws;
  void* out;
  int out_f32;
  // A layer of T tokens (ids != null).
  const void* ids;
  int ids64, first, T, topk;
  const void* vals;       // SUM
  int vals_bf16;
};

struct RwSmem {
  float scale[kRwMaxRows];
  uint32_t top[kRwThreads / 32];
  int src[kRwMaxRows];     // a row's place in memory
  int tok[kRwMaxRows];
  float val[kRwMaxRows];
  int e[kRwMaxRows], r0[kRwMaxRows], n[kRwMaxRows];  // an expert's rows, four at a time
  int rows, chunks;
};

__device__ __forceinline__ int dot16(uint4 a, uint4 b, int c) {
  c = __dp4a(int(a.x), int(b.x), c);
  c = __dp4a(int(a.y), int(b.y), c);
  c = __dp4a(int(a.z), int(b.z), c);
  return __dp4a(int(a.w), int(b.w), c);
}

// The loads of one round: kRwLoads vectors of 16 bytes per lane in all.
constexpr int kRwLoads = 4;
template <bool DUAL>
__device__ __forceinline__ void rw_load(const uint4* w, const uint4* w2, int v0, int V, int lane,
                                        uint4 (&buf)[kRwLoads]) {
  constexpr int U = DUAL ? kRwLoads / 2 : kRwLoads;
#pragma unroll
  for (int j = 0; j < U; ++j) {
    const int v = v0 + j * 32 + lane;
    const bool in = v < V;
    buf[j] = in ? ld_nc_v4(w + v) : make_uint4(0, 0, 0, 0);
    if constexpr (DUAL) buf[U + j] = in ? ld_nc_v4(w2 + v) : make_uint4(0, 0, 0, 0);
  }
}

// One channel's (DUAL: two channels') sums over K for the rows of chunk c.
// buf holds the first round's loads and leaves with those of the next channel
// (null: none).
template <bool DUAL, int NR>
__device__ __forceinline__ void rw_channel(const RwSmem& sm, const uint4* rows, int V, int c, const uint4* w,
                                           const uint4* w2, const uint4* nw, const uint4* nw2,
                                           uint4 (&buf)[kRwLoads], int (&s)[NR], int (&s2)[NR]) {
  constexpr int U = DUAL ? kRwLoads / 2 : kRwLoads;
  const int lane = threadIdx.x & 31, r0 = sm.r0[c], last = sm.n[c] - 1;  // NR > n: the last row again
  const uint4* row[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    row[r] = rows + sm.src[r0 + min(r, last)] * V;
    s[r] = s2[r] = 0;
  }
#pragma unroll 1
  for (int v0 = 0; v0 < V; v0 += 32 * U) {
    uint4 next[kRwLoads];
    const bool end = v0 + 32 * U >= V;
    rw_load<DUAL>(end ? nw : w, end ? nw2 : w2, end ? 0 : v0 + 32 * U, end && nw == nullptr ? 0 : V, lane, next);
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int v = min(v0 + j * 32 + lane, V - 1);  // (past the end the weights are zeros)
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const uint4 x = row[r][v];
        s[r] = dot16(buf[j], x, s[r]);
        if constexpr (DUAL) s2[r] = dot16(buf[U + j], x, s2[r]);
      }
    }
#pragma unroll
    for (int j = 0; j < kRwLoads; ++j) buf[j] = next[j];
  }
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    s[r] = __reduce_add_sync(0xffffffffu, s[r]);
    if constexpr (DUAL) s2[r] = __reduce_add_sync(0xffffffffu, s2[r]);
  }
}

template <typename In>
__device__ __forceinline__ void rw_quantize(const RwArgs& a, RwSmem& sm, unsigned char* rows, int count) {
  // The warps in equal groups, one for each row.
  int per = kRwThreads;
  while (per > 32 && per * count > kRwThreads) per /= 2;
  const int r = int(threadIdx.x) / per, c = int(threadIdx.x) % per, groups = a.K / 8;
  const int live = a.live ? min(max(*a.live, 0), count) : count;
  const bool on = r < live;
  const In* src = static_cast<const In*>(a.x) + int64_t(on ? (a.perm ? a.perm[r] : r) : 0) * a.K;
  RowTop<In> seen;
#pragma unroll 4
  for (int g = c; g < groups && on; g += per) {
    Raw8<In> v;
    v.load(src + g * 8);
    v.top(seen);
  }
  uint32_t top = __reduce_max_sync(0xffffffffu, seen.bits());
  if ((threadIdx.x & 31) == 0) sm.top[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll 4
  for (int w = 0; w < per / 32; ++w) top = max(top, sm.top[r * (per / 32) + w]);
  const RowScale rs(top);
  if (c == 0 && on) sm.scale[r] = rs.scale;
#pragma unroll 1
  for (int g = c; g < groups && on; g += per) {
    Raw8<In> raw;
    raw.load(src + g * 8);
    float v[8];
    raw.values(v);
    *reinterpret_cast<uint2*>(rows + r * a.K + g * 8) = rs.round8(v);
  }
}

// The table of rows and chunks, by one warp, from counts per expert.
__device__ __forceinline__ void rw_table_counts(const RwArgs& a, RwSmem& sm, int lane) {
  // Experts with rows, in order; counts that would pass the last row are cut.
  int row = 0, chunks = 0;
#pragma unroll 1
  for (int e0 = 0; e0 < a.E && row < a.rows; e0 += 32) {
    const int e = e0 + lane;
    int c = e < a.E ? (a.counts ? min(max(a.counts[e], 0), a.rows) : a.rows) : 0;
    int pre = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, pre, o);
      if (lane >= o) pre += v;
    }
    const int begin = min(row + pre - c, a.rows);
    c = min(row + pre, a.rows) - begin;
    const int mine = (c + kRwRows - 1) / kRwRows;
    int at = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, at, o);
      if (lane >= o) at += v;
    }
    for (int i = 0; i < mine; ++i) {
      const int k = chunks + at - mine + i;
      sm.e[k] = e;
      sm.r0[k] = begin + i * kRwRows;
      sm.n[k] = min(kRwRows, c - i * kRwRows);
    }
    row = min(row + __shfl_sync(0xffffffffu, pre, 31), a.rows);
    chunks += __shfl_sync(0xffffffffu, at, 31);
  }
  if (lane < a.rows) sm.src[lane] = lane;
  if (lane == 0) {
    sm.chunks = chunks;
    sm.rows = a.rows;
  }
}

// The same from a layer's ids, sorted by expert, then token (T * topk <= 32
// rows; an id repeated within a token's row counts once).
template <bool SUM>
__device__ __forceinline__ void rw_table_ids(const RwArgs& a, RwSmem& sm, int lane) {
  const int n = a.T * a.topk, t = lane / a.topk;
  long long e = -1;
  if (lane < n)
    e = (a.ids64 ? static_cast<const long long*>(a.ids)[lane] : static_cast<const int32_t*>(a.ids)[lane]) -
        (long long)a.first;
  const uint32_t none = 0xffffffffu;
  const uint32_t key = lane < n && e >= 0 && e < a.E ? uint32_t(e) * 32 + uint32_t(t) : none;
  const uint32_t same = __match_any_sync(0xffffffffu, key);
  const bool on = key != none && (same & ((1u << lane) - 1)) == 0;
  const uint32_t expert = on ? key >> 5 : none;
  const uint32_t peers = __match_any_sync(0xffffffffu, expert);
  // A row's rank among its expert's is that of its lane (tokens ascend with
  // the lane); every fourth opens a chunk.
  const int rank = __popc(peers & ((1u << lane) - 1));
  const bool head = on && rank % kRwRows == 0;
  const uint32_t hkey = head ? (expert * 32 + uint32_t(lane)) : none;
  int row = 0, at = 0;
#pragma unroll 4
  for (int j = 0; j < kRwMaxRows; ++j) {
    const uint32_t kj = __shfl_sync(0xffffffffu, on ? key : none, j);
    const uint32_t hj = __shfl_sync(0xffffffffu, hkey, j);
    row += on && kj < key;
    at += head && hj < hkey;
  }
  if (on) {
    sm.src[row] = SUM ? row : t;
    sm.tok[row] = t;
    if constexpr (SUM)
      sm.val[row] = a.vals_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(a.vals)[lane])
                                : static_cast<const float*>(a.vals)[lane];
  }
  if (head) {
    sm.e[at] = int(expert);
    sm.r0[at] = row;
    sm.n[at] = min(kRwRows, __popc(peers) - rank);
  }
  const uint32_t ons = __ballot_sync(0xffffffffu, on), heads = __ballot_sync(0xffffffffu, head);
  if (lane == 0) {
    sm.rows = SUM ? __popc(ons) : a.T;
    sm.chunks = __popc(heads);
  }
}

// PAIR: a warp takes two neighbouring channels at a time (two up to a row of
// the table; F even), so that a row's values are read from shared memory once
// for both.
template <bool GLU, bool SUM, bool PAIR>
__global__ void __launch_bounds__(kRwThreads, 2) w8a8_rows_kernel(const __grid_constant__ RwArgs a) {
  constexpr bool DUAL = GLU || PAIR;
  extern __shared__ __align__(16) unsigned char rw_rows[];
  __shared__ RwSmem sm;
  const int warp = int(threadIdx.x) >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    if (a.ids != nullptr) rw_table_ids<SUM>(a, sm, lane);
    else rw_table_counts(a, sm, lane);
  }
  __syncthreads();
  const int V = a.K / 16, warps = int(gridDim.x) * (kRwThreads / 32), chunks = sm.chunks;
  const int cols = PAIR ? a.F / 2 : a.F;
  // This warp's (chunk, channel) pairs: chunk by chunk, or (SUM) every chunk
  // of a channel, then the next channel.
  int c = 0, f = int(blockIdx.x) * (kRwThreads / 32) + warp;
  auto settle = [&](int& cc, int& ff) {  // whether the pair exists; channels past a chunk's last go to the next chunk
    if constexpr (!SUM) {
      while (ff >= cols && cc < chunks) {
        ff -= cols;
        ++cc;
      }
    }
    return cc < chunks && ff < cols;
  };
  auto weights = [&](int cc, int ff) {
    return reinterpret_cast<const uint4*>(a.wq) + (int64_t(sm.e[cc]) * a.N + (PAIR ? 2 * ff : ff)) * V;
  };
  uint4 buf[kRwLoads];
  bool more = settle(c, f);
  const uint4* w = more ? weights(c, f) : nullptr;
  const int64_t second = GLU ? int64_t(a.F) * V : V;  // to the up channel, or the pair's other one
  if (more) rw_load<DUAL>(w, w + second, 0, V, lane, buf);
  if (a.x != nullptr) {
    if (a.x_f32) rw_quantize<float>(a, sm, rw_rows, sm.rows);
    else rw_quantize<__nv_bfloat16>(a, sm, rw_rows, sm.rows);
  } else {
    for (int i = threadIdx.x; i < a.rows * V; i += kRwThreads)
      reinterpret_cast<uint4*>(rw_rows)[i] = reinterpret_cast<const uint4*>(a.xq)[i];
    if (int(threadIdx.x) < a.rows) sm.scale[threadIdx.x] = a.xs[threadIdx.x];
  }
  __syncthreads();
  const uint4* rows = reinterpret_cast<const uint4*>(rw_rows);
  auto store = [&](int row, int ff, float v, float v2) {  // one value, or a pair's two
    const int64_t at = int64_t(row) * a.F + (PAIR ? 2 * ff : ff);
    if (a.out_f32) {
      float* o = static_cast<float*>(a.out) + at;
      if constexpr (PAIR) *reinterpret_cast<float2*>(o) = make_float2(v, v2);
      else *o = v;
    } else {
      __nv_bfloat16* o = static_cast<__nv_bfloat16*>(a.out) + at;
      if constexpr (PAIR) *reinterpret_cast<__nv_bfloat162*>(o) = __floats2bfloat162_rn(v, v2);
      else *o = __float2bfloat16_rn(v);
    }
  };
  float y = 0.f, y2 = 0.f;  // SUM: lane t's token
  if (SUM && chunks == 0) {  // no token has an expert here
    for (; f < cols; f += warps)
      if (lane < a.T) store(lane, f, 0.f, 0.f);
  }
#pragma unroll 1
  while (more) {
    int nc = c, nf = f;
    if (SUM && c + 1 < chunks) {
      ++nc;
    } else {
      nf += warps;
      if (SUM) nc = 0;
    }
    more = settle(nc, nf);
    const uint4* nw = more ? weights(nc, nf) : nullptr;
    const float* sw = a.ws + int64_t(sm.e[c]) * a.N + (PAIR ? 2 * f : f);
    const float g = sw[0], u = DUAL ? sw[GLU ? a.F : 1] : 0.f;
    auto channel = [&](auto nr) {
      constexpr int NR = decltype(nr)::value;
      int s[NR], s2[NR];
      rw_channel<DUAL, NR>(sm, rows, V, c, w, w + second, nw, nw + second, buf, s, s2);
      const int r0 = sm.r0[c], n = sm.n[c];
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        if (r >= n) break;
        const float x = sm.scale[sm.src[r0 + r]], z = float(s[r]) * x * g, z2 = float(s2[r]) * x * u;
        if constexpr (SUM) {
          if (lane == sm.tok[r0 + r]) {
            y = fmaf(sm.val[r0 + r], z, y);
            if constexpr (PAIR) y2 = fmaf(sm.val[r0 + r], z2, y2);
          }
        } else if (lane == r) {
          store(r0 + r, f, GLU ? silu_mul(z, z2) : z, z2);
        }
      }
    };
    const int n = sm.n[c];
    if (n == 1) channel(std::integral_constant<int, 1>{});
    else if (n == 2) channel(std::integral_constant<int, 2>{});
    else channel(std::integral_constant<int, 4>{});
    if (SUM && nf != f) {
      if (lane < a.T) store(lane, f, y, y2);
      y = y2 = 0.f;
    }
    c = nc;
    f = nf;
    w = nw;
  }
}

// ---------------------------------------------------------------- quantisation
// TPR threads per row, each VPT groups of eight values in registers; rows
// longer than that are read again for the rounding.
template <typename In, int VPT, int THREADS>
__global__ void __launch_bounds__(THREADS)
    quant_rows_kernel(const In* __restrict__ x, int64_t rows, int K, const int32_t* __restrict__ perm,
                      const int32_t* __restrict__ live_rows, int tpr, int8_t* __restrict__ q,
                      float* __restrict__ scale) {
  __shared__ uint32_t top_s[THREADS / 32];
  const int per = THREADS / tpr, lr = threadIdx.x / tpr, c = threadIdx.x % tpr;
  const int64_t live = live_rows ? min(int64_t(max(*live_rows, 0)), rows) : rows;
  const int groups = K / 8;
#pragma unroll 1
  for (int64_t base = int64_t(blockIdx.x) * per; base < live; base += int64_t(gridDim.x) * per) {
    const int64_t r = base + lr;
    const bool on = r < live;
    const In* src = x + (on ? (perm ? int64_t(perm[r]) : r) : 0) * K;
    Raw8<In> v[VPT];
    RowTop<In> seen;
    if (on) {
#pragma unroll
      for (int j = 0; j < VPT; ++j)
        if (c + j * tpr < groups) v[j].load(src + (c + j * tpr) * 8);
#pragma unroll
      for (int j = 0; j < VPT; ++j)
        if (c + j * tpr < groups) v[j].top(seen);
#pragma unroll 1
      for (int g = c + VPT * tpr; g < groups; g += tpr) {
        Raw8<In> w;
        w.load(src + g * 8);
        w.top(seen);
      }
    }
    uint32_t top = __reduce_max_sync(0xffffffffu, seen.bits());
    if (tpr > 32) {
      __syncthreads();  // the last round's maxima have been read
      if ((threadIdx.x & 31) == 0) top_s[threadIdx.x >> 5] = top;
      __syncthreads();
      const int w0 = lr * (tpr / 32);
      for (int w = 0; w < tpr / 32; ++w) top = max(top, top_s[w0 + w]);
    }
    if (!on) continue;
    const RowScale rs(top);
    if (c == 0) scale[r] = rs.scale;
    int8_t* dst = q + r * K;
    auto put = [&](int g, float (&w)[8]) { *reinterpret_cast<uint2*>(dst + g * 8) = rs.round8(w); };
#pragma unroll
    for (int j = 0; j < VPT; ++j)
      if (c + j * tpr < groups) {
        float w[8];
        v[j].values(w);
        put(c + j * tpr, w);
      }
#pragma unroll 1
    for (int g = c + VPT * tpr; g < groups; g += tpr) {
      Raw8<In> raw;
      raw.load(src + g * 8);
      float w[8];
      raw.values(w);
      put(g, w);
    }
  }
}

template <typename In>
int launch_quant(const void* x, int64_t rows, int K, const int32_t* perm, const int32_t* live, void* q, float* scale,
                 int sms, cudaStream_t stream) {
  const In* xi = static_cast<const In*>(x);
  int8_t* qi = static_cast<int8_t*>(q);
  // The fewest threads per row that leave each at most four groups of eight,
  // in CTAs of 256, or of 512 for fp32 rows that need them (8192 x 14336: 98
  // us, 104 with eight groups in each of 256 threads; bf16 95 and 76 us, so
  // there the smaller CTAs stay).
  constexpr int kMost = sizeof(In) == 4 ? 512 : 256;
  int tpr = 32;
  while (tpr < kMost && K / 8 > 4 * tpr) tpr *= 2;
  const int vpt = (K / 8 + tpr - 1) / tpr, per = tpr < 256 ? 256 / tpr : 1;
  const unsigned g = unsigned(std::min<int64_t>((rows + per - 1) / per, int64_t(sms) * 8));
  if (vpt <= 1) quant_rows_kernel<In, 1, 256><<<g, 256, 0, stream>>>(xi, rows, K, perm, live, tpr, qi, scale);
  else if (vpt <= 2) quant_rows_kernel<In, 2, 256><<<g, 256, 0, stream>>>(xi, rows, K, perm, live, tpr, qi, scale);
  else if (tpr <= 256 && vpt <= 4)
    quant_rows_kernel<In, 4, 256><<<g, 256, 0, stream>>>(xi, rows, K, perm, live, tpr, qi, scale);
  else  // kMost threads per row
    quant_rows_kernel<In, 2048 / kMost, kMost><<<g, kMost, 0, stream>>>(xi, rows, K, perm, live, tpr, qi, scale);
  return cudaGetLastError() == cudaSuccess ? kOk : kCudaErr;
}

// ---------------------------------------------------------------- weighted sum of the experts' rows
// y[t] = sum over k of v[t, k] * rows[offsets[e] + slots[t, k]], e = ids[t, k];
// slot -1: not routed here.  fp32 in the order of k, one rounding to bf16.
constexpr int kSumThreads = 256;
template <typename In>
__global__ void __launch_bounds__(kSumThreads)
    weighted_sum_kernel(const In* __restrict__ src, const void* __restrict__ ids, int ids64, int first,
                        const void* __restrict__ vals, int vals_bf16, const int32_t* __restrict__ slots,
                        const int32_t* __restrict__ offsets, int64_t T, int K, int H, int E,
                        __nv_bfloat16* __restrict__ y) {
  const int vec = H / 8;
  const int64_t total = T * vec;
  for (int64_t i = int64_t(blockIdx.x) * kSumThreads + threadIdx.x; i < total;
       i += int64_t(gridDim.x) * kSumThreads) {
    const int64_t t = i / vec;
    const int f = int(i - t * vec) * 8;
    float acc[8] = {};
#pragma unroll 4
    for (int k = 0; k < K; ++k) {
      const int64_t o = t * K + k;
      const int slot = slots[o];
      const long long e =
          (ids64 ? static_cast<const long long*>(ids)[o] : static_cast<const int32_t*>(ids)[o]) - (long long)first;
      if (slot < 0 || e < 0 || e >= E) continue;
      const float v = vals_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(vals)[o])
                                : static_cast<const float*>(vals)[o];
      float w[8];
      load8(src + (int64_t(offsets[e]) + slot) * H + f, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] = fmaf(v, w[j], acc[j]);
    }
    __nv_bfloat162 o2[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) o2[j] = __floats2bfloat162_rn(acc[2 * j], acc[2 * j + 1]);
    *reinterpret_cast<uint4*>(y + t * H + f) = *reinterpret_cast<uint4*>(o2);
  }
}

// ---------------------------------------------------------------- host side
int sm_count(int* sms, int* device = nullptr) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return kCudaErr;
  if (device) *device = dev;
  return cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess ? kOk : kCudaErr;
}

bool misaligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }
bool misaligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) != 0; }

size_t q_smem_bytes(int E) {
  return 1024 + size_t(kQStages) * kQStageBytes + kQXBytes + sizeof(QSmem) + size_t(E + 1) * 8;
}
static_assert(1024 + size_t(kQStages) * kQStageBytes + kQXBytes + sizeof(QSmem) + size_t(kMaxExperts + 1) * 8 <=
                  227 * 1024,
              "shared memory plan exceeds 227 KB");
static_assert((kQStages * kQStageBytes + kQXBytes) % 16 == 0, "QSmem must start on a 16-byte boundary");

// Whether a product may have fewer tiles than kQWaves per pair.
bool q_split(int64_t rows, int N, int F, bool glu, int pairs) {
  const int64_t ft = glu ? (F + 127) / 128 : (N + 255) / 256;
  return (rows + kQTileRows - 1) / kQTileRows * ft < kQWaves * int64_t(pairs);
}

int encode_s8(CUtensorMap* m, int rank, const void* ptr, const cuuint64_t* dims, const cuuint64_t* strides,
              const cuuint32_t* box) {
  const cuuint32_t one[3] = {1, 1, 1};
  return driver().cuTensorMapEncodeTiled(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, cuuint32_t(rank), const_cast<void*>(ptr),
                                         dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? kOk
             : kCudaErr;
}

// Once per device and form: shared memory opted in to, and the CTA pairs that
// can be resident together (the split form's meet at a grid barrier).
constexpr int kMaxDevices = 64;
template <bool GLU, bool SPLIT>
int w8a8_pairs(int dev, int sms, cudaLaunchConfig_t cfg, int* out) {
  static std::atomic<int> known[kMaxDevices];
  if (dev < 0 || dev >= kMaxDevices) return kCudaErr;
  int n = known[dev].load(std::memory_order_acquire);
  if (n == 0) {
    const size_t smem = q_smem_bytes(kMaxExperts);
    if (cudaFuncSetAttribute(w8a8_kernel<GLU, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)) !=
        cudaSuccess)
      return kCudaErr;
    cfg.gridDim = dim3(unsigned(sms & ~1));
    cfg.dynamicSmemBytes = smem;
    if (cudaOccupancyMaxActiveClusters(&n, w8a8_kernel<GLU, SPLIT>, &cfg) != cudaSuccess || n < 1) return kCudaErr;
    n = std::min(n, sms / 2);
    known[dev].store(n, std::memory_order_release);
  }
  *out = n;
  return kOk;
}

// The form for a handful of rows: they have to fit shared memory twice per SM,
// and an expert's to be taken in one pass as a rule (21 rows over 8 experts of
// 14336 x 4096: 87.7 us against 80.5 with the tiles; 16 rows 55.9 against
// 56.1; 32 over 64 experts of 2816 x 2048: 29.7 against 36.3; one expert of
// 4096 x 7168 with 4 rows 10.7 against 13.1, with 6 rows 14.7 against 13.4).
bool one_pass(int64_t rows, int E) { return rows <= kRwRows || rows <= 2 * int64_t(E); }
bool fresh(int64_t rows, int K) { return rows <= kRwMaxFreshRows && rows * K <= kRwMaxFresh; }
bool rows_form(int64_t rows, int K, int E) {
  return rows <= kRwMaxRows && rows * K <= int64_t(kRwMaxSmem) && one_pass(rows, E);
}

template <bool GLU, bool SUM, bool PAIR>
int launch_rows_as(const RwArgs& a, int staged, int64_t items, int dev, int sms, cudaStream_t stream) {
  static std::atomic<bool> ready[kMaxDevices];
  if (dev < 0 || dev >= kMaxDevices) return kCudaErr;
  if (!ready[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(w8a8_rows_kernel<GLU, SUM, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             int(kRwMaxSmem)) != cudaSuccess)
      return kCudaErr;
    ready[dev].store(true, std::memory_order_release);
  }
  const int64_t blocks = std::min<int64_t>((items + kRwThreads / 32 - 1) / (kRwThreads / 32), 2 * int64_t(sms));
  w8a8_rows_kernel<GLU, SUM, PAIR><<<unsigned(blocks), kRwThreads, size_t(staged) * a.K, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? kOk : kCudaErr;
}
template <bool GLU, bool SUM>
int launch_rows(const RwArgs& a, int staged, int64_t items, int dev, int sms, cudaStream_t stream) {
  if constexpr (!GLU) {
    // Pairs of channels where rows share an expert and they still occupy
    // every warp: with several rows the shared memory reads bound the form.
    if (staged > 1 && items / 2 >= 2 * int64_t(sms) * (kRwThreads / 32))
      return launch_rows_as<GLU, SUM, true>(a, staged, items / 2, dev, sms, stream);
  }
  return launch_rows_as<GLU, SUM, false>(a, staged, items, dev, sms, stream);
}

template <bool GLU, bool SPLIT>
int launch_w8a8(const CUtensorMap& tw, const QRowMaps& tx, const QArgs& a, int dev, int sms, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 2;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeCooperative;
  at[1].val.cooperative = 1;
  cfg.blockDim = dim3(kQThreads);
  cfg.stream = stream;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  int pairs = 0;
  if (w8a8_pairs<GLU, SPLIT>(dev, sms, cfg, &pairs) != kOk) return kCudaErr;
  cfg.gridDim = dim3(unsigned(2 * pairs));
  cfg.dynamicSmemBytes = q_smem_bytes(a.E);
  cfg.numAttrs = SPLIT ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, w8a8_kernel<GLU, SPLIT>, tw, tx, a) == cudaSuccess ? kOk : kCudaErr;
}

bool q_sizes_ok(int64_t rows, int32_t K, int32_t N, int32_t E, int32_t glu) {
  if (rows < 0 || rows > (int64_t(1) << 30) || K <= 0 || K % 16 || K > kQMaxK) return false;
  if (N <= 0 || N % (glu ? 16 : 8) || E < 1 || E > kMaxExperts) return false;
  const int64_t ft = (N + 255) / 256;
  const int64_t tiles = ((rows + kQTileRows - 1) / kQTileRows + E) * ft;
  return tiles * ((K + kQKb - 1) / kQKb) <= (int64_t(1) << 30);
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" int moe_quant_rows(const void* x, int32_t x_is_f32, int64_t rows, int32_t K, const int32_t* perm,
                              const int32_t* live_rows, void* q, float* scale, void* stream) {
  if (rows < 0 || rows > (int64_t(1) << 30) || K <= 0 || K % 8) return kBadArg;
  if (rows == 0) return kOk;
  if (!x || !q || !scale || misaligned16(x) || (reinterpret_cast<uintptr_t>(q) & 7)) return kBadArg;
  int sms = 0;
  if (sm_count(&sms) != kOk) return kCudaErr;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return x_is_f32 ? launch_quant<float>(x, rows, K, perm, live_rows, q, scale, sms, s)
                  : launch_quant<__nv_bfloat16>(x, rows, K, perm, live_rows, q, scale, sms, s);
}

namespace {
// scratch: partial sums of the split form, then (x given, quantised by a
// launch of its own) the quantised rows and their scales.
struct QScratch {
  bool few, split, rows_outside;
  size_t xq, xs, total;
};
QScratch q_scratch(int64_t rows, int K, int N, int E, bool glu, bool with_x, int sms) {
  QScratch q;
  q.few = rows_form(rows, K, E);
  q.split = !q.few && q_split(rows, N, glu ? N / 2 : N, glu, sms / 2);
  q.rows_outside = with_x && !(q.few && fresh(rows, K));
  q.xq = q.split ? size_t(sms / 2) * 2 * kQSlotInts * 4 : 0;
  q.xs = q.xq + (q.rows_outside ? (size_t(rows) * K + 255) / 256 * 256 : 0);
  q.total = q.xs + (q.rows_outside ? size_t(rows) * 4 : 0);
  return q;
}
}  // namespace

extern "C" int moe_w8a8_scratch_bytes(int64_t rows, int32_t K, int32_t N, int32_t E, int32_t swiglu, int32_t with_x,
                                      int32_t device, size_t* out) {
  if (!out || !q_sizes_ok(rows, K, N, E, swiglu)) return kBadArg;
  int sms = 0;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) return kCudaErr;
  *out = q_scratch(rows, K, N, E, swiglu != 0, with_x != 0, sms).total;
  return kOk;
}

extern "C" int moe_w8a8_gemm(const moe_w8a8_params* p, void* stream) {
  if (!p || !q_sizes_ok(p->rows, p->K, p->N, p->experts, p->swiglu)) return kBadArg;
  if (p->rows == 0) return kOk;
  if ((!p->x && (!p->xq || !p->xs)) || !p->wq || !p->ws || !p->out || (!p->counts && p->experts != 1)) return kBadArg;
  if (misaligned16(p->x)) return kBadArg;
  if (misaligned16(p->xq) || misaligned16(p->wq) || misaligned16(p->out) || misaligned16(p->scratch) ||
      misaligned4(p->xs) || misaligned4(p->ws))
    return kBadArg;
  if (!driver().ok) return kCudaErr;
  int sms = 0, dev = 0;
  if (sm_count(&sms, &dev) != kOk) return kCudaErr;
  const bool glu = p->swiglu != 0;
  const QScratch sc = q_scratch(p->rows, p->K, p->N, p->experts, glu, p->x != nullptr, sms);
  unsigned char* scratch = static_cast<unsigned char*>(p->scratch);
  if (sc.total > 0 && (!scratch || p->scratch_bytes < sc.total)) return kBadArg;
  const int8_t* xq = static_cast<const int8_t*>(p->xq);
  const float* xs = p->xs;
  QArgs a = {};
  a.E = p->experts;
  a.K = p->K;
  a.N = p->N;
  a.rows = p->rows;
  a.F = glu ? p->N / 2 : p->N;
  a.counts = p->counts;
  a.ws = p->ws;
  a.out = p->out;
  a.out_f32 = p->out_is_f32;
  a.part = reinterpret_cast<int32_t*>(scratch);
  a.status_host = p->status_host;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (sc.rows_outside) {
    int8_t* q = reinterpret_cast<int8_t*>(scratch + sc.xq);
    float* scale = reinterpret_cast<float*>(scratch + sc.xs);
    const int rc = p->x_is_f32
                       ? launch_quant<float>(p->x, a.rows, a.K, p->perm, p->live_rows, q, scale, sms, s)
                       : launch_quant<__nv_bfloat16>(p->x, a.rows, a.K, p->perm, p->live_rows, q, scale, sms, s);
    if (rc != kOk) return rc;
    xq = q;
    xs = scale;
  }
  a.xs = xs;
  if (sc.few) {
    RwArgs w = {};
    w.E = a.E;
    w.K = a.K;
    w.N = a.N;
    w.F = a.F;
    w.rows = int(a.rows);
    w.counts = a.counts;
    w.xq = xq;
    w.xs = xs;
    w.x = sc.rows_outside ? nullptr : p->x;
    w.x_f32 = p->x_is_f32;
    w.perm = p->perm;
    w.live = p->live_rows;
    w.wq = static_cast<const int8_t*>(p->wq);
    w.ws = p->ws;
    w.out = p->out;
    w.out_f32 = p->out_is_f32;
    const int64_t items = int64_t(a.F) * std::min(w.rows, a.E);  // at least one chunk per expert with rows
    return glu ? launch_rows<true, false>(w, w.rows, items, dev, sms, s)
               : launch_rows<false, false>(w, w.rows, items, dev, sms, s);
  }
  const bool split = sc.split;
  CUtensorMap tw;
  QRowMaps tx;
  {
    const cuuint64_t dims[3] = {cuuint64_t(a.K), cuuint64_t(a.N), cuuint64_t(a.E)};
    const cuuint64_t str[2] = {cuuint64_t(a.K), cuuint64_t(a.K) * a.N};
    const cuuint32_t box[3] = {cuuint32_t(kQKb), glu ? 64u : 128u, 1};
    if (encode_s8(&tw, 3, p->wq, dims, str, box)) return kCudaErr;
  }
  // Boxes of 16, 32, ... rows, as far as half a tile's rows may need.
  for (int i = 0; i < kQRowMaps && (i == 0 || (8 << i) < (a.rows + 31) / 32 * 16); ++i) {
    const cuuint64_t dims[2] = {cuuint64_t(a.K), cuuint64_t(a.rows)};
    const cuuint64_t str[1] = {cuuint64_t(a.K)};
    const cuuint32_t box[2] = {cuuint32_t(kQKb), 16u << i};
    if (encode_s8(&tx.m[i], 2, xq, dims, str, box)) return kCudaErr;
  }
  if (glu)
    return split ? launch_w8a8<true, true>(tw, tx, a, dev, sms, s) : launch_w8a8<true, false>(tw, tx, a, dev, sms, s);
  return split ? launch_w8a8<false, true>(tw, tx, a, dev, sms, s) : launch_w8a8<false, false>(tw, tx, a, dev, sms, s);
}

extern "C" int moe_weighted_sum(const void* rows, int32_t rows_are_f32, const void* top_idxs, int32_t ids_are_int64, int32_t first_expert,
                                const void* top_vals, int32_t vals_are_bf16, const int32_t* slots,
                                const int32_t* offsets, int64_t T, int32_t K, int32_t H, int32_t experts, void* y,
                                void* stream) {
  if (T < 0 || T > (int64_t(1) << 30) || K < 1 || K > kMaxRouteK || H <= 0 || H % 8 || experts < 1 ||
      experts > kMaxExperts)
    return kBadArg;
  if (T == 0) return kOk;
  if (!rows || !top_idxs || !top_vals || !slots || !offsets || !y || misaligned16(rows) || misaligned16(y))
    return kBadArg;
  int sms = 0;
  if (sm_count(&sms) != kOk) return kCudaErr;
  const int64_t blocks = std::min<int64_t>((T * (H / 8) + kSumThreads - 1) / kSumThreads, int64_t(sms) * 8);
  const auto launch = [&](auto* src) {
    weighted_sum_kernel<<<unsigned(blocks), kSumThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        src, top_idxs, ids_are_int64, first_expert, top_vals, vals_are_bf16, slots, offsets, T, K, H, experts,
        static_cast<__nv_bfloat16*>(y));
  };
  if (rows_are_f32) launch(static_cast<const float*>(rows));
  else launch(static_cast<const __nv_bfloat16*>(rows));
  return cudaGetLastError() == cudaSuccess ? kOk : kCudaErr;
}

namespace {
size_t up256(size_t v) { return (v + 255) / 256 * 256; }

// The layer of a few tokens: where each expert has few rows (four tokens, or
// two rows per expert on average) the rows kernel finds them itself and sums
// them; its scratch is h, then what is quantised by launches of its own.
bool q_layer_few(int64_t T, int H, int F, int E, int K) {
  return T * K <= kRwMaxRows && T * H <= int64_t(kRwMaxSmem) && T * K * F <= int64_t(kRwMaxSmem) &&
         (T <= kRwRows || T * K <= 2 * int64_t(E));
}
struct QFewScratch {
  bool x_outside, h_outside;
  size_t xq, xs, hq, hs, total;
};
QFewScratch q_few_scratch(int64_t T, int H, int F, int K) {
  QFewScratch s;
  s.x_outside = !fresh(T, H);
  s.h_outside = !fresh(T * K, F);
  s.xq = up256(size_t(T) * K * F * 4);
  s.xs = s.xq + (s.x_outside ? up256(size_t(T) * H) : 0);
  s.hq = s.xs + (s.x_outside ? 256 : 0);
  s.hs = s.hq + (s.h_outside ? up256(size_t(T) * K * F) : 0);
  s.total = s.hs + (s.h_outside ? 256 : 0);
  return s;
}
// Else: the routing's vectors, h, the second product's rows, and what either
// product needs (the second after the first).
struct QManyScratch {
  size_t offsets, max_count, perm, slots, h, rows, product, total;
};
QManyScratch q_many_scratch(int64_t T, int H, int F, int E, int K, int sms) {
  const int64_t n = T * K;
  QManyScratch s;
  s.offsets = up256(size_t(E) * 4);
  s.max_count = s.offsets + up256(size_t(E + 1) * 4);
  s.perm = s.max_count + 256;
  s.slots = s.perm + up256(size_t(n) * 4);
  s.h = s.slots + up256(size_t(n) * 4);
  s.rows = s.h + up256(size_t(n) * F * 4);
  s.product = s.rows + up256(size_t(n) * H * 4);
  s.total = s.product + std::max(q_scratch(n, H, 2 * F, E, true, true, sms).total,
                                 q_scratch(n, F, H, E, false, true, sms).total);
  return s;
}
bool q_layer_ok(int64_t T, int32_t H, int32_t F, int32_t E, int32_t K) {
  return T >= 0 && T <= (int64_t(1) << 30) && K >= 1 && K <= kMaxRouteK && H > 0 && H % 16 == 0 && F > 0 &&
         F % 16 == 0 && F <= kQMaxK && q_sizes_ok(T * K, H, 2 * F, E, 1) && q_sizes_ok(T * K, F, H, E, 0);
}

// Routing, the two products with h in fp32 between them, and the sum of fp32
// rows: y is rounded once, as where no sum is split.
int q_layer_many(const moe_w8a8_layer_params* p, int sms, void* stream) {
  const int H = p->hidden, F = p->ffn, E = p->experts;
  const int64_t n = p->T * p->K;
  const QManyScratch sc = q_many_scratch(p->T, H, F, E, p->K, sms);
  if (p->scratch_bytes < sc.total) return kBadArg;
  unsigned char* base = static_cast<unsigned char*>(p->scratch);
  int32_t* counts = reinterpret_cast<int32_t*>(base);
  int32_t* offsets = reinterpret_cast<int32_t*>(base + sc.offsets);
  int32_t* perm = reinterpret_cast<int32_t*>(base + sc.perm);
  int32_t* slots = reinterpret_cast<int32_t*>(base + sc.slots);
  int rc = launch_route(p->top_idxs, p->ids_are_int64, p->T, p->K, p->first_expert, E, counts, offsets, perm, slots,
                        reinterpret_cast<int32_t*>(base + sc.max_count), static_cast<cudaStream_t>(stream));
  if (rc != kOk) return rc;
  moe_w8a8_params g = {};
  g.rows = n;
  g.experts = E;
  g.counts = counts;
  g.live_rows = offsets + E;
  g.scratch = base + sc.product;
  g.scratch_bytes = sc.total - sc.product;
  g.status_host = p->status_host;
  g.out_is_f32 = 1;
  g.K = H;
  g.N = 2 * F;
  g.swiglu = 1;
  g.wq = p->w13;
  g.ws = p->w13_scale;
  g.x = p->x;
  g.perm = perm;
  g.out = base + sc.h;
  rc = moe_w8a8_gemm(&g, stream);
  if (rc != kOk) return rc;
  g.K = F;
  g.N = H;
  g.swiglu = 0;
  g.wq = p->w2;
  g.ws = p->w2_scale;
  g.x = base + sc.h;
  g.x_is_f32 = 1;
  g.perm = nullptr;
  g.out = base + sc.rows;
  rc = moe_w8a8_gemm(&g, stream);
  if (rc != kOk) return rc;
  return moe_weighted_sum(base + sc.rows, 1, p->top_idxs, p->ids_are_int64, p->first_expert, p->top_vals,
                          p->vals_are_bf16, slots, offsets, p->T, p->K, H, E, p->y, stream);
}
}  // namespace

extern "C" int moe_w8a8_layer_scratch_bytes(int64_t T, int32_t H, int32_t F, int32_t E, int32_t K, int32_t device,
                                            size_t* out) {
  if (!out || !q_layer_ok(T, H, F, E, K)) return kBadArg;
  int sms = 0;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) return kCudaErr;
  *out = q_layer_few(T, H, F, E, K) ? q_few_scratch(T, H, F, K).total : q_many_scratch(T, H, F, E, K, sms).total;
  return kOk;
}

extern "C" int moe_w8a8_layer(const moe_w8a8_layer_params* p, void* stream) {
  if (!p || !q_layer_ok(p->T, p->hidden, p->ffn, p->experts, p->K) || p->first_expert < 0) return kBadArg;
  if (p->T == 0) return kOk;
  if (!p->x || !p->w13 || !p->w13_scale || !p->w2 || !p->w2_scale || !p->top_idxs || !p->top_vals || !p->y ||
      !p->scratch)
    return kBadArg;
  if (misaligned16(p->x) || misaligned16(p->w13) || misaligned16(p->w2) || misaligned16(p->y) ||
      misaligned16(p->scratch) || misaligned4(p->w13_scale) || misaligned4(p->w2_scale))
    return kBadArg;
  int sms = 0, dev = 0;
  if (sm_count(&sms, &dev) != kOk) return kCudaErr;
  if (!q_layer_few(p->T, p->hidden, p->ffn, p->experts, p->K)) return q_layer_many(p, sms, stream);
  const int T = int(p->T), H = p->hidden, F = p->ffn, K = p->K;
  const QFewScratch sc = q_few_scratch(T, H, F, K);
  if (p->scratch_bytes < sc.total) return kBadArg;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  unsigned char* base = static_cast<unsigned char*>(p->scratch);
  float* h = reinterpret_cast<float*>(base);
  RwArgs a = {};
  a.E = p->experts;
  a.K = H;
  a.N = 2 * F;
  a.F = F;
  a.rows = T;
  a.wq = static_cast<const int8_t*>(p->w13);
  a.ws = p->w13_scale;
  a.out = h;
  a.out_f32 = 1;
  a.ids = p->top_idxs;
  a.ids64 = p->ids_are_int64;
  a.first = p->first_expert;
  a.T = T;
  a.topk = K;
  a.vals = p->top_vals;
  a.vals_bf16 = p->vals_are_bf16;
  a.x = p->x;
  if (sc.x_outside) {
    int8_t* q = reinterpret_cast<int8_t*>(base + sc.xq);
    float* scale = reinterpret_cast<float*>(base + sc.xs);
    if (launch_quant<__nv_bfloat16>(p->x, T, H, nullptr, nullptr, q, scale, sms, s) != kOk) return kCudaErr;
    a.x = nullptr;
    a.xq = q;
    a.xs = scale;
  }
  if (launch_rows<true, false>(a, T, int64_t(F) * std::min(T * K, a.E), dev, sms, s) != kOk) return kCudaErr;
  // Rows of h that no id leads to were not written; they are not used either.
  a.K = F;
  a.N = a.F = H;
  a.rows = T * K;
  a.wq = static_cast<const int8_t*>(p->w2);
  a.ws = p->w2_scale;
  a.out = p->y;
  a.out_f32 = 0;
  a.x = h;
  a.x_f32 = 1;
  if (sc.h_outside) {
    int8_t* q = reinterpret_cast<int8_t*>(base + sc.hq);
    float* scale = reinterpret_cast<float*>(base + sc.hs);
    if (launch_quant<float>(h, T * K, F, nullptr, nullptr, q, scale, sms, s) != kOk) return kCudaErr;
    a.x = nullptr;
    a.xq = q;
    a.xs = scale;
  }
  return launch_rows<false, true>(a, T * K, H, dev, sms, s);
}
