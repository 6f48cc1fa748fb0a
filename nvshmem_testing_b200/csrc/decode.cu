// The whole gated MoE layer for a few tokens (T <= 64) in one kernel:
//   y[t] = sum_k v[t,k] * (silu(x_t W_gate,e) * (x_t W_up,e)) W_down,e
// with e = ids[t,k] - first_expert, and (routed form) ids and v from
// softmax(x R) and its top-k.  The reference routes, pads, exchanges and
// multiplies in separate steps (utils.py:23-75, baseline.py:18-50).
//
// With few tokens the layer is a stream of the active experts' weights
// (6*H*F bytes each), every byte used once for a handful of rows, so the
// kernel is built around that stream.  Persistent, one CTA per SM, launched
// cooperatively; two passes over the weights with a grid barrier between:
//   pass 1  units (active expert, 128 features of F, 64 of H): the gate and
//           the up block (2 x 128 features) are the MMA A operand
//           (tcgen05, M = 128 each, feature-contiguous as stored), all T
//           tokens the B operand; h = silu(gate) * up is written, in bf16,
//           for the tokens that chose the expert only.
//   pass 2  units (256 features of H, active expert, 64 of F): the rows of
//           h of one expert are B; the epilogue adds v * D to an fp32 sum
//           per token and feature in shared memory, so that the experts'
//           outputs meet without leaving the CTA.
// Each pass splits its list of 32 KB units evenly over the CTAs, at any k:
// every SM streams the same number of bytes whatever the number of experts
// or tiles.  A tile that ends up in several CTAs is summed by the last of
// them, from fp32 partials in CTA order, so results do not depend on timing.
// The weights' first stages of a pass are requested before the barrier in
// front of it; only the token rows wait for it.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <climits>

#include "moe_ep.h"
#include "moe_ep_internal.h"
#include "ptx.cuh"

namespace moe {
namespace {

namespace cg = cooperative_groups;

constexpr int kDecMaxT = 64;
constexpr int kDecMaxRows = 1024;                 // T * K
constexpr int kDecMaxH = 32768;
constexpr int kDecEpiWarps = 8;                   // two per TMEM lane quarter
constexpr int kDecEpi0 = 2;                       // warps: 0 loads, 1 MMA, 2.. epilogue
constexpr int kDecThreads = (kDecEpi0 + kDecEpiWarps) * 32;
constexpr int kDecMaxStages = 8;
constexpr uint32_t kDecABytes = 256 * 64 * 2;     // 256 features x 64 K
constexpr uint32_t kDecMaxSmem = 227 * 1024;
constexpr int kDecTokChunk = 8;                   // router: tokens whose logits a thread sums at a time
constexpr uint64_t kDecBoundNs = 2000000000ull;   // bug guard on every pipeline wait
constexpr int kBarEpi = 1;

struct DecArgs {
  int T, H, F, E, K, first;  // E: experts held here
  int NB;                    // T rounded to 16: B rows and MMA N of pass 1
  int stages;
  uint32_t stage_bytes, scratch_bytes;
  int maxact;                // min(E, T * K)
  int w2_atoms;              // w2 described in atoms of 64 features (H % 64 == 0)
  const __nv_bfloat16* x;
  const void* ids;
  const void* vals;
  int ids64, vals_bf16;
  __nv_bfloat16* hs;         // [T*K][F]
  float* part;               // [2 * grid][T][256]
  uint32_t* ctr;             // [2 * grid]
  __nv_bfloat16* y;
  int32_t* status_host;
  // Routed form (router_w != nullptr).
  const __nv_bfloat16* router_w;  // [H, Er]
  int Er, renorm;
  float* lpart;              // [grid][T][Er]
  void* out_ids;
  float* out_vals;
};

struct alignas(16) DecSmem {
  uint64_t full[kDecMaxStages];
  uint64_t empty[kDecMaxStages];
  uint64_t tfull[2];
  uint64_t tempty[2];
  uint64_t drain;
  uint32_t fills[kDecMaxStages];
  uint32_t tmem_base;
  int err;
  int nact, rows;
  int last;
};

__device__ bool dec_wait(uint64_t* bar, uint32_t parity, DecSmem& sm) {
  uint64_t deadline = 0;
  for (uint32_t spin = 0;; ++spin) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((spin & 63) == 63) {
      if (*reinterpret_cast<volatile int*>(&sm.err)) return false;
      const uint64_t now = globaltimer_ns();
      if (deadline == 0) deadline = now + kDecBoundNs;
      else if (now > deadline) return false;
    }
  }
}

__device__ void dec_fail(DecSmem& sm, const DecArgs& a, int detail) {
  if (atomicExch(&sm.err, 1) == 0 && a.status_host)
    *reinterpret_cast<volatile int32_t*>(a.status_host) = int32_t(status_word(kTimeout, kSitePipe, detail));
}

// Share of CTA c of `units`, and the CTA a unit belongs to (g CTAs, g <= units).
__device__ __forceinline__ int share_lo(int64_t units, int g, int c) { return int(units * c / g); }
__device__ __forceinline__ int share_owner(int64_t units, int g, int64_t u) {
  return int(((u + 1) * g - 1) / units);
}

__device__ __forceinline__ long long load_id(const DecArgs& a, const void* ids, int i) {
  return a.ids64 ? __ldcg(static_cast<const long long*>(ids) + i) : __ldcg(static_cast<const int*>(ids) + i);
}

// Tables in shared memory, built alike by every CTA from the routing.
struct DecTables {
  uint16_t* act_e;    // [maxact] active experts, ascending
  uint16_t* act_off;  // [maxact + 1] first row of each
  float* val;         // [T*K] routing weight of a row
  uint8_t* tok;       // [T*K] token of a row
};

__host__ __device__ inline uint32_t dec_table_bytes(int maxact, int rows) {
  return uint32_t(((rows * 4 + (2 * maxact + 1) * 2 + rows) + 15) / 16 * 16);
}

// One 64-bit mask of tokens per expert: an id repeated in a row counts once,
// ids outside [first, first + E) match none, and rows of an expert ascend by
// token, the same in every CTA.
__device__ void dec_build(const DecArgs& a, DecSmem& sm, const DecTables& tb, unsigned char* scratch, const void* ids,
                          const void* vals, int vals_bf16) {
  unsigned long long* mask = reinterpret_cast<unsigned long long*>(scratch);  // [E]
  uint16_t* off_e = reinterpret_cast<uint16_t*>(mask + a.E);                  // [E]
  const int tid = threadIdx.x, n = a.T * a.K;
  for (int e = tid; e < a.E; e += kDecThreads) mask[e] = 0;
  __syncthreads();
  for (int i = tid; i < n; i += kDecThreads) {
    const long long e = load_id(a, ids, i) - a.first;
    if (e >= 0 && e < a.E) atomicOr(&mask[e], 1ull << (i / a.K));
  }
  __syncthreads();
  if (tid < 32) {
    int act = 0, row = 0;
    for (int e0 = 0; e0 < a.E; e0 += 32) {
      const int e = e0 + tid;
      const int c = e < a.E ? __popcll(mask[e]) : 0;
      int pre = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, pre, o);
        if (tid >= o) pre += v;
      }
      const uint32_t live = __ballot_sync(0xffffffffu, c > 0);
      if (e < a.E) off_e[e] = uint16_t(row + pre - c);
      if (c > 0) {
        const int at = act + __popc(live & ((1u << tid) - 1));
        tb.act_e[at] = uint16_t(e);
        tb.act_off[at] = uint16_t(row + pre - c);
      }
      act += __popc(live);
      row += __shfl_sync(0xffffffffu, pre, 31);
    }
    if (tid == 0) {
      tb.act_off[act] = uint16_t(row);
      sm.nact = act;
      sm.rows = row;
    }
  }
  __syncthreads();
  for (int i = tid; i < n; i += kDecThreads) {
    const int t = i / a.K;
    const long long id = load_id(a, ids, i), e = id - a.first;
    if (e < 0 || e >= a.E) continue;
    bool again = false;
    for (int j = t * a.K; j < i; ++j) again |= load_id(a, ids, j) == id;
    if (again) continue;
    const int r = off_e[e] + __popcll(mask[e] & ((1ull << t) - 1));
    tb.tok[r] = uint8_t(t);
    tb.val[r] = vals_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(vals)[i])
                          : __ldcg(static_cast<const float*>(vals) + i);
  }
  __syncthreads();
}

// Router, step 1: this CTA's slice of H of every token's logits, in fp32.
// Threads hold two neighbouring experts each; groups of threads take every
// `groups`-th row of the slice and are summed in group order.
__device__ void dec_router_partial(const DecArgs& a, unsigned char* stage) {
  const int G = gridDim.x, c = blockIdx.x, tid = threadIdx.x;
  const int h0 = int(int64_t(a.H) * c / G), h1 = int(int64_t(a.H) * (c + 1) / G), nh = h1 - h0;
  float* red = reinterpret_cast<float*>(stage);                       // [groups][chunk][Er]
  float* xs = red + kDecThreads * 2 * kDecTokChunk;                   // [T][nh]
  for (int i = tid; i < a.T * nh; i += kDecThreads) {
    const int t = i / nh, h = i - t * nh;
    xs[i] = __bfloat162float(a.x[int64_t(t) * a.H + h0 + h]);
  }
  __syncthreads();
  const int P = a.Er / 2;
  const int groups = P < kDecThreads ? kDecThreads / P : 1;
  const int grp = tid / P;
  for (int t0 = 0; t0 < a.T; t0 += kDecTokChunk) {
    const int nt = min(kDecTokChunk, a.T - t0);
    for (int p0 = 0; p0 < P; p0 += kDecThreads) {  // more than one round only for Er > 2 * kDecThreads
      const int p = P < kDecThreads ? tid - grp * P : p0 + tid;
      const bool on = P < kDecThreads ? grp < groups : p < P;
      float2 s[kDecTokChunk];
#pragma unroll
      for (int j = 0; j < kDecTokChunk; ++j) s[j] = make_float2(0.f, 0.f);
      if (on) {
        const __nv_bfloat162* r = reinterpret_cast<const __nv_bfloat162*>(a.router_w + int64_t(h0) * a.Er) + p;
#pragma unroll 8
        for (int h = P < kDecThreads ? grp : 0; h < nh; h += groups) {
          const float2 w = __bfloat1622float2(r[int64_t(h) * P]);
#pragma unroll
          for (int j = 0; j < kDecTokChunk; ++j) {
            const float xv = j < nt ? xs[(t0 + j) * nh + h] : 0.f;
            s[j].x = fmaf(xv, w.x, s[j].x);
            s[j].y = fmaf(xv, w.y, s[j].y);
          }
        }
      }
      if (groups > 1) {
        if (on) {
#pragma unroll
          for (int j = 0; j < kDecTokChunk; ++j)
            *reinterpret_cast<float2*>(&red[(grp * kDecTokChunk + j) * a.Er + 2 * p]) = s[j];
        }
        __syncthreads();
        for (int i = tid; i < nt * a.Er; i += kDecThreads) {
          const int j = i / a.Er, e = i - j * a.Er;
          float v = 0.f;
          for (int g = 0; g < groups; ++g) v += red[(g * kDecTokChunk + j) * a.Er + e];
          a.lpart[(int64_t(c) * a.T + t0 + j) * a.Er + e] = v;
        }
        __syncthreads();
      } else if (on) {
        for (int j = 0; j < nt; ++j)
          *reinterpret_cast<float2*>(&a.lpart[(int64_t(c) * a.T + t0 + j) * a.Er + 2 * p]) = s[j];
      }
    }
  }
}

// Router, step 2: tokens c, c + grid, ...: the slices' sum in CTA order, the
// softmax over Er in fp32 and the K largest (equal logits: lowest id first).
__device__ void dec_router_topk(const DecArgs& a, unsigned char* stage, unsigned char* scratch) {
  const int G = gridDim.x, tid = threadIdx.x, lane = tid & 31;
  float* red = reinterpret_cast<float*>(stage);       // [parts][Er]
  float* lg = reinterpret_cast<float*>(scratch);      // [Er]
  const int parts = a.Er < kDecThreads ? kDecThreads / a.Er : 1;
  for (int t = blockIdx.x; t < a.T; t += G) {
    for (int i = tid; i < parts * a.Er; i += kDecThreads) {
      const int q = i / a.Er, e = i - q * a.Er;
      const int c0 = G * q / parts, c1 = G * (q + 1) / parts;
      float v = 0.f;
#pragma unroll 16
      for (int c = c0; c < c1; ++c) v += __ldcg(&a.lpart[(int64_t(c) * a.T + t) * a.Er + e]);
      red[i] = v;
    }
    __syncthreads();
    for (int e = tid; e < a.Er; e += kDecThreads) {
      float v = 0.f;
      for (int q = 0; q < parts; ++q) v += red[q * a.Er + e];
      lg[e] = v;
    }
    __syncthreads();
    if (tid < 32) {
      float m = -INFINITY;
      for (int e = lane; e < a.Er; e += 32) m = fmaxf(m, lg[e]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      float z = 0.f;
      for (int e = lane; e < a.Er; e += 32) z += expf(lg[e] - m);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
      uint32_t taken = 0;  // bit i: expert lane + 32 * i
      float mine = 0.f;    // lane k: the k-th probability
      int id = 0;
      float sum = 0.f;
      for (int k = 0; k < a.K; ++k) {
        float best = 0.f;
        int be = INT_MAX;
        for (int i = 0, e = lane; e < a.Er; ++i, e += 32) {
          const float v = lg[e];
          if (!((taken >> i) & 1) && (be == INT_MAX || v > best)) {
            best = v;
            be = e;
          }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const float ob = __shfl_xor_sync(0xffffffffu, best, o);
          const int oe = __shfl_xor_sync(0xffffffffu, be, o);
          // An empty hand (INT_MAX) loses; equal values, or values that do
          // not compare (NaN), go to the lower id: every lane agrees.
          const bool take = be == INT_MAX || (oe != INT_MAX && (ob > best || (!(best > ob) && oe < be)));
          if (take) {
            best = ob;
            be = oe;
          }
        }
        be = __shfl_sync(0xffffffffu, be, 0);
        best = __shfl_sync(0xffffffffu, best, 0);
        if ((be & 31) == lane) taken |= 1u << (be >> 5);
        const float pr = expf(best - m) / z;
        sum += pr;
        if (lane == k) {
          mine = pr;
          id = be;
        }
      }
      if (lane < a.K) {
        const int64_t o = int64_t(t) * a.K + lane;
        a.out_vals[o] = a.renorm ? mine / sum : mine;
        if (a.ids64) static_cast<long long*>(a.out_ids)[o] = id;
        else static_cast<int*>(a.out_ids)[o] = id;
      }
    }
    __syncthreads();
  }
}

// What one pass consists of.
struct Pass {
  int units;     // all CTAs
  int tile;      // units of one tile (the units whose sums belong together)
  int kb;        // units of one expert's K
  int g;         // CTAs that have units
  int lo, hi;    // this CTA's
};

__global__ void __launch_bounds__(kDecThreads, 1)
    decode_kernel(const __grid_constant__ CUtensorMap tm_w13, const __grid_constant__ CUtensorMap tm_w2,
                  const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_h,
                  const DecArgs a) {
  extern __shared__ unsigned char dec_dyn[];
  unsigned char* stage =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(dec_dyn) + 1023) & ~uintptr_t(1023));
  unsigned char* scratch = stage + size_t(a.stages) * a.stage_bytes;
  unsigned char* tables = scratch + a.scratch_bytes;
  const int maxrows = a.T * a.K;
  DecTables tb;
  tb.val = reinterpret_cast<float*>(tables);
  tb.act_e = reinterpret_cast<uint16_t*>(tb.val + maxrows);
  tb.act_off = tb.act_e + a.maxact;
  tb.tok = reinterpret_cast<uint8_t*>(tb.act_off + a.maxact + 1);
  DecSmem& sm = *reinterpret_cast<DecSmem*>(tables + dec_table_bytes(a.maxact, maxrows));
  float* acc = reinterpret_cast<float*>(scratch);  // pass 2: [T][256]

  cg::grid_group grid = cg::this_grid();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int S = a.stages;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], 1);
      sm.fills[i] = 0;
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.tfull[i], 1);
      mbar_init(&sm.tempty[i], kDecEpiWarps);
    }
    mbar_init(&sm.drain, 1);
    sm.err = 0;
    fence_mbar_init();
    prefetch_tensormap(&tm_w13);
    prefetch_tensormap(&tm_x);
    prefetch_tensormap(&tm_w2);
    prefetch_tensormap(&tm_h);
  }
  const uint32_t tmem_cols = a.NB <= 16 ? 64 : a.NB <= 32 ? 128 : 256;
  if (warp == 1) {
    __syncwarp();
    tmem_alloc(&sm.tmem_base, tmem_cols);
    tmem_relinquish();
  }
  // The tickets of split tiles start at zero: written here, ordered before
  // their first use by the first grid barrier.
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < 2 * int(gridDim.x); i += kDecThreads) a.ctr[i] = 0;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;

  if (a.router_w != nullptr) {
    dec_router_partial(a, stage);
    grid.sync();
    dec_router_topk(a, stage, scratch);
    fence_proxy_async_smem();  // the stages, written by threads so far, belong to the TMA from here
    grid.sync();
    dec_build(a, sm, tb, scratch, a.out_ids, a.out_vals, 0);
  } else {
    dec_build(a, sm, tb, scratch, a.ids, a.vals, a.vals_bf16);
  }
  const int nact = sm.nact;
  const int G = gridDim.x;

  auto make_pass = [&](int tiles, int tile, int kb) {
    Pass p;
    p.units = tiles * tile;
    p.tile = tile;
    p.kb = kb;
    p.g = min(G, p.units);
    const bool on = int(blockIdx.x) < p.g;
    p.lo = on ? share_lo(p.units, p.g, blockIdx.x) : 0;
    p.hi = on ? share_lo(p.units, p.g, blockIdx.x + 1) : 0;
    return p;
  };
  const int kb1 = (a.H + 63) / 64, nt1 = (a.F + 127) / 128;
  const int kb2 = (a.F + 63) / 64, nt2 = (a.H + 255) / 256;
  const Pass p1 = make_pass(nact * nt1, kb1, kb1);
  const Pass p2 = make_pass(nact > 0 ? nt2 : 0, nact * kb2, kb2);

  // ---- loads (one thread)
  uint32_t it = 0;  // stages used so far
  auto act_rows = [&](int ai) { return int(tb.act_off[ai + 1]) - int(tb.act_off[ai]); };
  // Weights of unit u of a pass into the next stage; the stage's expected
  // bytes include the rows that load_rows adds.
  auto load_weights = [&](int pass, const Pass& p, int u) -> bool {
    const int st = it % S;
    if (!dec_wait(&sm.empty[st], ((it / S) & 1) ^ 1, sm)) {
      dec_fail(sm, a, 1);
      return false;
    }
    unsigned char* dst = stage + size_t(st) * a.stage_bytes;
    const int tile = u / p.tile, k = u % p.kb;
    if (pass == 1) {
      const int ai = tile / nt1, f0 = (tile % nt1) * 128;
      mbar_arrive_expect_tx(&sm.full[st], kDecABytes + uint32_t(a.NB) * 128);
      tma_load_4d(&tm_w13, &sm.full[st], dst, f0, k * 64, 0, tb.act_e[ai]);
      tma_load_4d(&tm_w13, &sm.full[st], dst + 16384, f0 + 64, k * 64, 0, tb.act_e[ai]);
    } else {
      const int ai = (u % p.tile) / p.kb;
      mbar_arrive_expect_tx(&sm.full[st], kDecABytes + uint32_t((act_rows(ai) + 15) / 16) * 2048);
      if (a.w2_atoms) {
        tma_load_4d(&tm_w2, &sm.full[st], dst, 0, k * 64, tile * 4, tb.act_e[ai]);
      } else {
        for (int g = 0; g < 4; ++g)
          tma_load_3d(&tm_w2, &sm.full[st], dst + g * 8192, tile * 256 + g * 64, k * 64, tb.act_e[ai]);
      }
    }
    sm.fills[st] += 1;
    ++it;
    return true;
  };
  auto load_rows = [&](int pass, const Pass& p, int u, uint32_t at) {
    const int st = at % S;
    unsigned char* dst = stage + size_t(st) * a.stage_bytes + kDecABytes;
    const int k = u % p.kb;
    if (pass == 1) {
      tma_load_2d(&tm_x, &sm.full[st], dst, k * 64, 0);
    } else {
      const int ai = (u % p.tile) / p.kb;
      const int nb = (act_rows(ai) + 15) / 16;
      for (int b = 0; b < nb; ++b)
        tma_load_2d(&tm_h, &sm.full[st], dst + b * 2048, k * 64, int(tb.act_off[ai]) + b * 16);
    }
  };
  // The first stages of a pass: weights only, before the barrier.
  auto preload = [&](int pass, const Pass& p) {
    int n = 0;
    while (n < S && p.lo + n < p.hi && load_weights(pass, p, p.lo + n)) ++n;
    return n;
  };
  auto produce = [&](int pass, const Pass& p, int pre) {
    for (int i = 0; i < pre; ++i) load_rows(pass, p, p.lo + i, it - pre + i);
    for (int u = p.lo + pre; u < p.hi; ++u) {
      if (!load_weights(pass, p, u)) return;
      load_rows(pass, p, u, it - 1);
    }
  };

  // ---- MMA (one thread)
  uint32_t mi = 0, mseg = 0;  // stages and accumulators used so far
  auto multiply = [&](int pass, const Pass& p) {
    for (int u = p.lo; u < p.hi; ++u, ++mi) {
      const int k = u % p.kb;
      const bool begin = u == p.lo || k == 0, end = u + 1 == p.hi || k + 1 == p.kb;
      const uint32_t buf = mseg & 1;
      if (begin && !dec_wait(&sm.tempty[buf], ((mseg >> 1) & 1) ^ 1, sm)) {
        dec_fail(sm, a, 2);
        return;
      }
      const int st = mi % S;
      if (!dec_wait(&sm.full[st], (mi / S) & 1, sm)) {
        dec_fail(sm, a, 3);
        return;
      }
      tc_fence_after();
      int n = a.NB;
      if (pass == 2) n = (act_rows((u % p.tile) / p.kb) + 15) / 16 * 16;
      const uint32_t idesc = make_idesc_mn(/*bf16*/ 1, 128, uint32_t(n), /*A MN-major*/ 1, /*B K-major*/ 0);
      const uint32_t aa = smem_u32(stage + size_t(st) * a.stage_bytes), ba = aa + kDecABytes;
      // Pass 1: box g (64 features of each half) is [gate 64x64][up 64x64];
      // pass 2: four groups of 64 features in order.
      const uint32_t half = pass == 1 ? 8192 : 16384, group = pass == 1 ? 16384 : 8192;
      const uint32_t d = tmem + buf * 2 * uint32_t(a.NB);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        const uint64_t bd = smem_desc_sw128(ba + kk * 32, 16, 1024);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint64_t ad = smem_desc_sw128(aa + h * half + kk * 2048, group, 1024);
          tc_mma_f16(d + h * uint32_t(a.NB), ad, bd, idesc, (!begin || kk != 0) ? 1u : 0u);
        }
      }
      tc_commit(&sm.empty[st]);
      if (end) {
        tc_commit(&sm.tfull[buf]);
        ++mseg;
      }
    }
  };

  // ---- epilogue (8 warps: lane quarter = 32 features of 128; two warps each)
  uint32_t eseg = 0;
  const int quarter = warp & 3, sub = (warp - kDecEpi0) >> 2;
  const int etid = int(threadIdx.x) - kDecEpi0 * 32;
  const uint32_t tlane = tmem + (uint32_t(quarter * 32) << 16);
  // This CTA's sums of a split tile are in its slot; true for the CTA whose
  // ticket is the last of the tile's.
  auto last_part = [&](uint32_t* ctr, int parts) {
    __threadfence();
    named_bar_sync(kBarEpi, kDecEpiWarps * 32);
    if (etid == 0) {
      sm.last = atomicAdd(ctr, 1u) == uint32_t(parts - 1);
      __threadfence();
    }
    named_bar_sync(kBarEpi, kDecEpiWarps * 32);
    return sm.last != 0;
  };
  const size_t slot_floats = size_t(a.T) * 256;
  auto slot = [&](int cta, int which) { return a.part + (size_t(cta) * 2 + which) * slot_floats; };

  auto epilogue1 = [&](const Pass& p) {
    for (int u = p.lo; u < p.hi; ++eseg) {
      const int tile = u / p.kb, ai = tile / nt1;
      const int seg_end = min(p.hi, (tile + 1) * p.kb);
      const bool whole = u == tile * p.kb && seg_end == (tile + 1) * p.kb;
      const uint32_t buf = eseg & 1;
      if (!named_bar_and(kBarEpi, kDecEpiWarps * 32, dec_wait(&sm.tfull[buf], (eseg >> 1) & 1, sm))) {
        dec_fail(sm, a, 4);
        return;
      }
      tc_fence_after();
      const int n = act_rows(ai), r0 = tb.act_off[ai];
      const int fl = quarter * 32 + lane;              // feature within the tile
      const int f = (tile % nt1) * 128 + fl;
      const uint32_t d = tlane + buf * 2 * uint32_t(a.NB);
      float* mine = slot(blockIdx.x, u == tile * p.kb ? 1 : 0);
      for (int j0 = sub; j0 < n; j0 += 8) {
        uint32_t g[4], w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (j0 + 2 * q < n) {
            const uint32_t t = tb.tok[r0 + j0 + 2 * q];
            g[q] = tmem_ld_32x32b_x1(d + t);
            w[q] = tmem_ld_32x32b_x1(d + uint32_t(a.NB) + t);
          }
        tmem_ld_wait();
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int j = j0 + 2 * q;
          if (j >= n) break;
          const float gv = __uint_as_float(g[q]), uv = __uint_as_float(w[q]);
          if (whole) {
            if (f < a.F) a.hs[size_t(r0 + j) * a.F + f] = __float2bfloat16_rn(gv / (1.f + expf(-gv)) * uv);
          } else {
            mine[j * 256 + fl] = gv;
            mine[j * 256 + 128 + fl] = uv;
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.tempty[buf]);
      if (!whole) {
        const int c0 = share_owner(p.units, p.g, int64_t(tile) * p.kb);
        const int c1 = share_owner(p.units, p.g, int64_t(tile + 1) * p.kb - 1);
        if (last_part(&a.ctr[c0], c1 - c0 + 1) && f < a.F) {
          for (int j = sub; j < n; j += 2) {
            float gv = 0.f, uv = 0.f;
            for (int c = c0; c <= c1; ++c) {
              const float* ps = slot(c, c == c0 ? 1 : 0) + j * 256 + fl;
              gv += __ldcg(ps);
              uv += __ldcg(ps + 128);
            }
            a.hs[size_t(r0 + j) * a.F + f] = __float2bfloat16_rn(gv / (1.f + expf(-gv)) * uv);
          }
        }
      }
      u = seg_end;
    }
  };

  auto epilogue2 = [&](const Pass& p) {
    const int fl = sub * 128 + quarter * 32 + lane;  // feature within the tile: this thread's alone
    for (int u = p.lo; u < p.hi;) {
      const int tile = u / p.tile;
      const int tile_end = min(p.hi, (tile + 1) * p.tile);
      const bool starts = u == tile * p.tile;
      const bool whole = starts && tile_end == (tile + 1) * p.tile;
      const int f = tile * 256 + fl;
      for (int t = 0; t < a.T; ++t) acc[t * 256 + fl] = 0.f;
      for (; u < tile_end; ++eseg) {
        const int in = u % p.tile, ai = in / p.kb;
        const int seg_end = min(tile_end, tile * p.tile + (ai + 1) * p.kb);
        const uint32_t buf = eseg & 1;
        if (!named_bar_and(kBarEpi, kDecEpiWarps * 32, dec_wait(&sm.tfull[buf], (eseg >> 1) & 1, sm))) {
          dec_fail(sm, a, 5);
          return;
        }
        tc_fence_after();
        const int n = act_rows(ai), r0 = tb.act_off[ai];
        const uint32_t d = tlane + buf * 2 * uint32_t(a.NB) + uint32_t(sub) * uint32_t(a.NB);
        for (int j0 = 0; j0 < n; j0 += 4) {
          uint32_t v[4];
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (j0 + q < n) v[q] = tmem_ld_32x32b_x1(d + uint32_t(j0 + q));
          tmem_ld_wait();
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if (j0 + q >= n) break;
            float* s = &acc[int(tb.tok[r0 + j0 + q]) * 256 + fl];
            *s = fmaf(tb.val[r0 + j0 + q], __uint_as_float(v[q]), *s);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.tempty[buf]);
        u = seg_end;
      }
      if (whole) {
        if (f < a.H)
          for (int t = 0; t < a.T; ++t) a.y[size_t(t) * a.H + f] = __float2bfloat16_rn(acc[t * 256 + fl]);
      } else {
        float* mine = slot(blockIdx.x, starts ? 1 : 0);
        for (int t = 0; t < a.T; ++t) mine[t * 256 + fl] = acc[t * 256 + fl];
        const int c0 = share_owner(p.units, p.g, int64_t(tile) * p.tile);
        const int c1 = share_owner(p.units, p.g, int64_t(tile + 1) * p.tile - 1);
        if (last_part(&a.ctr[G + c0], c1 - c0 + 1) && f < a.H) {
          for (int t = 0; t < a.T; ++t) {
            float v = 0.f;
            for (int c = c0; c <= c1; ++c) v += __ldcg(slot(c, c == c0 ? 1 : 0) + t * 256 + fl);
            a.y[size_t(t) * a.H + f] = __float2bfloat16_rn(v);
          }
        }
      }
    }
  };

  // ---- the two passes
  int pre = 0;
  if (threadIdx.x == 0) pre = preload(1, p1);
  __syncwarp();
  if (a.router_w == nullptr) grid.sync();  // (routed: the router's barriers ordered the tickets)
  if (warp == 0 && lane == 0) produce(1, p1, pre);
  else if (warp == 1 && lane == 0) multiply(1, p1);
  else if (warp >= kDecEpi0) epilogue1(p1);
  __syncwarp();
  if (threadIdx.x == 0 && !*reinterpret_cast<volatile int*>(&sm.err)) pre = preload(2, p2);
  __syncwarp();
  fence_proxy_async_global();  // h, written by threads, is read by the TMA
  grid.sync();
  const bool ok = !*reinterpret_cast<volatile int*>(&sm.err);
  if (ok) {
    if (warp == 0 && lane == 0) {
      fence_proxy_async_global();
      produce(2, p2, pre);
    } else if (warp == 1 && lane == 0) {
      multiply(2, p2);
    } else if (warp >= kDecEpi0) {
      epilogue2(p2);
    }
  }
  if (nact == 0)  // no token has an expert here
    for (int64_t i = int64_t(blockIdx.x) * kDecThreads + threadIdx.x; i < int64_t(a.T) * a.H;
         i += int64_t(G) * kDecThreads)
      a.y[i] = __float2bfloat16_rn(0.f);
  __syncwarp();
  if (warp == 1 && lane == 0) tc_commit(&sm.drain);
  __syncthreads();
  // Teardown: after an abort, wait (bounded) for every issued load and MMA.
  if (threadIdx.x == 0 && *reinterpret_cast<volatile int*>(&sm.err)) {
    const uint64_t until = globaltimer_ns() + kDecBoundNs;
    for (int st = 0; st < S; ++st) {
      const uint32_t f = sm.fills[st];
      if (f == 0) continue;
      while (!mbar_try_wait(&sm.full[st], (f - 1) & 1) && globaltimer_ns() < until) {
      }
    }
    while (!mbar_try_wait(&sm.drain, 0) && globaltimer_ns() < until) {
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tmem, tmem_cols);
  }
}

int encode(CUtensorMap* m, int rank, const void* ptr, const cuuint64_t* dims, const cuuint64_t* strides,
           const cuuint32_t* box) {
  const cuuint32_t one[5] = {1, 1, 1, 1, 1};
  return driver().cuTensorMapEncodeTiled(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, cuuint32_t(rank),
                                         const_cast<void*>(ptr), dims, strides, box, one,
                                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? kOk
             : kCudaErr;
}

struct DecScratch {
  size_t hs, part, ctr, lpart, total;
};

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

DecScratch dec_scratch(int T, int K, int F, int Er, int sms) {
  DecScratch s;
  s.hs = 0;
  s.part = up256(size_t(T) * K * F * 2);
  s.ctr = s.part + up256(size_t(2) * sms * T * 256 * 4);
  s.lpart = s.ctr + up256(size_t(2) * sms * 4);
  s.total = s.lpart + up256(size_t(sms) * T * Er * 4);
  return s;
}

bool dec_sizes_ok(int64_t T, int32_t H, int32_t F, int32_t E, int32_t K, int32_t Er) {
  if (T < 0 || T > kDecMaxT || K < 1 || K > kMaxRouteK || T * K > kDecMaxRows) return false;
  if (H <= 0 || H % 8 || H > kDecMaxH || F <= 0 || F % 8 || E < 1 || E > kMaxExperts) return false;
  if (Er < 0 || Er > kMaxExperts || Er % 2 || (Er > 0 && K > Er)) return false;
  // Unit counts stay within 31 bits.
  const int64_t act = E < T * K ? E : T * K;
  const int64_t u1 = act * ((F + 127) / 128) * ((H + 63) / 64), u2 = act * ((H + 255) / 256) * ((F + 63) / 64);
  return u1 <= INT_MAX && u2 <= INT_MAX;
}

bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" int moe_decode_scratch_bytes(int64_t T, int32_t H, int32_t F, int32_t E, int32_t K, int32_t router_experts,
                                        int32_t device, size_t* out) {
  if (!out || !dec_sizes_ok(T, H, F, E, K, router_experts)) return kBadArg;
  int sms = 0;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) return kCudaErr;
  *out = dec_scratch(int(T), K, F, router_experts, sms).total;
  return kOk;
}

extern "C" int moe_decode_layer(const moe_decode_params* p, void* stream) {
  if (!p) return kBadArg;
  const int Er = p->router_w ? p->router_experts : 0;
  if (!dec_sizes_ok(p->T, p->hidden, p->ffn, p->experts, p->K, Er)) return kBadArg;
  if (p->router_w && Er < 2) return kBadArg;
  if (p->T == 0) return kOk;
  if (!p->x || !p->w13 || !p->w2 || !p->y || !p->top_idxs || !p->top_vals || !p->scratch) return kBadArg;
  if (misaligned(p->x) || misaligned(p->w13) || misaligned(p->w2) || misaligned(p->scratch)) return kBadArg;
  if (p->router_w && ((reinterpret_cast<uintptr_t>(p->router_w) & 3) || p->vals_are_bf16)) return kBadArg;
  if (!driver().ok) return kCudaErr;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return kCudaErr;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return kCudaErr;
  const int T = int(p->T), H = p->hidden, F = p->ffn, E = p->experts, K = p->K;
  const DecScratch sc = dec_scratch(T, K, F, Er, sms);
  if (p->scratch_bytes < sc.total) return kBadArg;
  unsigned char* base = static_cast<unsigned char*>(p->scratch);

  DecArgs a = {};
  a.T = T;
  a.H = H;
  a.F = F;
  a.E = E;
  a.K = K;
  a.first = p->first_expert;
  a.NB = (T + 15) / 16 * 16;
  a.x = static_cast<const __nv_bfloat16*>(p->x);
  a.ids = p->top_idxs;
  a.vals = p->top_vals;
  a.ids64 = p->ids_are_int64;
  a.vals_bf16 = p->vals_are_bf16;
  a.hs = reinterpret_cast<__nv_bfloat16*>(base + sc.hs);
  a.part = reinterpret_cast<float*>(base + sc.part);
  a.ctr = reinterpret_cast<uint32_t*>(base + sc.ctr);
  a.lpart = reinterpret_cast<float*>(base + sc.lpart);
  a.y = static_cast<__nv_bfloat16*>(p->y);
  a.status_host = p->status_host;
  a.router_w = static_cast<const __nv_bfloat16*>(p->router_w);
  a.Er = Er;
  a.renorm = p->renormalize;
  a.out_ids = p->top_idxs;
  a.out_vals = static_cast<float*>(p->top_vals);
  a.maxact = E < T * K ? E : T * K;
  a.stage_bytes = kDecABytes + uint32_t(a.NB) * 128;
  // Pass 2's sums [T][256] and, before them, the masks and offsets of the
  // routing tables and one token's logits.
  uint32_t scratch = uint32_t(T) * 1024;
  const uint32_t build = uint32_t(E) * 10 + 16, logits = uint32_t(Er) * 4;
  if (scratch < build) scratch = build;
  if (scratch < logits) scratch = logits;
  a.scratch_bytes = (scratch + 15) / 16 * 16;
  const uint32_t fixed = 1024 + a.scratch_bytes + dec_table_bytes(a.maxact, T * K) + uint32_t(sizeof(DecSmem));
  int stages = int((kDecMaxSmem - fixed) / a.stage_bytes);
  a.stages = stages > kDecMaxStages ? kDecMaxStages : stages;
  if (a.stages < 2) return kBadArg;
  const uint32_t smem = fixed + uint32_t(a.stages) * a.stage_bytes;
  // The router's slices use the stage memory.
  if (Er && uint32_t(a.stages) * a.stage_bytes < kDecThreads * 2 * kDecTokChunk * 4 + uint32_t(T) * ((H + sms - 1) / sms + 1) * 4)
    return kBadArg;

  CUtensorMap m13, m2, mx, mh;
  {
    const cuuint64_t dims[4] = {cuuint64_t(F), cuuint64_t(H), 2, cuuint64_t(E)};
    const cuuint64_t str[3] = {cuuint64_t(F) * 4, cuuint64_t(F) * 2, cuuint64_t(H) * F * 4};
    const cuuint32_t box[4] = {64, 64, 2, 1};
    if (encode(&m13, 4, p->w13, dims, str, box)) return kCudaErr;
  }
  a.w2_atoms = H % 64 == 0;
  if (a.w2_atoms) {
    const cuuint64_t dims[4] = {64, cuuint64_t(F), cuuint64_t(H / 64), cuuint64_t(E)};
    const cuuint64_t str[3] = {cuuint64_t(H) * 2, 128, cuuint64_t(H) * F * 2};
    const cuuint32_t box[4] = {64, 64, 4, 1};
    if (encode(&m2, 4, p->w2, dims, str, box)) return kCudaErr;
  } else {
    const cuuint64_t dims[3] = {cuuint64_t(H), cuuint64_t(F), cuuint64_t(E)};
    const cuuint64_t str[2] = {cuuint64_t(H) * 2, cuuint64_t(H) * F * 2};
    const cuuint32_t box[3] = {64, 64, 1};
    if (encode(&m2, 3, p->w2, dims, str, box)) return kCudaErr;
  }
  {
    const cuuint64_t dims[2] = {cuuint64_t(H), cuuint64_t(T)};
    const cuuint64_t str[1] = {cuuint64_t(H) * 2};
    const cuuint32_t box[2] = {64, cuuint32_t(a.NB)};
    if (encode(&mx, 2, p->x, dims, str, box)) return kCudaErr;
  }
  {
    const cuuint64_t dims[2] = {cuuint64_t(F), cuuint64_t(T) * K};
    const cuuint64_t str[1] = {cuuint64_t(F) * 2};
    const cuuint32_t box[2] = {64, 16};
    if (encode(&mh, 2, a.hs, dims, str, box)) return kCudaErr;
  }
  if (cudaFuncSetAttribute(decode_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)) != cudaSuccess)
    return kCudaErr;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(sms));
  cfg.blockDim = dim3(kDecThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeCooperative;
  at[0].val.cooperative = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, decode_kernel, m13, m2, mx, mh, a) == cudaSuccess ? kOk : kCudaErr;
}
