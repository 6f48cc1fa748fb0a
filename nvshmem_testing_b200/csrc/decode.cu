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
//           tokens the B operand; h = silu(gate) * up is written for the
//           tokens that chose the expert only.
//   pass 2  units (256 features of H, active expert, 64 of F): the rows of
//           h of one expert are B; the epilogue adds v * D to an fp32 sum
//           per token and feature in shared memory, so that the experts'
//           outputs meet without leaving the CTA.
// h passes as two bf16 values, its rounding and what that leaves: beside bf16
// weights the MMA takes bf16 only, and one value alone would double the
// squared error of the result (2-norm 0.0023; with two 0.0017, the rounding
// of y).  An expert's n rows and their n remainders lie next to each other,
// so that up to eight rows per expert are one 16-row block as before (one
// token, 64 experts: 35.6 -> 35.9 us; 48 tokens over 16 experts: 68.9 -> 69.9;
// 64 rows in each of four experts: 80.5 -> 83).
// Each pass splits its list of 32 KB units evenly over the CTAs, at any k:
// every SM streams the same number of bytes whatever the number of experts
// or tiles.  SMs do not get the same bandwidth, though (those of the fuller
// GPCs up to 14 % less, always the same ones), so of a long list the last
// eighth is left in small chunks for whoever is done first (7 tokens, 8
// experts of 352 MB: 410 -> 392 us; 705 MB in all: no gain), and more where
// the rows' alignment sets the SMs further apart.  A tile that ends
// up in several parts is summed from fp32 partials in the order of the list,
// so results depend neither on timing nor on who did what: in pass 1 by the
// last of its CTAs (few parts, few rows; otherwise by the grid), in pass 2,
// where 256 features may be spread over all CTAs, by the grid after another
// barrier.  The grid barriers are cooperative groups': the launch guarantees
// that all CTAs are resident, every wait of a CTA's own is bounded, and after
// an error a CTA skips work, not barriers.
// The weights' first stages of a pass are requested before the barrier in
// front of it; only the token rows wait for it.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <climits>
#include <type_traits>

#include "decode_parts.h"
#include "moe_ep.h"
#include "moe_ep_internal.h"
#include "ptx.cuh"

namespace moe {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxDevices = 64;
constexpr int kDecMaxT = 64;
constexpr int kDecMaxRows = 1024;                 // T * K
constexpr int kDecMaxH = 32768;
constexpr int kDecEpiWarps = 8;                   // two per TMEM lane quarter
constexpr int kDecEpi0 = 2;                       // warps: 0 loads, 1 MMA, 2.. epilogue
constexpr int kDecThreads = (kDecEpi0 + kDecEpiWarps) * 32;
constexpr int kDecMaxStages = 8;
constexpr uint32_t kDecABytes = 256 * 64 * 2;     // 256 features x 64 K
constexpr uint32_t kDecMaxSmem = 226 * 1024;      // dynamic; under 1 KB is static
constexpr int kDecTokChunk = 8;                   // router: tokens whose logits a thread sums at a time
constexpr uint64_t kDecBoundNs = 2000000000ull;   // bug guard on every pipeline wait
constexpr int kBarEpi = 1;

struct DecArgs {
  int T, H, F, E, K, first;  // E: experts held here
  int NB;                    // T rounded to 16: B rows and MMA N of pass 1
  int NB2;                   // 2 * T rounded to 16: the most of pass 2
  int stages;
  uint32_t stage_bytes, scratch_bytes;
  int maxact;                // min(E, T * K)
  const __nv_bfloat16* x;
  const void* ids;
  const void* vals;
  int ids64, vals_bf16;
  __nv_bfloat16* hs;         // [2*T*K][F]: an expert's n rows, then their remainders
  float* part;               // [2 * (grid + kDecMaxChunks)][T][256]
  uint32_t* ctr;             // [grid + kDecMaxChunks] tickets of pass 1's split tiles, [2] chunks handed out
  __nv_bfloat16* y;
  int32_t* status_host;
  // Routed form (router_w != nullptr).
  const __nv_bfloat16* router_w;  // [H, Er]
  int Er, renorm;
  int eparts;                // the router's experts in this many slices, H in grid / eparts
  float* lpart;              // [grid / eparts][T][Er]
  void* out_ids;
  float* out_vals;
};

struct alignas(16) DecSmem {
  uint64_t full[kDecMaxStages];
  uint64_t empty[kDecMaxStages];
  uint64_t tfull[2];
  uint64_t tempty[2];
  uint64_t drain;
  uint64_t run[kDecRunSlots];   // a chunk (or the end) has been taken
  int chunk[kDecRunSlots];
  uint32_t fills[kDecMaxStages];
  uint32_t tmem_base;
  int err;
  int nact;
  int last;
};

// The kernel runs most of its code once per launch, from a cold instruction
// cache: what is not in a unit's path is kept small (out of line, not
// unrolled).
__device__ __noinline__ bool dec_wait_slow(uint64_t* bar, uint32_t parity, DecSmem& sm) {
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
__device__ __forceinline__ bool dec_wait(uint64_t* bar, uint32_t parity, DecSmem& sm) {
  return mbar_try_wait(bar, parity) || dec_wait_slow(bar, parity, sm);
}

__device__ __noinline__ void dec_fail(DecSmem& sm, const DecArgs& a, int detail) {
  if (atomicExch(&sm.err, 1) == 0 && a.status_host)
    *reinterpret_cast<volatile int32_t*>(a.status_host) = int32_t(status_word(kTimeout, kSitePipe, detail));
}

__device__ __forceinline__ float silu_mul(float g, float u) { return g / (1.f + expf(-g)) * u; }

// h as the sum of two bf16 values: its rounding, and what that leaves (nothing
// where it left the finite numbers).
__device__ __forceinline__ __nv_bfloat16 rest_of(float h, __nv_bfloat16 hi) {
  const float r = h - __bfloat162float(hi);
  return __float2bfloat16_rn(fabsf(r) < INFINITY ? r : 0.f);
}
__device__ __forceinline__ void store_h(__nv_bfloat16* at, size_t to_rest, float h) {
  const __nv_bfloat16 hi = __float2bfloat16_rn(h);
  at[0] = hi;
  at[to_rest] = rest_of(h, hi);
}
__device__ __forceinline__ void store_h4(__nv_bfloat16* at, size_t to_rest, float4 g, float4 u) {
  const float h[4] = {silu_mul(g.x, u.x), silu_mul(g.y, u.y), silu_mul(g.z, u.z), silu_mul(g.w, u.w)};
  __nv_bfloat16 hi[4], lo[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    hi[i] = __float2bfloat16_rn(h[i]);
    lo[i] = rest_of(h[i], hi[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    *reinterpret_cast<__nv_bfloat162*>(at + i) = __nv_bfloat162(hi[i], hi[i + 1]);
    *reinterpret_cast<__nv_bfloat162*>(at + to_rest + i) = __nv_bfloat162(lo[i], lo[i + 1]);
  }
}

// Adds the values of the lane `o` away to this lane's (the same sum in both).
__device__ __forceinline__ void add_xor(float4& v, int o) {
  v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
  v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  v.z += __shfl_xor_sync(0xffffffffu, v.z, o);
  v.w += __shfl_xor_sync(0xffffffffu, v.w, o);
}

// The sum of parts lo..hi in order, `at(q)` giving part q's address: eight
// loads in flight at a time, the last group's too.
template <typename V, typename At>
__device__ __forceinline__ V sum_parts(int lo, int hi, At at) {
  V sum = {};
#pragma unroll 1
  for (int q = lo; q <= hi; q += 8) {
    V v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = q + j <= hi ? __ldcg(at(q + j)) : V{};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (sizeof(V) == 4) {
        sum += v[j];
      } else {
        sum.x += v[j].x;
        sum.y += v[j].y;
        if constexpr (sizeof(V) == 16) {
          sum.z += v[j].z;
          sum.w += v[j].w;
        }
      }
    }
  }
  return sum;
}

__device__ __forceinline__ long long load_id(const void* ids, int ids64, int i) {
  return ids64 ? static_cast<const long long*>(ids)[i] : static_cast<const int*>(ids)[i];
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
// token, the same in every CTA.  The routing is read once, into shared
// memory.
__device__ void dec_build(const DecArgs& a, DecSmem& sm, const DecTables& tb, unsigned char* scratch, const void* ids,
                          int ids64, const void* vals, int vals_bf16) {
  if (a.T * a.K <= 32) {
    // Few rows: one warp sorts them by expert, then token, by counting.
    const int lane = threadIdx.x;
    if (lane < 32) {
      const int n = a.T * a.K, t = lane / a.K;
      long long e = -1;
      float v = 0.f;
      if (lane < n) {
        e = load_id(ids, ids64, lane) - a.first;
        v = vals_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(vals)[lane])
                      : static_cast<const float*>(vals)[lane];
      }
      // The order of a row: expert, token, and (an id repeated within a
      // token's row counts once) its first place; what is not held here last.
      const uint32_t key = e >= 0 && e < a.E ? uint32_t(e) * 32 + uint32_t(t) : 0xffffffffu;
      const uint32_t same = __match_any_sync(0xffffffffu, key);
      const bool on = key != 0xffffffffu && (same & ((1u << lane) - 1)) == 0;
      const uint32_t expert = on ? key >> 5 : 0xffffffffu;
      const uint32_t peers = __match_any_sync(0xffffffffu, expert);  // rows of the same expert
      const bool head = on && (peers & ((1u << lane) - 1)) == 0;
      int row = 0, at = 0;
#pragma unroll 4
      for (int j = 0; j < 32; ++j) {
        const uint32_t kj = __shfl_sync(0xffffffffu, on ? key : 0xffffffffu, j);
        const uint32_t hj = __shfl_sync(0xffffffffu, head ? expert : 0xffffffffu, j);
        row += on && kj < key;
        at += on && hj < expert;
      }
      if (on) {
        tb.tok[row] = uint8_t(t);
        tb.val[row] = v;
      }
      // Rows of an expert are ascending by token: its head is the first.
      if (head) {
        tb.act_e[at] = uint16_t(expert);
        tb.act_off[at] = uint16_t(row);
      }
      const uint32_t ons = __ballot_sync(0xffffffffu, on), heads = __ballot_sync(0xffffffffu, head);
      if (lane == 0) {
        tb.act_off[__popc(heads)] = uint16_t(__popc(ons));
        sm.nact = __popc(heads);
      }
    }
    __syncthreads();
    return;
  }
  unsigned long long* mask = reinterpret_cast<unsigned long long*>(scratch);  // [E]
  float* v = reinterpret_cast<float*>(mask + a.E);                            // [T*K]
  uint16_t* off_e = reinterpret_cast<uint16_t*>(v + a.T * a.K);               // [E]
  int16_t* loc = reinterpret_cast<int16_t*>(off_e + a.E);                     // [T*K] expert here, or -1
  const int tid = threadIdx.x, n = a.T * a.K;
#pragma unroll 1
  for (int i = tid; i < n; i += kDecThreads) {
    const long long e = load_id(ids, ids64, i) - a.first;
    v[i] = vals_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(vals)[i])
                     : static_cast<const float*>(vals)[i];
    loc[i] = e >= 0 && e < a.E ? int16_t(e) : int16_t(-1);
  }
#pragma unroll 1
  for (int e = tid; e < a.E; e += kDecThreads) mask[e] = 0;
  __syncthreads();
#pragma unroll 1
  for (int i = tid; i < n; i += kDecThreads)
    if (loc[i] >= 0) atomicOr(&mask[loc[i]], 1ull << (i / a.K));
  __syncthreads();
  if (tid < 32) {
    int act = 0, row = 0;
#pragma unroll 1
    for (int e0 = 0; e0 < a.E; e0 += 32) {
      const int e = e0 + tid;
      const int c = e < a.E ? __popcll(mask[e]) : 0;
      const uint32_t live = __ballot_sync(0xffffffffu, c > 0);
      if (live == 0) continue;
      int pre = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, pre, o);
        if (tid >= o) pre += u;
      }
      if (c > 0) {
        const int at = act + __popc(live & ((1u << tid) - 1));
        off_e[e] = uint16_t(row + pre - c);
        tb.act_e[at] = uint16_t(e);
        tb.act_off[at] = uint16_t(row + pre - c);
      }
      act += __popc(live);
      row += __shfl_sync(0xffffffffu, pre, 31);
    }
    if (tid == 0) {
      tb.act_off[act] = uint16_t(row);
      sm.nact = act;
    }
  }
  __syncthreads();
#pragma unroll 1
  for (int i = tid; i < n; i += kDecThreads) {
    const int e = loc[i];
    if (e < 0) continue;
    const int t = i / a.K;
    bool again = false;
#pragma unroll 1
    for (int j = t * a.K; j < i; ++j) again |= loc[j] == e;
    if (again) continue;
    const int r = off_e[e] + __popcll(mask[e] & ((1ull << t) - 1));
    tb.tok[r] = uint8_t(t);
    tb.val[r] = v[i];
  }
  __syncthreads();
}

// Router, step 1: one slice of H of the logits of one slice of the experts,
// for every token, in fp32.  A thread holds two neighbouring experts and
// eight tokens; the threads left over take other tokens, then other rows of
// the slice, whose sums are added in a fixed order.
__device__ void dec_router_partial(const DecArgs& a, unsigned char* stage) {
  const int hparts = int(gridDim.x) / a.eparts, hp = int(blockIdx.x) / a.eparts, tid = threadIdx.x;
  if (hp >= hparts) return;
  const int Es = a.Er / a.eparts, e0 = (int(blockIdx.x) % a.eparts) * Es;
  const int h0 = int(int64_t(a.H) * hp / hparts), nh = int(int64_t(a.H) * (hp + 1) / hparts) - h0;
  float* red = reinterpret_cast<float*>(stage);                       // [groups][cpar][8][Es]
  float* xs = red + kDecThreads * 2 * kDecTokChunk;                   // [chunk][nh][8]
  const int chunks = (a.T + kDecTokChunk - 1) / kDecTokChunk;
#pragma unroll 1
  for (int i = tid; i < chunks * kDecTokChunk * nh; i += kDecThreads) {
    const int t = i / nh, h = i - t * nh;
    xs[((t / kDecTokChunk) * nh + h) * kDecTokChunk + t % kDecTokChunk] =
        t < a.T ? __bfloat162float(a.x[int64_t(t) * a.H + h0 + h]) : 0.f;
  }
  __syncthreads();
  const int P = Es / 2, rest = tid / P;
  const bool wide = P >= kDecThreads;  // more experts than threads: rounds over them instead
  const int cpar = wide ? 1 : min(chunks, kDecThreads / P);
  const int groups = wide ? 1 : kDecThreads / (P * cpar);
  const int cc = wide ? 0 : rest % cpar, grp = wide ? 0 : rest / cpar;
#pragma unroll 1
  for (int cb = 0; cb < chunks; cb += cpar) {
    const int ch = cb + cc;
#pragma unroll 1
    for (int p0 = 0; p0 < P; p0 += kDecThreads) {
      const int p = wide ? p0 + tid : tid - rest * P;
      const bool on = ch < chunks && (wide ? p < P : grp < groups);
      float2 s[kDecTokChunk];
#pragma unroll
      for (int j = 0; j < kDecTokChunk; ++j) s[j] = make_float2(0.f, 0.f);
      if (on) {
        const __nv_bfloat162* r =
            reinterpret_cast<const __nv_bfloat162*>(a.router_w + int64_t(h0) * a.Er + e0) + p;
        const int P0 = a.Er / 2;
        // Eight rows' loads in flight; rows past the slice count as zeros.
#pragma unroll 1
        for (int hb = grp; hb < nh; hb += 8 * groups) {
          __nv_bfloat162 w8[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int h = hb + i * groups;
            w8[i] = h < nh ? r[int64_t(h) * P0] : __nv_bfloat162{};
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int h = hb + i * groups;
            const float2 w = __bfloat1622float2(w8[i]);
            const float4* xv = reinterpret_cast<const float4*>(xs + (ch * nh + min(h, nh - 1)) * kDecTokChunk);
            float xr[kDecTokChunk];
#pragma unroll
            for (int j = 0; j < kDecTokChunk; j += 4)
              *reinterpret_cast<float4*>(&xr[j]) = h < nh ? xv[j / 4] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int j = 0; j < kDecTokChunk; ++j) {
              s[j].x = fmaf(xr[j], w.x, s[j].x);
              s[j].y = fmaf(xr[j], w.y, s[j].y);
            }
          }
        }
      }
      if (groups > 1) {
        if (on) {
#pragma unroll
          for (int j = 0; j < kDecTokChunk; ++j)
            *reinterpret_cast<float2*>(&red[((grp * cpar + cc) * kDecTokChunk + j) * Es + 2 * p]) = s[j];
        }
        __syncthreads();
#pragma unroll 1
        for (int i = tid; i < cpar * kDecTokChunk * Es; i += kDecThreads) {
          const int j = i / Es, t = cb * kDecTokChunk + j, e = i - j * Es;
          if (t >= a.T) break;
          float v = 0.f;
#pragma unroll 4
          for (int g = 0; g < groups; ++g) v += red[(g * cpar * kDecTokChunk + j) * Es + e];
          a.lpart[(int64_t(hp) * a.T + t) * a.Er + e0 + e] = v;
        }
        __syncthreads();
      } else if (on) {
#pragma unroll
        for (int j = 0; j < kDecTokChunk; ++j) {
          const int t = ch * kDecTokChunk + j;
          if (t < a.T) *reinterpret_cast<float2*>(&a.lpart[(int64_t(hp) * a.T + t) * a.Er + e0 + 2 * p]) = s[j];
        }
      }
    }
  }
}

// A logit's bits as an unsigned number of the same order (-0 and 0 alike, NaN
// lowest).
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t bits = __float_as_uint(v + 0.f);
  return v != v ? 0u : (bits >> 31) ? ~bits : (bits | 0x80000000u);
}
constexpr int kDecCountExperts = 128;

// Router, step 2: tokens t0, t0 + stride, ...: the slices' sum in order, the
// softmax over Er in fp32 and the K largest (equal logits: lowest id first).
// The last
// token's routing also stays in `keep`.
struct DecRouted {
  long long id[kMaxRouteK];
  float val[kMaxRouteK];
};
__device__ void dec_router_topk(const DecArgs& a, unsigned char* stage, unsigned char* scratch, int t0, int stride,
                                bool store, DecRouted& keep) {
  const int hparts = int(gridDim.x) / a.eparts, tid = threadIdx.x, lane = tid & 31;
  float* red = reinterpret_cast<float*>(stage);              // [parts][Er]
  float* lg = reinterpret_cast<float*>(scratch);             // [Er]
  uint2* cand = reinterpret_cast<uint2*>(lg + a.Er);         // [groups][K] (key, id)
  __shared__ int chosen[kMaxRouteK];
  __shared__ float norm[2];
  const int E4 = a.Er / 4;  // four experts per load
  const int parts = kDecThreads / E4;
  float4* red4 = reinterpret_cast<float4*>(red);
#pragma unroll 1
  for (int t = t0; t < a.T; t += stride) {
    if (tid < parts * E4) {
      const int q = tid / E4, e = tid - q * E4;
      const float4* at = reinterpret_cast<const float4*>(a.lpart + int64_t(t) * a.Er) + e;
      const int64_t step = int64_t(a.T) * E4;
      red4[tid] = sum_parts<float4>(hparts * q / parts, hparts * (q + 1) / parts - 1,
                                    [&](int c) { return at + c * step; });
    }
    __syncthreads();
#pragma unroll 1
    for (int e = tid; e < a.Er; e += kDecThreads) {
      float v = 0.f;
#pragma unroll 4
      for (int q = 0; q < parts; ++q) v += red[q * a.Er + e];
      lg[e] = v;
    }
    __syncthreads();
    // Few experts: an expert's place is the number of those before it,
    // counted by one thread each.  More (256: 5.3 us against 4.0): the K
    // largest of every 32, a warp each, then K times the largest of those.
    const int warp = tid >> 5, warps = kDecThreads / 32, groups = a.Er <= kDecCountExperts ? 0 : (a.Er + 31) / 32;
    if (groups == 0 && tid < a.Er) {
      const uint32_t mine = order_key(lg[tid]);
      int before = 0;
#pragma unroll 4
      for (int i = 0; i < E4; ++i) {  // a key before mine, or the same one at a lower id
        const float4 k = reinterpret_cast<const float4*>(lg)[i];
        before += int(order_key(k.x) >= mine + (4 * i >= tid)) + int(order_key(k.y) >= mine + (4 * i + 1 >= tid)) +
                  int(order_key(k.z) >= mine + (4 * i + 2 >= tid)) + int(order_key(k.w) >= mine + (4 * i + 3 >= tid));
      }
      if (before < a.K) chosen[before] = tid;
    }
#pragma unroll 1
    for (int g = warp; g < groups; g += warps) {
      const int e = g * 32 + lane;
      bool open = e < a.Er;
      const uint32_t key = order_key(open ? lg[e] : 0.f);
#pragma unroll 1
      for (int k = 0; k < a.K; ++k) {
        const uint32_t top = __reduce_max_sync(0xffffffffu, open ? key : 0u);
        const uint32_t have = __ballot_sync(0xffffffffu, open && key == top);
        if (have == 0) {  // fewer than K in the group
          if (lane == 0) cand[g * a.K + k] = make_uint2(0u, INT_MAX);
        } else if (lane == __ffs(have) - 1) {  // equal logits: the lowest id
          cand[g * a.K + k] = make_uint2(key, uint32_t(e));
          open = false;
        }
      }
    }
    if (groups > 0) __syncthreads();
    if (tid < 32) {
      // (An id of INT_MAX: taken, or none.)
      const int n = groups * a.K;
#pragma unroll 1
      for (int k = 0; k < a.K && groups > 0; ++k) {
        uint32_t best = 0, be = INT_MAX;
        int at = 0;
#pragma unroll 1
        for (int i = lane; i < n; i += 32) {
          const uint2 c = cand[i];
          if (c.y != INT_MAX && (be == INT_MAX || c.x > best || (c.x == best && c.y < be))) {
            best = c.x;
            be = c.y;
            at = i;
          }
        }
        const uint32_t top = __reduce_max_sync(0xffffffffu, best);
        const uint32_t pick = __reduce_min_sync(0xffffffffu, best == top ? be : INT_MAX);
        if (best == top && be == pick) cand[at].y = INT_MAX;
        if (lane == 0) chosen[k] = int(pick);
      }
      __syncwarp();
    } else if (tid < 64) {
      float m = -INFINITY;
#pragma unroll 1
      for (int e = lane; e < a.Er; e += 32) m = fmaxf(m, lg[e]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      float z = 0.f;
#pragma unroll 1
      for (int e = lane; e < a.Er; e += 32) z += expf(lg[e] - m);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
      if (lane == 0) {
        norm[0] = m;
        norm[1] = z;
      }
    }
    __syncthreads();
    if (tid < 32) {
      const float m = norm[0], z = norm[1];
      const int id = lane < a.K ? chosen[lane] : 0;
      const float pr = lane < a.K ? expf(lg[id] - m) / z : 0.f;
      float sum = pr;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane < a.K) {
        const int64_t o = int64_t(t) * a.K + lane;
        const float v = a.renorm ? pr / sum : pr;
        keep.id[lane] = id;
        keep.val[lane] = v;
        if (store) {
          a.out_vals[o] = v;
          if (a.ids64) static_cast<long long*>(a.out_ids)[o] = id;
          else static_cast<int*>(a.out_ids)[o] = id;
        }
      }
    }
    __syncthreads();
  }
}

// A position in a pass, moved on by additions: the loads and the MMAs each
// run in one thread, whose integer divisions (two per unit and more) took
// longer than a unit's share of the memory bandwidth.
struct Cursor {
  int ai, ft, k;  // active expert, tile of features, K
};
template <int PASS>
__device__ __forceinline__ Cursor cursor_at(const Pass& p, int nact, int u) {
  Cursor c;
  const int x = u / p.kb;
  c.k = u - x * p.kb;
  const int in = PASS == 1 ? p.nt : nact;
  const int hi = in > 0 ? x / in : 0;
  c.ai = PASS == 1 ? hi : x - hi * in;
  c.ft = PASS == 1 ? x - hi * in : hi;
  return c;
}
template <int PASS>
__device__ __forceinline__ void cursor_next_k(Cursor& c, const Pass& p, int nact) {  // the next run over K
  c.k = 0;
  if (PASS == 1) {
    if (++c.ft == p.nt) {
      c.ft = 0;
      ++c.ai;
    }
  } else {
    if (++c.ai == nact) {
      c.ai = 0;
      ++c.ft;
    }
  }
}
template <int PASS>
__device__ __forceinline__ void cursor_next(Cursor& c, const Pass& p, int nact) {
  if (++c.k == p.kb) cursor_next_k<PASS>(c, p, nact);
}

// The stage a thread has reached, and the parity of its round.
struct Ring {
  int st;
  uint32_t ph;
  __device__ __forceinline__ void next(int n) {
    if (++st == n) {
      st = 0;
      ph ^= 1;
    }
  }
};

__global__ void __launch_bounds__(kDecThreads, 1)
    decode_kernel(const __grid_constant__ CUtensorMap tm_w13, const __grid_constant__ CUtensorMap tm_w2,
                  const __grid_constant__ CUtensorMap tm_w2e,
                  const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_h,
                  const __grid_constant__ DecArgs a) {
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
    for (int i = 0; i < kDecRunSlots; ++i) mbar_init(&sm.run[i], 1);
    sm.err = 0;
    fence_mbar_init();
    prefetch_tensormap(&tm_w13);
    prefetch_tensormap(&tm_x);
    prefetch_tensormap(&tm_w2);
    prefetch_tensormap(&tm_h);
  }
  const uint32_t tmem_cols = a.NB2 <= 16 ? 64 : a.NB2 <= 32 ? 128 : a.NB2 <= 64 ? 256 : 512;
  if (warp == 1) {
    __syncwarp();
    tmem_alloc(&sm.tmem_base, tmem_cols);
    tmem_relinquish();
  }
  // The tickets of split tiles start at zero: written here, ordered before
  // their first use by the first grid barrier.
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < int(gridDim.x) + kDecMaxChunks + 2; i += kDecThreads) a.ctr[i] = 0;

  // (The block meets in each of the following steps before anything of the
  // above is used.)
  const void* ids = a.ids;
  const void* vals = a.vals;
  int ids64 = a.ids64;
  if (a.router_w != nullptr) {
    __shared__ DecRouted routed;
    dec_router_partial(a, stage);
    grid.sync();
    // One token: every CTA finds its experts for itself, which costs less
    // than handing them round through another barrier.
    const bool alone = a.T == 1;
    dec_router_topk(a, stage, scratch, alone ? 0 : blockIdx.x, alone ? 1 : int(gridDim.x), !alone || blockIdx.x == 0,
                    routed);
    fence_proxy_async_smem();  // the stages, written by threads so far, belong to the TMA from here
    if (alone) {
      ids = routed.id;
      vals = routed.val;
      ids64 = 1;
    } else {
      grid.sync();
    }
  }
  dec_build(a, sm, tb, scratch, ids, ids64, vals, a.vals_bf16);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  const int nact = sm.nact;
  const int G = gridDim.x;

  const int kb1 = (a.H + 63) / 64, nt1 = (a.F + 127) / 128;
  const int kb2 = (a.F + 63) / 64, nt2 = (a.H + 255) / 256;
  const Pass p1 = make_pass(a.T, G, blockIdx.x, nact * nt1, kb1, kb1, nt1, ragged_rows(a.F));
  const Pass p2 = make_pass(a.T, G, blockIdx.x, nact > 0 ? nt2 : 0, nact * kb2, kb2, nt2, false);
  auto take_run = [&](Runs& r, const Pass& p, int pass) {
    if (p.chunks == 0) return false;
    int chunk = int(atomicAdd(&a.ctr[G + kDecMaxChunks + pass - 1], 1u));
    if (chunk >= p.chunks) chunk = -1;
    sm.chunk[r.n % kDecRunSlots] = chunk;
    mbar_arrive(&sm.run[r.n % kDecRunSlots]);
    ++r.n;
    return set_run(r, p, chunk);
  };
  auto next_chunk = [&](Runs& r, const Pass& p) {
    return follow_run(
        r, p, [&](int slot, uint32_t parity) { return dec_wait(&sm.run[slot], parity, sm); },
        [&](int slot) { return *reinterpret_cast<volatile int*>(&sm.chunk[slot]); }, [&] { dec_fail(sm, a, 6); });
  };
  auto act_rows = [&](int ai) { return int(tb.act_off[ai + 1]) - int(tb.act_off[ai]); };
  auto blocks2 = [&](int ai) { return (2 * act_rows(ai) + 15) >> 4; };  // of 16 B rows in pass 2

  // ---- loads (one thread)
  Ring lr = {0, 0};  // next stage to fill
  // Weights are read once: they leave L2 first, so that activations, partial
  // sums and the kernel's own code stay.
  const uint64_t once = l2_policy_evict_first();
  // A unit's weights into the next stage; the stage's expected bytes include
  // the rows that load_rows adds.
  auto load_weights = [&](auto pass, const Cursor& c) -> bool {
    constexpr int PASS = decltype(pass)::value;
    uint64_t* full = &sm.full[lr.st];
    if (!dec_wait(&sm.empty[lr.st], lr.ph ^ 1, sm)) {
      dec_fail(sm, a, 1);
      return false;
    }
    unsigned char* dst = stage + uint32_t(lr.st) * a.stage_bytes;
    const int e = tb.act_e[c.ai];
    if constexpr (PASS == 1) {
      // Two boxes of 64 gate and the 64 up features (one of all four atoms
      // was no faster).
      mbar_arrive_expect_tx(full, kDecABytes + uint32_t(a.NB) * 128);
      tma_load_4d_hint(&tm_w13, full, dst, c.ft * 128, c.k * 64, 0, e, once);
      tma_load_4d_hint(&tm_w13, full, dst + 16384, c.ft * 128 + 64, c.k * 64, 0, e, once);
    } else {
      // One box of four atoms of 64 features; a tile whose last atom is a part
      // of one atom by atom, clipped at the row's end.
      mbar_arrive_expect_tx(full, kDecABytes + uint32_t(blocks2(c.ai)) * 2048);
      if (c.ft * 4 + 4 <= a.H / 64) {
        tma_load_4d_hint(&tm_w2, full, dst, 0, c.k * 64, c.ft * 4, e, once);
      } else {
#pragma unroll 1
        for (int g = 0; g < 4; ++g)
          tma_load_3d_hint(&tm_w2e, full, dst + g * 8192, c.ft * 256 + g * 64, c.k * 64, e, once);
      }
    }
    sm.fills[lr.st] += 1;
    lr.next(S);
    return true;
  };
  auto load_rows = [&](auto pass, const Cursor& c, int st) {
    constexpr int PASS = decltype(pass)::value;
    uint64_t* full = &sm.full[st];
    unsigned char* dst = stage + uint32_t(st) * a.stage_bytes + kDecABytes;
    if constexpr (PASS == 1) {
      tma_load_2d(&tm_x, full, dst, c.k * 64, 0);
    } else {
      const int r0 = 2 * tb.act_off[c.ai], nb = blocks2(c.ai);
      for (int b = 0; b < nb; ++b) tma_load_2d(&tm_h, full, dst + b * 2048, c.k * 64, r0 + b * 16);
    }
  };
  // The first stages of a pass: weights only, before the barrier.
  int pre = 0;     // units preloaded
  Ring pre_at = {0, 0};
  auto preload = [&](auto pass, const Pass& p) {
    constexpr int PASS = decltype(pass)::value;
    pre_at = lr;
    pre = 0;
    Cursor c = cursor_at<PASS>(p, nact, p.lo);
    const int n = min(S, p.hi - p.lo);
    for (; pre < n && load_weights(pass, c); ++pre) cursor_next<PASS>(c, p, nact);
  };
  Runs lruns = {0, 0, 0, 0};
  auto produce = [&](auto pass, const Pass& p) {
    constexpr int PASS = decltype(pass)::value;
    Runs& r = lruns;
    first_run(r, p, blockIdx.x);
    do {
      Cursor c = cursor_at<PASS>(p, nact, r.lo);
      for (int u = r.lo; u < r.hi; ++u) {
        if (pre > 0) {
          --pre;
          load_rows(pass, c, pre_at.st);
          pre_at.next(S);
        } else {
          const int st = lr.st;
          if (!load_weights(pass, c)) return;
          load_rows(pass, c, st);
        }
        cursor_next<PASS>(c, p, nact);
      }
    } while (take_run(r, p, PASS));
  };

  // ---- MMA (one thread)
  Ring mr = {0, 0};       // next stage to multiply
  Ring mseg = {0, 0};     // next accumulator (two)
  Runs mruns = {0, 0, 0, 0};
  auto multiply = [&](auto pass, const Pass& p) {
    constexpr int PASS = decltype(pass)::value;
    // Pass 1: box g (64 features of each half) is [gate 64x64][up 64x64];
    // pass 2: four groups of 64 features in order.
    constexpr uint32_t half = PASS == 1 ? 8192 : 16384, group = PASS == 1 ? 16384 : 8192;
    Runs& r = mruns;
    first_run(r, p, blockIdx.x);
    do {
      Cursor c = cursor_at<PASS>(p, nact, r.lo);
      bool begin = true;
      uint32_t idesc = 0;
      for (int u = r.lo; u < r.hi; ++u) {
        if (begin) {
          if (!dec_wait(&sm.tempty[mseg.st], mseg.ph ^ 1, sm)) {
            dec_fail(sm, a, 2);
            return;
          }
          const int n = PASS == 1 ? a.NB : blocks2(c.ai) * 16;
          idesc = make_idesc_mn(/*bf16*/ 1, 128, uint32_t(n), /*A MN-major*/ 1, /*B K-major*/ 0);
        }
        if (!dec_wait(&sm.full[mr.st], mr.ph, sm)) {
          dec_fail(sm, a, 3);
          return;
        }
        tc_fence_after();
        const uint32_t aa = smem_u32(stage + uint32_t(mr.st) * a.stage_bytes), ba = aa + kDecABytes;
        const uint32_t d = tmem + uint32_t(mseg.st) * 2 * uint32_t(a.NB2);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          const uint64_t bd = smem_desc_sw128(ba + kk * 32, 16, 1024);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint64_t ad = smem_desc_sw128(aa + h * half + kk * 2048, group, 1024);
            tc_mma_f16(d + h * uint32_t(a.NB2), ad, bd, idesc, (!begin || kk != 0) ? 1u : 0u);
          }
        }
        tc_commit(&sm.empty[mr.st]);
        mr.next(S);
        begin = c.k + 1 == p.kb;
        if (begin || u + 1 == r.hi) {
          tc_commit(&sm.tfull[mseg.st]);
          mseg.next(2);
        }
        cursor_next<PASS>(c, p, nact);
      }
    } while (next_chunk(r, p));
  };

  // ---- epilogue (8 warps: lane quarter = 32 features of 128; two warps each)
  Ring eseg = {0, 0};
  const int quarter = warp & 3, sub = (warp - kDecEpi0) >> 2;
  const int etid = int(threadIdx.x) - kDecEpi0 * 32;
  const uint32_t tlane = tmem + (uint32_t(quarter * 32) << 16);
  // Of a part's split tiles the one it starts goes to its slot 1, the one it
  // joins to slot 0.
  const size_t slot_floats = size_t(a.T) * 256;
  auto slot = [&](int part, int which) { return a.part + (size_t(part) * 2 + which) * slot_floats; };
  Runs eruns = {0, 0, 0, 0};
  // Every epilogue warp follows the same runs.
  auto next_run = [&](const Pass& p) {
    const bool more = next_chunk(eruns, p);
    return p.chunks != 0 && named_bar_and(kBarEpi, kDecEpiWarps * 32, more);
  };
  auto seg_full = [&](int site) {
    if (named_bar_and(kBarEpi, kDecEpiWarps * 32, dec_wait(&sm.tfull[eseg.st], eseg.ph, sm))) return true;
    dec_fail(sm, a, site);
    return false;
  };
  auto seg_done = [&]() {
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.tempty[eseg.st]);
    eseg.next(2);
  };

  // A short list with many rows per expert: the parts of its few tiles are
  // too much for one CTA each (56 rows of 20 parts: 64 us), so the grid adds
  // them up, behind a barrier of its own.
  const bool spread = nact > 0 && int(tb.act_off[nact]) >= 12 * nact && p1.units < 16 * G;
  auto join1 = [&](const Pass& p) {
    const int warps = kDecThreads / 32;
#pragma unroll 1
    for (int i = int(blockIdx.x) * warps + warp; i < nact * p.nt * kDecMaxT; i += G * warps) {
      const int tile = i / kDecMaxT, j = i % kDecMaxT, ai = tile / p.nt, l4 = lane * 4;
      const int c0 = p.part_of(tile * p.kb), c1 = p.part_of(tile * p.kb + p.kb - 1);
      const int f = (tile - ai * p.nt) * 128 + l4;
      if (j >= act_rows(ai) || c0 == c1) continue;
      auto at = [&](int q) { return reinterpret_cast<const float4*>(slot(q, q == c0 ? 1 : 0) + j * 256 + l4); };
      const float4 g = sum_parts<float4>(c0, c1, at);
      const float4 u = sum_parts<float4>(c0, c1, [&](int q) { return at(q) + 32; });
      if (f < a.F) {
        store_h4(a.hs + size_t(2 * tb.act_off[ai] + j) * a.F + f, size_t(act_rows(ai)) * a.F, g, u);
      }
    }
  };

  auto epilogue1 = [&](const Pass& p) {
    first_run(eruns, p, blockIdx.x);
    do {
      Cursor c = cursor_at<1>(p, nact, eruns.lo);
      for (int u = eruns.lo; u < eruns.hi;) {
        const int tile0 = u - c.k, seg_end = min(eruns.hi, tile0 + p.kb);
        const bool whole = c.k == 0 && seg_end == tile0 + p.kb;
        if (!seg_full(4)) return;
        tc_fence_after();
        const int n = act_rows(c.ai), r0 = tb.act_off[c.ai];
        const int fl = quarter * 32 + lane;              // feature within the tile
        const int f = c.ft * 128 + fl;
        const uint32_t d = tlane + uint32_t(eseg.st) * 2 * uint32_t(a.NB2);
        float* mine = slot(eruns.part, c.k == 0 ? 1 : 0);
        for (int j0 = sub; j0 < n; j0 += 8) {
          uint32_t g[4], w[4];
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (j0 + 2 * q < n) {
              const uint32_t t = tb.tok[r0 + j0 + 2 * q];
              g[q] = tmem_ld_32x32b_x1(d + t);
              w[q] = tmem_ld_32x32b_x1(d + uint32_t(a.NB2) + t);
            }
          tmem_ld_wait();
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int j = j0 + 2 * q;
            if (j >= n) break;
            const float gv = __uint_as_float(g[q]), uv = __uint_as_float(w[q]);
            if (whole) {
              if (f < a.F) store_h(a.hs + size_t(2 * r0 + j) * a.F + f, size_t(n) * a.F, silu_mul(gv, uv));
            } else {
              mine[j * 256 + fl] = gv;
              mine[j * 256 + 128 + fl] = uv;
            }
          }
        }
        seg_done();
        if (!whole && !spread) {
          // The part whose ticket is the tile's last adds them all up.
          const int c0 = p.part_of(tile0), c1 = p.part_of(tile0 + p.kb - 1);
          named_bar_sync(kBarEpi, kDecEpiWarps * 32);
          if (etid == 0) sm.last = atom_add_acq_rel(&a.ctr[c0], 1u) == uint32_t(c1 - c0);
          named_bar_sync(kBarEpi, kDecEpiWarps * 32);
          if (sm.last) {
            // Four gate or up features a thread, neighbours the same ones;
            // many parts: four such pairs, a quarter of the parts each.
            const int np = c1 - c0 + 1, quarters = np > 6 ? 4 : 1, lanes = 2 * quarters;
            const int upper = lane & 1, qt = quarters == 4 ? (lane >> 1) & 3 : 0;
#pragma unroll 1
            for (int i0 = (etid & ~31) / lanes; i0 < n * 32; i0 += kDecEpiWarps * 32 / lanes) {
              const int i = i0 + lane / lanes, j = i >> 5, l4 = (i & 31) * 4, f4 = c.ft * 128 + l4;
              float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
              if (j < n)
                v = sum_parts<float4>(c0 + np * qt / quarters, c0 + np * (qt + 1) / quarters - 1, [&](int q) {
                  return reinterpret_cast<const float4*>(slot(q, q == c0 ? 1 : 0) + j * 256 + upper * 128 + l4);
                });
              if (quarters == 4) {
                add_xor(v, 2);
                add_xor(v, 4);
              }
              float4 w;
              w.x = __shfl_xor_sync(0xffffffffu, v.x, 1);
              w.y = __shfl_xor_sync(0xffffffffu, v.y, 1);
              w.z = __shfl_xor_sync(0xffffffffu, v.z, 1);
              w.w = __shfl_xor_sync(0xffffffffu, v.w, 1);
              if (j < n && upper == 0 && qt == 0 && f4 < a.F) {
                store_h4(a.hs + size_t(2 * r0 + j) * a.F + f4, size_t(n) * a.F, v, w);
              }
            }
          }
        }
        u = seg_end;
        cursor_next_k<1>(c, p, nact);
      }
    } while (next_run(p));
  };

  auto epilogue2 = [&](const Pass& p) {
    const int fl = sub * 128 + quarter * 32 + lane;  // feature within the tile: this thread's alone
    first_run(eruns, p, blockIdx.x);
    do {
      Cursor c = cursor_at<2>(p, nact, eruns.lo);
      for (int u = eruns.lo; u < eruns.hi;) {
        const int tile0 = u - c.ai * p.kb - c.k, tile_end = min(eruns.hi, tile0 + p.tile);
        const bool starts = u == tile0, whole = starts && tile_end == tile0 + p.tile;
        const int f = c.ft * 256 + fl;
#pragma unroll 4
        for (int t = 0; t < a.T; ++t) acc[t * 256 + fl] = 0.f;
        while (u < tile_end) {
          if (!seg_full(5)) return;
          tc_fence_after();
          const int n = act_rows(c.ai), r0 = tb.act_off[c.ai];
          const uint32_t d = tlane + (uint32_t(eseg.st) * 2 + uint32_t(sub)) * uint32_t(a.NB2);
          for (int j0 = 0; j0 < n; j0 += 4) {
            uint32_t v[4], w[4];  // the products of h's two parts
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (j0 + q < n) {
                v[q] = tmem_ld_32x32b_x1(d + uint32_t(j0 + q));
                w[q] = tmem_ld_32x32b_x1(d + uint32_t(n + j0 + q));
              }
            tmem_ld_wait();
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              if (j0 + q >= n) break;
              float* s = &acc[int(tb.tok[r0 + j0 + q]) * 256 + fl];
              *s = fmaf(tb.val[r0 + j0 + q], __uint_as_float(v[q]) + __uint_as_float(w[q]), *s);
            }
          }
          seg_done();
          u = min(tile_end, u + p.kb - c.k);
          cursor_next_k<2>(c, p, nact);
        }
        if (whole) {
          if (f < a.H)
#pragma unroll 4
            for (int t = 0; t < a.T; ++t) a.y[size_t(t) * a.H + f] = __float2bfloat16_rn(acc[t * 256 + fl]);
        } else {
          float* mine = slot(eruns.part, starts ? 1 : 0);
#pragma unroll 4
          for (int t = 0; t < a.T; ++t) mine[t * 256 + fl] = acc[t * 256 + fl];
        }
      }
    } while (next_run(p));
  };

  // y of the tiles that lie in several parts: four features per four
  // threads, each of which adds a quarter of the parts.
  auto join2 = [&](const Pass& p) {
    const int per = a.T * 64, total = p.nt * per;
#pragma unroll 1
    for (int i0 = (int(blockIdx.x) * kDecThreads + int(threadIdx.x & ~31u)) >> 2; i0 < total;
         i0 += (G * kDecThreads) >> 2) {
      const int i = i0 + (lane >> 2), qt = lane & 3;
      const int tile = i / per, r = i - tile * per;
      const int t = r >> 6, fl = (r & 63) * 4, f = tile * 256 + fl;
      const int u0 = tile * p.tile;
      int c0 = 0, c1 = 0;
      if (i < total) {
        c0 = p.part_of(u0);
        c1 = p.part_of(u0 + p.tile - 1);
      }
      const bool split = c0 != c1;
      const int n = split ? c1 - c0 + 1 : 0;
      float4 v = sum_parts<float4>(c0 + n * qt / 4, c0 + n * (qt + 1) / 4 - 1, [&](int q) {
        return reinterpret_cast<const float4*>(slot(q, q == c0 ? 1 : 0) + t * 256 + fl);
      });
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) add_xor(v, o);
      if (split && f < a.H && qt == 0) {
        __nv_bfloat162* o = reinterpret_cast<__nv_bfloat162*>(a.y + size_t(t) * a.H + f);
        o[0] = __floats2bfloat162_rn(v.x, v.y);
        o[1] = __floats2bfloat162_rn(v.z, v.w);
      }
    }
  };

  // ---- the two passes
  using Pass1 = std::integral_constant<int, 1>;
  using Pass2 = std::integral_constant<int, 2>;
  if (threadIdx.x == 0) preload(Pass1{}, p1);
  __syncwarp();
  if (a.router_w == nullptr) grid.sync();  // (routed: the router's barriers ordered the tickets)
  if (warp == 0 && lane == 0) produce(Pass1{}, p1);
  else if (warp == 1 && lane == 0) multiply(Pass1{}, p1);
  else if (warp >= kDecEpi0) epilogue1(p1);
  __syncwarp();
  if (threadIdx.x == 0 && !*reinterpret_cast<volatile int*>(&sm.err)) preload(Pass2{}, p2);
  __syncwarp();
  if (spread) {
    grid.sync();
    join1(p1);
  }
  fence_proxy_async_global();  // h, written by threads, is read by the TMA
  grid.sync();
  if (!*reinterpret_cast<volatile int*>(&sm.err)) {
    if (warp == 0 && lane == 0) {
      fence_proxy_async_global();
      produce(Pass2{}, p2);
    } else if (warp == 1 && lane == 0) {
      multiply(Pass2{}, p2);
    } else if (warp >= kDecEpi0) {
      epilogue2(p2);
    }
  }
  __syncwarp();
  grid.sync();
  join2(p2);
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

// How much a miss brings into L2: 256 bytes where rows are multiples of that,
// else what is asked for with as little around it as the map allows.  Around
// pieces that start inside a 256-byte block lie columns that another CTA reads
// at another time, by when they are gone from L2 again (25 tokens, 64 experts,
// H 4352: F 1200 289 us with 256, 270 with 64; F 1184 271 and 254; aligned
// rows are up to 2 % faster with 256: 132.7 and 135.5 us at one token, 8 of
// 256 experts).
CUtensorMapL2promotion promotion(int row_bytes) {
  return row_bytes % 256 == 0 ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : CU_TENSOR_MAP_L2_PROMOTION_L2_64B;
}

int encode(CUtensorMap* m, int rank, const void* ptr, const cuuint64_t* dims, const cuuint64_t* strides,
           const cuuint32_t* box, int row_bytes) {
  const cuuint32_t one[5] = {1, 1, 1, 1, 1};
  return driver().cuTensorMapEncodeTiled(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, cuuint32_t(rank),
                                         const_cast<void*>(ptr), dims, strides, box, one,
                                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                         promotion(row_bytes), CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
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
  s.part = up256(size_t(T) * K * F * 4);
  const size_t parts = size_t(sms) + max_chunks(T, ragged_rows(F));
  s.ctr = s.part + up256(2 * parts * T * 256 * 4);
  s.lpart = s.ctr + up256((size_t(sms) + kDecMaxChunks + 2) * 4);
  s.total = s.lpart + up256(size_t(sms) * T * Er * 4);
  return s;
}

bool dec_sizes_ok(int64_t T, int32_t H, int32_t F, int32_t E, int32_t K, int32_t Er) {
  if (T < 0 || T > kDecMaxT || K < 1 || K > kMaxRouteK || T * K > kDecMaxRows) return false;
  if (H <= 0 || H % 8 || H > kDecMaxH || F <= 0 || F % 8 || E < 1 || E > kMaxExperts) return false;
  if (Er < 0 || Er > kMaxExperts || Er % 4 || (Er > 0 && K > Er)) return false;
  // Unit counts times CTAs stay within 32 bits (2^24 units are 512 GB).
  const int64_t act = E < T * K ? E : T * K;
  const int64_t u1 = act * ((F + 127) / 128) * ((H + 63) / 64), u2 = act * ((H + 255) / 256) * ((F + 63) / 64);
  return u1 <= (1 << 24) && u2 <= (1 << 24);
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
  if (p->router_w && Er < 4) return kBadArg;
  if (p->T == 0) return kOk;
  if (!p->x || !p->w13 || !p->w2 || !p->y || !p->top_idxs || !p->top_vals || !p->scratch) return kBadArg;
  if (misaligned(p->x) || misaligned(p->w13) || misaligned(p->w2) || misaligned(p->y) ||
      misaligned(p->scratch))
    return kBadArg;
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
  a.NB2 = (2 * T + 15) / 16 * 16;
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
  a.stage_bytes = kDecABytes + uint32_t(a.NB2) * 128;
  // Pass 2's sums [T][256] and, before them, the masks and offsets of the
  // routing tables and one token's logits.
  uint32_t scratch = uint32_t(T) * 1024;
  const uint32_t build = uint32_t(E) * 10 + uint32_t(T) * K * 6, logits = uint32_t(Er) * 4 + uint32_t((Er + 31) / 32 * K) * 8;
  if (scratch < build) scratch = build;
  if (scratch < logits) scratch = logits;
  a.scratch_bytes = (scratch + 15) / 16 * 16;
  const uint32_t fixed = 1024 + a.scratch_bytes + dec_table_bytes(a.maxact, T * K) + uint32_t(sizeof(DecSmem));
  int stages = int((kDecMaxSmem - fixed) / a.stage_bytes);
  a.stages = stages > kDecMaxStages ? kDecMaxStages : stages;
  if (a.stages < 2) return kBadArg;
  const uint32_t smem = fixed + uint32_t(a.stages) * a.stage_bytes;
  // The router's slices use the stage memory: tokens by H / (slices of H).
  // Slices of a quarter of the experts leave fewer parts to add per logit,
  // where a quarter is whole 16-byte pieces of a row and its rows fit.
  const uint32_t room = uint32_t(a.stages) * a.stage_bytes - kDecThreads * 2 * kDecTokChunk * 4;
  const uint32_t xrow = uint32_t(T + kDecTokChunk - 1) / kDecTokChunk * kDecTokChunk * 4;
  a.eparts = Er % 32 == 0 && sms >= 8 && (H / (sms / 4) + 1) * xrow <= room ? 4 : 1;
  if (Er && (H / (sms / a.eparts) + 1) * xrow > room) return kBadArg;

  CUtensorMap m13, m2, m2e, mx, mh;
  {
    const cuuint64_t dims[4] = {cuuint64_t(F), cuuint64_t(H), 2, cuuint64_t(E)};
    const cuuint64_t str[3] = {cuuint64_t(F) * 4, cuuint64_t(F) * 2, cuuint64_t(H) * F * 4};
    const cuuint32_t box[4] = {64, 64, 2, 1};
    if (encode(&m13, 4, p->w13, dims, str, box, F * 2)) return kCudaErr;
  }
  {
    // Whole atoms of 64 features (at least one is described; a row shorter
    // than one is never read through it).
    const cuuint64_t dims[4] = {64, cuuint64_t(F), cuuint64_t(H < 64 ? 1 : H / 64), cuuint64_t(E)};
    const cuuint64_t str[3] = {cuuint64_t(H) * 2, 128, cuuint64_t(H) * F * 2};
    const cuuint32_t box[4] = {64, 64, 4, 1};
    if (encode(&m2, 4, p->w2, dims, str, box, H * 2)) return kCudaErr;
  }
  {
    const cuuint64_t dims[3] = {cuuint64_t(H), cuuint64_t(F), cuuint64_t(E)};
    const cuuint64_t str[2] = {cuuint64_t(H) * 2, cuuint64_t(H) * F * 2};
    const cuuint32_t box[3] = {64, 64, 1};
    if (encode(&m2e, 3, p->w2, dims, str, box, H * 2)) return kCudaErr;
  }
  {
    const cuuint64_t dims[2] = {cuuint64_t(H), cuuint64_t(T)};
    const cuuint64_t str[1] = {cuuint64_t(H) * 2};
    const cuuint32_t box[2] = {64, cuuint32_t(a.NB)};
    if (encode(&mx, 2, p->x, dims, str, box, H * 2)) return kCudaErr;
  }
  {
    const cuuint64_t dims[2] = {cuuint64_t(F), cuuint64_t(2 * T) * K};
    const cuuint64_t str[1] = {cuuint64_t(F) * 2};
    const cuuint32_t box[2] = {64, 16};
    if (encode(&mh, 2, a.hs, dims, str, box, F * 2)) return kCudaErr;
  }
  // Once per device: shared memory opted in to.
  static std::atomic<bool> ready[kMaxDevices];
  if (dev < 0 || dev >= kMaxDevices) return kCudaErr;
  if (!ready[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(decode_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kDecMaxSmem)) !=
        cudaSuccess)
      return kCudaErr;
    ready[dev].store(true, std::memory_order_release);
  }
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
  return cudaLaunchKernelEx(&cfg, decode_kernel, m13, m2, m2e, mx, mh, a) == cudaSuccess ? kOk : kCudaErr;
}
