// Attention of one token for each of B streams over a paged cache, with a window and sinks.
//
//   o = sum_j softmax_j(scale q . k_j) v_j over the positions j that the stream's last one sees
//
// HBM-bound: the visible rows of K and V are read once for all the query heads that share them. A workgroup takes one stream,
// key head and chunk of tiles (position-aligned, TILE keys), its waves the chunk's tiles in turn, each for itself: a wave
// has its own stages in LDS, filled by loads straight into it (K and V of a tile, 16 KiB at D = 128) while the tile before
// is computed. S^T = K Q^T has a query a lane (16 columns, as many as heads share the key head), so that its softmax is
// within a lane but for one exchange over the lane groups, and S^T's own layout is the second operand of
// O^T = V^T P^T: keys in the order that S^T leaves them, V read transposed in the same order. The waves' parts (running
// maximum, sum, O) are joined in LDS, those of a stream's chunks by a second kernel, in order.
// What is not seen is loaded as zeros, so that nothing of it (a NaN, say) meets a weight of 0.
// Loads bypass the caches' retention, and the key heads of one chunk stand beside one another in the grid (a cache's row is all
// of them): a call of 64 streams over caches of 4096 .. 8192 rows, 16 heads on 4, D = 128: 150 us, 5.5 TB/s (202 us without
// both), of 256 streams over 3.2 GB 580 us, 5.6 TB/s, so that it is memory and not a cache that gives them: reads alone, a tenth
// faster than a copy (5.14). One stream over 32768 rows: 20.2 us where its bytes take 13; two launches and the first loads' chain
// (length and pages, rows, queries) are the rest.
// Sums, statistics and O are fp32; P is rounded to bf16 for the product where V is bf16 (at most 2^-8 of each weight, as V's own).
#include <algorithm>
#include <cmath>

#include "gdn_attn.h"
#include "zonos3_attn.h"

namespace zgdn {
namespace {

constexpr int WS_NW = 2, WS_WIDE = 8;  // waves a workgroup
constexpr long WS_PER_CU = 2;           // workgroups a CU
constexpr int WS_KEYS = 1024;   // keys of a chunk, at most
constexpr long MOST_ROOM = 1L << 30;  // positions of a stream
constexpr int WS_Q = 16;        // query heads of a workgroup, at most

struct WinStepArgs {
  const void* q;
  long q_ld;
  const void *kc, *vc;
  long kc_ld, vc_ld;
  const int32_t *lengths, *pages;
  int page_size, page_shift, n_pages;  // (pages NULL: one page a stream, of any size)
  long cache_pages;                    // pages in the cache
  void* o;
  int B, Hq, Hk, window, sinks;
  float c;            // scale log2(e)
  int q_groups, gq;   // groups of at most 16 query heads of a key head, heads of a group
  int chunk, splits;  // tiles of a chunk; chunks of a stream, at most
  float *part_o, *part_ml;  // [unit][split][gq][D], [unit][split][gq][2]
};

template <typename T>
struct WsCfg {
  static constexpr int TILE = sizeof(T) == 2 ? 32 : 16;
};

// Position-aligned tiles of TILE keys that the query at position `at` sees: those of the sinks, then those from the window's
// start on.
struct KeyTiles {
  int sinks, from, n;  // tiles of the sinks, the first of the window's, all
  __device__ __forceinline__ int at(int i) const { return i < sinks ? i : from + (i - sinks); }
};
template <int TILE>
__device__ __forceinline__ KeyTiles key_tiles(int at, int window, int sinks) {
  KeyTiles t;
  const int lo = window > 0 ? max(0, at - window + 1) : 0;
  t.from = lo / TILE;
  t.sinks = min((min(sinks, lo) + TILE - 1) / TILE, t.from);
  t.n = at < 0 ? 0 : t.sinks + at / TILE + 1 - t.from;
  return t;
}
// Those of stream b.
template <int TILE>
__device__ __forceinline__ KeyTiles stream_tiles(const WinStepArgs& a, int b, int& n, int& lo) {
  const long room = (long)a.page_size * a.n_pages;
  n = (int)max(0L, min((long)a.lengths[b], room));
  lo = a.window > 0 ? max(0, n - a.window) : 0;
  return key_tiles<TILE>(n - 1, a.window, a.sinks);
}

// NW waves of RING stages each: two waves of two, so that two workgroups (four and more at D = 64) share a CU and the start of
// one is hidden behind the others' loads; or, for a few short streams, eight waves that need no second kernel to join them.
template <typename T, int D, int NW, int RING>
__global__ __launch_bounds__(64 * NW) void win_step_kernel(WinStepArgs a) {
  constexpr bool BF = sizeof(T) == 2;
  constexpr int TILE = WsCfg<T>::TILE, ROWB = D * (int)sizeof(T), CH = ROWB / 16, RP = 64 / CH;
  constexpr int LI = TILE * ROWB / 1024;  // load instructions for a tile of K (and of V)
  constexpr int STAGE = 2 * TILE * ROWB;
  constexpr int DT = D / 16;
  __shared__ __align__(1024) uint8_t ring[NW][RING][STAGE];
  __shared__ int32_t page_of[WS_KEYS];
  static_assert(RING * STAGE >= WS_Q * (D + 2) * 4, "the waves' parts");
  const int lane = threadIdx.x & 63, wave = wave_id(), m = lane & 15, g = lane >> 4;
  // (the key heads of one stream's chunk beside one another: a row of the cache is all of them)
  const int per_chunk = a.Hk * a.q_groups, bs = blockIdx.x / per_chunk, b = bs / a.splits, split = bs - b * a.splits;
  const int unit = b * per_chunk + (blockIdx.x - bs * per_chunk), hk = (unit - b * per_chunk) / a.q_groups;
  const int qg = unit - b * per_chunk - hk * a.q_groups;
  int n, lo;
  const KeyTiles tiles = stream_tiles<TILE>(a, b, n, lo);
  const int first = split * a.chunk, count = min(a.chunk, tiles.n - first);  // the chunk's tiles
  const int G = a.Hq / a.Hk, h0 = hk * G + qg * a.gq, heads = min(a.gq, G - qg * a.gq);

  // queries as the second operand: column m, entries k of the lane's group
  uint4 qf[BF ? D / 32 : D / 16];
#pragma unroll
  for (int t = 0; t < (int)(sizeof(qf) / 16); ++t) {
    qf[t] = make_uint4(0, 0, 0, 0);
    if (m < heads) {
      const T* src = reinterpret_cast<const T*>(a.q) + (size_t)b * a.q_ld + (size_t)(h0 + m) * D;
      qf[t] = *reinterpret_cast<const uint4*>(src + (BF ? 32 * t + 8 * g : 16 * t + 4 * g));
    }
  }
  // the pages of the chunk's positions, one entry for each run of `gran` of them; -1 for one that is not in the cache. (Without
  // a window the positions do not depend on the length: the pages are read while it is.)
  const int gran = a.pages == nullptr ? TILE : min(a.page_size, TILE), per_tile = TILE / gran;
  bool missing = false;
  if (a.pages != nullptr) {
    const int room = a.page_size * a.n_pages;
    for (int i = threadIdx.x; i < a.chunk * per_tile; i += 64 * NW) {
      const int tile = a.window > 0 ? tiles.at(first + i / per_tile) : first + i / per_tile;
      const int p = tile * TILE + (i % per_tile) * gran;
      int32_t page = p < room ? a.pages[(size_t)b * a.n_pages + (p >> a.page_shift)] : -1;
      if (page < 0 || page >= a.cache_pages) {
        page = -1;
        missing = missing || (p < n && (p + gran > lo || p < a.sinks));
      }
      page_of[i] = page;
    }
    missing = __syncthreads_or(missing);
  }
  if (count <= 0) {
    if (a.splits == 1)  // nothing is seen
      for (int i = threadIdx.x; i < heads * D; i += 64 * NW)
        io<T>::store(reinterpret_cast<T*>(a.o) + ((size_t)b * a.Hq + h0) * D + i, 0.f);
    return;
  }
  const int sink_end = min(a.sinks, lo);
#pragma unroll
  for (int t = 0; t < (int)(sizeof(qf) / 16); ++t) asm volatile("" : "+v"(qf[t].x));  // (awaited here, not in the loop)

  auto seen = [&](int i, int p) {  // position p of the chunk's tile i
    bool s = p < n && (p >= lo || p < sink_end);
    if (missing) s = s && page_of[i * per_tile + (p % TILE) / gran] >= 0;
    return s;
  };
  const uint8_t* kb = reinterpret_cast<const uint8_t*>(a.kc) + (size_t)hk * ROWB;
  const uint8_t* vb = reinterpret_cast<const uint8_t*>(a.vc) + (size_t)hk * ROWB;
  const size_t kl = (size_t)a.kc_ld * sizeof(T), vl = (size_t)a.vc_ld * sizeof(T);
  uint32_t koff[LI], voff[LI];  // of a tile whose rows follow one another: the lane's pieces from its first row on
#pragma unroll
  for (int j = 0; j < LI; ++j) {
    const int r = j * RP + lane / CH;
    const uint32_t c = (uint32_t)((lane % CH) ^ swizzle<ROWB, T, 16>(r)) << 4;
    koff[j] = (uint32_t)r * (uint32_t)kl + c;
    voff[j] = (uint32_t)r * (uint32_t)vl + c;
  }
  auto whole_tile = [&](int p0) { return !missing && p0 + TILE <= n && (p0 >= lo || p0 + TILE <= sink_end); };
  auto issue = [&](int i, int stage) {  // tile i of the chunk
    const int p0 = tiles.at(first + i) * TILE;
    const uint32_t at = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)&ring[wave][stage][0]);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // what the stage held before has been read
    if (gran == TILE && whole_tile(p0)) {
      const size_t row = a.pages == nullptr ? (size_t)b * a.page_size + p0
                                            : (size_t)__builtin_amdgcn_readfirstlane(page_of[i]) * a.page_size +
                                                  (p0 & (a.page_size - 1));
      const uint8_t *kt = kb + row * kl, *vt = vb + row * vl;
#pragma unroll
      for (int j = 0; j < LI; ++j) load_lds_from(kt, koff[j], at + 1024 * j);
#pragma unroll
      for (int j = 0; j < LI; ++j) load_lds_from(vt, voff[j], at + TILE * ROWB + 1024 * j);
      return;
    }
#pragma unroll
    for (int j = 0; j < LI; ++j) {
      const int r = j * RP + lane / CH, p = p0 + r;
      const size_t c = (size_t)(((lane % CH) ^ swizzle<ROWB, T, 16>(r)) << 4);
      const bool s = seen(i, p);
      size_t row = (size_t)b * a.page_size + p;
      if (a.pages != nullptr) row = (size_t)page_of[i * per_tile + r / gran] * a.page_size + (p & (a.page_size - 1));
      load_lds_from(s ? (const void*)(kb + row * kl + c) : (const void*)zeros16, at + 1024 * j);
      load_lds_from(s ? (const void*)(vb + row * vl + c) : (const void*)zeros16, at + TILE * ROWB + 1024 * j);
    }
  };

  af32x4 o[DT] = {};
  float top = -INFINITY, sum = 0.f;  // of the lane's query; sum: of the lane's keys
  bool any = false;
  auto compute = [&](int i, int stage) {
    const uint8_t *ks = &ring[wave][stage][0], *vs = ks + TILE * ROWB;
    const int p0 = tiles.at(first + i) * TILE;
    constexpr int ST = TILE / 16;
    af32x4 st[ST] = {};
#pragma unroll
    for (int t = 0; t < ST; ++t) {
#pragma unroll
      for (int kk = 0; kk < (int)(sizeof(qf) / 16); ++kk) {
        const uint4 kf = *reinterpret_cast<const uint4*>(ks + row_chunk<ROWB, T, 16>(16 * t + m, 4 * kk + g));
        if constexpr (BF) {
          st[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(abf16x8, kf), __builtin_bit_cast(abf16x8, qf[kk]),
                                                          st[t], 0, 0, 0);
        } else {
          const uint32_t kw[4] = {kf.x, kf.y, kf.z, kf.w}, qw[4] = {qf[kk].x, qf[kk].y, qf[kk].z, qf[kk].w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            st[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kw[e]), __uint_as_float(qw[e]), st[t], 0, 0, 0);
        }
      }
    }
    const bool whole = whole_tile(p0);
    float best = -INFINITY;
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = st[t][e] * a.c;
        if (!whole) {
          const bool s = seen(i, p0 + 16 * t + 4 * g + e);
          any = any || s;
          x = s ? x : -INFINITY;
        }
        st[t][e] = x;
        best = fmaxf(best, x);
      }
    any = any || whole;
    const float next = fmaxf(top, max_over_groups(best));
    const float base = next == -INFINITY ? 0.f : next;
    const float keep = exp2_of(top - base);
    top = next;
    float add = 0.f;
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        st[t][e] = exp2_of(st[t][e] - base);
        add += st[t][e];
      }
    sum = fmaf(sum, keep, add);
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[d][e] *= keep;
    const int s = lane & 15;
    if constexpr (BF) {
      const uint4 pw = make_uint4(pack_bf16x2(st[0][0], st[0][1]), pack_bf16x2(st[0][2], st[0][3]),
                                  pack_bf16x2(st[1][0], st[1][1]), pack_bf16x2(st[1][2], st[1][3]));
      const abf16x8 pf = __builtin_bit_cast(abf16x8, pw);
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const int r = 4 * g + (s >> 2), c = 2 * d + ((s & 3) >> 1), low = 8 * (s & 1);
        const uint2 v0 = lds_transposed(vs + row_chunk<ROWB, T, 16>(r, c) + low);
        const uint2 v1 = lds_transposed(vs + row_chunk<ROWB, T, 16>(r + 16, c) + low);
        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(abf16x8, make_uint4(v0.x, v0.y, v1.x, v1.y)), pf,
                                                       o[d], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v = *reinterpret_cast<const float*>(vs + row_chunk<ROWB, T, 16>(4 * g + e, 4 * d + (s >> 2)) + 4 * (s & 3));
          o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, st[0][e], o[d], 0, 0, 0);
        }
    }
  };

  wait_own_loads<0>();
  if constexpr (RING == 1) {
    for (int i = wave; i < count; i += NW) {
      issue(i, 0);
      wait_own_loads<0>();
      compute(i, 0);
    }
  } else {
    if (wave < count) issue(wave, 0);
    for (int i = wave, stage = 0; i < count; i += NW, stage ^= 1) {
      if (i + NW < count) {
        issue(i + NW, stage ^ 1);
        wait_own_loads<2 * LI>();
      } else {
        wait_own_loads<0>();
      }
      compute(i, stage);
    }
  }

  // the waves' parts, joined in LDS: [wave][query][D + 2]
  sum = sum_over_groups(sum);
  any = __any(any);
  __syncthreads();
  float* mine = reinterpret_cast<float*>(&ring[0][0][0]) + (wave * WS_Q + m) * (D + 2);
  if (m < heads) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) mine[16 * d + 4 * g + e] = o[d][e];
    if (g == 0) {
      mine[D] = top;
      mine[D + 1] = any ? sum : -1.f;  // (below zero: the part saw nothing)
    }
  }
  __syncthreads();
  const float* parts = reinterpret_cast<const float*>(&ring[0][0][0]);
  for (int i = threadIdx.x; i < heads * D; i += 64 * NW) {
    const int h = i / D, d = i - h * D;
    float best = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) best = fmaxf(best, parts[(w * WS_Q + h) * (D + 2) + D]);
    const float base = best == -INFINITY ? 0.f : best;
    float x = 0.f, l = 0.f;
    bool saw = false;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float* p = parts + (w * WS_Q + h) * (D + 2);
      if (p[D + 1] < 0.f) continue;
      const float f = exp2_of(p[D] - base);
      x = fmaf(p[d], f, x);
      l = fmaf(p[D + 1], f, l);
      saw = true;
    }
    if (a.splits == 1) {
      io<T>::store(reinterpret_cast<T*>(a.o) + ((size_t)b * a.Hq + h0 + h) * D + d, saw ? x / l : 0.f);
    } else {
      const size_t at = ((size_t)unit * a.splits + split) * a.gq + h;
      a.part_o[at * D + d] = x;
      if (d == 0) {
        a.part_ml[2 * at] = best;
        a.part_ml[2 * at + 1] = saw ? l : -1.f;
      }
    }
  }
}

// A workgroup for each stream and query head joins its chunks' parts: groups of D / 4 lanes, JOIN_AT parts each at a time, in
// order, with a running maximum (so that a part's statistics and values are read at one time); then its first wave the groups'
// sums. The first parts are read while the length is, whether there are as many or not.
constexpr int JOIN_AT = 4, JOIN_MOST = 1024;  // parts a group at a time; threads, at most
template <typename T, int D>
__global__ __launch_bounds__(JOIN_MOST) void win_step_join_kernel(WinStepArgs a) {
  constexpr int LANES = D / 4, MOST = JOIN_MOST / LANES, EACH = D / 64;
  __shared__ __align__(16) float x_of[MOST][D];
  __shared__ float top_of[MOST], sum_of[MOST];
  static_assert(MOST <= 64, "a lane for each group");
  const int groups = blockDim.x / LANES;
  const int b = blockIdx.x / a.Hq, h = blockIdx.x - b * a.Hq, G = a.Hq / a.Hk, hk = h / G, qg = (h - hk * G) / a.gq;
  const size_t unit = ((size_t)b * a.Hk + hk) * a.q_groups + qg;
  const size_t at = unit * a.splits * a.gq + (h - hk * G - qg * a.gq);
  int n, lo;
  const KeyTiles tiles = stream_tiles<WsCfg<T>::TILE>(a, b, n, lo);
  const int used = (tiles.n + a.chunk - 1) / a.chunk;
  const int d = 4 * (threadIdx.x % LANES), jg = threadIdx.x / LANES;
  float top = -INFINITY, sum = 0.f;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  bool any = false;
  int i0 = jg;
  do {
    float2 ml[JOIN_AT];
    float4 u[JOIN_AT];
#pragma unroll
    for (int e = 0; e < JOIN_AT; ++e) {
      const size_t p = at + (size_t)min(i0 + e * groups, a.splits - 1) * a.gq;
      ml[e] = *reinterpret_cast<const float2*>(a.part_ml + 2 * p);
      u[e] = *reinterpret_cast<const float4*>(a.part_o + p * D + d);
    }
#pragma unroll
    for (int e = 0; e < JOIN_AT; ++e) {
      const bool saw = i0 + e * groups < used && !(ml[e].y < 0.f);  // (a sum below zero: the part saw nothing)
      if (!saw) continue;                                           // (what is not there may be any bits)
      const float next = fmaxf(top, ml[e].x), base = next == -INFINITY ? 0.f : next;
      const float keep = exp2_of(top - base), f = exp2_of(ml[e].x - base);
      top = next;
      sum = fmaf(sum, keep, ml[e].y * f);
      x = make_float4(fmaf(x.x, keep, u[e].x * f), fmaf(x.y, keep, u[e].y * f), fmaf(x.z, keep, u[e].z * f),
                      fmaf(x.w, keep, u[e].w * f));
      any = true;
    }
    i0 += JOIN_AT * groups;
  } while (i0 < used);
  *reinterpret_cast<float4*>(&x_of[jg][d]) = x;
  if (d == 0) {
    top_of[jg] = top;
    sum_of[jg] = any ? sum : -1.f;
  }
  __syncthreads();
  const int lane = threadIdx.x;
  if (lane >= 64) return;
  const float l = lane < groups ? sum_of[lane] : -1.f, t = lane < groups ? top_of[lane] : -INFINITY;
  const bool saw = !(l < 0.f);
  const float best = wave_max(t);
  const float f = saw ? exp2_of(t - (best == -INFINITY ? 0.f : best)) : 0.f, all = wave_sum(saw ? l * f : 0.f);
  float o[EACH] = {};
  for (int g = 0; g < groups; ++g) {
    const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), g));
#pragma unroll
    for (int e = 0; e < EACH; ++e) o[e] = fmaf(x_of[g][64 * e + lane], w, o[e]);
  }
  const bool seen = __any(saw);
#pragma unroll
  for (int e = 0; e < EACH; ++e)
    io<T>::store(reinterpret_cast<T*>(a.o) + (size_t)blockIdx.x * D + 64 * e + lane, seen ? o[e] / all : 0.f);
}

// How a call is cut: chunks of at most WS_KEYS keys, of at least a tile for each wave, two workgroups for each CU where the
// streams' visible positions have that many. Up to WS_KEYS keys of streams and key heads that a CU each can take are not cut.
struct StepPlan {
  int q_groups, gq, chunk, splits;
  bool wide;
};
StepPlan step_plan(int B, long room, int Hq, int Hk, int window, int sinks, int dtype) {
  StepPlan p;
  const int G = Hq / Hk;
  const long tile = dtype == ZGDN_BF16 ? WsCfg<bf16>::TILE : WsCfg<float>::TILE;
  p.q_groups = (G + WS_Q - 1) / WS_Q;
  p.gq = (G + p.q_groups - 1) / p.q_groups;
  long tiles = std::max(1L, (room + tile - 1) / tile);
  if (window > 0) tiles = std::min(tiles, (window + tile - 2) / tile + 1 + (sinks + tile - 1) / tile);
  const long units = (long)B * Hk * p.q_groups;
  p.wide = tiles <= WS_KEYS / tile && units <= device_cus();
  if (p.wide) {
    p.chunk = (int)tiles;
    p.splits = 1;
    return p;
  }
  const long want = (WS_PER_CU * device_cus() + units - 1) / units;  // chunks of a stream
  long chunk = std::min(std::max((tiles + want - 1) / want, (long)WS_NW), WS_KEYS / tile);
  p.splits = (int)((tiles + chunk - 1) / chunk);
  chunk = (tiles + p.splits - 1) / p.splits;  // (of equal size)
  p.chunk = (int)(chunk + WS_NW - 1) / WS_NW * WS_NW;
  p.splits = (int)((tiles + p.chunk - 1) / p.chunk);
  return p;
}
size_t step_bytes(const StepPlan& p, int B, int Hk, int D) {
  return p.splits == 1 ? 0 : (size_t)B * Hk * p.q_groups * p.splits * p.gq * (D + 2) * sizeof(float);
}

template <typename T, int D>
void launch_win_step(const WinStepArgs& a, bool wide, hipStream_t s) {
  const unsigned units = (unsigned)(a.B * a.Hk * a.q_groups);
  if (wide) {
    hipLaunchKernelGGL((win_step_kernel<T, D, WS_WIDE, 128 / D>), dim3(units), dim3(64 * WS_WIDE), 0, s, a);
    return;
  }
  hipLaunchKernelGGL((win_step_kernel<T, D, WS_NW, 2>), dim3(units * a.splits), dim3(64 * WS_NW), 0, s, a);
  if (a.splits == 1) return;
  constexpr int WAVE = 64 / (D / 4);  // groups of a wave
  const int waves = std::min((a.splits + JOIN_AT * WAVE - 1) / (JOIN_AT * WAVE), JOIN_MOST / 64);
  hipLaunchKernelGGL((win_step_join_kernel<T, D>), dim3((unsigned)(a.B * a.Hq)), dim3(64 * waves), 0, s, a);
}

bool step_sizes(int B, long room, int Hq, int Hk, int D, int window, int sinks, int dtype) {
  return B >= 0 && room >= 0 && room <= MOST_ROOM && Hq >= 1 && Hk >= 1 && Hq % Hk == 0 && (D == 64 || D == 128) &&
         window >= 0 && sinks >= 0 && (dtype == ZGDN_F32 || dtype == ZGDN_BF16);
}

}  // namespace
}  // namespace zgdn

extern "C" size_t zattn_window_step_workspace_bytes(int B, long room, int Hq, int Hk, int D, int window, int sinks,
                                                    int dtype) {
  using namespace zgdn;
  if (!step_sizes(B, room, Hq, Hk, D, window, sinks, dtype) || B == 0) return 0;
  return step_bytes(step_plan(B, room, Hq, Hk, window >= room ? 0 : window, std::min(sinks, 1 << 30), dtype), B, Hk, D);
}

// (for tests) Whether a call takes one launch of wide workgroups, and the chunks of a stream, for the same sizes.
extern "C" int zgdn_window_step_form(int B, long room, int Hq, int Hk, int window, int sinks, int dtype, int64_t* form) {
  using namespace zgdn;
  if (!step_sizes(B, room, Hq, Hk, 64, window, sinks, dtype) || B == 0)
    return fail(ZGDN_EINVAL, "zgdn_window_step_form: bad sizes");
  const StepPlan p = step_plan(B, room, Hq, Hk, window >= room ? 0 : window, std::min(sinks, 1 << 30), dtype);
  form[0] = p.wide;
  form[1] = p.splits;
  return ZGDN_OK;
}

extern "C" int zattn_window_step(const void* q, long q_ld, const void* k_cache, long kc_ld, const void* v_cache, long vc_ld,
                                 int dtype, const int32_t* lengths, const int32_t* pages, int page_size, int n_pages,
                                 long n_rows, void* o, int B, int Hq, int Hk, int D, int window, int sinks, float scale,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  using namespace zgdn;
  const char* fn = "zattn_window_step";
  if (B < 0 || Hq < 1 || Hk < 1 || page_size < 0 || n_pages < 0 || n_rows < 0 || window < 0 || sinks < 0)
    return fail(ZGDN_EINVAL, "%s: bad sizes B=%d Hq=%d Hk=%d page_size=%d n_pages=%d n_rows=%ld window=%d sinks=%d", fn, B, Hq,
                Hk, page_size, n_pages, n_rows, window, sinks);
  if (Hq % Hk) return fail(ZGDN_EINVAL, "%s: Hq=%d is not a multiple of Hk=%d", fn, Hq, Hk);
  if (D != 64 && D != 128) return fail(ZGDN_EUNSUPPORTED, "%s: D=%d (supported: 64 and 128)", fn, D);
  if (dtype != ZGDN_F32 && dtype != ZGDN_BF16) return fail(ZGDN_EINVAL, "%s: unknown dtype code %d", fn, dtype);
  if (pages == nullptr ? n_pages != 1 || n_rows < (long)B * page_size
                       : page_size < 1 || (page_size & (page_size - 1)) || n_rows % page_size)
    return fail(ZGDN_EINVAL, "%s: pages of %d rows, %d a stream, in a cache of %ld rows (with a table: a power of two, whole "
                "pages; without: one a stream)", fn, page_size, n_pages, n_rows);
  const long room = (long)page_size * n_pages;
  if (room > MOST_ROOM) return fail(ZGDN_EUNSUPPORTED, "%s: %ld positions a stream", fn, room);
  if (!std::isfinite(scale * LOG2E)) return fail(ZGDN_EINVAL, "%s: scale %g", fn, scale);
  if (window >= room) window = 0;  // (every position)
  sinks = std::min(sinks, 1 << 30);  // (more than positions reach)
  if (B == 0) return ZGDN_OK;
  if (!q || !o || !lengths || (n_rows > 0 && (!k_cache || !v_cache))) return fail(ZGDN_EINVAL, "%s: null tensor pointer", fn);
  const int ve = dtype == ZGDN_F32 ? 4 : 8;
  const long most = 1L << 22, wq = (long)Hq * D, wk = (long)Hk * D;
  auto bad = [&](long ld, long width) { return ld < width || ld > most || ld % ve; };
  if (bad(q_ld, wq) || bad(kc_ld, wk) || bad(vc_ld, wk))
    return fail(ZGDN_EINVAL, "%s: row strides q=%ld k_cache=%ld v_cache=%ld (multiples of %d elements, at least a row, at most "
                "2^22)", fn, q_ld, kc_ld, vc_ld, ve);
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)o | (uintptr_t)workspace) % 16)
    return fail(ZGDN_EINVAL, "%s: q, caches, o and workspace need 16-byte aligned bases", fn);
  if (((uintptr_t)lengths | (uintptr_t)pages) % 4) return fail(ZGDN_EINVAL, "%s: lengths, pages not on 4-byte boundaries", fn);
  const StepPlan p = step_plan(B, room, Hq, Hk, window, sinks, dtype);
  if ((long)B * Hk * p.q_groups * p.splits > (1L << 32) / (64 * WS_NW) - 1 || (long)B * Hq > (1L << 32) / JOIN_MOST - 1)
    return fail(ZGDN_EUNSUPPORTED, "%s: B=%d x Hq=%d x %d chunks", fn, B, Hq, p.splits);
  const size_t need = step_bytes(p, B, Hk, D);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(ZGDN_EINVAL, "%s: workspace of %zu bytes, %zu needed", fn, workspace == nullptr ? 0 : workspace_bytes, need);
  const size_t es = dtype == ZGDN_F32 ? 4 : 2, n = (size_t)B;
  const Region out = {o, n, wq * es, wq * es}, ws = {need ? workspace : nullptr, 1, need, need};
  const Region in[] = {{q, n, wq * es, q_ld * es}, {k_cache, (size_t)n_rows, wk * es, kc_ld * es},
                       {v_cache, (size_t)n_rows, wk * es, vc_ld * es}, {lengths, 1, n * 4, n * 4},
                       {pages, 1, n * n_pages * 4, n * n_pages * 4}};
  bool meet = regions_meet(out, ws);
  for (const Region& r : in) meet = meet || regions_meet(out, r) || regions_meet(ws, r);
  if (meet) return fail(ZGDN_EINVAL, "%s: o or the workspace overlap another operand", fn);
  float* part = reinterpret_cast<float*>(workspace);
  const size_t rows = (size_t)B * Hk * p.q_groups * p.splits * p.gq;
  WinStepArgs a{q, q_ld, k_cache, v_cache, kc_ld, vc_ld, lengths, pages, page_size,
                pages != nullptr ? __builtin_ctz((unsigned)page_size) : 0, n_pages, pages != nullptr ? n_rows / page_size : 0,
                o, B, Hq, Hk, window, sinks, scale * LOG2E, p.q_groups, p.gq, p.chunk, p.splits, part,
                need ? part + rows * D : nullptr};
  hipStream_t s = (hipStream_t)stream;
  if (dtype == ZGDN_F32)
    D == 128 ? launch_win_step<float, 128>(a, p.wide, s) : launch_win_step<float, 64>(a, p.wide, s);
  else
    D == 128 ? launch_win_step<bf16, 128>(a, p.wide, s) : launch_win_step<bf16, 64>(a, p.wide, s);
  return check_launch(fn);
}
