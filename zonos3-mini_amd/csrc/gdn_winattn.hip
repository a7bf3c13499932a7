// Causal attention over whole sequences with a sliding window and first tokens that stay visible (sinks), on MFMA.
//
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys j <= p_i with p_i - j < window or j < sinks
//
// The queries of the G heads that share a key head are one list of rows, row r = query r / G, head r % G: a workgroup's rows
// then stand at few positions, and its keys are read once for all of them. A wave holds 32 rows, a row a lane: S^T = K Q^T
// leaves a row's scores in one lane (and its partner, lane ^ 32), so that the softmax is within a lane but for one exchange,
// and S^T's layout is the second operand of O^T = V^T P^T as it stands: keys in the order that S^T leaves them, V read
// transposed from LDS in the same order. One pass over the keys with a running maximum and sum.
// Tiles of K and V are loaded straight into LDS, a tile ahead. Tiles that no row sees are left out, tiles that all rows of a
// wave see whole have no mask.
// Scores, statistics and O are fp32; P is rounded to bf16 for the product where V is bf16 (at most 2^-8 of each weight, as V's own).
// A masked weight is 0, but 0 times an infinity or a NaN of V is a NaN: in tiles that a row of the workgroup does not see
// whole, such entries are zeroed in LDS ahead of the product, and the rows that see one of them are computed again in the end,
// key by key (win_row).
#include <algorithm>

#include "gdn_attn.h"
#include "zonos3_attn.h"

namespace zgdn {
namespace {

struct WinArgs {
  const void *q, *k, *v;
  long q_ld, k_ld, v_ld;
  void* o;
  const int32_t *cu_q, *cu_k;
  int N, Tq, Tk, Hq, Hk, window, sinks;
  float c;    // scale log2(e)
  int tiles;  // of rows a key head, at most
};

__device__ __forceinline__ int prefix_count(int x) {  // over the lanes up to this one
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);
  return x;
}

// The rows that a workgroup takes: tile `tile` of a sequence's nq G rows, the last tiles first (they have the most keys).
struct RowTile {
  int q0, nq, k0, nk, tile;  // (q0, k0: the sequence's first row of q and of k)
};
template <int ROWS>
__device__ __forceinline__ bool find_rows(const WinArgs& a, int i, RowTile& t) {
  const int G = a.Hq / a.Hk;
  if (a.cu_q == nullptr) {
    const int per = a.tiles / a.N, s = i % a.N;
    t = {s * a.Tq, a.Tq, s * a.Tk, a.Tk, per - 1 - i / a.N};
    return true;
  }
  const int l = threadIdx.x & 63;
  int taken = 0;
  for (int s0 = 0; s0 < a.N; s0 += 64) {
    int b = 0, e = 0;
    if (s0 + l < a.N) seq_bounds(a.cu_q, s0 + l, a.Tq, b, e);
    const int mine = (int)(((long)(e - b) * G + ROWS - 1) / ROWS), upto = prefix_count(mine);
    const int all = __builtin_amdgcn_readlane(upto, 63);
    if (i < taken + all) {
      const int at = __builtin_ctzll(__ballot(i - taken < upto));
      int kb, ke;
      seq_bounds(a.cu_k, s0 + at, a.Tk, kb, ke);
      const int n = __builtin_amdgcn_readlane(mine, at), before = __builtin_amdgcn_readlane(upto, at) - n;
      b = __builtin_amdgcn_readlane(b, at);
      e = __builtin_amdgcn_readlane(e, at);
      kb = __builtin_amdgcn_readfirstlane(kb);
      ke = __builtin_amdgcn_readfirstlane(ke);
      t = {b, e - b, kb, ke - kb, n - 1 - (i - taken - before)};
      return true;
    }
    taken += all;
  }
  return false;
}

// Zeros in the place of a piece's infinities and NaN; whether there were any.
template <typename T>
__device__ __forceinline__ bool clear_odd(uint4& w) {
  uint32_t u[4] = {w.x, w.y, w.z, w.w};
  bool any = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool high = (u[i] & 0x7f800000u) == 0x7f800000u, low = sizeof(T) == 2 && (u[i] & 0x7f80u) == 0x7f80u;
    u[i] = high ? (sizeof(T) == 2 ? u[i] & 0xffffu : 0u) : u[i];
    u[i] = low ? u[i] & 0xffff0000u : u[i];
    any = any || high || low;
  }
  w = make_uint4(u[0], u[1], u[2], u[3]);
  return any;
}

// One row by one wave, in fp32 and from visible keys alone: q its query, k and v its key head's first rows, p its position.
template <typename T, int D>
__device__ __noinline__ void win_row(const T* q, const T* k, long k_ld, const T* v, long v_ld, T* o, int p, int window,
                                     int sinks, float c) {
  const int lane = threadIdx.x & 63;
  const int lo = window > 0 ? max(0, p - window + 1) : 0, s = min(sinks, lo), n = s + p + 1 - lo;  // visible keys
  float top = -INFINITY, sum = 0.f, acc[D / 64] = {};
  for (int i0 = 0; i0 < n; i0 += 64) {
    const int i = i0 + lane, j = i < s ? i : lo + i - s;
    float x = -INFINITY;
    if (i < n) {
      float dot = 0.f;
      for (int d = 0; d < D; ++d) dot = fmaf(io<T>::load(q + d), io<T>::load(k + (size_t)j * k_ld + d), dot);
      x = dot * c;
    }
    const float next = fmaxf(top, wave_max(x)), base = next == -INFINITY ? 0.f : next, keep = exp2_of(top - base);
    top = next;
    const float w = i < n ? exp2_of(x - base) : 0.f;
    sum = fmaf(sum, keep, wave_sum(w));
#pragma unroll
    for (int d = 0; d < D / 64; ++d) acc[d] *= keep;
    for (int e = 0; e < min(64, n - i0); ++e) {
      const int je = i0 + e < s ? i0 + e : lo + i0 + e - s;
      const float we = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), e));
#pragma unroll
      for (int d = 0; d < D / 64; ++d) acc[d] = fmaf(we, io<T>::load(v + (size_t)je * v_ld + 64 * d + lane), acc[d]);
    }
  }
#pragma unroll
  for (int d = 0; d < D / 64; ++d) io<T>::store(o + 64 * d + lane, acc[d] / sum);
}

template <typename T, int D, int NW>
__global__ __launch_bounds__(64 * NW) void win_attn_kernel(WinArgs a) {
  constexpr bool BF = sizeof(T) == 2;
  constexpr int ES = (int)sizeof(T), ROWB = D * ES, CH = ROWB / 16, RP = 64 / CH;
  constexpr int KT = BF ? 64 : 32, ST = KT / 32;  // keys of a tile
  constexpr int LW = KT * ROWB / 1024 / NW;       // a wave's load instructions for a tile of K (and of V)
  constexpr int STAGE = 2 * KT * ROWB, DT = D / 32, QF = D * ES / 32;
  constexpr int ROWS = 32 * NW;
  __shared__ __align__(1024) uint8_t lds[2][STAGE];
  __shared__ int dirty;  // something of V was zeroed
  const int lane = threadIdx.x & 63, wave = wave_id(), m = lane & 31, h = lane >> 5;
  const int hk = blockIdx.x % a.Hk, G = a.Hq / a.Hk;
  RowTile rt;
  if (!find_rows<ROWS>(a, blockIdx.x / a.Hk, rt)) return;
  const uint32_t rows = (uint32_t)rt.nq * G, r0 = (uint32_t)rt.tile * ROWS, rw = r0 + 32 * wave;
  const bool real = rw + m < rows;
  const uint32_t row = min(rw + m, rows - 1);  // (lanes behind the last row: as that one, without its stores)
  const int past = rt.nk - rt.nq;
  const int qi = (int)(row / G), hq = hk * G + (int)(row - (uint32_t)qi * G);
  const int p = past + qi;  // the lane's position
  // positions of the workgroup's and of the wave's rows
  const int first = past + (int)(r0 / G), last = past + (int)((min(rows, r0 + ROWS) - 1) / G);
  const int wfirst = past + (int)(min(rows - 1, rw) / G), wlast = past + (int)((min(rows, rw + 32) - 1) / G);
  const KeyTiles tiles = key_tiles<KT>(first, last, a.window, a.sinks);

  const T* qrow = reinterpret_cast<const T*>(a.q) + (size_t)(rt.q0 + qi) * a.q_ld + (size_t)hq * D;
  uint4 qf[QF];
#pragma unroll
  for (int t = 0; t < QF; ++t) qf[t] = *reinterpret_cast<const uint4*>(qrow + (BF ? 16 * t + 8 * h : 8 * t + 4 * h));
#pragma unroll
  for (int t = 0; t < QF; ++t) asm volatile("" : "+v"(qf[t].x));  // (awaited here, not in the loop)

  const T* kbase = reinterpret_cast<const T*>(a.k) + (size_t)rt.k0 * a.k_ld + (size_t)hk * D;
  const T* vbase = reinterpret_cast<const T*>(a.v) + (size_t)rt.k0 * a.v_ld + (size_t)hk * D;
  const uint32_t k_row = (uint32_t)a.k_ld * ES, v_row = (uint32_t)a.v_ld * ES;
  uint32_t koff[LW], voff[LW];
#pragma unroll
  for (int j = 0; j < LW; ++j) {
    const int r = (wave * LW + j) * RP + lane / CH;
    const uint32_t c = (uint32_t)((lane % CH) ^ swizzle<ROWB, T>(r)) << 4;
    koff[j] = (uint32_t)r * k_row + c;
    voff[j] = (uint32_t)r * v_row + c;
  }
  auto rsrc = [&](const T* base, long ld, uint32_t row_bytes, int p0) {
    const uint64_t at = (uint64_t)(uintptr_t)(base + (size_t)p0 * ld);
    const int there = min(KT, rt.nk - p0);
    return RsrcWords{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)at),
                     (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(at >> 32) & 0xffffu)),
                     (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(there - 1) * row_bytes + ROWB)), 0x00020000u};
  };
  auto issue = [&](int i, int stage) {
    const int p0 = tiles.at(i) * KT;
    const uint32_t at = (uint32_t)(uintptr_t)&lds[stage][0] + 1024 * LW * wave;
    const RsrcWords kr = rsrc(kbase, a.k_ld, k_row, p0), vr = rsrc(vbase, a.v_ld, v_row, p0);
#pragma unroll
    for (int j = 0; j < LW; ++j) load_lds(kr, koff[j], (uint32_t)__builtin_amdgcn_readfirstlane((int)(at + 1024 * j)));
#pragma unroll
    for (int j = 0; j < LW; ++j)
      load_lds(vr, voff[j], (uint32_t)__builtin_amdgcn_readfirstlane((int)(at + KT * ROWB + 1024 * j)));
  };

  af32x16 o[DT] = {};
  float top = -INFINITY, sum = 0.f;  // of the lane's row; sum: of the lane's keys
  auto edge = [&](int p0) {  // is there a row that does not see all of the tile
    return !(p0 + KT - 1 <= first && (a.window == 0 || last - p0 < a.window || p0 + KT <= a.sinks));
  };
  auto clean = [&](int stage) {  // zeros for what is not finite in V
    uint8_t* vs = &lds[stage][KT * ROWB];
#pragma unroll
    for (int j = 0; j < LW; ++j) {
      uint4* at = reinterpret_cast<uint4*>(vs + 1024 * (LW * wave + j) + 16 * lane);
      uint4 w = *at;
      if (clear_odd<T>(w)) {
        *at = w;
        dirty = 1;
      }
    }
  };
  auto compute = [&](int i, int stage) {
    const int p0 = tiles.at(i) * KT;
    // does a row of the wave see any of the tile, do all see all of it
    if (p0 > wlast || (a.window > 0 && p0 + KT <= wfirst - a.window + 1 && p0 >= a.sinks)) return;
    const bool whole = p0 + KT - 1 <= wfirst && (a.window == 0 || wlast - p0 < a.window || p0 + KT <= a.sinks);
    const uint8_t *ks = &lds[stage][0], *vs = ks + KT * ROWB;
    af32x16 st[ST] = {};
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
      for (int kk = 0; kk < QF; ++kk) {
        const uint4 kf = *reinterpret_cast<const uint4*>(ks + row_chunk<ROWB, T>(32 * t + m, 2 * kk + h));
        if constexpr (BF) {
          st[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(abf16x8, kf), __builtin_bit_cast(abf16x8, qf[kk]),
                                                          st[t], 0, 0, 0);
        } else {
          const uint32_t kw[4] = {kf.x, kf.y, kf.z, kf.w}, qw[4] = {qf[kk].x, qf[kk].y, qf[kk].z, qf[kk].w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            st[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(kw[e]), __uint_as_float(qw[e]), st[t], 0, 0, 0);
        }
      }
    float best = -INFINITY;
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        float x = st[t][e] * a.c;
        if (!whole) {
          const int j = p0 + 32 * t + 8 * (e >> 2) + 4 * h + (e & 3);
          x = j <= p && (a.window == 0 || p - j < a.window || j < a.sinks) ? x : -INFINITY;
        }
        st[t][e] = x;
        best = fmaxf(best, x);
      }
    const auto pair = __builtin_amdgcn_permlane32_swap(__float_as_uint(best), __float_as_uint(best), false, false);
    const float next = fmaxf(top, fmaxf(__uint_as_float(pair[0]), __uint_as_float(pair[1])));
    const float base = next == -INFINITY ? 0.f : next, keep = exp2_of(top - base);
    top = next;
    float add = 0.f;
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        st[t][e] = exp2_of(st[t][e] - base);
        add += st[t][e];
      }
    sum = fmaf(sum, keep, add);
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][e] *= keep;
    const int s = lane & 15;
    if constexpr (BF) {
#pragma unroll
      for (int t = 0; t < ST; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u) {  // 16 keys
          const abf16x8 pf = __builtin_bit_cast(
              abf16x8, make_uint4(pack_bf16x2(st[t][8 * u], st[t][8 * u + 1]), pack_bf16x2(st[t][8 * u + 2], st[t][8 * u + 3]),
                                  pack_bf16x2(st[t][8 * u + 4], st[t][8 * u + 5]), pack_bf16x2(st[t][8 * u + 6], st[t][8 * u + 7])));
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            const int r = 32 * t + 16 * u + 4 * h + (s >> 2), c = 4 * d + 2 * ((lane >> 4) & 1) + ((s & 3) >> 1);
            const uint2 v0 = lds_transposed(vs + row_chunk<ROWB, T>(r, c) + 8 * (s & 1));
            const uint2 v1 = lds_transposed(vs + row_chunk<ROWB, T>(r + 8, c) + 8 * (s & 1));
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(abf16x8, make_uint4(v0.x, v0.y, v1.x, v1.y)), pf,
                                                           o[d], 0, 0, 0);
          }
        }
    } else {
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int r = 8 * (e >> 2) + 4 * h + (e & 3);
          const float v = *reinterpret_cast<const float*>(vs + row_chunk<ROWB, T>(r, 8 * d + (m >> 2)) + 4 * (m & 3));
          o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, st[0][e], o[d], 0, 0, 0);
        }
    }
  };

  if (threadIdx.x == 0) dirty = 0;
  if (tiles.n > 0) issue(0, 0);
  for (int i = 0; i < tiles.n; ++i) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the tile is there, the other stage read
    if (i + 1 < tiles.n) issue(i + 1, (i + 1) & 1);
    if (edge(tiles.at(i) * KT)) {
      clean(i & 1);
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
    compute(i, i & 1);
  }

  const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
  sum = __uint_as_float(both[0]) + __uint_as_float(both[1]);
  const float inv = p < 0 ? 0.f : 1.f / sum;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] *= inv;
  uint32_t again = 0;  // the wave's rows that see what was zeroed
  if (tiles.n > 0 && dirty) {
    for (int i = 0; i < tiles.n; ++i) {
      const int p0 = tiles.at(i) * KT, j = p0 + lane;
      if (!edge(p0)) continue;
      bool bad = false;
      if (lane < KT && j < rt.nk)
        for (int c = 0; c < CH; ++c) {
          uint4 w = *reinterpret_cast<const uint4*>(vbase + (size_t)j * a.v_ld + c * (16 / ES));
          bad = clear_odd<T>(w) || bad;
        }
      if (__ballot(bad) == 0) continue;
      for (int l = 0; l < 32; ++l) {
        const int rp = __builtin_amdgcn_readlane(p, l);
        if (__ballot(bad && j <= rp && (a.window == 0 || rp - j < a.window || j < a.sinks))) again |= 1u << l;
      }
    }
    again &= (uint32_t)__ballot(real);
  }
  if (real && !(again >> m & 1)) {
    T* orow = reinterpret_cast<T*>(a.o) + ((size_t)(rt.q0 + qi) * a.Hq + hq) * D;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        io<T>::store4(orow + 32 * d + 2 * e + 4 * h, make_float4(o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]));
  }
  while (again != 0) {
    const int l = __builtin_ctz(again);
    again &= again - 1;
    const int lq = __builtin_amdgcn_readlane(qi, l), lh = __builtin_amdgcn_readlane(hq, l), lp = __builtin_amdgcn_readlane(p, l);
    win_row<T, D>(reinterpret_cast<const T*>(a.q) + (size_t)(rt.q0 + lq) * a.q_ld + (size_t)lh * D, kbase, a.k_ld, vbase,
                  a.v_ld, reinterpret_cast<T*>(a.o) + ((size_t)(rt.q0 + lq) * a.Hq + lh) * D, lp, a.window, a.sinks, a.c);
  }
}

template <int ROWS>
long row_tiles(const WinArgs& a) {
  const int G = a.Hq / a.Hk;
  if (a.cu_q == nullptr) return a.N * (((long)a.Tq * G + ROWS - 1) / ROWS);
  return ((long)a.Tq * G + ROWS - 1) / ROWS + a.N;  // (each sequence may leave a part of a tile)
}

template <typename T, int D, int NW>
bool launch_win_rows(WinArgs a, hipStream_t s) {
  const long tiles = row_tiles<32 * NW>(a);
  if (tiles * a.Hk > (1L << 32) / (64 * NW) - 1) return false;
  a.tiles = (int)tiles;
  hipLaunchKernelGGL((win_attn_kernel<T, D, NW>), dim3((unsigned)(tiles * a.Hk)), dim3(64 * NW), 0, s, a);
  return true;
}
// Rows of a workgroup: as many as leave one for every CU.
template <typename T, int D>
bool launch_win(const WinArgs& a, hipStream_t s) {
  const long cus = device_cus();
  if (row_tiles<256>(a) * a.Hk >= cus) return launch_win_rows<T, D, 8>(a, s);
  if (row_tiles<128>(a) * a.Hk >= cus) return launch_win_rows<T, D, 4>(a, s);
  return launch_win_rows<T, D, 2>(a, s);
}

}  // namespace
}  // namespace zgdn

extern "C" int zattn_window_fwd(const void* q, long q_ld, const void* k, long k_ld, const void* v, long v_ld, int dtype,
                                void* o, const int32_t* cu_q, const int32_t* cu_k, int n_seqs, int B, int Tq, int Tk, int Hq,
                                int Hk, int D, int window, int sinks, float scale, void* stream) {
  using namespace zgdn;
  const char* fn = "zattn_window_fwd";
  if (B < 1 || Tq < 0 || Tk < 0 || Hq < 1 || Hk < 1 || window < 0 || sinks < 0)
    return fail(ZGDN_EINVAL, "%s: bad sizes B=%d Tq=%d Tk=%d Hq=%d Hk=%d window=%d sinks=%d", fn, B, Tq, Tk, Hq, Hk, window,
                sinks);
  if (Hq % Hk) return fail(ZGDN_EINVAL, "%s: Hq=%d is not a multiple of Hk=%d", fn, Hq, Hk);
  if (D != 64 && D != 128) return fail(ZGDN_EUNSUPPORTED, "%s: D=%d (supported: 64 and 128)", fn, D);
  if (dtype != ZGDN_F32 && dtype != ZGDN_BF16) return fail(ZGDN_EINVAL, "%s: unknown dtype code %d", fn, dtype);
  if ((cu_q == nullptr) != (cu_k == nullptr)) return fail(ZGDN_EINVAL, "%s: cu_q and cu_k go together", fn);
  if (cu_q != nullptr && (B != 1 || n_seqs < 1))
    return fail(ZGDN_EINVAL, "%s: packed sequences need B == 1 and n_seqs >= 1 (B=%d n_seqs=%d)", fn, B, n_seqs);
  if ((long)B * Tq > (1L << 30) || (long)B * Tk > (1L << 30) || (long)B * Tq * Hq > (1L << 31))
    return fail(ZGDN_EUNSUPPORTED, "%s: B=%d x Tq=%d x Hq=%d, Tk=%d rows", fn, B, Tq, Hq, Tk);
  if (Tq == 0) return ZGDN_OK;
  if (!q || !o || (Tk > 0 && (!k || !v))) return fail(ZGDN_EINVAL, "%s: null tensor pointer", fn);
  const int ve = dtype == ZGDN_F32 ? 4 : 8;
  const long most = 1L << 22, wq = (long)Hq * D, wk = (long)Hk * D;
  auto bad = [&](long ld, long width) { return ld < width || ld > most || ld % ve; };
  if (bad(q_ld, wq) || bad(k_ld, wk) || bad(v_ld, wk))
    return fail(ZGDN_EINVAL, "%s: row strides q=%ld k=%ld v=%ld (multiples of %d elements, at least a row, at most 2^22)", fn,
                q_ld, k_ld, v_ld, ve);
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o) % 16)
    return fail(ZGDN_EINVAL, "%s: q, k, v and o need 16-byte aligned bases", fn);
  if (((uintptr_t)cu_q | (uintptr_t)cu_k) % 4) return fail(ZGDN_EINVAL, "%s: cu_q, cu_k not on 4-byte boundaries", fn);
  const size_t es = dtype == ZGDN_F32 ? 4 : 2, nq = (size_t)B * Tq, nk = (size_t)B * Tk, cu = ((size_t)n_seqs + 1) * 4;
  const Region out = {o, nq, wq * es, wq * es};
  const Region in[] = {{q, nq, wq * es, q_ld * es}, {k, nk, wk * es, k_ld * es}, {v, nk, wk * es, v_ld * es},
                       {cu_q, 1, cu, cu}, {cu_k, 1, cu, cu}};
  bool meet = false;
  for (const Region& r : in) meet = meet || regions_meet(out, r);
  if (meet) return fail(ZGDN_EINVAL, "%s: o overlaps another operand", fn);
  WinArgs a{q, k, v, q_ld, k_ld, v_ld, o, cu_q, cu_k, cu_q != nullptr ? n_seqs : B, Tq, Tk, Hq, Hk, window, sinks,
            scale * LOG2E, 0};
  hipStream_t s = (hipStream_t)stream;
  const bool ok = dtype == ZGDN_F32 ? (D == 128 ? launch_win<float, 128>(a, s) : launch_win<float, 64>(a, s))
                                    : (D == 128 ? launch_win<bf16, 128>(a, s) : launch_win<bf16, 64>(a, s));
  if (!ok) return fail(ZGDN_EUNSUPPORTED, "%s: B=%d x Tq=%d x Hq=%d rows", fn, B, Tq, Hq);
  return check_launch(fn);
}
