// y = act(x w^T + bias) + residual on bf16 MFMA, fp32 sums, the epilogue in fp32, rounded once.
//
// Tiles are computed transposed (A = rows of w, B = rows of x: v_mfma_f32_16x16x32_bf16, D: w row 4 g + e, x row lane % 16),
// two tiles of w rows interleaved, so that a lane ends with 8 neighbouring columns of one row of y: bias, residual and y
// are 16-byte accesses. Three forms, chosen by launch (below):
//   gemm_act_tile   BM x BN tiles, both operands by direct-to-LDS loads in blocks of 64 of K, several blocks ahead;
//   gemm_act_split  few rows (a decode step): small tiles, K split over the workgroup's waves;
//   gemm_act_any    rows off 16-byte boundaries, K not a multiple of 8: loads through registers.
#include <algorithm>
#include <atomic>

#include "gdn_common.h"
#include "zonos3_linear.h"

namespace zgdn {
namespace {

typedef __bf16 abf16x8 __attribute__((ext_vector_type(8)));
typedef float af32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t au32x4 __attribute__((ext_vector_type(4)));

struct ActArgs {
  const uint16_t *x, *w;
  long x_ld, w_ld;
  const void* bias;
  int bias_bf16, act;
  const uint16_t* res;
  long r_ld;
  uint16_t* y;
  long y_ld;
  int M, N, K;
  int vec;  // elements that one access of y and the residual may take: 8, 4 or 1
  int tiles_m, tiles_n;
};

template <int ACT>
__device__ __forceinline__ float act_of(float x) {
  if constexpr (ACT == ZLIN_RELU) return x > 0.f || x != x ? x : 0.f;
  if constexpr (ACT == ZLIN_SILU) return silu_fast(x);
  if constexpr (ACT == ZLIN_GELU) return 0.5f * x * (1.f + erff(x * 0.70710678118654752f));
  if constexpr (ACT == ZLIN_GELU_TANH)  // 0.5 (1 + tanh u) = 1 / (1 + exp(-2 u))
    return x * __builtin_amdgcn_rcpf(1.f + __expf(-2.f * 0.79788456080286536f * (x + 0.044715f * x * x * x)));
  return x;
}

__device__ __forceinline__ float bias_at(const ActArgs& a, int n) {
  return a.bias_bf16 ? bf16_to_f32(reinterpret_cast<const uint16_t*>(a.bias)[n]) : reinterpret_cast<const float*>(a.bias)[n];
}

// Columns n .. n + C - 1 of row m, sums c (bias added already).
template <int ACT, int C>
__device__ __forceinline__ void finish(const ActArgs& a, int m, int n, float (&c)[C]) {
  if (m >= a.M || n >= a.N) return;
#pragma unroll
  for (int e = 0; e < C; ++e) c[e] = act_of<ACT>(c[e]);
  const size_t yi = (size_t)m * a.y_ld + n, ri = (size_t)m * a.r_ld + n;
  if (a.vec >= C && n + C <= a.N) {
    uint32_t r[C / 2];
    if (a.res != nullptr) {
      if constexpr (C == 8) {
        const uint4 v = *reinterpret_cast<const uint4*>(a.res + ri);
        r[0] = v.x, r[1] = v.y, r[2] = v.z, r[3] = v.w;
      } else {
        const uint2 v = *reinterpret_cast<const uint2*>(a.res + ri);
        r[0] = v.x, r[1] = v.y;
      }
#pragma unroll
      for (int e = 0; e < C; e += 2) {
        c[e] += __uint_as_float(r[e / 2] << 16);
        c[e + 1] += __uint_as_float(r[e / 2] & 0xffff0000u);
      }
    }
#pragma unroll
    for (int e = 0; e < C; e += 2) r[e / 2] = pack_bf16x2(c[e], c[e + 1]);
    if constexpr (C == 8)
      *reinterpret_cast<uint4*>(a.y + yi) = make_uint4(r[0], r[1], r[2], r[3]);
    else
      *reinterpret_cast<uint2*>(a.y + yi) = make_uint2(r[0], r[1]);
  } else {
#pragma unroll
    for (int e = 0; e < C; ++e) {
      if (n + e >= a.N) break;
      float v = c[e];
      if (a.res != nullptr) v += bf16_to_f32(a.res[ri + e]);
      a.y[yi + e] = f32_to_bf16(v);
    }
  }
}

template <typename F>
__device__ __forceinline__ void with_act(int act, F f) {
  switch (act) {
    case ZLIN_RELU: return f(std::integral_constant<int, ZLIN_RELU>{});
    case ZLIN_SILU: return f(std::integral_constant<int, ZLIN_SILU>{});
    case ZLIN_GELU: return f(std::integral_constant<int, ZLIN_GELU>{});
    case ZLIN_GELU_TANH: return f(std::integral_constant<int, ZLIN_GELU_TANH>{});
    default: return f(std::integral_constant<int, ZLIN_NONE>{});
  }
}

__device__ __forceinline__ af32x4 amfma(abf16x8 a, abf16x8 b, af32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// A buffer of `rows` rows, K elements of each, for loads by byte offset (zeros behind its end).
__device__ __forceinline__ au32x4 rows_rsrc(const uint16_t* p, long ld, int rows, int K) {
  const uint64_t at = (uint64_t)(uintptr_t)p;
  const uint32_t bytes = rows > 0 ? (uint32_t)(rows - 1) * (uint32_t)ld * 2u + (uint32_t)K * 2u : 0u;
  return au32x4{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)at),
                (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(at >> 32) & 0xffffu)),
                (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
}

__device__ __forceinline__ uint32_t lds_at(const void* p) {
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)(uintptr_t)(__attribute__((address_space(3))) const void*)p);
}
constexpr uint32_t NOWHERE = 0x80000000u;  // a byte offset behind every buffer's end: such a lane gets zeros

template <int N>
__device__ __forceinline__ void wait_and_meet() {  // at most N of the wave's loads outstanding, then a barrier
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// ------------------------------------------------------------------------------------------------------- tiles
//
// 8 waves, WM of them along the rows of x: BM x BN tiles, a wave BM / WM x BN / WN of it. Blocks of BK = 64 of K in NS
// stages of LDS (128-byte rows, 16-byte chunk c of row r at c ^ f(r)): block kb computes while the next ones land. The
// fragments of a block's second half are read under the products of its first, those of the next block's first half under
// the products of its second (read right before their own products they cost the same within noise: 8192 x 4096 x 4096 221 us
// either way, 4096 x 2056 x 1024 22.9 and 22.7; the library's product of the first takes 178).
// Fragment reads touch 16 rows, one chunk each: f spreads rows 0 .. 15 (x) and rows 8 a + b, b < 4 (w, whose fragments
// interleave) over all 16 places of 256 bytes.
// FOLD: the at most 16 columns behind the last full tile are formed by the tiles (row block tm, column tile tn: rows
// 16 tn .. of its block), not by a column of tiles of their own (4096 x 2056 x 1024 with bias
// and SiLU, whole calls: 30.9 us, 22.7 so).

constexpr int BK = 64;

__device__ __forceinline__ int fx(int r) { return (r >> 1) & 7; }
__device__ __forceinline__ int fw(int r) { return (r >> 1 & 1) | (r >> 3 & 3) << 1; }

template <int BM, int BN, int WM, int NS_, bool FOLD>
struct TileCfg {
  static constexpr int WN = 8 / WM;
  static constexpr int TM = BM / WM / 16, TN = BN / WN / 32;  // 16-row tiles of x, 32-row pairs of w, a wave
  static constexpr int STAGE = (BM + BN + (FOLD ? 16 : 0)) * 128;
  static constexpr int NS = NS_;
  static constexpr int LDS = NS * STAGE;
  static constexpr int PX = BM / 8 / 8, PW = BN / 8 / 8;  // 1 KiB pieces (8 rows) of each operand a wave
  static constexpr int PER_CU = LDS <= 80 * 1024 ? 2 : 1;
  static_assert(!FOLD || NS == 2, "the folded rows' two pieces are not counted");
};

template <int BM, int BN, int WM, int NS, bool FOLD>
__global__ __launch_bounds__(512, (2 * TileCfg<BM, BN, WM, NS, FOLD>::PER_CU)) void gemm_act_tile_kernel(ActArgs a) {
  using C = TileCfg<BM, BN, WM, NS, FOLD>;
  constexpr int TM = C::TM, TN = C::TN;
  extern __shared__ uint4 act_lds[];
  uint8_t* lds = reinterpret_cast<uint8_t*>(act_lds);
  // workgroups go round-robin over the 8 XCDs: each XCD takes a run of tiles, in bands of 8 column tiles, row tile by row
  // tile, so that its L2 holds a band of w and the rows at hand
  const int total = a.tiles_m * a.tiles_n, per = (total + 7) / 8;
  const int t = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || t >= total) return;
  const int band = t / (8 * a.tiles_m), in = t - band * 8 * a.tiles_m, width = min(8, a.tiles_n - 8 * band);
  const int tm = in / width, tn = 8 * band + in - tm * width;
  const int m0 = __builtin_amdgcn_readfirstlane(tm * BM), n0 = __builtin_amdgcn_readfirstlane(tn * BN);
  const int wave = wave_id(), l = threadIdx.x & 63, m = l & 15, g = l >> 4;
  const int wm = (wave % WM) * (BM / WM), wn = (wave / WM) * (BN / C::WN);
  const au32x4 rx = rows_rsrc(a.x + (size_t)m0 * a.x_ld, a.x_ld, min(BM, a.M - m0), a.K);
  const au32x4 rw = rows_rsrc(a.w + (size_t)n0 * a.w_ld, a.w_ld, min(BN, a.N - n0), a.K);
  uint32_t ox[C::PX], ow[C::PW];  // the lane's offsets in its pieces (piece p: rows 8 p .. + 7)
  int cx[C::PX], cw[C::PW];       // and chunks
#pragma unroll
  for (int i = 0; i < C::PX; ++i) {
    const int r = 8 * (wave + 8 * i) + (l >> 3);
    cx[i] = (l & 7) ^ fx(r);
    ox[i] = (uint32_t)r * (uint32_t)a.x_ld * 2u + 16u * cx[i];
  }
#pragma unroll
  for (int i = 0; i < C::PW; ++i) {
    const int r = 8 * (wave + 8 * i) + (l >> 3);
    cw[i] = (l & 7) ^ fw(r);
    ow[i] = (uint32_t)r * (uint32_t)a.w_ld * 2u + 16u * cw[i];
  }
  // the folded columns: 16 rows of w, two pieces, by waves 0 and 1; their products by the wave that holds rows 16 tn
  const int nf0 = a.tiles_n * BN;
  const bool fold = FOLD && 16 * tn < BM, fold_mine = fold && wave == (16 * tn) / (BM / WM) + WM * (tn % C::WN);
  au32x4 rf = {0u, 0u, 0u, 0u};
  uint32_t of = 0;
  int cf = 0;
  af32x4 facc = {0.f, 0.f, 0.f, 0.f};
  if constexpr (FOLD) {
    rf = rows_rsrc(a.w + (size_t)nf0 * a.w_ld, a.w_ld, a.N - nf0, a.K);
    const int r = 8 * (wave & 1) + (l >> 3);
    cf = (l & 7) ^ fx(r);
    of = (uint32_t)r * (uint32_t)a.w_ld * 2u + 16u * cf;
  }
  const int nk = (a.K + BK - 1) / BK, tail = a.K - (nk - 1) * BK;  // elements of the last block
  const uint32_t base = lds_at(lds);
  auto issue = [&](int kb, int stage) {
    const uint32_t at = base + stage * C::STAGE + 1024 * wave, k = (uint32_t)min(kb, nk - 1) * BK * 2;
    const bool cut = kb >= nk - 1;  // (behind the last block: it again, unread)
#pragma unroll
    for (int i = 0; i < C::PX; ++i) load_lds(rx, cut && 8 * cx[i] >= tail ? NOWHERE : ox[i], k, at + 8192 * i);
#pragma unroll
    for (int i = 0; i < C::PW; ++i) load_lds(rw, cut && 8 * cw[i] >= tail ? NOWHERE : ow[i], k, at + BM * 128 + 8192 * i);
    if constexpr (FOLD) {
      if (fold && wave < 2) load_lds(rf, cut && 8 * cf >= tail ? NOWHERE : of, k, at + (BM + BN) * 128);
    }
  };

  af32x4 acc[TN][2][TM];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < TM; ++j) acc[i][u][j] = af32x4{0.f, 0.f, 0.f, 0.f};
  // w rows of fragment u of a pair: 8 (m / 4) + 4 u + m % 4
  const int rwl = wn + 8 * (m >> 2) + (m & 3), rxl = wm + m;
  struct Frags {
    abf16x8 x[TM], w[TN][2], fx_, fw_;
  };
  auto read = [&](Frags& f, int stage, int s) {
    const uint8_t* xs = lds + stage * C::STAGE;
    const uint8_t* ws = xs + BM * 128;
#pragma unroll
    for (int j = 0; j < TM; ++j)
      f.x[j] = *reinterpret_cast<const abf16x8*>(xs + (rxl + 16 * j) * 128 + (((4 * s + g) ^ fx(rxl)) << 4));
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int u = 0; u < 2; ++u)
        f.w[i][u] = *reinterpret_cast<const abf16x8*>(ws + (rwl + 32 * i + 4 * u) * 128 + (((4 * s + g) ^ fw(rwl)) << 4));
    if constexpr (FOLD) {
      if (fold_mine) {
        f.fx_ = *reinterpret_cast<const abf16x8*>(xs + (16 * tn + m) * 128 + (((4 * s + g) ^ fx(m)) << 4));
        f.fw_ = *reinterpret_cast<const abf16x8*>(ws + (BN + m) * 128 + (((4 * s + g) ^ fx(m)) << 4));
      }
    }
  };
  auto multiply = [&](const Frags& f) {
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][u][j] = amfma(f.w[i][u], f.x[j], acc[i][u][j]);
    if constexpr (FOLD) {
      if (fold_mine) facc = amfma(f.fw_, f.fx_, facc);
    }
  };
#pragma unroll
  for (int s = 0; s < NS - 1; ++s) issue(s, s);
  wait_and_meet<(NS - 2) * (C::PX + C::PW)>();
  issue(NS - 1, NS - 1);
  Frags f0, f1;
  read(f0, 0, 0);
  int st = 0;
  for (int kb = 0; kb < nk; ++kb) {
    read(f1, st, 1);
    __builtin_amdgcn_sched_barrier(0);
    multiply(f0);
    __builtin_amdgcn_sched_barrier(0);
    // block kb + 1 is there, and everybody has read all of block kb: its stage takes block kb + NS
    wait_and_meet<(NS - 2) * (C::PX + C::PW)>();
    issue(kb + NS, st);
    st = st == NS - 1 ? 0 : st + 1;
    read(f0, st, 0);
    __builtin_amdgcn_sched_barrier(0);
    multiply(f1);
    __builtin_amdgcn_sched_barrier(0);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  with_act(a.act, [&](auto act) {
    constexpr int ACT = decltype(act)::value;
    if (a.vec == 8 && n0 + BN <= a.N) {  // whole column tiles: rows behind M read zeros and are dropped by the buffers' bounds
      const int rows = min(BM, a.M - m0);
      const Rsrc ry = raw_rsrc(a.y + (size_t)m0 * a.y_ld,
                               (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(rows - 1) * (uint32_t)a.y_ld * 2u + (uint32_t)a.N * 2u)));
      const Rsrc rr = raw_rsrc(a.res + (size_t)m0 * a.r_ld,
                               (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(rows - 1) * (uint32_t)a.r_ld * 2u + (uint32_t)a.N * 2u)));
      au32x4 r[TN][TM];  // (all of a lane's, ahead of the first store: one wait for memory; 30526 x 1024 x 2048: 135 us half by half, 132 so)
      if (a.res != nullptr) {
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
          for (int j = 0; j < TM; ++j)
            r[i][j] = __builtin_amdgcn_raw_buffer_load_b128(
                rr, (uint32_t)(wm + 16 * j + m) * (uint32_t)a.r_ld * 2u + 2u * (n0 + wn + 32 * i + 8 * g), 0, 0);
      }
#pragma unroll
      for (int i = 0; i < TN; ++i) {
        const int n = n0 + wn + 32 * i + 8 * g;
        float b[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) b[e] = a.bias != nullptr ? bias_at(a, n + e) : 0.f;
#pragma unroll
        for (int j = 0; j < TM; ++j) {
          float c[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) c[e] = act_of<ACT>(acc[i][e >> 2][j][e & 3] + b[e]);
          if (a.res != nullptr) {
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
              c[e] += __uint_as_float(r[i][j][e / 2] << 16);
              c[e + 1] += __uint_as_float(r[i][j][e / 2] & 0xffff0000u);
            }
          }
          const au32x4 y = {pack_bf16x2(c[0], c[1]), pack_bf16x2(c[2], c[3]), pack_bf16x2(c[4], c[5]), pack_bf16x2(c[6], c[7])};
          __builtin_amdgcn_raw_buffer_store_b128(y, ry, (uint32_t)(wm + 16 * j + m) * (uint32_t)a.y_ld * 2u + 2u * n, 0, 0);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < TN; ++i) {
        const int n = n0 + wn + 32 * i + 8 * g;
        float b[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) b[e] = a.bias != nullptr ? bias_at(a, min(n + e, a.N - 1)) : 0.f;
#pragma unroll
        for (int j = 0; j < TM; ++j) {
          float c[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) c[e] = acc[i][e >> 2][j][e & 3] + b[e];
          finish<ACT>(a, m0 + wm + 16 * j + m, n, c);
        }
      }
    }
    if constexpr (FOLD) {
      if (fold_mine) {
        const int n = nf0 + 4 * g;
        float c[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e] = facc[e] + (a.bias != nullptr ? bias_at(a, min(n + e, a.N - 1)) : 0.f);
        finish<ACT>(a, m0 + 16 * tn + m, n, c);
      }
    }
  });
}

// ---------------------------------------------------------------------------------------------- K split over waves
//
// 16 R x 16 R tiles (R 1: a decode step's rows; R 2: more rows, still too few tiles of 64 x 128 for the CUs), K in slices of
// SL = 128 / R elements, slice q to wave q % 8: such a call is the weights' way from memory and a few round trips, so each
// wave keeps two slices of both operands on their way (direct-to-LDS, whole runs of 256 / R bytes of a row; chunk c of a
// row at c ^ f(row)) and waits for nobody before its products. The 8 partial tiles are added in LDS in wave order. The row
// tiles of one column tile run on one XCD where they can, and share its copy of the weights (whole column tiles by XCD leave
// most of the XCDs idle where there are fewer than 8: 21614 x 17 x 5168 307 us, 56 in runs of tiles).

constexpr int RW = 8;  // waves
template <int R>
struct SplitCfg {
  static constexpr int SL = 128 / R, RB = 2 * SL, CH = RB / 16;  // elements, bytes, chunks of a row's slice
  static constexpr int OP = 16 * R * RB;                         // bytes of one operand's slice: 4 KiB
  static constexpr int LDS = RW * 2 * 2 * OP;                    // two slices of both, a wave: 128 KiB
  __device__ static __forceinline__ int f(int r) { return R == 1 ? r & 15 : (r >> 1) & 7; }
};

struct __attribute__((packed, aligned(2))) Packed8 {
  uint32_t w[4];
};
// 8 elements from p on, wherever that is; of these only `n` (zeros behind them).
__device__ __forceinline__ uint4 fetch8(const uint16_t* p) {
  const Packed8 x = *reinterpret_cast<const Packed8*>(p);
  return make_uint4(x.w[0], x.w[1], x.w[2], x.w[3]);
}
__device__ __forceinline__ uint4 fetch8_upto(const uint16_t* p, int n) {
  if (n >= 8) return fetch8(p);
  uint32_t u[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) u[i] = i < n ? p[i] : 0u;
  return make_uint4(u[0] | u[1] << 16, u[2] | u[3] << 16, u[4] | u[5] << 16, u[6] | u[7] << 16);
}

// WIDE false: rows off 16-byte boundaries or K not a multiple of 8, the slices through registers.
template <int R, bool WIDE>
__global__ __launch_bounds__(64 * RW) void gemm_act_split_kernel(ActArgs a) {
  using C = SplitCfg<R>;
  extern __shared__ uint4 act_lds[];
  uint8_t* lds = reinterpret_cast<uint8_t*>(act_lds);
  // each XCD (workgroups go round-robin over the 8) takes a run of tiles, column tile by column tile
  const int total = a.tiles_m * a.tiles_n, per = (total + 7) / 8, t = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (t >= total) return;
  const int tn = t / a.tiles_m, tm = t - tn * a.tiles_m;
  const int wave = wave_id(), l = threadIdx.x & 63, m = l & 15, g = l >> 4;
  const int m0 = __builtin_amdgcn_readfirstlane(16 * R * tm), n0 = __builtin_amdgcn_readfirstlane(16 * R * tn);
  const au32x4 rx = rows_rsrc(a.x + (size_t)m0 * a.x_ld, a.x_ld, min(16 * R, a.M - m0), a.K);
  const au32x4 rw = rows_rsrc(a.w + (size_t)n0 * a.w_ld, a.w_ld, min(16 * R, a.N - n0), a.K);
  uint8_t* mine = lds + wave * 4 * C::OP;
  const uint32_t base = lds_at(mine);
  uint4 vw[4], vx[4];
  auto issue = [&](int q, int half) {  // slice q of the wave's
    const int k0 = (q * RW + wave) * C::SL;
#pragma unroll
    for (int p = 0; p < 4; ++p) {  // 1 KiB: 64 / CH rows
      const int r = p * (64 / C::CH) + l / C::CH, c = (l % C::CH) ^ C::f(r);
      if constexpr (!WIDE) {
        // (rows behind the last: the last, whose products nobody stores)
        vw[p] = fetch8_upto(a.w + (size_t)min(n0 + r, a.N - 1) * a.w_ld + k0 + 8 * c, a.K - k0 - 8 * c);
        vx[p] = fetch8_upto(a.x + (size_t)min(m0 + r, a.M - 1) * a.x_ld + k0 + 8 * c, a.K - k0 - 8 * c);
        continue;
      }
      const bool there = k0 + 8 * c < a.K;
      load_lds(rw, there ? (uint32_t)r * (uint32_t)a.w_ld * 2u + 16u * c : NOWHERE, (uint32_t)k0 * 2u, base + half * 2 * C::OP + 1024 * p);
      load_lds(rx, there ? (uint32_t)r * (uint32_t)a.x_ld * 2u + 16u * c : NOWHERE, (uint32_t)k0 * 2u, base + half * 2 * C::OP + C::OP + 1024 * p);
    }
  };
  const int slices = (a.K + C::SL * RW - 1) / (C::SL * RW);  // (a wave's last may lie behind K: zeros)
  af32x4 acc[R][R];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < R; ++j) acc[i][j] = af32x4{0.f, 0.f, 0.f, 0.f};
  issue(0, 0);
  for (int q = 0; q < slices; ++q) {
    if constexpr (!WIDE) {
      uint8_t* at = mine + (q & 1) * 2 * C::OP + 16 * l;
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        *reinterpret_cast<uint4*>(at + 1024 * p) = vw[p];
        *reinterpret_cast<uint4*>(at + C::OP + 1024 * p) = vx[p];
      }
      if (q + 1 < slices) issue(q + 1, 0);
    } else if (q + 1 < slices) {
      issue(q + 1, (q + 1) & 1);
      asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    const uint8_t* ws = mine + (q & 1) * 2 * C::OP;
#pragma unroll
    for (int s = 0; s < C::SL / 32; ++s) {
      abf16x8 fa[R], fb[R];
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int at = (16 * i + m) * C::RB + (((4 * s + g) ^ C::f(m)) << 4);
        fa[i] = *reinterpret_cast<const abf16x8*>(ws + at);
        fb[i] = *reinterpret_cast<const abf16x8*>(ws + C::OP + at);
      }
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < R; ++j) acc[i][j] = amfma(fa[i], fb[j], acc[i][j]);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the load after the next overwrites the slice)
  }
  __syncthreads();
  float* part = reinterpret_cast<float*>(lds);  // [tile][wave][lane][4]
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < R; ++j) *reinterpret_cast<af32x4*>(part + ((i * R + j) * RW + wave) * 256 + 4 * l) = acc[i][j];
  __syncthreads();
  if (wave < R * R) {
    float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < RW; ++w) {
      const af32x4 p = *reinterpret_cast<const af32x4*>(part + (wave * RW + w) * 256 + 4 * l);
#pragma unroll
      for (int e = 0; e < 4; ++e) c[e] += p[e];
    }
    const int n = n0 + 16 * (wave / R) + 4 * g;
    if (a.bias != nullptr) {
#pragma unroll
      for (int e = 0; e < 4; ++e) c[e] += bias_at(a, min(n + e, a.N - 1));
    }
    with_act(a.act, [&](auto act) { finish<decltype(act)::value>(a, m0 + 16 * (wave % R) + m, n, c); });
  }
}

// Any sizes and alignments: T x T tiles, 4 waves of T / 2 x T / 2, blocks of 64 of K through registers (loaded two blocks
// ahead: 8 elements of a row at a time from wherever it starts, one by one at the end of K; rows behind the last: the last,
// whose products nobody stores) into two stages of LDS (128-byte rows, 16-byte chunks swizzled by row).
template <int T>
__global__ __launch_bounds__(256) void gemm_act_any_kernel(ActArgs a) {
  constexpr int W = T / 32, L = T / 32;  // 16-row tiles a wave and side; 8-element pieces a thread and operand
  __shared__ uint4 sx[2][T * 8], sw[2][T * 8];
  // each XCD takes a run of tiles, row tile by row tile
  const int total = a.tiles_m * a.tiles_n, per = (total + 7) / 8, at = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (at >= total) return;
  const int n0 = (at % a.tiles_n) * T, m0 = (at / a.tiles_n) * T;
  const int wave = wave_id(), l = threadIdx.x & 63, m = l & 15, g = l >> 4;
  const int wm = (wave & 1) * (T / 2), wn = (wave >> 1) * (T / 2);
  af32x4 acc[W][W];
#pragma unroll
  for (int i = 0; i < W; ++i)
#pragma unroll
    for (int j = 0; j < W; ++j) acc[i][j] = af32x4{0.f, 0.f, 0.f, 0.f};
  const int c = threadIdx.x & 7;
  const uint16_t *xp[L], *wp[L];
#pragma unroll
  for (int i = 0; i < L; ++i) {
    const int r = (threadIdx.x >> 3) + 32 * i;
    xp[i] = a.x + (size_t)min(m0 + r, a.M - 1) * a.x_ld + 8 * c;
    wp[i] = a.w + (size_t)min(n0 + r, a.N - 1) * a.w_ld + 8 * c;
  }
  uint4 px[2][L], pw[2][L];
  auto load = [&](int kb, int s) {
    if (64 * kb + 64 <= a.K) {
#pragma unroll
      for (int i = 0; i < L; ++i) {
        px[s][i] = fetch8(xp[i] + 64 * kb);
        pw[s][i] = fetch8(wp[i] + 64 * kb);
      }
    } else {
#pragma unroll
      for (int i = 0; i < L; ++i) {
        px[s][i] = fetch8_upto(xp[i] + 64 * kb, a.K - 64 * kb - 8 * c);
        pw[s][i] = fetch8_upto(wp[i] + 64 * kb, a.K - 64 * kb - 8 * c);
      }
    }
  };
  const int nk = (a.K + 63) / 64;
  auto block = [&](int kb, int s) {
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const int r = (threadIdx.x >> 3) + 32 * i;
      sx[s][r * 8 + (c ^ fx(r))] = px[s][i];
      sw[s][r * 8 + (c ^ fx(r))] = pw[s][i];
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the block is there, the other stage read by everybody
    if (kb + 2 < nk) load(kb + 2, s);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      abf16x8 fa[W], fb[W];
#pragma unroll
      for (int i = 0; i < W; ++i) {
        fa[i] = __builtin_bit_cast(abf16x8, sw[s][(wn + 16 * i + m) * 8 + ((4 * t + g) ^ fx(m))]);
        fb[i] = __builtin_bit_cast(abf16x8, sx[s][(wm + 16 * i + m) * 8 + ((4 * t + g) ^ fx(m))]);
      }
#pragma unroll
      for (int i = 0; i < W; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j) acc[i][j] = amfma(fa[i], fb[j], acc[i][j]);
    }
  };
  load(0, 0);
  if (nk > 1) load(1, 1);
  for (int kb = 0; kb < nk; kb += 2) {
    block(kb, 0);
    if (kb + 1 < nk) block(kb + 1, 1);
  }
  with_act(a.act, [&](auto act) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int n = n0 + wn + 16 * i + 4 * g;
      float b[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) b[e] = a.bias != nullptr ? bias_at(a, min(n + e, a.N - 1)) : 0.f;
#pragma unroll
      for (int j = 0; j < W; ++j) {
        float c[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e] = acc[i][j][e] + b[e];
        finish<decltype(act)::value>(a, m0 + wm + 16 * j + m, n, c);
      }
    }
  });
}

// LDS above the default 64 KiB, allowed once per device and kernel; false when the device refuses.
template <typename F>
bool lds_ready(F kernel, int bytes, std::atomic<signed char>* state) {
  if (bytes <= 65536) return true;
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return false;
  const signed char s = state[dev].load(std::memory_order_acquire);
  if (s != 0) return s > 0;
  const bool ok = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess;
  if (!ok) (void)hipGetLastError();
  state[dev].store(ok ? 1 : -1, std::memory_order_release);
  return ok;
}

template <int R, bool WIDE>
int launch_split(const char* fn, ActArgs a, hipStream_t s) {
  using C = SplitCfg<R>;
  static std::atomic<signed char> state[64];
  if (!lds_ready(gemm_act_split_kernel<R, WIDE>, C::LDS, state)) return fail(ZGDN_EHIP, "%s: the device refused the LDS", fn);
  a.tiles_m = (a.M + 16 * R - 1) / (16 * R), a.tiles_n = (a.N + 16 * R - 1) / (16 * R);
  hipLaunchKernelGGL((gemm_act_split_kernel<R, WIDE>), dim3((unsigned)(((long)a.tiles_m * a.tiles_n + 7) / 8 * 8)), dim3(64 * RW), C::LDS, s, a);
  return ZGDN_OK;
}

template <int T>
int launch_any(ActArgs a, hipStream_t s) {
  a.tiles_m = (a.M + T - 1) / T, a.tiles_n = (a.N + T - 1) / T;
  hipLaunchKernelGGL(gemm_act_any_kernel<T>, dim3((unsigned)(((long)a.tiles_m * a.tiles_n + 7) / 8 * 8)), dim3(256), 0, s, a);
  return ZGDN_OK;
}

template <int BM, int BN, int WM, int NS, bool FOLD = false>
int launch_tiles(const char* fn, ActArgs a, hipStream_t s) {
  using C = TileCfg<BM, BN, WM, NS, FOLD>;
  static std::atomic<signed char> state[64];
  if (!lds_ready(gemm_act_tile_kernel<BM, BN, WM, NS, FOLD>, C::LDS, state))
    return fail(ZGDN_EHIP, "%s: the device refused the LDS", fn);
  a.tiles_m = (a.M + BM - 1) / BM, a.tiles_n = FOLD ? a.N / BN : (a.N + BN - 1) / BN;
  const long per = ((long)a.tiles_m * a.tiles_n + 7) / 8;
  hipLaunchKernelGGL((gemm_act_tile_kernel<BM, BN, WM, NS, FOLD>), dim3((unsigned)(8 * per)), dim3(512), C::LDS, s, a);
  return ZGDN_OK;
}

// Which form takes the least time, by what each was measured to take (us, MI355X, graph replays): a fixed part and, a round
// of workgroups over the CUs, a part for each block of K. `one`, `all`: with one workgroup a CU, with all that fit.
struct Form {
  int bm, bn, bk, per_cu, threads;
  double fixed, round, one, all;
};
enum FormCode { F_NONE, F_SPLIT16, F_SPLIT32, F_TILE64, F_FOLD, F_WIDE, F_TILE256, F_ANY64, F_ANY128, F_COUNT };
// The fit's points (M x N x K, us in graph replays), the form taken and the next best: 4 x 2056 x 1024 3.4 split 16, 4.0
// split 32; 64 x 1024 x 2048 4.4 split 16, 4.9 split 32; 64 x 2056 x 1024 4.1 split 32, 6.1 split 16; 200 x 1024 x 2048 5.5
// split 32, 11.9 tile 64 x 128; 400 x 2056 x 1024 8.0 tile 64 x 128, 11.5 split 32; 1000 x 2056 x 1024 12.4 tile 64 x 128,
// 13.9 128 x 128; 4096 x 2056 x 1024 23.8 tile 128 x 128 (its last 8 columns folded), 29.6 256 x 256; 30526 x 1024 x 2048
// 113 tile 256 x 256, 134 128 x 128 and 128 x 256. (128 x 128 without folded columns is no form: twice as many tiles of
// 64 x 128 take less at every size.) Between them the rule is off by up to a quarter where columns are few (us of calls, taken
// / best): 30000 x 32 x 1024 19.5 split 32 / 15.7 tile 64 x 128, 5104 x 72 x 2176 14.2 split 32 / 12.8 tile 64 x 128; it is
// right at 21614 x 17 x 5168 (56 split 32, 67) and 8192 x 64 x 4096 (25 split 32, 29).
// Rows off 16-byte boundaries, where the split forms go through registers at 2.1 times their figures (us of calls; the form
// taken in brackets):
//                          split 16   split 32   any 64   any 128
//   4 x 2056 x 1025          [6.8]       7.6      13.2     24.5
//   512 x 64 x 8193         [13.6]      23.4      74.6    149
//   64 x 2056 x 1025         14.4       [7.2]     13.0     25.9
//   1260 x 362 x 1869        50.5      [19.8]     22.1     43.3
//   3000 x 300 x 300         52.3       18.9      [6.8]    12.4
//   5836 x 1038 x 1501      562        185        68.7    [51.7]
//   20000 x 1000 x 1001    1209        412       122      [98.3]
constexpr Form FORMS[F_COUNT] = {
    {},
    {16, 16, 1024, 1, 512, 1.5, 1.0, 0.6, 0.6},
    {32, 32, 512, 1, 512, 1.5, 1.0, 0.7, 0.7},
    {64, 128, 64, 2, 512, 3.0, 0.0, 0.275, 0.52},
    {128, 128, 64, 2, 512, 3.0, 0.0, 0.66, 1.15},
    {128, 256, 64, 1, 512, 3.0, 0.0, 0.96, 0.98},
    {256, 256, 64, 1, 512, 3.0, 0.0, 1.62, 1.65},
    {64, 64, 64, 2, 256, 3.0, 0.0, 0.75, 1.0},
    {128, 128, 64, 1, 256, 3.0, 0.0, 1.2, 1.2},
};
constexpr double NEVER = 1e300;

// Columns behind the last whole tile of 128 that the tiles before them form as well (see gemm_act_tile_kernel); else 0.
int folded(int N) {
  const int over = N % 128;
  return over <= 16 && N / 128 >= 8 ? over : 0;
}
long workgroups(const Form& f, long M, long cols) {  // (whole rounds over the 8 XCDs)
  return (((M + f.bm - 1) / f.bm) * ((cols + f.bn - 1) / f.bn) + 7) / 8 * 8;
}
double form_us(const Form& f, long M, long cols, long K, long n_cu) {
  if (workgroups(f, M, cols) * f.threads >= 1L << 32) return NEVER;  // (a grid has fewer than 2^32 threads)
  const long tiles = ((M + f.bm - 1) / f.bm) * ((cols + f.bn - 1) / f.bn), blocks = (K + f.bk - 1) / f.bk;
  const long rounds = (tiles + n_cu * f.per_cu - 1) / (n_cu * f.per_cu);
  return f.fixed + rounds * f.round + blocks * (tiles <= n_cu ? f.one : rounds * f.all);
}
// The form of a product, F_NONE where none fits a grid. wide: rows on 16-byte boundaries (the forms with direct loads).
int choose(int M, int N, int K, bool wide, long n_cu) {
  int best = F_NONE;
  double least = NEVER;
  for (int f = F_SPLIT16; f < F_COUNT; ++f) {
    const bool split = f <= F_SPLIT32;
    if (f == F_FOLD && !folded(N)) continue;
    if (!split && wide != (f < F_ANY64)) continue;
    const double us = (split && !wide ? 2.1 : 1.0) * form_us(FORMS[f], M, f == F_FOLD ? N - folded(N) : N, K, n_cu);
    if (us < least) least = us, best = f;
  }
  return best;
}

}  // namespace
}  // namespace zgdn

extern "C" int zlin_gemm_act(const void* x, long x_ld, const void* w, long w_ld, const void* bias, int bias_dtype,
                             int act, const void* residual, long r_ld, void* y, long y_ld, int M, int N, int K, int dtype,
                             void* stream) {
  using namespace zgdn;
  const char* fn = "zlin_gemm_act";
  if (dtype != ZGDN_BF16) return fail(ZGDN_EUNSUPPORTED, "%s: bf16 only (dtype %d)", fn, dtype);
  if (bias != nullptr && bias_dtype != ZGDN_F32 && bias_dtype != ZGDN_BF16)
    return fail(ZGDN_EINVAL, "%s: unknown bias dtype code %d", fn, bias_dtype);
  if (act < ZLIN_NONE || act > ZLIN_GELU_TANH) return fail(ZGDN_EINVAL, "%s: unknown activation %d", fn, act);
  if (M < 0 || N < 1 || K < 1) return fail(ZGDN_EINVAL, "%s: bad sizes M=%d N=%d K=%d", fn, M, N, K);
  if (M == 0) return ZGDN_OK;
  if (!x || !w || !y) return fail(ZGDN_EINVAL, "%s: null pointer", fn);
  if (x_ld < K || w_ld < K || y_ld < N || (residual != nullptr && r_ld < N))
    return fail(ZGDN_EINVAL, "%s: row strides x=%ld w=%ld (at least K=%d), y=%ld residual=%ld (at least N=%d)", fn, x_ld, w_ld,
                K, y_ld, residual != nullptr ? r_ld : (long)N, N);
  if (((uintptr_t)x | (uintptr_t)w | (uintptr_t)y | (uintptr_t)residual) % 2 ||
      (uintptr_t)bias % (bias_dtype == ZGDN_F32 ? 4 : 2))
    return fail(ZGDN_EINVAL, "%s: pointers off their element's boundary", fn);
  if (M > INT32_MAX - 256 || N > INT32_MAX - 256 || K > INT32_MAX - 2048)
    return fail(ZGDN_EUNSUPPORTED, "%s: M=%d N=%d K=%d", fn, M, N, K);
  const Region ry = {y, (size_t)M, (size_t)N * 2, (size_t)y_ld * 2};
  const size_t bias_bytes = (size_t)N * (bias_dtype == ZGDN_F32 ? 4 : 2);
  if (regions_meet(ry, {x, (size_t)M, (size_t)K * 2, (size_t)x_ld * 2}) || regions_meet(ry, {w, (size_t)N, (size_t)K * 2, (size_t)w_ld * 2}) ||
      regions_meet(ry, {bias, 1, bias_bytes, bias_bytes}) ||
      (!(residual == y && r_ld == y_ld) && regions_meet(ry, {residual, (size_t)M, (size_t)N * 2, (size_t)r_ld * 2})))
    return fail(ZGDN_EINVAL, "%s: y overlaps another operand (it may only be the residual itself)", fn);
  ActArgs a{(const uint16_t*)x, (const uint16_t*)w, x_ld, w_ld, bias, bias_dtype == ZGDN_BF16, act,
            (const uint16_t*)residual, residual != nullptr ? r_ld : 0, (uint16_t*)y, y_ld, M, N, K, 1, 0, 0};
  auto takes = [&](int n) {  // accesses of n elements of y and the residual
    return y_ld % n == 0 && (uintptr_t)y % (2 * n) == 0 && (residual == nullptr || (r_ld % n == 0 && (uintptr_t)residual % (2 * n) == 0));
  };
  a.vec = takes(8) ? 8 : takes(4) ? 4 : 1;
  // wide loads: rows on 16-byte boundaries, and a tile's rows within 32-bit byte offsets of one another
  const bool wide = x_ld % 8 == 0 && w_ld % 8 == 0 && K % 8 == 0 && ((uintptr_t)x | (uintptr_t)w) % 16 == 0 &&
                    x_ld < (1 << 21) && w_ld < (1 << 21) && K < (1 << 21);
  if (y_ld >= (1 << 21) || r_ld >= (1 << 21)) a.vec = std::min(a.vec, 4);  // (likewise for the whole tiles' stores)
  hipStream_t s = (hipStream_t)stream;
  int st = ZGDN_OK;
  switch (choose(M, N, K, wide, device_cus())) {
    case F_SPLIT16: st = wide ? launch_split<1, true>(fn, a, s) : launch_split<1, false>(fn, a, s); break;
    case F_SPLIT32: st = wide ? launch_split<2, true>(fn, a, s) : launch_split<2, false>(fn, a, s); break;
    case F_TILE64: st = launch_tiles<64, 128, 2, 3>(fn, a, s); break;
    case F_FOLD: st = launch_tiles<128, 128, 2, 2, true>(fn, a, s); break;
    case F_WIDE: st = launch_tiles<128, 256, 2, 3>(fn, a, s); break;
    case F_TILE256: st = launch_tiles<256, 256, 2, 2>(fn, a, s); break;
    case F_ANY64: st = launch_any<64>(a, s); break;
    case F_ANY128: st = launch_any<128>(a, s); break;
    default: return fail(ZGDN_EUNSUPPORTED, "%s: M=%d N=%d K=%d: more tiles than a grid holds", fn, M, N, K);
  }
  return st != ZGDN_OK ? st : check_launch(fn);
}

// Host layer and tests (not part of the public header): the form that a product of these sizes takes and, where `groups` is
// not NULL, the workgroups of its launch. 0: none, the product is refused.
extern "C" int zgdn_gemm_act_form(int M, int N, int K, int wide, int64_t* groups) {
  using namespace zgdn;
  if (M < 1 || N < 1 || K < 1 || M > INT32_MAX - 256 || N > INT32_MAX - 256 || K > INT32_MAX - 2048) return F_NONE;
  const int f = choose(M, N, K, wide != 0, device_cus());
  if (groups != nullptr) *groups = f == F_NONE ? 0 : workgroups(FORMS[f], M, f == F_FOLD ? N - folded(N) : N);
  return f;
}
