// y = act(x w^T + bias) + residual on bf16 MFMA, fp32 sums, the epilogue in fp32, rounded once.
//
// Tiles are computed transposed (A = rows of w, B = rows of x: v_mfma_f32_16x16x32_bf16, D: w row 4 g + e, x row lane % 16),
// two tiles of w rows interleaved, so that a lane ends with 8 neighbouring columns of one row of y: bias, residual and y
// are 16-byte accesses. Three forms, chosen by launch (below):
//   gemm_act_tile   BM x BN tiles, both operands by direct-to-LDS loads in blocks of 64 of K, several blocks ahead;
//   gemm_act_rows   few rows (a decode step): 16 x 16 tiles, K split over the workgroup's waves;
//   gemm_act_any    rows off 16-byte boundaries, K not a multiple of 8: guarded loads through registers.
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
  if constexpr (ACT == ZLIN_SILU) return x / (1.f + __expf(-x));
  if constexpr (ACT == ZLIN_GELU) return 0.5f * x * (1.f + erff(x * 0.70710678118654752f));
  if constexpr (ACT == ZLIN_GELU_TANH)  // 0.5 (1 + tanh u) = 1 / (1 + exp(-2 u))
    return x / (1.f + __expf(-2.f * 0.79788456080286536f * (x + 0.044715f * x * x * x)));
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

// 16 bytes a lane from a buffer straight into LDS (lane i at lds + 16 i), `k` bytes on from the lane's offset. In assembly:
// the kernels' own waits count these loads. M0, which they use for nothing else, needs a wait state before the load.
__device__ __forceinline__ void load_lds(au32x4 rsrc, uint32_t off, uint32_t k, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(off), "s"(rsrc), "s"(k) : "memory");
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
// stages of LDS (128-byte rows, 16-byte chunk c of row r at c ^ f(r)): block kb computes while the NS - 1 after it land.
// Fragment reads touch 16 rows, one chunk each: f spreads rows 0 .. 15 (x) and rows 8 a + b, b < 4 (w, whose fragments
// interleave) over all 16 places of 256 bytes.

constexpr int BK = 64;

__device__ __forceinline__ int fx(int r) { return (r >> 1) & 7; }
__device__ __forceinline__ int fw(int r) { return (r >> 1 & 1) | (r >> 3 & 3) << 1; }

template <int BM, int BN, int WM, int NS_>
struct TileCfg {
  static constexpr int WN = 8 / WM;
  static constexpr int TM = BM / WM / 16, TN = BN / WN / 32;  // 16-row tiles of x, 32-row pairs of w, a wave
  static constexpr int STAGE = (BM + BN) * 128;
  static constexpr int NS = NS_;
  static constexpr int LDS = NS * STAGE;
  static constexpr int PX = BM / 8 / 8, PW = BN / 8 / 8;  // 1 KiB pieces (8 rows) of each operand a wave
  static constexpr int PER_CU = LDS <= 80 * 1024 ? 2 : 1;
};

template <int BM, int BN, int WM, int NS>
__global__ __launch_bounds__(512, (2 * TileCfg<BM, BN, WM, NS>::PER_CU)) void gemm_act_tile_kernel(ActArgs a) {
  using C = TileCfg<BM, BN, WM, NS>;
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
  const int nk = (a.K + BK - 1) / BK, tail = a.K - (nk - 1) * BK;  // elements of the last block
  const uint32_t base = lds_at(lds);
  auto issue = [&](int kb, int stage) {
    const uint32_t at = base + stage * C::STAGE + 1024 * wave, k = (uint32_t)min(kb, nk - 1) * BK * 2;
    const bool cut = kb >= nk - 1;  // (behind the last block: it again, unread)
#pragma unroll
    for (int i = 0; i < C::PX; ++i) load_lds(rx, cut && 8 * cx[i] >= tail ? NOWHERE : ox[i], k, at + 8192 * i);
#pragma unroll
    for (int i = 0; i < C::PW; ++i) load_lds(rw, cut && 8 * cw[i] >= tail ? NOWHERE : ow[i], k, at + BM * 128 + 8192 * i);
  };

  af32x4 acc[TN][2][TM];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < TM; ++j) acc[i][u][j] = af32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < NS - 1; ++s) issue(s, s);
  // w rows of fragment u of a pair: 8 (m / 4) + 4 u + m % 4
  const int rwl = wn + 8 * (m >> 2) + (m & 3), rxl = wm + m;
  int st = 0;
  for (int kb = 0; kb < nk; ++kb) {
    wait_and_meet<(NS - 2) * (C::PX + C::PW)>();
    issue(kb + NS - 1, st == 0 ? NS - 1 : st - 1);
    const uint8_t* xs = lds + st * C::STAGE;
    const uint8_t* ws = xs + BM * 128;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      abf16x8 fb[TM], fa[TN][2];
#pragma unroll
      for (int j = 0; j < TM; ++j)
        fb[j] = *reinterpret_cast<const abf16x8*>(xs + (rxl + 16 * j) * 128 + (((4 * s + g) ^ fx(rxl)) << 4));
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u)
          fa[i][u] = *reinterpret_cast<const abf16x8*>(ws + (rwl + 32 * i + 4 * u) * 128 + (((4 * s + g) ^ fw(rwl)) << 4));
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int j = 0; j < TM; ++j) acc[i][u][j] = amfma(fa[i][u], fb[j], acc[i][u][j]);
    }
    st = st == NS - 1 ? 0 : st + 1;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  with_act(a.act, [&](auto act) {
    constexpr int ACT = decltype(act)::value;
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
  });
}

// ----------------------------------------------------------------------------------------------------- few rows
//
// 16 rows x 16 columns a workgroup, K in slices of 128 (256 bytes of a row), slice q to wave q % 8: such a call is the
// weights' way from memory, so each wave keeps two slices of both operands on their way (direct-to-LDS, 4 rows x 256
// contiguous bytes a load; chunk c of row r at c ^ r) and waits for nobody before its products. The 8 partial tiles are
// added in LDS in wave order. The row tiles of one column tile run on one XCD and share its copy of the weights.

constexpr int RW = 8, RSL = 128;                // waves, elements of a slice
constexpr int RTILE = 16 * RSL * 2;             // bytes of one operand's slice: 4 KiB
constexpr int ROWS_LDS = RW * 2 * 2 * RTILE;    // two slices of both, a wave: 128 KiB

__global__ __launch_bounds__(64 * RW) void gemm_act_rows_kernel(ActArgs a) {
  extern __shared__ uint4 act_lds[];
  uint8_t* lds = reinterpret_cast<uint8_t*>(act_lds);
  const int grp = blockIdx.x / (8 * a.tiles_m), in = blockIdx.x - grp * 8 * a.tiles_m;
  const int tn = grp * 8 + (in & 7), tm = in >> 3;
  if (tn >= a.tiles_n) return;
  const int wave = wave_id(), l = threadIdx.x & 63, m = l & 15, g = l >> 4;
  const int m0 = __builtin_amdgcn_readfirstlane(16 * tm), n0 = __builtin_amdgcn_readfirstlane(16 * tn);
  const au32x4 rx = rows_rsrc(a.x + (size_t)m0 * a.x_ld, a.x_ld, min(16, a.M - m0), a.K);
  const au32x4 rw = rows_rsrc(a.w + (size_t)n0 * a.w_ld, a.w_ld, min(16, a.N - n0), a.K);
  uint8_t* mine = lds + wave * 4 * RTILE;
  const uint32_t base = lds_at(mine);
  auto issue = [&](int q, int half) {  // slice q of the wave's
    const int k0 = (q * RW + wave) * RSL;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const int r = 4 * p + g, c = m ^ r;  // the lane's row of the piece and the chunk its place holds
      const bool there = k0 + 8 * c < a.K;
      load_lds(rw, there ? (uint32_t)r * (uint32_t)a.w_ld * 2u + 16u * c : NOWHERE, (uint32_t)k0 * 2u, base + half * 2 * RTILE + 1024 * p);
      load_lds(rx, there ? (uint32_t)r * (uint32_t)a.x_ld * 2u + 16u * c : NOWHERE, (uint32_t)k0 * 2u, base + half * 2 * RTILE + RTILE + 1024 * p);
    }
  };
  const int slices = (a.K + RSL * RW - 1) / (RSL * RW);  // (a wave's last may lie behind K: zeros)
  af32x4 acc = {0.f, 0.f, 0.f, 0.f};
  issue(0, 0);
  for (int q = 0; q < slices; ++q) {
    if (q + 1 < slices) {
      issue(q + 1, (q + 1) & 1);
      asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    const uint8_t* ws = mine + (q & 1) * 2 * RTILE;
#pragma unroll
    for (int s = 0; s < RSL / 32; ++s) {
      const int at = m * 256 + (((4 * s + g) ^ m) << 4);
      acc = amfma(*reinterpret_cast<const abf16x8*>(ws + at), *reinterpret_cast<const abf16x8*>(ws + RTILE + at), acc);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the load after the next overwrites the slice)
  }
  __syncthreads();
  float* part = reinterpret_cast<float*>(lds);  // [wave][lane][4]
  *reinterpret_cast<af32x4*>(part + wave * 256 + 4 * l) = acc;
  __syncthreads();
  if (wave == 0) {
    float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < RW; ++w) {
      const af32x4 p = *reinterpret_cast<const af32x4*>(part + w * 256 + 4 * l);
#pragma unroll
      for (int e = 0; e < 4; ++e) c[e] += p[e];
    }
    const int n = n0 + 4 * g;
    if (a.bias != nullptr) {
#pragma unroll
      for (int e = 0; e < 4; ++e) c[e] += bias_at(a, min(n + e, a.N - 1));
    }
    with_act(a.act, [&](auto act) { finish<decltype(act)::value>(a, m0 + m, n, c); });
  }
}

// Any sizes and alignments: 64 x 64 tiles, 4 waves of 32 x 32, blocks of 64 of K through LDS (128-byte rows, 16-byte
// chunks swizzled by row), each thread fetching 8 elements of a row at a time, one by one.
__global__ __launch_bounds__(256) void gemm_act_any_kernel(ActArgs a) {
  __shared__ uint4 sx[64 * 8], sw[64 * 8];
  const int n0 = (blockIdx.x % a.tiles_n) * 64, m0 = (blockIdx.x / a.tiles_n) * 64;
  const int wave = wave_id(), l = threadIdx.x & 63, m = l & 15, g = l >> 4;
  const int wm = (wave & 1) * 32, wn = (wave >> 1) * 32;
  af32x4 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = af32x4{0.f, 0.f, 0.f, 0.f};
  auto fetch = [&](const uint16_t* base, long ld, int row, int rows, int k) {
    uint32_t u[8];
    const uint16_t* p = base + (size_t)min(row, rows - 1) * ld;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t v = p[min(k + i, a.K - 1)];
      u[i] = row < rows && k + i < a.K ? v : 0u;
    }
    return make_uint4(u[0] | u[1] << 16, u[2] | u[3] << 16, u[4] | u[5] << 16, u[6] | u[7] << 16);
  };
  for (int k0 = 0; k0 < a.K; k0 += 64) {
    uint4 fx_[2], fw_[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int e = threadIdx.x + 256 * i, r = e >> 3, c = e & 7;
      fx_[i] = fetch(a.x, a.x_ld, m0 + r, a.M, k0 + 8 * c);
      fw_[i] = fetch(a.w, a.w_ld, n0 + r, a.N, k0 + 8 * c);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int e = threadIdx.x + 256 * i, r = e >> 3, c = e & 7;
      sx[r * 8 + (c ^ (r >> 1 & 7))] = fx_[i];
      sw[r * 8 + (c ^ (r >> 1 & 7))] = fw_[i];
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      abf16x8 fa[2], fb[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int ra = wn + 16 * i + m, rb = wm + 16 * i + m;
        fa[i] = __builtin_bit_cast(abf16x8, sw[ra * 8 + ((4 * s + g) ^ (ra >> 1 & 7))]);
        fb[i] = __builtin_bit_cast(abf16x8, sx[rb * 8 + ((4 * s + g) ^ (rb >> 1 & 7))]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = amfma(fa[i], fb[j], acc[i][j]);
    }
  }
  with_act(a.act, [&](auto act) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int n = n0 + wn + 16 * i + 4 * g;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float c[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e] = acc[i][j][e] + (a.bias != nullptr ? bias_at(a, min(n + e, a.N - 1)) : 0.f);
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

template <int BM, int BN, int WM, int NS>
int launch_tiles(const char* fn, ActArgs a, hipStream_t s) {
  using C = TileCfg<BM, BN, WM, NS>;
  static std::atomic<signed char> state[64];
  if (!lds_ready(gemm_act_tile_kernel<BM, BN, WM, NS>, C::LDS, state)) return fail(ZGDN_EHIP, "%s: the device refused the LDS", fn);
  a.tiles_m = (a.M + BM - 1) / BM, a.tiles_n = (a.N + BN - 1) / BN;
  const long per = ((long)a.tiles_m * a.tiles_n + 7) / 8;
  hipLaunchKernelGGL((gemm_act_tile_kernel<BM, BN, WM, NS>), dim3((unsigned)(8 * per)), dim3(512), C::LDS, s, a);
  return ZGDN_OK;
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
  if (M > INT32_MAX - 256 || N > INT32_MAX - 256 || K > INT32_MAX - 2048 ||
      (long)((M + 63) / 64) * ((N + 63) / 64) > INT32_MAX / 64)
    return fail(ZGDN_EUNSUPPORTED, "%s: M=%d N=%d K=%d", fn, M, N, K);
  ActArgs a{(const uint16_t*)x, (const uint16_t*)w, x_ld, w_ld, bias, bias_dtype == ZGDN_BF16, act,
            (const uint16_t*)residual, residual != nullptr ? r_ld : 0, (uint16_t*)y, y_ld, M, N, K, 1, 0, 0};
  auto takes = [&](int n) {  // accesses of n elements of y and the residual
    return y_ld % n == 0 && (uintptr_t)y % (2 * n) == 0 && (residual == nullptr || (r_ld % n == 0 && (uintptr_t)residual % (2 * n) == 0));
  };
  a.vec = takes(8) ? 8 : takes(4) ? 4 : 1;
  // wide loads: rows on 16-byte boundaries, and a tile's rows within 32-bit byte offsets of one another
  const bool wide = x_ld % 8 == 0 && w_ld % 8 == 0 && K % 8 == 0 && ((uintptr_t)x | (uintptr_t)w) % 16 == 0 &&
                    x_ld < (1 << 21) && w_ld < (1 << 21) && K < (1 << 21);
  hipStream_t s = (hipStream_t)stream;
  int st = ZGDN_OK;
  if (!wide) {
    a.tiles_m = (M + 63) / 64, a.tiles_n = (N + 63) / 64;
    hipLaunchKernelGGL(gemm_act_any_kernel, dim3((unsigned)a.tiles_m * a.tiles_n), dim3(256), 0, s, a);
  } else if (M <= 64) {
    static std::atomic<signed char> state[64];
    if (!lds_ready(gemm_act_rows_kernel, ROWS_LDS, state)) return fail(ZGDN_EHIP, "%s: the device refused the LDS", fn);
    a.tiles_m = (M + 15) / 16, a.tiles_n = (N + 15) / 16;
    hipLaunchKernelGGL(gemm_act_rows_kernel, dim3((unsigned)((a.tiles_n + 7) / 8 * 8) * a.tiles_m), dim3(64 * RW), ROWS_LDS, s, a);
  } else {
    // the tile whose rounds over the CUs take the least work, larger tiles doing more of it a time
    const long n_cu = device_cus();
    auto cost = [&](long bm, long bn, int per_cu, double eff) {
      const long tiles = ((M + bm - 1) / bm) * ((N + bn - 1) / bn), slots = n_cu * per_cu;
      return (double)((tiles + slots - 1) / slots) * per_cu * bm * bn / eff;
    };
    const double c0 = cost(256, 256, 1, 1.0), c1 = cost(128, 256, 1, 0.8), c2 = cost(128, 128, 2, 0.65), c3 = cost(64, 128, 2, 0.5);
    const double best = std::min(std::min(c0, c1), std::min(c2, c3));
    st = best == c0 ? launch_tiles<256, 256, 2, 2>(fn, a, s)
         : best == c1 ? launch_tiles<128, 256, 2, 3>(fn, a, s)
         : best == c2 ? launch_tiles<128, 128, 2, 2>(fn, a, s)
                      : launch_tiles<64, 128, 2, 3>(fn, a, s);
  }
  return st != ZGDN_OK ? st : check_launch(fn);
}
