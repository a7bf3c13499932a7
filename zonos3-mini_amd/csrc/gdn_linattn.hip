// Linear attention with a decay per head over whole sequences, on MFMA.
//
//   S_t = exp(g_t) S_{t-1} + v_t k_t^T,   o_t = S_t (scale q_t)
//
// With S the state before a chunk of 64 tokens and G the running sum of g in it,
//   o_t = exp(G_t) S (scale q_t) + sum_{s <= t} exp(G_t - G_s) (scale q_t . k_s) v_s,
//   S' = exp(G_end) S + sum_s exp(G_end - G_s) v_s k_s^T.
// A workgroup walks the chunks of one sequence and head, S in registers. Where there are too few of these for the device a
// sequence is cut into segments, and then
//   1. a walk over all segments but the last sums what each adds to the state,
//   2. the join turns these into the states before the segments,
//   3. the walk over the segments from there has the outputs (and, last, the final state).
// Products are bf16 x bf16 with fp32 sums. States stay fp32: where a product takes a state or a weighted value it is
// split into bf16 terms whose sum has 16 (outputs: two terms) or 24 bits (states: three), so that an output keeps only
// its own rounding and a state that of fp32 sums. fp32 inputs take the same steps on the fp32 MFMA.
//
// Measured (the three kernels, us): 32 packed prompts of 64 .. 2048 tokens, 16 heads of 128 x 128: 5 + 5 + 173; one of 4096:
// 15 + 7 + 25; one of 32768, 16 heads of 128 x 64 on one key head: 40 + 9 + 88. What bounds it: a chunk's instructions, not
// its bytes (packed: 569 MB, 104 us at the rate of a copy).
//
// The exponents are sums within a chunk, prefix sums from its start and suffix sums to its end, of one sign where all g <= 0;
// P's are differences of the prefix sums. These are held so that many strong decays do not cost the slow ones behind
// them their digits: in doubles for fp32, for bf16 as sums of whole numbers (exact) and of what is left of each decay (at
// most 32 in all: a difference is off by 2^-18 at most; as plain fp32 sums 48 resets left 2^-11, outputs up to 10 times their
// bound off). g is taken as at least -200 (exp(-200) is zero in fp32), so that -inf resets a state.
#include <algorithm>
#include <atomic>

#include "gdn_common.h"
#include "zonos3_linear.h"

namespace zgdn {
namespace {

typedef __bf16 lbf16x8 __attribute__((ext_vector_type(8)));
typedef float lf32x4 __attribute__((ext_vector_type(4)));
typedef short lshort4 __attribute__((ext_vector_type(4)));

constexpr int CH = 64;  // tokens of a chunk
constexpr float G_MIN = -200.f;
constexpr long CUS = 256;

struct LinArgs {
  const void *q, *k, *v, *g;
  long q_ld, k_ld, v_ld, g_ld;  // (g_ld 0: g [Hv])
  int g_bf16;
  const float* s_in;
  float* s_out;
  void* o;
  const int32_t* cu;
  int N, T, Hk, Hv;
  float scale;
  int run, run_slots;  // tokens of a segment, at most; segments
  float *ends, *gtot;  // [run_slots][Hv][V * K], [run_slots][Hv]: what a segment adds (then the state before it), log decay
};

__device__ __forceinline__ lf32x4 mfma16(lbf16x8 a, lbf16x8 b, lf32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ lf32x4 mfma4(float a, float b, lf32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// Log decay of row t (of the call's rows), head h: as it is stored, then as a float.
__device__ __forceinline__ uint32_t g_bits(const LinArgs& a, size_t t, int h) {
  const size_t i = t * (size_t)a.g_ld + h;
  return a.g_bf16 ? reinterpret_cast<const uint16_t*>(a.g)[i] : reinterpret_cast<const uint32_t*>(a.g)[i];
}
__device__ __forceinline__ float g_value(const LinArgs& a, uint32_t bits) {
  const float x = __uint_as_float(a.g_bf16 ? bits << 16 : bits);
  return x < G_MIN ? G_MIN : x;  // (a NaN stays)
}

// x exp(G) as x + x expm1(G) for slow decays: the factor's own rounding, the same at every stage, would otherwise grow
// with the length of the memory.
struct Decay {
  float add, mul;
};
__device__ __forceinline__ Decay decay_of(float G) {
  Decay d;
  const bool slow = G > -0.5f;
  d.add = slow ? expm1f(G) : expf(G);
  d.mul = slow ? 1.f : 0.f;
  return d;
}
__device__ __forceinline__ float decayed(float x, const Decay& d) { return fmaf(x, d.add, x * d.mul); }

__device__ __forceinline__ int pieces(int len, int size) { return max(1, (len + size - 1) / size); }

__device__ __forceinline__ int prefix_count(int x) {  // over the lanes up to this one
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);
  return x;
}

// The segment that a workgroup of the walk takes, in scalar registers. A sequence of several is cut into equal ones (but for
// their last chunk). The state pass takes every sequence's but the last, in order. The walk over the outputs takes a packed
// batch's by length: the longest, one a CU, then the shortest beside them, then the ones between, so that CUs finish
// together. (Above 64 sequences: in order, there are many to a CU.)
struct Segment {
  int seq, bos, slot, first, n;  // slot: of all segments in order; first, n: its tokens in the sequence
  bool cut, last;                // one of several; the sequence's last
};
template <bool OUT>
__device__ __forceinline__ bool find_segment(const LinArgs& a, int i, int side, Segment& p) {
  int j, len, n;  // segment of the sequence, the sequence's tokens and segments
  if (a.cu == nullptr) {
    n = pieces(a.T, a.run);
    const int per = OUT ? n : n - 1;
    p.seq = i / per;
    j = i - p.seq * per;
    p.bos = p.seq * a.T;
    p.slot = p.seq * n + j;
    len = a.T;
    if (p.seq >= a.N) return false;
  } else {
    const int l = threadIdx.x & 63;
    int base = 0, taken = 0;
    bool found = false;
    for (int s0 = 0; s0 < a.N && !found; s0 += 64) {
      int bos = 0, eos = 0, mine = 0;
      if (s0 + l < a.N) {
        seq_bounds(a.cu, s0 + l, a.T, bos, eos);
        mine = pieces(eos - bos, a.run);
      }
      const int slots = prefix_count(mine);
      const int counts = OUT ? slots : prefix_count(max(0, mine - 1));
      const int all = __builtin_amdgcn_readlane(counts, 63);
      int before = counts - (OUT ? mine : max(0, mine - 1)), at = i - taken;
      if (OUT && a.N <= 64) {
        const int size = mine > 0 ? (eos - bos + mine - 1) / mine : 0;
        before = 0;
        for (int s = 0; s < a.N; ++s) {
          const int other = __builtin_amdgcn_readlane(size, s);
          before += other > size || (other == size && s < l) ? __builtin_amdgcn_readlane(mine, s) : 0;
        }
        if (at >= side && at < all) at = at < 2 * side ? all - 1 - (at - side) : at - side;
        if (i >= all) return false;
      }
      const uint64_t here = __ballot(before <= at && at < before + (OUT ? mine : mine - 1));
      if (here) {
        const int f = __builtin_ctzll(here);
        p.seq = s0 + f;
        p.bos = __builtin_amdgcn_readlane(bos, f);
        len = __builtin_amdgcn_readlane(eos, f) - p.bos;
        n = __builtin_amdgcn_readlane(mine, f);
        j = at - __builtin_amdgcn_readlane(before, f);
        p.slot = base + __builtin_amdgcn_readlane(slots, f) - n + j;
        found = true;
      }
      base += __builtin_amdgcn_readlane(slots, 63);
      taken += all;
    }
    if (!found) return false;
  }
  const int size = (((len + CH - 1) / CH + n - 1) / n) * CH;
  p.first = j * size;
  p.n = min(size, len - p.first);
  p.cut = n > 1;
  p.last = j == n - 1;
  return true;
}

// ---------------------------------------------------------------------------------------------- LDS tiles of rows
//
// Rows of ROWB bytes (128 .. 512), 16-byte chunk c of row r at c ^ mask(r): row fragments (16 rows, one chunk each) and
// transposing reads (4 rows, 32 bytes each, for each group of 16 lanes) then spread over the banks.

template <int ROWB, typename T = uint16_t>
__device__ __forceinline__ int chunk_at(int r, int c) {
  constexpr int n = ROWB / 16;
  constexpr bool wide = sizeof(T) == 4;  // (fp32 rows, 256 bytes and more, are read by whole chunks of 16 rows)
  const int f = wide ? r & 15 : n >= 16 ? (r & 7) << 1 | (r >> 3 & 1) : n == 8 ? (r >> 1) & 7 : (r >> 1) & 3;
  return r * ROWB + ((c ^ f) << 4);
}

typedef uint32_t lu32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t lu32x4 __attribute__((ext_vector_type(4)));

// ROWS rows of ROWB bytes from global memory (row stride ld_bytes, `rows` of them there, zeros behind them) into LDS, by
// NW waves; each wave instruction fills 1 KiB, so a lane fetches the chunk that belongs at its place. The places in a row
// repeat every PERIOD instructions of a wave: these byte offsets are kept, the others follow by whole rows.
template <int ROWB, int NW, typename T = uint16_t>
struct RowsAt {
  static constexpr int RP = 1024 / ROWB, PERIOD = ROWB >= 256 ? (16 + RP * NW - 1) / (RP * NW) : 1;
  static_assert(RP * NW * PERIOD % 16 == 0, "the swizzle's period");
  uint32_t off[PERIOD];
  __device__ __forceinline__ RowsAt(uint32_t ld_bytes, int wave) {
    constexpr int n = ROWB / 16;
    const int l = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < PERIOD; ++i) {
      const int r = (i * NW + wave) * RP + l / n;
      off[i] = (uint32_t)(r - i * NW * RP) * ld_bytes + (uint32_t)(chunk_at<ROWB, T>(r, l % n) - r * ROWB);
    }
  }
  __device__ __forceinline__ void anew() {  // (nothing formed from them is kept across)
#pragma unroll
    for (int i = 0; i < PERIOD; ++i) asm volatile("" : "+v"(off[i]));
  }
};
// (instructions i0 .. i1 - 1 of the wave's ROWS ROWB / 1024 / NW)
template <int ROWB, int ROWS, int NW, typename T>
__device__ __forceinline__ void load_rows(const RowsAt<ROWB, NW, T>& at_row, const void* base, uint32_t ld_bytes, int rows,
                                          uint8_t* lds, int wave, int i0 = 0, int i1 = ROWS * ROWB / 1024 / NW) {
  constexpr int RP = 1024 / ROWB;  // rows an instruction
  static_assert(ROWS % (RP * NW) == 0, "as many a wave");
  // (formed by scalar instructions; a clamp of the rows to 0 .. 64 would be a vector one, with five wait states behind it)
  const uint32_t bytes = rows > 0 ? (uint32_t)(rows - 1) * ld_bytes + ROWB : 0u;
  const uint64_t at = (uint64_t)(uintptr_t)base;
  const lu32x4 rs = {(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)at),
                     (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(at >> 32) & 0xffffu)),
                     (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
#pragma unroll
  for (int i = i0; i < i1; ++i)
    load_lds(rs, at_row.off[i % RowsAt<ROWB, NW, T>::PERIOD] + (uint32_t)(i * NW * RP) * ld_bytes,
             (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)(lds + 1024 * (i * NW + wave))));  // (in LDS: the low half)
}
__device__ __forceinline__ uint2 lds_tr(const uint8_t* p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) lshort4*)p));
}

__device__ __forceinline__ float lo_f32(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f32(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// a, b as N bf16 pairs whose sum approximates them to 8 N bits: the value rounded, then what is left, rounded, ...
template <int N>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t* w) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    w[i] = pack_bf16x2(a, b);
    a -= lo_f32(w[i]);
    b -= hi_f32(w[i]);
  }
}

__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int N>
__device__ __forceinline__ void wait_loads() {  // at most N of the wave's loads outstanding, then a barrier
  static_assert(N < 64, "counter");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// Sum over the lanes up to this one (DPP: within rows of 16, then rows 0 and 2 on 1 and 3, then the lower half on the upper).
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_rows(float x) {  // (zero where there is no source lane)
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ float prefix_sum(float x) {
  x += dpp_rows<0x111, 0xF>(x);
  x += dpp_rows<0x112, 0xF>(x);
  x += dpp_rows<0x114, 0xF>(x);
  x += dpp_rows<0x118, 0xF>(x);
  x += dpp_rows<0x142, 0xA>(x);
  x += dpp_rows<0x143, 0xC>(x);
  return x;
}

// ------------------------------------------------------------------------------------------- bf16: a walk over chunks
//
// A workgroup walks the 64-token chunks of one segment of a sequence for NH value heads that share a key head (NH V = 64 or
// 128 value columns, 16 U a wave). A wave keeps its U halves of 16 value rows of S in registers, as transposed tiles
// [U][K / 16] (D: key 32 (kt / 2) + 8 g + 4 (kt % 2) + e; value of lane m and half u: 8 (m / 4) + 4 u + m % 4, of one half m):
// a pair of key tiles, split into bf16 terms, is an MFMA operand with its keys in memory order, and the halves' rows of an
// output tile are 4 U neighbours.
// A chunk:
//   P^T [s, t] = K Q^T, scaled by exp(G_t - G_s) and masked, a few tiles a wave, as two bf16 terms into LDS for all;
//   O^T [v, t] = exp(G_t) S Q^T + V^T P^T;
//   S^T = exp(G_end) S^T + K^T V', V' = exp(G_end - G_s) V in three bf16 terms.
// V^T and K^T are read transposed from LDS. A chunk of 128 x 128 is 200 MFMAs (16 cycles) and 780 other vector instructions
// a wave; beside an MFMA two of these cost nothing and each further one 4.3 cycles, so the splits into terms run beside the
// products of the step before, 4900 cycles in all if nothing waited. Measured: 9700 a chunk with one workgroup on the CU,
// 7500 with two (the rest: P's chain of reads, products, exponentials and writes, 1700; barriers and loads 1000; V^T P^T
// and stores 1500). The three terms of V' are 32 of the MFMAs and 100 of the others more than two would be; two where a
// segment's end state is not kept took a second body of the loop and registers it did not have (97 spilled: 27 -> 32 us at
// 4096 tokens; with U = 1, below, there was room and nothing gained). OUT false: the state alone.
// U = 2 where workgroups share CUs, U = 1 where none has to: the same work by 8 waves, two on each SIMD, one of which computes
// while the other waits (U 2 / 1: the kernel of two prompts of 64 tokens 10.5 / 10.0 us, whole calls of one prompt of 4096,
// 16 heads, 48.3 / 46.2, of 32768 on one key head 136 / 126; two
// workgroups of 8 waves would not fit a CU's registers).

template <int K, int V, int NH, int U, bool OUT>
struct WalkCfg {
  static constexpr int WH = V / (16 * U), NW = NH * WH;  // waves a head, in all
  static constexpr int KB = 2 * K, VB = 2 * NH * V;  // bytes of a row
  static constexpr int KI = CH * KB / 1024 / NW, VI = CH * VB / 1024 / NW;  // a wave's load instructions for k (q) and v
  static constexpr int P_TERM = OUT ? 6 * 1024 : 0;  // 16 x 32 blocks of P in fragment order: t tiles 0, 1 one, 2, 3 two
  static constexpr int GC = WH;  // chunks whose decays are formed at a time, each by a wave a head
  static constexpr int G_FLOATS = 3 * CH + 4, G_BYTES = (GC + 1) * NH * G_FLOATS * 4;
  static constexpr int VS = OUT ? 1 : 2;  // stages of v (and q)
  static constexpr int REST = VS * CH * VB + (OUT ? CH * KB : 0) + NH * 2 * P_TERM + G_BYTES;
  static constexpr int LDS_MAX = (NW == 8 ? 160 : 80) * 1024;  // 8 waves a CU, in one workgroup or two
  static constexpr int KS = REST + 2 * CH * KB <= LDS_MAX ? 2 : 1;  // stages of k
  static constexpr int AT_V = KS * CH * KB, AT_Q = AT_V + VS * CH * VB;
  static constexpr int AT_P = AT_Q + (OUT ? CH * KB : 0);
  static constexpr int AT_G = AT_P + NH * 2 * P_TERM;
  static constexpr int LDS = AT_G + G_BYTES;
  static_assert(LDS <= LDS_MAX && (OUT || KS == 2), "LDS");
  // P's tiles (s tile i, t tile j, i <= j) by wave of the head, 4 i + j each, a nibble a tile, those of a wave in one row or
  // column where they can be
  static constexpr int MOST = WH == 8 ? 2 : WH == 4 ? 3 : 6;
  static constexpr uint32_t tiles(int w) {
    return WH == 8 ? (w == 0 ? 0x0 : w == 1 ? 0x2 : w == 2 ? 0x3 : w == 3 ? 0x7 : w == 4 ? 0xB : w == 5 ? 0xF : w == 6 ? 0x51 : 0xA6)
         : WH == 4 ? (w == 0 ? 0x73 : w == 1 ? 0xFB : w == 2 ? 0xA62 : 0x051)
                   : (w == 0 ? 0xFB73 : 0x051A62);
  }
  static constexpr int count(int w) { return WH == 8 ? (w < 6 ? 1 : 2) : WH == 4 ? (w < 2 ? 2 : 3) : (w == 0 ? 4 : 6); }
};

template <int U>
__device__ __forceinline__ int walk_row(int u, int m) {
  return U == 2 ? 8 * (m >> 2) + 4 * u + (m & 3) : m;
}

// The scheduler moves nothing across: regions of a few products and the other work that is to run beside them.
__device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0); }
// One product, then N other vector instructions, M times over: the order of a region's.
template <int M, int N>
__device__ __forceinline__ void interleave() {
#pragma unroll
  for (int i = 0; i < M; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x002, N, 0);
  }
}

template <int K, int V, int NH, int U, bool OUT>
__global__ __launch_bounds__((64 * WalkCfg<K, V, NH, U, OUT>::NW), 2) void lin_walk_kernel(LinArgs a) {
  using C = WalkCfg<K, V, NH, U, OUT>;
  constexpr int NW = C::NW, WH = C::WH, KT = K / 16, KK = K / 32;
  extern __shared__ uint4 lin_lds[];
  uint8_t* lds = reinterpret_cast<uint8_t*>(lin_lds);
  const int groups = a.Hv / NH;
  const int index = blockIdx.x / groups, h0 = (blockIdx.x - index * groups) * NH;
  Segment p;
  // (a table whose sequences overlap may name more segments than there are slots)
  if (!find_segment<OUT>(a, index, max(1, (int)CUS / groups), p) || p.slot >= a.run_slots) return;
  const int n = p.n;  // (0 for an empty sequence)
  const int wave = wave_id(), l = threadIdx.x & 63, g = l >> 4, m = l & 15;
  const int hh = wave / WH, wl = wave - hh * WH, h = h0 + hh;
  const size_t row0 = (size_t)p.bos + p.first;
  const size_t hk = (size_t)(h0 / (a.Hv / a.Hk)) * K;
  const uint16_t* qp = reinterpret_cast<const uint16_t*>(a.q) + row0 * a.q_ld + hk;
  const uint16_t* kp = reinterpret_cast<const uint16_t*>(a.k) + row0 * a.k_ld + hk;
  const uint16_t* vp = reinterpret_cast<const uint16_t*>(a.v) + row0 * a.v_ld + (size_t)h0 * V;
  float* gb = reinterpret_cast<float*>(lds + C::AT_G) + hh * C::G_FLOATS;  // + NH G_FLOATS a chunk, GC + 1 in turn
  uint8_t* pl = lds + C::AT_P + hh * 2 * C::P_TERM + 16 * l;
  const uint8_t* qs = lds + C::AT_Q;

  const int chunks = (n + CH - 1) / CH;
  auto rows_of = [&](int c) { return min(CH, n - c * CH); };  // (behind the last chunk 0 and less: zeros)
  RowsAt<C::KB, NW> k_at((uint32_t)a.k_ld * 2u, wave), q_at((uint32_t)a.q_ld * 2u, wave);
  RowsAt<C::VB, NW> v_at((uint32_t)a.v_ld * 2u, wave);
  auto issue = [&](const uint16_t* x, long ld, const auto& lanes, auto row_bytes, int at, int c, int i0, int i1) {
    const int rows = rows_of(c);
    load_rows<decltype(row_bytes)::value, CH, NW>(lanes, x + (rows > 0 ? (size_t)c * CH : 0) * ld, (uint32_t)ld * 2u, rows,
                                                  lds + at, wave, i0, i1);
  };
  auto issue_k = [&](int c, int i0 = 0, int i1 = C::KI) {
    issue(kp, a.k_ld, k_at, std::integral_constant<int, C::KB>{}, C::KS == 2 ? (c & 1) * CH * C::KB : 0, c, i0, i1);
  };
  auto issue_v = [&](int c, int i0 = 0, int i1 = C::VI) {
    issue(vp, a.v_ld, v_at, std::integral_constant<int, C::VB>{}, C::AT_V + (C::VS == 2 ? (c & 1) * CH * C::VB : 0), c, i0, i1);
  };
  auto issue_q = [&](int c, int i0 = 0, int i1 = C::KI) {
    issue(qp, a.q_ld, q_at, std::integral_constant<int, C::KB>{}, C::AT_Q, c, i0, i1);
  };
  // Log decays, GC chunks at a time, one of them a wave: lane l takes the chunk's tokens l (prefix sums) and 63 - l (suffix
  // sums: lanes in token order from the end).
  auto g_at = [&](int c) { return gb + (c % (C::GC + 1)) * NH * C::G_FLOATS; };
  struct G2 {
    uint32_t up, down;
  };
  auto g_load = [&](int c) {
    const int t = c * CH + l, u = c * CH + 63 - l;
    return G2{t < n ? g_bits(a, row0 + t, h) : 0u, u < n ? g_bits(a, row0 + u, h) : 0u};
  };
  auto g_store = [&](int c, const G2& x) {
    float* b = g_at(c);
    if constexpr (OUT) {  // (whole numbers and what is left of them: sums of the first are exact, those of the second small)
      const float up = g_value(a, x.up), whole = rintf(up);
      b[l] = prefix_sum(whole);
      b[CH + l] = prefix_sum(up - whole);
    }
    const float s = prefix_sum(g_value(a, x.down)), total = __shfl(s, 63);
    b[2 * CH + 63 - l] = expf(dpp_rows<0x138, 0xF>(s));
    const Decay d = decay_of(total);
    if (l == 0) *reinterpret_cast<lf32x4*>(b + 3 * CH) = lf32x4{d.add, d.mul, total, 0.f};
  };

  const size_t hs = (size_t)V * K;
  lf32x4 acc[U][KT];
  // a state [V][K] of the head in memory: the lane's tiles are 4 floats each, pairs of them 8
  const size_t lane_at = (size_t)(16 * U * wl + walk_row<U>(0, m)) * K + 8 * g;
  auto state_at = [&](int u, int kt) { return lane_at + 4 * u * K + 32 * (kt >> 1) + 4 * (kt & 1); };
  auto put = [&](float* dst) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) *reinterpret_cast<lf32x4*>(dst + state_at(u, kt)) = acc[u][kt];
  };

  G2 gv = g_load(wl);
  issue_k(0);
  if constexpr (OUT) issue_q(0);
  issue_v(0);
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) acc[u][kt] = lf32x4{0.f, 0.f, 0.f, 0.f};
  // the state before the segment: carried into it, or the initial one (a sequence of one segment)
  const float* s_in = nullptr;
  if constexpr (OUT) {
    s_in = p.cut ? a.ends + ((size_t)p.slot * a.Hv + h) * hs
           : a.s_in != nullptr ? a.s_in + ((size_t)p.seq * a.Hv + h) * hs
                               : nullptr;
    if (s_in != nullptr) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) acc[u][kt] = *reinterpret_cast<const lf32x4*>(s_in + state_at(u, kt));
    }
    // P's tiles above its diagonal blocks of 32 stay zero
    for (int e = wl; e < 2 * C::P_TERM / 1024; e += WH) *reinterpret_cast<uint4*>(pl + 1024 * e) = make_uint4(0, 0, 0, 0);
  }
  g_store(wl, gv);
  float gsum = 0.f;

  // Offsets of the lane's 16-byte chunks in rows of KB bytes: chunk c of the rows of one place mod 16 lies at the offset of
  // chunk 0 with c's bits flipped. Formed anew each chunk (held, all of them would take 30 registers).
  int at_row = chunk_at<C::KB>(m, g);                    // row m, chunk g
  int at_tr = chunk_at<C::KB>(4 * g + (m >> 2), m & 3);  // transposing reads of rows 4 g ..: a half of each of 4 chunks
  auto flip = [](int at, int c) { return at ^ (c << 4); };
  const bool keep = p.last && a.s_out != nullptr;  // whether the state behind the last chunk is wanted

  // (NT: terms of V')
  auto chunk = [&](int c, auto terms) {
    constexpr int NT = decltype(terms)::value;
    asm volatile("" : "+v"(at_row), "+v"(at_tr));
    k_at.anew(), v_at.anew();
    if constexpr (OUT) q_at.anew();
    // chunk c is there, and nobody reads what the next loads overwrite (the first chunk's state may still be on its way)
    if (OUT && c == 0 && s_in != nullptr)
      wait_loads<U * KT>();
    else
      wait_loads<0>();
    const int in_group = c & (C::GC - 1);
    if (in_group == 0 && c + C::GC < chunks) gv = g_load(c + C::GC + wl);
    if constexpr (!OUT) {
      issue_k(c + 1);
      issue_v(c + 1);
    }
    const uint8_t* ks = lds + (C::KS == 2 ? (c & 1) * CH * C::KB : 0);
    const uint8_t* vs = lds + C::AT_V + (C::VS == 2 ? (c & 1) * CH * C::VB : 0);
    const float* b = g_at(c);
    lf32x4 o[U][4];
    lbf16x8 vf[U][2];  // the wave's columns of V^T: [half][block of 32 tokens]
    auto read_v = [&] {
      const int r = 4 * g + (m >> 2), col = (hh * V + 16 * U * wl) / 8 + (U == 2 ? m & 3 : (m & 3) >> 1);
      const uint8_t* at = vs + chunk_at<C::VB>(r, col) + (U == 2 ? 0 : 8 * (m & 1));
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const uint2 x = lds_tr(at + 32 * s * C::VB + 8 * u), y = lds_tr(at + (32 * s + 16) * C::VB + 8 * u);
          vf[u][s] = __builtin_bit_cast(lbf16x8, make_uint4(x.x, x.y, y.x, y.y));
        }
    };
    // V' in terms, a pair of tokens at a time: word i of half u in block s
    uint32_t vt[2][U][NT][4];  // [block][half][term][word]
    lf32x4 vw[2][2];          // the weights of a block's tokens (rows 4 g .., 16 + 4 g ..)
    auto read_weights = [&](int s) {
      vw[s][0] = *reinterpret_cast<const lf32x4*>(b + 2 * CH + 32 * s + 4 * g);
      vw[s][1] = *reinterpret_cast<const lf32x4*>(b + 2 * CH + 32 * s + 16 + 4 * g);
    };
    auto v_pair = [&](int s, int u, int i) {
      const uint4 all = __builtin_bit_cast(uint4, vf[u][s]);
      const uint32_t x = i == 0 ? all.x : i == 1 ? all.y : i == 2 ? all.z : all.w;
      uint32_t t[NT];
      split_pair<NT>(lo_f32(x) * vw[s][i >> 1][2 * (i & 1)], hi_f32(x) * vw[s][i >> 1][2 * (i & 1) + 1], t);
#pragma unroll
      for (int k = 0; k < NT; ++k) vt[s][u][k][i] = t[k];
    };
    constexpr int SR = 2 * U;                   // regions of a step of S Q^T: a term of a half each
    constexpr int XS = 3 - U, GX = 2 * KK / XS;  // the update's steps: pairs of key tiles at a time, steps in all
    static_assert(!OUT || (C::KI + C::VI <= GX * NT && SR * KK % C::KI == 0), "regions for the loads");
    auto v_frag = [&](int s, int u, int k) {
      return __builtin_bit_cast(lbf16x8, make_uint4(vt[s][u][k][0], vt[s][u][k][1], vt[s][u][k][2], vt[s][u][k][3]));
    };
    bool apart = false;
    if constexpr (OUT) {
      // P^T tiles: the wave's all at once
      auto p_tiles = [&](auto wc) {
        constexpr int CNT = C::count(decltype(wc)::value);
        constexpr uint32_t CODE = C::tiles(decltype(wc)::value);
        lf32x4 d[CNT];
        lbf16x8 kf[4], qf[4];
#pragma unroll
        for (int x = 0; x < CNT; ++x) d[x] = lf32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            bool ki = false, qi = false;
#pragma unroll
            for (int x = 0; x < CNT; ++x) {
              ki |= ((CODE >> (4 * x) & 15) >> 2) == i;
              qi |= (CODE >> (4 * x) & 3) == i;
            }
            if (ki) kf[i] = *reinterpret_cast<const lbf16x8*>(ks + 16 * i * C::KB + flip(at_row, 4 * kk));
            if (qi) qf[i] = *reinterpret_cast<const lbf16x8*>(qs + 16 * i * C::KB + flip(at_row, 4 * kk));
          }
#pragma unroll
          for (int x = 0; x < CNT; ++x) d[x] = mfma16(kf[(CODE >> (4 * x) & 15) >> 2], qf[CODE >> (4 * x) & 3], d[x]);
        }
#pragma unroll
        for (int x = 0; x < CNT; ++x) {
          const int i = (CODE >> (4 * x) & 15) >> 2, j = CODE >> (4 * x) & 3;
          const lf32x4 ws = *reinterpret_cast<const lf32x4*>(b + 16 * i + 4 * g), rs = *reinterpret_cast<const lf32x4*>(b + CH + 16 * i + 4 * g);
          const float wt = b[16 * j + m], rt = b[CH + 16 * j + m];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            d[x][e] *= a.scale * __expf((wt - ws[e]) + (rt - rs[e]));
            if (i == j) d[x][e] = 4 * g + e <= m ? d[x][e] : 0.f;
          }
          uint32_t w0[2], w1[2];
          split_pair<2>(d[x][0], d[x][1], w0);
          split_pair<2>(d[x][2], d[x][3], w1);
          // the block of tile j and tokens 32 (i / 2) .. in fragment order: this very lane's, half i % 2
          const int at = 1024 * (j < 2 ? j : 2 * j - 2 + (i >> 1)) + 8 * (i & 1);
          *reinterpret_cast<uint2*>(pl + at) = make_uint2(w0[0], w1[0]);
          *reinterpret_cast<uint2*>(pl + C::P_TERM + at) = make_uint2(w0[1], w1[1]);
        }
      };
      switch (wl) {
        case 0: p_tiles(std::integral_constant<int, 0>{}); break;
        case 1: p_tiles(std::integral_constant<int, 1>{}); break;
        case 2:
          if constexpr (WH > 2) p_tiles(std::integral_constant<int, 2>{});
          break;
        case 3:
          if constexpr (WH > 2) p_tiles(std::integral_constant<int, 3>{});
          break;
        case 4:
          if constexpr (WH > 4) p_tiles(std::integral_constant<int, 4>{});
          break;
        case 5:
          if constexpr (WH > 4) p_tiles(std::integral_constant<int, 5>{});
          break;
        case 6:
          if constexpr (WH > 4) p_tiles(std::integral_constant<int, 6>{});
          break;
        default:
          if constexpr (WH > 4) p_tiles(std::integral_constant<int, 7>{});
      }
      // O^T = S Q^T, the state in two terms; beside each step's products the next one's terms and V's of the first block
      uint32_t st[2][U][2][4];  // [step % 2][half][term][word]
      lbf16x8 qf[2][4];
      auto q_read = [&](int kk) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          qf[kk & 1][j] = *reinterpret_cast<const lbf16x8*>(qs + 16 * j * C::KB + flip(at_row, 4 * kk));
      };
      auto s_pair = [&](int kk, int u, int i) {
        uint32_t t[2];
        const lf32x4 x = acc[u][2 * kk + (i >> 1)];
        split_pair<2>(x[2 * (i & 1)], x[2 * (i & 1) + 1], t);
        st[kk & 1][u][0][i] = t[0];
        st[kk & 1][u][1][i] = t[1];
      };
      fence();
      q_read(0);
      read_v();
      read_weights(0);
      float f[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = a.scale * __expf(b[16 * j + m] + b[CH + 16 * j + m]);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[u][j] = lf32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) s_pair(0, u, i);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        fence();
        if (kk + 1 < KK) q_read(kk + 1);
#pragma unroll
        for (int r = 0; r < SR; ++r) {  // term 1 - r / U of half r % U
          fence();
          const int x = 1 - r / U, u = r % U;
          const lbf16x8 sf = __builtin_bit_cast(lbf16x8, make_uint4(st[kk & 1][u][x][0], st[kk & 1][u][x][1], st[kk & 1][u][x][2], st[kk & 1][u][x][3]));
#pragma unroll
          for (int j = 0; j < 4; ++j) o[u][j] = mfma16(sf, qf[kk & 1][j], o[u][j]);
          if (kk + 1 < KK) {
            s_pair(kk + 1, r >> 1, 2 * (r & 1));
            s_pair(kk + 1, r >> 1, 2 * (r & 1) + 1);
          }
          const int at = SR * kk + r;  // (the 4 U pairs of V' over the SR KK regions)
          if (at * 2 % KK == 0) v_pair(0, at * 2 / KK >> 2, at * 2 / KK & 3);
          if constexpr (C::KS == 2) {  // the next k's loads, one at a time
            constexpr int every = SR * KK / C::KI;
            if (at % every == 0) issue_k(c + 1, at / every, at / every + 1);
          }
          interleave<4, 5>();
        }
      }
      fence();
      // (formed here, although only the update needs them)
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < NT; ++k)
          asm volatile("" : "+v"(vt[0][u][k][0]), "+v"(vt[0][u][k][1]), "+v"(vt[0][u][k][2]), "+v"(vt[0][u][k][3]));
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int u = 0; u < U; ++u) o[u][j] *= f[j];
      typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
      u16x2 top = {0, 0};  // the largest magnitude's bits
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const uint4 w = __builtin_bit_cast(uint4, vf[u][s]);
          const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, x[e] & 0x7fff7fffu));
        }
      apart = __ballot(top.x >= 0x7f80 || top.y >= 0x7f80) != 0;
      lds_barrier();  // P is there, and nobody reads q and v any more
      auto p_frag = [&](int j, int s, int term) {
        return *reinterpret_cast<const lbf16x8*>(pl + term * C::P_TERM + 1024 * (j < 2 ? j : 2 * j - 2 + s));
      };
      if (!apart) {
        lbf16x8 pf[2][4][2];
        auto p_read = [&](int s) {
#pragma unroll
          for (int x = 1; x >= 0; --x)
#pragma unroll
            for (int j = 2 * s; j < 4; ++j) pf[s][j][x] = p_frag(j, s, x);
        };
        auto pv = [&](int s, int x) {
          fence();
#pragma unroll
          for (int j = 2 * s; j < 4; ++j)
#pragma unroll
            for (int u = 0; u < U; ++u) o[u][j] = mfma16(vf[u][s], pf[s][j][x], o[u][j]);
          fence();
        };
        p_read(0);
        if constexpr (U == 1) {
          fence();
          issue_q(c + 1, 0, C::KI);
          issue_v(c + 1, 0, C::VI);
        }
        pv(0, 1);  // (the small terms first)
        p_read(1);
        pv(0, 0);
        pv(1, 1);
        pv(1, 0);
      } else {
        if constexpr (U == 1) {
          issue_q(c + 1, 0, C::KI);
          issue_v(c + 1, 0, C::VI);
        }
        // an infinity or a NaN among the values: a masked P is zero, and zero times it NaN. Token by token, each added
        // from its own row on
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const uint4 all = __builtin_bit_cast(uint4, vf[u][s]);
#pragma unroll 1
            for (int i = 0; i < 32; ++i) {  // the lane's fragment holds token i at place i % 4 + 4 (i / 16)
              const int at = (i & 3) + 4 * (i >> 4);
              const uint32_t half = (i >> 2 & 3) == g ? (at & 1 ? 0xffff0000u : 0x0000ffffu) : 0u;
              const lbf16x8 one = __builtin_bit_cast(
                  lbf16x8, make_uint4(at >> 1 == 0 ? all.x & half : 0u, at >> 1 == 1 ? all.y & half : 0u,
                                      at >> 1 == 2 ? all.z & half : 0u, at >> 1 == 3 ? all.w & half : 0u));
#pragma unroll
              for (int j = 2 * s; j < 4; ++j) {
                lf32x4 x = {0.f, 0.f, 0.f, 0.f};
                x = mfma16(one, p_frag(j, s, 1), x);
                x = mfma16(one, p_frag(j, s, 0), x);
                if (32 * s + i <= 16 * j + m) o[u][j] += x;
              }
            }
          }
      }
      // the lane holds values 4 U g .. of the wave's, of token 16 j + m (rows behind the segment are dropped)
      const uint32_t lb = (uint32_t)a.Hv * V * 2u;
      const Rsrc rs = raw_rsrc(reinterpret_cast<uint16_t*>(a.o) + ((row0 + (size_t)c * CH) * a.Hv + h) * V,
                               (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(rows_of(c) - 1) * lb + 2 * V)));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t at = (uint32_t)(16 * j + m) * lb + 2 * (16 * U * wl + 4 * U * g);
        const uint32_t w0 = pack_bf16x2(o[0][j][0], o[0][j][1]), w1 = pack_bf16x2(o[0][j][2], o[0][j][3]);
        if constexpr (U == 2)
          __builtin_amdgcn_raw_buffer_store_b128(
              lu32x4{w0, w1, pack_bf16x2(o[1][j][0], o[1][j][1]), pack_bf16x2(o[1][j][2], o[1][j][3])}, rs, at, 0, 0);
        else
          __builtin_amdgcn_raw_buffer_store_b64(lu32x2{w0, w1}, rs, at, 0, 0);
      }
    } else {
      read_v();
      read_weights(0);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) v_pair(0, u, i);
    }
    if (OUT && c + 1 == chunks && !keep) return;
    // S^T = exp(G_end) S^T + K^T V', a pair of key tiles at a time: beside the first block's products the decay of the next
    // pair and V' of the second block
    const lf32x4 all = *reinterpret_cast<const lf32x4*>(b + 3 * CH);
    gsum += all[2];
    const Decay dc = {all[0], all[1]};
    read_weights(1);
    lbf16x8 kf[2][XS][2];  // [step % 2][pair][tile of the pair]
    auto k_read = [&](int x) {  // pair x of 2 KK: pair x % KK of block x / KK
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint8_t* at = ks + 32 * (x / KK) * C::KB + flip(at_tr, 4 * (x % KK)) + 8 * i;
        const uint2 y = lds_tr(at), z = lds_tr(at + 16 * C::KB);
        kf[x / XS & 1][x % XS][i] = __builtin_bit_cast(lbf16x8, make_uint4(y.x, y.y, z.x, z.y));
      }
    };
    auto decay = [&](int y, int part) {  // of the tiles of step y, by halves
      const int kk = XS * y + (U == 2 ? 0 : part), u = U == 2 ? part : 0;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[u][2 * kk + i][e] = decayed(acc[u][2 * kk + i][e], dc);
    };
    fence();
#pragma unroll
    for (int x = 0; x < XS; ++x) k_read(x);
    decay(0, 0);
    decay(0, 1);
#pragma unroll
    for (int y = 0; y < GX; ++y) {
      const int s = 2 * y / GX;
      fence();
      if (y + 1 < GX) {
#pragma unroll
        for (int x = 0; x < XS; ++x) k_read(XS * (y + 1) + x);
      }
#pragma unroll
      for (int t = NT - 1; t >= 0; --t) {  // (the small terms first)
        fence();
#pragma unroll
        for (int x = 0; x < XS; ++x)
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const lbf16x8 vfr = v_frag(s, u, t);
            const int kk = (XS * y + x) % KK;
#pragma unroll
            for (int i = 0; i < 2; ++i) acc[u][2 * kk + i] = mfma16(kf[y & 1][x][i], vfr, acc[u][2 * kk + i]);
          }
        if constexpr (OUT && U == 2) {  // the next q's and v's loads, one at a time
          const int i = y * NT + NT - 1 - t;
          if (i < C::KI)
            issue_q(c + 1, i, i + 1);
          else if (i < C::KI + C::VI)
            issue_v(c + 1, i - C::KI, i - C::KI + 1);
        }
        if (s == 0) {
          if (2 * (y + 1) < GX && t < 2) decay(y + 1, t);
          constexpr int PER = 8 * U / GX;  // pairs of V' a step
#pragma unroll
          for (int q = t; q < PER; q += NT) v_pair(1, (PER * y + q) >> 2, (PER * y + q) & 3);
          interleave<4, 5>();
        }
      }
    }
    fence();
    if (in_group == C::GC - 1 && c + 1 < chunks) g_store(c + 1 + wl, gv);
    if constexpr (C::KS == 1) {
      lds_barrier();  // nobody reads k any more
      issue_k(c + 1);
    }
  };
  for (int c = 0; c < chunks; ++c) chunk(c, std::integral_constant<int, 3>{});
  if constexpr (OUT) {
    if (keep) put(a.s_out + ((size_t)p.seq * a.Hv + h) * hs);
  } else {
    const size_t at = (size_t)p.slot * a.Hv + h;
    put(a.ends + at * hs);
    if (wl == 0 && l == 0) a.gtot[at] = gsum;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (loads into LDS that nobody reads end before the workgroup does)
}

// ------------------------------------------------------------------------------------------- fp32: a walk over chunks
//
// The same steps on the fp32 MFMA (16 x 16, 4 terms), for one head a workgroup of 4 waves; a wave keeps U = V / 64 tiles of
// 16 value rows (value of row m and tile u: U m + u of the wave's), all keys. The 4 terms of a product are taken so that a
// register is an operand as it stands: for S Q^T keys 16 g + 4 i + x of a block of 64 (S^T's tile x holds the block's keys
// = x mod 4, so a lane's rows 4 g + i are these), for V^T P^T and K^T V' tokens 16 i + 4 g + e, the rows that P's tiles
// hold; a chunk's values are read once for both. A chunk of 64 x 64 is 216 MFMAs of 32 cycles a wave, 6900 cycles, and takes
// 13000: 6 prompts of 40 .. 1500 tokens of 8 such heads 11 + 4 + 22 us.

template <int K, int V, bool OUT>
struct Walk32Cfg {
  static constexpr int NW = 4, U = V / 64, KB = 4 * K, VB = 4 * V;
  static constexpr int VS = OUT ? 1 : 2;  // stages of v (and q); k has two
  static constexpr int AT_V = 2 * CH * KB, AT_Q = AT_V + VS * CH * VB, AT_P = AT_Q + (OUT ? CH * KB : 0);
  static constexpr int AT_G = AT_P + (OUT ? 10 * 1024 : 0);
  // a chunk's decays: prefix sums (doubles), scale exp of them, exp of the suffix sums, of all (Decay) and their sum;
  // formed 4 chunks at a time, one a wave
  static constexpr int G_FLOATS = 4 * CH + 4, RING = NW + 1;
  static constexpr int LDS = AT_G + RING * G_FLOATS * 4;
  static_assert(LDS <= 160 * 1024, "LDS");
};

template <int K, int V, bool OUT>
__global__ __launch_bounds__(256, (K * V > 8192 ? 1 : 2)) void lin_walk_f32_kernel(LinArgs a) {
  using C = Walk32Cfg<K, V, OUT>;
  constexpr int NW = C::NW, U = C::U, KH = K / 64;
  extern __shared__ uint4 lin_lds[];
  uint8_t* lds = reinterpret_cast<uint8_t*>(lin_lds);
  const int index = blockIdx.x / a.Hv, h = blockIdx.x - index * a.Hv;
  Segment p;
  if (!find_segment<OUT>(a, index, max(1, (int)CUS / a.Hv), p) || p.slot >= a.run_slots) return;  // (as above)
  const int n = p.n, wave = wave_id(), l = threadIdx.x & 63, g = l >> 4, m = l & 15;
  const size_t row0 = (size_t)p.bos + p.first, hk = (size_t)(h / (a.Hv / a.Hk)) * K;
  const float* qp = reinterpret_cast<const float*>(a.q) + row0 * a.q_ld + hk;
  const float* kp = reinterpret_cast<const float*>(a.k) + row0 * a.k_ld + hk;
  const float* vp = reinterpret_cast<const float*>(a.v) + row0 * a.v_ld + (size_t)h * V;
  float* gb = reinterpret_cast<float*>(lds + C::AT_G);

  const int chunks = (n + CH - 1) / CH;
  RowsAt<C::KB, NW, float> k_at((uint32_t)a.k_ld * 4u, wave), q_at((uint32_t)a.q_ld * 4u, wave);
  RowsAt<C::VB, NW, float> v_at((uint32_t)a.v_ld * 4u, wave);
  auto issue = [&](const float* x, long ld, const auto& lanes, auto row_bytes, int at, int c) {
    const int rows = min(CH, n - c * CH);  // (behind the last chunk 0 and less: zeros)
    load_rows<decltype(row_bytes)::value, CH, NW>(lanes, x + (rows > 0 ? (size_t)c * CH : 0) * ld, (uint32_t)ld * 4u, rows, lds + at, wave);
  };
  auto issue_k = [&](int c) { issue(kp, a.k_ld, k_at, std::integral_constant<int, C::KB>{}, (c & 1) * CH * C::KB, c); };
  auto issue_v = [&](int c) {
    issue(vp, a.v_ld, v_at, std::integral_constant<int, C::VB>{}, C::AT_V + (OUT ? 0 : (c & 1) * CH * C::VB), c);
  };
  auto issue_q = [&](int c) { issue(qp, a.q_ld, q_at, std::integral_constant<int, C::KB>{}, C::AT_Q, c); };
  auto g_at = [&](int c) { return gb + (c % C::RING) * C::G_FLOATS; };
  auto g_load = [&](int c) {  // lane l: tokens l, and 63 - l for the sums from the end
    const int t = c * CH + l, u = c * CH + 63 - l;
    return make_uint2(t < n ? g_bits(a, row0 + t, h) : 0u, u < n ? g_bits(a, row0 + u, h) : 0u);
  };
  auto g_store = [&](int c, uint2 x) {
    float* b = g_at(c);
    if constexpr (OUT) {
      double s = g_value(a, x.x);  // (differences of these go into exponents)
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const double y = __shfl_up(s, d);
        s += l >= d ? y : 0.;
      }
      reinterpret_cast<double*>(b)[l] = s;
      b[2 * CH + l] = a.scale * expf((float)s);
    }
    const float s = prefix_sum(g_value(a, x.y)), total = __shfl(s, 63);
    b[3 * CH + 63 - l] = expf(dpp_rows<0x138, 0xF>(s));
    const Decay d = decay_of(total);
    if (l == 0) *reinterpret_cast<lf32x4*>(b + 4 * CH) = lf32x4{d.add, d.mul, total, 0.f};
  };

  const size_t hs = (size_t)V * K;
  lf32x4 acc[U][KH][4];  // [tile][block of 64 keys][x]: element i is key 16 g + 4 i + x
  const int v0 = 16 * U * wave;
  auto state_at = [&](int u, int kh, int i) { return (size_t)(v0 + U * m + u) * K + 64 * kh + 16 * g + 4 * i; };
  auto put = [&](float* dst) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int kh = 0; kh < KH; ++kh)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<lf32x4*>(dst + state_at(u, kh, i)) =
              lf32x4{acc[u][kh][0][i], acc[u][kh][1][i], acc[u][kh][2][i], acc[u][kh][3][i]};
  };

  const uint2 g0 = g_load(wave);
  issue_k(0);
  if constexpr (OUT) issue_q(0);
  issue_v(0);
  const float* s_in = nullptr;
  if constexpr (OUT)
    s_in = p.cut ? a.ends + ((size_t)p.slot * a.Hv + h) * hs
                 : a.s_in != nullptr ? a.s_in + ((size_t)p.seq * a.Hv + h) * hs : nullptr;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int kh = 0; kh < KH; ++kh)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        lf32x4 x = {0.f, 0.f, 0.f, 0.f};
        if (OUT && s_in != nullptr) x = *reinterpret_cast<const lf32x4*>(s_in + state_at(u, kh, i));
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[u][kh][e][i] = x[e];
      }
  g_store(wave, g0);
  uint2 gv = g0;
  float gsum = 0.f;
  const bool keep = p.last && a.s_out != nullptr;

  for (int c = 0; c < chunks; ++c) {
    wait_loads<0>();  // chunk c is there, and nobody reads what the next loads overwrite
    const int in_group = c % NW;
    if (in_group == 0 && c + NW < chunks) gv = g_load(c + NW + wave);
    issue_k(c + 1);
    if constexpr (!OUT) issue_v(c + 1);
    const uint8_t* ks = lds + (c & 1) * CH * C::KB;
    const uint8_t* vs = lds + C::AT_V + (OUT ? 0 : (c & 1) * CH * C::VB);
    const uint8_t* qs = lds + C::AT_Q;
    uint8_t* ps = lds + C::AT_P + 16 * l;
    const float* b = g_at(c);
    float v[4][4][U];  // tokens 16 i + 4 g + e
    auto read_v = [&] {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int at = (v0 + U * m) * 4;  // (a lane's U values lie in one chunk)
          const uint8_t* src = vs + chunk_at<C::VB, float>(16 * i + 4 * g + e, at >> 4) + (at & 15);
          if constexpr (U == 2) {
            const float2 x = *reinterpret_cast<const float2*>(src);
            v[i][e][0] = x.x, v[i][e][1] = x.y;
          } else {
            v[i][e][0] = *reinterpret_cast<const float*>(src);
          }
        }
    };
    if constexpr (OUT) {
      // P^T's 10 tiles (s tile i, t tile j, i <= j), wave, wave + 4 and (waves 0, 1) wave + 8
      lf32x4 d[3];
      int ti[3], tj[3];
#pragma unroll
      for (int x = 0; x < 3; ++x) {
        const int t = min(wave + 4 * x, 9);
        tj[x] = t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3;
        ti[x] = t - tj[x] * (tj[x] + 1) / 2;
        d[x] = lf32x4{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int kk = 0; kk < K / 16; ++kk) {
#pragma unroll
        for (int x = 0; x < 3; ++x) {
          const lf32x4 kf = *reinterpret_cast<const lf32x4*>(ks + 16 * ti[x] * C::KB + chunk_at<C::KB, float>(m, 4 * kk + g));
          const lf32x4 qf = *reinterpret_cast<const lf32x4*>(qs + 16 * tj[x] * C::KB + chunk_at<C::KB, float>(m, 4 * kk + g));
#pragma unroll
          for (int e = 0; e < 4; ++e) d[x] = mfma4(kf[e], qf[e], d[x]);
        }
      }
      const double* pd = reinterpret_cast<const double*>(b);
#pragma unroll
      for (int x = 0; x < 3; ++x) {
        const double gt = pd[16 * tj[x] + m];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // (a masked place's exponent may be of any size)
          const float f = a.scale * __expf((float)(gt - pd[16 * ti[x] + 4 * g + e])) * d[x][e];
          d[x][e] = 16 * ti[x] + 4 * g + e <= 16 * tj[x] + m ? f : 0.f;
        }
        if (x < 2 || wave < 2) *reinterpret_cast<lf32x4*>(ps + 1024 * (wave + 4 * x)) = d[x];
      }
      lf32x4 o[U][4];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[u][j] = lf32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kh = 0; kh < KH; ++kh)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          lf32x4 qf[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            qf[j] = *reinterpret_cast<const lf32x4*>(qs + 16 * j * C::KB + chunk_at<C::KB, float>(m, 16 * kh + 4 * g + i));
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int u = 0; u < U; ++u) o[u][j] = mfma4(acc[u][kh][e][i], qf[j][e], o[u][j]);
        }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float f = b[2 * CH + 16 * j + m];
#pragma unroll
        for (int u = 0; u < U; ++u) o[u][j] *= f;
      }
      read_v();
      bool odd = false;  // (a comparison with a NaN is false)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int u = 0; u < U; ++u) odd |= !(fabsf(v[i][e][u]) < INFINITY);
      const bool apart = __ballot(odd) != 0;
      lds_barrier();  // P is there, and nobody reads q and v any more
      issue_q(c + 1);
      issue_v(c + 1);
      auto p_frag = [&](int i, int j) { return *reinterpret_cast<const lf32x4*>(ps + 1024 * (j * (j + 1) / 2 + i)); };
      if (!apart) {
        lf32x4 pf[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = i; j < 4; ++j) pf[i][j] = p_frag(i, j);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int j = i; j < 4; ++j)
#pragma unroll
              for (int u = 0; u < U; ++u) o[u][j] = mfma4(v[i][e][u], pf[i][j][e], o[u][j]);
      } else {
        // an infinity or a NaN among the values: a masked P is zero, and zero times it NaN. Token by token, each added
        // from its own row on
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i <= j; ++i) {
            const lf32x4 pf = p_frag(i, j);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int u = 0; u < U; ++u)
#pragma unroll 1
                for (int gg = 0; gg < 4; ++gg) {
                  const lf32x4 y = mfma4(g == gg ? v[i][e][u] : 0.f, pf[e], lf32x4{0.f, 0.f, 0.f, 0.f});
                  if (16 * i + 4 * gg + e <= 16 * j + m) o[u][j] += y;
                }
          }
      }
      // the lane holds values 4 U g .. + 4 U - 1 of the wave's, of token 16 j + m (rows behind the segment are dropped)
      const uint32_t lb = (uint32_t)a.Hv * V * 4u;
      const int rows = min(CH, n - c * CH);
      const Rsrc rs = raw_rsrc(reinterpret_cast<float*>(a.o) + ((row0 + (size_t)c * CH) * a.Hv + h) * V,
                               (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(rows - 1) * lb + 4 * V)));
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int y = 0; y < U; ++y) {
          lf32x4 w;
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = U == 2 ? o[e & 1][j][2 * y + (e >> 1)] : o[0][j][e];
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(lu32x4, w), rs,
                                                 (uint32_t)(16 * j + m) * lb + 4 * (v0 + 4 * U * g + 4 * y), 0, 0);
        }
      if (c + 1 == chunks && !keep) break;
    } else {
      read_v();
    }
    const lf32x4 decay = *reinterpret_cast<const lf32x4*>(b + 4 * CH);
    const Decay dc = {decay[0], decay[1]};
    gsum += decay[2];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int kh = 0; kh < KH; ++kh)
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[u][kh][x][i] = decayed(acc[u][kh][x][i], dc);
    lf32x4 kf[2][KH];  // k's fragments, read one step ahead
    auto k_read = [&](int x) {
#pragma unroll
      for (int kh = 0; kh < KH; ++kh)
        kf[x & 1][kh] = *reinterpret_cast<const lf32x4*>(ks + chunk_at<C::KB, float>(16 * (x >> 2) + 4 * g + (x & 3), 16 * kh + m));
    };
    k_read(0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const lf32x4 w = *reinterpret_cast<const lf32x4*>(b + 3 * CH + 16 * i + 4 * g);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int u = 0; u < U; ++u) v[i][e][u] *= w[e];
    }
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      fence();
      if (x + 1 < 16) k_read(x + 1);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int kh = 0; kh < KH; ++kh)
#pragma unroll
          for (int y = 0; y < 4; ++y) acc[u][kh][y] = mfma4(kf[x & 1][kh][y], v[x >> 2][x & 3][u], acc[u][kh][y]);
    }
    fence();
    if (in_group == NW - 1 && c + 1 < chunks) g_store(c + 1 + wave, gv);
  }
  if constexpr (OUT) {
    if (keep) put(a.s_out + ((size_t)p.seq * a.Hv + h) * hs);
  } else {
    const size_t at = (size_t)p.slot * a.Hv + h;
    put(a.ends + at * hs);
    if (wave == 0 && l == 0) a.gtot[at] = gsum;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (as above)
}

// The states before a sequence's runs, in place of what the runs add: c_0 the initial state, c_{j+1} = exp(G_j) c_j + E_j.
// A thread keeps 4 elements, 8 runs loaded ahead.
__global__ __launch_bounds__(256) void lin_join_kernel(LinArgs a, int hs) {
  const int unit = blockIdx.x, part = blockIdx.y;
  const int seq = unit / a.Hv, h = unit - seq * a.Hv;
  int slot0 = 0, n = 0;
  if (a.cu == nullptr) {
    n = pieces(a.T, a.run);
    slot0 = seq * n;
  } else {
    const int l = threadIdx.x & 63;
    int bos, eos;
    seq_bounds(a.cu, seq, a.T, bos, eos);
    n = pieces(eos - bos, a.run);
    if (n < 2) return;
    int sum = 0;
    for (int s = l; s < seq; s += 64) {
      seq_bounds(a.cu, s, a.T, bos, eos);
      sum += pieces(eos - bos, a.run);
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
    slot0 = sum;
  }
  n = min(n, a.run_slots - slot0);  // (tables whose sequences overlap may name more runs than there are slots)
  const size_t at = (size_t)part * 1024 + 4 * threadIdx.x;
  lf32x4 c = {0.f, 0.f, 0.f, 0.f};
  if (a.s_in != nullptr) c = *reinterpret_cast<const lf32x4*>(a.s_in + ((size_t)seq * a.Hv + h) * hs + at);
  constexpr int U = 8;
  for (int j0 = 0; j0 < n; j0 += U) {
    lf32x4 e[U];
    float gt[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const size_t u = (size_t)(slot0 + min(j0 + i, n - 1)) * a.Hv + h;  // (what the last run adds is not written)
      e[i] = *reinterpret_cast<const lf32x4*>(a.ends + u * hs + at);
      gt[i] = a.gtot[u];
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (j0 + i >= n) break;
      *reinterpret_cast<lf32x4*>(a.ends + ((size_t)(slot0 + j0 + i) * a.Hv + h) * hs + at) = c;
      const float d = expf(gt[i]);
#pragma unroll
      for (int x = 0; x < 4; ++x) c[x] = fmaf(c[x], d, e[i][x]);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------- host

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

struct Plan {
  int run, run_slots, single;
  size_t gtot, total;  // offset into the workspace (behind the segments' states), its size
};

// Value heads that a workgroup of the bf16 walk takes together: two of 64 columns where they share a key head.
int walk_heads(int Hk, int Hv, int V) { return V == 64 && Hv / Hk % 2 == 0 ? 2 : 1; }

Plan make_plan(bool packed, int N, int T, int Hk, int Hv, int K, int V, int dtype) {
  Plan p;
  // Segments of a CU's share of the chunks. Half as long, two to a CU, 4096 tokens of 16 heads of 128 x 128 take 53.3 us
  // instead of 46.2 (more states through the join and the state pass) and 32768 on one key head the same 127. Sequences that
  // fill the CUs uncut are not cut below 1.5 shares: 32 of 64 .. 2048 tokens, 16 heads, take 173 us so, and 198 cut to 16
  // chunks.
  const long rows = packed ? T : (long)N * T, groups = dtype == ZGDN_BF16 ? Hv / walk_heads(Hk, Hv, V) : Hv;
  const long share = (rows * groups + CUS * CH - 1) / (CUS * CH);
  p.run = (int)std::min(std::max(1L, N * groups >= CUS ? share + share / 2 : share) * CH, (long)INT32_MAX / 4);
  // (at most: a packed batch's sequences are not known here)
  p.run_slots = (int)(packed ? T / p.run + (long)N : N * std::max(1L, ((long)T + p.run - 1) / p.run));
  p.single = T <= p.run;
  p.gtot = p.single ? 0 : (size_t)p.run_slots * Hv * K * V * 4;
  p.total = p.gtot + (p.single ? 0 : ((size_t)p.run_slots * Hv * 4 + 255) / 256 * 256);
  return p;
}

bool sizes_ok(int Hk, int Hv, int K, int V, int dtype) {
  return Hk >= 1 && Hv >= 1 && Hv % Hk == 0 && (K == 64 || K == 128) && (V == 64 || V == 128) &&
         (dtype == ZGDN_F32 || dtype == ZGDN_BF16);
}

// The state pass over all segments but a sequence's last, the join, the walk over the outputs.
template <typename FS, typename FO>
int launch_walks(const char* fn, const LinArgs& a, const Plan& p, FS states, int states_lds, FO outputs, int outputs_lds,
                 std::atomic<signed char>* ready, int groups, int threads, int state_size, hipStream_t s) {
  if (!lds_ready(outputs, outputs_lds, ready) || !lds_ready(states, states_lds, ready + 64))
    return fail(ZGDN_EHIP, "%s: the device refused the LDS", fn);
  if (!p.single) {
    const int before_last = a.cu != nullptr ? a.T / a.run : a.N * ((a.T + a.run - 1) / a.run - 1);  // segments, at most
    hipLaunchKernelGGL(states, dim3((unsigned)(before_last * groups)), dim3(threads), states_lds, s, a);
    hipLaunchKernelGGL(lin_join_kernel, dim3((unsigned)(a.N * a.Hv), (unsigned)(state_size / 1024)), dim3(256), 0, s, a, state_size);
  }
  hipLaunchKernelGGL(outputs, dim3((unsigned)(p.run_slots * groups)), dim3(threads), outputs_lds, s, a);
  return ZGDN_OK;
}

template <int K, int V, int NH, int U>
int launch_bf16(const char* fn, const LinArgs& a, const Plan& p, hipStream_t s) {
  using CO = WalkCfg<K, V, NH, U, true>;
  using CS = WalkCfg<K, V, NH, U, false>;
  static std::atomic<signed char> ready[128];
  return launch_walks(fn, a, p, lin_walk_kernel<K, V, NH, U, false>, CS::LDS, lin_walk_kernel<K, V, NH, U, true>, CO::LDS, ready,
                      a.Hv / NH, 64 * CO::NW, K * V, s);
}

template <int K, int V>
int launch_f32(const char* fn, const LinArgs& a, const Plan& p, hipStream_t s) {
  using CO = Walk32Cfg<K, V, true>;
  using CS = Walk32Cfg<K, V, false>;
  static std::atomic<signed char> ready[128];
  return launch_walks(fn, a, p, lin_walk_f32_kernel<K, V, false>, CS::LDS, lin_walk_f32_kernel<K, V, true>, CO::LDS, ready,
                      a.Hv, 64 * CO::NW, K * V, s);
}

template <int K, int V>
int launch_all(const char* fn, const LinArgs& a, const Plan& p, int dtype, hipStream_t s) {
  if (dtype == ZGDN_F32) return launch_f32<K, V>(fn, a, p, s);
  if constexpr (V == 64) {
    if (walk_heads(a.Hk, a.Hv, V) == 2)
      return (long)p.run_slots * (a.Hv / 2) <= CUS ? launch_bf16<K, V, 2, 1>(fn, a, p, s) : launch_bf16<K, V, 2, 2>(fn, a, p, s);
  }
  return (long)p.run_slots * a.Hv <= CUS ? launch_bf16<K, V, 1, 1>(fn, a, p, s) : launch_bf16<K, V, 1, 2>(fn, a, p, s);
}

}  // namespace
}  // namespace zgdn

extern "C" size_t zlin_attn_workspace_bytes(int packed, int n_seqs, int T, int Hk, int Hv, int K, int V, int dtype) {
  using namespace zgdn;
  if (n_seqs < 1 || T < 0 || !sizes_ok(Hk, Hv, K, V, dtype)) return 0;
  return make_plan(packed != 0, n_seqs, T, Hk, Hv, K, V, dtype).total;
}

extern "C" int zlin_attn_fwd(const void* q, long q_ld, const void* k, long k_ld, const void* v, long v_ld, int dtype,
                             const void* g, long g_ld, int g_dtype, const float* initial_state, float* final_state,
                             void* o, const int32_t* cu_seqlens, int n_seqs, int B, int T, int Hk, int Hv, int K, int V,
                             float scale, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace zgdn;
  const char* fn = "zlin_attn_fwd";
  if (B < 1 || T < 0 || Hk < 1 || Hv < 1) return fail(ZGDN_EINVAL, "%s: bad sizes B=%d T=%d Hk=%d Hv=%d", fn, B, T, Hk, Hv);
  if (Hv % Hk) return fail(ZGDN_EINVAL, "%s: Hv=%d is not a multiple of Hk=%d", fn, Hv, Hk);
  if (!sizes_ok(Hk, Hv, K, V, ZGDN_BF16))
    return fail(ZGDN_EUNSUPPORTED, "%s: K=%d V=%d (supported: 64 and 128 each)", fn, K, V);
  for (int dt : {dtype, g_dtype})
    if (dt != ZGDN_F32 && dt != ZGDN_BF16) return fail(ZGDN_EINVAL, "%s: unknown dtype code %d", fn, dt);
  if ((T > 0 && (!q || !k || !v || !g || !o)) || (g_ld == 0 && !g)) return fail(ZGDN_EINVAL, "%s: null tensor pointer", fn);
  const int N = cu_seqlens != nullptr ? n_seqs : B;
  if (cu_seqlens != nullptr && B != 1) return fail(ZGDN_EINVAL, "%s: cu_seqlens needs B == 1 (got B=%d)", fn, B);
  if (N < 1) return fail(ZGDN_EINVAL, "%s: n_seqs=%d with cu_seqlens", fn, n_seqs);
  if (g_ld == 0 ? g_dtype != ZGDN_F32 : g_ld < Hv)
    return fail(ZGDN_EINVAL, "%s: g rows %ld apart (at least %d, or 0 for float32 decays a head)", fn, g_ld, Hv);
  const int ve = dtype == ZGDN_F32 ? 4 : 8;
  if (q_ld < (long)Hk * K || k_ld < (long)Hk * K || v_ld < (long)Hv * V || q_ld % ve || k_ld % ve || v_ld % ve ||
      q_ld > (1 << 22) || k_ld > (1 << 22) || v_ld > (1 << 22))
    return fail(ZGDN_EINVAL, "%s: row strides q=%ld k=%ld v=%ld (multiples of %d elements, at least a row, at most 2^22)", fn,
                q_ld, k_ld, v_ld, ve);
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o | (uintptr_t)initial_state | (uintptr_t)final_state |
       (uintptr_t)workspace) % 16)
    return fail(ZGDN_EINVAL, "%s: q, k, v, o, states and workspace need 16-byte aligned bases", fn);
  const size_t n_state = (size_t)N * Hv * K * V;
  if (initial_state != nullptr && final_state != nullptr && initial_state != final_state &&
      initial_state < final_state + n_state && final_state < initial_state + n_state)
    return fail(ZGDN_EINVAL, "%s: initial_state and final_state overlap without being the same", fn);
  if ((long)B * T > INT32_MAX) return fail(ZGDN_EUNSUPPORTED, "%s: B=%d x T=%d rows", fn, B, T);
  const Plan p = make_plan(cu_seqlens != nullptr, N, T, Hk, Hv, K, V, dtype);
  if ((long)p.run_slots * Hv >= 1 << 24)  // (a grid has 2^32 threads; slots: at least one a sequence)
    return fail(ZGDN_EUNSUPPORTED, "%s: %d segments of %d heads", fn, p.run_slots, Hv);
  if (workspace_bytes < p.total || (workspace == nullptr && p.total > 0))
    return fail(ZGDN_EINVAL, "%s: workspace of %zu bytes, %zu needed", fn, workspace_bytes, p.total);
  const size_t es = dtype == ZGDN_F32 ? 4 : 2, ge = g_dtype == ZGDN_F32 ? 4 : 2, rows = (size_t)B * T;
  const Region out = {o, rows, (size_t)Hv * V * es, (size_t)Hv * V * es}, end = {final_state, 1, n_state * 4, n_state * 4},
               work = {workspace, 1, p.total, p.total};
  const Region in[] = {{q, rows, (size_t)Hk * K * es, q_ld * es}, {k, rows, (size_t)Hk * K * es, k_ld * es},
                       {v, rows, (size_t)Hv * V * es, v_ld * es}, {g, g_ld == 0 ? 1 : rows, Hv * ge, g_ld == 0 ? Hv * ge : g_ld * ge},
                       {cu_seqlens, 1, (size_t)(N + 1) * 4, (size_t)(N + 1) * 4}, {initial_state, 1, n_state * 4, n_state * 4}};
  bool meet = regions_meet(out, end) || regions_meet(out, work) || regions_meet(end, work);
  for (const Region& r : in)
    meet = meet || regions_meet(out, r) || regions_meet(work, r) || (r.at != initial_state && regions_meet(end, r));
  if (meet) return fail(ZGDN_EINVAL, "%s: o, final_state or the workspace overlap another operand", fn);
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  LinArgs a{};
  a.q = q, a.k = k, a.v = v, a.g = g;
  a.q_ld = q_ld, a.k_ld = k_ld, a.v_ld = v_ld, a.g_ld = g_ld;
  a.g_bf16 = g_dtype == ZGDN_BF16;
  a.s_in = initial_state, a.s_out = final_state, a.o = o, a.cu = cu_seqlens;
  a.N = N, a.T = T, a.Hk = Hk, a.Hv = Hv, a.scale = scale;
  a.run = p.run, a.run_slots = p.run_slots;
  a.ends = (float*)ws, a.gtot = (float*)(ws + p.gtot);
  hipStream_t hs = (hipStream_t)stream;
  const int st = K == 128 ? (V == 128 ? launch_all<128, 128>(fn, a, p, dtype, hs) : launch_all<128, 64>(fn, a, p, dtype, hs))
                          : (V == 128 ? launch_all<64, 128>(fn, a, p, dtype, hs) : launch_all<64, 64>(fn, a, p, dtype, hs));
  return st != ZGDN_OK ? st : check_launch(fn);
}
