// Linear attention with a decay per head over whole sequences, on MFMA.
//
//   S_t = exp(g_t) S_{t-1} + v_t k_t^T,   o_t = S_t (scale q_t)
//
// A sequence is cut into segments of L tokens. With S the state before a segment and G the running sum of g in it,
//   o_t = exp(G_t) S (scale q_t) + sum_{s <= t} exp(G_t - G_s) (scale q_t . k_s) v_s,
// so the segments' outputs are independent given their start states, which come from sums over the tokens before:
//   1. lin_state: sequences are also cut into runs of whole segments. A run's state is summed in registers, 64 tokens at a
//      time, from zeros (a sequence's first run: from its initial state), and written down at each segment's start.
//   2. lin_carry (where a sequence may have several runs): the state before each run from the runs' end states.
//   3. lin_out: each segment's outputs from its start state (the written one plus the carried one, decayed) and its rows.
// Products are bf16 x bf16 with fp32 sums. States stay fp32: where a product takes a state or a weighted value it is
// split into bf16 terms whose sum has 16 (outputs: two terms) or 24 bits (states: three), so that an output keeps only
// its own rounding and a state that of fp32 sums. fp32 inputs take the same steps on the fp32 MFMA.
//
// The exponents are sums of one sign where all g <= 0: suffix sums to a block's end and prefix sums from its start, not
// differences of long sums. g is taken as at least -200 (exp(-200) is zero in fp32), so that -inf resets a state.
#include <algorithm>
#include <atomic>

#include "gdn_common.h"
#include "zonos3_linear.h"

namespace zgdn {
namespace {

typedef __bf16 lbf16x8 __attribute__((ext_vector_type(8)));
typedef float lf32x4 __attribute__((ext_vector_type(4)));
typedef short lshort4 __attribute__((ext_vector_type(4)));

constexpr int ST = 64;  // tokens of a stage of the state pass
constexpr int CH = 64;  // tokens of a chunk of the walk
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
  int seg, run;      // tokens of a segment, of a run (a multiple of seg)
  int seg_slots, run_slots;
  int direct;        // one run a sequence: its end is the final state
  int save_first;    // the first segment's start state is written down too (the final state overwrites the initial one)
  float *ckpt, *gcum;  // [seg_slots][Hv][V * K], [seg_slots][Hv]: state before a segment within its run, log decay from there
  float *ends, *gtot;  // [run_slots][Hv][V * K], [run_slots][Hv]: a run's end state (then the state before it), log decay
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
__device__ __forceinline__ float load_g(const LinArgs& a, size_t t, int h) { return g_value(a, g_bits(a, t, h)); }

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

// A sequence's piece of `size` tokens by its slot (pieces numbered sequence by sequence, at least one each), with the
// slot of the sequence's first piece of `other` tokens. Whole waves call it together.
struct Piece {
  int seq, j, bos, len, other0;
};
__device__ __forceinline__ bool find_piece(const int32_t* cu, int N, int T, int slot, int size, int other, Piece& p) {
  if (cu == nullptr) {
    const int per = pieces(T, size);
    p.seq = slot / per;
    p.j = slot - p.seq * per;
    p.bos = p.seq * T;
    p.len = T;
    p.other0 = p.seq * pieces(T, other);
    return p.seq < N;
  }
  const int l = threadIdx.x & 63;
  int base = 0, base2 = 0;
  for (int s0 = 0; s0 < N; s0 += 64) {
    int bos = 0, eos = 0, n = 0, n2 = 0;
    if (s0 + l < N) {
      seq_bounds(cu, s0 + l, T, bos, eos);
      n = pieces(eos - bos, size);
      n2 = pieces(eos - bos, other);
    }
    int i = n, i2 = n2;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int u = __shfl_up(i, d), u2 = __shfl_up(i2, d);
      i += l >= d ? u : 0;
      i2 += l >= d ? u2 : 0;
    }
    const uint64_t past = __ballot(base + i > slot);
    if (past) {
      const int f = __builtin_ctzll(past);
      p.seq = s0 + f;
      p.j = slot - base - (__shfl(i, f) - __shfl(n, f));
      p.bos = __shfl(bos, f);
      p.len = __shfl(eos, f) - p.bos;
      p.other0 = base2 + __shfl(i2, f) - __shfl(n2, f);
      return true;
    }
    base += __shfl(i, 63);
    base2 += __shfl(i2, 63);
  }
  return false;
}
// (the same values in scalar registers: buffer resources are built from them)
__device__ __forceinline__ void uniform(Piece& p) {
  p.seq = __builtin_amdgcn_readfirstlane(p.seq);
  p.j = __builtin_amdgcn_readfirstlane(p.j);
  p.bos = __builtin_amdgcn_readfirstlane(p.bos);
  p.len = __builtin_amdgcn_readfirstlane(p.len);
  p.other0 = __builtin_amdgcn_readfirstlane(p.other0);
}

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
// Rows of ROWB bytes (64 .. 512), 16-byte chunk c of row r at c ^ mask(r): row fragments (16 rows, one chunk each) and
// transposing reads (4 rows, 32 bytes each, for each group of 16 lanes) then spread over the banks.

template <int ROWB>
__device__ __forceinline__ int chunk_at(int r, int c) {
  constexpr int n = ROWB / 16;
  const int f = n >= 16 ? (r & 7) << 1 | (r >> 3 & 1) : n == 8 ? (r >> 1) & 7 : (r >> 1) & 3;
  return r * ROWB + ((c ^ f) << 4);
}

// 16 bytes a lane from a buffer straight into LDS, lane i at lds + 16 i. In assembly, since the compiler waits for every such
// load ahead of a transposing LDS read, whatever it reads: here the kernels' own waits are in charge. Nothing is written to a
// register; M0 (which these kernels use for nothing else) needs a wait state before the load.
typedef uint32_t lu32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void load_lds(lu32x4 rsrc, uint32_t off, const uint8_t* lds) {
  const uint32_t at = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)lds);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(at), "v"(off), "s"(rsrc) : "memory");
}

// ROWS rows of ROWB bytes from global memory (row stride ld_bytes, `rows` of them there, zeros behind them) into LDS, by
// NW waves; each wave instruction fills 1 KiB, so a lane fetches the chunk that belongs at its place. The places in a row
// repeat every PERIOD instructions of a wave: these byte offsets are kept, the others follow by whole rows.
template <int ROWB, int NW>
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
      off[i] = (uint32_t)(r - i * NW * RP) * ld_bytes + (uint32_t)(chunk_at<ROWB>(r, l % n) - r * ROWB);
    }
  }
  __device__ __forceinline__ void anew() {  // (nothing formed from them is kept across)
#pragma unroll
    for (int i = 0; i < PERIOD; ++i) asm volatile("" : "+v"(off[i]));
  }
};
// (instructions i0 .. i1 - 1 of the wave's ROWS ROWB / 1024 / NW)
template <int ROWB, int ROWS, int NW>
__device__ __forceinline__ void load_rows(const RowsAt<ROWB, NW>& at_row, const void* base, uint32_t ld_bytes, int rows,
                                          uint8_t* lds, int wave, int i0 = 0, int i1 = ROWS * ROWB / 1024 / NW) {
  constexpr int RP = 1024 / ROWB;  // rows an instruction
  static_assert(ROWS % (RP * NW) == 0, "as many a wave");
  const uint32_t bytes = rows > 0 ? (uint32_t)(rows - 1) * ld_bytes + ROWB : 0u;
  const uint64_t at = (uint64_t)(uintptr_t)base;
  const lu32x4 rs = {(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)at),
                     (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(at >> 32) & 0xffffu)),
                     (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
#pragma unroll
  for (int i = i0; i < i1; ++i)
    load_lds(rs, at_row.off[i % RowsAt<ROWB, NW>::PERIOD] + (uint32_t)(i * NW * RP) * ld_bytes, lds + 1024 * (i * NW + wave));
}
template <int ROWB, int ROWS, int NW>
__device__ __forceinline__ void load_rows(const void* base, uint32_t ld_bytes, int rows, uint8_t* lds, int wave) {
  load_rows<ROWB, ROWS, NW>(RowsAt<ROWB, NW>(ld_bytes, wave), base, ld_bytes, rows, lds, wave);
}

__device__ __forceinline__ uint2 lds_tr(const uint8_t* p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) lshort4*)p));
}
// Fragment of a tile's transpose: column c0 + (lane % 16) of rows r0 + 4 g + {0..3} and r0 + 16 + 4 g + {0..3}
// (g = lane / 16), the order in which two D tiles below one another hold their rows.
template <int ROWB>
__device__ __forceinline__ lbf16x8 tr_frag(const uint8_t* tile, int r0, int c0) {
  const int l = threadIdx.x & 63, g = l >> 4, s = l & 15;
  const int r = r0 + 4 * g + (s >> 2), c = c0 / 8 + ((s & 3) >> 1);
  const uint2 a = lds_tr(tile + chunk_at<ROWB>(r, c) + 8 * (s & 1));
  const uint2 b = lds_tr(tile + chunk_at<ROWB>(r + 16, c) + 8 * (s & 1));
  return __builtin_bit_cast(lbf16x8, make_uint4(a.x, a.y, b.x, b.y));
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
__device__ __forceinline__ void loads_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

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

// Sum over the lanes after this one (suffix, without it) and over all of the wave's.
__device__ __forceinline__ float suffix_sum(float x, float& total) {
  const int l = threadIdx.x & 63;
  float s = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const float u = __shfl_down(s, d);
    s += l + d < 64 ? u : 0.f;
  }
  total = __shfl(s, 0);
  const float n = __shfl_down(s, 1);
  return l == 63 ? 0.f : n;
}

// ------------------------------------------------------------------------------------------------- 1. run states
//
// A workgroup of NW waves sums 16 NW value rows of one (run, head); wave w keeps rows 16 w .. of S as the transposed
// tiles [K / 16] (D: key 4 g + e, value lane % 16). A stage's tokens enter as sum_s K^T (M = key) x weighted V (N = value)
// over the tokens, both read transposed from LDS; the weights exp(G_end - G_s) go on v, split into three bf16 terms.

template <typename T, int K, int V, int NW>
struct StateCfg {
  static constexpr int ES = sizeof(T);
  static constexpr int KB = K * ES, VB = 16 * NW * ES;  // bytes of a row
  static constexpr int STAGE = ST * (KB + VB);
  static constexpr int LDS = 2 * STAGE + NW * ST * 4;
};

template <int K>
__device__ __forceinline__ void put_state(float* dst, const lf32x4 (&acc)[K / 16], int v0) {  // dst [V][K] of one head
  const int l = threadIdx.x & 63, g = l >> 4, m = l & 15;
#pragma unroll
  for (int kt = 0; kt < K / 16; ++kt)
    *reinterpret_cast<lf32x4*>(dst + (size_t)(v0 + m) * K + 16 * kt + 4 * g) = acc[kt];
}

template <typename T, int K, int V, int NW>
__global__ __launch_bounds__(64 * NW) void lin_state_kernel(LinArgs a) {
  using C = StateCfg<T, K, V, NW>;
  extern __shared__ uint4 lin_lds[];
  uint8_t* lds = reinterpret_cast<uint8_t*>(lin_lds);
  constexpr int VG = V / (16 * NW);
  // units (run, head) one after the other, the VG workgroups of one unit on one XCD (ids equal mod 8)
  const int id = blockIdx.x, unit = id / (8 * VG) * 8 + id % 8, vg = id / 8 % VG;
  const int slot = unit / a.Hv, h = unit - slot * a.Hv;
  if (slot >= a.run_slots) return;
  Piece p;
  if (!find_piece(a.cu, a.N, a.T, slot, a.run, a.seg, p)) return;
  uniform(p);
  const int wave = wave_id(), l = threadIdx.x & 63, g = l >> 4, m = l & 15;
  const int first = p.j * a.run, n = min(a.run, p.len - first);  // (n 0 for an empty sequence)
  const int v0 = 16 * NW * vg + 16 * wave;
  const size_t row0 = (size_t)p.bos + first;
  const T* kp = reinterpret_cast<const T*>(a.k) + row0 * a.k_ld + (size_t)(h / (a.Hv / a.Hk)) * K;
  const T* vp = reinterpret_cast<const T*>(a.v) + row0 * a.v_ld + (size_t)h * V + 16 * NW * vg;
  const uint32_t k_lb = (uint32_t)a.k_ld * C::ES, v_lb = (uint32_t)a.v_ld * C::ES;
  float* wts = reinterpret_cast<float*>(lds + 2 * C::STAGE) + wave * ST;  // the wave's own

  auto issue = [&](int s) {
    uint8_t* at = lds + (s & 1) * C::STAGE;
    load_rows<C::KB, ST, NW>(kp + (size_t)s * ST * a.k_ld, k_lb, n - s * ST, at, wave);
    load_rows<C::VB, ST, NW>(vp + (size_t)s * ST * a.v_ld, v_lb, n - s * ST, at + ST * C::KB, wave);
  };
  auto g_of = [&](int s) { return s * ST + l < n ? load_g(a, row0 + s * ST + l, h) : 0.f; };

  const int stages = (n + ST - 1) / ST;
  if (stages > 0) issue(0);
  float gv = g_of(0), gsum = 0.f;

  lf32x4 acc[K / 16];
#pragma unroll
  for (int kt = 0; kt < K / 16; ++kt) acc[kt] = lf32x4{0.f, 0.f, 0.f, 0.f};
  const size_t hs = (size_t)V * K;
  if (p.j == 0 && a.s_in != nullptr) {
    const float* src = a.s_in + ((size_t)p.seq * a.Hv + h) * hs;
#pragma unroll
    for (int kt = 0; kt < K / 16; ++kt)
      acc[kt] = *reinterpret_cast<const lf32x4*>(src + (size_t)(v0 + m) * K + 16 * kt + 4 * g);
  }
  // (segments past the slots: only tables whose sequences overlap name so many)
  if (p.j == 0 && a.save_first && p.other0 < a.seg_slots) put_state<K>(a.ckpt + ((size_t)p.other0 * a.Hv + h) * hs, acc, v0);

  for (int s = 0; s < stages; ++s) {
    const int at = p.other0 + (first + s * ST) / a.seg;
    if (s > 0 && s * ST % a.seg == 0 && at < a.seg_slots) {
      const size_t c = (size_t)at * a.Hv + h;
      put_state<K>(a.ckpt + c * hs, acc, v0);
      if (vg == 0 && threadIdx.x == 0) a.gcum[c] = gsum;
    }
    loads_barrier();  // stage s is there, and nobody reads the other one any more
    if (s + 1 < stages) issue(s + 1);
    float total;
    const float w = expf(suffix_sum(gv, total));
    gv = g_of(s + 1);
    gsum += total;
    wts[l] = w;
    const Decay d = decay_of(total);
#pragma unroll
    for (int kt = 0; kt < K / 16; ++kt)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[kt][e] = decayed(acc[kt][e], d);
    const uint8_t* ks = lds + (s & 1) * C::STAGE;
    const uint8_t* vs = ks + ST * C::KB;
    {
#pragma unroll 1
      for (int b = 0; b < ST; b += 16) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // tokens b + 4 g + e
          const int r = b + 4 * g + e;
          const int cv = 16 * wave + m;
          const float x = *reinterpret_cast<const float*>(vs + chunk_at<C::VB>(r, cv / 4) + 4 * (cv & 3)) * wts[r];
#pragma unroll
          for (int kt = 0; kt < K / 16; ++kt) {
            const float y = *reinterpret_cast<const float*>(ks + chunk_at<C::KB>(r, 4 * kt + (m >> 2)) + 4 * (m & 3));
            acc[kt] = mfma4(y, x, acc[kt]);
          }
        }
      }
    }
  }
  if (a.direct) {
    if (a.s_out != nullptr) put_state<K>(a.s_out + ((size_t)p.seq * a.Hv + h) * hs, acc, v0);
  } else {
    const size_t c = (size_t)slot * a.Hv + h;
    put_state<K>(a.ends + c * hs, acc, v0);
    if (vg == 0 && threadIdx.x == 0) a.gtot[c] = gsum;
  }
}

// ---------------------------------------------------------------------------------------------------- 2. carries
//
// The end states of a sequence's runs, in place, become the states carried into them: c_0 = 0 (the first run starts from
// the initial state itself), c_{j+1} = exp(G_j) c_j + E_j; the last one is the final state. A thread keeps 4 elements.

__global__ __launch_bounds__(256) void lin_carry_kernel(LinArgs a, int hs) {
  const int per = hs / 1024, unit = blockIdx.x / per, part = blockIdx.x % per;
  const int seq = unit / a.Hv, h = unit - seq * a.Hv;
  int slot0 = 0, n = 0;
  if (a.cu == nullptr) {
    n = pieces(a.T, a.run);
    slot0 = seq * n;
  } else {
    const int l = threadIdx.x & 63;
    int sum = 0;
    for (int s = l; s < seq; s += 64) {
      int bos, eos;
      seq_bounds(a.cu, s, a.T, bos, eos);
      sum += pieces(eos - bos, a.run);
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
    slot0 = sum;
    int bos, eos;
    seq_bounds(a.cu, seq, a.T, bos, eos);
    n = pieces(eos - bos, a.run);
  }
  n = min(n, a.run_slots - slot0);  // (tables whose sequences overlap may name more runs than there are slots)
  const size_t at = (size_t)part * 1024 + 4 * threadIdx.x;
  lf32x4 c = {0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j < n; ++j) {
    const size_t u = (size_t)(slot0 + j) * a.Hv + h;
    lf32x4* p = reinterpret_cast<lf32x4*>(a.ends + u * hs + at);
    const lf32x4 e = *p;
    const float d = expf(a.gtot[u]);
    *p = c;
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = fmaf(c[i], d, e[i]);
  }
  if (a.s_out != nullptr) *reinterpret_cast<lf32x4*>(a.s_out + ((size_t)seq * a.Hv + h) * hs + at) = c;
}

// Whether any of a block's R rows holds an infinity or a NaN (each wave for its own block).
template <int ROWB, int R>
__device__ __forceinline__ bool rows_not_finite(const uint8_t* rows, int es) {
  uint32_t bad = 0;
#pragma unroll
  for (int i = 0; i < ROWB * R / 1024; ++i) {
    const uint4 w = *reinterpret_cast<const uint4*>(rows + 1024 * i + 16 * (threadIdx.x & 63));
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      bad |= (x[e] & 0x7f800000u) == 0x7f800000u;
      if (es == 2) bad |= (x[e] & 0x7f80u) == 0x7f80u;
    }
  }
  return __ballot(bad) != 0;
}

// ---------------------------------------------------------------------------------------------------- 3. outputs
//
// A workgroup takes one (segment, head); a wave 32 tokens (fp32: 16), which are the columns of its transposed tiles:
//   O^T [V, t] = S Q^T (rows scaled by exp(G_t)) + V^T P^T,   P^T [s, t] = K Q^T scaled and masked.
// P^T's D tiles (token s = 4 g + e of 16, t = lane % 16) are the B operand of the second product as they stand, with V^T
// read transposed from LDS in the same order of s. The start state is split into two bf16 terms in LDS, P into two in
// registers. exp(G_t - G_s) is exp(prefix_t + blocks between) exp(suffix_s) across blocks of 32 and one exponential an
// element within a block.

template <typename T, int K, int V, int L>
struct OutCfg {
  static constexpr int ES = sizeof(T), TW = ES == 2 ? 32 : 16;  // tokens a wave
  static constexpr int NW = L / TW;
  static constexpr int KB = K * ES, VB = V * ES;
  static constexpr int S_BYTES = V * K * 4;  // two bf16 terms, or fp32
  static constexpr int AT_K = S_BYTES, AT_V = AT_K + L * KB, AT_W = AT_V + L * VB;
  static constexpr int LDS = AT_W + 2 * L * 4 + NW * 4 + (ES == 4 ? L * 8 : 0);
};

template <typename T, int K, int V, int L>
__global__ __launch_bounds__((64 * OutCfg<T, K, V, L>::NW)) void lin_out_kernel(LinArgs a) {
  using C = OutCfg<T, K, V, L>;
  constexpr int TW = C::TW, NW = C::NW, NT = TW / 16;
  extern __shared__ uint4 lin_lds[];
  uint8_t* lds = reinterpret_cast<uint8_t*>(lin_lds);
  uint8_t *kt_ = lds + C::AT_K, *vt_ = lds + C::AT_V;
  float* wsuf = reinterpret_cast<float*>(lds + C::AT_W);  // exp(suffix) of each token to its block's end
  float* pre = wsuf + L;                                  // prefix within the block, the token's own g included
  float* tot = pre + L;                                   // each block's sum
  const int slot = blockIdx.x / a.Hv, h = blockIdx.x - slot * a.Hv;
  Piece p;
  if (!find_piece(a.cu, a.N, a.T, slot, a.seg, a.run, p)) return;
  uniform(p);
  const int first = p.j * L, n = min(L, p.len - first);
  if (n <= 0) return;  // (an empty sequence)
  const int wave = wave_id(), l = threadIdx.x & 63, g = l >> 4, m = l & 15;
  const size_t row0 = (size_t)p.bos + first;
  const size_t hk = (size_t)(h / (a.Hv / a.Hk)) * K;
  const T* qp = reinterpret_cast<const T*>(a.q) + row0 * a.q_ld + hk;
  const T* kp = reinterpret_cast<const T*>(a.k) + row0 * a.k_ld + hk;
  const T* vp = reinterpret_cast<const T*>(a.v) + row0 * a.v_ld + (size_t)h * V;

  // the start state: within the run as written down (or the initial state), and what is carried into the run
  const int run = first / a.run, in_run = first - run * a.run;
  const size_t hs = (size_t)V * K;
  const float* s_loc = in_run > 0 || (p.j == 0 && a.save_first) ? a.ckpt + ((size_t)slot * a.Hv + h) * hs
                       : p.j == 0 && a.s_in != nullptr          ? a.s_in + ((size_t)p.seq * a.Hv + h) * hs
                                                                : nullptr;
  const float* s_car = run > 0 && p.other0 + run < a.run_slots ? a.ends + ((size_t)(p.other0 + run) * a.Hv + h) * hs : nullptr;
  const bool has_state = s_loc != nullptr || s_car != nullptr;
  if (has_state) {
    const float dc = s_car == nullptr ? 0.f : in_run > 0 ? expf(a.gcum[(size_t)slot * a.Hv + h]) : 1.f;
    constexpr int THREADS = 64 * NW, PER = V * K / 4 / THREADS, BATCH = PER > 16 ? 16 : PER;
#pragma unroll 1
    for (int b = 0; b < PER; b += BATCH) {
      lf32x4 x[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const size_t at = 4 * ((size_t)(b + i) * THREADS + threadIdx.x);
        x[i] = s_loc != nullptr ? *reinterpret_cast<const lf32x4*>(s_loc + at) : lf32x4{0.f, 0.f, 0.f, 0.f};
      }
      if (s_car != nullptr) {
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
          const size_t at = 4 * ((size_t)(b + i) * THREADS + threadIdx.x);
          const lf32x4 y = *reinterpret_cast<const lf32x4*>(s_car + at);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[i][e] = fmaf(y[e], dc, x[i][e]);
        }
      }
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int at = 4 * ((b + i) * THREADS + (int)threadIdx.x), v = at / K, k = at % K;
        if constexpr (C::ES == 2) {
          uint32_t w0[2], w1[2];
          split_pair<2>(x[i][0], x[i][1], w0);
          split_pair<2>(x[i][2], x[i][3], w1);
          uint8_t* base = lds + (k / 32) * V * 128;  // rows of 64 bytes of first terms, 64 of second ones
          const int c = (k % 32) / 8, half = k & 4 ? 8 : 0;
          *reinterpret_cast<uint2*>(base + chunk_at<128>(v, c) + half) = make_uint2(w0[0], w1[0]);
          *reinterpret_cast<uint2*>(base + chunk_at<128>(v, 4 + c) + half) = make_uint2(w0[1], w1[1]);
        } else {
          *reinterpret_cast<lf32x4*>(lds + chunk_at<K * 4>(v, k / 4)) = x[i];
        }
      }
    }
  }
  load_rows<C::KB, L, NW>(kp, (uint32_t)a.k_ld * C::ES, n, kt_, wave);
  load_rows<C::VB, L, NW>(vp, (uint32_t)a.v_ld * C::ES, n, vt_, wave);

  // the wave's queries: lane's token m of each tile, 16 bytes of keys a step
  const int t0 = wave * TW;
  constexpr int QS = C::KB / 64;  // steps of 64 bytes of a row
  uint4 q[NT][QS];
  {
    const uint32_t lb = (uint32_t)a.q_ld * C::ES;
    const Rsrc rs = raw_rsrc(qp, (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(n - 1) * lb + C::KB)));
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < QS; ++i)
        q[j][i] = __builtin_bit_cast(
            uint4, __builtin_amdgcn_raw_buffer_load_b128(rs, (uint32_t)(t0 + 16 * j + m) * lb + 64 * i + 16 * g, 0, 0));
  }
  // decays of the wave's own block: lanes 0 .. TW - 1 a token each
  {
    const int i = l & (TW - 1), t = t0 + i;
    const float gv = t < n ? load_g(a, row0 + t, h) : 0.f;
    float s = gv, u = gv;  // prefix and suffix, inclusive
    double sd = (double)gv;
#pragma unroll
    for (int d = 1; d < TW; d <<= 1) {
      const float x = __shfl_up(s, d, TW), y = __shfl_down(u, d, TW);
      s += i >= d ? x : 0.f;
      u += i + d < TW ? y : 0.f;
      if constexpr (C::ES == 4) {
        const double z = __shfl_up(sd, d, TW);
        sd += i >= d ? z : 0.0;
      }
    }
    const float nx = __shfl_down(u, 1, TW);
    if (l < TW) {
      wsuf[t] = expf(i == TW - 1 ? 0.f : nx);
      pre[t] = s;
      if constexpr (C::ES == 4) reinterpret_cast<double*>(tot + NW + (NW & 1))[t] = sd;
      if (i == TW - 1) tot[wave] = s;
    }
  }
  loads_barrier();

  lf32x4 acc[V / 16][NT];
#pragma unroll
  for (int v = 0; v < V / 16; ++v)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[v][j] = lf32x4{0.f, 0.f, 0.f, 0.f};
  float pt[NT];  // the lane's tokens' prefixes
#pragma unroll
  for (int j = 0; j < NT; ++j) pt[j] = pre[t0 + 16 * j + m];

  if (has_state) {
    if constexpr (C::ES == 2) {
#pragma unroll
      for (int i = 0; i < K / 32; ++i) {
        const uint8_t* base = lds + i * V * 128;
#pragma unroll
        for (int v = 0; v < V / 16; ++v) {
          const lbf16x8 hi = *reinterpret_cast<const lbf16x8*>(base + chunk_at<128>(16 * v + m, g));
          const lbf16x8 lo = *reinterpret_cast<const lbf16x8*>(base + chunk_at<128>(16 * v + m, 4 + g));
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const lbf16x8 b = __builtin_bit_cast(lbf16x8, q[j][i]);
            acc[v][j] = mfma16(lo, b, acc[v][j]);
            acc[v][j] = mfma16(hi, b, acc[v][j]);
          }
        }
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < K / 16; ++i) {
#pragma unroll
        for (int v = 0; v < V / 16; ++v) {
          const lf32x4 x = *reinterpret_cast<const lf32x4*>(lds + chunk_at<K * 4>(16 * v + m, 4 * i + g));
          lf32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ii = 0; ii < QS; ++ii)
            if (ii == i) y = __builtin_bit_cast(lf32x4, q[0][ii]);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[v][0] = mfma4(x[e], y[e], acc[v][0]);
        }
      }
    }
    float before = 0.f;
    for (int b = 0; b < wave; ++b) before += tot[b];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const float f = a.scale * expf(before + pt[j]);
#pragma unroll
      for (int v = 0; v < V / 16; ++v) acc[v][j] *= f;
    }
  }

  float between = 0.f;  // sum of the blocks between the one at hand and the wave's own
  for (int sb = wave; sb >= 0; --sb) {
    const int s0 = sb * TW;
    lf32x4 pp[NT][NT];  // [s tile][t tile]
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int j = 0; j < NT; ++j) pp[i][j] = lf32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < QS; ++kk) {
        const uint4 kf = *reinterpret_cast<const uint4*>(kt_ + chunk_at<C::KB>(s0 + 16 * i + m, 4 * kk + g));
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          if constexpr (C::ES == 2) {
            pp[i][j] = mfma16(__builtin_bit_cast(lbf16x8, kf), __builtin_bit_cast(lbf16x8, q[j][kk]), pp[i][j]);
          } else {
            const lf32x4 x = __builtin_bit_cast(lf32x4, kf), y = __builtin_bit_cast(lf32x4, q[j][kk]);
#pragma unroll
            for (int e = 0; e < 4; ++e) pp[i][j] = mfma4(x[e], y[e], pp[i][j]);
          }
        }
      }
    }
    if (sb == wave) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int s = 16 * i + 4 * g + e, t = 16 * j + m;
            float d;
            if constexpr (C::ES == 4) {
              const double* pd = reinterpret_cast<const double*>(tot + NW + (NW & 1)) + s0;
              d = (float)(pd[t] - pd[s]);
            } else {
              d = pt[j] - pre[s0 + s];
            }
            pp[i][j][e] = s <= t ? pp[i][j][e] * (a.scale * expf(d)) : 0.f;
          }
    } else {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const float f = a.scale * expf(pt[j] + between);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const lf32x4 w = *reinterpret_cast<const lf32x4*>(wsuf + s0 + 16 * i + 4 * g);
#pragma unroll
          for (int e = 0; e < 4; ++e) pp[i][j][e] *= f * w[e];
        }
      }
      between += tot[sb];
    }
    if constexpr (C::ES == 2) {
      lbf16x8 ph[NT], pl[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        uint32_t w[4][2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          split_pair<2>(pp[i][j][0], pp[i][j][1], w[2 * i]);
          split_pair<2>(pp[i][j][2], pp[i][j][3], w[2 * i + 1]);
        }
        ph[j] = __builtin_bit_cast(lbf16x8, make_uint4(w[0][0], w[1][0], w[2][0], w[3][0]));
        pl[j] = __builtin_bit_cast(lbf16x8, make_uint4(w[0][1], w[1][1], w[2][1], w[3][1]));
      }
      if (sb == wave && rows_not_finite<C::VB, TW>(vt_ + s0 * C::VB, C::ES)) {
        // a masked P is zero, and zero times such a value is NaN: token by token, each added from its own row on
        for (int s = 0; s < TW; ++s) {
          const bool mine = (s >> 2 & 3) == g;  // the lane's fragment holds token s at place s % 4 + 4 (s / 16)
          const int at = (s & 3) + 4 * (s >> 4);
#pragma unroll
          for (int v = 0; v < V / 16; ++v) {
            uint4 w = __builtin_bit_cast(uint4, tr_frag<C::VB>(vt_, s0, 16 * v));
            const uint32_t half = mine ? (at & 1 ? 0xffff0000u : 0x0000ffffu) : 0u;
            w.x &= at >> 1 == 0 ? half : 0u;
            w.y &= at >> 1 == 1 ? half : 0u;
            w.z &= at >> 1 == 2 ? half : 0u;
            w.w &= at >> 1 == 3 ? half : 0u;
            const lbf16x8 vf = __builtin_bit_cast(lbf16x8, w);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              lf32x4 x = {0.f, 0.f, 0.f, 0.f};
              x = mfma16(vf, pl[j], x);
              x = mfma16(vf, ph[j], x);
              if (s <= 16 * j + m) acc[v][j] += x;
            }
          }
        }
      } else {
#pragma unroll
        for (int v = 0; v < V / 16; ++v) {
          const lbf16x8 vf = tr_frag<C::VB>(vt_, s0, 16 * v);
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            acc[v][j] = mfma16(vf, pl[j], acc[v][j]);
            acc[v][j] = mfma16(vf, ph[j], acc[v][j]);
          }
        }
      }
    } else {
      const bool apart = sb == wave && rows_not_finite<C::VB, TW>(vt_ + s0 * C::VB, C::ES);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = s0 + 4 * g + e;
#pragma unroll
        for (int v = 0; v < V / 16; ++v) {
          const float x = *reinterpret_cast<const float*>(vt_ + chunk_at<C::VB>(r, 4 * v + (m >> 2)) + 4 * (m & 3));
          if (!apart) {
            acc[v][0] = mfma4(x, pp[0][0][e], acc[v][0]);
          } else {  // (as above)
            for (int gg = 0; gg < 4; ++gg) {
              const lf32x4 y = mfma4(g == gg ? x : 0.f, pp[0][0][e], lf32x4{0.f, 0.f, 0.f, 0.f});
              if (4 * gg + e <= m) acc[v][0] += y;
            }
          }
        }
      }
    }
  }

  // the lane holds values 16 v + 4 g .. + 3 of its tokens
  T* op = reinterpret_cast<T*>(a.o) + (row0 * a.Hv + h) * V;
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int t = t0 + 16 * j + m;
    if (t < n) {
#pragma unroll
      for (int v = 0; v < V / 16; ++v) {
        T* dst = op + (size_t)t * a.Hv * V + 16 * v + 4 * g;
        if constexpr (C::ES == 2)
          *reinterpret_cast<uint2*>(dst) =
              make_uint2(pack_bf16x2(acc[v][j][0], acc[v][j][1]), pack_bf16x2(acc[v][j][2], acc[v][j][3]));
        else
          *reinterpret_cast<lf32x4*>(dst) = acc[v][j];
      }
    }
  }
}

// ------------------------------------------------------------------------------------------- bf16: a walk over chunks
//
// A workgroup walks the 64-token chunks of one segment of a sequence for NH value heads that share a key head (NH V = 64 or
// 128 value columns, 32 a wave). A wave keeps its 32 value rows of S in registers, as transposed tiles [2][K / 16] (D: key
// 32 (kt / 2) + 8 g + 4 (kt % 2) + e; value of lane m and half u: 8 (m / 4) + 4 u + m % 4): a pair of key tiles, split into
// bf16 terms, is an MFMA operand with its keys in memory order, and both halves' rows of an output tile are 8 neighbours.
// A chunk:
//   P^T [s, t] = K Q^T, scaled by exp(G_t - G_s) and masked, a few tiles a wave, as two bf16 terms into LDS for all;
//   O^T [v, t] = exp(G_t) S Q^T + V^T P^T;
//   S^T = exp(G_end) S^T + K^T V', V' = exp(G_end - G_s) V in three bf16 terms.
// V^T and K^T are read transposed from LDS. A chunk's 200 MFMAs a wave (16 cycles each) and 700 other vector instructions
// (4 each) take turns unless they are interleaved: the splits into terms run beside the products of the step before, and
// two workgroups share a CU. OUT false: the state alone.

template <int K, int V, int NH, bool OUT>
struct WalkCfg {
  static constexpr int WH = V / 32, NW = NH * WH;  // waves a head, in all
  static constexpr int KB = 2 * K, VB = 2 * NH * V;  // bytes of a row
  static constexpr int KI = CH * KB / 1024 / NW, VI = CH * VB / 1024 / NW;  // a wave's load instructions for k (q) and v
  static constexpr int P_TERM = OUT ? 6 * 1024 : 0;  // 16 x 32 blocks of P in fragment order: t tiles 0, 1 one, 2, 3 two
  static constexpr int GC = WH;  // chunks whose decays are formed at a time, each by a wave a head
  static constexpr int G_FLOATS = 3 * CH + 4, G_BYTES = (GC + 1) * NH * G_FLOATS * 4;
  static constexpr int VS = OUT ? 1 : 2;  // stages of v (and q)
  static constexpr int REST = VS * CH * VB + (OUT ? CH * KB : 0) + NH * 2 * P_TERM + G_BYTES;
  static constexpr int KS = REST + 2 * CH * KB <= 80 * 1024 ? 2 : 1;  // stages of k
  static constexpr int AT_V = KS * CH * KB, AT_Q = AT_V + VS * CH * VB;
  static constexpr int AT_P = AT_Q + (OUT ? CH * KB : 0);
  static constexpr int AT_G = AT_P + NH * 2 * P_TERM;
  static constexpr int LDS = AT_G + G_BYTES;
  static_assert(LDS <= 80 * 1024 && (OUT || KS == 2), "two workgroups a CU");
  // P's tiles (s tile i, t tile j, i <= j) by wave of the head, 4 i + j each, a nibble a tile: those of a wave share rows
  static constexpr uint32_t tiles(int w) {
    return WH == 4 ? (w == 0 ? 0x73 : w == 1 ? 0xFB : w == 2 ? 0xA62 : 0x051) : (w == 0 ? 0xFB73 : 0x051A62);
  }
  static constexpr int count(int w) { return WH == 4 ? (w < 2 ? 2 : 3) : (w == 0 ? 4 : 6); }
};

template <int N>
__device__ __forceinline__ void wait_loads() {  // at most N of the wave's loads outstanding, then a barrier
  static_assert(N < 64, "counter");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

__device__ __forceinline__ int walk_row(int u, int m) { return 8 * (m >> 2) + 4 * u + (m & 3); }

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

template <int K, int V, int NH, bool OUT>
__global__ __launch_bounds__((64 * WalkCfg<K, V, NH, OUT>::NW), 2) void lin_walk_kernel(LinArgs a) {
  using C = WalkCfg<K, V, NH, OUT>;
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
  auto rows_of = [&](int c) { return max(0, min(CH, n - c * CH)); };  // (behind the last chunk: none, zeros)
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
    if constexpr (OUT) {
      const float s = prefix_sum(g_value(a, x.up));
      b[l] = s;
      b[CH + l] = a.scale * expf(s);
    }
    const float s = prefix_sum(g_value(a, x.down)), total = __shfl(s, 63);
    b[2 * CH + 63 - l] = expf(dpp_rows<0x138, 0xF>(s));
    // S exp(G) as S + S expm1(G): of a slow decay the factor's own rounding, the same at every chunk, would grow with the
    // length of the memory; of a fast one what is left is off by 2^-25 of what was
    if (l == 0) *reinterpret_cast<float2*>(b + 3 * CH) = make_float2(expm1f(total), total);
  };

  const size_t hs = (size_t)V * K;
  lf32x4 acc[2][KT];
  // a state [V][K] of the head in memory: the lane's tiles are 4 floats each, pairs of them 8
  const size_t lane_at = (size_t)(32 * wl + walk_row(0, m)) * K + 8 * g;
  auto state_at = [&](int u, int kt) { return lane_at + 4 * u * K + 32 * (kt >> 1) + 4 * (kt & 1); };
  auto put = [&](float* dst) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) *reinterpret_cast<lf32x4*>(dst + state_at(u, kt)) = acc[u][kt];
  };

  G2 gv = g_load(wl);
  issue_k(0);
  if constexpr (OUT) issue_q(0);
  issue_v(0);
#pragma unroll
  for (int u = 0; u < 2; ++u)
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
      for (int u = 0; u < 2; ++u)
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
      wait_loads<2 * KT>();
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
    lf32x4 o[2][4];
    lbf16x8 vf[2][2];  // the wave's columns of V^T: [half][block of 32 tokens]
    auto read_v = [&] {
      const int r = 4 * g + (m >> 2), col = (hh * V + 32 * wl) / 8 + (m & 3);
      const uint8_t* at = vs + chunk_at<C::VB>(r, col);
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint2 x = lds_tr(at + 32 * s * C::VB + 8 * u), y = lds_tr(at + (32 * s + 16) * C::VB + 8 * u);
          vf[u][s] = __builtin_bit_cast(lbf16x8, make_uint4(x.x, x.y, y.x, y.y));
        }
    };
    // V' in terms, a pair of tokens at a time: word i of half u in block s
    uint32_t vt[2][2][NT][4];  // [block][half][term][word]
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
    static_assert(!OUT || (C::KI + C::VI <= 2 * KK * NT && 4 * KK % C::KI == 0), "regions for the loads");
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
          const lf32x4 gs = *reinterpret_cast<const lf32x4*>(b + 16 * i + 4 * g);
          const float gt = b[16 * j + m];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            d[x][e] *= a.scale * __expf(gt - gs[e]);
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
      if (wl == 0)
        p_tiles(std::integral_constant<int, 0>{});
      else if (wl == 1)
        p_tiles(std::integral_constant<int, 1>{});
      else if constexpr (WH == 4) {
        if (wl == 2)
          p_tiles(std::integral_constant<int, 2>{});
        else
          p_tiles(std::integral_constant<int, 3>{});
      }
      // O^T = S Q^T, the state in two terms; beside each step's products the next one's terms and V's of the first block
      uint32_t st[2][2][2][4];  // [step % 2][half][term][word]
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
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[u][j] = lf32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) s_pair(0, u, i);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        fence();
        if (kk + 1 < KK) q_read(kk + 1);
#pragma unroll
        for (int r = 0; r < 4; ++r) {  // term 1 - r / 2 of half r % 2
          fence();
          const int x = 1 - (r >> 1), u = r & 1;
          const lbf16x8 sf = __builtin_bit_cast(lbf16x8, make_uint4(st[kk & 1][u][x][0], st[kk & 1][u][x][1], st[kk & 1][u][x][2], st[kk & 1][u][x][3]));
#pragma unroll
          for (int j = 0; j < 4; ++j) o[u][j] = mfma16(sf, qf[kk & 1][j], o[u][j]);
          if (kk + 1 < KK) {
            s_pair(kk + 1, r >> 1, 2 * (r & 1));
            s_pair(kk + 1, r >> 1, 2 * (r & 1) + 1);
          }
          // (the 8 pairs of V' over the 4 KK regions)
          if constexpr (KK == 4) {
            if ((r & 1) == 0) v_pair(0, kk >> 1, 2 * (kk & 1) + (r >> 1));
          } else {
            v_pair(0, kk, r);
          }
          if constexpr (C::KS == 2) {  // the next k's loads, one at a time
            constexpr int every = 4 * KK / C::KI;
            if ((4 * kk + r) % every == 0) issue_k(c + 1, (4 * kk + r) / every, (4 * kk + r) / every + 1);
          }
          interleave<4, 5>();
        }
      }
      fence();
      // (formed here, although only the update needs them)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int k = 0; k < NT; ++k)
          asm volatile("" : "+v"(vt[0][u][k][0]), "+v"(vt[0][u][k][1]), "+v"(vt[0][u][k][2]), "+v"(vt[0][u][k][3]));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float f = b[CH + 16 * j + m];
#pragma unroll
        for (int u = 0; u < 2; ++u) o[u][j] *= f;
      }
      typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
      u16x2 top = {0, 0};  // the largest magnitude's bits
#pragma unroll
      for (int u = 0; u < 2; ++u)
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
            for (int u = 0; u < 2; ++u) o[u][j] = mfma16(vf[u][s], pf[s][j][x], o[u][j]);
          fence();
        };
        p_read(0);
        pv(0, 1);  // (the small terms first)
        p_read(1);
        pv(0, 0);
        pv(1, 1);
        pv(1, 0);
      } else {
        // an infinity or a NaN among the values: a masked P is zero, and zero times it NaN. Token by token, each added
        // from its own row on
#pragma unroll
        for (int u = 0; u < 2; ++u)
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
      // the lane holds values 8 g .. 8 g + 7 of the wave's, of token 16 j + m (rows behind the segment are dropped)
      const uint32_t lb = (uint32_t)a.Hv * V * 2u;
      const Rsrc rs = raw_rsrc(reinterpret_cast<uint16_t*>(a.o) + ((row0 + (size_t)c * CH) * a.Hv + h) * V,
                               (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(rows_of(c) - 1) * lb + 2 * V)));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const lu32x4 w = {pack_bf16x2(o[0][j][0], o[0][j][1]), pack_bf16x2(o[0][j][2], o[0][j][3]),
                          pack_bf16x2(o[1][j][0], o[1][j][1]), pack_bf16x2(o[1][j][2], o[1][j][3])};
        __builtin_amdgcn_raw_buffer_store_b128(w, rs, (uint32_t)(16 * j + m) * lb + 2 * (32 * wl + 8 * g), 0, 0);
      }
    } else {
      read_v();
      read_weights(0);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) v_pair(0, u, i);
    }
    if (OUT && c + 1 == chunks && !keep) return;
    // S^T = exp(G_end) S^T + K^T V', a pair of key tiles at a time: beside the first block's products the decay of the next
    // pair and V' of the second block
    gsum += b[3 * CH + 1];
    const float add = b[3 * CH];
    read_weights(1);
    lbf16x8 kf[2][2];  // [step % 2][tile of the pair]
    auto k_read = [&](int x) {  // of step x: pair x % KK of block x / KK
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint8_t* at = ks + 32 * (x / KK) * C::KB + flip(at_tr, 4 * (x % KK)) + 8 * i;
        const uint2 y = lds_tr(at), z = lds_tr(at + 16 * C::KB);
        kf[x & 1][i] = __builtin_bit_cast(lbf16x8, make_uint4(y.x, y.y, z.x, z.y));
      }
    };
    auto decay = [&](int kk, int u) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[u][2 * kk + i][e] = fmaf(acc[u][2 * kk + i][e], add, acc[u][2 * kk + i][e]);
    };
    fence();
    k_read(0);
    decay(0, 0);
    decay(0, 1);
#pragma unroll
    for (int x = 0; x < 2 * KK; ++x) {
      const int s = x / KK, kk = x % KK;
      fence();
      if (x + 1 < 2 * KK) k_read(x + 1);
#pragma unroll
      for (int t = NT - 1; t >= 0; --t) {  // (the small terms first)
        fence();
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const lbf16x8 vfr = v_frag(s, u, t);
#pragma unroll
          for (int i = 0; i < 2; ++i) acc[u][2 * kk + i] = mfma16(kf[x & 1][i], vfr, acc[u][2 * kk + i]);
        }
        if constexpr (OUT) {  // the next q's and v's loads, one at a time
          const int i = x * NT + NT - 1 - t;
          if (i < C::KI)
            issue_q(c + 1, i, i + 1);
          else if (i < C::KI + C::VI)
            issue_v(c + 1, i - C::KI, i - C::KI + 1);
        }
        if (s == 0) {
          if (kk + 1 < KK && t < 2) decay(kk + 1, t);
          // (the 8 pairs of V' over the NT KK regions)
          if constexpr (KK == 4) {
            if (t < 2) v_pair(1, kk >> 1, 2 * (kk & 1) + t);
          } else {
            v_pair(1, kk, t);
            if (t < 4 - NT) v_pair(1, kk, NT + t);
          }
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

// The states before a sequence's runs, in place of what the runs add: c_0 the initial state, c_{j+1} = exp(G_j) c_j + E_j.
// A thread keeps 4 elements, 8 runs loaded ahead.
__global__ __launch_bounds__(256) void lin_join_kernel(LinArgs a, int hs) {
  const int per = hs / 1024, unit = blockIdx.x / per, part = blockIdx.x % per;
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

constexpr int STATE_NW = 4;  // waves (of 16 value rows) a workgroup of the state pass

struct Plan {
  int seg, run, seg_slots, run_slots, single;
  size_t ckpt, gcum, ends, gtot, total;  // offsets into the workspace, its size
};

// Value heads that a workgroup of the bf16 walk takes together: two of 64 columns where they share a key head.
int walk_heads(int Hk, int Hv, int V) { return V == 64 && Hv / Hk % 2 == 0 ? 2 : 1; }

Plan make_plan(bool packed, int N, int T, int Hk, int Hv, int K, int V, int dtype) {
  Plan p;
  const bool walk = dtype == ZGDN_BF16;
  auto slots = [&](long size) {  // at most: a packed batch's sequences are not known here
    return (int)(packed ? T / size + N : N * std::max(1L, (T + size - 1) / size));
  };
  if (walk) {
    // Segments of a CU's share of the chunks. Half as long, two to a CU, costs 7 us at 4096 tokens of 16 heads of 128 x 128
    // (states 12 us in the join instead of 7, 17 instead of 15 in the state pass, against 1 us less in the outputs) and
    // gains 2 at 32768. Sequences that fill the CUs uncut are not cut below 1.5 shares: 32 of 64 .. 2048 tokens, 16 heads,
    // take 180 us so, and 203 cut to 16 chunks (33 in the state pass and 13 in the join against 14 less in the outputs).
    const long rows = packed ? T : (long)N * T, groups = Hv / walk_heads(Hk, Hv, V);
    const long share = (rows * groups + CUS * CH - 1) / (CUS * CH);
    const long seg = std::max(1L, N * groups >= CUS ? share + share / 2 : share) * CH;
    p.seg = (int)std::min(seg, (long)INT32_MAX / 4);
    p.run = p.seg;
  } else {
    p.seg = 64;
    const int vg = V / (16 * STATE_NW);
    p.run = (int)std::min((long)INT32_MAX / 128 * 64, std::max(1L, (T + 63L) / 64) * 64);
    while (p.run > 4 * p.seg && (long)slots(p.run) * Hv * vg < 256) p.run = (p.run / p.seg + 1) / 2 * p.seg;
  }
  p.run_slots = slots(p.run);
  p.seg_slots = slots(p.seg);
  p.single = T <= p.run;
  const bool cut = !walk;
  const size_t hs = (size_t)K * V * 4;
  auto round = [](size_t x) { return (x + 255) / 256 * 256; };
  p.ckpt = 0;
  p.gcum = p.ckpt + (cut ? (size_t)p.seg_slots * Hv * hs : 0);
  p.ends = p.gcum + (cut ? round((size_t)p.seg_slots * Hv * 4) : 0);
  p.gtot = p.ends + (p.single ? 0 : (size_t)p.run_slots * Hv * hs);
  p.total = p.gtot + (p.single ? 0 : round((size_t)p.run_slots * Hv * 4));
  return p;
}

bool sizes_ok(int Hk, int Hv, int K, int V, int dtype) {
  return Hk >= 1 && Hv >= 1 && Hv % Hk == 0 && (K == 64 || K == 128) && (V == 64 || V == 128) &&
         (dtype == ZGDN_F32 || dtype == ZGDN_BF16);
}

template <int K, int V, int NH>
int launch_walk(const char* fn, const LinArgs& a, const Plan& p, hipStream_t s) {
  using CO = WalkCfg<K, V, NH, true>;
  using CS = WalkCfg<K, V, NH, false>;
  static std::atomic<signed char> so[64], ss[64];
  if (!lds_ready(lin_walk_kernel<K, V, NH, true>, CO::LDS, so) || !lds_ready(lin_walk_kernel<K, V, NH, false>, CS::LDS, ss))
    return fail(ZGDN_EHIP, "%s: the device refused the LDS", fn);
  const int groups = a.Hv / NH;
  const int before_last = a.cu != nullptr ? a.T / a.run : a.N * ((a.T + a.run - 1) / a.run - 1);  // segments, at most
  if (!p.single)
    hipLaunchKernelGGL((lin_walk_kernel<K, V, NH, false>), dim3((unsigned)(before_last * groups)), dim3(64 * CS::NW), CS::LDS, s, a);
  if (!p.single)
    hipLaunchKernelGGL(lin_join_kernel, dim3((unsigned)(a.N * a.Hv * (V * K / 1024))), dim3(256), 0, s, a, V * K);
  hipLaunchKernelGGL((lin_walk_kernel<K, V, NH, true>), dim3((unsigned)(p.seg_slots * groups)), dim3(64 * CO::NW), CO::LDS, s, a);
  return ZGDN_OK;
}

template <int K, int V>
int launch_bf16(const char* fn, const LinArgs& a, const Plan& p, hipStream_t s) {
  if constexpr (V == 64) {
    if (walk_heads(a.Hk, a.Hv, V) == 2) return launch_walk<K, V, 2>(fn, a, p, s);
  }
  return launch_walk<K, V, 1>(fn, a, p, s);
}

template <int K, int V>
int launch_f32(const char* fn, const LinArgs& a, const Plan& p, hipStream_t s) {
  constexpr int NW = STATE_NW, VG = V / (16 * NW);
  using CS = StateCfg<float, K, V, NW>;
  using CO = OutCfg<float, K, V, 64>;
  static std::atomic<signed char> so[64], ss[64];
  if (!lds_ready(lin_out_kernel<float, K, V, 64>, CO::LDS, so) || !lds_ready(lin_state_kernel<float, K, V, NW>, CS::LDS, ss))
    return fail(ZGDN_EHIP, "%s: the device refused the LDS", fn);
  if (a.s_out != nullptr || a.T > p.seg) {
    const int units = p.run_slots * a.Hv;
    hipLaunchKernelGGL((lin_state_kernel<float, K, V, NW>), dim3((unsigned)((units + 7) / 8 * 8 * VG)), dim3(64 * NW), CS::LDS, s, a);
  }
  if (!p.single)
    hipLaunchKernelGGL(lin_carry_kernel, dim3((unsigned)(a.N * a.Hv * (V * K / 1024))), dim3(256), 0, s, a, V * K);
  if (a.T > 0)
    hipLaunchKernelGGL((lin_out_kernel<float, K, V, 64>), dim3((unsigned)(a.seg_slots * a.Hv)), dim3(64 * CO::NW), CO::LDS, s, a);
  return ZGDN_OK;
}

template <int K, int V>
int launch_all(const char* fn, const LinArgs& a, const Plan& p, int dtype, hipStream_t s) {
  return dtype == ZGDN_F32 ? launch_f32<K, V>(fn, a, p, s) : launch_bf16<K, V>(fn, a, p, s);
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
  if ((long)p.seg_slots * Hv > INT32_MAX / 16) return fail(ZGDN_EUNSUPPORTED, "%s: %d segments of %d heads", fn, p.seg_slots, Hv);
  if (workspace_bytes < p.total || (workspace == nullptr && p.total > 0))
    return fail(ZGDN_EINVAL, "%s: workspace of %zu bytes, %zu needed", fn, workspace_bytes, p.total);
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  LinArgs a{};
  a.q = q, a.k = k, a.v = v, a.g = g;
  a.q_ld = q_ld, a.k_ld = k_ld, a.v_ld = v_ld, a.g_ld = g_ld;
  a.g_bf16 = g_dtype == ZGDN_BF16;
  a.s_in = initial_state, a.s_out = final_state, a.o = o, a.cu = cu_seqlens;
  a.N = N, a.T = T, a.Hk = Hk, a.Hv = Hv, a.scale = scale;
  a.seg = p.seg, a.run = p.run, a.seg_slots = p.seg_slots, a.run_slots = p.run_slots;
  a.direct = p.single;
  a.save_first = initial_state != nullptr && initial_state == final_state;
  a.ckpt = (float*)(ws + p.ckpt), a.gcum = (float*)(ws + p.gcum), a.ends = (float*)(ws + p.ends), a.gtot = (float*)(ws + p.gtot);
  hipStream_t hs = (hipStream_t)stream;
  const int st = K == 128 ? (V == 128 ? launch_all<128, 128>(fn, a, p, dtype, hs) : launch_all<128, 64>(fn, a, p, dtype, hs))
                          : (V == 128 ? launch_all<64, 128>(fn, a, p, dtype, hs) : launch_all<64, 64>(fn, a, p, dtype, hs));
  return st != ZGDN_OK ? st : check_launch(fn);
}
