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
constexpr float G_MIN = -200.f;

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
// NW waves; each wave instruction fills 1 KiB, so a lane fetches the chunk that belongs at its place.
template <int ROWB, int ROWS, int NW>
__device__ __forceinline__ void load_rows(const void* base, uint32_t ld_bytes, int rows, uint8_t* lds, int wave) {
  constexpr int RP = 1024 / ROWB, P = ROWS / RP;  // rows a piece, pieces
  static_assert(ROWS % RP == 0 && P % NW == 0, "whole pieces, as many a wave");
  const uint32_t bytes = rows > 0 ? (uint32_t)(rows - 1) * ld_bytes + ROWB : 0u;
  const uint64_t at = (uint64_t)(uintptr_t)base;
  const lu32x4 rs = {(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)at),
                     (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(at >> 32) & 0xffffu)),
                     (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
  const int l = threadIdx.x & 63;
  constexpr int n = ROWB / 16;
#pragma unroll
  for (int p0 = 0; p0 < P; p0 += NW) {
    const int p = p0 + wave;
    const int r = p * RP + l / n, c = l % n;
    load_lds(rs, (uint32_t)r * ld_bytes + (uint32_t)(chunk_at<ROWB>(r, c) - r * ROWB), lds + 1024 * p);
  }
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
// A workgroup walks the 64-token chunks of one piece of a sequence for NH value heads that share a key head (NH V = 64 or
// 128 value columns, 32 a wave). A wave keeps its 32 value rows of S in registers, as transposed tiles [2][K / 16] (D: key
// 4 g + e; value of lane m and half u: 8 (m / 4) + 4 u + m % 4, so that both halves' rows of an output tile are 8
// neighbours), which as they stand are an MFMA operand once split into bf16 terms. A chunk:
//   P^T [s, t] = K Q^T, scaled by exp(G_t - G_s) and masked, a few tiles a wave, as two bf16 terms into LDS for all;
//   O^T [v, t] = exp(G_t) S Q^T + V^T P^T;
//   S^T = exp(G_end) S^T + K^T V', V' = exp(G_end - G_s) V in three bf16 terms.
// V^T and K^T are read transposed from LDS. The phases of one workgroup leave each of matrix unit, vector unit and LDS idle
// in turn: two workgroups run on a CU. OUT false: the state alone.

constexpr int CH = 64;  // tokens of a chunk

template <int K, int V, int NH, bool OUT>
struct WalkCfg {
  static constexpr int WH = V / 32, NW = NH * WH;  // waves a head, in all
  static constexpr int KB = 2 * K, VB = 2 * NH * V;  // bytes of a row
  static constexpr int KV_BYTES = CH * (KB + VB);
  static constexpr int NS = OUT ? 1 : 2;  // stages of k and v
  static constexpr int AT_Q = NS * KV_BYTES;
  static constexpr int P_TERM = OUT ? 6 * 1024 : 0;  // 16 x 32 blocks of P in fragment order: t tiles 0, 1 one, 2, 3 two
  static constexpr int AT_P = AT_Q + (OUT ? CH * KB : 0);
  static constexpr int GC = WH;  // chunks whose decays are formed at a time, each by a wave a head
  static constexpr int G_FLOATS = 3 * CH + 4;
  static constexpr int AT_G = AT_P + NH * 2 * P_TERM;
  static constexpr int LDS = AT_G + 2 * GC * NH * G_FLOATS * 4;
  static_assert(LDS <= 80 * 1024, "two workgroups a CU");
};

template <int K>
__device__ __forceinline__ int walk_row(int u, int m) { return 8 * (m >> 2) + 4 * u + (m & 3); }

// Fragment of V's transpose: the values of half u (of 32 columns from c0) in rows r0 + 4 g + {0..3}, r0 + 16 + 4 g + {0..3}.
template <int ROWB>
__device__ __forceinline__ lbf16x8 tr_frag_half(const uint8_t* tile, int r0, int c0, int u) {
  const int l = threadIdx.x & 63, g = l >> 4, s = l & 15;
  const int r = r0 + 4 * g + (s >> 2), c = c0 / 8 + (s & 3);
  const uint2 a = lds_tr(tile + chunk_at<ROWB>(r, c) + 8 * u);
  const uint2 b = lds_tr(tile + chunk_at<ROWB>(r + 16, c) + 8 * u);
  return __builtin_bit_cast(lbf16x8, make_uint4(a.x, a.y, b.x, b.y));
}

template <int K, int V, int NH, bool OUT>
__global__ __launch_bounds__((64 * WalkCfg<K, V, NH, OUT>::NW), 2) void lin_walk_kernel(LinArgs a) {
  using C = WalkCfg<K, V, NH, OUT>;
  constexpr int NW = C::NW, WH = C::WH, KT = K / 16;
  extern __shared__ uint4 lin_lds[];
  uint8_t* lds = reinterpret_cast<uint8_t*>(lin_lds);
  const int groups = a.Hv / NH;
  const int slot = blockIdx.x / groups, h0 = (blockIdx.x - slot * groups) * NH;
  const int size = OUT ? a.seg : a.run;
  Piece p;
  if (!find_piece(a.cu, a.N, a.T, slot, size, OUT ? a.run : a.seg, p)) return;
  uniform(p);
  const int first = p.j * size;
  const bool last = first + size >= p.len;
  int n = min(size, p.len - first);  // (0 for an empty sequence)
  if (!OUT && last) {  // a last run is walked up to its last segment (which has the final state in its outputs' walk)
    n = max(n - 1, 0) / a.seg * a.seg;
    if (n == 0) return;
  }
  const int wave = wave_id(), l = threadIdx.x & 63, g = l >> 4, m = l & 15;
  const int hh = wave / WH, wl = wave - hh * WH, h = h0 + hh;
  const size_t row0 = (size_t)p.bos + first;
  const size_t hk = (size_t)(h0 / (a.Hv / a.Hk)) * K;
  const uint16_t* qp = reinterpret_cast<const uint16_t*>(a.q) + row0 * a.q_ld + hk;
  const uint16_t* kp = reinterpret_cast<const uint16_t*>(a.k) + row0 * a.k_ld + hk;
  const uint16_t* vp = reinterpret_cast<const uint16_t*>(a.v) + row0 * a.v_ld + (size_t)h0 * V;
  float* gb = reinterpret_cast<float*>(lds + C::AT_G) + hh * C::G_FLOATS;  // + NH G_FLOATS a chunk, of 2 GC in turn
  uint8_t* pl = lds + C::AT_P + hh * 2 * C::P_TERM + 16 * l;
  const uint8_t* qs = lds + C::AT_Q;

  const int chunks = (n + CH - 1) / CH;
  auto rows_of = [&](int c) { return max(0, min(CH, n - c * CH)); };  // (behind the last chunk: none, zeros)
  auto issue_kv = [&](int c) {
    uint8_t* at = lds + (C::NS == 2 ? (c & 1) * C::KV_BYTES : 0);
    const int rows = rows_of(c);
    const size_t t = rows > 0 ? (size_t)c * CH : 0;
    load_rows<C::KB, CH, NW>(kp + t * a.k_ld, (uint32_t)a.k_ld * 2u, rows, at, wave);
    load_rows<C::VB, CH, NW>(vp + t * a.v_ld, (uint32_t)a.v_ld * 2u, rows, at + CH * C::KB, wave);
  };
  auto issue_q = [&](int c) {
    const int rows = rows_of(c);
    load_rows<C::KB, CH, NW>(qp + (rows > 0 ? (size_t)c * CH : 0) * a.q_ld, (uint32_t)a.q_ld * 2u, rows, lds + C::AT_Q, wave);
  };
  // Log decays, GC chunks at a time, one of them a wave: lane l takes the chunk's tokens l (prefix sums) and 63 - l (suffix
  // sums: lanes in token order from the end).
  auto g_at = [&](int c) { return gb + (c & (2 * C::GC - 1)) * NH * C::G_FLOATS; };
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
    const Decay d = decay_of(total);
    if (l == 0) *reinterpret_cast<float4*>(b + 3 * CH) = make_float4(d.add, d.mul, total, 0.f);
  };

  const size_t hs = (size_t)V * K;
  lf32x4 acc[2][KT];
  auto put = [&](float* dst) {  // [V][K] of the head
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
        *reinterpret_cast<lf32x4*>(dst + (size_t)(32 * wl + walk_row<K>(u, m)) * K + 16 * kt + 4 * g) = acc[u][kt];
  };
  auto add_in = [&](const float* src, float f) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        const lf32x4 x = *reinterpret_cast<const lf32x4*>(src + (size_t)(32 * wl + walk_row<K>(u, m)) * K + 16 * kt + 4 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[u][kt][e] = fmaf(x[e], f, acc[u][kt][e]);
      }
  };

  float gsum = 0.f;
  auto write_down = [&](int c) {  // the state before the segment that starts with chunk c of the run
    const int at = p.other0 + (first + c * CH) / a.seg;
    if (c == 0 && !(p.j == 0 && p.len <= a.run && a.save_first)) return;
    if (at >= a.seg_slots) return;  // (only tables whose sequences overlap have so many segments)
    put(a.ckpt + ((size_t)at * a.Hv + h) * hs);
    if (wl == 0 && l == 0) a.gcum[(size_t)at * a.Hv + h] = gsum;
  };

  G2 gv = g_load(wl);
  if constexpr (OUT) issue_q(0);
  issue_kv(0);
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) acc[u][kt] = lf32x4{0.f, 0.f, 0.f, 0.f};
  if constexpr (OUT) {
    // the state before the segment: in a sequence of one run the initial state or what the run's walk wrote down, else the
    // state carried into the run, decayed, and what the run's walk wrote down
    const int run = first / a.run, in_run = first - run * a.run;
    const size_t at = ((size_t)slot * a.Hv + h) * hs;
    if (p.len <= a.run) {
      if (in_run > 0 || (a.save_first && !last))
        add_in(a.ckpt + at, 1.f);
      else if (a.s_in != nullptr)
        add_in(a.s_in + ((size_t)p.seq * a.Hv + h) * hs, 1.f);
    } else {
      if (in_run > 0) add_in(a.ckpt + at, 1.f);
      if (p.other0 + run < a.run_slots)
        add_in(a.ends + ((size_t)(p.other0 + run) * a.Hv + h) * hs, in_run > 0 ? expf(a.gcum[(size_t)slot * a.Hv + h]) : 1.f);
    }
    // P's tiles above its diagonal blocks of 32 stay zero
    for (int e = wl; e < 2 * C::P_TERM / 1024; e += WH) *reinterpret_cast<uint4*>(pl + 1024 * e) = make_uint4(0, 0, 0, 0);
  } else if (p.len <= a.run && a.s_in != nullptr) {
    add_in(a.s_in + ((size_t)p.seq * a.Hv + h) * hs, 1.f);
  }
  g_store(wl, gv);

  // Offsets of the lane's 16-byte chunks in rows of KB bytes: chunk c of the rows of one place mod 16 lies at the offset of
  // chunk 0 with c's bits flipped. Formed anew each chunk (held, all of them would take 40 registers).
  int at_row = chunk_at<C::KB>(m, g);                                             // row m, chunk g
  int at_half = chunk_at<C::KB>(m, g >> 1) + 8 * (g & 1);                         // row m, 8 bytes at 8 g
  int at_tr = chunk_at<C::KB>(4 * g + (m >> 2), (m & 3) >> 1) + 8 * (m & 1);      // transposing reads, column 0
  auto flip = [](int at, int c) { return at ^ (c << 4); };

  for (int c = 0; c < chunks; ++c) {
    asm volatile("" : "+v"(at_row), "+v"(at_half), "+v"(at_tr));
    loads_barrier();  // chunk c is there, and nobody reads what the next loads overwrite
    const int in_group = c & (C::GC - 1);
    if (in_group == 0 && c + C::GC < chunks) gv = g_load(c + C::GC + wl);
    if constexpr (!OUT) issue_kv(c + 1);
    const uint8_t* ks = lds + (C::NS == 2 ? (c & 1) * C::KV_BYTES : 0);
    const uint8_t* vs = ks + CH * C::KB;
    const float* b = g_at(c);
    lf32x4 o[2][4];
    if constexpr (OUT) {
      // P^T tiles (s tile i, t tile j, i <= j), in the order 00 01 11 02 12 22 ...
      constexpr uint64_t TILES = 0xFB73A62510;  // 4 i + j of tile w in its bits 4 w ..
#pragma unroll
      for (int x = 0; x < (10 + WH - 1) / WH; ++x) {
        const int w = wl + x * WH;
        if (w < 10) {
          const int ij = (int)(TILES >> (4 * w)) & 15, i = ij >> 2, j = ij & 3;
          lf32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int kk = 0; kk < K / 32; ++kk) {
            const lbf16x8 kf = *reinterpret_cast<const lbf16x8*>(ks + 16 * i * C::KB + flip(at_row, 4 * kk));
            const lbf16x8 qf = *reinterpret_cast<const lbf16x8*>(qs + 16 * j * C::KB + flip(at_row, 4 * kk));
            d = mfma16(kf, qf, d);
          }
          const lf32x4 gs = *reinterpret_cast<const lf32x4*>(b + 16 * i + 4 * g);
          const float gt = b[16 * j + m];
#pragma unroll
          for (int e = 0; e < 4; ++e) d[e] *= a.scale * __expf(gt - gs[e]);
          if (i == j) {
#pragma unroll
            for (int e = 0; e < 4; ++e) d[e] = 4 * g + e <= m ? d[e] : 0.f;
          }
          uint32_t w0[2], w1[2];
          split_pair<2>(d[0], d[1], w0);
          split_pair<2>(d[2], d[3], w1);
          // the block of tile j and tokens 32 (i / 2) .. in fragment order: this very lane's, half i % 2
          const int at = 1024 * (j < 2 ? j : 2 * j - 2 + (i >> 1)) + 8 * (i & 1);
          *reinterpret_cast<uint2*>(pl + at) = make_uint2(w0[0], w1[0]);
          *reinterpret_cast<uint2*>(pl + C::P_TERM + at) = make_uint2(w0[1], w1[1]);
        }
      }
      // O^T = S Q^T, the state in two terms, keys in the order of its tiles
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[u][j] = lf32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < K / 32; ++kk) {
        lbf16x8 sf[2][2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint32_t t[4][2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            split_pair<2>(acc[u][2 * kk + i][0], acc[u][2 * kk + i][1], t[2 * i]);
            split_pair<2>(acc[u][2 * kk + i][2], acc[u][2 * kk + i][3], t[2 * i + 1]);
          }
#pragma unroll
          for (int x = 0; x < 2; ++x) sf[u][x] = __builtin_bit_cast(lbf16x8, make_uint4(t[0][x], t[1][x], t[2][x], t[3][x]));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint2 q0 = *reinterpret_cast<const uint2*>(qs + 16 * j * C::KB + flip(at_half, 4 * kk));
          const uint2 q1 = *reinterpret_cast<const uint2*>(qs + 16 * j * C::KB + flip(at_half, 4 * kk + 2));
          const lbf16x8 qf = __builtin_bit_cast(lbf16x8, make_uint4(q0.x, q0.y, q1.x, q1.y));
#pragma unroll
          for (int u = 0; u < 2; ++u) o[u][j] = mfma16(sf[u][1], qf, o[u][j]);
#pragma unroll
          for (int u = 0; u < 2; ++u) o[u][j] = mfma16(sf[u][0], qf, o[u][j]);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float f = b[CH + 16 * j + m];
#pragma unroll
        for (int u = 0; u < 2; ++u) o[u][j] *= f;
      }
      lds_barrier();  // P is there, and nobody reads q any more
      issue_q(c + 1);
    }
    lbf16x8 vf[2][2];  // [half][block of 32 tokens]
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int s = 0; s < 2; ++s) vf[u][s] = tr_frag_half<C::VB>(vs, 32 * s, hh * V + 32 * wl, u);
    if constexpr (OUT) {
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
      auto p_frag = [&](int j, int s, int term) {
        return *reinterpret_cast<const lbf16x8*>(pl + term * C::P_TERM + 1024 * (j < 2 ? j : 2 * j - 2 + s));
      };
      if (__ballot(top.x >= 0x7f80 || top.y >= 0x7f80) == 0) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int j = 2 * s; j < 4; ++j) {
            const lbf16x8 lo = p_frag(j, s, 1), hi = p_frag(j, s, 0);
#pragma unroll
            for (int u = 0; u < 2; ++u) o[u][j] = mfma16(vf[u][s], lo, o[u][j]);
#pragma unroll
            for (int u = 0; u < 2; ++u) o[u][j] = mfma16(vf[u][s], hi, o[u][j]);
          }
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
      // the lane holds values 8 g .. 8 g + 7 of the wave's, of token 16 j + m (rows behind the piece are dropped)
      const uint32_t lb = (uint32_t)a.Hv * V * 2u;
      const Rsrc rs = raw_rsrc(reinterpret_cast<uint16_t*>(a.o) + ((row0 + (size_t)c * CH) * a.Hv + h) * V,
                               (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(rows_of(c) - 1) * lb + 2 * V)));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const lu32x4 w = {pack_bf16x2(o[0][j][0], o[0][j][1]), pack_bf16x2(o[0][j][2], o[0][j][3]),
                          pack_bf16x2(o[1][j][0], o[1][j][1]), pack_bf16x2(o[1][j][2], o[1][j][3])};
        __builtin_amdgcn_raw_buffer_store_b128(w, rs, (uint32_t)(16 * j + m) * lb + 2 * (32 * wl + 8 * g), 0, 0);
      }
    } else if (c * CH % a.seg == 0) {
      write_down(c);
    }
    const float add = b[3 * CH];
    gsum += b[3 * CH + 2];
    if (__builtin_amdgcn_readfirstlane(__float_as_int(b[3 * CH + 1])) != 0) {  // (a slow decay)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[u][kt][e] = fmaf(acc[u][kt][e], add, acc[u][kt][e]);
    } else {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) acc[u][kt] *= add;
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const float4 w0 = *reinterpret_cast<const float4*>(b + 2 * CH + 32 * s + 4 * g);
      const float4 w1 = *reinterpret_cast<const float4*>(b + 2 * CH + 32 * s + 16 + 4 * g);
      uint32_t t[2][4][3];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint4 vw = __builtin_bit_cast(uint4, vf[u][s]);
        split_pair<3>(lo_f32(vw.x) * w0.x, hi_f32(vw.x) * w0.y, t[u][0]);
        split_pair<3>(lo_f32(vw.y) * w0.z, hi_f32(vw.y) * w0.w, t[u][1]);
        split_pair<3>(lo_f32(vw.z) * w1.x, hi_f32(vw.z) * w1.y, t[u][2]);
        split_pair<3>(lo_f32(vw.w) * w1.z, hi_f32(vw.w) * w1.w, t[u][3]);
      }
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        const uint2 k0 = lds_tr(ks + 32 * s * C::KB + flip(at_tr, 2 * kt));
        const uint2 k1 = lds_tr(ks + (32 * s + 16) * C::KB + flip(at_tr, 2 * kt));
        const lbf16x8 kf = __builtin_bit_cast(lbf16x8, make_uint4(k0.x, k0.y, k1.x, k1.y));
#pragma unroll
        for (int i = 2; i >= 0; --i)  // (the small terms first)
#pragma unroll
          for (int u = 0; u < 2; ++u)
            acc[u][kt] = mfma16(kf, __builtin_bit_cast(lbf16x8, make_uint4(t[u][0][i], t[u][1][i], t[u][2][i], t[u][3][i])), acc[u][kt]);
      }
    }
    if (in_group == C::GC - 1 && c + 1 < chunks) g_store(c + 1 + wl, gv);
    if constexpr (OUT) {
      lds_barrier();  // nobody reads k and v any more
      issue_kv(c + 1);
    }
  }
  if constexpr (OUT) {
    if (last && a.s_out != nullptr) put(a.s_out + ((size_t)p.seq * a.Hv + h) * hs);
  } else if (last) {
    write_down(chunks);
  } else {
    const size_t at = (size_t)slot * a.Hv + h;
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
    // segments as long as leave two workgroups for every CU
    const long rows = packed ? T : (long)N * T, groups = Hv / walk_heads(Hk, Hv, V);
    const long seg = std::max(1L, (rows * groups / 512 + CH - 1) / CH) * CH;
    p.seg = (int)std::min(seg, (long)INT32_MAX / 4);
    p.run = 2 * p.seg;
  } else {
    p.seg = 64;
    const int vg = V / (16 * STATE_NW);
    p.run = (int)std::min((long)INT32_MAX / 128 * 64, std::max(1L, (T + 63L) / 64) * 64);
    while (p.run > 4 * p.seg && (long)slots(p.run) * Hv * vg < 256) p.run = (p.run / p.seg + 1) / 2 * p.seg;
  }
  p.run_slots = slots(p.run);
  p.seg_slots = slots(p.seg);
  p.single = T <= p.run;
  const bool cut = !walk || T > p.seg;
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
  if (a.T > p.seg)
    hipLaunchKernelGGL((lin_walk_kernel<K, V, NH, false>), dim3((unsigned)(p.run_slots * groups)), dim3(64 * CS::NW), CS::LDS, s, a);
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
