// Causal attention over whole sequences with a sliding window and first tokens that stay visible (sinks), on MFMA.
//
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys j <= p_i with p_i - j < window or j < sinks
//
// The queries of the G heads that share a key head are one list of rows, row r = query r / G, head r % G: a workgroup's rows
// then stand at few positions, and its keys are read once for all of them. A wave holds 32 rows, a row a lane: S^T = K Q^T
// leaves a row's scores in one lane (and its partner, lane ^ 32), so that the softmax is within a lane but for one exchange,
// and S^T's layout is the second operand of O^T = V^T P^T as it stands: keys in the order that S^T leaves them, V read
// transposed from LDS in the same order. One pass over the keys with a running maximum and sum.
// Tiles of K and V are loaded straight into LDS, a tile ahead. The keys that a workgroup's rows see are one list, sinks then
// window, so that a few sinks share a tile with the window's first keys; tiles that all rows of a wave see whole have no mask.
// Scores, statistics and O are fp32; P is rounded to bf16 for the product where V is bf16 (at most 2^-8 of each weight, as V's own).
// What a row is divided by is the sum of its weights as they are at D = 128 and as they are rounded at D = 64, whichever costs
// fewer cycles there (RowWave::add): a weight's rounding is then the output's alone, or the sum's with it.
// The maximum may lag by 2^8: it is taken on, and O rescaled, only where a row's rises by more.
//
// What bounds it: matrix products, and the card's power. 16384 tokens of 16 heads on 4, D = 128: 977 .. 1094 us by card and by
// how long it has been busy, 1005 .. 1125 TFLOP/s, 81 .. 90 % of the rate of a large library product; the matrix units are busy
// for 62 % of the cycles, at a clock that falls to 1.5-1.8 GHz (1.3 times the cycles at 1.74 GHz took no longer). 32768 tokens
// through a window of 1024: 316 .. 335 us, eight rounds of two workgroups a CU of which 17 tiles of 64 keys take 33 us and start
// and end 6 each. fp32, 16 heads on 4: 8192 tokens 2355 us at D = 128 and 1140 at D = 64, 117 and 121 TFLOP/s of 154; 4096 tokens
// 765 and 311, 90 and 111.
//
// A masked weight is 0, but 0 times an infinity or a NaN of V is a NaN. A workgroup with an output that is not finite computes
// its rows once more, and in tiles that a row of it does not see whole zeroes such entries in LDS ahead of the product; what
// rows see of them is added in the end (patch_row). (Cleaned at once, with a barrier more, such tiles cost 32768 tokens
// through a window of 1024 9 us of 329.)
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>

#include "gdn_attn.h"
#include "zonos3_attn.h"

namespace zgdn {
namespace {

// n / d for n below 2^31, by a product: n mul / 2^(31 + shift), 2^shift >= d, with mul = 2^(31 + shift) / d rounded up by less
// than 1, so that the result is less than n / 2^(31 + shift) <= 1 / d too large. (A division is twenty vector instructions, of
// uniform numbers as well: 1000 tokens of 8 + 2 heads 14.6 -> 14.2 us, 64 rows behind 8192 keys 17.1 -> 16.6.)
struct Over {
  uint32_t mul, shift;
  Over() = default;
  explicit Over(uint32_t d) : shift(0) {
    while ((1ull << shift) < d) ++shift;
    mul = (uint32_t)(((1ull << (31 + shift)) + d - 1) / d);
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return __umulhi(n << 1, mul) >> shift; }
};

struct WinArgs {
  const void *q, *k, *v;
  long q_ld, k_ld, v_ld;
  void* o;
  const int32_t *cu_q, *cu_k;
  int N, Tq, Tk, Hq, Hk, window, sinks;
  float c;    // |scale| log2(e), or 2^-149 (not 0: a masked score, -inf, times c stays -inf, and any other vanishes)
  int flip;   // scale below zero: the queries change their signs
  int G, per;  // query heads of a key head; tiles of a sequence's rows, where all have as many
  Over over_G, over_Hk, over_N, over_splits;
  int paired;               // two workgroups a CU hold the whole call
  int splits;               // workgroups that share a tile of 32 rows
  float *part_o, *part_ml;  // [workgroup][32][D], [workgroup][32][maximum, sum, whether V was zeroed, -]
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

// The rows that a workgroup takes: tile `tile` of a sequence's nq G rows, the last tiles first (they have the most keys). Where
// all workgroups are on the device at one time (paired), the first tiles come second, so that CUs have one of many keys and one
// of few (4096 tokens, 16 heads: 93 -> 88 us; 8192 tokens, 8 heads 176 -> 167).
struct RowTile {
  int q0, nq, k0, nk, tile;  // (q0, k0: the sequence's first row of q and of k)
};
template <int ROWS>
__device__ __forceinline__ bool find_rows(const WinArgs& a, int i, RowTile& t) {
  if (a.cu_q == nullptr) {
    const int j = (int)a.over_N(i), s = i - j * a.N;
    t = {s * a.Tq, a.Tq, s * a.Tk, a.Tk, a.paired && 2 * j >= a.per ? j - (a.per + 1) / 2 : a.per - 1 - j};
    return true;
  }
  const int l = threadIdx.x & 63;
  int taken = 0;
  for (int s0 = 0; s0 < a.N; s0 += 64) {
    int b = 0, e = 0, kb = 0, ke = 0;
    if (s0 + l < a.N) {
      seq_bounds(a.cu_q, s0 + l, a.Tq, b, e);
      seq_bounds(a.cu_k, s0 + l, a.Tk, kb, ke);
    }
    const int mine = (int)(((uint32_t)(e - b) * a.G + (ROWS - 1)) / ROWS), upto = prefix_count(mine);
    const int all = __builtin_amdgcn_readlane(upto, 63);
    if (i < taken + all) {
      const int at = __builtin_ctzll(__ballot(i - taken < upto));
      const int n = __builtin_amdgcn_readlane(mine, at), before = __builtin_amdgcn_readlane(upto, at) - n;
      b = __builtin_amdgcn_readlane(b, at);
      e = __builtin_amdgcn_readlane(e, at);
      kb = __builtin_amdgcn_readlane(kb, at);
      ke = __builtin_amdgcn_readlane(ke, at);
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

// The keys that the rows at positions first .. last see, as a list of places: the sinks ahead of the window's start, then all
// from there on. Place u is position u, or u + shift behind the sinks.
struct KeyList {
  int s, shift, sunk, n;  // places of sinks; positions left out; places below sunk are seen whatever the window; tiles
  __device__ __forceinline__ int position(int u) const { return u < s ? u : u + shift; }
};
template <int KT>
__device__ __forceinline__ KeyList key_list(const WinArgs& a, int first, int last) {
  KeyList k;
  const int lo = a.window > 0 ? max(0, first - a.window + 1) : 0;
  k.s = min(a.sinks, lo);
  k.shift = lo - k.s;
  k.sunk = max(k.s, a.sinks - k.shift);
  k.n = last < 0 ? 0 : (last - k.shift) / KT + 1;
  return k;
}

struct WholeTiles {
  int to, from, sunk;  // those below `to` from `from` on, or below `sunk`
  __device__ __forceinline__ bool has(int i) const { return i < to && (i >= from || i < sunk); }
};

// Adds to a row that is stored what was zeroed of the values that it sees: w v for each infinity and NaN v, w its weight, by
// one wave. q, k, v, o: the row's and its key head's first entries; p its place, top its maximum.
template <typename T, int D, int KT>
__device__ __forceinline__ void patch_row(const WinArgs& a, const KeyList& keys, const WholeTiles& whole, int nk, const T* q,
                                       const T* k, const T* v, T* o, int p, float top) {
  const int lane = threadIdx.x & 63;
  for (int i = 0; i < keys.n; ++i) {
    if (whole.has(i)) continue;
    const int u = KT * i + lane, j = keys.position(u);
    bool odd = false;
    if (lane < KT && u <= p && j < nk && (a.window == 0 || p - u < a.window || u < keys.sunk))
      for (int c = 0; c < D * (int)sizeof(T) / 16; ++c) {
        uint4 w = *reinterpret_cast<const uint4*>(v + (size_t)j * a.v_ld + c * (16 / (int)sizeof(T)));
        odd = clear_odd<T>(w) || odd;
      }
    for (uint64_t left = __ballot(odd); left != 0; left &= left - 1) {
      const size_t key = (size_t)__builtin_amdgcn_readlane(j, __builtin_ctzll(left));
      float dot = 0.f;
#pragma unroll
      for (int d = lane; d < D; d += 64) dot = fmaf(io<T>::load(q + d), io<T>::load(k + key * a.k_ld + d), dot);
      dot = wave_sum(dot);
      const float w = exp2_of(((a.flip ? -dot : dot) - top) * a.c);
#pragma unroll
      for (int d = lane; d < D; d += 64) {
        const float x = io<T>::load(v + key * a.v_ld + d);
        if (x - x != 0.f) io<T>::store(o + d, io<T>::load(o + d) + w * x);
      }
    }
  }
}

// A workgroup's rows of a sequence and key head, and their keys. Positions, from here on, are places of the list's second part
// (p - shift): differences and bounds are the same.
template <int ROWS, int KT>
struct Rows {
  RowTile t;
  uint32_t rows, r0;
  int G, hk, past, first, last;  // past: position of query 0; first, last: places of the first and last row
  KeyList keys;
  __device__ __forceinline__ bool find(const WinArgs& a, int i, int key_head) {
    if (!find_rows<ROWS>(a, i, t)) return false;
    G = a.G;
    hk = key_head;
    rows = (uint32_t)t.nq * G;
    r0 = (uint32_t)t.tile * ROWS;
    past = t.nk - t.nq;
    first = past + (int)a.over_G(r0);
    last = past + (int)a.over_G(min(rows, r0 + ROWS) - 1);
    keys = key_list<KT>(a, first, last);
    first -= keys.shift;
    last -= keys.shift;
    return true;
  }
  // The tiles that rows at places f .. l all see whole.
  __device__ __forceinline__ WholeTiles whole(const WinArgs& a, int f, int l) const {
    WholeTiles w;
    w.to = f < 0 ? 0 : (f + 1) / KT;
    w.from = a.window == 0 || keys.sunk > l - a.window ? 0 : (l - a.window) / KT + 1;
    w.sunk = keys.sunk / KT;
    return w;
  }
  // patch_row for query qi, head hq, whose maximum is `top`.
  template <typename T, int D>
  __device__ __forceinline__ void patch(const WinArgs& a, const WholeTiles& w, int qi, int hq, float top) const {
    const size_t row = (size_t)(t.q0 + qi);
    patch_row<T, D, KT>(a, keys, w, t.nk, reinterpret_cast<const T*>(a.q) + row * a.q_ld + (size_t)hq * D,
                        reinterpret_cast<const T*>(a.k) + (size_t)t.k0 * a.k_ld + (size_t)hk * D,
                        reinterpret_cast<const T*>(a.v) + (size_t)t.k0 * a.v_ld + (size_t)hk * D,
                        reinterpret_cast<T*>(a.o) + (row * a.Hq + hq) * D, past + qi - keys.shift, top);
  }
};

// Loads of the tiles of K or of V straight into LDS, one after the other, by N instructions of a wave each, the first at row
// `at` of a tile. (What a tile costs in scalar instructions counts: a wave issues one instruction in four or five cycles.)
template <typename T, int D, int KT, int N>
struct TileLoads {
  static constexpr int ES = (int)sizeof(T), ROWB = D * ES, CH = ROWB / 16, RP = 64 / CH;
  const T* base;  // the sequence's first row
  long ld;
  uint32_t row_bytes, off[N];
  int at, next, last, split;    // the next tile; the last one; the one where the list's parts meet
  uint64_t from;                // of the next tile's first row
  uint32_t tile_bytes, last_bytes;
  __device__ __forceinline__ TileLoads(const void* p, long row_ld, const RowTile& t, int hk, int r0) {
    base = reinterpret_cast<const T*>(p) + (size_t)t.k0 * row_ld + (size_t)hk * D;
    ld = row_ld;
    row_bytes = (uint32_t)row_ld * ES;
    at = r0;
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int r = r0 + j * RP + lane / CH;
      off[j] = (uint32_t)r * row_bytes + ((uint32_t)((lane % CH) ^ swizzle<ROWB, T, 32>(r)) << 4);
    }
  }
  // From tile i on. Rows behind the last of nk keys are zeros.
  __device__ __forceinline__ void start(const KeyList& k, int nk, int i) {
    next = i;
    last = k.n - 1;
    split = k.s > 0 && k.shift > 0 ? k.s / KT : -1;
    tile_bytes = (KT - 1) * row_bytes + ROWB;
    last_bytes = (uint32_t)(min(KT, nk - (KT * last + k.shift)) - 1) * row_bytes + ROWB;  // (where the parts do not meet in it)
    from = (uint64_t)(uintptr_t)(base + (size_t)(KT * i + (i > split ? k.shift : 0)) * ld);
  }
  __device__ __forceinline__ void issue(const KeyList& k, int nk, uint32_t to) {
    if (next != split) {
      const RsrcWords rs = {(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)from),
                            (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(from >> 32) & 0xffffu)),
                            (uint32_t)__builtin_amdgcn_readfirstlane((int)(next == last ? last_bytes : tile_bytes)), 0x00020000u};
#pragma unroll
      for (int j = 0; j < N; ++j) load_lds(rs, off[j], (uint32_t)__builtin_amdgcn_readfirstlane((int)(to + 1024 * j)));
    } else {  // the last sinks and the window's first keys
      int lane = threadIdx.x & 63;
      asm volatile("" : "+v"(lane));  // (nothing of this is kept across a loop)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int r = at + j * RP + lane / CH, row = k.position(KT * next + r), c = (lane % CH) ^ swizzle<ROWB, T, 32>(r);
        const uint8_t* p = reinterpret_cast<const uint8_t*>(base + (size_t)row * ld) + 16 * c;
        load_lds_from(row < nk ? (const void*)p : (const void*)zeros16,
                      (uint32_t)__builtin_amdgcn_readfirstlane((int)(to + 1024 * j)));
      }
      from += (uint64_t)k.shift * row_bytes;
    }
    from += (uint64_t)KT * row_bytes;
    ++next;
  }
};

// Zeros for what is not finite in the pieces of V that TileLoad's N instructions brought to `at`; whether there was anything.
template <typename T, int N>
__device__ __forceinline__ bool clean_tile(uint8_t* at) {
  bool any = false;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    uint4* p = reinterpret_cast<uint4*>(at + 1024 * j + 16 * (threadIdx.x & 63));
    uint4 w = *p;
    if (clear_odd<T>(w)) {
      *p = w;
      any = true;
    }
  }
  return any;
}

// One wave's 32 rows, a row a lane and its partner (lane ^ 32).
template <typename T, int D, int KT>
struct RowWave {
  static constexpr bool BF = sizeof(T) == 2;
  static constexpr int ES = (int)sizeof(T), ROWB = D * ES, ST = KT / 32, DT = D / 32, QF = D * ES / 32;
  struct Scores {
    af32x16 t[ST];
  };
  uint4 qf[QF];      // the query as the second operand: entries k of the lane's half
  af32x16 o[DT];     // O^T
  float top, sum;    // of the row; of the lane's keys
  float c, lag;      // lag: how far the maximum may lag behind (weights up to 2^8)
  int m, h, l, l4;   // row, half, lane of 16, group of 16 of the half

  __device__ __forceinline__ void start(const WinArgs& a, const T* q) {
    const int lane = threadIdx.x & 63;
    m = lane & 31, h = lane >> 5, l = lane & 15, l4 = (lane >> 4) & 1;
    c = a.c, lag = fminf(8.f / a.c, FLT_MAX), top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int t = 0; t < QF; ++t) qf[t] = *reinterpret_cast<const uint4*>(q + (BF ? 16 * t + 8 * h : 8 * t + 4 * h));
    if (a.flip) {
      constexpr uint32_t signs = BF ? 0x80008000u : 0x80000000u;
#pragma unroll
      for (int t = 0; t < QF; ++t) qf[t] = make_uint4(qf[t].x ^ signs, qf[t].y ^ signs, qf[t].z ^ signs, qf[t].w ^ signs);
    }
#pragma unroll
    for (int t = 0; t < QF; ++t) asm volatile("" : "+v"(qf[t].x));  // (awaited here, not in the loop)
    float zero = 0.f;
    asm volatile("" : "+v"(zero));  // (a constant tuple would be kept in registers for the next start)
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][e] = zero;
  }
  // Where a stage's fragments are for the lane. Those of the other steps differ in some bits of the address alone (rows 32
  // apart have one mask, rows 8 apart masks that differ in one bit). Formed for each stage anew: the addresses of all steps,
  // kept across a loop, took 16 registers.
  __device__ __forceinline__ uint32_t key_at(const uint8_t* ks) const {
    uint32_t at = lds_address(ks) + row_chunk<ROWB, T, 32>(m, h);
    asm volatile("" : "+v"(at));
    return at;
  }
  static __device__ __forceinline__ uint4 key_frag(uint32_t at, int t, int kk) {  // rows 32 t + m, piece 2 kk + h
    return lds_piece((at ^ (kk << 5)) + 32 * t * ROWB);
  }
  __device__ __forceinline__ uint32_t value_at(const uint8_t* vs) const {
    uint32_t at = lds_address(vs) + row_chunk<ROWB, T, 32>(4 * h + (l >> 2), 2 * l4 + ((l & 3) >> 1)) + 8 * (l & 1);
    asm volatile("" : "+v"(at));
    return at;
  }
  static __device__ __forceinline__ uint4 value_frag(uint32_t at, int u, int d) {  // bf16: 16 keys u, 32 columns d
    constexpr int FLIP = (swizzle<ROWB, T, 32>(0) ^ swizzle<ROWB, T, 32>(8)) << 4;
    const uint2 v0 = lds_transposed((at ^ (d << 6)) + 16 * u * ROWB);
    const uint2 v1 = lds_transposed((at ^ (d << 6) ^ FLIP) + (16 * u + 8) * ROWB);
    return make_uint4(v0.x, v0.y, v1.x, v1.y);
  }
  __device__ __forceinline__ af32x16 score_step(const uint4& kf, int kk, af32x16 x) const {
    if constexpr (BF) {
      return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(abf16x8, kf), __builtin_bit_cast(abf16x8, qf[kk]), x, 0, 0, 0);
    } else {
      const uint32_t kw[4] = {kf.x, kf.y, kf.z, kf.w}, qw[4] = {qf[kk].x, qf[kk].y, qf[kk].z, qf[kk].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) x = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(kw[e]), __uint_as_float(qw[e]), x, 0, 0, 0);
      return x;
    }
  }
  // S^T: place 32 t + 8 (e / 4) + 4 h + e % 4 of the tile in t[t][e].
  __device__ __forceinline__ void scores(const uint8_t* ks, Scores& s) const {
    const uint32_t at = key_at(ks);
    if constexpr (BF) {
#pragma unroll
      for (int t = 0; t < ST; ++t) {
        s.t[t] = af32x16{};
#pragma unroll
        for (int kk = 0; kk < QF; ++kk) s.t[t] = score_step(key_frag(at, t, kk), kk, s.t[t]);
      }
    } else {  // (fragments read a step ahead, so that a step's four products wait for none)
      uint4 kf[2] = {key_frag(at, 0, 0)};
      s.t[0] = af32x16{};
#pragma unroll
      for (int kk = 0; kk < QF; ++kk) {
        if (kk + 1 < QF) kf[(kk + 1) & 1] = key_frag(at, 0, kk + 1);
        s.t[0] = score_step(kf[kk & 1], kk, s.t[0]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  static __device__ __forceinline__ float largest(const Scores& s) {  // of the lane's
    float best = s.t[0][0];
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
      for (int e = t == 0; e + 1 < 16; e += 2) best = fmaxf(fmaxf(best, s.t[t][e]), s.t[t][e + 1]);
    return fmaxf(best, s.t[0][15]);
  }
  // Which of the lane's places, a bit each, lie below place x of the tile.
  static __device__ __forceinline__ uint32_t places_below(int x) {
    x = min(max(x, 0), KT);
    const int n = (x >> 3) * 4 + min(x & 7, 4);
    return n >= 32 ? ~0u : (1u << n) - 1u;
  }
  // -inf for what the row at place p does not see of the tile at p0; the lane's largest of the rest.
  __device__ __forceinline__ float mask(const WinArgs& a, const KeyList& k, int p, int p0, Scores& s) const {
    const int at = p0 + 4 * h;
    uint32_t seen = a.window > 0 ? ~places_below(p - a.window + 1 - at) : ~0u;
    seen = places_below(p + 1 - at) & (seen | places_below(k.sunk - at));
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint32_t keep = (uint32_t)__builtin_amdgcn_sbfe((int)seen, 16 * t + e, 1);  // all ones or none
        s.t[t][e] = __uint_as_float((__float_as_uint(s.t[t][e]) & keep) | (0xff800000u & ~keep));
      }
    return largest(s);
  }
  // The running maximum, and what goes by it, where it is more than `lag` behind.
  __device__ __forceinline__ void settle(float best) {
    const auto pair = __builtin_amdgcn_permlane32_swap(__float_as_uint(best), __float_as_uint(best), false, false);
    const float next = fmaxf(top, fmaxf(__uint_as_float(pair[0]), __uint_as_float(pair[1])));
    if (__any(next > top + lag)) {
      const float keep = exp2_of((top - (next == -INFINITY ? 0.f : next)) * c);
      top = next;
      sum *= keep;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] *= keep;
    }
  }
  // O^T + V^T P^T. AHEAD: beside it the scores of the next tile and the lane's largest of them, given out over the weights.
  template <bool AHEAD>
  __device__ __forceinline__ void add(const uint8_t* vs, Scores& s, const uint8_t* next_ks, Scores& ahead, float& best) {
    const float base = top == -INFINITY ? 0.f : top * c;
    if constexpr (BF) {
      uint32_t w[2 * ST][4];
      auto weigh = [&](int n) {  // two weights, rounded, and their part of the sum
        const af32x16& x = s.t[n / 8];
        const float y0 = exp2_of(fmaf(x[2 * (n % 8)], c, -base)), y1 = exp2_of(fmaf(x[2 * (n % 8) + 1], c, -base));
        const uint32_t y = pack_bf16x2(y0, y1);
        // one sum of two products takes about as long as three additions: at D = 64 vector instructions bind and the count of
        // instructions tells (8192 tokens, 16 + 4 heads: 160 us, 164 with additions), at D = 128 it does not (1013, 1032 without)
        if constexpr (D == 64)
          sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(abf16x2, y), __builtin_bit_cast(abf16x2, 0x3f803f80u), sum, false);
        else
          sum += y0, sum += y1;
        w[n / 4][n % 4] = y;
      };
      constexpr int LATE = AHEAD ? 4 : 0;  // weights of the last 8 keys of the lane's, beside the product's first steps
      if constexpr (AHEAD) {
        const uint32_t kat = key_at(next_ks);
        constexpr int PF = D == 128 ? 2 : 1;  // steps that a fragment is read ahead (as many as registers allow)
        uint4 kf[PF + 1][ST];
#pragma unroll
        for (int t = 0; t < ST; ++t) ahead.t[t] = af32x16{};
#pragma unroll
        for (int kk = 0; kk < PF; ++kk)
#pragma unroll
          for (int t = 0; t < ST; ++t) kf[kk][t] = key_frag(kat, t, kk);
#pragma unroll
        for (int kk = 0; kk < QF; ++kk) {
          if (kk + PF < QF)
#pragma unroll
            for (int t = 0; t < ST; ++t) kf[(kk + PF) % (PF + 1)][t] = key_frag(kat, t, kk + PF);
#pragma unroll
          for (int t = 0; t < ST; ++t) ahead.t[t] = score_step(kf[kk % (PF + 1)][t], kk, ahead.t[t]);
#pragma unroll
          for (int n = (8 * ST - LATE) * kk / QF; n < (8 * ST - LATE) * (kk + 1) / QF; ++n) weigh(n);
        }
      } else {
#pragma unroll
        for (int n = 0; n < 8 * ST; ++n) weigh(n);
      }
      const uint32_t vat = value_at(vs);
      uint4 vf[2][DT];
#pragma unroll
      for (int d = 0; d < DT; ++d) vf[0][d] = value_frag(vat, 0, d);
#pragma unroll
      for (int u = 0; u < 2 * ST; ++u) {
        if (u + 1 < 2 * ST)
#pragma unroll
          for (int d = 0; d < DT; ++d) vf[(u + 1) & 1][d] = value_frag(vat, u + 1, d);
        const abf16x8 pf = __builtin_bit_cast(abf16x8, make_uint4(w[u][0], w[u][1], w[u][2], w[u][3]));
#pragma unroll
        for (int d = 0; d < DT; ++d)
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(abf16x8, vf[u & 1][d]), pf, o[d], 0, 0, 0);
        if constexpr (AHEAD) {
          if (u < 2) weigh(8 * ST - LATE + 2 * u), weigh(8 * ST - LATE + 2 * u + 1);
          if (u == 2) best = largest(ahead);
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s.t[0][e] = exp2_of(fmaf(s.t[0][e], c, -base));
        sum += s.t[0][e];
      }
      float v[2][DT];
      auto values = [&](int e) {
#pragma unroll
        for (int d = 0; d < DT; ++d)
          v[e & 1][d] = *reinterpret_cast<const float*>(
              vs + row_chunk<ROWB, T, 32>(8 * (e >> 2) + 4 * h + (e & 3), 8 * d + (m >> 2)) + 4 * (m & 3));
      };
      values(0);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        if (e + 1 < 16) values(e + 1);
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[e & 1][d], s.t[0][e], o[d], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (AHEAD) {
        scores(next_ks, ahead);
        best = largest(ahead);
      }
    }
  }
  // Is an entry of O's row not finite?
  __device__ __forceinline__ bool odd() const {
    float x = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) x = fmaf(o[d][e], 0.f, x);
    return x != 0.f;
  }
  // O's row times `by`, 16 bytes a lane: of two groups of four entries a half has every other one, so the halves exchange them.
  __device__ __forceinline__ void store(T* row, float by) const {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 8) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = o[d][e + i] * by;
        T* at = row + 32 * d + 2 * e + 8 * h;
        if constexpr (BF) {
          const auto u = __builtin_amdgcn_permlane32_swap(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[4], x[5]), false, false);
          const auto v = __builtin_amdgcn_permlane32_swap(pack_bf16x2(x[2], x[3]), pack_bf16x2(x[6], x[7]), false, false);
          *reinterpret_cast<uint4*>(at) = make_uint4(u[0], v[0], u[1], v[1]);
        } else {
          *reinterpret_cast<float4*>(row + 32 * d + 2 * e + 4 * h) = make_float4(x[0], x[1], x[2], x[3]);
          *reinterpret_cast<float4*>(row + 32 * d + 2 * e + 8 + 4 * h) = make_float4(x[4], x[5], x[6], x[7]);
        }
      }
  }
  // The row's sum over both halves.
  __device__ __forceinline__ float whole_sum() const {
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
    return __uint_as_float(both[0]) + __uint_as_float(both[1]);
  }
};

// Many rows: a wave for each 32 of a workgroup's, all on the same tiles. The scores of a tile are formed beside the product of
// the one before, so that matrix and vector instructions have each other to run beside; K is loaded a tile further ahead than V.
// (Three workgroups a CU at D = 64. For fp32 there 10 of a wave's registers are then spilled; two a CU, which would need none to
// be, have not been measured.)
template <typename T, int D, int NW>
__global__ __launch_bounds__(64 * NW, D == 64 ? 3 : sizeof(T) == 2 ? 2 : 1) void win_attn_kernel(WinArgs a) {
  constexpr int KT = sizeof(T) == 2 ? 64 : 32, ROWB = D * (int)sizeof(T), LW = KT * ROWB / 1024 / NW, ROWS = 32 * NW;
  using Wave = RowWave<T, D, KT>;
  using R = Rows<ROWS, KT>;
  __shared__ __align__(1024) uint8_t stages[4][KT * ROWB];
  __shared__ int dirty;  // something of V was zeroed
  auto k_lds = [&](int i) { return stages[i & 1]; };
  auto v_lds = [&](int i) { return stages[2 + (i & 1)]; };
  const int wave = wave_id(), m = threadIdx.x & 31;
  R r;
  const int of_keys = (int)a.over_Hk(blockIdx.x);
  if (!r.find(a, of_keys, blockIdx.x - of_keys * a.Hk)) return;
  const uint32_t rw = r.r0 + 32 * wave, row = min(rw + m, r.rows - 1);  // (lanes behind the last row: as that one, without stores)
  const bool real = rw + m < r.rows;
  const int qi = (int)a.over_G(row), hq = r.hk * r.G + (int)(row - (uint32_t)qi * r.G);
  const int shift = r.keys.shift, n = r.keys.n, p = r.past + qi - shift;
  const int wfirst = r.past + (int)a.over_G(min(r.rows - 1, rw)) - shift;
  const int wlast = r.past + (int)a.over_G(min(r.rows, rw + 32) - 1) - shift;
  constexpr int RP = 1024 / ROWB;
  const WholeTiles whole = r.whole(a, r.first, r.last), whole_w = r.whole(a, wfirst, wlast);
  TileLoads<T, D, KT, LW> load_k(a.k, a.k_ld, r.t, r.hk, wave * LW * RP), load_v(a.v, a.v_ld, r.t, r.hk, wave * LW * RP);
  auto issue_k = [&] { load_k.issue(r.keys, r.t.nk, lds_address(k_lds(load_k.next)) + 1024 * LW * wave); };
  auto issue_v = [&] { load_v.issue(r.keys, r.t.nk, lds_address(v_lds(load_v.next)) + 1024 * LW * wave); };

  if (threadIdx.x == 0) dirty = 0;
  const T* q = reinterpret_cast<const T*>(a.q) + (size_t)(r.t.q0 + qi) * a.q_ld + (size_t)hq * D;
  Wave w;
  using Scores = typename Wave::Scores;
  auto settle = [&](int i, Scores& s, float best) {
    if (!whole_w.has(i)) {
      asm volatile("");  // (a branch, not 100 instructions of every tile)
      best = w.mask(a, r.keys, p, KT * i, s);
    }
    w.settle(best);
  };
  for (bool cleaning = false;; cleaning = true) {
    int t0 = 0;
    asm volatile("" : "+s"(t0));  // (nothing of the first tile is kept for another pass)
    if (n > 0) {
      load_k.start(r.keys, r.t.nk, t0);
      load_v.start(r.keys, r.t.nk, t0);
      issue_k();
      issue_v();
      if (n > 1) issue_k();
    }
    w.start(a, q + t0);
    if (n > 0) {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the first tiles are there
      Scores one, two;
      w.scores(k_lds(0), one);
      settle(t0, one, w.largest(one));
      // (the tile behind the last one is scored too, on what its stage holds, and not used)
      auto step = [&](int i, Scores& s, Scores& ahead) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");  // V of tile i and K of the next are there
        if (i + 2 < n) issue_k();
        if (i + 1 < n) issue_v();
        if (cleaning && !whole.has(i)) {
          if (clean_tile<T, LW>(v_lds(i) + 1024 * LW * wave)) dirty = 1;
          asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
        float best;
        w.template add<true>(v_lds(i), s, k_lds(i + 1), ahead, best);
        if (i + 1 < n) settle(i + 1, ahead, best);
      };
      for (int i = t0;;) {
        step(i, one, two);
        if (++i >= n) break;
        step(i, two, one);
        if (++i >= n) break;
      }
    }
    if (cleaning || !__builtin_expect(__syncthreads_or(w.odd()), 0)) break;
  }
  const float inv = p + shift < 0 ? 0.f : 1.f / w.whole_sum();
  if (real) w.store(reinterpret_cast<T*>(a.o) + ((size_t)(r.t.q0 + qi) * a.Hq + hq) * D, inv);
  if (n > 0 && dirty) {
    __threadfence();
    for (uint32_t left = (uint32_t)__ballot(real); left != 0; left &= left - 1) {
      const int x = __builtin_ctz(left);
      r.template patch<T, D>(a, whole, __builtin_amdgcn_readlane(qi, x), __builtin_amdgcn_readlane(hq, x),
                             __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w.top), x)));
    }
  }
}

// Few rows: a workgroup for 32 rows and a share of their tiles (a.splits), whose waves take them in turn, each with stages of
// its own and no barrier; the waves' parts (maximum, sum, O) are joined in LDS, those of several workgroups by a second
// kernel, in order.
constexpr int FEW_NW = 4, FEW_KT = 32;
template <typename T, int D>
struct FewCfg {
  static constexpr int TILE = 2 * FEW_KT * D * (int)sizeof(T);  // bytes of K and V
  static constexpr int RING = TILE <= 16384 ? 2 : 1, PART = D + 4;
  static_assert(RING * TILE >= 32 * PART * 4, "the waves' parts");
};

template <typename T, int D>
__global__ __launch_bounds__(64 * FEW_NW, 2) void win_few_kernel(WinArgs a) {
  constexpr int KT = FEW_KT, ROWB = D * (int)sizeof(T), LI = KT * ROWB / 1024, RING = FewCfg<T, D>::RING, PART = FewCfg<T, D>::PART;
  using Wave = RowWave<T, D, KT>;
  using R = Rows<32, KT>;
  extern __shared__ __align__(1024) uint8_t tile_lds[];  // [wave][stage][K, V][KT rows]
  __shared__ float top_of[FEW_NW][32], sum_of[FEW_NW][32];
  __shared__ int dirty;  // something of V was zeroed
  const int wave = wave_id(), m = threadIdx.x & 31, h = (threadIdx.x >> 5) & 1;
  auto k_lds = [&](int stage) { return tile_lds + (wave * RING + stage) * FewCfg<T, D>::TILE; };
  auto v_lds = [&](int stage) { return k_lds(stage) + KT * ROWB; };
  const int ts = (int)a.over_Hk(blockIdx.x), tile = (int)a.over_splits(ts), split = ts - tile * a.splits;
  R r;
  if (!r.find(a, tile, blockIdx.x - ts * a.Hk)) return;
  const uint32_t row = min(r.r0 + m, r.rows - 1);
  const int qi = (int)a.over_G(row), hq = r.hk * r.G + (int)(row - (uint32_t)qi * r.G);
  const int p = r.past + qi - r.keys.shift;
  const int t0 = (int)((long)r.keys.n * split / a.splits), t1 = (int)((long)r.keys.n * (split + 1) / a.splits);
  const WholeTiles whole = r.whole(a, r.first, r.last);
  TileLoads<T, D, KT, LI> load_k(a.k, a.k_ld, r.t, r.hk, 0), load_v(a.v, a.v_ld, r.t, r.hk, 0);
  auto issue = [&](int i, int stage) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // what the stage held before has been read
    load_k.start(r.keys, r.t.nk, i);
    load_v.start(r.keys, r.t.nk, i);
    load_k.issue(r.keys, r.t.nk, lds_address(k_lds(stage)));
    load_v.issue(r.keys, r.t.nk, lds_address(v_lds(stage)));
  };
  if (t0 + wave < t1) issue(t0 + wave, 0);
  if (threadIdx.x == 0) dirty = 0;
  __syncthreads();
  Wave w;
  w.start(a, reinterpret_cast<const T*>(a.q) + (size_t)(r.t.q0 + qi) * a.q_ld + (size_t)hq * D);
  auto compute = [&](int i, int stage) {
    typename Wave::Scores s;
    float best;
    w.scores(k_lds(stage), s);
    if (whole.has(i)) {
      best = w.largest(s);
    } else {
      if (clean_tile<T, LI>(v_lds(stage))) dirty = 1;
      best = w.mask(a, r.keys, p, KT * i, s);
    }
    w.settle(best);
    w.template add<false>(v_lds(stage), s, nullptr, s, best);
  };
  for (int i = t0 + wave, stage = 0; i < t1; i += FEW_NW, stage ^= RING - 1) {
    if (RING == 2 && i + FEW_NW < t1) {
      issue(i + FEW_NW, stage ^ 1);
      wait_own_loads<2 * LI>();
    } else {
      wait_own_loads<0>();
    }
    compute(i, stage);
    if (RING == 1 && i + FEW_NW < t1) issue(i + FEW_NW, 0);
  }

  const float sum = w.whole_sum();
  __syncthreads();
  float* mine = reinterpret_cast<float*>(k_lds(0)) + m * PART;
#pragma unroll
  for (int d = 0; d < Wave::DT; ++d)
#pragma unroll
    for (int e = 0; e < 16; e += 4)
      *reinterpret_cast<float4*>(mine + 32 * d + 2 * e + 4 * h) = make_float4(w.o[d][e], w.o[d][e + 1], w.o[d][e + 2], w.o[d][e + 3]);
  if (h == 0) {
    top_of[wave][m] = w.top;
    sum_of[wave][m] = sum;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * D / 4; i += 64 * FEW_NW) {
    const int x = i / (D / 4), d = i % (D / 4) * 4;
    if (r.r0 + x >= r.rows) continue;
    float best = -INFINITY;
#pragma unroll
    for (int y = 0; y < FEW_NW; ++y) best = fmaxf(best, top_of[y][x]);
    const float base = best == -INFINITY ? 0.f : best;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    float all = 0.f;
#pragma unroll
    for (int y = 0; y < FEW_NW; ++y) {
      const float f = exp2_of((top_of[y][x] - base) * a.c);
      const float4 u = *reinterpret_cast<const float4*>(
          reinterpret_cast<const float*>(tile_lds + y * RING * FewCfg<T, D>::TILE) + x * PART + d);
      v = make_float4(fmaf(u.x, f, v.x), fmaf(u.y, f, v.y), fmaf(u.z, f, v.z), fmaf(u.w, f, v.w));
      all = fmaf(sum_of[y][x], f, all);
    }
    if (a.splits > 1) {
      const size_t at = (size_t)blockIdx.x * 32 + x;
      *reinterpret_cast<float4*>(a.part_o + at * D + d) = v;
      if (d == 0) *reinterpret_cast<float4*>(a.part_ml + 4 * at) = make_float4(best, all, dirty ? 1.f : 0.f, 0.f);
    } else {
      const uint32_t rr = r.r0 + x;
      const int q = (int)a.over_G(rr), hh = r.hk * r.G + (int)(rr - (uint32_t)q * r.G);
      const float inv = r.past + q < 0 ? 0.f : 1.f / all;
      io<T>::store4(reinterpret_cast<T*>(a.o) + ((size_t)(r.t.q0 + q) * a.Hq + hh) * D + d,
                    make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
    }
  }
  if (a.splits > 1 || !dirty) return;
  float top = -INFINITY;
#pragma unroll
  for (int y = 0; y < FEW_NW; ++y) top = fmaxf(top, top_of[y][m]);
  __threadfence();
  __syncthreads();
  for (int x = wave; x < 32; x += FEW_NW)
    if (r.r0 + x < r.rows)
      r.template patch<T, D>(a, whole, __builtin_amdgcn_readlane(qi, x), __builtin_amdgcn_readlane(hq, x),
                             __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(top), x)));
}

// A workgroup joins the parts of 8 rows, D / 4 lanes each.
template <typename T, int D>
__global__ __launch_bounds__(2 * D) void win_few_join_kernel(WinArgs a) {
  using R = Rows<32, FEW_KT>;
  const int t8 = (int)a.over_Hk(blockIdx.x), tile = t8 / 4;
  R r;
  if (!r.find(a, tile, blockIdx.x - t8 * a.Hk)) return;
  const int x = (t8 & 3) * 8 + threadIdx.x / (D / 4), d = threadIdx.x % (D / 4) * 4;
  const bool real = r.r0 + x < r.rows;
  float top = -INFINITY, sum = 0.f;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  bool odd = false;
  constexpr int AT = 4;  // parts read at a time
  for (int i0 = 0; i0 < a.splits; i0 += AT) {
    float4 ml[AT], u[AT];
#pragma unroll
    for (int e = 0; e < AT; ++e) {
      const size_t at = ((size_t)(tile * a.splits + min(i0 + e, a.splits - 1)) * a.Hk + r.hk) * 32 + (real ? x : 0);
      ml[e] = *reinterpret_cast<const float4*>(a.part_ml + 4 * at);
      u[e] = *reinterpret_cast<const float4*>(a.part_o + at * D + d);
    }
#pragma unroll
    for (int e = 0; e < AT; ++e)
      if (i0 + e < a.splits) {
        const float next = fmaxf(top, ml[e].x), base = next == -INFINITY ? 0.f : next;
        const float keep = exp2_of((top - base) * a.c), f = exp2_of((ml[e].x - base) * a.c);
        top = next;
        odd = odd || ml[e].z != 0.f;
        sum = fmaf(sum, keep, ml[e].y * f);
        v = make_float4(fmaf(v.x, keep, u[e].x * f), fmaf(v.y, keep, u[e].y * f), fmaf(v.z, keep, u[e].z * f),
                        fmaf(v.w, keep, u[e].w * f));
      }
  }
  const uint32_t rr = min(r.r0 + x, r.rows - 1);
  const int q = (int)a.over_G(rr), hq = r.hk * r.G + (int)(rr - (uint32_t)q * r.G);
  if (real) {
    const float inv = r.past + q < 0 ? 0.f : 1.f / sum;
    io<T>::store4(reinterpret_cast<T*>(a.o) + ((size_t)(r.t.q0 + q) * a.Hq + hq) * D + d,
                  make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
  }
  uint64_t left = __ballot(odd && real && d == 0);  // (a row's lanes are of one wave)
  if (left == 0) return;
  __threadfence();
  const WholeTiles whole = r.whole(a, r.first, r.last);
  for (; left != 0; left &= left - 1) {
    const int lane = __builtin_ctzll(left);
    r.template patch<T, D>(a, whole, __builtin_amdgcn_readlane(q, lane), __builtin_amdgcn_readlane(hq, lane),
                           __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(top), lane)));
  }
}

// How a call is cut: 128 rows a workgroup, or 32 rows and a share of their keys, whichever is estimated to take less. What a
// workgroup takes, in us: a start and end, then its tiles one after the other, in the first form (a tile of 64 keys for bf16, 32
// for fp32) alone on its CU or as its part of a CU's time, in the second (tiles of 32 for each of four waves) a round at a time.
// (Measured, first / second form, us: 1000 tokens of 8 + 2 heads 22.9 / 15.3, 1536 of 16 + 4 32 / 40, 2048 of 8 + 2 through a window
// of 256 12.2 / 21.5; fp32: 4096 of 8 + 2 569 / 325, through a window of 256 53 / 91, 8192 of 16 + 4 2354 / 2434.)
// Of the second form as many shares of the keys as there are CUs for, of two tiles for each wave at least.
struct WinCost {
  double alone, part, wave;  // a tile of the first form, alone and as a part; of the second
};
WinCost win_cost(int D, int dtype) {
  if (dtype == ZGDN_F32) return D == 128 ? WinCost{4.4, 4.4, 4.6} : WinCost{2.3, 2.3, 2.5};
  return D == 128 ? WinCost{1.05, 1.0, 1.0} : WinCost{0.85, 0.6, 0.7};
}
struct WinPlan {
  long tiles;  // of rows a key head
  int rows, splits;
};
long row_tiles(const WinArgs& a, int rows) {
  const long all = (long)a.Tq * (a.Hq / a.Hk);
  if (a.cu_q == nullptr) return a.N * ((all + rows - 1) / rows);
  return (all + rows - 1) / rows + a.N;  // (each sequence may leave a part of a tile)
}
WinPlan win_plan(const WinArgs& a, int D, int dtype) {
  constexpr double MANY = 6.0, FEW = 7.5, JOIN = 4.0;  // start and end, in us
  const double cus = device_cus(), kt = dtype == ZGDN_F32 ? 32 : 64;
  const WinCost cost = win_cost(D, dtype);
  WinPlan many{row_tiles(a, 128), 128, 1}, few{row_tiles(a, 32), 32, 1};
  // Keys of the longest list and of a list in the mean. The lengths of a packed batch are on the device: it is taken for
  // sequences of equal length, so that `most` is no bound there. One of 30008 keys among 63 of 108, 8 queries each: 496 us, its list
  // walked by one workgroup a key head, where it alone is shared out and takes 26.
  const double seqs = a.cu_q != nullptr ? a.N : 1, nk = a.Tk / seqs, nq = std::min(a.Tq / seqs, nk);
  const double reach = a.window > 0 ? (double)a.window + a.sinks + 32 : nk;
  const double most = std::min(nk, reach), mean = std::min(nk - nq / 2, reach);
  const double many_us = MANY + std::max(most / kt * cost.alone, many.tiles * a.Hk / cus * mean / kt * cost.part);
  const double slots = (D == 64 && dtype == ZGDN_BF16 ? 2 : 1) * cus, groups = (double)few.tiles * a.Hk;
  few.splits = (int)std::max(1.0, std::min(std::floor(most / (2 * FEW_NW * FEW_KT)), std::floor(cus / groups)));
  const double share = cost.wave / (FEW_NW * FEW_KT * few.splits);
  const double few_us = std::max(FEW + most * share, std::ceil(groups * few.splits / slots) * (FEW + mean * share)) +
                        (few.splits > 1 ? JOIN : 0.0);
  return few_us < many_us ? few : many;
}
size_t win_bytes(const WinPlan& p, const WinArgs& a, int D) {
  return p.splits == 1 ? 0 : (size_t)p.tiles * a.Hk * p.splits * 32 * (D + 4) * sizeof(float);
}

template <typename T, int D>
bool launch_win(WinArgs a, const WinPlan& p, hipStream_t s) {
  static std::atomic<signed char> ready[MAX_DEVICES];
  a.G = a.Hq / a.Hk;
  a.per = (int)(p.tiles / a.N);
  a.over_G = Over(a.G), a.over_Hk = Over(a.Hk), a.over_N = Over(a.N), a.over_splits = Over(p.splits);
  a.splits = p.splits;
  a.paired = p.rows == 128 && p.tiles * a.Hk <= 2 * device_cus();
  const unsigned n = (unsigned)(p.tiles * a.Hk);
  if (p.rows == 128) {
    hipLaunchKernelGGL((win_attn_kernel<T, D, 4>), dim3(n), dim3(256), 0, s, a);
    return true;
  }
  constexpr int LDS = FEW_NW * FewCfg<T, D>::RING * FewCfg<T, D>::TILE;
  const auto kernel = win_few_kernel<T, D>;
  if (!lds_ready((const void*)kernel, LDS, ready)) return false;
  hipLaunchKernelGGL(kernel, dim3(n * p.splits), dim3(64 * FEW_NW), LDS, s, a);
  if (p.splits > 1) hipLaunchKernelGGL((win_few_join_kernel<T, D>), dim3(4 * n), dim3(2 * D), 0, s, a);
  return true;
}

// What a plan goes by.
WinArgs plan_args(int packed, int n_seqs, int Tq, int Tk, int Hq, int Hk, int window, int sinks) {
  static const int32_t bounds = 0;  // (told from none by its address alone)
  WinArgs a{};
  a.cu_q = packed ? &bounds : nullptr;
  a.N = n_seqs, a.Tq = Tq, a.Tk = Tk, a.Hq = Hq, a.Hk = Hk;
  a.window = window >= Tk ? 0 : window, a.sinks = std::min(sinks, 1 << 30);
  return a;
}

bool win_sizes(int B, int Tq, int Tk, int Hq, int Hk, int D, int window, int sinks, int dtype) {
  return B >= 1 && Tq >= 0 && Tk >= 0 && Hq >= 1 && Hk >= 1 && Hq % Hk == 0 && (D == 64 || D == 128) && window >= 0 &&
         sinks >= 0 && (dtype == ZGDN_F32 || dtype == ZGDN_BF16) && (long)B * Tq <= 1L << 30 && (long)B * Tk <= 1L << 30 &&
         (long)B * Tq * Hq <= 1L << 31;
}

}  // namespace
}  // namespace zgdn

extern "C" size_t zattn_window_fwd_workspace_bytes(int packed, int n_seqs, int Tq, int Tk, int Hq, int Hk, int D, int window,
                                                   int sinks, int dtype) {
  using namespace zgdn;
  if (n_seqs < 1 || !win_sizes(packed ? 1 : n_seqs, Tq, Tk, Hq, Hk, D, window, sinks, dtype) || Tq == 0) return 0;
  const WinArgs a = plan_args(packed, n_seqs, Tq, Tk, Hq, Hk, window, sinks);
  return win_bytes(win_plan(a, D, dtype), a, D);
}

// (for tests) Rows of a workgroup and workgroups that share their keys, for the same sizes.
extern "C" int zgdn_window_fwd_form(int packed, int n_seqs, int Tq, int Tk, int Hq, int Hk, int D, int window, int sinks,
                                    int dtype, int64_t* form) {
  using namespace zgdn;
  if (n_seqs < 1 || !win_sizes(packed ? 1 : n_seqs, Tq, Tk, Hq, Hk, D, window, sinks, dtype))
    return fail(ZGDN_EINVAL, "zgdn_window_fwd_form: bad sizes");
  const WinPlan p = win_plan(plan_args(packed, n_seqs, Tq, Tk, Hq, Hk, window, sinks), D, dtype);
  form[0] = p.rows;
  form[1] = p.splits;
  return ZGDN_OK;
}

extern "C" int zattn_window_fwd(const void* q, long q_ld, const void* k, long k_ld, const void* v, long v_ld, int dtype,
                                void* o, const int32_t* cu_q, const int32_t* cu_k, int n_seqs, int B, int Tq, int Tk, int Hq,
                                int Hk, int D, int window, int sinks, float scale, void* workspace, size_t workspace_bytes, void* stream) {
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
  if (!std::isfinite(scale * LOG2E)) return fail(ZGDN_EINVAL, "%s: scale %g", fn, scale);
  if (Tq == 0) return ZGDN_OK;
  if (!q || !o || (Tk > 0 && (!k || !v))) return fail(ZGDN_EINVAL, "%s: null tensor pointer", fn);
  const int ve = dtype == ZGDN_F32 ? 4 : 8;
  const long most = 1L << 22, wq = (long)Hq * D, wk = (long)Hk * D;
  auto bad = [&](long ld, long width) { return ld < width || ld > most || ld % ve; };
  if (bad(q_ld, wq) || bad(k_ld, wk) || bad(v_ld, wk))
    return fail(ZGDN_EINVAL, "%s: row strides q=%ld k=%ld v=%ld (multiples of %d elements, at least a row, at most 2^22)", fn,
                q_ld, k_ld, v_ld, ve);
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o | (uintptr_t)workspace) % 16)
    return fail(ZGDN_EINVAL, "%s: q, k, v, o and workspace need 16-byte aligned bases", fn);
  if (((uintptr_t)cu_q | (uintptr_t)cu_k) % 4) return fail(ZGDN_EINVAL, "%s: cu_q, cu_k not on 4-byte boundaries", fn);
  const size_t es = dtype == ZGDN_F32 ? 4 : 2, nq = (size_t)B * Tq, nk = (size_t)B * Tk, cu = ((size_t)n_seqs + 1) * 4;
  if (window >= Tk) window = 0;        // (every key up to the query)
  sinks = std::min(sinks, 1 << 30);  // (more than positions reach)
  const float c = fabsf(scale) * LOG2E;
  WinArgs a{q, k, v, q_ld, k_ld, v_ld, o, cu_q, cu_k, cu_q != nullptr ? n_seqs : B, Tq, Tk, Hq, Hk, window, sinks,
            c > 0.f ? c : FLT_TRUE_MIN, scale < 0.f};
  const WinPlan p = win_plan(a, D, dtype);
  if (p.tiles * p.splits * Hk > (1L << 32) / 256 - 1) return fail(ZGDN_EUNSUPPORTED, "%s: B=%d x Tq=%d x Hq=%d rows", fn, B, Tq, Hq);
  const size_t need = win_bytes(p, a, D);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(ZGDN_EINVAL, "%s: workspace of %zu bytes, %zu needed", fn, workspace == nullptr ? 0 : workspace_bytes, need);
  const Region out = {o, nq, wq * es, wq * es}, ws = {need ? workspace : nullptr, 1, need, need};
  const Region in[] = {{q, nq, wq * es, q_ld * es}, {k, nk, wk * es, k_ld * es}, {v, nk, wk * es, v_ld * es},
                       {cu_q, 1, cu, cu}, {cu_k, 1, cu, cu}};
  bool meet = regions_meet(out, ws);
  for (const Region& r : in) meet = meet || regions_meet(out, r) || regions_meet(ws, r);
  if (meet) return fail(ZGDN_EINVAL, "%s: o or the workspace overlaps another operand", fn);
  if (need > 0) {
    a.part_o = reinterpret_cast<float*>(workspace);
    a.part_ml = a.part_o + (size_t)p.tiles * Hk * p.splits * 32 * D;
  }
  hipStream_t s = (hipStream_t)stream;
  const bool ok = dtype == ZGDN_F32 ? (D == 128 ? launch_win<float, 128>(a, p, s) : launch_win<float, 64>(a, p, s))
                                    : (D == 128 ? launch_win<bf16, 128>(a, p, s) : launch_win<bf16, 64>(a, p, s));
  if (!ok) return fail(ZGDN_EHIP, "%s: the device has too little LDS a workgroup", fn);
  return check_launch(fn);
}
