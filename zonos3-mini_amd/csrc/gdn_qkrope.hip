// Norms of queries and keys for each head, with the position rotation in the same pass and the cache's write behind it.
//
//   y = x * rsqrt(mean(x^2) + eps) * w, then pairs (a, b) -> (a cos t - b sin t, b cos t + a sin t), t = position * inv_freq[i]
//
// HBM-bound: q and k are read and written once. A head is D / 16 lanes, each with the two 8-entry pieces of 8 pairs (in halves:
// entries 8 u .. and R / 2 + 8 u ..; adjacent: 16 u .. 16 u + 15), so that pairs never leave a lane and the norm is one sum
// over 8 or 4 lanes. A wave takes one token: its lanes form the token's R / 2 angles once, one a lane, and hand them round
// through LDS; then up to three groups of 64 / (D / 16) heads, all loads first. A token of more groups, or each group of
// a few tokens, has a wave of its own.
// Measured: calls of 30526 rows of 16 + 2 heads, D = 128, on inputs that rotate: bf16 56 us, 5.05 TB/s, fp32 113 us, 4.96 (a copy:
// 5.14; on the same inputs again and again the bf16 kernel takes 50, for it finds some of them in the last-level cache); one token
// of 8 + 2 heads into a cache 2.8 us in a graph, a launch's own time.
// The angle is reduced to a quarter turn in float64: position * inv_freq has 24 bits in float32, and at position 2^20 the
// rest of them after the whole turns would be 7 (an error of 0.03).
#include <type_traits>

#include "gdn_common.h"
#include "zonos3_attn.h"

namespace zgdn {
namespace {

constexpr int QR_NW = 4;    // waves a workgroup
constexpr int QR_ITER = 3;  // groups of heads a wave, at most

struct RopeArgs {
  const void *q, *k, *v;
  long q_ld, k_ld, v_ld;
  const void* positions;
  int pos_i32;
  const void* inv_freq;
  int freq_f32;
  const void *q_weight, *k_weight;
  int w_bf16;
  float eps;
  void *q_out, *k_out, *k_cache, *v_cache;
  long kc_ld, vc_ld;
  const int64_t* rows;
  long n_cache_rows;
  int n_tokens, Hq, Hk, R;
  int groups, per, parts;  // groups of heads; groups a wave; waves a token
};

// Eight consecutive entries as loaded.
template <typename T>
struct Eight;
template <>
struct Eight<bf16> {
  uint4 w;
  __device__ __forceinline__ void load(const bf16* p) { w = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void floats(float* x) const {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(u[i] << 16), x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
  __device__ __forceinline__ static void store(bf16* p, const float* x) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                                              pack_bf16x2(x[6], x[7]));
  }
  __device__ __forceinline__ void keep(bf16* p) const { *reinterpret_cast<uint4*>(p) = w; }
};
template <>
struct Eight<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = reinterpret_cast<const float4*>(p)[0];
    b = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ void floats(float* x) const {
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  }
  __device__ __forceinline__ static void store(float* p, const float* x) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  }
  __device__ __forceinline__ void keep(float* p) const {
    reinterpret_cast<float4*>(p)[0] = a;
    reinterpret_cast<float4*>(p)[1] = b;
  }
};

// (cos, sin) of position * freq. Quarter turns n and the rest r in [-1/2, 1/2] of one, in float64; then the Taylor sums of
// sine (to x^9, the next term below 2e-9) and cosine (to x^10, below 2e-10) on |x| <= pi / 4.
__device__ __forceinline__ float2 turn_of(double position, double freq) {
  const double t = position * freq * 0.63661977236758134308;  // 2 / pi
  const double n = rint(t);
  const float x = (float)(t - n) * 1.57079632679489661923f;
  const double m = n - 4.0 * floor(0.25 * n);  // n mod 4 (a NaN stays in t - n)
  const int quarter = (int)m;
  const float y = x * x;
  const float s = fmaf(fmaf(fmaf(fmaf(2.7557319e-6f, y, -1.9841270e-4f), y, 8.3333333e-3f), y, -1.6666667e-1f) * y, x, x);
  const float c = fmaf(fmaf(fmaf(fmaf(fmaf(-2.7557319e-7f, y, 2.4801587e-5f), y, -1.3888889e-3f), y, 4.1666667e-2f), y, -0.5f),
                       y, 1.f);
  const float a = quarter & 1 ? s : c, b = quarter & 1 ? c : s;  // |cos|, |sin|
  return make_float2(quarter == 1 || quarter == 2 ? -a : a, quarter >= 2 ? -b : b);
}

template <typename T, int D, bool HALVES>
__global__ __launch_bounds__(64 * QR_NW) void qk_rope_kernel(RopeArgs a) {
  constexpr int LPH = D / 16, HPG = 64 / LPH;
  __shared__ __align__(16) float2 turns[QR_NW][64];
  const int lane = threadIdx.x & 63, wave = wave_id();
  const long item = (long)blockIdx.x * QR_NW + wave;
  const int t = (int)(item / a.parts), part = (int)(item - (long)t * a.parts);
  if (t >= a.n_tokens) return;
  const int u = lane % LPH;
  const bool turned = 16 * u < a.R;
  int p0, p1;  // where the lane's two pieces start in a head
  if (!HALVES || !turned) {
    p0 = 16 * u;
    p1 = p0 + 8;
  } else {
    p0 = 8 * u;
    p1 = a.R / 2 + 8 * u;
  }
  const int n_heads = a.Hq + a.Hk + (a.v != nullptr ? a.Hk : 0);
  const int first = part * a.per * HPG + lane / LPH;

  Eight<T> x0[QR_ITER], x1[QR_ITER];
#pragma unroll
  for (int i = 0; i < QR_ITER; ++i) {
    const int h = first + i * HPG;
    if (i < a.per && h < n_heads) {
      const T* src = h < a.Hq ? reinterpret_cast<const T*>(a.q) + (size_t)t * a.q_ld + (size_t)h * D
                     : h < a.Hq + a.Hk ? reinterpret_cast<const T*>(a.k) + (size_t)t * a.k_ld + (size_t)(h - a.Hq) * D
                                       : reinterpret_cast<const T*>(a.v) + (size_t)t * a.v_ld + (size_t)(h - a.Hq - a.Hk) * D;
      x0[i].load(src + p0);
      x1[i].load(src + p1);
    }
  }
  const int64_t row = a.rows != nullptr ? a.rows[t] : -1;
  if (2 * lane < a.R) {
    const double pos = a.pos_i32 ? (double)reinterpret_cast<const int32_t*>(a.positions)[t]
                                 : (double)reinterpret_cast<const int64_t*>(a.positions)[t];
    const double freq = a.freq_f32 ? (double)reinterpret_cast<const float*>(a.inv_freq)[lane]
                                   : reinterpret_cast<const double*>(a.inv_freq)[lane];
    turns[wave][lane] = turn_of(pos, freq);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (the wave's own part of LDS: no barrier)
  __builtin_amdgcn_wave_barrier();
  float c[8], s[8];
  if (turned) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 w = reinterpret_cast<const float4*>(&turns[wave][8 * u])[i];
      c[2 * i] = w.x, s[2 * i] = w.y, c[2 * i + 1] = w.z, s[2 * i + 1] = w.w;
    }
  }
  const bool cached = row >= 0 && row < a.n_cache_rows;

#pragma unroll
  for (int i = 0; i < QR_ITER; ++i) {
    const int h = first + i * HPG;
    if (i >= a.per || h >= n_heads) continue;
    if (h >= a.Hq + a.Hk) {  // v goes into the cache as it is
      if (cached) {
        T* dst = reinterpret_cast<T*>(a.v_cache) + (size_t)row * a.vc_ld + (size_t)(h - a.Hq - a.Hk) * D;
        x0[i].keep(dst + p0);
        x1[i].keep(dst + p1);
      }
      continue;
    }
    float x[16];
    x0[i].floats(x);
    x1[i].floats(x + 8);
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) sum = fmaf(x[j], x[j], sum);
    sum = group_sum<LPH>(sum);
    const float r = rsqrtf(sum * (1.f / D) + a.eps);
    const void* weight = h < a.Hq ? a.q_weight : a.k_weight;
    if (weight != nullptr) {
      float w[16];
      if (a.w_bf16) {
        Eight<bf16> w0, w1;
        w0.load(reinterpret_cast<const bf16*>(weight) + p0);
        w1.load(reinterpret_cast<const bf16*>(weight) + p1);
        w0.floats(w);
        w1.floats(w + 8);
      } else {
        Eight<float> w0, w1;
        w0.load(reinterpret_cast<const float*>(weight) + p0);
        w1.load(reinterpret_cast<const float*>(weight) + p1);
        w0.floats(w);
        w1.floats(w + 8);
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = x[j] * r * w[j];
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] *= r;
    }
    if (turned) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int ia = HALVES ? j : 2 * j, ib = HALVES ? j + 8 : 2 * j + 1;
        const float xa = x[ia], xb = x[ib];
        x[ia] = xa * c[j] - xb * s[j];
        x[ib] = xb * c[j] + xa * s[j];
      }
    }
    if (h < a.Hq) {
      T* dst = reinterpret_cast<T*>(a.q_out) + ((size_t)t * a.Hq + h) * D;
      Eight<T>::store(dst + p0, x);
      Eight<T>::store(dst + p1, x + 8);
    } else {
      if (a.k_out != nullptr) {
        T* dst = reinterpret_cast<T*>(a.k_out) + ((size_t)t * a.Hk + (h - a.Hq)) * D;
        Eight<T>::store(dst + p0, x);
        Eight<T>::store(dst + p1, x + 8);
      }
      if (cached) {
        T* dst = reinterpret_cast<T*>(a.k_cache) + (size_t)row * a.kc_ld + (size_t)(h - a.Hq) * D;
        Eight<T>::store(dst + p0, x);
        Eight<T>::store(dst + p1, x + 8);
      }
    }
  }
}

template <typename T, int D>
void launch_qk_rope(RopeArgs a, int interleaved, hipStream_t s) {
  constexpr int HPG = 64 / (D / 16);
  const int heads = a.Hq + a.Hk + (a.v != nullptr ? a.Hk : 0);
  a.groups = (heads + HPG - 1) / HPG;
  // few tokens: a wave for each group (its loads are all there is to wait for); else as few waves as hold the token's groups
  a.parts = (long)a.n_tokens * a.groups <= 4L * device_cus() ? a.groups : (a.groups + QR_ITER - 1) / QR_ITER;
  a.per = (a.groups + a.parts - 1) / a.parts;
  const long waves = (long)a.n_tokens * a.parts;
  const dim3 grid((unsigned)((waves + QR_NW - 1) / QR_NW)), block(64 * QR_NW);
  if (interleaved)
    hipLaunchKernelGGL((qk_rope_kernel<T, D, false>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((qk_rope_kernel<T, D, true>), grid, block, 0, s, a);
}

}  // namespace
}  // namespace zgdn

extern "C" int zattn_qk_norm_rope(const void* q, long q_ld, const void* k, long k_ld, const void* v, long v_ld, int dtype,
                                  const void* positions, int positions_i32, const void* inv_freq, int inv_freq_f32,
                                  const void* q_weight, const void* k_weight, int w_dtype, float eps, int interleaved,
                                  void* q_out, void* k_out, void* k_cache, long kc_ld, void* v_cache, long vc_ld,
                                  const int64_t* rows, long n_cache_rows, int n_tokens, int Hq, int Hk, int D, int R,
                                  void* stream) {
  using namespace zgdn;
  const char* fn = "zattn_qk_norm_rope";
  if (n_tokens < 0 || Hq < 1 || Hk < 1 || n_cache_rows < 0)
    return fail(ZGDN_EINVAL, "%s: bad sizes n_tokens=%d Hq=%d Hk=%d n_cache_rows=%ld", fn, n_tokens, Hq, Hk, n_cache_rows);
  if (D != 64 && D != 128) return fail(ZGDN_EUNSUPPORTED, "%s: D=%d (supported: 64 and 128)", fn, D);
  if (R < 0 || R > D || R % 16) return fail(ZGDN_EINVAL, "%s: R=%d (a multiple of 16, at most D=%d)", fn, R, D);
  for (int dt : {dtype, w_dtype})
    if (dt != ZGDN_F32 && dt != ZGDN_BF16) return fail(ZGDN_EINVAL, "%s: unknown dtype code %d", fn, dt);
  if (rows == nullptr ? k_cache != nullptr || v_cache != nullptr || v != nullptr
                      : n_cache_rows > 0 && (k_cache == nullptr || (v == nullptr) != (v_cache == nullptr)))
    return fail(ZGDN_EINVAL, "%s: rows and k_cache go together, and v and v_cache with them", fn);
  if (n_tokens > 0 && (!q || !k || !positions || !q_out || (R > 0 && !inv_freq)))
    return fail(ZGDN_EINVAL, "%s: null tensor pointer", fn);
  const int ve = dtype == ZGDN_F32 ? 4 : 8;
  const long most = 1L << 22, wq = (long)Hq * D, wk = (long)Hk * D;
  const bool caches = rows != nullptr, with_v = v != nullptr;
  auto bad = [&](long ld, long width) { return ld < width || ld > most || ld % ve; };
  if (bad(q_ld, wq) || bad(k_ld, wk) || (with_v && bad(v_ld, wk)) || (caches && bad(kc_ld, wk)) || (with_v && bad(vc_ld, wk)))
    return fail(ZGDN_EINVAL, "%s: row strides q=%ld k=%ld v=%ld k_cache=%ld v_cache=%ld (multiples of %d elements, at least a "
                "row, at most 2^22)", fn, q_ld, k_ld, v_ld, kc_ld, vc_ld, ve);
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_weight | (uintptr_t)k_weight | (uintptr_t)q_out |
       (uintptr_t)k_out | (uintptr_t)k_cache | (uintptr_t)v_cache) % 16)
    return fail(ZGDN_EINVAL, "%s: tensors need 16-byte aligned bases", fn);
  if ((uintptr_t)positions % (positions_i32 ? 4 : 8) || (uintptr_t)inv_freq % (inv_freq_f32 ? 4 : 8) || (uintptr_t)rows % 8)
    return fail(ZGDN_EINVAL, "%s: positions, inv_freq or rows not on a boundary of their type", fn);
  if (n_tokens == 0) return ZGDN_OK;
  if ((wq + 2 * wk) / 1024 / QR_ITER + 1 > (1L << 26) / n_tokens - 1)  // (waves: 2^32 threads at most in a grid)
    return fail(ZGDN_EUNSUPPORTED, "%s: n_tokens=%d x %d heads", fn, n_tokens, Hq + 2 * Hk);
  const size_t es = dtype == ZGDN_F32 ? 4 : 2, ws = w_dtype == ZGDN_F32 ? 4 : 2, n = (size_t)n_tokens;
  const size_t nc = (size_t)n_cache_rows;
  const Region out[] = {{q_out, n, wq * es, wq * es}, {k_out, n, wk * es, wk * es},
                        {k_cache, nc, wk * es, kc_ld * es}, {v_cache, nc, wk * es, vc_ld * es}};
  const Region in[] = {{q, n, wq * es, q_ld * es}, {k, n, wk * es, k_ld * es}, {v, n, wk * es, v_ld * es},
                       {positions, 1, n * (positions_i32 ? 4 : 8), n * 8}, {inv_freq, 1, (size_t)R / 2 * (inv_freq_f32 ? 4 : 8), 1},
                       {q_weight, 1, D * ws, D * ws}, {k_weight, 1, D * ws, D * ws}, {rows, 1, n * 8, n * 8}};
  bool meet = false;
  for (int i = 0; i < 4; ++i) {
    for (int j = 0; j < i; ++j) meet = meet || regions_meet(out[i], out[j]);
    for (const Region& r : in) meet = meet || regions_meet(out[i], r);
  }
  if (meet) return fail(ZGDN_EINVAL, "%s: an output overlaps another operand", fn);
  RopeArgs a{q, k, v, q_ld, k_ld, v_ld, positions, positions_i32, inv_freq, inv_freq_f32, q_weight, k_weight,
             w_dtype == ZGDN_BF16, eps, q_out, k_out, k_cache, v_cache, kc_ld, vc_ld, rows, n_cache_rows, n_tokens, Hq, Hk,
             R, 0, 0, 0};
  hipStream_t s = (hipStream_t)stream;
  if (dtype == ZGDN_F32)
    D == 128 ? launch_qk_rope<float, 128>(a, interleaved, s) : launch_qk_rope<float, 64>(a, interleaved, s);
  else
    D == 128 ? launch_qk_rope<bf16, 128>(a, interleaved, s) : launch_qk_rope<bf16, 64>(a, interleaved, s);
  return check_launch(fn);
}
