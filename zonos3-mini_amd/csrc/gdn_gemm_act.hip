// y = act(x w^T + bias) + residual on bf16 MFMA, fp32 sums, the epilogue in fp32, rounded once.
//
// Tiles are computed transposed (A = rows of w, B = rows of x), so that a lane of a D tile holds 4 neighbouring columns
// of one row of y: bias, residual and y are 8-byte accesses.
#include <algorithm>
#include <atomic>

#include "gdn_common.h"
#include "zonos3_linear.h"

namespace zgdn {
namespace {

typedef __bf16 abf16x8 __attribute__((ext_vector_type(8)));
typedef float af32x4 __attribute__((ext_vector_type(4)));

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
  int vec;  // y and the residual take 8-byte accesses
};

__device__ __forceinline__ float act_of(float x, int act) {
  switch (act) {
    case ZLIN_RELU:
      return x > 0.f || x != x ? x : 0.f;
    case ZLIN_SILU:
      return x / (1.f + __expf(-x));
    case ZLIN_GELU:
      return 0.5f * x * (1.f + erff(x * 0.70710678118654752f));
    case ZLIN_GELU_TANH:  // 0.5 (1 + tanh u) = 1 / (1 + exp(-2 u))
      return x / (1.f + __expf(-2.f * 0.79788456080286536f * (x + 0.044715f * x * x * x)));
    default:
      return x;
  }
}

// Four columns n .. n + 3 of row m.
__device__ __forceinline__ void finish(const ActArgs& a, int m, int n, af32x4 c) {
  if (m >= a.M || n >= a.N) return;
  const int left = min(4, a.N - n);
  if (a.bias != nullptr) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = n + min(e, left - 1);
      c[e] += a.bias_bf16 ? bf16_to_f32(reinterpret_cast<const uint16_t*>(a.bias)[i]) : reinterpret_cast<const float*>(a.bias)[i];
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) c[e] = act_of(c[e], a.act);
  const size_t yi = (size_t)m * a.y_ld + n, ri = (size_t)m * a.r_ld + n;
  if (a.vec && left == 4) {
    if (a.res != nullptr) {
      const uint2 r = *reinterpret_cast<const uint2*>(a.res + ri);
      c[0] += __uint_as_float(r.x << 16);
      c[1] += __uint_as_float(r.x & 0xffff0000u);
      c[2] += __uint_as_float(r.y << 16);
      c[3] += __uint_as_float(r.y & 0xffff0000u);
    }
    *reinterpret_cast<uint2*>(a.y + yi) = make_uint2(pack_bf16x2(c[0], c[1]), pack_bf16x2(c[2], c[3]));
  } else {
    for (int e = 0; e < left; ++e) {
      float v = c[e];
      if (a.res != nullptr) v += bf16_to_f32(a.res[ri + e]);
      a.y[yi + e] = f32_to_bf16(v);
    }
  }
}

// Any sizes and alignments: 64 x 64 tiles, 4 waves of 32 x 32, blocks of 64 of K through LDS (128-byte rows, 16-byte
// chunks swizzled by row), each thread fetching 8 elements of a row at a time, one by one where the rows do not start
// on 16-byte boundaries or K ends within them.
template <bool WIDE>
__global__ __launch_bounds__(256) void gemm_act_any_kernel(ActArgs a) {
  __shared__ uint4 sx[64 * 8], sw[64 * 8];
  const int n0 = blockIdx.x * 64, m0 = blockIdx.y * 64;
  const int wave = wave_id(), l = threadIdx.x & 63, m = l & 15, g = l >> 4;
  const int wm = (wave & 1) * 32, wn = (wave >> 1) * 32;
  af32x4 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = af32x4{0.f, 0.f, 0.f, 0.f};
  auto fetch = [&](const uint16_t* base, long ld, int row, int rows, int k) {
    uint4 r = make_uint4(0, 0, 0, 0);
    if (row >= rows || k >= a.K) return r;
    const uint16_t* p = base + (size_t)row * ld + k;
    if (WIDE && k + 8 <= a.K) return *reinterpret_cast<const uint4*>(p);
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = k + i < a.K ? p[i] : 0;
    return make_uint4(u[0] | u[1] << 16, u[2] | u[3] << 16, u[4] | u[5] << 16, u[6] | u[7] << 16);
  };
  for (int k0 = 0; k0 < a.K; k0 += 64) {
    uint4 fx[2], fw[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int e = threadIdx.x + 256 * i, r = e >> 3, c = e & 7;
      fx[i] = fetch(a.x, a.x_ld, m0 + r, a.M, k0 + 8 * c);
      fw[i] = fetch(a.w, a.w_ld, n0 + r, a.N, k0 + 8 * c);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int e = threadIdx.x + 256 * i, r = e >> 3, c = e & 7;
      sx[r * 8 + (c ^ (r >> 1 & 7))] = fx[i];
      sw[r * 8 + (c ^ (r >> 1 & 7))] = fw[i];
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
        for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[i], fb[j], acc[i][j], 0, 0, 0);
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) finish(a, m0 + wm + 16 * j + m, n0 + wn + 16 * i + 4 * g, acc[i][j]);
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
  if (M > INT32_MAX - 64 || N > INT32_MAX - 64 || K > INT32_MAX - 64 || (M + 63) / 64 > 65535)
    return fail(ZGDN_EUNSUPPORTED, "%s: M=%d N=%d K=%d", fn, M, N, K);
  ActArgs a{(const uint16_t*)x, (const uint16_t*)w, x_ld, w_ld, bias, bias_dtype == ZGDN_BF16, act,
            (const uint16_t*)residual, residual != nullptr ? r_ld : 0, (uint16_t*)y, y_ld, M, N, K, 0};
  a.vec = y_ld % 4 == 0 && (uintptr_t)y % 8 == 0 && (residual == nullptr || (r_ld % 4 == 0 && (uintptr_t)residual % 8 == 0));
  const bool wide = x_ld % 8 == 0 && w_ld % 8 == 0 && ((uintptr_t)x | (uintptr_t)w) % 16 == 0;
  const dim3 grid((N + 63) / 64, (M + 63) / 64);
  if (wide)
    hipLaunchKernelGGL((gemm_act_any_kernel<true>), grid, dim3(256), 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL((gemm_act_any_kernel<false>), grid, dim3(256), 0, (hipStream_t)stream, a);
  return check_launch(fn);
}
