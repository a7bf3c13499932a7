// Linear attention's single-token step on the streams' states, in place: S = exp(g) S + v k^T, o = S (scale q).
//
// HBM-bound: the state is read and written once, 8 V K bytes a stream and head, next to which the rest is nothing. A row
// of K state entries is held by K / 8 lanes (two 16-byte pieces each), so that a wave's load covers whole rows; o is one
// reduction a row over those lanes. A pass of a wave is 64 / (K / 8) rows of one stream and head (4 at K = 128, 8 at 64).
// Where there is work for three workgroups a CU, waves walk tiles of 4 passes with the next tile's loads issued before the
// current one is updated and stored; below, a tile is one pass and a wave has one (64 streams of 16 heads of 128 x 128:
// 20.8 us; one stream of 4 heads: 3.3).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "gdn_common.h"
#include "zonos3_linear.h"

namespace zgdn {
namespace {

constexpr int LS_NW = 4;  // waves a workgroup

struct StepArgs {
  const void *q, *k, *v, *g;
  long q_ld, k_ld, v_ld, g_ld;
  int g_bf16;
  float* state;
  const int64_t* slots;
  int n_slots;
  void* o;
  int B, Hk, Hv, V, n_tiles;
  float scale;
};

template <typename TIn>
__device__ __forceinline__ float4 ls_load4(const void* p, size_t i) {
  return io<TIn>::load4(reinterpret_cast<const TIn*>(p) + i);
}

// Where stream b's state is: its row of the table, or -1 where its slot is outside it or an earlier stream has it.
__device__ __forceinline__ long stream_row(const StepArgs& a, int b) {
  if (a.slots == nullptr) return b;
  const int64_t s = a.slots[b];
  if (s < 0 || s >= a.n_slots) return -1;
  const int l = threadIdx.x & 63;
  for (int i0 = 0; i0 < b; i0 += 64)
    if (__ballot(i0 + l < b && a.slots[min(i0 + l, b)] == s)) return -1;
  return (long)s;
}

template <typename TIn, int GPT>
struct LsTile {
  float4 s[GPT][2];
  float4 ka, kb, qa, qb;
  float vj[GPT];
  float g;
  long row;  // (wave-uniform)
};

template <typename TIn, int K, int GPT>
__global__ __launch_bounds__(64 * LS_NW) void lin_step_kernel(StepArgs a) {
  constexpr int LPR = K / 8, RPP = 64 / LPR, ROWS = RPP * GPT;
  const int lane = threadIdx.x & 63, sub = lane % LPR, rsub = lane / LPR;
  const int c0 = 4 * sub, c1 = K / 2 + 4 * sub;
  const int tph = a.V / ROWS;
  using Tile = LsTile<TIn, GPT>;

  auto load = [&](int ti, Tile& x) {
    const int nh = ti / tph, b = nh / a.Hv, h = nh - b * a.Hv, v0 = (ti - nh * tph) * ROWS + rsub;
    const size_t hk = (size_t)(h / (a.Hv / a.Hk)) * K;
    x.ka = ls_load4<TIn>(a.k, (size_t)b * a.k_ld + hk + c0);
    x.kb = ls_load4<TIn>(a.k, (size_t)b * a.k_ld + hk + c1);
    x.qa = ls_load4<TIn>(a.q, (size_t)b * a.q_ld + hk + c0);
    x.qb = ls_load4<TIn>(a.q, (size_t)b * a.q_ld + hk + c1);
#pragma unroll
    for (int j = 0; j < GPT; ++j)
      x.vj[j] = io<TIn>::load(reinterpret_cast<const TIn*>(a.v) + (size_t)b * a.v_ld + (size_t)h * a.V + v0 + j * RPP);
    const size_t gi = (size_t)b * a.g_ld + h;
    x.g = a.g_bf16 ? bf16_to_f32(reinterpret_cast<const uint16_t*>(a.g)[gi]) : reinterpret_cast<const float*>(a.g)[gi];
    x.row = stream_row(a, b);
    if (x.row >= 0) {
      const float* src = a.state + ((size_t)x.row * a.Hv + h) * a.V * K + (size_t)v0 * K;
#pragma unroll
      for (int j = 0; j < GPT; ++j) {
        x.s[j][0] = *reinterpret_cast<const float4*>(src + (size_t)j * RPP * K + c0);
        x.s[j][1] = *reinterpret_cast<const float4*>(src + (size_t)j * RPP * K + c1);
      }
    }
  };

  auto process = [&](int ti, const Tile& x) {
    const int nh = ti / tph, b = nh / a.Hv, h = nh - b * a.Hv, v0 = (ti - nh * tph) * ROWS + rsub;
    TIn* o = reinterpret_cast<TIn*>(a.o) + (size_t)nh * a.V + v0;
    if (x.row < 0) {
      if (sub == 0) {
#pragma unroll
        for (int j = 0; j < GPT; ++j) io<TIn>::store(o + j * RPP, 0.f);
      }
      return;
    }
    // exp(g) S as S + S expm1(g) for slow decays: the factor's rounding, the same at every step where g is fixed, would
    // otherwise grow with the length of the memory
    const bool slow = x.g > -0.5f;
    const float add = slow ? expm1f(x.g) : expf(x.g), mul = slow ? 1.f : 0.f;
    const float kk[8] = {x.ka.x, x.ka.y, x.ka.z, x.ka.w, x.kb.x, x.kb.y, x.kb.z, x.kb.w};
    const float qq[8] = {x.qa.x, x.qa.y, x.qa.z, x.qa.w, x.qb.x, x.qb.y, x.qb.z, x.qb.w};
    float* dst = a.state + ((size_t)x.row * a.Hv + h) * a.V * K + (size_t)v0 * K;
#pragma unroll
    for (int j = 0; j < GPT; ++j) {
      float st[8] = {x.s[j][0].x, x.s[j][0].y, x.s[j][0].z, x.s[j][0].w, x.s[j][1].x, x.s[j][1].y, x.s[j][1].z, x.s[j][1].w};
      float acc = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        st[i] = fmaf(st[i], add, fmaf(x.vj[j], kk[i], mul * st[i]));
        acc = fmaf(st[i], qq[i], acc);
      }
      *reinterpret_cast<float4*>(dst + (size_t)j * RPP * K + c0) = make_float4(st[0], st[1], st[2], st[3]);
      *reinterpret_cast<float4*>(dst + (size_t)j * RPP * K + c1) = make_float4(st[4], st[5], st[6], st[7]);
      acc = group_sum<LPR>(acc);
      if (sub == 0) io<TIn>::store(o + j * RPP, a.scale * acc);
    }
  };

  const int stride = gridDim.x * LS_NW;
  int ti = blockIdx.x * LS_NW + wave_id();
  if (ti >= a.n_tiles) return;
  Tile b0, b1;
  load(ti, b0);
  if (stride >= a.n_tiles) {  // one tile a wave
    process(ti, b0);
    return;
  }
  const int last = a.n_tiles - 1;
  for (;;) {  // two buffers in turn (the load after a wave's last tile repeats the last one and is not used)
    const int t1 = ti + stride;
    load(min(t1, last), b1);
    process(ti, b0);
    if (t1 >= a.n_tiles) break;
    const int t2 = t1 + stride;
    load(min(t2, last), b0);
    process(t1, b1);
    if (t2 >= a.n_tiles) break;
    ti = t2;
  }
}

template <typename TIn, int K>
void launch_lin_step(StepArgs a, hipStream_t s) {
  constexpr int RPP = 64 / (K / 8), PER_CU = 3;
  const long heads = (long)a.B * a.Hv, n_cu = device_cus();
  const long tiles4 = heads * (a.V / (4 * RPP));
  if (tiles4 >= PER_CU * n_cu * LS_NW) {
    a.n_tiles = (int)tiles4;
    hipLaunchKernelGGL((lin_step_kernel<TIn, K, 4>), dim3((unsigned)(PER_CU * n_cu)), dim3(64 * LS_NW), 0, s, a);
  } else {
    a.n_tiles = (int)(heads * (a.V / RPP));
    hipLaunchKernelGGL((lin_step_kernel<TIn, K, 1>), dim3((unsigned)((a.n_tiles + LS_NW - 1) / LS_NW)), dim3(64 * LS_NW), 0, s, a);
  }
}

}  // namespace
}  // namespace zgdn

extern "C" int zlin_attn_step(const void* q, long q_ld, const void* k, long k_ld, const void* v, long v_ld, int dtype,
                              const void* g, long g_ld, int g_dtype, float* state, const int64_t* slots, int n_slots,
                              void* o, int B, int Hk, int Hv, int K, int V, float scale, void* stream) {
  using namespace zgdn;
  const char* fn = "zlin_attn_step";
  if (B < 0 || Hk < 1 || Hv < 1 || n_slots < 0)
    return fail(ZGDN_EINVAL, "%s: bad sizes B=%d Hk=%d Hv=%d n_slots=%d", fn, B, Hk, Hv, n_slots);
  if (Hv % Hk) return fail(ZGDN_EINVAL, "%s: Hv=%d is not a multiple of Hk=%d", fn, Hv, Hk);
  if ((K != 64 && K != 128) || (V != 64 && V != 128))
    return fail(ZGDN_EUNSUPPORTED, "%s: K=%d V=%d (supported: 64 and 128 each)", fn, K, V);
  for (int dt : {dtype, g_dtype})
    if (dt != ZGDN_F32 && dt != ZGDN_BF16) return fail(ZGDN_EINVAL, "%s: unknown dtype code %d", fn, dt);
  if (B > 0 && (!q || !k || !v || !g || !o || !state)) return fail(ZGDN_EINVAL, "%s: null tensor pointer", fn);
  if (slots == nullptr && n_slots != B)
    return fail(ZGDN_EINVAL, "%s: states of %d streams for B=%d without slots", fn, n_slots, B);
  if (g_ld == 0 ? g_dtype != ZGDN_F32 : g_ld < Hv)
    return fail(ZGDN_EINVAL, "%s: g rows %ld apart (at least %d, or 0 for float32 decays a head)", fn, g_ld, Hv);
  const int ve = dtype == ZGDN_F32 ? 4 : 8;
  if (q_ld < (long)Hk * K || k_ld < (long)Hk * K || v_ld < (long)Hv * V || q_ld % ve || k_ld % ve || v_ld % ve)
    return fail(ZGDN_EINVAL, "%s: row strides q=%ld k=%ld v=%ld (multiples of %d elements, at least a row)", fn, q_ld, k_ld,
                v_ld, ve);
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o | (uintptr_t)state) % 16)
    return fail(ZGDN_EINVAL, "%s: q, k, v, o and state need 16-byte aligned bases", fn);
  if ((long)B * Hv * V >= INT32_MAX) return fail(ZGDN_EUNSUPPORTED, "%s: B=%d x Hv=%d x V=%d rows", fn, B, Hv, V);
  if (B == 0) return ZGDN_OK;
  const size_t es = dtype == ZGDN_F32 ? 4 : 2, ge = g_dtype == ZGDN_F32 ? 4 : 2, n = (size_t)B;
  const size_t table = (size_t)n_slots * Hv * V * K * 4;
  const Region out = {o, n, (size_t)Hv * V * es, (size_t)Hv * V * es}, st = {state, 1, table, table};
  const Region in[] = {{q, n, (size_t)Hk * K * es, q_ld * es}, {k, n, (size_t)Hk * K * es, k_ld * es},
                       {v, n, (size_t)Hv * V * es, v_ld * es}, {g, g_ld == 0 ? 1 : n, Hv * ge, g_ld == 0 ? Hv * ge : g_ld * ge},
                       {slots, 1, n * 8, n * 8}};
  bool meet = regions_meet(out, st);
  for (const Region& r : in) meet = meet || regions_meet(out, r) || regions_meet(st, r);
  if (meet) return fail(ZGDN_EINVAL, "%s: o or state overlap another operand", fn);
  StepArgs a{q, k, v, g, q_ld, k_ld, v_ld, g_ld, g_dtype == ZGDN_BF16, state, slots, n_slots, o, B, Hk, Hv, V, 0, scale};
  hipStream_t s = (hipStream_t)stream;
  if (dtype == ZGDN_F32)
    K == 128 ? launch_lin_step<float, 128>(a, s) : launch_lin_step<float, 64>(a, s);
  else
    K == 128 ? launch_lin_step<bf16, 128>(a, s) : launch_lin_step<bf16, 64>(a, s);
  return check_launch(fn);
}
