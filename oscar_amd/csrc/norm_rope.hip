// RMS norm of every query and key head with the position rotation, in one pass (gfx950).
//
// y = x / sqrt(mean(x^2) + eps) * (w + offset), then pairs of the first rotary_dim values
// turn by the token's angles.  A row (one head of one token) lies in head_dim / 8 lanes,
// 16 bytes of a 16-bit type each, so that its sum of squares is a reduction within 16 or
// 32 lanes and the other half of a rotated pair, rotary_dim / 2 values away, is whole lanes
// away.
#include "common.h"
#include "store_quant.h"

#include "../../include/oscar_operators.h"

namespace oscar {

namespace {

constexpr int kThreads = 256;

struct NormRopeParams {
  oscarop_norm_rope_args_v1 a;
  FastDiv div_heads;  // num_q_heads + num_kv_heads
  uint32_t rows;      // tokens x heads
};

// 8 elements at i of an array whose type is known at run time (uniform)
__device__ __forceinline__ void load8_of(const void* base, int32_t dtype, int64_t i, float* v) {
  if (dtype == OSCAR_BF16) load8<OSCAR_BF16>(base, i, v);
  else if (dtype == OSCAR_F16) load8<OSCAR_F16>(base, i, v);
  else load8<OSCAR_F32>(base, i, v);
}

template <int DT>
__device__ __forceinline__ void store8(void* base, int64_t i, const float* v) {
  if constexpr (DT == OSCAR_F32) {
    store4<DT>(base, i, v);
    store4<DT>(base, i + 4, v + 4);
  } else {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (DT == OSCAR_BF16)
        w[e] = f32_to_bf16_bits(v[2 * e]) | ((unsigned)f32_to_bf16_bits(v[2 * e + 1]) << 16);
      else
        w[e] = f32_to_f16_bits(v[2 * e]) | ((unsigned)f32_to_f16_bits(v[2 * e + 1]) << 16);
    }
    *(u32x4*)((uint16_t*)base + i) = w;
  }
}

template <int D, int DT>
__global__ __launch_bounds__(kThreads) void norm_rope_kernel(NormRopeParams P) {
  constexpr int L = D / 8;  // lanes of a row
  const oscarop_norm_rope_args_v1& A = P.a;
  const int lane = threadIdx.x & 63, e0 = 8 * (lane % L);
  const uint32_t row = (uint32_t)blockIdx.x * (kThreads / L) + threadIdx.x / L;
  const bool live = row < P.rows;  // whole lane groups; all lanes stay for the exchanges
  const uint32_t t = fdiv(live ? row : 0, P.div_heads);
  const int head = (int)((live ? row : 0) - t * P.div_heads.d);
  const bool is_q = head < A.num_q_heads;
  const int64_t in = is_q ? t * A.q_stride_token + (int64_t)head * D
                          : t * A.k_stride_token + (int64_t)(head - A.num_q_heads) * D;
  float x[8], w[8];
  load8<DT>(is_q ? A.q : A.k, in + e0, x);
  const int64_t pos = A.positions_int64 ? ((const int64_t*)A.positions)[t] : ((const int32_t*)A.positions)[t];
  const bool known = pos >= 0 && pos < A.cos_sin_rows;
  const void* weight = is_q ? A.q_weight : A.k_weight;
  if (weight != nullptr) {
    load8_of(weight, A.weight_dtype, e0, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] += A.weight_offset;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = 1.f;
  }
  float sum = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) sum = fmaf(x[e], x[e], sum);
  sum += dpp_row<kDppXor1>(sum);
  sum += dpp_row<kDppXor2>(sum);
  sum += dpp_row<kDppHalfMirror>(sum);
  sum += dpp_row<kDppMirror>(sum);
  if constexpr (L == 32) sum += swizzle_xor16(sum);
  const float r = 1.f / sqrtf(sum * (1.f / D) + A.eps);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = x[e] * r * w[e];
  const int half = (int)A.rotary_dim / 2;
  const int64_t table = (known ? pos : 0) * A.rotary_dim;
  float y[8];
  if (A.interleaved) {
    if (e0 < 2 * half) {
      float c[4], s[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        c[e] = load_elem(A.cos_sin, A.cos_sin_dtype, table + e0 / 2 + e);
        s[e] = load_elem(A.cos_sin, A.cos_sin_dtype, table + half + e0 / 2 + e);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        y[2 * e] = fmaf(x[2 * e], c[e], -(x[2 * e + 1] * s[e]));
        y[2 * e + 1] = fmaf(x[2 * e + 1], c[e], x[2 * e] * s[e]);
      }
    }
  } else {
    const bool low = e0 < half;
    const int other = lane + (low ? half / 8 : -(half / 8));  // a lane of the same row where e0 < rotary_dim
    float p[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = __shfl(x[e], e0 < 2 * half ? other : lane);
    if (e0 < 2 * half) {
      float c[8], s[8];
      load8_of(A.cos_sin, A.cos_sin_dtype, table + (low ? e0 : e0 - half), c);
      load8_of(A.cos_sin, A.cos_sin_dtype, table + half + (low ? e0 : e0 - half), s);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = fmaf(x[e], c[e], (low ? -p[e] : p[e]) * s[e]);
    }
  }
  if (!live) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    y[e] = e0 < 2 * half ? y[e] : x[e];
    y[e] = known ? y[e] : NAN;
  }
  if (is_q) store8<DT>(A.q_out, t * A.q_out_stride_token + (int64_t)head * D + e0, y);
  else store8<DT>(A.k_out, t * A.k_out_stride_token + (int64_t)(head - A.num_q_heads) * D + e0, y);
}

bool aligned16(const void* p) { return (((uintptr_t)p) & 15) == 0; }

}  // namespace

}  // namespace oscar

using namespace oscar;

extern "C" int oscarop_norm_rope_v1(const oscarop_norm_rope_args_v1* args, void* stream) {
  const char* name = "oscarop_norm_rope_v1";
  if (!args) return fail(-22, "%s: null args", name);
  const oscarop_norm_rope_args_v1& a = *args;
  const int64_t D = a.head_dim;
  if (D != 128 && D != 256) return fail(-22, "%s: head_dim %lld unsupported (128/256)", name, (long long)D);
  if (a.num_tokens < 0 || a.num_q_heads < 0 || a.num_kv_heads < 0) return fail(-22, "%s: negative size", name);
  auto is_dtype = [](int32_t t) { return t == OSCAR_F32 || t == OSCAR_F16 || t == OSCAR_BF16; };
  if (!is_dtype(a.dtype) || !is_dtype(a.cos_sin_dtype) || ((a.q_weight || a.k_weight) && !is_dtype(a.weight_dtype)))
    return fail(-22, "%s: types must be fp32, fp16 or bf16", name);
  if (!(a.eps >= 0.f)) return fail(-22, "%s: eps must not be negative", name);
  if (a.rotary_dim < 16 || a.rotary_dim > D || a.rotary_dim % 16)
    return fail(-22, "%s: rotary_dim %lld must be a multiple of 16 up to head_dim", name, (long long)a.rotary_dim);
  const int64_t heads = a.num_q_heads + a.num_kv_heads;
  if (a.num_tokens == 0 || heads == 0) return 0;
  if (heads >= (1 << 20) || a.num_tokens * heads >= (1ll << 31))
    return fail(-22, "%s: too many rows for one call", name);
  if (!a.positions || !a.cos_sin || a.cos_sin_rows < 1 || (a.num_q_heads && (!a.q || !a.q_out)) ||
      (a.num_kv_heads && (!a.k || !a.k_out)))
    return fail(-22, "%s: missing pointer", name);
  const int64_t v = a.dtype == OSCAR_F32 ? 4 : 8;  // elements of 16 bytes
  if (!aligned16(a.cos_sin) || !aligned16(a.q_weight) || !aligned16(a.k_weight) ||
      (a.num_q_heads && (!aligned16(a.q) || !aligned16(a.q_out) || a.q_stride_token % v || a.q_out_stride_token % v)) ||
      (a.num_kv_heads && (!aligned16(a.k) || !aligned16(a.k_out) || a.k_stride_token % v || a.k_out_stride_token % v)))
    return fail(-22, "%s: rows, weights and the table must be 16-byte aligned", name);
  // (a broadcast output would have several rows write one place)
  if (a.num_tokens > 1 && ((a.num_q_heads && a.q_out_stride_token < a.num_q_heads * D) ||
                           (a.num_kv_heads && a.k_out_stride_token < a.num_kv_heads * D)))
    return fail(-22, "%s: output tokens overlap", name);
  NormRopeParams p{};
  p.a = a;
  p.div_heads = FastDiv::of(heads);
  p.rows = (uint32_t)(a.num_tokens * heads);
  const int64_t per = kThreads / (D / 8);
  const dim3 grid((unsigned)((p.rows + per - 1) / per));
  hipStream_t s = (hipStream_t)stream;
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, s, p); };
  if (D == 256) {
    if (a.dtype == OSCAR_BF16) launch(norm_rope_kernel<256, OSCAR_BF16>);
    else if (a.dtype == OSCAR_F16) launch(norm_rope_kernel<256, OSCAR_F16>);
    else launch(norm_rope_kernel<256, OSCAR_F32>);
  } else {
    if (a.dtype == OSCAR_BF16) launch(norm_rope_kernel<128, OSCAR_BF16>);
    else if (a.dtype == OSCAR_F16) launch(norm_rope_kernel<128, OSCAR_F16>);
    else launch(norm_rope_kernel<128, OSCAR_F32>);
  }
  OSCAR_CHECK_LAUNCH("norm_rope_kernel");
  return 0;
}
