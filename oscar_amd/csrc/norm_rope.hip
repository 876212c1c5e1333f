// RMS norm of every query and key head with the position rotation, in one pass (gfx950).
//
// y = x / sqrt(mean(x^2) + eps) * (w + offset), then pairs of the first rotary_dim values
// turn by the token's angles.  A row (one head of one token) lies in head_dim / 8 lanes,
// 16 bytes of a 16-bit type each, so that its sum of squares is a reduction within 16 or
// 32 lanes and the other half of a rotated pair, rotary_dim / 2 values away, is whole lanes
// away.  Lanes take HPG heads of their token one after the other: the angles are loaded once
// for all of them and their rows are in flight together.  Bound by the rows' bytes.
#include <type_traits>

#include "common.h"
#include "store_quant.h"

#include "../../include/oscar_operators.h"

namespace oscar {

namespace {

constexpr int kThreads = 256;
// Four heads per lane group from this many bytes of rows on: fewer, longer waves, which cost
// more while there is one round of them and save once instructions and memory are the bound.
// One head / four, us: 600 tokens of 28 heads of 128 bf16 4.3 / 5.1, 1200 (9 MB) 7.4 / 6.9,
// 5000 18.8 / 16.7, 15361 (110 MB) 57.0 / 43.3 (5.1 TB/s in and out, a large copy's rate; 40.4 with
// interleaved pairs); 1200 of 7 heads of 256 4.3 / 5.4, 5000 (18 MB) 12.0 / 11.4;
// 5000 of 7 of 256 fp32 (36 MB) 17.3 / 15.6.
constexpr int64_t kManyBytes = 8 << 20;

typedef float __attribute__((ext_vector_type(2))) f32x2;
typedef __bf16 __attribute__((ext_vector_type(2))) bf16x2;
typedef _Float16 __attribute__((ext_vector_type(2))) f16x2;

struct NormRopeParams {
  oscarop_norm_rope_args_v1 a;
  FastDiv div_units;  // units of a token: HPG heads each
  uint32_t units;     // of all tokens
  int heads;          // num_q_heads + num_kv_heads
};

// 8 (or 4) elements at i of an array whose type is known at run time (uniform)
__device__ __forceinline__ void load8_of(const void* base, int32_t dtype, int64_t i, float* v) {
  if (dtype == OSCAR_BF16) load8<OSCAR_BF16>(base, i, v);
  else if (dtype == OSCAR_F16) load8<OSCAR_F16>(base, i, v);
  else load8<OSCAR_F32>(base, i, v);
}
__device__ __forceinline__ void load4_of(const void* base, int32_t dtype, int64_t i, float* v) {
  if (dtype == OSCAR_F32) {
    const f32x4 x = *(const f32x4*)((const float*)base + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = x[e];
  } else {
    const u32x2 x = *(const u32x2*)((const uint16_t*)base + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const unsigned short b = (unsigned short)(x[e / 2] >> (16 * (e & 1)));
      v[e] = dtype == OSCAR_BF16 ? bf16_bits_to_f32(b) : f16_bits_to_f32(b);
    }
  }
}

template <int DT>
__device__ __forceinline__ void store8(void* base, int64_t i, const float* v) {
  if constexpr (DT == OSCAR_F32) {
    store4<DT>(base, i, v);
    store4<DT>(base, i + 4, v + 4);
  } else {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {  // (to nearest even)
      if constexpr (DT == OSCAR_BF16) w[e] = __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{v[2 * e], v[2 * e + 1]}, bf16x2));
      else w[e] = __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{v[2 * e], v[2 * e + 1]}, f16x2));
    }
    *(u32x4*)((uint16_t*)base + i) = w;
  }
}

template <int D, int DT, int HPG>
__global__ __launch_bounds__(kThreads) void norm_rope_kernel(NormRopeParams P) {
  constexpr int L = D / 8;  // lanes of a row
  const oscarop_norm_rope_args_v1& A = P.a;
  const int lane = threadIdx.x & 63, e0 = 8 * (lane % L);
  const uint32_t unit = (uint32_t)blockIdx.x * (kThreads / L) + threadIdx.x / L;
  const bool live = unit < P.units;  // whole lane groups; all lanes stay for the exchanges
  const uint32_t t = fdiv(live ? unit : 0, P.div_units);
  const int head0 = (int)((live ? unit : 0) - t * P.div_units.d) * HPG;
  float x[HPG][8];
#pragma unroll
  for (int i = 0; i < HPG; ++i) {
    const int head = head0 + i < P.heads ? head0 + i : head0;
    if (head < A.num_q_heads) load8<DT>(A.q, t * A.q_stride_token + (int64_t)head * D + e0, x[i]);
    else load8<DT>(A.k, t * A.k_stride_token + (int64_t)(head - A.num_q_heads) * D + e0, x[i]);
  }
  const int64_t pos = A.positions_int64 ? ((const int64_t*)A.positions)[t] : ((const int32_t*)A.positions)[t];
  const bool known = pos >= 0 && pos < A.cos_sin_rows;
  // ---- this lane's angles: c and s of its 8 values' pairs (4 when interleaved), 1 and 0 past
  // the rotated ones
  const int half = (int)A.rotary_dim / 2;
  const bool turns = e0 < 2 * half, low = e0 < half;
  const int64_t table = (known ? pos : 0) * A.rotary_dim;
  float c[8], s[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    c[e] = 1.f;
    s[e] = 0.f;
  }
  if (turns) {
    if (A.interleaved) {
      load4_of(A.cos_sin, A.cos_sin_dtype, table + e0 / 2, c);
      load4_of(A.cos_sin, A.cos_sin_dtype, table + half + e0 / 2, s);
    } else {
      load8_of(A.cos_sin, A.cos_sin_dtype, table + (low ? e0 : e0 - half), c);
      load8_of(A.cos_sin, A.cos_sin_dtype, table + half + (low ? e0 : e0 - half), s);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] = low ? -s[e] : s[e];
    }
  }
  const bool all_turn = 2 * half == D;
  const int other = !turns ? lane : low ? lane + half / 8 : lane - half / 8;  // the lane of the pairs' other values
  float w[8];
#pragma unroll
  for (int i = 0; i < HPG; ++i) {
    const int head = head0 + i;
    const bool is_q = head < A.num_q_heads;
    if (i == 0 || head == A.num_q_heads) {  // another side's weights
      const void* weight = is_q ? A.q_weight : A.k_weight;
      if (weight != nullptr) {
        load8_of(weight, A.weight_dtype, e0, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] += A.weight_offset;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = 1.f;
      }
    }
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf(x[i][e], x[i][e], sum);
    sum += dpp_row<kDppXor1>(sum);
    sum += dpp_row<kDppXor2>(sum);
    sum += dpp_row<kDppHalfMirror>(sum);
    sum += dpp_row<kDppMirror>(sum);
    if constexpr (L == 32) sum += swizzle_xor16(sum);
    const float r = known ? 1.f / sqrtf(sum * (1.f / D) + A.eps) : NAN;
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[i][e] = x[i][e] * r * w[e];
    if (A.interleaved) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        y[2 * e] = fmaf(x[i][2 * e], c[e], -(x[i][2 * e + 1] * s[e]));
        y[2 * e + 1] = fmaf(x[i][2 * e + 1], c[e], x[i][2 * e] * s[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = fmaf(x[i][e], c[e], __shfl(x[i][e], other) * s[e]);
    }
    if (!all_turn) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = turns ? y[e] : x[i][e];  // (0 times an infinity beside it would be NaN)
    }
    if (!live || head >= P.heads) continue;
    if (is_q) store8<DT>(A.q_out, t * A.q_out_stride_token + (int64_t)head * D + e0, y);
    else store8<DT>(A.k_out, t * A.k_out_stride_token + (int64_t)(head - A.num_q_heads) * D + e0, y);
  }
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
  constexpr int64_t kMostHeads = 1 << 20, kMostRows = 1ll << 31;  // below
  const bool many = a.num_q_heads >= kMostHeads || a.num_kv_heads >= kMostHeads;
  const int64_t heads = many ? kMostHeads : a.num_q_heads + a.num_kv_heads;
  if (a.num_tokens == 0 || heads == 0) return 0;
  if (heads >= kMostHeads || a.num_tokens >= kMostRows || a.num_tokens * heads >= kMostRows)
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
  const int hpg = a.num_tokens * heads * D * (16 / v) >= kManyBytes ? 4 : 1;
  const int64_t units = (heads + hpg - 1) / hpg, per = kThreads / (D / 8);
  p.div_units = FastDiv::of(units);
  p.units = (uint32_t)(a.num_tokens * units);
  p.heads = (int)heads;
  const dim3 grid((unsigned)((p.units + per - 1) / per));
  hipStream_t s = (hipStream_t)stream;
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, s, p); };
  auto by_heads = [&](auto d, auto dt) {
    constexpr int DD = decltype(d)::value, DT = decltype(dt)::value;
    hpg == 4 ? launch(norm_rope_kernel<DD, DT, 4>) : launch(norm_rope_kernel<DD, DT, 1>);
  };
  using std::integral_constant;
  auto by_type = [&](auto d) {
    if (a.dtype == OSCAR_BF16) by_heads(d, integral_constant<int, OSCAR_BF16>{});
    else if (a.dtype == OSCAR_F16) by_heads(d, integral_constant<int, OSCAR_F16>{});
    else by_heads(d, integral_constant<int, OSCAR_F32>{});
  };
  if (D == 256) by_type(integral_constant<int, 256>{});
  else by_type(integral_constant<int, 128>{});
  OSCAR_CHECK_LAUNCH("norm_rope_kernel");
  return 0;
}
