// The score function of the attention kernels beside the plain scaled product: scores
// capped by a tanh and biased by the distance to the query's own position.
//   s' = cap tanh(s scale / cap) + slope (t - position)      (no cap: s scale + ...)
// in log2 units, as the softmax takes them.  SC is the template parameter of the kernels:
// 0 the plain product (no code of this file runs), 1 biased only, 2 capped (and biased
// where there are slopes).
#pragma once

#include "common.h"

#include "../../include/oscar_operators.h"

namespace oscar {

struct Score {
  float scale2;         // scale log2(e)
  float cap2;           // cap log2(e)
  float exp2_scale;     // 2 log2(e) scale / cap
  float over_cap;       // scale / cap
  const float* slopes;  // [num_q_heads], or null
};

constexpr float kScoreLog2e = 1.4426950408889634f;

// The caps that are taken: up to 2^10, since a capped score keeps cap 2^-22 (capped2), which
// has to stay below the roundings of a probability (2^-12 of it); from 2^-20, since scale / cap
// has to be a finite number.
constexpr float kLeastCap = 9.5367431640625e-7f, kMostCap = 1024.f;
constexpr char kBadCap[] = "%s: soft_cap must lie in [2^-20, 1024], 0 for none";

// 0, 1 or 2 (see above); -22 for a cap that is not taken
inline int score_of(const oscarop_score_v1* score, float scale, Score* out) {
  *out = Score{};
  out->scale2 = scale * kScoreLog2e;
  if (score == nullptr) return 0;
  const float cap = score->soft_cap;
  if (cap != 0.f && !(cap >= kLeastCap && cap <= kMostCap)) return -22;
  out->slopes = score->alibi_slopes;
  if (cap == 0.f) return out->slopes != nullptr ? 1 : 0;
  out->cap2 = cap * kScoreLog2e;
  out->over_cap = scale / cap;
  out->exp2_scale = 2.f * kScoreLog2e * out->over_cap;
  return 2;
}

// the slope of a head in log2 units
__device__ __forceinline__ float slope2_of(const Score& f, int head) {
  return f.slopes != nullptr ? f.slopes[head] * kScoreLog2e : 0.f;
}

// tanh(u) = 1 - 2 / (e^(2u) + 1): within 2^-22 of tanh for every u, infinities included
__device__ __forceinline__ float capped2(const Score& f, float s) {
  const float e = __builtin_amdgcn_exp2f(s * f.exp2_scale);
  return fmaf(-2.f * f.cap2, __builtin_amdgcn_rcpf(e + 1.f), f.cap2);
}

// The same with the relative error of a few roundings also where the score is small
// against the cap, where the form above keeps cap 2^-22: the series of tanh up to u^11 for
// u < kSmallTanh (the first term left out is below 2^-25 of it there).
constexpr float kSmallTanh = 0.35f;
__device__ __forceinline__ float capped2_small(const Score& f, float s) {
  const float u = s * f.over_cap, t = u * u;
  float p = fmaf(t, -1382.f / 155925.f, 62.f / 2835.f);
  p = fmaf(t, p, -17.f / 315.f);
  p = fmaf(t, p, 2.f / 15.f);
  p = fmaf(t, p, -1.f / 3.f);
  const float x = s * f.scale2;
  return fmaf(x * t, p, x);
}
__device__ __forceinline__ float capped2_fine(const Score& f, float s) {
  return fabsf(s * f.over_cap) < kSmallTanh ? capped2_small(f, s) : capped2(f, s);
}

// the score of a raw product s at `distance` = t - position
template <int SC>
__device__ __forceinline__ float score2(const Score& f, float s, float slope2, float distance) {
  static_assert(SC == 1 || SC == 2);
  return fmaf(slope2, distance, SC == 2 ? capped2(f, s) : s * f.scale2);
}

}  // namespace oscar
