// The attention weight that every cached token received from a batch's queries, added to
// what it had: weights[r][h][t] += sum over the rows of request r that KV head h serves of
// exp(s' - lse), s' the row's score of key t (score.h) and lse the row's log-sum-exp, as the
// attention call left it.  Keys are those the attention reads: the packed INT2 history, FP32
// window copies where the owner tag matches, and the current chunk's rows.
//
// A wave holds the K operands of one 32-token tile in registers for all rows and adds up
// probabilities per key, lane by lane (lane l: row l % 32 of a row block), so that the sum
// over the rows crosses lanes once, at the end.  The query operands of a block of 32 rows
// go through LDS, shared by the workgroup's waves.  Every weight has one owner, so nothing
// is atomic and results do not depend on the order of workgroups.
#include <type_traits>

#include "common.h"
#include "int2_tile.h"
#include "score.h"

#include "../../include/oscar_operators.h"

namespace oscar {

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kTile = 32;
constexpr float kLn2 = 0.6931471805599453f;

struct WeightsParams {
  oscarop_weights_args_v1 a;
  oscar_staging_v1 st;
  int has_stage;
  int group;  // Hq / Hk
  Score sc;
};

template <int D, int QT, int SC>
__global__ __launch_bounds__(kThreads) void weights_kernel(WeightsParams P) {
  constexpr int NCH = D / 32;  // 16-element chunks per lane half
  const oscarop_weights_args_v1& A = P.a;
  const int tid = threadIdx.x, lane = tid & 63, m = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int req = blockIdx.z, kvh = blockIdx.y, G = P.group;
  const int qa = A.query_start_loc[req], nq = A.query_start_loc[req + 1] - qa, seq = A.seq_lens[req];
  if (nq < 1) return;
  const bool has_new = A.k_new != nullptr;
  const int hist = has_new ? seq - nq : seq;
  const int before = seq - nq;  // query i sees keys [0, before + i + 1)
  const int bs = (int)A.cache.block_size;
  const int64_t hk = A.cache.num_kv_heads;
  float* out = A.weights + req * A.weights_stride_request + kvh * A.weights_stride_head;
  // a request that does not fit the call's arrays reads nothing and turns its weights, as
  // far as there are any, into NaN
  const bool bad = qa < 0 || (int64_t)qa + nq > A.num_tokens || hist < 0 || seq > A.weights_cols ||
                   (hist > 0 && (hist - 1) / bs >= A.block_table_cols);
  if (bad) {
    for (int64_t t = (int64_t)blockIdx.x * kThreads + tid; t < A.weights_cols && t < seq; t += (int64_t)gridDim.x * kThreads)
      out[t] = NAN;
    return;
  }
  __shared__ __attribute__((aligned(16))) u32x4 s_q[2 * NCH][64];  // Q^T operands of a row block
  const int nrows = nq * G;
  for (int tb = blockIdx.x * (kWaves * kTile); tb < seq; tb += gridDim.x * (kWaves * kTile)) {
    // ---- this wave's tile: lane (token m, half g) holds the K operands of its half
    const int t0 = tb + wave * kTile, t = t0 + m;
    u32x4 kop[2 * NCH];
    {
      int64_t blk = 0;
      bool staged = false;
      int64_t seat = 0;
      const int off = t % bs;
      if (t0 < hist) {
        blk = A.block_table[req * A.block_table_stride + t0 / bs];
        blk = blk < 0 || blk >= A.cache.num_blocks ? 0 : blk;  // a bad id must not fault
        if (P.has_stage && t < hist) {
          seat = blk % P.st.rows * bs + off;
          staged = P.st.owner[seat] == blk;
        }
      }
      const bool codes = t < hist && !staged, cur = has_new && t >= hist && t < seq;
      const uint8_t* slot = A.cache.k + blk * A.cache.k_stride[0] + off * A.cache.k_stride[1] + kvh * A.cache.k_stride[2];
      unsigned t_lo = 0, t_hi = 0;
      if (codes) byte_tables<QT>(*(const unsigned*)slot, t_lo, t_hi);
      const float* fp = P.st.stage_k + (seat * hk + kvh) * D + g * (D / 2);
      const uint16_t* row = (const uint16_t*)A.k_new + (int64_t)(qa + (cur ? t - hist : 0)) * A.k_new_stride_token + kvh * D +
                            g * (D / 2);
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        unsigned o[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
        if (codes) {
          lut16(*(const unsigned*)(slot + 32 + g * (D / 8) + 4 * c), t_lo, t_hi, o);
        } else if (staged) {
          f32x4 f[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) f[x] = *(const f32x4*)(fp + 16 * c + 4 * x);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            o[x] = hist_pair<QT>(f[0][x], f[1][x]);
            o[4 + x] = hist_pair<QT>(f[2][x], f[3][x]);
          }
        } else if (cur) {
          kpairs16(*(const u32x4*)(row + 16 * c), *(const u32x4*)(row + 16 * c + 8), o);
        }
        kop[2 * c] = u32x4{o[0], o[1], o[2], o[3]};
        kop[2 * c + 1] = u32x4{o[4], o[5], o[6], o[7]};
      }
    }
    float acc[16] = {};
    // ---- all rows that see the workgroup's first key
    const int first = tb > before ? (tb - before) * G : 0;
    for (int rb = first / 32; rb * 32 < nrows; ++rb) {
      const int n = 32 * rb + m;
      const bool row_ok = n < nrows;
      const int tok = row_ok ? n / G : 0, head = kvh * G + (row_ok ? n - tok * G : 0);
      const uint16_t* q = (const uint16_t*)A.q + (int64_t)(qa + tok) * A.q_stride_token + (int64_t)head * D + g * (D / 2);
      __syncthreads();  // the block before has been read
#pragma unroll
      for (int c = wave; c < NCH; c += kWaves) {
        unsigned o[8];
        kpairs16(*(const u32x4*)(q + 16 * c), *(const u32x4*)(q + 16 * c + 8), o);
        s_q[2 * c][lane] = u32x4{o[0], o[1], o[2], o[3]};
        s_q[2 * c + 1][lane] = u32x4{o[4], o[5], o[6], o[7]};
      }
      const float lse = A.lse[(int64_t)(qa + tok) * A.num_q_heads + head];
      __syncthreads();
      f32x16 S = {};
#pragma unroll
      for (int j = 0; j < 2 * NCH; ++j) S = mma16<QT>(kop[j], s_q[j][lane], S);
      // exp(s' - lse) = 2^(s2 - lse2) f, f the rest of lse's conversion to log2 units (a
      // rounding of up to 2^-20 there would show in every weight of the row)
      const float lse2 = lse * kScoreLog2e;
      const float f = fabsf(lse) < INFINITY ? 1.f - kLn2 * fmaf(lse, kScoreLog2e, -lse2) : 1.f;
      const float slope2 = SC ? slope2_of(P.sc, head) : 0.f;
      // keys of the lane's half that the row sees (none of a row that saw no key at all)
      const int limit = row_ok && lse != -INFINITY ? before + tok + 1 - t0 - 4 * g : 0;
      const float near = (float)(t0 + 4 * g - (before + tok));
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = out_tok(r, 0);
        float x;
        if constexpr (SC == 0) x = fmaf(S[r], P.sc.scale2, -lse2);
        else x = fmaf(slope2, near + key, (SC == 2 ? capped2_fine(P.sc, S[r]) : S[r] * P.sc.scale2) - lse2);
        const float p = key < limit ? __builtin_amdgcn_exp2f(x) : 0.f;
        acc[r] = fmaf(p, f, acc[r]);
      }
    }
    // ---- over the rows: the 32 lanes of each half
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float x = acc[r];
      x += dpp_row<kDppXor1>(x);
      x += dpp_row<kDppXor2>(x);
      x += dpp_row<kDppHalfMirror>(x);
      x += dpp_row<kDppMirror>(x);
      x += swizzle_xor16(x);
      if (m == r) sum = x;
    }
    const int mine = t0 + out_tok(m, g);  // lane m < 16 of each half
    if (m < 16 && mine < seq) out[mine] += sum;
  }
}

}  // namespace

}  // namespace oscar

using namespace oscar;

extern "C" int64_t oscarop_attn_weights_workspace_bytes_v1(const oscarop_weights_args_v1* args) {
  return args ? 0 : -22;
}

extern "C" int oscarop_attn_weights_v1(const oscarop_weights_args_v1* args, const oscarop_score_v1* score, void* stream) {
  const char* name = "oscarop_attn_weights_v1";
  if (!args) return fail(-22, "%s: null args", name);
  const oscarop_weights_args_v1& a = *args;
  WeightsParams p{};
  const int sc = score_of(score, a.scale, &p.sc);
  if (sc < 0) return fail(-22, "%s: soft_cap must be a finite number, 0 for none", name);
  const int64_t D = a.cache.head_dim;
  if (D != 128 && D != 256) return fail(-22, "%s: head_dim %lld unsupported (128/256)", name, (long long)D);
  if (a.num_reqs < 0 || a.num_tokens < 0 || a.max_seq_len < 0 || a.max_query_len < 0)
    return fail(-22, "%s: negative size", name);
  if (a.q_dtype != OSCAR_BF16 && a.q_dtype != OSCAR_F16)
    return fail(-22, "%s: q_dtype must be OSCAR_BF16 or OSCAR_F16", name);
  if (a.cache.num_kv_heads < 1 || a.num_q_heads < 1 || a.num_q_heads % a.cache.num_kv_heads)
    return fail(-22, "%s: Hq must be a multiple of Hk", name);
  if (a.num_reqs == 0 || a.num_tokens == 0 || a.max_seq_len == 0) return 0;
  if (!a.q || !a.lse || !a.weights || !a.query_start_loc || !a.seq_lens || !a.block_table || !a.cache.k)
    return fail(-22, "%s: missing pointer", name);
  if (a.num_reqs > 0xffff || a.cache.num_kv_heads > 0xffff || a.num_tokens * a.num_q_heads >= (1ll << 31))
    return fail(-22, "%s: too many requests or rows for one call", name);
  if (a.block_table_rows < a.num_reqs || a.block_table_cols < 1 || a.block_table_stride < a.block_table_cols)
    return fail(-22, "%s: Missing request block-table rows", name);
  if (a.cache.block_size < kTile || a.cache.block_size % kTile || a.cache.block_size > (1 << 20))
    return fail(-22, "%s: block_size %lld must be a multiple of %d (<= 2^20)", name, (long long)a.cache.block_size, kTile);
  if (a.weights_cols < 1 || a.weights_stride_head < a.weights_cols ||
      (a.num_reqs > 1 && a.weights_stride_request < a.weights_stride_head * a.cache.num_kv_heads))
    return fail(-22, "%s: weights of two heads or requests overlap", name);
  if ((a.cache.k_stride[0] & 15) || (a.cache.k_stride[1] & 15) || (a.cache.k_stride[2] & 15) || (((uintptr_t)a.cache.k) & 15))
    return fail(-22, "%s: cache slots must be 16-byte aligned", name);
  if ((a.q_stride_token & 7) || (((uintptr_t)a.q) & 15) ||
      (a.k_new && ((a.k_new_stride_token & 7) || (((uintptr_t)a.k_new) & 15))))
    return fail(-22, "%s: q / k_new rows must be 16-byte aligned", name);
  if (a.staging && (a.staging->rows < 1 || a.staging->rows * a.cache.block_size >= (1ll << 31) || !a.staging->owner ||
                    !a.staging->stage_k || (((uintptr_t)a.staging->stage_k) & 15)))
    return fail(-22, "%s: staging arena rows out of range or unaligned", name);
  p.a = a;
  p.has_stage = a.staging != nullptr;
  if (a.staging) p.st = *a.staging;
  p.group = (int)(a.num_q_heads / a.cache.num_kv_heads);
  hipStream_t s = (hipStream_t)stream;
  const int64_t per = kWaves * kTile;
  const dim3 grid((unsigned)((a.max_seq_len + per - 1) / per), (unsigned)a.cache.num_kv_heads, (unsigned)a.num_reqs);
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, s, p); };
  auto by_score = [&](auto d, auto qt) {
    constexpr int DD = decltype(d)::value, QT = decltype(qt)::value;
    if (sc == 0) launch(weights_kernel<DD, QT, 0>);
    else if (sc == 1) launch(weights_kernel<DD, QT, 1>);
    else launch(weights_kernel<DD, QT, 2>);
  };
  using std::integral_constant;
  if (D == 256) {
    if (a.q_dtype == OSCAR_F16) by_score(integral_constant<int, 256>{}, integral_constant<int, OSCAR_F16>{});
    else by_score(integral_constant<int, 256>{}, integral_constant<int, OSCAR_BF16>{});
  } else {
    if (a.q_dtype == OSCAR_F16) by_score(integral_constant<int, 128>{}, integral_constant<int, OSCAR_F16>{});
    else by_score(integral_constant<int, 128>{}, integral_constant<int, OSCAR_BF16>{});
  }
  OSCAR_CHECK_LAUNCH("weights_kernel");
  return 0;
}
