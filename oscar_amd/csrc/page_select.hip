// Bounds of the keys of each page, and the pages that promise the largest scores (gfx950).
//
// A query's product with any key of a page is at most
//   sum_d max(q_d low_d, q_d high_d) = sum_d (q_d m_d + |q_d| w_d),
// low and high being the least and the largest key of the page in channel d, m = (low + high) / 2
// and w = (high - low) / 2.  The products of 8 or 11 bits of a query with 12 of m or w are exact in
// 64 bits, and so are their sums unless the terms lie 2^30 apart: pages are told apart by
// their real order, whatever order the sums are taken in.
//
//   bounds_kernel   one workgroup per page: the codes of its tokens, each token's four values from a
//                   table, packed minimum and maximum
//   score_kernel    eight lanes a page, the bounds in registers, the queries from LDS
//   select_kernel   one workgroup per (request, KV head): the budget-th largest score by radix
//                   selection, then the chosen columns in their order
#include "common.h"
#include "int2_tile.h"

#include "../../include/oscar_operators.h"

namespace oscar {

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int64_t kMostAxis = 0xffff;  // requests, and KV heads: an axis of the grid each

// ------------------------------------------------------------------------ bounds
// NaN goes through both
__device__ __forceinline__ f16x2 pk_min(f16x2 a, f16x2 b) { return __builtin_elementwise_minimum(a, b); }
__device__ __forceinline__ f16x2 pk_max(f16x2 a, f16x2 b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ f16x2 as_f16x2(unsigned v) { return __builtin_bit_cast(f16x2, v); }
__device__ __forceinline__ unsigned as_u32(f16x2 v) { return __builtin_bit_cast(unsigned, v); }

template <int D>
__global__ __launch_bounds__(kThreads) void bounds_kernel(oscarop_bounds_args_v1 A) {
  constexpr int CH = D / 16;             // 16-channel chunks (a dword of codes each)
  constexpr int GROUPS = kThreads / CH;  // tokens at a time
  const int tid = threadIdx.x, r = blockIdx.z, h = blockIdx.y;
  const int bs = (int)A.cache.block_size;
  const int64_t before = A.lengths[r], after = A.seq_lens[r];
  if (before < 0 || after <= before || (after - 1) / bs >= A.block_table_cols) return;
  const int64_t col = before / bs + blockIdx.x;
  if (col * bs >= after) return;
  const int page = A.block_table[r * A.block_table_stride + col];
  if (page < 0 || page >= A.cache.num_blocks) return;
  const int held = after - col * bs < bs ? (int)(after - col * bs) : bs;
  const uint8_t* base = A.cache.k + (int64_t)page * A.cache.k_stride[0] + (int64_t)h * A.cache.k_stride[2];
  const int64_t ks1 = A.cache.k_stride[1];
  const int c = tid % CH, group = tid / CH;
  f16x2 low[8], high[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) low[k] = as_f16x2(0x7c007c00u), high[k] = as_f16x2(0xfc00fc00u);
  for (int t = group; t < held; t += GROUPS) {
    const uint8_t* slot = base + t * ks1;
    const unsigned consts = *(const unsigned*)slot, w = *(const unsigned*)(slot + 32 + 4 * c);
    unsigned lo, hi;
    value_table<OSCAR_F16>(consts, lo, hi);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      // channels k and k + 8 of the chunk
      const unsigned y = (w >> (2 * k)) & 0x00030003u;
      const f16x2 v = as_f16x2(__builtin_amdgcn_perm(hi, lo, y * 0x202u + 0x01000100u));
      low[k] = pk_min(low[k], v);
      high[k] = pk_max(high[k], v);
    }
  }
  __shared__ unsigned s_part[GROUPS][CH][17];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    s_part[group][c][k] = as_u32(low[k]);
    s_part[group][c][8 + k] = as_u32(high[k]);
  }
  __syncthreads();
  uint16_t* out = (uint16_t*)A.bounds + (((int64_t)page * A.cache.num_kv_heads + h) * 2) * D;
  if (tid < D) {
    const int chunk = tid / 16, k = tid % 16;
    f16x2 v = as_f16x2(s_part[0][chunk][k]);
    for (int g = 1; g < GROUPS; ++g) {
      const f16x2 o = as_f16x2(s_part[g][chunk][k]);
      v = k < 8 ? pk_min(v, o) : pk_max(v, o);
    }
    uint16_t* row = out + (k < 8 ? 0 : D) + 16 * chunk + (k & 7);
    row[0] = (uint16_t)as_u32(v);
    row[8] = (uint16_t)(as_u32(v) >> 16);
  }
}

// ------------------------------------------------------------------------ scores
constexpr int kLanes = 8;                               // lanes of a page
constexpr int kPages = kThreads / kLanes;               // pages of a workgroup at a time
constexpr int kRowsHeld = 32;                           // queries in LDS at a time

struct SelectParams {
  oscarop_select_args_v1 a;
  uint64_t* keys;     // [num_reqs][Hk][max_pages]
};

struct History {
  int q0, nq;        // queries
  int64_t pages;     // of the history; below 0 for a request that does not fit
};

__device__ __forceinline__ History history_of(const oscarop_select_args_v1& A, int r) {
  const int a = A.query_start_loc[r], b = A.query_start_loc[r + 1];
  const int64_t h = (int64_t)A.seq_lens[r] - (A.has_new ? (int64_t)b - a : 0);
  const int64_t pages = (h + A.block_size - 1) / A.block_size;
  const bool ok = a >= 0 && b >= a && b <= A.num_tokens && h >= 0 && pages <= A.block_table_cols && pages <= A.max_pages;
  return {a, b - a, ok ? pages : -1};
}

// scores in ascending order as unsigned numbers: +0 and -0 alike, NaN above everything
__device__ __forceinline__ uint64_t order_of(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
  return x != x ? ~0ull : u ^ ((uint64_t)((int64_t)u >> 63) | 0x8000000000000000ull);
}

template <int CTRL>
__device__ __forceinline__ double dpp_row64(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x);
  const unsigned lo = __builtin_amdgcn_update_dpp(0, (unsigned)u, CTRL, 0xf, 0xf, true);
  const unsigned hi = __builtin_amdgcn_update_dpp(0, (unsigned)(u >> 32), CTRL, 0xf, 0xf, true);
  return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}

template <int D, int QT>
__global__ __launch_bounds__(kThreads) void score_kernel(SelectParams P) {
  constexpr int STEPS = D / (8 * kLanes);  // 16-byte pieces of a lane
  const oscarop_select_args_v1& A = P.a;
  const int tid = threadIdx.x, h = blockIdx.y, r = blockIdx.z;
  const History x = history_of(A, r);
  if (x.pages <= A.budget) return;
  const int group = (int)(A.num_q_heads / A.num_kv_heads);
  const int first = A.first_pages, end = (int)x.pages - A.last_pages;
  const int j = tid % kLanes;
  __shared__ __attribute__((aligned(16))) float s_q[kRowsHeld][D];
  const int64_t rows = (int64_t)x.nq * group;
  for (int p0 = first + blockIdx.x * kPages; p0 < end; p0 += gridDim.x * kPages) {
    const int p = p0 + tid / kLanes;
    const bool in = p < end;
    int page = A.block_table[r * A.block_table_stride + (in ? p : first)];
    page = page < 0 || page >= A.num_blocks ? 0 : page;
    const uint16_t* b = (const uint16_t*)A.bounds + ((int64_t)page * A.num_kv_heads + h) * 2 * D + 8 * j;
    u32x4 lo[STEPS], hi[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      lo[s] = *(const u32x4*)(b + 8 * kLanes * s);
      hi[s] = *(const u32x4*)(b + D + 8 * kLanes * s);
    }
    double best = -INFINITY;
    bool nan = false;
    for (int64_t row0 = 0; row0 < rows; row0 += kRowsHeld) {
      const int held = rows - row0 < kRowsHeld ? (int)(rows - row0) : kRowsHeld;
      __syncthreads();  // the rows before have been read
      for (int i = tid; i < held * (D / 8); i += kThreads) {
        const int64_t row = row0 + i / (D / 8);
        const int e = i % (D / 8) * 8;
        float v[8];
        load8<QT>(A.q, (x.q0 + row / group) * A.q_stride_token + (h * group + row % group) * (int64_t)D + e, v);
        *(f32x4*)&s_q[i / (D / 8)][e] = f32x4{v[0], v[1], v[2], v[3]};
        *(f32x4*)&s_q[i / (D / 8)][e + 4] = f32x4{v[4], v[5], v[6], v[7]};
      }
      __syncthreads();
      double m[STEPS][8], w[STEPS][8];
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const double l = f16_bits_to_f32((lo[s][e / 2] >> (16 * (e & 1))) & 0xffff);
          const double u = f16_bits_to_f32((hi[s][e / 2] >> (16 * (e & 1))) & 0xffff);
          m[s][e] = 0.5 * (u + l);
          w[s][e] = 0.5 * (u - l);
        }
      for (int i = 0; i < held; ++i) {
        double sum = 0.0;
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const double q = s_q[i][8 * kLanes * s + 8 * j + e];
            sum = fma(q, m[s][e], sum);
            sum = fma(fabs(q), w[s][e], sum);
          }
        sum += dpp_row64<kDppXor1>(sum);
        sum += dpp_row64<kDppXor2>(sum);
        sum += dpp_row64<kDppHalfMirror>(sum);
        nan |= sum != sum;
        best = sum > best ? sum : best;
      }
    }
    if (in && j == 0) P.keys[((int64_t)r * A.num_kv_heads + h) * A.max_pages + p] = nan ? ~0ull : order_of(best);
  }
}

// ------------------------------------------------------------------------ selection
constexpr int kHeld = 4096;  // scores in LDS; more are read again in each pass

// exclusive prefix sum over the workgroup of one number per thread; *total gets the sum
__device__ __forceinline__ unsigned scan(unsigned x, unsigned* total, unsigned* s_part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  unsigned v = x;
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  __syncthreads();  // s_part of the call before has been read
  if (lane == 63) s_part[wave] = v;
  __syncthreads();
  unsigned before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    before += w < wave ? s_part[w] : 0;
    sum += s_part[w];
  }
  *total = sum;
  return before + v - x;
}

__global__ __launch_bounds__(kThreads) void select_kernel(SelectParams P) {
  const oscarop_select_args_v1& A = P.a;
  const int tid = threadIdx.x, h = blockIdx.x, r = blockIdx.y;
  const History x = history_of(A, r);
  const int64_t list = (int64_t)r * A.num_kv_heads + h;
  int32_t* table = A.table + list * A.budget;
  int32_t* pages = A.pages == nullptr ? nullptr : A.pages + list * A.budget;
  const int32_t* row = A.block_table + (int64_t)r * A.block_table_stride;
  auto put = [&](int at, int col) {
    table[at] = row[col];
    if (pages != nullptr) pages[at] = col;
  };
  const int many = (int)x.pages;
  if (many <= A.budget) {
    for (int i = tid; i < A.budget; i += kThreads) {
      if (i < many) put(i, i);
      else {
        table[i] = -1;
        if (pages != nullptr) pages[i] = -1;
      }
    }
    return;
  }
  const int first = A.first_pages, n = many - first - A.last_pages, want = A.budget - first - A.last_pages;
  const uint64_t* keys = P.keys + list * A.max_pages + first;
  __shared__ uint64_t s_key[kHeld];
  __shared__ int s_bin[256];
  __shared__ unsigned s_part[kWaves];
  __shared__ int s_found[3];  // digit, rest to take, size of its bin
  const bool held = n <= kHeld;
  if (held)
    for (int i = tid; i < n; i += kThreads) s_key[i] = keys[i];
  auto key = [&](int i) { return held ? s_key[i] : keys[i]; };
  uint64_t prefix = 0, mask = 0;
  unsigned rest = want, total;
  for (int shift = 56; shift >= 0; shift -= 8) {
    s_bin[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) {
      const uint64_t k = key(i);
      if ((k & mask) == prefix) atomicAdd(&s_bin[(int)(k >> shift) & 255], 1);
    }
    __syncthreads();
    // thread t: the t-th largest digit
    const int mine = s_bin[255 - tid];
    const unsigned above = scan(mine, &total, s_part);
    if (above < rest && above + mine >= rest) {
      s_found[0] = 255 - tid;
      s_found[1] = rest - above;
      s_found[2] = mine;
    }
    __syncthreads();
    prefix |= (uint64_t)s_found[0] << shift;
    mask |= 255ull << shift;
    rest = s_found[1];
    if ((unsigned)s_found[2] == rest) break;  // all of the bin
    __syncthreads();  // s_found has been read
  }
  // scores above the prefix, and the first `rest` that equal it: thread t looks at the columns
  // [t run, (t + 1) run)
  const int run = (n + kThreads - 1) / kThreads;
  const int a = min(tid * run, n), b = min(a + run, n);
  unsigned same = 0, over = 0;
  for (int i = a; i < b; ++i) {
    const uint64_t k = key(i) & mask;
    same += k == prefix;
    over += k > prefix;
  }
  unsigned ties = scan(same, &total, s_part);
  const unsigned taken = ties < rest ? min(same, rest - ties) : 0;
  unsigned at = first + scan(over + taken, &total, s_part);
  for (int i = a; i < b; ++i) {
    const uint64_t k = key(i) & mask;
    const bool tie = k == prefix;
    if (k > prefix || (tie && ties < rest)) put(at++, first + i);
    ties += tie;
  }
  for (int i = tid; i < first; i += kThreads) put(i, i);
  for (int i = tid; i < A.last_pages; i += kThreads) put(A.budget - A.last_pages + i, many - A.last_pages + i);
}

// -22 for sizes that are refused
int64_t select_workspace(const oscarop_select_args_v1& a) {
  if (a.num_reqs < 0 || a.num_reqs > kMostAxis || a.num_kv_heads < 1 || a.num_kv_heads > kMostAxis || a.max_pages < 0 ||
      a.max_pages > 1 << 24)
    return -22;
  // (at most 2^16 2^16 2^24 8 bytes)
  return a.max_pages > a.budget ? 8 * (int64_t)a.num_reqs * a.num_kv_heads * a.max_pages : 0;
}

}  // namespace

}  // namespace oscar

using namespace oscar;

extern "C" int oscarop_page_bounds_v1(const oscarop_bounds_args_v1* args, void* stream) {
  if (!args) return fail(-22, "oscarop_page_bounds_v1: null args");
  const oscarop_bounds_args_v1& a = *args;
  const int64_t d = a.cache.head_dim;
  if (d != 128 && d != 256) return fail(-22, "oscarop_page_bounds_v1: head_dim %lld unsupported", (long long)d);
  if (a.num_reqs < 0 || a.num_reqs > kMostAxis || a.cache.num_kv_heads < 1 || a.cache.num_kv_heads > kMostAxis)
    return fail(-22, "oscarop_page_bounds_v1: requests or KV heads out of range");
  if (a.cache.block_size < 1 || a.cache.block_size > 1 << 20 || a.cache.num_blocks < 0)
    return fail(-22, "oscarop_page_bounds_v1: block_size must lie in [1, 2^20]");
  if (a.max_new < 0 || a.max_new > 1 << 30) return fail(-22, "oscarop_page_bounds_v1: max_new out of range");
  if (a.num_reqs == 0 || a.max_new == 0) return 0;
  if (!a.cache.k || !a.block_table || !a.lengths || !a.seq_lens || !a.bounds)
    return fail(-22, "oscarop_page_bounds_v1: missing pointer");
  if (a.block_table_rows < a.num_reqs || a.block_table_cols < 1 || (a.num_reqs > 1 && a.block_table_stride < a.block_table_cols))
    return fail(-22, "oscarop_page_bounds_v1: Missing request block-table rows");
  if (((uintptr_t)a.cache.k & 15) || (a.cache.k_stride[0] & 15) || (a.cache.k_stride[1] & 15) || (a.cache.k_stride[2] & 15) ||
      ((uintptr_t)a.bounds & 15))
    return fail(-22, "oscarop_page_bounds_v1: cache slots and bounds must be 16-byte aligned");
  // max_new tokens that begin at a page's last place
  const int64_t pages = (a.max_new + a.cache.block_size - 2) / a.cache.block_size + 1;
  const dim3 grid((unsigned)(pages < a.block_table_cols ? pages : a.block_table_cols), (unsigned)a.cache.num_kv_heads,
                  (unsigned)a.num_reqs);
  if (d == 256) hipLaunchKernelGGL(bounds_kernel<256>, grid, dim3(kThreads), 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL(bounds_kernel<128>, grid, dim3(kThreads), 0, (hipStream_t)stream, a);
  OSCAR_CHECK_LAUNCH("bounds_kernel");
  return 0;
}

extern "C" int64_t oscarop_select_workspace_bytes_v1(const oscarop_select_args_v1* args) {
  return args == nullptr ? -22 : select_workspace(*args);
}

extern "C" int oscarop_select_v1(const oscarop_select_args_v1* args, void* stream) {
  if (!args) return fail(-22, "oscarop_select_v1: null args");
  const oscarop_select_args_v1& a = *args;
  if (a.head_dim != 128 && a.head_dim != 256)
    return fail(-22, "oscarop_select_v1: head_dim %lld unsupported", (long long)a.head_dim);
  if (a.q_dtype != OSCAR_BF16 && a.q_dtype != OSCAR_F16)
    return fail(-22, "oscarop_select_v1: q_dtype must be OSCAR_BF16 or OSCAR_F16");
  const int64_t need = select_workspace(a);
  if (need < 0) return fail(-22, "oscarop_select_v1: requests, KV heads or pages out of range");
  if (a.num_tokens < 0 || a.num_tokens > INT32_MAX || a.num_q_heads < 1 || a.num_q_heads % a.num_kv_heads ||
      a.num_q_heads / a.num_kv_heads > 1 << 16)
    return fail(-22, "oscarop_select_v1: Hq must be a multiple of Hk");
  if (a.block_size < 1 || a.block_size > 1 << 20) return fail(-22, "oscarop_select_v1: block_size must lie in [1, 2^20]");
  if (a.first_pages < 0 || a.last_pages < 1 || (int64_t)a.first_pages + a.last_pages >= a.budget || a.budget > 1 << 24)
    return fail(-22, "oscarop_select_v1: the budget must exceed first_pages + last_pages, last_pages be 1 at least");
  if (a.num_reqs == 0) return 0;
  if (!a.block_table || !a.query_start_loc || !a.seq_lens || !a.table)
    return fail(-22, "oscarop_select_v1: missing pointer");
  if (a.block_table_rows < a.num_reqs || a.block_table_cols < 0 || (a.num_reqs > 1 && a.block_table_stride < a.block_table_cols))
    return fail(-22, "oscarop_select_v1: Missing request block-table rows");
  SelectParams p{};
  p.a = a;
  p.keys = (uint64_t*)a.workspace;
  const hipStream_t s = (hipStream_t)stream;
  if (need > 0) {
    if (!a.q || !a.bounds || a.num_blocks < 1) return fail(-22, "oscarop_select_v1: missing pointer");
    if ((a.q_stride_token & 7) || ((uintptr_t)a.q & 15) || ((uintptr_t)a.bounds & 15))
      return fail(-22, "oscarop_select_v1: q rows and bounds must be 16-byte aligned");
    if (a.workspace_bytes < need || !a.workspace || ((uintptr_t)a.workspace & 15))
      return fail(-28, "oscarop_select_v1: workspace of %lld bytes < %lld", (long long)a.workspace_bytes, (long long)need);
    const int64_t scored = a.max_pages - a.first_pages - a.last_pages;
    const dim3 grid((unsigned)((scored + kPages - 1) / kPages), (unsigned)a.num_kv_heads, (unsigned)a.num_reqs);
    auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, s, p); };
    const bool f16 = a.q_dtype == OSCAR_F16;
    if (a.head_dim == 256) f16 ? launch(score_kernel<256, OSCAR_F16>) : launch(score_kernel<256, OSCAR_BF16>);
    else f16 ? launch(score_kernel<128, OSCAR_F16>) : launch(score_kernel<128, OSCAR_BF16>);
    OSCAR_CHECK_LAUNCH("score_kernel");
  }
  hipLaunchKernelGGL(select_kernel, dim3((unsigned)a.num_kv_heads, (unsigned)a.num_reqs), dim3(kThreads), 0, s, p);
  OSCAR_CHECK_LAUNCH("select_kernel");
  return 0;
}
