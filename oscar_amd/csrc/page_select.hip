// Bounds of the keys of each page, and the pages that promise the largest scores (gfx950).
//
// A query's product with any key of a page is at most
//   sum_d max(q_d low_d, q_d high_d) = sum_d (q_d m_d + |q_d| w_d),
// low and high being the least and the largest key of the page in channel d, m = (low + high) / 2
// and w = (high - low) / 2, of the keys as their slots hold them, fp16.  m and w have up to 41 bits, a query
// 8 or 11: their products are exact in 64 bits.  A sum's order is the same for every page and form of the
// kernel, so that equal bounds give equal scores; it is off by 13 (D 128) or 21 (D 256) additions'
// rounding at most, 21 2^-53 sum_d (|q_d m_d| + |q_d| w_d), and exact where the terms' bits all
// fit in 53 (values of one range mostly).
//
//   bounds_kernel   one workgroup per page (several in turn where a request grew by more than
//                   max_new): the codes of its tokens, each token's four values from a table,
//                   packed minimum and maximum
//   select_kernel   eight lanes a page, the bounds in registers, the queries in LDS in 64 bits; the
//                   last workgroup of a (request, KV head) finds the budget-th largest score by
//                   radix selection and writes the chosen columns in their order
//
// bounds_kernel is bound by latency: a page of 128 tokens is one round of loads.  4.1 us for 24 requests
// of four new tokens, 7.1 for 938 full pages of D 256 (9.1 MB of slots' bytes in use, 2.6 times the
// 1.9 us of a large copy).
//
// select_kernel: about 3.6 us of launch and the counters' line, 2 to 3 until the bounds are there, the
// products, then 4 to 6 for the choice, whose chain is the keys' stores, the counter, the keys' loads, two
// or three digits and the stores.  One list of 250 pages and 6 rows 9 us, 8 of 192 pages and 24 rows
// 12.4, 16 of 1024 pages and 6 rows 16 (16.8 MB of bounds; scores 4, choice 6), 12 ragged of up to 470 pages, two
// heads of D 128 and 16 rows 13.3.  A launch of its own for the choice costs the 4 to 5 us of a launch.
// Products in 32 bits would take half the time of a third of the kernel, and could miss the order of
// near scores.  What took the 16 lists from 19.9 us to 15.1 in a graph: counters a cache line apart (in one
// line the 512 arrivals wait for each other, 3.7 us), the last digit's candidates ranked by all waves (a loop
// over LDS in one took 1 to 2), 32 queries at a time.
#include <type_traits>

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
  __shared__ unsigned s_part[GROUPS][CH][17];
  // one page, unless a request grew by more than the launch was sized for
  for (int64_t col = before / bs + blockIdx.x; col * bs < after; col += gridDim.x) {
    const int page = A.block_table[r * A.block_table_stride + col];
    if (page < 0 || page >= A.cache.num_blocks) continue;
    const int held = after - col * bs < bs ? (int)(after - col * bs) : bs;
    const uint8_t* base = A.cache.k + (int64_t)page * A.cache.k_stride[0] + (int64_t)h * A.cache.k_stride[2];
    const int64_t ks1 = A.cache.k_stride[1];
    const int c = tid % CH, group = tid / CH;
    f16x2 low[8], high[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) low[k] = as_f16x2(0x7c007c00u), high[k] = as_f16x2(0xfc00fc00u);
    constexpr int BATCH = 128 / GROUPS;  // slots of a thread in flight: a page of 128 tokens at once
    for (int t0 = group; t0 < held; t0 += BATCH * GROUPS) {
      unsigned consts[BATCH], w[BATCH];
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        // (behind the page's tokens: the thread's first one again)
        const uint8_t* slot = base + (t0 + u * GROUPS < held ? t0 + u * GROUPS : t0) * ks1;
        consts[u] = *(const unsigned*)slot;
        w[u] = *(const unsigned*)(slot + 32 + 4 * c);
      }
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        unsigned lo, hi;
        value_table<OSCAR_F16>(consts[u], lo, hi);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          // channels k and k + 8 of the chunk
          const unsigned y = (w[u] >> (2 * k)) & 0x00030003u;
          const f16x2 v = as_f16x2(__builtin_amdgcn_perm(hi, lo, y * 0x202u + 0x01000100u));
          low[k] = pk_min(low[k], v);
          high[k] = pk_max(high[k], v);
        }
      }
    }
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
    __syncthreads();  // s_part is rewritten for the next page
  }
}

// ------------------------------------------------------------------------ scores and selection
constexpr int kLanes = 8;                // lanes of a page
constexpr int kPages = 64 / kLanes;      // pages of a workgroup at a time
constexpr int kHeld = 4096;              // scores in LDS; more are read again in each pass
constexpr int kFew = 64;                 // candidates that are ranked against each other
constexpr int kBatch = 4;                // scores of a thread in flight
constexpr int kRowsHeld = 32;            // queries in LDS at a time, in 64 bits: a conversion costs four products
// Workgroups up to which the waves of one share their pages, what the card holds at a time: 8 lists of
// 192 pages and 24 rows 192 workgroups of 8 pages.  Beyond, 32 pages: 6 lists of 1500 pages and 6 rows
// 16 us (8 pages: 22), 8 of 800 and 24 rows 19 (23), 8 of 700 with two heads of D 128 and 8 rows 13 (16).
constexpr int64_t kByRows = 512;

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

// what a wave's lanes give, combined into its last lane: within rows of 16 lanes, then the
// rows' last lanes into the rows behind them (0: what lanes without a neighbour take)
template <class Op>
__device__ __forceinline__ unsigned wave_prefix(unsigned v, Op op) {
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false));
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false));
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false));
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false));
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));
  return op(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));
}

// exclusive prefix sum over the workgroup of one number per thread
__device__ __forceinline__ unsigned scan(unsigned x, unsigned* s_part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned v = wave_prefix(x, [](unsigned a, unsigned b) { return a + b; });
  __syncthreads();  // s_part of the call before has been read
  if (lane == 63) s_part[wave] = v;
  __syncthreads();
  unsigned before = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) before += w < wave ? s_part[w] : 0;
  return before + v - x;
}

// One list's choice: the want-th largest key of `first` to `end`, then the chosen columns in
// their order.  The keys agree in their upper bits, so digits begin at the highest one in which two
// differ; the few candidates that are left in the digit's bin are ranked against each other.
__device__ void choose(const SelectParams& P, int many, int64_t list, const int32_t* row, uint64_t* s_key) {
  const oscarop_select_args_v1& A = P.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int32_t* table = A.table + list * A.budget;
  int32_t* pages = A.pages == nullptr ? nullptr : A.pages + list * A.budget;
  auto put = [&](int at, int col, int page) {
    table[at] = page;
    if (pages != nullptr) pages[at] = col;
  };
  const int first = A.first_pages, n = many - first - A.last_pages, want = A.budget - first - A.last_pages;
  const uint64_t* keys = P.keys + list * A.max_pages + first;
  __shared__ int s_bin[256];
  __shared__ unsigned s_part[kWaves];
  __shared__ unsigned s_diff[kWaves][2];
  __shared__ uint64_t s_few[kFew];
  __shared__ unsigned s_rank[kFew];
  __shared__ int s_found[3];       // digit, rest to take, size of its bin
  __shared__ uint64_t s_limit;
  const bool held = n <= kHeld;
  auto load = [&](int i) { return __hip_atomic_load(keys + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
  // at the end thread t looks at the columns [t run, (t + 1) run): its first ones' pages early
  const int run = (n + kThreads - 1) / kThreads;
  const int a = min(tid * run, n), b = min(a + run, n);
  int page[kBatch];
  auto load_pages = [&](int i) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) page[u] = row[first + min(i + u, n - 1)];
  };
  load_pages(a);
  for (int i = tid; i < first; i += kThreads) put(i, i, row[i]);
  for (int i = tid; i < A.last_pages; i += kThreads) put(A.budget - A.last_pages + i, many - A.last_pages + i, row[many - A.last_pages + i]);
  const uint64_t some = load(0);
  uint64_t diff = 0;
  for (int i = tid; i < n; i += kBatch * kThreads) {
    uint64_t k[kBatch];  // all on their way before the first is used
#pragma unroll
    for (int u = 0; u < kBatch; ++u) k[u] = load(min(i + u * kThreads, n - 1));
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (held && i + u * kThreads < n) s_key[i + u * kThreads] = k[u];
      diff |= k[u] ^ some;
    }
  }
  auto key = [&](int i) { return held ? s_key[i] : load(i); };
  auto both = [](unsigned a, unsigned b) { return a | b; };
  const unsigned low = wave_prefix((unsigned)diff, both), high = wave_prefix((unsigned)(diff >> 32), both);
  if (lane == 63) {
    s_diff[wave][0] = low;
    s_diff[wave][1] = high;
  }
  s_bin[tid] = 0;
  if (tid == 0) s_found[2] = 0;
  __syncthreads();
  diff = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) diff |= (uint64_t)s_diff[w][1] << 32 | s_diff[w][0];
  // keys are told apart by `mask`; those with `prefix` there are still to be told apart
  int left = diff == 0 ? 0 : 64 - __clzll((long long)diff);
  uint64_t mask = left >= 64 ? 0 : ~0ull << left, prefix = some & mask;
  unsigned rest = want;
  while (left > 0) {
    const int shift = left > 8 ? left - 8 : 0, digits = (1 << (left - shift)) - 1;
    for (int i = tid; i < n; i += kThreads) {
      const uint64_t k = key(i);
      if ((k & mask) == prefix) atomicAdd(&s_bin[(int)(k >> shift) & digits], 1);
    }
    __syncthreads();
    // thread t: the t-th largest digit
    const unsigned mine = s_bin[255 - tid], above = scan(mine, s_part);
    if (above < rest && above + mine >= rest) {
      s_found[0] = 255 - tid;
      s_found[1] = rest - above;
      s_found[2] = mine;
    }
    __syncthreads();
    prefix |= (uint64_t)s_found[0] << shift;
    mask |= (uint64_t)digits << shift;
    rest = s_found[1];
    left = shift;
    const unsigned size = s_found[2];
    if (size == rest) break;  // all of the bin
    s_bin[tid] = 0;
    if (size <= kFew && left > 0) {
      __syncthreads();  // s_found has been read
      if (tid == 0) s_found[2] = 0;
      if (tid < kFew) s_rank[tid] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += kThreads) {
        const uint64_t k = key(i);
        if ((k & mask) == prefix) s_few[atomicAdd(&s_found[2], 1)] = k;
      }
      __syncthreads();
      // each wave's share of the candidates, against a lane's one: those above it, and those alike
      const uint64_t own = s_few[lane < (int)size ? lane : 0];
      unsigned above = 0, alike = 0;
#pragma unroll
      for (int u = 0; u < kFew / kWaves; ++u) {
        const int at = wave * (kFew / kWaves) + u;
        const uint64_t o = s_few[at < (int)size ? at : 0];
        above += at < (int)size && o > own;
        alike += at < (int)size && o == own;
      }
      atomicAdd(&s_rank[lane], above << 16 | alike);
      __syncthreads();
      if (wave == 0) {
        const unsigned rank = s_rank[lane], over = rank >> 16;
        if (lane < (int)size && over < rest && over + (rank & 0xffffu) >= rest) {
          s_limit = own;
          s_found[1] = rest - over;  // of the keys that equal the limit
        }
      }
      __syncthreads();
      prefix = s_limit;
      mask = ~0ull;
      rest = s_found[1];
      break;
    }
    __syncthreads();  // s_found has been read, the bins are clear
  }
  // keys above the prefix, and the first `rest` that equal it
  unsigned same = 0, over = 0;
  for (int i = a; i < b; ++i) {
    const uint64_t k = key(i) & mask;
    same += k == prefix;
    over += k > prefix;
  }
  unsigned ties = scan(same, s_part);
  const unsigned taken = ties < rest ? min(same, rest - ties) : 0;
  unsigned at = first + scan(over + taken, s_part);
  for (int i0 = a; i0 < b; i0 += kBatch) {
    if (i0 > a) load_pages(i0);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (i0 + u >= b) break;
      const uint64_t k = key(i0 + u) & mask;
      const bool tie = k == prefix;
      if (k > prefix || (tie && ties < rest)) put(at++, first + i0 + u, page[u]);
      ties += tie;
    }
  }
}

// A workgroup scores eight pages at a time, its waves a quarter of the rows each (ROWS), or 32
// pages, eight a wave; the last one of a (request, KV head) to arrive makes the choice.
template <int D, int QT, bool ROWS>
__global__ __launch_bounds__(kThreads, 2) void select_kernel(SelectParams P) {
  constexpr int STEPS = D / (8 * kLanes);  // 16-byte pieces of a lane
  const oscarop_select_args_v1& A = P.a;
  const int tid = threadIdx.x, lane = tid & 63, h = blockIdx.y, r = blockIdx.z;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t list = (int64_t)r * A.num_kv_heads + h;
  const int32_t* table_row = A.block_table + (int64_t)r * A.block_table_stride;
  constexpr int kAtOnce = ROWS ? kPages : kWaves * kPages;
  const int j = lane % kLanes;
  const int64_t p0 = (int64_t)A.first_pages + (int64_t)blockIdx.x * kAtOnce, p = p0 + lane / kLanes + (ROWS ? 0 : kPages * wave);
  // the page and its bounds are on their way while the request's lengths come (behind the
  // last page: some page's)
  int page = -1;
  if (A.block_table_cols > 0) page = table_row[p < A.block_table_cols ? p : A.block_table_cols - 1];
  const History x = history_of(A, r);
  if (x.pages <= A.budget) {
    // all of them
    if (blockIdx.x > 0) return;
    for (int i = tid; i < A.budget; i += kThreads) {
      A.table[list * A.budget + i] = i < x.pages ? table_row[i] : -1;
      if (A.pages != nullptr) A.pages[list * A.budget + i] = i < x.pages ? i : -1;
    }
    return;
  }
  const int group = (int)(A.num_q_heads / A.num_kv_heads);
  const int64_t end = x.pages - A.last_pages;
  const int64_t rows = (int64_t)x.nq * group;
  __shared__ double s_best[kWaves][kPages];
  // the queries, and for the choice the scores
  __shared__ __attribute__((aligned(16))) uint64_t s_mem[kRowsHeld * D > kHeld ? kRowsHeld * D : kHeld];
  double(*s_q)[D] = (double(*)[D])s_mem;
  __shared__ int s_last;
  if (p0 < end) {
    page = page < 0 || page >= A.num_blocks ? 0 : page;
    const uint16_t* b = (const uint16_t*)A.bounds + ((int64_t)page * A.num_kv_heads + h) * 2 * D + 8 * j;
    u32x4 lo[STEPS], hi[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      lo[s] = *(const u32x4*)(b + 8 * kLanes * s);
      hi[s] = *(const u32x4*)(b + D + 8 * kLanes * s);
    }
    auto rows_from = [&](int64_t from, int many) {
      constexpr int PIECES = kRowsHeld * (D / 8) / kThreads;  // of eight elements, all on their way at once
      float v[PIECES][8];
#pragma unroll
      for (int u = 0; u < PIECES; ++u) {
        const int i = min(tid + u * kThreads, many * (D / 8) - 1);
        const int64_t row = from + i / (D / 8);
        load8<QT>(A.q, (x.q0 + row / group) * A.q_stride_token + (h * group + row % group) * (int64_t)D + i % (D / 8) * 8, v[u]);
      }
#pragma unroll
      for (int u = 0; u < PIECES; ++u) {
        const int i = tid + u * kThreads;
        if (i >= many * (D / 8)) break;
#pragma unroll
        for (int e = 0; e < 8; ++e) s_q[i / (D / 8)][i % (D / 8) * 8 + e] = v[u][e];
      }
      __syncthreads();
    };
    if (rows > 0) rows_from(0, rows < kRowsHeld ? (int)rows : kRowsHeld);
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
    double best = -INFINITY;
    for (int64_t from = 0; from < rows; from += kRowsHeld) {
      const int many = rows - from < kRowsHeld ? (int)(rows - from) : kRowsHeld;
      if (from > 0) {
        __syncthreads();  // the rows before have been read
        rows_from(from, many);
      }
      for (int row = ROWS ? wave : 0; row < many; row += ROWS ? kWaves : 1) {
        double part[4] = {0.0, 0.0, 0.0, 0.0};  // four sums at a time: one alone waits for itself
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const double v = s_q[row][8 * kLanes * s + 8 * j + e];
            part[e & 3] = fma(v, m[s][e], part[e & 3]);
            part[e & 3] = fma(fabs(v), w[s][e], part[e & 3]);
          }
        double sum = (part[0] + part[1]) + (part[2] + part[3]);
        sum += dpp_row64<kDppXor1>(sum);
        sum += dpp_row64<kDppXor2>(sum);
        sum += dpp_row64<kDppHalfMirror>(sum);
        // Finite bounds and queries have finite sums; m and w of an infinite bound give NaN or an
        // infinity by the query's sign, and all of these count alike (a NaN stays)
        sum = fabs(sum) < INFINITY ? sum : NAN;
        best = best != best || sum <= best ? best : sum;
      }
    }
    auto put = [&](int64_t at, uint64_t k) {
      __hip_atomic_store(P.keys + list * A.max_pages + at, k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    };
    if constexpr (ROWS) {
      if (j == 0) s_best[wave][lane / kLanes] = best;
      __syncthreads();
      if (tid < kPages && p0 + tid < end) {
        uint64_t k = 0;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
          const uint64_t o = order_of(s_best[i][tid]);
          k = o > k ? o : k;
        }
        put(p0 + tid, k);
      }
    } else if (j == 0 && p < end) {
      put(p, order_of(best));
    }
  }
  // The keys go past this XCD's L2 and are read past the reader's (agent-scope atomics), so that
  // the barrier, which waits for them, and the counter, which wraps to zero, order them; an agent-scope
  // fence would write back the whole L2 instead, for every workgroup (16 lists of 1024 pages: 64 us)
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (tid == 0) s_last = atomicInc((unsigned*)&A.arrivals[list * OSCAROP_SELECT_ARRIVAL], gridDim.x - 1) == gridDim.x - 1;
  __syncthreads();
  if (s_last) choose(P, (int)x.pages, list, table_row, s_mem);
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
  dim3 grid(1, (unsigned)a.num_kv_heads, (unsigned)a.num_reqs);
  bool by_rows = true;
  if (need > 0) {
    if ((a.num_tokens > 0 && !a.q) || !a.bounds || a.num_blocks < 1) return fail(-22, "oscarop_select_v1: missing pointer");
    if ((a.q_stride_token & 7) || ((uintptr_t)a.q & 15) || ((uintptr_t)a.bounds & 15))
      return fail(-22, "oscarop_select_v1: q rows and bounds must be 16-byte aligned");
    if (a.workspace_bytes < need || !a.workspace || ((uintptr_t)a.workspace & 15))
      return fail(-28, "oscarop_select_v1: workspace of %lld bytes < %lld", (long long)a.workspace_bytes, (long long)need);
    if (!a.arrivals) return fail(-22, "oscarop_select_v1: missing pointer");
    const int64_t scored = a.max_pages - a.first_pages - a.last_pages;
    grid.x = (unsigned)((scored + kPages - 1) / kPages);
    by_rows = (int64_t)grid.x * a.num_kv_heads * a.num_reqs <= kByRows;
    if (!by_rows) grid.x = (unsigned)((scored + kWaves * kPages - 1) / (kWaves * kPages));
  }
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, s, p); };
  const bool f16 = a.q_dtype == OSCAR_F16;
  auto launch_rows = [&](auto rows) {
    constexpr bool R = decltype(rows)::value;
    if (a.head_dim == 256) f16 ? launch(select_kernel<256, OSCAR_F16, R>) : launch(select_kernel<256, OSCAR_BF16, R>);
    else f16 ? launch(select_kernel<128, OSCAR_F16, R>) : launch(select_kernel<128, OSCAR_BF16, R>);
  };
  if (by_rows) launch_rows(std::true_type{});
  else launch_rows(std::false_type{});
  OSCAR_CHECK_LAUNCH("select_kernel");
  return 0;
}
