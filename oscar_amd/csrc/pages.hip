// Pages, slots and positions of a step's tokens, from lengths on the device (gfx950).
//
// Request r has length_r tokens in the cache and counts_r rows in the step, of which g_r
// (all, or those marked in `keep`) take places length_r, length_r + 1, ...
//   need_r = ceil((length_r + g_r) / bs) - ceil(length_r / bs)
// pages come off the top of the pool's stack for the requests whose running sum of needs
// still fits in it; the total T of those granted, request r's pages are
//   stack[free - T + sum_{s < r} need_s + i], i < need_r,
// and the slot of place p is table[r][p / bs] bs + p mod bs.
//
//   map_kernel    one workgroup: the sums over the requests, starts, lengths, the table's new
//                 columns and the pool's count; and the rows of a small step as well
//   rows_kernel   slots and positions of a larger step's rows, one a lane
//   release_kernel  one workgroup: pages behind the new lengths go back on the stack
//
// All of it is latency, a chain of a few dependent accesses and barriers: a step of one token
// reads and writes 37 bytes (map_kernel 4.5 us, release_kernel 2.3, an empty kernel 1.5 to 2), one of 256
// requests and 16600 rows 270 KB (6.7 and 4.1 in rows_kernel, release 5.0), one of 48 requests and 1536
// marked rows 27 KB (8.6, release 3.4).  One workgroup, since the sums go over all requests;
// rows beyond kSmallStep have a launch of their own, where one workgroup would take 1024 of them a round.
// The sums saturate at 2^32 - 1, which keeps them associative, and a
// saturated one is more than any pool or step holds.
#include "common.h"

#include "../../include/oscar_operators.h"

namespace oscar {

namespace {

constexpr int kMap = 1024;              // threads of the workgroup that looks at the requests
constexpr int kMapWaves = kMap / 64;
constexpr int kRows = 256;              // threads of a workgroup of rows
constexpr int64_t kMostReqs = 1 << 16;
constexpr int64_t kMostKeep = 1 << 16;  // rows of a step with marks: 1024 words of LDS
constexpr int kWords = kMostKeep / 64;
constexpr int64_t kMostRows = 1 << 30;
constexpr int kStarts = 4096;           // requests whose starts are held in LDS
constexpr int kOwnPages = 4;            // new pages that a request's own thread writes
constexpr int64_t kSmallStep = 2048;    // rows that the first workgroup serves as well

struct MapParams {
  oscarop_map_args_v1 a;
  int rows_too;          // map_kernel serves the rows
  uint32_t* kept_at;     // [num_reqs] marks before each request's first row (keep only)
  uint32_t* word_sum;    // [words] marks before each 64 rows
};

__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }

// exclusive prefix sum (saturating) over the workgroup, one number a thread; *total the sum
__device__ __forceinline__ uint32_t scan_sat(uint32_t x, uint32_t* total, uint32_t* s_part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t v = x;
  // within rows of 16 lanes, then the rows' last lanes to the rows behind them
  v = add_sat(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false));
  v = add_sat(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false));
  v = add_sat(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false));
  v = add_sat(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false));
  v = add_sat(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));
  v = add_sat(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));
  __syncthreads();  // s_part of the call before has been read
  if (lane == 63) s_part[wave] = v;
  __syncthreads();
  uint32_t before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < kMapWaves; ++w) {
    const uint32_t p = s_part[w];
    before = w < wave ? add_sat(before, p) : before;
    sum = add_sat(sum, p);
  }
  *total = sum;
  const uint32_t left = __shfl_up(v, 1);
  return lane == 0 ? before : add_sat(before, left);
}

// the request of a row: the last one that starts at or before it (requests without rows
// share their start with the next)
__device__ __forceinline__ int request_of_row(const int32_t* starts, int reqs, int row) {
  int lo = 0, hi = reqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (starts[mid] <= row) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// slot and position of a row (rank: its number among its request's placed rows)
__device__ __forceinline__ void write_row(const oscarop_map_args_v1& A, int row, int r, int start, bool real, bool placed,
                                          uint32_t rank) {
  int64_t slot = -1, position = 0;
  if (real) {
    const int64_t length = A.lengths[r];
    position = length < 0 ? 0 : length + (row - start);
    if (placed && A.granted[r]) {
      const uint32_t place = (uint32_t)length + rank, bs = (uint32_t)A.block_size;  // below 2^31: it was granted
      const int page = A.block_table[r * A.block_table_stride + place / bs];
      if (page >= 0) slot = (int64_t)page * bs + place % bs;
    }
  }
  A.slots[row] = slot;
  A.positions[row] = position;
}

__global__ __launch_bounds__(kMap) void map_kernel(MapParams P) {
  const oscarop_map_args_v1& A = P.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int reqs = A.num_reqs, bs = A.block_size;
  const int rows = (int)A.num_tokens;
  __shared__ uint32_t s_part[kMapWaves];
  __shared__ int32_t s_start[kStarts + 1];
  __shared__ uint64_t s_word[kWords + 1];
  __shared__ uint32_t s_pre[kWords + 1];
  __shared__ uint32_t s_most;
  const int words = (rows + 63) / 64;
  if (A.keep != nullptr) {
    for (int w = wave; w < words; w += kMapWaves) {
      const int i = 64 * w + lane;
      const uint64_t b = __ballot(i < rows && A.keep[i] != 0);
      if (lane == 0) s_word[w] = b;
    }
    if (tid == 0) s_word[words] = 0;
    __syncthreads();
    // words <= kWords = kMap: one a thread
    uint32_t total;
    const uint32_t mine = tid < words ? __popcll(s_word[tid]) : 0;
    const uint32_t before = scan_sat(mine, &total, s_part);
    if (tid < words) s_pre[tid] = before;
    if (tid == 0) s_pre[words] = total;
    if (!P.rows_too && tid < words) P.word_sum[tid] = before;
  }
  if (tid == 0) s_most = 0;
  __syncthreads();
  auto marks_before = [&](int row) {
    return s_pre[row >> 6] + __popcll(s_word[row >> 6] & ((1ull << (row & 63)) - 1));
  };
  // thread t: requests [t run, (t + 1) run)
  const int run = (reqs + kMap - 1) / kMap;
  const int first = min(tid * run, reqs), last = min(first + run, reqs);
  uint32_t mine = 0, total;
  for (int r = first; r < last; ++r) {
    const int c = A.counts[r];
    mine = add_sat(mine, c < 0 ? 0u : (uint32_t)c);
  }
  const uint32_t start = scan_sat(mine, &total, s_part);
  if (tid == 0) {
    const int end = total > (uint32_t)rows ? rows : (int)total;
    A.query_start_loc[reqs] = end;
    if (reqs <= kStarts) s_start[reqs] = end;
  }
  // what each request asks for: its growth, and its pages (0 where it does not fit)
  auto look = [&](int r, uint32_t at, int& length, uint32_t& grown, uint32_t& need, bool& fits) {
    length = A.lengths[r];
    const int count = max(A.counts[r], 0);
    fits = length >= 0 && (uint64_t)at + (uint64_t)count <= (uint64_t)rows;
    grown = 0;
    need = 0;
    if (!fits) return;
    grown = A.keep != nullptr ? marks_before((int)at + count) - marks_before((int)at) : (uint32_t)count;
    const int64_t upto = (int64_t)length + grown;
    const int64_t pages = (upto + bs - 1) / bs;
    fits = upto <= INT32_MAX && pages <= A.block_table_cols;
    if (fits) need = (uint32_t)(pages - ((int64_t)length + bs - 1) / bs);
  };
  uint32_t at = start, needs = 0;
  for (int r = first; r < last; ++r) {
    int length;
    uint32_t grown, need;
    bool fits;
    look(r, at, length, grown, need, fits);
    needs = add_sat(needs, need);
    at = add_sat(at, (uint32_t)max(A.counts[r], 0));
  }
  int free = *A.pool_count;
  free = free < 0 ? 0 : (free > A.pool_size ? (int)A.pool_size : free);
  const uint32_t before = scan_sat(needs, &total, s_part);
  // T: the largest running sum that fits
  uint32_t sum = before, most = 0;
  at = start;
  for (int r = first; r < last; ++r) {
    int length;
    uint32_t grown, need;
    bool fits;
    look(r, at, length, grown, need, fits);
    sum = add_sat(sum, need);
    if (sum <= (uint32_t)free) most = sum;
    at = add_sat(at, (uint32_t)max(A.counts[r], 0));
  }
  if (most > 0) atomicMax(&s_most, most);
  __syncthreads();
  const int base = free - (int)s_most;
  sum = before;
  at = start;
  for (int k = 0; k < run; ++k) {
    const int r = first + k;
    int from = 0, many = 0, column = 0;
    if (r < last) {
      int length;
      uint32_t grown, need;
      bool fits;
      look(r, at, length, grown, need, fits);
      sum = add_sat(sum, need);
      const bool granted = fits && (need == 0 || sum <= (uint32_t)free);
      const int begin = at > (uint32_t)rows ? rows : (int)at;
      A.query_start_loc[r] = begin;
      if (reqs <= kStarts) s_start[r] = begin;
      A.seq_lens[r] = granted ? length + (int)grown : length;
      A.granted[r] = granted;
      if (!P.rows_too && A.keep != nullptr) P.kept_at[r] = marks_before(begin);
      if (granted && need > 0) {
        from = base + (int)(sum - need);
        many = (int)need;
        column = (int)(((int64_t)length + bs - 1) / bs);
      }
      at = add_sat(at, (uint32_t)max(A.counts[r], 0));
    }
    // the table's new columns: a few by the request's own thread, more by its wave
    int32_t* row = A.block_table + (int64_t)(r < last ? r : 0) * A.block_table_stride + column;
    if (many <= kOwnPages) {
#pragma unroll
      for (int i = 0; i < kOwnPages; ++i)
        if (i < many) row[i] = A.pool_pages[from + i];
    }
    uint64_t large = __ballot(many > kOwnPages);
    while (large != 0) {
      const int who = __ffsll((unsigned long long)large) - 1;
      large &= large - 1;
      const int f = __builtin_amdgcn_readlane(from, who), n = __builtin_amdgcn_readlane(many, who);
      const int rr = __builtin_amdgcn_readlane(r, who), cc = __builtin_amdgcn_readlane(column, who);
      int32_t* to = A.block_table + (int64_t)rr * A.block_table_stride + cc;
      for (int i = lane; i < n; i += 64) to[i] = A.pool_pages[f + i];
    }
  }
  __syncthreads();  // the table, the starts and the grants are there for the rows
  if (tid == 0) *A.pool_count = base;
  if (!P.rows_too) return;
  const int32_t* starts = reqs <= kStarts ? s_start : A.query_start_loc;
  for (int row = tid; row < rows; row += kMap) {
    const int r = reqs > 0 ? request_of_row(starts, reqs, row) : 0;
    const bool real = reqs > 0 && row >= starts[0] && row < starts[reqs];
    const int begin = reqs > 0 ? starts[r] : 0;
    bool placed = real;
    uint32_t rank = real ? row - begin : 0;
    if (A.keep != nullptr) {
      placed = real && ((s_word[row >> 6] >> (row & 63)) & 1);
      rank = real ? marks_before(row) - marks_before(begin) : 0;
    }
    write_row(A, row, r, begin, real, placed, rank);
  }
}

__global__ __launch_bounds__(kRows) void rows_kernel(MapParams P) {
  const oscarop_map_args_v1& A = P.a;
  const int row = blockIdx.x * kRows + threadIdx.x, lane = threadIdx.x & 63;
  const int rows = (int)A.num_tokens, reqs = A.num_reqs;
  const int32_t* starts = A.query_start_loc;
  const bool in = row < rows;
  const int r = request_of_row(starts, reqs, row);
  const int begin = starts[r];
  const bool real = in && row < starts[reqs];
  bool placed = real;
  uint32_t rank = row - begin;
  if (A.keep != nullptr) {
    // a wave's rows are one word of marks
    const bool mark = in && A.keep[in ? row : 0] != 0;
    const uint64_t word = __ballot(mark);
    placed = real && mark;
    rank = real ? P.word_sum[row >> 6] + __popcll(word & ((1ull << lane) - 1)) - P.kept_at[r] : 0;
  }
  if (in) write_row(A, row, r, begin, real, placed, rank);
}

__global__ __launch_bounds__(kMap) void release_kernel(oscarop_release_args_v1 A) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int reqs = A.num_reqs, bs = A.block_size;
  __shared__ uint32_t s_part[kMapWaves];
  __shared__ uint32_t s_most;
  if (tid == 0) s_most = 0;
  int count = *A.pool_count;
  count = count < 0 ? 0 : (count > A.pool_size ? (int)A.pool_size : count);
  const uint32_t room = (uint32_t)(A.pool_size - count);
  const int run = (reqs + kMap - 1) / kMap;
  const int first = min(tid * run, reqs), last = min(first + run, reqs);
  auto look = [&](int r, int& column) -> uint32_t {
    const int64_t from = A.lengths[r], to = A.new_lengths[r];
    column = 0;
    if (to < 0 || to > from || (from + bs - 1) / bs > A.block_table_cols) return 0;
    column = (int)((to + bs - 1) / bs);
    return (uint32_t)((from + bs - 1) / bs - column);
  };
  uint32_t mine = 0, total;
  int column;
  for (int r = first; r < last; ++r) mine = add_sat(mine, look(r, column));
  uint32_t sum = scan_sat(mine, &total, s_part), most = 0;
  for (int k = 0; k < run; ++k) {
    const int r = first + k;
    int many = 0, to = 0;
    column = 0;
    if (r < last) {
      const uint32_t n = look(r, column);
      sum = add_sat(sum, n);
      if (sum <= room) {
        most = sum;
        many = (int)n;
        to = count + (int)(sum - n);
      }
    }
    const int32_t* row = A.block_table + (int64_t)(r < last ? r : 0) * A.block_table_stride + column;
    if (many <= kOwnPages) {
#pragma unroll
      for (int i = 0; i < kOwnPages; ++i)
        if (i < many) A.pool_pages[to + i] = row[i];
    }
    uint64_t large = __ballot(many > kOwnPages);
    while (large != 0) {
      const int who = __ffsll((unsigned long long)large) - 1;
      large &= large - 1;
      const int t = __builtin_amdgcn_readlane(to, who), n = __builtin_amdgcn_readlane(many, who);
      const int rr = __builtin_amdgcn_readlane(r, who), cc = __builtin_amdgcn_readlane(column, who);
      const int32_t* src = A.block_table + (int64_t)rr * A.block_table_stride + cc;
      for (int i = lane; i < n; i += 64) A.pool_pages[t + i] = src[i];
    }
  }
  if (most > 0) atomicMax(&s_most, most);
  __syncthreads();
  if (tid == 0) *A.pool_count = count + (int)s_most;
}

int64_t map_workspace(int64_t num_reqs, int64_t num_tokens, bool keep) {
  if (num_reqs < 0 || num_reqs > kMostReqs || num_tokens < 0 || num_tokens > kMostRows || (keep && num_tokens > kMostKeep))
    return -22;
  return keep && num_tokens > kSmallStep ? 4 * (num_reqs + (num_tokens + 63) / 64) : 0;
}

}  // namespace

}  // namespace oscar

using namespace oscar;

extern "C" int64_t oscarop_map_workspace_bytes_v1(int64_t num_reqs, int64_t num_tokens, int32_t keep) {
  return map_workspace(num_reqs, num_tokens, keep != 0);
}

extern "C" int oscarop_map_v1(const oscarop_map_args_v1* args, void* stream) {
  if (!args) return fail(-22, "oscarop_map_v1: null args");
  const oscarop_map_args_v1& a = *args;
  const int64_t need = map_workspace(a.num_reqs, a.num_tokens, a.keep != nullptr);
  if (need < 0)
    return fail(-22, "oscarop_map_v1: at most %lld requests, and %lld rows with marks", (long long)kMostReqs,
                (long long)kMostKeep);
  if (a.block_size < 1) return fail(-22, "oscarop_map_v1: block_size must be positive");
  if (!a.query_start_loc || !a.pool_count || a.pool_size < 0 || a.pool_size > INT32_MAX || (a.pool_size > 0 && !a.pool_pages) ||
      (a.num_tokens > 0 && (!a.slots || !a.positions)) ||
      (a.num_reqs > 0 && (!a.lengths || !a.counts || !a.seq_lens || !a.granted || !a.block_table)))
    return fail(-22, "oscarop_map_v1: missing pointer");
  if (a.num_reqs > 0 && (a.block_table_cols < 0 || a.block_table_rows < a.num_reqs ||
                         (a.num_reqs > 1 && a.block_table_stride < a.block_table_cols)))
    return fail(-22, "oscarop_map_v1: Missing request block-table rows");
  if (a.workspace_bytes < need || (need > 0 && (!a.workspace || ((uintptr_t)a.workspace & 3))))
    return fail(-28, "oscarop_map_v1: workspace of %lld bytes < %lld", (long long)a.workspace_bytes, (long long)need);
  MapParams p{};
  p.a = a;
  p.rows_too = a.num_tokens <= kSmallStep || a.num_reqs == 0;
  p.kept_at = (uint32_t*)a.workspace;
  p.word_sum = p.kept_at + a.num_reqs;
  const hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(map_kernel, dim3(1), dim3(kMap), 0, s, p);
  OSCAR_CHECK_LAUNCH("map_kernel");
  if (!p.rows_too) {
    hipLaunchKernelGGL(rows_kernel, dim3((unsigned)((a.num_tokens + kRows - 1) / kRows)), dim3(kRows), 0, s, p);
    OSCAR_CHECK_LAUNCH("rows_kernel");
  }
  return 0;
}

extern "C" int oscarop_release_v1(const oscarop_release_args_v1* args, void* stream) {
  if (!args) return fail(-22, "oscarop_release_v1: null args");
  const oscarop_release_args_v1& a = *args;
  if (a.num_reqs < 0 || a.num_reqs > kMostReqs)
    return fail(-22, "oscarop_release_v1: at most %lld requests", (long long)kMostReqs);
  if (a.block_size < 1) return fail(-22, "oscarop_release_v1: block_size must be positive");
  if (a.num_reqs == 0) return 0;
  if (!a.lengths || !a.new_lengths || !a.block_table || !a.pool_count || a.pool_size < 0 || a.pool_size > INT32_MAX ||
      (a.pool_size > 0 && !a.pool_pages))
    return fail(-22, "oscarop_release_v1: missing pointer");
  if (a.block_table_cols < 0 || a.block_table_rows < a.num_reqs || (a.num_reqs > 1 && a.block_table_stride < a.block_table_cols))
    return fail(-22, "oscarop_release_v1: Missing request block-table rows");
  hipLaunchKernelGGL(release_kernel, dim3(1), dim3(kMap), 0, (hipStream_t)stream, a);
  OSCAR_CHECK_LAUNCH("release_kernel");
  return 0;
}
