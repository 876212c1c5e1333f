// Eviction from the paged INT2 cache by accumulated attention weight (gfx950).
//
// Of request r's tokens [sink, tail) the `drop` of least weight go, per KV head, `drop`
// being whole pages: behind the new end (tail - drop) whole pages of the block table come
// free, and the tail's pages, with the tokens' FP32 window copies, stay where they are.
// Attention does not depend on the order of its keys, so nothing is compacted: the kept
// tokens behind the new end move into the places of the dropped ones before it (as many, as
// the counts say), the others stay.  The i-th place takes the i-th such token, both
// ascending, so that the result is fixed.
//
//   evict_select_kernel  one workgroup per (request, KV head): the drop-th smallest weight by
//                        radix selection, then the lists of places and movers and the new
//                        weights
//   evict_move_kernel    the slots' bytes and weights from mover to place, and the places'
//                        window tags
#include "common.h"

#include "../../include/oscar_operators.h"

namespace oscar {

namespace {

constexpr int kSelect = 1024;  // threads of a selecting workgroup
constexpr int kMove = 256;

struct EvictParams {
  oscarop_evict_args_v1 a;
  oscar_staging_v1 st;
  int has_stage;
  int64_t pairs;    // entries of a list at most
  int32_t* counts;  // [num_reqs][Hk]
  int32_t* places;  // [num_reqs][Hk][pairs]
  int32_t* movers;
};

struct Request {
  int seq, sink, tail, drop;
  bool ok;
};

// requests[r] = seq_len, sink, tail, drop; one that does not fit is left alone
__device__ __forceinline__ Request request_of(const oscarop_evict_args_v1& A, int r) {
  const int32_t* q = A.requests + 4 * (int64_t)r;
  Request x{q[0], q[1], q[2], q[3], true};
  const int bs = (int)A.cache.block_size;
  x.ok = x.sink >= 0 && x.drop >= 0 && x.tail <= x.seq && x.drop <= x.tail - x.sink && x.seq <= A.weights_cols &&
         x.drop <= A.max_drop && (x.seq <= 0 || (x.seq - 1) / bs < A.block_table_cols);
  return x;
}

// weights in ascending order as unsigned numbers: +0 and -0 alike, NaN above everything
__device__ __forceinline__ uint32_t order_of(float w) {
  uint32_t u = __float_as_uint(w);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if (u == 0x80000000u) u = 0;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// exclusive prefix sum over the workgroup of one number per thread; *total gets the sum
__device__ __forceinline__ int scan(int x, int* total, int* s_part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int v = x;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int y = __shfl_up(v, d);
    v += lane >= d ? y : 0;
  }
  __syncthreads();  // s_part of the call before has been read
  if (lane == 63) s_part[wave] = v;
  __syncthreads();
  int before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < kSelect / 64; ++w) {
    const int p = s_part[w];
    before += w < wave ? p : 0;
    sum += p;
  }
  *total = sum;
  return before + v - x;
}

__global__ __launch_bounds__(kSelect) void evict_select_kernel(EvictParams P) {
  const oscarop_evict_args_v1& A = P.a;
  const int tid = threadIdx.x, h = blockIdx.x, r = blockIdx.y;
  const int64_t hk = A.cache.num_kv_heads;
  const Request q = request_of(A, r);
  const float* w = A.weights + r * A.weights_stride_request + h * A.weights_stride_head;
  float* out = A.weights_out + r * A.out_stride_request + h * A.out_stride_head;
  const int64_t list = (int64_t)r * hk + h;
  if (!q.ok) {
    for (int64_t t = tid; t < A.weights_cols; t += kSelect) out[t] = w[t];
    if (tid == 0) P.counts[list] = 0;
    return;
  }
  const int end = q.tail - q.drop;  // where the tail goes
  // the tail's weights, then zeros
  for (int64_t t = end + tid; t < A.weights_cols; t += kSelect) out[t] = t < q.seq - q.drop ? w[t + q.drop] : 0.f;
  __shared__ int s_hist[256];
  __shared__ int s_part[kSelect / 64];
  __shared__ uint32_t s_prefix;
  __shared__ int s_left;
  // ---- the drop-th smallest: byte by byte from the top, `left` = its rank among those that
  // share the bytes found so far
  uint32_t prefix = 0;
  int left = q.drop;  // drop the `left` smallest
  if (q.drop > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kSelect) s_hist[i] = 0;
      __syncthreads();
      for (int t = q.sink + tid; t < q.tail; t += kSelect) {
        const uint32_t u = order_of(w[t]);
        if (shift == 24 || (u >> (shift + 8)) == prefix) atomicAdd(&s_hist[(u >> shift) & 255], 1);
      }
      __syncthreads();
      if (tid == 0) {
        int b = 0, sum = 0;
        while (sum + s_hist[b] < left) sum += s_hist[b++];
        s_prefix = prefix << 8 | b;
        s_left = left - sum;
      }
      __syncthreads();
      prefix = s_prefix;
      left = s_left;
    }
  }
  // weights below `prefix` go, and of those equal to it the last `left`: those whose rank
  // among the equal ones is at least equal - left
  int equal = 0;
  if (q.drop > 0) {
    int mine = 0;
    for (int t = q.sink + tid; t < q.tail; t += kSelect) mine += order_of(w[t]) == prefix;
    scan(mine, &equal, s_part);
  }
  int32_t* places = P.places + list * P.pairs;
  int32_t* movers = P.movers + list * P.pairs;
  for (int t = tid; t < q.sink && t < end; t += kSelect) out[t] = w[t];
  int n_equal = 0, n_place = 0, n_mover = 0, total;
  for (int t0 = q.sink; t0 < q.tail; t0 += kSelect) {
    const int t = t0 + tid;
    const bool in = t < q.tail;
    const float x = in ? w[t] : 0.f;
    const uint32_t u = order_of(x);
    const bool same = in && q.drop > 0 && u == prefix;
    const int rank = n_equal + scan(same, &total, s_part);
    n_equal += total;
    const bool gone = in && q.drop > 0 && (u < prefix || (same && rank >= equal - left));
    const bool place = gone && t < end, mover = in && !gone && t >= end;
    const int at = n_place + scan(place, &total, s_part);
    n_place += total;
    const int from = n_mover + scan(mover, &total, s_part);
    n_mover += total;
    if (place) places[at] = t;
    if (mover) movers[from] = t;
    if (in && !gone && t < end) out[t] = x;
  }
  if (tid == 0) P.counts[list] = n_place;
}

__global__ __launch_bounds__(kMove) void evict_move_kernel(EvictParams P) {
  const oscarop_evict_args_v1& A = P.a;
  const int h = blockIdx.y, r = blockIdx.z;
  const int64_t hk = A.cache.num_kv_heads, list = (int64_t)r * hk + h;
  const int many = P.counts[list];
  const int bs = (int)A.cache.block_size, words = (int)A.cache.head_dim / 16;  // 4-byte words of codes
  const int32_t* row = A.block_table + (int64_t)r * A.block_table_stride;
  // 32 lanes per move: two words of constants and `words` of codes for K, then for V
  const int lane = threadIdx.x & 31;
  for (int i = (blockIdx.x * kMove + threadIdx.x) / 32; i < many; i += gridDim.x * (kMove / 32)) {
    const int to = P.places[list * P.pairs + i], from = P.movers[list * P.pairs + i];
    const int64_t bt = row[to / bs], bf = row[from / bs];
    if (lane == 0)
      A.weights_out[r * A.out_stride_request + h * A.out_stride_head + to] =
          A.weights[r * A.weights_stride_request + h * A.weights_stride_head + from];
    if (bt < 0 || bt >= A.cache.num_blocks || bf < 0 || bf >= A.cache.num_blocks) continue;  // never out of the cache
    auto move = [&](uint8_t* base, const int64_t* stride, int at) {
      const int64_t head = h * stride[2] + at;
      *(uint32_t*)(base + bt * stride[0] + to % bs * stride[1] + head) =
          *(const uint32_t*)(base + bf * stride[0] + from % bs * stride[1] + head);
    };
    for (int x = lane; x < 2 + 2 * words; x += 32) {
      if (x < 2) move(A.cache.k, A.cache.k_stride, 4 * x);
      else if (x < 2 + words) move(A.cache.k, A.cache.k_stride, 32 + 4 * (x - 2));
      else move(A.cache.v, A.cache.v_stride, 4 * (x - 2 - words));
    }
    if (lane == 0 && P.has_stage) {
      int64_t* tag = P.st.owner + bt % P.st.rows * bs + to % bs;
      if (*tag == bt) *tag = -1;
    }
  }
}

}  // namespace

}  // namespace oscar

using namespace oscar;

extern "C" int64_t oscarop_evict_workspace_bytes_v1(int64_t num_reqs, int64_t num_kv_heads, int64_t max_drop) {
  if (num_reqs < 0 || num_kv_heads < 1 || max_drop < 0) return -22;
  return num_reqs * num_kv_heads * (2 * max_drop + 1) * (int64_t)sizeof(int32_t);
}

extern "C" int oscarop_evict_v1(const oscarop_evict_args_v1* args, void* stream) {
  const char* name = "oscarop_evict_v1";
  if (!args) return fail(-22, "%s: null args", name);
  const oscarop_evict_args_v1& a = *args;
  const int64_t D = a.cache.head_dim, hk = a.cache.num_kv_heads, bs = a.cache.block_size;
  if (D != 128 && D != 256) return fail(-22, "%s: head_dim %lld unsupported (128/256)", name, (long long)D);
  if (a.num_reqs < 0 || a.max_drop < 0) return fail(-22, "%s: negative size", name);
  if (a.num_reqs == 0) return 0;
  if (!a.weights || !a.weights_out || !a.block_table || !a.requests || !a.cache.k || !a.cache.v)
    return fail(-22, "%s: missing pointer", name);
  if (hk < 1 || hk > 0xffff || a.num_reqs > 0xffff || a.weights_cols < 1 || a.weights_cols >= (1ll << 30))
    return fail(-22, "%s: sizes out of range", name);
  if (bs < 1 || bs > (1 << 20) || a.max_drop % bs) return fail(-22, "%s: max_drop must be whole pages", name);
  if (a.block_table_rows < a.num_reqs || a.block_table_cols < 1 || a.block_table_stride < a.block_table_cols)
    return fail(-22, "%s: Missing request block-table rows", name);
  for (int i = 0; i < 3; ++i)
    if ((a.cache.k_stride[i] & 3) || (a.cache.v_stride[i] & 3)) return fail(-22, "%s: cache slots must be 4-byte aligned", name);
  if ((((uintptr_t)a.cache.k) & 3) || (((uintptr_t)a.cache.v) & 3))
    return fail(-22, "%s: cache slots must be 4-byte aligned", name);
  auto overlap = [&](int64_t head, int64_t request) {
    return (hk > 1 && head < a.weights_cols) || (a.num_reqs > 1 && request < (hk - 1) * head + a.weights_cols);
  };
  if (overlap(a.weights_stride_head, a.weights_stride_request) || overlap(a.out_stride_head, a.out_stride_request))
    return fail(-22, "%s: weights of two heads or requests overlap", name);
  auto end_of = [&](const float* p, int64_t head, int64_t request) {
    return p + (a.num_reqs - 1) * request + (hk - 1) * head + a.weights_cols;
  };
  if (a.weights_out < end_of(a.weights, a.weights_stride_head, a.weights_stride_request) &&
      a.weights < end_of(a.weights_out, a.out_stride_head, a.out_stride_request))
    return fail(-22, "%s: weights_out overlaps weights", name);
  if (a.staging && (a.staging->rows < 1 || !a.staging->owner)) return fail(-22, "%s: staging arena rows out of range", name);
  const int64_t need = oscarop_evict_workspace_bytes_v1(a.num_reqs, hk, a.max_drop);
  if (!a.workspace || a.workspace_bytes < need || (((uintptr_t)a.workspace) & 15))
    return fail(-22, "%s: 16-byte aligned workspace of %lld bytes required", name, (long long)need);
  EvictParams p{};
  p.a = a;
  p.has_stage = a.staging != nullptr;
  if (a.staging) p.st = *a.staging;
  p.pairs = a.max_drop;
  p.counts = (int32_t*)a.workspace;
  p.places = p.counts + a.num_reqs * hk;
  p.movers = p.places + a.num_reqs * hk * p.pairs;
  hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(evict_select_kernel, dim3((unsigned)hk, (unsigned)a.num_reqs), dim3(kSelect), 0, s, p);
  OSCAR_CHECK_LAUNCH("evict_select_kernel");
  if (a.max_drop == 0) return 0;
  const int64_t per = kMove / 32, wgs = (a.max_drop + per - 1) / per;
  hipLaunchKernelGGL(evict_move_kernel, dim3((unsigned)(wgs < 256 ? wgs : 256), (unsigned)hk, (unsigned)a.num_reqs), dim3(kMove), 0, s,
                     p);
  OSCAR_CHECK_LAUNCH("evict_move_kernel");
  return 0;
}
