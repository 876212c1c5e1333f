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
//                        radix selection, then the lists of places and movers, and the new
//                        weights up to the new end
//   evict_move_kernel    the slots' bytes and weights from mover to place, the places' window
//                        tags, and the new weights from the new end on
//
// The selection is bound by what one compute unit issues, some eighty instructions a token in
// all, not by the 4 bytes per token it reads (31000 tokens 23 us, a third of it the reading
// with the first digit and a third the lists): the weights lie in LDS as ordered numbers and
// every thread takes a run of consecutive tokens, so that marks and lists are counted without
// talk between lanes and only a thread's totals are scanned.  (More compute units a list would
// have to meet after the first digit and before the lists are written; not built.)
#include <type_traits>

#include "common.h"

#include "../../include/oscar_operators.h"

namespace oscar {

namespace {

constexpr int kSelect = 1024;          // threads of a selecting workgroup
constexpr int kSelectWaves = kSelect / 64;
constexpr int kRun = 32;               // consecutive tokens of a thread at most
constexpr int kLoads = 16;             // loads of a thread in flight
constexpr int kStep = 4;               // of them at a time; a run is a multiple of it
constexpr int kFew = 256;              // candidates whose ranks are counted pair by pair
constexpr int kBlock = kSelect * kRun; // tokens held at a time; longer lists are read again in every step
constexpr int kDigit = 11;             // bits of the second and third digit, two bins a thread
constexpr int kFirst = 10;             // bits of the first: sign, exponent and one more
constexpr int kCopies = 4;             // of its bins: most weights share a few exponents, and atomics of one bin take turns
constexpr int kBins = kCopies << kFirst;
constexpr int kMove = 256;
constexpr int64_t kMostLists = 0xffff;       // requests, and KV heads: an axis of the grid each
constexpr int64_t kMostTokens = 1ll << 30;   // of a list, below: places are offsets of 32 bits
// workgroups of evict_move_kernel: about one per 32 moves of a large call, since fewer than
// max_drop tokens move (128000 moves in 8192 / 4096 / 2048 workgroups: 14.9 / 13.6 / 14.5 us)
constexpr int64_t kMoveWorkgroups = 4096;

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
  x.ok = x.sink >= 0 && x.drop >= 0 && x.sink <= x.tail && x.tail <= x.seq && x.drop <= x.tail - x.sink && x.seq <= A.weights_cols &&
         x.drop <= A.max_drop && (x.seq <= 0 || (x.seq - 1) / bs < A.block_table_cols);
  return x;
}

// weights in ascending order as unsigned numbers: +0 and -0 alike, NaN above everything
__device__ __forceinline__ uint32_t order_of(float w) {
  const uint32_t u = __float_as_uint(w + 0.f);  // (-0 becomes +0)
  return w != w ? 0xffffffffu : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}

// exclusive prefix sum over the workgroup of one number per thread; *total gets the sum
__device__ __forceinline__ uint32_t scan(uint32_t x, uint32_t* total, uint32_t* s_part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // over the wave: within rows of 16 lanes by row_shr 1, 2, 4, 8, then the rows' last lanes
  // to the rows behind them (row_bcast 15, 31)
  uint32_t v = x;
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  __syncthreads();  // s_part of the call before has been read
  if (lane == 63) s_part[wave] = v;
  __syncthreads();
  uint32_t before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < kSelectWaves; ++w) {
    before += w < wave ? s_part[w] : 0;
    sum += s_part[w];
  }
  *total = sum;
  return before + v - x;
}

// element i < 2^30 of an array, by an offset of 32 bits
template <class T>
__device__ __forceinline__ T* at32(T* p, int i) {
  return (T*)((std::conditional_t<std::is_const_v<T>, const char*, char*>)p + (uint32_t)i * (uint32_t)sizeof(T));
}

// where number i of a block lies in s_buf: a word is left out every 32, so that the threads'
// runs start in different banks (four numbers from a multiple of four lie side by side, and
// 32 n further on is 33 n further on)
__device__ __forceinline__ int place_of(int i) { return i + i / 32; }
constexpr int kPitch = kSelect + kSelect / 32;

__global__ __launch_bounds__(kSelect) void evict_select_kernel(EvictParams P) {
  const oscarop_evict_args_v1& A = P.a;
  const int tid = threadIdx.x, lane = tid & 63, h = blockIdx.x, r = blockIdx.y;
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
  if (q.drop == 0) {
    for (int t = tid; t < end; t += kSelect) out[t] = w[t];
    if (tid == 0) P.counts[list] = 0;
    return;
  }
  const int n = q.tail - q.sink;  // token sink + i, i < n
  __shared__ uint32_t s_buf[kBlock + kBlock / 32];
  __shared__ int s_bin[kBins];
  __shared__ uint32_t s_part[kSelectWaves];
  __shared__ uint32_t s_prefix, s_low, s_high;
  __shared__ int s_left, s_equal, s_places, s_few;
  __shared__ uint32_t s_cand[kFew];
  for (int i = tid; i < kBins; i += kSelect) s_bin[i] = 0;
  if (tid == 0) {
    s_low = 0xffffffffu;
    s_high = 0;
    s_few = 0;
  }
  // ---- blocks of the list; thread t has the tokens base + t per + b, b < mine, of a block,
  // `per` being a multiple of kStep
  int base = 0, per = 0, mine = 0;
  auto load = [&](int at, auto first) __attribute__((always_inline)) {
    constexpr bool FIRST = decltype(first)::value;  // the list's first reading: counts the first digit, copies the weights
    const int many = n - at < kBlock ? n - at : kBlock;
    base = at;
    per = (many + kSelect * kStep - 1) / (kSelect * kStep) * kStep;
    mine = min(max(many - tid * per, 0), per);
    __syncthreads();  // s_buf of the block before has been read
    const int run = per;
    for (int b = 0; b < run; b += kLoads) {
      float x[kLoads];
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        const int i = (b + u) * kSelect + tid;
        x[u] = i < many ? *at32(w, q.sink + at + i) : 0.f;
      }
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        const int i = (b + u) * kSelect + tid;
        if (b + u >= run) break;
        const uint32_t k = i < many ? order_of(x[u]) : 0xffffffffu;
        s_buf[place_of(tid) + (b + u) * kPitch] = k;
        if constexpr (FIRST) {
          // (places get their movers' weights later)
          if (i < many && q.sink + at + i < end) *at32(out, q.sink + at + i) = x[u];
          if (i < many) atomicAdd(&s_bin[kCopies * (k >> (32 - kFirst)) + lane % kCopies], 1);
        }
      }
    }
    __syncthreads();
  };
  auto each = [&](auto use) __attribute__((always_inline)) {  // use(b, key, place): of every thread at once, b < mine or not
    for (int b = 0; b < per; b += kStep) {
      uint32_t k[kStep];
#pragma unroll
      for (int u = 0; u < kStep; ++u) k[u] = s_buf[place_of(tid * per + b) + u];
#pragma unroll
      for (int u = 0; u < kStep; ++u) use(b + u, k[u], place_of(tid * per + b) + u);
    }
  };
  const bool one = n <= kBlock;
  auto blocks = [&](auto step) __attribute__((always_inline)) {
    if (one) return step();
    for (int at = 0; at < n; at += kBlock) {
      load(at, std::false_type{});
      step();
    }
  };
  // ---- the drop-th smallest, digit by digit from the top.  The bin of the digit that holds
  // rank `left` among those that share the digits found so far:
  uint32_t prefix = 0;
  int left = q.drop, equal = 0;
  auto find = [&](int bits, auto first) __attribute__((always_inline)) {
    constexpr bool FIRST = decltype(first)::value;
    static_assert(kSelect == 1 << kFirst && 2 * kSelect == 1 << kDigit);
    __syncthreads();
    int c[FIRST ? kCopies : 2];
    int* mine_bins = s_bin + (FIRST ? kCopies : 2) * tid;
    uint32_t b0 = 0, b1 = 0, all;
#pragma unroll
    for (int i = 0; i < (FIRST ? kCopies : 2); ++i) {
      c[i] = mine_bins[i];
      mine_bins[i] = 0;
    }
    if constexpr (FIRST) {
#pragma unroll
      for (int i = 0; i < kCopies; ++i) b0 += c[i];
    } else {
      b0 = c[0];
      b1 = c[1];
    }
    const uint32_t before = scan(b0 + b1, &all, s_part);
    if (before < (uint32_t)left && (uint32_t)left <= before + b0 + b1) {
      const bool second = (uint32_t)left > before + b0;
      s_prefix = prefix << bits | (uint32_t)(FIRST ? tid : 2 * tid + second);
      s_left = left - (int)(before + (second ? b0 : 0));
      s_equal = second ? b1 : b0;
    }
    __syncthreads();
    prefix = s_prefix;
    left = s_left;
    equal = s_equal;
  };
  for (int at = 0; at < n; at += kBlock) load(at, std::true_type{});
  find(0, std::true_type{});
  // few candidates: every one's rank among them, pair by pair
  auto finish = [&](int shift) __attribute__((always_inline)) {
    blocks([&]() __attribute__((always_inline)) {
      each([&](int b, uint32_t k, int) __attribute__((always_inline)) {
        if (b < mine && k >> shift == prefix) s_cand[atomicAdd(&s_few, 1)] = k;
      });
    });
    __syncthreads();
    if (tid < equal) {
      const uint32_t k = s_cand[tid];
      int below = 0, same = 0;
      for (int i = 0; i < equal; ++i) {
        below += s_cand[i] < k;
        same += s_cand[i] == k;
      }
      if (below < left && left <= below + same) {  // equal candidates write the same
        s_prefix = k;
        s_left = left - below;
        s_equal = same;
      }
    }
    __syncthreads();
    prefix = s_prefix;
    left = s_left;
    equal = s_equal;
  };
  constexpr int kShift1 = 32 - kFirst, kShift2 = kShift1 - kDigit;
  static_assert(kShift2 == kDigit);
  if (equal <= kFew) {
    finish(kShift1);
  } else {
    // one value in the bin (equal weights) needs no further digits
    uint32_t low = 0xffffffffu, high = 0;
    blocks([&]() __attribute__((always_inline)) {
      each([&](int b, uint32_t k, int) __attribute__((always_inline)) {
        const bool in = b < mine && k >> kShift1 == prefix;
        low = min(low, in ? k : 0xffffffffu);
        high = max(high, in ? k : 0u);
      });
    });
#pragma unroll
    for (int d = 32; d > 0; d /= 2) {
      const uint32_t y = __shfl_xor(low, d), z = __shfl_xor(high, d);
      low = y < low ? y : low;
      high = z > high ? z : high;
    }
    if (lane == 0 && low <= high) {
      atomicMin(&s_low, low);
      atomicMax(&s_high, high);
    }
    __syncthreads();
    auto digit = [&](int shift, int bits) __attribute__((always_inline)) {
      blocks([&]() __attribute__((always_inline)) {
        each([&](int b, uint32_t k, int) __attribute__((always_inline)) {
          if (b < mine && k >> (shift + bits) == prefix) atomicAdd(&s_bin[(k >> shift) & ((1u << bits) - 1u)], 1);
        });
      });
      find(bits, std::false_type{});
    };
    if (s_low == s_high) {
      prefix = s_low;
    } else {
      digit(kShift2, kDigit);
      if (equal <= kFew) finish(kShift2);
      else digit(0, kShift2);
    }
  }
  // ---- weights below `prefix` go, and of those equal to it the last `left`: those with
  // `keep` of them before.  Of the tokens before one, L are below and E equal: L +
  // max(0, E - keep) of them go.
  const int keep = equal - left;
  auto gone_before = [&](int below, int same) __attribute__((always_inline)) { return below + (same > keep ? same - keep : 0); };
  // a thread's tokens' totals, and those of the tokens before its first
  struct Totals {
    int below, same;  // of the tokens before the thread's first
    int all_below, all_same;
  };
  auto totals = [&](const Totals& carry) __attribute__((always_inline)) {
    uint32_t mine_both = 0, all;  // below in the low half, equal in the high one: a block has 2^15 tokens
    each([&](int, uint32_t k, int) __attribute__((always_inline)) {
      // (numbers past the list, which may equal it, are the last ones)
      mine_both += k < prefix ? 1u : k == prefix ? 0x10000u : 0u;
    });
    const uint32_t before = scan(mine_both, &all, s_part);
    return Totals{carry.all_below + (int)(before & 0xffffu), carry.all_same + (int)(before >> 16),
                  carry.all_below + (int)(all & 0xffffu), carry.all_same + (int)(all >> 16)};
  };
  // how many go before the new end: the wave that has its token counts on from the thread's own
  Totals sum{};
  blocks([&]() __attribute__((always_inline)) {
    sum = totals(sum);
    const int to = end - q.sink - base - tid * per;  // this thread's tokens before the end
    const uint64_t has = __ballot(to >= 0 && to < mine);
    if (has) {
      const int from = __builtin_ctzll(has);
      const int many = __builtin_amdgcn_readlane(to, from), l = __builtin_amdgcn_readlane(sum.below, from), e = __builtin_amdgcn_readlane(sum.same, from);
      const uint32_t k = s_buf[place_of((tid - lane + from) * per + (lane < many ? lane : 0))];
      const int more_l = __popcll(__ballot(lane < many && k < prefix)), more_e = __popcll(__ballot(lane < many && k == prefix));
      if (lane == 0) s_places = gone_before(l + more_l, e + more_e);
    }
  });
  __syncthreads();
  const int places = s_places;
  // ---- the lists: a key's place gets the tokens that go before its own, and whether that
  // goes; then the block's tokens in order, so that the lists' parts are written side by side
  int32_t* place_list = P.places + list * P.pairs;
  int32_t* mover_list = P.movers + list * P.pairs;
  if (!one) sum = Totals{};
  blocks([&]() __attribute__((always_inline)) {
    if (!one) sum = totals(sum);
    int l = sum.below, e = sum.same;
    each([&](int, uint32_t k, int place) __attribute__((always_inline)) {
      const bool equal_one = k == prefix, gone = k < prefix || (equal_one && e >= keep);
      s_buf[place] = (uint32_t)gone_before(l, e) | (gone ? 0x80000000u : 0u);
      l += k < prefix;
      e += equal_one;
    });
    __syncthreads();
    const int many = n - base < kBlock ? n - base : kBlock;
    for (int i0 = 0; i0 < many; i0 += kStep * kSelect) {
      uint32_t m[kStep];
#pragma unroll
      for (int u = 0; u < kStep; ++u) m[u] = s_buf[place_of(i0) + place_of(tid) + u * kPitch];
#pragma unroll
      for (int u = 0; u < kStep; ++u) {
        const int i = i0 + u * kSelect + tid, t = q.sink + base + i, g = (int)(m[u] & 0x7fffffffu);
        const bool gone = m[u] >> 31;
        if (i < many && gone == (t < end)) *at32(gone ? place_list : mover_list, gone ? g : t - end - (g - places)) = t;
      }
    }
  });
  if (tid == 0) P.counts[list] = places;
}

// A group of D / 16 lanes per move: 8 bytes of constants and the codes of K and V, 16 bytes a
// lane (five lanes of eight at head dim 128, nine of sixteen at 256).  128000 moves at head dim
// 128 14 us: the lines that the scattered slots touch, two read and two written for each move,
// are 43 MB between the L2 and memory, 8.4 us at a large copy's rate.  A group's loads follow on
// each other, list, page, slot; four moves of a group in flight took 17 us.
template <int D>
__global__ __launch_bounds__(kMove) void evict_move_kernel(EvictParams P) {
  constexpr int L = D / 16, W = D / 64;  // lanes of a move; 16-byte parts of a side's codes
  const oscarop_evict_args_v1& A = P.a;
  const int h = blockIdx.y, r = blockIdx.z;
  const int64_t hk = A.cache.num_kv_heads, list = (int64_t)r * hk + h;
  const int many = P.counts[list], bs = (int)A.cache.block_size;
  const int32_t* row = A.block_table + (int64_t)r * A.block_table_stride;
  const float* w = A.weights + r * A.weights_stride_request + h * A.weights_stride_head;
  float* out = A.weights_out + r * A.out_stride_request + h * A.out_stride_head;
  // the first tokens' weights, the tail's, then zeros
  if (const Request q = request_of(A, r); q.ok) {
    for (int t = blockIdx.x * kMove + threadIdx.x; t < q.sink; t += gridDim.x * kMove) out[t] = w[t];
    for (int64_t t = q.tail - q.drop + (int64_t)blockIdx.x * kMove + threadIdx.x; t < A.weights_cols; t += (int64_t)gridDim.x * kMove)
      out[t] = t < q.seq - q.drop ? w[t + q.drop] : 0.f;
  }
  const int lane = threadIdx.x % L;
  const bool v_side = lane > W;
  const int64_t* stride = v_side ? A.cache.v_stride : A.cache.k_stride;
  const int64_t s0 = stride[0], s1 = stride[1];
  uint8_t* base = (v_side ? A.cache.v : A.cache.k) + h * stride[2] + (lane == 0 ? 0 : v_side ? 16 * (lane - 1 - W) : 32 + 16 * (lane - 1));
  for (int i = (blockIdx.x * kMove + threadIdx.x) / L; i < many; i += gridDim.x * (kMove / L)) {
    const int to = P.places[list * P.pairs + i], from = P.movers[list * P.pairs + i];
    const int64_t bt = row[to / bs], bf = row[from / bs];
    if (lane == L - 1) out[to] = w[from];
    if (bt < 0 || bt >= A.cache.num_blocks || bf < 0 || bf >= A.cache.num_blocks) continue;  // never out of the cache
    uint8_t* dst = base + bt * s0 + to % bs * s1;
    const uint8_t* src = base + bf * s0 + from % bs * s1;
    if (lane == 0) *(u32x2*)dst = *(const u32x2*)src;
    else if (lane <= 2 * W) *(u32x4*)dst = *(const u32x4*)src;
    if (lane == L - 2 && P.has_stage) {
      int64_t* tag = P.st.owner + bt % P.st.rows * bs + to % bs;
      if (*tag == bt) *tag = -1;
    }
  }
}

}  // namespace

}  // namespace oscar

using namespace oscar;

extern "C" int64_t oscarop_evict_workspace_bytes_v1(int64_t num_reqs, int64_t num_kv_heads, int64_t max_drop) {
  if (num_reqs < 0 || num_kv_heads < 1 || max_drop < 0 || num_reqs > kMostLists || num_kv_heads > kMostLists || max_drop >= kMostTokens)
    return -22;
  int64_t bytes;
  return __builtin_mul_overflow(num_reqs * num_kv_heads, (2 * max_drop + 1) * (int64_t)sizeof(int32_t), &bytes) ? -22 : bytes;
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
  if (hk < 1 || hk > kMostLists || a.num_reqs > kMostLists || a.weights_cols < 1 || a.weights_cols >= kMostTokens || a.max_drop >= kMostTokens)
    return fail(-22, "%s: sizes out of range", name);
  if (bs < 1 || bs > (1 << 20) || a.max_drop % bs) return fail(-22, "%s: max_drop must be whole pages", name);
  if (a.block_table_rows < a.num_reqs || a.block_table_cols < 1 || a.block_table_stride < a.block_table_cols)
    return fail(-22, "%s: Missing request block-table rows", name);
  if ((a.cache.k_stride[0] & 15) || (a.cache.k_stride[1] & 15) || (a.cache.k_stride[2] & 15) || (((uintptr_t)a.cache.k) & 15) ||
      (a.cache.v_stride[0] & 15) || (a.cache.v_stride[1] & 15) || (a.cache.v_stride[2] & 15) || (((uintptr_t)a.cache.v) & 15))
    return fail(-22, "%s: cache slots must be 16-byte aligned", name);
  const Rows2 in{{a.num_reqs, hk}, {a.weights_stride_request, a.weights_stride_head}, a.weights_cols};
  const Rows2 out{{a.num_reqs, hk}, {a.out_stride_request, a.out_stride_head}, a.weights_cols};
  if (in.overlap() || out.overlap()) return fail(-22, "%s: weights of two heads or requests overlap", name);
  if (in.meets(out, ((intptr_t)a.weights_out - (intptr_t)a.weights) / (intptr_t)sizeof(float)))
    return fail(-22, "%s: weights_out overlaps weights", name);
  if (a.staging && (a.staging->rows < 1 || !a.staging->owner)) return fail(-22, "%s: staging arena rows out of range", name);
  const int64_t need = oscarop_evict_workspace_bytes_v1(a.num_reqs, hk, a.max_drop);
  if (need < 0) return fail(-22, "%s: sizes out of range", name);
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
  const dim3 lists((unsigned)hk, (unsigned)a.num_reqs);
  hipLaunchKernelGGL(evict_select_kernel, lists, dim3(kSelect), 0, s, p);
  OSCAR_CHECK_LAUNCH("evict_select_kernel");
  // (moves, and the weights behind the new end: a few pages out of many columns)
  const int64_t per = kMove / (D / 16), moves = (a.max_drop + per - 1) / per, copies = (a.weights_cols + 4 * kMove - 1) / (4 * kMove);
  const int64_t wgs = moves > copies ? moves : copies;
  const int64_t most = (kMoveWorkgroups + hk * a.num_reqs - 1) / (hk * a.num_reqs);
  const dim3 grid((unsigned)(wgs < 1 ? 1 : wgs < most ? wgs : most), (unsigned)hk, (unsigned)a.num_reqs);
  if (D == 256) hipLaunchKernelGGL(evict_move_kernel<256>, grid, dim3(kMove), 0, s, p);
  else hipLaunchKernelGGL(evict_move_kernel<128>, grid, dim3(kMove), 0, s, p);
  OSCAR_CHECK_LAUNCH("evict_move_kernel");
  return 0;
}
