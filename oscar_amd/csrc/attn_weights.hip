// The attention weight that every cached token received from a batch's queries, added to
// what it had: weights[r][h][t] += sum over the rows of request r that KV head h serves of
// exp(s' - lse), s' the row's score of key t (score.h) and lse the row's log-sum-exp, as the
// attention call left it.  Keys are those the attention reads: the packed INT2 history, FP32
// window copies where the owner tag matches, and the current chunk's rows.
//
// S = Q K^T of 32 rows and 32 keys leaves a key's scores in one lane pair (lane % 32: the key;
// registers: the rows), so that the sum over the rows is a sum over registers and crosses
// lanes once.  Every number has one owner, so nothing is atomic and results do not depend on
// the order of workgroups; which kernel runs and where rows are cut depends on the call's sizes,
// and the last bits with them.
//
//   weights_few_kernel   a batch of at most 32 rows per KV head (decode, verification): the
//                        queries stay in LDS and every wave streams key tiles past them, the
//                        next tile's codes in flight.  8 requests of 24576 tokens, 24 rows:
//                        14.9 us; bound by the lookups of the K operands, and in a short
//                        call by what a wave waits for before its first tile
//   weights_many_kernel  more rows: a wave holds the K operands of two tiles in registers and
//                        the row blocks go past, through LDS and shared by the workgroup's
//                        waves; where the keys alone do not fill the chip the rows are cut
//                        into chunks, whose sums weights_sum_kernel adds in their order.  A
//                        block of 32 rows against 256 keys takes 2.1 us a workgroup with two
//                        of them on a compute unit.  2500 fresh tokens of 6 heads: 28.6 us a
//                        call (27 and 4 us by the profiler, which adds about a microsecond to
//                        each), of which the keys' way into registers is 6 us (eight waves of
//                        one tile each, their rows reordered through LDS instead of loaded one
//                        a lane, took as long in all)
#include <type_traits>

#include "common.h"
#include "int2_tile.h"
#include "score.h"
#include "store_quant.h"

#include "../../include/oscar_operators.h"

namespace oscar {

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kTile = 32;
constexpr int kFewRows = 32;                           // of a KV head, for weights_few_kernel
constexpr int kKeyTiles = 2;                           // per wave of weights_many_kernel
constexpr int kGroupKeys = kWaves * kKeyTiles * kTile;  // per workgroup
constexpr int kTable = 128;
constexpr int64_t kMostTokens = 1 << 24, kMostKeys = 1 << 30;
constexpr int64_t kMostLists = 0xffff;  // requests, and KV heads: an axis of the grid each
constexpr int64_t kMostHeads = 1 << 20;
constexpr float kLn2 = 0.6931471805599453f;

struct WeightsParams {
  oscarop_weights_args_v1 a;
  oscar_staging_v1 st;
  int has_stage;
  FastDiv group;  // Hq / Hk
  Score sc;
  int chunks;        // row chunks (1: sums go to the weights)
  int chunk_blocks;  // row blocks of a chunk; the last one takes what is left
  float* part;       // [num_reqs][chunks][Hk][weights_cols]
  // the chunks with rows of the key groups before one, and of all; plain_order: the groups do
  // not fit here, and workgroups lie in the order of the groups
  int first[kTable];
  int plain_order;
};

// The row chunks of the requests' key groups.  A key group's rows begin with the first that
// sees one of its keys.
struct Rows {
  int first, end;  // row blocks
};
__device__ __forceinline__ Rows rows_of(const WeightsParams& P, int chunk, int tb, int before, int nrows) {
  const int from = tb > before ? (int)(((int64_t)(tb - before) * P.group.d) / 32) : 0, blocks = (nrows + 31) / 32;
  const int a = chunk * P.chunk_blocks;
  Rows r;
  r.first = a > from ? a : from;
  r.end = chunk == P.chunks - 1 || blocks < a + P.chunk_blocks ? blocks : a + P.chunk_blocks;
  return r;
}

// Which request, KV head, key group and row chunk a workgroup takes.  Where there are several
// chunks the workgroups lie along one axis, and those that have rows in a batch of the call's
// largest sizes come first and side by side: workgroups go to the dies and their shader engines
// in turn, and one with more than its share would need a second round (6000 fresh tokens of 6
// heads on 1: 118 us in the order of the groups, 85 so).
struct Unit {
  int req, kvh, group, chunk, groups;
};
__device__ __forceinline__ Unit unit_of(const WeightsParams& P) {
  if (P.chunks == 1) return {(int)blockIdx.z, (int)blockIdx.y, (int)blockIdx.x, 0, (int)gridDim.x};
  const int hk = (int)P.a.cache.num_kv_heads, lists = P.a.num_reqs * hk, list = blockIdx.x % lists;
  const int i = blockIdx.x / lists, groups = gridDim.x / (lists * P.chunks);
  Unit u{list / hk, list % hk, i / P.chunks, i % P.chunks, groups};
  if (P.plain_order) return u;
  const int lane = threadIdx.x & 63, total = P.first[groups];
  // entries of a table that lie at or below x, less one; they ascend, past `groups` they do not count
  auto last = [&](int x, auto entry) __attribute__((always_inline)) {
    return __popcll(__ballot(lane < groups && entry(lane) <= x)) + __popcll(__ballot(64 + lane < groups && entry(64 + lane) <= x)) - 1;
  };
  if (i < total) {
    u.group = last(i, [&](int g) __attribute__((always_inline)) { return P.first[g]; });
    u.chunk = P.chunks - (P.first[u.group + 1] - i);
  } else {
    u.group = last(i - total, [&](int g) __attribute__((always_inline)) { return g * P.chunks - P.first[g]; });
    u.chunk = i - total - (u.group * P.chunks - P.first[u.group]);
  }
  return u;
}

// a request that does not fit the call's arrays
__device__ __forceinline__ bool misfit(const oscarop_weights_args_v1& A, int qa, int nq, int seq) {
  const int hist = A.k_new != nullptr ? seq - nq : seq;
  return qa < 0 || (int64_t)qa + nq > A.num_tokens || seq < 0 || hist < 0 || seq > A.weights_cols ||
         (hist > 0 && (hist - 1) / (int)A.cache.block_size >= A.block_table_cols);
}

// What a request's workgroups share.
struct Span {
  int qa, nq, seq, hist, before;  // first query, queries, length, cached tokens; query i sees keys [0, before + i + 1)
};
__device__ __forceinline__ Span span_of(const oscarop_weights_args_v1& A, int req) {
  Span x;
  x.qa = A.query_start_loc[req];
  x.nq = A.query_start_loc[req + 1] - x.qa;
  x.seq = A.seq_lens[req];
  x.before = x.seq - x.nq;
  x.hist = A.k_new != nullptr ? x.before : x.seq;
  return x;
}

// Row n of a request under KV head kvh: its token (0-based in the request) and query head.
struct RowRef {
  int tok, head;
  bool ok;
};
__device__ __forceinline__ RowRef row_of(const WeightsParams& P, int n, int nrows, int kvh) {
  RowRef r;
  r.ok = n < nrows;
  r.tok = (int)fdiv((uint32_t)(r.ok ? n : 0), P.group);
  r.head = kvh * (int)P.group.d + ((r.ok ? n : 0) - r.tok * (int)P.group.d);
  return r;
}

// One lane's token of a key tile: token t0 + lane % 32, half lane / 32 of its elements, as
// loaded.  What it is (KeyKind) shows only when the loads are in.
enum KeyKind { kNone = 0, kCodes = 1, kStaged = 2, kCurrent = 3 };  // past the length; history; its window copy; the chunk
template <int D>
struct KeyRegs {
  u32x4 word[D / 128];  // history: its half of the codes
  unsigned meta;        // history: scale and zero
  int tag;              // history: the low word of its seat's owner tag (tags are -1, -2 or block ids < 2^31)
  int blk, t;           // history: its block; the token
};

// the block of the history tile at t0 (0 off the history: a place that may be read)
__device__ __forceinline__ int block_of_tile(const oscarop_weights_args_v1& A, const Span& x, int req, int t0) {
  if (t0 >= x.hist) return 0;
  const int blk = A.block_table[req * A.block_table_stride + t0 / (int)A.cache.block_size];
  return blk < 0 || blk >= A.cache.num_blocks ? 0 : blk;  // a bad id must not fault
}

// first key of the i-th tile from t0, far past any length where it would overflow
__device__ __forceinline__ int tile_at(int t0, int i, int step) {
  const int64_t t = t0 + (int64_t)i * step;
  return t < 0x7fffffff ? (int)t : 0x7fffffff;
}

// (pages hold whole tiles: a tile that ends past the history is read within its page)
template <int D>
__device__ __forceinline__ void load_keys(const WeightsParams& P, const Span& x, int kvh, int t0, int blk, KeyRegs<D>& k) {
  const oscarop_weights_args_v1& A = P.a;
  const int lane = threadIdx.x & 63, g = lane >> 5, bs = (int)A.cache.block_size;
  k.t = t0 + (lane & 31);
  k.blk = blk;
  k.tag = -1;
  if (t0 < x.hist) {
    const int off = t0 % bs + (lane & 31);
    const uint8_t* slot = A.cache.k + blk * A.cache.k_stride[0] + off * A.cache.k_stride[1] + kvh * A.cache.k_stride[2];
    k.meta = *(const unsigned*)slot;
#pragma unroll
    for (int i = 0; i < D / 128; ++i) k.word[i] = *(const u32x4*)(slot + 32 + g * (D / 8) + 16 * i);
    if (P.has_stage) k.tag = ((const int*)P.st.owner)[2 * ((int64_t)((unsigned)blk % (unsigned)P.st.rows) * bs + off)];
  }
}

// The K operands of the lane's half, 16 elements (two operands) at a time: use(c, a, b).
template <int D, int QT, class Use>
__device__ __forceinline__ void key_operands(const WeightsParams& P, const Span& x, int kvh, const KeyRegs<D>& k, Use use) {
  constexpr int NCH = D / 32;
  const int kind = k.t < x.hist ? (k.tag == k.blk ? kStaged : kCodes) : P.a.k_new != nullptr && k.t < x.seq ? kCurrent : kNone;
  if (__all(kind == kCodes)) {
    unsigned t_lo, t_hi;
    byte_tables<QT>(k.meta, t_lo, t_hi);
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      unsigned o[8];
      lut16(k.word[c >> 2][c & 3], t_lo, t_hi, o);
      use(c, u32x4{o[0], o[1], o[2], o[3]}, u32x4{o[4], o[5], o[6], o[7]});
    }
    return;
  }
  const int g = (threadIdx.x & 63) >> 5, bs = (int)P.a.cache.block_size;
  const int64_t seat = (int64_t)((unsigned)k.blk % (unsigned)(P.has_stage ? P.st.rows : 1)) * bs + k.t % bs;
  const float* staged = P.st.stage_k + (seat * P.a.cache.num_kv_heads + kvh) * D + g * (D / 2);
  const uint16_t* row = (const uint16_t*)P.a.k_new + (int64_t)(x.qa + k.t - x.hist) * P.a.k_new_stride_token + kvh * D + g * (D / 2);
  unsigned t_lo = 0, t_hi = 0;
  if (kind == kCodes) byte_tables<QT>(k.meta, t_lo, t_hi);
  constexpr int kAhead = 4;  // chunks whose rows are in flight together: a tile is a chain of these
#pragma unroll
  for (int c0 = 0; c0 < NCH; c0 += kAhead) {
    f32x4 f[kAhead][4];
#pragma unroll
    for (int c = 0; c < kAhead; ++c) {
      if (kind == kStaged) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[c][i] = *(const f32x4*)(staged + 16 * (c0 + c) + 4 * i);
      } else if (kind == kCurrent) {
#pragma unroll
        for (int i = 0; i < 2; ++i) f[c][i] = *(const f32x4*)(row + 16 * (c0 + c) + 8 * i);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int c = 0; c < kAhead; ++c) {
      unsigned o[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
      if (kind == kCodes) {
        lut16(k.word[(c0 + c) >> 2][(c0 + c) & 3], t_lo, t_hi, o);
      } else if (kind == kStaged) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          o[i] = hist_pair<QT>(f[c][0][i], f[c][1][i]);
          o[4 + i] = hist_pair<QT>(f[c][2][i], f[c][3][i]);
        }
      } else if (kind == kCurrent) {
        kpairs16(__builtin_bit_cast(u32x4, f[c][0]), __builtin_bit_cast(u32x4, f[c][1]), o);
      }
      use(c0 + c, u32x4{o[0], o[1], o[2], o[3]}, u32x4{o[4], o[5], o[6], o[7]});
    }
  }
}

// What the rows of a block need to turn products into weights, in LDS by row:
// exp(s' - lse) = 2^(s2 - lse2) f, f being the rest of lse's conversion to log2 units (a
// rounding of up to 2^-20 there would show in every weight of the row).  Rows past the last
// and rows that saw no key have lse2 = inf and f = 0 (and zero queries).
struct RowConst {
  float lse2, f, slope2, tok;
};
struct BlockConst {
  __attribute__((aligned(16))) float lse2[32], f[32], slope2[32], tok[32];
};
template <int SC>
__device__ __forceinline__ RowConst row_const(const WeightsParams& P, const RowRef& r, float lse) {
  const bool sees = r.ok && lse != -INFINITY;
  RowConst c;
  c.lse2 = sees ? lse * kScoreLog2e : INFINITY;
  c.f = !sees ? 0.f : fabsf(lse) < INFINITY ? 1.f - kLn2 * fmaf(lse, kScoreLog2e, -c.lse2) : 1.f;
  c.slope2 = SC ? slope2_of(P.sc, r.head) : 0.f;
  c.tok = (float)r.tok;
  return c;
}
__device__ __forceinline__ void put_row(BlockConst& b, int row, const RowConst& c) {
  b.lse2[row] = c.lse2;
  b.f[row] = c.f;
  b.slope2[row] = c.slope2;
  b.tok[row] = c.tok;
}

// The sum over `rows` rows of the weights of this lane's key of a tile (both lanes of the key
// get it): register 4 q + i holds row 8 q + 4 g + i.  near: the key's distance to the
// request's first query; full: every row sees every key of the tile.
template <int SC>
__device__ __forceinline__ float sum_weights(const WeightsParams& P, const BlockConst& b, int rows, const f32x16& S, float near,
                                             bool full) {
  const int g = (threadIdx.x & 63) >> 5;
  float sum = 0.f;
  auto add = [&](auto all, auto fine) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (8 * q >= rows) break;
      const f32x4 lse2 = *(const f32x4*)&b.lse2[8 * q + 4 * g], f = *(const f32x4*)&b.f[8 * q + 4 * g];
      f32x4 slope2 = {}, tok = {};
      if constexpr (SC != 0) slope2 = *(const f32x4*)&b.slope2[8 * q + 4 * g];
      if constexpr (SC != 0 || !decltype(all)::value) tok = *(const f32x4*)&b.tok[8 * q + 4 * g];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float s = S[4 * q + i];
        float x;
        if constexpr (SC == 0) x = fmaf(s, P.sc.scale2, -lse2[i]);
        else x = fmaf(slope2[i], near - tok[i], (SC == 1 ? s * P.sc.scale2 : decltype(fine)::value ? capped2_small(P.sc, s) : capped2_fine(P.sc, s)) - lse2[i]);
        float p = __builtin_amdgcn_exp2f(x);
        if constexpr (!decltype(all)::value) p = near <= tok[i] ? p : 0.f;
        sum = fmaf(p, f[i], sum);
      }
    }
  };
  using std::false_type;
  using std::true_type;
  if constexpr (SC == 2) {
    // the whole tile's scores small against the cap, as they are for most: the series alone
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(S[e]));
    if (__all(top * fabsf(P.sc.over_cap) < kSmallTanh)) full ? add(true_type{}, true_type{}) : add(false_type{}, true_type{});
    else full ? add(true_type{}, false_type{}) : add(false_type{}, false_type{});
  } else {
    full ? add(true_type{}, false_type{}) : add(false_type{}, false_type{});
  }
  return sum + swap_halves(sum);
}

// the weights of a request that does not fit: nothing is read, they become NaN as far as
// there are any
__device__ __forceinline__ void poison(const oscarop_weights_args_v1& A, float* out, int seq, int part, int parts) {
  for (int64_t t = (int64_t)part * kThreads + threadIdx.x; t < A.weights_cols && t < seq; t += (int64_t)parts * kThreads) out[t] = NAN;
}

// This wave's part of a row block's queries, as MFMA operands: chunks wave, wave + kWaves, ...
template <int D>
struct QueryRegs {
  u32x4 v[D / 32 / kWaves][2];
  float lse;
  RowRef row;
};
template <int D>
__device__ __forceinline__ void load_queries(const WeightsParams& P, const Span& x, int kvh, int n0, QueryRegs<D>& q) {
  const oscarop_weights_args_v1& A = P.a;
  const int lane = threadIdx.x & 63, g = lane >> 5, wave = threadIdx.x >> 6;
  q.row = row_of(P, n0 + (lane & 31), x.nq * (int)P.group.d, kvh);
  const uint16_t* p = (const uint16_t*)A.q + (int64_t)(x.qa + q.row.tok) * A.q_stride_token + (int64_t)q.row.head * D + g * (D / 2);
#pragma unroll
  for (int i = 0; i < D / 32 / kWaves; ++i) {
    q.v[i][0] = *(const u32x4*)(p + 16 * (wave + kWaves * i));
    q.v[i][1] = *(const u32x4*)(p + 16 * (wave + kWaves * i) + 8);
  }
  q.lse = A.lse[(int64_t)(x.qa + q.row.tok) * A.num_q_heads + q.row.head];
}
template <int D, int SC>
__device__ __forceinline__ void put_queries(const WeightsParams& P, const QueryRegs<D>& q, u32x4 (*s_q)[64], BlockConst& s_row) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const bool sees = q.row.ok && q.lse != -INFINITY;
#pragma unroll
  for (int i = 0; i < D / 32 / kWaves; ++i) {
    const int c = wave + kWaves * i;
    unsigned o[8];
    kpairs16(q.v[i][0], q.v[i][1], o);
    const u32x4 a = {o[0], o[1], o[2], o[3]}, b = {o[4], o[5], o[6], o[7]}, zero = {0u, 0u, 0u, 0u};
    s_q[2 * c][lane] = sees ? a : zero;
    s_q[2 * c + 1][lane] = sees ? b : zero;
  }
  if (threadIdx.x < 32) put_row(s_row, threadIdx.x, row_const<SC>(P, q.row, q.lse));
}

template <int D, int QT, int SC>
__global__ __launch_bounds__(kThreads, 3) void weights_few_kernel(WeightsParams P) {
  constexpr int NCH = D / 32;  // 16-element chunks per lane half
  const oscarop_weights_args_v1& A = P.a;
  const int lane = threadIdx.x & 63, m = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int req = blockIdx.z, kvh = blockIdx.y;
  const Span x = span_of(A, req);
  if (x.nq < 1) return;
  float* out = A.weights + req * A.weights_stride_request + kvh * A.weights_stride_head;
  if (misfit(A, x.qa, x.nq, x.seq)) return poison(A, out, x.seq, blockIdx.x, gridDim.x);
  // neighbouring tiles go to different workgroups: the window's are slow ones (their rows come
  // one line a lane), and those of one compute unit would wait for each other
  const int step = gridDim.x * kWaves * kTile, t_first = (wave * gridDim.x + blockIdx.x) * kTile;
  if ((int)(blockIdx.x * kTile) >= x.seq) return;
  __shared__ __attribute__((aligned(16))) u32x4 s_q[2 * NCH][64];  // query operands of a row block
  __shared__ BlockConst s_row;
  const int nrows = x.nq * (int)P.group.d;
  for (int n0 = 0; n0 < nrows; n0 += 32) {  // once, unless the batch outgrew the call's max_query_len
    // lane i: the block of the wave's tile i (and, every 64 tiles, of the next 64)
    int blocks = block_of_tile(A, x, req, tile_at(t_first, lane, step));
    KeyRegs<D> next;
    float old_next = 0.f;
    load_keys<D>(P, x, kvh, t_first, __builtin_amdgcn_readlane(blocks, 0), next);
    if (t_first + m < x.seq) old_next = out[t_first + m];
    QueryRegs<D> q;
    load_queries<D>(P, x, kvh, n0, q);
    if (n0) __syncthreads();
    put_queries<D, SC>(P, q, s_q, s_row);
    __syncthreads();
    int tile = 0;
    for (int t0 = t_first; t0 < x.seq; t0 += step) {
      const KeyRegs<D> k = next;
      const float old = old_next;
      if (t0 + step < x.seq) {
        if (++tile == 64) {
          tile = 0;
          blocks = block_of_tile(A, x, req, tile_at(t0 + step, lane, step));
        }
        load_keys<D>(P, x, kvh, t0 + step, __builtin_amdgcn_readlane(blocks, tile), next);
        if (t0 + step + m < x.seq) old_next = out[t0 + step + m];
      }
      // the contraction in three parts: the partial sums stay smaller and fewer roundings
      // follow on each other (one token's weights over 500 keys, relative to 64 bits, mean of
      // twelve: 5.5e-7 so, 7.0e-7 in halves and 3% less time, 6.4e-7 in plain fp32)
      f32x16 S = {}, T = {};
      key_operands<D, QT>(P, x, kvh, k, [&](int c, u32x4 a, u32x4 b) {
        constexpr int kPart = (NCH + 2) / 3;
        T = mma16<QT>(s_q[2 * c][lane], a, c % kPart == 0 ? f32x16{} : T);
        T = mma16<QT>(s_q[2 * c + 1][lane], b, T);
        if (c % kPart == kPart - 1 || c == NCH - 1) S = c < kPart ? T : S + T;
      });
      const float sum = sum_weights<SC>(P, s_row, nrows - n0, S, (float)(t0 + m - x.before), t0 + kTile - 1 <= x.before);
      if (lane < 32 && t0 + m < x.seq) out[t0 + m] = old + sum;
    }
  }
}

template <int D, int QT, int SC>
__global__ __launch_bounds__(kThreads, 2) void weights_many_kernel(WeightsParams P) {
  constexpr int NCH = D / 32;
  const oscarop_weights_args_v1& A = P.a;
  const int lane = threadIdx.x & 63, m = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const auto [req, kvh, group0, chunk, groups] = unit_of(P);
  const Span x = span_of(A, req);
  if (x.nq < 1) return;
  float* out = P.chunks > 1 ? P.part + (((int64_t)req * P.chunks + chunk) * A.cache.num_kv_heads + kvh) * A.weights_cols
                            : A.weights + req * A.weights_stride_request + kvh * A.weights_stride_head;
  if (misfit(A, x.qa, x.nq, x.seq)) {
    if (P.chunks == 1) poison(A, out, x.seq, group0, groups);
    return;
  }
  __shared__ __attribute__((aligned(16))) u32x4 s_q[2][2 * NCH][64];  // query operands of a row block
  __shared__ BlockConst s_row[2];
  const int nrows = x.nq * (int)P.group.d;
  for (int tb = group0 * kGroupKeys; tb < x.seq; tb += groups * kGroupKeys) {
    const Rows rows = rows_of(P, chunk, tb, x.before, nrows);
    if (rows.first >= rows.end) continue;
    QueryRegs<D> q;
    load_queries<D>(P, x, kvh, 32 * rows.first, q);
    const int wave_t0 = tb + wave * kKeyTiles * kTile;
    u32x4 kop[kKeyTiles][2 * NCH];
#pragma unroll
    for (int i = 0; i < kKeyTiles; ++i) {
      KeyRegs<D> k;
      load_keys<D>(P, x, kvh, wave_t0 + i * kTile, block_of_tile(A, x, req, wave_t0 + i * kTile), k);
      key_operands<D, QT>(P, x, kvh, k, [&](int c, u32x4 a, u32x4 b) {
        kop[i][2 * c] = a;
        kop[i][2 * c + 1] = b;
      });
    }
    // (64 bits: a prompt of 131072 tokens adds 24576 blocks' sums here, of which as many fp32
    // additions lose 2e-4)
    double acc[kKeyTiles] = {};
    for (int rb = rows.first; rb < rows.end; ++rb) {
      const int buf = (rb - rows.first) & 1;
      put_queries<D, SC>(P, q, s_q[buf], s_row[buf]);
      if (rb + 1 < rows.end) load_queries<D>(P, x, kvh, 32 * (rb + 1), q);
      // one barrier a block: the buffer written next was read before the last barrier
      __syncthreads();
      f32x16 S[kKeyTiles] = {};
#pragma unroll
      for (int j = 0; j < 2 * NCH; ++j) {
        const u32x4 qop = s_q[buf][j][lane];
#pragma unroll
        for (int i = 0; i < kKeyTiles; ++i) S[i] = mma16<QT>(qop, kop[i][j], S[i]);
      }
      const int first_tok = (int)fdiv((uint32_t)(32 * rb), P.group);
#pragma unroll
      for (int i = 0; i < kKeyTiles; ++i) {
        const int t0 = wave_t0 + i * kTile;
        acc[i] += sum_weights<SC>(P, s_row[buf], nrows - 32 * rb, S[i], (float)(t0 + m - x.before), t0 + kTile - 1 <= x.before + first_tok);
      }
    }
#pragma unroll
    for (int i = 0; i < kKeyTiles; ++i) {
      const int t = wave_t0 + i * kTile + m;
      if (lane < 32 && t < x.seq) out[t] = (float)(P.chunks > 1 ? acc[i] : out[t] + acc[i]);
    }
    __syncthreads();  // the next key group's first block goes over a buffer still being read
  }
}

// weights += the chunks' sums, in a fixed order: 32 keys per workgroup, the chunks dealt to
// eight lanes of each
__global__ __launch_bounds__(256) void weights_sum_kernel(WeightsParams P) {
  const oscarop_weights_args_v1& A = P.a;
  const int req = blockIdx.z, kvh = blockIdx.y, lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const Span x = span_of(A, req);
  if (x.nq < 1) return;
  float* out = A.weights + req * A.weights_stride_request + kvh * A.weights_stride_head;
  if (misfit(A, x.qa, x.nq, x.seq)) return poison(A, out, x.seq, blockIdx.x, gridDim.x);
  __shared__ float s_sum[8][32];
  const int64_t pitch = A.cache.num_kv_heads * A.weights_cols;
  const float* p = P.part + ((int64_t)req * P.chunks * A.cache.num_kv_heads + kvh) * A.weights_cols;
  const int nrows = x.nq * (int)P.group.d, chunks = ((nrows + 31) / 32 + P.chunk_blocks - 1) / P.chunk_blocks;
  const int end = chunks < P.chunks ? chunks : P.chunks;
  for (int t0 = blockIdx.x * 32; t0 < x.seq; t0 += gridDim.x * 32) {
    const int t = t0 + lane;
    // the chunks with rows (rows_of), eight loads of a lane in flight
    const int tb = t0 / kGroupKeys * kGroupKeys, first = rows_of(P, 0, tb, x.before, nrows).first / P.chunk_blocks;
    const int begin = first < P.chunks ? first : P.chunks - 1;
    float sum = 0.f;
    if (t < x.seq)
      for (int c0 = begin + part; c0 < end; c0 += 64) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c0 + 8 * i < end ? p[(c0 + 8 * i) * pitch + t] : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += v[i];
      }
    __syncthreads();
    s_sum[part][lane] = sum;
    __syncthreads();
    if (part == 0 && t < x.seq) {
#pragma unroll
      for (int i = 1; i < 8; ++i) sum += s_sum[i][lane];
      out[t] += sum;
    }
  }
}

// Workgroups of weights_few_kernel that the chip holds, and key tiles of a wave at most.
constexpr int64_t kFewWorkgroups = 768;
constexpr int64_t kFewTiles = 16;

// Row chunks of a call: as many as leave the workgroups with any rows within one round of the
// chip, two per compute unit (the rows that see a key group's first key begin later in every
// group of a fresh prompt, and the chunks before them are empty).  A workgroup's key operands
// cost about as much to load as four row blocks, so the second workgroup of a compute unit pays
// from there on; the first always does.  Chunks of at least 4 / 2 / 1 blocks, us: 100 fresh
// tokens of 6 heads 16.0 / 12.6 / 10.9, 1000 (470 workgroups at one block) 18.0 / 15.2 / 18.0.
constexpr int64_t kUnits = 512;
constexpr int64_t kMinBlocks = 4;
constexpr int64_t kMaxPart = 256ll << 20;  // bytes of partial sums
struct Chunks {
  int64_t count, blocks;
};
// chunks of `per` blocks before key group g's first one with rows
int64_t empty_chunks(const oscarop_weights_args_v1& a, int64_t g, int64_t per, int64_t count) {
  const int64_t tokens = g * kGroupKeys - (a.max_seq_len - a.max_query_len);
  const int64_t none = tokens <= 0 ? 0 : tokens * (a.num_q_heads / a.cache.num_kv_heads) / 32 / per;
  return none < count ? none : count;
}
Chunks chunks_of(const oscarop_weights_args_v1& a) {
  const Chunks one = {1, 1 << 30};
  const int64_t hk = a.cache.num_kv_heads, rows = a.max_query_len * (a.num_q_heads / hk), blocks = (rows + 31) / 32;
  const int64_t groups = (a.max_seq_len + kGroupKeys - 1) / kGroupKeys, lists = a.num_reqs * hk;
  if (groups * lists < 1 || rows <= kFewRows || blocks < 2 || groups * lists >= kUnits) return one;
  const int64_t before = a.max_seq_len - a.max_query_len;
  const int64_t all = before < 0 ? 0 : before / kGroupKeys + 1;  // key groups that every row block sees
  auto fits = [&](int64_t per, int64_t units) {
    const int64_t count = (blocks + per - 1) / per;
    int64_t sum = all * count;
    for (int64_t g = all; g < groups; ++g) sum += count - empty_chunks(a, g, per, count);
    return sum * lists <= units;
  };
  const int64_t most = kMaxPart / (lists * a.weights_cols * (int64_t)sizeof(float));
  if (most < 2) return one;
  auto fewest = [&](int64_t low, int64_t units) {  // blocks a chunk that fit
    int64_t high = blocks;
    while (low < high) {
      const int64_t per = (low + high) / 2;
      if (fits(per, units)) high = per;
      else low = per + 1;
    }
    return low;
  };
  const int64_t least = (blocks + most - 1) / most;
  int64_t per = fewest(least, kUnits / 2);
  if (per > kMinBlocks) per = fewest(least < kMinBlocks ? kMinBlocks : least, kUnits);
  return per < blocks ? Chunks{(blocks + per - 1) / per, per} : one;
}

}  // namespace

}  // namespace oscar

using namespace oscar;

extern "C" int64_t oscarop_attn_weights_workspace_bytes_v1(const oscarop_weights_args_v1* args) {
  if (!args || args->num_reqs < 0 || args->max_seq_len < 0 || args->max_query_len < 0 || args->cache.num_kv_heads < 1 ||
      args->num_q_heads < 1 || args->num_q_heads % args->cache.num_kv_heads || args->weights_cols < 1 ||
      args->num_reqs > kMostLists || args->cache.num_kv_heads > kMostLists || args->num_q_heads > kMostHeads ||
      args->max_query_len > kMostTokens || args->max_seq_len > kMostKeys || args->weights_cols > kMostKeys)
    return -22;
  const Chunks c = chunks_of(*args);
  return c.count > 1 ? args->num_reqs * c.count * args->cache.num_kv_heads * args->weights_cols * (int64_t)sizeof(float) : 0;
}

extern "C" int oscarop_attn_weights_v1(const oscarop_weights_args_v1* args, const oscarop_score_v1* score, void* stream) {
  const char* name = "oscarop_attn_weights_v1";
  if (!args) return fail(-22, "%s: null args", name);
  const oscarop_weights_args_v1& a = *args;
  WeightsParams p{};
  const int sc = score_of(score, a.scale, &p.sc);
  if (sc < 0) return fail(-22, kBadCap, name);
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
  // (distances are counted in fp32, lengths and rows in int)
  if (a.num_reqs > kMostLists || a.cache.num_kv_heads > kMostLists || a.num_q_heads > kMostHeads ||
      a.num_tokens >= (1ll << 31) || a.num_tokens * a.num_q_heads >= (1ll << 31))
    return fail(-22, "%s: too many requests or rows for one call", name);
  if (a.num_tokens > kMostTokens || a.max_query_len > kMostTokens || a.max_seq_len > kMostKeys || a.weights_cols > kMostKeys)
    return fail(-22, "%s: too many tokens for one call", name);
  if (a.block_table_rows < a.num_reqs || a.block_table_cols < 1 || a.block_table_stride < a.block_table_cols)
    return fail(-22, "%s: Missing request block-table rows", name);
  if (a.cache.block_size < kTile || a.cache.block_size % kTile || a.cache.block_size > (1 << 20))
    return fail(-22, "%s: block_size %lld must be a multiple of %d (<= 2^20)", name, (long long)a.cache.block_size, kTile);
  const Rows2 lists{{a.num_reqs, a.cache.num_kv_heads}, {a.weights_stride_request, a.weights_stride_head}, a.weights_cols};
  if (a.weights_cols < 1 || a.weights_stride_head < a.weights_cols || lists.overlap())
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
  p.group = FastDiv::of(a.num_q_heads / a.cache.num_kv_heads);
  const Chunks chunks = chunks_of(a);
  const int64_t need = oscarop_attn_weights_workspace_bytes_v1(&a);
  if (need > 0 && (!a.workspace || a.workspace_bytes < need || (((uintptr_t)a.workspace) & 15)))
    return fail(-22, "%s: 16-byte aligned workspace of %lld bytes required", name, (long long)need);
  p.chunks = (int)chunks.count;
  p.chunk_blocks = (int)chunks.blocks;
  p.part = (float*)a.workspace;
  const int64_t key_groups = (a.max_seq_len + kGroupKeys - 1) / kGroupKeys;
  p.plain_order = key_groups >= kTable;
  if (p.chunks > 1 && !p.plain_order)
    for (int64_t g = 0; g < key_groups; ++g)
      p.first[g + 1] = p.first[g] + p.chunks - (int)empty_chunks(a, g, p.chunk_blocks, p.chunks);
  hipStream_t s = (hipStream_t)stream;
  const unsigned hk = (unsigned)a.cache.num_kv_heads, reqs = (unsigned)a.num_reqs;
  const bool few = a.max_query_len * (int64_t)p.group.d <= kFewRows;
  // few: a workgroup per key tile as long as the chip holds them all, then more tiles each
  const int64_t tiles = (a.max_seq_len + kTile - 1) / kTile;
  int64_t few_wgs = kFewWorkgroups / ((int64_t)hk * reqs);
  const int64_t least = (tiles + kWaves * kFewTiles - 1) / (kWaves * kFewTiles);
  few_wgs = few_wgs < least ? least : few_wgs > tiles ? tiles : few_wgs;
  const unsigned units = (unsigned)(few ? few_wgs : key_groups * chunks.count);
  const dim3 grid = chunks.count > 1 ? dim3(units * hk * reqs) : dim3(units, hk, reqs);
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, s, p); };
  auto by_score = [&](auto d, auto qt) {
    constexpr int DD = decltype(d)::value, QT = decltype(qt)::value;
    if (few) sc == 0 ? launch(weights_few_kernel<DD, QT, 0>) : sc == 1 ? launch(weights_few_kernel<DD, QT, 1>) : launch(weights_few_kernel<DD, QT, 2>);
    else sc == 0 ? launch(weights_many_kernel<DD, QT, 0>) : sc == 1 ? launch(weights_many_kernel<DD, QT, 1>) : launch(weights_many_kernel<DD, QT, 2>);
  };
  using std::integral_constant;
  if (D == 256) {
    if (a.q_dtype == OSCAR_F16) by_score(integral_constant<int, 256>{}, integral_constant<int, OSCAR_F16>{});
    else by_score(integral_constant<int, 256>{}, integral_constant<int, OSCAR_BF16>{});
  } else {
    if (a.q_dtype == OSCAR_F16) by_score(integral_constant<int, 128>{}, integral_constant<int, OSCAR_F16>{});
    else by_score(integral_constant<int, 128>{}, integral_constant<int, OSCAR_BF16>{});
  }
  OSCAR_CHECK_LAUNCH(few ? "weights_few_kernel" : "weights_many_kernel");
  if (p.chunks > 1) {
    const dim3 sums((unsigned)tiles, hk, reqs);
    hipLaunchKernelGGL(weights_sum_kernel, sums, dim3(256), 0, s, p);
    OSCAR_CHECK_LAUNCH("weights_sum_kernel");
  }
  return 0;
}
