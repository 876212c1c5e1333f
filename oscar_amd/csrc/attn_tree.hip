// Attention of drafted trees over the packed INT2 history (gfx950).
//
// A request of n nodes has M = n G rows per KV head (G query heads each), which all see its
// history; among each other nodes see by a mask.  The split-K decode (attn_decode.hip) takes 32 rows
// a wave and unpacks the codes for each 32 anew, which its vector unit pays for: two thirds of a
// tile's time.  Here a workgroup of eight waves holds up to 256 rows, 32 a wave, and unpacks a tile of
// keys once for all of them, into LDS.
//
// Work: the plan (oscarop_tree_plan_v1) cuts M into blocks of at most 256 rows and deals each
// block's tiles of KT = 8192 / D keys round-robin to items, one workgroup each: full tiles of the
// history to some, its ragged end and the chunk's tiles to others (SLOW), whose masks and second
// parts of P do not fit in registers beside the full tiles' loop.  Wave w holds rows [32 w, 32 w + 32)
// of the block: their queries (B operands) and O^T in registers.  For a tile t, with 32x32x16 MFMA,
//   S^T(t) = K(t) Q^T,   P(t) = exp2(scale S - m),   O^T += V(t)^T P(t)^T;
// S^T's layout (lane: a row, keys in fours) is already that of the B operand of P.  The items' O / l
// and log-sum-exps are merged by tree_merge_kernel.
//
// The loop: K and V have two buffers each in LDS, so one barrier a tile does; the codes of tile
// t + 2 are on their way while t is computed.  With more than 192 rows waves 0 to 3 unpack keys before
// their products and waves 4 to 7 values after theirs: the two waves of a SIMD are out of step, and
// give its matrix unit and its vector unit something to do at the same time.  With fewer, waves without
// rows unpack for those with them (192 rows 79 -> 72 us with the merge).  Each kind of wave has a
// loop of its own: with one for all, the queries did not stay in registers.
//
// LDS: K in operand order, 16 bytes a lane.  V one row per key, 32 elements of padding, its
// 16-byte units exchanged by the key's bits 2 and 3: rows then spread over all banks, for the
// stores of a key per lane as for the transposing reads of a column per lane.
//
// Values: K is the reference's bf16 or fp16 of fp16(code * scale + zero), V fp16(...)
// unrounded, the window's FP32 copies likewise; P fp16, up to 2^15, the reference m 2^7 below the
// largest score at its last move, so that keys of 2^-21 of the largest still keep 11 bits.  The chunk's
// V in bf16 have a wider range than fp16: chunk tiles multiply it by P in two bf16 parts, P at most 2^-16
// so that no sum of finite values overflows.  A
// value of the chunk that is not finite goes into LDS as zero and is added afterwards, to the
// rows alone that see its node.
//
// What bounds it: 8 requests of 24576 tokens with 32 nodes (192 rows, D 256) take 61 to 63 us, 0.62
// PFLOP/s in 39 GFLOP: 25 tiles a workgroup at 2.0 us and 12 us before and after them, of which
// 50 MB of partials; their merge takes another 10 us.  A tile's products alone take 1.0 us at the 2.0 to
// 2.1 GHz that the matrix units leave the clock, its softmax and unpacking (about 255 vector
// instructions a wave) as long again, and the two overlap in part (252 rows: the matrix unit busy for 36%
// of the cycles, the waves waiting for a third).  12 ragged requests of up to 64 nodes, D 128 with capped
// scores: 65 to 69 us, bound by the cap's exponentials and divides.  One request of 500 tokens and 16
// nodes: 15 us, latency.  Measured against it, at 8 x 24576 tokens: four waves of 16 or 64 rows with
// 16x16x32 products, 99 to 165 us; the softmax of tile t - 1 between the products of tile t in one
// wave, 86 to 114; slow tiles in the same loop, 113 (registers spill); two tiles a barrier, 14 us more; the
// products of values a tile late in the second wave of a SIMD, 4 us less with 252 rows, 2 more in
// ragged calls; LDS operands read once instead of anew for each product, 1 us (they are not the
// bound); two accumulators of S or a higher wave priority, no gain beyond the noise.
#include <type_traits>
#include <vector>

#include "common.h"
#include "int2_tile.h"
#include "score.h"

namespace oscar {

namespace {

constexpr int kWaves = 8;        // two a SIMD
constexpr int kThreads = 64 * kWaves;
constexpr int kMostRows = 32 * kWaves;  // of a workgroup
constexpr int kMostTiles = 512;  // of an item
constexpr int kAhead = 3, kAheadV = 3;  // operands of products read ahead
constexpr int kSlowCost = 3;      // a slow tile's time in full ones
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kBelow = 7.f;    // the reference below the maximum where it moves to,
constexpr float kMost = 15.f;    // and how far above it a score may come (log2 units)
// The same for tiles of a bf16 chunk, whose values reach 2^128: probabilities of at most 2^-16 keep the sums
// of an item's 2^15 keys below it (as two bf16 parts they lose nothing), and the merge's weights of at most
// 2^-12 the sums of its items.
constexpr float kChunk = -16.f;
constexpr float kWeight = 1.f / 4096.f;
typedef short __attribute__((ext_vector_type(4))) i16x4;

template <int D>
struct Cfg {
  static constexpr int KT = 8192 / D;        // keys of a tile: two dwords of codes a thread
  static constexpr int KSTEPS = D / 16;      // QK contraction steps
  static constexpr int KSUB = KT / 32;       // 32-key parts of a tile
  static constexpr int VSTEPS = KT / 16;     // PV contraction steps
  static constexpr int NB = D / 32;          // 32-wide parts of O^T
  static constexpr int VROW = D + 32;        // elements of a row of V in LDS
  static constexpr int KBYTES = KT * D * 2;
  static constexpr int VBYTES = KT * VROW * 2;
};

struct TreeParams {
  oscarop_tree_attn_args_v1 a;
  oscar_staging_v1 st;
  int has_stage;
  int group;
  float* part_o;    // [partial rows][D], columns in LDS order
  float* part_lse;  // [partial rows], log2 units
  Score sc;
};

// elements (e0, e4) (e1, e5) (e2, e6) (e3, e7) of eight: the order in which codes are looked up
__device__ __forceinline__ u32x4 kpairs8(const u32x4& x) {
  return u32x4{__builtin_amdgcn_perm(x[2], x[0], 0x05040100u), __builtin_amdgcn_perm(x[2], x[0], 0x07060302u),
               __builtin_amdgcn_perm(x[3], x[1], 0x05040100u), __builtin_amdgcn_perm(x[3], x[1], 0x07060302u)};
}

// element of a row in LDS order (kpairs8)
__device__ __forceinline__ int column(int i) { return (i & ~7) + ((i & 7) >> 1) + 4 * (i & 1); }

struct Item {
  int req, kvh, qa, n, hist, row0, rows, first, stride, count, part;
};

// where 32 tokens lie: their page, the offset of the first in it, and its seat in the window
struct Place {
  int page, off, seat, pad;
};

// The tiles of one item: full ones of the history, or (SLOW) its ragged end and the chunk's.  Apart, since
// what the latter need does not fit beside O and the queries in the others' loop.
template <int D, int QT, int SC, bool SLOW>
__device__ __forceinline__ void run_item(const TreeParams& P, const Item& I, uint8_t* s_k, uint8_t* s_v, const Place* s_place,
                                         uint32_t* s_odd) {
  using C = Cfg<D>;
  const oscarop_tree_attn_args_v1& T = P.a;
  const oscar_attn_args_v1& A = T.attn;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = P.group;
  const int htiles = (int)(((int64_t)I.hist + C::KT - 1) / C::KT);

  // ---- this lane's row and its queries: half g of a step holds 8 of its 16 elements
  const int m = lane & 31, g = lane >> 5;
  const int row = 32 * wave + m;
  const bool active = 32 * wave < I.rows;  // the wave has rows
  int node = -1;
  u32x4 q[C::KSTEPS];
  {
    const bool ok = row < I.rows;
    const int mm = I.row0 + (ok ? row : 0);
    if (ok) node = mm / G;
    const uint16_t* src = (const uint16_t*)A.q + (int64_t)(I.qa + mm / G) * A.q_stride_token + (int64_t)(I.kvh * G + mm % G) * D;
#pragma unroll
    for (int ks = 0; ks < C::KSTEPS; ++ks) {
      q[ks] = kpairs8(*(const u32x4*)(src + 16 * ks + 8 * g));
      if (!ok) q[ks] = u32x4{0u, 0u, 0u, 0u};
    }
  }

  // ---- filling, in eight units of 256 / 4 threads: 0 to 3 the keys, 4 to 7 the values; thread
  // (token, 32 codes)
  const uint8_t* kbase = A.cache.k + (int64_t)I.kvh * A.cache.k_stride[2];
  const uint8_t* vbase = A.cache.v + (int64_t)I.kvh * A.cache.v_stride[2];
  struct Unit {
    bool v;                            // values
    int tok, vec, sub, in32, to, turn;
    u32x2 codes;
    unsigned meta;
    int tag, page, seat;
  };
  auto unit_of = [&](int which) {
    Unit u;
    const int idx = 64 * (which & 3) + lane;
    u.v = which >= 4;
    u.tok = idx % C::KT, u.vec = idx / C::KT, u.sub = u.tok >> 5, u.in32 = u.tok & 31;
    // where piece i (8 elements) of the thread's four goes
    // (a row of values has its 16-byte units exchanged, within four, by the key's bits 2 and 3)
    u.to = u.v ? u.tok * (C::VROW * 2) + 64 * u.vec : (2 * u.vec * C::KSUB + u.sub) * 1024 + u.in32 * 16;
    u.turn = (u.tok >> 2) & 3;
    u.codes = u32x2{0u, 0u};
    u.meta = 0;
    u.tag = -1, u.page = 0, u.seat = 0;
    return u;
  };
  const int64_t ks0 = A.cache.k_stride[0], ks1 = A.cache.k_stride[1];
  const int64_t vs0 = A.cache.v_stride[0], vs1 = A.cache.v_stride[1];
  auto load_at = [&](Unit& u, const Place& x, int off) {
    u.page = x.page;
    u.seat = x.seat + off - x.off;
    const uint8_t* slot = u.v ? vbase + (int64_t)u.page * vs0 + (int64_t)off * vs1 : kbase + 32 + (int64_t)u.page * ks0 + (int64_t)off * ks1;
    u.codes = *(const u32x2*)(slot + 8 * u.vec);
    u.meta = *(const unsigned*)(kbase + (int64_t)u.page * ks0 + (int64_t)off * ks1 + (u.v ? 4 : 0));
    u.tag = P.has_stage ? ((const int32_t*)P.st.owner)[2 * (int64_t)u.seat] : -1;
  };
  auto load = [&](Unit& u, int j) {
    const Place x = s_place[(j < I.count ? j : I.count - 1) * C::KSUB + u.sub];
    load_at(u, x, x.off + u.in32);
  };
  auto dest = [&](const Unit& u, int i, int buf) -> u32x4* {
    if (u.v) return (u32x4*)(s_v + buf * C::VBYTES + u.to + 16 * (i ^ u.turn));
    return (u32x4*)(s_k + buf * C::KBYTES + u.to + (i >> 1) * (C::KSUB * 1024) + (i & 1) * 512);
  };
  auto fill_codes = [&](const Unit& u, bool some, int buf) {
    unsigned t_lo, t_hi;
    if (QT == OSCAR_F16 || u.v) byte_tables<OSCAR_F16>(u.meta, t_lo, t_hi);
    else byte_tables<OSCAR_BF16>(u.meta, t_lo, t_hi);
    if (!some) t_lo = t_hi = 0;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      unsigned o[8];
      lut16(u.codes[c], t_lo, t_hi, o);
      *dest(u, 2 * c, buf) = u32x4{o[0], o[1], o[2], o[3]};
      *dest(u, 2 * c + 1, buf) = u32x4{o[4], o[5], o[6], o[7]};
    }
  };
  // the window's copy of a token
  auto fill_staged = [&](const Unit& u, int buf) {
    const f32x4* src = (const f32x4*)((u.v ? P.st.stage_v : P.st.stage_k) + ((int64_t)u.seat * A.cache.num_kv_heads + I.kvh) * D + 32 * u.vec);
#pragma unroll 2
    for (int i = 0; i < 4; ++i) {
      const f32x4 a = src[2 * i], b = src[2 * i + 1];
      u32x4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = u.v ? hist_pair<OSCAR_F16>(a[e], b[e]) : hist_pair<QT>(a[e], b[e]);
      *dest(u, i, buf) = o;
    }
  };
  // tile j, loaded before, into its buffer
  auto fill = [&](const Unit& u, int j) {
    fill_codes(u, true, j & 1);
    if (__builtin_expect(u.tag == u.page, 0)) fill_staged(u, j & 1);
  };
  constexpr unsigned kInf = QT == OSCAR_BF16 ? 0x7f80u : 0x7c00u;  // the exponent of infinities and NaN
  // tile t at once: the history's ragged end (unseen keys zero), or one of the chunk's
  auto fill_slow = [&](Unit& own, int t, int j) {
    const bool chunk = t >= htiles;
    const int key = (chunk ? t - htiles : t) * C::KT + own.tok;
    if (!chunk) {
      const bool in = key < I.hist;
      const Place x = s_place[j * C::KSUB + (in ? own.sub : 0)];
      load_at(own, x, in ? x.off + own.in32 : x.off);
      fill_codes(own, in, 0);
      if (in && own.tag == own.page) fill_staged(own, 0);
      return;
    }
    const u32x4* src = (const u32x4*)((const uint16_t*)(own.v ? A.v_new : A.k_new) + (int64_t)(I.qa + (key < I.n ? key : 0)) * A.kv_new_stride_token +
                                      (int64_t)I.kvh * D + 32 * own.vec);
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u32x4 x = key < I.n ? kpairs8(src[i]) : u32x4{0u, 0u, 0u, 0u};
      if (own.v) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned low = x[e] & kInf, high = (x[e] >> 16) & kInf;
          odd |= low == kInf || high == kInf;
          x[e] &= (low == kInf ? 0u : 0xffffu) | (high == kInf ? 0u : 0xffff0000u);
        }
      }
      *dest(own, i, 0) = x;
    }
    if (odd) atomicOr(&s_odd[own.sub], 1u << own.in32);
  };

  // ---- running state of this lane's row
  float m_run = -INFINITY, l_run = 0.f;
  f32x16 O[C::NB];
#pragma unroll
  for (int b = 0; b < C::NB; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) O[b][r] = 0.f;
  const float c_score = A.scale * kLog2e;
  constexpr bool kScaled = SC == 2;  // the scores carry the scale already
  f32x16 S[C::KSUB];
  u32x4 ph[C::VSTEPS];

  auto qk = [&](int buf) {
    const u32x4* src = (const u32x4*)(s_k + buf * C::KBYTES) + lane;
#pragma unroll
    for (int a = 0; a < C::KSUB; ++a)
#pragma unroll
      for (int r = 0; r < 16; ++r) S[a][r] = 0.f;
#pragma unroll
    for (int ks = 0; ks < C::KSTEPS; ++ks)
#pragma unroll
      for (int a = 0; a < C::KSUB; ++a) S[a] = mma16<QT>(src[(ks * C::KSUB + a) * 64], q[ks], S[a]);
    // operands three products ahead: all of them at once do not fit beside O and the queries
    __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
    for (int i = 0; i < C::KSTEPS * C::KSUB; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    if constexpr (SC == 2) {
#pragma unroll
      for (int a = 0; a < C::KSUB; ++a)
#pragma unroll
        for (int r = 0; r < 16; ++r) S[a][r] = capped2(P.sc, S[a][r]);
    }
  };
  // unseen keys of a slow tile
  uint64_t sees = 0;  // the tile's keys that this lane's row sees
  auto mask = [&](int t) {
    const int j0 = (t - htiles) * C::KT;  // a multiple of 32
    const int left = I.hist - t * C::KT;  // keys of a history tile
    uint64_t see = left >= 64 ? ~0ull : (1ull << (left > 0 ? left : 0)) - 1;
    if (t >= htiles) {
      see = 0;
      if (node >= j0 && (j0 >> 6) < T.mask_words) {
        see = (uint64_t)T.mask[(int64_t)(I.qa + node) * T.mask_words + (j0 >> 6)] >> (j0 & 63);
        const int last = node - j0;  // no node after its own
        if (last < 63) see &= (2ull << last) - 1;
      }
    }
    sees = see;
#pragma unroll
    for (int a = 0; a < C::KSUB; ++a)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (!((see >> (32 * a + out_tok(r, g))) & 1)) S[a][r] = -INFINITY;
  };
  // O += p v for the values of key k of chunk tile t that are not finite, in the rows that see it;
  // p comes from the lane of the row that holds the key
  auto add_odd = [&](int t, int k) {
    float mine = 0.f;
#pragma unroll
    for (int a = 0; a < C::KSUB; ++a)
#pragma unroll
      for (int r = 0; r < 16; ++r) mine = 32 * a + out_tok(r, g) == k ? S[a][r] : mine;
    const float other = swap_halves(mine), p = ((k >> 2) & 1) == g ? mine : other;
    const bool seen = (sees >> k) & 1;
    const uint16_t* v = (const uint16_t*)A.v_new + (int64_t)(I.qa + (t - htiles) * C::KT + k) * A.kv_new_stride_token + (int64_t)I.kvh * D;
#pragma unroll
    for (int b = 0; b < C::NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const unsigned x = v[column(32 * b + out_tok(r, g))];
        if (seen && (x & kInf) == kInf) O[b][r] = fmaf(p, QT == OSCAR_BF16 ? bf16_bits_to_f32(x) : f16_bits_to_f32(x), O[b][r]);
      }
  };
  // p = exp2(score - reference); the reference moves, and O with it, where a score comes 2^most above it, to
  // 2^below under that
  auto softmax = [&](float below, float most) {
    float mx = -INFINITY;
#pragma unroll
    for (int a = 0; a < C::KSUB; ++a)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, S[a][r]);
    if (!kScaled) mx *= c_score;
    mx = fmaxf(mx, swap_halves(mx));
    const bool up = mx > m_run + most;
    if (__builtin_expect_with_probability(__any(up) != 0, 0, 0.999)) {
      const float to = up ? mx - below : m_run;
      const float f = !up ? 1.f : (m_run == -INFINITY ? 0.f : exp2f(m_run - to));
      l_run *= f;
      m_run = to;
#pragma unroll
      for (int b = 0; b < C::NB; ++b) {
        O[b] *= f;
        __builtin_amdgcn_sched_barrier(0);  // (not all of O in vector registers at a time)
      }
    }
    const float nm = m_run == -INFINITY ? 0.f : -m_run;
    float sum = 0.f;
#pragma unroll
    for (int a = 0; a < C::KSUB; ++a)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p = __builtin_amdgcn_exp2f(kScaled ? S[a][r] + nm : fmaf(S[a][r], c_score, nm));
        S[a][r] = p;
        sum += p;
      }
    l_run += sum;
  };
  auto half = [&]() {
#pragma unroll
    for (int s = 0; s < C::VSTEPS; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) ph[s][e] = q_pair<OSCAR_F16>(S[s >> 1][8 * (s & 1) + 2 * e], S[s >> 1][8 * (s & 1) + 2 * e + 1]);
  };
  // the A operand of O^T's part b in step s: eight keys of column lane % 32
  const int i16 = lane & 15, g16 = lane >> 4;
  const int vrow = (4 * (g16 >> 1) + (i16 >> 2)) * (C::VROW * 2) + 8 * (i16 & 1), unit = 2 * (g16 & 1) + ((i16 & 3) >> 1);
  const int vat0 = vrow + 16 * (unit ^ (g16 >> 1)), vat1 = vrow + 16 * (unit ^ (2 + (g16 >> 1)));
  auto vop = [&](int buf, int s, int b) {
    u32x4 v;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32x2 t = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(
                                                    s_v + buf * C::VBYTES + (h ? vat1 : vat0) + (16 * s + 8 * h) * (C::VROW * 2) + 64 * b)));
      v[2 * h] = t[0];
      v[2 * h + 1] = t[1];
    }
    return v;
  };
  auto pv = [&](int buf) {
#pragma unroll
    for (int b = 0; b < C::NB; ++b)
#pragma unroll
      for (int s = 0; s < C::VSTEPS; ++s) O[b] = mma16<OSCAR_F16>(vop(buf, s, b), ph[s], O[b]);
    __builtin_amdgcn_sched_group_barrier(0x100, 2 * kAheadV, 1);
#pragma unroll
    for (int i = 0; i < C::NB * C::VSTEPS; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
    }
  };
  // a chunk tile of bf16 values: P = hi + lo, both bf16
  auto pv_chunk = [&](int buf) {
#pragma unroll 1
    for (int part = 0; part < 2; ++part) {
#pragma unroll
      for (int s = 0; s < C::VSTEPS; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p0 = S[s >> 1][8 * (s & 1) + 2 * e], p1 = S[s >> 1][8 * (s & 1) + 2 * e + 1];
          const unsigned hb = q_pair<OSCAR_BF16>(p0, p1);
          ph[s][e] = hb;
          S[s >> 1][8 * (s & 1) + 2 * e] = p0 - q_half<OSCAR_BF16>(hb, 0);
          S[s >> 1][8 * (s & 1) + 2 * e + 1] = p1 - q_half<OSCAR_BF16>(hb, 1);
        }
#pragma unroll
      for (int b = 0; b < C::NB; ++b)
#pragma unroll
        for (int s = 0; s < C::VSTEPS; ++s) O[b] = mma16<OSCAR_BF16>(vop(buf, s, b), ph[s], O[b]);
    }
  };

  __syncthreads();  // s_place
  if constexpr (!SLOW) {
    // Who unpacks: waves without rows where there are enough of them, since a SIMD that has two waves
    // with rows has the most to do (wave w runs on SIMD w % 4)
    const int busy = (I.rows + 31) / 32;
    // a wave without rows: the units from, from + step and from + 2 step - 2
    auto serve = [&](auto units, int from, int step) {
      constexpr int N = decltype(units)::value;
      // tiles on their way: with at most 128 rows a tile takes less time than its codes take to
      // come (8 x 24576 tokens, 30 rows 51 -> 46 us, 126 62 -> 57); three or four gain no more
      constexpr int E = N == 2 ? 2 : 1;
      Unit u[E][N > 0 ? N : 1];
#pragma unroll
      for (int i = 0; i < N; ++i) u[0][i] = unit_of(from + step * i - (i == 2 ? 2 : 0));
#pragma unroll
      for (int i = 0; i < N; ++i) load(u[0][i], 0);
#pragma unroll
      for (int e = 1; e < E; ++e)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          u[e][i] = u[0][i];
          load(u[e][i], e);
        }
      auto next = [&](int e, int j) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          fill(u[e][i], j);
          load(u[e][i], j + E);
        }
      };
      next(0, 0);
#pragma unroll 1
      for (int j = 0; j < I.count; j += E) {
        __syncthreads();  // tile j is there, and tile j - 1 has been read
        next(E - 1, j + 1);
        if (E > 1 && j + 1 < I.count) {
          __syncthreads();
          next(0, j + 2);
        }
      }
    };
    if (!active) {
      if (wave < 4 || (wave == 5 && busy == 5)) serve(std::integral_constant<int, 0>{}, 0, 0);
      else if (busy <= 4) serve(std::integral_constant<int, 2>{}, wave - 4, 4);
      else if (busy <= 6) serve(std::integral_constant<int, 3>{}, wave - 6, 4);
      else serve(std::integral_constant<int, 1>{}, wave, 0);
      return;
    }
    // a wave with rows, and a unit of the keys (1), of the values (2) or none
    auto compute = [&](auto kind) {
      constexpr int K = decltype(kind)::value;
      Unit u = unit_of(K == 2 ? 4 + (wave & 3) : wave & 3);
      u.v = K == 2;
      if (K) {
        load(u, 0);
        fill(u, 0);
        load(u, 1);
      }
#pragma unroll 1
      for (int j = 0; j < I.count; ++j) {
        __syncthreads();  // tile j is there, and tile j - 1 has been read
        auto next = [&]() {
          fill(u, j + 1);
          load(u, j + 2);
          __builtin_amdgcn_sched_barrier(0);  // the scores and what unpacking takes share registers
        };
        // The two waves of a SIMD out of step: one unpacks before its products, the other after
        if (K == 1) next();
        qk(j & 1);
        __builtin_amdgcn_sched_barrier(0);
        softmax(kBelow, kMost);
        half();
        __builtin_amdgcn_sched_barrier(0);
        pv(j & 1);
        __builtin_amdgcn_sched_barrier(0);
        if (K == 2) next();
      }
    };
    if (busy > 6 || (busy > 4 && (wave & 6) == 2)) wave < 4 ? compute(std::integral_constant<int, 1>{}) : compute(std::integral_constant<int, 2>{});
    else compute(std::integral_constant<int, 0>{});
  } else {
    Unit own = unit_of(wave);
    auto scores = [&](int j) {
      const int t = I.first + I.stride * j;
      __syncthreads();  // the buffers and s_odd have been read
      if (tid < 2) s_odd[tid] = 0;
      __syncthreads();
      fill_slow(own, t, j);
      __syncthreads();
      qk(0);
      mask(t);
      const bool chunk = QT == OSCAR_BF16 && t >= htiles;
      softmax(chunk ? kChunk : kBelow, chunk ? kChunk : kMost);
    };
    int j = 0;
    if (I.first < htiles) {  // the ragged end
      scores(j++);
      half();
      pv(0);
    }
#pragma unroll 1
    for (; j < I.count; ++j) {
      scores(j);
#pragma unroll 1
      for (int a = 0; a < C::KSUB; ++a)
        for (uint32_t odd = __builtin_amdgcn_readfirstlane(s_odd[a]); odd != 0; odd &= odd - 1)
          add_odd(I.first + I.stride * j, 32 * a + __builtin_ctz(odd));
      if constexpr (QT == OSCAR_BF16) {
        pv_chunk(0);
      } else {
        half();
        pv(0);
      }
    }
  }

  // ---- the item's partial: O / l and the log-sum-exp
  const float l = l_run + swap_halves(l_run);
  if (row >= I.rows) return;
  const float f = l > 0.f ? 1.f / l : (l != l ? NAN : 0.f);
  float* out = P.part_o + (int64_t)(I.part + row) * D + 4 * g;
#pragma unroll
  for (int b = 0; b < C::NB; ++b)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      *(f32x4*)(out + 32 * b + 8 * e) = f32x4{O[b][4 * e], O[b][4 * e + 1], O[b][4 * e + 2], O[b][4 * e + 3]} * f;
  if (g == 0) P.part_lse[I.part + row] = l != l ? NAN : (l > 0.f ? m_run + log2f(l) : -INFINITY);
}

template <int D, int QT, int SC>
__global__ __launch_bounds__(kThreads, 2) void tree_main_kernel(TreeParams P) {
  using C = Cfg<D>;
  const oscarop_tree_attn_args_v1& T = P.a;
  const oscar_attn_args_v1& A = T.attn;
  const int32_t* it = A.items + (int64_t)blockIdx.x * OSCAROP_TREE_ITEM_INTS;
  const Item I{it[0], it[1], it[2], it[3], it[4], it[5], it[6], it[7], it[8], it[9], it[10]};
  const int bs = (int)A.cache.block_size, tid = threadIdx.x;
  const int G = P.group;
  const int htiles = (int)(((int64_t)I.hist + C::KT - 1) / C::KT);
  const int64_t tiles = htiles + ((int64_t)I.n + C::KT - 1) / C::KT;
  // an item that breaks the plan's rules reads nothing; its rows become NaN where they lie in
  // the partials at all
  if (I.rows < 1 || I.rows > kMostRows || I.part < 0 || (int64_t)I.part + I.rows > T.partial_rows) return;
  if (I.req < 0 || I.req >= A.num_reqs || I.kvh < 0 || I.kvh >= A.cache.num_kv_heads || I.n < 1 || I.hist < 0 || I.qa < 0 ||
      (int64_t)I.qa + I.n > A.num_tokens || I.row0 < 0 || (int64_t)I.row0 + I.rows > (int64_t)I.n * G || I.first < 0 ||
      I.stride < 1 || I.count < 1 || I.count > kMostTiles || I.first + (int64_t)I.stride * (I.count - 1) >= tiles ||
      (I.first < I.hist / C::KT && I.first + (int64_t)I.stride * (I.count - 1) >= I.hist / C::KT) ||
      (I.hist > 0 && (I.hist - 1) / bs >= A.block_table_cols)) {
    for (int i = tid; i < I.rows; i += kThreads) P.part_lse[I.part + i] = NAN;
    return;
  }
  __shared__ __attribute__((aligned(16))) uint8_t s_k[2 * C::KBYTES];
  __shared__ __attribute__((aligned(16))) uint8_t s_v[2 * C::VBYTES];
  __shared__ Place s_place[kMostTiles * C::KSUB];
  __shared__ uint32_t s_odd[2];  // a chunk tile's keys whose values are not all finite
  if (tid < 2) s_odd[tid] = 0;
  const int full = I.hist / C::KT;  // full tiles of the history
  for (int i = tid; i < I.count * C::KSUB; i += kThreads) {
    const int64_t key = (int64_t)(I.first + I.stride * (i / C::KSUB)) * C::KT + 32 * (i % C::KSUB);
    Place x{0, 0, 0, 0};
    if (key < I.hist) {
      x.page = A.block_table[(int64_t)I.req * A.block_table_stride + key / bs];
      x.page = x.page < 0 || x.page >= A.cache.num_blocks ? 0 : x.page;
      x.off = (int)(key % bs);
      if (P.has_stage) x.seat = (int)((unsigned)x.page % (unsigned)P.st.rows) * bs + x.off;
    }
    s_place[i] = x;
  }

  if (I.first >= full) run_item<D, QT, SC, true>(P, I, s_k, s_v, s_place, s_odd);
  else run_item<D, QT, SC, false>(P, I, s_k, s_v, s_place, s_odd);
}

// The items of a block of rows, merged by their log-sum-exps.  One row a 64-lane (D 256) or
// 32-lane (D 128) group, four columns a lane.  Bound by memory: 50 MB of partials of
// 8 x 24576 tokens with 32 nodes in 10 us, eight items' loads of a row in flight at a time.
constexpr int kBatch = 8;
constexpr int kMergeThreads = 256;

template <int D>
__global__ __launch_bounds__(kMergeThreads) void tree_merge_kernel(TreeParams P) {
  const oscarop_tree_attn_args_v1& T = P.a;
  const oscar_attn_args_v1& A = T.attn;
  const int32_t* gr = A.groups + (int64_t)blockIdx.x * OSCAR_GROUP_INTS;
  const int kvh = gr[0], qa = gr[1], row0 = gr[2], rows = gr[3], part = gr[4], many = gr[5], step = gr[6];
  const int lanes = D / 4;
  const int col = threadIdx.x % lanes, G = P.group;
  const int row = blockIdx.y * (kMergeThreads / lanes) + threadIdx.x / lanes;
  if (row >= rows) return;
  const int m = row0 + row;
  const int64_t token = (int64_t)qa + m / G;
  if (row0 < 0 || kvh < 0 || kvh >= A.cache.num_kv_heads || qa < 0 || token >= A.num_tokens) return;
  bool nan = part < 0 || many < 0 || step < rows || (int64_t)part + (int64_t)step * (many - 1) + rows > T.partial_rows;
  const int n = nan ? 0 : many;
  const float* lse = P.part_lse + part + row;
  const f32x4* po = (const f32x4*)(P.part_o + (int64_t)(nan ? 0 : part + row) * D) + col;
  float M = -INFINITY, L = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < n; i += kBatch) {
    float l[kBatch];
    f32x4 x[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const bool in = i + u < n;
      l[u] = in ? lse[(int64_t)(i + u) * step] : -INFINITY;
      x[u] = in ? po[(int64_t)(i + u) * step * (D / 4)] : f32x4{0.f, 0.f, 0.f, 0.f};
    }
    float top = M;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      nan |= l[u] != l[u];
      top = fmaxf(top, l[u]);
    }
    if (top == -INFINITY) continue;
    const float f = M == -INFINITY ? 0.f : exp2f(M - top);
    acc *= f;
    L *= f;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const float w = l[u] == -INFINITY ? 0.f : exp2f(l[u] - top) * kWeight;
      L += w;
      acc += w > 0.f ? x[u] * w : f32x4{0.f, 0.f, 0.f, 0.f};
    }
    M = top;
  }
  const bool some = M != -INFINITY && L > 0.f;
  acc = nan ? f32x4{NAN, NAN, NAN, NAN} : (some ? acc * (1.f / L) : f32x4{0.f, 0.f, 0.f, 0.f});
  const int head = kvh * G + m % G;
  // columns 4 i .. 4 i + 3 of a part in LDS order are elements e, e + 4, e + 1, e + 5
  const int e = 16 * (col / 4) + 8 * ((col & 3) >> 1) + 2 * (col & 1);
  float* out = A.out_rot + (token * A.num_q_heads + head) * D + e;
  *(float2*)out = make_float2(acc[0], acc[2]);
  *(float2*)(out + 4) = make_float2(acc[1], acc[3]);
  if (col == 0) A.lse[token * A.num_q_heads + head] = nan ? NAN : (some ? (M + log2f(L / kWeight)) * kLn2 : -INFINITY);
}

template <int D>
int launch_tree(const TreeParams& p, int sc, hipStream_t s) {
  const oscar_attn_args_v1& a = p.a.attn;
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(a.num_items), dim3(kThreads), 0, s, p); };
  const bool f16 = a.q_dtype == OSCAR_F16;
  if (sc == 0) f16 ? launch(tree_main_kernel<D, OSCAR_F16, 0>) : launch(tree_main_kernel<D, OSCAR_BF16, 0>);
  else f16 ? launch(tree_main_kernel<D, OSCAR_F16, 2>) : launch(tree_main_kernel<D, OSCAR_BF16, 2>);
  OSCAR_CHECK_LAUNCH("tree_main_kernel");
  constexpr int kRows = kMergeThreads / (D / 4);
  hipLaunchKernelGGL(tree_merge_kernel<D>, dim3(a.num_groups, kMostRows / kRows), dim3(kMergeThreads), 0, s, p);
  OSCAR_CHECK_LAUNCH("tree_merge_kernel");
  return 0;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct Block {
  int req, kvh, qa, n, hist, row0, rows, waves;
  int64_t full, slow;  // tiles: full ones of the history; its ragged end and the chunk's
};

}  // namespace

}  // namespace oscar

using namespace oscar;

extern "C" int oscarop_tree_plan_v1(const int32_t* qsl, const int32_t* seqs, int32_t num_reqs, int32_t num_kv_heads, int32_t group,
                                    int32_t head_dim, int32_t target_items, int32_t* items, int32_t max_items, int32_t* groups,
                                    int32_t max_groups, oscarop_tree_sizes_v1* plan) try {
  if (!qsl || !seqs || !plan || num_reqs < 0 || num_kv_heads < 1 || num_kv_heads > 0xffff || group < 1 || group > 1 << 16)
    return fail(-22, "oscarop_tree_plan_v1: invalid arguments");
  if (head_dim != 128 && head_dim != 256) return fail(-22, "oscarop_tree_plan_v1: head_dim %d unsupported (128/256)", head_dim);
  const int kt = 8192 / head_dim;
  if (target_items < 1) target_items = 1;
  std::vector<Block> blocks;
  for (int r = 0; r < num_reqs; ++r) {
    const int64_t n = (int64_t)qsl[r + 1] - qsl[r];
    if (n <= 0) continue;
    if (qsl[r] < 0 || seqs[r] < n) return fail(-22, "oscarop_tree_plan_v1: sequence length must cover its query chunk");
    const int64_t rows = n * group;
    if (rows > 1 << 24) return fail(-22, "oscarop_tree_plan_v1: query chunk of request %d too long", r);
    // as few blocks of at most kMostRows rows as there can be, alike
    const int64_t count = ceil_div(rows, kMostRows), each = ceil_div(rows, count);
    if ((int64_t)blocks.size() + count * num_kv_heads > 1 << 20)
      return fail(-22, "oscarop_tree_plan_v1: too many request x kv-head groups");
    for (int64_t a = 0; a < rows; a += each) {
      const int64_t b = a + each < rows ? a + each : rows;
      const int hist = seqs[r] - (int)n;
      // the block's last node sees no later one
      const int64_t slow = (hist % kt != 0) + ceil_div((b - 1) / group + 1, kt);
      for (int h = 0; h < num_kv_heads; ++h)
        blocks.push_back({r, h, qsl[r], (int)n, hist, (int)a, (int)(b - a), (int)ceil_div(b - a, 32), hist / kt, slow});
    }
  }
  // an item costs its tiles, and a tile its rows and its unpacking, a slow one more; the smallest bound
  // that keeps to target_items (one for each block's kind of tiles at least)
  auto items_of = [&](int64_t tiles, int64_t cost, int64_t most) {
    const int64_t cap = most / cost < 1 ? 1 : (most / cost > kMostTiles ? kMostTiles : most / cost);
    return ceil_div(tiles, cap);
  };
  auto fast_items = [&](const Block& b, int64_t most) { return items_of(b.full, b.waves + 2, most); };
  auto split = [&](const Block& b, int64_t most) { return fast_items(b, most) + items_of(b.slow, kSlowCost * (b.waves + 2), most); };
  int64_t lo = 1, hi = (int64_t)kSlowCost * (kWaves + 2) * kMostTiles;
  while (lo < hi) {
    const int64_t mid = (lo + hi) / 2;
    int64_t total = 0;
    for (const Block& b : blocks) total += split(b, mid);
    if (total <= target_items) hi = mid;
    else lo = mid + 1;
  }
  int64_t num = 0, part = 0, longest = 0;
  for (const Block& b : blocks) {
    const int64_t k = split(b, lo);
    num += k;
    part += k * b.rows;
    longest = k > longest ? k : longest;
  }
  if (num > 1 << 24 || part > INT32_MAX) return fail(-22, "oscarop_tree_plan_v1: too many work items");
  plan->num_items = (int32_t)num;
  plan->num_groups = (int32_t)blocks.size();
  plan->partial_rows = part;
  plan->partial_bytes = part * (head_dim + 1) * (int64_t)sizeof(float);
  if (items == nullptr || groups == nullptr) return (int)num;  // size query
  if (num > max_items || (int64_t)blocks.size() > max_groups) return fail(-28, "oscarop_tree_plan_v1: buffers too small");
  int64_t at = 0;
  std::vector<int64_t> first(blocks.size());
  for (size_t g = 0; g < blocks.size(); ++g) {
    const Block& b = blocks[g];
    first[g] = at;
    int32_t* gr = groups + g * OSCAR_GROUP_INTS;
    const int64_t k = split(b, lo);
    const int32_t record[OSCAR_GROUP_INTS] = {b.kvh, b.qa, b.row0, b.rows, (int32_t)at, (int32_t)k, b.rows, 0};
    for (int i = 0; i < OSCAR_GROUP_INTS; ++i) gr[i] = record[i];
    at += k * b.rows;
  }
  // item p of every block, then p + 1: blocks progress together
  int64_t out = 0;
  for (int64_t p = 0; p < longest; ++p)
    for (size_t g = 0; g < blocks.size(); ++g) {
      const Block& b = blocks[g];
      const int64_t kf = fast_items(b, lo), k = split(b, lo);
      if (p >= k) continue;
      // the slow items first: theirs are the longest
      const int64_t ks = k - kf, x = p < ks ? p : p - ks, of = p < ks ? ks : kf;
      const int64_t begin = p < ks ? b.full + x : x, tiles = p < ks ? b.slow : b.full;
      int32_t* it = items + out++ * OSCAROP_TREE_ITEM_INTS;
      const int32_t record[OSCAROP_TREE_ITEM_INTS] = {b.req, b.kvh, b.qa, b.n, b.hist, b.row0, b.rows, (int32_t)begin,
                                                      (int32_t)of, (int32_t)ceil_div(tiles - x, of),
                                                      (int32_t)(first[g] + p * b.rows), 0};
      for (int i = 0; i < OSCAROP_TREE_ITEM_INTS; ++i) it[i] = record[i];
    }
  return (int)num;
} catch (const std::bad_alloc&) {
  return fail(-12, "oscarop_tree_plan_v1: out of memory");
}

extern "C" int oscarop_attn_tree_v1(const oscarop_tree_attn_args_v1* args, const oscarop_score_v1* score, void* stream) {
  const char* name = "oscarop_attn_tree_v1";
  if (!args) return fail(-22, "%s: null args", name);
  const oscar_attn_args_v1& a = args->attn;
  TreeParams p{};
  const int sc = score_of(score, a.scale, &p.sc);
  if (sc < 0) return fail(-22, kBadCap, name);
  if (p.sc.slopes != nullptr) return fail(-22, "%s: no alibi_slopes with a mask", name);
  const int64_t d = a.cache.head_dim;
  if (d != 128 && d != 256) return fail(-22, "%s: head_dim %lld unsupported", name, (long long)d);
  if (a.num_items <= 0 || a.num_groups <= 0) return 0;
  if (const int rc = attn_check_args(a, name)) return rc;
  if (a.phases != 0) return fail(-22, "%s: phases must be 0", name);
  if (!a.k_new) return fail(-22, "%s: a tree's attention needs its nodes' K and V", name);
  if (!args->mask || ((uintptr_t)args->mask & 7) || args->mask_words < 1)
    return fail(-22, "%s: a mask of at least one word a row, 8-byte aligned", name);
  if (a.num_q_heads / a.cache.num_kv_heads > 1 << 16 || a.cache.num_kv_heads > 0xffff || a.num_groups > 1 << 20)
    return fail(-22, "%s: too many heads or groups", name);
  const int64_t need = args->partial_rows * (d + 1) * (int64_t)sizeof(float);
  if (args->partial_rows < 1 || args->partial_rows > INT32_MAX || !a.workspace || ((uintptr_t)a.workspace & 15) ||
      a.workspace_bytes < need)
    return fail(-22, "%s: workspace of %lld bytes < %lld", name, (long long)a.workspace_bytes, (long long)need);
  // (the largest product is the largest score)
  if (!(a.scale > 0.f) || a.scale > 3e38f) return fail(-22, "%s: scale must be positive and finite", name);
  p.a = *args;
  p.has_stage = a.staging != nullptr;
  if (a.staging) p.st = *a.staging;
  p.group = (int)(a.num_q_heads / a.cache.num_kv_heads);
  p.part_o = (float*)a.workspace;
  p.part_lse = p.part_o + args->partial_rows * d;
  return d == 256 ? launch_tree<256>(p, sc, (hipStream_t)stream) : launch_tree<128>(p, sc, (hipStream_t)stream);
}
