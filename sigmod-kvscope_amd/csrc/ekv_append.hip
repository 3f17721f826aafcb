// Tokens on their way from the projection to attention: norms of each query and key head, the rotation of
// their positions, and the keys' and values' place in a paged cache.  One kernel does a token's heads in one
// pass; ekv_rotate_heads leaves the cache out.
//
// Mathematics.  A head is a vector x of dim elements.  Its norm is y = x * rsqrt(mean(x^2) + eps) * w; pair p of it
// is a complex number that turns by pos * f_p radians.  Angles of far positions lose everything in float32 (a
// million radians have steps of 1/16), so pos * f_p / 2 pi is float64 until its whole turns are gone.
//
// Bound.  Every input is read once and every output written once, 3 or 4 flop an element: bandwidth, or a launch's
// latency where the tokens are few.  Measured (32 query and 8 KV heads of 128, bf16): 38241 tokens of prompts, 940 MB, 155 us
// (6.1 TB/s; a bare copy of the same pattern 155), the norms of 16384 tokens, 335 MB, 57 us (5.9 TB/s), 128 tokens of a
// decode step 4.1 us.
//
// Layout.  A head's pairs are cut into units of 8, a unit a lane: the 8 elements of the first halves and the 8 of the
// second ones, two loads of 16 bytes (of 16-bit types).  A lane then holds whole pairs in either order of them and
// needs nothing of another lane for the rotation; elements that do not rotate are units of the same shape.  (16 lanes a
// head, 1 KB an instruction and partners 8 lanes apart, copied no faster: 153 and 155 us.)  The lanes of a head (a power of
// two; a head dim that is none leaves some idle) lie in one row of 16 lanes, so that the sum of squares is a few DPP moves.
// A wave has 64 / lanes heads of one token and one kind at a time, the next ones on their way.  The cosines and sines of a
// token are computed once a wave, a pair a lane, and pass through LDS to the lanes whose units they turn, 8 times fewer than
// if each lane computed its own; weights that every head shares wait in LDS too (held in registers they cost a quarter of
// the waves, and 69 us where these take 63).
//
// Rounding.  Everything is float32 (angles float64) until one rounding to the output's type, half a step.  A cache's scale
// is multiplied by its rounded reciprocal: one more step of float32, next to nothing beside e4m3's.
#include "ekv_attention.hpp"

namespace ekv {
namespace append {

using attn::f32x4;
using attn::pack2;
using attn::u32x2;
using attn::u32x4;

constexpr int kWaves = 4;         // of a workgroup
constexpr int kMostPairs = 128;   // of a head
constexpr int kUnit = 8;          // pairs of a lane

struct Heads {  // one tensor [tokens, heads, dim]: strides in bytes
  const char *at;
  int64_t token, head;
};
// The stride of an axis of one element is whatever it is, and not used.
inline Heads heads_of(const void *at, int64_t token, int64_t head, int tokens, int heads, int bytes) {
  return {(const char *)at, tokens > 1 ? token * bytes : 0, heads > 1 ? head * bytes : 0};
}

enum Kind { kQuery, kKey, kValue };
enum Past { kNothing, kLoads, kAll };    // what of a pass goes past the caches: nothing, its loads, its queries too
enum Norm { kNone, kShared, kOfHeads };  // no weights; the same of every head; each head's own

struct Params {
  Heads in[3], out[2];  // by Kind
  char *keys, *values;  // the cache, strides in bytes
  int64_t st_block, st_pos, st_head, blocks;
  const int32_t *table;
  int64_t table_stride;
  int32_t *lens, *seen;
  const int32_t *first;
  int64_t first_stride;
  const int32_t *q_start, *positions;
  int64_t positions_stride;
  const double *frequencies;
  const int32_t *axes;
  const char *q_weight, *k_weight;
  int64_t q_weight_stride, k_weight_stride;  // bytes
  float *scores;
  int64_t sc_row, sc_head;
  int32_t *slot_positions;
  int64_t sp_row, sp_head;
  int rows, width, tokens, max_query, q_heads, kv_heads, dim, pairs, axis_count, block_size;
  uint32_t bs_mul;  // page_divisor(block_size)
  int bs_shift;
  bool adjacent, advance, saturate, weight_f32;
  int parts;                // waves of a token: 1, 2 or 4
  int crowd;                // tokens of a wave of crowd_kernel
  PageDivisor by_q_heads, by_kv_heads, by_pairs;
  int lanes_log;            // of a head: 2, 4, 8 or 16 lanes
  int q_passes, kv_passes;  // of 64 / lanes heads, that the queries and that the keys (and the values) of a token take
  float rotary_scale, eps, weight_offset, k_inverse, v_inverse, mean;  // mean: 1 / dim
};

// -- elements -------------------------------------------------------------------------------------

template <class T>
struct Unit {  // 8 elements as they lie in memory (16 of an fp8 cache)
  u32x4 w;
};
template <>
struct Unit<float> {
  u32x4 w, more;
};

// Accesses that go PAST the caches are non-temporal (launch_norm says when).
template <class T, bool PAST>
__device__ __forceinline__ Unit<T> load_unit(const char *at) {
  const auto *p = as_global((const u32x4 *)at);
  Unit<T> u;
  if constexpr (PAST) {
    u.w = __builtin_nontemporal_load(p);
    if constexpr (sizeof(T) == 4) u.more = __builtin_nontemporal_load(p + 1);
  } else {
    u.w = p[0];
    if constexpr (sizeof(T) == 4) u.more = p[1];
  }
  return u;
}

__device__ __forceinline__ void widen(const Unit<float> &u, float (&x)[kUnit]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[e] = __builtin_bit_cast(f32x4, u.w)[e];
    x[4 + e] = __builtin_bit_cast(f32x4, u.more)[e];
  }
}
__device__ __forceinline__ void widen(const Unit<__bf16> &u, float (&x)[kUnit]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[2 * e] = __builtin_bit_cast(float, u.w[e] << 16);
    x[2 * e + 1] = __builtin_bit_cast(float, u.w[e] & 0xffff0000u);
  }
}
__device__ __forceinline__ void widen(const Unit<_Float16> &u, float (&x)[kUnit]) {
  const attn::f16x8 h = __builtin_bit_cast(attn::f16x8, u.w);
#pragma unroll
  for (int e = 0; e < kUnit; ++e) x[e] = (float)h[e];
}

template <class T>
__device__ __forceinline__ void load_weights(const char *at, float (&x)[kUnit]) {
  const auto *p = as_global((const u32x4 *)at);
  if constexpr (sizeof(T) == 4) widen(Unit<T>{p[0], p[1]}, x);
  else widen(Unit<T>{p[0]}, x);
}

// The largest finite e4m3 value for what passes it; NaN stays.
__device__ __forceinline__ float within_e4m3(float x) {
  return __builtin_elementwise_maximum(__builtin_elementwise_minimum(x, 448.f), -448.f);
}

template <class C>
__device__ __forceinline__ Unit<C> narrow(const float (&x)[kUnit]) {
  if constexpr (std::is_same<C, float>::value) {
    return {__builtin_bit_cast(u32x4, f32x4{x[0], x[1], x[2], x[3]}), __builtin_bit_cast(u32x4, f32x4{x[4], x[5], x[6], x[7]})};
  } else {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = pack2(x[2 * e], x[2 * e + 1], C{});
    return {w};
  }
}
__device__ __forceinline__ u32x2 narrow_e4m3(const float (&x)[kUnit], bool saturate) {
  float y[kUnit];
#pragma unroll
  for (int e = 0; e < kUnit; ++e) y[e] = saturate ? within_e4m3(x[e]) : x[e];
  u32x2 w;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int word = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h], y[4 * h + 1], 0, false);
    w[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h + 2], y[4 * h + 3], word, true);
  }
  return w;
}
template <class C, bool PAST>
__device__ __forceinline__ void store_unit(char *at, const Unit<C> &u) {
  auto *p = as_global((u32x4 *)at);
  if constexpr (PAST) {
    __builtin_nontemporal_store(u.w, p);
    if constexpr (sizeof(C) == 4) __builtin_nontemporal_store(u.more, p + 1);
  } else {
    p[0] = u.w;
    if constexpr (sizeof(C) == 4) p[1] = u.more;
  }
}
// A lane's two units of 8 bytes.  Where a lane and its neighbour hold 16 bytes of the first unit and 16 of the second
// beside each other (`paired`), one stores the first and one the second: whole pieces of 128 bytes of a head, where 8 bytes
// a lane leave lines half written.
__device__ __forceinline__ void store_e4m3(char *at, int a, int b, u32x2 x, u32x2 y, bool paired) {
  if (paired) {
    const bool odd = lane_id() & 1;
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      // the neighbour's share: the even lane gives its second unit for the odd lane's first
      const uint32_t got = (uint32_t)dpp_move<0xB1>((int)(odd ? x[i] : y[i]));
      w[i] = odd ? got : x[i];
      w[2 + i] = odd ? y[i] : got;
    }
    store_unit<attn::FP8, true>(at + (odd ? b - kUnit : a), {w});
  } else {
    *as_global((u32x2 *)(at + a)) = x;
    *as_global((u32x2 *)(at + b)) = y;
  }
}

// Sum over the lanes of a head (2, 4, 8 or 16), every one of them receiving it.  All lanes of the wave are active.
__device__ __forceinline__ float head_sum(float v, int lanes) {
  auto add = [&](auto ctrl) {
    v += __builtin_bit_cast(float, dpp_move<decltype(ctrl)::value>(__builtin_bit_cast(int, v)));
  };
  add(std::integral_constant<int, 0xB1>());                   // quad_perm [1, 0, 3, 2]
  if (lanes >= 4) add(std::integral_constant<int, 0x4E>());   // quad_perm [2, 3, 0, 1]
  if (lanes >= 8) add(std::integral_constant<int, 0x141>());  // row_half_mirror: the other quad of 8 lanes
  if (lanes >= 16) add(std::integral_constant<int, 0x140>()); // row_mirror: the other 8 of 16 lanes
  return v;
}

// i / divisor, 0 <= i < 2^31
__device__ __forceinline__ int quotient(int i, const PageDivisor &d) { return (int)(__umulhi((uint32_t)i << 1, d.mul) >> d.shift); }

// -- the arithmetic of a head ---------------------------------------------------------------------
//
// Which products are fused with which sums is written out, so that a head's result is the same bits in every kernel.

// 1 / the root mean square of the head whose elements the lanes hold, two units each (a lane that is not `mine` holds none).
// Elements whose squares vanish beside an eps next to 0, or pass float32, come back scaled, and the result is theirs.
// All lanes of the wave are active.
__device__ __forceinline__ float over_rms(const Params &p, float (&x)[kUnit], float (&y)[kUnit], bool mine, int lanes) {
  float squares = 0.f;
#pragma unroll
  for (int e = 0; e < kUnit; ++e) squares = __builtin_fmaf(x[e], x[e], __builtin_fmaf(y[e], y[e], squares));
  squares = head_sum(mine ? squares : 0.f, lanes);
  const float mean = __builtin_fmaf(squares, p.mean, p.eps);
  float over = rsqrtf(mean);
  // From 2^-100 on, squares below float32's least are nothing beside the others or eps.  A mean below it, or squares past
  // float32: again, of scaled elements.  2^100 is exact, float32's least becomes 2^-49 and what has a mean below 2^-100 stays
  // below 2^54.  2^-70 takes the largest to 2^58, and bits of elements below 2^-56 alone, beside one of 2^60 or more.
  const bool vanish = mean < 0x1p-100f, past = squares == __builtin_inff();
  if (__any(mine && (vanish || past))) {
    const float by = vanish ? 0x1p100f : past ? 0x1p-70f : 1.f;
    squares = 0.f;
#pragma unroll
    for (int e = 0; e < kUnit; ++e) {
      x[e] *= by;
      y[e] *= by;
      squares = __builtin_fmaf(x[e], x[e], __builtin_fmaf(y[e], y[e], squares));
    }
    squares = head_sum(mine ? squares : 0.f, lanes);
    over = rsqrtf(__builtin_fmaf(squares, p.mean, p.eps * by * by));
  }
  return over;
}

// The weights of one head's own, of queries or keys (1 without): elements [a, a + 8) and [b, b + 8).
template <class T>
__device__ __forceinline__ void own_weights(const Params &p, int kind, int head, int a, int b, float (&wa)[kUnit],
                                            float (&wb)[kUnit]) {
  const char *const weight = kind == kQuery ? p.q_weight : p.k_weight;
#pragma unroll
  for (int e = 0; e < kUnit; ++e) wa[e] = wb[e] = 1.f;
  if (weight == nullptr) return;
  const char *row = weight + head * (kind == kQuery ? p.q_weight_stride : p.k_weight_stride);
  if (p.weight_f32) {
    load_weights<float>(row + a * 4, wa);
    load_weights<float>(row + b * 4, wb);
  } else {
    load_weights<T>(row + a * sizeof(T), wa);
    load_weights<T>(row + b * sizeof(T), wb);
  }
#pragma unroll
  for (int e = 0; e < kUnit; ++e) {
    wa[e] += p.weight_offset;
    wb[e] += p.weight_offset;
  }
}

// Weights that every head shares, of queries and of keys: asked for as they lie in memory (converting one at once would wait
// for it at once), then kept in LDS (1 without).
template <class T>
struct SharedWeights {
  static constexpr int kHeld = 2 * kMostPairs / kWave;  // of a lane, for each kind
  uint32_t raw[2][kHeld];
  __device__ __forceinline__ void load(const Params &p) {
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      const int i = k * kWave + lane_id();
#pragma unroll
      for (int kind = 0; kind < 2; ++kind) {
        const char *const weight = kind == kQuery ? p.q_weight : p.k_weight;
        raw[kind][k] = 0;
        if (weight != nullptr && i < p.dim)
          raw[kind][k] = p.weight_f32 ? as_global((const uint32_t *)weight)[i] : as_global((const uint16_t *)weight)[i];
      }
    }
  }
  __device__ __forceinline__ void keep(const Params &p, float (&to)[2][2 * kMostPairs]) const {
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
#pragma unroll
      for (int kind = 0; kind < 2; ++kind) {
        const uint32_t w = raw[kind][k];
        const float x = p.weight_f32 || sizeof(T) == 4 ? __builtin_bit_cast(float, w)
                        : std::is_same<T, __bf16>::value ? __builtin_bit_cast(float, w << 16)
                                                         : (float)__builtin_bit_cast(_Float16, (uint16_t)w);
        const bool weighs = (kind == kQuery ? p.q_weight : p.k_weight) != nullptr;
        to[kind][k * kWave + lane_id()] = weighs ? p.weight_offset + x : 1.f;
      }
    }
  }
};

// The cosine and sine, times the rotary scale, of a position times a frequency.
__device__ __forceinline__ void turn_of(const Params &p, double pos, double frequency, float &cosine, float &sine) {
  const double angle = pos * frequency, whole = __builtin_rint(angle * 0.15915494309189533577);  // 1 / 2 pi
  const float x = (float)__builtin_fma(angle, 0.15915494309189533577, -whole);
  float s, c;
  sincospif(2.f * x, &s, &c);
  cosine = c * p.rotary_scale;
  sine = s * p.rotary_scale;
}

// The lane's 8 pairs turned: x[e] with y[e], or adjacent elements of x and then of y.
template <bool ADJACENT>
__device__ __forceinline__ void rotate(float (&x)[kUnit], float (&y)[kUnit], const float (&cosine)[kUnit],
                                       const float (&sine)[kUnit]) {
  auto turn = [&](float &u, float &v, float c, float s) {
    const float was = u;
    u = __builtin_fmaf(was, c, -(v * s));
    v = __builtin_fmaf(was, s, v * c);
  };
#pragma unroll
  for (int e = 0; e < kUnit; ++e) {
    if constexpr (!ADJACENT) turn(x[e], y[e], cosine[e], sine[e]);
    else if (e < 4) turn(x[2 * e], x[2 * e + 1], cosine[e], sine[e]);
    else turn(y[2 * e - 8], y[2 * e - 7], cosine[e], sine[e]);
  }
}

// What a lane holds of a head.
struct Share {
  bool active;  // an idle lane reads what the first lane of its head does, and writes nothing
  bool turns;   // its elements are rotated
  int nth;      // the head of the pass
  int a, b;     // its elements: [a, a + 8) and [b, b + 8)
  int low, high;  // the pairs of its cosines: [low, low + 4) and [high, high + 4)
};
template <bool ADJACENT>
__device__ __forceinline__ Share share_of(const Params &p) {
  const int lane = lane_id(), lanes = 1 << p.lanes_log, turning = p.pairs / kUnit, rest = p.dim - 2 * p.pairs;
  Share s;
  s.nth = lane >> p.lanes_log;
  s.active = (lane & (lanes - 1)) * 2 * kUnit < p.dim;
  const int unit = s.active ? lane & (lanes - 1) : 0;
  s.turns = unit < turning;
  s.a = s.turns ? unit * kUnit : 2 * p.pairs + (unit - turning) * kUnit;
  s.b = s.turns ? p.pairs + s.a : s.a + rest / 2;
  // adjacent: [a, a + 8) are pairs a / 2 .. a / 2 + 3, [b, b + 8) those from b / 2 on
  s.low = !s.turns ? 0 : ADJACENT ? s.a / 2 : s.a;
  s.high = !s.turns ? 0 : ADJACENT ? s.b / 2 : s.a + 4;
  return s;
}

// -- where a token belongs ------------------------------------------------------------------------

struct Place {
  bool live;      // the token is one of a row's first max_query
  int row;
  int64_t slot, index;
  bool in_table;  // the slot is one of the row's table
  int64_t page;   // of the slot, -1 for none
};

__device__ __forceinline__ int capacity(const Params &p) { return p.width * p.block_size; }  // below 2^31 - 4096

// The row of a token: the last of the ascending start[0 .. rows) that is at most `token`.  load() asks for a window of 254
// starts (of more rows, those between two of every rows / 64-th, and so on) and for their neighbours on both sides; find()
// counts in it.  Between the two a wave asks for its first heads: what a wave asked for first is there first, so that the
// row is known while the heads are on their way.
struct RowSearch {
  static constexpr int kHeld = 4;
  int32_t value[kHeld];
  int below, n;  // start[0 .. below) are at most `token`, start[below + n ..] are not

  __device__ __forceinline__ void load(const int32_t *start, int rows, int token) {
    const int lane = lane_id();
    below = 0;
    n = rows;
    while (n > kHeld * kWave - 2) {
      const int step = (n + kWave - 1) / kWave, i = (lane + 1) * step - 1;
      const bool low = i < n && start[below + i] <= token;
      const int whole = __popcll(__ballot(low)) * step;
      below += whole;
      n = min(step, n - whole);
    }
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      const int j = k * kWave + lane, i = below - 1 + j;  // the first is the last one known to be at most `token`
      value[k] = j <= n + 1 && i >= 0 ? start[i] : 0;
    }
  }
  // (row, its first token, the next row's); row -1 for a token before the first
  __device__ __forceinline__ void find(int token, int &row, int &begin, int &end) const {
    const int lane = lane_id();
    int found = 0;
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      const int j = k * kWave + lane;
      found += __popcll(__ballot(j >= 1 && j <= n && value[k] <= token));
    }
    auto at = [&](int j) {
      int v = __builtin_amdgcn_readlane(value[0], j & (kWave - 1));
#pragma unroll
      for (int k = 1; k < kHeld; ++k)
        if (j / kWave == k) v = __builtin_amdgcn_readlane(value[k], j & (kWave - 1));
      return v;
    };
    row = below + found - 1;
    begin = at(found);
    end = at(found + 1);
  }
};

__device__ __forceinline__ Place place_of(const Params &p, int token, const RowSearch &search) {
  Place at{false, 0, 0, 0, false, -1};
  int count = 1, nth = 0;
  at.row = token;
  if (p.q_start != nullptr) {
    int begin, end;
    search.find(token, at.row, begin, end);
    if (at.row < 0) return at;
    const int a = min(max(begin, 0), p.tokens);
    const int b = min(max(end, a), p.tokens);
    count = b - a;
    nth = token - a;
  }
  at.live = nth < count && nth < p.max_query;
  if (!at.live) return at;
  const int len = min(max(p.lens[at.row], 0), capacity(p));
  const int back = p.advance ? 0 : count;
  at.slot = (int64_t)len - back + nth;
  at.index = p.seen != nullptr ? (int64_t)p.seen[at.row] - back + nth : at.slot;
  at.in_table = at.slot >= 0 && at.slot < capacity(p);
  if (at.in_table) {
    const int32_t page = p.table[at.row * p.table_stride + (int)(__umulhi((uint32_t)at.slot << 1, p.bs_mul) >> p.bs_shift)];
    at.page = page >= 0 && page < p.blocks ? page : -1;
  }
  return at;
}

// What a row of t tokens becomes when they are in.
__device__ __forceinline__ void advance_row(const Params &p, int row, int t) {
  const int kept = min(t, p.max_query), len = min(max(p.lens[row], 0), capacity(p));
  if (kept <= 0) return;
  p.lens[row] = len + min(kept, capacity(p) - len);
  if (p.seen != nullptr) p.seen[row] += kept;
}

// -- the pass ---------------------------------------------------------------------------------------

// T: the inputs' type.  C: the cache's (FP8 or T).  PAGED: with a cache and values; else keys go to k_out.  NORM: what
// weights there are.  ADJACENT: the order of the pairs.  PAST: what goes past the caches.
// Waves a SIMD: those of 16-bit heads with their own weights are asked for (one fewer, by two registers, took 68.5 us where
// 16384 tokens of 32 query and 8 KV heads of 128 into an fp8 cache take 65, and 41.5 where crowd_kernel takes 36 for 65536
// tokens of 4 and 1 heads); the others come out at 5 to 8 by themselves.
template <class T, class C, bool PAGED, Norm NORM, bool ADJACENT, Past PAST>
__global__ __launch_bounds__(kWaves *kWave, (sizeof(T) == 2 && NORM == kOfHeads ? 6 : 1)) void heads_kernel(Params p) {
  __shared__ __align__(16) float s_cos[kWaves][kMostPairs], s_sin[kWaves][kMostPairs];
  __shared__ __align__(16) float s_weight[NORM == kShared ? kWaves : 1][2][2 * kMostPairs];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = lane_id();
  const int lanes = 1 << p.lanes_log, per = kWave >> p.lanes_log;  // of a head; heads of a pass
  const int64_t item = (int64_t)blockIdx.x * kWaves + wave;
  const int token = (int)(item / p.parts), part = (int)(item % p.parts);

  const Share share = share_of<ADJACENT>(p);
  const bool active = share.active, turns = share.turns;
  const int nth = share.nth, a = share.a, b = share.b;
  const bool paired = p.pairs / kUnit % 2 == 0 && p.dim % 32 == 0;  // fp8 caches: store_e4m3

  // The passes of the queries, then the keys, then the values; the wave takes every parts-th.  A pass has heads of one
  // kind, so that what depends on the kind is scalar.
  const int passes = p.q_passes + (PAGED ? 2 : 1) * p.kv_passes;
  auto kind_of = [&](int pass) { return pass < p.q_passes ? kQuery : pass < p.q_passes + p.kv_passes ? kKey : kValue; };
  auto first_head = [&](int pass, int kind) {
    return (pass - (kind == kQuery ? 0 : p.q_passes + (kind == kValue ? p.kv_passes : 0))) * per;
  };
  auto heads_of = [&](int kind) { return kind == kQuery ? p.q_heads : p.kv_heads; };
  Unit<T> ua, ub;
  auto fetch = [&](int pass) {
    const int kind = kind_of(pass), head = min(first_head(pass, kind) + nth, heads_of(kind) - 1);
    const Heads &from = p.in[kind];
    const char *x = from.at + token * from.token + head * from.head;
    ua = load_unit<T, PAST != kNothing>(x + a * sizeof(T));
    ub = load_unit<T, PAST != kNothing>(x + b * sizeof(T));
  };

  if (token < p.tokens) {
    // What the token's place, its angles and the norms are made of is asked for ahead of the heads.
    RowSearch search;
    if (PAGED && p.q_start != nullptr) search.load(p.q_start, p.rows, token);
    constexpr int kTurns = kMostPairs / kWave;  // pairs of a lane
    double frequency[kTurns];
    int axis[kTurns];
#pragma unroll
    for (int k = 0; k < kTurns; ++k) {
      const int i = k * kWave + lane;
      frequency[k] = i < p.pairs ? p.frequencies[i] : 0.0;
      axis[k] = p.axes != nullptr && i < p.pairs ? p.axes[i] : 0;
    }
    SharedWeights<T> weights;
    if constexpr (NORM == kShared) weights.load(p);
    if (part < passes) fetch(part);

    Place at{true, 0, 0, 0, false, -1};
    if constexpr (PAGED) at = place_of(p, token, search);
    if constexpr (NORM == kShared) weights.keep(p, s_weight[wave]);

    // the token's cosines and sines
    float cosine[kUnit], sine[kUnit];
    if (p.pairs > 0) {
      int64_t own = at.index;
      if (PAGED && p.first != nullptr && at.live) own += p.first[at.row * p.first_stride];
#pragma unroll
      for (int k = 0; k < kTurns; ++k) {
        const int i = k * kWave + lane;
        if (k * kWave >= p.pairs) break;
        double pos = (double)own;
        if (p.positions != nullptr) {  // the axes' positions are scalar
          int32_t mine = 0;
          for (int x = 0; x < p.axis_count; ++x) {
            const int32_t there = __builtin_amdgcn_readfirstlane(p.positions[x * p.positions_stride + token]);
            mine = axis[k] == x ? there : mine;
          }
          pos = (double)mine;
        }
        turn_of(p, pos, frequency[k], s_cos[wave][i], s_sin[wave][i]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      cosine[e] = s_cos[wave][share.low + e];
      sine[e] = s_sin[wave][share.low + e];
      cosine[4 + e] = s_cos[wave][share.high + e];
      sine[4 + e] = s_sin[wave][share.high + e];
    }

    int64_t in_page = 0;
    if constexpr (PAGED) {
      if (at.page >= 0) {
        const int64_t block = __umulhi((uint32_t)at.slot << 1, p.bs_mul) >> p.bs_shift;
        in_page = at.page * p.st_block + (at.slot - block * p.block_size) * p.st_pos;
      }
      if (part == 0 && at.live && at.in_table && (p.scores != nullptr || p.slot_positions != nullptr)) {
        for (int h = lane; h < p.kv_heads; h += kWave) {  // a new slot has no weight yet
          if (p.scores != nullptr) p.scores[at.row * p.sc_row + h * p.sc_head + at.slot] = 0.f;
          if (p.slot_positions != nullptr) p.slot_positions[at.row * p.sp_row + h * p.sp_head + at.slot] = (int32_t)at.index;
        }
      }
    }

    for (int pass = part; pass < passes; pass += p.parts) {
      const int kind = kind_of(pass), head = first_head(pass, kind) + nth, heads = heads_of(kind);
      const bool mine = active && head < heads;
      const Unit<T> va = ua, vb = ub;
      if (pass + p.parts < passes) fetch(pass + p.parts);
      // where a token of no row has nothing to write but 0 for its queries
      if (PAGED && (kind == kQuery ? !at.live : at.page < 0)) {
        if (kind == kQuery && mine) {
          char *to = (char *)p.out[kQuery].at + token * p.out[kQuery].token + head * p.out[kQuery].head;
          store_unit<T, PAST == kAll>(to + a * sizeof(T), Unit<T>{});
          store_unit<T, PAST == kAll>(to + b * sizeof(T), Unit<T>{});
        }
        continue;
      }
      float x[kUnit], y[kUnit];
      widen(va, x);
      widen(vb, y);
      if (NORM != kNone && (!PAGED || kind != kValue)) {
        const float over = (kind == kQuery ? p.q_weight : p.k_weight) == nullptr ? 1.f : over_rms(p, x, y, mine, lanes);
        float wa[kUnit], wb[kUnit];
        if constexpr (NORM == kShared) {
#pragma unroll
          for (int e = 0; e < kUnit; ++e) {
            wa[e] = s_weight[wave][kind][a + e];
            wb[e] = s_weight[wave][kind][b + e];
          }
        } else {
          own_weights<T>(p, kind, min(head, heads - 1), a, b, wa, wb);
        }
#pragma unroll
        for (int e = 0; e < kUnit; ++e) {
          x[e] *= over * wa[e];
          y[e] *= over * wb[e];
        }
      }
      if (turns && (!PAGED || kind != kValue)) rotate<ADJACENT>(x, y, cosine, sine);
      if (!PAGED || kind == kQuery) {
        if (mine) {
          const Heads &out = p.out[kind];
          char *to = (char *)out.at + (int64_t)token * out.token + head * out.head;
          store_unit<T, PAST == kAll>(to + a * sizeof(T), narrow<T>(x));
          store_unit<T, PAST == kAll>(to + b * sizeof(T), narrow<T>(y));
        }
      } else {  // the slot's key or value
        const float inverse = kind == kValue ? p.v_inverse : p.k_inverse;
#pragma unroll
        for (int e = 0; e < kUnit; ++e) {
          x[e] *= inverse;
          y[e] *= inverse;
        }
        char *to = (kind == kValue ? p.values : p.keys) + in_page + head * p.st_head;
        if constexpr (std::is_same<C, attn::FP8>::value) {
          const u32x2 xa = narrow_e4m3(x, p.saturate), yb = narrow_e4m3(y, p.saturate);
          if (mine) store_e4m3(to, a, b, xa, yb, paired);
        } else if (mine) {
          store_unit<T, true>(to + a * sizeof(T), narrow<T>(x));
          store_unit<T, true>(to + b * sizeof(T), narrow<T>(y));
        }
      }
    }
  }
  if constexpr (PAGED) {
    // Without q_start a row's token is one workgroup's, whose waves have all read the row's length by now; else
    // advance_kernel runs behind this one.
    if (p.advance && p.q_start == nullptr) {
      __syncthreads();
      if (token < p.tokens && part == 0 && lane == 0) advance_row(p, token, 1);
    }
  }
}

// Heads without a cache, several tokens a wave: where a token's heads leave most of a pass idle, a pass takes the heads of one
// kind of `crowd` tokens in a row.  Their angles are spread over all lanes, and each lane reads its token's for each pass.
template <class T, Norm NORM, bool ADJACENT, Past PAST>
__global__ __launch_bounds__(kWaves *kWave, (sizeof(T) == 2 && NORM == kOfHeads ? 8 : 1)) void crowd_kernel(Params p) {
  constexpr int kMostTurns = kWave * kUnit;  // of the wave's tokens: no more than a pass has heads, 8 pairs a lane
  __shared__ __align__(16) float s_cos[kWaves][kMostTurns], s_sin[kWaves][kMostTurns];
  __shared__ __align__(16) float s_weight[NORM == kShared ? kWaves : 1][2][2 * kMostPairs];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = lane_id();
  const int lanes = 1 << p.lanes_log, per = kWave >> p.lanes_log;  // of a head; heads of a pass
  const int64_t first = ((int64_t)blockIdx.x * kWaves + wave) * p.crowd;
  if (first >= p.tokens) return;
  const int n = (int)min((int64_t)p.crowd, p.tokens - first);
  const Share share = share_of<ADJACENT>(p);
  const int a = share.a, b = share.b;
  const int q_passes = (n * p.q_heads + per - 1) / per, passes = q_passes + (n * p.kv_heads + per - 1) / per;
  struct Item {
    int t, head;  // of the wave's tokens, of its heads of the kind
    bool there;
  };
  auto item_of = [&](int pass, int kind) {
    const int heads = kind == kQuery ? p.q_heads : p.kv_heads;
    const int i = (pass - (kind == kQuery ? 0 : q_passes)) * per + share.nth, last = n * heads - 1;
    const int within = min(i, last), t = quotient(within, kind == kQuery ? p.by_q_heads : p.by_kv_heads);
    return Item{t, within - t * heads, i <= last};
  };
  Unit<T> ua, ub;
  auto fetch = [&](int pass) {
    const int kind = pass < q_passes ? kQuery : kKey;
    const Item item = item_of(pass, kind);
    const char *x = p.in[kind].at + (first + item.t) * p.in[kind].token + item.head * p.in[kind].head;
    ua = load_unit<T, PAST != kNothing>(x + a * sizeof(T));
    ub = load_unit<T, PAST != kNothing>(x + b * sizeof(T));
  };
  SharedWeights<T> weights;
  if constexpr (NORM == kShared) weights.load(p);
  fetch(0);
  if constexpr (NORM == kShared) weights.keep(p, s_weight[wave]);
  for (int i = lane; i < n * p.pairs; i += kWave) {
    const int t = quotient(i, p.by_pairs), pair = i - t * p.pairs, axis = p.axes != nullptr ? p.axes[pair] : 0;
    double pos = 0.0;
    if ((uint32_t)axis < (uint32_t)p.axis_count) pos = (double)p.positions[axis * p.positions_stride + first + t];
    turn_of(p, pos, p.frequencies[pair], s_cos[wave][i], s_sin[wave][i]);
  }
  __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
  __builtin_amdgcn_wave_barrier();
  for (int pass = 0; pass < passes; ++pass) {
    const int kind = pass < q_passes ? kQuery : kKey;
    const Item item = item_of(pass, kind);
    const bool mine = share.active && item.there;
    float x[kUnit], y[kUnit];
    widen(ua, x);
    widen(ub, y);
    if (pass + 1 < passes) fetch(pass + 1);
    if constexpr (NORM != kNone) {
      const float over = (kind == kQuery ? p.q_weight : p.k_weight) == nullptr ? 1.f : over_rms(p, x, y, mine, lanes);
      float wa[kUnit], wb[kUnit];
      if constexpr (NORM == kShared) {
#pragma unroll
        for (int e = 0; e < kUnit; ++e) {
          wa[e] = s_weight[wave][kind][a + e];
          wb[e] = s_weight[wave][kind][b + e];
        }
      } else {
        own_weights<T>(p, kind, item.head, a, b, wa, wb);
      }
#pragma unroll
      for (int e = 0; e < kUnit; ++e) {
        x[e] *= over * wa[e];
        y[e] *= over * wb[e];
      }
    }
    if (share.turns) {
      float cosine[kUnit], sine[kUnit];
      const int at = item.t * p.pairs;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        cosine[e] = s_cos[wave][at + share.low + e];
        sine[e] = s_sin[wave][at + share.low + e];
        cosine[4 + e] = s_cos[wave][at + share.high + e];
        sine[4 + e] = s_sin[wave][at + share.high + e];
      }
      rotate<ADJACENT>(x, y, cosine, sine);
    }
    if (mine) {
      char *to = (char *)p.out[kind].at + (first + item.t) * p.out[kind].token + item.head * p.out[kind].head;
      store_unit<T, PAST == kAll>(to + a * sizeof(T), narrow<T>(x));
      store_unit<T, PAST == kAll>(to + b * sizeof(T), narrow<T>(y));
    }
  }
}

__global__ __launch_bounds__(256) void advance_kernel(Params p) {
  const int row = blockIdx.x * 256 + threadIdx.x;
  if (row >= p.rows) return;
  const int a = min(max(p.q_start[row], 0), p.tokens);
  const int b = min(max(p.q_start[row + 1], a), p.tokens);
  advance_row(p, row, b - a);
}

// -- host -----------------------------------------------------------------------------------------

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
constexpr int64_t kMostWaves = (1ll << 26) - 64;  // a launch has fewer than 2^32 threads

template <class T, class C, bool PAGED, Norm NORM, Past PAST>
int launch_pairs(const Params &p, hipStream_t stream, const char *who) {
  if constexpr (!PAGED) {
    if (p.crowd > 1) {
      const dim3 grid((unsigned)ceil_div(ceil_div(p.tokens, p.crowd), kWaves)), block(kWaves * kWave);
      if (p.adjacent) hipLaunchKernelGGL((crowd_kernel<T, NORM, true, PAST>), grid, block, 0, stream, p);
      else hipLaunchKernelGGL((crowd_kernel<T, NORM, false, PAST>), grid, block, 0, stream, p);
      return check_hip(hipGetLastError(), who);
    }
  }
  const dim3 grid((unsigned)ceil_div((int64_t)p.tokens * p.parts, kWaves)), block(kWaves * kWave);
  if (p.adjacent) hipLaunchKernelGGL((heads_kernel<T, C, PAGED, NORM, true, PAST>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((heads_kernel<T, C, PAGED, NORM, false, PAST>), grid, block, 0, stream, p);
  return check_hip(hipGetLastError(), who);
}

template <class T, class C, bool PAGED, Norm NORM>
int launch_norm(Params p, hipStream_t stream, const char *who) {
  p.lanes_log = p.dim <= 32 ? 1 : p.dim <= 64 ? 2 : p.dim <= 128 ? 3 : 4;
  p.q_passes = (int)ceil_div(p.q_heads, kWave >> p.lanes_log);
  p.kv_passes = (int)ceil_div(p.kv_heads, kWave >> p.lanes_log);
  const int passes = p.q_passes + (PAGED ? 2 : 1) * p.kv_passes;
  // What goes past the 256 MB Infinity Cache, by what the launch moves (cache pages do in any launch, but for fp8 units of 8
  // bytes).  Measured, us, alone / with a kernel behind that reads the rotated queries, as nothing, the loads, loads and
  // queries go past; MiB.  32 query and 8 KV heads of 128 in bf16: 120 25.5 / 45.0, 24.4 / 41.3, 25.2 / 43.8; 220 46.9 / 77.9,
  // 40.9 / 69.6, 41.4 / 74.8; 280 56.9 / 99.6, 54.4 / 86.8, 51.7 / 92.6; 340 68 / 116, 67 / 109, 62 / 111; 500 98 / 165,
  // 97 / 161, 90 / 159; into a cache 900 172 / 277, 182 / 283, 163 / 268.  Pieces that do not fill lines of 128 bytes are read
  // twice past the caches, which the next kernel's reads make good for in smaller launches alone: heads of 80 180 41.2 / 65.9,
  // 41.1 / 64.1, 46.6 / 74.1; 280 59.5 / 100, 63.8 / 96, 70.0 / 110; 340 71 / 118, 77 / 118, 84 / 132; 500 101 / 168, 110 / 179,
  // 121 / 190; of 96 the same.  fp32 heads of 128, nothing and loads: 180 42.3 / 67.5, 39.7 / 63.6; 280 59.5 / 100, 60.0 / 93;
  // 340 71 / 119, 74 / 116; 500 100 / 170, 104 / 174.
  const int64_t cache_bytes = std::is_same<C, attn::FP8>::value ? 1 : sizeof(T);
  const int64_t moved = p.tokens * (int64_t)p.dim *
                        ((2ll * p.q_heads + 2 * p.kv_heads) * sizeof(T) + (PAGED ? 2 * p.kv_heads * cache_bytes : 0));
  const bool whole = sizeof(T) == 2 && p.pairs % 64 == 0 && (p.dim / 2 - p.pairs) % 64 == 0;
  const Past past = moved < 160ll << 20 ? kNothing : moved < 300ll << 20 ? kLoads : whole ? kAll : kNothing;
  // Waves of a token: four while that does not fill the chip, so that a pass of the heads is not behind another (a decode
  // step's 128 tokens 4.1 us, 4.7 with two, 6.4 with one).  Where there are tokens enough a wave needs passes enough for what
  // it does once, its token's place and angles: two waves from five passes on (16384 tokens' norms, five passes, 60 us, 61
  // with one, 66 with four; 9536 tokens of 16 query and 2 KV heads into a cache, four passes, 21.8, 20.6 with one, 29.3 with
  // four; of 8 and 1, three, 19.3, 16.7, 27.4), and four where the launch outlasts its caches, has no weights to load and six
  // passes (38000 tokens of 32 query and 8 KV heads 156 us, 167 with two, 173 with one; no other shape was measured).
  const bool few = p.tokens * 4ll <= 16ll * cu_count();
  p.parts = few || (past == kAll && NORM == kNone && passes > 5) ? 4 : passes >= 5 ? 2 : 1;
  while (p.parts > 1 && p.parts / 2 >= passes) p.parts /= 2;
  while (p.parts > 1 && (int64_t)p.tokens * p.parts >= kMostWaves) p.parts /= 2;
  // Eight tokens a wave (four of the widest heads), where passes of one token would be more than five eighths idle and the
  // waves stay four a compute unit: 32768 tokens of one query and one KV head of 96, normed, 13 us against 27 one by one, of
  // 4 and 1 of 128 20 / 29, of 16 and 4 of 32 18 / 28; of 4 and 4 of 128, half idle, 31 / 24 without norms.
  p.crowd = 1;
  const int heads_of_pass = kWave >> p.lanes_log, crowd = heads_of_pass < 8 ? heads_of_pass : 8;
  if (!PAGED && (p.q_heads + p.kv_heads) * 8ll <= 3ll * passes * heads_of_pass && p.tokens >= crowd * 4 * cu_count()) {
    p.crowd = crowd;
    if (p.q_heads > 0) p.by_q_heads = page_divisor(p.q_heads);
    if (p.kv_heads > 0) p.by_kv_heads = page_divisor(p.kv_heads);
    if (p.pairs > 0) p.by_pairs = page_divisor(p.pairs);
  }
  if constexpr (sizeof(T) == 2)
    if (past == kAll) return launch_pairs<T, C, PAGED, NORM, kAll>(p, stream, who);
  return past == kLoads ? launch_pairs<T, C, PAGED, NORM, kLoads>(p, stream, who)
                        : launch_pairs<T, C, PAGED, NORM, kNothing>(p, stream, who);
}

template <class T, class C, bool PAGED>
int launch(const Params &p, hipStream_t stream, const char *who) {
  if (p.q_weight == nullptr && p.k_weight == nullptr) return launch_norm<T, C, PAGED, kNone>(p, stream, who);
  if (p.q_weight_stride == 0 && p.k_weight_stride == 0) return launch_norm<T, C, PAGED, kShared>(p, stream, who);
  return launch_norm<T, C, PAGED, kOfHeads>(p, stream, who);
}

template <class T>
int launch_cache(const Params &p, bool fp8, hipStream_t stream) {
  return fp8 ? launch<T, attn::FP8, true>(p, stream, "ekv_append_tokens launch")
             : launch<T, T, true>(p, stream, "ekv_append_tokens launch");
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }
int bytes_of(int dtype) { return dtype == EKV_F32 ? 4 : dtype == EKV_FP8_E4M3 ? 1 : 2; }

// The checks and parameters that both entry points share; `Block` is either one's arguments.
template <class Block>
int fill(const Block *a, Params &p, const char *who) {
  if (a->dtype != EKV_F32 && a->dtype != EKV_F16 && a->dtype != EKV_BF16)
    return fail(EKV_EUNSUPPORTED, "%s: heads of type %d", who, a->dtype);
  if ((a->q_weight != nullptr || a->k_weight != nullptr) && a->weight_dtype != a->dtype && a->weight_dtype != EKV_F32)
    return fail(EKV_EUNSUPPORTED, "%s: weights of type %d with heads of type %d", who, a->weight_dtype, a->dtype);
  if (a->head_dim < 16 || a->head_dim > 256 || a->head_dim % 16 != 0)
    return fail(EKV_EUNSUPPORTED, "%s: head dim %d (a multiple of 16, at most 256)", who, a->head_dim);
  if (a->pairs < 0 || a->pairs % kUnit != 0 || 2 * a->pairs > a->head_dim)
    return fail(EKV_EUNSUPPORTED, "%s: %d rotated pairs of a head of %d (a multiple of 8, at most half)", who, a->pairs,
                a->head_dim);
  if (a->tokens < 0 || a->q_heads < 0 || a->kv_heads < 0 || a->q_heads > (1 << 20) || a->kv_heads > (1 << 20))
    return fail(EKV_EINVAL, "%s: tokens %d, heads %d / %d", who, a->tokens, a->q_heads, a->kv_heads);
  if (a->pairs > 0 && a->frequencies == nullptr) return fail(EKV_EINVAL, "%s: null pointer (frequencies)", who);
  if (a->pairs > 0 && a->positions != nullptr &&
      (a->axis_count < 1 || a->positions_stride < 0))
    return fail(EKV_EINVAL, "%s: positions of %d axes, stride %lld", who, a->axis_count, (long long)a->positions_stride);
  if (!(a->eps >= 0.f)) return fail(EKV_EINVAL, "%s: eps %g", who, a->eps);
  const int e = bytes_of(a->dtype), we = bytes_of(a->weight_dtype);
  p = Params{};
  p.in[kQuery] = heads_of(a->query, a->q_stride_token, a->q_stride_head, a->tokens, a->q_heads, e);
  p.out[kQuery] = heads_of(a->q_out, a->q_out_stride_token, a->q_out_stride_head, a->tokens, a->q_heads, e);
  p.positions = a->pairs > 0 ? a->positions : nullptr;
  p.positions_stride = a->positions_stride;
  p.frequencies = a->frequencies;
  p.axes = a->axes;
  p.q_weight = a->q_heads > 0 ? (const char *)a->q_weight : nullptr;
  p.k_weight = (const char *)a->k_weight;
  p.q_weight_stride = a->q_weight_stride * we;
  p.k_weight_stride = a->k_weight_stride * we;
  p.tokens = a->tokens;
  p.q_heads = a->q_heads;
  p.kv_heads = a->kv_heads;
  p.dim = a->head_dim;
  p.pairs = a->pairs;
  p.axis_count = a->axis_count;
  p.adjacent = a->adjacent != 0;
  p.weight_f32 = a->weight_dtype == EKV_F32;
  p.rotary_scale = a->rotary_scale;
  p.eps = a->eps;
  p.weight_offset = a->weight_offset;
  p.mean = 1.f / a->head_dim;
  return EKV_OK;
}

bool row_aligned(const Heads &h) { return aligned16(h.at) && h.token % 16 == 0 && h.head % 16 == 0; }
bool weight_aligned(const char *at, int64_t stride) { return aligned16(at) && stride % 16 == 0; }

// Whether no two of the rows [tokens, heads] of `bytes` bytes share memory.
bool apart(const Heads &h, int64_t tokens, int64_t heads, int64_t bytes) {
  typedef unsigned __int128 Wide;  // products of strides and counts
  const Wide token = h.token < 0 ? -(Wide)h.token : (Wide)h.token, head = h.head < 0 ? -(Wide)h.head : (Wide)h.head;
  if (tokens < 1 || heads < 1) return true;
  if ((tokens > 1 && token < (Wide)bytes) || (heads > 1 && head < (Wide)bytes)) return false;
  if (tokens < 2 || heads < 2 || token >= head * (Wide)(heads - 1) + bytes || head >= token * (Wide)(tokens - 1) + bytes) return true;
  for (int64_t j = 1; j < heads; ++j) {  // neither axis lies within the other's steps: the tokens nearest to j heads on
    const Wide n = head * (Wide)j / token, off = head * (Wide)j % token;
    if ((n < (Wide)tokens && off < (Wide)bytes) || (n + 1 < (Wide)tokens && token - off < (Wide)bytes)) return false;
  }
  return true;
}

// Whether m counts from a and n from b have one in common.
bool share(const int32_t *a, int64_t m, const int32_t *b, int64_t n) {
  return a != nullptr && b != nullptr && (uintptr_t)a < (uintptr_t)(b + n) && (uintptr_t)b < (uintptr_t)(a + m);
}

}  // namespace append
}  // namespace ekv

using namespace ekv;
using append::kKey;
using append::kQuery;
using append::kValue;

extern "C" int ekv_rotate_heads(const ekv_rotation_t *a, void *stream) {
  const char *who = "ekv_rotate_heads";
  if (a == nullptr) return fail(EKV_EINVAL, "%s: null argument block", who);
  append::Params p;
  const int rc = append::fill(a, p, who);
  if (rc != EKV_OK) return rc;
  const int e = append::bytes_of(a->dtype);
  p.in[kKey] = append::heads_of(a->key, a->k_stride_token, a->k_stride_head, a->tokens, a->kv_heads, e);
  p.out[kKey] = append::heads_of(a->k_out, a->k_out_stride_token, a->k_out_stride_head, a->tokens, a->kv_heads, e);
  if (p.tokens == 0 || p.q_heads + p.kv_heads == 0) return EKV_OK;
  if ((p.q_heads > 0 && (p.in[kQuery].at == nullptr || p.out[kQuery].at == nullptr)) ||
      (p.kv_heads > 0 && (p.in[kKey].at == nullptr || p.out[kKey].at == nullptr)) ||
      (p.pairs > 0 && p.positions == nullptr))
    return fail(EKV_EINVAL, "%s: null pointer", who);
  if (!append::row_aligned(p.in[kQuery]) || !append::row_aligned(p.out[kQuery]) || !append::row_aligned(p.in[kKey]) ||
      !append::row_aligned(p.out[kKey]) || !append::weight_aligned(p.q_weight, p.q_weight_stride) ||
      !append::weight_aligned(p.k_weight, p.k_weight_stride))
    return fail(EKV_EINVAL, "%s: heads and weights start at multiples of 16 bytes", who);
  if (!append::apart(p.out[kQuery], p.tokens, p.q_heads, (int64_t)p.dim * e) ||
      !append::apart(p.out[kKey], p.tokens, p.kv_heads, (int64_t)p.dim * e))
    return fail(EKV_EINVAL, "%s: heads of an output share memory", who);
  if (p.tokens >= append::kMostWaves) return fail(EKV_EINVAL, "%s: %d tokens pass the threads of a launch", who, p.tokens);
  hipStream_t s = (hipStream_t)stream;
  switch (a->dtype) {
    case EKV_F32: return append::launch<float, float, false>(p, s, "ekv_rotate_heads launch");
    case EKV_F16: return append::launch<_Float16, _Float16, false>(p, s, "ekv_rotate_heads launch");
    default: return append::launch<__bf16, __bf16, false>(p, s, "ekv_rotate_heads launch");
  }
}

extern "C" int ekv_append_tokens(const ekv_append_t *a, void *stream) {
  const char *who = "ekv_append_tokens";
  if (a == nullptr) return fail(EKV_EINVAL, "%s: null argument block", who);
  append::Params p;
  const int rc = append::fill(a, p, who);
  if (rc != EKV_OK) return rc;
  if (a->kv_dtype != a->dtype && a->kv_dtype != EKV_FP8_E4M3)
    return fail(EKV_EUNSUPPORTED, "%s: tokens of type %d for a cache of type %d", who, a->dtype, a->kv_dtype);
  if (a->rows < 0 || a->width < 0 || a->max_query < 1 || a->kv_heads < 1 || a->block_size < 1 || a->blocks < 0)
    return fail(EKV_EINVAL, "%s: rows %d, width %d, at most %d tokens a row, %d KV heads, block size %d", who, a->rows,
                a->width, a->max_query, a->kv_heads, a->block_size);
  if (a->q_start == nullptr && (a->tokens != a->rows || a->max_query != 1))
    return fail(EKV_EINVAL, "%s: %d tokens, at most %d a row, of %d rows need q_start", who, a->tokens, a->max_query,
                a->rows);
  if ((int64_t)a->width * a->block_size >= attn::kMostKeys)
    return fail(EKV_EINVAL, "%s: a table of %d blocks of %d tokens passes 2^31 - 4096", who, a->width, a->block_size);
  if (!(a->k_scale > 0.f) || !(a->v_scale > 0.f))
    return fail(EKV_EINVAL, "%s: scales %g and %g", who, a->k_scale, a->v_scale);
  const int e = append::bytes_of(a->dtype), ce = append::bytes_of(a->kv_dtype);
  p.in[kKey] = append::heads_of(a->new_keys, a->k_stride_token, a->k_stride_head, a->tokens, a->kv_heads, e);
  p.in[kValue] = append::heads_of(a->new_values, a->v_stride_token, a->v_stride_head, a->tokens, a->kv_heads, e);
  p.keys = (char *)a->keys;
  p.values = (char *)a->values;
  p.st_block = a->blocks > 1 ? a->kv_stride_block * ce : 0;
  p.st_pos = a->block_size > 1 ? a->kv_stride_pos * ce : 0;
  p.st_head = a->kv_heads > 1 ? a->kv_stride_head * ce : 0;
  p.blocks = a->blocks;
  p.table = a->table;
  p.table_stride = a->table_stride;
  p.lens = a->lens;
  p.seen = a->seen;
  p.first = a->first;
  p.first_stride = a->first_stride;
  p.q_start = a->q_start;
  p.scores = a->scores;
  p.sc_row = a->scores_stride_row;
  p.sc_head = a->scores_stride_head;
  p.slot_positions = a->slot_positions;
  p.sp_row = a->slot_positions_stride_row;
  p.sp_head = a->slot_positions_stride_head;
  p.rows = a->rows;
  p.width = a->width;
  p.max_query = a->max_query;
  p.block_size = a->block_size;
  const PageDivisor d = page_divisor(a->block_size);
  p.bs_mul = d.mul;
  p.bs_shift = d.shift;
  p.advance = a->advance != 0;
  p.saturate = a->saturate != 0;
  p.k_inverse = (float)(1.0 / a->k_scale);
  p.v_inverse = (float)(1.0 / a->v_scale);
  if (p.tokens == 0) return EKV_OK;
  if (p.rows == 0) return fail(EKV_EINVAL, "%s: %d tokens of no row", who, p.tokens);
  if (p.first != nullptr && p.first_stride < 0)
    return fail(EKV_EINVAL, "%s: first of stride %lld", who, (long long)p.first_stride);
  if (p.in[kKey].at == nullptr || p.in[kValue].at == nullptr || p.lens == nullptr ||
      (p.q_heads > 0 && (p.in[kQuery].at == nullptr || p.out[kQuery].at == nullptr)) ||
      (p.width > 0 && (p.keys == nullptr || p.values == nullptr || p.table == nullptr)))
    return fail(EKV_EINVAL, "%s: null pointer", who);
  if (p.blocks < 1 && p.width > 0) return fail(EKV_EINVAL, "%s: tables of an empty cache", who);
  if (!append::row_aligned(p.in[kQuery]) || !append::row_aligned(p.out[kQuery]) || !append::row_aligned(p.in[kKey]) ||
      !append::row_aligned(p.in[kValue]) || !append::aligned16(p.keys) || !append::aligned16(p.values) || p.st_block % 16 != 0 ||
      p.st_pos % 16 != 0 || p.st_head % 16 != 0 || !append::weight_aligned(p.q_weight, p.q_weight_stride) ||
      !append::weight_aligned(p.k_weight, p.k_weight_stride))
    return fail(EKV_EINVAL, "%s: heads, weights and the cache's rows start at multiples of 16 bytes", who);
  if (!append::apart(p.out[kQuery], p.tokens, p.q_heads, (int64_t)p.dim * e))
    return fail(EKV_EINVAL, "%s: heads of an output share memory", who);
  if (p.table_stride < p.width)
    return fail(EKV_EINVAL, "%s: table rows of %d blocks, stride %lld", who, p.width, (long long)p.table_stride);
  if (p.tokens >= append::kMostWaves) return fail(EKV_EINVAL, "%s: %d tokens pass the threads of a launch", who, p.tokens);
  if (p.advance) {  // a row's counts grow while other rows' are read, and each of them once
    const int64_t n = p.rows, reach = p.first == nullptr ? 0 : 1 + (n - 1) * p.first_stride;
    if (append::share(p.lens, n, p.seen, n) || append::share(p.first, reach, p.lens, n) || append::share(p.first, reach, p.seen, n))
      return fail(EKV_EINVAL, "%s: lens, seen and first share memory", who);
  }
  hipStream_t s = (hipStream_t)stream;
  const bool fp8 = a->kv_dtype == EKV_FP8_E4M3;
  int status;
  switch (a->dtype) {
    case EKV_F32: status = append::launch_cache<float>(p, fp8, s); break;
    case EKV_F16: status = append::launch_cache<_Float16>(p, fp8, s); break;
    default: status = append::launch_cache<__bf16>(p, fp8, s); break;
  }
  if (status != EKV_OK || !p.advance || p.q_start == nullptr) return status;
  hipLaunchKernelGGL(append::advance_kernel, dim3((unsigned)append::ceil_div(p.rows, 256)), dim3(256), 0, s, p);
  return check_hip(hipGetLastError(), "ekv_append_tokens advance launch");
}
