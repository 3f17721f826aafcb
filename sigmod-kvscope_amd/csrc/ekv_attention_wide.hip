// Attention of many query rows against one set of keys: prompt chunks over a prefix and their own keys, and
// the queries of a whole group over its shared prefix.  The arithmetic bounds it, so the keys and values of
// a step are staged through LDS once for all the waves of a workgroup, and both products run on the 16-bit
// matrix instruction of 32 x 32 x 16.
//
// A wave has 32 query rows.  S^T = K Q^T leaves a lane one query's logits (keys 8a + 4h + b of each 32, in
// lane half h), so the softmax of a row is in-lane work and one exchange between the halves.  The product
// over keys is a sum, so its order is free as long as both operands agree: O^T = V^T P^T takes a lane's
// weights where they lie, rounded to 16 bits, and the values through the transposing LDS read, four keys
// of one dim a lane.  The weights' rounding (half a step of the type, relative) is of the size of the
// output's own; their sum, the maxima and the outputs are float32.
//
// Measured, head dim 128: 3200 f16 query rows a KV head against prefixes of 32768 tokens 550 to 614 us as the clock goes
// (740 TFLOP/s at best, with the own tokens and the join); bf16 prompt chunks of up to 4096 rows 273 us (675 TFLOP/s).  The narrow form of the
// same calls, one wave for 16 query rows, took 2456 and 1247 us.
#include "ekv_attention.hpp"

namespace ekv {
namespace attn {

template <class T, int D>
struct Wide {
  static constexpr int kWaves = 4;
  static constexpr int kThreads = kWaves * kWave;
  static constexpr int kKeys = D == 256 ? 32 : 64;  // of a step
  static constexpr int kRow = Lds<T, D>::kRow;
  typedef Stage<T, D, kKeys, kThreads> Step;
  static constexpr int kTile = Step::kTile;
};

// One step's rows of 16-bit keys or values from memory straight to LDS, 1 KB an instruction: a lane's 16 bytes land at
// 16 times its number, so which piece of its row a lane asks for makes the permutation.  This saves the 32 registers
// that a step on its way would hold (with them the kernel spilled, and read the operands of one product at a time).
template <class T, int D>
struct Direct {
  using W = Wide<T, D>;
  using L = Lds<T, D>;
  typedef typename W::Step St;
  static constexpr int kPieces = W::kRow / 16;
  static constexpr int kAll = W::kKeys * kPieces;
  static constexpr int kLoads = (kAll + W::kThreads - 1) / W::kThreads;
  // The instruction has no register to return, and waits are for all loads in flight, so the compiler need not know of
  // it.  M0 holds the LDS address, which takes a wait state to arrive.
  __device__ static __forceinline__ void fetch(uint32_t lds, const char *base, uint32_t off) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory");
  }
  __device__ static __forceinline__ void fetch(uint32_t lds, const char *from) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(from) : "memory");
  }
  // the byte of its row that a lane asks for in load i
  template <bool VALUES>
  __device__ static __forceinline__ uint32_t source(int i) {
    const int row = St::first_row(i) + lane_id() / kPieces, at = lane_id() % kPieces;
    return VALUES ? L::value_at(row, at * 16) - row * W::kRow : L::key_at(row, at) - row * W::kRow;
  }
  // The rows from row 16 on are permuted as the first 16, so the loads of rows 16 apart have one lane offset.
  static constexpr int kStep = W::kThreads / kPieces;  // rows from a load to the next
  static constexpr int kOffsets = kStep >= 16 ? 1 : 16 / kStep;
  typedef uint32_t Offsets[kOffsets];
  template <bool VALUES>
  __device__ static __forceinline__ void offsets(const Params &p, Offsets &off) {
#pragma unroll
    for (int i = 0; i < kOffsets; ++i) off[i] = source<VALUES>(i) + (p.whole ? St::lane_offset(p) : 0);
  }
  __device__ static __forceinline__ void load(const Params &p, int64_t place, const char *from, const Offsets &off, char *tile) {
    const uint32_t to = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)tile);
    if (p.whole) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int first = St::first_row(i);
        if (kAll % W::kThreads != 0 && first >= W::kKeys) break;
        fetch(to + first * W::kRow, from + St::place_of(place, first), off[i % kOffsets]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int first = St::first_row(i);
        if (kAll % W::kThreads != 0 && first >= W::kKeys) break;
        fetch(to + first * W::kRow, from + St::shuffled(place, first + lane_id() / kPieces) + off[i % kOffsets]);
      }
    }
  }
  // the wave's rows of values that are not there become 0, once all of its loads have landed (0 * NaN is no zero)
  __device__ static __forceinline__ void clear(uint64_t ok, char *values) {
    const int lane = lane_id();
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int first = St::first_row(i);
      if (kAll % W::kThreads != 0 && first >= W::kKeys) break;
      if (!(ok >> (first + lane / kPieces) & 1)) *(u32x4 *)(values + first * W::kRow + lane * 16) = u32x4{0, 0, 0, 0};
    }
  }
};
// every load of this wave has landed
__device__ __forceinline__ void loads_landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// What a workgroup works on.
struct Item : Range {
  int first, rows, m0;  // first token, query rows, the tile's first one
  int slot;
  int see;              // query token i sees keys below own + see + i
};

// Out 0 and lse -inf for the tokens [from, to) of KV head `head`.
template <class Q, int D>
__device__ __forceinline__ void clear_tokens(const Params &p, int from, int to, int head, int threads) {
  const int64_t n = (int64_t)max(to - from, 0) * p.group;
  for (int64_t i = threadIdx.x; i < n * D; i += threads) {
    const int64_t m = i / D;
    const int token = from + (int)(m / p.group), q_head = head * p.group + (int)(m % p.group);
    ((Q *)p.out)[token * p.o_st + q_head * p.o_sh + i % D] = (Q)0.f;
    if (i % D == 0) p.lse[(int64_t)token * p.q_heads + q_head] = -INFINITY;
  }
}

template <class T, int D>
__device__ __forceinline__ bool own_item(const Params &p, uint32_t index, Item &s) {
  using W = Wide<T, D>;
  s.head = (int)(index % p.kv_heads);
  index /= p.kv_heads;
  s.slot = (int)(index % p.s_own);
  index /= p.s_own;
  int row, tile;
  if (p.packed) {
    auto tiles_of = [&](int r) {  // the first and the last row clear tokens of no row, with queries or without
      const int n = (int)ceil_div((int64_t)min(row_queries(p, r).count, p.max_query) * p.group, p.tile_own);
      return r == 0 || r == p.rows - 1 ? max(n, 1) : n;
    };
    if (!find_tile(p.rows, (int)index, tiles_of, row, tile)) return false;
  } else {  // the last tiles of a row see the most keys: they start first
    row = (int)(index % p.rows);
    tile = p.tiles_own - 1 - (int)(index / p.rows);
  }
  const int len = row_length(p, row);
  const RowQueries t = row_queries(p, row);
  const int count = min(t.count, p.max_query);
  if (p.direct && tile == 0) {  // tokens that no tile writes
    typedef typename T::Query Q;
    clear_tokens<Q, D>(p, t.first + count, t.first + t.count, s.head, W::kThreads);
    if (row == 0) clear_tokens<Q, D>(p, 0, t.first, s.head, W::kThreads);
    if (row == p.rows - 1) clear_tokens<Q, D>(p, t.first + t.count, p.tokens, s.head, W::kThreads);
  }
  s.first = t.first;
  s.rows = count * p.group;
  s.m0 = tile * p.tile_own;
  if (s.m0 >= s.rows) return false;
  s.table = p.table + (int64_t)row * p.table_stride;
  s.ptable = nullptr;
  s.plen = 0;
  const int g = p.wide_pre ? -1 : group_of(p, row);
  if (g >= 0) {
    s.ptable = p.ptable + (int64_t)g * p.ptable_stride;
    s.plen = group_length(p, g);
  }
  s.own = own_begin(s.plen);
  s.see = own_see(p, len, t);
  const int last = (min(s.m0 + p.tile_own, s.rows) - 1) / p.group;
  const int64_t begin = (int64_t)s.slot * p.chunk_own;
  const int seen = min(len, s.see + last);
  s.end = (int)min(begin + p.chunk_own, (int64_t)(seen > 0 ? s.own + seen : s.plen));
  s.begin = (int)min(begin, (int64_t)INT32_MAX);
  return s.begin < s.end || p.direct;
}

// The other lane half's value.
__device__ __forceinline__ float other_half_max(float v) {
  float a, b;
  row_swap32(v, a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float other_half_sum(float v) {
  float a, b;
  row_swap32(v, a, b);
  return a + b;
}

// A running maximum is kept while no row of the wave passes it by more than kSlack (powers of two), so that most steps
// leave the outputs unscaled.  Weights then reach 2^kSlack: 2^8 in bf16, and in f16 2^1, which leaves 2^14 of its lift.
template <class H>
constexpr float kSlack = kLift<H> > 0.f ? 1.f : 8.f;
template <class H>
constexpr float kWideLift = kLift<H> > 0.f ? kLift<H> - kSlack<H> : 0.f;

template <class T, int D>
__device__ __forceinline__ void attend_wide(const Params &p, const Item &s, char *lds) {
  using W = Wide<T, D>;
  typedef typename T::Half H;
  constexpr int KT = W::kKeys / 32, DT = D / 32;
  const int lane = lane_id(), half = lane / 32, n = lane % 32;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int w0 = s.m0 + wave * 32;  // the wave's first query row
  const int m = w0 + n;
  const bool live = m < s.rows;
  const int i_q = live ? m / p.group : 0;
  const int token = s.first + i_q, q_head = s.head * p.group + (live ? m - i_q * p.group : 0);
  const bool any = w0 < s.rows;
  const int limit = live ? min(s.end, s.own + max(0, s.see + i_q)) : 0;  // this lane's query sees keys below it
  const int every = min(s.end, s.own + max(0, s.see + w0 / p.group));    // and every query of the wave keys below this
  const int last_row = min(w0 + 31, s.rows - 1);
  const int most = any ? min(s.end, s.own + max(0, s.see + last_row / p.group)) : 0;  // none sees keys from here on

  // a negative scale turns the query's sign; the smallest one keeps a masked logit at -inf where scale is 0
  const float scale2 = fmaxf(fabsf(p.scale2), 0x1p-126f);
  const uint32_t flip = p.scale2 < 0.f ? 0x80008000u : 0u;
  u32x4 q[D / 16];
#pragma unroll
  for (int c = 0; c < D / 16; ++c) {
    q[c] = u32x4{0, 0, 0, 0};
    if (live) {
      q[c] = *as_global((const u32x4 *)(p.q + ((int64_t)token * p.q_st + (int64_t)q_head * p.q_sh + c * 16 + half * 8) * 2));
      q[c] ^= flip;
    }
  }

  // LDS offsets of this lane's reads
  int key_off[D / 16], value_off[DT];
#pragma unroll
  for (int c = 0; c < D / 16; ++c) key_off[c] = Lds<T, D>::key_at(n, 2 * c + half);
#pragma unroll
  for (int d = 0; d < DT; ++d)
    value_off[d] = W::kTile + Lds<T, D>::value_at(4 * half + lane % 16 / 4, d * 64 + lane / 16 % 2 * 32 + lane % 4 * 8);

  f32x16 acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = f32x16{};
  float top = -INFINITY, sum = 0.f;
  bool far = false;  // a query of the wave has a maximum of kRounded or more, either sign

  // The softmax of a step's logits runs beside the next step's products, so keys are a step ahead of values: step t
  // has its logits already, stores keys t + 2 over keys t, and values t + 1 over values t - 1.
  typedef typename W::Step St;
  typedef Direct<T, D> Di;
  constexpr bool kDirect = T::kBytes == 2;  // fp8 rows pass through registers, where they are widened
  typename St::Rows keys, vals;
  f32x16 xa[KT], xb[KT];
  uint64_t ok = 0, ok1 = 0;  // the keys of this step and the next that are there
  int page2 = -1;     // the pages of the step after the next
  int64_t place1 = 0;  // the rows of the next step
  typename Di::Offsets key_from, value_from;
  if constexpr (kDirect) {
    Di::template offsets<false>(p, key_from);
    Di::template offsets<true>(p, value_from);
  }
  auto products = [&](f32x16 *x, const char *buffer) {
#pragma unroll
    for (int k = 0; k < KT; ++k) x[k] = f32x16{};
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
#pragma unroll
      for (int k = 0; k < KT; ++k)
        x[k] = mfma32(*(const u32x4 *)(buffer + key_off[c] + k * 32 * W::kRow), q[c], x[k], H{});
  };
  if (s.begin < s.end) {
    const int page = St::look(p, s, s.begin), page1 = St::look(p, s, s.begin + W::kKeys);
    page2 = St::look(p, s, s.begin + 2 * W::kKeys);
    ok = St::there(p, page);
    ok1 = St::there(p, page1);
    const int64_t place = St::place(p, s, s.begin, page);
    place1 = St::place(p, s, s.begin + W::kKeys, page1);
    if constexpr (kDirect) {
      Di::load(p, place, p.k, key_from, lds);
      Di::load(p, place, p.v, value_from, lds + W::kTile);
      Di::load(p, place1, p.k, key_from, lds + 2 * W::kTile);
      loads_landed();
      if (ok != ~0ull) Di::clear(ok, lds + W::kTile);
    } else {
      St::load(p, place, p.k, keys);
      St::load(p, place, p.v, vals);
      St::store_keys(keys, lds);
      St::load(p, place1, p.k, keys);
      St::store_values(vals, ok, lds + W::kTile);
      St::store_keys(keys, lds + 2 * W::kTile);
    }
    lds_barrier();
    if (s.begin < most) products(xa, lds);
  }

  // One step: x its logits, y the next one's; `even` holds K and V of its parity, `odd` the other's.
  auto step = [&](int base, f32x16 *x, f32x16 *y, char *even, char *odd) {
    lds_barrier();
    const int next = base + W::kKeys;
    const bool more = next < s.end;
    uint64_t ok2 = 0;
    if (more) {
      const int64_t place2 = St::place(p, s, next + W::kKeys, page2);
      if constexpr (kDirect) {
        Di::load(p, place1, p.v, value_from, odd + W::kTile);
        Di::load(p, place2, p.k, key_from, even);
      } else {
        St::load(p, place1, p.v, vals);
        St::load(p, place2, p.k, keys);
      }
      place1 = place2;
      ok2 = St::there(p, page2);
      page2 = St::look(p, s, next + 2 * W::kKeys);
    }
    if (base < most) {
      if (base + W::kKeys > every || ok != ~0ull) {
        const uint64_t mine = ok >> (4 * half);
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int at = 32 * k + 8 * (i / 4) + i % 4;
            if (!(mine >> at & 1) || base + at + 4 * half >= limit) x[k][i] = -INFINITY;
          }
      }
      float high = x[0][0];
#pragma unroll
      for (int k = 0; k < KT; ++k)
#pragma unroll
        for (int i = 0; i < 16; ++i) high = fmaxf(high, x[k][i]);
      high = lifted<H>(other_half_max(high) * scale2, kWideLift<H>);
      if (!__all(high <= top + kSlack<H>)) {
        const float peak = fmaxf(top, high);
        const float shrink = __builtin_amdgcn_exp2f(top - (peak == -INFINITY ? 0.f : peak));
        sum *= shrink;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[d] *= shrink;
        top = peak;
        far = __any(fabsf(top) >= kRounded && top != -INFINITY);
      }
      const float ref = top == -INFINITY ? 0.f : top;
      // ref is a rounded product, the weights' products are not: a common factor of all weights, less than half a step of f16
      // from 1 below kRounded.  Far out it could be any power of two (and was NaN or 0 at the lowest values of a type), so
      // from there on the products are rounded as ref was.
      float factor = scale2;
      if (far) {
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
          for (int i = 0; i < 16; ++i) x[k][i] *= scale2;
        factor = 1.f;
      }
      products(y, odd);  // past the last step from keys that nothing needs
#pragma unroll
      for (int k = 0; k < KT; ++k)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          x[k][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[k][i], factor, -ref));
          sum += x[k][i];
        }
#pragma unroll
      for (int t = 0; t < W::kKeys / 16; ++t) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack2(x[t / 2][8 * (t % 2) + 2 * i], x[t / 2][8 * (t % 2) + 2 * i + 1], H{});
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const char *from = even + value_off[d] + t * 16 * W::kRow;
          const u32x2 a = read_transposed(from), b = read_transposed(from + 8 * W::kRow);
          acc[d] = mfma32(u32x4{a[0], a[1], b[0], b[1]}, w, acc[d], H{});
        }
      }
    }
    ok = ok1;
    ok1 = ok2;
    if (more) {
      if constexpr (kDirect) {
        loads_landed();
        if (ok != ~0ull) Di::clear(ok, odd + W::kTile);
      } else {
        St::store_keys(keys, even);
        St::store_values(vals, ok, odd + W::kTile);
      }
    }
  };
  char *other = lds + 2 * W::kTile;
  for (int base = s.begin; base < s.end;) {
    step(base, xa, xb, lds, other);
    base += W::kKeys;
    if (base >= s.end) break;
    step(base, xb, xa, other, lds);
    base += W::kKeys;
  }

  sum = other_half_sum(sum);
  if (!live) return;
  if (p.direct) {
    typedef typename T::Query Q;
    const bool none = sum == 0.f;
    const float inv = none ? 0.f : p.v_scale / sum;
    char *o = p.out + ((int64_t)token * p.o_st + (int64_t)q_head * p.o_sh + 4 * half) * 2;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        Q *dst = (Q *)(o + (d * 32 + a * 8) * 2);
#pragma unroll
        for (int b = 0; b < 4; ++b) dst[b] = (Q)(none ? 0.f : acc[d][4 * a + b] * inv);
      }
    if (half == 0) p.lse[(int64_t)token * p.q_heads + q_head] = none ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
    return;
  }
  const int64_t at = ((int64_t)s.slot * p.tokens + token) * p.q_heads + q_head;
  if (half == 0) p.part_ml[at] = make_float2(top, sum);
  float *o = p.part_o + at * D + 4 * half;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int a = 0; a < 4; ++a)
      *(f32x4 *)(o + d * 32 + a * 8) = f32x4{acc[d][4 * a], acc[d][4 * a + 1], acc[d][4 * a + 2], acc[d][4 * a + 3]};
}

template <class T, int D>
__global__ __launch_bounds__((Wide<T, D>::kThreads), (D == 256 ? 1 : 2)) void wide_kernel(const Params p) {
  __shared__ __attribute__((aligned(16))) char lds[4 * Wide<T, D>::kTile];
  Item s;
  if (own_item<T, D>(p, blockIdx.x, s)) attend_wide<T, D>(p, s, lds);
}

// The prefixes: the steps of every (group, tile) are one list, which the workgroups that the chip holds share
// equally.  (In chunks of equal length 648 workgroups had work where 512 fit: 1.24 waves a SIMD over the launch, 574 us
// for 3200 query rows against prefixes of 32768 tokens; in equal shares 558 us at the time, now 470 to 500.)
template <class T, int D>
__global__ __launch_bounds__((Wide<T, D>::kThreads), (D == 256 ? 1 : 2)) void wide_prefix_kernel(const Params p) {
  using W = Wide<T, D>;
  __shared__ __attribute__((aligned(16))) char lds[4 * W::kTile];
  __shared__ int s_group;
  __shared__ int64_t s_at;
  Item s;
  s.head = (int)(blockIdx.x % p.kv_heads);
  const int j = (int)(blockIdx.x / p.kv_heads);
  auto tiles_of = [&](int rows) { return (rows + p.tile_pre - 1) / p.tile_pre; };
  const Share share = share_out<W::kWaves, 1>(
      p.groups, p.share_pre, 2, p.s_pre, [&](int) { return j; },
      [&](int g, int64_t &steps) {
        steps = (group_length(p, g) + W::kKeys - 1) / W::kKeys;
        return steps * tiles_of(group_queries(p, g).count * p.group);
      }, &s_group, &s_at);
  if (j >= share.share) return;
  int64_t at = (int64_t)j * share.total / share.share;
  const int64_t stop = (int64_t)(j + 1) * share.total / share.share;
  int g = uniform(s_group);
  int64_t group_at = uniform(s_at);
  s.table = nullptr;
  s.see = INT32_MIN / 2;  // no own keys, whatever the query token: own + see + i would pass 2^31 behind the longest prefixes
  while (true) {
    const RowQueries t = group_queries(p, g);
    s.plen = s.own = uniform(group_length(p, g));
    s.ptable = p.ptable + (int64_t)g * p.ptable_stride;
    s.first = uniform(t.first);
    s.rows = uniform(t.count * p.group);
    const int steps = (s.plen + W::kKeys - 1) / W::kKeys;
    const int64_t end = group_at + (int64_t)steps * tiles_of(s.rows);
    while (at < min(stop, end)) {
      const int tile = (int)((at - group_at) / steps);
      const int64_t tile_at = group_at + (int64_t)tile * steps;
      const int u0 = (int)(at - tile_at), u1 = (int)(min(stop, tile_at + steps) - tile_at);
      const int j0 = share.worker_of(tile_at);
      s.m0 = tile * p.tile_pre;
      s.slot = p.s_own + j - j0;
      s.begin = u0 * W::kKeys;
      s.end = (int)min((int64_t)u1 * W::kKeys, (int64_t)s.plen);
      if (s.head == 0 && j == j0 && s.m0 + (int)threadIdx.x < s.rows && (int)threadIdx.x < p.tile_pre)
        p.pre_slots[(int64_t)s.first * p.group + s.m0 + threadIdx.x] = share.worker_of(tile_at + steps - 1) - j0 + 1;
      lds_barrier();  // the piece before has been read
      attend_wide<T, D>(p, s, lds);
      at = tile_at + u1;
    }
    if (at >= stop) break;
    group_at = end;
    ++g;
  }
}

// -- the running weights of prompt chunks ----------------------------------------------------------------
//
// A workgroup per (row, KV head, 64 keys).  The keys stay in registers as the matrix instruction's rows, the query
// rows pass by in tiles of 32, wave after wave: S^T = K Q^T again, weights exp2(s - lse), and each lane adds up its
// keys' weights over the queries of its column.  Columns, then waves are summed in one order at the end.  A tile of
// queries is read from L2 once per 64 keys, a tile ahead of its use.  Measured: 777 queries of 7 heads a KV head
// against up to 2047 keys, three rows of 4 KV heads of 64: 43 us (289 us in tiles of 16 query rows, a wave to 64 keys).
// The waves of a workgroup: 8 leave two a SIMD where a few hundred workgroups are all (the 43 us above; 4 waves took 53);
// head dim 256 has registers for one.
template <int D>
constexpr int kPerGroup = D == 256 ? 4 : 8;
constexpr int kWeighKeys = 64;

template <class T, int D>
__global__ __launch_bounds__((kPerGroup<D> * kWave), (D == 256 ? 1 : 2)) void weigh_wide_kernel(const Params p, int pieces) {
  typedef typename T::Half H;
  constexpr int KT = kWeighKeys / 32, C = D / 16;
  __shared__ float s_total[kPerGroup<D>][kWeighKeys];
  const uint32_t block = blockIdx.x;
  const int head = (int)(block % p.kv_heads), piece = (int)(block / p.kv_heads % pieces);
  const int row = (int)(block / p.kv_heads / pieces), begin = piece * kWeighKeys;
  const int len = row_length(p, row), end = min(begin + kWeighKeys, len);
  if (begin >= end) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = lane_id(), half = lane / 32, n = lane % 32;
  const RowQueries t = row_queries(p, row);
  const int see = own_see(p, len, t), rows = min(t.count, p.max_query) * p.group;
  const int32_t *table = p.table + (int64_t)row * p.table_stride;
  const int at = begin + lane;
  int page = -1;
  if (at < end) page = table[page_of(p, at)];
  const bool good = (uint32_t)page < (uint64_t)p.blocks;
  const uint64_t ok = __ballot(good);
  const int64_t off = ((int64_t)(good ? page : 0) * p.st_block + (int64_t)(good ? at - page_of(p, at) * p.block_size : 0) * p.st_pos +
                       (int64_t)head * p.st_head) * T::kBytes;
  const int lo = (int)(uint32_t)off, hi = (int)(off >> 32);
  u32x4 key[KT][C];
#pragma unroll
  for (int k = 0; k < KT; ++k) {
    const char *from = p.k + (int64_t)(((uint64_t)(uint32_t)__shfl(hi, 32 * k + n) << 32) | (uint32_t)__shfl(lo, 32 * k + n));
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if constexpr (T::kBytes == 1) {
        const u32x2 x = *as_global((const u32x2 *)(from + (2 * c + half) * 8));
        key[k][c] = widen(x[0], x[1]);
      } else {
        key[k][c] = *as_global((const u32x4 *)(from + (2 * c + half) * 16));
      }
    }
  }
  struct Queries {
    u32x4 q[C];
    float lse2;  // +inf where the query sees nothing or is none: its weights are 0
    int limit;   // it sees keys below this
  };
  auto fetch = [&](Queries &x, int m0) {
    const int m = m0 + n;
    const bool live = m < rows;
    const int i_q = live ? m / p.group : 0;
    const int token = t.first + i_q, q_head = head * p.group + (live ? m - i_q * p.group : 0);
    const char *from = p.q + ((int64_t)token * p.q_st + (int64_t)q_head * p.q_sh) * 2 + half * 16;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      x.q[c] = u32x4{0, 0, 0, 0};
      if (live) x.q[c] = *as_global((const u32x4 *)(from + c * 32));
    }
    const float lse = live ? p.lse[(int64_t)token * p.q_heads + q_head] : -INFINITY;
    x.lse2 = lse == -INFINITY ? INFINITY : lse * kLog2e;
    x.limit = lse == -INFINITY ? 0 : min(end, see + i_q);
  };
  float total[KT][16];
#pragma unroll
  for (int k = 0; k < KT; ++k)
#pragma unroll
    for (int i = 0; i < 16; ++i) total[k][i] = 0.f;
  auto add = [&](const Queries &y) {
    f32x16 x[KT];
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      x[k] = f32x16{};
#pragma unroll
      for (int c = 0; c < C; ++c) x[k] = mfma32(key[k][c], y.q[c], x[k], H{});
    }
    float factor = p.scale2, lse2 = y.lse2;
    if (__any(fabsf(y.lse2) >= kRounded && y.lse2 != INFINITY)) {
#pragma unroll
      for (int k = 0; k < KT; ++k)
#pragma unroll
        for (int i = 0; i < 16; ++i) x[k][i] = below_one(x[k][i] * p.scale2 - y.lse2);
      factor = 1.f;
      lse2 = 0.f;
    }
    if (~ok != 0 || !__all(y.limit >= begin + kWeighKeys)) {
      const uint64_t mine = ok >> (4 * half);
#pragma unroll
      for (int k = 0; k < KT; ++k)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int j = 32 * k + 8 * (i / 4) + i % 4;
          const bool sees = (mine >> j & 1) != 0 && begin + j + 4 * half < y.limit;
          total[k][i] += sees ? __builtin_amdgcn_exp2f(__builtin_fmaf(x[k][i], factor, -lse2)) : 0.f;
        }
    } else {
#pragma unroll
      for (int k = 0; k < KT; ++k)
#pragma unroll
        for (int i = 0; i < 16; ++i) total[k][i] += __builtin_amdgcn_exp2f(__builtin_fmaf(x[k][i], factor, -lse2));
    }
  };
  // queries before the first key see none of them
  const int64_t before = (int64_t)max(0, begin - see + 1) * p.group;
  constexpr int kStride = 32 * kPerGroup<D>;
  int m0 = (int)min(before, (int64_t)rows) / 32 * 32 + 32 * wave;
  Queries a, b;
  if (m0 < rows) fetch(a, m0);
  while (m0 < rows) {
    if (m0 + kStride < rows) fetch(b, m0 + kStride);
    add(a);
    m0 += kStride;
    if (m0 >= rows) break;
    if (m0 + kStride < rows) fetch(a, m0 + kStride);
    add(b);
    m0 += kStride;
  }
#pragma unroll
  for (int k = 0; k < KT; ++k)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = total[k][i];
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) v += shfl_xor(v, d);
      if (n == i) s_total[wave][32 * k + 8 * (i / 4) + 4 * half + i % 4] = v;
    }
  __syncthreads();
  if (threadIdx.x >= kWeighKeys || at >= end) return;
  float v = 0.f;
#pragma unroll
  for (int w = 0; w < kPerGroup<D>; ++w) v += s_total[w][lane];
  float *out = p.scores + (int64_t)row * p.sc_row + (int64_t)head * p.sc_head;
  out[at] = p.decay * out[at] + v;
}

template <class T, int D>
int launch_weigh(const Params &p, hipStream_t stream) {
  const int pieces = (int)ceil_div((int64_t)p.width * p.block_size, kWeighKeys);
  hipLaunchKernelGGL((weigh_wide_kernel<T, D>), dim3((unsigned)((int64_t)p.rows * pieces * p.kv_heads)),
                     dim3(kPerGroup<D> * kWave), 0, stream, p, pieces);
  return check_hip(hipGetLastError(), "ekv_prefix_attention weights launch");
}

template <class T, int D>
int launch_wide(const Params &p, bool own, hipStream_t stream) {
  if (own)
    hipLaunchKernelGGL((wide_kernel<T, D>), dim3((unsigned)p.items_own), dim3(Wide<T, D>::kThreads), 0, stream, p);
  else
    hipLaunchKernelGGL((wide_prefix_kernel<T, D>), dim3((unsigned)(p.kv_heads * p.share_pre)), dim3(Wide<T, D>::kThreads),
                       0, stream, p);
  return check_hip(hipGetLastError(), "ekv_prefix_attention wide launch");
}

template <class T>
int weigh_dim(const Params &p, int head_dim, hipStream_t stream) {
  switch (head_dim) {
    case 32: return launch_weigh<T, 32>(p, stream);
    case 64: return launch_weigh<T, 64>(p, stream);
    case 128: return launch_weigh<T, 128>(p, stream);
    default: return launch_weigh<T, 256>(p, stream);
  }
}

template <class T>
int wide_dim(const Params &p, int head_dim, bool own, hipStream_t stream) {
  switch (head_dim) {
    case 32: return launch_wide<T, 32>(p, own, stream);
    case 64: return launch_wide<T, 64>(p, own, stream);
    case 128: return launch_wide<T, 128>(p, own, stream);
    default: return launch_wide<T, 256>(p, own, stream);
  }
}

int wide_resident(int head_dim) { return head_dim == 256 ? 1 : 2; }

int wide_tile_rows() { return Wide<BF16, 128>::kWaves * 32; }

int wide_attention(const Params &p, int kv_dtype, int head_dim, bool own, hipStream_t stream) {
  switch (kv_dtype) {
    case EKV_F16: return wide_dim<F16>(p, head_dim, own, stream);
    case EKV_BF16: return wide_dim<BF16>(p, head_dim, own, stream);
    default: return wide_dim<FP8>(p, head_dim, own, stream);
  }
}

int wide_weights(const Params &p, int kv_dtype, int head_dim, hipStream_t stream) {
  switch (kv_dtype) {
    case EKV_F16: return weigh_dim<F16>(p, head_dim, stream);
    case EKV_BF16: return weigh_dim<BF16>(p, head_dim, stream);
    default: return weigh_dim<FP8>(p, head_dim, stream);
  }
}

}  // namespace attn
}  // namespace ekv
