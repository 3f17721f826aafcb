// Attention over the paged cache for a batch whose rows share prefixes, and the running attention weight
// of each cached token.
//
//   s_qj = scale * k_scale * <q, k_j>            over the keys j that query q sees
//   out_q = v_scale * sum_j exp(s_qj - lse_q) v_j,   lse_q = log sum_j exp(s_qj)
//   scores[row, head, j] = decay * scores[row, head, j] + sum_{q of the row and head} exp(s_qj - lse_q)
//
// A query sees the whole prefix of its row's group and its row's own keys up to itself.  The keys are cut
// into pieces; a piece leaves its maximum, sum and unnormalised output for each of its query rows, which
// combine_kernel joins:
//   m = max_c m_c,  l = sum_c l_c 2^(m_c - m),  out = sum_c o_c 2^(m_c - m) / l.
// A prefix is read once per tile of its group's query rows and not once per row, unless the rows' own tiles are as few
// or joining costs more (pays_together).
#include "ekv_attention.hpp"

namespace ekv {
namespace attn {

// What one wave works on.
struct Segment : Range {
  int first, rows;  // first token, query rows (tokens * group)
  int m0;           // the tile's first query row
  int row, slot;    // the batch row (own keys; -1: a prefix), the slot of the partial results
  int see;          // query token i sees own keys below see + i, and a prefix's all
};

__device__ __forceinline__ bool prefix_segment(const Params &p, uint32_t item, Segment &s) {
  s.head = (int)(item % p.kv_heads);
  item /= p.kv_heads;
  const int chunk = (int)(item % p.s_pre);
  int g, tile;
  if (!find_tile(p.groups, (int)(item / p.s_pre), [&](int e) { return (int)ceil_div((int64_t)group_queries(p, e).count * p.group, kRowsPerTile); }, g, tile))
    return false;
  const RowQueries t = group_queries(p, g);
  s.table = p.ptable + (int64_t)g * p.ptable_stride;
  s.ptable = nullptr;
  s.plen = s.own = 0;
  s.row = -1;
  s.first = t.first;
  s.rows = t.count * p.group;
  s.m0 = tile * kRowsPerTile;
  s.slot = p.s_own + chunk;
  const int64_t begin = (int64_t)chunk * p.chunk_pre;
  s.end = (int)min(begin + p.chunk_pre, (int64_t)group_length(p, g));
  s.begin = (int)min(begin, (int64_t)INT32_MAX);
  return s.begin < s.end;
}

// The shapes of one instance: one wave's step of about 8 KB (fp8) or 16 KB of keys and values on their way while
// the step before is worked on, so that the 8 waves of a compute unit have 64 to 128 KB in flight.
template <class T, int D>
struct Narrow {
  static constexpr int kRow = Lds<T, D>::kRow;
  static constexpr int kKeys = std::is_same<T, F32>::value ? (D <= 64 ? 32 : 16) : (D <= 64 ? 64 : 32);
  typedef Stage<T, D, kKeys, kWave> Step;
  static constexpr int kBytes = 2 * Step::kTile;  // LDS of a wave
  static constexpr int kWaves = kBytes > 16384 ? 2 : 4;
  static constexpr int kThreads = kWaves * kWave;
  // waves of a compute unit: as many as LDS has room for, 2 a SIMD (1 at head dim 256) at most for their registers
  static constexpr int kFit = 163840 / (kWaves * kBytes + 1024) * kWaves;
  static constexpr int kResident = kFit < (D == 256 ? 4 : 8) ? kFit : (D == 256 ? 4 : 8);
  static constexpr int kPieceDims = D >= 64 ? 4 : 2;  // float32: dims of a value row that a lane reads at once
};

// One wave per item.  S^T = K Q^T on the matrix cores leaves each lane the logits of four keys (4g + i of each 16,
// in lane group g) of one query row.  O^T = V^T P^T takes as its P operand what the lane already holds, its weights
// rounded to 16 bits (half a step of the type, relative: the size of the output's own rounding; float32 caches keep
// float32 weights), and as its V operand the same keys' values by the transposing LDS read, so no weight moves
// between lanes.  The LDS is the wave's own: nothing waits for another wave.
template <class T, int D>
__device__ __forceinline__ void attend(const Params &p, const Segment &s, char *lds) {
  using N = Narrow<T, D>;
  using L = Lds<T, D>;
  constexpr int E = sizeof(typename T::Query), KT = N::kKeys / 16, QP = N::kRow / 64;
  const int lane = lane_id(), g = lane / 16, n = lane % 16;
  const int m = s.m0 + n;
  const bool live = m < s.rows;
  const int i_q = live ? m / p.group : 0;
  const int token = s.first + i_q, q_head = s.head * p.group + (live ? m - i_q * p.group : 0);
  const bool own = s.row >= 0;
  const int limit = !live ? 0 : own ? min(s.end, s.see + i_q) : s.end;  // this lane's query sees keys below it
  const int every = own ? min(s.end, s.see + s.m0 / p.group) : s.end;   // and every query of the tile keys below this

  typedef typename N::Step St;
  int page = s.begin < s.end ? St::look(p, s, s.begin) : -1;
  u32x4 q[QP];
#pragma unroll
  for (int c = 0; c < QP; ++c) {
    q[c] = u32x4{0, 0, 0, 0};
    if (live)
      q[c] = *as_global((const u32x4 *)(p.q + ((int64_t)token * p.q_st + (int64_t)q_head * p.q_sh) * E + (4 * c + g) * 16));
  }
  typename St::Rows keys, vals;
  uint64_t coming = 0;  // the keys of the step on its way that are there
  if (s.begin < s.end) {
    coming = St::there(p, page);
    const int64_t place = St::place(p, s, s.begin, page);
    St::load(p, place, p.k, keys);
    St::load(p, place, p.v, vals);
    page = St::look(p, s, s.begin + N::kKeys);
  }

  int key_off[QP];
#pragma unroll
  for (int c = 0; c < QP; ++c) key_off[c] = L::key_at(n, 4 * c + g);
  const char *values = lds + St::kTile;
  float *logits = nullptr;  // of this lane's query row
  if (p.logits != nullptr && own && live)
    logits = p.logits + (((int64_t)s.row * p.kv_heads + s.head) * p.logit_rows + m) * p.logit_stride;

  f32x4 acc[D / 16];
#pragma unroll
  for (int d = 0; d < D / 16; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  float top = -INFINITY, sum = 0.f;

  for (int base = s.begin; base < s.end; base += N::kKeys) {
    const uint64_t ok = coming;
    St::store_keys(keys, lds);
    St::store_values(vals, ok, lds + St::kTile);
    asm volatile("" ::: "memory");  // the lanes of the wave read what others wrote, in order
    if (base + N::kKeys < s.end) {
      coming = St::there(p, page);
      const int64_t place = St::place(p, s, base + N::kKeys, page);
      St::load(p, place, p.k, keys);
      St::load(p, place, p.v, vals);
      page = St::look(p, s, base + 2 * N::kKeys);
    }
    f32x4 x[KT];
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      x[k] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < QP; ++c) x[k] = dot_piece<T>(*(const u32x4 *)(lds + key_off[c] + k * 16 * N::kRow), q[c], x[k]);
      x[k] *= p.scale2;
    }
    if (base + N::kKeys > every || ~ok != 0) {
      const uint64_t mine = ok >> (4 * g);
#pragma unroll
      for (int k = 0; k < KT; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!(mine >> (16 * k + i) & 1) || base + 16 * k + 4 * g + i >= limit) x[k][i] = -INFINITY;
    }
    if (logits != nullptr) {
#pragma unroll
      for (int k = 0; k < KT; ++k)
        if (base + 16 * k + 4 * g < s.end) *(f32x4 *)(logits + base + 16 * k + 4 * g) = x[k];
    }
    float high = x[0][0];
#pragma unroll
    for (int k = 0; k < KT; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) high = fmaxf(high, x[k][i]);
    const float peak = fmaxf(top, lifted<typename T::Half>(rows_max(high), kLift<typename T::Half>));
    const float ref = peak == -INFINITY ? 0.f : peak;
    if (!__all(top == peak)) {
      const float shrink = __builtin_amdgcn_exp2f(top - ref);
      sum *= shrink;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) acc[d] *= shrink;
    }
    top = peak;
#pragma unroll
    for (int k = 0; k < KT; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[k][i] = __builtin_amdgcn_exp2f(x[k][i] - ref);
        sum += x[k][i];
      }
    if constexpr (std::is_same<T, F32>::value) {
      constexpr int PD = N::kPieceDims;
      typedef float Piece __attribute__((ext_vector_type(PD)));
#pragma unroll
      for (int k = 0; k < KT; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int c = 0; c < D / 16 / PD; ++c) {
            const Piece v = *(const Piece *)(values + L::value_at(16 * k + 4 * g + i, (c * 16 + n) * PD * 4));
#pragma unroll
            for (int j = 0; j < PD; ++j)
              acc[c * PD + j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[j], x[k][i], acc[c * PD + j], 0, 0, 0);
          }
    } else {
      typedef typename T::Half H;
#pragma unroll
      for (int k = 0; k < KT; k += 2) {
        const u32x4 w = {pack2(x[k][0], x[k][1], H{}), pack2(x[k][2], x[k][3], H{}), pack2(x[k + 1][0], x[k + 1][1], H{}),
                         pack2(x[k + 1][2], x[k + 1][3], H{})};
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          const char *from = values + L::value_at(4 * g + n / 4, d * 32 + n % 4 * 8) + k * 16 * N::kRow;
          const u32x2 v = read_transposed(from), u = read_transposed(from + 16 * N::kRow);
          acc[d] = mfma16(u32x4{v[0], v[1], u[0], u[1]}, w, acc[d], H{});
        }
      }
    }
    asm volatile("" ::: "memory");  // the next step overwrites what this one read
  }

  sum = rows_sum(sum);
  if (!live) return;
  const int64_t at = ((int64_t)s.slot * p.tokens + token) * p.q_heads + q_head;
  if (g == 0) p.part_ml[at] = make_float2(top, sum);
  float *o = p.part_o + at * D;
  if constexpr (std::is_same<T, F32>::value) {
    constexpr int PD = N::kPieceDims;
#pragma unroll
    for (int c = 0; c < D / 16 / PD; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int j = 0; j < PD; ++j) o[c * 16 * PD + (4 * g + e) * PD + j] = acc[c * PD + j][e];
  } else {
#pragma unroll
    for (int d = 0; d < D / 16; ++d) *(f32x4 *)(o + 16 * d + 4 * g) = acc[d];
  }
}

constexpr int kThreads = 256;

// The own keys of a decode step stream at the rate that memory has only if every wave has the same share of them to
// the end: rows have lengths that the host does not know, and items of a fixed length left the last ones running
// alone (128 rows of 512 to 8192 tokens: 427 us in chunks of 256 or 1024 keys against 358 us, 6.4 TB/s).  So the steps of
// all rows, one row after the other, are one list; each (KV head, query tile) has `share` waves, and wave j of them
// takes steps j T / share to (j + 1) T / share of the T, in at most kMaxSlots pieces a row.
template <class T, int D>
__global__ __launch_bounds__((Narrow<T, D>::kThreads), (D == 256 ? 1 : 2)) void narrow_kernel(const Params p) {
  using N = Narrow<T, D>;
  __shared__ __attribute__((aligned(16))) char lds[N::kWaves * N::kBytes];
  __shared__ int s_row[N::kWaves];
  __shared__ int64_t s_at[N::kWaves];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  char *mine = lds + wave * N::kBytes;
  const int64_t shared = ceil_div(p.items_pre, N::kWaves);  // the prefixes' items come first
  Segment s;
  if (blockIdx.x < shared) {
    const int64_t item = (int64_t)blockIdx.x * N::kWaves + wave;
    if (item < p.items_pre && prefix_segment(p, (uint32_t)item, s)) attend<T, D>(p, s, mine);
    return;
  }
  const int64_t first = (blockIdx.x - shared) * N::kWaves;
  const int each = p.kv_heads * p.tiles_own;
  const Share share = share_out<N::kWaves, N::kWaves>(
      p.rows, p.share, 1, p.s_own, [&](int w) { return (first + w) / each; },
      [&](int r, int64_t &steps) {
        steps = (row_length(p, r) + N::kKeys - 1) / N::kKeys;
        return steps;
      }, s_row, s_at);
  const int j = (int)((first + wave) / each), part = (int)((first + wave) % each);
  if (j >= share.share) return;
  s.head = part % p.kv_heads;
  s.m0 = part / p.kv_heads * kRowsPerTile;
  s.ptable = nullptr;
  s.plen = s.own = 0;
  int64_t at = (int64_t)j * share.total / share.share;
  const int64_t stop = (int64_t)(j + 1) * share.total / share.share;
  s.row = uniform(s_row[wave]);
  int64_t row_at = uniform(s_at[wave]);  // the units before the row
  while (true) {
    const int len = uniform(row_length(p, s.row)), units = (len + N::kKeys - 1) / N::kKeys;
    if (units > 0) {
      const int j0 = share.worker_of(row_at), j1 = share.worker_of(row_at + units - 1);
      if (part == 0 && j == j0 && lane_id() == 0) p.row_slots[s.row] = j1 - j0 + 1;
      const RowQueries t = row_queries(p, s.row);
      s.table = p.table + (int64_t)s.row * p.table_stride;
      s.first = uniform(t.first);
      s.rows = uniform(min(t.count, p.max_query) * p.group);
      s.see = uniform(len - t.count + 1);
      s.slot = j - j0;
      const int u0 = (int)(at - row_at), u1 = (int)(min(stop, row_at + units) - row_at);
      s.begin = u0 * N::kKeys;
      if (s.m0 < s.rows) {
        const int last = (min(s.m0 + kRowsPerTile, s.rows) - 1) / p.group;
        s.end = (int)min((int64_t)u1 * N::kKeys, (int64_t)min(len, s.see + last));  // may be before s.begin: the partial result is empty
        attend<T, D>(p, s, mine);
      }
      at = row_at + u1;
      row_at += units;
    }
    if (at >= stop) break;
    ++s.row;
  }
}

// -- joining the chunks ---------------------------------------------------------------------------------

// The row of a token: the last one whose first token is <= it.
__device__ __forceinline__ int row_of(const Params &p, int token) {
  if (p.q_start == nullptr) return token;
  int lo = 0, hi = p.rows;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.q_start[mid] <= token) lo = mid;
    else hi = mid;
  }
  return lo;
}
// W waves per (token, query head), each with a share of the slots: lane t weighs slot t of 64, then the slots'
// outputs are summed in slot order, and the waves' sums in wave order.  Few queries (one row of 8192 tokens has 32
// of 254 slots) are a matter of latency and take 8 waves each; many have few slots each and take one (128 rows of
// 32 heads: 4.7 us, where 4 waves took 9.2).
template <class Q, int D, int W>
__global__ __launch_bounds__(W == 1 ? kThreads : W *kWave) void combine_kernel(const Params p) {
  constexpr int kWaves = W == 1 ? kThreads / kWave : W;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t item = ((int64_t)blockIdx.x * kWaves + wave) / W;
  const int part = wave % W;
  if (item >= (int64_t)p.tokens * p.q_heads) return;  // W > 1: the whole workgroup
  const int lane = lane_id();
  const int token = (int)(item / p.q_heads), q_head = (int)(item - (int64_t)token * p.q_heads);
  const int row = row_of(p, token);
  const RowQueries t = row_queries(p, row);
  const int i_q = token - t.first;
  int own = 0, pre = 0;  // slots written for this query
  if (i_q >= 0 && i_q < min(t.count, p.max_query)) {
    const int len = row_length(p, row);
    const int seen = min(len, len - t.count + 1 + i_q);
    const int g = group_of(p, row);
    const int n = g >= 0 ? group_length(p, g) : 0;
    if (p.wide_own) {
      const int ahead = p.wide_pre ? 0 : n;  // keys before the own ones on their axis
      const int64_t all = seen > 0 ? (int64_t)own_begin(ahead) + seen : ahead;
      own = all > 0 ? (int)((all - 1) / p.chunk_own) + 1 : 0;
    } else {
      own = seen > 0 ? p.row_slots[row] : 0;
    }
    if (n > 0 && p.wide_pre) pre = p.pre_slots[(int64_t)token * p.group + q_head % p.group];
    else if (n > 0 && !p.wide_own) pre = (n - 1) / p.chunk_pre + 1;
  }
  constexpr int kPer = D > 64 ? D / 64 : 1;
  constexpr int kLanes = D / kPer;
  constexpr int kFlight = W == 1 ? 8 : 16;
  typedef float Piece __attribute__((ext_vector_type(kPer)));
  Piece acc = {};
  float top = -INFINITY, sum = 0.f;
  const int64_t plane = (int64_t)p.tokens * p.q_heads;
  const int each = (own + pre + W - 1) / W;
  const int end = min((part + 1) * each, own + pre);
  auto slot = [&](int k) { return k < own ? k : p.s_own + k - own; };
  for (int k0 = part * each; k0 < end; k0 += kWave) {
    const int n = min(end - k0, kWave);
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < n) ml = p.part_ml[(int64_t)slot(k0 + lane) * plane + item];
    const float peak = fmaxf(top, wave_max(ml.x));
    const float ref = peak == -INFINITY ? 0.f : peak;
    const float shrink = __builtin_amdgcn_exp2f(top - ref);
    const float w = ml.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml.x - ref);
    sum = sum * shrink + wave_sum(ml.y * w);
    acc *= shrink;
    top = peak;
    const float *o = p.part_o + item * D + (lane % kLanes) * kPer;
    // past the last slot the weight is 0 and the last slot is read again
    for (int k = 0; k < n; k += kFlight) {
      Piece x[kFlight];
#pragma unroll
      for (int u = 0; u < kFlight; ++u) x[u] = *(const Piece *)(o + (int64_t)slot(k0 + min(k + u, n - 1)) * plane * D);
#pragma unroll
      for (int u = 0; u < kFlight; ++u)
        acc += __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), k + u)) * x[u];
    }
  }
  if constexpr (W > 1) {
    __shared__ float s_top[W], s_sum[W];
    __shared__ Piece s_acc[W][kLanes];
    if (lane < kLanes) s_acc[part][lane] = acc;
    s_top[part] = top;
    s_sum[part] = sum;
    __syncthreads();
    if (part != 0) return;
#pragma unroll
    for (int w = 1; w < W; ++w) {
      const float peak = fmaxf(top, s_top[w]);
      const float ref = peak == -INFINITY ? 0.f : peak;
      const float a = __builtin_amdgcn_exp2f(top - ref), b = __builtin_amdgcn_exp2f(s_top[w] - ref);
      sum = sum * a + s_sum[w] * b;
      acc = acc * a + s_acc[w][lane % kLanes] * b;
      top = peak;
    }
  }
  // no key seen, or none with any weight: the sum is empty
  const bool none = sum == 0.f;
  const float inv = none ? 0.f : p.v_scale / sum;
  if (lane < kLanes) {
    Q *o = (Q *)p.out + (int64_t)token * p.o_st + (int64_t)q_head * p.o_sh + lane * kPer;
#pragma unroll
    for (int j = 0; j < kPer; ++j) o[j] = (Q)(none ? 0.f : acc[j] * inv);
  }
  if (lane == 0) p.lse[item] = none ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

// -- the running weights ------------------------------------------------------------------------------

// The logits were kept: a thread per four keys of a (row, KV head).
template <int THREADS>
__global__ __launch_bounds__(THREADS) void fold_kernel(const Params p, int pieces) {
  const uint32_t block = blockIdx.x;
  const int head = (int)(block % p.kv_heads), row = (int)(block / p.kv_heads / pieces);
  const int key = ((int)(block / p.kv_heads % pieces) * THREADS + threadIdx.x) * 4;
  const int len = row_length(p, row);
  if (key >= len) return;
  const RowQueries t = row_queries(p, row);
  const int see = len - t.count + 1, rows = min(t.count, p.max_query) * p.group;
  const float *logits = p.logits + ((int64_t)row * p.kv_heads + head) * p.logit_rows * p.logit_stride + key;
  float total[4] = {0.f, 0.f, 0.f, 0.f};
  for (int m = 0; m < rows; ++m) {
    const int i_q = m / p.group;
    const float lse = p.lse[(int64_t)(t.first + i_q) * p.q_heads + head * p.group + (m - i_q * p.group)];
    if (lse == -INFINITY || key >= see + i_q) continue;  // it sees none of them (nor wrote their logits)
    const f32x4 x = *(const f32x4 *)(logits + (int64_t)m * p.logit_stride);
#pragma unroll
    for (int i = 0; i < 4; ++i)  // unseen ones are -inf, and get nothing from a query of NaN either
      total[i] += x[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(below_one(x[i] - lse * kLog2e));
  }
  float *out = p.scores + (int64_t)row * p.sc_row + (int64_t)head * p.sc_head;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (key + i < len) out[key + i] = p.decay * out[key + i] + total[i];
}

// The logits again: one wave per (row, KV head, 64 keys), the logits of every query row against them, their weights
// exp(s - lse) summed over the query rows in one order, and one addition to each key's running score.
constexpr int kWeighKeys = 64;

template <class T, int D>
__global__ __launch_bounds__(kThreads) void weigh_kernel(const Params p, int pieces) {
  constexpr int E = sizeof(typename T::Query), KT = kWeighKeys / 16, QP = Lds<T, D>::kRow / 64;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  int64_t item = (int64_t)blockIdx.x * (kThreads / kWave) + wave;
  if (item >= (int64_t)p.rows * pieces * p.kv_heads) return;
  const int head = (int)(item % p.kv_heads);
  item /= p.kv_heads;
  const int row = (int)(item / pieces), begin = (int)(item % pieces) * kWeighKeys;
  const int len = row_length(p, row), end = min(begin + kWeighKeys, len);
  if (begin >= end) return;
  const int32_t *table = p.table + (int64_t)row * p.table_stride;
  const RowQueries t = row_queries(p, row);
  const int see = len - t.count + 1, rows = min(t.count, p.max_query) * p.group;
  const int lane = lane_id(), g = lane / 16, n = lane % 16;
  const int mine = min(begin + lane, end - 1);
  const int page_mine = table[page_of(p, mine)];
  const uint64_t ok = __ballot((uint32_t)page_mine < (uint64_t)p.blocks) >> (4 * g);
  // the key rows' pieces 4c + g, read where they lie: 64 bytes of 16 rows a load
  u32x4 key[KT][QP];
#pragma unroll
  for (int k = 0; k < KT; ++k) {
    const int pos = min(begin + 16 * k + n, end - 1);
    int page = __shfl(page_mine, 16 * k + n);
    if ((uint32_t)page >= (uint64_t)p.blocks) page = 0;
    const char *from = p.k + ((int64_t)page * p.st_block + (int64_t)(pos - page_of(p, pos) * p.block_size) * p.st_pos +
                              (int64_t)head * p.st_head) * T::kBytes;
#pragma unroll
    for (int c = 0; c < QP; ++c) {
      if constexpr (T::kBytes == 1) {
        const u32x2 x = *as_global((const u32x2 *)(from + (4 * c + g) * 8));
        key[k][c] = widen(x[0], x[1]);
      } else {
        key[k][c] = *as_global((const u32x4 *)(from + (4 * c + g) * 16));
      }
    }
  }
  float total[KT][4];
#pragma unroll
  for (int k = 0; k < KT; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) total[k][i] = 0.f;
  // queries before the first key see none of them
  const int64_t before = (int64_t)max(0, begin - see + 1) * p.group;
  for (int m0 = (int)min(before, (int64_t)rows) / kRowsPerTile * kRowsPerTile; m0 < rows; m0 += kRowsPerTile) {
    const int m = m0 + n;
    const bool live = m < rows;
    const int i_q = live ? m / p.group : 0;
    const int token = t.first + i_q, q_head = head * p.group + (live ? m - i_q * p.group : 0);
    u32x4 q[QP];
#pragma unroll
    for (int c = 0; c < QP; ++c) {
      q[c] = u32x4{0, 0, 0, 0};
      if (live)
        q[c] = *as_global((const u32x4 *)(p.q + ((int64_t)token * p.q_st + (int64_t)q_head * p.q_sh) * E + (4 * c + g) * 16));
    }
    const float lse = live ? p.lse[(int64_t)token * p.q_heads + q_head] : -INFINITY;
    const float lse2 = lse * kLog2e;
    const int limit = lse == -INFINITY ? 0 : min(end, see + i_q);
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < QP; ++c) x = dot_piece<T>(key[k][c], q[c], x);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool sees = (ok >> (16 * k + i) & 1) != 0 && begin + 16 * k + 4 * g + i < limit;
        total[k][i] += sees ? __builtin_amdgcn_exp2f(below_one(x[i] * p.scale2 - lse2)) : 0.f;
      }
    }
  }
  float *out = p.scores + (int64_t)row * p.sc_row + (int64_t)head * p.sc_head;
#pragma unroll
  for (int k = 0; k < KT; ++k) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float v = total[k][i];
#pragma unroll
      for (int d = 1; d < 16; d <<= 1) v += shfl_xor(v, d);
      const int pos = begin + 16 * k + 4 * g + i;
      if (n == i && pos < end) out[pos] = p.decay * out[pos] + v;
    }
  }
}

// -- the launches ---------------------------------------------------------------------------------------

// How a prefix's keys are cut where the narrow kernel reads them: so that the items fill the chip several times
// over, but no chunk is shorter than 64 keys, and the partial outputs stay below 256 MB.
void split(int64_t keys, int64_t items_per_chunk, int64_t queries, int head_dim, int &chunk, int &slots) {
  const int64_t target = 32 * (int64_t)cu_count();
  int64_t n = ceil_div(target, items_per_chunk > 0 ? items_per_chunk : 1);
  n = n < ceil_div(keys, 1024) ? ceil_div(keys, 1024) : n;
  const int64_t fit = (256ll << 20) / ((queries > 0 ? queries : 1) * (head_dim * 4 + 8));
  n = n > fit ? fit : n;
  n = n > kMaxChunks ? kMaxChunks : n < 1 ? 1 : n;
  chunk = (int)(ceil_div(ceil_div(keys, n), 64) * 64);
  if (chunk < 64) chunk = 64;
  slots = (int)ceil_div(keys, chunk);
  if (slots < 1) slots = 1;
}

// The wide kernel's: a few workgroups for each that the chip holds, no chunk shorter than 512 keys (its
// partial outputs, written and read again, are as much traffic as 64 keys and values).
void split_wide(int64_t keys, int64_t items_per_chunk, int64_t queries, int head_dim, int &chunk, int &slots) {
  int64_t n = ceil_div(2 * (int64_t)cu_count(), items_per_chunk > 0 ? items_per_chunk : 1);
  const int64_t fit = (256ll << 20) / ((queries > 0 ? queries : 1) * (head_dim * 4 + 8));
  n = n > fit ? fit : n;
  n = n > kMaxChunks ? kMaxChunks : n < 1 ? 1 : n;
  const int64_t each = ceil_div(ceil_div(keys, n), 64) * 64;
  chunk = (int)(each < 512 ? 512 : each > (1 << 30) ? INT32_MAX : each);
  slots = (int)ceil_div(keys, chunk);
  if (slots < 1) slots = 1;
}

// The narrow kernel's resident waves of a compute unit and keys of a step.
struct Shape {
  int waves, keys;
};
template <class T>
Shape narrow_shape(int head_dim) {
  auto of = [](auto n) { return Shape{decltype(n)::kResident, decltype(n)::kKeys}; };
  return head_dim == 32 ? of(Narrow<T, 32>{}) : head_dim == 64 ? of(Narrow<T, 64>{})
         : head_dim == 128 ? of(Narrow<T, 128>{}) : of(Narrow<T, 256>{});
}
Shape narrow_shape(int kv_dtype, int head_dim) {
  return kv_dtype == EKV_F32 ? narrow_shape<F32>(head_dim) : kv_dtype == EKV_FP8_E4M3 ? narrow_shape<FP8>(head_dim)
                                                                                     : narrow_shape<BF16>(head_dim);
}

// Where the wide kernel takes the own keys: whether the prefixes are read for all queries of a group together, as for
// fewer query rows, and joined to the own keys' results.  Else each of the rows' `alone` tiles walks its prefix by itself,
// ahead of its own keys, with nothing to join: the better way where rows fill their tiles (a prompt chunk each) or the
// prefix is short.  Told apart by what the two cost the chip: a key and its value 26, 30, 38 or 108 ps a tile at head dims
// 32 to 256, a partial result its bytes written and read at 4 TB/s, the launches more 12 us.  Measured, a walk for each
// tile against together, 8 KV heads of 128, 4 query heads each: 200 rows of 5 queries behind two prefixes of 32768 tokens
// 3652 against 793 us, of 8 queries 3675 against 1432; 128 rows of 5, 8, 16, 20, 24 and 32 queries behind 8192 tokens 476,
// 482, 539, 574, 578 and 656 against 209, 267, 434, 520, 603 and 776, of 5 behind 1024 tokens 122 against 129; 2048 queries
// among 127 single tokens behind 8192, 2048 and 256 tokens 814, 299 and 138 against 491, 269 and 208.
bool pays_together(const Params &p, int head_dim, int64_t alone) {
  const int64_t together = ceil_div((int64_t)p.tokens * p.group, wide_tile_rows()) + p.groups;
  const int64_t workers = (int64_t)cu_count() * wide_resident(head_dim) / p.kv_heads;
  const double slots = 2.0 + (double)workers / together;
  const double key = (22.0 + head_dim / 8.0) * 2 / wide_resident(head_dim) * 1e-3;  // ns
  const double saved = (double)(alone - together) * p.kv_heads * p.pwidth * p.block_size * key;
  const double join = 12000.0 + (double)p.tokens * p.q_heads * slots * (head_dim * 4 + 8) / 2000.0;
  return saved > join;
}

void plan(Params &p, int head_dim, int kv_dtype) {
  p.whole = p.block_size % 16 == 0 && p.st_pos >= 0 && p.st_pos < 1 << 24;
  const int64_t queries = (int64_t)p.tokens * p.q_heads;
  const int64_t own_rows = (int64_t)p.max_query * p.group;
  const bool half = kv_dtype != EKV_F32;
  const int64_t axis = (int64_t)(p.width + (p.groups > 0 ? p.pwidth : 0)) * p.block_size + 64;
  const int least = head_dim == 256 ? kWideRows256 : kWideRows;
  p.wide_own = half && own_rows >= least && axis < (1 << 30);
  p.tile_own = p.wide_own ? wide_tile_rows() : kRowsPerTile;
  p.tiles_own = (int)ceil_div(own_rows, p.tile_own);
  const int64_t own_keys = (int64_t)p.width * p.block_size, prefix_keys = p.groups > 0 ? (int64_t)p.pwidth * p.block_size : 0;
  // Rows of different query counts (a prompt chunk among single tokens): the tiles there can be in all, found by a search
  // over the rows, where every row's most would be over twice as many.  (2048 queries among 63 single tokens of long rows:
  // 286 us, 541 us with a workgroup for every row's most; among 255 of short rows 425 against 1001.)
  const int64_t tiles_most = (int64_t)p.rows * p.tiles_own, tiles_all = ceil_div((int64_t)p.tokens * p.group, p.tile_own) + p.rows;
  p.packed = p.wide_own && tiles_most > 2 * tiles_all;
  const int64_t own_items = (p.packed ? tiles_all : tiles_most) * p.kv_heads;
  if (p.wide_own)
    p.wide_pre = p.groups > 0 && pays_together(p, head_dim, tiles_most < tiles_all ? tiles_most : tiles_all);
  else
    p.wide_pre = half && p.groups > 0 && (int64_t)p.tokens * p.group / p.groups >= least;
  p.tile_pre = p.wide_pre ? wide_tile_rows() : kRowsPerTile;
  p.items_pre = 0;
  p.s_pre = 0;
  p.chunk_pre = 64;
  const int64_t fit = (256ll << 20) / ((queries > 0 ? queries : 1) * (head_dim * 4 + 8));  // partial results of 256 MB
  if (p.wide_own) {
    split_wide((p.wide_pre ? 0 : own_begin(prefix_keys)) + own_keys, own_items, queries, head_dim, p.chunk_own, p.s_own);
  } else {
    // waves that a (KV head, tile) has: all together those that the chip holds, and no more than there are steps
    const Shape shape = narrow_shape(kv_dtype, head_dim);
    const int64_t each = (int64_t)p.kv_heads * p.tiles_own, row_steps = ceil_div(own_keys, shape.keys);
    int64_t share = (int64_t)cu_count() * shape.waves / each;
    share = share > p.rows * row_steps ? p.rows * row_steps : share;
    p.share = (int)(share < 1 ? 1 : share);
    int64_t slots = row_steps + 2;
    slots = slots > fit ? fit : slots;
    p.s_own = (int)(slots > kMaxSlots ? kMaxSlots : slots < 3 ? 3 : slots);
    p.waves_own = each * p.share;
  }
  if (p.wide_pre) {
    // workgroups that a KV head has: all together those that the chip holds
    const int64_t groups = (int64_t)cu_count() * wide_resident(head_dim) / p.kv_heads;
    p.share_pre = (int)(groups < 1 ? 1 : groups);
    const int64_t most = ceil_div(prefix_keys, 32) + 2;
    const int64_t limit = most > fit ? fit : most;
    p.s_pre = (int)(limit > kMaxChunks ? kMaxChunks : limit < 3 ? 3 : limit);
  } else if (p.groups > 0 && !p.wide_own) {
    p.tiles_pre = (int)(ceil_div((int64_t)p.tokens * p.group, p.tile_pre) + p.groups);
    const int64_t items = (int64_t)p.kv_heads * p.tiles_pre;
    split(prefix_keys, items, queries, head_dim, p.chunk_pre, p.s_pre);
    p.items_pre = items * p.s_pre;
  }
  p.items_own = p.wide_own ? own_items * p.s_own : 0;
  // The logits of a decode step's few query rows are kept (4 bytes each, written and read, against the key read
  // again) where they stay below a gigabyte and fold_kernel's launch below 2^32 threads.
  p.logit_rows = p.logit_stride = 0;
  if (p.scores != nullptr && own_rows <= kRowsPerTile && p.tokens > 0) {
    const int64_t stride = ceil_div(own_keys, 4) * 4, segments = (int64_t)p.rows * p.kv_heads;
    if (stride * segments * own_rows <= (256ll << 20) && segments * ceil_div(own_keys, 4 * kThreads) < (1ll << 24)) {
      p.logit_rows = (int)own_rows;
      p.logit_stride = stride;
    }
  }
  p.direct = p.wide_own && !p.wide_pre && p.s_own == 1;
}

size_t partial_bytes(const Params &p, int head_dim) {
  return p.direct ? 0 : (size_t)(p.s_own + p.s_pre) * p.tokens * p.q_heads * ((size_t)head_dim * 4 + 8);
}
size_t workspace_bytes(const Params &p, int head_dim) {
  return (partial_bytes(p, head_dim) + 15) / 16 * 16 + (size_t)p.rows * p.kv_heads * p.logit_rows * p.logit_stride * 4 +
         (size_t)p.rows * 4 + (p.wide_pre ? (size_t)p.tokens * p.group * 4 : 0) + 16;
}

constexpr int kJoinWide = 1024;  // up to so many queries, 8 waves join the partial results of one

template <class T, int D>
int launch(const Params &p, hipStream_t stream) {
  int rc = EKV_OK;
  if (p.tokens > 0) {
    if (p.wide_pre) rc = wide_attention(p, T::kType, D, false, stream);
    if (rc == EKV_OK && p.wide_own) rc = wide_attention(p, T::kType, D, true, stream);
    using N = Narrow<T, D>;
    const unsigned grid = (unsigned)(ceil_div(p.items_pre, N::kWaves) + ceil_div(p.waves_own, N::kWaves));
    if (rc == EKV_OK && grid > 0) {
      hipLaunchKernelGGL((narrow_kernel<T, D>), dim3(grid), dim3(N::kThreads), 0, stream, p);
      rc = check_hip(hipGetLastError(), "ekv_prefix_attention launch");
    }
    if (rc == EKV_OK && !p.direct) {
      const int64_t queries = (int64_t)p.tokens * p.q_heads;
      typedef typename T::Query Q;
      if (queries <= kJoinWide)
        hipLaunchKernelGGL((combine_kernel<Q, D, 8>), dim3((unsigned)queries), dim3(8 * kWave), 0, stream, p);
      else
        hipLaunchKernelGGL((combine_kernel<Q, D, 1>), dim3((unsigned)ceil_div(queries, 4)), dim3(kThreads), 0, stream, p);
      rc = check_hip(hipGetLastError(), "ekv_prefix_attention combine launch");
    }
  }
  if (rc != EKV_OK || p.scores == nullptr || p.width == 0) return rc;
  const int64_t capacity = (int64_t)p.width * p.block_size, segments = (int64_t)p.rows * p.kv_heads;
  if (p.wide_own && (int64_t)p.max_query * p.group >= kWeighWide &&
      segments * ceil_div(capacity, kWeighKeys) < kWeighWaves * (int64_t)cu_count())
    return wide_weights(p, T::kType, D, stream);
  if (p.logits != nullptr) {
    const int pieces = (int)ceil_div(capacity, 4 * kThreads);
    hipLaunchKernelGGL((fold_kernel<kThreads>), dim3((unsigned)(segments * pieces)), dim3(kThreads), 0, stream, p, pieces);
  } else {
    const int pieces = (int)ceil_div(capacity, kWeighKeys);
    const unsigned weigh = (unsigned)ceil_div(segments * pieces, kThreads / kWave);
    hipLaunchKernelGGL((weigh_kernel<T, D>), dim3(weigh), dim3(kThreads), 0, stream, p, pieces);
  }
  return check_hip(hipGetLastError(), "ekv_prefix_attention weights launch");
}

template <class T>
int launch_dim(const Params &p, int head_dim, hipStream_t stream) {
  switch (head_dim) {
    case 32: return launch<T, 32>(p, stream);
    case 64: return launch<T, 64>(p, stream);
    case 128: return launch<T, 128>(p, stream);
    default: return launch<T, 256>(p, stream);
  }
}

// The checks both entry points share, and the parameters they fill.
int fill(const ekv_attention_t *a, Params &p) {
  const char *who = "ekv_prefix_attention";
  if (a == nullptr) return fail(EKV_EINVAL, "%s: null argument block", who);
  const int pair = a->q_dtype == a->kv_dtype ? a->q_dtype : a->q_dtype == EKV_BF16 && a->kv_dtype == EKV_FP8_E4M3 ? 3 : -1;
  if (pair < 0 || (pair != EKV_F32 && pair != EKV_F16 && pair != EKV_BF16 && a->kv_dtype != EKV_FP8_E4M3) ||
      a->q_dtype == EKV_FP8_E4M3)
    return fail(EKV_EUNSUPPORTED, "%s: queries of type %d with keys of type %d", who, a->q_dtype, a->kv_dtype);
  if (a->head_dim != 32 && a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256)
    return fail(EKV_EUNSUPPORTED, "%s: head dim %d (32, 64, 128 or 256)", who, a->head_dim);
  if (a->rows < 0 || a->tokens < 0 || a->width < 0 || a->max_query < 1 || a->kv_heads < 1 || a->q_heads < 1 ||
      a->q_heads % a->kv_heads != 0 || a->block_size < 1 || a->prefix_groups < 0 || a->prefix_width < 0 || a->blocks < 0)
    return fail(EKV_EINVAL, "%s: rows %d, tokens %d, width %d, queries %d, heads %d / %d, block size %d, groups %d x %d",
                who, a->rows, a->tokens, a->width, a->max_query, a->q_heads, a->kv_heads, a->block_size,
                a->prefix_groups, a->prefix_width);
  if (a->q_start == nullptr && (a->tokens != a->rows || a->max_query != 1))
    return fail(EKV_EINVAL, "%s: %d tokens, at most %d a row, of %d rows need q_start", who, a->tokens, a->max_query,
                a->rows);
  if ((int64_t)a->width * a->block_size >= kMostKeys || (int64_t)a->prefix_width * a->block_size >= kMostKeys)
    return fail(EKV_EINVAL, "%s: a table of %d or %d blocks of %d tokens passes 2^31 - 4096", who, a->width, a->prefix_width,
                a->block_size);
  if ((int64_t)a->tokens * a->q_heads >= INT32_MAX - 65536 || (int64_t)a->max_query * a->q_heads >= INT32_MAX - 65536)
    return fail(EKV_EINVAL, "%s: %d tokens of %d heads pass 2^31", who, a->tokens, a->q_heads);
  if (a->prefix_groups > 1 && a->prefix_rows == nullptr)
    return fail(EKV_EINVAL, "%s: %d prefixes need prefix_rows", who, a->prefix_groups);
  p = Params{};
  p.q = (const char *)a->query;
  p.q_st = a->q_stride_token;
  p.q_sh = a->q_stride_head;
  p.k = (const char *)a->keys;
  p.v = (const char *)a->values;
  p.st_block = a->kv_stride_block;
  p.st_pos = a->kv_stride_pos;
  p.st_head = a->kv_stride_head;
  p.blocks = a->blocks;
  p.table = a->table;
  p.table_stride = a->table_stride;
  p.lens = a->lens;
  p.q_start = a->q_start;
  p.ptable = a->prefix_table;
  p.ptable_stride = a->prefix_stride;
  p.plens = a->prefix_lens;
  p.prows = a->prefix_rows;
  p.scores = a->scores;
  p.sc_row = a->scores_stride_row;
  p.sc_head = a->scores_stride_head;
  p.out = (char *)a->out;
  p.o_st = a->out_stride_token;
  p.o_sh = a->out_stride_head;
  p.lse = a->lse;
  p.rows = a->rows;
  p.width = a->width;
  p.groups = a->prefix_width > 0 ? a->prefix_groups : 0;
  p.pwidth = a->prefix_width;
  p.tokens = a->tokens;
  p.max_query = a->max_query;
  p.q_heads = a->q_heads;
  p.kv_heads = a->kv_heads;
  p.group = a->q_heads / a->kv_heads;
  p.block_size = a->block_size;
  const PageDivisor d = page_divisor(a->block_size);
  p.bs_mul = d.mul;
  p.bs_shift = d.shift;
  p.scale2 = a->scale * a->k_scale * kLog2e;
  p.v_scale = a->v_scale;
  p.decay = a->decay;
  plan(p, a->head_dim, a->kv_dtype);
  // a launch has fewer than 2^32 threads: 64 a wave or item of the narrow kernel and of the weights read again, 256 an
  // item of the wide one
  if (p.waves_own + p.items_pre >= (1ll << 26) - 64 || p.items_own >= (1ll << 24) ||
      (int64_t)p.tokens * p.q_heads >= (1ll << 26) - 64 ||
      (p.scores != nullptr &&
       (int64_t)p.rows * p.kv_heads * ceil_div((int64_t)p.width * p.block_size, kWeighKeys) >= (1ll << 26) - 64))
    return fail(EKV_EINVAL, "%s: %d rows of %d blocks and %d tokens of %d heads pass the threads of a launch", who,
                p.rows, p.width, p.tokens, p.q_heads);
  return EKV_OK;
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace attn
}  // namespace ekv

using namespace ekv;

extern "C" size_t ekv_prefix_attention_workspace(const ekv_attention_t *a) {
  attn::Params p;
  if (attn::fill(a, p) != EKV_OK) return 0;
  return attn::workspace_bytes(p, a->head_dim);
}

extern "C" int ekv_prefix_attention(const ekv_attention_t *a, void *workspace, size_t workspace_bytes, void *stream) {
  attn::Params p;
  const int rc = attn::fill(a, p);
  if (rc != EKV_OK) return rc;
  if (p.tokens == 0 && (p.scores == nullptr || p.rows == 0)) return EKV_OK;
  if (p.rows == 0) return fail(EKV_EINVAL, "ekv_prefix_attention: %d tokens of no row", p.tokens);
  if (((p.k == nullptr || p.v == nullptr) && (p.width > 0 || p.groups > 0)) || p.lens == nullptr ||
      (p.tokens > 0 && (p.q == nullptr || p.out == nullptr || p.lse == nullptr)) ||
      (p.table == nullptr && p.width > 0) || (p.groups > 0 && (p.ptable == nullptr || p.plens == nullptr)))
    return fail(EKV_EINVAL, "ekv_prefix_attention: null pointer");
  if (p.blocks < 1 && (p.width > 0 || p.groups > 0))
    return fail(EKV_EINVAL, "ekv_prefix_attention: tables of an empty cache");
  const int qe = a->q_dtype == EKV_F32 ? 4 : 2, ke = a->kv_dtype == EKV_F32 ? 4 : a->kv_dtype == EKV_FP8_E4M3 ? 1 : 2;
  if (!attn::aligned16(p.q) || !attn::aligned16(p.k) || !attn::aligned16(p.v) || p.q_st * qe % 16 || p.q_sh * qe % 16 ||
      p.st_block * ke % 16 || p.st_pos * ke % 16 || p.st_head * ke % 16)
    return fail(EKV_EINVAL, "ekv_prefix_attention: query, key and value rows start at multiples of 16 bytes");
  if (p.table_stride < p.width || (p.groups > 0 && p.ptable_stride < p.pwidth))
    return fail(EKV_EINVAL, "ekv_prefix_attention: table rows of %d and %d blocks, strides %lld and %lld", p.width,
                p.pwidth, (long long)p.table_stride, (long long)p.ptable_stride);
  const size_t need = attn::workspace_bytes(p, a->head_dim);
  if (workspace == nullptr || workspace_bytes < need || !attn::aligned16(workspace))
    return fail(EKV_EINVAL, "ekv_prefix_attention: a workspace of %zu bytes, %zu needed at a multiple of 16",
                workspace_bytes, need);
  const int64_t queries = (int64_t)p.tokens * p.q_heads;
  p.part_o = (float *)workspace;
  p.part_ml = (float2 *)(p.part_o + (int64_t)(p.s_own + p.s_pre) * queries * a->head_dim);
  char *more = (char *)workspace + (attn::partial_bytes(p, a->head_dim) + 15) / 16 * 16;
  if (p.logit_rows > 0) p.logits = (float *)more;
  p.row_slots = (int32_t *)(more + (size_t)p.rows * p.kv_heads * p.logit_rows * p.logit_stride * 4);
  p.pre_slots = p.row_slots + p.rows;
  hipStream_t s = (hipStream_t)stream;
  switch (a->kv_dtype) {
    case EKV_F32: return attn::launch_dim<attn::F32>(p, a->head_dim, s);
    case EKV_F16: return attn::launch_dim<attn::F16>(p, a->head_dim, s);
    case EKV_BF16: return attn::launch_dim<attn::BF16>(p, a->head_dim, s);
    default: return attn::launch_dim<attn::FP8>(p, a->head_dim, s);
  }
}
