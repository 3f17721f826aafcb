// Attention over the paged cache for a batch whose rows share prefixes, and the running attention weight
// of each cached token.
//
//   s_qj = scale * k_scale * <q, k_j>            over the keys j that query q sees
//   out_q = v_scale * sum_j exp(s_qj - lse_q) v_j,   lse_q = log sum_j exp(s_qj)
//   scores[row, head, j] = decay * scores[row, head, j] + sum_{q of the row and head} exp(s_qj - lse_q)
//
// A query sees the whole prefix of its row's group and its row's own keys up to itself.  The keys are cut
// into chunks, every (chunk, KV head, tile of query rows) is one item of work, and an item leaves its
// maximum, sum and unnormalised output, which combine_kernel joins:
//   m = max_c m_c,  l = sum_c l_c 2^(m_c - m),  out = sum_c o_c 2^(m_c - m) / l.
// A prefix is one set of items for all the queries of its group: its keys and values are read once per
// tile of them and not once per row.
#include "ekv_attention.hpp"

namespace ekv {
namespace attn {

// What one wave works on: keys [begin, end) behind `table`, query rows [m0, M) of the tokens from `first`.
struct Segment {
  const int32_t *table;
  int begin, end;
  int first, rows;  // first token, query rows (tokens * group)
  int m0;
  int head, slot;
  int see;  // query token i sees keys below see + i (own pages), or INT_MAX / 2 (a prefix)
};

template <int TILE>
__device__ __forceinline__ bool own_segment(const Params &p, int64_t item, Segment &s) {
  s.head = (int)(item % p.kv_heads);
  item /= p.kv_heads;
  const int tile = (int)(item % p.tiles_own);
  item /= p.tiles_own;
  const int chunk = (int)(item % p.s_own);
  const int row = (int)(item / p.s_own);
  const int len = row_length(p, row);
  const RowQueries t = row_queries(p, row);
  s.table = p.table + (int64_t)row * p.table_stride;
  s.first = t.first;
  s.rows = min(t.count, p.max_query) * p.group;
  s.m0 = tile * TILE;
  s.see = len - t.count + 1;
  s.slot = chunk;
  if (s.m0 >= s.rows) return false;
  const int last = (min(s.m0 + TILE, s.rows) - 1) / p.group;
  const int64_t begin = (int64_t)chunk * p.chunk_own;
  s.end = (int)min(begin + p.chunk_own, (int64_t)min(len, s.see + last));
  s.begin = (int)min(begin, (int64_t)INT32_MAX);
  return s.begin < s.end;
}

template <int TILE>
__device__ __forceinline__ bool prefix_segment(const Params &p, int64_t item, Segment &s) {
  s.head = (int)(item % p.kv_heads);
  item /= p.kv_heads;
  const int chunk = (int)(item % p.s_pre);
  int g, tile;
  if (!find_tile(p, (int)(item / p.s_pre), TILE, g, tile)) return false;
  const RowQueries t = group_queries(p, g);
  s.table = p.ptable + (int64_t)g * p.ptable_stride;
  s.first = t.first;
  s.rows = t.count * p.group;
  s.m0 = tile * TILE;
  s.see = INT32_MAX / 2;
  s.slot = p.s_own + chunk;
  const int64_t begin = (int64_t)chunk * p.chunk_pre;
  s.end = (int)min(begin + p.chunk_pre, (int64_t)group_length(p, g));
  s.begin = (int)min(begin, (int64_t)INT32_MAX);
  return s.begin < s.end;
}

// The keys and values of 16 consecutive slots, one lane's part: key l % 16, and the values of the four
// keys 4 * (l / 16) + i, whose dims the 16 lanes of a lane group share out.
template <class T, int D>
struct Tile {
  static constexpr int kLaneDims = D / 16;  // of one value row
  static constexpr int kPieceDims = kLaneDims * T::kBytes > 16 ? 16 / T::kBytes : kLaneDims;
  static constexpr int kValuePieces = kLaneDims / kPieceDims;
  static constexpr int kPieceBytes = kPieceDims * T::kBytes;
  static constexpr int kPieceWords = kPieceBytes < 4 ? 1 : kPieceBytes / 4;
  KeyRow<T, D> key;
  uint32_t value[4][kValuePieces * kPieceWords];
  uint32_t ok;  // bit i: key 4 * (l / 16) + i has a page in the cache

  // WHOLE: the 16 slots lie in one page (block sizes that are multiples of 16), so its id is uniform.
  template <bool WHOLE>
  __device__ __forceinline__ void load(const Params &p, const Segment &s, int base, bool values) {
    const int lane = lane_id(), g = lane / 16, n = lane % 16;
    const int64_t head = (int64_t)s.head * p.st_head;
    if constexpr (WHOLE) {
      const int index = page_of(p, base);
      int page = s.table[index];
      const bool good = (uint32_t)page < (uint64_t)p.blocks;
      ok = good ? 15u : 0u;
      if (!good) page = 0;
      const int at = base - index * p.block_size;
      const int64_t origin = ((int64_t)page * p.st_block + (int64_t)at * p.st_pos + head) * T::kBytes;
      key.load(p.k + origin + (int64_t)n * p.st_pos * T::kBytes, g);
      if (values) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          load_value(p.v + origin + (int64_t)(4 * g + i) * p.st_pos * T::kBytes, n, i);
      }
    } else {
      ok = 0;
      {
        const int pos = min(base + n, s.end - 1), index = page_of(p, pos);
        int page = s.table[index];
        if ((uint32_t)page >= (uint64_t)p.blocks) page = 0;
        key.load(p.k + ((int64_t)page * p.st_block + (int64_t)(pos - index * p.block_size) * p.st_pos + head) *
                           T::kBytes, g);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int pos = min(base + 4 * g + i, s.end - 1), index = page_of(p, pos);
        int page = s.table[index];
        const bool good = (uint32_t)page < (uint64_t)p.blocks;
        ok |= good ? 1u << i : 0u;
        if (!good) page = 0;
        if (values)
          load_value(p.v + ((int64_t)page * p.st_block + (int64_t)(pos - index * p.block_size) * p.st_pos + head) *
                               T::kBytes, n, i);
      }
    }
  }
  __device__ __forceinline__ void load_value(const char *row, int n, int i) {
#pragma unroll
    for (int c = 0; c < kValuePieces; ++c)
      load_bytes<kPieceBytes>(row + (c * 16 + n) * kPieceBytes, value[i] + c * kPieceWords);
  }
};

// One wave per item.  S^T = K Q^T on the matrix cores leaves each lane the logits of four keys of one query
// row.  O^T = V^T P^T is summed by the float32 matrix instruction of four keys: its P operand is what the
// lane already holds (key 4g + i for step i, the weights never rounded), and its V operand one element of
// the lane's own 16 bytes of a value row, so neither product moves data between lanes or through LDS.  The
// float32 instruction has a sixteenth of the 16-bit one's rate, which for 16 query rows still outruns HBM.
// Loads run one step (KT tiles) ahead in registers.
template <class T, int D, bool WHOLE, int KT>
__device__ __forceinline__ void attend(const Params &p, const Segment &s) {
  using Tl = Tile<T, D>;
  constexpr int E = sizeof(typename T::Query);
  const int lane = lane_id(), g = lane / 16, n = lane % 16;
  const int m = s.m0 + n;
  const bool live = m < s.rows;
  const int i_q = live ? m / p.group : 0;
  const int token = s.first + i_q, q_head = s.head * p.group + (live ? m - i_q * p.group : 0);
  QueryRow<T, D> q;
  q.load(p.q + ((int64_t)token * p.q_st + (int64_t)q_head * p.q_sh) * E, g, live);
  const int limit = live ? min(s.end, s.see + i_q) : 0;   // this lane's query sees keys below it
  const int every = min(s.end, s.see + s.m0 / p.group);    // and every query of the tile keys below this
  const int last = s.begin + ((s.end - 1 - s.begin) & ~15);  // the last tile that starts before the end

  f32x4 acc[D / 16];
#pragma unroll
  for (int a = 0; a < D / 16; ++a) acc[a] = f32x4{0.f, 0.f, 0.f, 0.f};
  float top = -INFINITY, sum = 0.f;

  auto step = [&](Tl *t, int base) {
    float x[KT][4];
    float high = -INFINITY;
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      const f32x4 c = dot_tile<T, D>(t[k].key, q);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[k][i] = c[i] * p.scale2;
      const int tile = base + 16 * k;
      if (!__all(tile + 16 <= every && t[k].ok == 15u)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int pos = tile + 4 * g + i;
          const bool there = (t[k].ok >> i & 1u) != 0;
          x[k][i] = there && pos < limit ? x[k][i] : -INFINITY;
          if (!there || pos >= s.end) {  // what lies there may be anything: 0 * NaN is no zero
#pragma unroll
            for (int w = 0; w < Tl::kValuePieces * Tl::kPieceWords; ++w) t[k].value[i][w] = 0;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) high = fmaxf(high, x[k][i]);
    }
    const float peak = fmaxf(top, rows_max(high));
    const float ref = peak == -INFINITY ? 0.f : peak;
    const float shrink = __builtin_amdgcn_exp2f(top - ref);
    if (!__all(top == peak)) {
      sum *= shrink;
#pragma unroll
      for (int a = 0; a < D / 16; ++a) acc[a] *= shrink;
    }
    top = peak;
#pragma unroll
    for (int k = 0; k < KT; ++k) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float w = __builtin_amdgcn_exp2f(x[k][i] - ref);
        sum += w;
#pragma unroll
        for (int c = 0; c < Tl::kValuePieces; ++c) {
#pragma unroll
          for (int j = 0; j < Tl::kPieceDims; ++j)
            acc[c * Tl::kPieceDims + j] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                element<T>(t[k].value[i] + c * Tl::kPieceWords, j), w, acc[c * Tl::kPieceDims + j], 0, 0, 0);
        }
      }
    }
  };
  auto fetch = [&](Tl *t, int base) {
#pragma unroll
    for (int k = 0; k < KT; ++k) t[k].template load<WHOLE>(p, s, min(base + 16 * k, last), true);
  };

  Tl a[KT], b[KT];
  constexpr int kStep = 16 * KT;
  fetch(a, s.begin);
  for (int base = s.begin;;) {
    fetch(b, base + kStep);
    step(a, base);
    base += kStep;
    if (base >= s.end) break;
    fetch(a, base + kStep);
    step(b, base);
    base += kStep;
    if (base >= s.end) break;
  }

  sum = rows_sum(sum);
  if (!live) return;
  const int64_t at = ((int64_t)s.slot * p.tokens + token) * p.q_heads + q_head;
  if (g == 0) p.part_ml[at] = make_float2(top, sum);
  float *o = p.part_o + at * D;
#pragma unroll
  for (int c = 0; c < Tl::kValuePieces; ++c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float *dst = o + c * 16 * Tl::kPieceDims + (4 * g + e) * Tl::kPieceDims;
#pragma unroll
      for (int j = 0; j < Tl::kPieceDims; ++j) dst[j] = acc[c * Tl::kPieceDims + j][e];
    }
  }
}

constexpr int kThreads = 256;

// tiles of a step: about 8 KB of keys and values in flight per wave
template <class T, int D>
constexpr int kTiles = D * T::kBytes <= 128 ? 4 : D * T::kBytes <= 256 ? 2 : 1;

template <class T, int D, bool WHOLE>
__global__ __launch_bounds__(kThreads, D *T::kBytes <= 512 ? 2 : 1) void narrow_kernel(const Params p) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t item = (int64_t)blockIdx.x * (kThreads / kWave) + wave;
  const int64_t shared = p.wide_pre ? 0 : p.items_pre;  // items of the prefixes come first
  Segment s;
  if (item < shared) {
    if (!prefix_segment<kRowsPerTile>(p, item, s)) return;
  } else {
    if (item - shared >= p.items_own) return;
    if (!own_segment<kRowsPerTile>(p, item - shared, s)) return;
  }
  attend<T, D, WHOLE, kTiles<T, D>>(p, s);
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
__device__ __forceinline__ void store(float *dst, float v) { *dst = v; }
__device__ __forceinline__ void store(__bf16 *dst, float v) { *dst = (__bf16)v; }
__device__ __forceinline__ void store(_Float16 *dst, float v) { *dst = (_Float16)v; }

// One wave per (token, query head): lane t weighs slot t, then the slots' outputs are summed in slot order.
template <class Q, int D>
__global__ __launch_bounds__(kThreads) void combine_kernel(const Params p) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t item = (int64_t)blockIdx.x * (kThreads / kWave) + wave;
  if (item >= (int64_t)p.tokens * p.q_heads) return;
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
      const int64_t all = (int64_t)n + max(seen, 0);
      own = all > 0 ? (int)((all - 1) / p.chunk_own) + 1 : 0;
    } else {
      own = seen > 0 ? (seen - 1) / p.chunk_own + 1 : 0;
      pre = n > 0 ? (n - 1) / p.chunk_pre + 1 : 0;
    }
  }
  constexpr int kPer = D > 64 ? D / 64 : 1;
  constexpr int kLanes = D / kPer;
  float acc[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) acc[j] = 0.f;
  float top = -INFINITY, sum = 0.f;
  const int64_t plane = (int64_t)p.tokens * p.q_heads;
  for (int part = 0; part < 2; ++part) {
    const int slots = part == 0 ? own : pre, first = part == 0 ? 0 : p.s_own;
    if (slots == 0) continue;
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < slots) ml = p.part_ml[(int64_t)(first + lane) * plane + item];
    const float peak = fmaxf(top, wave_max(ml.x));
    const float ref = peak == -INFINITY ? 0.f : peak;
    const float shrink = __builtin_amdgcn_exp2f(top - ref);
    const float w = ml.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml.x - ref);
    sum = sum * shrink + wave_sum(ml.y * w);
#pragma unroll
    for (int j = 0; j < kPer; ++j) acc[j] *= shrink;
    top = peak;
    const float *o = p.part_o + ((int64_t)first * plane + item) * D + (lane % kLanes) * kPer;
    // four slots' loads in flight; past the last slot the weight is 0 and the last slot is read again
    for (int k = 0; k < slots; k += 4) {
      float x[4][kPer];
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int j = 0; j < kPer; ++j) x[u][j] = o[(int64_t)min(k + u, slots - 1) * plane * D + j];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float wk = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), k + u));
#pragma unroll
        for (int j = 0; j < kPer; ++j) acc[j] += k + u < slots ? wk * x[u][j] : 0.f;
      }
    }
  }
  // no key seen, or none with any weight: the sum is empty
  const bool none = sum == 0.f;
  const float inv = none ? 0.f : p.v_scale / sum;
  if (lane < kLanes) {
    Q *o = (Q *)p.out + (int64_t)token * p.o_st + (int64_t)q_head * p.o_sh + lane * kPer;
#pragma unroll
    for (int j = 0; j < kPer; ++j) store(o + j, none ? 0.f : acc[j] * inv);
  }
  if (lane == 0) p.lse[item] = none ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

// -- the running weights ------------------------------------------------------------------------------

constexpr int kWeighKeys = 64;  // keys of one wave

// One wave per (row, KV head, 64 keys): the logits of every query row against them again, their weights
// exp(s - lse) summed over the query rows in one order, and one addition to each key's running score.
template <class T, int D, bool WHOLE>
__global__ __launch_bounds__(kThreads) void weigh_kernel(const Params p, int pieces) {
  constexpr int E = sizeof(typename T::Query);
  constexpr int KT = kWeighKeys / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  int64_t item = (int64_t)blockIdx.x * (kThreads / kWave) + wave;
  if (item >= (int64_t)p.rows * pieces * p.kv_heads) return;
  Segment s;
  s.head = (int)(item % p.kv_heads);
  item /= p.kv_heads;
  const int row = (int)(item / pieces);
  s.begin = (int)(item % pieces) * kWeighKeys;
  const int len = row_length(p, row);
  s.end = min(s.begin + kWeighKeys, len);
  if (s.begin >= s.end) return;
  s.table = p.table + (int64_t)row * p.table_stride;
  const RowQueries t = row_queries(p, row);
  const int see = len - t.count + 1, rows = min(t.count, p.max_query) * p.group;
  const int lane = lane_id(), g = lane / 16, n = lane % 16;
  const int last = s.begin + ((s.end - 1 - s.begin) & ~15);
  Tile<T, D> tile[KT];
#pragma unroll
  for (int k = 0; k < KT; ++k) tile[k].template load<WHOLE>(p, s, min(s.begin + 16 * k, last), false);
  float total[KT][4];
#pragma unroll
  for (int k = 0; k < KT; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) total[k][i] = 0.f;
  // queries before the first key see none of them
  const int m_first = max(0, (s.begin - see + 1)) * p.group / kRowsPerTile * kRowsPerTile;
  for (int m0 = m_first; m0 < rows; m0 += kRowsPerTile) {
    const int m = m0 + n;
    const bool live = m < rows;
    const int i_q = live ? m / p.group : 0;
    const int token = t.first + i_q, q_head = s.head * p.group + (live ? m - i_q * p.group : 0);
    QueryRow<T, D> q;
    q.load(p.q + ((int64_t)token * p.q_st + (int64_t)q_head * p.q_sh) * E, g, live);
    const float lse = live ? p.lse[(int64_t)token * p.q_heads + q_head] : -INFINITY;
    const float lse2 = lse * kLog2e;
    const int limit = lse == -INFINITY ? 0 : min(s.end, see + i_q);
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      const f32x4 c = dot_tile<T, D>(tile[k].key, q);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool sees = (tile[k].ok >> i & 1u) != 0 && s.begin + 16 * k + 4 * g + i < limit;
        total[k][i] += sees ? __builtin_amdgcn_exp2f(c[i] * p.scale2 - lse2) : 0.f;
      }
    }
  }
  float *out = p.scores + (int64_t)row * p.sc_row + (int64_t)s.head * p.sc_head;
#pragma unroll
  for (int k = 0; k < KT; ++k) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float v = total[k][i];
#pragma unroll
      for (int d = 1; d < 16; d <<= 1) v += shfl_xor(v, d);
      const int pos = s.begin + 16 * k + 4 * g + i;
      if (n == i && pos < s.end) out[pos] = p.decay * out[pos] + v;
    }
  }
}

// -- the launches ---------------------------------------------------------------------------------------

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How the keys are cut.  A long table is cut so that the items fill the chip several times over (rows have
// different lengths and the host knows only the widest), but no chunk is shorter than 64 keys, and the
// partial outputs stay below 256 MB.
void split(int64_t keys, int64_t items_per_chunk, int64_t queries, int head_dim, int &chunk, int &slots) {
  const int64_t target = 32 * (int64_t)cu_count();
  int64_t n = ceil_div(target, items_per_chunk > 0 ? items_per_chunk : 1);
  n = n < ceil_div(keys, 1024) ? ceil_div(keys, 1024) : n;
  const int64_t fit = (256ll << 20) / ((queries > 0 ? queries : 1) * (head_dim * 4 + 8));
  n = n > fit ? fit : n;
  n = n > kMaxSlots ? kMaxSlots : n < 1 ? 1 : n;
  chunk = (int)(ceil_div(ceil_div(keys, n), 64) * 64);
  if (chunk < 64) chunk = 64;
  slots = (int)ceil_div(keys, chunk);
  if (slots < 1) slots = 1;
}

// The wide kernel's: a few workgroups for each that the chip holds, no chunk shorter than 512 keys (its
// partial outputs, written and read again, are as much traffic as 64 keys and values).
void split_wide(int64_t keys, int64_t items_per_chunk, int64_t queries, int head_dim, int &chunk, int &slots) {
  int64_t n = ceil_div(4 * (int64_t)cu_count(), items_per_chunk > 0 ? items_per_chunk : 1);
  const int64_t fit = (256ll << 20) / ((queries > 0 ? queries : 1) * (head_dim * 4 + 8));
  n = n > fit ? fit : n;
  n = n > kMaxSlots ? kMaxSlots : n < 1 ? 1 : n;
  const int64_t each = ceil_div(ceil_div(keys, n), 64) * 64;
  chunk = (int)(each < 512 ? 512 : each > (1 << 30) ? INT32_MAX : each);
  slots = (int)ceil_div(keys, chunk);
  if (slots < 1) slots = 1;
}

void plan(Params &p, int head_dim, int kv_dtype) {
  const int64_t queries = (int64_t)p.tokens * p.q_heads;
  const int64_t own_rows = (int64_t)p.max_query * p.group;
  const bool half = kv_dtype != EKV_F32;
  const int64_t axis = (int64_t)(p.width + (p.groups > 0 ? p.pwidth : 0)) * p.block_size;
  p.wide_own = half && own_rows >= kWideRows && axis < (1 << 30);
  p.wide_pre = half && !p.wide_own && p.groups > 0 && (int64_t)p.tokens * p.group / p.groups >= kWideRows;
  p.tile_own = p.wide_own ? wide_tile_rows() : kRowsPerTile;
  p.tile_pre = p.wide_pre ? wide_tile_rows() : kRowsPerTile;
  p.tiles_own = (int)ceil_div(own_rows, p.tile_own);
  const int64_t own_keys = (int64_t)p.width * p.block_size, prefix_keys = p.groups > 0 ? (int64_t)p.pwidth * p.block_size : 0;
  const int64_t own_items = (int64_t)p.rows * p.kv_heads * p.tiles_own;
  p.items_pre = 0;
  p.s_pre = 0;
  p.chunk_pre = 64;
  if (p.wide_own) {
    split_wide(own_keys + prefix_keys, own_items, queries, head_dim, p.chunk_own, p.s_own);
  } else {
    split(own_keys, own_items, queries, head_dim, p.chunk_own, p.s_own);
    if (p.groups > 0) {
      p.tiles_pre = (int)(ceil_div((int64_t)p.tokens * p.group, p.tile_pre) + p.groups);
      const int64_t items = (int64_t)p.kv_heads * p.tiles_pre;
      if (p.wide_pre) split_wide(prefix_keys, items, queries, head_dim, p.chunk_pre, p.s_pre);
      else split(prefix_keys, items, queries, head_dim, p.chunk_pre, p.s_pre);
      p.items_pre = items * p.s_pre;
    }
  }
  p.items_own = own_items * p.s_own;
  p.direct = p.wide_own && p.s_own == 1;
}

int64_t narrow_items(const Params &p) { return p.wide_own ? 0 : p.items_own + (p.wide_pre ? 0 : p.items_pre); }

size_t workspace_bytes(const Params &p, int head_dim) {
  if (p.direct) return 16;
  return (size_t)(p.s_own + p.s_pre) * p.tokens * p.q_heads * ((size_t)head_dim * 4 + 8);
}

template <class T, int D>
int launch(const Params &p, hipStream_t stream) {
  const bool whole = p.block_size % 16 == 0;
  int rc = EKV_OK;
  if (p.tokens > 0) {
    if (p.wide_own || p.wide_pre) rc = wide_attention(p, T::kType, D, p.wide_own, stream);
    const unsigned grid = (unsigned)ceil_div(narrow_items(p), kThreads / kWave);
    if (rc == EKV_OK && grid > 0) {
      if (whole) hipLaunchKernelGGL((narrow_kernel<T, D, true>), dim3(grid), dim3(kThreads), 0, stream, p);
      else hipLaunchKernelGGL((narrow_kernel<T, D, false>), dim3(grid), dim3(kThreads), 0, stream, p);
      rc = check_hip(hipGetLastError(), "ekv_prefix_attention launch");
    }
    if (rc == EKV_OK && !p.direct) {
      const unsigned joins = (unsigned)ceil_div((int64_t)p.tokens * p.q_heads, kThreads / kWave);
      hipLaunchKernelGGL((combine_kernel<typename T::Query, D>), dim3(joins), dim3(kThreads), 0, stream, p);
      rc = check_hip(hipGetLastError(), "ekv_prefix_attention combine launch");
    }
  }
  if (rc != EKV_OK || p.scores == nullptr) return rc;
  if (p.width == 0) return rc;
  const int pieces = (int)ceil_div((int64_t)p.width * p.block_size, kWeighKeys);
  const unsigned weigh = (unsigned)ceil_div((int64_t)p.rows * pieces * p.kv_heads, kThreads / kWave);
  if (whole) hipLaunchKernelGGL((weigh_kernel<T, D, true>), dim3(weigh), dim3(kThreads), 0, stream, p, pieces);
  else hipLaunchKernelGGL((weigh_kernel<T, D, false>), dim3(weigh), dim3(kThreads), 0, stream, p, pieces);
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
  if ((int64_t)a->width * a->block_size >= INT32_MAX || (int64_t)a->prefix_width * a->block_size >= INT32_MAX)
    return fail(EKV_EINVAL, "%s: a table of %d or %d blocks of %d tokens passes 2^31", who, a->width, a->prefix_width,
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
  // a launch has fewer than 2^32 threads: 64 an item of the narrow kernel, 256 of the wide one
  if (narrow_items(p) >= (1ll << 26) - 64 || (p.wide_own ? p.items_own : p.wide_pre ? p.items_pre : 0) >= (1ll << 24) ||
      (int64_t)p.tokens * p.q_heads >= (1ll << 26) - 64 ||
      (p.scores != nullptr && (int64_t)p.rows * p.kv_heads * ceil_div((int64_t)p.width * p.block_size, kWeighKeys) >= (1ll << 26) - 64))
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
  hipStream_t s = (hipStream_t)stream;
  switch (a->kv_dtype) {
    case EKV_F32: return attn::launch_dim<attn::F32>(p, a->head_dim, s);
    case EKV_F16: return attn::launch_dim<attn::F16>(p, a->head_dim, s);
    case EKV_BF16: return attn::launch_dim<attn::BF16>(p, a->head_dim, s);
    default: return attn::launch_dim<attn::FP8>(p, a->head_dim, s);
  }
}
