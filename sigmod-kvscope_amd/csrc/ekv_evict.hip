// Eviction of cached tokens by accumulated attention weight.
//
// For each (row, KV head) of n tokens and budget b = min(n, budget): the b tokens that come first in the
// order (protected first, higher score, lower slot) stay.  A token is protected when its position is below
// `sinks` or at least seen - recent.  NaN ranks with -inf, -0 with +0.
//
// Attention does not depend on the order of a cache's slots, so nothing is shifted: the k-th token kept
// behind slot b moves into the k-th freed slot below it, and every other token stays where it is.  Sources
// are at b or above and destinations below, so all moves can run at once, in place.
//
// select_kernel, a workgroup per (row, head), holds the row's scores and positions in registers (up to 16384
// slots; longer rows pass through memory again and again, stream_kernel), finds the b-th by three passes over 11,
// 11 and 10 bits of the keys, writes scores, positions and lengths, and copies the keys and values of the tokens
// that move.  Where a few workgroups would copy much, they list the moves for move_kernel instead, which spreads
// them over the chip.  Bound: the scores and positions, read and written once, and the rows that move.
// Measured, 128 rows of 8 KV heads of 128, bf16: a few tokens past a budget of 4096 29 us, half of 512 to 8192
// tokens 254 us (78 and 321 us with eight passes through memory and a copy kernel behind them).
#include "ekv_common.hpp"

namespace ekv {
namespace evict {

constexpr int kThreads = 512;
constexpr int kBins = 256;
constexpr int kMoveThreads = 256;

struct Params {
  const int32_t *table;
  int64_t table_stride;
  const int32_t *lens, *budget, *seen;
  const float *scores;
  const int32_t *positions;
  int64_t s_row, s_head, p_row, p_head;
  float *new_scores;
  int32_t *new_positions;
  int64_t ns_row, ns_head, np_row, np_head;
  int32_t *new_lens;
  char *k, *v;
  int64_t st_block, st_pos, st_head;  // bytes
  int64_t blocks;
  int32_t *count;   // [rows * heads]
  int2 *moves;      // [rows * heads][capacity / 2]: from, to
  int rows, heads, width, block_size, capacity, half, fixed_budget, recent, sinks, row_bytes;
  uint32_t bs_mul;
  int bs_shift;
};

__device__ __forceinline__ int page_of(const Params &p, int pos) {
  return (int)(__umulhi((uint32_t)pos << 1, p.bs_mul) >> p.bs_shift);
}

// Unsigned keys in the order of the scores.
__device__ __forceinline__ uint32_t order_of(float f) {
  if (f != f) f = -INFINITY;
  const uint32_t b = __builtin_bit_cast(uint32_t, f + 0.f);  // -0 + 0 = +0
  return (b >> 31) ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ bool is_protected(const Params &p, int position, int64_t newest) {
  return position < p.sinks || position >= newest;
}

// A token that keeps its slot: copied where the new buffers are not the old ones.
__device__ __forceinline__ void keep_in_place(const Params &p, int j, const float *scores, const int32_t *positions,
                                              float *new_scores, int32_t *new_positions) {
  if (new_scores != scores) new_scores[j] = scores[j];
  if (new_positions != positions) new_positions[j] = positions[j];
}

// -- rows that registers hold ----------------------------------------------------------------------------

// Of NT threads each has 4 consecutive slots of each of R rounds: slots 4 NT i + 4 tid + e.
constexpr int kDigit = 2048;  // bins of a pass
typedef float Float4 __attribute__((ext_vector_type(4), aligned(4)));
typedef int Int4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t Row16 __attribute__((ext_vector_type(4)));

// Exclusive sums of the threads' values in slot order (round by round, thread by thread).  Contains barriers.
template <int NT, int R>
__device__ __forceinline__ int ordered_scan(const int (&v)[R], int (&before)[R], int *scratch) {
  constexpr int kWaves = NT / kWave;
  static_assert(R * kWaves <= kWave, "a wave scans the waves' sums");
  const int lane = lane_id(), wave = threadIdx.x / kWave;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int inc = wave_inclusive_scan(v[i]);
    before[i] = inc - v[i];
    if (lane == kWave - 1) scratch[i * kWaves + wave] = inc;
  }
  __syncthreads();
  // every wave scans the waves' sums of the rounds
  const int sum = lane < R * kWaves ? scratch[lane] : 0;
  const int inc = wave_inclusive_scan(sum);
#pragma unroll
  for (int i = 0; i < R; ++i) before[i] += __shfl(inc - sum, i * kWaves + wave);
  __syncthreads();
  return __builtin_amdgcn_readlane(inc, kWave - 1);
}

// The key and value rows of `count` moves that move(k) names, 16 bytes a lane, four moves in flight.  A slot whose
// table entry is no page of the cache is not read or written.
template <int THREADS, class Move>
__device__ __forceinline__ void copy_rows(const Params &p, int row, int head, int count, int first, int stride, Move move) {
  const int pieces = p.row_bytes / 16;  // a power of two, 2 to 64
  const int per = THREADS / pieces, piece = threadIdx.x % pieces;
  const int32_t *table = p.table + (int64_t)row * p.table_stride;
  constexpr int kFlight = 4;
  for (int k0 = first * per + threadIdx.x / pieces; k0 < count; k0 += stride * per * kFlight) {
    int64_t src[kFlight], dst[kFlight];
    bool good[kFlight];
    int2 m[kFlight];
    int a[kFlight], b[kFlight];
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      const int k = k0 + u * stride * per;
      good[u] = k < count;
      m[u] = good[u] ? move(k) : make_int2(0, 0);
    }
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      a[u] = table[page_of(p, m[u].x)];
      b[u] = table[page_of(p, m[u].y)];
    }
    Row16 x[kFlight] = {}, y[kFlight] = {};
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      good[u] = good[u] && (uint32_t)a[u] < (uint64_t)p.blocks && (uint32_t)b[u] < (uint64_t)p.blocks;
      const int from = m[u].x - page_of(p, m[u].x) * p.block_size, to = m[u].y - page_of(p, m[u].y) * p.block_size;
      src[u] = (int64_t)a[u] * p.st_block + (int64_t)from * p.st_pos + head * p.st_head + piece * 16;
      dst[u] = (int64_t)b[u] * p.st_block + (int64_t)to * p.st_pos + head * p.st_head + piece * 16;
      if (good[u]) {
        x[u] = *(const Row16 *)(p.k + src[u]);
        y[u] = *(const Row16 *)(p.v + src[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      if (!good[u]) continue;
      *(Row16 *)(p.k + dst[u]) = x[u];
      *(Row16 *)(p.v + dst[u]) = y[u];
    }
  }
}

// Waves a SIMD that the registers are kept to.  Where the workgroups copy, up to three rounds fit 64, with which a compute
// unit holds four workgroups, all of 128 rows at once (29 us for a few tokens past a budget of 4096, 33 with two); four
// rounds would spill there (284 us for half of 8192, 254 with two).  Where they list the moves there are few workgroups, and
// 128 registers, or 96 for four rounds, hold a row without a spill (with eight and four waves 35 to 104 registers spilled:
// 8 rows of 8 heads and 8192 tokens cut in half 57 us, 42 without; 32 rows of 4096 and 8192 tokens 80 and 163, 66 and 147).
template <int NT, int R, bool COPY>
constexpr int kSelectWaves = COPY ? (NT == 512 && R <= 3 ? 8 : 4) : (R <= 3 ? 4 : 5);

template <int NT, int R, bool COPY>
__global__ __launch_bounds__(NT, (kSelectWaves<NT, R, COPY>)) void select_kernel(const Params p) {
  constexpr int kRound = 4 * NT, kBinsEach = kDigit / NT;
  typedef int Bins __attribute__((ext_vector_type(kBinsEach), aligned(4)));
  __shared__ __attribute__((aligned(16))) int s_bins[kDigit];
  __shared__ int s_scan[64];
  __shared__ int s_pick[3];
  __shared__ uint16_t s_from[R * kRound / 2], s_to[R * kRound / 2];  // the k-th survivor's slot, the k-th freed slot
  const int segment = blockIdx.x, row = segment / p.heads, head = segment - row * p.heads;
  const int tid = threadIdx.x;
  const int n = min(max(p.lens[row], 0), p.capacity);
  const int b = min(n, max(p.budget != nullptr ? p.budget[row] : p.fixed_budget, 0));
  const int64_t newest = (int64_t)p.seen[row] - p.recent;
  const float *scores = p.scores + (int64_t)row * p.s_row + (int64_t)head * p.s_head;
  const int32_t *positions = p.positions + (int64_t)row * p.p_row + (int64_t)head * p.p_head;
  float *new_scores = p.new_scores + (int64_t)row * p.ns_row + (int64_t)head * p.ns_head;
  int32_t *new_positions = p.new_positions + (int64_t)row * p.np_row + (int64_t)head * p.np_head;

  Float4 s[R];
  Int4 at[R];
  uint32_t keep = 0, safe = 0;  // bits 4 i + e
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int j = i * kRound + 4 * tid;
    s[i] = Float4{0.f, 0.f, 0.f, 0.f};
    at[i] = Int4{0, 0, 0, 0};
    if (j + 4 <= n) {
      s[i] = *(const Float4 *)(scores + j);
      at[i] = *(const Int4 *)(positions + j);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (j + e < n) {
          s[i][e] = scores[j + e];
          at[i][e] = positions[j + e];
        }
    }
  }
  // Which of the thread's slots there are
  auto there = [&](int i, int e) { return i * kRound + 4 * tid + e < n; };
  if (b < n) {
    int mine = 0;
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (there(i, e) && is_protected(p, at[i][e], newest)) {
          safe |= 1u << (4 * i + e);
          ++mine;
        }
    // the class that the cut falls into: the protected tokens if there are b of them or more
    const int guarded = block_sum<NT, int>(mine, s_scan);
    const bool among_safe = guarded >= b;
    // the `want`-th highest key of that class, digit by digit; `equal` tokens have that very key
    int want = among_safe ? b : b - guarded, equal = 0;
    uint32_t cut = 0;
    auto candidate = [&](int i, int e) { return there(i, e) && ((safe >> (4 * i + e) & 1) != 0) == among_safe; };
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
      if (want == 0) break;  // b is 0, or the protected tokens are b
      *(Bins *)(s_bins + kBinsEach * tid) = Bins{};
      __syncthreads();
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (i * kRound >= n || !candidate(i, e)) continue;
          const uint32_t key = order_of(s[i][e]);
          if (pass == 0 || key >> (shift + bits) == cut >> (shift + bits)) atomicAdd(&s_bins[key >> shift & ((1u << bits) - 1)], 1);
        }
      __syncthreads();
      // the threads' bins from the highest down: the one where the running count reaches `want`
      const int low = kDigit - kBinsEach * (tid + 1);
      const Bins c = *(const Bins *)(s_bins + low);
      int total, sum = 0;
#pragma unroll
      for (int e = 0; e < kBinsEach; ++e) sum += c[e];
      int before = block_exclusive_scan<NT>(sum, s_scan, total);
#pragma unroll
      for (int e = kBinsEach - 1; e >= 0; --e) {
        if (before < want && before + c[e] >= want) {
          s_pick[0] = low + e;
          s_pick[1] = want - before;
          s_pick[2] = c[e];
        }
        before += c[e];
      }
      __syncthreads();
      cut |= (uint32_t)s_pick[0] << shift;
      want = s_pick[1];
      equal = s_pick[2];
    }
    // of the tokens equal to the cut the first `want` stay
    uint32_t ties = 0;
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (!there(i, e)) continue;
        const uint32_t bit = 1u << (4 * i + e), key = order_of(s[i][e]);
        if (!candidate(i, e)) keep |= safe & bit;
        else if (equal > 0 && key >= cut) (key == cut ? ties : keep) |= bit;
      }
    int count[R], before[R];
    if (want < equal) {
#pragma unroll
      for (int i = 0; i < R; ++i) count[i] = __popc(ties >> (4 * i) & 15u);
      ordered_scan<NT, R>(count, before, s_scan);
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t bit = 1u << (4 * i + e);
          if ((ties & bit) != 0 && before[i]++ < want) keep |= bit;
        }
    } else {
      keep |= ties;
    }
    // freed slots and survivors behind them, each in slot order
    uint32_t hole = 0, late = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = i * kRound + 4 * tid + e;
        const uint32_t bit = 1u << (4 * i + e);
        if (j < b && !(keep & bit)) hole |= bit;
        if (j >= b && (keep & bit) != 0) late |= bit;
      }
      count[i] = __popc(hole >> (4 * i) & 15u) | __popc(late >> (4 * i) & 15u) << 16;
    }
    const int moved = ordered_scan<NT, R>(count, before, s_scan) & 0xffff;  // as many survivors as freed slots
#pragma unroll
    for (int i = 0; i < R; ++i) {
      int free = before[i] & 0xffff, come = before[i] >> 16;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = i * kRound + 4 * tid + e;
        if (hole >> (4 * i + e) & 1) s_to[free++] = (uint16_t)j;
        if (late >> (4 * i + e) & 1) s_from[come++] = (uint16_t)j;
      }
    }
    __syncthreads();
    // survivors to their new slots, the others where they are, nothing behind the budget
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int j = i * kRound + 4 * tid;
      int come = before[i] >> 16;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (late >> (4 * i + e) & 1) {
          const int to = s_to[come++];
          new_scores[to] = s[i][e];
          new_positions[to] = at[i][e];
        }
      const uint32_t holes = hole >> (4 * i) & 15u;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (j + e >= b) {
          s[i][e] = 0.f;
          at[i][e] = -1;
        }
      if (j + 4 <= p.capacity && holes == 0) {
        if (j >= b || new_scores != scores || j + 4 > b) *(Float4 *)(new_scores + j) = s[i];
        if (j >= b || new_positions != positions || j + 4 > b) *(Int4 *)(new_positions + j) = at[i];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (j + e < p.capacity && !(holes >> e & 1)) {
            new_scores[j + e] = s[i][e];
            new_positions[j + e] = at[i][e];
          }
      }
    }
    if (COPY) {
      copy_rows<NT>(p, row, head, moved, 0, 1, [&](int k) { return make_int2(s_from[k], s_to[k]); });
    } else {
      int2 *moves = p.moves + (int64_t)segment * p.half;
      for (int k = tid; k < moved; k += NT) moves[k] = make_int2(s_from[k], s_to[k]);
      if (tid == 0) p.count[segment] = moved;
    }
  } else {  // everything stays
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int j = i * kRound + 4 * tid;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (j + e >= n) at[i][e] = -1;  // the score is 0
      if (j + 4 <= p.capacity) {
        if (j + 4 > n || new_scores != scores) *(Float4 *)(new_scores + j) = s[i];
        if (j + 4 > n || new_positions != positions) *(Int4 *)(new_positions + j) = at[i];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (j + e < p.capacity) {
            new_scores[j + e] = s[i][e];
            new_positions[j + e] = at[i][e];
          }
      }
    }
    if (!COPY && tid == 0) p.count[segment] = 0;
  }
  if (tid == 0 && head == 0) p.new_lens[row] = b;
}

// -- longer rows -----------------------------------------------------------------------------------------

__global__ __launch_bounds__(kThreads) void stream_kernel(const Params p) {
  __shared__ int s_bins[kBins];
  __shared__ int s_scan[kThreads / kWave];
  __shared__ int s_pick[2];
  const int segment = blockIdx.x, row = segment / p.heads, head = segment - row * p.heads;
  const int tid = threadIdx.x;
  const int n = min(max(p.lens[row], 0), p.capacity);
  const int b = min(n, max(p.budget != nullptr ? p.budget[row] : p.fixed_budget, 0));
  const int64_t newest = (int64_t)p.seen[row] - p.recent;
  const float *scores = p.scores + (int64_t)row * p.s_row + (int64_t)head * p.s_head;
  const int32_t *positions = p.positions + (int64_t)row * p.p_row + (int64_t)head * p.p_head;
  float *new_scores = p.new_scores + (int64_t)row * p.ns_row + (int64_t)head * p.ns_head;
  int32_t *new_positions = p.new_positions + (int64_t)row * p.np_row + (int64_t)head * p.np_head;
  int2 *moves = p.moves + (int64_t)segment * p.half;

  int moved = 0;
  if (b < n) {
    // the class that the cut falls into: the protected tokens if there are b of them or more
    int mine = 0;
    for (int j = tid; j < n; j += kThreads) mine += is_protected(p, positions[j], newest);
    const int safe = block_sum<kThreads, int>(mine, s_scan);
    const bool among_safe = safe >= b;
    // the `want`-th highest key of that class, digit by digit
    int want = among_safe ? b : b - safe;
    uint32_t cut = 0;
    for (int shift = 24; shift >= 0 && want > 0; shift -= 8) {
      for (int i = tid; i < kBins; i += kThreads) s_bins[i] = 0;
      __syncthreads();
      for (int j = tid; j < n; j += kThreads) {
        if (is_protected(p, positions[j], newest) != among_safe) continue;
        const uint32_t key = order_of(scores[j]);
        if (shift == 24 || (key >> (shift + 8)) == (cut >> (shift + 8))) atomicAdd(&s_bins[key >> shift & 255u], 1);
      }
      __syncthreads();
      // bins from the highest down: the one where the running count reaches `want`
      const int bin = kBins - 1 - tid;
      const int c = tid < kBins ? s_bins[bin] : 0;
      int total;
      const int before = block_exclusive_scan<kThreads>(c, s_scan, total);
      if (before < want && before + c >= want) {
        s_pick[0] = bin;
        s_pick[1] = want - before;
      }
      __syncthreads();
      cut |= (uint32_t)s_pick[0] << shift;
      want = s_pick[1];
      __syncthreads();
    }
    // survivors and freed slots in slot order; of the keys equal to the cut the first `want` stay
    int equal = 0, freed = 0, late = 0;
    for (int base = 0; base < n; base += kThreads) {
      const int j = base + tid;
      bool kept = false, tie = false;
      if (j < n) {
        const bool s = is_protected(p, positions[j], newest);
        const uint32_t key = order_of(scores[j]);
        if (s != among_safe) kept = s;
        else if (b > 0) {
          kept = key > cut;
          tie = key == cut;
        }
      }
      int total;
      const int rank = block_exclusive_scan<kThreads>(tie ? 1 : 0, s_scan, total);
      if (tie && equal + rank < want) kept = true;
      equal += total;
      if (kept && j < b) keep_in_place(p, j, scores, positions, new_scores, new_positions);
      const bool hole = j < b && !kept, survivor = j >= b && j < n && kept;
      const int both = block_exclusive_scan<kThreads>((hole ? 1 : 0) | (survivor ? 1 << 16 : 0), s_scan, total);
      if (hole) moves[freed + (both & 0xffff)].y = j;
      if (survivor) moves[late + (both >> 16)].x = j;
      freed += total & 0xffff;
      late += total >> 16;
    }
    moved = freed;  // as many survivors behind b as slots freed below it
  } else {
    for (int j = tid; j < n; j += kThreads) keep_in_place(p, j, scores, positions, new_scores, new_positions);
  }
  __syncthreads();
  for (int k = tid; k < moved; k += kThreads) {
    const int2 m = moves[k];
    new_scores[m.y] = scores[m.x];
    new_positions[m.y] = positions[m.x];
  }
  __syncthreads();  // in place, the survivors are read before the slots behind b are cleared
  for (int j = b + tid; j < p.capacity; j += kThreads) {
    new_scores[j] = 0.f;
    new_positions[j] = -1;
  }
  if (tid == 0) {
    p.count[segment] = moved;
    if (head == 0) p.new_lens[row] = b;
  }
}

// The moves that were listed, several workgroups a segment.
__global__ __launch_bounds__(kMoveThreads) void move_kernel(const Params p) {
  const int segment = blockIdx.x, row = segment / p.heads, head = segment - row * p.heads;
  const int2 *moves = p.moves + (int64_t)segment * p.half;
  copy_rows<kMoveThreads>(p, row, head, p.count[segment], blockIdx.y, gridDim.y, [&](int k) { return moves[k]; });
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

template <int NT, int R>
void launch_select(const Params &p, bool copy, dim3 grid, hipStream_t stream) {
  if (copy) hipLaunchKernelGGL((select_kernel<NT, R, true>), grid, dim3(NT), 0, stream, p);
  else hipLaunchKernelGGL((select_kernel<NT, R, false>), grid, dim3(NT), 0, stream, p);
}

size_t workspace_bytes(int64_t segments, int64_t capacity) {
  return (size_t)(ceil_div(segments * 4, 256) * 256 + segments * (capacity / 2) * 8);
}

}  // namespace evict
}  // namespace ekv

using namespace ekv;

extern "C" size_t ekv_evict_tokens_workspace(int32_t rows, int32_t kv_heads, int32_t capacity) {
  if (rows < 0 || kv_heads < 1 || capacity < 0) return 0;
  return evict::workspace_bytes((int64_t)rows * kv_heads, capacity);
}

extern "C" int ekv_evict_tokens(const ekv_eviction_t *a, void *workspace, size_t workspace_bytes, void *stream) {
  const char *who = "ekv_evict_tokens";
  if (a == nullptr) return fail(EKV_EINVAL, "%s: null argument block", who);
  const int bytes = a->kv_dtype == EKV_F32 ? 4 : a->kv_dtype == EKV_F16 || a->kv_dtype == EKV_BF16 ? 2
                    : a->kv_dtype == EKV_FP8_E4M3 ? 1 : 0;
  if (bytes == 0) return fail(EKV_EUNSUPPORTED, "%s: element type %d", who, a->kv_dtype);
  if (a->head_dim != 32 && a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256)
    return fail(EKV_EUNSUPPORTED, "%s: head dim %d (32, 64, 128 or 256)", who, a->head_dim);
  if (a->rows < 0 || a->kv_heads < 1 || a->width < 0 || a->block_size < 1 || a->blocks < 0 || a->recent < 0 ||
      a->sinks < 0 || (a->budget == nullptr && a->fixed_budget < 0))
    return fail(EKV_EINVAL, "%s: rows %d, heads %d, width %d, block size %d, budget %d, recent %d, sinks %d", who,
                a->rows, a->kv_heads, a->width, a->block_size, a->fixed_budget, a->recent, a->sinks);
  const int64_t capacity = (int64_t)a->width * a->block_size, segments = (int64_t)a->rows * a->kv_heads;
  if (capacity >= INT32_MAX)
    return fail(EKV_EINVAL, "%s: a table of %d blocks of %d tokens passes 2^31", who, a->width, a->block_size);
  if (segments >= (1 << 23)) return fail(EKV_EINVAL, "%s: %d rows of %d heads", who, a->rows, a->kv_heads);
  if (a->rows == 0) return EKV_OK;
  if (a->lens == nullptr || a->seen == nullptr || a->new_lens == nullptr ||
      (a->width > 0 && (a->table == nullptr || a->keys == nullptr || a->values == nullptr || a->scores == nullptr ||
                        a->positions == nullptr || a->new_scores == nullptr || a->new_positions == nullptr)))
    return fail(EKV_EINVAL, "%s: null pointer", who);
  if (a->new_lens == a->lens) return fail(EKV_EINVAL, "%s: the new lengths may not overwrite the old ones", who);
  if (a->table_stride < a->width) return fail(EKV_EINVAL, "%s: table rows of %d blocks, stride %lld", who, a->width,
                                              (long long)a->table_stride);
  if (((uintptr_t)a->keys | (uintptr_t)a->values) % 16 || a->kv_stride_block * bytes % 16 ||
      a->kv_stride_pos * bytes % 16 || a->kv_stride_head * bytes % 16)
    return fail(EKV_EINVAL, "%s: key and value rows start at multiples of 16 bytes", who);
  const size_t need = evict::workspace_bytes(segments, capacity);
  if (workspace == nullptr || workspace_bytes < need || (uintptr_t)workspace % 16)
    return fail(EKV_EINVAL, "%s: a workspace of %zu bytes, %zu needed at a multiple of 16", who, workspace_bytes, need);
  evict::Params p{};
  p.table = a->table;
  p.table_stride = a->table_stride;
  p.lens = a->lens;
  p.budget = a->budget;
  p.seen = a->seen;
  p.scores = a->scores;
  p.positions = a->positions;
  p.s_row = a->scores_stride_row;
  p.s_head = a->scores_stride_head;
  p.p_row = a->positions_stride_row;
  p.p_head = a->positions_stride_head;
  p.new_scores = a->new_scores;
  p.new_positions = a->new_positions;
  p.ns_row = a->new_scores_stride_row;
  p.ns_head = a->new_scores_stride_head;
  p.np_row = a->new_positions_stride_row;
  p.np_head = a->new_positions_stride_head;
  p.new_lens = a->new_lens;
  p.k = (char *)a->keys;
  p.v = (char *)a->values;
  p.st_block = a->kv_stride_block * bytes;
  p.st_pos = a->kv_stride_pos * bytes;
  p.st_head = a->kv_stride_head * bytes;
  p.blocks = a->blocks;
  p.count = (int32_t *)workspace;
  p.moves = (int2 *)((char *)workspace + evict::ceil_div(segments * 4, 256) * 256);
  p.rows = a->rows;
  p.heads = a->kv_heads;
  p.width = a->width;
  p.block_size = a->block_size;
  p.capacity = (int)capacity;
  p.half = (int)(capacity / 2);
  p.fixed_budget = a->fixed_budget;
  p.recent = a->recent;
  p.sinks = a->sinks;
  p.row_bytes = a->head_dim * bytes;
  const PageDivisor d = page_divisor(a->block_size);
  p.bs_mul = d.mul;
  p.bs_shift = d.shift;
  hipStream_t s = (hipStream_t)stream;
  // A workgroup copies its own moves unless there are too few of them for the rows that may move.
  const bool copy = segments >= 2 * (int64_t)cu_count() || capacity * p.row_bytes <= 512 << 10;
  const bool held = capacity <= 16384;
  const dim3 grid((unsigned)segments);
  if (!held) hipLaunchKernelGGL(evict::stream_kernel, grid, dim3(evict::kThreads), 0, s, p);
  else if (capacity <= 2048) evict::launch_select<512, 1>(p, copy, grid, s);
  else if (capacity <= 4096) evict::launch_select<512, 2>(p, copy, grid, s);
  else if (capacity <= 6144) evict::launch_select<512, 3>(p, copy, grid, s);
  else if (capacity <= 8192) evict::launch_select<512, 4>(p, copy, grid, s);
  else evict::launch_select<1024, 4>(p, copy, grid, s);
  int rc = check_hip(hipGetLastError(), "ekv_evict_tokens select launch");
  if (rc != EKV_OK || capacity < 2 || (held && copy)) return rc;
  // workgroups a segment: enough to fill the chip, no more than its longest list has work for
  const int64_t per = evict::kMoveThreads / (p.row_bytes / 16);
  int64_t y = evict::ceil_div(16 * (int64_t)cu_count(), segments);
  const int64_t most = evict::ceil_div(p.half, 4 * per);
  y = y > most ? most : y;
  hipLaunchKernelGGL(evict::move_kernel, dim3((unsigned)segments, (unsigned)y), dim3(evict::kMoveThreads), 0, s, p);
  return check_hip(hipGetLastError(), "ekv_evict_tokens move launch");
}
