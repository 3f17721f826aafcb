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
// Two kernels: select_kernel finds the survivors, lists the moves and writes scores, positions and lengths;
// move_kernel copies the keys and values of the listed tokens.
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

__global__ __launch_bounds__(kThreads) void select_kernel(const Params p) {
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

// The key and value rows of the listed tokens, 16 bytes a thread.  A slot whose table entry is no page of
// the cache is not read or written.
__global__ __launch_bounds__(kMoveThreads) void move_kernel(const Params p) {
  const int segment = blockIdx.x, row = segment / p.heads, head = segment - row * p.heads;
  const int pieces = p.row_bytes / 16;  // a power of two, 2 to 64
  const int count = p.count[segment];
  const int per = kMoveThreads / pieces, piece = threadIdx.x % pieces;
  const int32_t *table = p.table + (int64_t)row * p.table_stride;
  const int2 *moves = p.moves + (int64_t)segment * p.half;
  for (int k = blockIdx.y * per + threadIdx.x / pieces; k < count; k += gridDim.y * per) {
    const int2 m = moves[k];
    const int from = page_of(p, m.x), to = page_of(p, m.y);
    const int a = table[from], b = table[to];
    if ((uint32_t)a >= (uint64_t)p.blocks || (uint32_t)b >= (uint64_t)p.blocks) continue;
    const int64_t src = (int64_t)a * p.st_block + (int64_t)(m.x - from * p.block_size) * p.st_pos + head * p.st_head;
    const int64_t dst = (int64_t)b * p.st_block + (int64_t)(m.y - to * p.block_size) * p.st_pos + head * p.st_head;
    const uint4 x = *(const uint4 *)(p.k + src + piece * 16), y = *(const uint4 *)(p.v + src + piece * 16);
    *(uint4 *)(p.k + dst + piece * 16) = x;
    *(uint4 *)(p.v + dst + piece * 16) = y;
  }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

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
  hipLaunchKernelGGL(evict::select_kernel, dim3((unsigned)segments), dim3(evict::kThreads), 0, s, p);
  int rc = check_hip(hipGetLastError(), "ekv_evict_tokens select launch");
  if (rc != EKV_OK || capacity < 2) return rc;
  // workgroups a segment: enough to fill the chip, no more than its longest list has work for
  const int64_t per = evict::kMoveThreads / (p.row_bytes / 16);
  int64_t y = evict::ceil_div(16 * (int64_t)cu_count(), segments);
  const int64_t most = evict::ceil_div(p.half, per);
  y = y > most ? most : y;
  hipLaunchKernelGGL(evict::move_kernel, dim3((unsigned)segments, (unsigned)y), dim3(evict::kMoveThreads), 0, s, p);
  return check_hip(hipGetLastError(), "ekv_evict_tokens move launch");
}
