// Shared by the attention kernels over the paged cache: the call's parameters, the page lookup, the
// element types' loads and matrix products, and the segments of work.
#pragma once

#include "ekv_common.hpp"

namespace ekv {
namespace attn {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kRowsPerTile = 16;  // query rows of one narrow tile (the matrix instruction's columns)
constexpr int kWideRows = 64;     // from so many query rows a set of keys on, the wide kernel
constexpr int kMaxSlots = 64;     // partial results a query row can have from its own pages, and from its prefix

struct Params {
  const char *q;
  int64_t q_st, q_sh;  // elements
  const char *k, *v;
  int64_t st_block, st_pos, st_head;  // elements
  int64_t blocks;
  const int32_t *table;
  int64_t table_stride;
  const int32_t *lens, *q_start;
  const int32_t *ptable;
  int64_t ptable_stride;
  const int32_t *plens, *prows;
  float *scores;
  int64_t sc_row, sc_head;
  char *out;
  int64_t o_st, o_sh;
  float *lse;
  float *part_o;   // [slots][tokens][q_heads][head_dim], unnormalised
  float2 *part_ml;  // [slots][tokens][q_heads]: maximum (in powers of two) and sum
  int rows, width, groups, pwidth, tokens, max_query, q_heads, kv_heads, group, block_size;
  uint32_t bs_mul;  // page_divisor(block_size)
  int bs_shift;
  float scale2, v_scale, decay;  // scale2: scale * k_scale * log2(e)
  // the split: own pages in s_own chunks of chunk_own keys, prefixes in s_pre chunks of chunk_pre
  int chunk_own, s_own, tiles_own, chunk_pre, s_pre, tiles_pre;
  int tile_own, tile_pre;  // query rows of a tile
  int64_t items_own, items_pre;
  // wide_own: the own keys of a row go through the wide kernel, behind its prefix's on one axis (no items of
  // the prefix's own); wide_pre: the prefixes do.  direct: one chunk holds everything a query sees, so the
  // wide kernel writes the result.
  bool wide_own, wide_pre, direct;
};

__device__ __forceinline__ int page_of(const Params &p, int pos) {
  return (int)(__umulhi((uint32_t)pos << 1, p.bs_mul) >> p.bs_shift);
}

// -- element types --------------------------------------------------------------------------------
//
// A key row is the A operand of the matrix product S^T = K Q^T: lane l holds key l % 16 and, of its
// head_dim elements, those of its lane group g = l / 16.  The contraction runs over all of them, so
// which dims a lane group holds is free as long as the query operand agrees: each takes whole 16-byte
// pieces.  Products of 16-bit (and fp8, converted exactly to bf16) elements are exact in the float32
// they are summed in.

struct F32 {
  static constexpr int kType = EKV_F32;
  static constexpr int kBytes = 4;
  static constexpr int kStepDims = 4;  // dims of one matrix instruction
  typedef float Query;
};
struct F16 {
  static constexpr int kType = EKV_F16;
  static constexpr int kBytes = 2;
  static constexpr int kStepDims = 32;
  typedef _Float16 Query;
};
struct BF16 {
  static constexpr int kType = EKV_BF16;
  static constexpr int kBytes = 2;
  static constexpr int kStepDims = 32;
  typedef __bf16 Query;
};
struct FP8 {  // keys and values e4m3, queries bf16
  static constexpr int kType = EKV_FP8_E4M3;
  static constexpr int kBytes = 1;
  static constexpr int kStepDims = 32;
  typedef __bf16 Query;
};

// 8 consecutive e4m3 values as bf16: both formats hold them exactly
__device__ __forceinline__ bf16x8 widen(uint32_t lo, uint32_t hi) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, 1.0f, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, 1.0f, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, 1.0f, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, 1.0f, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// element j of the dwords at w, as float32
template <class T>
__device__ __forceinline__ float element(const uint32_t *w, int j) {
  if constexpr (std::is_same<T, F32>::value) {
    return __builtin_bit_cast(float, w[j]);
  } else if constexpr (std::is_same<T, BF16>::value) {
    return __builtin_bit_cast(float, (j & 1) ? (w[j / 2] & 0xffff0000u) : (w[j / 2] << 16));
  } else if constexpr (std::is_same<T, F16>::value) {
    const f16x2 h = __builtin_bit_cast(f16x2, w[j / 2]);
    return (float)h[j & 1];
  } else {
    const f32x2 f = (j & 2) ? __builtin_amdgcn_cvt_pk_f32_fp8((int)w[j / 4], true)
                            : __builtin_amdgcn_cvt_pk_f32_fp8((int)w[j / 4], false);
    return f[j & 1];
  }
}

// BYTES (2, 4, 8 or a multiple of 16) from global memory into dwords
template <int BYTES>
__device__ __forceinline__ void load_bytes(const char *src, uint32_t *dst) {
  if constexpr (BYTES == 2) {
    dst[0] = *as_global((const uint16_t *)src);
  } else if constexpr (BYTES == 4) {
    dst[0] = *as_global((const uint32_t *)src);
  } else if constexpr (BYTES == 8) {
    const u32x2 x = *as_global((const u32x2 *)src);
    dst[0] = x[0];
    dst[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const u32x4 x = *as_global((const u32x4 *)(src + 16 * i));
#pragma unroll
      for (int e = 0; e < 4; ++e) dst[4 * i + e] = x[e];
    }
  }
}

// The first dim of the 8 (16-bit, fp8) or 4 (float32) that lane group g supplies in piece c of a row.
template <class T, int D>
__device__ __forceinline__ int piece_dim(int c, int g) {
  if constexpr (std::is_same<T, F32>::value) return c * 16 + g * 4;
  else if constexpr (std::is_same<T, FP8>::value && D >= 64) return (c / 2) * 64 + g * 16 + (c & 1) * 8;
  else return c * 32 + g * 8;
}
template <class T, int D>
constexpr int kPieces = std::is_same<T, F32>::value ? D / 16 : D / 32;

// The lane's part of one key row: D / 4 elements.
template <class T, int D>
struct KeyRow {
  static constexpr int kLoad = (std::is_same<T, FP8>::value && D == 32) ? 8 : 16;  // bytes of a load
  static constexpr int kLoads = D * T::kBytes / 4 / kLoad;
  uint32_t w[D * T::kBytes / 16];
  __device__ __forceinline__ void load(const char *row, int g) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load_bytes<kLoad>(row + (i * 4 + g) * kLoad, w + i * kLoad / 4);
  }
};

// The lane's part of one query row, in the order of the key rows' pieces.
template <class T, int D>
struct QueryRow {
  static constexpr int kDwords = std::is_same<T, F32>::value ? D / 4 : D / 8;
  uint32_t w[kDwords];
  __device__ __forceinline__ void load(const char *row, int g, bool live) {
    constexpr int E = sizeof(typename T::Query);
#pragma unroll
    for (int c = 0; c < kPieces<T, D>; ++c) {
      if (live) load_bytes<16>(row + piece_dim<T, D>(c, g) * E, w + 4 * c);
      else w[4 * c] = w[4 * c + 1] = w[4 * c + 2] = w[4 * c + 3] = 0;
    }
  }
};

// S^T of 16 keys and 16 query rows: lane l receives keys 4 * (l / 16) + i of query row l % 16.
template <class T, int D>
__device__ __forceinline__ f32x4 dot_tile(const KeyRow<T, D> &k, const QueryRow<T, D> &q) {
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < kPieces<T, D>; ++c) {
    if constexpr (std::is_same<T, F32>::value) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, k.w[4 * c + e]),
                                                   __builtin_bit_cast(float, q.w[4 * c + e]), acc, 0, 0, 0);
    } else if constexpr (std::is_same<T, FP8>::value) {
      const bf16x8 a = widen(k.w[2 * c], k.w[2 * c + 1]);
      const bf16x8 b = __builtin_bit_cast(bf16x8, u32x4{q.w[4 * c], q.w[4 * c + 1], q.w[4 * c + 2], q.w[4 * c + 3]});
      acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0);
    } else {
      const u32x4 ka = {k.w[4 * c], k.w[4 * c + 1], k.w[4 * c + 2], k.w[4 * c + 3]};
      const u32x4 qb = {q.w[4 * c], q.w[4 * c + 1], q.w[4 * c + 2], q.w[4 * c + 3]};
      if constexpr (std::is_same<T, BF16>::value)
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, ka), __builtin_bit_cast(bf16x8, qb),
                                                      acc, 0, 0, 0);
      else
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, ka), __builtin_bit_cast(f16x8, qb), acc,
                                                     0, 0, 0);
    }
  }
  return acc;
}

// -- segments of work -------------------------------------------------------------------------------

// A row's query tokens: [first, first + count), all of them within the call's tokens.
struct RowQueries {
  int first, count;
};
__device__ __forceinline__ RowQueries row_queries(const Params &p, int row) {
  if (p.q_start == nullptr) return {row, 1};
  const int a = min(max(p.q_start[row], 0), p.tokens);
  const int b = min(max(p.q_start[row + 1], a), p.tokens);
  return {a, b - a};
}
__device__ __forceinline__ int row_length(const Params &p, int row) {
  return min(max(p.lens[row], 0), p.width * p.block_size);  // the host keeps width * block_size below 2^31
}
// The token ranges and lengths of the prefix groups.
__device__ __forceinline__ RowQueries group_queries(const Params &p, int g) {
  int r0 = 0, r1 = p.rows;
  if (p.prows != nullptr) {
    r0 = min(max(p.prows[g], 0), p.rows);
    r1 = min(max(p.prows[g + 1], r0), p.rows);
  }
  if (p.q_start == nullptr) return {r0, r1 - r0};
  const int a = min(max(p.q_start[r0], 0), p.tokens);
  const int b = min(max(p.q_start[r1], a), p.tokens);
  return {a, b - a};
}
__device__ __forceinline__ int group_length(const Params &p, int g) {
  return min(max(p.plens[g], 0), p.pwidth * p.block_size);
}

// The group of a row, or -1.
__device__ __forceinline__ int group_of(const Params &p, int row) {
  if (p.groups == 0) return -1;
  if (p.prows == nullptr) return 0;
  if (row < p.prows[0] || row >= p.prows[p.groups]) return -1;
  int lo = 0, hi = p.groups;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.prows[mid] <= row) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Group and tile of tile number `index` when every group's queries are cut into tiles of `rows` query
// rows; false past the last.  All 64 lanes call it with one index and receive one answer.
__device__ __forceinline__ bool find_tile(const Params &p, int index, int rows, int &g, int &tile) {
  int before = 0;
  for (int base = 0; base < p.groups; base += kWave) {
    const int mine = base + lane_id();
    int n = 0;
    if (mine < p.groups) {
      const RowQueries t = group_queries(p, mine);
      n = (int)(((int64_t)t.count * p.group + rows - 1) / rows);
    }
    const int inc = wave_inclusive_scan(n);
    const uint64_t past = __ballot(before + inc > index);
    if (past != 0) {
      const int lane = __builtin_ctzll(past);
      g = base + lane;
      tile = index - before - __shfl(inc - n, lane);
      return true;
    }
    before += __builtin_amdgcn_readlane(inc, kWave - 1);
  }
  return false;
}

// The wide kernel (16-bit and fp8 keys): query rows of its tiles, and the launch over the own keys or the prefixes.
int wide_tile_rows();
int wide_attention(const Params &p, int kv_dtype, int head_dim, bool own, hipStream_t stream);

}  // namespace attn
}  // namespace ekv
