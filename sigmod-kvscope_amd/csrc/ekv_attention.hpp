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
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kRowsPerTile = 16;  // query rows of one narrow tile (the matrix instruction's columns)
// From so many query rows a set of keys on (a row's own keys, a group's prefix), the wide kernel: it reads the keys once
// where the narrow one reads them once for each 16 rows.  Own keys alone, 64 rows of 1000 to 4000 tokens with 20, 32, 48 and
// 60 query rows a KV head: 163, 160, 167 and 167 us against the narrow kernel's 251, 257, 277 and 359; at head dim 256, where
// the narrow kernel streams and the wide one has one workgroup a compute unit, 538 us with 20 to 64 query rows against 474,
// 477 (32), 513 (48) and 663 (64).
constexpr int kWideRows = 17, kWideRows256 = 64;
// The running weights: a workgroup for 64 keys from so many query rows on, where a wave for 64 keys would leave the chip
// unfilled (2 rows of 1000 to 4000 tokens: 70, 98, 157 and 219 us with 512, 1024, 2048 and 4000 query rows a KV head, 74,
// 119, 207 and 343 us with a wave; 55 against 51 with 256; 32 rows, 2048: 1425 against 1357).
constexpr int kWeighWide = 512, kWeighWaves = 16;  // query rows, waves a compute unit
constexpr int kMostKeys = INT32_MAX - 4095;  // of a table row: a step past its last key is still an int
constexpr int kMaxSlots = 128;    // partial results a query row can have from the equal shares of its own keys
constexpr int kMaxChunks = 64;    // and from chunks of keys

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
  float *logits;   // [rows][kv_heads][logit_rows][logit_stride], in powers of two, or null
  int64_t logit_stride;
  int logit_rows;
  int rows, width, groups, pwidth, tokens, max_query, q_heads, kv_heads, group, block_size;
  uint32_t bs_mul;  // page_divisor(block_size)
  int bs_shift;
  float scale2, v_scale, decay;  // scale2: scale * k_scale * log2(e)
  int32_t *row_slots;  // [rows]: the slots that a row's own keys have partial results in (narrow kernel)
  // the split: at most s_own slots for the own keys (wide kernel: chunks of chunk_own keys; narrow kernel: the
  // pieces of `share` waves a head and tile, waves_own in all), prefixes in s_pre chunks of chunk_pre (wide
  // kernel: in at most s_pre pieces of share_pre workgroups a head)
  int32_t *pre_slots;  // [tokens * group]: the slots that a query row's prefix has partial results in (wide kernel)
  int share, share_pre;
  int64_t waves_own;
  int chunk_own, s_own, tiles_own, chunk_pre, s_pre, tiles_pre;
  int tile_own, tile_pre;  // query rows of a tile
  bool packed;             // own items are the tiles that rows have, not the most that one can have for each row
  int64_t items_own, items_pre;
  // wide_own: the own keys of a row go through the wide kernel; wide_pre: the prefixes do, each for all queries of
  // its group.  wide_own alone: a row's tiles walk its prefix ahead of the own keys, on one axis.  direct: one chunk
  // holds everything a query sees, so the wide kernel writes the result.
  bool wide_own, wide_pre, direct;
  bool whole;  // 16 slots from a multiple of 16 on lie in one page, at offsets below 2^31
};

__device__ __forceinline__ int page_of(const Params &p, int pos) {
  return (int)(__umulhi((uint32_t)pos << 1, p.bs_mul) >> p.bs_shift);
}

// -- element types --------------------------------------------------------------------------------
//
// Keys and values meet the matrix instructions out of LDS: fp8 ones are widened to bf16 on the way there,
// which holds them exactly, the others keep their type.  Products of 16-bit elements are exact in the float32
// they are summed in.

// kLift: weights are 2^kLift times what they are against the running maximum, and so is their sum.  f16 has no values below
// 2^-24, and steps of that below 2^-14: lifted to its upper end the weights keep their relative rounding down to 2^-29 and
// are lost only below 2^-40.
template <class H>
constexpr float kLift = 0.f;
template <>
inline constexpr float kLift<_Float16> = 15.f;
// From so large logits on (in powers of two) float32's steps are too coarse to tell weights apart by, and nothing is lifted:
// a lift that is rounded up passes f16's largest value.
constexpr float kFar = 0x1p20f;
// Below this the rounding of a logit is less than half a step of f16 in its weight.
constexpr float kRounded = 0x1p12f;
// What the weights beside the largest logit `high` are against.
template <class H>
__device__ __forceinline__ float lifted(float high, float lift) {
  if constexpr (kLift<H> == 0.f) return high;
  return fabsf(high) < kFar ? high - lift : high;
}

struct F32 {
  static constexpr int kType = EKV_F32;
  static constexpr int kBytes = 4;  // of an element in the cache
  static constexpr int kLds = 4;    // and in LDS
  typedef float Query;
  typedef float Half;
};
struct F16 {
  static constexpr int kType = EKV_F16;
  static constexpr int kBytes = 2;
  static constexpr int kLds = 2;
  typedef _Float16 Query;
  typedef _Float16 Half;  // the 16-bit type that keys, values and weights meet in
};
struct BF16 {
  static constexpr int kType = EKV_BF16;
  static constexpr int kBytes = 2;
  static constexpr int kLds = 2;
  typedef __bf16 Query;
  typedef __bf16 Half;
};
struct FP8 {  // keys and values e4m3, queries bf16
  static constexpr int kType = EKV_FP8_E4M3;
  static constexpr int kBytes = 1;
  static constexpr int kLds = 2;
  typedef __bf16 Query;
  typedef __bf16 Half;
};

// 8 consecutive e4m3 values as bf16: both formats hold them exactly
__device__ __forceinline__ u32x4 widen(uint32_t lo, uint32_t hi) {
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, 1.0f, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, 1.0f, true)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, 1.0f, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, 1.0f, true))};
}

// two weights as 16-bit ones
__device__ __forceinline__ uint32_t pack2(float a, float b, __bf16) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, _Float16) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), f16x2));
}

// products of 16 or 32 rows and columns over 32 or 16 of the contracted index
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c, __bf16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c, _Float16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c, __bf16) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c, _Float16) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// 16 x 16 over the 16 (float32) or 32 elements that one 16-byte piece a lane holds
template <class T>
__device__ __forceinline__ f32x4 dot_piece(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (std::is_same<T, F32>::value) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], c, 0, 0, 0);
    return c;
  } else {
    return mfma16(a, b, c, typename T::Half{});
  }
}

// Keys and values of a step in LDS, row by row.  The 16-byte pieces of a key row are permuted by the row's number
// so that the reads of one piece of 16 (32) rows meet every bank; the 32-byte pieces of a 16-bit value row so that
// the transposing reads, 4 (8) rows of 64 (32) bytes for half a wave, do.
template <class T, int D>
struct Lds {
  static constexpr int kRow = D * T::kLds;
  static constexpr int kLine = kRow < 256 ? 256 / kRow : 1;  // rows in 256 bytes
  __device__ static __forceinline__ int key_at(int row, int piece) {
    return row * kRow + (piece ^ (row / kLine & (kRow / 16 - 1) & 15)) * 16;
  }
  // the byte of a value row; the 16 from a multiple of 16 on are together
  __device__ static __forceinline__ int value_at(int row, int byte) {
    if constexpr (T::kLds == 4) return row * kRow + byte;
    const int chunk = byte / 64 ^ (row / kLine & (kRow / 64 - 1) & 3);
    return row * kRow + chunk * 64 + ((byte & 32) ^ (row & 4) * 8) + byte % 32;
  }
};

// The keys that a wave or workgroup reads, [begin, end) of one axis: a prefix's first, the own ones from `own` on, a
// multiple of 64 (between the two there are none), so that 16 keys from a multiple of 16 on are of one page where the
// block size is a multiple of 16.
struct Range {
  const int32_t *ptable, *table;
  int plen, own, begin, end, head;
};
__host__ __device__ __forceinline__ int own_begin(int plen) { return (plen + 63) / 64 * 64; }

// One step of KEYS keys and values on its way from memory through registers to LDS.  Loads take whole rows, 16
// bytes a lane, the form that memory serves fastest.  The pages come a step ahead of the rows, a lookup a lane:
// loads return in order, so a lookup right before its rows would wait for every row ahead of it.
template <class T, int D, int KEYS, int THREADS>
struct Stage {
  static constexpr int kPieces = D * T::kBytes / 16;  // 16-byte pieces of a row in memory
  static constexpr int kAll = KEYS * kPieces;
  static constexpr int kLoads = (kAll + THREADS - 1) / THREADS;  // of a thread, for K and for V
  static constexpr int kTile = KEYS * Lds<T, D>::kRow;           // LDS bytes of K, and of V
  typedef u32x4 Rows[kLoads];

  // the thread's i-th piece, and whether there is one (KEYS * pieces is a multiple of 64, so a wave agrees)
  __device__ static __forceinline__ bool piece(int i, int &row, int &col) {
    const int at = (THREADS == kWave ? lane_id() : (int)threadIdx.x) + i * THREADS;
    row = at / kPieces;
    col = at % kPieces;
    return kAll % THREADS == 0 || at < kAll;
  }
  // the page of this lane's key of the step at `base`; -1: there is none
  __device__ static __forceinline__ int look(const Params &p, const Range &s, int base) {
    const int at = base + lane_id() % KEYS;
    int page = -1;
    if (at < s.end && (at < s.plen || at >= s.own)) {
      const bool shared = at < s.plen;
      page = (shared ? s.ptable : s.table)[page_of(p, shared ? at : at - s.own)];
    }
    return page;
  }
  // the keys of a step that are there (KEYS below 64: again and again)
  __device__ static __forceinline__ uint64_t there(const Params &p, int page) {
    return __ballot((uint32_t)page < (uint64_t)p.blocks);
  }
  // where this lane's key of the step at `base` lies, in bytes; page 0's first slot for one that is not there
  __device__ static __forceinline__ int64_t place(const Params &p, const Range &s, int base, int page) {
    const int at = base + lane_id() % KEYS;
    const bool good = (uint32_t)page < (uint64_t)p.blocks;
    const int pos = good ? at < s.plen ? at : at - s.own : 0;
    return ((good ? page : 0) * p.st_block + (pos - page_of(p, pos) * p.block_size) * p.st_pos + s.head * p.st_head) * T::kBytes;
  }
  // Where the rows of one load are of one page (whole): its first row's place, a lane's offset from it the same in
  // every load.
  static constexpr bool kScalar = kWave / kPieces <= 16;
  __device__ static __forceinline__ int first_row(int i) {
    const int wave = THREADS == kWave ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    return (wave * kWave + i * THREADS) / kPieces;
  }
  __device__ static __forceinline__ int64_t place_of(int64_t place, int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)place, lane);
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(place >> 32), lane) << 32 | lo);
  }
  __device__ static __forceinline__ uint32_t lane_offset(const Params &p) {
    return (uint32_t)(lane_id() / kPieces) * (uint32_t)(p.st_pos * T::kBytes);
  }
  __device__ static __forceinline__ int64_t shuffled(int64_t place, int lane) {
    const uint32_t lo = __shfl((int)(uint32_t)place, lane);
    return (int64_t)((uint64_t)(uint32_t)__shfl((int)(place >> 32), lane) << 32 | lo);
  }
  // the rows at `place`, keys (from p.k) or values (from p.v)
  __device__ static __forceinline__ void load(const Params &p, int64_t place, const char *from, Rows &to) {
    if (kScalar && p.whole) {
      const uint32_t off = lane_offset(p) + lane_id() % kPieces * 16;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int first = first_row(i);
        if (kAll % THREADS != 0 && first >= KEYS) break;
        to[i] = fetch(from + place_of(place, first) + off);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        int row, col;
        if (!piece(i, row, col)) break;
        to[i] = fetch(from + shuffled(place, row) + col * 16);
      }
    }
  }
  __device__ static __forceinline__ u32x4 fetch(const char *from) {
    // a wave's rows are read once: the stream leaves the caches to others (2.3 GB of rows: 427 us, not 455)
    if constexpr (THREADS == kWave) return __builtin_nontemporal_load(as_global((const u32x4 *)from));
    else return *as_global((const u32x4 *)from);
  }
  __device__ static __forceinline__ void store_keys(const Rows &k, char *keys) {
    using L = Lds<T, D>;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      int row, col;
      if (!piece(i, row, col)) break;
      if constexpr (T::kBytes == 1) {
        *(u32x4 *)(keys + L::key_at(row, 2 * col)) = widen(k[i][0], k[i][1]);
        *(u32x4 *)(keys + L::key_at(row, 2 * col + 1)) = widen(k[i][2], k[i][3]);
      } else {
        *(u32x4 *)(keys + L::key_at(row, col)) = k[i];
      }
    }
  }
  // the values of keys that are not there as 0 (0 * NaN is no zero)
  __device__ static __forceinline__ void store_values(Rows &v, uint64_t ok, char *values) {
    using L = Lds<T, D>;
    if (ok != ~0ull) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        int row, col;
        if (!piece(i, row, col)) break;
        if (!(ok >> row & 1)) v[i] = u32x4{0, 0, 0, 0};
      }
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      int row, col;
      if (!piece(i, row, col)) break;
      if constexpr (T::kBytes == 1) {
        *(u32x4 *)(values + L::value_at(row, 32 * col)) = widen(v[i][0], v[i][1]);
        *(u32x4 *)(values + L::value_at(row, 32 * col + 16)) = widen(v[i][2], v[i][3]);
      } else {
        *(u32x4 *)(values + L::value_at(row, 16 * col)) = v[i];
      }
    }
  }
};

// Four values of one dim a lane out of LDS: in a group of 16 lanes, lane 4j + c gives the place of dims 4c .. 4c + 3
// of key j, and lane n receives dim n of the four keys.
__device__ __forceinline__ u32x2 read_transposed(const char *from) {
  typedef __attribute__((address_space(3))) s16x4 *Ptr;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(from)));
}

// A key's logit less its query's lse.  The weight, 2 to that power, is at most 1: where logits are so large that their
// roundings are whole powers of two, a difference above 0 is one of those.  NaN stays NaN.
__device__ __forceinline__ float below_one(float difference) { return __builtin_elementwise_minimum(difference, 0.f); }

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

// Of a list of tiles, entry after entry with tiles_of(entry) each, the entry that tile number `index` is in and its number
// there; false past the last.  All 64 lanes call it with one index and receive one answer.
template <class Tiles>
__device__ __forceinline__ bool find_tile(int entries, int index, Tiles tiles_of, int &entry, int &tile) {
  int64_t before = 0;
  for (int base = 0; base < entries; base += kWave) {
    const int mine = base + lane_id();
    const int n = mine < entries ? tiles_of(mine) : 0;
    const int inc = wave_inclusive_scan(n);
    const uint64_t past = __ballot(before + inc > index);
    if (past != 0) {
      const int lane = __builtin_ctzll(past);
      entry = base + lane;
      tile = (int)(index - before) - __builtin_amdgcn_readlane(inc - n, lane);
      return true;
    }
    before += __builtin_amdgcn_readlane(inc, kWave - 1);
  }
  return false;
}

// -- equal shares -------------------------------------------------------------------------------------
//
// A list of work is the units of its entries (rows, groups), one entry after the other; `share` workers take a
// stretch each, worker j units j total / share to (j + 1) total / share.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)x), hi = __builtin_amdgcn_readfirstlane((int)(x >> 32));
  return (int64_t)((uint64_t)hi << 32 | lo);
}

struct Share {
  int64_t total;
  int share;
  // the worker that unit x is with
  __device__ __forceinline__ int worker_of(int64_t x) const { return (int)(((x + 1) * share - 1) / total); }
};

// Every thread of the workgroup: the list's size, the workers that share it (at most `workers`, each with `least`
// units, and so many that a run of units that must not be cut into more than `slots` pieces is not), and for each of
// this workgroup's WORKERS workers, number worker(w) of all, the entry that its first unit is in and the units before
// that entry.  size(entry, run): its units, and the longest run in it.
template <int WAVES, int WORKERS, class Worker, class Size>
__device__ __forceinline__ Share share_out(int entries, int workers, int least, int slots, Worker worker, Size size,
                                           int *start_entry, int64_t *start_at) {
  constexpr int kN = WAVES * kWave;
  __shared__ int64_t s_sum[WAVES], s_max[WAVES];
  const int wave = threadIdx.x / kWave, per = (entries + kN - 1) / kN;
  const int e0 = min((int)threadIdx.x * per, entries), e1 = min(e0 + per, entries);
  int64_t mine = 0, longest = 0;
  for (int e = e0; e < e1; ++e) {
    int64_t run;
    mine += size(e, run);
    longest = max(longest, run);
  }
  int64_t inclusive = mine;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int64_t other = __shfl_up(inclusive, d);
    if (lane_id() >= d) inclusive += other;
    longest = max(longest, (int64_t)__shfl_xor(longest, d));
  }
  if (lane_id() == kWave - 1) s_sum[wave] = inclusive;
  if (lane_id() == 0) s_max[wave] = longest;
  __syncthreads();
  int64_t before = inclusive - mine, total = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    before += w < wave ? s_sum[w] : 0;
    total += s_sum[w];
    longest = max(longest, s_max[w]);
  }
  int64_t share = min((int64_t)workers, (total + least - 1) / least);
  // a run of u units meets at most u share / total + 2 workers
  if (longest > 0) share = min(share, max((int64_t)1, total * (slots - 2) / longest));
  Share s;
  s.total = uniform(total);
  s.share = uniform((int)share);
#pragma unroll
  for (int w = 0; w < WORKERS; ++w) {
    const int64_t j = worker(w);
    if (j >= share) continue;
    const int64_t x = j * total / share;
    if (x < before || x >= before + mine) continue;
    int64_t at = before;
    for (int e = e0; e < e1; ++e) {
      int64_t run;
      const int64_t n = size(e, run);
      if (x < at + n) {
        start_entry[w] = e;
        start_at[w] = at;
        break;
      }
      at += n;
    }
  }
  __syncthreads();
  return s;
}

// The wide kernel (16-bit and fp8 keys): query rows of its tiles, and the launch over the own keys or the prefixes.
int wide_tile_rows();
int wide_resident(int head_dim);  // workgroups of a compute unit
int wide_attention(const Params &p, int kv_dtype, int head_dim, bool own, hipStream_t stream);
// The running weights where the own keys went through it.
int wide_weights(const Params &p, int kv_dtype, int head_dim, hipStream_t stream);

__host__ __device__ __forceinline__ int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace attn
}  // namespace ekv
