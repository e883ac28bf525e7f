// Tiles, fragments and document lookup of the attention kernels.
//
// Every product is an outer product of 32x32 tiles (v_mfma_f32_32x32x16_bf16, or eight
// v_mfma_f32_32x32x2_f32 in float32) arranged so that a wavefront's lane owns one query (or, in the
// key and value gradients, one key): lane l holds column l % 32 of the accumulator and, with
// h = l / 32, its rows 8 (r / 4) + 4 h + r % 4 for r = 0 .. 15. Scores are therefore formed
// transposed (keys down, queries across): a query's maximum, sum, log-sum-exp and rescaling factor
// are scalars of its lane, and the probabilities are already the B operand of the next product if
// that product's A operand lists the contraction indexes in the order the accumulator has them
// (slots 0 .. 7 of half h = rows 4 h + 0 .. 3 and 8 + 4 h + 0 .. 3 of a group of 16): no value moves
// between lanes.
#pragma once

#include <float.h>

#include "gs_host.h"

namespace gs {

using bf16x8 = __bf16 __attribute__((ext_vector_type(8)));
using bf16x4 = __bf16 __attribute__((ext_vector_type(4)));
using f32x8 = float __attribute__((ext_vector_type(8)));
using f32x4 = float __attribute__((ext_vector_type(4)));
using f32x16 = float __attribute__((ext_vector_type(16)));
using i16x4 = short __attribute__((ext_vector_type(4)));


// Eight contraction slots of one row (A) or column (B) per lane.
template <typename T>
struct FragOf;
template <>
struct FragOf<__bf16> {
  using type = bf16x8;
};
template <>
struct FragOf<float> {
  using type = f32x8;
};
template <typename T>
using Frag = typename FragOf<T>::type;

__device__ __forceinline__ void mma(f32x16& c, bf16x8 a, bf16x8 b) {
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x16& c, f32x8 a, f32x8 b) {
#pragma unroll
  for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
}

// Accumulator registers 8 k .. 8 k + 7 as a B operand. In bfloat16 the probabilities (and their
// gradients) are rounded here, to nearest; every sum of them is taken in float32.
template <typename T>
__device__ __forceinline__ Frag<T> acc_frag(const f32x16& c, int k) {
  Frag<T> f;
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = static_cast<T>(c[8 * k + j]);
  return f;
}

// A tile in LDS: rows of DP elements, the 16-byte chunks of a row permuted by XOR with bits of the
// row number so that the reads below fall on distinct banks (256 bytes of them). Along a row: sixteen
// consecutive rows at one chunk. Across, in bfloat16: four consecutive rows at four consecutive chunks
// (32 lanes), so the lowest two row bits have to go to other chunk bits than the lowest two; in float32
// rows 4 apart at eight consecutive chunks.
template <typename T, int DP>
struct Tile {
  static constexpr int kRowBytes = DP * static_cast<int>(sizeof(T));
  static constexpr int kChunks = kRowBytes / 16;
  static constexpr int kElemsPerChunk = 16 / static_cast<int>(sizeof(T));
  static __device__ __forceinline__ int swizzle(int row) {
    if constexpr (kChunks == 8) return ((row & 2) << 1) | ((row & 4) >> 1) | ((row >> 3) & 1);  // (row & 1: by layout)
    if constexpr (sizeof(T) == 2) return ((row & 3) << 2) | ((row & 4) >> 1) | ((row >> 3) & 1);
    return ((row << 1) & 14) | ((row >> 3) & 1);
  }
  static __device__ __forceinline__ int at(int row, int chunk) {
    return row * kRowBytes + ((chunk ^ swizzle(row)) << 4);
  }
  // A operand: row row0 + l % 32, elements 16 c + 8 h .. + 7
  static __device__ __forceinline__ Frag<T> rows(const char* lds, int row0, int c, int lane) {
    const int row = row0 + (lane & 31), h = lane >> 5;
    if constexpr (sizeof(T) == 2) {
      return *reinterpret_cast<const bf16x8*>(lds + at(row, 2 * c + h));
    } else {
      const f32x4 a = *reinterpret_cast<const f32x4*>(lds + at(row, 4 * c + 2 * h));
      const f32x4 b = *reinterpret_cast<const f32x4*>(lds + at(row, 4 * c + 2 * h + 1));
      return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
  }
  // A operand of the transposed tile: element col0 + l % 32, rows row0 + 4 h + 0 .. 3 and
  // row0 + 8 + 4 h + 0 .. 3. In bfloat16 the LDS unit transposes: of 16 lanes, lane i gives the
  // address of four elements of row i / 4 and receives column i of the four rows.
  static __device__ __forceinline__ Frag<T> cols(const char* lds, int col0, int row0, int lane) {
    const int h = lane >> 5;
    if constexpr (sizeof(T) == 2) {
      typedef __attribute__((address_space(3))) i16x4* lds_ptr;
      const int i = lane & 15;
      const int col = col0 + (lane & 16) + 4 * (i & 3);
      const int r = row0 + 4 * h + (i >> 2);
      const int in = (col & 7) * 2;
      const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(lds + at(r, col >> 3) + in));
      const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(lds + at(r + 8, col >> 3) + in));
      using i16x8 = short __attribute__((ext_vector_type(8)));
      return __builtin_bit_cast(bf16x8, i16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
    } else {
      const int col = col0 + (lane & 31);
      f32x8 f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int r = row0 + (j & 4) * 2 + 4 * h + (j & 3);
        f[j] = *reinterpret_cast<const float*>(lds + at(r, col >> 2) + (col & 3) * 4);
      }
      return f;
    }
  }
};

// Eight elements of a row from global memory (16-byte aligned), zero outside.
template <typename T>
__device__ __forceinline__ Frag<T> load_frag(const T* p, bool valid) {
  Frag<T> f;
  if (valid) {
    if constexpr (sizeof(T) == 2) {
      f = *reinterpret_cast<const bf16x8*>(p);
    } else {
      const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
      f = f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = static_cast<T>(0.0f);
  }
  return f;
}

struct AttnArgs {
  const void *q, *k, *v;
  void *out, *out_low;
  float* lse;
  const int32_t *q_offsets, *k_offsets, *k_lengths, *prefix;
  int64_t q_tokens, k_tokens;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;  // strides in elements
  int docs, heads, kv_heads, group, dim, causal;
  uint32_t group_magic;  // ceil(2^20 / group)
  float softcap, scale;
  // backward
  const void* d_out;
  void *d_q, *d_k, *d_v;
  float* delta;
  int n_tiles;
  // keys of a row tile cut into up to `splits` pieces of at least split_keys, multiples of split_unit (what
  // a workgroup takes in one step), for about split_blocks workgroups in all; joined by a second launch
  int splits, split_keys, split_unit, split_blocks;
  float* part;        // [splits][q_tokens][heads][dim], unnormalised
  float* part_stat;   // [splits][q_tokens][heads][2]: maximum (base 2), sum
  int32_t* part_n;    // [q_tokens][heads] pieces
  // backward: the rows of a key tile cut into `row_parts`, the keys of a row tile into `key_parts`, each
  // part's gradients in float32
  int row_parts, key_parts;
  float* part_q;      // [key_parts][q_tokens][heads][dim]
  float* part_kv;     // [dK, dV][row_parts][k_tokens][kv_heads][dim]
};

// A value that is the same in every lane, as a scalar (the compiler cannot always tell).
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
template <typename T>
__device__ __forceinline__ T* uniform(T* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
  return reinterpret_cast<T*>(static_cast<uint64_t>(hi) << 32 | lo);
}

// Rows [0, rows) of a strided matrix as a buffer: loads beyond the last row, and at kNowhere, give
// zero. Its base is set per tile, so that offsets stay within 32 bits however long the matrix is
// (token strides are below 2^22 elements, tiles have at most 64 rows: 2^30 bytes, so kNowhere is
// outside with any row's offset added).
constexpr uint32_t kNowhere = 0x80000000u;
template <typename T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_buffer(const T* base, int64_t stride, int rows, int dim) {
  const int bytes = rows > 0 ? static_cast<int>(((rows - 1) * stride + dim) * static_cast<int64_t>(sizeof(T))) : 0;
  return __builtin_amdgcn_make_buffer_rsrc(uniform(const_cast<T*>(base)), 0, uniform(bytes), 0x00027000);
}
__device__ __forceinline__ f32x4 load16(__amdgpu_buffer_rsrc_t b, uint32_t offset) {
  using u32x4 = uint32_t __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(f32x4, static_cast<u32x4>(__builtin_amdgcn_raw_buffer_load_b128(b, offset, 0, 0)));
}

// Copies a tile from a row_buffer straight to LDS (no registers), rows beyond the buffer's and columns
// beyond `dim` as zeros. The copy is under way when the call returns: copies_done() waits for the
// wavefront's own, a barrier after it for the others'. The LDS side is linear in the lanes, so it is
// the global side that a lane permutes: it fetches the chunk that belongs to its place in the tile.
// The instruction is written out because the compiler, given its builtin, waits for every copy under
// way before each transposed LDS read. It has no output registers. The LDS base is an
// input in M0, so that the compiler, which uses that register too, knows what it holds. The resource comes from
// v_readfirstlane, and a vector-memory instruction may read a scalar register five wait states after a vector
// instruction wrote it at the earliest (M0: one after any write): the hardware does not wait, and the compiler
// adds none inside the block. s_nop 4 is five.
template <typename T, int DP, int ROWS, int THREADS>
struct TileCopy {
  using L = Tile<T, DP>;
  static constexpr int kRowsPerStep = THREADS / L::kChunks;
  static constexpr bool kOneOffset = kRowsPerStep % 16 == 0;  // rows 16 apart are permuted alike
  uint32_t offset, step;
  int64_t stride;
  int dim;
  __device__ __forceinline__ uint32_t at(int row) const {
    const int c = ((threadIdx.x % L::kChunks) ^ L::swizzle(row)) * L::kElemsPerChunk;
    return c < dim ? static_cast<uint32_t>((row * stride + c) * sizeof(T)) : kNowhere;
  }
  __device__ __forceinline__ TileCopy(int64_t stride_, int dim_) : stride(stride_), dim(dim_) {
    offset = at(threadIdx.x / L::kChunks);
    step = static_cast<uint32_t>(kRowsPerStep * stride * sizeof(T));
  }
  __device__ __forceinline__ void operator()(char* lds, __amdgpu_buffer_rsrc_t src) const {
    typedef __attribute__((address_space(3))) char* lds_ptr;
    const uint32_t to = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_ptr)lds)) +
                        __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) * (kWave * 16);
#pragma unroll
    for (int i = 0; i < ROWS / kRowsPerStep; ++i) {
      const uint32_t from = kOneOffset ? offset + i * step : at(threadIdx.x / L::kChunks + i * kRowsPerStep);
      asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                   :: "{m0}"(to + i * (THREADS * 16)), "v"(from), "s"(src) : "memory");
    }
  }
};
// The same for rows that are (token, head of the group) pairs. The first row's token and head are kept
// as a pair and advanced, a row's own are found by a multiplication: (n magic) >> 20 is n / group for
// n < group + 64 (group <= 512).
struct RowStart {
  int token, g;
  __device__ __forceinline__ void advance(const AttnArgs& a, int rows) {
    g += rows;
    const int t = static_cast<int>((static_cast<uint32_t>(g) * a.group_magic) >> 20);
    token += t;
    g -= t * a.group;
  }
};
template <typename T, int DP, int ROWS, int THREADS>
struct RowTileCopy {
  using L = Tile<T, DP>;
  static constexpr int kRowsPerStep = THREADS / L::kChunks;
  int64_t token_stride, head_stride;
  // base: the first token's first head of the group. Rows from `valid` on, and columns from dim on, are zero.
  __device__ __forceinline__ void operator()(const AttnArgs& a, char* lds, const T* base, int g0, int valid) const {
    typedef __attribute__((address_space(3))) char* lds_ptr;
    const auto src = __builtin_amdgcn_make_buffer_rsrc(uniform(const_cast<T*>(base)), 0, 0x7fffffff, 0x00027000);
    const uint32_t to = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_ptr)lds)) +
                        __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) * (kWave * 16);
#pragma unroll
    for (int i = 0; i < ROWS / kRowsPerStep; ++i) {
      const int row = threadIdx.x / L::kChunks + i * kRowsPerStep;
      const int c = ((threadIdx.x % L::kChunks) ^ L::swizzle(row)) * L::kElemsPerChunk;
      const uint32_t n = g0 + row, t = (n * a.group_magic) >> 20;
      const uint32_t at = t * static_cast<uint32_t>(token_stride) +
                          (n - t * a.group) * static_cast<uint32_t>(head_stride) + c;
      const uint32_t from = row < valid && c < a.dim ? at * static_cast<uint32_t>(sizeof(T)) : kNowhere;
      asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                   :: "{m0}"(to + i * (THREADS * 16)), "v"(from), "s"(src) : "memory");
    }
  }
};
__device__ __forceinline__ void copies_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Four consecutive accumulator rows of one column, rounded to nearest and stored.
__device__ __forceinline__ void store4(__bf16* p, float a, float b, float c, float d) {
  *reinterpret_cast<bf16x4*>(p) = bf16x4{static_cast<__bf16>(a), static_cast<__bf16>(b), static_cast<__bf16>(c),
                                         static_cast<__bf16>(d)};
}
__device__ __forceinline__ void store4(float* p, float a, float b, float c, float d) {
  *reinterpret_cast<f32x4*>(p) = f32x4{a, b, c, d};
}

// What the rounding to bfloat16 took off, rounded to bfloat16 again: with it a row is known to 2^-17.
__device__ __forceinline__ float rounding_of(float v) { return v - static_cast<float>(static_cast<__bf16>(v)); }

// v of lane l and of lane l ^ 32, added (or the larger one): the two halves of a query's keys.
__device__ __forceinline__ float half_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// 2^x by the hardware instruction (1 ulp; results below the smallest normal number are zero).
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// How scores become base-2 exponents.
enum { kPlain = 0, kCap = 1, kCapFar = 2 };
// bfloat16, capped: kCap's tanh has an absolute error of 2e-7, so the score is off by that much of the cap: 6e-5 at
// kFarCap, beside the 4e-3 of a probability's rounding. Larger caps take the library's tanh, whose error is
// relative (8192 tokens, 16 heads of 64, cap 300: forward 428 us by the exponential, 602 by the library; backward 1301 and
// 1585).
constexpr float kFarCap = 256.0f;
template <typename T, int MODE>
constexpr bool kByExp = sizeof(T) == 2 && MODE == kCap;

// The piece of [0, end) that workgroup `split` takes: keys [begin, stop) of `n` pieces (at least one) of
// at least `share`.
struct Piece {
  int begin, stop, n;
};
__device__ __forceinline__ Piece piece_of(const AttnArgs& a, int end, int split, int share) {
  if (a.splits == 1) return {0, end, 1};
  const int per = (max((end + a.splits - 1) / a.splits, share) + a.split_unit - 1) / a.split_unit * a.split_unit;
  const int n = max(1, (end + per - 1) / per);
  const int begin = split < n ? split * per : end;
  return {begin, begin + min(per, end - begin), n};
}

// The tokens in order belong to docs + 2 stretches: those before the first document's offset, the
// documents, those after the last one's. The two outer ones have no keys. Offsets are clamped to
// the tensors, so whatever the arrays hold every access stays inside.
__device__ __forceinline__ int64_t edge(const int32_t* off, int64_t tokens, int docs, int i) {
  if (i <= 0) return 0;
  if (i >= docs + 2) return tokens;
  if (off == nullptr) return i == 1 ? 0 : tokens;
  const int64_t v = off[i - 1];
  return v < 0 ? 0 : (v > tokens ? tokens : v);
}

struct Doc {
  int64_t q0, k0;   // first token
  int64_t q_len;
  int64_t k_cap;    // tokens of the key stretch
  int64_t k_len;    // of them valid
  int64_t prefix;
};

// Finds the stretch and the tile in it of tile t, where stretch i (of `per` rows a token, by the offsets
// `off` of the queries or the keys) starts at tile floor(edge(i) per / rows) + i: at least as many tiles
// as it needs, with no sums over the documents. Up to 62 documents: a lane looks at one each and has
// loaded all that describes it in the same round trip to memory. More: 64 probes a step over the
// offsets, then the description.
struct Found {
  Doc doc;
  int64_t first;  // the stretch's first tile
  int share;      // with splits: keys of a piece, the same for all documents
};
__device__ __forceinline__ int64_t pick(int64_t v, int lane) {
  const int lo = __builtin_amdgcn_readlane(static_cast<int>(v), lane);
  const int hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane);
  return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(hi)) << 32 | static_cast<uint32_t>(lo));
}
template <bool BY_KEYS>
__device__ __forceinline__ Found find_doc(const AttnArgs& a, int64_t per, int rows, int64_t t) {
  const int lane = threadIdx.x & (kWave - 1);
  const int32_t* off = BY_KEYS ? a.k_offsets : a.q_offsets;
  const int64_t tokens = BY_KEYS ? a.k_tokens : a.q_tokens;
  Found f;
  Doc& d = f.doc;
  f.share = a.split_keys;
  int i;
  int64_t q1, k1, len = INT32_MAX, prefix = 0;
  if (a.docs + 2 <= kWave) {
    const int64_t q = edge(a.q_offsets, a.q_tokens, a.docs, lane), k = edge(a.k_offsets, a.k_tokens, a.docs, lane);
    const bool real = lane >= 1 && lane <= a.docs;
    const int32_t n = real && a.k_lengths ? a.k_lengths[lane - 1] : INT32_MAX;
    const int32_t p = real && a.prefix ? a.prefix[lane - 1] : 0;
    const int64_t start = (BY_KEYS ? k : q) * per / rows + lane;
    const uint64_t b = __ballot(lane < a.docs + 2 && start <= t);
    i = b ? 63 - __builtin_clzll(b) : 0;
    f.first = pick(start, i);
    d.q0 = pick(q, i);
    d.k0 = pick(k, i);
    q1 = i + 1 < a.docs + 2 ? pick(q, i + 1) : a.q_tokens;
    k1 = i + 1 < a.docs + 2 ? pick(k, i + 1) : a.k_tokens;
    len = __builtin_amdgcn_readlane(n, i);
    prefix = __builtin_amdgcn_readlane(p, i);
    if (!BY_KEYS && a.splits > 1) {
      // pieces of a length that gives all row tiles' keys together split_blocks workgroups
      const int64_t q_next = edge(a.q_offsets, a.q_tokens, a.docs, lane + 1);
      const int64_t k_next = edge(a.k_offsets, a.k_tokens, a.docs, lane + 1);
      const float tiles = static_cast<float>((max<int64_t>(q_next - q, 0) * per + rows - 1) / rows);
      float work = real ? tiles * static_cast<float>(max<int64_t>(min<int64_t>(k_next - k, n), 0)) : 0.0f;
#pragma unroll
      for (int b = 1; b < kWave; b *= 2) work += __shfl_xor(work, b);
      f.share = uniform(max(f.share, static_cast<int>(fminf(work * a.kv_heads / a.split_blocks, 1e9f))));
    }
  } else {
    int lo = 0, n = a.docs + 2;  // the answer is in [lo, lo + n)
    while (n > 1) {
      const int step = (n + kWave - 1) / kWave;
      const int at = lo + lane * step;
      const bool before = lane * step < n && edge(off, tokens, a.docs, at) * per / rows + at <= t;
      const uint64_t b = __ballot(before);
      const int last = b ? 63 - __builtin_clzll(b) : 0;
      n = min(step, n - last * step);
      lo += last * step;
    }
    i = lo;
    f.first = edge(off, tokens, a.docs, i) * per / rows + i;
    d.q0 = edge(a.q_offsets, a.q_tokens, a.docs, i);
    d.k0 = edge(a.k_offsets, a.k_tokens, a.docs, i);
    q1 = edge(a.q_offsets, a.q_tokens, a.docs, i + 1);
    k1 = edge(a.k_offsets, a.k_tokens, a.docs, i + 1);
    if (i >= 1 && i <= a.docs) {
      if (a.k_lengths) len = a.k_lengths[i - 1];
      if (a.prefix) prefix = a.prefix[i - 1];
    }
  }
  d.q_len = q1 > d.q0 ? q1 - d.q0 : 0;
  d.k_cap = k1 > d.k0 ? k1 - d.k0 : 0;
  d.k_len = i < 1 || i > a.docs || len < 0 ? 0 : (len < d.k_cap ? len : d.k_cap);
  d.prefix = prefix;
  return f;
}

// Keys that token t of the document sees: always the first so many.
__device__ __forceinline__ int visible(const AttnArgs& a, const Doc& d, int64_t t) {
  if (!a.causal) return static_cast<int>(d.k_len);
  int64_t n = t + 1 + d.k_len - d.q_len;
  if (n < d.prefix) n = d.prefix;
  return static_cast<int>(n < 0 ? 0 : (n < d.k_len ? n : d.k_len));
}

}  // namespace gs
