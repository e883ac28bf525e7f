// Projections with their epilogue, out = act(x W^T + b) + residual, and their gradients
//
//   dz = dout act'(z);   dx = dz W;   dW = dz^T x;   db = sum over rows of dz
//
// on the matrix cores. One tile kernel makes all three products: each of its operands is a matrix whose rows or whose
// columns run along the contraction. Both sides of a tile are copied to LDS straight from memory (gs_attention.h), 128
// bytes of contraction at a time, one stage ahead of the products; operands whose rows run along the
// contraction are read as they lie, the others through the LDS unit's transpose (bfloat16) or word by word (float32).
// Products accumulate in float32 (v_mfma_f32_32x32x16_bf16, or v_mfma_f32_32x32x2_f32 in float32). The result goes
// through LDS once, so that bias, activation, residual and stores see eight neighbouring columns a lane, and is
// rounded once. The last tiles, which would leave CUs idle, are cut along the contraction into float32 parts, which a
// second launch sums in order and finishes (gemm_plan).
//
// Large products: bfloat16 8192 x 8192 x 8192 846 us (1300 TF/s), 8192 x 4096 x 4096 226 us (1217), 16384 x 8192 x 2048 467 us
// (1176; with bias and residual 498). The matrix units are busy for half of that (51%), the one wavefront a SIMD waits for a
// quarter (27%), and a plain library product takes 674, 196 and 355 us. float32 4096 x 4096 x 4096 is bound by the matrix units: 1002 us,
// 137 of the 157 TF/s there are. 8203 x 1024 x 4096 takes 87 us bare, and 105 with a bias, gelu and both results stored, 201 MB
// of them, for which the matrix units stand still. Products of a few tiles are bound by the chain of a tile's stages, 0.3 us each:
// 181 x 1024 x 1024 8.1 us (four stages ahead of the products instead of one: 8.6).
//
// Few rows are bound by reading W once: linear_few_kernel streams it past the matrix unit without LDS.
#include <algorithm>
#include <type_traits>

#include "gs_attention.h"
#include "gs_rows.h"

namespace gs {

enum { kActNone = GS_ACT_NONE, kActRelu = GS_ACT_RELU, kActGelu = GS_ACT_GELU, kActGeluTanh = GS_ACT_GELU_TANH,
       kActSilu = GS_ACT_SILU, kActs };

// ---- activations -------------------------------------------------------------------------------------

// T is the operands' type here: beside operands known to 2^-8 of themselves the forms below that are off by some 2^-17 lose
// nothing, in float32 results too (a float32 residual's), and save a sixth of a product of 1024 inputs.

// exp(v), v <= 0: in bfloat16 by the hardware's exponential, off by 2^-23 |v| of itself.
template <typename T>
__device__ __forceinline__ float exp_down(float v) {
  if constexpr (sizeof(T) == 2) return exp2_hw(v * kLog2e);
  return expf(v);
}
template <typename T>
__device__ __forceinline__ float recip(float v) {
  if constexpr (sizeof(T) == 2) return __builtin_amdgcn_rcpf(v);
  return 1.0f / v;
}
template <typename T>
__device__ __forceinline__ float sigmoid(float v) {
  const float e = exp_down<T>(-fabsf(v));
  const float r = recip<T>(1.0f + e);
  return v >= 0.0f ? r : e * r;
}
// The normal distribution function, and exp(-z^2 / 2). float32: the library's erfc. bfloat16: Phi(-u) = exp(-u^2 / 2)
// t P(t), t = 1 / (1 + 0.27 u), P of degree six fitted to erfcx(u / sqrt 2) / 2 over t by reweighted least squares: off by
// 1.3e-6 of itself up to u = 14, where Phi(-u) is below float32's smallest number. The exponential's argument adds 2^-23 u^2 / 2, so
// that in all it is 1.6e-6 of itself up to u = 3, 3.1e-6 at 6, 6.9e-6 at 12 (8203 x 1024 x 4096: 97 us, with erfc 115).
template <typename T>
__device__ __forceinline__ float normal_cdf(float z, float& bell) {
  bell = exp_down<T>(-0.5f * z * z);
  if constexpr (sizeof(T) != 2) {
    return 0.5f * erfcf(z * -0.70710678118654752f);
  } else {
    const float u = fabsf(z), t = recip<T>(fmaf(0.27f, u, 1.0f));
    float p = -0.06105639412999153f;
    p = fmaf(p, t, 0.15936046838760376f);
    p = fmaf(p, t, -0.025581030175089836f);
    p = fmaf(p, t, 0.11871293932199478f);
    p = fmaf(p, t, 0.09232588112354279f);
    p = fmaf(p, t, 0.10856088250875473f);
    p = fmaf(p, t, 0.10767664760351181f);
    const float q = bell * (p * t);
    return z >= 0.0f ? 1.0f - q : q;
  }
}
constexpr float kTanhOuter = 1.5957691216057308f, kTanhInner = 0.044715f;  // 2 sqrt(2 / pi)

// Beyond 100 in size the exponentials are below float32's smallest number: values and slopes are taken there, so that
// their products do not become infinity times zero.
constexpr float kFar = 100.0f;

// Eight values, the kind chosen once for all of them.
template <typename F>
__device__ __forceinline__ void each8(float (&v)[8], F f) {
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = f(v[j]);
}
template <typename T>
__device__ __forceinline__ void activate8(int act, float (&v)[8]) {
  const auto near = [](float z) { return z < -kFar ? -kFar : z; };  // NaN stays
  switch (act) {
    case kActRelu: return each8(v, [](float z) { return z < 0.0f ? 0.0f : z; });
    case kActGelu:
      return each8(v, [&](float z) {
        float bell;
        z = near(z);
        return z * normal_cdf<T>(z, bell);
      });
    case kActGeluTanh:
      return each8(v, [&](float z) {
        z = near(z);
        return z * sigmoid<T>(kTanhOuter * fmaf(kTanhInner * z * z, z, z));
      });
    case kActSilu:
      return each8(v, [&](float z) {
        z = near(z);
        return z * sigmoid<T>(z);
      });
    default: return;
  }
}
// d act'(z) in place of d. relu passes d or does not: where z is not positive the gradient is 0 whatever arrives, and where z is
// NaN it goes on.
template <typename T>
__device__ __forceinline__ void slope8(int act, float (&v)[8], float (&d)[8]) {
  const auto near = [](float z) { return z < -kFar ? -kFar : (z > kFar ? kFar : z); };
  switch (act) {
    case kActRelu:
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] = v[j] <= 0.0f ? 0.0f : d[j];
      return;
    case kActGelu:
      each8(v, [&](float z) {
        float bell;
        z = near(z);
        const float p = normal_cdf<T>(z, bell);
        return fmaf(z * 0.3989422804014327f, bell, p);
      });
      break;
    case kActGeluTanh:
      each8(v, [&](float z) {
        z = near(z);
        const float p = sigmoid<T>(kTanhOuter * fmaf(kTanhInner * z * z, z, z));
        return fmaf(z * p * (1.0f - p), kTanhOuter * fmaf(3.0f * kTanhInner * z, z, 1.0f), p);
      });
      break;
    case kActSilu:
      each8(v, [&](float z) {
        z = near(z);
        const float p = sigmoid<T>(z);
        return fmaf(z * p, 1.0f - p, p);
      });
      break;
    default: return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) d[j] *= v[j];
}

// ---- the tile kernel ---------------------------------------------------------------------------------

// A product out[m][n] = sum over k of a(m, k) b(n, k) and its epilogue.
struct GemmArgs {
  const void *a, *b;
  int64_t lda, ldb;  // strides in elements: of rows m, n, or where these are columns of rows k
  int64_t m, k;
  int n;
  int act;
  const void *bias, *residual;
  int64_t residual_stride;
  void *out, *z;     // [m][n], contiguous; z: before the activation (NULL: not wanted)
  bool bias_bf16, residual_bf16, out_bf16, z_bf16;
  int tiles_m, tiles_n;
  int whole, splits; // tiles that one workgroup makes; parts of each of the others
  int64_t split_k;   // contraction of a part, a multiple of a stage's
  float* part;       // [other tiles][splits][rows of a tile][columns of a tile]
};

// The first row and column of tile t. Tiles are taken in groups of a few rows of them, down a group's columns, and an XCD has a
// contiguous share of that order: what its 32 CUs work on together is a block of four by eight tiles of 256, or eight by
// eight of 128 (two a CU), which reads the least of both operands. With eight by four of 256, a second turn reads the long
// operand again: 16384 x 8192 x 4096 in groups of 4, 8, 16 rows 895, 960 and 966 us; of 128 8203 x 1024 x 4096 89, 88 and 89.
struct TileAt {
  int64_t m0;
  int n0;
  __device__ __forceinline__ TileAt(const GemmArgs& g, int t, int bm, int bn) {
    const int rows = bm == 256 ? 4 : 8;
    const int group = t / (rows * g.tiles_n), first = group * rows;
    const int high = min(rows, g.tiles_m - first), in = t - first * g.tiles_n;
    m0 = static_cast<int64_t>(first + in % high) * bm;
    n0 = in / high * bn;
  }
};

// The epilogue of columns col .. col + 7 of a row (the first n of them): bias, activation, residual and store. The residual is
// loaded apart, long before.
struct Epilogue8 {
  RawAny8 residual;
  __device__ __forceinline__ void load(const GemmArgs& g, int64_t row, int col, int n) {
    if (g.residual) residual.load(g.residual, g.residual_bf16, row * g.residual_stride + col, n);
  }
  template <typename T>
  __device__ __forceinline__ void finish(const GemmArgs& g, int64_t row, int col, int n, const float (&bias)[8],
                                         float (&v)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += bias[j];
    if (g.z) store8(g.z, g.z_bf16, row * g.n + col, n, v);
    if (g.act != kActNone) activate8<T>(g.act, v);
    if (g.residual) {
      float r[8];
      residual.to(r);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += r[j];
    }
    store8(g.out, g.out_bf16, row * g.n + col, n, v);
  }
};
__device__ __forceinline__ void bias8(const GemmArgs& g, int col, int n, float (&bias)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) bias[j] = 0.0f;
  if (g.bias) load8(g.bias, g.bias_bf16, col, n, bias);
}
template <typename T>
__device__ __forceinline__ void finish8(const GemmArgs& g, int64_t row, int col, int n, float (&v)[8]) {
  Epilogue8 e;
  float bias[8];
  e.load(g, row, col, n);
  bias8(g, col, n, bias);
  e.template finish<T>(g, row, col, n, bias, v);
}

template <typename T>
constexpr int kVec = 16 / static_cast<int>(sizeof(T));

// One side of a tile: ROWS rows (or columns) of an operand, in LDS a stage of KB of the contraction. ALONG: the operand's
// rows run along the contraction.
template <typename T, int KB, bool ALONG, int ROWS, int THREADS>
struct Side {
  static constexpr int kWidth = ALONG ? KB : (ROWS * static_cast<int>(sizeof(T)) < 256 ? ROWS : 256 / static_cast<int>(sizeof(T)));
  static constexpr int kSubs = ALONG ? 1 : ROWS / kWidth;
  static constexpr int kBytes = ROWS * KB * static_cast<int>(sizeof(T));
  using L = Tile<T, kWidth>;
  using Copy = TileCopy<T, kWidth, THREADS / L::kChunks, THREADS>;  // one step
  static_assert(Copy::kOneOffset, "steps are whole periods of the chunks' permutation");
  const T* base;
  int64_t ld;
  int rows;  // there are from the tile's first on
  __device__ __forceinline__ Side(const void* p, int64_t ld_, int64_t row0, int64_t all)
      : base(static_cast<const T*>(p) + row0 * (ALONG ? ld_ : 1)), ld(ld_),
        rows(static_cast<int>(all - row0 < ROWS ? all - row0 : ROWS)) {}
  // A stage's copy, contraction k0 .. of `left` more, which kSteps instructions of every lane make. What is past the operand's
  // end is zero. Rows are there to a whole vector: where they run along the contraction its rest is zero in one operand
  // at least, where columns are copied it ends in results that are not stored.
  static constexpr int kSteps = kBytes / (THREADS * 16), kSubSteps = kSteps / kSubs;
  struct Stage {
    uint32_t offset[kSubs];
    __amdgpu_buffer_rsrc_t src[kSubs];
  };
  __device__ __forceinline__ Stage stage(int64_t k0, int64_t left) const {
    const int n = left < 0 ? 0 : (left < KB ? static_cast<int>(left) : KB);
    if constexpr (ALONG) {
      const int whole = (n + kVec<T> - 1) / kVec<T> * kVec<T>;
      return {{Copy(ld, whole).offset}, {row_buffer(base + k0, ld, rows, whole)}};
    } else {
      const auto cols = [&](int s) {
        const int c = (rows + kVec<T> - 1) / kVec<T> * kVec<T> - s * kWidth;
        return c < 0 ? 0 : (c < kWidth ? c : kWidth);
      };
      const auto src = [&](int s) {
        return row_buffer(base + k0 * ld + s * kWidth, ld, cols(s) ? n : 0, cols(s));
      };
      static_assert(kSubs <= 2, "at most two side by side");
      if constexpr (kSubs == 1) return {{Copy(ld, cols(0)).offset}, {src(0)}};
      else return {{Copy(ld, cols(0)).offset, Copy(ld, cols(1)).offset}, {src(0), src(1)}};
    }
  }
  __device__ __forceinline__ void step(char* lds, const Stage& st, int i) const {
    Copy c(ld, kWidth);
    c.offset = st.offset[i / kSubSteps] + i % kSubSteps * c.step;  // (kNowhere stays outside)
    c(lds + i * (THREADS * 16), st.src[i / kSubSteps]);
  }
  __device__ __forceinline__ void steps(char* lds, const Stage& st) const {
#pragma unroll
    for (int i = 0; i < kSteps; ++i) step(lds, st, i);
  }

  // Rows row0 + l % 32, contraction slots of group c of sixteen: both sides list them in the same order.
  static __device__ __forceinline__ Frag<T> frag(const char* lds, int row0, int c, int lane) {
    if constexpr (ALONG && sizeof(T) == 2) {
      return L::rows(lds, row0, c, lane);
    } else if constexpr (ALONG) {
      const int row = row0 + (lane & 31), h = lane >> 5;
      const f32x4 a = *reinterpret_cast<const f32x4*>(lds + L::at(row, 4 * c + h));
      const f32x4 b = *reinterpret_cast<const f32x4*>(lds + L::at(row, 4 * c + 2 + h));
      return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    } else {
      lds += row0 / kWidth * (KB * L::kRowBytes);
      row0 %= kWidth;
      if constexpr (sizeof(T) == 4) {
        return L::cols(lds, row0, 16 * c, lane);
      } else {
        typedef __attribute__((address_space(3))) i16x4* lds_ptr;
        const int i = lane & 15, col = row0 + (lane & 16) + 4 * (i & 3), r = 16 * c + 8 * (lane >> 5) + (i >> 2);
        const int in = (col & 7) * 2;
        const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(lds + L::at(r, col >> 3) + in));
        const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(lds + L::at(r + 4, col >> 3) + in));
        using i16x8 = short __attribute__((ext_vector_type(8)));
        return __builtin_bit_cast(bf16x8, i16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
      }
    }
  }
};

// BM x BN results by WM x WN wavefronts.
template <typename T, int BM, int BN, int WM, int WN, bool A_ALONG, bool B_ALONG>
__global__ __launch_bounds__(WM* WN* kWave) void gemm_kernel(GemmArgs g) {
  constexpr int kThreads = WM * WN * kWave;
  constexpr int TM = BM / WM / 32, TN = BN / WN / 32;  // 32 x 32 results of a wavefront
  constexpr bool kDeep = TM * TN == 16;
  constexpr int KB = 128 / static_cast<int>(sizeof(T)), kStages = 2, kGroups = KB / 16;
  using A = Side<T, KB, A_ALONG, BM, kThreads>;
  using B = Side<T, KB, B_ALONG, BN, kThreads>;
  constexpr int kStageBytes = A::kBytes + B::kBytes;
  constexpr int kRowFloats = TN * 32 + 4;  // of the epilogue's rows, padded against bank conflicts
  constexpr int kOutBytes = WM * WN * 32 * kRowFloats * 4;
  __shared__ __attribute__((aligned(16))) char lds[kStages * kStageBytes > kOutBytes ? kStages * kStageBytes : kOutBytes];
  const bool whole = static_cast<int>(blockIdx.x) < g.whole;
  const int other = whole ? 0 : xcd_tile(blockIdx.x - g.whole, gridDim.x - g.whole), split = other % g.splits;
  const TileAt at(g, whole ? xcd_tile(blockIdx.x, g.whole) : g.whole + other / g.splits, BM, BN);
  const int64_t m0 = at.m0;
  const int n0 = at.n0;
  const int64_t k_begin = whole ? 0 : split * g.split_k;
  const int64_t k_end = whole || g.k - k_begin < g.split_k ? g.k : k_begin + g.split_k;
  const A a(g.a, g.lda, m0, g.m);
  const B b(g.b, g.ldb, n0, g.n);
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
  f32x16 acc[TM][TN] = {};
  const auto stage = [&](char* to, int64_t k0) {
    a.steps(to, a.stage(k0, k_end - k0));
    b.steps(to + A::kBytes, b.stage(k0, k_end - k0));
  };
  if constexpr (kDeep) {
    // One wavefront a SIMD, so that what a tile's sides read of LDS is least; nothing else runs while it waits. Fragments are read
    // one group of sixteen ahead of the products. Past a stage's last reads the wavefronts meet: the next stage has been
    // copied, and this one may be overwritten. Reads and copies are sent between products, one at a time: together they
    // would leave the matrix unit idle while they are issued.
    char *now = lds, *next = lds + kStageBytes;
    Frag<T> fa[2][TM], fb[2][TN];
    const auto fetch = [&](const char* from, int c, int to, int i) {
      if (i < TM) fa[to][i] = A::frag(from, wm + 32 * i, c, lane);
      else if (i < TM + TN) fb[to][i - TM] = B::frag(from + A::kBytes, wn + 32 * (i - TM), c, lane);
    };
    if (k_begin < k_end) {
      stage(now, k_begin);
      copies_done();
      __syncthreads();
      if (k_begin + KB < k_end) stage(next, k_begin + KB);
#pragma unroll
      for (int i = 0; i < TM + TN; ++i) fetch(now, 0, 0, i);
    }
    // one stage; MORE: another follows, MOST: one more after that, which is copied here
    const auto turn = [&](auto more, auto most, int64_t k0) {
      constexpr bool MORE = decltype(more)::value, MOST = decltype(most)::value;
      typename A::Stage sa;
      typename B::Stage sb;
#pragma unroll
      for (int c = 0; c < kGroups; ++c) {
        const bool last = c + 1 == kGroups;
        if (last && MORE) {
          copies_done();
          __syncthreads();
        }
#pragma unroll
        for (int t = 0; t < TM * TN; ++t) {
          mma(acc[t / TN][t % TN], fb[c % 2][t % TN], fa[c % 2][t / TN]);
          if (!last) fetch(now, c + 1, (c + 1) % 2, t);
          else if (MORE) fetch(next, 0, 0, t);
          if (MOST && c == 1 && t == 8) sa = a.stage(k0 + 2 * KB, k_end - k0 - 2 * KB);
          if (MOST && c == 2 && t == 8) sb = b.stage(k0 + 2 * KB, k_end - k0 - 2 * KB);
          if (MOST && last) {
            if (t < A::kSteps) a.step(now, sa, t);
            else b.step(now + A::kBytes, sb, t - A::kSteps);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      char* s = now;
      now = next;
      next = s;
    };
    static_assert(A::kSteps + B::kSteps == TM * TN && kGroups == 4, "a copy for each product of the last group");
    using Yes = std::true_type;
    using No = std::false_type;
    int64_t k0 = k_begin;
    for (; k0 + 2 * KB < k_end; k0 += KB) turn(Yes{}, Yes{}, k0);
    if (k0 + KB < k_end) {
      turn(Yes{}, No{}, k0);
      k0 += KB;
    }
    if (k0 < k_end) turn(No{}, No{}, k0);
  } else {
    char *now = lds, *next = lds + kStageBytes;
    if (k_begin < k_end) stage(now, k_begin);
    for (int64_t k0 = k_begin; k0 < k_end; k0 += KB) {
      copies_done();
      __syncthreads();  // everyone's copies are there, and everyone has left the other stage
      if (k0 + KB < k_end) stage(next, k0 + KB);
#pragma unroll
      for (int c = 0; c < kGroups; ++c) {
        Frag<T> fa[TM], fb[TN];
#pragma unroll
        for (int i = 0; i < TM; ++i) fa[i] = A::frag(now, wm + 32 * i, c, lane);
#pragma unroll
        for (int j = 0; j < TN; ++j) fb[j] = B::frag(now + A::kBytes, wn + 32 * j, c, lane);
        if constexpr (sizeof(T) == 2) {
#pragma unroll
          for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) mma(acc[i][j], fb[j], fa[i]);
        } else {  // one pair of slots over all results, then the next: no product waits for the one before it
#pragma unroll
          for (int s = 0; s < 8; ++s)
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
              for (int j = 0; j < TN; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(fb[j][s], fa[i][s], acc[i][j], 0, 0, 0);
        }
      }
      char* s = now;
      now = next;
      next = s;
    }
  }
  __syncthreads();
  // A lane holds row l % 32 and of every 32 columns 8 (r / 4) + 4 (l / 32) + r % 4: 32 rows at a time through the
  // wavefront's own LDS, then eight neighbouring columns a lane, residuals loaded before (more than two turns ahead
  // the code of 16 x 32 x 32 results is longer than the compiler unrolls, which leaves the results in memory).
  constexpr int kLanes = TN * 4, kRows = kWave / kLanes, kAhead = TN == 4 ? 2 : 32 / kRows;
  float* own = reinterpret_cast<float*>(lds) + wave * 32 * kRowFloats;
  const int c8 = lane % kLanes * 8, col = n0 + wn + c8;
  const int64_t m_lane = m0 + wm + lane / kLanes;
  const auto left = [&](int r) { return m_lane + r < g.m ? g.n - col : 0; };
  float bias[8];
  if (whole) bias8(g, col, g.n - col, bias);
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    Epilogue8 e[kAhead];
    if (whole) {
#pragma unroll
      for (int q = 0; q < kAhead; ++q) e[q].load(g, m_lane + 32 * i + q * kRows, col, left(32 * i + q * kRows));
    }
    wave_sync();
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        store4(own + (lane & 31) * kRowFloats + 32 * j + 2 * r + 4 * (lane >> 5), acc[i][j][r], acc[i][j][r + 1],
               acc[i][j][r + 2], acc[i][j][r + 3]);
    wave_sync();
#pragma unroll 1
    for (int r0 = 0; r0 < 32; r0 += kAhead * kRows) {
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        const int r = r0 + q * kRows, in = 32 * i + r, n = left(in);
        const float* at = own + (r + lane / kLanes) * kRowFloats + c8;
        const f32x4 lo = *reinterpret_cast<const f32x4*>(at), hi = *reinterpret_cast<const f32x4*>(at + 4);
        float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        if (whole) {
          if (n > 0) e[q].template finish<T>(g, m_lane + in, col, n, bias, v);
          if (r + kAhead * kRows < 32) e[q].load(g, m_lane + in + kAhead * kRows, col, left(in + kAhead * kRows));
        } else {
          store8(g.part + (static_cast<int64_t>(other) * BM + wm + in + lane / kLanes) * BN + wn + c8, 8, v);
        }
      }
    }
  }
}

// Sums the parts of the tiles after the whole ones in order and finishes them: eight columns a thread.
constexpr int kFinishThreads = 256;
template <typename T, int TILE>
__global__ __launch_bounds__(kFinishThreads) void gemm_finish_kernel(GemmArgs g) {
  constexpr int kBlocks = TILE * TILE / 8 / kFinishThreads;  // of a tile
  const int other = blockIdx.x / kBlocks, i = blockIdx.x % kBlocks * kFinishThreads + threadIdx.x;
  const TileAt at(g, g.whole + other, TILE, TILE);
  const int row = i / (TILE / 8), c = i % (TILE / 8) * 8;
  const int n = at.m0 + row < g.m ? g.n - at.n0 - c : 0;
  if (n <= 0) return;
  const float* p = g.part + (static_cast<int64_t>(other) * g.splits * TILE + row) * TILE + c;
  float v[8] = {};
  for (int s = 0; s < g.splits; ++s, p += TILE * TILE) {
    const f32x4 lo = *reinterpret_cast<const f32x4*>(p), hi = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += lo[j], v[4 + j] += hi[j];
  }
  finish8<T>(g, at.m0 + row, at.n0 + c, n, v);
}

// ---- few rows ----------------------------------------------------------------------------------------

// Sixteen columns a workgroup, up to sixteen rows: its wavefronts take the contraction in turn, from memory straight into
// the matrix instruction's operands, four loads of W sent while the four before them are multiplied, and are joined in
// LDS. Rows at any address and stride: loads are of an element's alignment. Reading W bounds it, and at 1024 columns that
// 64 workgroups leave most CUs without loads: one row of 1024 x 4096 takes 3.5 us on the GPU, 4096 x 1024 6.6,
// 8192 x 8192 27.8 (4.8 TB/s); with eight wavefronts 3.7, 6.9 and 25.5. (32 rows in two sets read x twice as often as W:
// 1024 x 4096 5.1 us, by tiles 8.1; 4096 x 1024 12.8 and 11.9; 8192 x 8192 45 and 26: those go to the tiles. With 16 rows
// these take 4.2 and 8.0, 9.3 and 11.4, 31 and 25.)
constexpr int kFewWaves = 4, kFewUnroll = 4;
template <typename T>
__global__ __launch_bounds__(kFewWaves* kWave) void linear_few_kernel(GemmArgs g) {
  constexpr int kGroup = 128 / static_cast<int>(sizeof(T));  // contraction of two loads: a cache line of every row
  constexpr int kTurn = kFewWaves * kGroup, kStep = kFewUnroll / 2 * kTurn;
  __shared__ __attribute__((aligned(16))) float join[kFewWaves][16][16 + 4];
  typedef T Vec __attribute__((ext_vector_type(kVec<T>), aligned(sizeof(T))));
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, row = lane % 16;
  const int n0 = blockIdx.x * 16, k_lane = wave * kGroup + lane / 16 * 2 * kVec<T>;
  // (rows past the last repeat it: their results are not stored)
  const T* w = static_cast<const T*>(g.b) + min(n0 + row, g.n - 1) * g.ldb;
  const T* x = static_cast<const T*>(g.a) + min(row, static_cast<int>(g.m) - 1) * g.lda;
  const int k_all = static_cast<int>(g.k), k_whole = k_all / kVec<T> * kVec<T>;
  f32x4 acc = {};
  const auto product = [&](const Vec& fw, const Vec& fx) {
    if constexpr (sizeof(T) == 2) {
      acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw, fx, acc, 0, 0, 0);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(fw[j], fx[j], acc, 0, 0, 0);
    }
  };
  // Whole vectors: lanes past the last one load it again, so that no load needs a branch, and take zeros.
  struct Step {
    Vec w[kFewUnroll], x[kFewUnroll];
  };
  const auto fetch = [&](Step& s, int k) {
#pragma unroll
    for (int u = 0; u < kFewUnroll; ++u)
      s.w[u] = *reinterpret_cast<const Vec*>(w + min(k + u / 2 * kTurn + u % 2 * kVec<T>, k_whole - kVec<T>));
#pragma unroll
    for (int u = 0; u < kFewUnroll; ++u)
      s.x[u] = *reinterpret_cast<const Vec*>(x + min(k + u / 2 * kTurn + u % 2 * kVec<T>, k_whole - kVec<T>));
  };
  if (k_whole > 0) {
    Step next;
    fetch(next, k_lane);
    for (int k = 0; k < k_whole; k += kStep) {
      const Step now = next;
      if (k + kStep < k_whole) fetch(next, k + kStep + k_lane);
#pragma unroll
      for (int u = 0; u < kFewUnroll; ++u) {
        const bool has = k + k_lane + u / 2 * kTurn + u % 2 * kVec<T> < k_whole;
        product(has ? now.w[u] : Vec{}, has ? now.x[u] : Vec{});
      }
    }
  }
  if (k_whole < k_all && wave == 0) {  // the contraction's last vector, element by element
    Vec fw = {}, fx = {};
#pragma unroll
    for (int j = 0; j < kVec<T>; ++j)
      if (lane < 16 && k_whole + j < k_all) {
        fw[j] = w[k_whole + j];
        fx[j] = x[k_whole + j];
      }
    product(fw, fx);
  }
  // a lane holds row l % 16 and columns 4 (l / 16) .. + 3
  store4(&join[wave][row][lane / 16 * 4], acc[0], acc[1], acc[2], acc[3]);
  __syncthreads();
  const int r = threadIdx.x / 2, c = threadIdx.x % 2 * 8, n = g.n - n0 - c;
  if (r >= g.m || n <= 0) return;
  float v[8] = {};
#pragma unroll
  for (int s = 0; s < kFewWaves; ++s)
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += join[s][r][c + j];
  finish8<T>(g, r, n0 + c, n, v);
}

// ---- the activation's gradient -----------------------------------------------------------------------

// dz = dout act'(z) in the operands' type, rows padded with zeros to a multiple of 16 bytes, and the column sums of
// the unrounded dz over a workgroup's rows. Rounded to bfloat16, since that is what the matrix instruction takes: half a step of every
// term, so that the gradients of x and weight are off by 2.3e-3 of themselves where rounding them alone is 1.7e-3 (2-norm, 8203 x
// 1024 -> 4096); a second term for the rest would double the products. A bias' gradient has no such rounding.
// Memory bounds it: 8203 x 4096 of bfloat16 with z in float32 54 us (268 MB, 5.0 TB/s).
constexpr int kSlopeThreads = 256;
struct SlopeArgs {
  const void *d_out, *z;
  void* dz;       // NULL: only sums
  float* parts;   // [workgroups down][n], NULL: no sums
  int64_t m, ld;
  int n, act, rows;  // rows: of a workgroup
  bool z_bf16;
};
template <typename T, typename O>
__global__ __launch_bounds__(kSlopeThreads) void slope_kernel(SlopeArgs a) {
  constexpr int kGroups = kSlopeThreads / kWave;
  __shared__ float join[kGroups][kWave * 8 + 4];
  const int lane = threadIdx.x % kWave, col = (blockIdx.y * kWave + lane) * 8, n = a.n - col;
  float sum[8] = {};
  const int64_t from = static_cast<int64_t>(blockIdx.x) * a.rows, end = a.m - from < a.rows ? a.m : from + a.rows;
  for (int64_t row = from + threadIdx.x / kWave; row < end; row += kGroups) {
    float d[8], z[8];
    load8(static_cast<const O*>(a.d_out) + row * a.n + col, n, d);
    if (a.act != kActNone) {
      load8(a.z, a.z_bf16, row * a.n + col, n, z);
      slope8<T>(a.act, z, d);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[j] += d[j];
    if (a.dz && col < a.ld) store8(static_cast<T*>(a.dz) + row * a.ld + col, static_cast<int>(a.ld - col), d);
  }
  if (a.parts == nullptr) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) join[threadIdx.x / kWave][lane * 8 + j] = sum[j];
  __syncthreads();
  for (int c = threadIdx.x; c < kWave * 8; c += kSlopeThreads) {
    const int at = blockIdx.y * kWave * 8 + c;
    if (at >= a.n) continue;
    float s = join[0][c];
#pragma unroll
    for (int i = 1; i < kGroups; ++i) s += join[i][c];
    a.parts[static_cast<int64_t>(blockIdx.x) * a.n + at] = s;
  }
}

// Rows copied to rows of a multiple of eight elements, the rest zero: up to two matrices in one launch.
struct PackArgs {
  struct {
    const void* src;
    void* dst;
    int64_t vecs, cols, stride;  // vecs: of eight elements, in all
    int per_row;                 // of them
  } m[2];
};
template <typename T>
__global__ __launch_bounds__(kFinishThreads) void pack_kernel(PackArgs a) {
  int64_t i = static_cast<int64_t>(blockIdx.x) * kFinishThreads + threadIdx.x;
  const bool second = i >= a.m[0].vecs;
  if (second) i -= a.m[0].vecs;
  const auto& m = a.m[second];
  if (i >= m.vecs) return;
  const int64_t row = i / m.per_row, c = (i - row * m.per_row) * 8, left = m.cols - c;
  float v[8];  // (float32 holds both types exactly)
  load8(static_cast<const T*>(m.src) + row * m.stride + c, left < 8 ? static_cast<int>(left) : 8, v);
  store8(static_cast<T*>(m.dst) + i * 8, 8, v);
}

// ---- plans and launches ------------------------------------------------------------------------------

constexpr int kCus = 256;
constexpr int kFewRows = GS_LINEAR_FEW_ROWS;

struct GemmPlan {
  int tile;          // side: 256, 128 or 64
  int tiles_m, tiles_n, whole, splits;
  int64_t split_k;
  size_t part;       // bytes
};
// What a stage of 128 bytes of contraction takes a tile in us: of a CU's time where enough workgroups share it, and at
// least, where there are few. bfloat16: 8192 x 4096 x 4096 in tiles of 256, 128, 64 takes 225, 258 and 371 us; 256 tiles of
// 128 over 129 stages, one a CU, 87 us; 48 tiles of 64 over 16 stages 8 us. float32 (tiles of 256 have no
// registers left for it): 4096 x 4096 x 4096 in tiles of 128 and 64 takes 1006 and 1052 us; 256 tiles of 128 over 32 stages,
// one a CU, 77 us; 44 tiles of 64 over 18 stages 16 us.
struct TileCost {
  int side, share;  // workgroups that share a CU
  float busy, alone;
};
constexpr TileCost kTileCost[2][3] = {{{128, 2, 1.96f, 2.4f}, {64, 4, 0.51f, 0.75f}, {0, 1, 0.0f, 0.0f}},
                                      {{256, 1, 1.76f, 1.76f}, {128, 2, 0.48f, 0.67f}, {64, 4, 0.18f, 0.4f}}};
// Chooses the side of the tiles and how many of them are made whole, one workgroup each: all; or as many as fill
// every CU alike, where a few are left over; or none, where there are too few. The others are cut into parts of at least four
// stages, which costs a second launch, and the parts written and read. 8203 rows are 65 tiles of 128, so that 512 of 65 x 8
// tiles fill the chip and the other eight would take half as long again: 8203 x 1024 results over 4096 take 103 us
// whole, 77 us with those eight in sixteen parts each; 4096 x 1024 over 8203 88 us in 256 tiles, 73 us in 2 x 256 parts.
static GemmPlan gemm_plan(int64_t m, int64_t n, int64_t k, size_t es, size_t result, bool cut = true) {
  GemmPlan best = {};
  float least = FLT_MAX;
  const int64_t stage = 128 / static_cast<int64_t>(es);
  const int stages = static_cast<int>(std::max<int64_t>(1, (k + stage - 1) / stage));
  for (const TileCost& c : kTileCost[es == 2]) {
    if (c.side == 0) continue;
    const int64_t tiles_m = (m + c.side - 1) / c.side, tiles_n = (n + c.side - 1) / c.side;
    const int tiles = static_cast<int>(tiles_m * tiles_n);
    const float area = static_cast<float>(c.side) * c.side;
    const float store = area * result / 19500.0f;  // through a CU's share of the memory, bytes a us
    const auto take = [&](int others, int len) {
      const int whole = tiles - others, parts = (stages + len - 1) / len;
      const int turns = (whole + kCus - 1) / kCus, more = (others * parts + kCus - 1) / kCus;
      float t = std::max((static_cast<float>(turns) * stages + static_cast<float>(more) * len) * c.busy,
                         (turns ? stages : len) * c.alone) + turns * store;
      if (turns > 1 && turns % c.share == 1) t += stages * (c.alone - c.busy);  // the last ones have a CU each
      if (others) t += 6.0f + others * parts * 8.0f * area / 6e6f;
      if (t >= least) return;
      least = t;
      best = {c.side, static_cast<int>(tiles_m), static_cast<int>(tiles_n), whole, parts, len * stage,
              static_cast<size_t>(others) * parts * c.side * c.side * sizeof(float)};
    };
    take(0, stages);
    const int others = tiles <= kCus ? tiles : tiles % kCus;
    if (!cut || others == 0 || (tiles > kCus && others > kCus / 2)) continue;
    for (const int p : {2, 3, 4, 6, 8, 12, 16, 24, 32}) {
      if (stages < 4 * p) break;
      take(others, (stages + p - 1) / p);
    }
  }
  return best;
}

template <typename T, int TILE, int WM, int WN, bool A_ALONG, bool B_ALONG>
static int launch_gemm(const GemmArgs& g, const char* what, hipStream_t st) {
  const unsigned others = static_cast<unsigned>(g.tiles_m) * g.tiles_n - g.whole;
  hipLaunchKernelGGL((gemm_kernel<T, TILE, TILE, WM, WN, A_ALONG, B_ALONG>), dim3(g.whole + others * g.splits),
                     dim3(WM * WN * kWave), 0, st, g);
  if (const int rc = check_launch(what)) return rc;
  if (others == 0) return GS_OK;
  hipLaunchKernelGGL((gemm_finish_kernel<T, TILE>), dim3(others * (TILE * TILE / 8 / kFinishThreads)), dim3(kFinishThreads), 0,
                     st, g);
  return check_launch(what);
}
template <typename T, bool A_ALONG, bool B_ALONG>
static int run_gemm(GemmArgs g, const GemmPlan& p, void* workspace, const char* what, hipStream_t st) {
  g.tiles_m = p.tiles_m;
  g.tiles_n = p.tiles_n;
  g.whole = p.whole;
  g.splits = p.splits;
  g.split_k = p.split_k;
  g.part = static_cast<float*>(workspace);
  if constexpr (sizeof(T) == 2) {
    if (p.tile == 256) return launch_gemm<T, 256, 2, 2, A_ALONG, B_ALONG>(g, what, st);
  }
  if (p.tile == 128) return launch_gemm<T, 128, 2, 2, A_ALONG, B_ALONG>(g, what, st);
  return launch_gemm<T, 64, 2, 2, A_ALONG, B_ALONG>(g, what, st);
}
// A call that keeps z gives the same bits as one that does not: where the contraction is cut goes without z. Tiles that are made whole sum in one
// order whatever their side is, so that z's stores may choose it.
static GemmPlan forward_plan(const gs_linear* p) {
  const size_t es = row_type_bytes(p->dtype), result = row_type_bytes(p->out_dtype) * (p->residual ? 2 : 1);
  const GemmPlan g = gemm_plan(p->rows, p->outputs, p->inputs, es, result);
  if (!p->z || g.part) return g;
  return gemm_plan(p->rows, p->outputs, p->inputs, es, result + row_type_bytes(p->z_dtype), false);
}
// of d_x and of d_weight
static GemmPlan input_plan(const gs_linear* p) {
  const size_t es = row_type_bytes(p->dtype);
  return gemm_plan(p->rows, p->inputs, p->outputs, es, es);
}
static GemmPlan weight_plan(const gs_linear* p) {
  const size_t es = row_type_bytes(p->dtype);
  return gemm_plan(p->outputs, p->inputs, p->rows, es, es);
}

template <typename T>
static int run_forward(const gs_linear* p, const GemmArgs& g, void* workspace, hipStream_t st) {
  const dim3 grid((g.n + 15) / 16), block(kFewWaves * kWave);
  static_assert(kFewRows == 16, "rows of a matrix instruction");
  if (g.m > kFewRows) return run_gemm<T, true, true>(g, forward_plan(p), workspace, "linear", st);
  hipLaunchKernelGGL(linear_few_kernel<T>, grid, block, 0, st, g);
  return check_launch("linear");
}

static size_t round16(size_t n) { return (n + 15) / 16 * 16; }

// Workspace of the backward pass: dz, the bias gradient's parts, the products' parts (one after the other).
struct BackPlan {
  bool make_dz;
  int64_t ld;
  int rows, down;  // of a workgroup of the slope kernel, and workgroups down a column
  size_t dz, parts, product;
};
static BackPlan back_plan(const gs_linear* p) {
  BackPlan b = {};
  const size_t es = row_type_bytes(p->dtype);
  const int64_t per = 16 / static_cast<int64_t>(es);
  // the output's gradient is the product's operand as it is where there is no activation, no rounding and no padding
  b.make_dz = p->activation != kActNone || p->out_dtype != p->dtype || p->outputs % per != 0;
  b.ld = (p->outputs + per - 1) / per * per;
  // some thousand workgroups, of at most 64 rows (more only where a grid would pass its limit), of one for each wavefront at least
  const int64_t across = (p->outputs + kWave * 8 - 1) / (kWave * 8);
  b.rows = static_cast<int>(std::max<int64_t>(4, std::min<int64_t>(64, p->rows * across / 1024 / 4 * 4)));
  b.rows = static_cast<int>(std::max<int64_t>(b.rows, p->rows * across >> 23));
  b.down = static_cast<int>((p->rows + b.rows - 1) / b.rows);
  b.dz = b.make_dz ? round16(static_cast<size_t>(p->rows) * b.ld * es) : 0;
  b.parts = round16(static_cast<size_t>(b.down) * p->outputs * sizeof(float));
  b.product = std::max(input_plan(p).part, weight_plan(p).part);
  return b;
}

static int check_linear(const gs_linear* p, bool backward) {
  GS_REQUIRE(p, GS_ERR_ARG, "linear: args is NULL");
  GS_REQUIRE(row_type(p->dtype) && row_type(p->out_dtype), GS_ERR_ARG, "linear: dtypes must be GS_FLOAT32 or GS_BFLOAT16");
  GS_REQUIRE(p->dtype == GS_BFLOAT16 || p->out_dtype == GS_FLOAT32, GS_ERR_ARG,
             "linear: float32 products have a float32 result");
  GS_REQUIRE(!p->bias || row_type(p->bias_dtype), GS_ERR_ARG, "linear: bias dtype must be GS_FLOAT32 or GS_BFLOAT16");
  GS_REQUIRE(!p->z || (row_type(p->z_dtype) && (p->dtype == GS_BFLOAT16 || p->z_dtype == GS_FLOAT32)), GS_ERR_ARG,
             "linear: z must be GS_FLOAT32, or GS_BFLOAT16 of bfloat16 products");
  GS_REQUIRE(p->activation >= 0 && p->activation < kActs, GS_ERR_ARG, "linear: unknown activation");
  GS_REQUIRE(p->rows >= 0 && p->rows < (int64_t(1) << 31), GS_ERR_ARG, "linear: invalid row count");
  GS_REQUIRE(p->inputs >= 1 && p->inputs <= GS_LINEAR_MAX_WIDTH && p->outputs >= 1 && p->outputs <= GS_LINEAR_MAX_WIDTH,
             GS_ERR_ARG, "linear: %d inputs and %d outputs: 1 to %d are provided", p->inputs, p->outputs, GS_LINEAR_MAX_WIDTH);
  const size_t es = row_type_bytes(p->dtype);
  const int per = static_cast<int>(16 / es);
  GS_REQUIRE(p->rows == 0 || (p->x && p->weight && (backward || p->out)), GS_ERR_ARG, "linear: null pointer");
  const size_t os = row_type_bytes(p->out_dtype);
  const bool few = !backward && p->rows <= kFewRows;  // rows are read at any address and stride
  for (const int64_t s : {p->x_stride, p->weight_stride})
    GS_REQUIRE(s >= 0 && s < GS_LINEAR_MAX_STRIDE && (few || s % per == 0), GS_ERR_ALIGN,
               "linear: row strides must be multiples of 16 bytes below %d elements", GS_LINEAR_MAX_STRIDE);
  GS_REQUIRE(aligned(p->x, few ? es : 16) && aligned(p->weight, few ? es : 16) && aligned(p->z, row_type_bytes(p->z_dtype)) &&
                 aligned(p->bias, row_type_bytes(p->bias_dtype)) && aligned(p->residual, os) && aligned(p->out, os),
             GS_ERR_ALIGN, "linear: misaligned tensor (x and weight: 16 bytes)");
  // The gradients' products run over rows, and what is past the last one is outside the operand (Side::stage) only where rows do not overlap.
  GS_REQUIRE(!backward || ((p->rows <= 1 || p->x_stride >= p->inputs) && (p->outputs == 1 || p->weight_stride >= p->inputs)),
             GS_ERR_ARG, "linear: rows that overlap have no backward pass: copy them first");
  // grids of a dimension below 2^32 threads; results indexed below 2^62
  const int64_t m = p->rows, n = p->outputs, k = p->inputs;
  GS_REQUIRE((m + 63) / 64 * ((std::max(n, k) + 63) / 64) < (int64_t(1) << 23) && m * ((std::max(n, k) + 7) / 8) < (int64_t(1) << 32),
             GS_ERR_ARG, "linear: too many results");
  return GS_OK;
}

}  // namespace gs

using namespace gs;

extern "C" int gs_rows_pack(const gs_rows* sets, int n, int dtype, void* stream) {
  clear_error();
  GS_REQUIRE(row_type(dtype), GS_ERR_ARG, "row pack: dtype must be GS_FLOAT32 or GS_BFLOAT16");
  GS_REQUIRE(n >= 0 && n <= 2 && (n == 0 || sets), GS_ERR_ARG, "row pack: up to two sets of rows");
  PackArgs a = {};
  int64_t all = 0;
  for (int i = 0; i < n; ++i) {
    const gs_rows& r = sets[i];
    GS_REQUIRE(r.rows >= 0 && r.cols >= 0 && r.dst_stride >= r.cols && r.dst_stride % 8 == 0, GS_ERR_ARG,
               "row pack: invalid size");
    const int64_t per = r.dst_stride / 8;
    GS_REQUIRE(r.rows < (int64_t(1) << 32) && per < (int64_t(1) << 31) && r.rows * per < (int64_t(1) << 31), GS_ERR_ARG,
               "row pack: too many elements");
    GS_REQUIRE(r.rows * per == 0 || (r.src && r.dst), GS_ERR_ARG, "row pack: null pointer");
    GS_REQUIRE(aligned(r.src, row_type_bytes(dtype)) && aligned(r.dst, 16), GS_ERR_ALIGN, "row pack: misaligned tensor");
    a.m[i] = {r.src, r.dst, r.rows * per, r.cols, r.src_stride, static_cast<int>(per)};
    all += r.rows * per;
  }
  GS_REQUIRE(all < (int64_t(1) << 32) - kFinishThreads, GS_ERR_ARG, "row pack: too many elements");
  if (all == 0) return GS_OK;
  const dim3 grid(static_cast<unsigned>((all + kFinishThreads - 1) / kFinishThreads)), block(kFinishThreads);
  if (dtype == GS_BFLOAT16) hipLaunchKernelGGL(pack_kernel<__bf16>, grid, block, 0, as_stream(stream), a);
  else hipLaunchKernelGGL(pack_kernel<float>, grid, block, 0, as_stream(stream), a);
  return check_launch("row pack");
}

extern "C" int gs_linear_plan(const gs_linear* p, int product, int32_t* tile, int32_t* whole, int32_t* parts) {
  clear_error();
  GS_REQUIRE(tile && whole && parts, GS_ERR_ARG, "linear plan: null pointer");
  GS_REQUIRE(product >= GS_LINEAR_FORWARD && product <= GS_LINEAR_D_WEIGHT, GS_ERR_ARG, "linear plan: unknown product");
  if (const int rc = check_linear(p, product != GS_LINEAR_FORWARD)) return rc;
  GemmPlan g = {};
  if (product == GS_LINEAR_D_WEIGHT) g = weight_plan(p);
  else if (product == GS_LINEAR_D_X && p->rows > 0) g = input_plan(p);
  else if (product == GS_LINEAR_FORWARD && p->rows > kFewRows) g = forward_plan(p);
  *tile = g.tile;
  *whole = g.whole;
  *parts = g.whole < g.tiles_m * g.tiles_n ? g.splits : 0;
  return GS_OK;
}

extern "C" size_t gs_linear_fwd_workspace_size(const gs_linear* p) {
  clear_error();
  if (!p || p->rows <= kFewRows || p->inputs <= 0 || p->outputs <= 0 || !row_type(p->dtype)) return 0;
  return forward_plan(p).part;
}

extern "C" int gs_linear_fwd(const gs_linear* p, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  if (const int rc = check_linear(p, false)) return rc;
  const size_t need = gs_linear_fwd_workspace_size(p);
  GS_REQUIRE(workspace_bytes >= need && (workspace || need == 0), GS_ERR_WORKSPACE, "linear: workspace too small");
  GS_REQUIRE(aligned(workspace, 16), GS_ERR_ALIGN, "linear: misaligned workspace");
  if (p->rows == 0) return GS_OK;
  GemmArgs g = {};
  g.a = p->x;
  g.b = p->weight;
  g.lda = p->x_stride;
  g.ldb = p->weight_stride;
  g.m = p->rows;
  g.n = p->outputs;
  g.k = p->inputs;
  g.act = p->activation;
  g.bias = p->bias;
  g.bias_bf16 = p->bias_dtype == GS_BFLOAT16;
  g.residual = p->residual;
  g.residual_stride = p->residual_stride;
  g.residual_bf16 = g.out_bf16 = p->out_dtype == GS_BFLOAT16;
  g.out = p->out;
  g.z = p->z;
  g.z_bf16 = p->z_dtype == GS_BFLOAT16;
  return p->dtype == GS_BFLOAT16 ? run_forward<__bf16>(p, g, workspace, as_stream(stream))
                                 : run_forward<float>(p, g, workspace, as_stream(stream));
}

extern "C" size_t gs_linear_bwd_workspace_size(const gs_linear* p) {
  clear_error();
  if (!p || p->rows <= 0 || p->inputs <= 0 || p->outputs <= 0 || !row_type(p->dtype)) return 0;
  const BackPlan b = back_plan(p);
  return b.dz + b.parts + b.product;
}

template <typename T>
static int run_backward(const gs_linear* p, const void* d_out, void* d_x, void* d_weight, void* d_bias, void* workspace,
                        hipStream_t st) {
  const BackPlan b = back_plan(p);
  char* ws = static_cast<char*>(workspace);
  float* parts = reinterpret_cast<float*>(ws + b.dz);
  void* product = ws + b.dz + b.parts;
  const bool make_dz = b.make_dz && (d_x || d_weight);
  if ((make_dz || d_bias) && p->rows > 0) {
    const SlopeArgs s = {d_out, p->z, make_dz ? ws : nullptr, d_bias ? parts : nullptr, p->rows, b.ld, p->outputs, p->activation, b.rows,
                         p->z_dtype == GS_BFLOAT16};
    const dim3 grid(b.down, (p->outputs + kWave * 8 - 1) / (kWave * 8)), block(kSlopeThreads);
    if (p->out_dtype == GS_FLOAT32) hipLaunchKernelGGL((slope_kernel<T, float>), grid, block, 0, st, s);
    else hipLaunchKernelGGL((slope_kernel<T, __bf16>), grid, block, 0, st, s);
    if (const int rc = check_launch("linear backward (activation)")) return rc;
  }
  if (d_bias) {
    ColumnSums s = {};
    s.parts = parts;
    s.n = b.down;
    s.sums = 1;
    s.width = p->outputs;
    s.out[0] = d_bias;
    s.bf16[0] = p->bias_dtype == GS_BFLOAT16;
    if (const int rc = column_sums(s, "linear backward (bias)", st)) return rc;
  }
  GemmArgs g = {};
  g.out_bf16 = sizeof(T) == 2;
  const void* dz = make_dz ? static_cast<const void*>(ws) : d_out;
  const int64_t ld = make_dz ? b.ld : p->outputs;
  // a single row's stride says nothing, and may be 0
  const int64_t per = 16 / static_cast<int64_t>(sizeof(T)), apart = (p->inputs + per - 1) / per * per;
  if (d_x && p->rows > 0) {
    g.a = dz;
    g.lda = ld;
    g.b = p->weight;
    g.ldb = std::max(p->weight_stride, apart);
    g.m = p->rows;
    g.n = p->inputs;
    g.k = p->outputs;
    g.out = d_x;
    if (const int rc = run_gemm<T, true, false>(g, input_plan(p), product, "linear backward (input)", st)) return rc;
  }
  if (d_weight) {
    g.a = dz;
    g.lda = ld;
    g.b = p->x;
    g.ldb = std::max(p->x_stride, apart);
    g.m = p->outputs;
    g.n = p->inputs;
    g.k = p->rows;
    g.out = d_weight;
    if (const int rc = run_gemm<T, false, false>(g, weight_plan(p), product, "linear backward (weight)", st)) return rc;
  }
  return GS_OK;
}

extern "C" int gs_linear_bwd(const gs_linear* p, const void* d_out, void* d_x, void* d_weight, void* d_bias,
                             void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  if (const int rc = check_linear(p, true)) return rc;
  GS_REQUIRE(p->rows == 0 || d_out, GS_ERR_ARG, "linear: null gradient");
  GS_REQUIRE(p->rows == 0 || p->activation == kActNone || p->z, GS_ERR_ARG, "linear: the activation's gradient needs z");
  const size_t need = gs_linear_bwd_workspace_size(p), es = row_type_bytes(p->dtype);
  GS_REQUIRE(workspace_bytes >= need && (workspace || need == 0), GS_ERR_WORKSPACE, "linear: workspace too small");
  GS_REQUIRE(aligned(workspace, 16) && aligned(d_out, 16) && aligned(d_x, es) &&
                 aligned(d_weight, es) && aligned(d_bias, row_type_bytes(p->bias_dtype)),
             GS_ERR_ALIGN, "linear: misaligned gradient or workspace");
  const hipStream_t st = as_stream(stream);
  return p->dtype == GS_BFLOAT16 ? run_backward<__bf16>(p, d_out, d_x, d_weight, d_bias, workspace, st)
                                 : run_backward<float>(p, d_out, d_x, d_weight, d_bias, workspace, st);
}
