// Rows of float32 or bfloat16 in vectors of eight elements, at any address and stride (the memory system splits
// an access that crosses a line), the last vector of a row cut short.
#pragma once

#include "gs_host.h"

namespace gs {

// N elements as they lie in memory. Loads leave them so: turned to float inside the branch that loads them, every load
// would be waited for before the next is sent.
template <typename T, int N>
struct RawN {
  static constexpr int kPer = N * sizeof(T) > 16 ? 16 / sizeof(T) : N, kParts = N / kPer;
  typedef T Vec __attribute__((ext_vector_type(kPer), aligned(sizeof(T))));
  Vec part[kParts];
  // Elements p[0 .. n) of N, the others zero.
  __device__ __forceinline__ void load(const T* p, int n) {
    if (n >= N) {
#pragma unroll
      for (int i = 0; i < kParts; ++i) part[i] = *reinterpret_cast<const Vec*>(p + i * kPer);
    } else {
#pragma unroll
      for (int i = 0; i < kParts; ++i) part[i] = 0;
      if (n > 0) {
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (j < n) part[j / kPer][j % kPer] = p[j];
      }
    }
  }
  __device__ __forceinline__ void to(float (&v)[N]) const {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = static_cast<float>(part[j / kPer][j % kPer]);
  }
};
template <typename T>
using Raw8 = RawN<T, 8>;

// Elements p[0 .. n) of eight as float, the others zero.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int n, float (&v)[8]) {
  Raw8<T> r;
  r.load(p, n);
  r.to(v);
}
// The same of a tensor whose type is known at run time.
__device__ __forceinline__ void load8(const void* p, bool bf16, int64_t at, int n, float (&v)[8]) {
  if (bf16) load8(static_cast<const __bf16*>(p) + at, n, v);
  else load8(static_cast<const float*>(p) + at, n, v);
}

// Eight elements of a tensor whose type is known at run time, as they lie in memory.
struct RawAny8 {
  Raw8<float> f;  // bfloat16: in the first part
  bool bf16;
  __device__ __forceinline__ void load(const void* p, bool bf16_, int64_t at, int n) {
    bf16 = bf16_;
    if (bf16) {
      Raw8<__bf16> h;
      h.load(static_cast<const __bf16*>(p) + at, n);
      f.part[0] = __builtin_bit_cast(Raw8<float>::Vec, h.part[0]);
    } else {
      f.load(static_cast<const float*>(p) + at, n);
    }
  }
  __device__ __forceinline__ void to(float (&v)[8]) const {
    if (bf16) {
      const auto h = __builtin_bit_cast(Raw8<__bf16>::Vec, f.part[0]);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = static_cast<float>(h[j]);
    } else {
      f.to(v);
    }
  }
};

// Rounded once, to nearest.
template <typename T>
__device__ __forceinline__ void store8(T* p, int n, const float (&v)[8]) {
  using R = Raw8<T>;
  if (n >= 8) {
#pragma unroll
    for (int i = 0; i < R::kParts; ++i) {
      typename R::Vec a;
#pragma unroll
      for (int j = 0; j < R::kPer; ++j) a[j] = static_cast<T>(v[i * R::kPer + j]);
      *reinterpret_cast<typename R::Vec*>(p + i * R::kPer) = a;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = static_cast<T>(v[j]);
  }
}
__device__ __forceinline__ void store8(void* p, bool bf16, int64_t at, int n, const float (&v)[8]) {
  if (bf16) store8(static_cast<__bf16*>(p) + at, n, v);
  else store8(static_cast<float*>(p) + at, n, v);
}

// Sums of parts, column by column in a fixed order: out[k][c] = sum over p of parts[p][k][c]. 64 columns of one sum a
// workgroup, its wavefronts take the parts in turn.
constexpr int kSumThreads = 1024;
struct ColumnSums {
  const float* parts;
  int n, sums, width;
  void* out[5];
  bool bf16[5];
};
static __global__ __launch_bounds__(kSumThreads) void column_sums_kernel(ColumnSums a) {
  __shared__ float part[kSumThreads];
  const int k = blockIdx.y, c = blockIdx.x * kWave + threadIdx.x % kWave, w = threadIdx.x / kWave;
  constexpr int kStep = kSumThreads / kWave;
  float s[4] = {};
  if (c < a.width) {
    const auto at = [&](int i) { return a.parts[(static_cast<int64_t>(i) * a.sums + k) * a.width + c]; };
    int p = w;
    for (; p + 3 * kStep < a.n; p += 4 * kStep) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] += at(p + i * kStep);
    }
    for (; p < a.n; p += kStep) s[0] += at(p);
  }
  part[threadIdx.x] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  if (w == 0 && c < a.width) {
    float t = 0.0f;
    for (int i = 0; i < kStep; ++i) t += part[i * kWave + threadIdx.x];
    if (a.bf16[k]) static_cast<__bf16*>(a.out[k])[c] = static_cast<__bf16>(t);
    else static_cast<float*>(a.out[k])[c] = t;
  }
}
inline int column_sums(const ColumnSums& a, const char* what, hipStream_t st) {
  hipLaunchKernelGGL(column_sums_kernel, dim3((a.width + kWave - 1) / kWave, a.sums), dim3(kSumThreads), 0, st, a);
  return check_launch(what);
}

inline bool row_type(int dtype) { return dtype == GS_FLOAT32 || dtype == GS_BFLOAT16; }
inline size_t row_type_bytes(int dtype) { return dtype == GS_BFLOAT16 ? 2 : 4; }

}  // namespace gs
