// The global norm of many gradient tensors, and clipping by it. The tensors' table travels in the
// kernel arguments, up to kClipTensors of them a launch; each workgroup sums a piece of one tensor in
// float64 (squares of any float32 or bfloat16 value fit, and the order is fixed, so the norm is
// reproducible), one workgroup joins the pieces. Both passes are HBM-bound: 16-byte accesses, four in
// flight a thread, at whatever address a tensor begins (the memory system splits an access that
// crosses a line; tensors of odd sizes in one flat buffer are the rule, not the exception).
// The norm of those 394 MB takes 96 us (4.1 TB/s), of 236 MB that a cache holds 39 us.
#include <algorithm>

#include "gs_host.h"

namespace gs {

constexpr int kClipTensors = 128;
constexpr int kClipThreads = 256;
constexpr int kClipUnroll = 4;                                       // 16-byte accesses a thread
constexpr int64_t kClipStepBytes = kClipThreads * 16 * kClipUnroll;  // 16 KB
constexpr int kJoinThreads = 1024;

struct ClipTable {
  const void* in[kClipTensors];
  void* out[kClipTensors];
  int64_t n[kClipTensors];
  int32_t block0[kClipTensors];  // first workgroup; INT32_MAX past `count`
  uint8_t bf16[kClipTensors];
  int64_t piece_bytes;           // of a workgroup, a multiple of kClipStepBytes
};

// The tensor that workgroup b works on (block0 is non-decreasing), by votes of 64 entries.
__device__ __forceinline__ int tensor_of(const ClipTable& t, int b) {
  static_assert(kClipTensors % kWave == 0, "whole votes");
  const int lane = threadIdx.x & (kWave - 1);
  int n = -1;
#pragma unroll
  for (int i = 0; i < kClipTensors; i += kWave) n += __popcll(__ballot(t.block0[i + lane] <= b));
  return n;
}

template <int THREADS>
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[THREADS / kWave];
#pragma unroll
  for (int o = kWave / 2; o > 0; o >>= 1) v += __shfl_down(v, o);
  if ((threadIdx.x & (kWave - 1)) == 0) part[threadIdx.x / kWave] = v;
  __syncthreads();
  double s = 0.0;
  for (int i = 0; i < THREADS / kWave; ++i) s += part[i];
  return s;
}

// 16 bytes of elements at an element's alignment.
template <typename T>
struct Pack {
  static constexpr int kN = 16 / sizeof(T);
  typedef T Vec __attribute__((ext_vector_type(kN), aligned(sizeof(T))));
};

// Calls f(index, element vector) for the whole vectors of [from, to) and g(index) for the elements after
// them, four loads of a thread in flight.
template <typename T, typename F, typename G>
__device__ __forceinline__ void each(const T* in, int64_t from, int64_t to, F f, G g) {
  using Vec = typename Pack<T>::Vec;
  constexpr int N = Pack<T>::kN;
  constexpr int64_t kStep = kClipThreads * N * kClipUnroll;
  int64_t e = from;
  for (; e + kStep <= to; e += kStep) {
    Vec v[kClipUnroll];
#pragma unroll
    for (int i = 0; i < kClipUnroll; ++i)
      v[i] = *reinterpret_cast<const Vec*>(in + e + (i * kClipThreads + threadIdx.x) * N);
#pragma unroll
    for (int i = 0; i < kClipUnroll; ++i) f(e + (i * kClipThreads + threadIdx.x) * N, v[i]);
  }
  for (e += threadIdx.x * N; e + N <= to; e += kClipThreads * N) f(e, *reinterpret_cast<const Vec*>(in + e));
  // at most one thread has a partial vector
  for (; e < to; ++e) g(e);
}

template <typename T>
__device__ __forceinline__ double piece_sum(const T* in, int64_t from, int64_t to) {
  double s[4] = {0.0, 0.0, 0.0, 0.0};
  each<T>(in, from, to,
          [&](int64_t, typename Pack<T>::Vec v) {
#pragma unroll
            for (int k = 0; k < Pack<T>::kN; ++k) {
              const double x = static_cast<double>(static_cast<float>(v[k]));
              s[k % 4] = fma(x, x, s[k % 4]);
            }
          },
          [&](int64_t e) {
            const double x = static_cast<double>(static_cast<float>(in[e]));
            s[0] = fma(x, x, s[0]);
          });
  return (s[0] + s[1]) + (s[2] + s[3]);
}

__global__ __launch_bounds__(kClipThreads) void norm_kernel(ClipTable t, double* sums) {
  const int i = __builtin_amdgcn_readfirstlane(tensor_of(t, blockIdx.x));
  const int64_t per = t.piece_bytes / (t.bf16[i] ? 2 : 4);
  const int64_t from = (static_cast<int64_t>(blockIdx.x) - t.block0[i]) * per;
  const int64_t to = min(from + per, t.n[i]);
  double s = t.bf16[i] ? piece_sum(static_cast<const __bf16*>(t.in[i]), from, to)
                       : piece_sum(static_cast<const float*>(t.in[i]), from, to);
  s = block_sum<kClipThreads>(s);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

__global__ __launch_bounds__(kJoinThreads) void norm_join_kernel(const double* sums, int64_t n, double max_norm,
                                                                 float* norm, float* coef) {
  double s[4] = {0.0, 0.0, 0.0, 0.0};
  int64_t i = threadIdx.x;
  for (; i + 3 * kJoinThreads < n; i += 4 * kJoinThreads) {
#pragma unroll
    for (int k = 0; k < 4; ++k) s[k] += sums[i + k * kJoinThreads];
  }
  for (; i < n; i += kJoinThreads) s[0] += sums[i];
  const double r = sqrt(block_sum<kJoinThreads>((s[0] + s[1]) + (s[2] + s[3])));
  if (threadIdx.x != 0) return;
  *norm = static_cast<float>(r);
  if (coef) {
    const double c = max_norm / (r + 1e-6);
    *coef = c > 1.0 ? 1.0f : static_cast<float>(c);  // NaN stays
  }
}

template <bool STREAMED, typename T>
__device__ __forceinline__ void piece_scale(const T* in, T* out, int64_t from, int64_t to, float c) {
  using Vec = typename Pack<T>::Vec;
  each<T>(in, from, to,
          [&](int64_t e, Vec v) {
            Vec r;
#pragma unroll
            for (int k = 0; k < Pack<T>::kN; ++k) r[k] = static_cast<T>(static_cast<float>(v[k]) * c);
            if constexpr (STREAMED) __builtin_nontemporal_store(r, reinterpret_cast<Vec*>(out + e));
            else *reinterpret_cast<Vec*>(out + e) = r;
          },
          [&](int64_t e) { out[e] = static_cast<T>(static_cast<float>(in[e]) * c); });
}

template <bool STREAMED>
__global__ __launch_bounds__(kClipThreads) void scale_kernel(ClipTable t, const float* coef) {
  // From the last piece to the first: what the norm's pass read last is still in the last-level cache; and
  // outputs too large to stay there go past it, so as not to put it out (118M mixed gradients, 394 MB: 240
  // us in order, 231 us backwards, 207 us past the caches).
  const int b = gridDim.x - 1 - blockIdx.x;
  const int i = __builtin_amdgcn_readfirstlane(tensor_of(t, b));
  const float c = *coef;
  if (c == 1.0f && t.in[i] == t.out[i]) return;  // every value is its own product with 1
  const int64_t per = t.piece_bytes / (t.bf16[i] ? 2 : 4);
  const int64_t from = (static_cast<int64_t>(b) - t.block0[i]) * per;
  const int64_t to = min(from + per, t.n[i]);
  const auto in_f = static_cast<const float*>(t.in[i]);
  const auto in_b = static_cast<const __bf16*>(t.in[i]);
  const auto out_f = static_cast<float*>(t.out[i]);
  const auto out_b = static_cast<__bf16*>(t.out[i]);
  if (t.bf16[i]) piece_scale<STREAMED>(in_b, out_b, from, to, c);
  else piece_scale<STREAMED>(in_f, out_f, from, to, c);
}

// Bytes of a workgroup's piece: one step of its threads, and more where that would be over kClipPieces
// pieces, so that the join stays short. 2 bytes an element are assumed, the fewest: the workspace query
// has no types.
constexpr int64_t kClipPieces = 16384;
static int64_t piece_bytes_of(const int64_t* sizes, int n) {
  int64_t total = 0;
  for (int i = 0; i < n; ++i) total += std::max<int64_t>(sizes[i], 0);
  return std::max<int64_t>(1, (total * 2 / kClipPieces + kClipStepBytes - 1) / kClipStepBytes) * kClipStepBytes;
}
static int64_t pieces_of(int64_t size, int bytes, int64_t piece) {
  const int64_t per = piece / bytes;
  return (size + per - 1) / per;
}

static int check_tensors(const void* const* in, const int64_t* sizes, const int32_t* dtypes, int n, int64_t* pieces) {
  GS_REQUIRE(n >= 0 && (n == 0 || (in && sizes && dtypes)), GS_ERR_ARG, "gradients: null table or negative count");
  for (int i = 0; i < n; ++i) {
    GS_REQUIRE(sizes[i] >= 0 && sizes[i] < (int64_t(1) << 40), GS_ERR_ARG, "gradient %d: invalid size", i);
    GS_REQUIRE(dtypes[i] == GS_FLOAT32 || dtypes[i] == GS_BFLOAT16, GS_ERR_ARG,
               "gradient %d: dtype must be GS_FLOAT32 or GS_BFLOAT16", i);
    GS_REQUIRE(sizes[i] == 0 || in[i], GS_ERR_ARG, "gradient %d: null pointer", i);
    GS_REQUIRE(aligned(in[i], dtypes[i] == GS_BFLOAT16 ? 2 : 4), GS_ERR_ALIGN, "gradient %d: misaligned", i);
  }
  const int64_t piece = piece_bytes_of(sizes, n);
  int64_t total = 0;
  for (int i = 0; i < n; ++i) total += pieces_of(sizes[i], dtypes[i] == GS_BFLOAT16 ? 2 : 4, piece);
  GS_REQUIRE(total < (int64_t(1) << 31), GS_ERR_ARG, "gradients: too many elements");
  *pieces = total;
  return GS_OK;
}

// Calls f(table, workgroups, first piece) for launches of up to kClipTensors tensors, the last launch's
// tensors first if `backwards`; empty tensors are left out.
template <typename F>
static int each_table(const void* const* in, void* const* out, const int64_t* sizes, const int32_t* dtypes, int n,
                      bool backwards, F f) {
  ClipTable t;
  t.piece_bytes = piece_bytes_of(sizes, n);
  int64_t done = 0;
  const int launches = (n + kClipTensors - 1) / kClipTensors;
  for (int l = 0; l < launches; ++l) {
    const int first = (backwards ? launches - 1 - l : l) * kClipTensors;
    int64_t blocks = 0;
    int count = 0;
    for (int i = first; i < std::min(first + kClipTensors, n); ++i) {
      if (sizes[i] == 0) continue;
      const int k = count++;
      t.in[k] = in[i];
      t.out[k] = out ? out[i] : nullptr;
      t.n[k] = sizes[i];
      t.bf16[k] = dtypes[i] == GS_BFLOAT16;
      t.block0[k] = static_cast<int32_t>(blocks);
      blocks += pieces_of(sizes[i], dtypes[i] == GS_BFLOAT16 ? 2 : 4, t.piece_bytes);
    }
    if (count == 0) continue;
    for (int k = count; k < kClipTensors; ++k) t.block0[k] = INT32_MAX;
    if (const int rc = f(t, blocks, done)) return rc;
    done += blocks;
  }
  return GS_OK;
}

}  // namespace gs

using namespace gs;

static size_t norm_workspace(const int64_t* sizes, int n) {
  const int64_t piece = piece_bytes_of(sizes, n);
  int64_t total = 0;  // enough for either type
  for (int i = 0; i < n; ++i) total += pieces_of(std::max<int64_t>(sizes[i], 0), 4, piece);
  return static_cast<size_t>(total) * sizeof(double);
}

extern "C" size_t gs_grad_norm_workspace_size(const int64_t* sizes, int n) {
  clear_error();
  return sizes == nullptr || n <= 0 ? 0 : norm_workspace(sizes, n);
}

extern "C" int gs_grad_norm(const void* const* grads, const int64_t* sizes, const int32_t* dtypes, int n,
                            double max_norm, float* norm, float* coef, void* workspace, size_t workspace_bytes,
                            void* stream) {
  clear_error();
  int64_t pieces;
  if (const int rc = check_tensors(grads, sizes, dtypes, n, &pieces)) return rc;
  GS_REQUIRE(norm, GS_ERR_ARG, "gradient norm: null output");
  GS_REQUIRE(coef == nullptr || max_norm >= 0.0, GS_ERR_ARG, "gradient norm: max_norm must be >= 0");
  GS_REQUIRE(workspace_bytes >= norm_workspace(sizes, n) && (workspace || pieces == 0),
             GS_ERR_WORKSPACE, "gradient norm: workspace too small");
  GS_REQUIRE(aligned(workspace, 8) && aligned(norm, 4) && aligned(coef, 4), GS_ERR_ALIGN,
             "gradient norm: misaligned workspace or output");
  const hipStream_t st = as_stream(stream);
  double* sums = static_cast<double*>(workspace);
  const int rc = each_table(grads, nullptr, sizes, dtypes, n, false, [&](const ClipTable& t, int64_t blocks, int64_t at) {
    hipLaunchKernelGGL(norm_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kClipThreads), 0, st, t, sums + at);
    return check_launch("gradient norm");
  });
  if (rc) return rc;
  hipLaunchKernelGGL(norm_join_kernel, dim3(1), dim3(kJoinThreads), 0, st, sums, pieces, max_norm, norm, coef);
  return check_launch("gradient norm (join)");
}

extern "C" int gs_grad_scale(const void* const* grads, void* const* out, const int64_t* sizes, const int32_t* dtypes,
                             int n, const float* coef, void* stream) {
  clear_error();
  int64_t pieces;
  if (const int rc = check_tensors(grads, sizes, dtypes, n, &pieces)) return rc;
  GS_REQUIRE(coef && (n == 0 || out), GS_ERR_ARG, "gradient scale: null pointer");
  for (int i = 0; i < n; ++i) {
    GS_REQUIRE(sizes[i] == 0 || out[i], GS_ERR_ARG, "gradient scale: output %d is NULL", i);
    GS_REQUIRE(aligned(out[i], dtypes[i] == GS_BFLOAT16 ? 2 : 4), GS_ERR_ALIGN, "gradient scale: output %d misaligned", i);
  }
  GS_REQUIRE(aligned(coef, 4), GS_ERR_ALIGN, "gradient scale: misaligned coefficient");
  const hipStream_t st = as_stream(stream);
  int64_t bytes = 0;
  for (int i = 0; i < n; ++i) bytes += sizes[i] * (dtypes[i] == GS_BFLOAT16 ? 2 : 4);
  const bool streamed = bytes > (int64_t(64) << 20);
  return each_table(grads, out, sizes, dtypes, n, true, [&](const ClipTable& t, int64_t blocks, int64_t) {
    const dim3 grid(static_cast<unsigned>(blocks)), block(kClipThreads);
    if (streamed) hipLaunchKernelGGL(scale_kernel<true>, grid, block, 0, st, t, coef);
    else hipLaunchKernelGGL(scale_kernel<false>, grid, block, 0, st, t, coef);
    return check_launch("gradient scale");
  });
}
