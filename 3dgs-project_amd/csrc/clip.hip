// The global norm of many gradient tensors, and clipping by it. The tensors' table travels in the
// kernel arguments, up to kClipTensors of them a launch; each workgroup sums a fixed piece of one
// tensor in float64 (squares of any float32 or bfloat16 value fit, and the order is fixed, so the
// norm is reproducible), one workgroup joins the pieces.
#include "gs_host.h"

namespace gs {

constexpr int kClipTensors = 128;
constexpr int kClipThreads = 256;
constexpr int64_t kClipPiece = 16384;  // elements of a workgroup

struct ClipTable {
  const void* in[kClipTensors];
  void* out[kClipTensors];
  int64_t n[kClipTensors];
  int32_t block0[kClipTensors];  // first workgroup; the launch's end for the rest
  int8_t bf16[kClipTensors];
  int count;
};

// The tensor that workgroup b works on (block0 is non-decreasing).
__device__ __forceinline__ int tensor_of(const ClipTable& t, int b) {
  int lo = 0, hi = t.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (t.block0[mid] <= b) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[kClipThreads / kWave];
#pragma unroll
  for (int o = kWave / 2; o > 0; o >>= 1) v += __shfl_down(v, o);
  if ((threadIdx.x & (kWave - 1)) == 0) part[threadIdx.x / kWave] = v;
  __syncthreads();
  double s = 0.0;
  for (int i = 0; i < kClipThreads / kWave; ++i) s += part[i];
  return s;
}

__global__ __launch_bounds__(kClipThreads) void norm_kernel(ClipTable t, double* sums) {
  const int i = tensor_of(t, blockIdx.x);
  const int64_t from = (static_cast<int64_t>(blockIdx.x) - t.block0[i]) * kClipPiece;
  const int64_t to = min(from + kClipPiece, t.n[i]);
  double s = 0.0;
  for (int64_t e = from + threadIdx.x; e < to; e += kClipThreads) {
    const double g = t.bf16[i] ? static_cast<double>(static_cast<float>(static_cast<const __bf16*>(t.in[i])[e]))
                               : static_cast<double>(static_cast<const float*>(t.in[i])[e]);
    s = fma(g, g, s);
  }
  s = block_sum(s);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

__global__ __launch_bounds__(kClipThreads) void norm_join_kernel(const double* sums, int64_t n, double max_norm,
                                                                 float* norm, float* coef) {
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += kClipThreads) s += sums[i];
  s = sqrt(block_sum(s));
  if (threadIdx.x != 0) return;
  *norm = static_cast<float>(s);
  if (coef) {
    const double c = max_norm / (s + 1e-6);
    *coef = c > 1.0 ? 1.0f : static_cast<float>(c);  // NaN stays
  }
}

__global__ __launch_bounds__(kClipThreads) void scale_kernel(ClipTable t, const float* coef) {
  const int i = tensor_of(t, blockIdx.x);
  const int64_t from = (static_cast<int64_t>(blockIdx.x) - t.block0[i]) * kClipPiece;
  const int64_t to = min(from + kClipPiece, t.n[i]);
  const float c = *coef;
  for (int64_t e = from + threadIdx.x; e < to; e += kClipThreads) {
    if (t.bf16[i])
      static_cast<__bf16*>(t.out[i])[e] = static_cast<__bf16>(static_cast<float>(static_cast<const __bf16*>(t.in[i])[e]) * c);
    else
      static_cast<float*>(t.out[i])[e] = static_cast<const float*>(t.in[i])[e] * c;
  }
}

static int check_tensors(const void* const* in, const int64_t* sizes, const int32_t* dtypes, int n, int64_t* pieces) {
  GS_REQUIRE(n >= 0 && (n == 0 || (in && sizes && dtypes)), GS_ERR_ARG, "gradients: null table or negative count");
  int64_t total = 0;
  for (int i = 0; i < n; ++i) {
    GS_REQUIRE(sizes[i] >= 0 && sizes[i] < (int64_t(1) << 40), GS_ERR_ARG, "gradient %d: invalid size", i);
    GS_REQUIRE(dtypes[i] == GS_FLOAT32 || dtypes[i] == GS_BFLOAT16, GS_ERR_ARG,
               "gradient %d: dtype must be GS_FLOAT32 or GS_BFLOAT16", i);
    GS_REQUIRE(sizes[i] == 0 || in[i], GS_ERR_ARG, "gradient %d: null pointer", i);
    GS_REQUIRE(aligned(in[i], dtypes[i] == GS_BFLOAT16 ? 2 : 4), GS_ERR_ALIGN, "gradient %d: misaligned", i);
    total += (sizes[i] + kClipPiece - 1) / kClipPiece;
  }
  GS_REQUIRE(total < (int64_t(1) << 31), GS_ERR_ARG, "gradients: too many elements");
  *pieces = total;
  return GS_OK;
}

// Calls f(table, workgroups, first piece) for launches of up to kClipTensors tensors; empty ones are left out.
template <typename F>
static int each_table(const void* const* in, void* const* out, const int64_t* sizes, const int32_t* dtypes, int n,
                      F f) {
  int64_t done = 0;
  for (int i = 0; i < n;) {
    ClipTable t = {};
    int64_t blocks = 0;
    for (; i < n && t.count < kClipTensors; ++i) {
      if (sizes[i] == 0) continue;
      const int k = t.count++;
      t.in[k] = in[i];
      t.out[k] = out ? out[i] : nullptr;
      t.n[k] = sizes[i];
      t.bf16[k] = dtypes[i] == GS_BFLOAT16;
      t.block0[k] = static_cast<int32_t>(blocks);
      blocks += (sizes[i] + kClipPiece - 1) / kClipPiece;
    }
    if (t.count == 0) continue;
    if (const int rc = f(t, blocks, done)) return rc;
    done += blocks;
  }
  return GS_OK;
}

}  // namespace gs

using namespace gs;

extern "C" size_t gs_grad_norm_workspace_size(const int64_t* sizes, int n) {
  clear_error();
  int64_t total = 0;
  for (int i = 0; sizes && i < n; ++i)
    if (sizes[i] > 0) total += (sizes[i] + kClipPiece - 1) / kClipPiece;
  return static_cast<size_t>(total) * sizeof(double);
}

extern "C" int gs_grad_norm(const void* const* grads, const int64_t* sizes, const int32_t* dtypes, int n,
                            double max_norm, float* norm, float* coef, void* workspace, size_t workspace_bytes,
                            void* stream) {
  clear_error();
  int64_t pieces;
  if (const int rc = check_tensors(grads, sizes, dtypes, n, &pieces)) return rc;
  GS_REQUIRE(norm, GS_ERR_ARG, "gradient norm: null output");
  GS_REQUIRE(coef == nullptr || max_norm >= 0.0, GS_ERR_ARG, "gradient norm: max_norm must be >= 0");
  GS_REQUIRE(workspace_bytes >= static_cast<size_t>(pieces) * sizeof(double) && (workspace || pieces == 0),
             GS_ERR_WORKSPACE, "gradient norm: workspace too small");
  GS_REQUIRE(aligned(workspace, 8) && aligned(norm, 4) && aligned(coef, 4), GS_ERR_ALIGN,
             "gradient norm: misaligned workspace or output");
  const hipStream_t st = as_stream(stream);
  double* sums = static_cast<double*>(workspace);
  const int rc = each_table(grads, nullptr, sizes, dtypes, n, [&](const ClipTable& t, int64_t blocks, int64_t at) {
    hipLaunchKernelGGL(norm_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kClipThreads), 0, st, t, sums + at);
    return check_launch("gradient norm");
  });
  if (rc) return rc;
  hipLaunchKernelGGL(norm_join_kernel, dim3(1), dim3(kClipThreads), 0, st, sums, pieces, max_norm, norm, coef);
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
  return each_table(grads, out, sizes, dtypes, n, [&](const ClipTable& t, int64_t blocks, int64_t) {
    hipLaunchKernelGGL(scale_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kClipThreads), 0, st, t, coef);
    return check_launch("gradient scale");
  });
}
