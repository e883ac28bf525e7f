// Rotary positions with several axes: pair p of a head (elements (p, p + P) or (2p, 2p + 1) of the
// first 2P) is turned by the angle position[axis(p)] * frequency(p); elements from 2P on are copied.
// The gradient is the same with the angle negated.
#include <float.h>

#include <algorithm>

#include "gs_host.h"

namespace gs {

struct RotaryTensor {
  const void* in;
  void* out;
  int64_t token_stride, head_stride;  // of `in`, in elements; `out` is contiguous
  int heads;
};

struct RotaryArgs {
  RotaryTensor x[2];
  const float* positions;
  int64_t tokens;
  int axes, pairs, dim, adjacent;
  int tokens_per_block;
  int section_end[GS_ROTARY_MAX_AXES];
  float sign;
  double freq[GS_ROTARY_MAX_PAIRS];  // in turns
};

constexpr int kRotaryThreads = 256;
constexpr int kRotaryTable = 1024;  // (token, pair) angles of a workgroup

// cos and sin of 2 pi pos f. The product is formed in float64 and reduced to a turn before it is rounded to
// float32, so the angle's error does not grow with the position until the product's own rounding counts: n
// turns are known to about n 2^-52 of a turn, less than float32's 2^-24 up to 2^28 turns, a position of 2^30 at a
// frequency of 1.
__device__ __forceinline__ float2 turn(float pos, double f) {
  const double t = static_cast<double>(pos) * f;
  float2 r;
  sincospif(2.0f * static_cast<float>(t - rint(t)), &r.y, &r.x);
  return r;
}

template <typename T>
__device__ __forceinline__ void rotate(T u, T w, float2 cs, T* u1, T* w1) {
  const float f = static_cast<float>(u), g = static_cast<float>(w);
  *u1 = static_cast<T>(fmaf(f, cs.x, -(g * cs.y)));
  *w1 = static_cast<T>(fmaf(f, cs.y, g * cs.x));
}

// HBM-bound: every element is read and written once, in vectors of V. A workgroup takes a few tokens:
// it forms their angles' cos and sin once, in LDS, for all heads of both tensors (a sincos costs as much
// as moving some 30 elements), then its threads run over (token, head, V pairs), neighbours in memory
// next to each other. V is 16 bytes' worth at whatever address (the memory system splits an access that
// crosses a line), less only where a head has fewer pairs or copied elements than that. The last vector of
// the pairs and of the rest ends where they end: where V does not divide them it overlaps the one before,
// and two threads write the same values to the same place. (One element a thread wherever 16 bytes do not
// divide all: 30000 tokens, 24 bfloat16 heads of 96 with 45 pairs 147 us, so 84; 16 + 4 heads of 64 with 31
// pairs 69 us, so 46; 4099 tokens, 9 float32 heads of 72 with 31 pairs 10.9 us, so 8.1.) 32771 tokens, 16 + 16 heads of 64 bfloat16 out of a
// packed projection: 61 us, 4.4 TB/s (171 us with the angles formed per head and one element a thread).
template <typename T, int V>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(RotaryArgs a) {
  typedef T Vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  __shared__ float2 table[kRotaryTable];
  const int64_t token0 = static_cast<int64_t>(blockIdx.x) * a.tokens_per_block;
  const int n_tokens = static_cast<int>(min<int64_t>(a.tokens_per_block, a.tokens - token0));
  for (int e = threadIdx.x; e < n_tokens * a.pairs; e += kRotaryThreads) {
    const int t = e / a.pairs, p = e - t * a.pairs;
    int axis = 0;
    while (axis + 1 < a.axes && p >= a.section_end[axis]) ++axis;
    float2 cs = turn(a.positions[(token0 + t) * a.axes + axis], a.freq[p]);
    cs.y *= a.sign;
    table[e] = cs;
  }
  __syncthreads();
  const int turns = (a.pairs + V - 1) / V, rest = a.dim - 2 * a.pairs, per_head = turns + (rest + V - 1) / V;
  const int heads = a.x[0].heads + a.x[1].heads;
  const int per_token = heads * per_head;
  // four items of a thread at a time, their loads first
  constexpr int U = 4;
  const int n = n_tokens * per_token;
  for (int e0 = threadIdx.x; e0 < n; e0 += U * kRotaryThreads) {
    Vec b0[U], b1[U];
    T* to[U];
    int at[U];  // first angle, or -1: copied elements
#pragma unroll
    for (int q = 0; q < U; ++q) {
      const int e = min(e0 + q * kRotaryThreads, n - 1);
      const int t = e / per_token, th = e - t * per_token;
      int head = th / per_head;
      const int c = th - head * per_head;
      const int which = head >= a.x[0].heads;
      head -= which ? a.x[0].heads : 0;
      const RotaryTensor& x = a.x[which];
      const int64_t token = token0 + t;
      const int p = min(c * V, a.pairs - V);
      const int i = c >= turns ? 2 * a.pairs + min((c - turns) * V, rest - V) : a.adjacent ? 2 * p : p;
      const T* in = static_cast<const T*>(x.in) + token * x.token_stride + head * x.head_stride + i;
      to[q] = static_cast<T*>(x.out) + (token * x.heads + head) * a.dim + i;
      at[q] = c >= turns ? -1 : t * a.pairs + p;
      b0[q] = *reinterpret_cast<const Vec*>(in);
      b1[q] = c >= turns ? b0[q] : *reinterpret_cast<const Vec*>(in + (a.adjacent ? V : a.pairs));
    }
#pragma unroll
    for (int q = 0; q < U; ++q) {
      if (e0 + q * kRotaryThreads >= n) break;
      if (at[q] < 0) {
        *reinterpret_cast<Vec*>(to[q]) = b0[q];
        continue;
      }
      const float2* cs = table + at[q];
      Vec y0, y1;
      if (a.adjacent) {
        T u[2 * V], y[2 * V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
          u[k] = b0[q][k];
          u[V + k] = b1[q][k];
        }
#pragma unroll
        for (int k = 0; k < V; ++k) rotate(u[2 * k], u[2 * k + 1], cs[k], &y[2 * k], &y[2 * k + 1]);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          y0[k] = y[k];
          y1[k] = y[V + k];
        }
      } else {
#pragma unroll
        for (int k = 0; k < V; ++k) {
          T f, w;
          rotate(static_cast<T>(b0[q][k]), static_cast<T>(b1[q][k]), cs[k], &f, &w);
          y0[k] = f;
          y1[k] = w;
        }
      }
      *reinterpret_cast<Vec*>(to[q]) = y0;
      *reinterpret_cast<Vec*>(to[q] + (a.adjacent ? V : a.pairs)) = y1;
    }
  }
}

}  // namespace gs

using namespace gs;

extern "C" int gs_rotary_axes(const gs_rotary* p, void* stream) {
  clear_error();
  GS_REQUIRE(p != nullptr, GS_ERR_ARG, "rotary: arguments are NULL");
  GS_REQUIRE(p->dtype == GS_FLOAT32 || p->dtype == GS_BFLOAT16, GS_ERR_ARG,
             "rotary: dtype must be GS_FLOAT32 or GS_BFLOAT16");
  GS_REQUIRE(p->axes >= 1 && p->axes <= GS_ROTARY_MAX_AXES, GS_ERR_ARG, "rotary: 1 to %d axes", GS_ROTARY_MAX_AXES);
  GS_REQUIRE(p->tokens >= 0 && p->tokens < (int64_t(1) << 31) && p->q_heads >= 0 && p->k_heads >= 0 &&
                 p->q_heads + p->k_heads >= 1 && p->q_heads <= (1 << 16) && p->k_heads <= (1 << 16),
             GS_ERR_ARG, "rotary: invalid token or head count");
  GS_REQUIRE(p->base > 0.0 && p->base <= DBL_MAX, GS_ERR_ARG, "rotary: base must be positive and finite");
  RotaryArgs a = {};
  for (int i = 0; i < p->axes; ++i) {
    GS_REQUIRE(p->sections[i] >= 0 && p->sections[i] <= GS_ROTARY_MAX_PAIRS, GS_ERR_ARG,
               "rotary: section %d of %d pairs", i, p->sections[i]);
    a.pairs += p->sections[i];
    a.section_end[i] = a.pairs;
  }
  GS_REQUIRE(a.pairs >= 1 && a.pairs <= GS_ROTARY_MAX_PAIRS && 2 * a.pairs <= p->dim && p->dim <= (1 << 16),
             GS_ERR_ARG, "rotary: %d pairs do not fit a head of %d elements (at most %d pairs)", a.pairs, p->dim,
             GS_ROTARY_MAX_PAIRS);
  const bool work = p->tokens > 0;
  GS_REQUIRE(!work || (p->positions && (!p->q_heads || (p->q && p->q_out)) && (!p->k_heads || (p->k && p->k_out))),
             GS_ERR_ARG, "rotary: null pointer");
  const size_t es = p->dtype == GS_BFLOAT16 ? 2 : 4;
  GS_REQUIRE(aligned(p->q, es) && aligned(p->k, es) && aligned(p->q_out, es) && aligned(p->k_out, es) &&
                 aligned(p->positions, 4), GS_ERR_ALIGN, "rotary: misaligned tensor");
  if (!work) return GS_OK;
  a.x[0] = {p->q, p->q_out, p->q_token_stride, p->q_head_stride, p->q_heads};
  a.x[1] = {p->k, p->k_out, p->k_token_stride, p->k_head_stride, p->k_heads};
  a.positions = p->positions;
  a.tokens = p->tokens;
  a.axes = p->axes;
  a.dim = p->dim;
  a.adjacent = p->flags & GS_ROTARY_ADJACENT ? 1 : 0;
  a.sign = p->flags & GS_ROTARY_INVERSE ? -1.0f : 1.0f;
  const double ln = log(p->base);
  for (int axis = 0, i = 0; axis < p->axes; ++axis)
    for (int j = 0; j < p->sections[axis]; ++j, ++i) {
      const double x = p->flags & GS_ROTARY_SHARED ? static_cast<double>(i) / a.pairs
                                                   : static_cast<double>(j) / p->sections[axis];
      a.freq[i] = exp(-x * ln) * 0.15915494309189533577;
    }
  // the widest vector that fits into the pairs and into the rest
  const int rest = p->dim - 2 * a.pairs;
  int v = static_cast<int>(16 / es);
  while (v > 1 && (a.pairs < v || (rest > 0 && rest < v))) v /= 2;
  // Tokens of a workgroup: eight items a thread, if that leaves workgroups for the whole chip.
  const int64_t items = static_cast<int64_t>(p->q_heads + p->k_heads) * ((a.pairs + v - 1) / v + (rest + v - 1) / v);
  GS_REQUIRE(items < (1 << 26), GS_ERR_ARG, "rotary: too many heads");
  int64_t per = (8 * kRotaryThreads + items - 1) / items;
  per = std::min<int64_t>({per, kRotaryTable / a.pairs, (p->tokens + 1023) / 1024});
  a.tokens_per_block = static_cast<int>(std::max<int64_t>(1, per));
  const int64_t blocks = (p->tokens + a.tokens_per_block - 1) / a.tokens_per_block;
  GS_REQUIRE(blocks * kRotaryThreads < (int64_t(1) << 32), GS_ERR_ARG, "rotary: too many tokens");
  const dim3 grid(static_cast<unsigned>(blocks));
  const dim3 block(kRotaryThreads);
  const hipStream_t st = as_stream(stream);
  const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, st, a); };
  if (p->dtype == GS_BFLOAT16) {
    if (v == 8) launch(rotary_kernel<__bf16, 8>);
    else if (v == 4) launch(rotary_kernel<__bf16, 4>);
    else if (v == 2) launch(rotary_kernel<__bf16, 2>);
    else launch(rotary_kernel<__bf16, 1>);
  } else {
    if (v == 4) launch(rotary_kernel<float, 4>);
    else if (v == 2) launch(rotary_kernel<float, 2>);
    else launch(rotary_kernel<float, 1>);
  }
  return check_launch("rotary");
}
