// Rotary positions with several axes: pair p of a head (elements (p, p + P) or (2p, 2p + 1) of the
// first 2P) is turned by the angle position[axis(p)] * frequency(p); elements from 2P on are copied.
// The gradient is the same with the angle negated.
#include <float.h>

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
  int section_end[GS_ROTARY_MAX_AXES];
  float sign;
  // frequency in turns, as the sum of two floats
  float freq_hi[GS_ROTARY_MAX_PAIRS], freq_lo[GS_ROTARY_MAX_PAIRS];
};

constexpr int kRotaryThreads = 256;

// cos and sin of 2 pi pos f. The product is formed to about 48 bits and reduced to a turn before
// anything is rounded, so the angle's error does not grow with the position.
__device__ __forceinline__ void turn(float pos, float hi, float lo, float* c, float* s) {
  const float ph = pos * hi;
  const float pl = fmaf(pos, lo, fmaf(pos, hi, -ph));
  const float f = (ph - rintf(ph)) + pl;
  sincospif(2.0f * f, s, c);
}

template <typename T>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(RotaryArgs a) {
  const int per_head = a.dim - a.pairs;  // pairs, then copied elements
  const int heads = a.x[0].heads + a.x[1].heads;
  const int64_t e = static_cast<int64_t>(blockIdx.x) * kRotaryThreads + threadIdx.x;
  if (e >= a.tokens * heads * per_head) return;
  const int p = static_cast<int>(e % per_head);
  const int64_t th = e / per_head;
  int head = static_cast<int>(th % heads);
  const int64_t token = th / heads;
  const int which = head >= a.x[0].heads;
  head -= which ? a.x[0].heads : 0;
  const RotaryTensor& x = a.x[which];
  const T* in = static_cast<const T*>(x.in) + token * x.token_stride + head * x.head_stride;
  T* out = static_cast<T*>(x.out) + (token * x.heads + head) * a.dim;
  if (p >= a.pairs) {
    out[p + a.pairs] = in[p + a.pairs];
    return;
  }
  int axis = 0;
  while (axis + 1 < a.axes && p >= a.section_end[axis]) ++axis;
  float c, s;
  turn(a.positions[token * a.axes + axis], a.freq_hi[p], a.freq_lo[p], &c, &s);
  s *= a.sign;
  const int i = a.adjacent ? 2 * p : p, j = a.adjacent ? 2 * p + 1 : p + a.pairs;
  const float u = static_cast<float>(in[i]), w = static_cast<float>(in[j]);
  out[i] = static_cast<T>(fmaf(u, c, -(w * s)));
  out[j] = static_cast<T>(fmaf(u, s, w * c));
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
      const double f = exp(-x * ln) * 0.15915494309189533577;  // turns
      a.freq_hi[i] = static_cast<float>(f);
      a.freq_lo[i] = static_cast<float>(f - a.freq_hi[i]);
    }
  const int64_t n = p->tokens * (p->q_heads + p->k_heads) * (p->dim - a.pairs);
  const int64_t blocks = (n + kRotaryThreads - 1) / kRotaryThreads;
  GS_REQUIRE(blocks < (int64_t(1) << 31), GS_ERR_ARG, "rotary: too many elements");
  const dim3 grid(static_cast<unsigned>(blocks)), block(kRotaryThreads);
  if (p->dtype == GS_BFLOAT16)
    hipLaunchKernelGGL(rotary_kernel<__bf16>, grid, block, 0, as_stream(stream), a);
  else
    hipLaunchKernelGGL(rotary_kernel<float>, grid, block, 0, as_stream(stream), a);
  return check_launch("rotary");
}
