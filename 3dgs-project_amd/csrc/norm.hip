// Norms before and after a block, fused with what lies between them, forward and backward:
//
//   b = y, or post(y) = w' y^ + b'        y^ = (y - mean) / sqrt(var + eps), or without a mean y / sqrt(mean y^2 + eps)
//   h = x + scale gate k b                k: the dropout's factors, formed from the counter (gs_philox.h)
//   n = w h^ + b                          h^: h standardised in the same way
//
// and dropout alone. A row is held in the registers of 64 to 512 lanes from its one reading to its one writing;
// deviations are taken from the mean, not from the sum of squares. The backward pass forms h and its
// standardised rows again from x, y and four saved statistics a row, so that nothing else is kept:
//
//   t = dn w;  D = dh + (t - h^ mean(t h^) [- mean t]) / dev        dx = D
//   dgate = sum or each of scale D k b;   v = scale D gate k;   dw' = sum v y^, db' = sum v;  dw = sum dn h^, db = sum dn
//   q = v w';  dy = (q - y^ mean(q y^) [- mean q]) / dev'
//
// Column sums are kept in registers over the rows of a workgroup, joined in LDS, written as one part a workgroup
// and summed in a fixed order: no atomics, the same inputs give the same bits.
//
// Memory bounds all of it: 32771 x 1024 of a float32 stream and a bfloat16 branch, rms norms, gate and dropout, forward
// 403 MB in 76 us (5.3 TB/s), backward 604 MB in 139 us (4.3 TB/s; its two sums over a row stand between loads and stores),
// the column sums' join 5 us; one row 4.0 us. Widths above 4096 go backward at less than half of that: see with_bwd.
#include <algorithm>

#include "gs_philox.h"
#include "gs_rows.h"

namespace gs {

struct NormArgs {
  const void *x, *y, *weight, *bias, *post_weight, *post_bias, *gate;
  void *h, *n;
  float* stats;  // [rows][4]: mean and 1 / deviation of h, of y
  int64_t rows, x_stride, y_stride, gate_stride;
  int64_t first;  // row of a forward launch
  int width;
  bool layer, post, weights_bf16, gate_bf16;
  float eps, scale, inv_width;
  DropRule drop;
  // backward
  const void *d_h, *d_n;
  void *d_x, *d_y, *d_gate_rows;
  float* parts;      // [workgroups][sums][width]
  int sums;          // of the five column sums
  int8_t slot[5];    // where they are among these, -1: not wanted
};
enum { kSumWeight = 0, kSumBias, kSumPostWeight, kSumPostBias, kSumGate };

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 1; o < kWave; o *= 2) v += __shfl_xor(v, o);
  return v;
}

// Sums of two values over the G lanes of a row; `turn` alternates between two sets of LDS words, so that one barrier
// a sum is enough.
template <int G, int GROUPS>
struct RowSum {
  float2 (*lds)[GROUPS][G / kWave];
  int turn = 0;
  __device__ __forceinline__ float2 operator()(float a, float b) {
    a = wave_sum(a);
    b = wave_sum(b);
    if constexpr (G > kWave) {
      const int group = threadIdx.x / G, wave = threadIdx.x % G / kWave;
      if (threadIdx.x % kWave == 0) lds[turn][group][wave] = make_float2(a, b);
      __syncthreads();
      a = b = 0.0f;
#pragma unroll
      for (int i = 0; i < G / kWave; ++i) {
        a += lds[turn][group][i].x;
        b += lds[turn][group][i].y;
      }
      turn ^= 1;
    }
    return make_float2(a, b);
  }
};

// Where a lane's vector of eight lies in a row, and how many of its elements are the row's. WHOLE: the width is a multiple of
// eight, so that a vector is the row's or not; lanes past the end then load the last one and are masked, and
// no load needs a branch.
template <bool WHOLE>
struct Piece8 {
  int col, n;
  Piece8() = default;
  __device__ __forceinline__ Piece8(int col_, int width) : col(col_), n(width - col_) {
    if constexpr (WHOLE) {
      col = min(col_, width - 8);
      n = n > 0 ? 8 : 0;
    }
  }
  __device__ __forceinline__ int loaded() const { return WHOLE ? 8 : n; }
  __device__ __forceinline__ bool has(int j) const { return WHOLE ? n > 0 : j < n; }
};

// Mean and 1 / deviation of a row held in registers (elements that are not the row's are zero).
template <int NV, bool WHOLE, typename S>
__device__ __forceinline__ float2 row_stats(const NormArgs& a, const float (&v)[NV][8], const Piece8<WHOLE> (&at)[NV], S& sum) {
  float mean = 0.0f;
  if (a.layer) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[i][j];
    mean = sum(s, 0.0f).x * a.inv_width;
  }
  float q = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float d = at[i].has(j) ? v[i][j] - mean : 0.0f;
      q = fmaf(d, d, q);
    }
  const float var = sum(q, 0.0f).x * a.inv_width;
  return make_float2(mean, 1.0f / sqrtf(var + a.eps));
}

// What lies between y and h of eight elements, as loaded.
struct Between8 {
  RawAny8 w, b, g;
  template <bool WHOLE>
  __device__ __forceinline__ void load(const NormArgs& a, int64_t row, const Piece8<WHOLE>& at) {
    if (a.post) w.load(a.post_weight, a.weights_bf16, at.col, at.loaded());
    if (a.post_bias) b.load(a.post_bias, a.weights_bf16, at.col, at.loaded());
    if (a.gate) g.load(a.gate, a.gate_bf16, row * a.gate_stride + at.col, at.loaded());
  }
  // u = k b from y (given standardised as `hat`), and the factors f = scale gate and k.
  __device__ __forceinline__ void form(const NormArgs& a, uint64_t seed, int64_t row, int col, const float (&hat)[8],
                                       float (&f)[8], float (&k)[8], float (&u)[8]) const {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = hat[j], f[j] = a.scale, k[j] = 1.0f;
    if (a.post) {
      w.to(v);
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] *= v[j];
      if (a.post_bias) {
        b.to(v);
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] += v[j];
      }
    }
    if (a.gate) {
      g.to(v);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] *= v[j];
    }
    if (a.drop.threshold) {
      keep8(a.drop, seed, static_cast<uint32_t>(row), col / 8, k);
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = k[j] != 0.0f ? u[j] * k[j] : 0.0f;
    }
  }
};

// G lanes a row, each NV vectors of eight: vector i of lane l begins at 8 (l + G i).
template <typename X, typename Y, int G, int NV, bool WHOLE>
__global__ __launch_bounds__(G > 256 ? G : 256) void norm_fwd_kernel(NormArgs a) {
  constexpr int kGroups = G > 256 ? 1 : 256 / G;
  __shared__ float2 lds[2][kGroups][G / kWave];
  RowSum<G, kGroups> sum{lds};
  const int lane = threadIdx.x % G;
  const int64_t row_at = a.first + static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / G;
  // (groups past the last row repeat it without writing: every lane meets every barrier)
  const bool mine = row_at < a.rows;
  const int64_t row = mine ? row_at : a.rows - 1;
  Piece8<WHOLE> at[NV];
  Raw8<X> rx[NV];
  Raw8<Y> ry[NV];
  RawAny8 rw[NV], rb[NV];
  Between8 mid[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    at[i] = {8 * (lane + G * i), a.width};
    rx[i].load(static_cast<const X*>(a.x) + row * a.x_stride + at[i].col, at[i].loaded());
    if (a.y) {
      ry[i].load(static_cast<const Y*>(a.y) + row * a.y_stride + at[i].col, at[i].loaded());
      mid[i].load(a, row, at[i]);
    }
    if (a.weight) rw[i].load(a.weight, a.weights_bf16, at[i].col, at[i].loaded());
    if (a.bias) rb[i].load(a.bias, a.weights_bf16, at[i].col, at[i].loaded());
  }
  float h[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    rx[i].to(h[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) h[i][j] = at[i].has(j) ? h[i][j] : 0.0f;
  }
  if (a.y) {
    float b[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      ry[i].to(b[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) b[i][j] = at[i].has(j) ? b[i][j] : 0.0f;
    }
    float2 st = {0.0f, 1.0f};
    if (a.post) st = row_stats(a, b, at, sum);
    if (mine && lane == 0 && a.stats) {
      a.stats[4 * row + 2] = st.x;
      a.stats[4 * row + 3] = st.y;
    }
    const uint64_t seed = a.drop.threshold ? seed_of(a.drop) : 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float f[8], k[8], u[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) b[i][j] = (b[i][j] - st.x) * st.y;  // (without a post norm y itself)
      mid[i].form(a, seed, row, at[i].col, b[i], f, k, u);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[i][j] = at[i].has(j) ? fmaf(f[j], u[j], h[i][j]) : 0.0f;
      if (mine && at[i].n > 0) store8(static_cast<X*>(a.h) + row * a.width + at[i].col, at[i].n, h[i]);
    }
  }
  const float2 st = row_stats(a, h, at, sum);
  if (mine && lane == 0 && a.stats) {
    a.stats[4 * row] = st.x;
    a.stats[4 * row + 1] = st.y;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float w[8], n[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) n[j] = (h[i][j] - st.x) * st.y;
    if (a.weight) {
      rw[i].to(w);
#pragma unroll
      for (int j = 0; j < 8; ++j) n[j] *= w[j];
    }
    if (a.bias) {
      rb[i].to(w);
#pragma unroll
      for (int j = 0; j < 8; ++j) n[j] += w[j];
    }
    if (mine && at[i].n > 0) store8(static_cast<Y*>(a.n) + row * a.width + at[i].col, at[i].n, n);
  }
}

// NV 1: what differs from row to row is loaded a row ahead, which takes the registers that 256 lanes' workgroups of two
// wavefronts a SIMD have left (32771 x 1024: 168 us without, 139 with; sixteen elements a lane, a row a wavefront: 217).
template <typename X, typename Y, int G, int NV, bool WHOLE>
__global__ __launch_bounds__(G > 256 ? G : 256, 2) void norm_bwd_kernel(NormArgs a) {
  constexpr int kGroups = G > 256 ? 1 : 256 / G;
  constexpr int kWidth = 8 * G * NV;
  __shared__ float2 lds[2][kGroups][G / kWave];
  __shared__ float join[kGroups > 1 ? kGroups * kWidth : 1];
  RowSum<G, kGroups> sum{lds};
  const int lane = threadIdx.x % G;
  // Column sums: in registers, or with sixteen elements a lane, but for the bias', in the lane's own place in LDS
  constexpr bool kInLds = NV > 1;
  __shared__ float4 held[kInLds ? 4 : 1][kInLds ? NV : 1][2][kInLds ? G : 1];
  float col_sum[5][NV][8] = {};
  const auto place = [&](int k, int i, int half) -> float4& { return held[k - (k > kSumBias)][i][half][lane]; };
  const auto add = [&](int k, int i, const float (&p)[8], const float (&q)[8]) {
    if (kInLds && k != kSumBias) {
      if (a.slot[k] < 0) return;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float4& to = place(k, i, half);
        float4 c = to;
        c.x = fmaf(p[4 * half], q[4 * half], c.x);
        c.y = fmaf(p[4 * half + 1], q[4 * half + 1], c.y);
        c.z = fmaf(p[4 * half + 2], q[4 * half + 2], c.z);
        c.w = fmaf(p[4 * half + 3], q[4 * half + 3], c.w);
        to = c;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) col_sum[k][i][j] = fmaf(p[j], q[j], col_sum[k][i][j]);
    }
  };
  constexpr float kOnes[8] = {1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f};
  if constexpr (kInLds) {
    for (int k = 0; k < 5; ++k)
      for (int i = 0; i < NV; ++i)
        if (k != kSumBias) place(k, i, 0) = place(k, i, 1) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  Piece8<WHOLE> at[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) at[i] = {8 * (lane + G * i), a.width};
  const uint64_t seed = a.drop.threshold ? seed_of(a.drop) : 0;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
  struct Row {
    Raw8<X> x[NV], d_h[NV];
    Raw8<Y> y[NV], d_n[NV];
    float4 stats;
  };
  const auto fetch = [&](Row& r, int64_t row) {
    row = row < a.rows ? row : a.rows - 1;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = at[i].col, n = at[i].loaded();
      r.x[i].load(static_cast<const X*>(a.x) + row * a.x_stride + col, n);
      r.d_n[i].load(static_cast<const Y*>(a.d_n) + row * a.width + col, a.d_n ? n : 0);
      r.d_h[i].load(static_cast<const X*>(a.d_h) + row * a.width + col, a.d_h ? n : 0);
      if (a.y) r.y[i].load(static_cast<const Y*>(a.y) + row * a.y_stride + col, n);
    }
    r.stats = *reinterpret_cast<const float4*>(a.stats + 4 * row);
  };
  constexpr bool kAhead = NV == 1;
  Row next;
  if (kAhead) fetch(next, static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / G);
  // (the groups of a workgroup take as many turns as its first one: barriers are met by all)
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * kGroups; first < a.rows; first += step) {
    const int64_t row_at = first + threadIdx.x / G;
    const bool mine = row_at < a.rows;
    const int64_t row = mine ? row_at : a.rows - 1;
    if (!kAhead) fetch(next, row_at);
    const Row now = next;
    RawAny8 rw[NV];
    Between8 mid[NV];
    const auto weights = [&](int i) {
      if (a.weight) rw[i].load(a.weight, a.weights_bf16, at[i].col, at[i].loaded());
      if (a.y) mid[i].load(a, row, at[i]);
    };
    if (!kInLds) {
#pragma unroll
      for (int i = 0; i < NV; ++i) weights(i);
    }
    if (kAhead) fetch(next, row_at + step);
    const float4 st = now.stats;
    float hat[NV][8], t[NV][8], b[NV][8], u[NV][8], fk[NV][8];
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (kInLds) weights(i);
      now.x[i].to(hat[i]);
      if (a.y) {
        float f[8], k[8];
        now.y[i].to(b[i]);
        if (a.post) {
#pragma unroll
          for (int j = 0; j < 8; ++j) b[i][j] = (b[i][j] - st.z) * st.w;
        }
        mid[i].form(a, seed, row, at[i].col, b[i], f, k, u[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          hat[i][j] = fmaf(f[j], u[i][j], hat[i][j]);
          // (+0 + -0 is +0: only what is dropped has -0, so that its gradient can be zero whatever arrives)
          fk[i][j] = k[j] != 0.0f ? fmaf(f[j], k[j], 0.0f) : -0.0f;
        }
      }
      now.d_n[i].to(t[i]);
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = 1.0f;
      if (a.weight) rw[i].to(w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool has = mine && a.d_n && at[i].has(j);
        hat[i][j] = has ? (hat[i][j] - st.x) * st.y : 0.0f;
        t[i][j] = has ? t[i][j] : 0.0f;
      }
      add(kSumWeight, i, t[i], hat[i]);
      add(kSumBias, i, t[i], kOnes);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        t[i][j] = mine && at[i].has(j) ? t[i][j] * w[j] : 0.0f;
        s1 = fmaf(t[i][j], hat[i][j], s1);
        s2 += t[i][j];
      }
      if (kInLds) __builtin_amdgcn_sched_barrier(0);
    }
    const float2 m = sum(s1, s2);
    const float m1 = m.x * a.inv_width, m2 = a.layer ? m.y * a.inv_width : 0.0f;
    const float inv = a.d_n ? st.y : 0.0f;  // (a norm whose result goes nowhere adds nothing, whatever the row holds)
    s1 = s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const bool some = mine && at[i].n > 0;
      float d[8];
      now.d_h[i].to(d);
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] += inv * (t[i][j] - fmaf(hat[i][j], m1, m2));
      if (a.d_x && some) store8(static_cast<X*>(a.d_x) + row * a.width + at[i].col, at[i].n, d);
      if (!a.y) continue;
      float e[8], w[8];
      if (a.post && kInLds) mid[i].w.load(a.post_weight, a.weights_bf16, at[i].col, at[i].loaded());
      if (a.post) mid[i].w.to(w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool has = mine && at[i].has(j);
        e[j] = has ? a.scale * d[j] * u[i][j] : 0.0f;  // of the gate
        t[i][j] = has && __float_as_uint(fk[i][j]) != 0x80000000u ? d[j] * fk[i][j] : 0.0f;
        if (a.post) b[i][j] = has ? b[i][j] : 0.0f;
      }
      add(kSumGate, i, e, kOnes);
      if (a.post) {
        add(kSumPostWeight, i, t[i], b[i]);
        add(kSumPostBias, i, t[i], kOnes);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          t[i][j] = mine && at[i].has(j) ? t[i][j] * w[j] : 0.0f;
          s1 = fmaf(t[i][j], b[i][j], s1);
          s2 += t[i][j];
        }
      }
      if (a.d_gate_rows && some) store8(a.d_gate_rows, a.gate_bf16, row * a.width + at[i].col, at[i].n, e);
      if (kInLds) __builtin_amdgcn_sched_barrier(0);
    }
    if (!a.y) continue;
    if (a.post) {
      const float2 p = sum(s1, s2);
      const float p1 = p.x * a.inv_width, p2 = a.layer ? p.y * a.inv_width : 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) t[i][j] = st.w * (t[i][j] - fmaf(b[i][j], p1, p2));
    }
    if (a.d_y) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (mine && at[i].n > 0) store8(static_cast<Y*>(a.d_y) + row * a.width + at[i].col, at[i].n, t[i]);
    }
  }
#pragma unroll
  for (int k = 0; k < 5; ++k) {
    if (a.slot[k] < 0) continue;
    float* part = a.parts + (static_cast<int64_t>(blockIdx.x) * a.sums + a.slot[k]) * a.width;
    if constexpr (kGroups == 1) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (kInLds && k != kSumBias) {
          const float4 lo = place(k, i, 0), hi = place(k, i, 1);
          const float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
          if (at[i].n > 0) store8(part + at[i].col, at[i].n, v);
        } else if (at[i].n > 0) {
          store8(part + at[i].col, at[i].n, col_sum[k][i]);
        }
      }
    } else {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) join[(threadIdx.x / G) * kWidth + 8 * (lane + G * i) + j] = col_sum[k][i][j];
      __syncthreads();
      for (int c = threadIdx.x; c < a.width; c += 256) {
        float s = join[c];
#pragma unroll
        for (int g = 1; g < kGroups; ++g) s += join[g * kWidth + c];
        part[c] = s;
      }
    }
  }
}

// Dropout alone: a vector of eight a thread. 8203 x 4096 in bfloat16 22.5 us (6.0 TB/s, partly from the last-level cache),
// 32768 x 4096 88 us (6.1 TB/s), 8203 x 4096 in float32 41 us: memory bounds it, the generator's 20 products for
// eight elements lie under its loads.
constexpr int kDropThreads = 256;
template <typename T>
__global__ __launch_bounds__(kDropThreads) void dropout_kernel(const T* x, T* out, int64_t rows, int64_t stride,
                                                               int width, int groups, DropRule drop) {
  const uint64_t seed = seed_of(drop);
  const int64_t all = rows * groups;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kDropThreads + threadIdx.x;
  if (i >= all) return;
  const int64_t row = i / groups;
  const int group = static_cast<int>(i - row * groups), n = width - 8 * group;
  float v[8], keep[8];
  load8(x + row * stride + 8 * group, n, v);
  keep8(drop, seed, static_cast<uint32_t>(row), group, keep);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = keep[j] != 0.0f ? v[j] * keep[j] : 0.0f;
  store8(out + row * width + 8 * group, n, v);
}

// Workgroups of the backward pass: two a CU, so that the parts stay small beside the rows (at 1024 columns and
// three sums 6 MB written and read).
constexpr int64_t kNormParts = 512;
static int64_t norm_parts(int64_t rows) { return std::min<int64_t>(kNormParts, rows); }

// Workgroups of one launch of the forward, below the 2^32 threads that a grid may have: more rows take several.
constexpr int64_t kNormLaunch = 1 << 22;

static int check_norm(const gs_residual_norm* p, bool backward, NormArgs* a) {
  GS_REQUIRE(p, GS_ERR_ARG, "residual norm: args is NULL");
  GS_REQUIRE(row_type(p->x_dtype) && row_type(p->y_dtype), GS_ERR_ARG,
             "residual norm: dtypes must be GS_FLOAT32 or GS_BFLOAT16");
  GS_REQUIRE(p->x_dtype == GS_FLOAT32 || p->y_dtype == GS_BFLOAT16, GS_ERR_ARG,
             "residual norm: a bfloat16 stream takes a bfloat16 branch and norm");
  GS_REQUIRE((!p->weight && !p->bias && !p->post_weight && !p->post_bias) || row_type(p->weight_dtype), GS_ERR_ARG,
             "residual norm: weight dtype must be GS_FLOAT32 or GS_BFLOAT16");
  GS_REQUIRE(!p->gate || row_type(p->gate_dtype), GS_ERR_ARG, "residual norm: gate dtype must be GS_FLOAT32 or GS_BFLOAT16");
  GS_REQUIRE(p->rows >= 0 && p->rows < (int64_t(1) << 31), GS_ERR_ARG, "residual norm: invalid row count");
  GS_REQUIRE(p->width >= 1 && p->width <= GS_NORM_MAX_WIDTH, GS_ERR_ARG, "residual norm: width %d: 1 to %d are provided",
             p->width, GS_NORM_MAX_WIDTH);
  GS_REQUIRE(p->rows * p->width < (int64_t(1) << 38), GS_ERR_ARG, "residual norm: too many elements");
  GS_REQUIRE(p->eps > 0.0f && p->eps <= 1e30f, GS_ERR_ARG, "residual norm: eps must be positive and finite");
  GS_REQUIRE(p->scale - p->scale == 0.0f, GS_ERR_ARG, "residual norm: scale must be finite");
  GS_REQUIRE(p->dropout >= 0.0 && p->dropout < 1.0, GS_ERR_ARG, "residual norm: dropout must be at least 0 and below 1");
  GS_REQUIRE(p->y || (!p->gate && !p->post_weight && !p->post_bias && p->dropout == 0.0), GS_ERR_ARG,
             "residual norm: a gate, a post norm or dropout needs y");
  GS_REQUIRE(!p->post_bias || p->post_weight, GS_ERR_ARG, "residual norm: a post bias needs a post weight");
  GS_REQUIRE(p->rows == 0 || (p->x && (backward || (p->n && (!p->y || p->h)))), GS_ERR_ARG, "residual norm: null pointer");
  const size_t xs = row_type_bytes(p->x_dtype), ys = row_type_bytes(p->y_dtype), ws = row_type_bytes(p->weight_dtype);
  GS_REQUIRE(aligned(p->x, xs) && aligned(p->h, xs) && aligned(p->y, ys) && aligned(p->n, ys) && aligned(p->weight, ws) &&
                 aligned(p->bias, ws) && aligned(p->post_weight, ws) && aligned(p->post_bias, ws) &&
                 aligned(p->gate, row_type_bytes(p->gate_dtype)) && aligned(p->stats, 16) && aligned(p->seed_at, 8),
             GS_ERR_ALIGN, "residual norm: misaligned tensor");
  *a = {};
  a->x = p->x;
  a->y = p->y;
  a->weight = p->weight;
  a->bias = p->bias;
  a->post_weight = p->post_weight;
  a->post_bias = p->post_bias;
  a->gate = p->gate;
  a->h = p->h;
  a->n = p->n;
  a->stats = p->stats;
  a->rows = p->rows;
  a->x_stride = p->x_stride;
  a->y_stride = p->y_stride;
  a->gate_stride = p->gate_rows ? p->gate_stride : 0;
  a->width = p->width;
  a->layer = p->layer != 0;
  a->post = p->post_weight != nullptr;
  a->weights_bf16 = p->weight_dtype == GS_BFLOAT16;
  a->gate_bf16 = p->gate_dtype == GS_BFLOAT16;
  a->eps = p->eps;
  a->scale = p->scale;
  a->inv_width = static_cast<float>(1.0 / p->width);
  a->drop = drop_rule(p->dropout, p->seed_at, p->seed, p->draw);
  return GS_OK;
}

// Calls f(kernel, lanes a row) with the instance for a width: as many lanes as leave eight elements each (sixteen in the
// forward, where a wavefront's own row needs no barrier). Above 4096 the backward has too few registers: it keeps its column sums in
// LDS and loads the weights twice, and still some of a row goes through memory: 4096 x 8192 trained by 512 lanes of
// sixteen 412 us (829 with the sums in registers), by 1024 of eight 511; rows wider than 8192 are refused. Widths that
// are no multiple of eight take branches for their last vector: 32771 x 1024 by those instances 88 us forward and 220 with
// its backward, so 77 and 211.
template <typename X, typename Y, bool WHOLE, typename F>
static int with_fwd(int width, F f) {
  if (width <= 512) return f(norm_fwd_kernel<X, Y, 64, 1, WHOLE>, 64);
  if (width <= 1024) return f(norm_fwd_kernel<X, Y, 64, 2, WHOLE>, 64);
  if (width <= 2048) return f(norm_fwd_kernel<X, Y, 256, 1, WHOLE>, 256);
  if (width <= 4096) return f(norm_fwd_kernel<X, Y, 256, 2, WHOLE>, 256);
  return f(norm_fwd_kernel<X, Y, 512, 2, WHOLE>, 512);
}
template <typename X, typename Y, bool WHOLE, typename F>
static int with_bwd(int width, F f) {
  if (width <= 512) return f(norm_bwd_kernel<X, Y, 64, 1, WHOLE>, 64);
  if (width <= 1024) return f(norm_bwd_kernel<X, Y, 128, 1, WHOLE>, 128);
  if (width <= 2048) return f(norm_bwd_kernel<X, Y, 256, 1, WHOLE>, 256);
  if (width <= 4096) return f(norm_bwd_kernel<X, Y, 512, 1, WHOLE>, 512);
  return f(norm_bwd_kernel<X, Y, 512, 2, WHOLE>, 512);
}
template <typename F>
static int with_types(const gs_residual_norm* p, F f) {
  if (p->x_dtype == GS_BFLOAT16) return f(__bf16{}, __bf16{});
  if (p->y_dtype == GS_BFLOAT16) return f(float{}, __bf16{});
  return f(float{}, float{});
}

}  // namespace gs

using namespace gs;

extern "C" int gs_residual_norm_fwd(const gs_residual_norm* p, void* stream) {
  clear_error();
  NormArgs a;
  if (const int rc = check_norm(p, false, &a)) return rc;
  if (a.rows == 0) return GS_OK;
  const auto run = [&](auto kernel, int lanes) -> int {
    const int groups = std::max(1, 256 / lanes);
    for (a.first = 0; a.first < a.rows; a.first += kNormLaunch * groups) {
      const int64_t blocks = std::min(kNormLaunch, (a.rows - a.first + groups - 1) / groups);
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(std::max(256, lanes)), 0, as_stream(stream), a);
      if (const int rc = check_launch("residual norm")) return rc;
    }
    return GS_OK;
  };
  return with_types(p, [&](auto x, auto y) {
    using X = decltype(x);
    using Y = decltype(y);
    return a.width % 8 == 0 ? with_fwd<X, Y, true>(a.width, run) : with_fwd<X, Y, false>(a.width, run);
  });
}

extern "C" size_t gs_residual_norm_bwd_workspace_size(const gs_residual_norm* p) {
  clear_error();
  if (!p || p->rows <= 0 || p->width <= 0) return 0;
  return static_cast<size_t>(norm_parts(p->rows)) * 5 * static_cast<size_t>(p->width) * sizeof(float);
}

extern "C" int gs_residual_norm_bwd(const gs_residual_norm* p, const void* d_h, const void* d_n, void* d_x, void* d_y,
                                    void* d_weight, void* d_bias, void* d_post_weight, void* d_post_bias, void* d_gate,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  NormArgs a;
  if (const int rc = check_norm(p, true, &a)) return rc;
  GS_REQUIRE(a.rows == 0 || a.stats, GS_ERR_ARG, "residual norm: the backward pass needs the statistics");
  GS_REQUIRE(a.y || (!d_y && !d_gate && !d_post_weight && !d_post_bias && !d_h), GS_ERR_ARG,
             "residual norm: gradients of a branch that is not there");
  GS_REQUIRE((a.gate || !d_gate) && (a.post || (!d_post_weight && !d_post_bias)), GS_ERR_ARG,
             "residual norm: gradients of a gate or post norm that is not there");
  GS_REQUIRE(workspace_bytes >= gs_residual_norm_bwd_workspace_size(p) && (workspace || a.rows == 0), GS_ERR_WORKSPACE,
             "residual norm: workspace too small");
  const size_t xs = row_type_bytes(p->x_dtype), ys = row_type_bytes(p->y_dtype), ws = row_type_bytes(p->weight_dtype);
  GS_REQUIRE(aligned(d_h, xs) && aligned(d_x, xs) && aligned(d_n, ys) && aligned(d_y, ys) && aligned(d_weight, ws) &&
                 aligned(d_bias, ws) && aligned(d_post_weight, ws) && aligned(d_post_bias, ws) &&
                 aligned(d_gate, row_type_bytes(p->gate_dtype)) && aligned(workspace, 16),
             GS_ERR_ALIGN, "residual norm: misaligned gradient or workspace");
  a.d_h = d_h;
  a.d_n = d_n;
  a.d_x = d_x;
  a.d_y = d_y;
  const bool gate_column = p->gate_rows == 0;
  a.d_gate_rows = gate_column ? nullptr : d_gate;
  void* const outs[5] = {d_weight, d_bias, d_post_weight, d_post_bias, gate_column ? d_gate : nullptr};
  ColumnSums s = {};
  for (int k = 0; k < 5; ++k) {
    a.slot[k] = outs[k] ? static_cast<int8_t>(a.sums) : int8_t(-1);
    if (!outs[k]) continue;
    s.out[a.sums] = outs[k];
    s.bf16[a.sums++] = k == kSumGate ? a.gate_bf16 : a.weights_bf16;
  }
  a.parts = static_cast<float*>(workspace);
  const hipStream_t st = as_stream(stream);
  int64_t blocks = 0;
  if (a.rows > 0) {
    const auto run = [&](auto kernel, int lanes) {
      const int groups = std::max(1, 256 / lanes);
      blocks = std::min<int64_t>(norm_parts(a.rows), (a.rows + groups - 1) / groups);
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(std::max(256, lanes)), 0, st, a);
      return check_launch("residual norm backward");
    };
    const int rc = with_types(p, [&](auto x, auto y) {
      using X = decltype(x);
      using Y = decltype(y);
      return a.width % 8 == 0 ? with_bwd<X, Y, true>(a.width, run) : with_bwd<X, Y, false>(a.width, run);
    });
    if (rc) return rc;
  }
  if (a.sums == 0) return GS_OK;
  s.parts = a.parts;
  s.n = static_cast<int>(blocks);  // (no rows: the sums are zero)
  s.sums = a.sums;
  s.width = a.width;
  return column_sums(s, "residual norm backward (sums)", st);
}

extern "C" int gs_dropout(const void* x, void* out, int64_t rows, int64_t stride, int width, int dtype, double p,
                          const int64_t* seed_at, uint64_t seed, uint64_t draw, void* stream) {
  clear_error();
  GS_REQUIRE(row_type(dtype), GS_ERR_ARG, "dropout: dtype must be GS_FLOAT32 or GS_BFLOAT16");
  GS_REQUIRE(rows >= 0 && rows < (int64_t(1) << 32) && width >= 0, GS_ERR_ARG, "dropout: invalid size");
  GS_REQUIRE(p >= 0.0 && p < 1.0, GS_ERR_ARG, "dropout: p must be at least 0 and below 1");
  GS_REQUIRE(rows == 0 || width == 0 || (x && out), GS_ERR_ARG, "dropout: null pointer");
  const size_t es = row_type_bytes(dtype);
  GS_REQUIRE(aligned(x, es) && aligned(out, es) && aligned(seed_at, 8), GS_ERR_ALIGN, "dropout: misaligned tensor");
  const int64_t groups = (static_cast<int64_t>(width) + 7) / 8, all = rows * groups;
  const int64_t blocks = (all + kDropThreads - 1) / kDropThreads;
  GS_REQUIRE(blocks * kDropThreads < (int64_t(1) << 32), GS_ERR_ARG, "dropout: too many elements");
  if (all == 0) return GS_OK;
  const DropRule d = drop_rule(p, seed_at, seed, draw);
  const dim3 grid(static_cast<unsigned>(blocks)), block(kDropThreads);
  if (dtype == GS_BFLOAT16) {
    hipLaunchKernelGGL(dropout_kernel<__bf16>, grid, block, 0, as_stream(stream), static_cast<const __bf16*>(x),
                       static_cast<__bf16*>(out), rows, stride, width, static_cast<int>(groups), d);
  } else {
    hipLaunchKernelGGL(dropout_kernel<float>, grid, block, 0, as_stream(stream), static_cast<const float*>(x),
                       static_cast<float*>(out), rows, stride, width, static_cast<int>(groups), d);
  }
  return check_launch("dropout");
}
