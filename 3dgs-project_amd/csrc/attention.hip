// Softmax attention over packed documents, forward and backward (see gs_attention.h for the layout
// of the products). A query row is a (token, head of the group) pair: the heads that share a key
// head are rows of one tile, so a key tile is read once for all of them and the gradients of shared
// heads are summed inside one workgroup, in a fixed order, without atomics.
#include <algorithm>
#include <type_traits>

#include "gs_attention.h"

namespace gs {

constexpr int kAttnWaves = 4;
constexpr int kAttnThreads = kAttnWaves * kWave;
constexpr int kAttnRows = kAttnWaves * 32;  // query rows (or keys, in the key gradients) of a workgroup
constexpr int kAttnKeys = 64;               // keys (or query rows) of a tile in LDS

// Kernels are instances for heads of up to DU = 32, 64, 96 or 128 elements: what they multiply and hold in
// registers. A row of a tile in LDS is a power of two, so that its chunks can be permuted.
// With instances for 64 and 128 alone, forward and backward: 8192 bfloat16 tokens, 16 heads of 96 513 and 2007
// us, so 457 and 1765; of 32 323 and 933 us, so 265 and 740; 2500 float32 tokens, 16 heads of 96, causal, 368
// and 1731 us, so 284 and 942. 64 and 128 are the same either way.
constexpr int row_of(int du) { return du > 64 ? 128 : 64; }

// Scores as base-2 exponents, x = gain z + bias: z is what tiles of scores are kept as (monotone in the score,
// -infinity where masked), so that maxima are taken of z and a probability is p = 2^(gain z + (bias - m)),
// one fma and one exponential.
struct Rule {
  float gain, bias;
  float in_scale;  // capped: scale / cap
  float cap2;      // capped: cap log2 e
  float twice;     // capped: 2 log2 e scale / cap
};

// Capped scores, s' = cap tanh x, x = scale s / cap. In bfloat16 tanh x = 1 - 2 r with r = 1 / (1 + e^2x)
// from the hardware exponential and reciprocal (absolute error 2e-7, both ends saturate), and z = -r; the
// slope is 1 - tanh^2 = 4 r (1 - r). float32, and bfloat16 under far caps, take the library's tanh, whose relative
// error near zero is small too, as z.
__device__ __forceinline__ float cap_r(const Rule& u, float s) {
  return __builtin_amdgcn_rcpf(1.0f + exp2_hw(s * u.twice));
}
template <typename T, int MODE>
__device__ __forceinline__ Rule rule_of(const AttnArgs& a) {
  const float scale = fabsf(a.scale);
  // (a scale of 0 becomes the smallest that takes a masked -infinity along)
  if constexpr (MODE == kPlain) return {fmaxf(scale * kLog2e, FLT_MIN), 0.0f, 0.0f, 0.0f, 0.0f};
  const float cap2 = a.softcap * kLog2e;
  const bool r = kByExp<T, MODE>;
  return {r ? 2.0f * cap2 : cap2, r ? cap2 : 0.0f, scale / a.softcap, cap2, 2.0f * kLog2e * scale / a.softcap};
}
template <typename T, int MODE>
__device__ __forceinline__ float z_of(const Rule& u, float s) {
  if constexpr (MODE == kPlain) return s;
  if constexpr (kByExp<T, MODE>) return -cap_r(u, s);
  return tanhf(s * u.in_scale);
}
__device__ __forceinline__ float prob(const Rule& u, float z, float m) {
  return exp2_hw(fmaf(z, u.gain, u.bias - m));
}

// Softmax state of a lane's query: running maximum of the exponents (kept within 2^8 of the true one:
// the accumulators are rescaled only when some lane's maximum grows by more), sum.
struct Softmax {
  float m = -INFINITY, l = 0.0f;
};

// Turns N tiles of 32 scores into probabilities; `o` is rescaled where the reference moves. Key i of the
// lane's registers is seen if it is below `vis`.
template <typename T, int MODE, int N, int M>
__device__ __forceinline__ void softmax_step(const Rule& u, f32x16 (&s)[N], f32x16 (&o)[M], Softmax& st, bool mask,
                                             int vis, int h) {
  float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int t = 0; t < N; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) s[t][r] = z_of<T, MODE>(u, s[t][r]);
  if (mask) {
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (32 * t + 8 * (r / 4) + 4 * h + r % 4 >= vis) s[t][r] = -INFINITY;
  }
#pragma unroll
  for (int t = 0; t < N; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) top[r % 4] = fmaxf(top[r % 4], s[t][r]);
  const float x = fmaf(half_max(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]))), u.gain, u.bias);
  if (__any(x > st.m + 8.0f)) {
    const float m = fmaxf(st.m, x);
    const float f = exp2_hw(st.m - (m == -INFINITY ? 0.0f : m));
    st.m = m;
    st.l *= f;
#pragma unroll
    for (int i = 0; i < M; ++i) o[i] *= f;
  }
  const float ref = st.m == -INFINITY ? 0.0f : st.m;
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int t = 0; t < N; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[t][r] = prob(u, s[t][r], ref);
      sum[r % 4] += s[t][r];
    }
  st.l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

// Four elements of a row of the output and, for a backward pass to come, what rounding took off them.
template <typename T>
__device__ __forceinline__ void store_out(const AttnArgs& a, int64_t at, f32x4 x) {
  store4(static_cast<T*>(a.out) + at, x[0], x[1], x[2], x[3]);
  if constexpr (sizeof(T) == 2) {
    if (a.out_low)
      store4(static_cast<T*>(a.out_low) + at, rounding_of(x[0]), rounding_of(x[1]), rounding_of(x[2]), rounding_of(x[3]));
  }
}

// The query's sign takes the scale's, so that scores are scaled by |scale|.
template <typename T>
__device__ __forceinline__ Frag<T> load_query(const AttnArgs& a, const T* p, bool valid) {
  Frag<T> f = load_frag<T>(p, valid);
  if (a.scale < 0.0f) f = -f;
  return f;
}

// Keeps the instructions on either side apart: groups of LDS reads are issued together, ahead of the
// products that use them, where the compiler would read, wait and multiply one by one.
template <typename T>
__device__ __forceinline__ void keep_order() {
  if constexpr (sizeof(T) == 2) __builtin_amdgcn_sched_barrier(0);
}

// A masked key's probability is 0, but 0 times an infinity or a NaN among its values is not. Such values
// reach the sums of queries that do not see them only under the causal mask, where some queries of a tile
// see a key and others do not; they are then visible in the sums, which are formed again here over the
// keys that each query sees, one by one. Finite values never come here.
template <int M>
__device__ __forceinline__ bool any_not_finite(const f32x16 (&o)[M]) {
  float t = 0.0f;
#pragma unroll
  for (int i = 0; i < M; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) t = fmaf(o[i][r], 0.0f, t);
  return __any(!(t == 0.0f));
}
// Keys begin .. begin + 31, then `step` further on, below `vis`.
template <typename T, int DU, int MODE>
__device__ __forceinline__ void sums_of_seen(const AttnArgs& a, const Rule& u, const Frag<T> (&q)[DU / 16], const T* kp,
                                             const T* vp, float m, int begin, int step, int vis, int h,
                                             f32x16 (&o)[DU / 32]) {
  const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
  for (int i = 0; i < DU / 32; ++i) o[i] = f32x16{};
  for (int k0 = begin; k0 < vis; k0 += step)
    for (int key = k0; key < min(k0 + 32, vis); ++key) {
      float s = 0.0f;
#pragma unroll
      for (int c = 0; c < DU / 16; ++c) {
        const int d = 16 * c + 8 * h;
        const Frag<T> k = load_frag<T>(kp + key * a.k_token + d, d < a.dim);
#pragma unroll
        for (int j = 0; j < 8; ++j) s = fmaf(static_cast<float>(q[c][j]), static_cast<float>(k[j]), s);
      }
      const float p = static_cast<float>(static_cast<T>(prob(u, z_of<T, MODE>(u, half_sum(s)), ref)));
#pragma unroll
      for (int dt = 0; dt < DU / 32; ++dt)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
          const int d = 32 * dt + 2 * r + 4 * h;
          if (d >= a.dim) continue;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            o[dt][r + j] = fmaf(p, static_cast<float>(vp[key * a.v_token + d + j]), o[dt][r + j]);
        }
    }
}

// Three workgroups a CU for up to 64 elements without the causal mask: a packed batch's last round is then
// shorter (8203 tokens in 4 documents, 16 heads of 64: 115 -> 104 us, capped 151 -> 144; 8192 in one 344 -> 336),
// for a register spilled at 64. The causal instance, of 178 registers, gains plain (8192 tokens 182 -> 174 us) but
// loses capped (245 -> 251) and over caches (100 queries on eight of 3000 30 -> 32, capped 37 -> 42). Of the
// instances with two workgroups those for 128 elements under the causal mask spill one to three of 256.
template <typename T, int DU, int MODE, bool CAUSAL>
__global__ __launch_bounds__(kAttnThreads, sizeof(T) == 2 ? (DU <= 64 && !CAUSAL ? 3 : 2) : 1) void attn_fwd_kernel(AttnArgs a) {
  using L = Tile<T, row_of(DU)>;
  constexpr int C = DU / 16;
  constexpr int kTileBytes = kAttnKeys * L::kRowBytes;
  __shared__ __attribute__((aligned(16))) char lds[4 * kTileBytes];
  const int hk = static_cast<int>(blockIdx.x % a.kv_heads);
  const int64_t tile = a.n_tiles - 1 - static_cast<int64_t>(blockIdx.x / a.kv_heads);
  const Found found = find_doc<false>(a, a.group, kAttnRows, tile);
  const Doc& doc = found.doc;
  const int rows = static_cast<int>(doc.q_len) * a.group;
  const int64_t base = (tile - found.first) * kAttnRows;
  if (base >= rows) return;
  const int row0 = static_cast<int>(base);
  const Piece piece = piece_of(a, visible(a, doc, (min(row0 + kAttnRows, rows) - 1) / a.group), blockIdx.y, found.share);
  if (static_cast<int>(blockIdx.y) >= piece.n) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int wrow = row0 + wave * 32;
  const int row = wrow + (lane & 31);
  const bool live = row < rows;
  const int rc = live ? row : rows - 1;
  const int tok = rc / a.group, head = hk * a.group + rc - tok * a.group;
  const T* qp = static_cast<const T*>(a.q) + (doc.q0 + tok) * a.q_token + head * a.q_head;
  Frag<T> q[C];
#pragma unroll
  for (int c = 0; c < C; ++c) q[c] = load_query<T>(a, qp + 16 * c + 8 * h, 16 * c + 8 * h < a.dim);
  const int vis = visible(a, doc, tok);
  const int wave_min = visible(a, doc, min(wrow, rows - 1) / a.group);
  const Rule rule = rule_of<T, MODE>(a);
  f32x16 o[DU / 32] = {};
  Softmax st;
  const T* kp = static_cast<const T*>(a.k) + doc.k0 * a.k_token + hk * a.k_head;
  const T* vp = static_cast<const T*>(a.v) + doc.k0 * a.v_token + hk * a.v_head;
  const TileCopy<T, row_of(DU), kAttnKeys, kAttnThreads> copy_k(a.k_token, a.dim), copy_v(a.v_token, a.dim);
  const auto fetch = [&](int k0, char* to) {
    const int valid = min(kAttnKeys, static_cast<int>(doc.k_len) - k0);
    copy_k(to, row_buffer(kp + k0 * a.k_token, a.k_token, valid, a.dim));
    copy_v(to + kTileBytes, row_buffer(vp + k0 * a.v_token, a.v_token, valid, a.dim));
  };
  if (piece.begin < piece.stop) fetch(piece.begin, lds);
  int buf = 0;
  for (int k0 = piece.begin; k0 < piece.stop; k0 += kAttnKeys, buf ^= 1) {
    const char* lk = lds + buf * 2 * kTileBytes;
    const char* lv = lk + kTileBytes;
    copies_done();
    __syncthreads();
    if (k0 + kAttnKeys < piece.stop) fetch(k0 + kAttnKeys, lds + (buf ^ 1) * 2 * kTileBytes);
    // a wavefront past the last row only copies: its SIMD is the other workgroup's (8192 causal tokens, 16
    // heads of 64: 209 -> 182 us, of 128 297 -> 286; in the gradients' kernels it gains nothing)
    if (uniform(wrow) >= rows) continue;
    f32x16 s[2] = {};
    {
      Frag<T> ka[C], kb[C];
#pragma unroll
      for (int c = 0; c < C; ++c) ka[c] = L::rows(lk, 0, c, lane);
#pragma unroll
      for (int c = 0; c < C; ++c) kb[c] = L::rows(lk, 32, c, lane);
      keep_order<T>();
#pragma unroll
      for (int c = 0; c < C; ++c) mma(s[0], ka[c], q[c]);
#pragma unroll
      for (int c = 0; c < C; ++c) mma(s[1], kb[c], q[c]);
    }
    Frag<T> v[2][DU / 32];
#pragma unroll
    for (int dt = 0; dt < DU / 32; ++dt) v[0][dt] = L::cols(lv, 32 * dt, 0, lane);
    keep_order<T>();
    softmax_step<T, MODE>(rule, s, o, st, k0 + kAttnKeys > wave_min, vis - k0, h);
    // the wavefront that has its probabilities goes first: its products then run while the SIMD's other
    // wavefront is at its exponentials, and not the two in step (8192 tokens, 16 heads of 128: 562 -> 547 us,
    // causal 311 -> 286, capped 689 -> 669; both together lose a little, 365 -> 370)
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int kc = 0; kc < 4; ++kc) {
      if (kc < 3) {
#pragma unroll
        for (int dt = 0; dt < DU / 32; ++dt) v[(kc + 1) & 1][dt] = L::cols(lv, 32 * dt, 16 * (kc + 1), lane);
        keep_order<T>();
      }
      const Frag<T> p = acc_frag<T>(s[kc / 2], kc % 2);
#pragma unroll
      for (int dt = 0; dt < DU / 32; ++dt) mma(o[dt], v[kc & 1][dt], p);
    }
    __builtin_amdgcn_s_setprio(0);
  }
  // only where queries of a tile see different keys (8192 causal tokens, 16 heads of 128, with and without this
  // code 286 and 287 us; of 64, capped, 245 and 246)
  if constexpr (CAUSAL) {
    if (any_not_finite(o))
      sums_of_seen<T, DU, MODE>(a, rule, q, kp, vp, st.m, piece.begin, 32, min(vis, piece.stop), h, o);
  }
  if (!live) return;
  const float m = st.m, l = half_sum(st.l);
  if (a.splits > 1) {
    const int64_t at = (doc.q0 + tok) * a.heads + head;
    const int64_t part = blockIdx.y * a.q_tokens * a.heads + at;
    float* pp = a.part + part * a.dim;
#pragma unroll
    for (int dt = 0; dt < DU / 32; ++dt)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int d = 32 * dt + 2 * r + 4 * h;
        if (d < a.dim) store4(pp + d, o[dt][r], o[dt][r + 1], o[dt][r + 2], o[dt][r + 3]);
      }
    if (h == 0) {
      a.part_stat[2 * part] = m;
      a.part_stat[2 * part + 1] = l;
      if (blockIdx.y == 0) a.part_n[at] = piece.n;
    }
    return;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int64_t at = (doc.q0 + tok) * a.heads + head;
#pragma unroll
  for (int dt = 0; dt < DU / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int d = 32 * dt + 2 * r + 4 * h;
      if (d >= a.dim) continue;
      store_out<T>(a, at * a.dim + d, f32x4{o[dt][r], o[dt][r + 1], o[dt][r + 2], o[dt][r + 3]} * inv);
    }
  if (h == 0) a.lse[at] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// Few query rows (single tokens) against long keys (24 documents of 16k keys, 32 heads on 8 of 128: 276
// us, 5.8 TB/s; one of 777, 8 heads of 64: 7.7 us, 10.0 with four wavefronts): HBM-bound, so a workgroup's wavefronts each walk
// over keys of their own, 32 at a time, for the same 32 rows, and join at the end. The next keys' and
// values' loads (16 KB a wavefront at 128 elements of bfloat16) are in flight while the present ones are
// multiplied; they pass through the wavefront's own LDS (rows to be read across and along), with no
// barrier in the loop.
// bfloat16: eight wavefronts, so that a short document is a few steps long. float32's tiles allow four.
template <typename T>
constexpr int kFewWaves = sizeof(T) == 2 ? 8 : 4;
template <typename T, int DU, int MODE, bool CAUSAL>
__global__ __launch_bounds__(kFewWaves<T> * kWave) void attn_few_kernel(AttnArgs a) {
  constexpr int kWaves = kFewWaves<T>;
  using L = Tile<T, row_of(DU)>;
  constexpr int C = DU / 16;
  constexpr int kLoads = 32 * L::kChunks / kWave;  // 16-byte loads a lane for 32 rows
  constexpr int kTileBytes = 32 * L::kRowBytes;
  static_assert(2 * kTileBytes >= 32 * DU * 4, "the join reuses the wavefront's tiles");
  __shared__ __attribute__((aligned(16))) char lds[kWaves * 2 * kTileBytes];
  __shared__ float l_m[kWaves][32], l_l[kWaves][32];
  const int hk = static_cast<int>(blockIdx.x % a.kv_heads);
  const int64_t tile = static_cast<int64_t>(blockIdx.x / a.kv_heads);
  const Found found = find_doc<false>(a, a.group, 32, tile);
  const Doc& doc = found.doc;
  const int rows = static_cast<int>(doc.q_len) * a.group;
  const int64_t base = (tile - found.first) * 32;
  if (base >= rows) return;
  const int row0 = static_cast<int>(base);
  const int n_rows = min(32, rows - row0);
  const Piece piece = piece_of(a, visible(a, doc, (row0 + n_rows - 1) / a.group), blockIdx.y, found.share);
  if (static_cast<int>(blockIdx.y) >= piece.n) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int row = row0 + (lane & 31);
  const bool live = row < rows;
  const int rc = live ? row : rows - 1;
  const int tok = rc / a.group, head = hk * a.group + rc - tok * a.group;
  const T* qp = static_cast<const T*>(a.q) + (doc.q0 + tok) * a.q_token + head * a.q_head;
  const int vis = min(visible(a, doc, tok), piece.stop);
  const int all_min = min(visible(a, doc, row0 / a.group), piece.stop);
  const Rule rule = rule_of<T, MODE>(a);
  f32x16 o[DU / 32] = {};
  Softmax st;
  const T* kp = static_cast<const T*>(a.k) + doc.k0 * a.k_token + hk * a.k_head;
  const T* vp = static_cast<const T*>(a.v) + doc.k0 * a.v_token + hk * a.v_head;
  char* lk = lds + wave * 2 * kTileBytes;
  char* lv = lk + kTileBytes;
  f32x4 pk[kLoads], pv[kLoads];
  uint32_t at_k[kLoads], at_v[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int e = i * kWave + lane, r = e / L::kChunks, c = (e % L::kChunks) * L::kElemsPerChunk;
    at_k[i] = c < a.dim ? static_cast<uint32_t>((r * a.k_token + c) * sizeof(T)) : kNowhere;
    at_v[i] = c < a.dim ? static_cast<uint32_t>((r * a.v_token + c) * sizeof(T)) : kNowhere;
  }
  const auto fetch = [&](int k0) {
    const auto bk = row_buffer(kp + k0 * a.k_token, a.k_token, min(32, piece.stop - k0), a.dim);
    const auto bv = row_buffer(vp + k0 * a.v_token, a.v_token, min(32, piece.stop - k0), a.dim);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) pk[i] = load16(bk, at_k[i]);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) pv[i] = load16(bv, at_v[i]);
  };
  int k0 = piece.begin + __builtin_amdgcn_readfirstlane(wave) * 32;
  if (k0 < piece.stop) fetch(k0);
  Frag<T> q[C];
#pragma unroll
  for (int c = 0; c < C; ++c) q[c] = load_query<T>(a, qp + 16 * c + 8 * h, 16 * c + 8 * h < a.dim);
  for (; k0 < piece.stop; k0 += kWaves * 32) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int e = i * kWave + lane;
      *reinterpret_cast<f32x4*>(lk + L::at(e / L::kChunks, e % L::kChunks)) = pk[i];
      *reinterpret_cast<f32x4*>(lv + L::at(e / L::kChunks, e % L::kChunks)) = pv[i];
    }
    wave_sync();
    if (k0 + kWaves * 32 < piece.stop) fetch(k0 + kWaves * 32);
    f32x16 s[1] = {};
#pragma unroll
    for (int c = 0; c < C; ++c) mma(s[0], L::rows(lk, 0, c, lane), q[c]);
    softmax_step<T, MODE>(rule, s, o, st, k0 + 32 > all_min, vis - k0, h);
#pragma unroll
    for (int kc = 0; kc < 2; ++kc) {
      const Frag<T> p = acc_frag<T>(s[0], kc);
      // Here the matrix unit has time to spare, so what rounding took off the probabilities is multiplied
      // too: the output is off by its own rounding alone.
      Frag<T> low = {};
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int j = 0; j < 8; ++j) low[j] = static_cast<T>(s[0][8 * kc + j] - static_cast<float>(p[j]));
      }
#pragma unroll
      for (int dt = 0; dt < DU / 32; ++dt) {
        const Frag<T> v = L::cols(lv, 32 * dt, 16 * kc, lane);
        mma(o[dt], v, p);
        if constexpr (sizeof(T) == 2) mma(o[dt], v, low);
      }
    }
    wave_sync();
  }
  if constexpr (CAUSAL) {
    if (any_not_finite(o))
      sums_of_seen<T, DU, MODE>(a, rule, q, kp, vp, st.m, piece.begin + wave * 32, kWaves * 32, vis, h, o);
  }
  // join: every wavefront leaves its rows, statistics and (in its own tiles) sums; then all threads
  // take the same rows' elements and add the wavefronts' in order
  const float m = st.m, l = half_sum(st.l);
  float* own = reinterpret_cast<float*>(lk);
  if (live) {
    if (h == 0) {
      l_m[wave][lane & 31] = m;
      l_l[wave][lane & 31] = l;
    }
#pragma unroll
    for (int dt = 0; dt < DU / 32; ++dt)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        store4(own + (lane & 31) * DU + 32 * dt + 2 * r + 4 * h, o[dt][r], o[dt][r + 1], o[dt][r + 2], o[dt][r + 3]);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < n_rows * (DU / 4); e += kWaves * kWave) {
    const int i = e / (DU / 4), d = e % (DU / 4) * 4;
    float top = l_m[0][i];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, l_m[w][i]);
    const float ref = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = exp2_hw(l_m[w][i] - ref);
      sum += f * l_l[w][i];
      x += f * *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + w * 2 * kTileBytes) + i * DU + d);
    }
    const int t = (row0 + i) / a.group;
    const int64_t at = (doc.q0 + t) * a.heads + hk * a.group + row0 + i - t * a.group;
    if (a.splits > 1) {
      const int64_t part = blockIdx.y * a.q_tokens * a.heads + at;
      if (d < a.dim) *reinterpret_cast<f32x4*>(a.part + part * a.dim + d) = x;
      if (d == 0) {
        a.part_stat[2 * part] = top;
        a.part_stat[2 * part + 1] = sum;
        if (blockIdx.y == 0) a.part_n[at] = piece.n;
      }
    } else {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      if (d < a.dim) store_out<T>(a, at * a.dim + d, x * inv);
      if (d == 0) a.lse[at] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
    }
  }
}

// Joins the pieces of a (token, head), in order: 32 lanes take four elements each, and a piece's
// statistics each. Rows outside every document have no keys, hence one piece.
template <typename T>
__global__ __launch_bounds__(kAttnThreads) void attn_join_kernel(AttnArgs a) {
  constexpr int kLanes = 32;
  const int64_t at = (static_cast<int64_t>(blockIdx.x) * kAttnThreads + threadIdx.x) / kLanes;
  const int64_t all = a.q_tokens * a.heads;
  if (at >= all) return;
  const int lane = threadIdx.x % kLanes, d = 4 * lane;
  const int n = max(0, min(a.part_n[at], a.splits));  // (offsets that decrease leave some unwritten)
  float top = -INFINITY, sum = 0.0f;
  f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int i0 = 0; i0 < n; i0 += kLanes) {
    const int64_t mine = (i0 + lane) * all + at;
    const bool in = i0 + lane < n;
    const float m = in ? a.part_stat[2 * mine] : -INFINITY;
    const float l = in ? a.part_stat[2 * mine + 1] : 0.0f;
    float up = fmaxf(top, m);
#pragma unroll
    for (int b = 1; b < kLanes; b *= 2) up = fmaxf(up, __shfl_xor(up, b, kLanes));
    const float ref = up == -INFINITY ? 0.0f : up;
    const float keep = exp2_hw(top - ref), w = exp2_hw(m - ref);
    float part = w * l;
#pragma unroll
    for (int b = 1; b < kLanes; b *= 2) part += __shfl_xor(part, b, kLanes);
    sum = sum * keep + part;
    x *= keep;
    top = up;
    const int here = min(kLanes, n - i0);
    for (int i = 0; i < here; i += 8) {  // eight pieces' loads at a time
      f32x4 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        v[k] = d < a.dim ? *reinterpret_cast<const f32x4*>(a.part + ((i0 + min(i + k, here - 1)) * all + at) * a.dim + d)
                         : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float f = __shfl(w, min(i + k, kLanes - 1), kLanes);
        if (i + k < here) x += f * v[k];
      }
    }
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  if (d < a.dim) store_out<T>(a, at * a.dim + d, x * inv);
  if (lane == 0) a.lse[at] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

// Lays out the instructions since the last keep_order as M times one matrix instruction and V vector
// ones, after N LDS reads: the vector work then runs in the products' shadow within one wavefront.
template <int N, int M, int V>
__device__ __forceinline__ void interleave() {
  if constexpr (N > 0) __builtin_amdgcn_sched_group_barrier(0x100, N, 0);  // LDS reads
#pragma unroll
  for (int i = 0; i < M; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);  // matrix
    __builtin_amdgcn_sched_group_barrier(0x2, V, 0);  // vector
  }
}

// The fragments of 32 rows of a tile, along (rows) and across (cols).
template <typename T, int DU>
struct Rows {
  Frag<T> f[DU / 16];
  __device__ __forceinline__ void read(const char* lds, int row0, int lane) {
#pragma unroll
    for (int c = 0; c < DU / 16; ++c) f[c] = Tile<T, row_of(DU)>::rows(lds, row0, c, lane);
  }
  __device__ __forceinline__ void times(const Frag<T> (&b)[DU / 16], f32x16& acc) const {
    acc = f32x16{};
#pragma unroll
    for (int c = 0; c < DU / 16; ++c) mma(acc, f[c], b[c]);
  }
};
template <typename T, int DU>
struct Cols {
  Frag<T> f[2][DU / 32];
  __device__ __forceinline__ void read(const char* lds, int row0, int lane) {
#pragma unroll
    for (int kc = 0; kc < 2; ++kc)
#pragma unroll
      for (int dt = 0; dt < DU / 32; ++dt) f[kc][dt] = Tile<T, row_of(DU)>::cols(lds, 32 * dt, row0 + 16 * kc, lane);
  }
  __device__ __forceinline__ void add_times(const Frag<T> (&p)[2], f32x16 (&acc)[DU / 32]) const {
#pragma unroll
    for (int kc = 0; kc < 2; ++kc)
#pragma unroll
      for (int dt = 0; dt < DU / 32; ++dt) mma(acc[dt], f[kc][dt], p[kc]);
  }
};
template <typename T>
__device__ __forceinline__ void acc_frags(const f32x16& c, Frag<T> (&f)[2]) {
  f[0] = acc_frag<T>(c, 0);
  f[1] = acc_frag<T>(c, 1);
}

// The same products in float32, whose fragments are twice as large: read as they are used.
template <int DU>
__device__ __forceinline__ void rows_times(const char* lds, int row0, int lane, const f32x8 (&b)[DU / 16], f32x16& acc) {
  acc = f32x16{};
#pragma unroll
  for (int c = 0; c < DU / 16; ++c) {
    mma(acc, Tile<float, row_of(DU)>::rows(lds, row0, c, lane), b[c]);
    if (c % 2) __builtin_amdgcn_sched_barrier(0);
  }
}
template <int DU>
__device__ __forceinline__ void add_cols_times(const char* lds, int row0, int lane, const f32x16& p,
                                               f32x16 (&acc)[DU / 32]) {
#pragma unroll
  for (int kc = 0; kc < 2; ++kc) {
    const f32x8 f = acc_frag<float>(p, kc);
#pragma unroll
    for (int dt = 0; dt < DU / 32; ++dt) {
      mma(acc[dt], Tile<float, row_of(DU)>::cols(lds, 32 * dt, row0 + 16 * kc, lane), f);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// Probability of a score, p = e^(s - lse), and (capped) the score's slope 1 - tanh^2. The raw score's
// gradient is p slope (dp - delta).
// `base` is the row's, from base_of its log-sum-exp.
template <typename T, int MODE>
__device__ __forceinline__ float base_of(const Rule& u, float lse) {
  const float lse2 = lse == -INFINITY ? 0.0f : lse * kLog2e;
  return kByExp<T, MODE> ? u.cap2 - lse2 : -lse2;
}
template <typename T, int MODE>
__device__ __forceinline__ float prob_of(const Rule& u, float s, float base, float* slope) {
  if constexpr (MODE == kPlain) return exp2_hw(fmaf(s, u.gain, base));
  if constexpr (kByExp<T, MODE>) {
    const float r = cap_r(u, s), r4 = 4.0f * r;
    *slope = fmaf(-r4, r, r4);
    return exp2_hw(fmaf(-2.0f * u.cap2, r, base));
  }
  const float t = tanhf(s * u.in_scale);
  *slope = fmaf(-t, t, 1.0f);
  return exp2_hw(fmaf(u.cap2, t, base));
}

// Query gradients, and delta_i = dO_i . O_i for the key gradients. Like the forward, a lane owns a
// query; its score gradients are the B operand of dQ = dS K.
template <typename T, int DU, int MODE>
__global__ __launch_bounds__(kAttnThreads, sizeof(T) == 2 ? 2 : 1) void attn_bwd_q_kernel(AttnArgs a) {
  using L = Tile<T, row_of(DU)>;
  constexpr int C = DU / 16;
  constexpr int kTileBytes = kAttnKeys * L::kRowBytes;
  __shared__ __attribute__((aligned(16))) char lds[4 * kTileBytes];
  const int hk = static_cast<int>(blockIdx.x % a.kv_heads);
  const int64_t tile = a.n_tiles - 1 - static_cast<int64_t>(blockIdx.x / a.kv_heads);
  const Found found = find_doc<false>(a, a.group, kAttnRows, tile);
  const Doc& doc = found.doc;
  const int rows = static_cast<int>(doc.q_len) * a.group;
  const int64_t base = (tile - found.first) * kAttnRows;
  if (base >= rows) return;
  const int row0 = static_cast<int>(base);
  // with key_parts: this part's keys. A part without any writes zeros.
  int end = visible(a, doc, (min(row0 + kAttnRows, rows) - 1) / a.group), begin = 0;
  if (a.key_parts > 1) {
    const int per = (end + a.key_parts * kAttnKeys - 1) / (a.key_parts * kAttnKeys) * kAttnKeys;
    begin = min(static_cast<int>(blockIdx.y) * per, end);
    end = min(begin + per, end);
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int wrow = row0 + wave * 32;
  const int row = wrow + (lane & 31);
  const bool live = row < rows;
  const int rc = live ? row : rows - 1;
  const int tok = rc / a.group, head = hk * a.group + rc - tok * a.group;
  const T* kp = static_cast<const T*>(a.k) + doc.k0 * a.k_token + hk * a.k_head;
  const T* vp = static_cast<const T*>(a.v) + doc.k0 * a.v_token + hk * a.v_head;
  const TileCopy<T, row_of(DU), kAttnKeys, kAttnThreads> copy_k(a.k_token, a.dim), copy_v(a.v_token, a.dim);
  const auto fetch = [&](int k0, char* to) {
    const int valid = min(kAttnKeys, static_cast<int>(doc.k_len) - k0);
    copy_k(to, row_buffer(kp + k0 * a.k_token, a.k_token, valid, a.dim));
    copy_v(to + kTileBytes, row_buffer(vp + k0 * a.v_token, a.v_token, valid, a.dim));
  };
  if (begin < end) fetch(begin, lds);
  const T* qp = static_cast<const T*>(a.q) + (doc.q0 + tok) * a.q_token + head * a.q_head;
  const int64_t at = ((doc.q0 + tok) * a.heads + head) * a.dim;
  const T* gp = static_cast<const T*>(a.d_out) + at;
  const T* op = static_cast<const T*>(a.out) + at;
  const T* lp = static_cast<const T*>(a.out_low) + at;
  Frag<T> q[C], g[C];
  float delta = 0.0f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const bool in = 16 * c + 8 * h < a.dim;
    q[c] = load_query<T>(a, qp + 16 * c + 8 * h, in);
    g[c] = load_frag<T>(gp + 16 * c + 8 * h, in);
    const Frag<T> o = load_frag<T>(op + 16 * c + 8 * h, in);
    const Frag<T> low = load_frag<T>(lp + 16 * c + 8 * h, in && a.out_low);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      delta = fmaf(static_cast<float>(g[c][j]), static_cast<float>(o[j]) + static_cast<float>(low[j]), delta);
  }
  delta = half_sum(delta);
  const int64_t stat = (doc.q0 + tok) * a.heads + head;
  if (live && h == 0 && blockIdx.y == 0) a.delta[stat] = delta;
  const Rule rule = rule_of<T, MODE>(a);
  const float row_base = base_of<T, MODE>(rule, a.lse[stat]);
  const int vis = live ? visible(a, doc, tok) : 0;
  const int wave_min = wrow + 31 < rows ? visible(a, doc, wrow / a.group) : 0;
  f32x16 dq[DU / 32] = {};
  int buf = 0;
  for (int k0 = begin; k0 < end; k0 += kAttnKeys, buf ^= 1) {
    const char* lk = lds + buf * 2 * kTileBytes;
    const char* lv = lk + kTileBytes;
    copies_done();
    __syncthreads();
    if (k0 + kAttnKeys < end) fetch(k0 + kAttnKeys, lds + (buf ^ 1) * 2 * kTileBytes);
    const auto body = [&](auto masked) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        f32x16 s, dp;
        const auto probs = [&] {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            float slope = 1.0f;
            s[r] = prob_of<T, MODE>(rule, s[r], row_base, &slope);
            if constexpr (MODE != kPlain) s[r] *= slope;
            if (masked.value && k0 + 32 * t + 8 * (r / 4) + 4 * h + r % 4 >= vis) s[r] = 0.0f;
          }
        };
        const auto grads = [&] {
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] *= dp[r] - delta;
        };
        if constexpr (sizeof(T) == 2) {
          Rows<T, DU> x, y;
          Cols<T, DU> z;
          Frag<T> f[2];
          x.read(lk, 32 * t, lane);
          y.read(lv, 32 * t, lane);
          x.times(q, s);
          keep_order<T>();
          y.times(g, dp);
          probs();
          interleave<0, C, MODE == kPlain ? 6 : 12>();
          keep_order<T>();
          z.read(lk, 32 * t, lane);
          grads();
          acc_frags<T>(s, f);
          z.add_times(f, dq);
          keep_order<T>();
        } else {
          rows_times<DU>(lk, 32 * t, lane, q, s);
          rows_times<DU>(lv, 32 * t, lane, g, dp);
          probs();
          grads();
          add_cols_times<DU>(lk, 32 * t, lane, s, dq);
        }
      }
    };
    if (k0 + kAttnKeys > wave_min) body(std::true_type{});
    else body(std::false_type{});
  }
  if (!live) return;
  T* to = static_cast<T*>(a.d_q) + at;
#pragma unroll
  for (int dt = 0; dt < DU / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int d = 32 * dt + 2 * r + 4 * h;
      if (d >= a.dim) continue;
      const f32x4 x = f32x4{dq[dt][r], dq[dt][r + 1], dq[dt][r + 2], dq[dt][r + 3]} * a.scale;
      if (a.key_parts > 1)
        *reinterpret_cast<f32x4*>(a.part_q + blockIdx.y * a.q_tokens * a.heads * a.dim + at + d) = x;
      else
        store4(to + d, x[0], x[1], x[2], x[3]);
    }
}

// Key and value gradients: a lane owns one key, the workgroup walks over the query rows that see it,
// 64 at a time. Rows past the document's end need no mask: their q, dO and delta are zero (and p finite), and so
// is what they add. The lanes of keys past the valid length gather nothing that is kept.
//
// At 96 and 128 elements of bfloat16 both gradients' accumulators (128 registers beside K and V's 64) leave no
// room for a second wavefront on the SIMD, and the compiler then moves operands between the register
// files. There, workgroups with blockIdx.y = 0 gather dK (three products) and the others dV (S again, two
// products): five products for four, but two wavefronts a SIMD that fill each other's gaps. Measured at
// 8192 tokens, 16 heads of 128, the whole backward: 2199 us together with one wavefront a SIMD, 2008 apart; causal
// 1263 and 1123. In float32 it is 128 elements at which both do not fit one wavefront's 512 registers (115
// spilled). The whole backward together and apart, 16 heads: 700 tokens 337 and 283 us, causal 257 and 225; 2500
// tokens 2680 and 2711, causal 1789 and 1430, capped 3348 and 3009, both 2074 and 1576; 6000 tokens 11319 and 11662,
// causal 7305 and 6179, capped 16734 and 12871. Apart loses 1 to 3% in long plain documents without the mask and
// gains elsewhere, so it is taken throughout. Smaller heads keep both in one.
constexpr bool split_kv(bool bf16, int dim) { return dim > (bf16 ? 64 : 96); }
template <typename T, int DU>
constexpr bool kSplitKv = split_kv(sizeof(T) == 2, DU);

constexpr int kKvRows = 64;  // query rows of a tile
template <typename T, int DU>
struct KvShared {
  char tiles[4 * kKvRows * Tile<T, row_of(DU)>::kRowBytes];
  float base[2][kKvRows], delta[2][kKvRows];
  int vis[2][kKvRows];
};

template <typename T, int DU, int MODE, bool DK, bool DV>
__device__ __forceinline__ void attn_bwd_kv(const AttnArgs& a, KvShared<T, DU>& sh) {
  using L = Tile<T, row_of(DU)>;
  constexpr int C = DU / 16;
  constexpr int R = kKvRows;
  constexpr int kTileBytes = R * L::kRowBytes;
  char* lds = sh.tiles;
  const auto &l_base = sh.base, &l_delta = sh.delta;
  const auto& l_vis = sh.vis;
  const int hk = static_cast<int>(blockIdx.x % a.kv_heads);
  const int64_t tile = blockIdx.x / a.kv_heads;
  const Found found = find_doc<true>(a, 1, kAttnRows, tile);
  const Doc& doc = found.doc;
  const int64_t base = (tile - found.first) * kAttnRows;
  if (base >= doc.k_cap) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int key0 = static_cast<int>(base), wkey = key0 + wave * 32;
  const int key = wkey + (lane & 31);
  const bool live = key < doc.k_len;
  const int rows = static_cast<int>(doc.q_len) * a.group;
  // the first token that sees key0 (none of this tile's keys is seen by one before it)
  RowStart start = {0, 0};
  if (a.causal && key0 >= doc.prefix) {
    const int64_t t = key0 - doc.k_len + doc.q_len;
    if (t > 0) start.token = static_cast<int>(t < doc.q_len ? t : doc.q_len);
  }
  int row_begin = key0 >= doc.k_len ? rows : start.token * a.group;
  int row_end = rows;
  if (a.row_parts > 1) {
    const int part = blockIdx.z, per = ((rows - row_begin) / a.row_parts + R) / R * R;
    const int from = min(part * per, rows - row_begin);
    start.token += from / a.group;
    start.g = from % a.group;
    row_begin += from;
    row_end = min(row_begin + per, rows);
  }
  const RowTileCopy<T, row_of(DU), R, kAttnThreads> copy_q = {a.q_token, a.q_head};
  const RowTileCopy<T, row_of(DU), R, kAttnThreads> copy_g = {static_cast<int64_t>(a.heads) * a.dim, a.dim};
  const Rule rule = rule_of<T, MODE>(a);
  float n_lse = 0.0f, n_delta = 0.0f;
  int n_vis = 0;
  const auto fetch = [&](int r0, char* to) {
    const int64_t token = doc.q0 + start.token;
    copy_q(a, to, static_cast<const T*>(a.q) + token * a.q_token + hk * a.group * a.q_head, start.g, row_end - r0);
    copy_g(a, to + kTileBytes, static_cast<const T*>(a.d_out) + (token * a.heads + hk * a.group) * a.dim, start.g,
           row_end - r0);
    if (threadIdx.x < R) {
      n_lse = n_delta = 0.0f;
      n_vis = 0;
      if (r0 + static_cast<int>(threadIdx.x) < row_end) {
        const int n = start.g + threadIdx.x, t = static_cast<int>((n * a.group_magic) >> 20);
        const int64_t stat = (token + t) * a.heads + hk * a.group + n - t * a.group;
        n_lse = a.lse[stat];
        n_delta = a.delta[stat];
        n_vis = visible(a, doc, start.token + t);
      }
    }
    start.advance(a, R);
  };
  const auto keep = [&](int b) {
    if (threadIdx.x < R) {
      sh.base[b][threadIdx.x] = base_of<T, MODE>(rule, n_lse);
      sh.delta[b][threadIdx.x] = n_delta;
      sh.vis[b][threadIdx.x] = n_vis;
    }
  };
  if (row_begin < row_end) fetch(row_begin, lds);
  Frag<T> k[C], v[C];
  const T* kp = static_cast<const T*>(a.k) + (doc.k0 + key) * a.k_token + hk * a.k_head;
  const T* vp = static_cast<const T*>(a.v) + (doc.k0 + key) * a.v_token + hk * a.v_head;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const bool in = live && 16 * c + 8 * h < a.dim;
    k[c] = load_frag<T>(kp + 16 * c + 8 * h, in);
    if (a.scale < 0.0f) k[c] = -k[c];
    if constexpr (DK) v[c] = load_frag<T>(vp + 16 * c + 8 * h, in);
  }
  f32x16 dk[DU / 32] = {}, dv[DU / 32] = {};
  int buf = 0;
  for (int r0 = row_begin; r0 < row_end; r0 += R, buf ^= 1) {
    const char* lq = lds + buf * 2 * kTileBytes;
    const char* lg = lq + kTileBytes;
    keep(buf);
    copies_done();
    __syncthreads();
    // every row of the tile sees all of this wavefront's keys?
    const bool mask = a.causal && __builtin_amdgcn_readfirstlane(l_vis[buf][0]) < wkey + 32;
    if (r0 + R < row_end) fetch(r0 + R, lds + (buf ^ 1) * 2 * kTileBytes);
    const auto body = [&](auto masked) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        f32x16 s, dp, sl;
        const auto probs = [&] {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int at = 32 * t + 8 * i + 4 * h;
            const f32x4 base = *reinterpret_cast<const f32x4*>(&l_base[buf][at]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int r = 4 * i + j;
              float slope = 1.0f;
              s[r] = prob_of<T, MODE>(rule, s[r], base[j], &slope);
              if constexpr (MODE != kPlain && DV) sl[r] = slope;
              if constexpr (MODE != kPlain && !DV) s[r] *= slope;
              if (masked.value && key >= l_vis[buf][at + j]) s[r] = 0.0f;
            }
          }
        };
        const auto grads = [&] {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f32x4 delta = *reinterpret_cast<const f32x4*>(&l_delta[buf][32 * t + 8 * i + 4 * h]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int r = 4 * i + j;
              dp[r] = s[r] * (dp[r] - delta[j]);
              if constexpr (MODE != kPlain && DV) dp[r] *= sl[r];
            }
          }
        };
        if constexpr (sizeof(T) == 2) {
          // products of C matrix instructions; the probabilities are formed in the second's shadow, the
          // score gradients in the third's, and an operand is read during the product before its own
          Rows<T, DU> x, y;
          Cols<T, DU> zg, zq;
          Frag<T> f[2], e[2];
          x.read(lq, 32 * t, lane);
          if constexpr (DK && DV) y.read(lg, 32 * t, lane);
          x.times(k, s);
          if constexpr (DV) zg.read(lg, 32 * t, lane);
          keep_order<T>();
          if constexpr (DK && !DV) y.read(lg, 32 * t, lane);
          if constexpr (DK) y.times(v, dp);
          probs();
          if constexpr (DV) acc_frags<T>(s, f);
          if constexpr (DK && DV) zq.read(lq, 32 * t, lane);
          if constexpr (DK) interleave<0, C, MODE == kPlain ? 7 : 13>();
          keep_order<T>();
          if constexpr (DK && !DV) zq.read(lq, 32 * t, lane);
          if constexpr (DV) zg.add_times(f, dv);
          if constexpr (DK) {
            grads();
            acc_frags<T>(dp, e);
            if constexpr (DV) {
              interleave<0, C, MODE == kPlain ? 5 : 7>();
              keep_order<T>();
            }
            zq.add_times(e, dk);
          }
          keep_order<T>();
        } else {
          rows_times<DU>(lq, 32 * t, lane, k, s);
          if constexpr (DK) rows_times<DU>(lg, 32 * t, lane, v, dp);
          probs();
          if constexpr (DK) grads();
          if constexpr (DV) add_cols_times<DU>(lg, 32 * t, lane, s, dv);
          if constexpr (DK) add_cols_times<DU>(lq, 32 * t, lane, dp, dk);
        }
      }
    };
    if (mask) body(std::true_type{});
    else body(std::false_type{});
  }
  if (key >= doc.k_cap) return;
  const int64_t at = ((doc.k0 + key) * a.kv_heads + hk) * a.dim;
  T* dkp = static_cast<T*>(a.d_k) + at;
  T* dvp = static_cast<T*>(a.d_v) + at;
#pragma unroll
  for (int dt = 0; dt < DU / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int d = 32 * dt + 2 * r + 4 * h;
      if (d >= a.dim) continue;
      f32x4 x = {}, y = {};
      if (live) {
        x = f32x4{dk[dt][r], dk[dt][r + 1], dk[dt][r + 2], dk[dt][r + 3]} * a.scale;
        y = f32x4{dv[dt][r], dv[dt][r + 1], dv[dt][r + 2], dv[dt][r + 3]};
      }
      if (a.row_parts > 1) {
        const int64_t all = a.k_tokens * a.kv_heads * a.dim;
        float* to = a.part_kv + blockIdx.z * all + at + d;
        if constexpr (DK) *reinterpret_cast<f32x4*>(to) = x;
        if constexpr (DV) *reinterpret_cast<f32x4*>(to + a.row_parts * all) = y;
        continue;
      }
      if constexpr (DK) store4(dkp + d, x[0], x[1], x[2], x[3]);
      if constexpr (DV) store4(dvp + d, y[0], y[1], y[2], y[3]);
    }
}

template <typename T, int DU, int MODE>
__global__ __launch_bounds__(kAttnThreads, sizeof(T) == 2 ? 2 : 1) void attn_bwd_kv_kernel(AttnArgs a) {
  __shared__ __attribute__((aligned(16))) KvShared<T, DU> sh;
  if constexpr (!kSplitKv<T, DU>) attn_bwd_kv<T, DU, MODE, true, true>(a, sh);
  else if (blockIdx.y == 0) attn_bwd_kv<T, DU, MODE, true, false>(a, sh);
  else attn_bwd_kv<T, DU, MODE, false, true>(a, sh);
}

// Adds parts' gradients, in order, four elements a thread: blockIdx.y picks the first or the second.
template <typename T>
__global__ __launch_bounds__(kAttnThreads) void attn_sum_kernel(const float* parts, int n, int64_t all, T* first,
                                                                T* second) {
  const int64_t e = (static_cast<int64_t>(blockIdx.x) * kAttnThreads + threadIdx.x) * 4;
  if (e >= all) return;
  const float* from = parts + blockIdx.y * n * all + e;
  f32x4 x = *reinterpret_cast<const f32x4*>(from);
  for (int i = 1; i < n; ++i) x += *reinterpret_cast<const f32x4*>(from + i * all);
  store4((blockIdx.y ? second : first) + e, x[0], x[1], x[2], x[3]);
}

// ---------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------
static int attn_setup(const gs_attention* p, AttnArgs& a) {
  GS_REQUIRE(p != nullptr, GS_ERR_ARG, "attention: arguments are NULL");
  GS_REQUIRE(p->dtype == GS_FLOAT32 || p->dtype == GS_BFLOAT16, GS_ERR_ARG,
             "attention: dtype must be GS_FLOAT32 or GS_BFLOAT16");
  GS_REQUIRE(p->heads >= 1 && p->kv_heads >= 1 && p->heads % p->kv_heads == 0, GS_ERR_ARG,
             "attention: %d heads are not a multiple of %d key heads", p->heads, p->kv_heads);
  GS_REQUIRE(p->dim >= 8 && p->dim <= GS_ATTENTION_MAX_DIM && p->dim % 8 == 0, GS_ERR_ARG,
             "attention: head size must be a multiple of 8 up to %d (got %d)", GS_ATTENTION_MAX_DIM, p->dim);
  GS_REQUIRE(p->docs >= 1, GS_ERR_ARG, "attention: need at least one document");
  GS_REQUIRE(p->docs == 1 || (p->q_offsets && p->k_offsets), GS_ERR_ARG,
             "attention: several documents need their offsets");
  GS_REQUIRE(p->q_tokens >= 0 && p->k_tokens >= 0, GS_ERR_ARG, "attention: token counts must be >= 0");
  const int64_t group = p->heads / p->kv_heads;
  GS_REQUIRE(p->q_tokens * group < (int64_t(1) << 30) && p->k_tokens < (int64_t(1) << 30) &&
                 p->docs < (1 << 26), GS_ERR_ARG, "attention: too many tokens or documents");
  GS_REQUIRE(group <= 512, GS_ERR_ARG, "attention: at most 512 heads share a key head");
  GS_REQUIRE(p->prefix == nullptr || p->causal, GS_ERR_ARG, "attention: a prefix needs the causal mask");
  GS_REQUIRE(p->scale == 0.0f || (fabsf(p->scale) >= FLT_MIN && fabsf(p->scale) <= 0x1p126f), GS_ERR_ARG,
             "attention: scale must be finite, 0 or between 2^-126 and 2^126 in size");
  // in float32, and so that scores over the cap neither over- nor underflow where they count
  const float per_cap = p->softcap != 0.0f && p->scale != 0.0f ? fabsf(p->scale) / p->softcap : 1.0f;
  GS_REQUIRE(p->softcap == 0.0f || (p->softcap >= 0x1p-96f && p->softcap <= 0x1p96f), GS_ERR_ARG,
             "attention: softcap must be 0 or between 2^-96 and 2^96");
  GS_REQUIRE(per_cap >= FLT_MIN && per_cap <= 0x1p125f, GS_ERR_ARG,
             "attention: scale / softcap must be between 2^-126 and 2^125");
  const bool has_q = p->q_tokens > 0, has_k = p->k_tokens > 0;
  GS_REQUIRE((!has_q || (p->q && p->out && p->lse)) && (!has_k || (p->k && p->v)), GS_ERR_ARG,
             "attention: null pointer");
  const int64_t elems = p->dtype == GS_BFLOAT16 ? 8 : 4;
  const int64_t strides[6] = {p->q_token_stride, p->q_head_stride, p->k_token_stride,
                              p->k_head_stride, p->v_token_stride, p->v_head_stride};
  for (int i = 0; i < 6; ++i)
    GS_REQUIRE(strides[i] >= 0 && strides[i] < (int64_t(1) << (i % 2 ? 40 : 22)) && strides[i] % elems == 0,
               GS_ERR_ALIGN, "attention: strides must be multiples of 16 bytes, token strides below 2^22 elements "
               "(got %lld)", static_cast<long long>(strides[i]));
  // what 64 consecutive rows (token, head of a group) of q span, 2^31 bytes at most
  GS_REQUIRE((64 / group + 2) * p->q_token_stride + group * p->q_head_stride < (int64_t(1) << 28), GS_ERR_ALIGN,
             "attention: q's strides are too large");
  GS_REQUIRE(aligned(p->q, 16) && aligned(p->k, 16) && aligned(p->v, 16) && aligned(p->out, 16) &&
                 aligned(p->out_low, 16) && aligned(p->lse, 4), GS_ERR_ALIGN, "attention: tensors must be 16-byte aligned");
  a = {};
  a.q = p->q;
  a.k = p->k;
  a.v = p->v;
  a.out = p->out;
  a.out_low = p->dtype == GS_BFLOAT16 ? p->out_low : nullptr;
  a.lse = p->lse;
  a.q_offsets = p->q_offsets;
  a.k_offsets = p->k_offsets;
  a.k_lengths = p->k_lengths;
  a.prefix = p->prefix;
  a.q_tokens = p->q_tokens;
  a.k_tokens = p->k_tokens;
  a.q_token = p->q_token_stride;
  a.q_head = p->q_head_stride;
  a.k_token = p->k_token_stride;
  a.k_head = p->k_head_stride;
  a.v_token = p->v_token_stride;
  a.v_head = p->v_head_stride;
  a.docs = p->docs;
  a.heads = p->heads;
  a.kv_heads = p->kv_heads;
  a.group = static_cast<int>(group);
  a.dim = p->dim;
  a.group_magic = static_cast<uint32_t>(((1 << 20) + group - 1) / group);
  a.causal = p->causal != 0;
  a.softcap = p->softcap;
  a.scale = p->scale;
  a.splits = 1;
  a.row_parts = a.key_parts = 1;
  return GS_OK;
}

// Tiles of `rows` rows that `tokens` tokens of `per` rows in docs + 2 stretches can take.
static int64_t tiles_of(int64_t tokens, int64_t per, int rows, int docs) { return tokens * per / rows + docs + 2; }

template <template <typename, int, int> class K, typename T, int DU>
static void launch_mode(const AttnArgs& a, dim3 grid, hipStream_t st) {
  if (a.softcap == 0.0f) K<T, DU, kPlain>::launch(a, grid, st);
  else if (sizeof(T) == 2 && a.softcap > kFarCap) K<T, DU, sizeof(T) == 2 ? kCapFar : kCap>::launch(a, grid, st);
  else K<T, DU, kCap>::launch(a, grid, st);
}
template <template <typename, int, int> class K>
static void launch_attn(const AttnArgs& a, int dtype, int64_t blocks, int parts, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(parts), static_cast<unsigned>(a.row_parts));
  const auto by_type = [&](auto du) {
    if (dtype == GS_BFLOAT16) launch_mode<K, __bf16, du.value>(a, grid, st);
    else launch_mode<K, float, du.value>(a, grid, st);
  };
  if (a.dim > 96) by_type(std::integral_constant<int, 128>{});
  else if (a.dim > 64) by_type(std::integral_constant<int, 96>{});
  else if (a.dim > 32) by_type(std::integral_constant<int, 64>{});
  else by_type(std::integral_constant<int, 32>{});
}
// Forward kernels have an instance for the causal mask, the backward's do not.
#define GS_ATTN_FORWARD(NAME, KERNEL, THREADS)                                                            \
  template <typename T, int DU, int MODE>                                                                 \
  struct NAME {                                                                                           \
    static void launch(const AttnArgs& a, dim3 grid, hipStream_t st) {                                    \
      if (a.causal) hipLaunchKernelGGL((KERNEL<T, DU, MODE, true>), grid, dim3(THREADS), 0, st, a);       \
      else hipLaunchKernelGGL((KERNEL<T, DU, MODE, false>), grid, dim3(THREADS), 0, st, a);               \
    }                                                                                                     \
  }
#define GS_ATTN_BACKWARD(NAME, KERNEL)                                                                    \
  template <typename T, int DU, int MODE>                                                                 \
  struct NAME {                                                                                           \
    static void launch(const AttnArgs& a, dim3 grid, hipStream_t st) {                                    \
      hipLaunchKernelGGL((KERNEL<T, DU, MODE>), grid, dim3(kAttnThreads), 0, st, a);                      \
    }                                                                                                     \
  }
GS_ATTN_FORWARD(FwdKernel, attn_fwd_kernel, kAttnThreads);
GS_ATTN_FORWARD(FewKernel, attn_few_kernel, kFewWaves<T> * kWave);
GS_ATTN_BACKWARD(BwdQKernel, attn_bwd_q_kernel);
GS_ATTN_BACKWARD(BwdKvKernel, attn_bwd_kv_kernel);
#undef GS_ATTN_FORWARD
#undef GS_ATTN_BACKWARD

// How a forward call is laid out, by sizes alone (so that the workspace can be asked for first).
struct FwdPlan {
  bool few;       // the kernel for few rows
  int64_t tiles;  // row tiles
  int splits;     // pieces of the keys
};
// Measured: pieces of the tile kernel for 512 workgroups against 1024: 181 queries on three caches of 5000
// 38 us against 43, 300 on two of 16000 87 us against 83; of the few-row kernel for 1024 against 2048: one
// token on 32k keys 39 us against 43, on 131k (2 key heads) 51 us against 70. Pieces of one length for all
// documents against as many pieces for each: 100 queries on caches of 9000 and seven of 500 40 us against
// 48, on eight of 3000 33 against 31 (workgroups that find no piece); 300 on 16000 and 1000 69 against 84.
// Provided for a document six times the average rather than twice: 41, 43 and 69 us.
constexpr int kFewSplitKeys = 1024, kTileSplitKeys = 256;
constexpr int kFewBlocks = 1024, kTileBlocks = 512, kMaxSplits = 256, kLongest = 2;

static FwdPlan plan_fwd(const AttnArgs& a) {
  FwdPlan f;
  // few: at most 32 rows to a document and key head on average. There the tile kernel's 128 rows are
  // mostly padding and each workgroup's keys one long chain.
  f.few = a.q_tokens * a.group <= 32 * static_cast<int64_t>(a.docs);
  f.tiles = tiles_of(a.q_tokens, a.group, f.few ? 32 : kAttnRows, a.docs);
  // Pieces until the chip has its workgroups, each of split_keys at least. A document's part of them goes
  // by its length, which is known on the device only: up to kLongest times the average is provided for, a
  // longer one gets longer pieces.
  const int64_t work = (f.few ? std::max<int64_t>(a.docs, a.q_tokens * a.group / 32)
                              : a.q_tokens * a.group / kAttnRows + 1) * a.kv_heads;
  const int64_t longest = std::min<int64_t>(a.docs, kLongest);
  const int64_t keys = a.k_tokens / a.docs * longest;
  const int64_t want = (f.few ? kFewBlocks : kTileBlocks) * longest / work;
  const int64_t most = keys / (f.few ? kFewSplitKeys : kTileSplitKeys);
  f.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, most, kMaxSplits})));
  return f;
}

static size_t fwd_workspace(const AttnArgs& a, const FwdPlan& f) {
  if (f.splits == 1) return 0;
  const size_t rows = static_cast<size_t>(a.q_tokens) * a.heads;
  return rows * (static_cast<size_t>(f.splits) * (a.dim + 2) + 1) * sizeof(float);
}

}  // namespace gs

using namespace gs;

extern "C" size_t gs_attention_fwd_workspace_size(const gs_attention* p) {
  clear_error();
  AttnArgs a;
  if (attn_setup(p, a) || p->q_tokens == 0) return 0;
  return fwd_workspace(a, plan_fwd(a));
}

extern "C" int gs_attention_fwd(const gs_attention* p, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  AttnArgs a;
  if (const int rc = attn_setup(p, a)) return rc;
  if (p->q_tokens == 0) return GS_OK;
  const FwdPlan f = plan_fwd(a);
  // a launch holds fewer than 2^32 threads
  const int64_t threads = f.few ? (p->dtype == GS_BFLOAT16 ? kFewWaves<__bf16> : kFewWaves<float>) * kWave : kAttnThreads;
  GS_REQUIRE(f.tiles * a.kv_heads * threads < (int64_t(1) << 32), GS_ERR_ARG,
             "attention: too many tokens, documents or heads");
  GS_REQUIRE(workspace_bytes >= fwd_workspace(a, f) && (workspace || f.splits == 1), GS_ERR_WORKSPACE,
             "attention: workspace too small");
  GS_REQUIRE(aligned(workspace, 16), GS_ERR_ALIGN, "attention: workspace must be 16-byte aligned");
  const hipStream_t st = as_stream(stream);
  a.n_tiles = static_cast<int>(f.tiles);
  a.splits = f.splits;
  a.split_keys = f.few ? kFewSplitKeys : kTileSplitKeys;
  a.split_unit = f.few ? 8 * 32 : kAttnKeys;
  a.split_blocks = f.few ? kFewBlocks : kTileBlocks;
  const int64_t rows = a.q_tokens * a.heads;
  a.part = static_cast<float*>(workspace);
  a.part_stat = a.part + rows * a.splits * a.dim;
  a.part_n = reinterpret_cast<int32_t*>(a.part_stat + rows * a.splits * 2);
  if (f.few)
    launch_attn<FewKernel>(a, p->dtype, f.tiles * a.kv_heads, a.splits, st);
  else
    launch_attn<FwdKernel>(a, p->dtype, f.tiles * a.kv_heads, a.splits, st);
  if (const int rc = check_launch("attention")) return rc;
  if (a.splits == 1) return GS_OK;
  const dim3 grid(static_cast<unsigned>((rows * 32 + kAttnThreads - 1) / kAttnThreads)), block(kAttnThreads);
  if (p->dtype == GS_BFLOAT16)
    hipLaunchKernelGGL(attn_join_kernel<__bf16>, grid, block, 0, st, a);
  else
    hipLaunchKernelGGL(attn_join_kernel<float>, grid, block, 0, st, a);
  return check_launch("attention (join)");
}

namespace gs {

// How a backward call is laid out. A key tile's workgroup walks over every row that sees it, times the
// heads of its group: with few key heads that is one long chain on a part of the chip. The rows are then
// cut into parts, until the longest chain is about half of what each of the chip's 512 workgroups has to
// do on average (a causal tile has half the rows on average); the parts' sums are joined in float32.
// Measured at 8192 causal tokens, 16 heads on 4 of 128, capped: backward 1983 us in one part, 1509 us in 4.
struct BwdPlan {
  int64_t q_tiles, k_tiles;
  int kv_roles, row_parts, key_parts;
  size_t delta, part_q, part_kv;  // workspace floats
};
static BwdPlan plan_bwd(const AttnArgs& a, int dtype) {
  BwdPlan b;
  b.q_tiles = tiles_of(a.q_tokens, a.group, kAttnRows, a.docs);
  b.k_tiles = tiles_of(a.k_tokens, 1, kAttnRows, a.docs);
  b.kv_roles = split_kv(dtype == GS_BFLOAT16, a.dim) ? 2 : 1;
  const int64_t blocks = (a.k_tokens + kAttnRows - 1) / kAttnRows * a.kv_heads * b.kv_roles;
  const int64_t rows = a.q_tokens * a.group / a.docs;
  const int64_t want = blocks > 0 ? (a.causal ? 4 : 2) * 512 / blocks : 1;
  b.row_parts = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, rows / (dtype == GS_BFLOAT16 ? 256 : 128), 8})));
  b.delta = (static_cast<size_t>(a.q_tokens) * a.heads + 3) / 4 * 4;
  b.part_kv = b.row_parts > 1 ? 2 * static_cast<size_t>(b.row_parts) * a.k_tokens * a.kv_heads * a.dim : 0;
  // Query gradients: the keys in parts, until there are 512 workgroups (2000 tokens, 8 heads of 64: backward
  // 112 us in one part, 104 us in 4).
  const int64_t q_blocks = (a.q_tokens * a.group + kAttnRows - 1) / kAttnRows * a.kv_heads;
  const int64_t q_want = q_blocks > 0 ? 512 / q_blocks : 1;
  const int64_t keys = a.k_tokens / a.docs;
  b.key_parts = static_cast<int>(
      std::max<int64_t>(1, std::min<int64_t>({q_want, keys / (dtype == GS_BFLOAT16 ? 256 : 64), 8})));
  b.part_q = b.key_parts > 1 ? static_cast<size_t>(b.key_parts) * a.q_tokens * a.heads * a.dim : 0;
  return b;
}

}  // namespace gs

extern "C" size_t gs_attention_bwd_workspace_size(const gs_attention* p) {
  clear_error();
  AttnArgs a;
  if (attn_setup(p, a)) return 0;
  const BwdPlan b = plan_bwd(a, p->dtype);
  return (b.delta + b.part_q + b.part_kv) * sizeof(float);
}

extern "C" int gs_attention_bwd(const gs_attention* p, const void* d_out, void* d_q, void* d_k, void* d_v,
                                void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  AttnArgs a;
  if (const int rc = attn_setup(p, a)) return rc;
  GS_REQUIRE((p->q_tokens == 0 || (d_out && d_q)) && (p->k_tokens == 0 || (d_k && d_v)), GS_ERR_ARG,
             "attention backward: null pointer");
  GS_REQUIRE(aligned(d_out, 16) && aligned(d_q, 16) && aligned(d_k, 16) && aligned(d_v, 16), GS_ERR_ALIGN,
             "attention backward: tensors must be 16-byte aligned");
  // d_out is contiguous, whatever q's strides: 64 of its rows, like those of q
  GS_REQUIRE((64 / a.group + 2) * static_cast<int64_t>(a.heads) * a.dim < (int64_t(1) << 28), GS_ERR_ARG,
             "attention backward: too many heads");
  const BwdPlan b = plan_bwd(a, p->dtype);
  const size_t need = (b.delta + b.part_q + b.part_kv) * sizeof(float);
  GS_REQUIRE(workspace_bytes >= need && (workspace || need == 0), GS_ERR_WORKSPACE,
             "attention backward: workspace too small");
  GS_REQUIRE(aligned(workspace, 16), GS_ERR_ALIGN, "attention backward: workspace must be 16-byte aligned");
  GS_REQUIRE(std::max(b.q_tiles, b.k_tiles) * a.kv_heads * kAttnThreads < (int64_t(1) << 32), GS_ERR_ARG,
             "attention: too many tokens, documents or heads");
  a.d_out = d_out;
  a.d_q = d_q;
  a.d_k = d_k;
  a.d_v = d_v;
  a.delta = static_cast<float*>(workspace);
  a.part_q = a.delta + b.delta;
  a.part_kv = a.part_q + b.part_q;
  const hipStream_t st = as_stream(stream);
  const auto sum = [&](const float* parts, int n, int64_t all, void* first, void* second) {
    const dim3 grid(static_cast<unsigned>((all / 4 + kAttnThreads - 1) / kAttnThreads), second ? 2 : 1);
    if (p->dtype == GS_BFLOAT16)
      hipLaunchKernelGGL(attn_sum_kernel<__bf16>, grid, dim3(kAttnThreads), 0, st, parts, n, all,
                         static_cast<__bf16*>(first), static_cast<__bf16*>(second));
    else
      hipLaunchKernelGGL(attn_sum_kernel<float>, grid, dim3(kAttnThreads), 0, st, parts, n, all,
                         static_cast<float*>(first), static_cast<float*>(second));
    return check_launch("attention backward (sums)");
  };
  if (p->q_tokens > 0) {
    a.n_tiles = static_cast<int>(b.q_tiles);
    a.key_parts = b.key_parts;
    launch_attn<BwdQKernel>(a, p->dtype, b.q_tiles * a.kv_heads, b.key_parts, st);
    if (const int rc = check_launch("attention backward (queries)")) return rc;
    if (b.key_parts > 1)
      if (const int rc = sum(a.part_q, b.key_parts, a.q_tokens * a.heads * a.dim, d_q, nullptr)) return rc;
  }
  if (p->k_tokens > 0) {
    a.n_tiles = static_cast<int>(b.k_tiles);
    a.row_parts = b.row_parts;
    launch_attn<BwdKvKernel>(a, p->dtype, b.k_tiles * a.kv_heads, b.kv_roles, st);
    if (const int rc = check_launch("attention backward (keys)")) return rc;
    if (b.row_parts > 1) return sum(a.part_kv, b.row_parts, a.k_tokens * a.kv_heads * a.dim, d_k, d_v);
  }
  return GS_OK;
}
