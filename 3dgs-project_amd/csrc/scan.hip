// A gated linear recurrence over packed documents, forward and backward:
//
//   a = sigmoid(f);  h_t = a_t h_(t-1) + (1 - a_t) x_t;  y_t = h_t, or h_t silu(o_t)
//   l_t = dy_t silu(o_t) + a_(t+1) l_(t+1)   (at a document's last token the state's gradient in place of the second term)
//   dx = (1 - a) l;  df = l (h_(t-1) - x) a (1 - a);  do = dy h silu'(o);  dinitial = a l at the first token
//
// A step is the map h -> E + P h, and maps compose, so the tokens are cut into chunks of 16 that a wavefront walks, a
// lane holding four channels: scan_sums_kernel forms every chunk's map and, in LDS, the maps from the start of
// a part (the chunks of one workgroup) to each of its chunks; scan_parts_kernel joins the parts; scan_apply_kernel has so every
// chunk's state, and walks the tokens again with it. The inputs are so read twice, the second time from the last-level
// cache as far as it holds them. (One pass that waits for the workgroups before it would read them once, but
// needs them to be running; nothing here waits for another workgroup.)
//
// Memory bounds it beside the chain of a chunk's steps: 32771 x 1024 with a gate in bfloat16, forward sums 41 us, parts 10,
// walk 56 (268 MB, 4.8 TB/s); backward sums 51, parts 10, walk 128 (470 MB, 3.7 TB/s); one pass over inputs and
// results alone 737 MB, at a copy's 5.1 TB/s 145 us. With the loads of all sixteen tokens sent together
// the sums took 43 and 70 us, the walk 71.
//
// A document's first token replaces the state, so P = 0 there, and a map with P = 0 drops what came before it whatever
// that was: documents do not see each other's infinities and NaN.
//
// Accuracy: long memories have a near 1, where 1 - a is what counts. The smaller of a and 1 - a is formed
// directly, s = e / (1 + e) with e = exp(-|f|), by the hardware's exponential and reciprocal in both types: s is off by 2^-23 |f|
// and a few 2^-24 of itself, beside float32 roundings of the steps. These are taken as h + s (x - h) or x + s (h - x). A chunk's P
// is kept as 1 - P while that is the smaller one; a chunk's sum starts at zero, so its rounding is relative to what the
// chunk adds; chunks and parts are joined in float64. Rounding so does not pile up over the length of the sequence.
#include <algorithm>
#include <type_traits>

#include "gs_attention.h"
#include "gs_rows.h"

namespace gs {

constexpr int kScanChunk = 16;                           // tokens of a chunk
constexpr int kScanWaves = 8;
constexpr int kScanThreads = kScanWaves * kWave;
constexpr int kWalkWaves = 4;                            // of a workgroup where every wavefront has a chunk
constexpr int kScanVec = 4;                              // channels of a lane
constexpr int kScanGroup = kWave * kScanVec;             // channels of a workgroup
constexpr int kScanParts = 512;
constexpr int kScanBatch = 8;                            // tokens whose loads are in flight together

struct ScanArgs {
  const void *x, *f, *o;
  const float* initial;
  void* y;
  float *state, *carry;  // carry [chunks][width]: the state before every chunk
  const int32_t* offsets;
  int64_t tokens, x_stride, f_stride, o_stride;
  int docs, width, reverse;
  int groups;                 // of kScanGroup channels
  int chunks, parts, blocks;  // blocks: of a part
  int serial;                 // one wavefront walks all chunks
  int single;                 // one wavefront walks a document's
  float2* prefix;             // [chunks][width]: the map from the part's start to the chunk
  float2* part;               // [parts][width]: the map of a part
  float* before;              // [parts][width]: the state that a part starts with
  // backward
  const void* d_y;
  const float* d_state;
  void *d_x, *d_f, *d_o;
  float* d_initial;
};

template <typename T>
using Raw4 = RawN<T, 4>;
template <typename T>
__device__ __forceinline__ void put4(T* p, int n, const float (&v)[4]) {
  typedef T Vec __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  if (n >= 4) {
    Vec a;
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = static_cast<T>(v[j]);
    *reinterpret_cast<Vec*>(p) = a;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) p[j] = static_cast<T>(v[j]);
  }
}

// sigmoid(v): the larger of it and its complement, and the smaller.
struct Sigmoid {
  float large, small;
  bool up;  // the larger one is sigmoid(v)
  __device__ __forceinline__ explicit Sigmoid(float v) {
    const float e = exp2_hw(-fabsf(v) * kLog2e);
    large = __builtin_amdgcn_rcpf(1.0f + e);
    small = e * large;
    up = v >= 0.0f;
  }
  __device__ __forceinline__ float value() const { return up ? large : small; }
  __device__ __forceinline__ float rest() const { return up ? small : large; }
  __device__ __forceinline__ float step(float h, float x) const {
    const float from = up ? h : x, to = up ? x : h;
    return fmaf(small, to - from, from);
  }
  __device__ __forceinline__ float times(float v) const { return up ? fmaf(-small, v, v) : small * v; }
};

// The factor P of a chunk: its product, and 1 minus it from sums of its own.
struct Factor {
  float p = 1.0f, q = 0.0f;
  __device__ __forceinline__ void by(const Sigmoid& a) {
    p *= a.value();
    q = fmaf(a.rest(), 1.0f - q, q);
  }
  __device__ __forceinline__ void drop() {
    p = 0.0f;
    q = 1.0f;
  }
};
// One word for it: 1 - P where that is at most a half, -P otherwise (the sign tells them apart, -0 too).
__device__ __forceinline__ float packed(float p, float q) { return q <= 0.5f ? q : -p; }
__device__ __forceinline__ double factor_of(float w) {
  return __float_as_uint(w) >> 31 ? -static_cast<double>(w) : 1.0 - static_cast<double>(w);
}
__device__ __forceinline__ float packed(double p) {
  return p >= 0.5 ? fabsf(static_cast<float>(1.0 - p)) : -static_cast<float>(p);
}
// E + P h where P = 0 drops h.
__device__ __forceinline__ double mapped(double e, double p, double h) { return p == 0.0 ? e : fma(p, h, e); }

// Place i of the documents' edges in walking order: from the front, or from the back when reversed.
__device__ __forceinline__ int64_t scan_edge(const ScanArgs& a, int i) {
  const int k = a.reverse ? a.docs - i : i;
  int64_t v = a.offsets ? a.offsets[k] : (k ? a.tokens : 0);
  v = v < 0 ? 0 : (v > a.tokens ? a.tokens : v);
  return a.reverse ? a.tokens - v : v;
}
__device__ __forceinline__ int doc_at(const ScanArgs& a, int i) { return a.reverse ? a.docs - 1 - i : i; }
__device__ __forceinline__ int64_t token_at(const ScanArgs& a, int64_t p) { return a.reverse ? a.tokens - 1 - p : p; }

// What the tokens of a chunk at places p0 .. p0 + 15 are: bits for those inside a document, its first, its last; and
// in lane k the document of token k.
struct Places {
  uint32_t inside, first, last;
  uint32_t mine = 0;  // of one document's: are walked with it
  int doc;
  // of one document, places from .. to, walked with all of lo .. hi
  __device__ __forceinline__ Places(const ScanArgs& a, int64_t p0, int doc_, int from, int to, int lo, int hi) : doc(doc_at(a, doc_)) {
    const auto bits = [&](int b, int e) {
      const auto up_to = [&](int p) { return (1u << min(max(static_cast<int>(p - p0), 0), kScanChunk)) - 1; };
      return up_to(e) & ~up_to(b);
    };
    inside = bits(from, to);
    mine = bits(lo, hi);
    first = inside & bits(from, from + 1);
    last = inside & bits(to - 1, to);
  }
  __device__ __forceinline__ Places(const ScanArgs& a, int64_t p0) {
    const int lane = threadIdx.x % kWave;
    const int64_t p = p0 + lane;
    const bool there = lane < kScanChunk && p < a.tokens;
    // i: the last edge at or before p, so that empty documents are passed over
    int i = -1;
    int64_t at = -1, next = -1;
    if (a.docs < kWave) {
      const int64_t e = scan_edge(a, min(lane, a.docs));
#pragma unroll
      for (int k = 0; k < kScanChunk; ++k) {
        const uint64_t b = __ballot(lane <= a.docs && e <= p0 + k);
        if (lane == k) i = static_cast<int>(__popcll(b)) - 1;
      }
      at = __shfl(e, max(i, 0));
      next = __shfl(e, min(i + 1, a.docs));
    } else if (there) {
      int lo = 0, hi = a.docs + 1;  // edges before lo are at or before p, those from hi on are not
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (scan_edge(a, mid) <= p) lo = mid + 1;
        else hi = mid;
      }
      i = lo - 1;
      at = scan_edge(a, max(i, 0));
      next = scan_edge(a, min(i + 1, a.docs));
    }
    const bool in = there && i >= 0 && i < a.docs;
    doc = in ? doc_at(a, i) : 0;
    inside = static_cast<uint32_t>(__ballot(in));
    first = static_cast<uint32_t>(__ballot(in && at == p));
    last = static_cast<uint32_t>(__ballot(in && next == p + 1));
  }
  __device__ __forceinline__ int doc_of(int k) const { return __builtin_amdgcn_readlane(doc, k); }
};

// A lane's four channels. Lanes past the width, and the last one where the width is no multiple of four, take the last four
// channels: what two lanes hold alike they also write alike, and no access needs a branch. Only rows of fewer than
// four channels (SMALL) are read and written element by element. at_of: the channels' place in a row whose address is the same for
// all lanes, which takes scalar registers and 32 bits of the lane's.
template <bool SMALL>
struct Channels {
  int at, n;
  __device__ __forceinline__ Channels(const ScanArgs& a, int group)
      : at(SMALL ? 0 : min((group * kWave + static_cast<int>(threadIdx.x % kWave)) * kScanVec, a.width - kScanVec)),
        n(SMALL ? a.width : kScanVec) {}
  template <typename T>
  __device__ __forceinline__ T* at_of(T* row) const {
    using Byte = std::conditional_t<std::is_const_v<T>, const char, char>;
    return reinterpret_cast<T*>(reinterpret_cast<Byte*>(row) + static_cast<uint32_t>(at * static_cast<int>(sizeof(T))));
  }
  // Row `row` of a tensor of whole rows; a tensor that is not there is zero.
  template <typename T>
  __device__ __forceinline__ void load(const ScanArgs& a, const T* p, int64_t row, float (&v)[4]) const {
    Raw4<T> r;
    r.load(at_of(p + row * a.width), p ? (SMALL ? n : kScanVec) : 0);
    r.to(v);
  }
  template <typename T>
  __device__ __forceinline__ void store(T* row, const float (&v)[4]) const {
    put4(at_of(row), SMALL ? n : kScanVec, v);
  }
};

// Rows of the tokens at places p0 .. p0 + 7, whatever they belong to (so that no load waits for the documents); past the last
// token that one's again. within: outside lo .. hi - 1 the nearest one's again.
template <typename T, bool SMALL>
struct Batch {
  Raw4<T> row[kScanBatch];
  __device__ __forceinline__ void load(const ScanArgs& a, const void* p, int64_t stride, int64_t p0, const Channels<SMALL>& c) {
#pragma unroll
    for (int k = 0; k < kScanBatch; ++k) at(a, k, p, stride, min<int64_t>(p0 + k, a.tokens - 1), c);
  }
  __device__ __forceinline__ void within(const ScanArgs& a, const void* p, int64_t stride, int64_t p0, const Channels<SMALL>& c,
                                         int lo, int hi) {
#pragma unroll
    for (int k = 0; k < kScanBatch; ++k) at(a, k, p, stride, min(max<int64_t>(p0 + k, lo), int64_t(hi) - 1), c);
  }
  __device__ __forceinline__ void at(const ScanArgs& a, int k, const void* p, int64_t stride, int64_t place, const Channels<SMALL>& c) {
    row[k].load(c.at_of(static_cast<const T*>(p) + token_at(a, place) * stride), SMALL ? c.n : kScanVec);
  }
};

// ---- the maps of chunks and parts --------------------------------------------------------------------
// BACK: of l, whose walk starts at a chunk's last token.

template <typename T, bool BACK, bool SMALL>
__global__ __launch_bounds__(kScanThreads) void scan_sums_kernel(ScanArgs a) {
  __shared__ float2 maps[kScanWaves][kScanGroup];
  const Channels<SMALL> c(a, blockIdx.x);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  // the running map of the part, of one channel a thread (the first four wavefronts)
  double e_run = 0.0, p_run = 1.0;
  const int own = blockIdx.x * kScanGroup + threadIdx.x;
  for (int block = 0; block < a.blocks; ++block) {
    const int n0 = (blockIdx.y * a.blocks + block) * kScanWaves;  // in walking order
    if (n0 >= a.chunks) break;
    const int n = n0 + wave;
    float e[4] = {};
    Factor f[4];
    if (n < a.chunks) {
      const int64_t p0 = static_cast<int64_t>(BACK ? a.chunks - 1 - n : n) * kScanChunk;
      const Places pl(a, p0);
#pragma unroll
      for (int b = 0; b < kScanChunk / kScanBatch; ++b) {
        const int k0 = (BACK ? kScanChunk / kScanBatch - 1 - b : b) * kScanBatch;
        Batch<T, SMALL> bf, bx, bo;
        bf.load(a, a.f, a.f_stride, p0 + k0, c);
        bx.load(a, BACK ? a.d_y : a.x, BACK ? a.width : a.x_stride, p0 + k0, c);
        if (BACK && a.o) bo.load(a, a.o, a.o_stride, p0 + k0, c);
#pragma unroll
        for (int i = 0; i < kScanBatch; ++i) {
          const int k = BACK ? k0 + kScanBatch - 1 - i : k0 + i, r = k - k0;
          if (!((pl.inside >> k) & 1)) continue;
          if (((BACK ? pl.last : pl.first) >> k) & 1) {
            const float* from = BACK ? a.d_state : a.initial;
            c.load(a, from, pl.doc_of(k), e);
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j].drop();
          }
          float vf[4], vx[4], vo[4];
          bf.row[r].to(vf);
          bx.row[r].to(vx);
          if (BACK && a.o) {
            bo.row[r].to(vo);
#pragma unroll
            for (int j = 0; j < 4; ++j) vx[j] *= vo[j] * Sigmoid(vo[j]).value();
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const Sigmoid s(vf[j]);
            if constexpr (BACK) e[j] = s.times(e[j] + vx[j]);
            else e[j] = s.step(e[j], vx[j]);
            f[j].by(s);
          }
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int ch = c.at + j - static_cast<int>(blockIdx.x) * kScanGroup;  // (the last four may begin in the group before)
      if (ch >= 0) maps[wave][ch] = make_float2(e[j], packed(f[j].p, f[j].q));
    }
    __syncthreads();
    if (threadIdx.x < kScanGroup && own < a.width) {
      for (int w = 0; w < kScanWaves && n0 + w < a.chunks; ++w) {
        a.prefix[static_cast<int64_t>(n0 + w) * a.width + own] = make_float2(static_cast<float>(e_run), packed(p_run));
        const float2 m = maps[w][threadIdx.x];
        const double p = factor_of(m.y);
        e_run = mapped(m.x, p, e_run);
        p_run = p == 0.0 ? 0.0 : p_run * p;
      }
    }
  }
  if (a.parts > 1 && threadIdx.x < kScanGroup && own < a.width)
    a.part[static_cast<int64_t>(blockIdx.y) * a.width + own] = make_float2(static_cast<float>(e_run), packed(p_run));
}

// The state that every part starts with: the maps of the parts before it, joined. 32 lanes have a channel each, and 32 runs of
// parts are joined side by side, first to the runs' own maps and then, from what comes before a run, part by part.
constexpr int kRuns = 32, kRunParts = kScanParts / kRuns, kJoinThreads = kRuns * 32;
__global__ __launch_bounds__(kJoinThreads) void scan_parts_kernel(ScanArgs a) {
  __shared__ double2 maps[kRuns][32];
  const int lane = threadIdx.x % 32, run = threadIdx.x / 32, ch = blockIdx.x * 32 + lane, first = run * kRunParts;
  float2 m[kRunParts];
#pragma unroll
  for (int i = 0; i < kRunParts; ++i)
    m[i] = ch < a.width && first + i < a.parts ? a.part[static_cast<int64_t>(first + i) * a.width + ch] : make_float2(0.0f, 0.0f);
  double e = 0.0, p = 1.0;
#pragma unroll
  for (int i = 0; i < kRunParts; ++i) {
    const double f = factor_of(m[i].y);
    e = mapped(m[i].x, f, e);
    p = f == 0.0 ? 0.0 : p * f;
  }
  maps[run][lane] = make_double2(e, p);
  __syncthreads();
  double h = 0.0;
#pragma unroll 4
  for (int r = 0; r < run; ++r) h = mapped(maps[r][lane].x, maps[r][lane].y, h);
  if (ch >= a.width) return;
#pragma unroll
  for (int i = 0; i < kRunParts; ++i) {
    if (first + i < a.parts) a.before[static_cast<int64_t>(first + i) * a.width + ch] = static_cast<float>(h);
    h = mapped(m[i].x, factor_of(m[i].y), h);
  }
}

// The state that chunk n (in walking order) starts with.
template <bool SMALL>
__device__ __forceinline__ void state_before(const ScanArgs& a, int n, const Channels<SMALL>& c, float (&h)[4]) {
  float from[4];
  c.load(a, a.before, n / (a.blocks * kScanWaves), from);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (SMALL && j >= c.n) continue;
    const float2 m = a.prefix[static_cast<int64_t>(n) * a.width + c.at + j];
    h[j] = static_cast<float>(mapped(m.x, factor_of(m.y), from[j]));
  }
}

// Documents without tokens: their state goes through as it is, and so does its gradient.
template <bool SMALL>
__device__ __forceinline__ void pass_empty(const ScanArgs& a, const Channels<SMALL>& c, const float* from, float* to) {
  if (to == nullptr) return;
  const int lane = threadIdx.x % kWave, waves = gridDim.x / a.groups * (blockDim.x / kWave);
  for (int64_t d0 = (blockIdx.x / a.groups * (blockDim.x / kWave) + threadIdx.x / kWave) * int64_t(kWave); d0 < a.docs;
       d0 += static_cast<int64_t>(waves) * kWave) {
    const int d = static_cast<int>(min<int64_t>(d0 + lane, a.docs - 1));
    uint64_t empty = __ballot(d0 + lane < a.docs && scan_edge(a, d) >= scan_edge(a, d + 1));
    for (; empty; empty &= empty - 1) {
      const int64_t row = doc_at(a, static_cast<int>(d0) + __builtin_ctzll(empty));
      float v[4];
      c.load(a, from, row, v);
      c.store(to + row * a.width, v);
    }
  }
}

// ---- the walk ----------------------------------------------------------------------------------------

// The chunks that a wavefront walks: one; in serial mode all of them. ONE: those of its document (and of what belongs to none
// before the first document or behind the last).
template <bool ONE>
struct Walk {
  int first, end;
  int doc, from, to, lo, hi;  // ONE: in walking order, its places, and the places walked
  __device__ __forceinline__ explicit Walk(const ScanArgs& a) {
    if constexpr (ONE) {
      doc = blockIdx.x / a.groups;
      from = __builtin_amdgcn_readfirstlane(static_cast<int>(scan_edge(a, doc)));
      to = max(from, __builtin_amdgcn_readfirstlane(static_cast<int>(scan_edge(a, doc + 1))));
      lo = doc == 0 ? 0 : from;
      hi = doc == a.docs - 1 ? static_cast<int>(a.tokens) : to;
      first = lo / kScanChunk;
      end = hi > lo ? (hi - 1) / kScanChunk + 1 : first;
    } else {
      // the last ones first: what the sums' kernel read last is still in the cache
      const int n = (gridDim.x - 1 - blockIdx.x) / a.groups * (blockDim.x / kWave) + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
      first = a.serial ? 0 : n;
      end = a.serial ? a.chunks : min(n + 1, a.chunks);
    }
  }
  __device__ __forceinline__ Places places(const ScanArgs& a, int64_t p0) const {
    if constexpr (ONE) return Places(a, p0, doc, from, to, lo, hi);
    else return Places(a, p0);
  }
  template <typename B, typename C>
  __device__ __forceinline__ void load(B& b, const ScanArgs& a, const void* p, int64_t stride, int64_t p0, const C& c) const {
    if constexpr (ONE) b.within(a, p, stride, p0, c, lo, hi);
    else b.load(a, p, stride, p0, c);
  }
  // Token k of a chunk, at place p, is walked here.
  __device__ __forceinline__ bool has(const ScanArgs& a, const Places& pl, int k, int64_t p) const {
    return ONE ? (pl.mine >> k) & 1 : p < a.tokens;
  }
  __device__ __forceinline__ bool some(const ScanArgs& a, const Places& pl, int k, int64_t p) const {
    return ONE ? ((pl.mine >> k) & ((1u << kScanBatch) - 1)) != 0 : p < a.tokens;
  }
};

template <typename T, bool SMALL, bool ONE>
__global__ __launch_bounds__(kWalkWaves* kWave, 3) void scan_apply_kernel(ScanArgs a) {
  const Channels<SMALL> c(a, blockIdx.x % a.groups);
  pass_empty(a, c, a.initial, a.state);
  float h[4] = {};
  const Walk<ONE> w(a);
  for (int n = w.first; n < w.end; ++n) {
    const int64_t p0 = static_cast<int64_t>(n) * kScanChunk;
    if (!ONE && !a.serial) state_before(a, n, c, h);
    const Places pl = w.places(a, p0);
    if (a.carry && w.has(a, pl, 0, p0)) c.store(a.carry + static_cast<int64_t>(n) * a.width, h);
#pragma unroll
    for (int k0 = 0; k0 < kScanChunk; k0 += kScanBatch) {
      if (!w.some(a, pl, k0, p0 + k0)) continue;
      Batch<T, SMALL> bf, bx, bo;
      w.load(bf, a, a.f, a.f_stride, p0 + k0, c);
      w.load(bx, a, a.x, a.x_stride, p0 + k0, c);
      if (a.o) w.load(bo, a, a.o, a.o_stride, p0 + k0, c);
      Raw4<float> first[kScanBatch];
      if ((pl.first >> k0) & ((1u << kScanBatch) - 1)) {
#pragma unroll
        for (int k = 0; k < kScanBatch; ++k)
          if ((pl.first >> (k0 + k)) & 1)
            first[k].load(c.at_of(a.initial + static_cast<int64_t>(pl.doc_of(k0 + k)) * a.width), a.initial ? (SMALL ? c.n : kScanVec) : 0);
      }
#pragma unroll
      for (int k = 0; k < kScanBatch; ++k) {
        const int64_t p = p0 + k0 + k;
        if (!w.has(a, pl, k0 + k, p)) continue;
        float y[4] = {};
        if ((pl.inside >> (k0 + k)) & 1) {
          if ((pl.first >> (k0 + k)) & 1) first[k].to(h);
          float vf[4], vx[4], vo[4];
          bf.row[k].to(vf);
          bx.row[k].to(vx);
#pragma unroll
          for (int j = 0; j < 4; ++j) y[j] = h[j] = Sigmoid(vf[j]).step(h[j], vx[j]);
          if (a.o) {
            bo.row[k].to(vo);
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] *= vo[j] * Sigmoid(vo[j]).value();
          }
          if (a.state && ((pl.last >> (k0 + k)) & 1)) c.store(a.state + static_cast<int64_t>(pl.doc_of(k0 + k)) * a.width, h);
        }
        c.store(static_cast<T*>(a.y) + token_at(a, p) * a.width, y);
      }
    }
  }
}

// Eight tokens at a time from the chunk's end: the states before them are walked to from the chunk's start and held in
// registers. (All sixteen at once took 235 registers and two wavefronts a SIMD: 32771 x 1024 175 us.)
template <typename T, bool SMALL, bool ONE>
__global__ __launch_bounds__(kWalkWaves* kWave, 2) void scan_bwd_kernel(ScanArgs a) {
  const Channels<SMALL> c(a, blockIdx.x % a.groups);
  pass_empty(a, c, a.d_state, a.d_initial);
  float l[4] = {};  // a l of the token after
  const Walk<ONE> w(a);
  for (int n = w.first; n < w.end; ++n) {
    const int chunk = (ONE ? w.first + w.end : a.chunks) - 1 - n;
    if (!ONE && !a.serial) state_before(a, n, c, l);
    const Places pl = w.places(a, static_cast<int64_t>(chunk) * kScanChunk);
#pragma unroll 1
    for (int half = kScanChunk / kScanBatch - 1; half >= 0; --half) {
      const int64_t p0 = static_cast<int64_t>(chunk) * kScanChunk + half * kScanBatch;
      const uint32_t inside = pl.inside >> (half * kScanBatch), first = pl.first >> (half * kScanBatch),
                     last = pl.last >> (half * kScanBatch);
      if (!w.some(a, pl, half * kScanBatch, p0)) continue;
      float before[kScanBatch][4], h[4];
      c.load(a, a.carry, chunk, h);
      const auto begin = [&](int k) {  // the state before token k of the chunk where it is a document's first
        c.load(a, a.initial, pl.doc_of(k), h);
      };
      Batch<T, SMALL> bf, bx, bd, bo;
      if (half) {
        w.load(bf, a, a.f, a.f_stride, p0 - kScanBatch, c);
        w.load(bx, a, a.x, a.x_stride, p0 - kScanBatch, c);
#pragma unroll
        for (int k = 0; k < kScanBatch; ++k) {
          if ((pl.first >> k) & 1) begin(k);
          float vf[4], vx[4];
          bf.row[k].to(vf);
          bx.row[k].to(vx);
#pragma unroll
          for (int j = 0; j < 4; ++j) h[j] = Sigmoid(vf[j]).step(h[j], vx[j]);
        }
      }
      w.load(bf, a, a.f, a.f_stride, p0, c);
      w.load(bx, a, a.x, a.x_stride, p0, c);
      w.load(bd, a, a.d_y, a.width, p0, c);
      if (a.o) w.load(bo, a, a.o, a.o_stride, p0, c);
#pragma unroll
      for (int k = 0; k < kScanBatch; ++k) {
        if ((first >> k) & 1) begin(half * kScanBatch + k);
        float vf[4], vx[4];
        bf.row[k].to(vf);
        bx.row[k].to(vx);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          before[k][j] = h[j];
          h[j] = Sigmoid(vf[j]).step(h[j], vx[j]);
        }
      }
#pragma unroll
      for (int k = kScanBatch - 1; k >= 0; --k) {
        const int64_t p = p0 + k;
        if (!w.has(a, pl, half * kScanBatch + k, p)) continue;
        float dx[4] = {}, df[4] = {}, dg[4] = {};
        if ((inside >> k) & 1) {
          if ((last >> k) & 1)
            c.load(a, a.d_state, pl.doc_of(half * kScanBatch + k), l);
          float vf[4], vx[4], vo[4], vd[4];
          bf.row[k].to(vf);
          bx.row[k].to(vx);
          bd.row[k].to(vd);
          if (a.o) bo.row[k].to(vo);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const Sigmoid s(vf[j]);
            const float was = before[k][j];
            float d = vd[j];
            if (a.o) {
              const Sigmoid g(vo[j]);
              const float open = vo[j] * g.value();
              dg[j] = d * s.step(was, vx[j]) * fmaf(vo[j], g.large * g.small, g.value());
              d *= open;
            }
            const float whole = d + l[j];
            dx[j] = whole * s.rest();
            df[j] = whole * (was - vx[j]) * (s.large * s.small);
            l[j] = s.times(whole);
          }
          if (a.d_initial && ((first >> k) & 1))
            c.store(a.d_initial + static_cast<int64_t>(pl.doc_of(half * kScanBatch + k)) * a.width, l);
        }
        const int64_t at = token_at(a, p) * a.width;
        if (a.d_x) c.store(static_cast<T*>(a.d_x) + at, dx);
        if (a.d_f) c.store(static_cast<T*>(a.d_f) + at, df);
        if (a.d_o) c.store(static_cast<T*>(a.d_o) + at, dg);
      }
    }
  }
}

// Up to so many tokens one wavefront a channel group walks them all, in one launch: 1, 16, 24 (of 24 documents), 32 and 48
// tokens of 1024 channels 4.1, 9.3, 14.6, 16.2 and 23.1 us, by chunks 8.1, 15.8, 18.3, 16.2 and 16.3.
constexpr int kScanSerial = 32;
// Documents of few tokens, no more than 32 of them together or than there are documents, are walked by a wavefront each, which
// is what single tokens of many scenes want: 24, 64, 256 of 1024 channels 3.9, 3.9 and 4.2 us, by the rules above 14.5, 21.3 and
// 30.4. Lengths are not known here: if one document has all 256 tokens it takes 134 us for 39, and with
// 1024 documents 519 for 42 (single tokens 7.1 for 34), so that more than 256 go by chunks.
constexpr int kScanWalkers = 256;

struct ScanPlan {
  int chunks, parts, blocks, serial;
  size_t prefix, part;  // bytes
};
static ScanPlan scan_plan(int64_t tokens, int width) {
  ScanPlan s = {};
  s.chunks = static_cast<int>((tokens + kScanChunk - 1) / kScanChunk);
  s.serial = tokens <= kScanSerial;
  if (s.serial) {
    s.parts = 1;
    s.blocks = s.chunks;
    return s;
  }
  const int all = (s.chunks + kScanWaves - 1) / kScanWaves;
  s.blocks = (all + kScanParts - 1) / kScanParts;
  s.parts = (all + s.blocks - 1) / s.blocks;
  s.prefix = (static_cast<size_t>(s.chunks) * width * sizeof(float2) + 15) / 16 * 16;
  s.part = s.parts > 1 ? static_cast<size_t>(s.parts) * width * (sizeof(float2) + sizeof(float)) : 0;
  return s;
}

static int check_scan(const gs_gated_scan* p, void* workspace, size_t workspace_bytes, ScanArgs* a) {
  GS_REQUIRE(p, GS_ERR_ARG, "gated scan: args is NULL");
  GS_REQUIRE(row_type(p->dtype), GS_ERR_ARG, "gated scan: dtype must be GS_FLOAT32 or GS_BFLOAT16");
  GS_REQUIRE(p->tokens >= 0 && p->tokens < (int64_t(1) << 31), GS_ERR_ARG, "gated scan: invalid token count");
  GS_REQUIRE(p->width >= 1 && p->width <= GS_SCAN_MAX_WIDTH, GS_ERR_ARG, "gated scan: width %d: 1 to %d are provided",
             p->width, GS_SCAN_MAX_WIDTH);
  GS_REQUIRE(p->docs >= 1 && p->docs < (1 << 30) && (p->offsets || p->docs == 1), GS_ERR_ARG,
             "gated scan: at least one document, and offsets for more than one");
  GS_REQUIRE(p->tokens == 0 || (p->x && p->forget), GS_ERR_ARG, "gated scan: null pointer");
  const size_t es = row_type_bytes(p->dtype);
  GS_REQUIRE(aligned(p->x, es) && aligned(p->forget, es) && aligned(p->gate, es) && aligned(p->y, es) &&
                 aligned(p->initial, 4) && aligned(p->state, 4) && aligned(p->carry, 4) && aligned(p->offsets, 4) &&
                 aligned(workspace, 16), GS_ERR_ALIGN, "gated scan: misaligned tensor or workspace");
  const ScanPlan s = scan_plan(p->tokens, p->width);
  GS_REQUIRE((s.chunks + int64_t(kWalkWaves)) * ((p->width + kScanGroup - 1) / kScanGroup) < (int64_t(1) << 26), GS_ERR_ARG,
             "gated scan: too many elements");
  GS_REQUIRE(workspace_bytes >= s.prefix + s.part && (workspace || s.prefix == 0), GS_ERR_WORKSPACE,
             "gated scan: workspace too small");
  *a = {};
  a->x = p->x;
  a->f = p->forget;
  a->o = p->gate;
  a->initial = p->initial;
  a->y = p->y;
  a->state = p->state;
  a->carry = p->carry;
  a->offsets = p->offsets;
  a->tokens = p->tokens;
  a->x_stride = p->x_stride;
  a->f_stride = p->forget_stride;
  a->o_stride = p->gate_stride;
  a->docs = p->docs;
  a->width = p->width;
  a->reverse = p->reverse != 0;
  a->groups = (p->width + kScanGroup - 1) / kScanGroup;
  a->chunks = s.chunks;
  a->parts = s.parts;
  a->blocks = s.blocks;
  a->single = p->docs > 1 && p->docs <= kScanWalkers && (s.serial || p->tokens <= p->docs);
  a->serial = s.serial && !a->single;
  a->prefix = static_cast<float2*>(workspace);
  a->part = reinterpret_cast<float2*>(static_cast<char*>(workspace) + s.prefix);
  if (s.parts > 1) a->before = reinterpret_cast<float*>(a->part + static_cast<size_t>(s.parts) * p->width);
  return GS_OK;
}

template <typename T, bool BACK, bool SMALL, bool ONE>
static int run_walk(const ScanArgs& a, hipStream_t st) {
  const int walkers = ONE ? a.docs : (a.serial ? 1 : (a.chunks + kWalkWaves - 1) / kWalkWaves);
  const dim3 grid(static_cast<unsigned>(a.groups) * walkers), block(ONE || a.serial ? kWave : kWalkWaves * kWave);
  if constexpr (BACK) hipLaunchKernelGGL((scan_bwd_kernel<T, SMALL, ONE>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((scan_apply_kernel<T, SMALL, ONE>), grid, block, 0, st, a);
  return check_launch("gated scan");
}
template <typename T, bool BACK, bool SMALL>
static int run_scan(const ScanArgs& a, hipStream_t st) {
  if (a.single) return run_walk<T, BACK, SMALL, true>(a, st);
  if (!a.serial) {
    hipLaunchKernelGGL((scan_sums_kernel<T, BACK, SMALL>), dim3(a.groups, a.parts), dim3(kScanThreads), 0, st, a);
    if (const int rc = check_launch("gated scan (sums)")) return rc;
  }
  if (a.parts > 1) {
    hipLaunchKernelGGL(scan_parts_kernel, dim3((a.width + 31) / 32), dim3(kJoinThreads), 0, st, a);
    if (const int rc = check_launch("gated scan (parts)")) return rc;
  }
  return run_walk<T, BACK, SMALL, false>(a, st);
}

template <bool BACK>
static int run_scan(const ScanArgs& a, int dtype, hipStream_t st) {
  const bool small = a.width < kScanVec;
  if (dtype == GS_BFLOAT16) return small ? run_scan<__bf16, BACK, true>(a, st) : run_scan<__bf16, BACK, false>(a, st);
  return small ? run_scan<float, BACK, true>(a, st) : run_scan<float, BACK, false>(a, st);
}

}  // namespace gs

using namespace gs;

extern "C" int64_t gs_gated_scan_chunks(int64_t tokens) { return tokens <= 0 ? 0 : (tokens + kScanChunk - 1) / kScanChunk; }

extern "C" size_t gs_gated_scan_workspace_size(int64_t tokens, int width) {
  clear_error();
  if (tokens <= 0 || width <= 0) return 0;
  const ScanPlan s = scan_plan(tokens, width);
  return s.prefix + s.part;
}

extern "C" int gs_gated_scan_fwd(const gs_gated_scan* p, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  ScanArgs a;
  if (const int rc = check_scan(p, workspace, workspace_bytes, &a)) return rc;
  GS_REQUIRE(a.tokens == 0 || a.y, GS_ERR_ARG, "gated scan: null pointer");
  if (a.tokens == 0 && a.state == nullptr) return GS_OK;
  return run_scan<false>(a, p->dtype, as_stream(stream));
}

extern "C" int gs_gated_scan_bwd(const gs_gated_scan* p, const void* d_y, const float* d_state, void* d_x, void* d_forget,
                                 void* d_gate, float* d_initial, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  ScanArgs a;
  if (const int rc = check_scan(p, workspace, workspace_bytes, &a)) return rc;
  GS_REQUIRE(a.tokens == 0 || (a.carry && d_y), GS_ERR_ARG, "gated scan: the backward pass needs the carried states and d_y");
  GS_REQUIRE(a.o || !d_gate, GS_ERR_ARG, "gated scan: the gradient of a gate that is not there");
  const size_t es = row_type_bytes(p->dtype);
  GS_REQUIRE(aligned(d_y, es) && aligned(d_x, es) && aligned(d_forget, es) && aligned(d_gate, es) && aligned(d_state, 4) &&
                 aligned(d_initial, 4), GS_ERR_ALIGN, "gated scan: misaligned gradient");
  a.d_y = d_y;
  a.d_state = d_state;
  a.d_x = d_x;
  a.d_f = d_forget;
  a.d_o = d_gate;
  a.d_initial = d_initial;
  if (a.tokens == 0 && d_initial == nullptr) return GS_OK;
  return run_scan<true>(a, p->dtype, as_stream(stream));
}
