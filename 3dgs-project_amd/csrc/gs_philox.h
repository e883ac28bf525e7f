// Random bits for dropout from a counter, so that a mask is never stored: the backward pass, or a replayed
// graph, forms the same bits again from the seed.
//
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011): ten
// rounds of two 32x32 -> 64 bit products under a key that grows by Weyl constants. Here the key is the 64-bit
// seed and the counter (column / 8, row, draw low, draw high), so that eight neighbouring elements of a row,
// one 16-byte vector of bfloat16, share one call: element j takes half j % 2 (low first) of word j / 2, 16
// bits, and is dropped where these are below the threshold. The probability is a multiple of 2^-16 and the kept
// elements' factor goes by that multiple, so the expectation is exact. (With 32 bits an element, two calls for eight,
// dropout alone over 8203 x 4096 in bfloat16 took 28.7 us, with 16 it takes 22.5.)
#pragma once

#include <stdint.h>

#include "gs_host.h"

namespace gs {

struct DropRule {
  const int64_t* seed_at;  // device memory, or NULL
  uint64_t seed, draw;
  uint32_t threshold;      // of 2^16; 0: nothing is dropped
  float factor;            // of what is kept
};

// The key, the same in every lane.
__device__ __forceinline__ uint64_t seed_of(const DropRule& d) {
  return d.seed_at ? static_cast<uint64_t>(*d.seed_at) : d.seed;
}

// Factors of elements 8 group .. 8 group + 7 of a row.
__device__ __forceinline__ void keep8(const DropRule& d, uint64_t seed, uint32_t row, uint32_t group, float (&f)[8]) {
  uint32_t c0 = group, c1 = row, c2 = static_cast<uint32_t>(d.draw), c3 = static_cast<uint32_t>(d.draw >> 32);
  uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = static_cast<uint64_t>(c0) * 0xD2511F53u, b = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(b);
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  const uint32_t w[4] = {c0, c1, c2, c3};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f[2 * j] = (w[j] & 0xffffu) >= d.threshold ? d.factor : 0.0f;
    f[2 * j + 1] = (w[j] >> 16) >= d.threshold ? d.factor : 0.0f;
  }
}

// The rule of a probability 0 <= p < 1, which is rounded to a multiple of 2^-16 (at most 1 - 2^-16).
inline DropRule drop_rule(double p, const int64_t* seed_at, uint64_t seed, uint64_t draw) {
  uint32_t t = static_cast<uint32_t>(p * 65536.0 + 0.5);
  if (t > 65535u) t = 65535u;
  return {seed_at, seed, draw, t, static_cast<float>(65536.0 / (65536.0 - t))};
}

}  // namespace gs
