// The dropout masks of this library: 16 random bits per element from a counter-based generator, so
// that a mask is computed again wherever it is needed (forward, weight gradient, input gradient)
// and never stored.
//
// Generator: Philox-4x32 with ten rounds (Salmon, Moraes, Dror and Shaw, "Parallel random numbers:
// as easy as 1, 2, 3", SC 2011). For an element (r, c) of a matrix with C columns: the 128-bit block
// with counter (block's low word, high word, site, low word of key[1]) and the 64-bit key key[0],
// block = r ceil(C / 8) + c / 8; its halfword c % 8 (low half of word 0 first) is the element's 16 bits.
// The element is kept when they are at least `threshold` = round(p 2^16); kept values are
// multiplied by 2^16 / (2^16 - threshold), the reciprocal of the exact share that is kept. Eight
// columns are one 16-byte chunk of fp16 and one block of the generator.
//
// A round is two 32 x 32 -> 64-bit products (v_mad_u64_u32, a quarter of the VALU rate) and two
// three-operand exclusive ors.
#pragma once

#include "common.h"

namespace talm {
namespace {

struct DropArgs {
  const int64_t* key;  // [2], device memory (null: no dropout)
  uint32_t site;
  uint32_t threshold;  // 0: no dropout
};

struct DropKey {
  uint32_t k0, k1, word3, site, threshold;
  __device__ __forceinline__ DropKey(const int64_t* key, uint32_t site_, uint32_t threshold_)
      : k0(0), k1(0), word3(0), site(site_), threshold(threshold_) {
    if (threshold) {
      const uint64_t k = static_cast<uint64_t>(key[0]);
      k0 = static_cast<uint32_t>(k);
      k1 = static_cast<uint32_t>(k >> 32);
      word3 = static_cast<uint32_t>(key[1]);
    }
  }
};

__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
  return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);  // v_bitop3_b32 with the table of a ^ b ^ c
}

__device__ __forceinline__ uint4 philox_block(uint64_t block, const DropKey& d) {
  uint32_t c0 = static_cast<uint32_t>(block), c1 = static_cast<uint32_t>(block >> 32), c2 = d.site,
           c3 = d.word3, k0 = d.k0, k1 = d.k1;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = static_cast<uint64_t>(c0) * 0xD2511F53u, b = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = xor3(static_cast<uint32_t>(b >> 32), c1, k0);
    c1 = static_cast<uint32_t>(b);
    c2 = xor3(static_cast<uint32_t>(a >> 32), c3, k1);
    c3 = static_cast<uint32_t>(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// Two packed 16-bit values with the dropped ones cleared: `bits` is their word of the block.
__device__ __forceinline__ uint32_t keep2(uint32_t x, uint32_t bits, uint32_t threshold) {
  const uint32_t lo = (bits & 0xffffu) >= threshold ? 0xffffu : 0u;
  const uint32_t hi = (bits >> 16) >= threshold ? 0xffff0000u : 0u;
  return x & (lo | hi);
}
// Eight of them: the columns of block `r`.
__device__ __forceinline__ uint4 keep8(uint4 x, uint4 r, uint32_t threshold) {
  return make_uint4(keep2(x.x, r.x, threshold), keep2(x.y, r.y, threshold), keep2(x.z, r.z, threshold),
                    keep2(x.w, r.w, threshold));
}
// Bit e: column e of the block is kept.
__device__ __forceinline__ uint32_t keep_bits(uint4 r, uint32_t threshold) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
  uint32_t bits = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    bits |= ((e & 1 ? w[e >> 1] >> 16 : w[e >> 1] & 0xffffu) >= threshold ? 1u : 0u) << e;
  return bits;
}

inline uint32_t drop_threshold(float p) {
  const double t = static_cast<double>(p) * 65536.0 + 0.5;
  return t >= 65535.0 ? 65535u : static_cast<uint32_t>(t);
}
inline float drop_factor(uint32_t threshold) { return 65536.f / static_cast<float>(65536u - threshold); }

}  // namespace
}  // namespace talm
