// Counter-based random bits for dropout: Philox4x32 with seven rounds (Salmon, Moraes, Dror, Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", SC 2011; seven rounds are the fewest that the authors found to pass BigCrush).
//
// Every dropout of this library uses one map from places to bits, so no mask is ever stored and any kernel can ask for
// any place again: column c of row r (all leading dimensions counted as one) takes bits 16 * (c & 7) .. + 15 of the
// 128-bit output at counter (c >> 3, r mod 2^32, r >> 32, 0), keyed by the 64-bit seed, and is dropped where that
// number is below the threshold round(p * 65536). Eight neighbouring columns cost one evaluation: 28 products, about
// 60 instructions. The threshold is below 65536 (the callers refuse p that rounds to 1).
#pragma once
#include <stdint.h>

namespace philox {

struct Seed {
  const unsigned long long* ptr;  // device memory, or null: `value`
  unsigned long long value;
};

__device__ __forceinline__ uint2 load_key(const Seed& s) {
  const unsigned long long v = s.ptr ? __ldg(s.ptr) : s.value;
  return make_uint2(static_cast<uint32_t>(v), static_cast<uint32_t>(v >> 32));
}

__device__ __forceinline__ uint4 words(uint32_t group, unsigned long long row, uint2 key) {
  uint32_t c0 = group, c1 = static_cast<uint32_t>(row), c2 = static_cast<uint32_t>(row >> 32), c3 = 0;
  uint32_t k0 = key.x, k1 = key.y;
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const unsigned long long a = static_cast<unsigned long long>(c0) * 0xD2511F53u;
    const unsigned long long b = static_cast<unsigned long long>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(b);
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// f[j] = f[j] * scale where column 8 * group + j of the row is kept, 0 where it is dropped
__device__ __forceinline__ void apply8(float (&f)[8], uint32_t group, unsigned long long row, uint2 key,
                                       uint32_t threshold, float scale) {
  const uint4 w = words(group, row, key);
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f[2 * j] = (u[j] & 0xffffu) >= threshold ? f[2 * j] * scale : 0.f;
    f[2 * j + 1] = (u[j] >> 16) >= threshold ? f[2 * j + 1] * scale : 0.f;
  }
}

// whether column j of the eight is kept; high = threshold << 16
__device__ __forceinline__ bool keeps(const uint4& w, int j, uint32_t high) {
  const uint32_t u = j < 2 ? w.x : (j < 4 ? w.y : (j < 6 ? w.z : w.w));
  return (j & 1 ? u : u << 16) >= high;
}

}  // namespace philox
