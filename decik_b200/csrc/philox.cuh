// The counter-based generator of the dropout kernels: Philox4x32 with 7 rounds (Salmon, Moraes, Dror,
// Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011: 7 is the fewest rounds that pass
// BigCrush). One call gives the 8 16-bit lanes of 8 consecutive values:
//   key = seed, counter = (group, offset + stream), group = index / 8,
//   lane j of a group = the (j % 2)-th half (low first) of word j / 2,
//   keep value j iff lane >= cut, cut = floor(p 65536 + 1/2); kept values are scaled by
//   65536 / (65536 - cut), so that the expectation is exact for the p that the 16 bits can hold.
// A mask is therefore a function of (seed, offset + stream, index): it is never stored.
#pragma once

#include <cmath>

#include "common.cuh"

namespace decik {
namespace philox {

struct Key {
  uint32_t k0, k1, o0, o1;  // seed, offset + stream
};

// The key is the same in every lane. Broadcasting it says so: its schedule then lives in uniform
// registers, where the 12 additions of a call's rounds were vector instructions before (an eighth of
// all that the LoRA kernels execute).
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }

__device__ __forceinline__ Key make_key(const int64_t* __restrict__ rng, int64_t stream_id) {
  const unsigned long long seed = static_cast<unsigned long long>(__ldg(reinterpret_cast<const long long*>(rng)));
  const unsigned long long off = static_cast<unsigned long long>(__ldg(reinterpret_cast<const long long*>(rng) + 1)) +
                                 static_cast<unsigned long long>(stream_id);
  return {uniform(static_cast<uint32_t>(seed)), uniform(static_cast<uint32_t>(seed >> 32)),
          uniform(static_cast<uint32_t>(off)), uniform(static_cast<uint32_t>(off >> 32))};
}

// the four words of group g
__device__ __forceinline__ uint4 words(const Key& k, unsigned long long g) {
  uint32_t c0 = static_cast<uint32_t>(g), c1 = static_cast<uint32_t>(g >> 32), c2 = k.o0, c3 = k.o1;
  uint32_t k0 = k.k0, k1 = k.k1;
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const unsigned long long p0 = static_cast<unsigned long long>(c0) * 0xD2511F53u;
    const unsigned long long p1 = static_cast<unsigned long long>(c2) * 0xCD9E8D57u;
    const uint32_t n0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ k0, n2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ k1;
    c1 = static_cast<uint32_t>(p1);
    c3 = static_cast<uint32_t>(p0);
    c0 = n0;
    c2 = n2;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// keep of lane j (0..7); cut_hi = cut << 16, or with cut = 65536 (p = 1) never
__device__ __forceinline__ bool keep_lane(const uint4& w, int j, uint32_t cut) {
  const uint32_t v = j < 2 ? w.x : j < 4 ? w.y : j < 6 ? w.z : w.w;
  return ((j & 1) ? v >> 16 : v & 0xFFFFu) >= cut;
}

// host: the cut of a probability (0..65536) and the kept values' scale (0 when nothing is kept)
inline uint32_t cut_of(double p) { return static_cast<uint32_t>(std::floor(p * 65536.0 + 0.5)); }
inline float scale_of(uint32_t cut) {
  return cut >= 65536u ? 0.f : static_cast<float>(65536.0 / (65536.0 - static_cast<double>(cut)));
}
inline bool valid_p(double p) { return p >= 0.0 && p <= 1.0; }  // false for NaN

}  // namespace philox
}  // namespace decik
