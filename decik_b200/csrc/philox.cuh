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

constexpr int kRounds = 7;

// The keys of the rounds, the same for every mask of a seed.
struct Key {
  uint32_t k[kRounds][2];
};
// A stream's half of the counter, offset + stream.
struct Stream {
  uint32_t lo, hi;
};

// Broadcasting a value that is the same in every lane tells the compiler so, and keeps it from computing
// the value again at each use: with the schedule left to it, its 12 additions came back in every call
// (an eighth of all that the LoRA kernels executed).
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }

__device__ __forceinline__ Key make_key(const int64_t* __restrict__ rng) {
  const unsigned long long seed = static_cast<unsigned long long>(__ldg(reinterpret_cast<const long long*>(rng)));
  Key key;
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    key.k[r][0] = uniform(static_cast<uint32_t>(seed) + r * 0x9E3779B9u);
    key.k[r][1] = uniform(static_cast<uint32_t>(seed >> 32) + r * 0xBB67AE85u);
  }
  return key;
}
__device__ __forceinline__ Stream make_stream(const int64_t* __restrict__ rng, int64_t stream_id) {
  const unsigned long long off = static_cast<unsigned long long>(__ldg(reinterpret_cast<const long long*>(rng) + 1)) +
                                 static_cast<unsigned long long>(stream_id);
  return {uniform(static_cast<uint32_t>(off)), uniform(static_cast<uint32_t>(off >> 32))};
}

// the four words of group g
__device__ __forceinline__ uint4 words(const Key& key, const Stream& o, unsigned long long g) {
  uint32_t c0 = static_cast<uint32_t>(g), c1 = static_cast<uint32_t>(g >> 32), c2 = o.lo, c3 = o.hi;
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const unsigned long long p0 = static_cast<unsigned long long>(c0) * 0xD2511F53u;
    const unsigned long long p1 = static_cast<unsigned long long>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ key.k[r][0];
    c2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ key.k[r][1];
    c1 = static_cast<uint32_t>(p1);
    c3 = static_cast<uint32_t>(p0);
  }
  return make_uint4(c0, c1, c2, c3);
}

// keep of lane j (0..7)
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
