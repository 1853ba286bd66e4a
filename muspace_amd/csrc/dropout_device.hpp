// Dropout from a counter-based generator, shared by dropout and the residual norm
// (include/muspace_layer.h): whether element i of a tensor is kept follows from
// (seed, offset, i) alone, so that the mask is computed where it is needed, in the
// forward and again in the backward, and is stored nowhere.
//
// The generator is Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", 2011): ten rounds of two 32 x 32 -> 64 bit products over
// a counter of four words under a key of two. Counter (i / 4, offset), key seed; its
// four words are those of elements i to i + 3. An element is kept if its word is at or
// over p 2^32: probabilities are exact to 2^-32, at four elements a call. A round is
// two v_mad_u64_u32 at a quarter of the vector unit's rate: 1.1e12 elements a second,
// just above what 16-bit tensors can be read and written at.
#pragma once

#include "linear_device.hpp"

namespace dense {

struct Drop {
  uint64_t seed, offset;
  const int64_t *device_seed;  // read by the kernel in place of seed (0: none)
  uint32_t last;               // the largest word that is dropped
  float scale;                 // 1 / (1 - p)
  int on;                      // 0: every element is kept
};

__device__ __forceinline__ uint64_t seed_of(const Drop &d) {
  return d.device_seed != nullptr ? static_cast<uint64_t>(*d.device_seed) : d.seed;
}

__device__ __forceinline__ u32x4 philox(uint64_t counter, uint64_t offset, uint64_t seed) {
  uint32_t c0 = static_cast<uint32_t>(counter), c1 = static_cast<uint32_t>(counter >> 32);
  uint32_t c2 = static_cast<uint32_t>(offset), c3 = static_cast<uint32_t>(offset >> 32);
  uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
  for (int round = 0; round < 10; ++round) {
    const uint64_t p0 = static_cast<uint64_t>(c0) * 0xD2511F53u;
    const uint64_t p1 = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(p1);
    c2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(p0);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return u32x4{c0, c1, c2, c3};
}

// Bit e: element `index` + e is kept, e in 0..kCount - 1 (kCount a multiple of four).
template <int kCount>
__device__ __forceinline__ uint32_t kept_bits(const Drop &d, uint64_t seed, int64_t index) {
  const uint64_t counter = static_cast<uint64_t>(index) >> 2;
  const uint32_t skip = static_cast<uint32_t>(index) & 3u;
  uint32_t bits = 0;
#pragma unroll
  for (int j = 0; j <= kCount / 4; ++j) {
    if (j == kCount / 4 && skip == 0) break;  // elements that start a counter's words
    const u32x4 w = philox(counter + j, d.offset, seed);
#pragma unroll
    for (int e = 0; e < 4; ++e) bits |= (w[e] > d.last ? 1u : 0u) << (4 * j + e);
  }
  return bits >> skip;
}

// A tensor's elements by chunks: out = kept ? x scale : 0, plus the residual. x is not
// read as a factor where it is dropped: an infinity or NaN there is gone. Two chunks a
// thread are in flight; the last, short chunk is read value by value.
template <typename T>
__global__ __launch_bounds__(kThreads) void dropout_elements(const T *x, const T *residual, T *out,
                                                             int64_t count, const Drop d) {
  constexpr int kV = Piece<T>::kValues;
  constexpr int kAhead = 2;
  const uint64_t seed = seed_of(d);
  const int64_t chunks = (count + kV - 1) / kV;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  auto finish = [&](int64_t at, const u32x4 &xv, const u32x4 &rv, int left) {
    float v[kV], r[kV];
    unpack<T>(xv, v);
    const uint32_t bits = d.on ? kept_bits<kV>(d, seed, at) : ~0u;
#pragma unroll
    for (int e = 0; e < kV; ++e) v[e] = (bits >> e) & 1u ? v[e] * d.scale : 0.0f;
    if (residual != nullptr) {
      unpack<T>(rv, r);
#pragma unroll
      for (int e = 0; e < kV; ++e) v[e] += r[e];
    }
    loose_store(out + at, pack<T>(v), left);
  };
  int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  for (; i + (kAhead - 1) * step < count / kV; i += kAhead * step) {
    u32x4 xv[kAhead], rv[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int64_t at = (i + a * step) * kV;
      xv[a] = reinterpret_cast<const Loose16 *>(x + at)->v;
      rv[a] = u32x4{0, 0, 0, 0};
      if (residual != nullptr) rv[a] = reinterpret_cast<const Loose16 *>(residual + at)->v;
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a) finish((i + a * step) * kV, xv[a], rv[a], kV);
  }
  for (; i < chunks; i += step) {
    const int64_t at = i * kV;
    const int left = static_cast<int>(count - at < kV ? count - at : kV);
    finish(at, loose_load<T>(x + at, left),
           residual != nullptr ? loose_load<T>(residual + at, left) : u32x4{0, 0, 0, 0}, left);
  }
}

}  // namespace dense
