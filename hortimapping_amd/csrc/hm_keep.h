// Counter-based keep decisions of dropout (hm_dropout.hip) and of the dropout on the input of low-rank adapters
// (hm_adapter.hip), and the element types that both take.
//
// Generator: Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011).
//   key     = (low, high word of the seed)
//   counter = (column / 8, row low, row high, tag)
// One call gives four 32-bit words = eight 16-bit draws (word j / 2, low half first) for the eight columns of one block, so
// that a lane that holds eight consecutive values of a row needs ONE call, and a decision depends on (seed, tag, row, column)
// alone: not on the number of columns, the strides, the launch or the kernel that asks.  A value is kept where its draw is
// >= threshold = round(65536 p).  16 bits instead of 32 per draw halve the cost of the generator (20 wide products per call);
// the price is that p is taken to the nearest 1 / 65536, and the factor of what is kept is 65536 / (65536 - threshold), that
// of the p actually used, so the expectation of the output is exact.
#pragma once
#include "hm_common.h"

namespace hm {

struct KeepArgs {
  uint64_t seed;
  const uint64_t* d_seed;   // optional device word added to seed: what a captured graph changes between replays
  uint64_t row0;            // row number of the first row of the call
  uint32_t tag;
  uint32_t threshold;       // 0 .. 65536
  float up;                 // 65536 / (65536 - threshold), 0 at p = 1
};

// false: p is not in [0, 1] (a NaN included)
inline bool keep_args(KeepArgs* k, double p, unsigned long long seed, const unsigned long long* d_seed, unsigned tag,
                      unsigned long long row0) {
  if (!(p >= 0.0 && p <= 1.0)) return false;
  uint32_t thr = (uint32_t)(p * 65536.0 + 0.5);
  if (thr == 65536 && p < 1.0) thr = 65535;        // 1 - 2^-17 < p < 1: something is kept
  k->seed = seed;
  k->d_seed = reinterpret_cast<const uint64_t*>(d_seed);
  k->row0 = row0;
  k->tag = tag;
  k->threshold = thr;
  k->up = thr == 65536 ? 0.f : (float)(65536.0 / (65536 - thr));
  return true;
}

struct KeepKey { uint32_t k0, k1; };

__device__ __forceinline__ KeepKey keep_key(const KeepArgs& a) {
  uint64_t s = a.seed;
  if (a.d_seed != nullptr) s += *a.d_seed;
  return {(uint32_t)s, (uint32_t)(s >> 32)};
}

// bit j: column 8 * block + j of `row` (counted from the first row of the call) is kept
__device__ __forceinline__ uint32_t keep8(const KeepArgs& a, KeepKey key, uint64_t row, uint32_t block) {
  row += a.row0;
  uint32_t c0 = block, c1 = (uint32_t)row, c2 = (uint32_t)(row >> 32), c3 = a.tag, k0 = key.k0, k1 = key.k1;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)p1;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  const uint32_t w[4] = {c0, c1, c2, c3};
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m |= (uint32_t)(((w[j >> 1] >> (16 * (j & 1))) & 0xffffu) >= a.threshold) << j;
  return m;
}

// ---- element types: HM_TYPE_F32 / F16 / BF16 of the public header.  Arithmetic is in 32 bits; a result is rounded once
// (to nearest even) where it is stored.
typedef __bf16 bf16;
typedef _Float16 f16;

template <typename T> struct alignas(sizeof(T)) Pack8 { T v[8]; };     // eight values at the alignment of one

// eight consecutive values in one or two 16-byte accesses whatever the alignment (global memory takes any here)
template <typename T> __device__ __forceinline__ void load8(float* o, const T* p) {
  const Pack8<T> u = *reinterpret_cast<const Pack8<T>*>(p);
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = (float)u.v[j];
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float* v) {
  Pack8<T> u;
#pragma unroll
  for (int j = 0; j < 8; ++j) u.v[j] = (T)v[j];
  *reinterpret_cast<Pack8<T>*>(p) = u;
}

}  // namespace hm
