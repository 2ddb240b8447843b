// Dropout whose mask is never stored (gfx950): element i is kept when word i % 4 of Philox4x32 with 7 rounds
// (Salmon, Moraes, Dror, Shaw 2011: the fewest rounds of this width that passed all their tests), counter i / 4,
// key = the seed, is below (1 - p) 2^32. The backward pass is the same call on the gradient.
//
// Memory bound: 2 + 2 (4 + 4) bytes a value; a Philox call is 14 32x32-bit products for 4 values.
#include "bh/api.h"
#include "bh/device.h"
#include "bh/qk_rope_api.h"

#include <algorithm>
#include <stdexcept>
#include <string>

namespace bh {
namespace {

constexpr int kThreads = 256;

BH_DEVICE uint4 philox7(uint64_t seed, uint64_t ctr) {
  uint4 c = make_uint4((uint32_t)ctr, (uint32_t)(ctr >> 32), 0u, 0u);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint64_t p0 = (uint64_t)c.x * 0xD2511F53u, p1 = (uint64_t)c.z * 0xCD9E8D57u;
    c = make_uint4((uint32_t)(p1 >> 32) ^ c.y ^ k0, (uint32_t)p1, (uint32_t)(p0 >> 32) ^ c.w ^ k1, (uint32_t)p0);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return c;
}

// a thread takes 8 neighbouring values (two counters) a step
template <typename T>
__global__ __launch_bounds__(kThreads) void k_counter_dropout(const T* x, T* y, int64_t n, uint32_t thresh, float scale,
                                                              uint64_t seed, const int64_t* __restrict__ seed_dev,
                                                              bool aligned) {
  if (seed_dev) seed ^= (uint64_t)*seed_dev * 0x9E3779B97F4A7C15ull;
  const int64_t step = (int64_t)gridDim.x * kThreads * kVec;
  for (int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * kVec; i < n; i += step) {
    float r[kVec];
    load_vec<T>(x, i, n, aligned, r);
    const uint4 a = philox7(seed, (uint64_t)i >> 2), b = philox7(seed, ((uint64_t)i >> 2) + 1);
    const uint32_t u[kVec] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int k = 0; k < kVec; ++k) r[k] = u[k] < thresh ? r[k] * scale : 0.f;
    store_vec<T>(y, i, n, aligned, r);
  }
}

}  // namespace

void counter_dropout(int dt, const void* x, void* y, int64_t n, uint32_t thresh, float scale, uint64_t seed,
                     const int64_t* seed_dev, hipStream_t st) {
  if (n <= 0) return;
  const bool aligned = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 15) == 0;
  const int64_t per = (int64_t)kThreads * kVec;
  const unsigned grid = (unsigned)std::min<int64_t>((n + per - 1) / per, 256 * 32);
#define BH_DROP(T)                                                                                             \
  hipLaunchKernelGGL((k_counter_dropout<T>), dim3(grid), dim3(kThreads), 0, st, reinterpret_cast<const T*>(x), \
                     reinterpret_cast<T*>(y), n, thresh, scale, seed, seed_dev, aligned)
  switch (dt) {
    case kF32: BH_DROP(float); break;
    case kF16: BH_DROP(f16); break;
    case kBF16: BH_DROP(bf16); break;
    default: throw std::runtime_error("counter_dropout: fp32 / fp16 / bf16 only");
  }
#undef BH_DROP
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) throw std::runtime_error(std::string("counter_dropout: ") + hipGetErrorString(e));
}

}  // namespace bh
