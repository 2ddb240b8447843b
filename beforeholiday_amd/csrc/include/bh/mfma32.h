// Building blocks of the 32x32x16 MFMA attention kernels (gfx950): the matrix instruction, packing of
// accumulator registers into 16-bit operands, half-wave exchange, LDS-DMA through buffer resources, and the
// counter hash of attention dropout (the same function of (seed, head, query, key) in every kernel).
#pragma once

#include "bh/device.h"

namespace bh {
namespace m32 {

typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef float f4v __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef int i4v __attribute__((ext_vector_type(4)));
typedef int i2v __attribute__((ext_vector_type(2)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4v* lds_s4_ptr;

// D = A (32 x 16) . B (16 x 32) + C. Lane l holds A[l % 32][8 (l / 32) + 0..7] and B[8 (l / 32) + 0..7][l % 32];
// register i of the result is D[(i & 3) + 8 (i >> 2) + 4 (l / 32)][l % 32].
template <typename T> struct Mfma;
template <> struct Mfma<f16> {
  static BH_DEVICE f16v run(i4v a, i4v b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8v, a), __builtin_bit_cast(h8v, b), c, 0, 0, 0);
  }
};
template <> struct Mfma<bf16> {
  static BH_DEVICE f16v run(i4v a, i4v b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0,
                                                   0);
  }
};
BH_DEVICE f16v zero16() {
  f16v z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}
// accumulator register i <-> row offset inside the 32-row tile, without the lane's 4 (l / 32)
BH_HD constexpr int acc_row(int i) { return (i & 3) + 8 * (i >> 2); }

// registers 8u .. 8u+7 of an accumulator tile as a 16-bit operand (k = those 8 rows of each half-wave)
template <typename T> BH_DEVICE i4v pack8(const f16v& x, int u) {
  typedef T t8v __attribute__((ext_vector_type(8)));
  t8v v;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = from_f<T>(x[8 * u + j]);
  return __builtin_bit_cast(i4v, v);
}
template <typename T> BH_DEVICE void store4(T* dst, float a, float b, float c, float d) {
  typedef T t4v __attribute__((ext_vector_type(4)));
  *reinterpret_cast<t4v*>(dst) = t4v{from_f<T>(a), from_f<T>(b), from_f<T>(c), from_f<T>(d)};
}
// max / sum of a value over the two half-waves (lanes l and l ^ 32): one v_permlane32_swap
BH_DEVICE float half_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x),
                                                  false, false);
  return fmaxf(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
}
BH_DEVICE float half_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x),
                                                  false, false);
  return __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
}

// ---- LDS-DMA ---------------------------------------------------------------------------------------------
// One instruction moves 16 (4) bytes per lane from a buffer resource to LDS bytes [lds, lds + 1024 (256)),
// lane-linear; lanes whose offset is past the resource's end write zeros. Issued as inline asm because the
// compiler cannot tell the DMA's LDS writes from reads of the other buffer and would wait for every one of
// them; the kernels order them themselves (wait_vmcnt + barrier).
constexpr unsigned kRsrcWord3 = 0x00020000u;
constexpr int kOutOfRange = 0x7ffffff0;  // a lane offset past every resource made here
BH_DEVICE i4v make_rsrc(const void* base, uint32_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  return i4v{(int)(uint32_t)a, (int)((a >> 32) & 0xffff), (int)bytes, (int)kRsrcWord3};
}
BH_DEVICE unsigned lds_addr(const void* p) {
  typedef const __attribute__((address_space(3))) char* lds_cptr;
  return (unsigned)(uintptr_t)((lds_cptr)p);
}
BH_DEVICE void dma16(i4v rs, int voff, unsigned lds) {
  asm volatile(
      "s_mov_b32 m0, %1\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %0, %2, 0 offen lds" ::"v"(voff),
      "s"(lds), "s"(rs)
      : "memory", "m0");
}
BH_DEVICE void dma4(i4v rs, int voff, unsigned lds) {
  asm volatile(
      "s_mov_b32 m0, %1\n\t"
      "s_nop 0\n\t"
      "buffer_load_dword %0, %2, 0 offen lds" ::"v"(voff),
      "s"(lds), "s"(rs)
      : "memory", "m0");
}
template <int N> BH_DEVICE void wait_vmcnt() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
// this wave's LDS reads are done, then the workgroup barrier (nothing LDS moves across it)
BH_DEVICE void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// ---- attention dropout -----------------------------------------------------------------------------------
// A 32-bit avalanche hash of (seed, head, query) per row; per pair of keys a Weyl step, a fold, one 32-bit
// multiply and a fold: its low / high 16 bits decide about the even / odd key. No lane layout enters, so the
// kernels with the query on the lane and those with the key on the lane regenerate the same mask.
BH_DEVICE uint32_t mix32(uint32_t x) {
  x ^= x >> 16;
  x *= 0x7feb352du;
  x ^= x >> 15;
  x *= 0x846ca68bu;
  x ^= x >> 16;
  return x;
}
BH_DEVICE uint32_t row_hash(uint64_t seed, int bh, int q) {
  return mix32((uint32_t)seed ^
               mix32((uint32_t)(seed >> 32) ^ ((uint32_t)bh * 0x9E3779B1u) ^ ((uint32_t)q * 0x85EBCA77u)));
}
BH_DEVICE uint32_t fold16(uint32_t x) { return x ^ (x >> 16); }
// the pair's hash before its last fold: keep16(fold16(x), t) is the even key's decision, x < t << 16 the odd one's
BH_DEVICE uint32_t pair_hash(uint32_t rowh, int k) {
  return fold16(rowh + (uint32_t)(k >> 1) * 0x9E3779B9u) * 0x7feb352du;
}
BH_DEVICE bool keep16(uint32_t x, uint32_t thresh) { return (uint16_t)x < (uint16_t)thresh; }  // thresh <= 65535
BH_DEVICE bool keep_even(uint32_t x, uint32_t thresh) { return keep16(fold16(x), thresh); }
BH_DEVICE bool keep_odd(uint32_t x, uint32_t thresh) { return x < thresh << 16; }

}  // namespace m32
}  // namespace bh
