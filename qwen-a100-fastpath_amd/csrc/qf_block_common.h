// Device helpers shared by the kernels of libqf_block.so (gfx950).
#ifndef QF_BLOCK_COMMON_H
#define QF_BLOCK_COMMON_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>

#include "qf_block.h"

namespace qfb {

constexpr int kWave = 64;

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// bf16 <-> fp32 on 32-bit words (element order: low half first)
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ float bf16_f32(uint16_t h) { return __uint_as_float((uint32_t)h << 16); }
// two fp32 -> two bf16 (round to nearest even), `a` in the low half
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{a, b}), bf16x2_t));
}
__device__ __forceinline__ void unpack8(u32x4_t v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = bf16_lo(v[i]);
    f[2 * i + 1] = bf16_hi(v[i]);
  }
}
__device__ __forceinline__ u32x4_t pack8(const float (&f)[8]) {
  u32x4_t v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = pack_bf16(f[2 * i], f[2 * i + 1]);
  return v;
}

// Lane v of a DPP permutation of x (lanes without a source give 0).
template <int CTRL>
__device__ __forceinline__ float dpp_f32(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, false));
}
// Sum over groups of L lanes (8, 16, 32 or 64), the same in each lane of a group: rotations within rows of 16 lanes, then
// the wider exchanges.  Every lane of the wavefront active.
template <int L>
__device__ __forceinline__ float group_sum(float v) {
  v += dpp_f32<0xB1>(v);   // quad_perm 1 0 3 2
  v += dpp_f32<0x4E>(v);   // quad_perm 2 3 0 1
  v += dpp_f32<0x141>(v);  // row_half_mirror: the other quad of 8 lanes
  if constexpr (L >= 16) v += dpp_f32<0x140>(v);  // row_mirror: the other 8 of 16 lanes
  if constexpr (L >= 32) v += __shfl_xor(v, 16);
  if constexpr (L >= 64) v += __shfl_xor(v, 32);
  return v;
}

template <int L>
__device__ __forceinline__ float group_max(float v) {  // NaN only where every value is
  v = fmaxf(v, dpp_f32<0xB1>(v));
  v = fmaxf(v, dpp_f32<0x4E>(v));
  v = fmaxf(v, dpp_f32<0x141>(v));
  if constexpr (L >= 16) v = fmaxf(v, dpp_f32<0x140>(v));
  if constexpr (L >= 32) v = fmaxf(v, __shfl_xor(v, 16));
  if constexpr (L >= 64) v = fmaxf(v, __shfl_xor(v, 32));
  return v;
}

// Inclusive scan of sums over the wavefront's 64 lanes (every lane active).
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8: within 16 lanes
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast 15: row 0 into 1, row 2 into 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast 31: rows 0, 1 into 2, 3
  return v;
}
// Maximum over groups of 16 or all 64 lanes, the same in each lane of a group.
template <int L>
__device__ __forceinline__ uint32_t group_max_u32(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, false));
  if constexpr (L == 64) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false));  // rows 1 and 3 with the rows before
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false));  // rows 2 and 3 with row 1
    v = (uint32_t)__builtin_amdgcn_readlane((int)v, kWave - 1);
  }
  return v;
}

// 16 e4m3 values (a lane's bytes of a weight fragment) as two fragments of 8 bf16; exact (v_cvt_scalef32_pk_bf16_fp8).
__device__ __forceinline__ void widen16(u32x4_t v, bf16x8_t& lo, bf16x8_t& hi) {
  u32x4_t a, b;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    a[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[i], 1.f, false));
    a[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[i], 1.f, true));
    b[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 + i], 1.f, false));
    b[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 + i], 1.f, true));
  }
  lo = __builtin_bit_cast(bf16x8_t, a);
  hi = __builtin_bit_cast(bf16x8_t, b);
}

// s_waitcnt with vmcnt = N and the other counters unconstrained.
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0F70);
}

// 32-bit LDS address of a pointer into the workgroup's LDS
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

// A pointer that is the same in every lane, in scalar registers.
__device__ __forceinline__ const uint8_t* scalar_ptr(const uint8_t* p) {
  const uint64_t v = (uint64_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)v);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32));
  return (const uint8_t*)(((uint64_t)hi << 32) | lo);
}

// A 32-bit lane offset whose extension to an address is done here: a load then takes a scalar base and this register.
__device__ __forceinline__ uint32_t here(uint32_t offset) {
  asm volatile("" : "+v"(offset));
  return offset;
}

// Every wavefront is done with the reads before; the copies that it makes visible are those waited for.
__device__ __forceinline__ void ring_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" : : : "memory");
}

// A block of K of one weight tile times its token fragments, from zero.  `second` (the block has its second half) is the same
// in all lanes; matrix instructions run whatever the lane mask is, so the branch has to be a scalar one.
__device__ __forceinline__ f32x4_t block_product(const u32x4_t (&w)[2], const u32x4_t (&x)[2][2], bool second) {
  f32x4_t blk = {0.f, 0.f, 0.f, 0.f};
  bf16x8_t lo, hi;
  widen16(w[0], lo, hi);
  blk = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo, __builtin_bit_cast(bf16x8_t, x[0][0]), blk, 0, 0, 0);
  blk = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi, __builtin_bit_cast(bf16x8_t, x[0][1]), blk, 0, 0, 0);
  if (__builtin_amdgcn_readfirstlane(second)) {
    widen16(w[1], lo, hi);
    blk = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo, __builtin_bit_cast(bf16x8_t, x[1][0]), blk, 0, 0, 0);
    blk = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi, __builtin_bit_cast(bf16x8_t, x[1][1]), blk, 0, 0, 0);
  }
  return blk;
}

__device__ __forceinline__ u32x4_t load_once(const uint8_t* p) {  // read once: not kept in the caches
  return __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p));
}

constexpr int kDefaultLds = 64 * 1024;  // of a workgroup, static and dynamic

// Lets `fn` have `bytes` of dynamic LDS on the current device; `raised` holds the devices where it has.  Called where static
// and dynamic LDS together may pass kDefaultLds.
inline bool raise_lds(const void* fn, int bytes, std::atomic<uint64_t>& raised) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return false;
  const uint64_t bit = dev < 64 ? (uint64_t)1 << dev : 0;
  if (bit & raised.load(std::memory_order_relaxed)) return true;
  if (hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) return false;
  raised.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

// A launch's threads along x: below 2^32.
inline bool grid_fits(int64_t groups, int threads) { return groups * threads <= 0xffffffffll; }

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

}  // namespace qfb

#endif
