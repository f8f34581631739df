// Device helpers of the kernels of libqf_kv4.so: the 4-bit cache's records (include/qf_kv4.h).
#ifndef QF_KV4_COMMON_H
#define QF_KV4_COMMON_H

#include "qf_block_common.h"
#include "qf_kv4.h"
#include "qf_kv4_places.h"

#include <algorithm>
#include <atomic>

namespace qfk {

using namespace qfb;

constexpr int kGroup = 32;  // values that share a scale

// Division of 0 <= n < 2^31 by an invariant d >= 1 (Granlund and Montgomery, PLDI 1994): with l = ceil(log2 d) and
// m = ceil(2^(31 + l) / d), which has 32 bits, floor(n / d) = (n * m) >> (31 + l).
struct Divisor {
  uint32_t m;
  int shift;  // l
};
inline Divisor divisor(int d) {
  int l = 0;
  while (((int64_t)1 << l) < d) ++l;
  return Divisor{(uint32_t)((((uint64_t)1 << (31 + l)) + d - 1) / d), l};
}
__device__ __forceinline__ int divide(int n, Divisor d) { return (int)(((uint64_t)(uint32_t)n * d.m) >> (31 + d.shift)); }

inline int compute_units() {  // of the current device
  static std::atomic<int> cus[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  int n = cus[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n < 1) n = 256;
    cus[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// Offsets in a record of 16 positions of a head of D values.
template <int D>
struct Record {
  static constexpr int kWidth = (D < 128 ? D : 128) / 16;  // neighbouring values of a lane's byte run
  static constexpr int kHalves = D / (16 * kWidth);
  static constexpr int kValues = 8 * D, kKeyScales = 16 * D, kValueScales = 16 * D + D / 2, kBytes = 17 * D;
  __device__ static __forceinline__ int key(int p, int d) { return p * (D / 2) + d / 2; }  // of the byte that holds value d
  __device__ static __forceinline__ int value(int p, int d) {
    const int h = d / (16 * kWidth), c = d % (16 * kWidth) / kWidth, n = d % kWidth;
    return kValues + h * (128 * kWidth) + ((p / 4 * 16 + c) * 4 + p % 4) * (kWidth / 2) + n / 2;
  }
  __device__ static __forceinline__ int key_scale(int p, int d) { return kKeyScales + d / kGroup * kTile + p; }
  __device__ static __forceinline__ int value_scale(int p, int d) { return kValueScales + d / kGroup * kTile + p; }
};

// Byte I of a dword of scale bytes where a conversion looks for its scale: it reads the exponent of an fp32 alone (measured: the
// sign and the mantissa change nothing, and the exponent 255 gives NaN), so the bits around it may stay.
template <int I>
__device__ __forceinline__ float scale_of(uint32_t w) {
  return __uint_as_float(I < 3 ? w << (23 - 8 * I) : w >> 1);
}

// Two codes (byte B of w) times a scale as two bf16, the low nibble's in the low half.
template <int B>
__device__ __forceinline__ uint32_t widen2(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, B));
}
// Four dwords of bf16 from a dword of 8 codes.
__device__ __forceinline__ u32x4_t widen8(uint32_t w, float scale) {
  return u32x4_t{widen2<0>(w, scale), widen2<1>(w, scale), widen2<2>(w, scale), widen2<3>(w, scale)};
}

}  // namespace qfk

#endif
