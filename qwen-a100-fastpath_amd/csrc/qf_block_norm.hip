// qf_block_norm.hip — the norms before and after a block, fused with the block's gate and residual scale (gfx950).
//
//   p = x * rsqrt(mean(x^2) + eps) * (offset + w_post)      (p = x without w_post)
//   y = residual + alpha * act(gate) * p
//   h = y * rsqrt(mean(y^2) + eps) * (offset + w_pre)
//
// One pass: a row's values are read once into registers, 16 bytes a lane and piece, the two sums of squares meet by DPP
// (and through LDS where a row spans wavefronts), and y (before its rounding) feeds the second norm from registers.  All
// arithmetic is fp32 in a fixed order, each output rounded once.  Bound by memory: 8 bytes a value with a bf16 residual,
// 12 with fp32, 2 more with a gate a value.  Measured: 2048 x 5120, fp32 residual, 24 us (5.2 TB/s, a large copy's rate; 28
// and 4.4 TB/s where the rows come from HBM); 8191 x 2568 with a gate a value 35 us (6.0 TB/s; 37 and 5.7); one row of 5120
// 3.1 us, a launch and three trips to memory and LDS.
#include "qf_block_common.h"

namespace qfb {

struct NormArgs {
  const uint16_t* x;
  int64_t ldx;
  const void* residual;
  int64_t ldr;
  const uint16_t* w_post;
  const uint16_t* w_pre;
  const uint16_t* gate;
  int64_t ldg;
  void* y;
  int64_t ldy;
  uint16_t* h;
  int64_t ldh;
  int M, N, pieces;  // pieces = N / 8
  int gate_kind, sigmoid;
  float offset, alpha, eps, inv_n;
};

// 1 / (1 + exp(-g)): exp2 and the reciprocal are good to an ulp each, the product with log2 e adds |g| half ulps.
__device__ __forceinline__ float sigmoid(float g) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.4426950408889634f));
}

// Sum over a row's threads of their shares of the mean: groups of L lanes, or (L = 0) the whole workgroup.
template <int L>
__device__ __forceinline__ float row_sum(float v, float* exchange) {
  if constexpr (L > 0) return group_sum<L>(v);
  v = group_sum<64>(v);
  const int waves = blockDim.x / kWave;
  if (waves == 1) return v;
  if ((threadIdx.x & (kWave - 1)) == 0) exchange[threadIdx.x / kWave] = v;
  __syncthreads();
  v = 0.f;
  for (int w = 0; w < waves; ++w) v += exchange[w];
  return v;
}

// A row's mean square, of the P pieces of 8 values of a thread that piece(i, f) gives.  A thread's squares may overflow where
// the mean does not: such a row's are taken again, of the values' 2^-8 (exact but for what vanishes beside them), which
// keeps rows of up to 2^15 values in range.  The branch is uniform over the wavefront, and over the workgroup where rows span
// wavefronts (its threads add the same sums in the same order); the other rows of a wavefront keep their own mean.
template <int L, int P, typename F>
__device__ __forceinline__ float mean_square(float inv_n, float* exchange, F piece) {
  static_assert(QF_BLOCK_NORM_MAX_N <= 1 << 15, "2^-16 of a row's squares stays below their mean");
  float f[8], sum = 0.f;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    piece(i, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += f[e] * f[e];
  }
  const float mean = row_sum<L>(sum * inv_n, exchange);
  if (__builtin_expect(!__any(!(mean < __builtin_inff())), 1)) return mean;
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    piece(i, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += (f[e] * 0x1p-8f) * (f[e] * 0x1p-8f);
  }
  if constexpr (L == 0) __syncthreads();  // the first sums have been read
  const float again = row_sum<L>(sum * (inv_n * 0x1p16f), exchange);
  return mean < __builtin_inff() ? mean : again;
}

// L lanes a row with 256 / L rows a workgroup (L > 0), or a workgroup a row (L = 0); P pieces of 8 values a thread.
template <int L, int P, bool WIDE>
__global__ void __launch_bounds__(L > 0 ? 256 : 1024) block_norm_kernel(const NormArgs a) {
  __shared__ float exchange[2][16];
  const int threads = L > 0 ? L : (int)blockDim.x;  // of a row
  const int t = L > 0 ? (int)threadIdx.x % (L > 0 ? L : 1) : (int)threadIdx.x;
  const int64_t row = L > 0 ? (int64_t)blockIdx.x * (256 / (L > 0 ? L : 1)) + threadIdx.x / (L > 0 ? L : 1) : blockIdx.x;
  const bool live = row < a.M;  // rows past the last: their lanes take part in the exchanges only
  const int64_t m = live ? row : a.M - 1;

  u32x4_t xv[P], gv[P], rv[P][WIDE ? 2 : 1];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int j = t + i * threads;
    xv[i] = gv[i] = rv[i][0] = u32x4_t{0u, 0u, 0u, 0u};
    if constexpr (WIDE) rv[i][1] = rv[i][0];
    if (j < a.pieces) {
      xv[i] = *reinterpret_cast<const u32x4_t*>(a.x + m * a.ldx + (int64_t)j * 8);
      if constexpr (WIDE) {
        const u32x4_t* r = reinterpret_cast<const u32x4_t*>(static_cast<const float*>(a.residual) + m * a.ldr + (int64_t)j * 8);
        rv[i][0] = r[0];
        rv[i][1] = r[1];
      } else {
        rv[i][0] = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(a.residual) + m * a.ldr + (int64_t)j * 8);
      }
      if (a.gate_kind == QF_GATE_FULL) gv[i] = *reinterpret_cast<const u32x4_t*>(a.gate + m * a.ldg + (int64_t)j * 8);
      if (a.gate_kind == QF_GATE_CHANNEL) gv[i] = *reinterpret_cast<const u32x4_t*>(a.gate + (int64_t)j * 8);
    }
  }
  float row_gate = a.alpha;  // alpha, times the token's gate
  if (a.gate_kind == QF_GATE_TOKEN) {
    const float g = bf16_f32(a.gate[m * a.ldg]);
    row_gate *= a.sigmoid ? sigmoid(g) : g;
  }

  if (a.w_post != nullptr) {
    const float mean = mean_square<L, P>(a.inv_n, exchange[0], [&](int i, float(&f)[8]) { unpack8(xv[i], f); });
    row_gate *= 1.f / sqrtf(mean + a.eps);
  }

  float y[P][8];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int j = t + i * threads;
    float f[8];
    unpack8(xv[i], f);
    if (a.w_post != nullptr) {
      float w[8];
      unpack8(j < a.pieces ? *reinterpret_cast<const u32x4_t*>(a.w_post + (int64_t)j * 8) : u32x4_t{0u, 0u, 0u, 0u}, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= a.offset + w[e];
    }
    if (a.gate_kind == QF_GATE_FULL || a.gate_kind == QF_GATE_CHANNEL) {
      float g[8];
      unpack8(gv[i], g);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= a.sigmoid ? sigmoid(g[e]) : g[e];
    }
    if constexpr (WIDE) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[i][e] = __uint_as_float(rv[i][e / 4][e % 4]);
    } else {
      unpack8(rv[i][0], y[i]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y[i][e] += row_gate * f[e];
      if (j >= a.pieces) y[i][e] = 0.f;  // an infinite row_gate times the padding's zeros is no number
    }
    if (live && j < a.pieces) {
      if constexpr (WIDE) {
        u32x4_t* o = reinterpret_cast<u32x4_t*>(static_cast<float*>(a.y) + m * a.ldy + (int64_t)j * 8);
        u32x4_t v[2];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e / 4][e % 4] = __float_as_uint(y[i][e]);
        o[0] = v[0];
        o[1] = v[1];
      } else {
        *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(a.y) + m * a.ldy + (int64_t)j * 8) = pack8(y[i]);
      }
    }
  }
  const float mean = mean_square<L, P>(a.inv_n, exchange[1], [&](int i, float(&f)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = y[i][e];
  });
  const float inv = 1.f / sqrtf(mean + a.eps);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int j = t + i * threads;
    if (!live || j >= a.pieces) continue;
    float o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = y[i][e] * inv;
    if (a.w_pre != nullptr) {
      float w[8];
      unpack8(*reinterpret_cast<const u32x4_t*>(a.w_pre + (int64_t)j * 8), w);
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] *= a.offset + w[e];
    }
    *reinterpret_cast<u32x4_t*>(a.h + m * a.ldh + (int64_t)j * 8) = pack8(o);
  }
}

template <int L, int P>
int launch_norm(bool wide, unsigned grid, unsigned threads, hipStream_t s, const NormArgs& a) {
  if (!grid_fits(grid, (int)threads)) return QF_ERR_UNSUPPORTED;
  if (wide) {
    hipLaunchKernelGGL((block_norm_kernel<L, P, true>), dim3(grid), dim3(threads), 0, s, a);
  } else {
    hipLaunchKernelGGL((block_norm_kernel<L, P, false>), dim3(grid), dim3(threads), 0, s, a);
  }
  return hipGetLastError() == hipSuccess ? QF_OK : QF_ERR_HIP;
}

}  // namespace qfb

using namespace qfb;

extern "C" int qf_block_norm_rows(const uint16_t* x, int64_t ldx, const void* residual, int64_t ldr, int residual_f32,
                                  const uint16_t* post_weight, const uint16_t* pre_weight, float weight_offset,
                                  const uint16_t* gate, int64_t ldg, int gate_kind, int gate_act, float alpha, float eps,
                                  int M, int N, void* y, int64_t ldy, uint16_t* h, int64_t ldh, void* stream) {
  if (x == nullptr || residual == nullptr || y == nullptr || h == nullptr || M < 1 || N < 1) return QF_ERR_INVALID_ARG;
  if (gate_kind < QF_GATE_NONE || gate_kind > QF_GATE_FULL || gate_act < QF_ACT_NONE || gate_act > QF_ACT_SIGMOID ||
      (gate_kind != QF_GATE_NONE) != (gate != nullptr) || !(eps >= 0.f))
    return QF_ERR_INVALID_ARG;
  if (N % 8 || N > QF_BLOCK_NORM_MAX_N) return QF_ERR_UNSUPPORTED;
  const int64_t r_align = residual_f32 ? 4 : 8;
  if (ldx < 0 || ldr < 0 || ldg < 0 || (M > 1 && (ldy < N || ldh < N))) return QF_ERR_INVALID_ARG;
  if (ldx % 8 || ldr % r_align || ldy % r_align || ldh % 8 || (gate_kind == QF_GATE_FULL && ldg % 8))
    return QF_ERR_UNSUPPORTED;
  if (!aligned16(x) || !aligned16(residual) || !aligned16(y) || !aligned16(h) || !aligned16(post_weight) ||
      !aligned16(pre_weight) || (gate_kind != QF_GATE_TOKEN && !aligned16(gate)))
    return QF_ERR_UNSUPPORTED;
  NormArgs a;
  a.x = x;
  a.ldx = ldx;
  a.residual = residual;
  a.ldr = ldr;
  a.w_post = post_weight;
  a.w_pre = pre_weight;
  a.gate = gate;
  a.ldg = ldg;
  a.y = y;
  a.ldy = ldy;
  a.h = h;
  a.ldh = ldh;
  a.M = M;
  a.N = N;
  a.pieces = N / 8;
  a.gate_kind = gate_kind;
  a.sigmoid = gate_act == QF_ACT_SIGMOID;
  a.offset = weight_offset;
  a.alpha = alpha;
  a.eps = eps;
  a.inv_n = 1.f / (float)N;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool wide = residual_f32 != 0;
  // Rows of one piece a lane: 8192 rows in us, against a workgroup a row: N = 64 3.5 (5.7), 128 3.6 (5.8), 256 4.7 (6.3).
  // Longer rows want the workgroup: 512 values 8.1 (32 lanes with two pieces 8.7, a wavefront 9.1), one row of them 2.0 (2.8
  // with two pieces).  A thread takes 2 or 4 pieces only where 1024 threads do not reach.
  if (a.pieces <= 16) return launch_norm<16, 1>(wide, (unsigned)((M + 15ll) / 16), 256, s, a);
  if (a.pieces <= 32) return launch_norm<32, 1>(wide, (unsigned)((M + 7ll) / 8), 256, s, a);
  const int P = a.pieces <= 1024 ? 1 : a.pieces <= 2048 ? 2 : 4;
  const unsigned threads = (unsigned)(((a.pieces + P - 1) / P + kWave - 1) / kWave * kWave);
  if (P == 1) return launch_norm<0, 1>(wide, (unsigned)M, threads, s, a);
  if (P == 2) return launch_norm<0, 2>(wide, (unsigned)M, threads, s, a);
  return launch_norm<0, 4>(wide, (unsigned)M, threads, s, a);
}
