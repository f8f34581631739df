// qf_block_fp8.hip — matrix products with block-scaled e4m3 weights for MI355X (gfx950); the C ABI is in
// include/qf_block.h.
//
//   y[m, n] = sum over blocks kb of 128 k: s[n / 128, kb] * sum_{k in kb} x[m, k] q[n, k]          (M <= 16)
//   y[m, n] = sum over kb: s_a[m, kb] s[n / 128, kb] * sum_{k in kb} xq[m, k] q[n, k]              (any M)
//
// A block's products meet in an MFMA accumulator that starts at zero, and the scaled block is added to the running fp32
// sum with one multiply-add a value.
#include <type_traits>

#include "qf_block_common.h"

namespace qfb {

typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef const void __attribute__((address_space(1)))* gptr_t;
typedef void __attribute__((address_space(3)))* lptr_t;

constexpr int kTileN = 16;   // channels of a weight tile
constexpr int kStepK = 64;   // k of a TILED tile
constexpr int kBlock = QF_FP8_BLOCK;
constexpr int64_t kMaxStride = (int64_t)1 << 26;  // elements: 16 rows within 2^31 bytes
constexpr int kXcds = 8;
constexpr int kMaxLds = 160 * 1024;
constexpr int kCounterStride = 16;  // a counter a cache line
constexpr int kTokenPad = 256;  // the token scales' rows are padded to this many tokens

struct Fp8Args {
  const uint16_t* x;  // decode
  int64_t ldx;
  const uint8_t* xt;   // tiled e4m3 activations [token tiles][2 kblocks] KiB
  const float* s_tok;  // [kblocks][m_pad]
  int m_pad;
  const uint8_t* w;
  int64_t ldw;
  const float* scale;  // [nblocks][kblocks]
  const uint16_t* bias;
  void* y;
  int64_t ldy;
  int out_f32, vec_out;  // vec_out: 4 values of a row may be stored at once
  int M, N, ksteps, kblocks, ntiles;
  uint64_t* partial;   // K split: decode [split][ntiles][2][64 lanes], else [tile][split][wavefront][FA][FB][2][64 lanes]
  unsigned* counters;  // arrivals of a run (counter_stride apart, zero between calls) or a tile (zeroed by the quantiser)
  int counter_stride;
  int runs, splits;    // runs: decode
};

// 4 channels n .. n + 3 of one output row (cnt of them exist), the bias added, rounded once.
__device__ __forceinline__ void store4(const Fp8Args& a, int m, int n, f32x4_t v) {
  const int cnt = min(4, a.N - n);
  if (a.bias != nullptr) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < cnt) v[e] += bf16_f32(a.bias[n + e]);
  }
  if (a.out_f32) {
    float* p = static_cast<float*>(a.y) + (int64_t)m * a.ldy + n;
    if (a.vec_out && cnt == 4) {
      *reinterpret_cast<f32x4_t*>(p) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < cnt) p[e] = v[e];
    }
    return;
  }
  uint16_t* p = static_cast<uint16_t*>(a.y) + (int64_t)m * a.ldy + n;
  const u32x2_t o = {pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
  if (a.vec_out && cnt == 4) {
    *reinterpret_cast<u32x2_t*>(p) = o;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < cnt) p[e] = (uint16_t)(o[e / 2] >> (16 * (e & 1)));
  }
}

// The hardware hands workgroup i to XCD i % kXcds; consecutive logical indexes share an XCD and its L2.
__device__ __forceinline__ int xcd_order(int i, int n) {
  const int xcd = i % kXcds, per = n / kXcds, rem = n % kXcds;
  return xcd * per + min(xcd, rem) + i / kXcds;
}

// ---------------------------------------------------------------------------------------------
// Decode product, M <= 16: bf16 activations, the weights widened to bf16 in registers (exact).
//
// The grid is (runs of 16-channel tiles, K splits).  A workgroup's W wavefronts interleave over the blocks of its K range:
// wavefront v takes the blocks v, v + W, ... (S at most) of every tile of the run, holds their x in LDS or registers, and
// streams its blocks, tile after tile, S of them in flight: TILED weights through registers, each block's reloaded for the
// next tile as soon as it is multiplied; row-major ones through kRowSlots 2 KiB LDS slots of the wavefront's own, by
// direct-to-LDS copies of whole lines (a lane's 16-byte piece p of row n comes from piece p ^ ((n >> 1) & 7), which spreads a
// fragment read's 16 rows over the banks).  No barrier before the sums.  Lane (g, r) holds channel r (or token r) at k
// 16 g .. 16 g + 15 of each half block, so the fragments need no exchange.  Each wavefront parks its partial tile in LDS;
// wavefront v then adds the W partials of tiles v, v + W, ... in wavefront order; with a K split the last workgroup of a run
// adds the splits in split order.
//
// Bound by the weights' bytes: 5 x 34816 x 5120 30.4 us (5.9 TB/s), 1 x 5120 x 5120 8.6, 16 x 5120 x 17408 19.2 (row-major
// 21), over three sets of weights, part of them in the last-level cache; over 1.5 GB of them, a call in a graph, 33.6 (5.3
// TB/s), 8.3 and row-major 24.5.  A request behind a run's last tile cost 0.5 us there and 1.6 at 34816 channels.  Row-major slots a wavefront, 5 x
// 34816 x 5120: 2 35.7 us, 3 36.8, 4 40.2.  The nontemporal hint: TILED 30.4 us, 32 without it where the weights do not stand
// in the last-level cache; row-major copies with it 5% faster there and 20% slower where they do.
// ---------------------------------------------------------------------------------------------
constexpr int kRowSlots = 2;
constexpr int kJoinBatch = 4;
__host__ __device__ constexpr int decode_ring(int layout, int W) {
  return layout == QF_LAYOUT_TILED ? 0 : W * kRowSlots * 2048;
}

template <int LAYOUT, int S, int XL>
__global__ void __launch_bounds__(1024) __attribute__((amdgpu_waves_per_eu(4)))
fp8_decode_kernel(const Fp8Args a) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int last_arrival;
  constexpr int D = kRowSlots;
  const int W = blockDim.x / kWave;
  const int lane = threadIdx.x & (kWave - 1);
  const int v = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int g = lane >> 4, r = lane & 15;
  const int split = blockIdx.x / a.runs, run = blockIdx.x - split * a.runs;
  const int t0 = (int)((int64_t)run * a.ntiles / a.runs);
  const int nt = (int)((int64_t)(run + 1) * a.ntiles / a.runs) - t0;  // >= 1: no more runs than tiles
  const int kb0 = (int)((int64_t)split * a.kblocks / a.splits);
  const int kb1 = (int)((int64_t)(split + 1) * a.kblocks / a.splits);
  const int mine = kb1 - kb0 > v ? (kb1 - kb0 - v + W - 1) / W : 0;  // at most S
  uint8_t* const xs = smem + decode_ring(LAYOUT, W) + v * S * XL * 1024;  // [W][S][XL] KiB
  f32x4_t* const part = reinterpret_cast<f32x4_t*>(smem + decode_ring(LAYOUT, W) + W * S * XL * 1024);  // [nt][W][64 lanes]

  if (mine > 0) {  // uniform
    // x fragments of the wavefront's blocks.  XL > 0 (up to 4 XL tokens): in LDS for the whole run, a copy fetching 4 rows x
    // 256 bytes of a block, piece p of row n landing at p ^ n.  XL = 0: in registers, read straight from the caches; columns
    // past the last token stay zero and cost no requests.
    u32x4_t xf[XL ? 1 : S][2][2];
    if constexpr (XL == 0) {
#pragma unroll
      for (int p = 0; p < S; ++p) xf[p][0][0] = xf[p][0][1] = xf[p][1][0] = xf[p][1][1] = u32x4_t{0u, 0u, 0u, 0u};
      if (r < a.M) {
        const uint16_t* const xp = a.x + (int64_t)r * a.ldx + 16 * g;
#pragma unroll
        for (int p = 0; p < S; ++p)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int step = min(2 * (kb0 + v + p * W) + h, a.ksteps - 1);
            const u32x4_t* q = reinterpret_cast<const u32x4_t*>(xp + (int64_t)step * kStepK);
            xf[p][h][0] = q[0];
            xf[p][h][1] = q[1];
          }
      }
    } else {
      const int row = lane >> 4;
#pragma unroll
      for (int p = 0; p < S; ++p) {
        const int kb = kb0 + v + min(p, mine - 1) * W;
#pragma unroll
        for (int i = 0; i < XL; ++i) {
          const int n = 4 * i + row, piece = (lane & 15) ^ n;
          const int piece_in = 2 * kb + 1 < a.ksteps ? piece : piece & 7;  // a last half block: its values twice
          __builtin_amdgcn_global_load_lds((gptr_t)(a.x + (int64_t)min(n, a.M - 1) * a.ldx + (int64_t)kb * kBlock + piece_in * 8),
                                           (lptr_t)(xs + (p * XL + i) * 1024), 16, 0, 0);
        }
      }
    }
    auto x_of = [&](int p, u32x4_t (&f)[2][2]) {
      if constexpr (XL == 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int q = 0; q < 2; ++q) f[h][q] = xf[p][h][q];
      } else {
        const int n = r & (4 * XL - 1);  // columns past the last token: any row, never stored
        const uint32_t base = lds_addr(xs) + p * XL * 1024 + n * 256;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int q = 0; q < 2; ++q)
            asm volatile("ds_read_b128 %0, %1" : "=v"(f[h][q]) : "v"(base + (((8 * h + 2 * g + q) ^ n) << 4)));
        asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(f[0][0]), "+v"(f[0][1]), "+v"(f[1][0]), "+v"(f[1][1]));
      }
    };
    __builtin_amdgcn_sched_barrier(0);
    float sc[S];
    auto scales = [&](int t) {  // another block of channels: its scales
      const float* row = a.scale + (int64_t)((t0 + t) / (kBlock / kTileN)) * a.kblocks + kb0 + v;
#pragma unroll
      for (int p = 0; p < S; ++p) sc[p] = row[p < mine ? p * W : 0];
    };
    auto whole = [&](int p) { return 2 * (kb0 + v + p * W) + 1 < a.ksteps; };  // or half a block, the last one

    if constexpr (LAYOUT == QF_LAYOUT_TILED) {
      const uint32_t w_lane = (uint32_t)lane * 16;
      u32x4_t w[S][2];
      auto load = [&](int t, int p) {  // (blocks past the range: the last one again, not used)
        const uint8_t* q = a.w + ((int64_t)(t0 + t) * a.ksteps + 2 * (kb0 + v + min(p, mine - 1) * W)) * 1024;
        w[p][0] = load_once(q + w_lane);
        w[p][1] = load_once(q + (whole(min(p, mine - 1)) ? 1024 : 0) + w_lane);
      };
#pragma unroll
      for (int p = 0; p < S; ++p) load(0, p);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (XL > 0) wait_vmcnt<2 * S>();  // x, ahead of the weights
      auto tile = [&](int t, auto reload) {
        if (t == 0 || (t0 + t) % (kBlock / kTileN) == 0) scales(t);
        f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int p = 0; p < S; ++p) {
          if (p < mine) {
            u32x4_t x[2][2];
            x_of(p, x);
            acc += block_product(w[p], x, whole(p)) * sc[p];
          }
          if constexpr (decltype(reload)::value) load(t + 1, p);
        }
        part[(t * W + v) * kWave + lane] = acc;
      };
      for (int t = 0; t + 1 < nt; ++t) tile(t, std::true_type());
      tile(nt - 1, std::false_type());
    } else {
      // The copy cursor: block cp of tile ct, into slot cslot.  Past the last block it goes round the last tile again
      // (in-bounds re-reads into slots that are read no more), so that every copy is made and counted.
      uint8_t* const ring = smem + v * D * 2048;
      const int lrow = lane >> 3, piece = (lane & 7) ^ (lrow >> 1);  // rows 8 .. 15 flip piece bit 2 besides
      int ct = 0, cp = 0;
      uint32_t cslot = 0;
      const uint8_t *row0, *row1;
      auto enter = [&]() {
        const int n = (t0 + ct) * kTileN + lrow;
        row0 = a.w + (int64_t)min(n, a.N - 1) * a.ldw;
        row1 = a.w + (int64_t)min(n + 8, a.N - 1) * a.ldw;
      };
      enter();
      auto copy = [&]() {
        const bool both = whole(cp);  // else a last half block: its bytes twice, the second ones not used
        uint8_t* dst = ring + cslot;
        const int q0 = both ? piece : piece & 3, q1 = both ? piece ^ 4 : (piece ^ 4) & 3;
        const int64_t k = (int64_t)(kb0 + v + cp * W) * kBlock;
        __builtin_amdgcn_global_load_lds((gptr_t)(row0 + k + q0 * 16), (lptr_t)dst, 16, 0, 0);
        __builtin_amdgcn_global_load_lds((gptr_t)(row1 + k + q1 * 16), (lptr_t)(dst + 1024), 16, 0, 0);
        cslot = cslot == (D - 1) * 2048 ? 0 : cslot + 2048;
        if (++cp == mine) {
          cp = 0;
          if (ct < nt - 1) {
            ++ct;
            enter();
          }
        }
      };
#pragma unroll
      for (int d = 0; d < D; ++d) copy();
      if constexpr (XL > 0) wait_vmcnt<2 * D>();  // x, ahead of the weights
      const uint32_t f0 = lds_addr(ring) + r * 128 + ((g ^ ((r >> 1) & 7)) << 4);
      const uint32_t f1 = lds_addr(ring) + r * 128 + (((4 + g) ^ ((r >> 1) & 7)) << 4);
      uint32_t slot = 0;
      for (int t = 0; t < nt; ++t) {
        if (t == 0 || (t0 + t) % (kBlock / kTileN) == 0) scales(t);
        f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int p = 0; p < S; ++p) {
          if (p < mine) {  // uniform
            wait_vmcnt<2 * (D - 1)>();  // this block's copies have landed
            // Read by inline assembly, waits included: before a plain LDS read the compiler may wait for every copy in flight.
            u32x4_t w[2];
            asm volatile(
                "ds_read_b128 %0, %2\n\t"
                "ds_read_b128 %1, %3\n\t"
                "s_waitcnt lgkmcnt(0)"
                : "=&v"(w[0]), "=&v"(w[1])
                : "v"(f0 + slot), "v"(f1 + slot)
                : "memory");
            copy();  // the reads have returned: into the slot they read
            slot = slot == (D - 1) * 2048 ? 0 : slot + 2048;
            u32x4_t x[2][2];
            x_of(p, x);
            acc += block_product(w, x, whole(p)) * sc[p];
          }
        }
        part[(t * W + v) * kWave + lane] = acc;
      }
      wait_vmcnt<0>();  // no copy lands once the workgroup's LDS is given back
    }
  } else {
    for (int t = 0; t < nt; ++t) part[(t * W + v) * kWave + lane] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  __syncthreads();
  // a split's partial tile: 64 lanes x 16 bytes, as two planes of 8 bytes a lane
  auto slot = [&](int split, int t) { return a.partial + ((int64_t)split * a.ntiles + t0 + t) * 2 * kWave + lane; };
  for (int t = v; t < nt; t += W) {
    f32x4_t sum = part[t * W * kWave + lane];
    for (int u = 1; u < W; ++u) sum += part[(t * W + u) * kWave + lane];
    const int n = (t0 + t) * kTileN + 4 * g;
    if (r >= a.M) continue;
    if (a.splits == 1) {
      if (n < a.N) store4(a, r, n, sum);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        __hip_atomic_store(slot(split, t) + i * kWave, __builtin_bit_cast(uint64_t, f32x2_t{sum[2 * i], sum[2 * i + 1]}),
                           __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  if (a.splits == 1) return;
  // The splits' sums are in device memory (device-scope stores, waited for) before the run's counter is raised; the last
  // arrival reads them with device-scope loads issued after its increment returned, and returns the counter to zero.
  wait_vmcnt<0>();
  __syncthreads();
  if (threadIdx.x == 0) {
    const unsigned prev = __hip_atomic_fetch_add(a.counters + run * a.counter_stride, 1u, __ATOMIC_RELAXED,
                                                 __HIP_MEMORY_SCOPE_AGENT);
    last_arrival = prev == (unsigned)(a.splits - 1);
  }
  __syncthreads();
  if (!last_arrival) return;
  for (int t = v; t < nt; t += W) {
    const int n = (t0 + t) * kTileN + 4 * g;
    if (r < a.M && n < a.N) {
      f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
      for (int j = 0; j < a.splits; j += kJoinBatch) {  // a batch's loads are all in flight at once
        f32x2_t q[kJoinBatch][2];
#pragma unroll
        for (int k = 0; k < kJoinBatch; ++k)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            q[k][i] = __builtin_bit_cast(f32x2_t, __hip_atomic_load(slot(min(j + k, a.splits - 1), t) + i * kWave,
                                                                    __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
#pragma unroll
        for (int k = 0; k < kJoinBatch; ++k) {
          const f32x4_t p = {q[k][0].x, q[k][0].y, q[k][1].x, q[k][1].y};
          if (j + k < a.splits) sum = j + k == 0 ? p : sum + p;
        }
      }
      store4(a, r, n, sum);
    }
  }
  if (threadIdx.x == 0)
    __hip_atomic_store(a.counters + run * a.counter_stride, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ---------------------------------------------------------------------------------------------
// Token quantiser: 8 lanes a (token, block of 128), 16 values a lane, a workgroup 16 tokens by 2 blocks (so the 8
// tokens of a wavefront store 128 bytes side by side).  TILED writes the product's operand image (KiB tiles of 16 tokens
// x 64 k, as the weights'; the last half block's second half is zero, rows past M are not written) and the scales block by
// block; otherwise row-major values and scales.
//
// The quotient f / s is rounded correctly by r = 1 / s, q0 = f r, q = q0 + (f - q0 s) r, the remainder exact in an fma
// (Markstein): r is correctly rounded, and s = max / 448 has no significand of ones alone, the case the theorem leaves out
// (max has 8 bits, and a repeating fraction of sevenths holds zeros).  Small s are scaled up by 2^60 with f, so that neither
// r overflows nor a remainder that matters is subnormal: quotients below 2^-11 are zero in e4m3 whatever their last bits.
//
// Bound by the memory rate: 2048 x 5120 (32 MB in and out) 6.6 us, 4096 x 17408 37 us, 5.8 TB/s.  With 8 values a lane, a
// division each and 4 blocks a workgroup it took 10.2 and 52 us; 16 values and 4 blocks a workgroup, 7.8 and 38.
// ---------------------------------------------------------------------------------------------
struct QuantArgs {
  const uint16_t* x;
  int64_t ldx;
  uint8_t* xq;
  int64_t ldq;
  float* s;
  int m_pad;
  int M, ksteps, kblocks;
  unsigned* counters;  // the product's arrival counters, zeroed here
  int n_counters;
};

constexpr int kQuantBlocks = 2;  // blocks of 128 a workgroup

template <bool TILED>
__global__ void __launch_bounds__(256) quantize_tokens_fp8_kernel(const QuantArgs a) {
  if (TILED && blockIdx.x == 0 && blockIdx.y == 0)
    for (int c = threadIdx.x; c < a.n_counters; c += 256) a.counters[c] = 0;
  const int i = threadIdx.x & 7;
  const int m = blockIdx.x * 16 + (threadIdx.x >> 3 & 15);
  const int kb = blockIdx.y * kQuantBlocks + (threadIdx.x >> 7);
  if (kb >= a.kblocks || m >= a.M) return;
  const bool in = i < 4 || 2 * kb + 1 < a.ksteps;
  u32x4_t v[2] = {{0u, 0u, 0u, 0u}, {0u, 0u, 0u, 0u}};
  if (in) {
    const u32x4_t* p = reinterpret_cast<const u32x4_t*>(a.x + (int64_t)m * a.ldx + (int64_t)kb * kBlock + 16 * i);
    v[0] = p[0];
    v[1] = p[1];
  }
  float f[16], top = 0.f;
  unpack8(v[0], reinterpret_cast<float(&)[8]>(f[0]));
  unpack8(v[1], reinterpret_cast<float(&)[8]>(f[8]));
#pragma unroll
  for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(f[e]));
  const float s = group_max<8>(top) / 448.f;
  const float up = s < 0x1p-60f ? 0x1p60f : 1.f;
  const bool ok = s > 0.f && s < __builtin_inff();  // otherwise zeros, or NaN from NaN and infinity
  const float d = ok ? s * up : 0.f, r = ok ? 1.f / d : 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const float n = f[e] * up, q0 = n * r;
    f[e] = copysignf(fmaf(fmaf(-q0, d, n), r, q0), n);  // (-0 keeps its sign)
  }
  u32x4_t q;
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    const int p = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * h], f[4 * h + 1], 0, false);
    q[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * h + 2], f[4 * h + 3], p, true);
  }
  if constexpr (TILED) {
    const int64_t tile = ((int64_t)(m >> 4) * 2 * a.kblocks + 2 * kb + (i >> 2)) * kWave + (i & 3) * 16 + (m & 15);
    *reinterpret_cast<u32x4_t*>(a.xq + tile * 16) = q;
    if (i == 0) a.s[(int64_t)kb * a.m_pad + m] = s;
  } else {
    if (in) {
      u32x2_t* p = reinterpret_cast<u32x2_t*>(a.xq + (int64_t)m * a.ldq + (int64_t)kb * kBlock + 16 * i);
      p[0] = u32x2_t{q[0], q[1]};
      p[1] = u32x2_t{q[2], q[3]};
    }
    if (i == 0) a.s[(int64_t)m * a.kblocks + kb] = s;
  }
}

// ---------------------------------------------------------------------------------------------
// W8A8 product: LDS-tiled, v_mfma_f32_16x16x128_f8f6f4 (one instruction a block of K and 16 x 16 outputs).
//
// A workgroup of WN x WM wavefronts owns 16 FA WN channels x 16 FB WM tokens.  A stage is one block of K: its weight and
// activation fragments (16 rows x 128 k, 2 KiB) go global -> LDS by direct-to-LDS copies, lane l's 16 bytes of each half
// landing at 16 l, so a fragment read is two conflict-free 16-byte reads a lane; S stages form a ring.  Lane (g, r) of a
// fragment holds row r at k 16 g .. + 15 of both halves: the instruction sums over all of k, so its order within the block
// does not matter as long as both operands share it.  The accumulator's columns are tokens: a lane's token scale is one value a
// column, times the block's weight scale (one for the wavefront: its channels lie in one block of 128).
//
// What the instruction rounds: it adds the 8 products of 8 neighbouring k of a lane aligned to the largest exponent sum e
// among them and drops what lies below 2^(e - 13); the groups' sums and the running sums are fp32.  Against exact sums
// that is 1.5e-5 to 3.6e-5 of a result's size (normal values, K = 128 to 5120), a hundredth of an e4m3 activation's own
// rounding.  The narrower f8 instruction (16x16x32) drops the same and runs at a third of the rate (1.42 against 4.58
// PFLOP/s); the widened bf16 product of the decode kernel keeps everything, at half of it.
//
// Measured: 2048 x 32768 x 5120 (four rounds of 256 x 256) 315 to 330 us, 2.1 PFLOP/s, the matrix cores half busy at 2.2
// GHz.  Without its copies (in a copy of the kernel, for timing) a round takes 57 us instead of 82; 256 x 128 tiles with two
// stages ahead, all of a stage's copies at once, activations stored block by block, or weights read ahead into L2 change
// nothing or cost time.  128 x 128 tiles reach 1.9 PFLOP/s: the LDS traffic of a step (96 KiB read, 32 written) is 0.47 of its
// 0.57 us; 4 wavefronts of 64 x 64 read 64 KiB and take 0.7, as one wavefront a SIMD hides nothing.
// ---------------------------------------------------------------------------------------------
template <int FA_, int FB_, int WN_, int WM_, int S_>
struct Tile {
  static constexpr int FA = FA_, FB = FB_, WN = WN_, WM = WM_, S = S_;
  static constexpr int waves = WN * WM;
  static constexpr int channels = 16 * FA * WN, tokens = 16 * FB * WM;
  static constexpr int frags = FA * WN + FB * WM;
  static constexpr int own = frags / waves;  // fragments a wavefront copies
  static_assert(frags % waves == 0 && 8 % FA == 0 && kTokenPad % tokens == 0, "tile shape");
  static constexpr int copies = 2 * own + 1;  // with its tokens' scales
  static constexpr int stage = frags * 2048;
  static constexpr int slot = stage + waves * 256;
  static constexpr int lds = S * slot;
  static constexpr int max_kblocks = (kMaxLds - lds) / (4 * WN);  // the weight scales stand behind the ring
  static_assert(waves * FA * FB * 512 <= lds && max_kblocks >= QF_FP8_MAX_W8A8_K / kBlock, "LDS");
};

template <int LAYOUT, typename T, int MINW, int MAXW>
__global__ void __launch_bounds__(T::waves* kWave) __attribute__((amdgpu_waves_per_eu(MINW, MAXW)))
fp8_tile_kernel(const Fp8Args a) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int FA = T::FA, FB = T::FB, S = T::S;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wn = wave % T::WN, wm = wave / T::WN;
  const int g = lane >> 4, r = lane & 15;
  const int mblocks = (a.M + T::tokens - 1) / T::tokens;
  const int place = xcd_order(blockIdx.x, gridDim.x);
  const int tile = place / a.splits, split = place - tile * a.splits;
  const int nb = tile / mblocks, mb = tile - nb * mblocks;
  const int tile0 = nb * (T::channels / 16);
  const int m0 = mb * T::tokens;
  const int k0 = (int)((int64_t)split * a.kblocks / a.splits);  // this workgroup's blocks of K
  const int nsteps = (int)((int64_t)(split + 1) * a.kblocks / a.splits) - k0;

  // fragment f of the stage: the FA WN weight fragments, then the FB WM activation fragments; channels and tokens past
  // the matrix read its last tile, their outputs are not stored
  constexpr int kHalf = LAYOUT == QF_LAYOUT_TILED ? kTileN * kStepK : kStepK;
  // fragment's bytes: a scalar base and a 32-bit lane offset (the host bounds 16 rows of row-major weights by 2^31 bytes)
  const uint8_t* src[T::own];
  uint32_t src_lane[T::own];
#pragma unroll
  for (int j = 0; j < T::own; ++j) {
    const int f = wave * T::own + j;
    src_lane[j] = (uint32_t)lane * 16;
    if (f < FA * T::WN) {
      const int t = min(tile0 + f, a.ntiles - 1);
      if constexpr (LAYOUT == QF_LAYOUT_TILED) {
        src[j] = a.w + (int64_t)t * a.ksteps * 1024;
      } else {
        src[j] = a.w + (int64_t)t * kTileN * a.ldw;
        src_lane[j] = (uint32_t)min(r, a.N - 1 - t * kTileN) * (uint32_t)a.ldw + 16 * g;
      }
    } else {
      const int t = min((m0 >> 4) + f - FA * T::WN, (a.M - 1) >> 4);
      src[j] = a.xt + (int64_t)t * 2 * a.kblocks * 1024;
    }
    src[j] = scalar_ptr(src[j]);
  }
  const float* const ssrc = a.s_tok + m0 + 16 * FB * wm;
  const uint32_t s_src_lane = (uint32_t)(lane & (16 * FB - 1)) * 4;
  // Stage s in own + 1 pieces, a fragment each and the token scales (past the last stage: the last again, into a slot that
  // nothing reads any more).
  auto copy_piece = [&](int s, int slot_at, int j) {
    uint8_t* slot = smem + slot_at * T::slot;
    const int kb = k0 + min(s, nsteps - 1);
    if (j < T::own) {
      const int f = wave * T::own + j;
      const int half = f < FA * T::WN ? kHalf : kTileN * kStepK;
      const uint8_t* p = src[j] + (int64_t)kb * 2 * half;
      // a last half block: the weights' first half again, times the activations' zeros
      const uint8_t* q = p + (2 * kb + 1 < a.ksteps || f >= FA * T::WN ? half : 0);
      __builtin_amdgcn_global_load_lds((gptr_t)(scalar_ptr(p) + here(src_lane[j])), (lptr_t)(slot + f * 2048), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((gptr_t)(scalar_ptr(q) + here(src_lane[j])), (lptr_t)(slot + f * 2048 + 1024), 16, 0, 0);
    } else {
      const uint8_t* p = reinterpret_cast<const uint8_t*>(ssrc + (int64_t)kb * a.m_pad);
      __builtin_amdgcn_global_load_lds((gptr_t)(scalar_ptr(p) + here(s_src_lane)), (lptr_t)(slot + T::stage + wave * 256), 4, 0, 0);
    }
  };
  const int n_first = (tile0 + FA * wn) * kTileN;  // this wavefront's first channel
  const float* srow = a.scale + (int64_t)min(n_first / kBlock, (a.N - 1) / kBlock) * a.kblocks + k0;
  // all of its blocks' scales, in LDS behind the ring (a row for each of the WN channel groups)
  float* const sw = reinterpret_cast<float*>(smem + T::lds) + wn * nsteps;
  for (int k = wm * kWave + lane; k < nsteps; k += T::WM * kWave) sw[k] = srow[k];
  wait_vmcnt<0>();  // the copies below are counted

  f32x4_t acc[FA][FB];
#pragma unroll
  for (int i = 0; i < FA; ++i)
#pragma unroll
    for (int j = 0; j < FB; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < S - 1; ++s)
#pragma unroll
    for (int j = 0; j <= T::own; ++j) copy_piece(s, s, j);

  // LDS reads are issued by inline assembly and waited for by count (before a plain read's use the compiler waits for all of
  // LDS while copies are in flight); their registers are tied to the waits, so nothing uses them before.
  const uint32_t lane16 = (uint32_t)lane * 16, r4 = (uint32_t)r * 4;
  const uint32_t a_at = lds_addr(smem) + FA * wn * 2048;
  const uint32_t b_at = lds_addr(smem) + (FA * T::WN + FB * wm) * 2048;
  const uint32_t s_at = lds_addr(smem) + T::stage + wave * 256;
  const uint32_t w_at = lds_addr(sw);
  auto read_frag = [](uint32_t at) {
    i32x4_t lo, hi;
    asm volatile("ds_read_b128 %0, %1" : "=v"(lo) : "v"(at));
    asm volatile("ds_read_b128 %0, %1 offset:1024" : "=v"(hi) : "v"(at));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  auto read_tokens = [&](int s, uint32_t slot, i32x8_t (&B)[FB], float (&sc)[FB], float& w) {  // fragments, both scales
    asm volatile("ds_read_b32 %0, %1" : "=v"(w) : "v"(w_at + 4 * min(s, nsteps - 1)));
#pragma unroll
    for (int j = 0; j < FB; ++j) asm volatile("ds_read_b32 %0, %1" : "=v"(sc[j]) : "v"(here(r4) + (s_at + slot + 64 * j)));
#pragma unroll
    for (int j = 0; j < FB; ++j) B[j] = read_frag(here(lane16) + (b_at + slot + j * 2048));
  };
  auto tie = [](i32x8_t (&B)[FB], float (&sc)[FB], float& w) {
    asm volatile("" : "+v"(w));
#pragma unroll
    for (int j = 0; j < FB; ++j) asm volatile("" : "+v"(B[j]), "+v"(sc[j]));
  };
  // Products wait one row of fragments in t before they are scaled and added, so that the additions run beside the next
  // row's matrix instructions; each weight fragment is read a row ahead, the next stage's first ones ahead of the last row.
  // No branch in a stage: the compiler would move additions across it and keep every product alive.
  // The copies of the stage that refills the slot of stage s - 1 go out between the rows of stage s.
  constexpr int per_row = S == 2 ? 2 : (T::own + FA - 1) / (FA - 1);  // pieces: own + 1 over FA - 1 rows; early with one stage ahead
  f32x4_t t[FB];
#pragma unroll
  for (int j = 0; j < FB; ++j) t[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  i32x8_t A[2], B0[FB], B1[FB];
  float s0[FB], s1[FB], w;
  int at = 0, free_at = S - 1;  // ring slots of stage s, and of the one before it
  // (Bn, scn): the stage before (its scales), then the next
  auto step = [&](int s, i32x8_t (&B)[FB], float (&sc)[FB], i32x8_t (&Bn)[FB], float (&scn)[FB]) {
    const int next_at = at + 1 == S ? 0 : at + 1;
#pragma unroll
    for (int i = 0; i < FA; ++i) {
      if (i == 1) {
#pragma unroll
        for (int j = 0; j < FB; ++j) sc[j] *= w;
      }
      if (i + 1 < FA) {
        A[(i + 1) & 1] = read_frag(here(lane16) + (a_at + (uint32_t)at * T::slot + (i + 1) * 2048));
        asm volatile("s_waitcnt lgkmcnt(2)" : "+v"(A[i & 1]) : : "memory");
        if (i == 0) tie(B, sc, w);
      } else {  // (past the last stage: a stage that is copied again, not used)
        wait_vmcnt<T::copies*(S - 2)>();
        ring_barrier();  // stage s + 1 has landed, and nothing reads stage s any more
        asm volatile("" : "+v"(A[i & 1]));
        read_tokens(s + 1, (uint32_t)next_at * T::slot, Bn, scn, w);
        A[(i + 1) & 1] = read_frag(here(lane16) + (a_at + (uint32_t)next_at * T::slot));
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < FB; ++j) {
        acc[(i + FA - 1) % FA][j] += t[j] * (i == 0 ? scn[j] : sc[j]);
        t[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A[i & 1], B[j], f32x4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (i + 1 < FA) {
#pragma unroll
        for (int j = i * per_row; j < (i + 1) * per_row && j <= T::own; ++j) copy_piece(s + S - 1, free_at, j);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    free_at = at;
    at = next_at;
  };
  static_assert(FA % 2 == 0, "the weight fragments' two buffers alternate through a stage");
#pragma unroll
  for (int j = 0; j < FB; ++j) s1[j] = 0.f;
  wait_vmcnt<T::copies*(S - 2)>();
  ring_barrier();
  read_tokens(0, 0, B0, s0, w);
  A[0] = read_frag(here(lane16) + a_at);
  int s = 0;
  for (; s + 1 < nsteps; s += 2) {
    step(s, B0, s0, B1, s1);
    step(s + 1, B1, s1, B0, s0);
  }
  const bool odd = s < nsteps;
  if (odd) step(s, B0, s0, B1, s1);
  asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(A[0]), "+v"(A[1]) : : "memory");  // the reads past the last stage have returned
  tie(B0, s0, w);
  tie(B1, s1, w);
#pragma unroll
  for (int j = 0; j < FB; ++j) {
    const float even_s = s1[j], odd_s = s0[j];
    acc[FA - 1][j] += t[j] * (odd ? odd_s : even_s);
  }
  wait_vmcnt<0>();  // the last copies have landed before LDS is reused or released

  if (a.splits > 1) {
    // The splits of a tile meet through the workspace: each leaves its sums, lane for lane, by device-scope stores and waits
    // for them; one thread counts the arrival; the last one to arrive reads the others' by device-scope loads, issued after its
    // increment returned, and adds all in split order.
    auto slot = [&](int split, int i, int j) {
      return a.partial + ((((int64_t)tile * a.splits + split) * T::waves + wave) * (FA * FB) + i * FB + j) * 2 * kWave + lane;
    };
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
      for (int j = 0; j < FB; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          __hip_atomic_store(slot(split, i, j) + h * kWave, __builtin_bit_cast(uint64_t, f32x2_t{acc[i][j][2 * h], acc[i][j][2 * h + 1]}),
                             __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    wait_vmcnt<0>();
    __syncthreads();
    int* const last = reinterpret_cast<int*>(smem);
    if (threadIdx.x == 0)
      *last = __hip_atomic_fetch_add(a.counters + tile, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
              (unsigned)(a.splits - 1);
    __syncthreads();
    if (!*last) return;
    __syncthreads();  // before LDS is written again
    for (int o = 0; o < a.splits; ++o) {
#pragma unroll
      for (int i = 0; i < FA; ++i) {
        f32x4_t p[FB];
#pragma unroll
        for (int j = 0; j < FB; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const f32x2_t v = __builtin_bit_cast(f32x2_t, __hip_atomic_load(slot(o, i, j) + h * kWave, __ATOMIC_RELAXED,
                                                                            __HIP_MEMORY_SCOPE_AGENT));
            p[j][2 * h] = v.x;
            p[j][2 * h + 1] = v.y;
          }
#pragma unroll
        for (int j = 0; j < FB; ++j) acc[i][j] = o == 0 ? p[j] : acc[i][j] + p[j];
      }
    }
  }

  // Lane (g, r) holds channels 4 g .. 4 g + 3 of a tile, token r.
  if (!a.out_f32 && a.vec_out && a.ldy % 8 == 0 && (reinterpret_cast<uintptr_t>(a.y) & 15) == 0) {
    // each wavefront's block through its own LDS (16-byte chunk c of token t at c ^ (t % NC)): whole row pieces are stored
    constexpr int NC = 2 * FA;
    __syncthreads();
    uint8_t* blk = smem + wave * (FA * FB * 512);
#pragma unroll
    for (int i = 0; i < FA; ++i) {
      float b[4] = {0.f, 0.f, 0.f, 0.f};
      if (a.bias != nullptr) {
        const int n = n_first + 16 * i + 4 * g;
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = n + e < a.N ? bf16_f32(a.bias[n + e]) : 0.f;
      }
#pragma unroll
      for (int j = 0; j < FB; ++j) {
        const int t = 16 * j + r;
        const f32x4_t v = acc[i][j];
        const int c = 2 * i + (g >> 1);
        *reinterpret_cast<u32x2_t*>(blk + t * 16 * NC + ((c ^ (t % NC)) << 4) + 8 * (g & 1)) =
            u32x2_t{pack_bf16(v[0] + b[0], v[1] + b[1]), pack_bf16(v[2] + b[2], v[3] + b[3])};
      }
    }
    __syncthreads();
    const int c = lane % NC;
    const int n0 = n_first + 8 * c;
#pragma unroll
    for (int q = 0; q < 16 * FB * NC / kWave; ++q) {
      const int t = (kWave / NC) * q + lane / NC;
      const int m = m0 + 16 * FB * wm + t;
      const u32x4_t v = *reinterpret_cast<const u32x4_t*>(blk + t * 16 * NC + ((c ^ (t % NC)) << 4));
      if (m < a.M) {
        uint16_t* row = static_cast<uint16_t*>(a.y) + (int64_t)m * a.ldy + n0;
        if (n0 + 8 <= a.N) {
          *reinterpret_cast<u32x4_t*>(row) = v;
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (n0 + k < a.N) row[k] = (uint16_t)(v[k >> 1] >> (16 * (k & 1)));
        }
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < FA; ++i) {
    const int n = n_first + 16 * i + 4 * g;
#pragma unroll
    for (int j = 0; j < FB; ++j) {
      const int m = m0 + 16 * FB * wm + 16 * j + r;
      if (m < a.M && n < a.N) store4(a, m, n, acc[i][j]);
    }
  }
}

typedef Tile<8, 4, 2, 4, 2> BigTile;    // 256 channels x 256 tokens
typedef Tile<4, 2, 2, 4, 4> MidTile;    // 128 x 128
typedef Tile<2, 4, 4, 1, 3> SmallTile;  // 128 x 64
typedef Tile<2, 2, 2, 2, 4> TinyTile;   // 64 x 64

template <int LAYOUT, typename T, int MINW, int MAXW>
int launch_tile(const Fp8Args& a, hipStream_t s) {
  static std::atomic<uint64_t> raised{0};
  if (!raise_lds(reinterpret_cast<const void*>(&fp8_tile_kernel<LAYOUT, T, MINW, MAXW>), kMaxLds, raised)) return QF_ERR_HIP;
  const int64_t grid = (int64_t)((a.N + T::channels - 1) / T::channels) * ((a.M + T::tokens - 1) / T::tokens) * a.splits;
  const int share = (a.kblocks + a.splits - 1) / a.splits;
  if (!grid_fits(grid, T::waves * kWave)) return QF_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((fp8_tile_kernel<LAYOUT, T, MINW, MAXW>), dim3((unsigned)grid), dim3(T::waves * kWave),
                     T::lds + T::WN * share * 4, s, a);
  return hipGetLastError() == hipSuccess ? QF_OK : QF_ERR_HIP;
}

// The tile shapes' launch figures: us a block of K takes one workgroup a CU and two (0: LDS holds one), and what joining
// s splits adds, join + s * more (a tile's last arrival reads the others' sums).  Measured over M = 17 to 2048, N = 2000 to
// 34816, K = 2048 to 8192; the estimates below are within 15% of the times there, but for weights that come from HBM once.
struct TileFigures {
  int channels, tokens;
  double step, step2, join, more;
};
enum TileKind { kBig, kMid, kSmall, kTiny, kKinds };
constexpr TileFigures kFigures[kKinds] = {
    {256, 256, 1.70, 0, 6.0, 5.0}, {128, 128, 0.57, 0, 2.5, 2.2}, {128, 64, 0.48, 0.85, 1.2, 0.8}, {64, 64, 0.31, 0.50, 1.0, 0.5}};
constexpr int kCus = 256;
constexpr double kLaunch = 4.0;  // us

// One launch over N channels, and where main_n > 0 one of whole rounds of 256 x 256 tiles over the first main_n before it.
struct TilePlan {
  int kind, splits, main_n;
  double cost;
};

int64_t tiles_of(int kind, int M, int N) {
  const TileFigures& f = kFigures[kind];
  return (int64_t)((N - 1) / f.channels + 1) * ((M - 1) / f.tokens + 1);
}

TilePlan plan_single(int M, int N, int kblocks) {
  TilePlan best = {kTiny, 1, 0, 0};
  for (int kind = 0; kind < kKinds; ++kind) {
    const TileFigures& f = kFigures[kind];
    const int64_t tiles = tiles_of(kind, M, N);
    for (int splits = 1; splits <= 4 && splits <= kblocks && (splits == 1 || tiles * splits <= kCus); ++splits) {
      const int64_t wgs = tiles * splits;
      const int steps = (kblocks + splits - 1) / splits;
      const double round = wgs > kCus && f.step2 > 0 ? ((wgs + 2 * kCus - 1) / (2 * kCus)) * f.step2 : ((wgs + kCus - 1) / kCus) * f.step;
      const double cost = kLaunch + round * steps + (splits > 1 ? f.join + splits * f.more : 0);
      if (best.cost == 0 || cost < best.cost) best = TilePlan{kind, splits, 0, cost};
    }
  }
  return best;
}

// Past whole rounds of 256 x 256 tiles the channels left over may take a second launch of smaller ones (2048 x 34816 x
// 5120: 1088 tiles, 4.25 rounds).
TilePlan plan_tiles(int M, int N, int kblocks) {
  TilePlan best = plan_single(M, N, kblocks);
  const TileFigures& f = kFigures[kBig];
  const int mblocks = (M - 1) / f.tokens + 1;
  const int64_t rounds = tiles_of(kBig, M, N) / kCus;
  const int64_t main_n = rounds * kCus / mblocks * f.channels;
  if (main_n > 0 && main_n < N) {
    TilePlan tail = plan_single(M, N - (int)main_n, kblocks);
    tail.cost += kLaunch + rounds * f.step * kblocks;
    tail.main_n = (int)main_n;
    if (tail.cost < best.cost) best = tail;
  }
  return best;
}

template <int LAYOUT>
int launch_kind(const Fp8Args& a, int kind, hipStream_t s) {
  switch (kind) {
    case kBig: return launch_tile<LAYOUT, BigTile, 2, 2>(a, s);
    case kMid: return launch_tile<LAYOUT, MidTile, 2, 2>(a, s);
    case kSmall: return launch_tile<LAYOUT, SmallTile, 1, 2>(a, s);
    default: return launch_tile<LAYOUT, TinyTile, 1, 2>(a, s);
  }
}

template <int LAYOUT>
int launch_w8a8(Fp8Args a, const TilePlan& p, hipStream_t s) {
  if (p.main_n > 0) {
    Fp8Args m = a;
    m.N = p.main_n;
    m.ntiles = p.main_n / kTileN;
    m.splits = 1;
    const int st = launch_kind<LAYOUT>(m, kBig, s);
    if (st != QF_OK) return st;
    // the channels from main_n (a multiple of 256) on
    a.w += LAYOUT == QF_LAYOUT_TILED ? (int64_t)m.ntiles * a.ksteps * 1024 : (int64_t)p.main_n * a.ldw;
    a.scale += (int64_t)(p.main_n / kBlock) * a.kblocks;
    if (a.bias != nullptr) a.bias += p.main_n;
    a.y = static_cast<uint8_t*>(a.y) + (int64_t)p.main_n * (a.out_f32 ? 4 : 2);
    a.N -= p.main_n;
    a.ntiles -= m.ntiles;
  }
  a.splits = p.splits;
  return launch_kind<LAYOUT>(a, p.kind, s);
}

int check_product(const uint16_t* x, int64_t ldx, const uint8_t* w, int64_t ldw, int layout, const float* scale,
                  const void* y, int64_t ldy, int out_dtype, int M, int N, int K) {
  if (x == nullptr || w == nullptr || scale == nullptr || y == nullptr || M < 1 || N < 1 || K < 1) return QF_ERR_INVALID_ARG;
  if ((out_dtype != QF_DTYPE_BF16 && out_dtype != QF_DTYPE_F32) || ldx < 0 || (M > 1 && (ldx < K || ldy < N)))
    return QF_ERR_INVALID_ARG;
  if (layout != QF_LAYOUT_ROWMAJOR && layout != QF_LAYOUT_TILED) return QF_ERR_INVALID_ARG;
  if (layout == QF_LAYOUT_ROWMAJOR && N > 1 && ldw < K) return QF_ERR_INVALID_ARG;
  if (K % kStepK || ldx % 8 || !aligned16(x) || !aligned16(w) || (layout == QF_LAYOUT_ROWMAJOR && ldw % 16))
    return QF_ERR_UNSUPPORTED;
  if (ldx > kMaxStride || (layout == QF_LAYOUT_ROWMAJOR && ldw > kMaxStride)) return QF_ERR_UNSUPPORTED;
  if (N > 0x7fffffff - 255 || K > 0x7fffffff - 255 || M > 0x7fffffff - 255) return QF_ERR_UNSUPPORTED;
  return QF_OK;
}

void fill(Fp8Args& a, const uint16_t* x, int64_t ldx, const uint8_t* w, int64_t ldw, const float* scale,
          const uint16_t* bias, void* y, int64_t ldy, int out_dtype, int M, int N, int K) {
  a = Fp8Args{};
  a.x = x;
  a.ldx = ldx;
  a.w = w;
  a.ldw = ldw;
  a.scale = scale;
  a.bias = bias;
  a.y = y;
  a.ldy = ldy;
  a.out_f32 = out_dtype == QF_DTYPE_F32;
  a.vec_out = ldy % 4 == 0 && ((uintptr_t)y & (a.out_f32 ? 15u : 7u)) == 0;
  a.M = M;
  a.N = N;
  a.ksteps = K / kStepK;
  a.kblocks = (K + kBlock - 1) / kBlock;
  a.ntiles = (N + kTileN - 1) / kTileN;
}

// Runs of tiles and splits of K of a decode call.
constexpr int kMaxRuns = QF_W8A16_COUNTER_BYTES / 4;
constexpr int kMaxWaves = 16;   // a workgroup's: with at most 128 registers a lane, as many as a CU holds
constexpr int kDecodeGrid = 256;

struct DecodePlan {
  int waves, runs, splits, blocks, xl;  // blocks: S
  size_t lds;
};

// One workgroup a CU (a second round costs 3.5 us: 272 tiles 11.7 us against 8.3 for 256, K = 5120), so runs as long as that
// takes, and the cheapest number of splits by what a CU then has to fetch (28 bytes a ns under load) and what joining them
// costs: 3 us and 0.25 + 0.06 splits a tile of the run.  Splits pay where x is large beside a run's weights.  Measured at M
// = 16 in us, K = 5120, without a split and with the chosen ones: N = 1280 9.4 -> 7.2, 5120 13.0 -> 12.3, 10240 16.1 (2 splits 17.8);
// 5120 x 8192 20.4 -> 15.2.  x in LDS (xl) where it fits beside the run's partials, else in registers, 3 blocks a
// wavefront at most.
DecodePlan plan_decode(int layout, int M, int ntiles, int kblocks) {
  DecodePlan best = {};
  double best_cost = 0;
  for (int xl : {M <= 4 ? 1 : M <= 8 ? 2 : 4, 0}) {
    const int most_blocks = xl || layout == QF_LAYOUT_ROWMAJOR ? 5 : 3;
    const int most = kMaxWaves * most_blocks;
    const int least = (kblocks + most - 1) / most;
    for (int splits = least; splits < least + 8 && splits <= kblocks; ++splits) {
      const int share = (kblocks + splits - 1) / splits;
      for (int waves : {kMaxWaves, kMaxWaves / 2}) {
        int S = (share + waves - 1) / waves;
        if (S == 4) S = 5;
        if (S > most_blocks) continue;
        const int W = (share + S - 1) / S;
        const int fixed = decode_ring(layout, W) + W * S * xl * 1024;
        const int room = ((int)kMaxLds - 1024 - fixed) / (W * 1024);
        if (room < 1) continue;
        const int slots = splits < kDecodeGrid ? kDecodeGrid / splits : 1;
        const int run = (ntiles + slots - 1) / slots < room ? (ntiles + slots - 1) / slots : room;
        const int64_t runs = (ntiles + run - 1) / run;
        const int64_t rounds = (runs * splits + kDecodeGrid - 1) / kDecodeGrid;
        const double kb = 0.128 * share * (16.0 * run + 2 * M);  // thousand bytes a workgroup
        const double cost = rounds * (kb / 28 * (W < 12 ? 1.04 : 1) + (xl ? 0 : 0.3 * S)) + 3.5 * (rounds - 1) +
                            (splits > 1 ? 3.0 + run * (0.25 + 0.06 * splits) : 0);
        if (best.waves == 0 || cost < best_cost) {
          best_cost = cost;
          best = DecodePlan{W, (int)runs, splits, S, xl, (size_t)fixed + (size_t)run * W * 1024};
        }
      }
    }
  }
  return best;
}

template <int LAYOUT, int S, int XL>
int launch_decode(const Fp8Args& a, const DecodePlan& p, hipStream_t s) {
  static std::atomic<uint64_t> raised{0};
  if (!raise_lds(reinterpret_cast<const void*>(&fp8_decode_kernel<LAYOUT, S, XL>), kMaxLds - 512, raised)) return QF_ERR_HIP;
  hipLaunchKernelGGL((fp8_decode_kernel<LAYOUT, S, XL>), dim3((unsigned)(p.runs * p.splits)), dim3(p.waves * kWave),
                     p.lds, s, a);
  return hipGetLastError() == hipSuccess ? QF_OK : QF_ERR_HIP;
}

template <int LAYOUT, int XL>
int decode_by_blocks(const Fp8Args& a, const DecodePlan& p, hipStream_t s) {
  switch (p.blocks) {
    case 1: return launch_decode<LAYOUT, 1, XL>(a, p, s);
    case 2: return launch_decode<LAYOUT, 2, XL>(a, p, s);
    case 3: return launch_decode<LAYOUT, 3, XL>(a, p, s);
    case 5:
      if constexpr (XL > 0 || LAYOUT == QF_LAYOUT_ROWMAJOR) return launch_decode<LAYOUT, 5, XL>(a, p, s);
      return QF_ERR_UNSUPPORTED;
    default: return QF_ERR_UNSUPPORTED;
  }
}

template <int LAYOUT>
int decode(const Fp8Args& a, const DecodePlan& p, hipStream_t s) {
  switch (p.xl) {
    case 0: return decode_by_blocks<LAYOUT, 0>(a, p, s);
    case 1: return decode_by_blocks<LAYOUT, 1>(a, p, s);
    case 2: return decode_by_blocks<LAYOUT, 2>(a, p, s);
    default: return decode_by_blocks<LAYOUT, 4>(a, p, s);
  }
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

struct W8a8Plan {
  int m_pad, kblocks;
  TilePlan tiles;
  int64_t n_tiles;
  size_t image, counters, partial, total;  // offsets in the workspace; the token scales first
};

int plan_w8a8(int M, int N, int K, W8a8Plan* p) {
  if (M < 1 || N < 1 || K < 1 || K % kStepK || K > QF_FP8_MAX_W8A8_K || N > 0x7fffffff - 255 || M > 0x7fffffff - 255 ||
      !grid_fits((M + 15) / 16, 256))
    return QF_ERR_UNSUPPORTED;
  p->kblocks = (K + kBlock - 1) / kBlock;
  p->m_pad = (M + kTokenPad - 1) / kTokenPad * kTokenPad;
  p->tiles = plan_tiles(M, N, p->kblocks);
  p->n_tiles = p->tiles.splits > 1 ? tiles_of(p->tiles.kind, M, N - p->tiles.main_n) : 0;
  p->image = round256((size_t)p->kblocks * p->m_pad * 4);
  p->counters = p->image + round256((size_t)((M + 15) / 16) * 16 * p->kblocks * kBlock);
  p->partial = p->counters + round256((size_t)p->n_tiles * 4);
  p->total = p->partial + (size_t)p->n_tiles * p->tiles.splits * kFigures[p->tiles.kind].channels * kFigures[p->tiles.kind].tokens * 4;
  return QF_OK;
}

}  // namespace qfb

using namespace qfb;

extern "C" {

int qf_block_abi_version(void) { return QF_BLOCK_ABI_VERSION; }

size_t qf_fp8_w8a16_workspace_bytes(int M, int N, int K, int layout) {
  if (M < 1 || M > QF_FP8_MAX_DECODE_M || N < 1 || K < kStepK || K % kStepK || N > 0x7fffffff - 255 ||
      (layout != QF_LAYOUT_ROWMAJOR && layout != QF_LAYOUT_TILED))
    return 0;
  const int ntiles = (N - 1) / kTileN + 1;
  const int splits = plan_decode(layout, M, ntiles, (K - 1) / kBlock + 1).splits;
  return splits == 1 ? 0 : QF_W8A16_COUNTER_BYTES + (size_t)splits * ntiles * 1024;
}

int qf_fp8_w8a16_gemm(const uint16_t* x, int64_t ldx, const uint8_t* w, int64_t ldw, int layout, const float* scale,
                      const uint16_t* bias, void* y, int64_t ldy, int out_dtype, int M, int N, int K, void* workspace,
                      size_t workspace_bytes, void* stream) {
  const int st = check_product(x, ldx, w, ldw, layout, scale, y, ldy, out_dtype, M, N, K);
  if (st != QF_OK) return st;
  if (M > QF_FP8_MAX_DECODE_M) return QF_ERR_UNSUPPORTED;
  Fp8Args a;
  fill(a, x, ldx, w, ldw, scale, bias, y, ldy, out_dtype, M, N, K);
  const DecodePlan p = plan_decode(layout, M, a.ntiles, a.kblocks);
  if (p.waves == 0) return QF_ERR_UNSUPPORTED;
  if (p.splits > 1) {
    if (p.runs > kMaxRuns || (int64_t)p.runs * p.splits > 0x7fffffff) return QF_ERR_UNSUPPORTED;
    if (workspace == nullptr || workspace_bytes < qf_fp8_w8a16_workspace_bytes(M, N, K, layout) || !aligned16(workspace))
      return QF_ERR_WORKSPACE;
    a.counters = static_cast<unsigned*>(workspace);
    a.counter_stride = p.runs * kCounterStride <= kMaxRuns ? kCounterStride : 1;
    a.partial = reinterpret_cast<uint64_t*>(static_cast<uint8_t*>(workspace) + QF_W8A16_COUNTER_BYTES);
  }
  a.runs = p.runs;
  a.splits = p.splits;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return layout == QF_LAYOUT_TILED ? decode<QF_LAYOUT_TILED>(a, p, s) : decode<QF_LAYOUT_ROWMAJOR>(a, p, s);
}

int qf_quantize_tokens_fp8(const uint16_t* x, int64_t ldx, int M, int K, uint8_t* xq, int64_t ldq, float* s_a,
                           void* stream) {
  if (x == nullptr || xq == nullptr || s_a == nullptr || M < 1 || K < 1 || (M > 1 && (ldx < K || ldq < K)))
    return QF_ERR_INVALID_ARG;
  if (K % kStepK || ldx % 8 || ldq % 8 || !aligned16(x) || ((uintptr_t)xq & 7) || M > 0x7fffffff - 255)
    return QF_ERR_UNSUPPORTED;
  const int kblocks = (K + kBlock - 1) / kBlock;
  if (kblocks > 65535 * kQuantBlocks || !grid_fits((M + 15) / 16, 256)) return QF_ERR_UNSUPPORTED;
  const QuantArgs q = {x, ldx, xq, ldq, s_a, 0, M, K / kStepK, kblocks, nullptr, 0};
  hipLaunchKernelGGL(quantize_tokens_fp8_kernel<false>, dim3((unsigned)((M + 15) / 16), (unsigned)((kblocks + kQuantBlocks - 1) / kQuantBlocks)),
                     dim3(256), 0, static_cast<hipStream_t>(stream), q);
  return hipGetLastError() == hipSuccess ? QF_OK : QF_ERR_HIP;
}

size_t qf_fp8_w8a8_workspace_bytes(int M, int N, int K) {
  W8a8Plan p;
  return plan_w8a8(M, N, K, &p) == QF_OK ? p.total : 0;
}

int qf_fp8_w8a8_linear(const uint16_t* x, int64_t ldx, const uint8_t* w, int64_t ldw, int layout, const float* scale,
                       const uint16_t* bias, void* y, int64_t ldy, int out_dtype, int M, int N, int K,
                       void* workspace, size_t workspace_bytes, void* stream) {
  int st = check_product(x, ldx, w, ldw, layout, scale, y, ldy, out_dtype, M, N, K);
  if (st != QF_OK) return st;
  W8a8Plan p;
  st = plan_w8a8(M, N, K, &p);
  if (st != QF_OK) return st;
  if (workspace == nullptr || workspace_bytes < p.total || !aligned16(workspace)) return QF_ERR_WORKSPACE;
  Fp8Args a;
  fill(a, x, ldx, w, ldw, scale, bias, y, ldy, out_dtype, M, N, K);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.s_tok = reinterpret_cast<const float*>(ws);
  a.xt = ws + p.image;
  a.m_pad = p.m_pad;
  a.counters = reinterpret_cast<unsigned*>(ws + p.counters);
  a.partial = reinterpret_cast<uint64_t*>(ws + p.partial);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const QuantArgs q = {x, ldx, ws + p.image, 0, reinterpret_cast<float*>(ws), p.m_pad, M, a.ksteps, a.kblocks, a.counters, (int)p.n_tiles};
  hipLaunchKernelGGL(quantize_tokens_fp8_kernel<true>, dim3((unsigned)((M + 15) / 16), (unsigned)((a.kblocks + kQuantBlocks - 1) / kQuantBlocks)),
                     dim3(256), 0, s, q);
  if (hipGetLastError() != hipSuccess) return QF_ERR_HIP;
  return layout == QF_LAYOUT_TILED ? launch_w8a8<QF_LAYOUT_TILED>(a, p.tiles, s) : launch_w8a8<QF_LAYOUT_ROWMAJOR>(a, p.tiles, s);
}

}  // extern "C"
