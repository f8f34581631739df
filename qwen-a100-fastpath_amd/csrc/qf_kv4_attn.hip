// qf_kv4_attn.hip — attention over a paged cache held in 4 bits (gfx950).
//
// A wavefront takes 16 RT packed query rows (token, head of the kv head's group) and walks over positions in steps of 32, two
// cache records: S^T = K Q^T on v_mfma_f32_16x16x32_bf16 with the keys as the A operand, an online softmax in base 2, and
// O^T += V^T P^T on the same instruction.  The records are laid out so that a lane's 16 bytes are its part of an operand: the
// codes go from global memory to registers in whole KiB, without LDS, and are widened there (a scale and two codes an
// instruction).  A lane's accumulator of S^T holds 4 positions of one row for each record, which are its 8 values of the B
// operand P^T: the softmax weights never leave the lane.
//
//   attn_split_kernel    few rows (decode, verification): the positions of a request are split over workgroups and, in a
//                        workgroup, over 4 wavefronts, whose states meet in LDS; attn_combine_kernel adds the splits
//   attn_tile_kernel     many rows (prompt chunks): each wavefront its own rows, all their positions
#include "qf_kv4_common.h"

#include <mutex>

namespace qfk {

constexpr int kAttnThreads = 256;
constexpr int kAttnWaves = kAttnThreads / kWave;
constexpr int kStep = 2 * kTile;  // positions of a step
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMinChunk = 4 * kStep;

struct AttnArgs {
  const uint16_t* q;
  int64_t sq_t, sq_h;
  uint16_t* out;
  int64_t so_t, so_h;
  const uint8_t* cache;
  int64_t stride;
  int64_t num_blocks;
  const int32_t* bt;
  int64_t sbt;
  const int32_t *seq_lens, *cu_q;
  int B, Q, T, H, HKV, G, page, max_blocks;
  int rows;     // of a request: at most Q * G
  int workers;  // split kernel: positions are split so that about this many workgroups a kv head share the batch
  float qk_scale;
  Divisor by_g, by_page;
  float* o_part;   // [HKV][slots][rows][D]
  float2* ml_part; // [HKV][slots][rows]: exponent reference, sum
  int2* plan;      // [B]: first slot and slots of a request
  int slots;
};

// A request's tokens and positions, kept inside the tables.
struct Request {
  int tok0, n, seq;
};
__device__ __forceinline__ Request request(const AttnArgs& a, int b) {
  Request r;
  if (a.cu_q != nullptr) {
    r.tok0 = min(max(a.cu_q[b], 0), a.T);
    r.n = min(min(max(a.cu_q[b + 1] - r.tok0, 0), a.Q), a.T - r.tok0);
  } else {
    r.tok0 = b * a.Q;
    r.n = a.Q;
  }
  r.seq = max(a.seq_lens[b], 0);
  if ((int64_t)a.max_blocks * a.page < r.seq) r.seq = a.max_blocks * a.page;
  return r;
}

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ float quarters_max(float v) {  // over the 4 lanes l, l^16, l^32, l^48
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float quarters_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// A lane's bytes of two records (a step).
template <int D>
struct StepData {
  static constexpr int kDwords = D < 128 ? 2 : 4;  // of a half's keys, and of its values
  static constexpr int kHalves = Record<D>::kHalves;
  uint32_t k[2][kHalves][kDwords], v[2][kHalves][kDwords], ks[2][kHalves], vs[2][kHalves];
};

template <int D, int RT>
struct Walk {
  using R = Record<D>;
  using Data = StepData<D>;
  static constexpr int kHalves = R::kHalves;
  static constexpr int kDwords = Data::kDwords;
  static constexpr int kKSteps = D / 32;          // matrix instructions of a score
  static constexpr int kDTiles = D / 16;          // of the output
  static constexpr int kPerHalf = R::kWidth;      // d tiles of a half: value n of each lane's run
  static constexpr float kRescale = 8.f;

  const AttnArgs& a;
  int lane, l16, qg;
  bf16x8_t qf[RT][kKSteps];
  int last[RT];   // last visible position of the lane's row
  int diag;       // positions from here on are not seen by every row of the wavefront
  float m[RT], l[RT];
  f32x4_t o[RT][kDTiles];
  const uint8_t* base;   // the kv head's first record in block 0
  const int32_t* bt_row;

  __device__ __forceinline__ explicit Walk(const AttnArgs& args) : a(args) {
    lane = threadIdx.x % kWave;
    l16 = lane & 15;
    qg = lane >> 4;
  }

  // Rows r0 .. r0 + 16 RT - 1 of request r (rows past its last repeat it).
  __device__ __forceinline__ void start(const Request& r, int b, int hkv, int r0) {
    const int R_b = r.n * a.G;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int row = min(r0 + rt * 16 + l16, R_b - 1);
      const int qi = divide(row, a.by_g);
      const uint16_t* p = a.q + (int64_t)(r.tok0 + qi) * a.sq_t + (int64_t)(hkv * a.G + (row - qi * a.G)) * a.sq_h;
#pragma unroll
      for (int s = 0; s < kKSteps; ++s)
        qf[rt][s] = *reinterpret_cast<const bf16x8_t*>(p + s / kDwords * 128 + qg * 8 * kDwords + s % kDwords * 8);
      last[rt] = r.seq - r.n + qi;
      m[rt] = -__builtin_inff();
      l[rt] = 0.f;
#pragma unroll
      for (int u = 0; u < kDTiles; ++u) o[rt][u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    diag = r.seq - r.n + divide(min(r0, R_b - 1), a.by_g) + 1;
    base = a.cache + (int64_t)hkv * (a.page / kTile) * R::kBytes;
    bt_row = a.bt + (int64_t)b * a.sbt;
  }

  // The record that holds position pos (a multiple of 16), the same in every lane.
  __device__ __forceinline__ const uint8_t* record(int pos) const {
    const int pg = divide(pos, a.by_page);
    int64_t block = bt_row[pg];
    block = block < 0 ? 0 : block >= a.num_blocks ? a.num_blocks - 1 : block;
    return base + block * a.stride + (pos - pg * a.page) / kTile * R::kBytes;
  }

  __device__ __forceinline__ void load(Data& s, const uint8_t* r0, const uint8_t* r1) const {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint8_t* r = t == 0 ? r0 : r1;
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        const uint8_t* kp = r + l16 * (D / 2) + h * 64 + qg * (4 * kDwords);
        const uint8_t* vp = r + R::kValues + h * 1024 + lane * (4 * kDwords);
        if constexpr (kDwords == 4) {
          const u32x4_t kk = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(kp));
          const u32x4_t vv = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(vp));
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s.k[t][h][i] = kk[i];
            s.v[t][h][i] = vv[i];
          }
          s.ks[t][h] = r[R::kKeyScales + (4 * h + qg) * kTile + l16];
          s.vs[t][h] = *reinterpret_cast<const uint32_t*>(r + R::kValueScales + (4 * h + l16 / 4) * kTile + 4 * qg);
        } else {
          const u32x2_t kk = __builtin_nontemporal_load(reinterpret_cast<const u32x2_t*>(kp));
          const u32x2_t vv = __builtin_nontemporal_load(reinterpret_cast<const u32x2_t*>(vp));
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            s.k[t][h][i] = kk[i];
            s.v[t][h][i] = vv[i];
          }
          s.ks[t][h] = r[R::kKeyScales + qg / 2 * kTile + l16];
          s.vs[t][h] = *reinterpret_cast<const uint32_t*>(r + R::kValueScales + l16 / 8 * kTile + 4 * qg);
        }
      }
    }
  }

  // A value's block of NaN at a position that some rows see and others do not: the product would give it to all rows.  Where a
  // step holds one, its scales are cleared for the product and the rows that see it are made NaN here.
  __device__ __forceinline__ void masked_nan(Data& s, int pos, const uint8_t* r0, const uint8_t* r1) {
    bool any = false;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) any |= (s.vs[t][h] >> (8 * i) & 255u) == 255u;
    if (!__any(any)) return;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if ((s.vs[t][h] >> (8 * i) & 255u) == 255u) {
            s.vs[t][h] &= ~(255u << (8 * i));
            s.vs[t][h] |= 127u << (8 * i);
            clear(s, t, h, i);
          }
    // the lane's outputs are values 128 h + 32 qg .. of its rows (D = 64: 16 qg ..): one block each
    for (int p = 0; p < kStep; ++p) {
      const uint8_t* r = (p < kTile ? r0 : r1) + p % kTile;
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        const uint32_t byte = r[R::kValueScales + (kDwords == 4 ? 4 * h + qg : qg / 2) * kTile];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          if (byte == 255u && pos + p <= last[rt]) {
#pragma unroll
            for (int u = 0; u < kPerHalf; ++u) o[rt][h * kPerHalf + u] = o[rt][h * kPerHalf + u] + __builtin_nanf("");
          }
      }
    }
  }

  // The codes of position 4 qg + i of record t, half h: +0.
  __device__ __forceinline__ void clear(Data& s, int t, int h, int i) const {
    if constexpr (kDwords == 4) {
      s.v[t][h][i] = 0;
    } else {
      s.v[t][h][i / 2] &= i % 2 ? 0xffffu : 0xffff0000u;
    }
  }

  // Positions pos .. pos + 31, those from `end` on hold nothing.  r0, r1: the records (read again in a rare case only).
  __device__ __forceinline__ void step(Data& s, int pos, int end, const uint8_t* r0, const uint8_t* r1) {
    f32x4_t sc[RT][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) sc[rt][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        const float ks = scale_f32(s.ks[t][h]);
#pragma unroll
        for (int c = 0; c < kDwords; ++c) {
          const bf16x8_t kf = __builtin_bit_cast(bf16x8_t, widen8(s.k[t][h][c], ks));
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
            sc[rt][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[rt][h * kDwords + c], sc[rt][t], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int t = 0; t < 2; ++t) sc[rt][t] *= a.qk_scale;
    if (pos + kStep > diag || pos + kStep > end) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int p0 = pos + t * kTile + 4 * qg;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            sc[rt][t][i] = p0 + i < end && p0 + i <= last[rt] ? sc[rt][t][i] : -__builtin_inff();
        // what stands behind the end may be anything, a NaN among it: weight 0 times 0
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (p0 + i >= end) {
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
              s.vs[t][h] &= ~(255u << (8 * i));
              s.vs[t][h] |= 127u << (8 * i);
              clear(s, t, h, i);
            }
          }
      }
      masked_nan(s, pos, r0, r1);
    }
    // The row's exponent reference moves only when a score exceeds it by 2^8: the weights stay below that, and the
    // accumulators are rarely rescaled.  The result is that of the running maximum up to rounding.
    bool above = false;
    float mx[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      mx[rt] = fmaxf(fmaxf(fmaxf(sc[rt][0][0], sc[rt][0][1]), fmaxf(sc[rt][0][2], sc[rt][0][3])),
                     fmaxf(fmaxf(sc[rt][1][0], sc[rt][1][1]), fmaxf(sc[rt][1][2], sc[rt][1][3])));
      above |= mx[rt] > m[rt] + kRescale;
    }
    if (__any(above)) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const float top = fmaxf(m[rt], quarters_max(mx[rt]));
        const float keep = fast_exp2(m[rt] - (top == -__builtin_inff() ? 0.f : top));
        m[rt] = top;
        l[rt] *= keep;
#pragma unroll
        for (int u = 0; u < kDTiles; ++u) o[rt][u] *= keep;
      }
    }
    bf16x8_t pf[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const float ref = m[rt] == -__builtin_inff() ? 0.f : m[rt];  // a row that has seen nothing yet
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = fast_exp2(sc[rt][i / 4][i % 4] - ref);
      l[rt] += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
      pf[rt] = __builtin_bit_cast(bf16x8_t, pack8(w));
    }
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      float vs[2][4];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) vs[t][i] = scale_f32(s.vs[t][h] >> (8 * i) & 255u);
      auto values = [&](auto byte) {  // value n = 2 byte and 2 byte + 1 of the lane's run, as operands over the 8 positions
        constexpr int kB = decltype(byte)::value;
        u32x4_t even, odd;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          uint32_t x[4];
          if constexpr (kDwords == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = widen2<kB>(s.v[t][h][i], vs[t][i]);
          } else {
            x[0] = widen2<kB>(s.v[t][h][0], vs[t][0]);
            x[1] = widen2<kB + 2>(s.v[t][h][0], vs[t][1]);
            x[2] = widen2<kB>(s.v[t][h][1], vs[t][2]);
            x[3] = widen2<kB + 2>(s.v[t][h][1], vs[t][3]);
          }
          even[2 * t] = __builtin_amdgcn_perm(x[1], x[0], 0x05040100);
          even[2 * t + 1] = __builtin_amdgcn_perm(x[3], x[2], 0x05040100);
          odd[2 * t] = __builtin_amdgcn_perm(x[1], x[0], 0x07060302);
          odd[2 * t + 1] = __builtin_amdgcn_perm(x[3], x[2], 0x07060302);
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          f32x4_t& oe = o[rt][h * kPerHalf + 2 * kB];
          f32x4_t& oo = o[rt][h * kPerHalf + 2 * kB + 1];
          oe = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, even), pf[rt], oe, 0, 0, 0);
          oo = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, odd), pf[rt], oo, 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      };
      values(std::integral_constant<int, 0>{});
      values(std::integral_constant<int, 1>{});
      if constexpr (kDwords == 4) {
        values(std::integral_constant<int, 2>{});
        values(std::integral_constant<int, 3>{});
      }
    }
  }

  // Steps first, first + by, ... below n_steps, of positions from `begin` on.
  __device__ __forceinline__ void run(int begin, int end, int first, int by) {
    const int n_steps = (end - begin + kStep - 1) / kStep;
    const int last_tile = (end - 1) / kTile * kTile;
    if (first >= n_steps) return;
    Data s[2];
    const uint8_t *r0[2], *r1[2];
    auto fetch = [&](int i, int u) {
      const int pos = begin + min(i, n_steps - 1) * kStep;
      r0[u] = record(pos);
      r1[u] = record(min(pos + kTile, last_tile));
      load(s[u], r0[u], r1[u]);
    };
    fetch(first, 0);
#pragma unroll 1
    for (int i = first; i < n_steps; i += 2 * by) {
      fetch(i + by, 1);
      step(s[0], begin + i * kStep, end, r0[0], r1[0]);
      fetch(i + 2 * by, 0);
      if (i + by < n_steps) step(s[1], begin + (i + by) * kStep, end, r0[1], r1[1]);
    }
  }

  // The lane's outputs of its row in row tile rt: value v of the row is o[rt][h kPerHalf + n][i] with v = 16 kWidth h +
  // kWidth (4 qg + i) + n.
  __device__ __forceinline__ int value_at(int h, int i) const { return 16 * R::kWidth * h + R::kWidth * (4 * qg + i); }

  __device__ __forceinline__ void write(const Request& r, int hkv, int row, int rt) const {
    const int qi = divide(row, a.by_g);
    uint16_t* p = a.out + (int64_t)(r.tok0 + qi) * a.so_t + (int64_t)(hkv * a.G + (row - qi * a.G)) * a.so_h;
    const float inv = last[rt] < 0 ? 0.f : 1.f / l[rt];
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t w[kPerHalf / 2];
#pragma unroll
        for (int n = 0; n < kPerHalf / 2; ++n)
          w[n] = pack_bf16(o[rt][h * kPerHalf + 2 * n][i] * inv, o[rt][h * kPerHalf + 2 * n + 1][i] * inv);
        if constexpr (kPerHalf == 8) {
          *reinterpret_cast<u32x4_t*>(p + value_at(h, i)) = u32x4_t{w[0], w[1], w[2], w[3]};
        } else {
          *reinterpret_cast<u32x2_t*>(p + value_at(h, i)) = u32x2_t{w[0], w[1]};
        }
      }
  }
};

// The batch's split: one chunk length for all requests, so that about `workers` chunks hold them (at least kMinChunk
// positions), and one more chunk a request for its end: at most workers + B slots are used.  Workgroup `slot` finds its
// request; lane-parallel over 64 requests at a time.  false: a slot of no request.
struct Place {
  int b, split, splits, first, chunk;
};
__device__ __forceinline__ bool place_of(const AttnArgs& a, int slot, Place& p) {
  const int lane = threadIdx.x % kWave;
  uint64_t total = 0;
  for (int base = 0; base < a.B; base += kWave) {
    const int b = base + lane;
    if (b < a.B) {
      const Request r = request(a, b);
      total += r.n > 0 ? (uint32_t)r.seq : 0u;
    }
  }
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const uint32_t lo = __shfl_xor((int)(uint32_t)total, d), hi = __shfl_xor((int)(uint32_t)(total >> 32), d);
    total += ((uint64_t)hi << 32) | lo;
  }
  const uint64_t even = (total + a.workers - 1) / (uint32_t)a.workers;
  const uint64_t chunk = (max(even, (uint64_t)kMinChunk) + kStep - 1) / kStep * kStep;
  p.chunk = chunk > 0x7fffffe0 ? 0x7fffffe0 : (int)chunk;
  int before = 0;
  bool found = false;
  for (int base = 0; base < a.B; base += kWave) {
    const int b = base + lane;
    int n = 0;
    if (b < a.B) {
      const Request r = request(a, b);
      n = r.n > 0 ? max((int)(((uint32_t)r.seq + (uint32_t)(p.chunk - 1)) / (uint32_t)p.chunk), 1) : 0;
    }
    const int upto = before + wave_scan(n);
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < kWave && b < a.B) a.plan[b] = make_int2(upto - n, n);
    const uint64_t mine = __ballot(slot >= upto - n && slot < upto);
    if (mine != 0 && !found) {
      const int i = __builtin_ctzll(mine);
      p.b = base + i;
      p.first = __builtin_amdgcn_readlane(upto - n, i);
      p.splits = __builtin_amdgcn_readlane(n, i);
      p.split = slot - p.first;
      found = true;
      if (blockIdx.x != 0) break;
    }
    before = __builtin_amdgcn_readlane(upto, kWave - 1);
  }
  return found;
}

// RG groups of 16 RT rows; the wavefronts of a group share its positions.
template <int D, int RT, int RG>
__global__ __launch_bounds__(kAttnThreads) void attn_split_kernel(AttnArgs a) {
  using W = Walk<D, RT>;
  constexpr int kShare = kAttnWaves / RG;  // wavefronts of a row group
  extern __shared__ __align__(16) float lds[];  // [2][RT][D / 16][64 lanes x 4]
  __shared__ float row_m[kAttnWaves][RT][16], row_l[kAttnWaves][RT][16];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int rg = wave % RG, share = wave / RG;
  const int hkv = blockIdx.y;
  Place p;
  if (!place_of(a, blockIdx.x, p)) return;
  p.b = __builtin_amdgcn_readfirstlane(p.b);
  p.split = __builtin_amdgcn_readfirstlane(p.split);
  p.splits = __builtin_amdgcn_readfirstlane(p.splits);
  p.chunk = __builtin_amdgcn_readfirstlane(p.chunk);
  const Request r = request(a, p.b);
  W w(a);
  w.start(r, p.b, hkv, rg * RT * 16);
  const int begin = p.split * p.chunk;  // below 2^31: split s > 0 starts inside the sequence
  const int end = min(r.seq - begin, p.chunk) + begin;
  if (begin < end) w.run(begin, end, share, kShare);

  // ---- the wavefronts' states against their common reference ----
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) w.l[rt] = quarters_sum(w.l[rt]);
  if (w.qg == 0) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) row_m[wave][rt][w.l16] = w.m[rt];
  }
  __syncthreads();
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    float top = row_m[rg][rt][w.l16];
#pragma unroll
    for (int i = 1; i < kShare; ++i) top = fmaxf(top, row_m[i * RG + rg][rt][w.l16]);
    const float keep = fast_exp2(w.m[rt] - (top == -__builtin_inff() ? 0.f : top));
    w.m[rt] = top;
    w.l[rt] *= keep;
#pragma unroll
    for (int u = 0; u < W::kDTiles; ++u) w.o[rt][u] *= keep;
    if (w.qg == 0) row_l[wave][rt][w.l16] = w.l[rt];
  }
  auto at = [&](int half, int rt, int u) {
    return reinterpret_cast<f32x4_t*>(lds) + ((half * RT + rt) * W::kDTiles + u) * kWave + w.lane;
  };
#pragma unroll
  for (int from = kAttnWaves / 2; from >= RG; from /= 2) {  // wavefronts from .. 2 from - 1 hand theirs to 0 .. from - 1
    if (wave >= from && wave < 2 * from) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int u = 0; u < W::kDTiles; ++u) *at(wave - from, rt, u) = w.o[rt][u];
    }
    __syncthreads();
    if (wave < from) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int u = 0; u < W::kDTiles; ++u) w.o[rt][u] += *at(wave, rt, u);
    }
    if (from > RG) __syncthreads();
  }
  if (share != 0) return;
  const int rows = r.n * a.G;
  const int64_t part = ((int64_t)hkv * a.slots + blockIdx.x) * a.rows;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int row = (rg * RT + rt) * 16 + w.l16;
    w.l[rt] = row_l[rg][rt][w.l16];
#pragma unroll
    for (int i = 1; i < kShare; ++i) w.l[rt] += row_l[i * RG + rg][rt][w.l16];
    if (row >= rows) continue;
    if (p.splits == 1) {
      w.write(r, hkv, row, rt);
      continue;
    }
    float* to = a.o_part + (part + row) * D;
#pragma unroll
    for (int h = 0; h < W::kHalves; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int n = 0; n < W::kPerHalf; n += 4) {
          const int u = h * W::kPerHalf + n;
          *reinterpret_cast<f32x4_t*>(to + w.value_at(h, i) + n) =
              f32x4_t{w.o[rt][u][i], w.o[rt][u + 1][i], w.o[rt][u + 2][i], w.o[rt][u + 3][i]};
        }
    if (w.qg == 0) a.ml_part[part + row] = make_float2(w.m[rt], w.l[rt]);
  }
}

// A workgroup a packed row: D / 4 threads a split, the splits over 256 / (D / 4) groups of threads, then the groups in LDS.
template <int D>
__global__ __launch_bounds__(kAttnThreads) void attn_combine_kernel(AttnArgs a) {
  constexpr int kLanes = D / 4, kGroups = kAttnThreads / kLanes;
  __shared__ float sm_m[kGroups], sm_l[kGroups];
  __shared__ __align__(16) f32x4_t sm_o[kGroups][kLanes];
  const int b = blockIdx.x, row = blockIdx.y, hkv = blockIdx.z;
  const Request r = request(a, b);
  const int2 place = a.plan[b];
  if (row >= r.n * a.G || place.y < 2) return;
  const int g = threadIdx.x / kLanes, j = threadIdx.x % kLanes;
  const int64_t part = ((int64_t)hkv * a.slots + place.x) * a.rows + row;
  float m = -__builtin_inff(), l = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  for (int s = g; s < place.y; s += kGroups) {
    const float2 ml = a.ml_part[part + (int64_t)s * a.rows];
    const f32x4_t v = *reinterpret_cast<const f32x4_t*>(a.o_part + (part + (int64_t)s * a.rows) * D + 4 * j);
    const float top = fmaxf(m, ml.x);
    const float ref = top == -__builtin_inff() ? 0.f : top;
    const float keep = fast_exp2(m - ref), w = fast_exp2(ml.x - ref);
    o = o * keep + v * w;
    l = l * keep + ml.y * w;
    m = top;
  }
  if (j == 0) {
    sm_m[g] = m;
    sm_l[g] = l;
  }
  sm_o[g][j] = o;
  __syncthreads();
  if (g != 0) return;
  float top = sm_m[0];
#pragma unroll
  for (int i = 1; i < kGroups; ++i) top = fmaxf(top, sm_m[i]);
  const float ref = top == -__builtin_inff() ? 0.f : top;
  o = f32x4_t{0.f, 0.f, 0.f, 0.f};
  l = 0.f;
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    const float w = fast_exp2(sm_m[i] - ref);
    o += sm_o[i][j] * w;
    l += sm_l[i] * w;
  }
  const int qi = divide(row, a.by_g);
  const float inv = r.seq - r.n + qi < 0 ? 0.f : 1.f / l;
  uint16_t* to = a.out + (int64_t)(r.tok0 + qi) * a.so_t + (int64_t)(hkv * a.G + (row - qi * a.G)) * a.so_h + 4 * j;
  *reinterpret_cast<u32x2_t*>(to) = u32x2_t{pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv)};
}

// Rows 32 (4 x + wavefront) .. + 31 of request z, kv head y.
constexpr int kTileRT = 2;
template <int D>
__global__ __launch_bounds__(kAttnThreads) void attn_tile_kernel(AttnArgs a) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int hkv = blockIdx.y, b = blockIdx.z;
  const Request r = request(a, b);
  const int r0 = (blockIdx.x * kAttnWaves + wave) * 16 * kTileRT;
  if (r0 >= r.n * a.G) return;
  Walk<D, kTileRT> w(a);
  w.start(r, b, hkv, r0);
  const int last_row = min(r0 + 16 * kTileRT, r.n * a.G) - 1;
  const int end = max(r.seq - r.n + divide(last_row, a.by_g) + 1, 0);
  if (end > 0) w.run(0, end, 0, 1);
#pragma unroll
  for (int rt = 0; rt < kTileRT; ++rt) {
    w.l[rt] = quarters_sum(w.l[rt]);
    const int row = r0 + rt * 16 + w.l16;
    if (row < r.n * a.G) w.write(r, hkv, row, rt);
  }
}

typedef void (*AttnFn)(AttnArgs);

template <int D>
AttnFn split_kernel(int rt) {
  return rt == 1 ? &attn_split_kernel<D, 1, 1> : rt == 2 ? &attn_split_kernel<D, 2, 1> : &attn_split_kernel<D, 2, 2>;
}

int compute_units() {
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

// How a call runs: its launches and the parts of its workspace.
struct Plan {
  bool split;
  int workers, slots, rows;
  size_t o, ml, plan, bytes;  // offsets and size of the workspace
};
size_t round256(size_t n) { return (n + 255) / 256 * 256; }

Plan plan_of(const qf_kv4_attention_args& u) {
  Plan p = {};
  const int64_t rows = (int64_t)u.q_len * (u.num_heads / u.num_kv_heads);
  p.split = rows <= QF_KV4_MAX_ROWS;
  if (!p.split) return p;
  p.rows = (int)rows;
  const int cus = compute_units();
  p.workers = (cus + u.num_kv_heads - 1) / u.num_kv_heads;
  p.slots = p.workers + u.num_reqs;
  size_t n = QF_W8A16_COUNTER_BYTES;
  const size_t parts = (size_t)u.num_kv_heads * p.slots * p.rows;
  p.o = n;
  n += round256(parts * u.head_size * sizeof(float));
  p.ml = n;
  n += round256(parts * sizeof(float2));
  p.plan = n;
  p.bytes = n + round256((size_t)u.num_reqs * sizeof(int2));
  return p;
}

bool sizes_fit(const qf_kv4_attention_args& u) {
  return u.num_reqs >= 1 && u.q_len >= 1 && u.num_heads >= 1 && u.num_kv_heads >= 1 && u.num_heads % u.num_kv_heads == 0 &&
         (u.head_size == 64 || u.head_size == 128 || u.head_size == 256) &&
         (int64_t)u.q_len * (u.num_heads / u.num_kv_heads) <= 0x3fffffff && u.num_kv_heads <= 65535 && u.num_reqs <= 65535;
}

std::atomic<uint64_t> g_raised[3][5];

int launch(AttnFn fn, dim3 grid, size_t lds, std::atomic<uint64_t>& raised, hipStream_t s, const AttnArgs& a) {
  if (lds + 4096 > kDefaultLds && !raise_lds(reinterpret_cast<const void*>(fn), (int)lds, raised)) return QF_ERR_HIP;
  hipLaunchKernelGGL(fn, grid, dim3(kAttnThreads), lds, s, a);
  return hipGetLastError() == hipSuccess ? QF_OK : QF_ERR_HIP;
}

}  // namespace qfk

using namespace qfk;

extern "C" size_t qf_kv4_attention_workspace_bytes(const qf_kv4_attention_args* args) {
  return args && sizes_fit(*args) ? plan_of(*args).bytes : 0;
}

extern "C" int qf_kv4_attention(const qf_kv4_attention_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  if (!args) return QF_ERR_INVALID_ARG;
  const qf_kv4_attention_args& u = *args;
  if (!u.query.data || !u.out.data || !u.cache || !u.block_table || !u.seq_lens || u.num_blocks < 1 || u.max_blocks < 1 ||
      u.bt_stride < 0 || u.num_tokens < 1 || u.num_reqs < 1 || u.q_len < 1 || u.num_heads < 1 || u.num_kv_heads < 1 ||
      u.page_size < 1 || !(u.scale == u.scale) || (!u.cu_q && (int64_t)u.num_reqs * u.q_len > u.num_tokens))
    return QF_ERR_INVALID_ARG;
  if (!sizes_fit(u) || u.page_size % kTile || u.cache_stride % 16 || !aligned16(u.cache) ||
      u.cache_stride < (int64_t)u.num_kv_heads * (u.page_size / kTile) * 17 * u.head_size)
    return QF_ERR_UNSUPPORTED;
  for (const qf_heads* h : {&u.query, &u.out})
    if (h->stride_tok < 0 || h->stride_head < 0 || h->stride_tok % 8 || h->stride_head % 8 || !aligned16(h->data))
      return QF_ERR_UNSUPPORTED;
  const Plan p = plan_of(u);
  if (p.bytes && (!workspace || workspace_bytes < p.bytes || !aligned16(workspace))) return QF_ERR_WORKSPACE;
  uint8_t* const ws = static_cast<uint8_t*>(workspace);
  AttnArgs a = {};
  a.q = u.query.data;
  a.sq_t = u.query.stride_tok;
  a.sq_h = u.query.stride_head;
  a.out = u.out.data;
  a.so_t = u.out.stride_tok;
  a.so_h = u.out.stride_head;
  a.cache = static_cast<const uint8_t*>(u.cache);
  a.stride = u.cache_stride;
  a.num_blocks = u.num_blocks;
  a.bt = u.block_table;
  a.sbt = u.bt_stride;
  a.seq_lens = u.seq_lens;
  a.cu_q = u.cu_q;
  a.B = u.num_reqs;
  a.Q = u.q_len;
  a.T = u.num_tokens;
  a.H = u.num_heads;
  a.HKV = u.num_kv_heads;
  a.G = u.num_heads / u.num_kv_heads;
  a.page = u.page_size;
  a.max_blocks = u.max_blocks;
  a.rows = p.rows;
  a.workers = p.workers;
  a.slots = p.slots;
  a.qk_scale = u.scale * kLog2e;
  a.by_g = divisor(a.G);
  a.by_page = divisor(u.page_size);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int D = u.head_size, di = D == 64 ? 0 : D == 128 ? 1 : 2;
  if (!p.split) {
    const int64_t rows = (int64_t)u.q_len * a.G;
    const int per = kAttnWaves * 16 * kTileRT;
    const AttnFn fn = D == 64 ? &attn_tile_kernel<64> : D == 128 ? &attn_tile_kernel<128> : &attn_tile_kernel<256>;
    return launch(fn, dim3((unsigned)((rows + per - 1) / per), a.HKV, a.B), 0, g_raised[di][0], s, a);
  }
  a.o_part = reinterpret_cast<float*>(ws + p.o);
  a.ml_part = reinterpret_cast<float2*>(ws + p.ml);
  a.plan = reinterpret_cast<int2*>(ws + p.plan);
  const int rt = (p.rows + 15) / 16;
  const AttnFn fn = D == 64 ? split_kernel<64>(rt) : D == 128 ? split_kernel<128>(rt) : split_kernel<256>(rt);
  const AttnFn comb = D == 64 ? &attn_combine_kernel<64> : D == 128 ? &attn_combine_kernel<128> : &attn_combine_kernel<256>;
  const size_t lds = (size_t)2 * (rt == 1 ? 1 : 2) * 16 * D * sizeof(float);  // the first round of the wavefronts' merge
  const int st = launch(fn, dim3(p.slots, a.HKV), lds, g_raised[di][rt], s, a);
  if (st != QF_OK) return st;
  return launch(comb, dim3(a.B, p.rows, a.HKV), 0, g_raised[di][0], s, a);
}
