// qf_kv4_attn.hip — attention over a paged cache held in 4 bits (gfx950).
//
// A wavefront takes 16 RT packed query rows (token, head of the kv head's group) and walks over positions in steps of 32, two
// cache records: S^T = K Q^T on v_mfma_f32_16x16x32_bf16 with the keys as the A operand, an online softmax in base 2, and
// O^T += V^T P^T on the same instruction.  The records are laid out so that a lane's 16 bytes are its part of an operand, which
// one instruction widens for two codes and their scale.  A lane's accumulator of S^T holds 4 positions of one row for each
// record, which are its 8 values of the B operand P^T: the softmax weights never leave the lane.
//
//   attn_split_kernel    few rows (decode, verification): the positions of the batch are split over workgroups and, in a
//                        workgroup, over 4 wavefronts, whose states meet in LDS; attn_combine_kernel adds the splits.  Bound by the
//                        cache's bytes where it is long (100 000 positions, 64 heads over 8, D = 128: 109 MB in 31 us with the
//                        join, 3.5 TB/s; a wavefront's own step of 2000 cycles is what keeps it from more), by the chain lengths,
//                        block ids, codes, states, partial results where it is short (1000 positions: 5.4 us and 4.3 us)
//   attn_tile_kernel     many rows (prompt chunks): each wavefront its own rows, all of a workgroup the same positions.  Bound by
//                        the matrix cores at D = 128 (2048 tokens behind 8192 positions, 64 heads over 8: 514 us, 1.21 PFLOP/s).
//                        At D = 256 (16 rows a wavefront: twice the operand reads a product) by no unit alone: with row tiles that
//                        fill the machine twice LDS is busy 55% of the time and the matrix cores 40%, the chain product, softmax,
//                        product behind a barrier a stage has two wavefronts a SIMD to hide it; in a ragged batch by its longest
//                        request, whose row tiles come last to an end
#include "qf_kv4_common.h"

#include <math.h>
#include <string.h>

namespace qfk {

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
  int rows;     // split kernel: the most rows of a request that it takes
  int few;      // tile kernel: requests of up to so many rows are the split kernel's
  int workers;  // split kernel: positions are split so that about this many workgroups a kv head share the batch
  float qk_scale;  // |scale| * log2(e): scores are kept in base 2
  uint32_t flip;   // the queries' signs, changed for a negative scale
  Divisor by_g, by_page, by_workers;
  float* o_part;   // [HKV][slots][rows][D]
  float2* ml_part; // [HKV][slots][rows]: exponent reference, sum
  int2* plan;      // [B]: first slot and slots of a request
  int cus;  // compute units
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
  r.seq = min(max(a.seq_lens[b], 0), a.max_blocks * a.page);  // below 2^31 - 63
  return r;
}

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// The largest, NaN where one is.  (fmaxf, which leaves NaN out, would first quiet each operand that comes from a matrix
// instruction.)
__device__ __forceinline__ float largest(float x, float y) { return __builtin_elementwise_maximum(x, y); }

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
  typedef uint32_t Run __attribute__((ext_vector_type(kDwords)));
  Run k[2][kHalves], v[2][kHalves];
  uint32_t ks[2][kHalves], vs[2][kHalves];
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
        qf[rt][s] = __builtin_bit_cast(
            bf16x8_t, *reinterpret_cast<const u32x4_t*>(p + s / kDwords * 128 + qg * 8 * kDwords + s % kDwords * 8) ^ a.flip);
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

  // Offset from `base` of the record that holds position pos (a multiple of 16).
  __device__ __forceinline__ int64_t record(int pos) const {
    const int pg = divide(pos, a.by_page);
    int64_t block = bt_row[pg];
    block = block < 0 ? 0 : block >= a.num_blocks ? a.num_blocks - 1 : block;
    return block * a.stride + (pos - pg * a.page) / kTile * R::kBytes;
  }

  // A value's block of NaN at a position that some rows see and others do not: the product would give it to all rows.  Where a
  // step holds one, its scales are cleared for the product and the rows that see it are made NaN here.
  __device__ __forceinline__ void masked_nan(Data& s, int pos, int end) {
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
    mark_nan(pos, min(pos + kStep, end));
  }

  // NaN into the outputs of the rows that see a value's block of NaN among positions from .. to - 1 (the lane's outputs are values
  // 128 h + 32 qg .. of its rows, for D = 64 16 qg ..: one block each).
  __device__ __forceinline__ void mark_nan(int from, int to) {
    for (int p = from; p < to; ++p) {
      const uint8_t* r = base + record(p / kTile * kTile) + p % kTile;
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        const uint32_t byte = r[R::kValueScales + (kDwords == 4 ? 4 * h + qg : qg / 2) * kTile];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          if (byte == 255u && p <= last[rt]) {
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

  typedef f32x4_t Scores[RT][2];

  // The lane's byte of a dword of 4 positions' scales, turned to an fp32's exponent.  (`here`: where it is used; moved up to its
  // load, the instruction would wait for it.)
  __device__ __forceinline__ float key_scale(uint32_t w) const {
    w = here(w);
    return __uint_as_float(__builtin_amdgcn_alignbit(w, w, (uint32_t)(8 * (l16 & 3) + 9)));
  }

  // S^T of a step's 32 positions, 2 RT chains of matrix instructions side by side.
  __device__ __forceinline__ void scores(const Data& s, Scores& sc) const {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) sc[rt][0] = sc[rt][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      const float k0 = key_scale(s.ks[0][h]), k1 = key_scale(s.ks[1][h]);
#pragma unroll
      for (int c = 0; c < kDwords; ++c) {
        const bf16x8_t f0 = __builtin_bit_cast(bf16x8_t, widen8(s.k[0][h][c], k0));
        const bf16x8_t f1 = __builtin_bit_cast(bf16x8_t, widen8(s.k[1][h][c], k1));
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          sc[rt][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f0, qf[rt][h * kDwords + c], sc[rt][0], 0, 0, 0);
          sc[rt][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f1, qf[rt][h * kDwords + c], sc[rt][1], 0, 0, 0);
        }
      }
    }
  }

  // -inf where a row does not see a position.
  __device__ __forceinline__ void mask(Scores& sc, int pos) const {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int p0 = pos + t * kTile + 4 * qg;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[rt][t][i] = p0 + i <= last[rt] ? sc[rt][t][i] : -__builtin_inff();
    }
  }

  // The rows' exponent references brought up to the scores.  A reference moves only when a score exceeds it by 2^8: the weights
  // stay below that, and the accumulators are rarely rescaled.  The result is that of the running maximum up to rounding.
  template <int N>
  __device__ __forceinline__ void refer(const Scores (&sc)[N]) {
    bool above = false;
    float mx[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float top = sc[0][rt][0][0];
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const f32x4_t x = sc[n][rt][0], y = sc[n][rt][1];
        top = largest(largest(top, x[1]), n == 0 ? x[2] : x[0]);
        top = largest(largest(top, n == 0 ? x[3] : x[2]), y[0]);
        top = largest(largest(top, y[1]), y[2]);
        top = n == 0 ? largest(top, y[3]) : largest(largest(top, x[3]), y[3]);
      }
      mx[rt] = a.qk_scale * top;
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
  }

  // The softmax weights of the scores, rounded to bf16, as the operand P^T: the matrix instructions take 16-bit operands, those of fp32 at
  // a sixteenth of the rate.  Their sum l takes them unrounded, so an output is off by the weights' own roundings, 2^-8 of each at
  // most (error against 64 bits with weights of fp32 and so: 1000 positions 0.0016 and 0.0017, 38 000 0.0016 and 0.0021, a chunk of
  // 2048 tokens 0.0017 and 0.0023; the output's rounding is in both).
  __device__ __forceinline__ void weigh(const Scores& sc, bf16x8_t (&pf)[RT]) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const float ref = m[rt] == -__builtin_inff() ? 0.f : m[rt];  // a row that has seen nothing yet
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = fast_exp2(__builtin_fmaf(sc[rt][i / 4][i % 4], a.qk_scale, -ref));
      l[rt] += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
      pf[rt] = __builtin_bit_cast(bf16x8_t, pack8(w));
    }
  }

  // Positions pos .. pos + 31, those from `end` on hold nothing.
  __device__ __forceinline__ void step(Data& s, int pos, int end) {
    Scores all[1];
    Scores& sc = all[0];
    scores(s, sc);
    if (pos + kStep > diag || pos + kStep > end) {
      mask(sc, pos);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int p0 = pos + t * kTile + 4 * qg;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (p0 + i < end) continue;
          // what stands behind the end may be anything, a NaN among it: weight 0 times 0
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) sc[rt][t][i] = -__builtin_inff();
#pragma unroll
          for (int h = 0; h < kHalves; ++h) {
            s.vs[t][h] &= ~(255u << (8 * i));
            s.vs[t][h] |= 127u << (8 * i);
            clear(s, t, h, i);
          }
        }
      }
      masked_nan(s, pos, end);
    }
    refer(all);
    bf16x8_t pf[RT];
    weigh(sc, pf);
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      float vs[2][4];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        vs[t][0] = scale_of<0>(s.vs[t][h]);
        vs[t][1] = scale_of<1>(s.vs[t][h]);
        vs[t][2] = scale_of<2>(s.vs[t][h]);
        vs[t][3] = scale_of<3>(s.vs[t][h]);
      }
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

  // ---- the split kernel's way: steps through LDS ----
  // A lane's bytes go from global memory to LDS and from there to the same lane's registers, so LDS is a place to wait in, without
  // registers, for the step after the one that is computed.
  static constexpr int kCodes = 2 * 2 * kHalves * kDwords * 4 * kWave;         // a step's codes, keys then values
  static constexpr int kScales = D < 128 ? 256 : 2 * D;                        // and scales (D = 64: half of it is not read)
  static constexpr int kSlot = kCodes + kScales;
  static constexpr int kCopies = kCodes / 1024 + kScales / 256;                // instructions of a step
  typedef const void __attribute__((address_space(1)))* gptr_t;
  typedef void __attribute__((address_space(3)))* lptr_t;

  __device__ __forceinline__ void copy(const uint8_t* from, uint8_t* to) const {
    // 2: read once, not kept (one request of 100 000 positions 36 us, 39 kept; 48 requests out of 12 layers' caches 26.3, 27.6)
    __builtin_amdgcn_global_load_lds((gptr_t)from, (lptr_t)to, 16, 0, 2);
  }
  __device__ __forceinline__ void copy_step(const uint8_t* r0, const uint8_t* r1, uint8_t* slot) const {
    if constexpr (kDwords == 4) {
      const uint32_t key = (uint32_t)(l16 * (D / 2) + qg * 16), value = (uint32_t)(R::kValues + lane * 16);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          const uint8_t* r = t == 0 ? r0 : r1;
          copy(r + h * 64 + key, slot + (t * kHalves + h) * 1024);
          copy(r + h * 1024 + value, slot + (2 * kHalves + t * kHalves + h) * 1024);
        }
    } else {  // a record's codes are a KiB, the keys' half first
      copy(r0 + lane * 16, slot);
      copy(r1 + lane * 16, slot + 1024);
    }
    uint8_t* const to = slot + kCodes;
    if constexpr (D == 256) {
      __builtin_amdgcn_global_load_lds((gptr_t)(r0 + R::kKeyScales + lane * 4), (lptr_t)to, 4, 0, 2);
      __builtin_amdgcn_global_load_lds((gptr_t)(r1 + R::kKeyScales + lane * 4), (lptr_t)(to + 256), 4, 0, 2);
    } else {  // both records' scales in one instruction
      constexpr int kLanes = D / 4;
      const uint8_t* r = lane / kLanes % 2 == 0 ? r0 : r1;
      __builtin_amdgcn_global_load_lds((gptr_t)(r + R::kKeyScales + lane % kLanes * 4), (lptr_t)to, 4, 0, 2);
    }
  }

  // The step's data out of its slot.  One block with its own wait: the compiler would wait for every copy in flight before
  // an LDS read that it sees.
  __device__ __forceinline__ void read_step(Data& s, const uint8_t* slot) const {
    const uint32_t at = lds_addr(slot);
    const uint32_t ks = at + kCodes + (uint32_t)((kDwords == 4 ? qg : qg / 2) * kTile + (l16 & 12));
    const uint32_t vs = at + kCodes + (uint32_t)(D / 2 + (kDwords == 4 ? l16 / 4 : l16 / 8) * kTile + 4 * qg);
    if constexpr (D == 64) {
      const uint32_t k = at + (uint32_t)(l16 * 32 + qg * 8), v = at + 512 + (uint32_t)(lane * 8);
      u32x2_t k0, k1, v0, v1;
      asm volatile(
          "ds_read_b64 %0, %8\n\tds_read_b64 %1, %8 offset:1024\n\tds_read_b32 %4, %10\n\tds_read_b32 %5, %10 offset:64\n\t"
          "ds_read_b64 %2, %9\n\tds_read_b64 %3, %9 offset:1024\n\tds_read_b32 %6, %11\n\tds_read_b32 %7, %11 offset:64\n\t"
          "s_waitcnt lgkmcnt(0)"
          : "=&v"(k0), "=&v"(k1), "=&v"(v0), "=&v"(v1), "=&v"(s.ks[0][0]), "=&v"(s.ks[1][0]), "=&v"(s.vs[0][0]), "=&v"(s.vs[1][0])
          : "v"(k), "v"(v), "v"(ks), "v"(vs)
          : "memory");
      s.k[0][0] = k0;
      s.k[1][0] = k1;
      s.v[0][0] = v0;
      s.v[1][0] = v1;
    } else if constexpr (D == 128) {
      u32x4_t k0, k1, v0, v1;
      asm volatile(
          "ds_read_b128 %0, %8\n\tds_read_b128 %1, %8 offset:1024\n\tds_read_b32 %4, %9\n\tds_read_b32 %5, %9 offset:128\n\t"
          "ds_read_b128 %2, %8 offset:2048\n\tds_read_b128 %3, %8 offset:3072\n\tds_read_b32 %6, %10\n\t"
          "ds_read_b32 %7, %10 offset:128\n\ts_waitcnt lgkmcnt(0)"
          : "=&v"(k0), "=&v"(k1), "=&v"(v0), "=&v"(v1), "=&v"(s.ks[0][0]), "=&v"(s.ks[1][0]), "=&v"(s.vs[0][0]), "=&v"(s.vs[1][0])
          : "v"(at + (uint32_t)lane * 16), "v"(ks), "v"(vs)
          : "memory");
      s.k[0][0] = k0;
      s.k[1][0] = k1;
      s.v[0][0] = v0;
      s.v[1][0] = v1;
    } else {
      u32x4_t k[4], v[4];
      uint32_t a0, a1, a2, a3, b0, b1, b2, b3;
      asm volatile(
          "ds_read_b128 %0, %16\n\tds_read_b128 %1, %16 offset:1024\n\tds_read_b128 %2, %16 offset:2048\n\t"
          "ds_read_b128 %3, %16 offset:3072\n\tds_read_b32 %8, %17\n\tds_read_b32 %9, %17 offset:64\n\t"
          "ds_read_b32 %10, %17 offset:256\n\tds_read_b32 %11, %17 offset:320\n\tds_read_b128 %4, %16 offset:4096\n\t"
          "ds_read_b128 %5, %16 offset:5120\n\tds_read_b128 %6, %16 offset:6144\n\tds_read_b128 %7, %16 offset:7168\n\t"
          "ds_read_b32 %12, %18\n\tds_read_b32 %13, %18 offset:64\n\tds_read_b32 %14, %18 offset:256\n\t"
          "ds_read_b32 %15, %18 offset:320\n\ts_waitcnt lgkmcnt(0)"
          : "=&v"(k[0]), "=&v"(k[1]), "=&v"(k[2]), "=&v"(k[3]), "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(a0),
            "=&v"(a1), "=&v"(a2), "=&v"(a3), "=&v"(b0), "=&v"(b1), "=&v"(b2), "=&v"(b3)
          : "v"(at + (uint32_t)lane * 16), "v"(ks), "v"(vs)
          : "memory");
      s.ks[0][0] = a0;
      s.ks[0][kHalves - 1] = a1;
      s.ks[1][0] = a2;
      s.ks[1][kHalves - 1] = a3;
      s.vs[0][0] = b0;
      s.vs[0][kHalves - 1] = b1;
      s.vs[1][0] = b2;
      s.vs[1][kHalves - 1] = b3;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          s.k[t][h] = k[(t * kHalves + h) % 4];
          s.v[t][h] = v[(t * kHalves + h) % 4];
        }
    }
  }

  // Steps first, first + by, ... of the positions begin .. end - 1, through two slots of kSlot bytes (100 000 positions 36 us, with
  // three slots 39, with four 40: what is in flight is enough, and more of it in other places of the cache is read slower).  The
  // records of 32 steps are looked up at once, a record a lane.
  __device__ __forceinline__ void run(int begin, int end, int first, int by, uint8_t* slots) {
    const int n_steps = (end - begin + kStep - 1) / kStep;
    const int mine = first < n_steps ? (n_steps - 1 - first) / by + 1 : 0;
    const int last_tile = (end - 1) / kTile * kTile;
    uint32_t rec_lo = 0, rec_hi = 0;
    auto look_up = [&](int i) {
      const int pos = begin + (first + min(i + lane / 2, mine - 1) * by) * kStep + lane % 2 * kTile;
      const int64_t at = record(min(pos, last_tile));
      rec_lo = (uint32_t)at;
      rec_hi = (uint32_t)(at >> 32);
    };
    auto where = [&](int l) {
      const uint32_t lo = __builtin_amdgcn_readlane(rec_lo, l), hi = __builtin_amdgcn_readlane(rec_hi, l);
      return base + (int64_t)(((uint64_t)hi << 32) | lo);
    };
    auto issue = [&](int i) {
      if (i % 32 == 0 && i > 0) {
        look_up(i);
        wait_vmcnt<0>();
      }
      copy_step(where(2 * (i % 32)), where(2 * (i % 32) + 1), slots + i % 2 * kSlot);
    };
    if (mine > 0) look_up(0);
    wait_vmcnt<0>();  // the queries too: the copies alone are counted below
    if (mine > 0) issue(0);
#pragma unroll 1
    for (int i = 0; i < mine; ++i) {
      if (i + 1 < mine) {
        issue(i + 1);  // into the slot of step i - 1, whose reads have returned
        wait_vmcnt<kCopies>();
      } else {
        wait_vmcnt<0>();
      }
      asm volatile("" ::: "memory");
      Data now;
      read_step(now, slots + i % 2 * kSlot);
      step(now, begin + (first + i * by) * kStep, end);
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
  auto steps = [&](int b) {  // of request b: -1 where it has no tokens, or too many
    if (b >= a.B) return -1;
    const Request r = request(a, b);
    return r.n > 0 && r.n * a.G <= a.rows ? (r.seq + kStep - 1) / kStep : -1;
  };
  int mine = steps(lane);
  uint32_t most;  // steps of a chunk
  {
    uint32_t sum = max(mine, 0);
    uint64_t total = 0;
    if (a.B > kWave) {
      uint64_t all = sum;
      for (int b = lane + kWave; b < a.B; b += kWave) all += (uint32_t)max(steps(b), 0);
#pragma unroll
      for (int d = 1; d < kWave; d *= 2) {
        const uint32_t lo = __shfl_xor((int)(uint32_t)all, d), hi = __shfl_xor((int)(uint32_t)(all >> 32), d);
        all += ((uint64_t)hi << 32) | lo;
      }
      total = all;
    } else {
      total = (uint32_t)__builtin_amdgcn_readlane(wave_scan((int)sum), kWave - 1);  // at most 64 * 2^26
    }
    most = total < 0x80000000u ? (uint32_t)divide((int)total, a.by_workers) + 1 : chunk_steps(total, (uint32_t)a.workers);
    most = min(max(most, (uint32_t)(kMinChunk / kStep)), kMostSteps);
  }
  p.chunk = (int)min(most * kStep, 0x7fffffe0u);
  int before = 0;
  for (int base = 0;; base += kWave) {
    if (base > 0) mine = steps(base + lane);
    const int n = mine < 0 ? 0 : max((int)(((uint32_t)mine + most - 1) / most), 1);
    const int upto = before + wave_scan(n);
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < kWave && base + lane < a.B) a.plan[base + lane] = make_int2(upto - n, n);
    const uint64_t here = __ballot(slot >= upto - n && slot < upto);
    if (here != 0) {
      const int i = __builtin_ctzll(here);
      p.b = base + i;
      p.first = __builtin_amdgcn_readlane(upto - n, i);
      p.splits = __builtin_amdgcn_readlane(n, i);
      p.split = slot - p.first;
      if (blockIdx.x != 0) return true;
    }
    before = __builtin_amdgcn_readlane(upto, kWave - 1);
    if (base + kWave >= a.B) break;
  }
  return blockIdx.x == 0 ? before > 0 : false;
}

// 4 wavefronts a workgroup: several workgroups a CU then hide each other's start, merge and end (48 requests of up to 9000
// positions, 64 heads over 8: 25 us, 33 with 8 wavefronts and four slots each; 38000 positions, D = 256: 27.7 and 29.5).
constexpr int kSplitWaves = 4;
template <int D, int RT>
constexpr int split_lds() {  // the slots, then the wavefronts' tiles
  constexpr int slots = kSplitWaves * 2 * Walk<D, RT>::kSlot, merge = kSplitWaves * RT * D * 64;
  return slots > merge ? slots : merge;
}

// RG groups of 16 RT rows; the wavefronts of a group share its positions.  A partial result is a tile of 16 rows x 16 values a
// KiB, as the accumulators hold it: lane (row l16, quarter qg), the value that Walk::value_at names.  attn_combine_kernel adds them.
// (Adding them in this launch, by the last split to arrive, took longer: its reads wait for the others' writes, their count and each
// other, 1000 positions 9.6 against 8.8 us, 8000 positions 18.6 against 12.)
template <int D, int RT, int RG>
__global__ __launch_bounds__(kSplitWaves * kWave) void attn_split_kernel(AttnArgs a) {
  using W = Walk<D, RT>;
  constexpr int kWaves = kSplitWaves, kShare = kWaves / RG;  // wavefronts of a row group
  constexpr int kTiles = RG * RT * W::kDTiles;
  extern __shared__ __align__(16) uint8_t lds[];  // the slots, then [wavefront][RT][D / 16] tiles
  __shared__ float row_m[kWaves][RT][16], row_l[kWaves][RT][16], row_inv[RG * RT][16];
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
  w.run(begin, end, share, kShare, lds + wave * 2 * W::kSlot);

  // ---- the wavefronts' states against their common reference, through LDS ----
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) w.l[rt] = quarters_sum(w.l[rt]);
  if (w.qg == 0) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) row_m[wave][rt][w.l16] = w.m[rt];
  }
  __syncthreads();  // and every slot is done with
  f32x4_t* const tiles = reinterpret_cast<f32x4_t*>(lds);
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    float top = row_m[rg][rt][w.l16];
#pragma unroll
    for (int i = 1; i < kShare; ++i) top = fmaxf(top, row_m[i * RG + rg][rt][w.l16]);
    const float keep = fast_exp2(w.m[rt] - (top == -__builtin_inff() ? 0.f : top));
    w.m[rt] = top;
#pragma unroll
    for (int u = 0; u < W::kDTiles; ++u) tiles[((wave * RT + rt) * W::kDTiles + u) * kWave + w.lane] = w.o[rt][u] * keep;
    if (w.qg == 0) row_l[wave][rt][w.l16] = w.l[rt] * keep;
  }
  __syncthreads();
  const int rows = r.n * a.G;
  const int64_t slot = (int64_t)hkv * a.slots + blockIdx.x;
  auto none_seen = [&](int row) { return r.seq - r.n + divide(row, a.by_g) < 0; };
  if (share == 0 && w.qg == 0) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int row = (rg * RT + rt) * 16 + w.l16;
      float l = row_l[rg][rt][w.l16];
#pragma unroll
      for (int i = 1; i < kShare; ++i) l += row_l[i * RG + rg][rt][w.l16];
      row_inv[rg * RT + rt][w.l16] = none_seen(row) ? 0.f : 1.f / l;
      if (p.splits > 1 && row < rows) a.ml_part[slot * a.rows + row] = make_float2(w.m[rt], l);
    }
  }
#pragma unroll 1
  for (int k = wave; k < kTiles; k += kWaves) {  // tile u of row tile rt of row group g
    const int g = k / (RT * W::kDTiles), at = (k - g * RT * W::kDTiles) * kWave + w.lane;
    f32x4_t sum = tiles[g * RT * W::kDTiles * kWave + at];
#pragma unroll
    for (int i = 1; i < kShare; ++i) sum += tiles[(i * RG + g) * RT * W::kDTiles * kWave + at];
    if (p.splits == 1) {
      tiles[k * kWave + w.lane] = sum;  // (tile k of wavefront 0's, or of wavefront 1's where that is the second row group)
    } else if (k / W::kDTiles * 16 + w.l16 < rows) {
      reinterpret_cast<f32x4_t*>(a.o_part)[(slot * kTiles + k) * kWave + w.lane] = sum;
    }
  }
  if (p.splits > 1) return;
  __syncthreads();
  const float* const sums = reinterpret_cast<const float*>(lds);
#pragma unroll 1
  for (int k = wave; k < RG * RT * W::kHalves * 4; k += kWaves) {  // component i of half h of row tile rt
    const int i = k % 4, h = k / 4 % W::kHalves, rt = k / (4 * W::kHalves), row = rt * 16 + w.l16;
    if (row >= rows) continue;
    const int qi = divide(row, a.by_g);
    const float inv = row_inv[rt][w.l16];
    uint32_t v[W::kPerHalf / 2];
#pragma unroll
    for (int n = 0; n < W::kPerHalf / 2; ++n) {
      const float* t = sums + ((rt * W::kDTiles + h * W::kPerHalf + 2 * n) * kWave + w.lane) * 4 + i;
      v[n] = pack_bf16(t[0] * inv, t[4 * kWave] * inv);
    }
    uint16_t* to = a.out + (int64_t)(r.tok0 + qi) * a.so_t + (int64_t)(hkv * a.G + (row - qi * a.G)) * a.so_h + w.value_at(h, i);
    if constexpr (W::kPerHalf == 8) {
      *reinterpret_cast<u32x4_t*>(to) = u32x4_t{v[0], v[1], v[2], v[3]};
    } else {
      *reinterpret_cast<u32x2_t*>(to) = u32x2_t{v[0], v[1]};
    }
  }
}

// Many rows: 8 wavefronts with 16 kRT rows each walk over the same positions, 64 a stage.  A stage's keys and values are widened
// once for all of them, an eighth a wavefront, into LDS, in the order of the operands (8 KiB of fragments a wavefront and step of
// either, at D = 128): two buffers, one barrier a stage.  (2048 tokens behind 8192 positions, 64 heads over 8, before
// attn_tile_kernel's order of workgroups: 555 us; keys widened by each wavefront for itself 681; 4 wavefronts of 64 rows, whose
// accumulators move between register files, 928.)
template <int D>
struct TileShape {
  static constexpr int kRT = D == 256 ? 1 : 2;
  static constexpr int kWaves = 8;
  static constexpr int kRows = 16 * kRT * kWaves;
  static constexpr int kFragments = 4 * (D / 32) + 2 * (D / 16);  // KiB of a stage: 4 records' keys, 2 steps' values
  static constexpr int kLds = 2 * kFragments * 1024;
};

// The stages of a row tile that sees the positions below `end`, over at most `most` workgroups of 4 stages or more.
__device__ __forceinline__ void stage_splits(int end, int most, int& splits, int& per) {
  const int n = max((end + kStage - 1) / kStage, 1);
  splits = min(most, max(n / 4, 1));
  per = (n + splits - 1) / splits;
  splits = (n + per - 1) / per;
}

// The row tiles that a batch holds, of the requests that are not the split kernel's, in an order: request by request, the longest
// first where there are up to 64 (a lane each), each one's last tile, which sees most, first.  Every workgroup finds it out for
// itself from the lengths, so that the launch is as large as the batch at most and nothing is read back.
// (Chunks of up to 700 tokens, the longest given last: 13 requests 164 -> 151 us, D = 256, 15 requests 185 -> 169.  Splits by what
// the batch holds instead of what it could hold: 7 chunks of up to 24 tokens behind up to 5800 positions, 48 heads of 256 over
// 8: 118 -> 67 us; 9 of up to 165 behind 9000, 20 of 64 over 4: 110 -> 70; 40 chunks that fill the machine 146 -> 152.)
constexpr int kMostSplits = 16;
template <int ROWS>
struct Batch {
  static constexpr int kCap = 1 << 30;  // 64 requests more of at most 2^24 tiles each stay below 2^31
  const AttnArgs& a;
  int lane, mine, before, total;

  __device__ __forceinline__ int tiles_of(const Request& r) const {
    const int rows = r.n * a.G;
    return rows > a.few ? (rows + ROWS - 1) / ROWS : 0;
  }
  __device__ __forceinline__ int tiles_of(int b) const { return b < a.B ? tiles_of(request(a, b)) : 0; }

  __device__ __forceinline__ explicit Batch(const AttnArgs& args) : a(args) {
    lane = threadIdx.x % kWave;
    total = before = mine = 0;
    if (a.B <= kWave) {
      const Request r = request(a, min(lane, a.B - 1));
      mine = lane < a.B ? tiles_of(r) : 0;
      for (int j = 0; j < a.B; ++j) {
        const int tiles = __builtin_amdgcn_readlane(mine, j), seq = __builtin_amdgcn_readlane(r.seq, j);
        if (seq > r.seq || (seq == r.seq && j < lane)) before += tiles;
        total += tiles;
      }
    } else {
      for (int base = 0; base < a.B; base += kWave)
        total = min(total + __builtin_amdgcn_readlane(wave_scan(tiles_of(base + lane)), kWave - 1), kCap);
    }
  }

  // Workgroups that share the positions of a row tile: several where the batch's tiles leave compute units idle.  There are at
  // most a.cus partial results then.
  __device__ __forceinline__ int splits() const {
    const int64_t groups = (int64_t)total * a.HKV;
    return groups > a.cus ? 1 : min(a.cus / max((int)groups, 1), kMostSplits);
  }

  // Tile t of the order: its request and its place among the request's; false where the batch has fewer.
  __device__ __forceinline__ bool find(int t, int& b, int& row_tile) const {
    int n = mine, first = before;
    for (int base = 0, done = 0;; base += kWave) {
      if (a.B > kWave) {
        n = tiles_of(base + lane);
        first = done + wave_scan(n) - n;
        done = min(__builtin_amdgcn_readlane(first + n, kWave - 1), kCap);
      }
      const uint64_t here = __ballot(t >= first && t < first + n);
      if (here != 0) {
        const int i = __builtin_ctzll(here);
        b = base + i;
        row_tile = __builtin_amdgcn_readlane(n, i) - 1 - (t - __builtin_amdgcn_readlane(first, i));
        return true;
      }
      if (base + kWave >= a.B) return false;
    }
  }
};

template <int D>
__global__ __launch_bounds__(TileShape<D>::kWaves * kWave) void attn_tile_kernel(AttnArgs a) {
  using S = TileShape<D>;
  using W = Walk<D, S::kRT>;
  using R = Record<D>;
  extern __shared__ __align__(16) uint8_t lds[];
  __shared__ uint32_t odd[2][S::kWaves];  // a wavefront met a block of NaN that not all rows see
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  // The heads of a row tile stand together: those that see most come first over all heads, and where the heads are a multiple of
  // 8 an XCD's L2 holds its own heads' positions (4096 tokens of 32 heads over 8 from the start 234 -> 137 us; 2048 of 64 over 8
  // behind 8192 positions 556 -> 514; D = 256 341 -> 300).  With positions split a head's workgroups do (34.7 us, 37.6).
  const Batch<S::kRows> batch(a);
  const int most = batch.splits(), x = blockIdx.x;
  int t, hkv, split = 0;
  if (most == 1) {
    t = x / a.HKV;
    hkv = x - t * a.HKV;
  } else {
    if (batch.total == 0) return;
    hkv = x / (batch.total * most);
    if (hkv >= a.HKV) return;
    t = (x - hkv * batch.total * most) / most;
    split = (x - hkv * batch.total * most) % most;
  }
  int b, row_tile;
  if (!batch.find(t, b, row_tile)) return;
  const Request r = request(a, b);
  const int rows = r.n * a.G;
  const int row0 = row_tile * S::kRows;
  const int r0 = row0 + wave * 16 * S::kRT;
  W w(a);
  w.start(r, b, hkv, r0);
  auto seen = [&](int row) { return max(r.seq - r.n + divide(min(row, rows - 1), a.by_g) + 1, 0); };
  const int own_end = r0 < rows ? seen(r0 + 16 * S::kRT - 1) : 0;  // positions that a row of this wavefront sees
  const int end = seen(row0 + S::kRows - 1), all_see = seen(row0);
  int splits, per;
  stage_splits(end, most, splits, per);
  if (split >= splits) return;
  const int first_stage = split * per, n_stages = min((end + kStage - 1) / kStage, first_stage + per);
  const int last_tile = (end - 1) / kTile * kTile;

  // fragment f of a stage's keys (record f / (D / 32)), and of its values (step f / (D / 16))
  auto key_at = [&](int buffer, int f) { return lds + ((buffer * S::kFragments + f) * kWave + w.lane) * 16; };
  auto value_at = [&](int buffer, int f) { return key_at(buffer, 4 * W::kKSteps + f); };

  // The records of 16 stages are looked up at once, a record a lane.
  uint32_t rec_lo = 0, rec_hi = 0;
  auto look_up = [&](int stage) {
    const int64_t at = w.record(stage_record(stage, w.lane, last_tile));
    rec_lo = (uint32_t)at;
    rec_hi = (uint32_t)(at >> 32);
  };
  auto where = [&](int l) {
    const uint32_t lo = __builtin_amdgcn_readlane(rec_lo, l), hi = __builtin_amdgcn_readlane(rec_hi, l);
    return w.base + (int64_t)(((uint64_t)hi << 32) | lo);
  };

  // This wavefront's share of a stage: of record `mine` a half of each lane's run (D = 256: one of its halves).
  const int mine = wave / 2, part = wave % 2, half = D == 256 ? part : 0;
  constexpr int kKeyDwords = D == 256 ? 4 : W::kDwords / 2;  // of each lane's keys
  constexpr int kBytes = D == 256 ? 4 : D / 64;              // of each lane's run of values: 2 kBytes tiles
  const int byte0 = D == 256 ? 0 : part * kBytes;
  typedef uint32_t Keys __attribute__((ext_vector_type(kKeyDwords)));
  Keys k;
  typename W::Data::Run v;
  uint32_t ks, vs;
  auto load_share = [&](int stage) {
    const uint8_t* rec = where(stage % 16 * 4 + mine);
    k = *reinterpret_cast<const Keys*>(rec + w.l16 * (D / 2) + half * 64 + w.qg * (4 * W::kDwords) +
                                       (D == 256 ? 0 : part * 4 * kKeyDwords));
    v = *reinterpret_cast<const typename W::Data::Run*>(rec + R::kValues + half * 1024 + w.lane * 4 * W::kDwords);
    ks = *reinterpret_cast<const uint32_t*>(rec + R::kKeyScales + (W::kDwords == 4 ? 4 * half + w.qg : w.qg / 2) * kTile +
                                            (w.l16 & 12));
    vs = *reinterpret_cast<const uint32_t*>(rec + R::kValueScales + (W::kDwords == 4 ? 4 * half + w.l16 / 4 : w.l16 / 8) * kTile +
                                            4 * w.qg);
  };
  auto widen_share = [&](int stage) {
    const int pos = stage * kStage + mine * kTile, buffer = stage & 1;
    const float scale = w.key_scale(ks);
    const int f = mine * W::kKSteps + (D == 256 ? half * W::kDwords : part * kKeyDwords);
#pragma unroll
    for (int c = 0; c < kKeyDwords; ++c) *reinterpret_cast<u32x4_t*>(key_at(buffer, f + c)) = widen8(k[c], scale);
    if (pos + kTile > all_see) {  // behind the end anything may stand; a block of NaN would reach rows that do not see it
      bool any = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool gone = pos + 4 * w.qg + i >= end, nan = (vs >> (8 * i) & 255u) == 255u;
        any |= nan && !gone;
        if (gone || nan) {
          vs = (vs & ~(255u << (8 * i))) | 127u << (8 * i);
          if constexpr (W::kDwords == 4) {
            v[i] = 0;
          } else {
            v[i / 2] &= i % 2 ? 0xffffu : 0xffff0000u;
          }
        }
      }
      const bool met = __any(any);
      if (w.lane == 0) odd[buffer][wave] = met;
    }
    const uint32_t bytes = here(vs);
    const float s[4] = {scale_of<0>(bytes), scale_of<1>(bytes), scale_of<2>(bytes), scale_of<3>(bytes)};
    auto pair = [&](auto byte) {
      constexpr int kB = decltype(byte)::value;
      uint32_t x[4];
      if constexpr (D == 256) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = widen2<kB>(v[i], s[i]);
      } else if constexpr (D == 128) {  // bytes byte0 + kB, moved down
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = widen2<kB>(v[i] >> (8 * byte0), s[i]);
      } else {
        const uint32_t lo = v[0] >> (8 * byte0), hi = v[1] >> (8 * byte0);
        x[0] = widen2<0>(lo, s[0]);
        x[1] = widen2<2>(lo, s[1]);
        x[2] = widen2<0>(hi, s[2]);
        x[3] = widen2<2>(hi, s[3]);
      }
      const int u = mine / 2 * W::kDTiles + half * W::kPerHalf + 2 * (byte0 + kB);
      *reinterpret_cast<u32x2_t*>(value_at(buffer, u) + mine % 2 * 8) =
          u32x2_t{__builtin_amdgcn_perm(x[1], x[0], 0x05040100), __builtin_amdgcn_perm(x[3], x[2], 0x05040100)};
      *reinterpret_cast<u32x2_t*>(value_at(buffer, u + 1) + mine % 2 * 8) =
          u32x2_t{__builtin_amdgcn_perm(x[1], x[0], 0x07060302), __builtin_amdgcn_perm(x[3], x[2], 0x07060302)};
    };
    pair(std::integral_constant<int, 0>{});
    if constexpr (kBytes > 1) pair(std::integral_constant<int, 1>{});
    if constexpr (kBytes > 2) {
      pair(std::integral_constant<int, 2>{});
      pair(std::integral_constant<int, 3>{});
    }
  };

  auto compute = [&](int pos, int buffer) {
    if (pos >= own_end) return;
    typename W::Scores sc[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int rt = 0; rt < S::kRT; ++rt) sc[n][rt][0] = sc[n][rt][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < W::kKSteps; ++c) {
        const bf16x8_t f0 = *reinterpret_cast<const bf16x8_t*>(key_at(buffer, 2 * n * W::kKSteps + c));
        const bf16x8_t f1 = *reinterpret_cast<const bf16x8_t*>(key_at(buffer, (2 * n + 1) * W::kKSteps + c));
#pragma unroll
        for (int rt = 0; rt < S::kRT; ++rt) {
          sc[n][rt][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f0, w.qf[rt][c], sc[n][rt][0], 0, 0, 0);
          sc[n][rt][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f1, w.qf[rt][c], sc[n][rt][1], 0, 0, 0);
        }
      }
    }
    constexpr int kAhead = W::kDTiles < 8 ? W::kDTiles : 8;  // operands requested before they are needed
    bf16x8_t vf[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) vf[u] = *reinterpret_cast<const bf16x8_t*>(value_at(buffer, u));
    if (pos + kStage > w.diag) {
      w.mask(sc[0], pos);
      w.mask(sc[1], pos + kStep);
    }
    w.refer(sc);
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      bf16x8_t pf[S::kRT];
      w.weigh(sc[n], pf);
#pragma unroll
      for (int u = 0; u < W::kDTiles; ++u) {
        const int f = n * W::kDTiles + u;
#pragma unroll
        for (int rt = 0; rt < S::kRT; ++rt)
          w.o[rt][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[f % kAhead], pf[rt], w.o[rt][u], 0, 0, 0);
        if (f + kAhead < 2 * W::kDTiles) vf[f % kAhead] = *reinterpret_cast<const bf16x8_t*>(value_at(buffer, f + kAhead));
      }
    }
  };
  if (first_stage < n_stages) {
    look_up(first_stage / 16 * 16);
    load_share(first_stage);
    widen_share(first_stage);
    if ((first_stage + 1) % 16 == 0) look_up(first_stage + 1);
    load_share(first_stage + 1);  // past the last stage: the last record again
  }
#pragma unroll 1
  for (int stage = first_stage; stage < n_stages; ++stage) {
    ring_barrier();  // this stage's fragments stand, the stage before is done with
    if (stage + 1 < n_stages) widen_share(stage + 1);
    if ((stage + 2) % 16 == 0) look_up(stage + 2);
    load_share(stage + 2);
    compute(stage * kStage, stage & 1);
    if ((stage + 1) * kStage > all_see) {
      uint32_t met = 0;
#pragma unroll
      for (int i = 0; i < S::kWaves; ++i) met |= (stage * kStage + i / 2 * kTile + kTile > all_see) ? odd[stage & 1][i] : 0u;
      if (met != 0) w.mark_nan(max(stage * kStage, all_see / kTile * kTile), min((stage + 1) * kStage, end));
    }
  }
#pragma unroll
  for (int rt = 0; rt < S::kRT; ++rt) {
    w.l[rt] = quarters_sum(w.l[rt]);
    const int row = r0 + rt * 16 + w.l16;
    if (row >= rows) continue;
    if (splits == 1) {
      w.write(r, hkv, row, rt);
      continue;
    }
    const int64_t slot = ((int64_t)t * a.HKV + hkv) * most + split;
    const int at = wave * S::kRT + rt;
#pragma unroll
    for (int u = 0; u < W::kDTiles; ++u)
      reinterpret_cast<f32x4_t*>(a.o_part)[((slot * (S::kRows / 16) + at) * W::kDTiles + u) * kWave + w.lane] = w.o[rt][u];
    if (w.qg == 0) a.ml_part[slot * S::kRows + at * 16 + w.l16] = make_float2(w.m[rt], w.l[rt]);
  }
}

// A workgroup a slice (SLICES of them, 2 or 4) of a pair of tiles (values n and n + 1 of each lane's run): the splits are shared by
// its wavefronts, and by halves of a wavefront where SLICES is 4, 4 requested by each at once (they come from other XCDs'
// writes, a microsecond away); then the shares through LDS.
template <int D, int SLICES, int WAVES>
__device__ __forceinline__ void combine(const AttnArgs& a, const Request& r, int hkv, int row0, int pair, int slice, int64_t slot,
                                        int splits, int tiles, int slot_rows) {
  using W = Walk<D, 1>;
  constexpr int kSlice = kWave / SLICES;  // lanes of a tile
  constexpr int kGroups = WAVES * SLICES / 2;
  __shared__ float2 sm_ml[kGroups][kSlice];
  __shared__ __align__(16) f32x4_t sm_o[kGroups][2][kSlice];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int at = lane % kSlice, odd = lane / kSlice % 2, g = wave * (SLICES / 2) + lane / (2 * kSlice);
  const int tile_lane = slice * kSlice + at, tile = 2 * pair + odd;
  const int l16 = tile_lane % 16, qg = tile_lane / 16, part_row = tile / W::kDTiles * 16 + l16;
  const int row = row0 + part_row, rows = r.n * a.G;
  if (row - l16 >= rows) return;
  float m = -__builtin_inff(), l = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  if (row < rows) {
    const f32x4_t* from = reinterpret_cast<const f32x4_t*>(a.o_part) + (slot * tiles + tile) * kWave + tile_lane;
    const float2* stats = a.ml_part + slot * slot_rows + part_row;
    auto add = [&](int s, auto batch) {  // the splits s, s + kGroups, ... that there are, `batch` of them
      constexpr int kBatch = decltype(batch)::value;
      float2 ml[kBatch];
      f32x4_t v[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int n = min(s + i * kGroups, splits - 1);
        ml[i] = stats[(int64_t)n * slot_rows];
        v[i] = from[(int64_t)n * (tiles * kWave)];
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (s + i * kGroups >= splits) break;
        const float top = fmaxf(m, ml[i].x);
        const float ref = top == -__builtin_inff() ? 0.f : top;
        const float keep = fast_exp2(m - ref), weight = fast_exp2(ml[i].x - ref);
        o = o * keep + v[i] * weight;
        l = l * keep + ml[i].y * weight;
        m = top;
      }
    };
    int s = g;
    for (; s + 2 * kGroups < splits; s += 4 * kGroups) add(s, std::integral_constant<int, 4>{});
    if (s < splits) add(s, std::integral_constant<int, 2>{});
  }
  if (odd == 0) sm_ml[g][at] = make_float2(m, l);
  sm_o[g][odd][at] = o;
  __syncthreads();
  if (threadIdx.x >= kSlice || row >= rows) return;
  float top = sm_ml[0][at].x;
#pragma unroll
  for (int i = 1; i < kGroups; ++i) top = fmaxf(top, sm_ml[i][at].x);
  const float ref = top == -__builtin_inff() ? 0.f : top;
  f32x4_t evens = {0.f, 0.f, 0.f, 0.f}, odds = evens;
  l = 0.f;
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    const float2 ml = sm_ml[i][at];
    const float weight = fast_exp2(ml.x - ref);
    evens += sm_o[i][0][at] * weight;
    odds += sm_o[i][1][at] * weight;
    l += ml.y * weight;
  }
  const int qi = divide(row, a.by_g);
  const float inv = r.seq - r.n + qi < 0 ? 0.f : 1.f / l;
  using Rec = Record<D>;
  const int u = tile % W::kDTiles, h = u / W::kPerHalf, n = u % W::kPerHalf;
  uint16_t* to = a.out + (int64_t)(r.tok0 + qi) * a.so_t + (int64_t)(hkv * a.G + (row - qi * a.G)) * a.so_h +
                 16 * Rec::kWidth * h + Rec::kWidth * 4 * qg + n;
#pragma unroll
  for (int i = 0; i < 4; ++i) *reinterpret_cast<uint32_t*>(to + Rec::kWidth * i) = pack_bf16(evens[i] * inv, odds[i] * inv);
}

template <int D, int SLICES, int WAVES>
__global__ __launch_bounds__(WAVES * kWave) void attn_combine_kernel(AttnArgs a) {
  const int hkv = blockIdx.y, b = blockIdx.z;
  const int2 place = a.plan[b];
  if (place.y < 2) return;
  combine<D, SLICES, WAVES>(a, request(a, b), hkv, 0, blockIdx.x / SLICES, blockIdx.x % SLICES, (int64_t)hkv * a.slots + place.x,
                            place.y, gridDim.x / SLICES * 2, a.rows);
}

// Of the tile kernel's splits: workgroups over the slices of all row tiles that have several.
// (With cu_q so many whatever the batch holds: 40 chunks that split nothing 153 us, 156 with 2048; 7 that split 67 and 66.)
constexpr int kTileCombine = 1024;
template <int D>
__global__ __launch_bounds__(4 * kWave) void attn_tile_combine_kernel(AttnArgs a) {
  using S = TileShape<D>;
  constexpr int kSlices = 2, kPairs = S::kRows / 16 * (D / 16) / 2;
  const Batch<S::kRows> batch(a);
  const int most = batch.splits();
  if (most < 2) return;
  for (int u = blockIdx.x; u < batch.total * a.HKV * (kPairs * kSlices); u += gridDim.x) {
    const int unit = u / (kPairs * kSlices), part = u % (kPairs * kSlices), t = unit / a.HKV;
    int b, row_tile, splits, per;
    if (!batch.find(t, b, row_tile)) continue;
    const Request r = request(a, b);
    const int last_row = min((row_tile + 1) * S::kRows, r.n * a.G) - 1;
    stage_splits(max(r.seq - r.n + divide(last_row, a.by_g) + 1, 0), most, splits, per);
    if (splits < 2) continue;
    combine<D, kSlices, 4>(a, r, unit - t * a.HKV, row_tile * S::kRows, part / kSlices, part % kSlices, (int64_t)unit * most, splits,
                           2 * kPairs, S::kRows);
    __syncthreads();  // what it left in LDS has been read
  }
}

typedef void (*AttnFn)(AttnArgs);

struct Split {
  AttnFn fn;
  int row_tiles, threads, lds;
};
template <int D>
Split split_kernel(int rt) {
  constexpr int threads = kSplitWaves * kWave;
  if (rt == 1) return {&attn_split_kernel<D, 1, 1>, 1, threads, split_lds<D, 1>()};
  if (rt == 2) return {&attn_split_kernel<D, 2, 1>, 2, threads, split_lds<D, 2>()};
  return {&attn_split_kernel<D, 2, 2>, 4, threads, split_lds<D, 2>()};
}
Split split_of(int D, int rows) {
  const int rt = (rows + 15) / 16;
  return D == 64 ? split_kernel<64>(rt) : D == 128 ? split_kernel<128>(rt) : split_kernel<256>(rt);
}

struct Combine {
  AttnFn fn;
  int slices, threads;
};
template <int SLICES, int WAVES>
Combine combine_of(int D) {
  return {D == 64    ? &attn_combine_kernel<64, SLICES, WAVES>
          : D == 128 ? &attn_combine_kernel<128, SLICES, WAVES>
                     : &attn_combine_kernel<256, SLICES, WAVES>,
          SLICES, WAVES * kWave};
}

// How a call runs: its launches and the parts of its workspace.
struct Plan {
  bool tiles, split;  // the tile kernel; the split kernel with the combination
  int workers, slots, rows;         // split kernel
  int row_tiles;                    // tile kernel: of a request at most
  int64_t tile_groups;              // its workgroups
  bool cut;                         // it may split positions
  int combine_groups;               // whose results are added by as many
  size_t o, ml, plan, tile_o, tile_ml, bytes;  // offsets and size of the workspace
};
size_t round256(size_t n) { return (n + 255) / 256 * 256; }

int tile_rows(int D) { return D == 256 ? TileShape<256>::kRows : D == 128 ? TileShape<128>::kRows : TileShape<64>::kRows; }

// Requests of up to QF_KV4_MAX_ROWS packed rows are split over positions, larger ones tiled over rows; a batch with lengths of its
// own may hold both kinds (a chunk of 700 tokens beside single ones of 4000 positions).
Plan plan_of(const qf_kv4_attention_args& u) {
  Plan p = {};
  const int64_t rows = (int64_t)u.q_len * (u.num_heads / u.num_kv_heads);
  p.tiles = rows > QF_KV4_MAX_ROWS;
  p.split = !p.tiles || u.cu_q != nullptr;
  size_t n = 0;
  if (p.tiles) {
    const int per = tile_rows(u.head_size);
    p.row_tiles = (int)((rows + per - 1) / per);
    // The row tiles of the batch: as many as all requests could have, or with cu_q as the tokens fill, each request's last one being
    // short.  Positions are split where the tiles that the requests turn out to have leave compute units idle (100 tokens behind
    // 4000 positions, 64 heads over 8: 115 -> 34 us): without cu_q that is known here.
    const int64_t all = (int64_t)p.row_tiles * u.num_reqs;
    const int64_t by_tokens = ((int64_t)u.num_tokens * (u.num_heads / u.num_kv_heads) + per - 1) / per + u.num_reqs;
    p.tile_groups = (u.cu_q && by_tokens < all ? by_tokens : all) * u.num_kv_heads;
    p.cut = u.cu_q || compute_units() / p.tile_groups >= 2;
    if (p.cut) {
      p.combine_groups = u.cu_q ? kTileCombine : (int)p.tile_groups * (per / 16) * (u.head_size / 16);
      p.tile_groups = std::max<int64_t>(p.tile_groups, compute_units());
      p.tile_o = n;
      n += (size_t)compute_units() * per * u.head_size * sizeof(float);
      p.tile_ml = n;
      n += round256((size_t)compute_units() * per * sizeof(float2));
    }
  }
  if (!p.split) {
    p.bytes = n;
    return p;
  }
  p.rows = rows < QF_KV4_MAX_ROWS ? (int)rows : QF_KV4_MAX_ROWS;
  // A workgroup a compute unit.  Three where the requests by themselves fill the machine, so that the longest of them is cut finer and
  // one's waits are another's work: 48 requests of up to 9000 positions over 8 kv heads 28.0 us with one, 24.9 with two, 23.0 with
  // three; 16 requests, which do not fill it, 18.6 with one, 22.9 with two.  Not where the registers of a workgroup (over 180 a
  // lane) leave no room for three (40 requests of 32 rows 29.8, 32.9, 33.0; D = 256, 70 requests of 30 rows 39.9, 46.4, 55.1), nor
  // where each workgroup's look at all requests counts (260 over one kv head 16.3, 17.6, 18.9; 400 over 8 heads 56, 58, 60).
  // About 128 requests neither is the better one throughout (three, one; 64 heads of 128 over 8): of up to 2000 positions 64 requests
  // 26.9 and 23.9, 96 34.2 and 37.3, 128 44.8 and 39.6, 160 51.3 and 51.5, 260 71.7 and 70.3; of up to 9000 128 149.5 and 144.1, 160
  // 169 and 179; 32 heads of 64 over 4, of up to 4000, 128 22.4 and 32.6, 160 30.2 and 38.1.
  const int row_tiles = split_of(u.head_size, p.rows).row_tiles;
  const bool full = (int64_t)u.num_reqs * u.num_kv_heads >= compute_units();
  const int cus = compute_units() * (full && std::min(row_tiles, 2) * u.head_size <= 128 && u.num_reqs <= 128 ? 3 : 1);
  p.workers = (cus + u.num_kv_heads - 1) / u.num_kv_heads;
  p.slots = p.workers + u.num_reqs;
  const size_t parts = (size_t)u.num_kv_heads * p.slots;
  p.o = n;
  n += parts * row_tiles * 16 * u.head_size * sizeof(float);
  p.ml = n;
  n += round256(parts * p.rows * sizeof(float2));
  p.plan = n;
  p.bytes = n + round256((size_t)u.num_reqs * sizeof(int2));
  return p;
}

bool sizes_fit(const qf_kv4_attention_args& u) {
  return u.num_reqs >= 1 && u.q_len >= 1 && u.num_heads >= 1 && u.num_kv_heads >= 1 && u.num_heads % u.num_kv_heads == 0 &&
         (u.head_size == 64 || u.head_size == 128 || u.head_size == 256) &&
         (int64_t)u.q_len * (u.num_heads / u.num_kv_heads) <= 0x3fffffff && u.num_kv_heads <= QF_KV4_MAX_REQS &&
         u.num_reqs <= QF_KV4_MAX_REQS;
}

constexpr int kAloneLds = 82 * 1024;  // of 160 KiB
constexpr int kManyPositions = 4096;

// |scale| log2 e.  A masked score is -inf, which 0 would make no number: then 2^-149, the least number there is (the kernels keep such
// numbers), which moves no score of fp32 by more than 2^-21.  By its bits: a host thread may flush it to 0.
float base2_scale(float scale) {
  const float s = fabsf(scale) * kLog2e;
  uint32_t bits;
  memcpy(&bits, &s, sizeof bits);
  bits = std::max(bits, 1u);
  float out;
  memcpy(&out, &bits, sizeof out);
  return out;
}
std::atomic<uint64_t> g_raised[3][5];

int launch(AttnFn fn, dim3 grid, int threads, size_t lds, std::atomic<uint64_t>& raised, hipStream_t s, const AttnArgs& a) {
  if (!grid_fits(grid.x, threads)) return QF_ERR_UNSUPPORTED;
  if (lds + 4096 > kDefaultLds && !raise_lds(reinterpret_cast<const void*>(fn), std::max((int)lds, kAloneLds), raised))
    return QF_ERR_HIP;
  hipLaunchKernelGGL(fn, grid, dim3(threads), lds, s, a);
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
  if (!sizes_fit(u) || (int64_t)u.max_blocks * u.page_size > 0x7fffffc0 || u.page_size % kTile || u.cache_stride % 16 ||
      !aligned16(u.cache) ||
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
  a.few = p.split ? p.rows : 0;
  a.workers = p.workers;
  a.slots = p.slots;
  a.qk_scale = base2_scale(u.scale);
  a.flip = u.scale < 0 ? 0x80008000u : 0;
  a.by_g = divisor(a.G);
  a.by_page = divisor(u.page_size);
  a.by_workers = divisor(p.split ? p.workers : 1);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int D = u.head_size, di = D == 64 ? 0 : D == 128 ? 1 : 2;
  a.cus = compute_units();
  if (p.tiles) {
    a.o_part = reinterpret_cast<float*>(ws + p.tile_o);
    a.ml_part = reinterpret_cast<float2*>(ws + p.tile_ml);
    static_assert(TileShape<64>::kWaves == TileShape<128>::kWaves && TileShape<256>::kWaves == TileShape<128>::kWaves, "one shape");
    const AttnFn fn = D == 64 ? &attn_tile_kernel<64> : D == 128 ? &attn_tile_kernel<128> : &attn_tile_kernel<256>;
    const int lds = D == 64 ? TileShape<64>::kLds : D == 128 ? TileShape<128>::kLds : TileShape<256>::kLds;
    if (!grid_fits(p.tile_groups, TileShape<128>::kWaves * kWave)) return QF_ERR_UNSUPPORTED;
    int st = launch(fn, dim3((unsigned)p.tile_groups), TileShape<128>::kWaves * kWave, lds, g_raised[di][3], s, a);
    if (st != QF_OK) return st;
    if (p.cut) {
      const AttnFn comb = D == 64    ? &attn_tile_combine_kernel<64>
                          : D == 128 ? &attn_tile_combine_kernel<128>
                                     : &attn_tile_combine_kernel<256>;
      st = launch(comb, dim3(p.combine_groups), 4 * kWave, 0, g_raised[di][0], s, a);
      if (st != QF_OK) return st;
    }
    if (!p.split) return QF_OK;
  }
  a.o_part = reinterpret_cast<float*>(ws + p.o);
  a.ml_part = reinterpret_cast<float2*>(ws + p.ml);
  a.plan = reinterpret_cast<int2*>(ws + p.plan);
  const Split k = split_of(D, p.rows);
  const int64_t pairs = (int64_t)k.row_tiles * (D / 32) * a.HKV * a.B;
  // Small slices where that gives a compute unit a few workgroups at most (3 queries behind 38 000 positions, 64 splits of 18 rows of
  // 256: 26.4 -> 23.1 us with the splits themselves, 7 requests of 4 queries 12.6 -> 10.8; 16 requests of up to 3000 18.5, 18.7).
  const Combine c = 4 * pairs <= 4 * compute_units() ? combine_of<4, 8>(D) : combine_of<2, 4>(D);
  // Where a workgroup a compute unit is all there is, none takes two of them: each asks for more than half of the LDS (100 000
  // positions 35.7 -> 30.8 us, 30 000 17.0 -> 15.5, D = 256 19.6 -> 16.5; at 1000 8.6 -> 8.9, so not for tables that end there).
  // The lengths are on the device, the table's width stands for them: a short request behind a server's wide table pays for it
  // (64 heads of 128 over 8 behind 2560 pages of 16: 1000 positions 8.4 -> 8.7 us, 2000 8.4 -> 8.8, 4000 9.4 -> 9.5, 100 and 300 level).
  const bool alone = (int64_t)p.slots * a.HKV <= compute_units() * 5 / 4 && (int64_t)a.max_blocks * a.page >= kManyPositions;
  const int lds = alone ? std::max(k.lds, kAloneLds) : k.lds;
  const int st = launch(k.fn, dim3(p.slots, a.HKV), k.threads, lds, g_raised[di][k.row_tiles], s, a);
  if (st != QF_OK) return st;
  return launch(c.fn, dim3(k.row_tiles * D / 32 * c.slices, a.HKV, a.B), c.threads, 0, g_raised[di][0], s, a);
}
