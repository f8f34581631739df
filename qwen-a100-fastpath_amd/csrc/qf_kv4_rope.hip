// qf_kv4_rope.hip — norms of query and key heads with the position rotation and the write into the cache (gfx950).
//
// A row is a head of a token: D / 8 lanes of 16 bytes each, 64 / (D / 8) rows of one kind (query, key, value) a chunk, side by side
// in a wavefront.  Per row: the mean of squares over its lanes (DPP adds), the norm's factor, the rotation (the other value of a
// pair stands in the same lane, or rot / 16 lanes away and comes by a lane permutation), one rounding to bf16, and for keys and
// values their page, or blocks of 32 values (4 lanes) to 4 bits.
//
// A wavefront takes several chunks of one kind, the next one's rows requested before the last one's work, and the angles and
// weights, which a lane needs for one token only, once for all of them.  Queries: the chunks are heads of one token.  Keys and
// values: a chunk is one head of 64 / L neighbouring tokens, whose bytes of a 4-bit record stand together, and the 4 wavefronts
// of a workgroup take further neighbours.
//
// Memory bounds it where there are many rows (2048 tokens of 64 + 8 heads of 128 into 4 bits: 80 MB in 19 us, 4.2 TB/s; 8191 of 16 + 2
// into bf16 pages: 86 MB in 16.8 us, 5.1 TB/s, part of it in the caches), the chain position, angles, stores where there are few
// (5 tokens 3.7 us).  The fp64 rows of keys are one in eight to ten (64 + 8 + 8 heads: 10%, 24 + 4 + 4: 12%) and cost no registers: 78
// a lane, 6 wavefronts a SIMD.
#include "qf_kv4_common.h"

namespace qfk {

constexpr int kRopeThreads = 256;
constexpr int kRopeWaves = kRopeThreads / kWave;

// Chunks of a wavefront: one until each compute unit has 8 wavefronts, then up to 4.  Measured with 1, 2, 4 and 8 chunks: 5 tokens of
// 64 + 8 heads of 128 (112 chunks) 5.7, 6.3, 7.8, 10.7 us; 333 of 24 + 4 of 256 (5300) 8.8, 8.4, 9.7, 11.8; 2048 of 64 + 8 of 128
// (41 000) 30.9, 27.3, 25.0, 24.8; 8191 of 16 + 2 of 128 (41 000, into pages) 27.7, 22.4, 22.1, 26.5.
constexpr int kWavesBeforeMore = 8;
constexpr int kMostChunks = 4;

struct RopeArgs {
  qf_qk_norm_rope_args u;
  Divisor by_page, by_q, by_kv;
  int chunks;            // of a wavefront
  int kv_waves;          // wavefronts of keys and values, whole workgroups; those of queries follow
  int q_items;           // wavefronts of a token's queries
  int k_items, v_items;  // workgroups of 4 * 64 / L tokens' keys and values
};

template <typename T>
__device__ __forceinline__ void load8(float (&f)[8], const T* p);
template <>
__device__ __forceinline__ void load8<float>(float (&f)[8], const float* p) {
  const f32x4_t lo = *reinterpret_cast<const f32x4_t*>(p), hi = *reinterpret_cast<const f32x4_t*>(p + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = lo[i];
    f[4 + i] = hi[i];
  }
}
template <>
__device__ __forceinline__ void load8<uint16_t>(float (&f)[8], const uint16_t* p) {
  unpack8(*reinterpret_cast<const u32x4_t*>(p), f);
}
template <typename T>
__device__ __forceinline__ void load4(float (&f)[4], const T* p);
template <>
__device__ __forceinline__ void load4<float>(float (&f)[4], const float* p) {
  const f32x4_t v = *reinterpret_cast<const f32x4_t*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = v[i];
}
template <>
__device__ __forceinline__ void load4<uint16_t>(float (&f)[4], const uint16_t* p) {
  const u32x2_t v = *reinterpret_cast<const u32x2_t*>(p);
  f[0] = bf16_lo(v.x);
  f[1] = bf16_hi(v.x);
  f[2] = bf16_lo(v.y);
  f[3] = bf16_hi(v.y);
}

// What a row's 8 values of a lane become is n_i = factor (x_i a_i + o_i b_i): o the values that pair with x, a and b the norm's
// weights times the angle's cosine and (with its sign) sine.
struct Turn {
  u32x4_t w, wo;     // the weights of x and of o, bf16
  float c[8], s[8];  // -s where a value is the first of its pair; c = 1 and s = -0 outside the rotation
  double offset, eps;
  bool norm;
};

template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xf, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xf, 0xf, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int L>
__device__ __forceinline__ double group_sum(double v) {  // as the sum of floats
  v += dpp_f64<0xB1>(v);
  v += dpp_f64<0x4E>(v);
  v += dpp_f64<0x141>(v);
  if constexpr (L >= 16) v += dpp_f64<0x140>(v);
  if constexpr (L >= 32) v += __shfl_xor(v, 16);
  return v;
}

template <int L, bool INTERLEAVED>
__device__ __forceinline__ void paired(u32x4_t x, int other, bool turn, float (&o)[8]) {
  if constexpr (INTERLEAVED) {
    unpack8(x, o);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float first = o[i];
      o[i] = turn ? o[i + 1] : 0.0f;
      o[i + 1] = turn ? first : 0.0f;
    }
  } else {
    u32x4_t y;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t from = (uint32_t)__shfl((int)x[i], other);
      y[i] = turn ? from : 0;  // (an infinity times no sine is not a number)
    }
    unpack8(y, o);
  }
}

// In fp32, a and b as computed once for all rows of a wavefront.
template <int L>
__device__ __forceinline__ u32x4_t turned(u32x4_t mine, float (&o)[8], const Turn& at, const float (&a)[8], const float (&b)[8]) {
  float x[8];
  unpack8(mine, x);
  float factor = 1.0f;
  if (at.norm) {
    float sum = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
    sum = group_sum<L>(sum);
    float eps = (float)at.eps;
    // Squares outside fp32's range (their sum does not hold them, nor is it nothing beside eps): the row times a power of two.
    if (!(sum <= 0x1p+126f && (sum >= 0x1p-90f || at.eps >= 0x1p-110))) {
      const float up = sum < 1.0f ? 0x1p+100f : 0x1p-80f;
      sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] *= up;
        o[i] *= up;
        sum = fmaf(x[i], x[i], sum);
      }
      sum = group_sum<L>(sum);
      eps = (float)(at.eps * ((double)up * up));
    }
    factor = 1.0f / sqrtf(fmaf(sum, 1.0f / (8 * L), eps));
  }
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = fmaf(o[i] * factor, b[i], x[i] * factor * a[i]);
  return pack8(y);
}

// In fp64: the result, rounded to bf16, does not depend on the order of the sums.
template <int L>
__device__ __forceinline__ u32x4_t turned(u32x4_t mine, const float (&o)[8], const Turn& at) {
  float x[8], w[8], wo[8], y[8];
  unpack8(mine, x);
  unpack8(at.w, w);
  unpack8(at.wo, wo);
  double factor = 1;
  if (at.norm) {
    double sum = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fma((double)x[i], (double)x[i], sum);
    factor = 1.0 / sqrt(fma(group_sum<L>(sum), 1.0 / (8 * L), at.eps));
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const double n = (double)x[i] * factor * (at.offset + (double)w[i]), m = (double)o[i] * factor * (at.offset + (double)wo[i]);
    y[i] = (float)fma(m, (double)at.s[i], n * (double)at.c[i]);
    if (i % 2) __builtin_amdgcn_sched_barrier(0);  // (8 values in work at once take 60 registers more)
  }
  return pack8(y);
}

// A lane's 8 bf16 values of a block of 32 (4 neighbouring lanes) as codes (a dword) and the block's scale byte.
__device__ __forceinline__ uint32_t four_bits(u32x4_t v, uint32_t* byte) {
  uint32_t top = 0;  // the largest magnitude's bits, as bf16
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, max(v[i] & 0x7fffu, v[i] >> 16 & 0x7fffu));
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xf, 0xf, false));
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xf, 0xf, false));
  // below 7 * 2^e: from mantissa 1.75 on the exponent is one more; 6 * 2^125 is the largest value (2^128 would be infinite)
  const uint32_t e = min(max((top + 0x20u) >> 7, 4u) - 2, 252u);
  if (top >= 0x7f80u) {
    *byte = 255;
    return 0;
  }
  *byte = e;
  const float scale = __uint_as_float(e << 23);
  const uint32_t v0 = v[0], v1 = v[1], v2 = v[2], v3 = v[3];  // (a bit cast of a vector's element takes its first one)
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_t, v0), scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_t, v1), scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_t, v2), scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_t, v3), scale, 3);
}

enum { kQuery, kKey, kKey4, kValue };  // kKey4: a key for the 4-bit cache

// Chunks of a token's heads from `head` on, `step` heads apart.
template <int D, bool INTERLEAVED, typename TABLE, int KIND>
__device__ __forceinline__ void run_chunks(const RopeArgs& args, int t, int head, int step) {
  const qf_qk_norm_rope_args& a = args.u;
  constexpr int L = D / 8;  // lanes of a row
  const qf_heads& from = KIND == kQuery ? a.query : KIND == kValue ? a.value : a.key;
  const qf_heads& to = KIND == kQuery ? a.query_out : a.key_out;
  const int heads = t < a.num_tokens ? (KIND == kQuery ? a.num_heads : a.num_kv_heads) : 0;
  const int lane = threadIdx.x % kWave, j = lane % L;  // this lane's place in its row: values 8 j .. 8 j + 7
  const bool turn = KIND != kValue && 8 * j < a.rot && heads > 0;
  int64_t pos = 0, slot = -1;
  if (turn) pos = a.positions[t];
  if (KIND != kQuery && a.cache_kind != QF_CACHE_NONE && heads > 0) slot = a.slots[t];
  const uint16_t* p = from.data + t * from.stride_tok + head * from.stride_head + 8 * j;
  u32x4_t next = {0, 0, 0, 0};
  if (head < heads) next = *reinterpret_cast<const u32x4_t*>(p);

  const int half = a.rot / 16;  // lanes from a pair's first value to its second
  const int other = INTERLEAVED || !turn ? j : j < half ? j + half : j - half;
  const int partner = lane - j + other;
  Turn at;
  float fa[8], fb[8];
  if constexpr (KIND != kValue) {
    const uint16_t* weight = KIND == kQuery ? a.q_weight : a.k_weight;
    at.norm = weight != nullptr;
    at.offset = at.norm ? a.weight_offset : 1.0;
    at.eps = a.eps;
    at.w = at.wo = u32x4_t{0, 0, 0, 0};
    if (at.norm) {
      at.w = *reinterpret_cast<const u32x4_t*>(weight + 8 * j);
      at.wo = *reinterpret_cast<const u32x4_t*>(weight + 8 * other);
      if constexpr (INTERLEAVED) {
#pragma unroll
        for (int i = 0; i < 4; ++i) at.wo[i] = __builtin_amdgcn_alignbit(at.w[i], at.w[i], 16);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      at.c[i] = 1.0f;
      at.s[i] = -0.0f;
    }
    if (turn) {
      pos = pos < 0 ? 0 : pos >= a.num_positions ? a.num_positions - 1 : pos;
      const TABLE* cs = static_cast<const TABLE*>(a.cos_sin) + pos * a.rot;
      if constexpr (INTERLEAVED) {
        float c[4], s[4];
        load4(c, cs + 4 * j);
        load4(s, cs + a.rot / 2 + 4 * j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          at.c[2 * i] = at.c[2 * i + 1] = c[i];
          at.s[2 * i] = -s[i];
          at.s[2 * i + 1] = s[i];
        }
      } else {
        const int first = 8 * (j < half ? j : other);
        load8(at.c, cs + first);
        load8(at.s, cs + a.rot / 2 + first);
#pragma unroll
        for (int i = 0; i < 8; ++i) at.s[i] = j < half ? -at.s[i] : at.s[i];
      }
    }
    if constexpr (KIND != kKey4) {
      unpack8(at.w, fa);
      unpack8(at.wo, fb);
      const float offset = (float)at.offset;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        fa[i] = (offset + fa[i]) * at.c[i];
        fb[i] = (offset + fb[i]) * at.s[i];
      }
    }
  }
  const bool kept = KIND != kQuery && slot >= 0 && slot < a.num_blocks * a.page_size;
  int64_t block = 0;
  if (kept) block = slot <= 0x7fffffff ? divide((int)slot, args.by_page) : slot / a.page_size;
  const int place = kept ? (int)(slot - block * a.page_size) : 0;
  uint16_t* out = KIND == kValue || to.data == nullptr ? nullptr : to.data + t * to.stride_tok + head * to.stride_head + 8 * j;
#pragma unroll 1
  for (int c = 0; c < args.chunks; ++c) {
    u32x4_t x = next;
    const bool in = head < heads;
    head += step;
    p += step * from.stride_head;
    if (c + 1 < args.chunks && head < heads) next = *reinterpret_cast<const u32x4_t*>(p);
    if constexpr (KIND != kValue) {
      float o[8];
      if constexpr (KIND == kKey4) {
        // Widened anew for each chunk: kept, the weights and angles would take 64 registers in fp64.
#pragma unroll
        for (int i = 0; i < 8; ++i) asm volatile("" : "+v"(at.c[i]), "+v"(at.s[i]));
        asm volatile("" : "+v"(at.w), "+v"(at.wo));
        paired<L, INTERLEAVED>(x, partner, turn, o);
        x = turned<L>(x, o, at);
      } else {
        paired<L, INTERLEAVED>(x, partner, turn, o);
        x = turned<L>(x, o, at, fa, fb);
      }
      if (out != nullptr) {
        if (in) *reinterpret_cast<u32x4_t*>(out) = x;
        out += step * to.stride_head;
      }
    }
    if constexpr (KIND != kQuery) {
      if (!(kept && in)) continue;
      if (KIND == kKey4 || (KIND == kValue && a.cache_kind == QF_CACHE_KV4)) {
        using R = Record<D>;
        uint8_t* rec = static_cast<uint8_t*>(a.cache) + block * a.cache_stride +
                       ((int64_t)(head - step) * (a.page_size / kTile) + place / kTile) * R::kBytes;
        const int q = place % kTile;
        uint32_t byte;
        const uint32_t codes = four_bits(x, &byte);
        if constexpr (KIND == kKey4) {
          *reinterpret_cast<uint32_t*>(rec + R::key(q, 8 * j)) = codes;
        } else if constexpr (R::kWidth == 8) {
          *reinterpret_cast<uint32_t*>(rec + R::value(q, 8 * j)) = codes;
        } else {
          *reinterpret_cast<uint16_t*>(rec + R::value(q, 8 * j)) = (uint16_t)codes;
          *reinterpret_cast<uint16_t*>(rec + R::value(q, 8 * j + 4)) = (uint16_t)(codes >> 16);
        }
        if (j % 4 == 0) rec[KIND == kKey4 ? R::key_scale(q, 8 * j) : R::value_scale(q, 8 * j)] = (uint8_t)byte;
      } else {
        const qf_pages& pages = KIND == kValue ? a.value_pages : a.key_pages;
        *reinterpret_cast<u32x4_t*>(pages.data + block * pages.stride_block + place * pages.stride_tok +
                                    (head - step) * pages.stride_head + 8 * j) = x;
      }
    }
  }
}

template <int D, bool INTERLEAVED, typename TABLE>
__global__ __launch_bounds__(kRopeThreads) void qk_norm_rope_kernel(RopeArgs args) {
  constexpr int kRows = kWave / (D / 8);  // rows of a chunk
  const int row = threadIdx.x % kWave / (D / 8);
  const int wave = __builtin_amdgcn_readfirstlane(blockIdx.x * kRopeWaves + threadIdx.x / kWave);
  if (wave >= args.kv_waves) {
    const int t = divide(wave - args.kv_waves, args.by_q);
    const int item = wave - args.kv_waves - t * args.q_items;
    run_chunks<D, INTERLEAVED, TABLE, kQuery>(args, t, item * args.chunks * kRows + row, kRows);
    return;
  }
  const int n = wave / kRopeWaves, tokens = divide(n, args.by_kv);
  const int item = n - tokens * (args.k_items + args.v_items);
  const int t = (tokens * kRopeWaves + wave % kRopeWaves) * kRows + row;
  if (item >= args.k_items) {
    run_chunks<D, INTERLEAVED, TABLE, kValue>(args, t, (item - args.k_items) * args.chunks, 1);
  } else if (args.u.cache_kind == QF_CACHE_KV4) {
    run_chunks<D, INTERLEAVED, TABLE, kKey4>(args, t, item * args.chunks, 1);
  } else {
    run_chunks<D, INTERLEAVED, TABLE, kKey>(args, t, item * args.chunks, 1);
  }
}

struct LoadArgs {
  const uint8_t* cache;
  int64_t stride, num_blocks;
  int page, HK, T;
  const int64_t* slots;
  uint16_t *key, *value;
  Divisor by_heads, by_page;
};

// D / 8 lanes a head of a token: 8 values each of the key and of the value (2048 tokens of 8 heads of 128: 10.6 MB in 4.8 us).
template <int D>
__global__ __launch_bounds__(kRopeThreads) void kv4_load_kernel(LoadArgs a) {
  using R = Record<D>;
  constexpr int L = D / 8;
  const uint32_t i = blockIdx.x * kRopeThreads + threadIdx.x;  // (a launch has less than 2^32 threads)
  const int j = i % L;
  const int64_t at = i / L;  // token * HK + head
  if (at >= (int64_t)a.T * a.HK) return;
  const int t = divide((int)at, a.by_heads), head = (int)at - t * a.HK;
  const int64_t slot = a.slots[t];
  u32x4_t k = {0, 0, 0, 0}, v = k;
  if (slot >= 0 && slot < a.num_blocks * a.page) {
    const int64_t block = slot <= 0x7fffffff ? divide((int)slot, a.by_page) : slot / a.page;
    const int p = (int)(slot - block * a.page), q = p % kTile;
    const uint8_t* rec = a.cache + block * a.stride + ((int64_t)head * (a.page / kTile) + p / kTile) * R::kBytes;
    uint32_t w;
    if constexpr (R::kWidth == 8) {
      w = *reinterpret_cast<const uint32_t*>(rec + R::value(q, 8 * j));
    } else {
      w = *reinterpret_cast<const uint16_t*>(rec + R::value(q, 8 * j)) |
          (uint32_t)*reinterpret_cast<const uint16_t*>(rec + R::value(q, 8 * j + 4)) << 16;
    }
    k = widen8(*reinterpret_cast<const uint32_t*>(rec + R::key(q, 8 * j)), scale_of<0>(rec[R::key_scale(q, 8 * j)]));
    v = widen8(w, scale_of<0>(rec[R::value_scale(q, 8 * j)]));
  }
  *reinterpret_cast<u32x4_t*>(a.key + at * D + 8 * j) = k;
  *reinterpret_cast<u32x4_t*>(a.value + at * D + 8 * j) = v;
}

typedef void (*RopeFn)(RopeArgs);

template <int D>
RopeFn rope_kernel(bool interleaved, bool f32) {
  if (interleaved) return f32 ? &qk_norm_rope_kernel<D, true, float> : &qk_norm_rope_kernel<D, true, uint16_t>;
  return f32 ? &qk_norm_rope_kernel<D, false, float> : &qk_norm_rope_kernel<D, false, uint16_t>;
}

bool blocks_fit(int64_t blocks, int page) { return blocks <= (int64_t)1 << 40 && blocks <= ((int64_t)1 << 62) / page; }
bool strides_fit(int64_t a, int64_t b, const void* p) { return a >= 0 && b >= 0 && a % 8 == 0 && b % 8 == 0 && aligned16(p); }

}  // namespace qfk

using namespace qfk;

extern "C" int qf_qk_norm_rope(const qf_qk_norm_rope_args* args, void* stream) {
  if (!args) return QF_ERR_INVALID_ARG;
  const qf_qk_norm_rope_args& u = *args;
  const bool query = u.query.data != nullptr, cache = u.cache_kind != QF_CACHE_NONE;
  if (!u.key.data || u.num_tokens < 1 || u.num_kv_heads < 1 || (query && u.num_heads < 1) || query != (u.query_out.data != nullptr) ||
      u.cache_kind < QF_CACHE_NONE || u.cache_kind > QF_CACHE_KV4 || cache != (u.value.data != nullptr) ||
      (!cache && !u.key_out.data) || !(u.eps >= 0) || u.rot < 0 || u.rot > u.head_size ||
      (u.rot > 0 && (!u.positions || !u.cos_sin || u.num_positions < 1)))
    return QF_ERR_INVALID_ARG;
  if (cache && (!u.slots || u.num_blocks < 1 || u.page_size < 1)) return QF_ERR_INVALID_ARG;
  if (u.cache_kind == QF_CACHE_KV4 && !u.cache) return QF_ERR_INVALID_ARG;
  if (u.cache_kind == QF_CACHE_PAGES && (!u.key_pages.data || !u.value_pages.data)) return QF_ERR_INVALID_ARG;
  const int D = u.head_size;
  if ((D != 64 && D != 128 && D != 256) || u.rot % 16) return QF_ERR_UNSUPPORTED;
  for (const qf_heads* h : {&u.query, &u.key, &u.value, &u.query_out, &u.key_out})
    if (h->data && !strides_fit(h->stride_tok, h->stride_head, h->data)) return QF_ERR_UNSUPPORTED;
  if (!aligned16(u.q_weight) || !aligned16(u.k_weight) || (u.rot > 0 && !aligned16(u.cos_sin))) return QF_ERR_UNSUPPORTED;
  if (u.cache_kind == QF_CACHE_KV4 && (u.page_size % kTile || u.cache_stride % 16 || !aligned16(u.cache) ||
                                       u.cache_stride < (int64_t)u.num_kv_heads * (u.page_size / kTile) * 17 * D))
    return QF_ERR_UNSUPPORTED;
  if (u.cache_kind == QF_CACHE_PAGES)
    for (const qf_pages* p : {&u.key_pages, &u.value_pages})
      if (!strides_fit(p->stride_tok, p->stride_head, p->data) || p->stride_block < 0 || p->stride_block % 8)
        return QF_ERR_UNSUPPORTED;
  const int64_t rows = kWave / (D / 8), T = u.num_tokens;
  auto over = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  const int64_t q_chunks = query ? over(u.num_heads, rows) : 0;
  const int64_t all = T * q_chunks + over(T, rows) * u.num_kv_heads * (cache ? 2 : 1);
  const int ch = (int)std::min<int64_t>(std::max<int64_t>(all / (kWavesBeforeMore * (int64_t)compute_units()), 1), kMostChunks);
  const int64_t q_items = over(q_chunks, ch), k_items = over(u.num_kv_heads, ch), v_items = cache ? k_items : 0;
  if (q_items > 0xffffff || k_items > 0xffffff) return QF_ERR_UNSUPPORTED;
  const int64_t kv_waves = over(T, kRopeWaves * rows) * kRopeWaves * (k_items + v_items);
  const int64_t waves = kv_waves + over(T * q_items, kRopeWaves) * kRopeWaves;
  // wavefronts are counted in 31 bits, slots in 62
  if (waves > 0x7fffffff - kRopeWaves || (cache && !blocks_fit(u.num_blocks, u.page_size))) return QF_ERR_UNSUPPORTED;
  const int64_t groups = waves / kRopeWaves;
  if (!grid_fits(groups, kRopeThreads)) return QF_ERR_UNSUPPORTED;
  RopeArgs a = {u, divisor(cache ? u.page_size : 1), divisor(query ? (int)q_items : 1), divisor((int)(k_items + v_items)), ch,
                (int)kv_waves, (int)q_items, (int)k_items, (int)v_items};
  const RopeFn fn = D == 64    ? rope_kernel<64>(u.interleaved, u.cos_sin_f32)
                    : D == 128 ? rope_kernel<128>(u.interleaved, u.cos_sin_f32)
                               : rope_kernel<256>(u.interleaved, u.cos_sin_f32);
  hipLaunchKernelGGL(fn, dim3((unsigned)groups), dim3(kRopeThreads), 0, static_cast<hipStream_t>(stream), a);
  return hipGetLastError() == hipSuccess ? QF_OK : QF_ERR_HIP;
}

extern "C" int qf_kv4_load(const void* cache, int64_t cache_stride, int64_t num_blocks, int page_size, int num_kv_heads,
                           int head_size, const int64_t* slots, int num_tokens, uint16_t* key, uint16_t* value, void* stream) {
  if (!cache || !slots || !key || !value || num_blocks < 1 || page_size < 1 || num_kv_heads < 1 || num_tokens < 1)
    return QF_ERR_INVALID_ARG;
  const int D = head_size;
  if ((D != 64 && D != 128 && D != 256) || page_size % kTile || cache_stride % 16 || !aligned16(cache) || !aligned16(key) ||
      !aligned16(value) || !blocks_fit(num_blocks, page_size) ||
      cache_stride < (int64_t)num_kv_heads * (page_size / kTile) * 17 * D)
    return QF_ERR_UNSUPPORTED;
  if ((int64_t)num_tokens * num_kv_heads > 0x7fffffff) return QF_ERR_UNSUPPORTED;  // heads are counted in 31 bits
  const int64_t groups = ((int64_t)num_tokens * num_kv_heads * (D / 8) + kRopeThreads - 1) / kRopeThreads;
  if (!grid_fits(groups, kRopeThreads)) return QF_ERR_UNSUPPORTED;
  const LoadArgs a = {static_cast<const uint8_t*>(cache), cache_stride, num_blocks, page_size, num_kv_heads, num_tokens, slots,
                      key, value, divisor(num_kv_heads), divisor(page_size)};
  const auto fn = D == 64 ? &kv4_load_kernel<64> : D == 128 ? &kv4_load_kernel<128> : &kv4_load_kernel<256>;
  hipLaunchKernelGGL(fn, dim3((unsigned)groups), dim3(kRopeThreads), 0, static_cast<hipStream_t>(stream), a);
  return hipGetLastError() == hipSuccess ? QF_OK : QF_ERR_HIP;
}
