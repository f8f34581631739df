// qf_kv4_rope.hip — norms of query and key heads with the position rotation and the write into the cache (gfx950).
//
// A row is a head of a token: D / 8 lanes of 16 bytes each, 64 / (D / 8) rows a wavefront side by side; the rows of a token
// are its query heads, its key heads and its value heads in this order.  Per row: the mean of squares over its lanes (DPP
// adds), the norm's factor, the rotation (the other value of a pair stands in the same lane, or rot / 16 lanes away and comes
// by a lane permutation), one rounding to bf16, and for keys and values their page, or blocks of 32 values (4 lanes) to 4 bits.
#include "qf_kv4_common.h"

namespace qfk {

constexpr int kRopeThreads = 256;
constexpr int kRopeWaves = kRopeThreads / kWave;

struct RopeArgs {
  qf_qk_norm_rope_args u;
  Divisor by_page, by_parts;
  int rows;   // of a token
  int parts;  // wavefronts of a token
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

// The angles of a lane's 8 values: of each value (halves: value i and i + rot / 2 turn by one angle), or of its 4 pairs.
struct Angles {
  float c[8], s[8];
};

// The lane's 8 values of a row turned and normalised, in R (fp32 or fp64).  `other`: the bf16 values that pair with these.
// sign: -1 where these are the first of their pairs, 1 where they are the second, 0 outside the rotation.
template <int L, bool INTERLEAVED, typename R>
__device__ __forceinline__ u32x4_t turned(u32x4_t mine, u32x4_t other, bool norm, const float (&w)[8], const float (&wo)[8],
                                          const Angles& at, int sign, R offset, R eps) {
  float x[8], o[8], y[8];
  unpack8(mine, x);
  unpack8(other, o);
  R factor = 1;
  if (norm) {
    R sum = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += (R)x[i] * (R)x[i];
    if constexpr (sizeof(R) == 8) {
#pragma unroll
      for (int m = 1; m < L; m *= 2) sum += __shfl_xor(sum, m);
    } else {
      sum = group_sum<L>(sum);
      // squares outside fp32's range (their sum is not a number that holds them): this row in fp64
      if (!(sum >= 0x1p-90f && sum <= 0x1p+126f))
        return turned<L, INTERLEAVED, double>(mine, other, norm, w, wo, at, sign, (double)offset, (double)eps);
    }
    const R mean = sum * (R)(1.0 / (8 * L)) + eps;
    if constexpr (sizeof(R) == 8) {
      factor = 1.0 / sqrt(mean);
    } else {
      factor = 1.0f / sqrtf(mean);
    }
  }
  R n[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) n[i] = norm ? (R)x[i] * factor * (offset + (R)w[i]) : (R)x[i];
  if (sign != 0) {
    if constexpr (INTERLEAVED) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const R a = n[2 * i], b = n[2 * i + 1], c = at.c[i], s = at.s[i];
        n[2 * i] = a * c - b * s;
        n[2 * i + 1] = b * c + a * s;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const R m = norm ? (R)o[i] * factor * (offset + (R)wo[i]) : (R)o[i];
        n[i] = n[i] * (R)at.c[i] + (sign < 0 ? -m : m) * (R)at.s[i];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = (float)n[i];
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

template <int D, bool INTERLEAVED, typename TABLE>
__global__ __launch_bounds__(kRopeThreads) void qk_norm_rope_kernel(RopeArgs args) {
  const qf_qk_norm_rope_args& a = args.u;
  constexpr int L = D / 8;          // lanes of a row
  constexpr int kRows = kWave / L;  // rows of a wavefront
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(blockIdx.x * kRopeWaves + threadIdx.x / kWave);
  const int t = divide(wave, args.by_parts);
  if (t >= a.num_tokens) return;
  const int part = wave - t * args.parts;
  const int j = lane % L;  // this lane's place in its row: values 8 j .. 8 j + 7
  const int row = part * kRows + lane / L;
  const bool live = row < args.rows;
  const int H = a.query.data != nullptr ? a.num_heads : 0;
  const int HK = a.num_kv_heads;
  const bool is_q = row < H, is_k = !is_q && row < H + HK;
  const int head = is_q ? row : is_k ? row - H : row - H - HK;
  const qf_heads& from = is_q ? a.query : is_k ? a.key : a.value;

  u32x4_t x = {0, 0, 0, 0};
  if (live) x = *reinterpret_cast<const u32x4_t*>(from.data + t * from.stride_tok + head * from.stride_head + 8 * j);

  float w[8], wo[8];
  Angles at;
  const uint16_t* weight = is_q ? a.q_weight : is_k ? a.k_weight : nullptr;
  const bool norm = live && weight != nullptr;
  const int half = a.rot / 16;  // lanes from a pair's first value to its second
  const int other = INTERLEAVED || 8 * j >= a.rot ? j : j < half ? j + half : j - half;
  if (norm) {
    load8(w, weight + 8 * j);
    load8(wo, weight + 8 * other);
  }
  int sign = 0;
  if (8 * j < a.rot && (is_q || is_k)) {
    int64_t pos = a.positions[t];
    pos = pos < 0 ? 0 : pos >= a.num_positions ? a.num_positions - 1 : pos;
    const TABLE* cs = static_cast<const TABLE*>(a.cos_sin) + pos * a.rot;
    if constexpr (INTERLEAVED) {
      sign = 1;
      float c[4], s[4];
      load4(c, cs + 4 * j);
      load4(s, cs + a.rot / 2 + 4 * j);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        at.c[i] = c[i];
        at.s[i] = s[i];
      }
    } else {
      sign = j < half ? -1 : 1;
      const int first = 8 * (j < half ? j : other);
      load8(at.c, cs + first);
      load8(at.s, cs + a.rot / 2 + first);
    }
  }
  u32x4_t xo = x;
  if constexpr (!INTERLEAVED) {
#pragma unroll
    for (int i = 0; i < 4; ++i) xo[i] = (uint32_t)__shfl((int)x[i], lane - j + other);
  }

  // Keys for the 4-bit cache in fp64: their codes do not depend on how a sum was ordered.
  u32x4_t y = x;
  const bool wide = a.cache_kind == QF_CACHE_KV4;
  if (is_q || (is_k && !wide)) {
    y = turned<L, INTERLEAVED, float>(x, xo, norm, w, wo, at, sign, (float)a.weight_offset, (float)a.eps);
  } else if (is_k) {
    y = turned<L, INTERLEAVED, double>(x, xo, norm, w, wo, at, sign, a.weight_offset, a.eps);
  }
  if (!live) return;
  if (is_q || (is_k && a.key_out.data != nullptr)) {
    const qf_heads& to = is_q ? a.query_out : a.key_out;
    *reinterpret_cast<u32x4_t*>(to.data + t * to.stride_tok + head * to.stride_head + 8 * j) = y;
  }
  if (is_q || a.cache_kind == QF_CACHE_NONE) return;
  const int64_t slot = a.slots[t];
  if (slot < 0 || slot >= a.num_blocks * a.page_size) return;
  const int64_t block = slot <= 0x7fffffff ? divide((int)slot, args.by_page) : slot / a.page_size;
  const int p = (int)(slot - block * a.page_size);
  if (a.cache_kind == QF_CACHE_PAGES) {
    const qf_pages& to = is_k ? a.key_pages : a.value_pages;
    *reinterpret_cast<u32x4_t*>(to.data + block * to.stride_block + p * to.stride_tok + head * to.stride_head + 8 * j) = y;
    return;
  }
  using R = Record<D>;
  uint8_t* rec = static_cast<uint8_t*>(a.cache) + block * a.cache_stride +
                 ((int64_t)head * (a.page_size / kTile) + p / kTile) * R::kBytes;
  const int q = p % kTile;
  uint32_t byte;
  const uint32_t codes = four_bits(y, &byte);
  if (is_k) {
    *reinterpret_cast<uint32_t*>(rec + R::key(q, 8 * j)) = codes;
  } else if constexpr (R::kWidth == 8) {
    *reinterpret_cast<uint32_t*>(rec + R::value(q, 8 * j)) = codes;
  } else {
    *reinterpret_cast<uint16_t*>(rec + R::value(q, 8 * j)) = (uint16_t)codes;
    *reinterpret_cast<uint16_t*>(rec + R::value(q, 8 * j + 4)) = (uint16_t)(codes >> 16);
  }
  if (j % 4 == 0) rec[is_k ? R::key_scale(q, 8 * j) : R::value_scale(q, 8 * j)] = (uint8_t)byte;
}

struct LoadArgs {
  const uint8_t* cache;
  int64_t stride, num_blocks;
  int page, HK, T;
  const int64_t* slots;
  uint16_t *key, *value;
};

// D / 8 lanes a head of a token: 8 values each of the key and of the value.
template <int D>
__global__ __launch_bounds__(kRopeThreads) void kv4_load_kernel(LoadArgs a) {
  using R = Record<D>;
  constexpr int L = D / 8;
  const int64_t i = (int64_t)blockIdx.x * kRopeThreads + threadIdx.x;
  const int j = (int)(i % L);
  const int64_t at = i / L;  // token * HK + head
  if (at >= (int64_t)a.T * a.HK) return;
  const int t = (int)(at / a.HK), head = (int)(at - (int64_t)t * a.HK);
  const int64_t slot = a.slots[t];
  u32x4_t k = {0, 0, 0, 0}, v = k;
  if (slot >= 0 && slot < a.num_blocks * a.page) {
    const int64_t block = slot / a.page;
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
  const int64_t rows = (query ? u.num_heads : 0) + (int64_t)u.num_kv_heads * (cache ? 2 : 1);
  const int per_wave = kWave / (D / 8);
  const int64_t parts = (rows + per_wave - 1) / per_wave;
  // wavefronts are counted in 31 bits
  if (rows > 0x7fffffff || u.num_tokens * parts > 0x7fffffff - kRopeWaves || u.num_blocks > ((int64_t)1 << 40))
    return QF_ERR_UNSUPPORTED;
  const int64_t groups = (u.num_tokens * parts + kRopeWaves - 1) / kRopeWaves;
  if (!grid_fits(groups, kRopeThreads)) return QF_ERR_UNSUPPORTED;
  RopeArgs a = {u, divisor(cache ? u.page_size : 1), divisor((int)parts), (int)rows, (int)parts};
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
      !aligned16(value) || num_blocks > ((int64_t)1 << 40) ||
      cache_stride < (int64_t)num_kv_heads * (page_size / kTile) * 17 * D)
    return QF_ERR_UNSUPPORTED;
  const int64_t groups = ((int64_t)num_tokens * num_kv_heads * (D / 8) + kRopeThreads - 1) / kRopeThreads;
  if (!grid_fits(groups, kRopeThreads)) return QF_ERR_UNSUPPORTED;
  const LoadArgs a = {static_cast<const uint8_t*>(cache), cache_stride, num_blocks, page_size, num_kv_heads, num_tokens, slots,
                      key, value};
  const auto fn = D == 64 ? &kv4_load_kernel<64> : D == 128 ? &kv4_load_kernel<128> : &kv4_load_kernel<256>;
  hipLaunchKernelGGL(fn, dim3((unsigned)groups), dim3(kRopeThreads), 0, static_cast<hipStream_t>(stream), a);
  return hipGetLastError() == hipSuccess ? QF_OK : QF_ERR_HIP;
}
