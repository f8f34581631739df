// qf_block_moe.hip — a whole mixture-of-experts layer for up to 16 tokens, block-scaled e4m3 experts, in two launches
// (gfx950).  The C ABI is in include/qf_block.h.
//
//   a_e = bf16(silu(Wgate_e x) * (Wup_e x)),   y[t] = sum over the chosen experts e of c[t, e] * W2_e a_e
//
// 1. moe_up_kernel: every workgroup works the routing out for itself (a few thousand cycles, no launch and no trip through
//    memory between), then takes (chosen expert, 16 gate rows with their 16 up rows) items in turn; workgroup 0
//    leaves the routing for the second launch.
// 2. moe_down_kernel: a workgroup owns 16 output channels; its wavefronts share out the (expert, block of I) units, the
//    columns of the accumulator are the tokens, and a unit is weighed by its block's scale times c[t, e].
// An expert's weights are read once for all its tokens.  Products are exact (weights widened to bf16 in registers), sums
// fp32 in a fixed order.  Bound by the memory rate over the chosen experts' weights.
#include "qf_block_common.h"

namespace qfb {

constexpr int kTileN = 16;
constexpr int kStepK = 64;
constexpr int kBlock = QF_FP8_BLOCK;
constexpr int kMaxT = QF_FP8_MAX_DECODE_M;
constexpr int kMaxPairs = kMaxT * QF_MOE_MAX_TOP_K;          // (token, chosen expert) pairs, so chosen experts too
constexpr int kPerLane = QF_MOE_MAX_EXPERTS / kWave;         // experts a lane in the routing
constexpr int kMoeWaves = 8;
constexpr int kUpBatch = 2;    // blocks of K a wavefront has in flight
constexpr int kDownBatch = 3;  // units a wavefront has in flight

// What the first launch leaves for the second.
struct Routing {
  int active;                       // chosen experts
  int pad[3];
  uint16_t expert[kMaxPairs];       // in ascending order
  int16_t pair[kMaxPairs][kMaxT];   // row of a_e of (chosen expert, token), -1: not routed
  float weight[kMaxPairs][kMaxT];   // c, 0 where not routed
};

struct MoeArgs {
  const uint16_t* x;
  int64_t ldx;
  const void* logits;
  int64_t ldl;
  int logits_f32;
  const uint8_t* w13;
  const float* s13;
  const uint8_t* w2;
  const float* s2;
  uint16_t* y;
  int64_t ldy;
  Routing* routing;
  uint16_t* a;  // [pairs][I]
  int T, E, k, H, I, renormalize;
  int h_steps, h_blocks, i_steps, i_blocks;
};

struct RoutingLds {
  uint32_t tokens[QF_MOE_MAX_EXPERTS];  // an expert's tokens, a bit each
  uint16_t place[QF_MOE_MAX_EXPERTS];   // its place among the chosen ones
  uint16_t expert[kMaxPairs];
  uint16_t first[kMaxPairs + 1];        // first pair of a chosen expert
  uint8_t token[kMaxPairs];             // of a pair
  int16_t id[kMaxT][QF_MOE_MAX_TOP_K];  // -1: not routed
  float weight[kMaxT][QF_MOE_MAX_TOP_K];
  int active;
};

// A float's place in the order of the numbers (NaN above all), never 0.
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t u = __float_as_uint(f + 0.f);  // -0 counts as 0
  if (f != f) return 0xffffffffu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return k == 0xffffffffu ? __builtin_nanf("") : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// The routing of all tokens into LDS (every thread of the workgroup; ends with a barrier).
__device__ __forceinline__ void route(const MoeArgs& a, RoutingLds& s) {
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int waves = blockDim.x / kWave;
  const int per = (a.E + kWave - 1) / kWave;
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) s.tokens[e] = 0;
  __syncthreads();
  for (int t = wave; t < a.T; t += waves) {
    uint32_t key[kPerLane];  // of experts lane * per .. + per - 1; 0: none, or taken
#pragma unroll
    for (int p = 0; p < kPerLane; ++p) {
      const int e = lane * per + p;
      key[p] = 0;
      if (p < per && e < a.E) {
        const int64_t at = t * a.ldl + e;
        key[p] = order_key(a.logits_f32 ? static_cast<const float*>(a.logits)[at]
                                        : bf16_f32(static_cast<const uint16_t*>(a.logits)[at]));
      }
    }
    float sum = 0.f;  // of the whole softmax's terms, relative to the largest
    uint32_t mine = 0, top = 0;
    int id = 0;
    for (int j = 0; j < a.k; ++j) {
      uint32_t best = 0;
#pragma unroll
      for (int p = 0; p < kPerLane; ++p) best = max(best, key[p]);
      const uint32_t m = wave_max_u32(best);
      if (j == 0) {
        top = m;
        if (!a.renormalize) {
          const float f = key_value(m);
#pragma unroll
          for (int p = 0; p < kPerLane; ++p)
            if (key[p] != 0) sum += expf(key_value(key[p]) - f);
          sum = group_sum<64>(sum);
        }
      }
      const int from = __builtin_ctzll(__ballot(best == m));  // the first lane that has it: the lowest experts
      int at = 0;
#pragma unroll
      for (int p = kPerLane - 1; p >= 0; --p) at = key[p] == m ? p : at;
      at = __builtin_amdgcn_readlane(at, from);
#pragma unroll
      for (int p = 0; p < kPerLane; ++p)
        if (lane == from && p == at) key[p] = 0;
      if (lane == j) {
        mine = m;
        id = from * per + at;
      }
    }
    const float f = key_value(top);
    float c = lane < a.k ? expf(key_value(mine) - f) : 0.f;
    if (a.renormalize) sum = group_sum<64>(c);
    c = f == -__builtin_inff() ? 0.f : c / sum;
    if (lane < a.k) {
      s.id[t][lane] = c != 0.f ? (int16_t)id : (int16_t)-1;
      s.weight[t][lane] = c;
      if (c != 0.f) atomicOr(&s.tokens[id], 1u << t);
    }
  }
  __syncthreads();
  if (wave == 0) {  // the chosen experts in ascending order, with their first pairs
    int experts = 0, pairs = 0;
    for (int p = 0; p < per; ++p) {
      const int e = lane * per + p;
      const uint32_t bits = e < a.E ? s.tokens[e] : 0u;
      experts += bits != 0;
      pairs += __builtin_popcount(bits);
    }
    const int to = wave_scan(experts), pair_to = wave_scan(pairs);
    int at = to - experts, pair = pair_to - pairs;
    for (int p = 0; p < per; ++p) {
      const int e = lane * per + p;
      const uint32_t bits = e < a.E ? s.tokens[e] : 0u;
      if (bits == 0) continue;
      s.place[e] = (uint16_t)at;
      s.expert[at] = (uint16_t)e;
      s.first[at] = (uint16_t)pair;
      ++at;
      pair += __builtin_popcount(bits);
    }
    if (lane == kWave - 1) {
      s.active = to;
      s.first[to] = (uint16_t)pair_to;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.T * a.k; i += blockDim.x) {
    const int t = i / a.k, id = s.id[t][i % a.k];
    if (id >= 0) s.token[s.first[s.place[id]] + __builtin_popcount(s.tokens[id] & ((1u << t) - 1))] = (uint8_t)t;
  }
  __syncthreads();
}

// A block of K of one weight tile times its token fragments, from zero.
__device__ __forceinline__ f32x4_t block_product(const u32x4_t (&w)[2], const u32x4_t (&x)[2][2], bool second) {
  f32x4_t blk = {0.f, 0.f, 0.f, 0.f};
  bf16x8_t lo, hi;
  widen16(w[0], lo, hi);
  blk = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo, __builtin_bit_cast(bf16x8_t, x[0][0]), blk, 0, 0, 0);
  blk = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi, __builtin_bit_cast(bf16x8_t, x[0][1]), blk, 0, 0, 0);
  if (second) {
    widen16(w[1], lo, hi);
    blk = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo, __builtin_bit_cast(bf16x8_t, x[1][0]), blk, 0, 0, 0);
    blk = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi, __builtin_bit_cast(bf16x8_t, x[1][1]), blk, 0, 0, 0);
  }
  return blk;
}

__global__ void __launch_bounds__(kMoeWaves* kWave) moe_up_kernel(const MoeArgs a) {
  __shared__ RoutingLds s;
  __shared__ f32x4_t part[2][kMoeWaves][2][kWave];
  const int lane = threadIdx.x & (kWave - 1);
  const int v = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int g = lane >> 4, r = lane & 15;
  route(a, s);
  if (blockIdx.x == 0) {
    const int active = s.active;
    if (threadIdx.x == 0) a.routing->active = active;
    for (int i = threadIdx.x; i < active; i += blockDim.x) a.routing->expert[i] = s.expert[i];
    for (int i = threadIdx.x; i < active * kMaxT; i += blockDim.x) {
      const int at = i / kMaxT, t = i % kMaxT, e = s.expert[at];
      const bool in = s.tokens[e] >> t & 1;
      float c = 0.f;
      if (in)
        for (int j = 0; j < a.k; ++j) c = s.id[t][j] == e ? s.weight[t][j] : c;
      a.routing->weight[at][t] = c;
      a.routing->pair[at][t] = in ? (int16_t)(s.first[at] + __builtin_popcount(s.tokens[e] & ((1u << t) - 1))) : (int16_t)-1;
    }
  }
  const int row_tiles = a.I / kTileN;
  const int items = __builtin_amdgcn_readfirstlane(s.active) * row_tiles;
  int turn = 0;
  for (int item = blockIdx.x; item < items; item += gridDim.x, ++turn) {
    const int at = item / row_tiles, j = item - at * row_tiles;
    const int e = __builtin_amdgcn_readfirstlane(s.expert[at]);
    const int first = __builtin_amdgcn_readfirstlane(s.first[at]);
    const int n_tok = __builtin_amdgcn_readfirstlane(s.first[at + 1]) - first;
    const uint16_t* xp = a.x + (int64_t)s.token[first + min(r, n_tok - 1)] * a.ldx + 16 * g;
    const uint8_t* wg = a.w13 + (((int64_t)e * 2 * row_tiles + j) * a.h_steps * kWave + lane) * 16;
    const uint8_t* wu = wg + (int64_t)row_tiles * a.h_steps * kWave * 16;
    const float* sg = a.s13 + ((int64_t)e * 2 * a.i_blocks + j * kTileN / kBlock) * a.h_blocks;
    const float* su = sg + (int64_t)a.i_blocks * a.h_blocks;
    f32x4_t acc_g = {0.f, 0.f, 0.f, 0.f}, acc_u = acc_g;
    for (int base = v; base < a.h_blocks; base += kMoeWaves * kUpBatch) {
      u32x4_t g_w[kUpBatch][2], u_w[kUpBatch][2], xf[kUpBatch][2][2];
      float s_g[kUpBatch], s_u[kUpBatch];
#pragma unroll
      for (int b = 0; b < kUpBatch; ++b) {
        const int kb = min(base + b * kMoeWaves, a.h_blocks - 1);
        const int64_t half = 2 * kb + 1 < a.h_steps ? 1 : 0;  // a last half block: its first half again, not used
        g_w[b][0] = load_once(wg + (int64_t)kb * 2048);
        g_w[b][1] = load_once(wg + (int64_t)kb * 2048 + half * 1024);
        u_w[b][0] = load_once(wu + (int64_t)kb * 2048);
        u_w[b][1] = load_once(wu + (int64_t)kb * 2048 + half * 1024);
        s_g[b] = sg[kb];
        s_u[b] = su[kb];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const u32x4_t* p = reinterpret_cast<const u32x4_t*>(xp + (int64_t)kb * kBlock + (h ? half * kStepK : 0));
          xf[b][h][0] = p[0];
          xf[b][h][1] = p[1];
        }
      }
#pragma unroll
      for (int b = 0; b < kUpBatch; ++b) {
        const int kb = base + b * kMoeWaves;
        if (kb >= a.h_blocks) break;
        const bool second = 2 * kb + 1 < a.h_steps;
        acc_g += block_product(g_w[b], xf[b], second) * s_g[b];
        acc_u += block_product(u_w[b], xf[b], second) * s_u[b];
      }
    }
    // the wavefronts' sums, in their order; one wavefront adds them up while the others go on to the next item
    f32x4_t(&buf)[kMoeWaves][2][kWave] = part[turn & 1];
    buf[v][0][lane] = acc_g;
    buf[v][1][lane] = acc_u;
    __syncthreads();
    if (v == turn % kMoeWaves && r < n_tok) {
      f32x4_t gate = buf[0][0][lane], up = buf[0][1][lane];
      for (int u = 1; u < kMoeWaves; ++u) {
        gate += buf[u][0][lane];
        up += buf[u][1][lane];
      }
      float o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = gate[i] / (1.f + expf(-gate[i])) * up[i];
      *reinterpret_cast<u32x2_t*>(a.a + (int64_t)(first + r) * a.I + j * kTileN + 4 * g) =
          u32x2_t{pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3])};
    }
  }
}

__global__ void __launch_bounds__(kMoeWaves* kWave) moe_down_kernel(const MoeArgs a) {
  __shared__ int16_t pair[kMaxPairs][kMaxT];
  __shared__ float weight[kMaxPairs][kMaxT];
  __shared__ uint16_t expert[kMaxPairs];
  __shared__ f32x4_t part[kMoeWaves][kWave];
  const int lane = threadIdx.x & (kWave - 1);
  const int v = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int g = lane >> 4, r = lane & 15;
  const int nt = blockIdx.x;
  const int active = a.routing->active;
  for (int i = threadIdx.x; i < active * kMaxT; i += blockDim.x) {
    (&pair[0][0])[i] = (&a.routing->pair[0][0])[i];
    (&weight[0][0])[i] = (&a.routing->weight[0][0])[i];
  }
  for (int i = threadIdx.x; i < active; i += blockDim.x) expert[i] = a.routing->expert[i];
  __syncthreads();
  const int units = active * a.i_blocks;
  const int h_tiles = a.H / kTileN;
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
  for (int base = v; base < units; base += kMoeWaves * kDownBatch) {
    u32x4_t w[kDownBatch][2], xf[kDownBatch][2][2];
    float s[kDownBatch];
    bool in[kDownBatch];
#pragma unroll
    for (int b = 0; b < kDownBatch; ++b) {
      const int u = min(base + b * kMoeWaves, units - 1);
      const int at = u / a.i_blocks, kb = u - at * a.i_blocks;
      const int e = __builtin_amdgcn_readfirstlane(expert[at]);
      const int64_t half = 2 * kb + 1 < a.i_steps ? 1 : 0;
      const uint8_t* wp = a.w2 + ((((int64_t)e * h_tiles + nt) * a.i_steps + 2 * kb) * kWave + lane) * 16;
      w[b][0] = load_once(wp);
      w[b][1] = load_once(wp + half * 1024);
      const int p = pair[at][r];
      in[b] = p >= 0;
      s[b] = a.s2[((int64_t)e * ((a.H + kBlock - 1) / kBlock) + nt * kTileN / kBlock) * a.i_blocks + kb] * weight[at][r];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          xf[b][h][q] = u32x4_t{0u, 0u, 0u, 0u};  // a token that is not routed here: zeros, whatever a_e holds
          if (p >= 0)
            xf[b][h][q] = *reinterpret_cast<const u32x4_t*>(a.a + (int64_t)p * a.I + (int64_t)kb * kBlock +
                                                            (h ? half * kStepK : 0) + 16 * g + 8 * q);
        }
    }
#pragma unroll
    for (int b = 0; b < kDownBatch; ++b) {
      const int u = base + b * kMoeWaves;
      if (u >= units) break;
      const f32x4_t add = block_product(w[b], xf[b], 2 * (u % a.i_blocks) + 1 < a.i_steps) * s[b];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] += in[b] ? add[i] : 0.f;  // NaN weights of an expert reach its own tokens only
    }
  }
  part[v][lane] = acc;
  __syncthreads();
  if (v == 0 && r < a.T) {
    f32x4_t sum = part[0][lane];
    for (int u = 1; u < kMoeWaves; ++u) sum += part[u][lane];
    *reinterpret_cast<u32x2_t*>(a.y + (int64_t)r * a.ldy + nt * kTileN + 4 * g) =
        u32x2_t{pack_bf16(sum[0], sum[1]), pack_bf16(sum[2], sum[3])};
  }
}

bool moe_sizes_ok(int T, int E, int top_k, int H, int I) {
  return T >= 1 && T <= kMaxT && E >= 1 && E <= QF_MOE_MAX_EXPERTS && top_k >= 1 && top_k <= QF_MOE_MAX_TOP_K &&
         top_k <= E && H >= kStepK && H % kStepK == 0 && I >= kStepK && I % kStepK == 0 && H <= (1 << 24) && I <= (1 << 22);
}

constexpr size_t kRoutingBytes = (sizeof(Routing) + 255) / 256 * 256;

}  // namespace qfb

using namespace qfb;

extern "C" {

size_t qf_moe_few_workspace_bytes(int T, int E, int top_k, int H, int I) {
  if (!moe_sizes_ok(T, E, top_k, H, I)) return 0;
  return kRoutingBytes + ((size_t)T * top_k * I * 2 + 255) / 256 * 256;
}

int qf_moe_few_tokens(const uint16_t* x, int64_t ldx, const void* logits, int64_t ldl, int logits_f32, const uint8_t* w13,
                      const float* s13, const uint8_t* w2, const float* s2, uint16_t* y, int64_t ldy, int T, int E,
                      int top_k, int H, int I, int renormalize, void* workspace, size_t workspace_bytes, void* stream) {
  if (x == nullptr || logits == nullptr || w13 == nullptr || s13 == nullptr || w2 == nullptr || s2 == nullptr || y == nullptr)
    return QF_ERR_INVALID_ARG;
  if (T < 1 || E < 1 || top_k < 1 || H < 1 || I < 1 || (T > 1 && (ldx < H || ldl < E || ldy < H))) return QF_ERR_INVALID_ARG;
  if (!moe_sizes_ok(T, E, top_k, H, I)) return QF_ERR_UNSUPPORTED;
  if (ldx % 8 || ldy % 4 || !aligned16(x) || !aligned16(w13) || !aligned16(w2) || ((uintptr_t)y & 7)) return QF_ERR_UNSUPPORTED;
  if (workspace == nullptr || workspace_bytes < qf_moe_few_workspace_bytes(T, E, top_k, H, I) || !aligned16(workspace))
    return QF_ERR_WORKSPACE;
  MoeArgs a;
  a.x = x;
  a.ldx = ldx;
  a.logits = logits;
  a.ldl = ldl;
  a.logits_f32 = logits_f32;
  a.w13 = w13;
  a.s13 = s13;
  a.w2 = w2;
  a.s2 = s2;
  a.y = y;
  a.ldy = ldy;
  a.routing = static_cast<Routing*>(workspace);
  a.a = reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(workspace) + kRoutingBytes);
  a.T = T;
  a.E = E;
  a.k = top_k;
  a.H = H;
  a.I = I;
  a.renormalize = renormalize;
  a.h_steps = H / kStepK;
  a.h_blocks = (H + kBlock - 1) / kBlock;
  a.i_steps = I / kStepK;
  a.i_blocks = (I + kBlock - 1) / kBlock;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t chosen = (int64_t)T * top_k < E ? (int64_t)T * top_k : E;
  const int64_t items = chosen * (I / kTileN);
  const unsigned grid = (unsigned)(items < 768 ? items : 768);
  hipLaunchKernelGGL(moe_up_kernel, dim3(grid), dim3(kMoeWaves * kWave), 0, s, a);
  if (hipGetLastError() != hipSuccess) return QF_ERR_HIP;
  hipLaunchKernelGGL(moe_down_kernel, dim3((unsigned)(H / kTileN)), dim3(kMoeWaves * kWave), 0, s, a);
  return hipGetLastError() == hipSuccess ? QF_OK : QF_ERR_HIP;
}

}  // extern "C"
