// qf_block_moe.hip — a whole mixture-of-experts layer for up to 16 tokens, block-scaled e4m3 experts, in two launches
// (gfx950).  The C ABI is in include/qf_block.h.
//
//   a_e = silu(Wgate_e x) * (Wup_e x),   y[t] = sum over the chosen experts e of c[t, e] * W2_e a_e
//
// 1. moe_up_kernel: every workgroup works the routing out for itself (a few thousand cycles, no launch and no trip through
//    memory between), then takes (chosen expert, 16 gate rows with their 16 up rows) items in turn; workgroup 0
//    leaves the routing for the second launch.
// 2. moe_down_kernel: a workgroup owns 16 output channels; its wavefronts share out the (expert, block of I) units, the
//    columns of the accumulator are the tokens, and a unit is weighed by its block's scale times c[t, e].
// An expert's weights are read once for all its tokens.  Products are exact (weights widened to bf16 in registers), sums
// fp32 in a fixed order.  Between the launches an activation is the sum of two bf16 numbers (16 bits of it are kept): one
// bf16 alone put 2^-9 of noise into every a_e, half as much again as the output's own rounding (2.6e-3 against 1.7e-3 from
// the exact result); the second product costs no weight bytes.  Bound by the memory rate over the chosen experts' weights.
#include "qf_block_common.h"

namespace qfb {

constexpr int kTileN = 16;
constexpr int kStepK = 64;
constexpr int kBlock = QF_FP8_BLOCK;
constexpr int kMaxT = QF_FP8_MAX_DECODE_M;
constexpr int kMaxPairs = kMaxT * QF_MOE_MAX_TOP_K;          // (token, chosen expert) pairs, so chosen experts too
constexpr int kPerLane = QF_MOE_MAX_EXPERTS / kWave;         // experts a lane in the routing
constexpr int kMoeWaves = 8;
constexpr int kDownWaves = 16;
constexpr int kUpDepth = 2;    // blocks of H a wavefront requests ahead
constexpr int kDownDepth = 3;  // units a wavefront requests ahead; odd: the activations' two buffers alternate with the ring
static_assert(kDownDepth % 2 == 1, "an even ring");

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
  uint16_t* a;  // [pairs][2][I]: the activations, each as the sum of two bf16 numbers
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

__global__ void __launch_bounds__(kMoeWaves* kWave) __attribute__((amdgpu_waves_per_eu(4))) moe_up_kernel(const MoeArgs a) {
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
  // this workgroup's run of (chosen expert, 16 gate rows and their up rows) items, as one stream of blocks of H
  const int row_tiles = a.I / kTileN;
  const int items = __builtin_amdgcn_readfirstlane(s.active) * row_tiles;
  const int first_item = (int)((int64_t)blockIdx.x * items / gridDim.x);
  const int n_items = (int)((int64_t)(blockIdx.x + 1) * items / gridDim.x) - first_item;
  const int steps = (a.h_blocks - v + kMoeWaves - 1) / kMoeWaves;  // of this wavefront in an item, maybe none
  const int total = n_items * steps;
  struct Step {
    u32x4_t gate[2], up[2], x[2][2];
    float s_gate, s_up;
  };
  Step buf[kUpDepth + 1];
  const uint32_t w_lane = (uint32_t)lane * 16;
  int pi = first_item, pj = 0;  // the next request
  const uint8_t* p_gate;
  const float* p_scale;
  uint32_t x_lane;
  auto enter = [&](int item) {
    const int at = item / row_tiles, j = item - at * row_tiles;
    const int64_t e = __builtin_amdgcn_readfirstlane(s.expert[at]);
    const int first = __builtin_amdgcn_readfirstlane(s.first[at]);
    const int n_tok = __builtin_amdgcn_readfirstlane(s.first[at + 1]) - first;
    x_lane = s.token[first + min(r, n_tok - 1)] * (uint32_t)a.ldx * 2 + 32 * g;
    p_gate = a.w13 + (e * 2 * row_tiles + j) * a.h_steps * (kWave * 16);
    p_scale = a.s13 + (e * 2 * a.i_blocks + j * kTileN / kBlock) * a.h_blocks;
  };
  auto load = [&](Step& b) {
    const int kb = v + pj * kMoeWaves;
    const int half = 2 * kb + 1 < a.h_steps ? 1 : 0;  // a last half block: its first half again, not used
    const uint8_t* p = p_gate + (int64_t)kb * 2048;
    const uint8_t* q = p + (int64_t)row_tiles * a.h_steps * (kWave * 16);
    b.gate[0] = load_once(p + w_lane);
    b.gate[1] = load_once(p + half * 1024 + w_lane);
    b.up[0] = load_once(q + w_lane);
    b.up[1] = load_once(q + half * 1024 + w_lane);
    const uint8_t* xp = reinterpret_cast<const uint8_t*>(a.x + (int64_t)kb * kBlock);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32x4_t* c = reinterpret_cast<const u32x4_t*>(xp + (h ? half * 2 * kStepK : 0) + x_lane);
      b.x[h][0] = c[0];
      b.x[h][1] = c[1];
    }
    b.s_gate = p_scale[kb];
    b.s_up = p_scale[(int64_t)a.i_blocks * a.h_blocks + kb];
    if (++pj == steps) {
      if (pi + 1 < first_item + n_items) {
        enter(++pi);
        pj = 0;
      } else {
        pj = steps - 1;
      }
    }
  };
  // The wavefronts' partial tiles meet in LDS (two buffers, one barrier an item); one wavefront, another one each time, adds
  // them in wavefront order while the others stream on.
  f32x4_t acc_gate = {0.f, 0.f, 0.f, 0.f}, acc_up = acc_gate;
  auto leave = [&](int i) {
    f32x4_t(&slot)[kMoeWaves][2][kWave] = part[i & 1];
    slot[v][0][lane] = acc_gate;
    slot[v][1][lane] = acc_up;
    acc_gate = acc_up = f32x4_t{0.f, 0.f, 0.f, 0.f};
    ring_barrier();
    if (v != i % kMoeWaves) return;
    const int item = first_item + i, at = item / row_tiles, j = item - at * row_tiles;
    const int first = s.first[at];
    if (r >= s.first[at + 1] - first) return;
    f32x4_t gate = slot[0][0][lane], up = slot[0][1][lane];
    for (int u = 1; u < kMoeWaves; ++u) {
      gate += slot[u][0][lane];
      up += slot[u][1][lane];
    }
    // the activation as two bf16 parts, the rounded value and what the rounding left
    float hi[4], lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float o = gate[e] / (1.f + expf(-gate[e])) * up[e];
      hi[e] = bf16_lo(pack_bf16(o, 0.f));
      lo[e] = fabsf(hi[e]) < __builtin_inff() ? o - hi[e] : 0.f;
    }
    uint16_t* row = a.a + (int64_t)(first + r) * 2 * a.I + j * kTileN + 4 * g;
    *reinterpret_cast<u32x2_t*>(row) = u32x2_t{pack_bf16(hi[0], hi[1]), pack_bf16(hi[2], hi[3])};
    *reinterpret_cast<u32x2_t*>(row + a.I) = u32x2_t{pack_bf16(lo[0], lo[1]), pack_bf16(lo[2], lo[3])};
  };
  if (n_items == 0) return;
  if (steps == 0) {  // fewer blocks of H than wavefronts: this one has only its place in the sums
    for (int i = 0; i < n_items; ++i) leave(i);
    return;
  }
  enter(pi);
#pragma unroll
  for (int d = 0; d < kUpDepth; ++d) load(buf[d]);
  int ci = 0, cj = 0;
  for (int base = 0; base < total; base += kUpDepth + 1) {
#pragma unroll
    for (int d = 0; d <= kUpDepth; ++d) {
      load(buf[(d + kUpDepth) % (kUpDepth + 1)]);
      __builtin_amdgcn_sched_barrier(0);  // the requests go out ahead of this step's math
      if (base + d < total) {             // uniform
        const Step& b = buf[d];
        const bool second = 2 * (v + cj * kMoeWaves) + 1 < a.h_steps;
        acc_gate += block_product(b.gate, b.x, second) * b.s_gate;
        acc_up += block_product(b.up, b.x, second) * b.s_up;
        if (++cj == steps) {
          leave(ci++);
          cj = 0;
        }
      }
    }
  }
}

__global__ void __launch_bounds__(kDownWaves* kWave) moe_down_kernel(const MoeArgs a) {
  __shared__ int16_t pair[kMaxPairs][kMaxT];
  __shared__ float weight[kMaxPairs][kMaxT];
  __shared__ uint16_t expert[kMaxPairs];
  __shared__ f32x4_t part[kDownWaves][kWave];
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
  // (chosen expert, block of I) units, interleaved over the wavefronts; weights kDownDepth units ahead, activations one
  const int units = active * a.i_blocks;
  const int total = units > v ? (units - v + kDownWaves - 1) / kDownWaves : 0;
  const int h_tiles = a.H / kTileN;
  const int64_t h_blocks = a.h_blocks;
  const uint32_t w_lane = (uint32_t)lane * 16;
  struct Weights {
    u32x4_t w[2];
    float s;
  };
  struct Acts {
    u32x4_t hi[2][2], lo[2][2];
    float c;
    bool in;
  };
  Weights wb[kDownDepth + 1];
  Acts xb[2];
  auto load_w = [&](int i, Weights& b) {
    const int u = v + min(i, total - 1) * kDownWaves;
    const int at = u / a.i_blocks, kb = u - at * a.i_blocks;
    const int64_t e = __builtin_amdgcn_readfirstlane(expert[at]);
    const int half = 2 * kb + 1 < a.i_steps ? 1 : 0;
    const uint8_t* p = a.w2 + ((e * h_tiles + nt) * a.i_steps + 2 * kb) * (kWave * 16);
    b.w[0] = load_once(p + w_lane);
    b.w[1] = load_once(p + half * 1024 + w_lane);
    b.s = a.s2[(e * h_blocks + nt * kTileN / kBlock) * a.i_blocks + kb];
  };
  auto load_x = [&](int i, Acts& b) {
    const int u = v + min(i, total - 1) * kDownWaves;
    const int at = u / a.i_blocks, kb = u - at * a.i_blocks;
    const int half = 2 * kb + 1 < a.i_steps ? 1 : 0;
    const int p = pair[at][r];
    b.c = weight[at][r];
    b.in = p >= 0;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        b.hi[h][q] = b.lo[h][q] = u32x4_t{0u, 0u, 0u, 0u};  // a token that is not routed here: zeros, whatever `a` holds
        if (b.in) {
          const uint16_t* c = a.a + (int64_t)p * 2 * a.I + kb * kBlock + (h ? half * kStepK : 0) + 16 * g + 8 * q;
          b.hi[h][q] = *reinterpret_cast<const u32x4_t*>(c);
          b.lo[h][q] = *reinterpret_cast<const u32x4_t*>(c + a.I);
        }
      }
  };
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
  if (total > 0) {
#pragma unroll
    for (int d = 0; d < kDownDepth; ++d) load_w(d, wb[d]);
    load_x(0, xb[0]);
    for (int base = 0; base < total; base += kDownDepth + 1) {
#pragma unroll
      for (int d = 0; d <= kDownDepth; ++d) {
        const int i = base + d;
        load_w(i + kDownDepth, wb[(d + kDownDepth) % (kDownDepth + 1)]);
        load_x(i + 1, xb[(d + 1) & 1]);
        __builtin_amdgcn_sched_barrier(0);
        if (i < total) {  // uniform
          const Weights& b = wb[d];
          const Acts& x = xb[d & 1];
          const bool second = 2 * ((v + i * kDownWaves) % a.i_blocks) + 1 < a.i_steps;
          const f32x4_t add = (block_product(b.w, x.hi, second) + block_product(b.w, x.lo, second)) * (b.s * x.c);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] += x.in ? add[e] : 0.f;  // NaN weights of an expert reach its own tokens only
        }
      }
    }
  }
  part[v][lane] = acc;
  __syncthreads();
  if (v == 0 && r < a.T) {
    f32x4_t sum = part[0][lane];
    for (int u = 1; u < kDownWaves; ++u) sum += part[u][lane];
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
  return kRoutingBytes + ((size_t)T * top_k * I * 4 + 255) / 256 * 256;
}

int qf_moe_few_tokens(const uint16_t* x, int64_t ldx, const void* logits, int64_t ldl, int logits_f32, const uint8_t* w13,
                      const float* s13, const uint8_t* w2, const float* s2, uint16_t* y, int64_t ldy, int T, int E,
                      int top_k, int H, int I, int renormalize, void* workspace, size_t workspace_bytes, void* stream) {
  if (x == nullptr || logits == nullptr || w13 == nullptr || s13 == nullptr || w2 == nullptr || s2 == nullptr || y == nullptr)
    return QF_ERR_INVALID_ARG;
  if (T < 1 || E < 1 || top_k < 1 || H < 1 || I < 1 || (T > 1 && (ldx < H || ldl < E || ldy < H))) return QF_ERR_INVALID_ARG;
  if (!moe_sizes_ok(T, E, top_k, H, I)) return QF_ERR_UNSUPPORTED;
  if (ldx > ((int64_t)1 << 26) || ldx % 8 || ldy % 4 || !aligned16(x) || !aligned16(w13) || !aligned16(w2) || ((uintptr_t)y & 7)) return QF_ERR_UNSUPPORTED;
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
  const unsigned grid = (unsigned)(items < 512 ? items : 512);
  hipLaunchKernelGGL(moe_up_kernel, dim3(grid), dim3(kMoeWaves * kWave), 0, s, a);
  if (hipGetLastError() != hipSuccess) return QF_ERR_HIP;
  hipLaunchKernelGGL(moe_down_kernel, dim3((unsigned)(H / kTileN)), dim3(kDownWaves * kWave), 0, s, a);
  return hipGetLastError() == hipSuccess ? QF_OK : QF_ERR_HIP;
}

}  // extern "C"
