// qf_block_moe.hip — a whole mixture-of-experts layer for up to 16 tokens, block-scaled e4m3 experts, in two launches
// (gfx950).  The C ABI is in include/qf_block.h.
//
//   a_e = silu(Wgate_e x) * (Wup_e x),   y[t] = sum over the chosen experts e of c[t, e] * W2_e a_e
//
// 1. moe_up_kernel: every workgroup works the routing out for itself (a few thousand cycles, no launch and no trip through
//    memory between).  Workgroup 0 leaves it for the second launch; the others each stream a run of (chosen expert, 16 gate
//    rows with their 16 up rows) items, the wavefronts sharing out the blocks of H, two in flight each.
// 2. moe_down_kernel: a workgroup owns 32 output channels and a part of the (expert, block of I) units, its wavefronts share
//    these out; the columns of the accumulator are the tokens, and a unit is weighed by its block's scale times c[t, e].  The
//    last of a channel group's workgroups to arrive adds their sums, in split order.
// An expert's weights are read once for all its tokens.  Products are exact (weights widened to bf16 in registers), sums
// fp32 in a fixed order.  Between the launches an activation is the sum of two bf16 numbers (16 bits of it are kept): one
// bf16 alone put 2^-9 of noise into every a_e, half as much again as the output's own rounding (2.6e-3 against 1.7e-3 from
// the exact result); the second product costs no weight bytes.  Bound by the memory rate over the chosen experts' weights.
//
// Measured, H 2048, I 768, 8 experts a token: 1 token (38 MB of weights) 10.8 + 7.1 us; 16 tokens of 128 experts (about 390
// MB) 48 + 28 us, 5.2 TB/s.  The second launch took 61 us with 16 output channels a workgroup, 16 wavefronts and all units
// (the activations' 1 KiB a token and unit, read again for every 16 channels, were the larger part of its loads); with 32
// channels and the units split it is 28 with 8 wavefronts, 32 with 6, 30 with 4 and two workgroups a CU, 28 with 48 channels
// (8 against 7 at one token) and 38 with 64.
#include "qf_block_common.h"

namespace qfb {

constexpr int kTileN = 16;
constexpr int kStepK = 64;
constexpr int kBlock = QF_FP8_BLOCK;
constexpr int kMaxT = QF_FP8_MAX_DECODE_M;
constexpr int kMaxPairs = kMaxT * QF_MOE_MAX_TOP_K;          // (token, chosen expert) pairs, so chosen experts too
constexpr int kMaxUpWaves = 16;
constexpr int kUpWaveLds = 4096;  // a wavefront's partial tiles: gate and up, two buffers
constexpr int kDownGrid = 256;  // workgroups of the second launch where it splits: one a CU
constexpr int kDownWaves = 8;
constexpr int kDownTiles = 2;  // tiles of 16 output channels a workgroup

// What the first launch leaves for the second.
struct Routing {
  int active;                       // chosen experts
  int pad[3];
  unsigned arrivals[kDownGrid / 2];  // of the second launch's splits, a group of tiles each; zeroed by the first
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
  uint64_t* partial;  // [split][tile][2][64 lanes]
  int splits;
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
  float pair_weight[kMaxPairs];
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

// The routing of all tokens into LDS (every thread of the workgroup; ends with a barrier): L lanes a token, each with up to
// kPerLane experts, one chosen expert a round.
template <int L, int kPerLane>
__device__ __forceinline__ void route(const MoeArgs& a, RoutingLds& s) {
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int waves = blockDim.x / kWave;
  const int per = (a.E + kWave - 1) / kWave;
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) s.tokens[e] = 0;
  __syncthreads();
  const int i = lane & (L - 1), share = (a.E + L - 1) / L;
  for (int t0 = wave * (kWave / L); t0 < a.T; t0 += waves * (kWave / L)) {
    const int t = t0 + lane / L;  // past the last token: the last one's values, not kept
    uint32_t key[kPerLane];       // of experts i * share .. + share - 1; 0: none, or taken
    const int64_t row = (int64_t)min(t, a.T - 1) * a.ldl;
#pragma unroll
    for (int p = 0; p < kPerLane; ++p) {
      const int e = i * share + p;
      key[p] = 0;
      if (p < share && e < a.E)
        key[p] = order_key(a.logits_f32 ? static_cast<const float*>(a.logits)[row + e]
                                        : bf16_f32(static_cast<const uint16_t*>(a.logits)[row + e]));
    }
    float sum = 0.f;  // of the whole softmax's terms, relative to the largest
    uint32_t mine = 0, top = 0;
    for (int j = 0; j < a.k; ++j) {
      uint32_t best = 0;
#pragma unroll
      for (int p = 0; p < kPerLane; ++p) best = max(best, key[p]);
      const uint32_t m = group_max_u32<L>(best);
      if (j == 0) {
        top = m;
        if (!a.renormalize) {
          const float f = key_value(m);
#pragma unroll
          for (int p = 0; p < kPerLane; ++p)
            if (key[p] != 0) sum += expf(key_value(key[p]) - f);
          sum = group_sum<L>(sum);
        }
      }
      // the first lane that has it, and its first one: the lowest expert
      const uint64_t have = __ballot(best == m);
      const int from = L == kWave ? __builtin_ctzll(have) : __builtin_ctz((uint32_t)(have >> (lane & ~(L - 1))) & 0xffffu);
      if (i == from) {
        int at = 0;
#pragma unroll
        for (int p = kPerLane - 1; p >= 0; --p) at = key[p] == m ? p : at;
#pragma unroll
        for (int p = 0; p < kPerLane; ++p)
          if (p == at) key[p] = 0;
        if (t < a.T) s.id[t][j] = (int16_t)(i * share + at);
      }
      if (i == j) mine = m;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the ids that other lanes wrote
    const float f = key_value(top);
    float c = i < a.k ? expf(key_value(mine) - f) : 0.f;
    if (a.renormalize) sum = group_sum<L>(c);
    c = f == -__builtin_inff() ? 0.f : c / sum;
    if (i < a.k && t < a.T) {
      s.weight[t][i] = c;
      if (c != 0.f)
        atomicOr(&s.tokens[s.id[t][i]], 1u << t);
      else
        s.id[t][i] = -1;
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
    if (id < 0) continue;
    const int pair = s.first[s.place[id]] + __builtin_popcount(s.tokens[id] & ((1u << t) - 1));
    s.token[pair] = (uint8_t)t;
    s.pair_weight[pair] = s.weight[t][i % a.k];
  }
  __syncthreads();
}

template <int L, int kPerLane>
__global__ void __launch_bounds__(kMaxUpWaves* kWave) __attribute__((amdgpu_waves_per_eu(4))) moe_up_kernel(const MoeArgs a) {
  __shared__ RoutingLds s;
  extern __shared__ __align__(16) uint8_t smem[];
  const int W = blockDim.x / kWave;
  f32x4_t* const part = reinterpret_cast<f32x4_t*>(smem);  // [2][W][2][64 lanes]
  const int lane = threadIdx.x & (kWave - 1);
  const int v = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int g = lane >> 4, r = lane & 15;
  route<L, kPerLane>(a, s);
  if (blockIdx.x == 0) {  // leaves the routing for the second launch; the other workgroups share out the items
    const int active = s.active;
    if (threadIdx.x == 0) a.routing->active = active;
    if (threadIdx.x < kDownGrid / 2) a.routing->arrivals[threadIdx.x] = 0;
    for (int i = threadIdx.x; i < active; i += blockDim.x) a.routing->expert[i] = s.expert[i];
    for (int i = threadIdx.x; i < active * kMaxT; i += blockDim.x) {
      const int at = i / kMaxT, t = i % kMaxT;
      const uint32_t tokens = s.tokens[s.expert[at]];
      const int pair = s.first[at] + __builtin_popcount(tokens & ((1u << t) - 1));
      const bool in = tokens >> t & 1;
      a.routing->pair[at][t] = in ? (int16_t)pair : (int16_t)-1;
      a.routing->weight[at][t] = in ? s.pair_weight[pair] : 0.f;
    }
    return;
  }
  // This workgroup's run of (chosen expert, 16 gate rows and their up rows) items, as one stream of chunks of two blocks of
  // H a wavefront; a chunk's registers are loaded again for the next one as soon as they are multiplied.  (A wavefront without
  // a block in a chunk reads one line and multiplies nothing.)
  const int row_tiles = a.I / kTileN;
  const int items = __builtin_amdgcn_readfirstlane(s.active) * row_tiles;
  const int share = gridDim.x - 1, place = blockIdx.x - 1;
  const int first_item = (int)((int64_t)place * items / share);
  const int n_items = (int)((int64_t)(place + 1) * items / share) - first_item;
  const int chunks = (a.h_blocks + 2 * W - 1) / (2 * W);  // of an item
  if (n_items == 0) return;
  struct Step {
    u32x4_t gate[2], up[2], x[2][2];
    float s_gate, s_up;
  };
  Step buf[2];
  int pi = first_item, pj = 0;  // the next chunk to load
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
  auto block = [&](int j, int p) { return v + (2 * j + p) * W; };
  auto load = [&](int j, int p, Step& b) {
    const bool in = block(j, p) < a.h_blocks;
    const int kb = in ? block(j, p) : 0;
    const int half = 2 * kb + 1 < a.h_steps ? 1 : 0;  // a last half block: its first half again, not used
    const uint32_t w_lane = in ? (uint32_t)lane * 16 : 0u, x_at = in ? x_lane : 0u;
    const uint8_t* w = p_gate + (int64_t)kb * 2048;
    const uint8_t* q = w + (int64_t)row_tiles * a.h_steps * (kWave * 16);
    b.gate[0] = load_once(w + w_lane);
    b.gate[1] = load_once(w + half * 1024 + w_lane);
    b.up[0] = load_once(q + w_lane);
    b.up[1] = load_once(q + half * 1024 + w_lane);
    const uint8_t* xp = reinterpret_cast<const uint8_t*>(a.x + (int64_t)kb * kBlock);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32x4_t* c = reinterpret_cast<const u32x4_t*>(xp + (h ? half * 2 * kStepK : 0) + x_at);
      b.x[h][0] = c[0];
      b.x[h][1] = c[1];
    }
    b.s_gate = p_scale[kb];
    b.s_up = p_scale[(int64_t)a.i_blocks * a.h_blocks + kb];
  };
  auto advance = [&]() {
    if (++pj == chunks) {
      pj = 0;
      enter(++pi);
    }
  };
  // The wavefronts' partial tiles meet in LDS (two buffers, one barrier an item); one wavefront, another one each time, adds
  // them in wavefront order while the others stream on.
  f32x4_t acc_gate = {0.f, 0.f, 0.f, 0.f}, acc_up = acc_gate;
  auto leave = [&](int i) {
    f32x4_t* const slot = part + (i & 1) * W * 2 * kWave + lane;
    slot[2 * v * kWave] = acc_gate;
    slot[(2 * v + 1) * kWave] = acc_up;
    acc_gate = acc_up = f32x4_t{0.f, 0.f, 0.f, 0.f};
    ring_barrier();
    if (v != i % W) return;
    const int item = first_item + i, at = item / row_tiles, j = item - at * row_tiles;
    const int first = s.first[at];
    if (r >= s.first[at + 1] - first) return;
    f32x4_t gate = slot[0], up = slot[kWave];
    for (int u = 1; u < W; ++u) {
      gate += slot[2 * u * kWave];
      up += slot[(2 * u + 1) * kWave];
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
  enter(pi);
  load(0, 0, buf[0]);
  load(0, 1, buf[1]);
  int ci = 0, cj = 0;
  const int total = n_items * chunks;
  for (int n = 0; n + 1 < total; ++n) {
    advance();
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      if (block(cj, p) < a.h_blocks) {  // uniform
        const bool second = 2 * block(cj, p) + 1 < a.h_steps;
        acc_gate += block_product(buf[p].gate, buf[p].x, second) * buf[p].s_gate;
        acc_up += block_product(buf[p].up, buf[p].x, second) * buf[p].s_up;
      }
      load(pj, p, buf[p]);
    }
    if (++cj == chunks) {
      leave(ci++);
      cj = 0;
    }
  }
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    if (block(cj, p) < a.h_blocks) {
      const bool second = 2 * block(cj, p) + 1 < a.h_steps;
      acc_gate += block_product(buf[p].gate, buf[p].x, second) * buf[p].s_gate;
      acc_up += block_product(buf[p].up, buf[p].x, second) * buf[p].s_up;
    }
  }
  leave(ci);
}

// The grid is (groups of kDownTiles tiles, splits of the units).
__global__ void __launch_bounds__(kDownWaves* kWave) moe_down_kernel(const MoeArgs a) {
  __shared__ int16_t pair[kMaxPairs][kMaxT];
  __shared__ float weight[kMaxPairs][kMaxT];
  __shared__ uint16_t expert[kMaxPairs];
  __shared__ f32x4_t part[kDownWaves][kDownTiles][kWave];
  __shared__ int last_arrival;
  const int lane = threadIdx.x & (kWave - 1);
  const int v = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int g = lane >> 4, r = lane & 15;
  const int h_tiles = a.H / kTileN, nt = blockIdx.x * kDownTiles;
  const int active = a.routing->active;
  for (int i = threadIdx.x; i < active * kMaxT; i += blockDim.x) {
    (&pair[0][0])[i] = (&a.routing->pair[0][0])[i];
    (&weight[0][0])[i] = (&a.routing->weight[0][0])[i];
  }
  for (int i = threadIdx.x; i < active; i += blockDim.x) expert[i] = a.routing->expert[i];
  __syncthreads();
  // this split's (chosen expert, block of I) units, interleaved over the wavefronts, two of a wavefront's in flight
  const int units = active * a.i_blocks;
  const int u0 = (int)((int64_t)blockIdx.y * units / a.splits), u1 = (int)((int64_t)(blockIdx.y + 1) * units / a.splits);
  const int total = u1 - u0 > v ? (u1 - u0 - v + kDownWaves - 1) / kDownWaves : 0;
  struct Unit {
    u32x4_t w[kDownTiles][2], hi[2][2], lo[2][2];
    float s[kDownTiles];
    bool in, second;
  };
  Unit buf[2];
  auto load = [&](int i, Unit& b) {
    const bool some = i < total;
    const int u = some ? u0 + v + i * kDownWaves : u0 + v;
    const int at = u / a.i_blocks, kb = u - at * a.i_blocks;
    const int64_t e = __builtin_amdgcn_readfirstlane(expert[at]);
    b.second = 2 * kb + 1 < a.i_steps;
    const int half = b.second ? 1 : 0;
    const uint32_t w_lane = some ? (uint32_t)lane * 16 : 0u;
    const int p = some ? pair[at][r] : -1;
    b.in = p >= 0;
    const float c = weight[at][r];
#pragma unroll
    for (int t = 0; t < kDownTiles; ++t) {
      const int tile = min(nt + t, h_tiles - 1);
      const uint8_t* q = a.w2 + ((e * h_tiles + tile) * a.i_steps + 2 * kb) * (kWave * 16);
      b.w[t][0] = load_once(q + w_lane);
      b.w[t][1] = load_once(q + half * 1024 + w_lane);
      b.s[t] = a.s2[(e * a.h_blocks + tile * kTileN / kBlock) * a.i_blocks + kb] * c;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int q = 0; q < 2; ++q) b.hi[h][q] = b.lo[h][q] = u32x4_t{0u, 0u, 0u, 0u};
    if (b.in) {  // a token that is not routed here: zeros, whatever `a` holds
      const uint16_t* c = a.a + (int64_t)p * 2 * a.I + kb * kBlock + 16 * g;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          b.hi[h][q] = *reinterpret_cast<const u32x4_t*>(c + (h ? half * kStepK : 0) + 8 * q);
          b.lo[h][q] = *reinterpret_cast<const u32x4_t*>(c + a.I + (h ? half * kStepK : 0) + 8 * q);
        }
    }
  };
  f32x4_t acc[kDownTiles];
#pragma unroll
  for (int t = 0; t < kDownTiles; ++t) acc[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  auto use = [&](const Unit& b) {
#pragma unroll
    for (int t = 0; t < kDownTiles; ++t) {
      const f32x4_t add = (block_product(b.w[t], b.hi, b.second) + block_product(b.w[t], b.lo, b.second)) * b.s[t];
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[t][e] += b.in ? add[e] : 0.f;  // NaN weights of an expert reach its own tokens only
    }
  };
  if (total > 0) {
    load(0, buf[0]);
    load(1, buf[1]);
    int i = 0;
    for (; i + 2 < total; i += 2) {
      use(buf[0]);
      load(i + 2, buf[0]);
      use(buf[1]);
      load(i + 3, buf[1]);
    }
    use(buf[0]);
    if (i + 1 < total) use(buf[1]);
  }
#pragma unroll
  for (int t = 0; t < kDownTiles; ++t) part[v][t][lane] = acc[t];
  __syncthreads();
  auto store = [&](int tile, f32x4_t sum) {
    *reinterpret_cast<u32x2_t*>(a.y + (int64_t)r * a.ldy + tile * kTileN + 4 * g) =
        u32x2_t{pack_bf16(sum[0], sum[1]), pack_bf16(sum[2], sum[3])};
  };
  const bool mine = v < kDownTiles && nt + v < h_tiles && r < a.T;  // wavefront t adds tile t up
  auto slot = [&](int split) { return a.partial + ((int64_t)split * h_tiles + nt + v) * 2 * kWave + lane; };
  if (mine) {
    f32x4_t sum = part[0][v][lane];
    for (int u = 1; u < kDownWaves; ++u) sum += part[u][v][lane];
    if (a.splits == 1) {
      store(nt + v, sum);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        __hip_atomic_store(slot(blockIdx.y) + h * kWave, __builtin_bit_cast(uint64_t, f32x2_t{sum[2 * h], sum[2 * h + 1]}),
                           __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  if (a.splits == 1) return;
  // The splits' sums are in device memory (device-scope stores, waited for) before the group's arrival is counted; the last
  // one reads them with device-scope loads issued after its increment returned, and adds them in split order.
  wait_vmcnt<0>();
  __syncthreads();
  if (threadIdx.x == 0)
    last_arrival = __hip_atomic_fetch_add(&a.routing->arrivals[blockIdx.x], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                   (unsigned)(a.splits - 1);
  __syncthreads();
  if (!last_arrival || !mine) return;
  f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j < a.splits; j += 4) {  // a batch's loads are all in flight at once
    f32x2_t q[4][2];
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        q[k][h] = __builtin_bit_cast(f32x2_t, __hip_atomic_load(slot(min(j + k, a.splits - 1)) + h * kWave, __ATOMIC_RELAXED,
                                                                __HIP_MEMORY_SCOPE_AGENT));
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const f32x4_t p = {q[k][0].x, q[k][0].y, q[k][1].x, q[k][1].y};
      if (j + k < a.splits) sum = j + k == 0 ? p : sum + p;
    }
  }
  store(nt + v, sum);
}

// Wavefronts of the first launch's workgroups, each with two blocks of H in flight: the fewest passes over an item's blocks,
// evenly filled.  17 blocks (H 2112, 7 tokens): 27 us with 9 wavefronts and one workgroup a CU, 32 with 8 in two passes and
// two workgroups; 16 blocks: 48 with 8, 50 with 9 or 4, 60 with 5.
constexpr int kCus = 256;
constexpr int kSimdWaves = 4;  // of this kernel, by its registers; a workgroup's wavefronts go round the 4 SIMDs
int up_waves(int h_blocks) {
  const int passes = (h_blocks + 2 * kMaxUpWaves - 1) / (2 * kMaxUpWaves);
  const int waves = (h_blocks + 2 * passes - 1) / (2 * passes);
  return waves < 4 ? 4 : waves;
}

// The first launch's kernels by the routing's shape.  With 15 or 16 wavefronts the partial tiles and the routing pass the LDS
// that a launch may have unasked.
struct UpKernel {
  void (*fn)(MoeArgs);
  std::atomic<uint64_t> raised;
};
UpKernel& up_kernel(bool shared_waves, int E) {
  static UpKernel kernels[] = {{&moe_up_kernel<16, 4>, {0}}, {&moe_up_kernel<16, 8>, {0}}, {&moe_up_kernel<64, 1>, {0}},
                               {&moe_up_kernel<64, 2>, {0}}, {&moe_up_kernel<64, 4>, {0}}, {&moe_up_kernel<64, 8>, {0}}};
  if (shared_waves && E <= 128) return kernels[E <= 64 ? 0 : 1];
  return kernels[E <= 64 ? 2 : E <= 128 ? 3 : E <= 256 ? 4 : 5];
}

// Splits of the second launch: one workgroup a CU where the tile groups alone are fewer, and a unit a wavefront at least, as
// joining them takes about 2 us (H 512: 4 units 4.2 us, 7.0 in 16 splits; 16 units 5.7 and 7.9; H 1024: 30 units 7.4 in
// one, 6.4 in 2 or 8).
int down_groups(int H) { return (H / kTileN + kDownTiles - 1) / kDownTiles; }
int down_splits(int T, int E, int top_k, int H, int I) {
  const int64_t chosen = T * top_k < E ? T * top_k : E, units = chosen * ((I + kBlock - 1) / kBlock);  // at most
  const int64_t splits = down_groups(H) <= kDownGrid / 2 ? kDownGrid / down_groups(H) : 1;
  return (int)(units / kDownWaves < 1 ? 1 : units / kDownWaves < splits ? units / kDownWaves : splits);
}

bool moe_sizes_ok(int T, int E, int top_k, int H, int I) {
  return T >= 1 && T <= kMaxT && E >= 1 && E <= QF_MOE_MAX_EXPERTS && top_k >= 1 && top_k <= QF_MOE_MAX_TOP_K &&
         top_k <= E && H >= kStepK && H % kStepK == 0 && I >= kStepK && I % kStepK == 0 && H <= (1 << 24) && I <= (1 << 22);
}

constexpr size_t kRoutingBytes = (sizeof(Routing) + 255) / 256 * 256;
size_t partial_bytes(int splits, int H) { return splits > 1 ? (size_t)splits * (H / kTileN) * 1024 : 0; }

}  // namespace qfb

using namespace qfb;

extern "C" {

size_t qf_moe_few_workspace_bytes(int T, int E, int top_k, int H, int I) {
  if (!moe_sizes_ok(T, E, top_k, H, I)) return 0;
  return kRoutingBytes + partial_bytes(down_splits(T, E, top_k, H, I), H) + ((size_t)T * top_k * I * 4 + 255) / 256 * 256;
}

int qf_moe_few_tokens(const uint16_t* x, int64_t ldx, const void* logits, int64_t ldl, int logits_f32, const uint8_t* w13,
                      const float* s13, const uint8_t* w2, const float* s2, uint16_t* y, int64_t ldy, int T, int E,
                      int top_k, int H, int I, int renormalize, void* workspace, size_t workspace_bytes, void* stream) {
  if (x == nullptr || logits == nullptr || w13 == nullptr || s13 == nullptr || w2 == nullptr || s2 == nullptr || y == nullptr)
    return QF_ERR_INVALID_ARG;
  if (T < 1 || E < 1 || top_k < 1 || H < 1 || I < 1 || (T > 1 && (ldx < H || ldl < E || ldy < H))) return QF_ERR_INVALID_ARG;
  if (!moe_sizes_ok(T, E, top_k, H, I)) return QF_ERR_UNSUPPORTED;
  if (ldx > ((int64_t)1 << 26) || ldx % 8 || ldy % 4 || !aligned16(x) || !aligned16(w13) || !aligned16(w2) ||
      ((uintptr_t)y & 7))
    return QF_ERR_UNSUPPORTED;
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
  a.partial = reinterpret_cast<uint64_t*>(static_cast<uint8_t*>(workspace) + kRoutingBytes);
  a.splits = down_splits(T, E, top_k, H, I);
  a.a = reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(workspace) + kRoutingBytes + partial_bytes(a.splits, H));
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
  const int waves = up_waves(a.h_blocks), resident = kCus * (kSimdWaves / ((waves + 3) / 4));
  const unsigned grid = (unsigned)(items < resident - 1 ? items + 1 : resident);
  // Routing: a wavefront a token where there are as many, else 16 lanes a token, so that 4 tokens share a round's latency (16
  // tokens, 8 of 16 experts, H 512, I 128: 9.8 -> 6.8 us; 16 lanes for one token: +0.5 us).
  UpKernel& up = up_kernel(T > waves, E);
  const int lds = waves * kUpWaveLds;
  if (lds + (int)sizeof(RoutingLds) > kDefaultLds && !raise_lds(reinterpret_cast<const void*>(up.fn), kMaxUpWaves * kUpWaveLds, up.raised))
    return QF_ERR_HIP;
  hipLaunchKernelGGL(up.fn, dim3(grid), dim3(waves * kWave), lds, s, a);
  if (hipGetLastError() != hipSuccess) return QF_ERR_HIP;
  hipLaunchKernelGGL(moe_down_kernel, dim3((unsigned)down_groups(H), (unsigned)a.splits), dim3(kDownWaves * kWave), 0, s, a);
  return hipGetLastError() == hipSuccess ? QF_OK : QF_ERR_HIP;
}

}  // extern "C"
