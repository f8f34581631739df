// qf_kv4_tables.hip — a step's tables from request lengths (gfx950).
//
// Every workgroup scans the requests' lengths for itself (cu_q and the pages' places, in LDS) and then writes its share of
// the tokens and of the new table entries: a token finds its request, an entry its row, by bisection.  So the whole is one
// launch without a word between workgroups, and what bounds it is that launch: the lengths' latency, a scan of one workgroup
// and the bisection (12 steps of LDS latency for 4096 requests).  1 request 2.8 us, 333 requests with 26 000 tokens 5.1 us.
#include "qf_kv4_common.h"

namespace qfk {

constexpr int kTableThreads = 256;
constexpr int kTableWaves = kTableThreads / kWave;

struct TableArgs {
  const int32_t *context, *q_lens, *held;
  int32_t* table;
  int64_t bt_stride;
  const int32_t *stack, *count;
  int max_blocks, num_free, B, page, T;
  Divisor by_page;
  int32_t *cu_q, *seq_lens;
  int64_t *positions, *slots;
  int32_t *held_out, *count_out, *fits;
};

// Sums that stop at `cap` (at most 2^30): whatever passes it does not fit anyway, and no sum overflows.
__device__ __forceinline__ int capped(int a, int b, int cap) { return min(a + b, cap); }

// The last i of [0, n] with at[i] <= v, at[0] = 0 and rising; n where at[n] <= v.
__device__ __forceinline__ int find(const int* at, int n, int v) {
  int lo = 0, hi = n + 1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (at[mid] <= v) {
      lo = mid;
    } else {
      hi = mid;
    }
  }
  return lo;
}

__global__ __launch_bounds__(kTableThreads) void step_tables_kernel(TableArgs a) {
  extern __shared__ int lds[];
  int* const cu = lds;               // [B + 1] first token of each request
  int* const first = lds + a.B + 1;  // [B + 1] its first new page's place below the stack's top
  __shared__ int wave_q[kTableWaves], wave_need[kTableWaves], wave_bad[kTableWaves];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int count = *a.count;
  const int cap_q = a.T + 1, cap_need = a.num_free + 1;
  const int per = (a.B + kTableThreads - 1) / kTableThreads;  // requests of a thread

  int q_sum = 0, need_sum = 0;
  bool bad = count < 0 || count > a.num_free;
  for (int i = 0; i < per; ++i) {
    const int b = threadIdx.x * per + i;
    if (b >= a.B) break;
    const int context = a.context[b], q = a.q_lens[b], held = a.held[b];
    const int64_t seq = (int64_t)context + q;
    bad |= context < 0 || q < 0 || held < 0 || held > a.max_blocks || seq > 0x7fffffff;
    const int pages = seq > 0 && seq <= 0x7fffffff ? divide((int)seq - 1, a.by_page) + 1 : 0;
    bad |= pages > a.max_blocks;
    q_sum = capped(q_sum, min(max(q, 0), cap_q), cap_q);
    need_sum = capped(need_sum, min(max(pages - max(held, 0), 0), cap_need), cap_need);
  }
  int q_upto = q_sum, need_upto = need_sum;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const int q = __shfl_up(q_upto, d), need = __shfl_up(need_upto, d);
    if (lane >= d) {
      q_upto = capped(q_upto, q, cap_q);
      need_upto = capped(need_upto, need, cap_need);
    }
  }
  if (lane == kWave - 1) {
    wave_q[wave] = q_upto;
    wave_need[wave] = need_upto;
  }
  const bool wave_any = __any(bad);
  if (lane == 0) wave_bad[wave] = wave_any;
  // what stands before this thread in its wavefront (a difference of capped sums would be wrong past the cap)
  int q_before = __shfl_up(q_upto, 1), need_before = __shfl_up(need_upto, 1);
  if (lane == 0) q_before = need_before = 0;
  __syncthreads();
  int tokens = 0, pages = 0;
  bad = false;
#pragma unroll
  for (int w = 0; w < kTableWaves; ++w) {
    if (w == wave) {
      q_before = capped(q_before, tokens, cap_q);
      need_before = capped(need_before, pages, cap_need);
    }
    tokens = capped(tokens, wave_q[w], cap_q);
    pages = capped(pages, wave_need[w], cap_need);
    bad |= wave_bad[w] != 0;
  }
  const bool fits = !bad && tokens <= a.T && pages <= count;
  if (!fits) tokens = pages = 0;
  for (int i = 0; i < per; ++i) {
    const int b = threadIdx.x * per + i;
    if (b >= a.B) break;
    const int context = a.context[b], q = fits ? a.q_lens[b] : 0, held = a.held[b];
    const int seq = context + q;
    const int need = fits && seq > 0 ? max(divide(seq - 1, a.by_page) + 1 - held, 0) : 0;
    cu[b] = fits ? q_before : 0;
    first[b] = fits ? need_before : 0;
    if (blockIdx.x == 0) {
      a.cu_q[b] = cu[b];
      a.seq_lens[b] = seq;
      a.held_out[b] = held + need;
    }
    q_before += q;
    need_before += need;
  }
  if (threadIdx.x == 0) {
    cu[a.B] = tokens;
    first[a.B] = pages;
    if (blockIdx.x == 0) {
      a.cu_q[a.B] = tokens;
      *a.count_out = count - pages;
      *a.fits = fits;
    }
  }
  __syncthreads();

  const int threads = gridDim.x * kTableThreads;
  for (int t = blockIdx.x * kTableThreads + threadIdx.x; t < a.T; t += threads) {
    int64_t pos = 0, slot = -1;
    if (t < tokens) {
      const int b = find(cu, a.B, t);
      pos = a.context[b] + (t - cu[b]);
      const int page = divide((int)pos, a.by_page);
      const int held = a.held[b];
      const int id = page < held ? a.table[b * a.bt_stride + page] : a.stack[count - 1 - first[b] - (page - held)];
      slot = (int64_t)id * a.page + (pos - (int64_t)page * a.page);
    }
    a.positions[t] = pos;
    a.slots[t] = slot;
  }
  for (int j = blockIdx.x * kTableThreads + threadIdx.x; j < pages; j += threads) {
    const int b = find(first, a.B, j);
    a.table[b * a.bt_stride + a.held[b] + (j - first[b])] = a.stack[count - 1 - j];
  }
}

}  // namespace qfk

using namespace qfk;

extern "C" int qf_kv4_abi_version(void) { return QF_KV4_ABI_VERSION; }

extern "C" int qf_step_tables(const int32_t* context, const int32_t* q_lens, const int32_t* held, int32_t* block_table,
                              int64_t bt_stride, int max_blocks, const int32_t* free_blocks, const int32_t* free_count,
                              int num_free, int num_reqs, int page_size, int num_tokens, int32_t* cu_q, int32_t* seq_lens,
                              int64_t* positions, int64_t* slots, int32_t* held_out, int32_t* free_count_out, int32_t* fits,
                              void* stream) {
  if (!context || !q_lens || !held || !block_table || !free_count || !cu_q || !seq_lens || !held_out || !free_count_out ||
      !fits || num_reqs < 1 || page_size < 1 || num_tokens < 0 || num_free < 0 || max_blocks < 1 || bt_stride < max_blocks ||
      (num_tokens > 0 && (!positions || !slots)) || (num_free > 0 && !free_blocks))
    return QF_ERR_INVALID_ARG;
  if (num_reqs > QF_STEP_MAX_REQS || num_tokens > QF_STEP_MAX_TOKENS || num_free > QF_STEP_MAX_TOKENS ||
      max_blocks > QF_STEP_MAX_TOKENS)
    return QF_ERR_UNSUPPORTED;
  TableArgs a = {context, q_lens, held, block_table, bt_stride, free_blocks, free_count, max_blocks, num_free, num_reqs,
                 page_size, num_tokens, divisor(page_size), cu_q, seq_lens, positions, slots, held_out, free_count_out, fits};
  const int groups = num_tokens <= kTableThreads ? 1 : (num_tokens + kTableThreads - 1) / kTableThreads;
  step_tables_kernel<<<groups < 512 ? groups : 512, kTableThreads, 2 * (num_reqs + 1) * sizeof(int),
                       static_cast<hipStream_t>(stream)>>>(a);
  return hipGetLastError() == hipSuccess ? QF_OK : QF_ERR_HIP;
}
