// Page allocation, slot map and positions of a step, from the sequences' lengths (ea_plan_step_cuda),
// and the serving operators' error text.
//
// Everything follows from two prefix sums over the batch, of the new tokens and of the fresh pages
//   fresh_b = ceil((ctx_b + new_b) / ps) - ceil(ctx_b / ps),
// so every block computes both sums for itself in shared memory (8 bytes a sequence, from L2) and then
// works on its share of the tokens and of the fresh pages: one launch, no block waits for another.
// A token's page is found without the table entries that this launch writes: a page past the owned ones
// is free_pages[free_head + (fresh pages of earlier sequences) + its number].
// Bound by latency: 64 sequences 7 to 8 us a call, 509 sequences with 262,000 tokens (5.3 MB) 8 to 9 us, of which the
// host takes 7.
#include <stdio.h>
#include <string.h>

#include "ea_serving.cuh"

namespace ea {
namespace serving {

static thread_local char g_msg[256] = "";

int fail(int code, const char* msg) {
  snprintf(g_msg, sizeof g_msg, "%s", msg);
  return code;
}
int cuda_rc(cudaError_t e) { return e == cudaSuccess ? 0 : fail(-4, cudaGetErrorString(e)); }

int sm_count() {
  static int cached[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev < 64 && cached[dev]) return cached[dev];
  int n = 0;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  if (dev < 64) cached[dev] = n;
  return n;
}

namespace {

constexpr int THREADS = 256;
constexpr int PER_THREAD = 4;  // consecutive tokens: one 16-byte store of positions and of sequences

// first index i of the nondecreasing a[1 .. n] with a[i] > x, i.e. the segment b = i - 1 that holds x
__device__ __forceinline__ int segment_of(const int32_t* a, int n, int32_t x) {
  int lo = 0, hi = n;  // a[lo] <= x < a[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// 64 bits: a context and its new tokens together may need 2^32 pages of one row.
__device__ __forceinline__ int64_t pages_of(int64_t n, int ps) { return (n + ps - 1) / ps; }

// Prefix sums saturate at INT32_MAX, so a step with too many tokens still gives ordered sums.
__device__ __forceinline__ int32_t saturate(int64_t x) { return (int32_t)(x < 0x7FFFFFFF ? x : 0x7FFFFFFF); }

__global__ void __launch_bounds__(THREADS) plan_step_kernel(ea_plan_step_t a, FastDiv by_page, bool vec) {
  begin();
  extern __shared__ int32_t sm[];
  int32_t* tok = sm;                  // (batch + 1) prefix sums of the new tokens
  int32_t* frs = sm + a.batch + 1;    // (batch + 1) prefix sums of the fresh pages
  __shared__ int64_t wsum[2][THREADS / 32];
  __shared__ int too_long;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) too_long = 0;
  // per thread a run of consecutive sequences
  const int run = (a.batch + THREADS - 1) / THREADS;
  const int b0 = min(a.batch, tid * run), b1 = min(a.batch, b0 + run);
  int64_t st = 0, sf = 0;
  for (int b = b0; b < b1; ++b) {
    const int32_t ctx = max(0, a.context_lens[b]), nw = max(0, a.new_lens[b]);
    st += nw;
    sf += pages_of((int64_t)ctx + nw, a.page_size) - pages_of(ctx, a.page_size);
  }
  int64_t pt = st, pf = sf;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, pt, o), y = __shfl_up_sync(0xffffffffu, pf, o);
    if (lane >= o) pt += x, pf += y;
  }
  if (lane == 31) wsum[0][warp] = pt, wsum[1][warp] = pf;
  __syncthreads();
  pt -= st, pf -= sf;
  for (int w = 0; w < warp; ++w) pt += wsum[0][w], pf += wsum[1][w];
  bool over = false;
  for (int b = b0; b < b1; ++b) {
    const int32_t ctx = max(0, a.context_lens[b]), nw = max(0, a.new_lens[b]);
    tok[b] = saturate(pt), frs[b] = saturate(pf);
    const int64_t need = pages_of((int64_t)ctx + nw, a.page_size);
    pt += nw, pf += need - pages_of(ctx, a.page_size);
    over |= need > a.max_pages;
    if (blockIdx.x == b % gridDim.x) {
      a.q_start[b] = tok[b];
      a.seq_lens[b] = saturate((int64_t)ctx + nw);
    }
  }
  if (b1 == a.batch && b0 < b1) tok[a.batch] = saturate(pt), frs[a.batch] = saturate(pf);
  if (a.batch == 0 && tid == 0) tok[0] = frs[0] = 0;
  if (over) too_long = 1;
  __syncthreads();

  const int32_t total = tok[a.batch], fresh = frs[a.batch];
  const int32_t head = a.free_head ? max(0, *a.free_head) : 0;
  if (blockIdx.x == 0 && tid == 0) {
    a.q_start[a.batch] = total;
    *a.next_free_head = (int32_t)min((int64_t)a.num_free, (int64_t)head + fresh);
    *a.status = ((int64_t)head + fresh > a.num_free ? EA_PLAN_NO_PAGES : 0) | (too_long ? EA_PLAN_TABLE_FULL : 0) |
                (total > a.max_tokens ? EA_PLAN_TOO_MANY : 0);
  }

  // fresh pages into the table
  for (int32_t f = blockIdx.x * THREADS + tid; f < fresh; f += gridDim.x * THREADS) {
    const int b = segment_of(frs, a.batch, f);
    const int64_t col = pages_of(max(0, a.context_lens[b]), a.page_size) + (f - frs[b]);
    const int64_t at = (int64_t)head + f;
    if (col < a.max_pages) a.page_table[b * a.table_stride + col] = at < a.num_free ? a.free_pages[at] : -1;
    if (f > 0x7FFFFFFF - (int32_t)(gridDim.x * THREADS)) break;
  }

  // tokens
  const int64_t t0 = ((int64_t)blockIdx.x * THREADS + tid) * PER_THREAD;
  if (t0 >= a.max_tokens) return;
  int64_t slot[PER_THREAD];
  int32_t pos[PER_THREAD], seq[PER_THREAD];
  int b = t0 < total ? segment_of(tok, a.batch, (int32_t)t0) : a.batch;
  int32_t ctx = 0, first = 0, owned = 0;
  bool fetch = true;
#pragma unroll
  for (int j = 0; j < PER_THREAD; ++j) {
    const int32_t t = (int32_t)t0 + j;
    slot[j] = -1, pos[j] = 0, seq[j] = -1;
    if (t >= total || t >= a.max_tokens) continue;
    while (tok[b + 1] <= t) ++b, fetch = true;
    if (fetch) {
      ctx = max(0, a.context_lens[b]), first = tok[b];
      owned = (int32_t)pages_of(ctx, a.page_size);
      fetch = false;
    }
    const int32_t i = t - first;
    seq[j] = b;
    pos[j] = ctx + (a.depths ? a.depths[t] : i);
    const int32_t p = ctx + i;
    const uint32_t col = div_by((uint32_t)p, by_page);
    int32_t page = -1;
    if (p >= 0 && col < (uint32_t)a.max_pages) {
      const int64_t at = (int64_t)head + frs[b] + ((int64_t)col - owned);
      if ((int32_t)col < owned) page = a.page_table[b * a.table_stride + col];
      else if (at < a.num_free) page = a.free_pages[at];
    }
    if (page >= 0) slot[j] = (int64_t)page * a.page_size + (p - (int64_t)col * a.page_size);
  }
  if (vec && t0 + PER_THREAD <= a.max_tokens) {
    *(int4*)(a.positions + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
    *(int4*)(a.token_seq + t0) = make_int4(seq[0], seq[1], seq[2], seq[3]);
    *(longlong2*)(a.slot_map + t0) = make_longlong2(slot[0], slot[1]);
    *(longlong2*)(a.slot_map + t0 + 2) = make_longlong2(slot[2], slot[3]);
  } else {
#pragma unroll
    for (int j = 0; j < PER_THREAD; ++j)
      if (t0 + j < a.max_tokens) a.positions[t0 + j] = pos[j], a.token_seq[t0 + j] = seq[j], a.slot_map[t0 + j] = slot[j];
  }
}

}  // namespace
}  // namespace serving
}  // namespace ea

extern "C" const char* ea_serving_last_error(void) { return ea::serving::g_msg; }

extern "C" int ea_plan_step_cuda(const ea_plan_step_t* a, void* stream) {
  using namespace ea::serving;
  if (!a || a->batch < 0 || a->max_pages < 0 || a->page_size <= 0 || a->num_free < 0 || a->max_tokens < 0)
    return fail(-1, "plan_step: negative size, or no page size");
  if (a->batch > EA_PLAN_MAX_SEQS) return fail(-1, "plan_step: more than EA_PLAN_MAX_SEQS sequences");
  if (!a->q_start || !a->next_free_head || !a->status ||
      (a->batch && (!a->context_lens || !a->new_lens || !a->seq_lens || (a->max_pages && !a->page_table))) ||
      (a->num_free && !a->free_pages) || (a->max_tokens && (!a->slot_map || !a->positions || !a->token_seq)))
    return fail(-1, "plan_step: a required pointer is NULL");
  if (a->next_free_head == a->free_head) return fail(-1, "plan_step: next_free_head may not be free_head");
  const auto smem_of = [](int batch) { return 2 * (int)sizeof(int32_t) * (batch + 1); };
  // Room for the largest batch, once per device: the attribute belongs to the device, so a call that set it to its own
  // batch's would take it from a larger one that another thread is about to launch.
  static bool ready[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !ready[dev])) {
    e = cudaFuncSetAttribute(plan_step_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_of(EA_PLAN_MAX_SEQS));
    if (e == cudaSuccess && dev < 64) ready[dev] = true;
  }
  if (e != cudaSuccess) return cuda_rc(e);
  const int per_block = THREADS * PER_THREAD;
  const int grid = a->max_tokens > per_block ? (int)(((int64_t)a->max_tokens + per_block - 1) / per_block) : 1;
  const bool vec = (((uintptr_t)a->slot_map | (uintptr_t)a->positions | (uintptr_t)a->token_seq) & 15) == 0;
  return cuda_rc(launch_early(plan_step_kernel, grid, THREADS, smem_of(a->batch), (cudaStream_t)stream, *a, fast_div((uint32_t)a->page_size), vec));
}
