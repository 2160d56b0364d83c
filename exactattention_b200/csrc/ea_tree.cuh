// Work schedule and split partials of the tree attention kernels (ea_tree.cu, ea_tree_tc.cu).
//
// The work is cut into units of KT keys for one row tile (ROWS query rows of one sequence and kv head):
// unit order is (sequence, kv head, row tile, key tile). `workers` blocks take equal contiguous shares of
// the units, so lengths may differ freely without idle blocks and without the host knowing them: every
// block finds its share from the prefix sums of the sequences' units. An item (all key tiles of one row
// tile) that crosses shares leaves one partial (row maximum, row sum, unnormalised output) per share,
// which the block of the combine kernel that belongs to the item's first share adds up in share order.
#pragma once
#include "ea_serving.cuh"

namespace ea {
namespace serving {
namespace tree {

struct Args {
  ea_tree_attention_t t;
  FastDiv by_page, by_group;
  int group;     // query heads per kv head
  int workers;   // blocks that share the units
  int dp;        // channels of a partial: d rounded up
};

struct Item {
  int b, h, m;            // sequence, kv head, row tile
  int q0, new_tokens;     // first token of the step and their number
  int len;                // keys, the step's own included
  int kt0, kt1, tiles;    // key tiles of this share, and of the item
};

__device__ __forceinline__ int seq_len(const Args& a, int b) {
  return (int)min((int64_t)max(a.t.seq_lens[b], 0), (int64_t)a.t.max_pages * a.t.page_size);
}
__device__ __forceinline__ void seq_tokens(const Args& a, int b, int& q0, int& n) {
  const int64_t lo = max(a.t.q_start[b], 0), hi = min((int64_t)a.t.q_start[b + 1], a.t.tokens);
  q0 = (int)lo, n = (int)max(hi - lo, (int64_t)0);
}

template <int ROWS, int KT>
struct Schedule {
  const uint32_t* prefix;  // (batch + 1) in shared memory
  uint32_t total, workers;  // units; blocks that get some (a block past them has nothing to do)

  // Every thread of the block calls this; `sums` holds batch + 1 words, `scratch` 32.
  __device__ void build(const Args& a, uint32_t* sums, uint64_t* scratch) {
    const int n = a.t.batch, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    uint64_t carry = 0;  // sums saturate, so they stay ordered whatever q_start holds
    for (int base = 0; base < n; base += blockDim.x) {
      const int b = base + tid;
      uint64_t u = 0;
      if (b < n) {
        int q0, nt;
        seq_tokens(a, b, q0, nt);
        u = (uint64_t)a.t.kv_heads * (uint32_t)((nt * a.group + ROWS - 1) / ROWS) *
            (uint32_t)max(1, (seq_len(a, b) + KT - 1) / KT);
      }
      uint64_t s = u;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t x = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += x;
      }
      if (lane == 31) scratch[warp] = s;
      __syncthreads();
      uint64_t before = carry, all = carry;
      for (int w = 0; w < warps; ++w) {
        if (w < warp) before += scratch[w];
        all += scratch[w];
      }
      if (b < n) sums[b] = (uint32_t)min((unsigned long long)(before + s - u), 0x7FFFFFFFull);
      carry = all;
      __syncthreads();
    }
    carry = min((unsigned long long)carry, 0x7FFFFFFFull);
    if (tid == 0) sums[n] = (uint32_t)carry;
    __syncthreads();
    prefix = sums, total = (uint32_t)carry, workers = min((uint32_t)a.workers, total);
  }
  // First unit of a share; none of the `workers` shares is empty.
  __device__ uint32_t share(uint32_t worker) const {
    return worker >= workers ? total : (uint32_t)((uint64_t)total * worker / workers);
  }
  // The item of unit `pos` and how far it goes before `end`.
  __device__ Item item(const Args& a, uint32_t pos, uint32_t end) const {
    int lo = 0, hi = a.t.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid] <= pos) lo = mid;
      else hi = mid;
    }
    Item it;
    it.b = lo;
    seq_tokens(a, lo, it.q0, it.new_tokens);
    it.len = seq_len(a, lo);
    it.tiles = max(1, (it.len + KT - 1) / KT);
    const uint32_t mt = (uint32_t)((it.new_tokens * a.group + ROWS - 1) / ROWS);
    const uint32_t rel = pos - prefix[lo], idx = rel / (uint32_t)it.tiles;
    it.kt0 = (int)(rel - idx * it.tiles);
    it.kt1 = (int)min((uint32_t)it.tiles, it.kt0 + (end - pos));
    it.h = (int)(idx / mt), it.m = (int)(idx - it.h * mt);
    return it;
  }
};

// A share's partials: slot 2 w is the item it began inside of (its first), slot 2 w + 1 the one it leaves
// unfinished. Layout of a slot: ROWS x dp floats, ROWS maxima, ROWS sums.
__device__ __forceinline__ float* slot_of(const Args& a, int slot, int rows) {
  return (float*)a.t.workspace + (int64_t)slot * rows * (a.dp + 2);
}

// Kernel for more than 16 rows per kv head (ea_tree_tc.cu): 256-row items with `pair`, else 128-row ones.
constexpr int MANY_MAX_SEQS = 6000;  // what its shared memory has room for
int launch_many(const Args& a, bool pair, cudaStream_t st);

// Adds up the partials of the item that share blockIdx.x left unfinished, 16 rows a block (blockIdx.y).
template <typename T, int ROWS, int KT, int THREADS>
__global__ void __launch_bounds__(THREADS) combine_kernel(Args a) {
  extern __shared__ uint32_t sums[];
  __shared__ uint64_t scratch[32];
  Schedule<ROWS, KT> sch;
  sch.build(a, sums, scratch);
  const int w = blockIdx.x;
  const uint32_t lo = sch.share(w), hi = sch.share(w + 1);
  if (lo >= hi) return;
  const Item it = sch.item(a, hi - 1, hi);
  const uint32_t begin = hi - 1 - it.kt0;  // the item's first unit
  const uint32_t end = begin + it.tiles;
  if (begin < lo || end <= hi) return;  // begun earlier, or finished here
  int last = w;
  while (sch.share(last + 1) < end) ++last;
  const int r0 = blockIdx.y * 16, rows = min(16, min(ROWS, it.new_tokens * a.group - it.m * ROWS) - r0);
  const int stride = ROWS * (a.dp + 2);
  const float* first = slot_of(a, 2 * w + 1, ROWS);
  const float* rest = slot_of(a, 2 * w, ROWS);  // share w' > w: rest + (w' - w) * 2 * stride
  const int cols = a.dp;
  for (int e = threadIdx.x; e < rows * cols; e += THREADS) {
    const int r = r0 + e / cols, c = e % cols;
    float m = first[ROWS * a.dp + r];
    for (int i = 1; i <= last - w; ++i) m = fmaxf(m, rest[(int64_t)i * 2 * stride + ROWS * a.dp + r]);
    const float base = m == -INFINITY ? 0.0f : m;
    float s = exp2f(first[ROWS * a.dp + r] - base);
    float l = first[ROWS * (a.dp + 1) + r] * s, o = first[r * a.dp + c] * s;
    for (int i = 1; i <= last - w; ++i) {
      const float* p = rest + (int64_t)i * 2 * stride;
      s = exp2f(p[ROWS * a.dp + r] - base);
      l = fmaf(p[ROWS * (a.dp + 1) + r], s, l);
      o = fmaf(p[r * a.dp + c], s, o);
    }
    const int R = it.m * ROWS + r, i = (int)div_by((uint32_t)R, a.by_group), j = R - i * a.group;
    const int64_t head = (int64_t)(it.q0 + i) * a.t.q_heads + it.h * a.group + j;
    if (c < a.t.d) ((T*)a.t.out)[head * a.t.d + c] = from_f<T>(l == 0.0f ? 0.0f : o / l);
    if (c == 0 && a.t.lse) a.t.lse[head] = l == 0.0f ? -INFINITY : m + log2f(l);
  }
}

}  // namespace tree
}  // namespace serving
}  // namespace ea
