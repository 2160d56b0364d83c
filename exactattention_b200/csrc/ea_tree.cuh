// Work schedule and split partials of the tree attention kernels (ea_tree.cu, ea_tree_tc.cu).
//
// The work is cut into units of KT keys for one row tile (ROWS query rows of one sequence and kv head):
// unit order is (sequence, kv head, row tile, key tile). `workers` blocks take equal contiguous shares of
// the units, so lengths may differ freely without idle blocks and without the host knowing them: every
// block finds its share from the prefix sums of the sequences' units. An item (all key tiles of one row
// tile) that crosses shares leaves one partial (row maximum, row sum, unnormalised output) per share,
// which the block of the combine kernel that belongs to the item's first share adds up in share order.
#pragma once
#include <type_traits>

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
  int wait_debug;  // test hook (ea_set_test_hooks): the bounded waits report expiry
};

// The reference m of a row's weights 2^(s - m), in powers of two. When it moves it is put DOWN below the largest score seen;
// it moves only when a score passes m + DOWN by more than LAZY, so that most tiles rescale nothing. Sums, outputs, partials
// and the log-sum-exp all refer to m, whatever it is.
// bf16 has binary32's exponents: a weight keeps its relative error at any size, and DOWN is 0. fp16 loses bits below
// 2^-14 and everything below 2^-25, where the long tail behind one dominant key lies: DOWN + LAZY = 15 uses its range up to
// 2^15, so that the product takes a weight to within 2^-35 of the row's largest (the sum takes it unrounded). A DOWN of 11
// moves the reference so often that 2048 rows over 16384 keys take 340 us instead of 328; with 10 or 9 they take what they
// took without.
template <typename T>
struct Reference {
  static constexpr bool HALF = std::is_same<T, __half>::value;
  static constexpr float DOWN = HALF ? 10.0f : 0.0f, LAZY = HALF ? 5.0f : 8.0f;
  // Whether a score moves m. In fp16 by the difference, which is what the weight will be: m + 15 may round up.
  static __device__ __forceinline__ bool passed(float score, float m) {
    return HALF ? score - m > DOWN + LAZY : score > m + LAZY;
  }
};

struct Item {
  int b, h, m;            // sequence, kv head, row tile
  int q0, new_tokens;     // first token of the step and their number
  int len;                // keys that the page table has room for, the step's own included
  int ctx;                // keys before the step's own
  int kt0, kt1, tiles;    // key tiles of this share (none: kt0 >= kt1), and of the item
  uint32_t next;          // unit after the share's part of the item
};

// Keys of a sequence, as far as its row of the page table goes: keys past it have no page.
__device__ __forceinline__ int seq_len(const Args& a, int b) {
  return (int)min((int64_t)max(a.t.seq_lens[b], 0), (int64_t)a.t.max_pages * a.t.page_size);
}
// The step's tokens of a sequence that q has rows for.
__device__ __forceinline__ void seq_tokens(const Args& a, int b, int& q0, int& n) {
  const int64_t lo = max(a.t.q_start[b], 0), hi = min((int64_t)a.t.q_start[b + 1], a.t.tokens);
  q0 = (int)lo, n = (int)max(hi - lo, (int64_t)0);
}
// Keys before the step's own: from the lengths as they are given, whatever the table and q have room for. Negative where the step
// has more tokens than the sequence keys, but so that key - ctx stays within 32 bits for every key of a tile.
__device__ __forceinline__ int seq_ctx(const Args& a, int b, int len) {
  const int64_t n = max((int64_t)a.t.q_start[b + 1] - a.t.q_start[b], (int64_t)0);
  return (int)max(max(a.t.seq_lens[b], 0) - n, (int64_t)len - 0x7FFFFF00);
}

template <int ROWS, int KT, int EXTRA>
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
            (uint32_t)(max(1, (seq_len(a, b) + KT - 1) / KT) + EXTRA);
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
    it.ctx = seq_ctx(a, lo, it.len);
    it.tiles = max(1, (it.len + KT - 1) / KT);
    const uint32_t mt = (uint32_t)((it.new_tokens * a.group + ROWS - 1) / ROWS);
    const uint32_t units = it.tiles + EXTRA, rel = pos - prefix[lo], idx = rel / units, at = rel - idx * units;
    it.kt0 = (int)at;
    it.kt1 = (int)min((uint32_t)it.tiles, at + (end - pos));
    it.next = pos + min(end - pos, units - at);
    it.h = (int)(idx / mt), it.m = (int)(idx - it.h * mt);
    return it;
  }
};

// A share's partials: slot 2 w is the item it began inside of (its first), slot 2 w + 1 the one it leaves
// unfinished. Layout of a slot: dp / 4 x ROWS x 4 floats (a row per thread stores and loads whole lines), ROWS maxima,
// ROWS sums.
__device__ __forceinline__ float* slot_of(const Args& a, int slot, int rows) {
  return (float*)a.t.workspace + (int64_t)slot * rows * (a.dp + 2);
}

// Kernel for more than 16 rows per kv head (ea_tree_tc.cu): 256-row items with `pair`, else 128-row ones.
constexpr int MANY_MAX_SEQS = 6000;  // what its shared memory has room for
int launch_many(const Args& a, bool pair, cudaStream_t st);

// Adds up the partials of the item that share blockIdx.x left unfinished, 16 rows a block (blockIdx.y). It starts
// while the attention kernel still runs and finds its item meanwhile.
// Thread (share group, four channels, row): the groups take every G-th share; the groups' sums are joined in a fixed
// order. A round is COMBINE_SHARES shares; between rounds what has been added up is rescaled to the new maximum.
// Bound by the latency of loads from L2. A round's maxima and sums are asked for together, of its values COMBINE_AHEAD a
// thread: all of them where there are four groups or more (64 cells: 2 rows of 128 channels), a quarter with one group (7
// rows), the rest one after the other. That is what one item over many shares waits for: one token over 16384 keys of one kv head
// (256 partials, 1.3 us of bytes) takes 61 us a call with 2 rows and 123 us with 8; 131072 keys (296 partials) 84 and 155 us.
constexpr int COMBINE_THREADS = 256, COMBINE_SHARES = 16, COMBINE_AHEAD = 4;  // values a thread has in flight

template <typename T, int ROWS, int KT, int EXTRA>
__global__ void __launch_bounds__(COMBINE_THREADS) combine_kernel(Args a) {
  extern __shared__ uint32_t sums[];
  __shared__ uint64_t scratch[32];
  __shared__ float weight[COMBINE_SHARES][16], rescale[16], top[16], total[16];
  __shared__ float4 joined[COMBINE_THREADS];
  Schedule<ROWS, KT, EXTRA> sch;
  sch.build(a, sums, scratch);
  const int w = blockIdx.x, tid = threadIdx.x, r0 = blockIdx.y * 16;
  const uint32_t lo = sch.share(w), hi = sch.share(w + 1);
  Item it;
  int rows = 0, n = 2;  // rows of this block, shares of the item
  if (lo < hi) {
    it = sch.item(a, hi - 1, hi);
    const uint32_t begin_unit = hi - 1 - it.kt0, end_unit = begin_unit + it.tiles;  // the item's units
    if (begin_unit >= lo && end_unit > hi) {  // begun here and not finished here
      rows = min(16, min(ROWS, it.new_tokens * a.group - it.m * ROWS) - r0);
      while (sch.share(w + n) < end_unit) ++n;
    }
  }
  if (tid < 16) top[tid] = -INFINITY, total[tid] = 0.0f;
  begin();
  if (rows <= 0) return;
  // partial i of the item: slot 2 w + 1, then slots 2 (w + i)
  const auto part = [&](int i) { return slot_of(a, i ? 2 * (w + i) : 2 * w + 1, ROWS); };
  const int vecs = a.dp / 4, cells = rows * vecs;  // at most 512: two cells a thread where there are many rows
  const int groups = max(1, COMBINE_THREADS / cells);
  const int grp = min(tid / cells, groups), cell0 = cells > COMBINE_THREADS ? tid : tid - tid / cells * cells;
  const int mr = tid >> 4, ms = tid & 15;  // the row and share whose maximum and sum this thread reads
  float4 acc[2] = {make_float4(0, 0, 0, 0), make_float4(0, 0, 0, 0)};
  for (int i0 = 0; i0 < n; i0 += COMBINE_SHARES) {
    const int m = min(COMBINE_SHARES, n - i0);
    float pm = -INFINITY, pl = 0.0f;
    if (mr < rows && ms < m) {
      const float* p = part(i0 + ms) + ROWS * a.dp + r0 + mr;
      pm = p[0], pl = p[ROWS];
    }
    float4 x[2][COMBINE_AHEAD];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int cell = cell0 + c * COMBINE_THREADS, v = cell / rows, at = (v * ROWS + r0 + cell - v * rows) * 4;
#pragma unroll
      for (int j = 0; j < COMBINE_AHEAD; ++j)
        if (grp < groups && cell < cells && grp + j * groups < m) x[c][j] = *(const float4*)(part(i0 + grp + j * groups) + at);
    }
    float best = pm;
#pragma unroll
    for (int o = 8; o; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
    __syncthreads();  // the last round's weights are used (and top is set)
    const float was = top[mr], now = fmaxf(was, best), base = now == -INFINITY ? 0.0f : now;
    const float f = exp2f(pm - base), old = exp2f(was - base);
    float l = pl * f;
#pragma unroll
    for (int o = 8; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    weight[ms][mr] = f;
    __syncwarp();  // top and total are read by the row's lanes, which are in one warp
    if (ms == 0) top[mr] = now, total[mr] = fmaf(total[mr], old, l), rescale[mr] = old;
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int cell = cell0 + c * COMBINE_THREADS;
      if (grp >= groups || cell >= cells) continue;
      const int v = cell / rows, r = cell - v * rows, at = (v * ROWS + r0 + r) * 4;
      if (i0) acc[c].x *= rescale[r], acc[c].y *= rescale[r], acc[c].z *= rescale[r], acc[c].w *= rescale[r];
      int j = 0;
      for (int i = grp; i < m; i += groups, ++j) {
        float4 y;
        if (j < COMBINE_AHEAD) {
#pragma unroll
          for (int k = 0; k < COMBINE_AHEAD; ++k)
            if (k == j) y = x[c][k];
        } else {
          y = *(const float4*)(part(i0 + i) + at);
        }
        const float g = weight[i][r];
        acc[c].x = fmaf(y.x, g, acc[c].x), acc[c].y = fmaf(y.y, g, acc[c].y);
        acc[c].z = fmaf(y.z, g, acc[c].z), acc[c].w = fmaf(y.w, g, acc[c].w);
      }
    }
  }
  if (groups > 1) {
    joined[tid] = acc[0];
    __syncthreads();
    if (tid < cells)
      for (int g = 1; g < groups; ++g) {
        const float4 y = joined[g * cells + tid];
        acc[0].x += y.x, acc[0].y += y.y, acc[0].z += y.z, acc[0].w += y.w;
      }
  }
  if (grp > 0) return;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int cell = cell0 + c * COMBINE_THREADS;
    if (cell >= cells) break;
    const int v = cell / rows, r = cell - v * rows, ch = v * 4;
    const int R = it.m * ROWS + r0 + r, i = (int)div_by((uint32_t)R, a.by_group), j = R - i * a.group;
    const int64_t head = (int64_t)(it.q0 + i) * a.t.q_heads + it.h * a.group + j;
    const float l = total[r], inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (ch < a.t.d) {  // d is a multiple of 8
      T y[4] = {from_f<T>(acc[c].x * inv), from_f<T>(acc[c].y * inv), from_f<T>(acc[c].z * inv), from_f<T>(acc[c].w * inv)};
      *(uint2*)((T*)a.t.out + head * a.t.d + ch) = *(const uint2*)y;
    }
    if (ch == 0 && a.t.lse) a.t.lse[head] = l == 0.0f ? -INFINITY : top[r] + log2f(l);
  }
}

// Launches the combine kernel right after an attention kernel on the stream.
template <typename T, int ROWS, int KT, int EXTRA>
int launch_combine(const Args& a, cudaStream_t st) {
  if (a.workers <= 1) return 0;
  return cuda_rc(launch_early(combine_kernel<T, ROWS, KT, EXTRA>, dim3((unsigned)a.workers, (ROWS + 15) / 16), COMBINE_THREADS,
                              4 * (size_t)(a.t.batch + 1), st, a));
}

}  // namespace tree
}  // namespace serving
}  // namespace ea
