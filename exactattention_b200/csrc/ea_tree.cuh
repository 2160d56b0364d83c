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
// unfinished. Layout of a slot: dp / 4 x ROWS x 4 floats (a row per thread stores and loads whole lines), ROWS maxima,
// ROWS sums.
__device__ __forceinline__ float* slot_of(const Args& a, int slot, int rows) {
  return (float*)a.t.workspace + (int64_t)slot * rows * (a.dp + 2);
}

// Kernel for more than 16 rows per kv head (ea_tree_tc.cu): 256-row items with `pair`, else 128-row ones.
constexpr int MANY_MAX_SEQS = 6000;  // what its shared memory has room for
int launch_many(const Args& a, bool pair, cudaStream_t st);

// Adds up the partials of the item that share blockIdx.x left unfinished, 16 rows a block (blockIdx.y). It starts
// while the attention kernel still runs (programmatic dependent launch) and finds its item meanwhile.
// Thread (share group, row, four channels): the groups take every G-th share, with all of a row's weights
// 2^(m - max) computed once; the groups' sums are joined in a fixed order.
constexpr int COMBINE_THREADS = 256, COMBINE_SHARES = 64;  // shares whose weights are held at a time

template <typename T, int ROWS, int KT>
__global__ void __launch_bounds__(COMBINE_THREADS) combine_kernel(Args a) {
  extern __shared__ uint32_t sums[];
  __shared__ uint64_t scratch[32];
  __shared__ float weight[COMBINE_SHARES][16], top[16], total[16];
  __shared__ float4 joined[COMBINE_THREADS];
  Schedule<ROWS, KT> sch;
  sch.build(a, sums, scratch);
  const int w = blockIdx.x, tid = threadIdx.x, r0 = blockIdx.y * 16;
  const uint32_t lo = sch.share(w), hi = sch.share(w + 1);
  Item it;
  int rows = 0, n = 2;  // rows of this block, shares of the item
  if (lo < hi) {
    it = sch.item(a, hi - 1, hi);
    const uint32_t begin = hi - 1 - it.kt0, end = begin + it.tiles;  // the item's units
    if (begin >= lo && end > hi) {                                   // begun here and not finished here
      rows = min(16, min(ROWS, it.new_tokens * a.group - it.m * ROWS) - r0);
      while (sch.share(w + n) < end) ++n;
    }
  }
  cudaGridDependencySynchronize();
  if (rows <= 0) return;
  // partial i of the item: slot 2 w + 1, then slots 2 (w + i)
  const auto part = [&](int i) { return slot_of(a, i ? 2 * (w + i) : 2 * w + 1, ROWS); };

  // maxima of the rows: 16 lanes a row
  {
    const int r = tid >> 4;
    float m = -INFINITY;
    if (r < rows)
      for (int i = tid & 15; i < n; i += 16) m = fmaxf(m, part(i)[ROWS * a.dp + r0 + r]);
#pragma unroll
    for (int o = 8; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((tid & 15) == 0) top[r] = m, total[r] = 0.0f;
  }
  const int vecs = a.dp / 4, cells = rows * vecs;  // at most 512: two cells a thread where there are many rows
  int groups = COMBINE_THREADS / cells;            // groups of threads that take every groups-th share
  if (groups < 1) groups = 1;
  const int grp = min(tid / cells, groups), cell0 = cells > COMBINE_THREADS ? tid : tid - tid / cells * cells;
  float4 acc[2] = {make_float4(0, 0, 0, 0), make_float4(0, 0, 0, 0)};
  for (int i0 = 0; i0 < n; i0 += COMBINE_SHARES) {
    const int m = min(COMBINE_SHARES, n - i0);
    __syncthreads();
    {
      const int r = tid >> 4;
      float l = 0.0f;
      if (r < rows) {
        const float base = top[r] == -INFINITY ? 0.0f : top[r];
        for (int i = tid & 15; i < m; i += 16) {
          const float* p = part(i0 + i) + ROWS * a.dp + r0 + r;
          const float f = exp2f(p[0] - base);
          weight[i][r] = f;
          l = fmaf(p[ROWS], f, l);
        }
      }
#pragma unroll
      for (int o = 8; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
      if ((tid & 15) == 0) total[r] += l;
    }
    __syncthreads();
    if (grp < groups)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int cell = cell0 + c * COMBINE_THREADS;
        if (cell >= cells) break;
        const int v = cell / rows, r = cell - v * rows, at = (v * ROWS + r0 + r) * 4;
#pragma unroll 4
        for (int i = grp; i < m; i += groups) {
          const float4 x = *(const float4*)(part(i0 + i) + at);
          const float f = weight[i][r];
          acc[c].x = fmaf(x.x, f, acc[c].x), acc[c].y = fmaf(x.y, f, acc[c].y);
          acc[c].z = fmaf(x.z, f, acc[c].z), acc[c].w = fmaf(x.w, f, acc[c].w);
        }
      }
  }
  if (groups > 1) {
    joined[tid] = acc[0];
    __syncthreads();
    if (tid < cells)
      for (int g = 1; g < groups; ++g) {
        const float4 x = joined[g * cells + tid];
        acc[0].x += x.x, acc[0].y += x.y, acc[0].z += x.z, acc[0].w += x.w;
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
template <typename T, int ROWS, int KT>
int launch_combine(const Args& a, cudaStream_t st) {
  if (a.workers <= 1) return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.workers, ROWS / 16), cfg.blockDim = dim3(COMBINE_THREADS);
  cfg.dynamicSmemBytes = 4 * (size_t)(a.t.batch + 1), cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr, cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, combine_kernel<T, ROWS, KT>, a);
  if (e == cudaSuccess) e = cudaGetLastError();
  return cuda_rc(e);
}

}  // namespace tree
}  // namespace serving
}  // namespace ea
