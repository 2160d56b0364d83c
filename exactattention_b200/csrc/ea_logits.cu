// Penalties for repeated tokens, biases and grammar masks on logits (ea_process_logits_cuda).
//
// Bound by HBM: a row's logits are read once and written once. Two kernels:
//   dense_kernel   streams every row through, setting what its grammar mask forbids to -inf;
//   sparse_kernel  a block a row: collects the tokens that penalties or biases change in a hash table in shared
//                  memory and corrects those tokens of the output. Its table is built while the dense kernel drains
//                  (programmatic dependent launch); only the corrections wait for it.
// One kernel with a table of counts beside each chunk of the vocabulary was measured first: 68 us against 35 us for
// 256 rows of 131072 16-bit logits with 4096 history entries, because every chunk scans the whole history and lanes
// with and without a token take turns.
// A table entry's word: bits 0-19 how often the token was generated, bits 20-30 which bias entry it has first
// (EA_LOGITS_MAX_BIASES - entry, 0: none), bit 31 whether the prompt holds it. The words are integers, so the order of
// the atomics cannot change them.
#include "ea_serving.cuh"

namespace ea {
namespace serving {
namespace {

constexpr int DENSE_THREADS = 256, UNROLL = 4;  // 16-byte pieces a thread has in flight
constexpr int SPARSE_THREADS = 512, BATCH = 8;  // entries a thread works on at a time
constexpr int MAX_SLOTS = 16384, FILL = 12288;  // table entries, and how many tokens one pass puts into them
constexpr uint32_t COUNT = 0xFFFFFu, PROMPT = 0x80000000u;
constexpr int CODE_SHIFT = 20;

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

// The row's mask bits, nullptr where every token is allowed.
__device__ __forceinline__ const uint32_t* mask_of(const ea_process_logits_t& a, int64_t row) {
  if (!a.allowed_bits) return nullptr;
  const int b = a.row_seq ? a.row_seq[row] : (int)row;
  const int m = a.mask_rows ? a.mask_rows[row] : (int)row;
  return b >= 0 && b < a.batch && m >= 0 && m < a.num_masks ? (const uint32_t*)a.allowed_bits + m * a.mask_stride : nullptr;
}

// Thread `tid` of `threads` streams pieces tid, tid + threads, .. (UNROLL of them) of a row from piece `first` on.
template <typename T, int VEC>
__device__ __forceinline__ void stream_row(const ea_process_logits_t& a, int64_t row, const uint32_t* bits, int first, int tid,
                                           int threads) {
  using P = Pack<T, VEC>;
  const T* src = (const T*)a.logits + row * a.logits_stride;
  T* dst = (T*)a.out + row * a.out_stride;
  // Pieces are aligned in memory, so the row's first one may begin before its first token.
  const int v0 = (first + tid) * VEC - (int)(((uintptr_t)src / sizeof(T)) % VEC);
  P x[UNROLL];
#pragma unroll
  for (int j = 0; j < UNROLL; ++j) {
    const int v = v0 + j * threads * VEC;
    if (v >= 0 && v + VEC <= a.vocab) x[j] = *(const P*)(src + v);
  }
#pragma unroll
  for (int j = 0; j < UNROLL; ++j) {
    const int v = v0 + j * threads * VEC;
    if (v >= a.vocab || v + VEC <= 0) continue;
    const bool whole = v >= 0 && v + VEC <= a.vocab;
    if (!whole) {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (v + e >= 0 && v + e < a.vocab) x[j].v[e] = src[v + e];
    }
    if (bits) {
      // bit e of `no`: token v + e is forbidden; the piece may lie in two words
      const int lo = max(v, 0), hi = min(v + VEC, a.vocab) - 1;
      const uint32_t no = ~__funnelshift_r(bits[lo >> 5], bits[hi >> 5], lo & 31) << (lo - v);
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if ((no >> e) & 1) x[j].v[e] = from_f<T>(-INFINITY);
    }
    if (whole) {
      *(P*)(dst + v) = x[j];
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (v + e >= 0 && v + e < a.vocab) dst[v + e] = x[j].v[e];
    }
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(DENSE_THREADS) dense_kernel(ea_process_logits_t a, FastDiv by_chunks, int chunks) {
  cudaTriggerProgrammaticLaunchCompletion();
  const int64_t row = div_by(blockIdx.x, by_chunks);
  const int part = (int)(blockIdx.x - row * chunks);
  stream_row<T, VEC>(a, row, mask_of(a, row), part * UNROLL * DENSE_THREADS, threadIdx.x, DENSE_THREADS);
}

// VEC 0: the dense kernel has written the rows; else this block streams its row itself.
template <typename T, int VEC>
__global__ void __launch_bounds__(SPARSE_THREADS) sparse_kernel(ea_process_logits_t a, int slots, int shift) {
  extern __shared__ uint32_t keys[];  // token + 1, 0: free; then the words
  uint32_t* words = keys + slots;
  __shared__ int dup;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const int b = a.row_seq ? a.row_seq[row] : (int)row;
  const bool real = b >= 0 && b < a.batch;
  // the first history entries, asked for before their number is known
  const int32_t* hist = a.history ? a.history + (int64_t)(real ? b : 0) * a.history_stride : nullptr;
  uint32_t tok[BATCH];
  const auto fetch = [&](int first, int n) {
#pragma unroll
    for (int e = 0; e < BATCH; ++e) {
      const int i = first + e * SPARSE_THREADS + tid;
      tok[e] = i < n ? (uint32_t)hist[i] : 0xFFFFFFFFu;
    }
  };
  if (real && hist) fetch(0, a.max_history);
  const uint32_t* bits = mask_of(a, row);
  const float rep = real && a.repetition ? a.repetition[b] : 1.0f, freq = real && a.frequency ? a.frequency[b] : 0.0f,
              pres = real && a.presence ? a.presence[b] : 0.0f;
  const bool counts = rep != 1.0f || freq != 0.0f || pres != 0.0f;
  // the lists: history, path (drafted tokens), biases
  const int n_hist = counts && hist ? min(max(a.history_lens[b], 0), a.max_history) : 0;
  const int n_prompt = n_hist && a.prompt_lens ? min(max(a.prompt_lens[b], 0), n_hist) : 0;
  int n_path = 0;
  const int32_t* path = nullptr;
  if (counts && a.draft_tokens) {
    const int64_t q0 = a.q_start[b], q1 = min((int64_t)a.q_start[b + 1], a.rows);
    if (q0 >= 0 && q0 < q1) {
      n_path = (int)max(min(min(q1 - q0, (int64_t)EA_LOGITS_MAX_PATH), a.tree_mask ? (int64_t)a.tree_words * 32 : row - q0 + 1), (int64_t)0);
      path = a.draft_tokens + q0;
    }
  }
  const uint32_t* seen = a.tree_mask ? (const uint32_t*)a.tree_mask + row * a.tree_words : nullptr;
  const int n_bias = real ? a.num_biases : 0;
  const int32_t* ids = a.bias_ids + (int64_t)b * n_bias;
  const float* vals = a.bias_values + (int64_t)b * n_bias;
  const int64_t all = (int64_t)n_hist + n_path + n_bias;
  if (VEC == 0 && all == 0) {
    cudaGridDependencySynchronize();  // nothing after this kernel may overtake the dense one
    return;
  }
  // One pass where the lists fit; else as many as the vocabulary needs, pass p taking the tokens that are p modulo
  // their number, so that no pass can overfill the table.
  const uint32_t vocab = (uint32_t)a.vocab, passes = all <= slots / 4 * 3 ? 1u : (vocab + FILL - 1) / FILL;
  const auto slot_of = [&](uint32_t t) -> uint32_t* {
    for (uint32_t h = (t * 2654435761u) >> shift;; h = (h + 1) & (uint32_t)(slots - 1)) {
      uint32_t k = keys[h];
      if (k == 0) k = atomicCAS(keys + h, 0u, t + 1);
      if (k == 0 || k == t + 1) return words + h;
    }
  };
  for (uint32_t pass = 0; pass < passes; ++pass) {
    const auto mine = [&](uint32_t t) { return t < vocab && (passes == 1 || t % passes == pass); };
    for (int i = tid; i < slots / 2; i += SPARSE_THREADS) ((uint4*)keys)[i] = make_uint4(0, 0, 0, 0);
    if (tid == 0) dup = 0;
    __syncthreads();
    for (int first = 0; first < n_hist; first += BATCH * SPARSE_THREADS) {
      if (first || pass) fetch(first, n_hist);
#pragma unroll
      for (int e = 0; e < BATCH; ++e) {
        const int i = first + e * SPARSE_THREADS + tid;
        if (i >= n_hist || !mine(tok[e])) continue;
        if (i < n_prompt) atomicOr(slot_of(tok[e]), PROMPT);
        else atomicAdd(slot_of(tok[e]), 1u);
      }
    }
    for (int j = tid; j < n_path; j += SPARSE_THREADS) {
      if (seen && !((seen[j >> 5] >> (j & 31)) & 1)) continue;
      const uint32_t t = (uint32_t)path[j];
      if (mine(t)) atomicAdd(slot_of(t), 1u);
    }
    __syncthreads();
    for (int e = tid; e < n_bias; e += SPARSE_THREADS) {
      const uint32_t t = (uint32_t)ids[e];
      if (!mine(t)) continue;
      uint32_t* w = slot_of(t);
      const uint32_t old = atomicMax(w, (*w & (PROMPT | COUNT)) | (uint32_t)(EA_LOGITS_MAX_BIASES - e) << CODE_SHIFT);
      if ((old >> CODE_SHIFT) & 0x7FFu) dup = 1;
    }
    __syncthreads();
    // values and mask words of up to BATCH entries a thread at a time
    for (int i0 = tid; i0 < slots; i0 += BATCH * SPARSE_THREADS) {
      T old[BATCH];
      uint32_t mask[BATCH];
#pragma unroll
      for (int e = 0; e < BATCH; ++e) {
        const int i = i0 + e * SPARSE_THREADS;
        tok[e] = i < slots ? keys[i] : 0;
        mask[e] = 0xFFFFFFFFu;
        if (tok[e]) {
          const uint32_t t = tok[e] - 1;
          old[e] = ((const T*)a.logits)[row * a.logits_stride + t];
          if (bits) mask[e] = bits[t >> 5];
        }
      }
      if (pass == 0 && i0 == tid) {  // the row is written
        if constexpr (VEC == 0) cudaGridDependencySynchronize();
        else {
          const int pieces = (int)((vocab + 2 * VEC - 2) / VEC);
          for (int first = 0; first < pieces; first += UNROLL * SPARSE_THREADS)
            stream_row<T, VEC>(a, row, bits, first, tid, SPARSE_THREADS);
          __syncthreads();
        }
      }
#pragma unroll
      for (int e = 0; e < BATCH; ++e) {
        const uint32_t t = tok[e] - 1;
        if (!tok[e] || !((mask[e] >> (t & 31)) & 1)) continue;
        const uint32_t w = words[i0 + e * SPARSE_THREADS], cnt = w & COUNT, code = (w >> CODE_SHIFT) & 0x7FFu;
        float x = to_f(old[e]);
        if (cnt || (w & PROMPT)) x = x > 0.0f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
        x = __fsub_rn(x, __fmul_rn(freq, (float)cnt));
        if (cnt) x = __fsub_rn(x, pres);
        if (code) {
          int f = EA_LOGITS_MAX_BIASES - (int)code;
          x = __fadd_rn(x, vals[f]);
          if (dup)
            for (++f; f < n_bias; ++f)
              if ((uint32_t)ids[f] == t) x = __fadd_rn(x, vals[f]);
        }
        ((T*)a.out)[row * a.out_stride + t] = from_f<T>(x);
      }
    }
    __syncthreads();
  }
}

template <typename T, int VEC>
int launch(const ea_process_logits_t& a, cudaStream_t st) {
  const bool counts = (a.repetition || a.frequency || a.presence) && (a.history || a.draft_tokens);
  const bool sparse = counts || a.num_biases, dense = a.allowed_bits || a.out != a.logits;
  // Few short rows: a block that streams its row before it corrects it saves the second launch (6 us against 9 us for one
  // row of 32000 tokens).
  const bool together = sparse && dense && a.rows <= sm_count() && a.vocab <= 3 * UNROLL * SPARSE_THREADS * VEC;
  if (dense && !together) {
    const int per_block = UNROLL * DENSE_THREADS * VEC;
    const int chunks = (int)(((int64_t)a.vocab + VEC - 1 + per_block - 1) / per_block);
    const int64_t blocks = a.rows * chunks;
    if (blocks >= (1ll << 31)) return fail(-1, "process_logits: too many rows");
    dense_kernel<T, VEC><<<(unsigned)blocks, DENSE_THREADS, 0, st>>>(a, fast_div((uint32_t)chunks), chunks);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_rc(e);
  }
  if (!sparse) return 0;
  // table: four thirds of the longest lists the sizes allow, at most MAX_SLOTS (then several passes)
  const int64_t longest = (int64_t)a.max_history + a.num_biases + (a.draft_tokens ? (a.tree_mask ? a.tree_words * 32 : 1024) : 0);
  int log2 = 10;
  while ((1 << log2) < MAX_SLOTS && (1 << log2) / 4 * 3 < longest) ++log2;
  const int slots = 1 << log2;
  const auto kernel = together ? sparse_kernel<T, VEC> : sparse_kernel<T, 0>;
  static bool ready[2][64];  // per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !ready[together][dev])) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SLOTS * 8);
    if (e == cudaSuccess && dev < 64) ready[together][dev] = true;
  }
  if (e != cudaSuccess) return cuda_rc(e);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.rows), cfg.blockDim = dim3(SPARSE_THREADS), cfg.dynamicSmemBytes = (size_t)slots * 8;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr, cfg.numAttrs = dense && !together ? 1 : 0;  // after the dense kernel only
  e = cudaLaunchKernelEx(&cfg, kernel, a, slots, 32 - log2);
  if (e == cudaSuccess) e = cudaGetLastError();
  return cuda_rc(e);
}

template <typename T>
int launch_type(const ea_process_logits_t& a, cudaStream_t st) {
  constexpr int VEC = 16 / (int)sizeof(T);
  // 16-byte pieces where input and output rows are equally far from a 16-byte boundary
  const bool same = ((uintptr_t)a.logits - (uintptr_t)a.out) % 16 == 0 &&
                    (a.rows <= 1 || (a.logits_stride - a.out_stride) % VEC == 0);
  return same ? launch<T, VEC>(a, st) : launch<T, 1>(a, st);
}

}  // namespace
}  // namespace serving
}  // namespace ea

extern "C" int ea_process_logits_cuda(const ea_process_logits_t* a, void* stream) {
  using namespace ea::serving;
  if (!a || a->rows < 0 || a->vocab < 0 || a->batch < 0 || a->max_history < 0 || a->num_biases < 0 || a->num_masks < 0 ||
      a->tree_words < 0)
    return fail(-1, "process_logits: negative size");
  if (a->max_history > EA_LOGITS_MAX_HISTORY || a->num_biases > EA_LOGITS_MAX_BIASES || a->vocab > (1 << 30))
    return fail(-1, "process_logits: history, biases or vocabulary above their limits");
  if (a->rows == 0 || a->vocab == 0) return 0;
  if (!a->logits || !a->out || (a->history && !a->history_lens) || (a->num_biases && (!a->bias_ids || !a->bias_values)) ||
      (a->draft_tokens && !a->q_start))
    return fail(-1, "process_logits: a required pointer is NULL");
  cudaStream_t st = (cudaStream_t)stream;
  switch (a->dtype) {
    case EA_BF16: return launch_type<__nv_bfloat16>(*a, st);
    case EA_FP16: return launch_type<__half>(*a, st);
    case EA_FP32: return launch_type<float>(*a, st);
  }
  return fail(-9, "process_logits: unknown element type");
}
