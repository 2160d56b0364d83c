// Penalties for repeated tokens, biases and grammar masks on logits (ea_process_logits_cuda).
//
// Bound by HBM: a row's logits are read once and written once. A block owns a chunk of one row's vocabulary. It
// streams the chunk through, setting what the mask forbids to -inf, and corrects the few tokens that penalties or
// biases change afterwards. Which these are is in a table of one 32-bit word per token of the chunk in shared memory,
// built from the row's history, path and bias list while the first logits are on their way:
//   bits 0-19 how often the token was generated, bits 20-30 which bias entry it has first
//   (EA_LOGITS_MAX_BIASES - entry, 0: none), bit 31 whether the prompt holds it.
// The words are integers, so the order of the atomics cannot change them. Whoever finds a token's word zero puts the
// token on a list, from which the corrections are then done with full warps (in place, lanes with and without a
// token in their part of the history took turns: 80 us for 256 rows of 131072 tokens with 4096 history entries). So the
// dense part reads no table, and the cost of the sparse part follows the lists' lengths. Rows without penalties
// and biases build no table.
#include "ea_serving.cuh"

namespace ea {
namespace serving {
namespace {

constexpr int THREADS = 512;
constexpr int UNROLL = 4;  // 16-byte pieces a thread has in flight
constexpr int BATCH = 8;   // history entries of a thread at a time
constexpr uint32_t COUNT = 0xFFFFFu, PROMPT = 0x80000000u;
constexpr int CODE_SHIFT = 20;

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

struct Row {
  float rep, freq, pres;
  const int32_t* ids;
  const float* vals;
  bool dup;
};

// The row's rule for one token whose table word is not zero.
__device__ __forceinline__ float adjust(float x, uint32_t w, int token, const Row& r, int num_biases) {
  const uint32_t cnt = w & COUNT, code = (w >> CODE_SHIFT) & 0x7FFu;
  if (cnt || (w & PROMPT)) x = x > 0.0f ? __fdiv_rn(x, r.rep) : __fmul_rn(x, r.rep);
  x = __fsub_rn(x, __fmul_rn(r.freq, (float)cnt));
  if (cnt) x = __fsub_rn(x, r.pres);
  if (code) {
    int e = EA_LOGITS_MAX_BIASES - (int)code;
    x = __fadd_rn(x, r.vals[e]);
    if (r.dup)
      for (++e; e < num_biases; ++e)
        if (r.ids[e] == token) x = __fadd_rn(x, r.vals[e]);
  }
  return x;
}

template <typename T, int VEC>
__global__ void __launch_bounds__(THREADS, 2) logits_kernel(ea_process_logits_t a, int chunk, FastDiv by_chunks,
                                                            int chunks) {
  using P = Pack<T, VEC>;
  extern __shared__ uint4 table4[];
  uint32_t* table = (uint32_t*)table4;
  uint16_t* list = (uint16_t*)(table + chunk);  // tokens with a nonzero word
  __shared__ int dup, listed;
  const int tid = threadIdx.x;
  const int64_t row = div_by(blockIdx.x, by_chunks);
  const int part = (int)(blockIdx.x - row * chunks);
  const T* src = (const T*)a.logits + row * a.logits_stride;
  T* dst = (T*)a.out + row * a.out_stride;
  // Pieces are aligned in memory: place i of the chunk is token v0 + i, and the row's first piece may
  // begin before its first token.
  const int mis = (int)(((uintptr_t)src / sizeof(T)) % VEC);
  const int v0 = part * chunk - mis;
  if (v0 >= a.vocab) return;

  P x[UNROLL];
#pragma unroll
  for (int j = 0; j < UNROLL; ++j) {
    const int i = (j * THREADS + tid) * VEC, v = v0 + i;
    if (i < chunk && v >= 0 && v + VEC <= a.vocab) x[j] = *(const P*)(src + v);
  }

  const int b = a.row_seq ? a.row_seq[row] : (int)row;
  const bool real = b >= 0 && b < a.batch;
  const int m = a.allowed_bits && real ? (a.mask_rows ? a.mask_rows[row] : (int)row) : -1;
  const uint32_t* bits = m >= 0 && m < a.num_masks ? (const uint32_t*)a.allowed_bits + m * a.mask_stride : nullptr;
  Row r;
  r.rep = real && a.repetition ? a.repetition[b] : 1.0f;
  r.freq = real && a.frequency ? a.frequency[b] : 0.0f;
  r.pres = real && a.presence ? a.presence[b] : 0.0f;
  const bool counts = real && (r.rep != 1.0f || r.freq != 0.0f || r.pres != 0.0f) && (a.history || a.draft_tokens);
  const bool biased = real && a.num_biases > 0;
  const bool tabled = counts || biased;
  // the chunk's tokens, and the lists: history, path (drafted tokens), biases
  const uint32_t lo = (uint32_t)max(v0, 0), span = (uint32_t)(min(a.vocab, v0 + chunk)) - lo;
  int n_hist = 0, n_prompt = 0, n_path = 0;
  const int32_t *hist = nullptr, *path = nullptr;
  const uint32_t* seen = nullptr;
  bool hist4 = false;
  uint32_t tok[BATCH];  // places in the chunk of the thread's first history entries (>= span: elsewhere)
  // entries first + 4 (512 j + tid) + 0 .. 3, j = 0, 1
  const auto fetch = [&](int first) {
#pragma unroll
    for (int j = 0; j < BATCH / 4; ++j) {
      const int i = first + 4 * (j * THREADS + tid);
      int4 h = make_int4(-1, -1, -1, -1);
      if (hist4 && i + 4 <= a.max_history) {
        h = *(const int4*)(hist + i);
      } else {
        if (i < a.max_history) h.x = hist[i];
        if (i + 1 < a.max_history) h.y = hist[i + 1];
        if (i + 2 < a.max_history) h.z = hist[i + 2];
        if (i + 3 < a.max_history) h.w = hist[i + 3];
      }
      tok[4 * j] = (uint32_t)h.x - lo, tok[4 * j + 1] = (uint32_t)h.y - lo;
      tok[4 * j + 2] = (uint32_t)h.z - lo, tok[4 * j + 3] = (uint32_t)h.w - lo;
    }
  };
  const auto entry = [&](int first, int e) { return first + 4 * ((e >> 2) * THREADS + tid) + (e & 3); };
  // puts a token on the list if its word was zero before
  const auto touch = [&](uint32_t t, uint32_t before) {
    if (before) return;
    const uint32_t together = __activemask(), below = together & ((1u << (tid & 31)) - 1);
    int at = 0;
    if (!below) at = atomicAdd(&listed, __popc(together));
    at = __shfl_sync(together, at, __ffs(together) - 1);
    list[at + __popc(below)] = (uint16_t)t;
  };
  if (tabled) {
    if (counts && a.history) {
      hist = a.history + (int64_t)b * a.history_stride;
      hist4 = ((uintptr_t)hist & 15) == 0;
      fetch(0);
      n_hist = min(max(a.history_lens[b], 0), a.max_history);
      n_prompt = a.prompt_lens ? min(max(a.prompt_lens[b], 0), n_hist) : 0;
    }
    if (counts && a.draft_tokens) {
      const int64_t q0 = a.q_start[b], q1 = min((int64_t)a.q_start[b + 1], a.rows);
      if (q0 >= 0 && q0 < q1) {
        n_path = (int)min(min(q1 - q0, (int64_t)(a.tree_mask ? a.tree_words * 32 : row - q0 + 1)), (int64_t)EA_LOGITS_MAX_PATH);
        path = a.draft_tokens + q0;
        if (a.tree_mask) seen = (const uint32_t*)a.tree_mask + row * a.tree_words;
      }
    }
    r.ids = a.bias_ids + (int64_t)b * a.num_biases;
    r.vals = a.bias_values + (int64_t)b * a.num_biases;
    for (int i = tid; i < (int)(span + 3) / 4; i += THREADS) table4[i] = make_uint4(0, 0, 0, 0);
    if (tid == 0) dup = listed = 0;
    __syncthreads();
    for (int first = 0; first < n_hist; first += BATCH * THREADS) {
      if (first) fetch(first);
#pragma unroll
      for (int e = 0; e < BATCH; ++e) {
        const int i = entry(first, e);
        if (tok[e] < span && i < n_hist) {
          touch(tok[e], i < n_prompt ? atomicOr(table + tok[e], PROMPT) : atomicAdd(table + tok[e], 1u));
        }
      }
    }
    for (int j = tid; j < n_path; j += THREADS) {
      if (seen && !((seen[j >> 5] >> (j & 31)) & 1)) continue;
      const uint32_t t = (uint32_t)path[j] - lo;
      if (t < span) touch(t, atomicAdd(table + t, 1u));
    }
    __syncthreads();
    if (biased) {
      for (int e = tid; e < a.num_biases; e += THREADS) {
        const uint32_t t = (uint32_t)r.ids[e] - lo;
        if (t < span) {
          const uint32_t code = (uint32_t)(EA_LOGITS_MAX_BIASES - e) << CODE_SHIFT;
          const uint32_t old = atomicMax(table + t, (table[t] & (PROMPT | COUNT)) | code);
          if ((old >> CODE_SHIFT) & 0x7FFu) dup = 1;
          touch(t, old);
        }
      }
    }
  }

  for (int i0 = 0; i0 < chunk; i0 += UNROLL * THREADS * VEC) {
    if (i0) {
#pragma unroll
      for (int j = 0; j < UNROLL; ++j) {
        const int i = i0 + (j * THREADS + tid) * VEC, v = v0 + i;
        if (i < chunk && v >= 0 && v + VEC <= a.vocab) x[j] = *(const P*)(src + v);
      }
    }
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      const int i = i0 + (j * THREADS + tid) * VEC, v = v0 + i;
      if (i >= chunk || v >= a.vocab || v + VEC <= 0) continue;
      const bool whole = v >= 0 && v + VEC <= a.vocab;
      if (!whole) {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (v + e >= 0 && v + e < a.vocab) x[j].v[e] = src[v + e];
      }
      if (bits) {
        // bit e of `no`: token v + e is forbidden; the piece may lie in two words
        const int first = max(v, 0), last = min(v + VEC, a.vocab) - 1;
        uint32_t no = ~__funnelshift_r(bits[first >> 5], bits[last >> 5], first & 31) << (first - v);
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
  if (!tabled) return;

  __syncthreads();  // the chunk is written and the table complete
  r.dup = dup != 0;
  for (int i = tid; i < listed; i += THREADS) {
    const uint32_t t = list[i];
    const int v = (int)(lo + t);
    if (bits && !((bits[v >> 5] >> (v & 31)) & 1)) continue;
    dst[v] = from_f<T>(adjust(to_f(src[v]), table[t], v, r, a.num_biases));
  }
}

template <typename T, int VEC>
int launch(const ea_process_logits_t& a, cudaStream_t st) {
  // The largest chunk whose blocks still fill the GPU twice: fewer chunks read the history less often.
  int chunk = 16384;
  while (chunk > 2048 && a.rows * ((a.vocab + chunk - 1) / chunk) < 2 * sm_count()) chunk >>= 1;
  const int chunks = (int)(((int64_t)a.vocab + VEC - 1 + chunk - 1) / chunk);
  chunk = (int)((((int64_t)a.vocab + VEC - 1 + chunks - 1) / chunks + 15) & ~15ll);  // equal chunks
  const int64_t blocks = a.rows * chunks;
  if (blocks > 0x7FFFFFFF) return fail(-1, "process_logits: too many rows");
  const size_t smem = (size_t)chunk * 6;
  static bool ready[64];  // per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !ready[dev])) {
    e = cudaFuncSetAttribute(logits_kernel<T, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, 6 * 16400);
    if (e == cudaSuccess && dev < 64) ready[dev] = true;
  }
  if (e != cudaSuccess) return cuda_rc(e);
  logits_kernel<T, VEC><<<(unsigned)blocks, THREADS, smem, st>>>(a, chunk, fast_div((uint32_t)chunks), chunks);
  return cuda_rc(cudaGetLastError());
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
