// Penalties for repeated tokens, biases and grammar masks on logits (ea_process_logits_cuda).
//
// Bound by HBM: a row's logits are read once and written once; what the grammar mask forbids becomes -inf on the way, and
// the few tokens that penalties or biases change are corrected afterwards. Which these are is kept in 32-bit words:
//   bits 0-19 how often the token was generated, bits 20-30 which bias entry it has first
//   (EA_LOGITS_MAX_BIASES - entry, 0: none), bit 31 whether the prompt holds it.
// The words are integers, so the order of the atomics cannot change them. Who finds a word (or a table entry) fresh
// puts it on a list, from which the corrections are done with full warps.
//   Many rows: dense_kernel streams all rows through; sparse_kernel, a block a row, collects the row's history, path and
//   biases in a hash table in shared memory and corrects their tokens. It is launched to start while the dense kernel
//   drains; only its stores wait for it.
//   Few rows (up to four blocks for every SM): chunk_kernel alone, with a word for every token of its chunk of the row's
//   vocabulary; every chunk reads the whole history, which is cheaper than a second launch (6 us against 13 us for one
//   row of 32000 tokens).
// Measured otherwise for 256 rows of 131072 16-bit logits with 4096 history entries: the chunk kernel for all 68 us; with
// a cluster of blocks sharing the scan through distributed shared memory 99 us; with a kernel before it that sorts
// every row's history by chunk 60 us; dense and sparse kernel 54 us, of which the dense one alone takes 23 us. With the
// dense kernel as one wave that leaves room for the sparse one's blocks from the start they take 71 to 85 us together: the
// scattered reads get into the way of the stream. An atomic for every new list entry instead of one a warp: 56 us.
#include <type_traits>

#include "ea_serving.cuh"

namespace ea {
namespace serving {
namespace {

constexpr int THREADS = 512;        // of the chunk and the sparse kernel
constexpr int DENSE_THREADS = 256;
constexpr int UNROLL = 4;           // 16-byte pieces a thread has in flight
constexpr int BATCH = 8;            // history entries a thread asks for at a time
constexpr int LIST = 4096;          // tokens a chunk lists; more: its table is searched
constexpr int MAX_CHUNK = 16384 + 16;
constexpr int MAX_SLOTS = 16384;    // entries of a hash table
constexpr uint32_t COUNT = 0xFFFFFu, PROMPT = 0x80000000u;
constexpr int CODE_SHIFT = 20;

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

// -inf in the elements whose bit of `no` is set
template <typename T, int VEC>
__device__ __forceinline__ void forbid(Pack<T, VEC>& p, uint32_t no) {
  if constexpr (sizeof(T) == 2 && VEC == 8) {
    constexpr uint32_t INF2 = std::is_same<T, __half>::value ? 0xFC00FC00u : 0xFF80FF80u;
    uint32_t* w = (uint32_t*)&p;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // four bits to four bytes of 0 or 255, then every byte twice
      const uint32_t b = (((no >> 4 * h & 15u) * 0x00204081u) & 0x01010101u) * 255u;
      const uint32_t m0 = __byte_perm(b, 0, 0x1100), m1 = __byte_perm(b, 0, 0x3322);
      w[2 * h] = (w[2 * h] & ~m0) | (INF2 & m0);
      w[2 * h + 1] = (w[2 * h + 1] & ~m1) | (INF2 & m1);
    }
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if ((no >> e) & 1) p.v[e] = from_f<T>(-INFINITY);
  }
}

// A row's sequence and lists.
struct Row {
  int b, n_hist, n_prompt, n_path;
  bool counts;  // history and path matter
  float rep, freq, pres;
  const int32_t *hist, *path;
  const uint32_t* seen;  // path members, nullptr: all
};
__device__ __forceinline__ Row row_of(const ea_process_logits_t& a, int64_t row) {
  Row r;
  const int b = a.row_seq ? a.row_seq[row] : (int)row;
  r.b = b >= 0 && b < a.batch ? b : -1;
  r.rep = r.b >= 0 && a.repetition ? a.repetition[b] : 1.0f;
  r.freq = r.b >= 0 && a.frequency ? a.frequency[b] : 0.0f;
  r.pres = r.b >= 0 && a.presence ? a.presence[b] : 0.0f;
  r.counts = r.b >= 0 && (r.rep != 1.0f || r.freq != 0.0f || r.pres != 0.0f) && (a.history || a.draft_tokens);
  r.n_hist = r.n_prompt = r.n_path = 0;
  r.hist = r.path = nullptr, r.seen = nullptr;
  if (!r.counts) return r;
  if (a.history) {
    r.hist = a.history + (int64_t)b * a.history_stride;
    r.n_hist = min(max(a.history_lens[b], 0), a.max_history);
    r.n_prompt = a.prompt_lens ? min(max(a.prompt_lens[b], 0), r.n_hist) : 0;
  }
  if (a.draft_tokens) {
    const int64_t q0 = a.q_start[b], q1 = min((int64_t)a.q_start[b + 1], a.rows);
    if (q0 >= 0 && q0 < q1) {
      const int64_t most = a.tree_mask ? (int64_t)a.tree_words * 32 : row - q0 + 1;
      r.n_path = (int)max(min(min(q1 - q0, (int64_t)EA_LOGITS_MAX_PATH), most), (int64_t)0);
      r.path = a.draft_tokens + q0;
      if (a.tree_mask) r.seen = (const uint32_t*)a.tree_mask + row * a.tree_words;
    }
  }
  return r;
}
// Token j of the lists: history, then path; EMPTY where there is none or the path leaves it out.
constexpr uint32_t EMPTY = 0xFFFFFFFFu;
__device__ __forceinline__ uint32_t token_of(const Row& r, int j) {
  if (j < r.n_hist) return (uint32_t)r.hist[j];
  j -= r.n_hist;
  if (j >= r.n_path || (r.seen && !((r.seen[j >> 5] >> (j & 31)) & 1))) return EMPTY;
  return (uint32_t)r.path[j];
}
template <typename T, int VEC>
__device__ __forceinline__ int misalignment(const ea_process_logits_t& a, int64_t row) {
  return (int)(((uintptr_t)((const T*)a.logits + row * a.logits_stride) / sizeof(T)) % VEC);
}

// The row's mask bits, nullptr where every token is allowed.
__device__ __forceinline__ const uint32_t* mask_of(const ea_process_logits_t& a, int64_t row, bool real) {
  const int m = a.allowed_bits && real ? (a.mask_rows ? a.mask_rows[row] : (int)row) : -1;
  return m >= 0 && m < a.num_masks ? (const uint32_t*)a.allowed_bits + m * a.mask_stride : nullptr;
}
// The logit of a token whose word is not zero.
__device__ __forceinline__ float adjust(float x, uint32_t w, uint32_t token, const Row& r, const int32_t* ids, const float* vals,
                                        int n_bias, bool dup) {
  const uint32_t cnt = w & COUNT, code = (w >> CODE_SHIFT) & 0x7FFu;
  if (cnt || (w & PROMPT)) x = x > 0.0f ? __fdiv_rn(x, r.rep) : __fmul_rn(x, r.rep);
  x = __fsub_rn(x, __fmul_rn(r.freq, (float)cnt));
  if (cnt) x = __fsub_rn(x, r.pres);
  if (code) {
    int e = EA_LOGITS_MAX_BIASES - (int)code;
    x = __fadd_rn(x, vals[e]);
    if (dup)
      for (++e; e < n_bias; ++e)
        if ((uint32_t)ids[e] == token) x = __fadd_rn(x, vals[e]);
  }
  return x;
}

template <typename T, int VEC>
__global__ void __launch_bounds__(DENSE_THREADS) dense_kernel(ea_process_logits_t a, int chunks, FastDiv by_chunks) {
  using P = Pack<T, VEC>;
  begin();
  const int64_t row = div_by(blockIdx.x, by_chunks);
  const int part = (int)(blockIdx.x - row * chunks);
  const T* src = (const T*)a.logits + row * a.logits_stride;
  T* dst = (T*)a.out + row * a.out_stride;
  // Pieces are aligned in memory, so the row's first one may begin before its first token.
  const int v0 = (part * UNROLL * DENSE_THREADS + (int)threadIdx.x) * VEC - misalignment<T, VEC>(a, row);
  P x[UNROLL];
#pragma unroll
  for (int j = 0; j < UNROLL; ++j) {
    const int v = v0 + j * DENSE_THREADS * VEC;
    if (v >= 0 && v + VEC <= a.vocab) x[j] = *(const P*)(src + v);
  }
  const int b = a.row_seq ? a.row_seq[row] : (int)row;
  const uint32_t* bits = mask_of(a, row, b >= 0 && b < a.batch);
#pragma unroll
  for (int j = 0; j < UNROLL; ++j) {
    const int v = v0 + j * DENSE_THREADS * VEC;
    if (v >= a.vocab || v + VEC <= 0) continue;
    const bool whole = v >= 0 && v + VEC <= a.vocab;
    if (!whole) {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (v + e >= 0 && v + e < a.vocab) x[j].v[e] = src[v + e];
    }
    if (bits) {
      // bit e: token v + e is allowed; the piece may lie in two words
      const int lo = max(v, 0), hi = min(v + VEC, a.vocab) - 1;
      forbid<T, VEC>(x[j], ~__funnelshift_r(bits[lo >> 5], bits[hi >> 5], lo & 31) << (lo - v));
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

template <typename T>
__global__ void __launch_bounds__(THREADS, 2) sparse_kernel(ea_process_logits_t a, int slots, int shift, bool alone) {
  if (alone) begin();
  extern __shared__ uint32_t keys[];  // token + 1, 0: free; then the words, then the list of used entries
  uint32_t* words = keys + slots;
  uint16_t* list = (uint16_t*)(words + slots);
  __shared__ int dup, listed;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const Row r = row_of(a, row);
  const uint32_t* bits = mask_of(a, row, r.b >= 0);
  const int n_bias = r.b >= 0 ? a.num_biases : 0, n = r.n_hist + r.n_path;
  const int32_t* ids = a.bias_ids + (int64_t)r.b * n_bias;
  const float* vals = a.bias_values + (int64_t)r.b * n_bias;
  const T* src = (const T*)a.logits + row * a.logits_stride;
  T* dst = (T*)a.out + row * a.out_stride;
  const uint32_t vocab = (uint32_t)a.vocab;
  if (n + n_bias == 0) {
    begin();  // nothing after this kernel may overtake the dense one
    return;
  }
  // One pass where the lists fit; else as many as the vocabulary needs, pass p taking the tokens that are p modulo
  // their number, so that no pass can overfill the table.
  const uint32_t fill = slots / 4 * 3, passes = n + n_bias <= (int)fill ? 1u : (vocab + fill - 1) / fill;
  // The entry of token t, and whether it is new. The table never fills up; the bound on the search is for safety.
  const auto entry_of = [&](uint32_t t, bool& fresh) -> uint32_t {
    uint32_t h = (t * 2654435761u) >> shift;
    for (int i = 0; i < slots; ++i, h = (h + 1) & (uint32_t)(slots - 1)) {
      uint32_t k = keys[h];
      if (k == 0) {
        k = atomicCAS(keys + h, 0u, t + 1);
        if (k == 0) {
          fresh = true;
          break;
        }
      }
      if (k == t + 1) break;
    }
    return h;
  };
  // Puts the new entries of a warp on the list, with one atomic for all of them.
  const auto append = [&](uint32_t h, bool fresh) {
    const uint32_t who = __ballot_sync(0xffffffffu, fresh);
    if (!who) return;
    int at = 0;
    if ((tid & 31) == 0) at = atomicAdd(&listed, __popc(who));
    at = __shfl_sync(0xffffffffu, at, 0) + __popc(who & ((1u << (tid & 31)) - 1));
    if (fresh) list[at] = (uint16_t)h;
  };
  for (uint32_t pass = 0; pass < passes; ++pass) {
    const auto mine = [&](uint32_t t) { return t < vocab && (passes == 1 || t % passes == pass); };
    for (int i = tid; i < slots / 2; i += THREADS) ((uint4*)keys)[i] = make_uint4(0, 0, 0, 0);
    if (tid == 0) dup = listed = 0;
    uint32_t tok[BATCH];
#pragma unroll
    for (int e = 0; e < BATCH; ++e) tok[e] = token_of(r, e * THREADS + tid);
    __syncthreads();
    for (int first = 0; first < n; first += BATCH * THREADS) {
      if (first) {
#pragma unroll
        for (int e = 0; e < BATCH; ++e) tok[e] = token_of(r, first + e * THREADS + tid);
      }
#pragma unroll
      for (int e = 0; e < BATCH; ++e) {
        uint32_t h = 0;
        bool fresh = false;
        if (mine(tok[e])) {
          h = entry_of(tok[e], fresh);
          if (first + e * THREADS + tid < r.n_prompt) atomicOr(words + h, PROMPT);
          else atomicAdd(words + h, 1u);
        }
        append(h, fresh);
      }
    }
    __syncthreads();
    for (int e0 = 0; e0 < n_bias; e0 += THREADS) {  // whole warps come here
      const int e = e0 + tid;
      const uint32_t t = e < n_bias ? (uint32_t)ids[e] : EMPTY;
      uint32_t h = 0;
      bool fresh = false;
      if (mine(t)) {
        h = entry_of(t, fresh);
        const uint32_t old = atomicMax(words + h, (words[h] & (PROMPT | COUNT)) | (uint32_t)(EA_LOGITS_MAX_BIASES - e) << CODE_SHIFT);
        if ((old >> CODE_SHIFT) & 0x7FFu) dup = 1;
      }
      append(h, fresh);
    }
    __syncthreads();
    const int used = listed;
    for (int first = 0; first < used; first += BATCH * THREADS) {
      T old[BATCH];
      uint32_t ok = 0;
#pragma unroll
      for (int e = 0; e < BATCH; ++e) {
        const int i = first + e * THREADS + tid;
        tok[e] = i < used ? list[i] : 0;
        if (i < used) {
          const uint32_t t = keys[tok[e]] - 1;
          old[e] = src[t];
          ok |= (bits ? (bits[t >> 5] >> (t & 31)) & 1u : 1u) << e;
        }
      }
      if (pass == 0 && first == 0) begin();  // the dense kernel's rows are written
#pragma unroll
      for (int e = 0; e < BATCH; ++e) {
        if (!((ok >> e) & 1)) continue;
        const uint32_t t = keys[tok[e]] - 1;
        dst[t] = from_f<T>(adjust(to_f(old[e]), words[tok[e]], t, r, ids, vals, n_bias, dup != 0));
      }
    }
    if (pass == 0 && used == 0) begin();
    __syncthreads();
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(THREADS, 2) chunk_kernel(ea_process_logits_t a, int chunk, int chunks, FastDiv by_chunks) {
  using P = Pack<T, VEC>;
  begin();
  extern __shared__ uint4 table4[];
  uint32_t* table = (uint32_t*)table4;
  __shared__ uint16_t list[LIST];
  __shared__ int dup, listed;
  const int tid = threadIdx.x;
  const int64_t row = div_by(blockIdx.x, by_chunks);
  const int part = (int)(blockIdx.x - row * chunks);
  const T* src = (const T*)a.logits + row * a.logits_stride;
  T* dst = (T*)a.out + row * a.out_stride;
  // Pieces are aligned in memory: place i of the chunk is token v0 + i, and the row's first piece may begin before its
  // first token.
  const int v0 = part * chunk - misalignment<T, VEC>(a, row);

  P x[UNROLL];
#pragma unroll
  for (int j = 0; j < UNROLL; ++j) {
    const int i = (j * THREADS + tid) * VEC, v = v0 + i;
    if (i < chunk && v >= 0 && v + VEC <= a.vocab) x[j] = *(const P*)(src + v);
  }

  const Row r = row_of(a, row);
  const uint32_t* bits = mask_of(a, row, r.b >= 0);
  const int n_bias = r.b >= 0 ? a.num_biases : 0;
  const bool tabled = r.counts || n_bias > 0;
  const int32_t* ids = a.bias_ids + (int64_t)r.b * n_bias;
  const float* vals = a.bias_values + (int64_t)r.b * n_bias;
  uint32_t id = tid < n_bias ? (uint32_t)ids[tid] : EMPTY;
  if (tabled) {
    for (int i = tid; i < chunk / 4; i += THREADS) table4[i] = make_uint4(0, 0, 0, 0);
    if (tid == 0) dup = listed = 0;
    __syncthreads();
  }
  // Puts a token on the list if its word was zero before.
  const auto touch = [&](uint32_t at, uint32_t before) {
    if (before) return;
    const int k = atomicAdd(&listed, 1);
    if (k < LIST) list[k] = (uint16_t)at;
  };
  if (r.counts) {
    const int n = r.n_hist + r.n_path;
#pragma unroll 4
    for (int j = tid; j < n; j += THREADS) {
      const uint32_t t = token_of(r, j), at = t - (uint32_t)v0;
      if (t < (uint32_t)a.vocab && at < (uint32_t)chunk)
        touch(at, j < r.n_prompt ? atomicOr(table + at, PROMPT) : atomicAdd(table + at, 1u));
    }
  }
  if (n_bias) {
    __syncthreads();  // the counts are complete
    for (int e = tid; e < n_bias; e += THREADS) {
      if (e != tid) id = (uint32_t)ids[e];
      const uint32_t t = id, at = t - (uint32_t)v0;
      if (t >= (uint32_t)a.vocab || at >= (uint32_t)chunk) continue;
      const uint32_t old = atomicMax(table + at, (table[at] & (PROMPT | COUNT)) | (uint32_t)(EA_LOGITS_MAX_BIASES - e) << CODE_SHIFT);
      if ((old >> CODE_SHIFT) & 0x7FFu) dup = 1;
      touch(at, old);
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
        // bit e: token v + e is allowed; the piece may lie in two words
        const int lo = max(v, 0), hi = min(v + VEC, a.vocab) - 1;
        forbid<T, VEC>(x[j], ~__funnelshift_r(bits[lo >> 5], bits[hi >> 5], lo & 31) << (lo - v));
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

  __syncthreads();  // the chunk is written, the table and its list are complete
  const bool search = listed > LIST;
  const int n = search ? chunk : listed;
  for (int i = tid; i < n; i += THREADS) {
    const int at = search ? i : list[i], v = v0 + at;
    const uint32_t w = table[at];
    if (!w || (bits && !((bits[v >> 5] >> (v & 31)) & 1))) continue;
    dst[v] = from_f<T>(adjust(to_f(src[v]), w, (uint32_t)v, r, ids, vals, n_bias, dup != 0));
  }
}

int vec_of(const ea_process_logits_t& a) {
  const int size = a.dtype == EA_FP32 ? 4 : 2, vec = 16 / size;
  // 16-byte pieces where input and output rows are equally far from a 16-byte boundary
  const bool same = ((uintptr_t)a.logits - (uintptr_t)a.out) % 16 == 0 &&
                    (a.rows <= 1 || (a.logits_stride - a.out_stride) % vec == 0);
  return same ? vec : 1;
}

// Room for `bytes` of dynamic shared memory, once per kernel and device.
template <auto kernel>
cudaError_t allow_smem(int bytes) {
  static bool ready[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && ready[dev])) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) ready[dev] = true;
  return e;
}

template <typename T, int VEC>
int launch(const ea_process_logits_t& a, cudaStream_t st) {
  const bool counts = (a.repetition || a.frequency || a.presence) && (a.history || a.draft_tokens);
  const bool sparse = counts || a.num_biases, dense = a.allowed_bits || a.out != a.logits;
  // a row's places: its tokens, and those before it in its first 16-byte piece
  const bool aligned = (uintptr_t)a.logits % 16 == 0 && (a.rows <= 1 || a.logits_stride * sizeof(T) % 16 == 0);
  const int64_t places = (int64_t)a.vocab + (aligned ? 0 : VEC - 1);
  cudaError_t e;
  int chunk = 16384;
  while (chunk > 2048 && a.rows * ((places + chunk - 1) / chunk) < 2 * sm_count()) chunk >>= 1;
  int64_t chunks = (places + chunk - 1) / chunk;
  if (sparse && a.rows * chunks <= 4 * sm_count()) {
    chunk = (int)(((places + chunks - 1) / chunks + 15) & ~15ll);
    if ((e = allow_smem<chunk_kernel<T, VEC>>(4 * MAX_CHUNK)) != cudaSuccess) return cuda_rc(e);
    return cuda_rc(launch_early(chunk_kernel<T, VEC>, (unsigned)(a.rows * chunks), THREADS, 4 * (size_t)chunk, st, a, chunk,
                                (int)chunks, fast_div((uint32_t)chunks)));
  }
  if (dense) {
    const int per_block = UNROLL * DENSE_THREADS * VEC;
    chunks = (places + per_block - 1) / per_block;
    if (a.rows * chunks >= (1ll << 31)) return fail(-1, "process_logits: too many rows");
    e = launch_early(dense_kernel<T, VEC>, (unsigned)(a.rows * chunks), DENSE_THREADS, 0, st, a, (int)chunks, fast_div((uint32_t)chunks));
    if (e != cudaSuccess) return cuda_rc(e);
  }
  if (!sparse) return 0;
  if (a.rows >= (1ll << 31)) return fail(-1, "process_logits: too many rows");
  // table: four thirds of the longest lists the sizes allow, at most MAX_SLOTS (then several passes)
  const int64_t longest = (int64_t)a.max_history + a.num_biases + (a.draft_tokens ? (a.tree_mask ? a.tree_words * 32 : 1024) : 0);
  int log2 = 10;
  while ((1 << log2) < MAX_SLOTS && (1 << log2) / 4 * 3 < longest) ++log2;
  if ((e = allow_smem<sparse_kernel<T>>(MAX_SLOTS * 10)) != cudaSuccess) return cuda_rc(e);
  // alone (in place, without masks) it has to wait for what is before it; behind the dense kernel that one has
  return cuda_rc(launch_early(sparse_kernel<T>, (unsigned)a.rows, THREADS, (size_t)10 << log2, st, a, 1 << log2, 32 - log2, !dense));
}

template <typename T>
int launch_type(const ea_process_logits_t& a, cudaStream_t st) {
  constexpr int VEC = 16 / (int)sizeof(T);
  return vec_of(a) == VEC ? launch<T, VEC>(a, st) : launch<T, 1>(a, st);
}

}  // namespace
}  // namespace serving
}  // namespace ea

extern "C" int ea_process_logits_cuda(const ea_process_logits_t* a, void* stream) {
  using namespace ea::serving;
  if (!a || a->rows < 0 || a->vocab < 0 || a->batch < 0 || a->max_history < 0 || a->num_biases < 0 || a->num_masks < 0 ||
      a->tree_words < 0)
    return fail(-1, "process_logits: negative size");
  if (a->batch > EA_LOGITS_MAX_SEQS || a->max_history > EA_LOGITS_MAX_HISTORY || a->num_biases > EA_LOGITS_MAX_BIASES || a->vocab > (1 << 30))
    return fail(-1, "process_logits: sequences, history, biases or vocabulary above their limits");
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
