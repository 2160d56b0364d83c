// Attention of a step's tokens over the paged cache (ea_tree_attention_cuda): the entry, and the kernel for
// few query rows per kv head.
//
// Row statistics (maximum, sum) and outputs are binary32. The kernel below keeps the query rows of one sequence and kv
// head (tokens x the heads of a group, 8 or 16) in registers as the narrow operand of 16 x 8 x 16 matrix instructions:
// keys are the M side of the scores, channels the M side of the outputs, rows the N side of both, so few rows
// cost few instructions. With rows on the M side two rows cost what sixteen do: 64 sequences of 4096 to 32768 keys,
// 2 rows, d = 128 took 776 us in bursts and 860 us in a long loop, where the 1000 W limit lowered the SM clock to 1.7 to
// 1.85 GHz; this way round takes 737 us and 790 us. Sixteen rows, which have the same products either way and turn
// their weights over on top, pay for it: 895 us before, 915 us now in a long loop (d = 128). A warp owns 16 of a tile's 64 keys with a running maximum, sum and output of its
// own, so the warps of a block stream their keys without waiting for one another and join once per item. Bound by HBM: a
// 16-key slice is 8 KB of K and V at d = 128, for which an SM has about 350 cycles at the measured copy rate, and
// needs 24 matrix instructions (8 rows; 48 for 16) and 16 ldmatrix of its four sub-partitions.
// Weights enter P.V as a pair of 16-bit numbers, their rounding and its remainder (relative error 2^-17 for bf16
// instead of 2^-9; for fp16 2^-22 or 2^-35 of the row's largest weight, whichever is more), which is 8 of those 24
// instructions: the tensor pipe has the room. A row's reference moves seldom (Reference in ea_tree.cuh), so most slices need no
// reduction over lanes.
#include "ea_tree.cuh"

namespace ea {
namespace serving {
namespace tree {

namespace {

constexpr int MAX_ROWS = 16, WARPS = 4, KT = 16 * WARPS, THREADS = 32 * WARPS, STAGES = 3, EXTRA = 1;

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// 16 bytes: `bytes` (16 or 0) from src, the rest zeros
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t a, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
// an 8 x 8 matrix of 16-bit numbers, two of a row in each lane, turned over
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <typename T>
__device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
      "%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__half>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
      "%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// two weights as their roundings and the roundings of what is left
template <typename T>
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo);
template <>
__device__ __forceinline__ void split2<__nv_bfloat16>(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  hi = *(const uint32_t*)&h;
  const __nv_bfloat162 r = __floats2bfloat162_rn(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xFFFF0000u));
  lo = *(const uint32_t*)&r;
}
template <>
__device__ __forceinline__ void split2<__half>(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  hi = *(const uint32_t*)&h;
  const float2 f = __half22float2(h);
  const __half2 r = __floats2half2_rn(x - f.x, y - f.y);
  lo = *(const uint32_t*)&r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// the two 16-bit numbers with infinities and NaN replaced by zeros
template <typename T>
__device__ __forceinline__ uint32_t finite2(uint32_t v) {
  constexpr uint32_t EXP = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
  if ((v & EXP) == EXP) v &= 0xFFFF0000u;
  if ((v & EXP << 16) == EXP << 16) v &= 0xFFFFu;
  return v;
}
template <int DP>
struct Smem {
  static constexpr int ROW_BYTES = DP * 2;
  static constexpr int SLICE = 16 * ROW_BYTES;                    // K or V of 16 keys
  static constexpr int STAGE = 2 * SLICE;                         // one warp's
  static constexpr int POOL = WARPS * STAGES * STAGE + 256;       // aligned to 256 bytes; also the join's scratch
  static_assert(POOL - 256 >= WARPS * MAX_ROWS * DP * 4, "the join fits into the stages");
};

template <int DP>
__device__ __forceinline__ uint32_t swz(int row, int piece) {
  return (uint32_t)(row * Smem<DP>::ROW_BYTES + ((piece ^ (row & 7)) << 4));
}

// Issues the copies of 16 keys from `key0` of the item into a stage. `page` is this lane's page of key
// key0 + lane % 16 (-1: none).
template <typename T, int DP>
__device__ __forceinline__ void load_slice(const Args& a, const Item& it, int key0, int page, uint32_t stage, int lane) {
  constexpr int PIECES = DP / 8, LANES_PER_ROW = PIECES < 8 ? PIECES : 8, RPI = 32 / LANES_PER_ROW;
  const int sub = lane / LANES_PER_ROW, c0 = lane % LANES_PER_ROW;
#pragma unroll
  for (int r0 = 0; r0 < 16; r0 += RPI) {
    const int r = r0 + sub, key = key0 + r;
    const int pg = __shfl_sync(0xffffffffu, page, r);
    const bool ok = key < it.len && pg >= 0;
    const int64_t off = ok ? key - (int64_t)div_by((uint32_t)key, a.by_page) * a.t.page_size : 0;
    const int64_t p = ok ? pg : 0;
    const T* ks = (const T*)a.t.k_cache + p * a.t.k_page_stride + it.h * a.t.k_head_stride + off * a.t.k_row_stride;
    const T* vs = (const T*)a.t.v_cache + p * a.t.v_page_stride + it.h * a.t.v_head_stride + off * a.t.v_row_stride;
#pragma unroll
    for (int c = c0; c < PIECES; c += LANES_PER_ROW) {
      const bool in = ok && c * 8 < a.t.d;
      cp16(stage + swz<DP>(r, c), in ? ks + c * 8 : (const T*)a.t.k_cache, in ? 16 : 0);
      cp16(stage + Smem<DP>::SLICE + swz<DP>(r, c), in ? vs + c * 8 : (const T*)a.t.v_cache, in ? 16 : 0);
    }
  }
}

// Whether query row R of the item (token i of the step) sees key `key`.
__device__ __forceinline__ bool sees(const Args& a, const Item& it, int i, int key, int page_ok) {
  if (key >= it.len || !page_ok) return false;
  if (key < it.ctx) return true;
  const int j = key - it.ctx;
  if (!a.t.tree_mask) return j <= i;
  return (j >> 5) < a.t.mask_words && ((a.t.tree_mask[(int64_t)(it.q0 + i) * a.t.mask_words + (j >> 5)] >> (j & 31)) & 1);
}

template <typename T, int DP, int NT>
__global__ void __launch_bounds__(THREADS, 2) few_rows_kernel(Args a) {
  using S = Smem<DP>;
  constexpr int ROWS = 8 * NT;
  begin();
  extern __shared__ uint8_t raw[];
  uint8_t* pool = (uint8_t*)(((uintptr_t)raw + 255) & ~(uintptr_t)255);
  uint32_t* sums = (uint32_t*)(raw + S::POOL);
  __shared__ uint64_t scratch[32];
  __shared__ float join_m[WARPS][ROWS], join_l[WARPS][ROWS];
  Schedule<ROWS, KT, EXTRA> sch;
  sch.build(a, sums, scratch);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t base = smem_addr(pool) + warp * STAGES * S::STAGE;
  uint32_t pos = sch.share(blockIdx.x);
  const uint32_t end = sch.share(blockIdx.x + 1);
  const float alpha = a.t.alpha;
  const bool in_page = a.t.page_size % 16 == 0;  // a slice lies in one page

  // copies of a whole slice from one page: this lane's piece of rows lane / LPR, + RPI, ..; lanes past d fill in zeros
  constexpr int LPR = DP / 8 < 8 ? DP / 8 : 8, RPI = 32 / LPR;
  const int c0 = lane % LPR;
  const int bytes0 = c0 * 8 < a.t.d ? 16 : 0, bytes1 = (c0 + 8) * 8 < a.t.d ? 16 : 0;
  const int64_t k_lane = (lane / LPR) * a.t.k_row_stride + (bytes0 ? c0 * 8 : 0);
  const int64_t v_lane = (lane / LPR) * a.t.v_row_stride + (bytes0 ? c0 * 8 : 0);
  // fragment addresses inside a slice; a step of 16 channels flips address bits 5 and up
  const uint32_t k_frag = (lane & 15) * S::ROW_BYTES + (((lane >> 4) ^ (lane & 7)) << 4);
  const uint32_t v_frag = S::SLICE + ((lane & 7) + ((lane >> 4) << 3)) * S::ROW_BYTES + ((((lane >> 3) & 1) ^ (lane & 7)) << 4);

  while (pos < end) {
    const Item it = sch.item(a, pos, end);
    pos = it.next;
    if (it.kt0 >= it.kt1) continue;
    const int rows = min(ROWS, it.new_tokens * a.group - it.m * ROWS);
    const int R0 = it.m * ROWS;

    // Q as B fragments: row 8 nt + lane / 4; and the tokens of the rows whose statistics this lane keeps, 8 nt +
    // 2 (lane % 4) + e
    uint32_t qf[NT][DP / 16][2];
    int tok[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int R = R0 + min(8 * nt + lane / 4, rows - 1), i = (int)div_by((uint32_t)R, a.by_group);
      const T* q = (const T*)a.t.q + (int64_t)(it.q0 + i) * a.t.q_stride + (int64_t)(it.h * a.group + R - i * a.group) * a.t.q_head_stride;
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const int c = ks * 16 + p * 8 + (lane & 3) * 2;
          qf[nt][ks][p] = c < a.t.d ? *(const uint32_t*)(q + c) : 0u;
        }
#pragma unroll
      for (int e = 0; e < 2; ++e) tok[nt][e] = (int)div_by((uint32_t)(R0 + min(8 * nt + 2 * (lane & 3) + e, rows - 1)), a.by_group);
    }
    const int n = it.kt1 - it.kt0;
    const int key_w = it.kt0 * KT + warp * 16;
    const T* k_head = (const T*)a.t.k_cache + it.h * a.t.k_head_stride + k_lane;
    const T* v_head = (const T*)a.t.v_cache + it.h * a.t.v_head_stride + v_lane;
    const int32_t* pages = a.t.page_table + it.b * a.t.table_stride;
    // the page of a slice, fetched one slice ahead of its copies: the slice's (in_page) or the lane's key's
    const auto page_of = [&](int key0) {
      const int key = in_page ? key0 : key0 + (lane & 15);
      if (key >= it.len) return -1;
      const int p = pages[div_by((uint32_t)key, a.by_page)];
      return p >= 0 && p < a.t.num_pages ? p : -1;
    };
    // issues a slice's copies; which of its keys exist
    const auto load = [&](int key0, int page, uint32_t stage) -> uint32_t {
      if (in_page && page >= 0 && key0 + 16 <= it.len) {
        const int off = key0 - (int)div_by((uint32_t)key0, a.by_page) * a.t.page_size;
        const T* ks = k_head + page * a.t.k_page_stride + off * a.t.k_row_stride;
        const T* vs = v_head + page * a.t.v_page_stride + off * a.t.v_row_stride;
#pragma unroll
        for (int r0 = 0; r0 < 16; r0 += RPI) {
          const uint32_t at = stage + swz<DP>(r0 + lane / LPR, c0);
          cp16(at, ks, bytes0);
          cp16(at + S::SLICE, vs, bytes0);
          if (DP == 128) {
            cp16(at ^ 128, ks + 64, bytes1);  // piece c0 + 8
            cp16((at ^ 128) + S::SLICE, vs + 64, bytes1);
          }
          ks += RPI * a.t.k_row_stride;
          vs += RPI * a.t.v_row_stride;
        }
        return 0xFFFFu;
      }
      if (in_page && key0 + (lane & 15) >= it.len) page = -1;
      load_slice<T, DP>(a, it, key0, page, stage, lane);
      return __ballot_sync(0xffffffffu, page >= 0) & 0xFFFFu;
    };

    // o: channels 16 nn + lane / 4 (+ 8), rows 8 nt + 2 (lane % 4) (+ 1)
    float o[NT][DP / 16][4], m[NT][2], l[NT][2];
    // The first pass takes the values as they are. An infinity or NaN among them may not meet the zero weight of a row
    // that does not see its key, nor a weight's remainder: if any output is not finite, a second pass takes
    // such values out of the product and adds them to the rows that see them one by one.
    for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int nn = 0; nn < DP / 16; ++nn)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[nt][nn][e] = 0.0f;
        m[nt][0] = m[nt][1] = -INFINITY, l[nt][0] = l[nt][1] = 0.0f;
      }
      uint32_t exist[STAGES];  // of the slices under way, oldest first
      int page = page_of(key_w);
#pragma unroll
      for (int s = 0; s < STAGES - 1; ++s) {
        exist[s] = s < n ? load(key_w + s * KT, page, base + s * S::STAGE) : 0;
        cp_commit();
        page = page_of(key_w + (s + 1) * KT);
      }
      uint32_t cur = base, ahead = base + (STAGES - 1) * S::STAGE;
      for (int t = 0; t < n; ++t) {
        cp_wait<STAGES - 2>();
        __syncwarp();
        const int coming = t + STAGES - 1;
        exist[STAGES - 1] = coming < n ? load(key_w + coming * KT, page, ahead) : 0;
        cp_commit();
        page = page_of(key_w + (coming + 1) * KT);
        const int key0 = key_w + t * KT;
        const uint32_t okm = exist[0];

        // scores: keys lane / 4 (+ 8), rows 8 nt + 2 (lane % 4) (+ 1)
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nt][e] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          if (ks * 16 < a.t.d) {
            uint32_t f[4];
            ldsm4((cur + k_frag) ^ (ks * 32), f);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma<T>(s[nt], f, qf[nt][ks][0], qf[nt][ks][1]);
          }
        }
        const bool masked = key0 + 16 > it.ctx || okm != 0xFFFFu;
        uint32_t hi[NT][2], lo[NT][2];
        bool grows = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[nt][e] *= alpha;
            if (masked) {
              const int kk = (lane >> 2) + 8 * (e >> 1);
              if (!sees(a, it, tok[nt][e & 1], key0 + kk, (okm >> kk) & 1)) s[nt][e] = -INFINITY;
            }
            grows |= Reference<T>::passed(s[nt][e], m[nt][e & 1]);
          }
        if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float mx = fmaxf(s[nt][e], s[nt][2 + e]);
#pragma unroll
              for (int w = 4; w < 32; w <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
              // where another row's score passed, this row keeps its reference: its bits do not depend on others
              const float to = Reference<T>::passed(mx, m[nt][e]) ? mx - Reference<T>::DOWN : m[nt][e];
              const float scale = ex2(m[nt][e] - (to == -INFINITY ? 0.0f : to));
              const float f = m[nt][e] == to ? 1.0f : scale;
              m[nt][e] = to, l[nt][e] *= f;
#pragma unroll
              for (int nn = 0; nn < DP / 16; ++nn) o[nt][nn][e] *= f, o[nt][nn][2 + e] *= f;
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float ref = m[nt][e] == -INFINITY ? 0.0f : m[nt][e];
            s[nt][e] = ex2(s[nt][e] - ref), s[nt][2 + e] = ex2(s[nt][2 + e] - ref);
            l[nt][e] += s[nt][e] + s[nt][2 + e];
          }
          // the weights as B fragments: keys 2 (lane % 4) (+ 1) (+ 8), row lane / 4
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            split2<T>(s[nt][2 * h], s[nt][2 * h + 1], hi[nt][h], lo[nt][h]);
            hi[nt][h] = transpose8(hi[nt][h]), lo[nt][h] = transpose8(lo[nt][h]);
          }
        }
#pragma unroll
        for (int nn = 0; nn < DP / 16; ++nn) {
          if (nn * 16 < a.t.d) {
            uint32_t f[4];
            ldsm4_t((cur + v_frag) ^ (nn * 32), f);
            if (pass) {
#pragma unroll
              for (int e = 0; e < 4; ++e) f[e] = finite2<T>(f[e]);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma<T>(o[nt][nn], f, hi[nt][0], hi[nt][1]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma<T>(o[nt][nn], f, lo[nt][0], lo[nt][1]);
          }
        }
        if (pass) {
          for (int kk = 0; kk < 16; ++kk) {
            bool see[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 2; ++e) see[nt][e] = sees(a, it, tok[nt][e], key0 + kk, (okm >> kk) & 1);
#pragma unroll
            for (int nn = 0; nn < DP / 16; ++nn)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int c = nn * 16 + 8 * h + (lane >> 2);
                const float f = to_f(*(const T*)(pool + (cur - smem_addr(pool)) + S::SLICE + swz<DP>(kk, c >> 3) + (c & 7) * 2));
                if (isfinite(f)) continue;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                  for (int e = 0; e < 2; ++e)
                    if (see[nt][e]) o[nt][nn][2 * h + e] += f;
              }
          }
          __syncwarp();
        }
#pragma unroll
        for (int i = 0; i + 1 < STAGES; ++i) exist[i] = exist[i + 1];
        cur = cur == base + (STAGES - 1) * S::STAGE ? base : cur + S::STAGE;
        ahead = ahead == base + (STAGES - 1) * S::STAGE ? base : ahead + S::STAGE;
      }
      cp_wait<0>();
      __syncwarp();
      float probe = 0.0f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int nn = 0; nn < DP / 16; ++nn)
#pragma unroll
          for (int e = 0; e < 4; ++e) probe = fmaf(o[nt][nn][e], 0.0f, probe);  // NaN if one is not finite
      if (!__any_sync(0xffffffffu, probe != 0.0f)) break;
    }

    // join the warps
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], w);
        if (lane < 4) join_m[warp][8 * nt + 2 * lane + e] = m[nt][e], join_l[warp][8 * nt + 2 * lane + e] = l[nt][e];
      }
    __syncthreads();  // every warp's copies have landed and its stages are free
    float* acc = (float*)pool + warp * ROWS * DP;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * nt + 2 * (lane & 3) + e;
        if (r >= rows) continue;
        float mm = join_m[0][r];
#pragma unroll
        for (int w = 1; w < WARPS; ++w) mm = fmaxf(mm, join_m[w][r]);
        const float sc = exp2f(m[nt][e] - (mm == -INFINITY ? 0.0f : mm));
#pragma unroll
        for (int nn = 0; nn < DP / 16; ++nn)
#pragma unroll
          for (int h = 0; h < 2; ++h) acc[r * DP + nn * 16 + 8 * h + (lane >> 2)] = o[nt][nn][2 * h + e] * sc;
      }
    __syncthreads();
    const bool whole = it.kt0 == 0 && it.kt1 == it.tiles;
    float* slot = slot_of(a, 2 * blockIdx.x + (it.kt0 == 0 ? 1 : 0), ROWS);
    for (int e = tid; e < rows * DP; e += THREADS) {
      const int r = e / DP, c = e % DP;
      float mm = join_m[0][r], ll = 0.0f, x = 0.0f;
#pragma unroll
      for (int w = 1; w < WARPS; ++w) mm = fmaxf(mm, join_m[w][r]);
      const float ref = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        ll = fmaf(join_l[w][r], exp2f(join_m[w][r] - ref), ll);
        x += ((const float*)pool)[(w * ROWS + r) * DP + c];
      }
      if (whole) {
        const int R = R0 + r, i = (int)div_by((uint32_t)R, a.by_group), j = R - i * a.group;
        const int64_t head = (int64_t)(it.q0 + i) * a.t.q_heads + it.h * a.group + j;
        if (c < a.t.d) ((T*)a.t.out)[head * a.t.d + c] = from_f<T>(ll == 0.0f ? 0.0f : x / ll);
        if (c == 0 && a.t.lse) a.t.lse[head] = ll == 0.0f ? -INFINITY : mm + log2f(ll);
      } else {
        slot[((c >> 2) * ROWS + r) * 4 + (c & 3)] = x;
        if (c == 0) slot[ROWS * DP + r] = mm, slot[ROWS * (DP + 1) + r] = ll;
      }
    }
    __syncthreads();  // before the next item's copies
  }
}

template <typename T, int DP, int NT>
int launch(Args& a, cudaStream_t st) {
  const size_t smem = Smem<DP>::POOL + 4 * (size_t)(a.t.batch + 1);
  static bool ready[64];  // per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !ready[dev])) {
    e = cudaFuncSetAttribute(few_rows_kernel<T, DP, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             Smem<DP>::POOL + 4 * (EA_TREE_MAX_SEQS + 1));
    if (e == cudaSuccess && dev < 64) ready[dev] = true;
  }
  if (e != cudaSuccess) return cuda_rc(e);
  e = launch_early(few_rows_kernel<T, DP, NT>, a.workers, THREADS, smem, st, a);
  if (e != cudaSuccess) return cuda_rc(e);
  return launch_combine<T, 8 * NT, KT, EXTRA>(a, st);
}

template <typename T>
int launch_few(Args& a, int rows, cudaStream_t st) {
  if (a.dp == 64) return rows == 8 ? launch<T, 64, 1>(a, st) : launch<T, 64, 2>(a, st);
  return rows == 8 ? launch<T, 128, 1>(a, st) : launch<T, 128, 2>(a, st);
}

// Most units a call can have, from the sizes the host knows.
int64_t most_units(const ea_tree_attention_t& t, int rows, int kt) {
  const int64_t group = t.q_heads / t.kv_heads;
  const int64_t tiles = ((int64_t)t.max_pages * t.page_size + kt - 1) / kt;
  // row tiles: every sequence's last one may be partly filled
  const int64_t row_tiles = t.tokens * group / rows + t.batch;
  return row_tiles * t.kv_heads * ((tiles > 0 ? tiles : 1) + 4);  // and an item's units without keys
}

// Which kernel, by the query rows per sequence and kv head: at most 8 or 16 (few_rows_kernel), below 512 the tensor-core
// kernel with 128-row items, else with 256-row items, which take half the traffic from L2 but keep one of two slots
// idle where an item has 128 rows or fewer. Eight sequences behind 16384 keys, 4 kv heads of 128, us with 128- / 256-row items:
// 64 rows 70 / 90, 128 rows 78 / 94, 192 rows 113 / 105, 256 rows 116 / 111, 320 rows 145 / 171, 384 rows 147 / 173,
// 512 rows 198 / 179, 768 rows 285 / 266, 1024 rows 370 / 340; from 1536 rows on they are within the clock's changes of one
// another, and behind 1000 to 4000 keys 128-row items are ahead up to 1024 rows (100 / 102). max_new is a hint, so any choice
// is right for any lengths.
struct Choice {
  int rows, kt, per_sm;
};
Choice choose(const ea_tree_attention_t& t) {
  const int64_t rows = (int64_t)(t.max_new > 0 ? t.max_new : 1) * (t.q_heads / t.kv_heads);
  if (rows <= MAX_ROWS || t.batch > MANY_MAX_SEQS) return {rows <= 8 ? 8 : MAX_ROWS, KT, 2};
  return {rows < 512 ? 128 : 256, 128, 1};
}
int check(const ea_tree_attention_t* t) {
  if (!t || t->tokens < 0 || t->batch < 0 || t->q_heads <= 0 || t->kv_heads <= 0 || t->d <= 0 || t->page_size <= 0 ||
      t->max_pages < 0 || t->num_pages < 0 || t->mask_words < 0)
    return fail(-1, "tree_attention: negative or zero size");
  if (t->q_heads % t->kv_heads) return fail(-1, "tree_attention: q_heads is no multiple of kv_heads");
  if (t->batch > EA_TREE_MAX_SEQS) return fail(-1, "tree_attention: more than EA_TREE_MAX_SEQS sequences");
  if (t->d % 8 || t->d > 128) return fail(-9, "tree_attention: d is no multiple of 8 up to 128");
  if (t->dtype != EA_BF16 && t->dtype != EA_FP16) return fail(-9, "tree_attention: element type is neither bf16 nor fp16");
  if (t->tokens * t->q_heads >= (1ll << 31) || (int64_t)t->max_pages * t->page_size >= (1ll << 31))
    return fail(-1, "tree_attention: too many tokens or keys");
  const Choice c = choose(*t);
  if (most_units(*t, c.rows, c.kt) >= (1ll << 31))
    return fail(-1, "tree_attention: 2^31 tiles or more, by the tokens, the table's width and max_new");
  return 0;
}

int workers_for(const ea_tree_attention_t& t, const Choice& c) {
  const int64_t most = most_units(t, c.rows, c.kt), fill = (int64_t)c.per_sm * sm_count();
  return (int)(most < fill ? (most > 0 ? most : 1) : fill);
}

}  // namespace
}  // namespace tree
}  // namespace serving
}  // namespace ea

extern "C" int64_t ea_tree_attention_workspace(const ea_tree_attention_t* t) {
  using namespace ea::serving;
  if (tree::check(t)) return -1;
  const int dp = t->d <= 64 ? 64 : 128;
  const tree::Choice c = tree::choose(*t);
  return (int64_t)tree::workers_for(*t, c) * 2 * c.rows * (dp + 2) * 4;
}

extern "C" int ea_tree_attention_cuda(const ea_tree_attention_t* t, void* stream) {
  using namespace ea::serving;
  const int rc = tree::check(t);
  if (rc) return rc;
  if (t->tokens == 0 || t->batch == 0) return 0;
  if (!t->q || !t->out || !t->q_start || !t->seq_lens || !t->workspace ||
      (t->max_pages && (!t->page_table || !t->k_cache || !t->v_cache)))
    return fail(-1, "tree_attention: a required pointer is NULL");
  const uintptr_t base = (uintptr_t)t->q | (uintptr_t)t->k_cache | (uintptr_t)t->v_cache | (uintptr_t)t->out | (uintptr_t)t->workspace;
  const auto used = [](int64_t extent, int64_t stride, int64_t other) { return extent > 1 ? stride | other : 0; };
  const int64_t strides = used(t->tokens, t->q_stride, 0) | used(t->q_heads, t->q_head_stride, 0) |
                          used(t->num_pages, t->k_page_stride, t->v_page_stride) |
                          used(t->kv_heads, t->k_head_stride, t->v_head_stride) |
                          used(t->page_size, t->k_row_stride, t->v_row_stride);
  if (base % 16 || strides % 8) return fail(-9, "tree_attention: rows of q, the caches or out, or the workspace, are not on 16-byte boundaries");
  tree::Args a;
  a.t = *t;
  a.group = t->q_heads / t->kv_heads;
  a.by_page = fast_div((uint32_t)t->page_size);
  a.by_group = fast_div((uint32_t)a.group);
  a.dp = t->d <= 64 ? 64 : 128;
  a.wait_debug = wait_debug_hook();
  const tree::Choice c = tree::choose(*t);
  a.workers = tree::workers_for(*t, c);
  cudaStream_t st = (cudaStream_t)stream;
  if (c.rows > tree::MAX_ROWS) return tree::launch_many(a, c.rows == 256, st);
  return t->dtype == EA_BF16 ? tree::launch_few<__nv_bfloat16>(a, c.rows, st) : tree::launch_few<__half>(a, c.rows, st);
}
