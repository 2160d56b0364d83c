// Rotary positions (ea_rope_cuda): pair i of every head is turned by positions[axis(i)] * inv_freq[i],
//   (x, y) -> (x c - y s, y c + x s),
// optionally with the write of the turned keys and of the values into paged cache rows.
//
// Bound by HBM: every element is read once and written once. A thread owns one piece (two 16-byte parts of a head
// that hold VEC pairs) of one token and takes it from up to four heads: it loads all of them, the block computes the
// cos / sin of its tokens into shared memory while the loads are under way, once per (token, frequency), and the
// thread turns and stores its pieces with them. The angle is reduced in 32 bits without loss: turns = position * f
// with f = inv_freq / 2 pi as a sum of two numbers, the product's rounding error recovered by an FMA, the nearest
// integer taken off the large part (exact); what is left of 2^-47 relative error is far below a 32-bit result's
// rounding. sincospif then sees an argument in [-1, 1] whatever the position. Positions of 2^24 and more, which
// binary32 does not hold, and angles of 2^24 and more, whose 2^-47 would show, are reduced the same way in binary64.
// Measured on one B200: 16927 tokens, 16 q and 8 kv heads of 128, three axes, written into a paged cache: 53 us for 278 MB
// (80% of the copy rate); with the angles computed per thread in binary64 127 us.
#include "ea_serving.cuh"

namespace ea {
namespace serving {
namespace {

constexpr double INV_2PI = 0.15915494309189533577, INV_2PI_LO = -9.839338337591243e-18;  // their sum is 1 / (2 pi) to 2^-109

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

// Keeps the compiler from widening a piece's numbers before this point, which would double the registers it takes
// across the barrier.
template <typename T, int VEC>
__device__ __forceinline__ void keep_packed(Pack<T, VEC>& p) {
  if constexpr (sizeof(p) == 16) {
    uint32_t* w = (uint32_t*)&p;
    asm volatile("" : "+r"(w[0]), "+r"(w[1]), "+r"(w[2]), "+r"(w[3]));
  }
}

struct Plan {
  int units, turn_units;  // pieces of a head: those that are turned first, then copied ones
  int tokens, lanes;      // of a block: tokens, and heads that are worked on at the same time
  int head_blocks, all_heads;
  FastDiv by_units, by_lanes, by_half, by_page, by_head_blocks;
};

__device__ __forceinline__ float2 cos_sin(int pos, float freq, bool inverse) {
  float r;
  const float p = (float)pos;
  if (fabsf(p) < 0x1p24f && fabsf(p * freq) < 0x1p24f) {
    const float c_hi = 0.15915494f;                              // 1 / (2 pi) = c_hi + c_lo
    const float c_lo = (float)(INV_2PI - (double)0.15915494f);
    const float f_hi = freq * c_hi, f_lo = fmaf(freq, c_lo, fmaf(freq, c_hi, -f_hi));
    const float t = p * f_hi, e = fmaf(p, f_lo, fmaf(p, f_hi, -t));
    r = (t - rintf(t)) + e;
  } else {
    const double x = (double)pos * freq, left = fma((double)pos, (double)freq, -x), n = rint(x * INV_2PI);
    const double v = fma(x, INV_2PI, -n) + fma(x, INV_2PI_LO, left * INV_2PI);
    r = (float)(v - rint(v));
  }
  float2 cs;
  sincospif(2.0f * r, &cs.y, &cs.x);
  if (inverse) cs.y = -cs.y;
  return cs;
}

template <typename T, int VEC, int ITEMS, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS > 256 ? 1 : ITEMS == 4 ? 3 : 5) rope_kernel(ea_rope_t a, Plan p) {
  using P = Pack<T, VEC>;
  begin();
  extern __shared__ float2 cs[];  // (tokens, rot / 2)
  const uint32_t group = div_by(blockIdx.x, p.by_head_blocks);
  const int64_t tok0 = (int64_t)group * p.tokens;
  const int nk = a.q_heads + a.kv_heads, half = a.rot / 2;
  const int toks = (int)min((int64_t)p.tokens, a.tokens - tok0);
  const uint32_t th = div_by(threadIdx.x, p.by_units);
  const int u = (int)(threadIdx.x - th * p.units), tl = (int)div_by(th, p.by_lanes);
  const int h0 = (int)(blockIdx.x - group * p.head_blocks) * p.lanes * ITEMS + (int)(th - tl * p.lanes);
  const int64_t tok = tok0 + tl;
  const bool turn = u < p.turn_units, live = tl < toks;
  // turned units hold VEC pairs; a copied unit is the one piece at rot + VEC c
  const int o = !turn ? a.rot + VEC * (u - p.turn_units) : a.adjacent ? 2 * VEC * u : VEC * u;
  const int apart = a.adjacent ? VEC : half;  // from the first part of a piece to the second

  int64_t k_row = 0, v_row = 0;
  bool stored = true;  // the token's key and value have a place
  if (a.slot_map && live) {
    const int64_t slot = a.slot_map[tok];
    stored = slot >= 0 && slot < a.num_slots;
    const int64_t page = slot < 0x7FFFFFFF ? (int64_t)div_by((uint32_t)slot, p.by_page) : slot / a.page_size;
    const int64_t off = slot - page * a.page_size;
    k_row = page * a.k_page_stride + off * a.k_row_stride;
    v_row = page * a.v_page_stride + off * a.v_row_stride;
  }
  P x[ITEMS], y[ITEMS];
  T* dst[ITEMS];  // nullptr: nothing to do
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int h = h0 + i * p.lanes;
    dst[i] = nullptr;
    if (!live || h >= p.all_heads || (h >= a.q_heads && !stored)) continue;
    const T* src;
    if (h < a.q_heads) {
      src = (const T*)a.q + tok * a.q_stride + h * a.q_head_stride;
      dst[i] = (T*)a.q_out + (tok * a.q_heads + h) * a.d + o;
    } else if (h < nk) {
      const int kh = h - a.q_heads;
      src = (const T*)a.k + tok * a.k_stride + kh * a.k_head_stride;
      dst[i] = (a.slot_map ? (T*)a.k_cache + k_row + kh * a.k_cache_head_stride
                           : (T*)a.k_out + (tok * a.kv_heads + kh) * a.d) + o;
    } else {
      src = (const T*)a.v + tok * a.v_stride + (h - nk) * a.v_head_stride;
      dst[i] = (T*)a.v_cache + v_row + (h - nk) * a.v_cache_head_stride + o;
    }
    x[i] = *(const P*)(src + o);
    if (turn) y[i] = *(const P*)(src + o + apart);
  }

  for (uint32_t e = threadIdx.x; e < (uint32_t)(toks * half); e += THREADS) {
    const int t = (int)div_by(e, p.by_half), f = (int)(e - t * half);
    const int ax = a.axes ? min(max(a.axes[f], 0), a.num_axes - 1) : 0;
    cs[e] = cos_sin(a.positions[ax * a.axis_stride + tok0 + t], a.inv_freq[f], a.inverse);
  }
  __syncthreads();
  float c[VEC], s[VEC];
  if (turn && live) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float2 t = cs[tl * half + u * VEC + j];
      c[j] = t.x, s[j] = t.y;
    }
  }

#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    if (!dst[i]) continue;
    keep_packed(x[i]), keep_packed(y[i]);
    if (turn && h0 + i * p.lanes < nk) {
      float e[2 * VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) e[j] = to_f(x[i].v[j]), e[VEC + j] = to_f(y[i].v[j]);
      if (a.adjacent) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float f = e[2 * j], g = e[2 * j + 1];
          e[2 * j] = fmaf(f, c[j], -(g * s[j])), e[2 * j + 1] = fmaf(g, c[j], f * s[j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float f = e[j], g = e[VEC + j];
          e[j] = fmaf(f, c[j], -(g * s[j])), e[VEC + j] = fmaf(g, c[j], f * s[j]);
        }
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[i].v[j] = from_f<T>(e[j]), y[i].v[j] = from_f<T>(e[VEC + j]);
    }
    *(P*)dst[i] = x[i];
    if (turn) *(P*)(dst[i] + apart) = y[i];
  }
}

template <typename T, int VEC, int ITEMS, int THREADS>
int launch_items(const ea_rope_t& a, Plan p, cudaStream_t st) {
  const int want = (p.all_heads + ITEMS - 1) / ITEMS;  // lanes for all heads in one block
  p.lanes = min(want, THREADS / p.units);
  p.head_blocks = (p.all_heads + p.lanes * ITEMS - 1) / (p.lanes * ITEMS);
  p.tokens = p.head_blocks > 1 ? 1 : max(1, THREADS / (p.units * p.lanes));
  p.by_lanes = fast_div((uint32_t)p.lanes);
  p.by_head_blocks = fast_div((uint32_t)p.head_blocks);
  const int64_t blocks = (a.tokens + p.tokens - 1) / p.tokens * p.head_blocks;
  if (blocks >= (1ll << 31)) return fail(-1, "rope: too many tokens");
  // at most THREADS / units tokens of rot / 2 <= units * VEC pairs: 8 KB per VEC
  return cuda_rc(launch_early(rope_kernel<T, VEC, ITEMS, THREADS>, (unsigned)blocks, THREADS, sizeof(float2) * p.tokens * (a.rot / 2), st, a, p));
}

template <typename T, int VEC>
int launch(const ea_rope_t& a, cudaStream_t st) {
  Plan p;
  p.turn_units = a.rot / 2 / VEC;
  p.units = p.turn_units + (a.d - a.rot) / VEC;
  p.all_heads = a.q_heads + a.kv_heads * (a.slot_map ? 2 : 1);
  p.by_units = fast_div((uint32_t)p.units);
  p.by_half = fast_div((uint32_t)max(1, a.rot / 2));
  p.by_page = fast_div((uint32_t)max(1, a.page_size));
  if constexpr (VEC == 1) {
    return launch_items<T, 1, 1, 1024>(a, p, st);  // up to 1024 single pairs a head
  } else {
    // four pieces a thread keep enough bytes in flight; one where that would leave SMs without a block
    const int64_t items = a.tokens * p.units * p.all_heads;
    if (items > 4 * 256 * 2 * (int64_t)sm_count()) return launch_items<T, VEC, 4, 256>(a, p, st);
    return launch_items<T, VEC, 1, 256>(a, p, st);
  }
}

template <typename T>
int launch_type(const ea_rope_t& a, cudaStream_t st) {
  constexpr int VEC = 16 / (int)sizeof(T);
  // 16-byte pieces where every head starts on a 16-byte boundary and the pieces divide the head's two
  // halves; single pairs otherwise
  const uintptr_t base = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.q_out | (uintptr_t)a.k_out |
                         (uintptr_t)a.k_cache | (uintptr_t)a.v_cache;
  int64_t strides = a.d | (a.q_heads ? a.q_stride | a.q_head_stride : 0) |
                    (a.kv_heads ? a.k_stride | a.k_head_stride : 0);
  if (a.slot_map)
    strides |= a.v_stride | a.v_head_stride | a.k_page_stride | a.k_cache_head_stride | a.k_row_stride |
               a.v_page_stride | a.v_cache_head_stride | a.v_row_stride;
  if (base % 16 == 0 && strides % VEC == 0 && (a.rot / 2) % VEC == 0) return launch<T, VEC>(a, st);
  return launch<T, 1>(a, st);
}

}  // namespace
}  // namespace serving
}  // namespace ea

extern "C" int ea_rope_cuda(const ea_rope_t* a, void* stream) {
  using namespace ea::serving;
  if (!a || a->tokens < 0 || a->q_heads < 0 || a->kv_heads < 0 || a->d <= 0 || a->rot < 0 || a->rot > a->d ||
      a->rot % 2 != 0 || a->num_axes < 1)
    return fail(-1, "rope: negative size, or rot odd or above d");
  if (a->d > 1024 || a->q_heads > 65536 || a->kv_heads > 65536) return fail(-9, "rope: d above 1024 or above 65536 heads");
  if (a->tokens == 0 || a->q_heads + a->kv_heads == 0) return 0;
  if ((a->rot && (!a->positions || !a->inv_freq)) || (a->q_heads && (!a->q || !a->q_out)) || (a->kv_heads && !a->k))
    return fail(-1, "rope: a required pointer is NULL");
  if (a->slot_map ? (a->kv_heads && (!a->v || !a->k_cache || !a->v_cache || a->page_size <= 0 || a->num_slots < 0))
                  : (a->kv_heads && !a->k_out))
    return fail(-1, "rope: a required pointer is NULL, or no page size");
  cudaStream_t st = (cudaStream_t)stream;
  switch (a->dtype) {
    case EA_BF16: return launch_type<__nv_bfloat16>(*a, st);
    case EA_FP16: return launch_type<__half>(*a, st);
    case EA_FP32: return launch_type<float>(*a, st);
  }
  return fail(-9, "rope: unknown element type");
}
