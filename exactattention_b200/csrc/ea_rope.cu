// Rotary positions (ea_rope_cuda): pair i of every head is turned by positions[axis(i)] * inv_freq[i],
//   (x, y) -> (x c - y s, y c + x s),
// optionally with the write of the turned keys and of the values into paged cache rows.
//
// Bound by HBM: every element is read once and written once. A thread owns VEC consecutive pairs
// of one token (two 16-byte pieces of a head), computes their cos / sin once and walks over heads with
// them, so the trigonometry costs little per byte. The angle is reduced in binary64
// (turns = position * inv_freq / 2 pi, minus its nearest integer: the product of a 31-bit and a 24-bit
// number rounds at 2^-53), then sincospif sees an argument in [-1, 1] whatever the position.
#include "ea_serving.cuh"

namespace ea {
namespace serving {
namespace {

constexpr int THREADS = 256;
constexpr double INV_2PI = 0.15915494309189533577;  // 1 / (2 pi)

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

struct Plan {
  int units, turn_units;  // pieces of a head: those that are turned first, then copied ones
  int groups;             // head groups: thread (token, group, unit) takes heads group, group + groups, ..
  FastDiv by_units, by_groups, by_page;
};

// The two pieces of a unit, in elements from the head's start. Turned units hold VEC pairs; a copied unit is
// the piece at rot + VEC c alone.
template <int VEC>
__device__ __forceinline__ void unit_offsets(const ea_rope_t& a, int u, int turn_units, int& o0, int& o1) {
  if (u < turn_units) {
    o0 = a.adjacent ? 2 * VEC * u : VEC * u;
    o1 = a.adjacent ? o0 + VEC : o0 + a.rot / 2;
  } else {
    o0 = a.rot + VEC * (u - turn_units);
    o1 = -1;
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(THREADS) rope_kernel(ea_rope_t a, Plan p) {
  using P = Pack<T, VEC>;
  const int64_t item = (int64_t)blockIdx.x * THREADS + threadIdx.x;
  const int per_tok = p.units * p.groups;
  const int64_t tok = item / per_tok;
  if (tok >= a.tokens) return;
  const uint32_t rem = (uint32_t)(item - tok * per_tok);
  const int grp = (int)div_by(rem, p.by_units), u = (int)(rem - grp * p.units);
  int o0, o1;
  unit_offsets<VEC>(a, u, p.turn_units, o0, o1);
  const bool turn = u < p.turn_units;

  float c[VEC], s[VEC];
  if (turn) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int f = u * VEC + i;
      const int ax = a.axes ? min(max(a.axes[f], 0), a.num_axes - 1) : 0;
      const double turns = (double)a.positions[ax * a.axis_stride + tok] * (double)a.inv_freq[f] * INV_2PI;
      const float r = (float)(turns - rint(turns));
      sincospif(2.0f * r, &s[i], &c[i]);
      if (a.inverse) s[i] = -s[i];
    }
  }
  int64_t kdst = 0, vdst = 0;
  bool store_kv = true;
  if (a.slot_map) {
    const int64_t slot = a.slot_map[tok];
    store_kv = slot >= 0 && slot < a.num_slots;
    if (store_kv) {
      const int64_t page = slot < 0x7FFFFFFF ? (int64_t)div_by((uint32_t)slot, p.by_page) : slot / a.page_size;
      const int64_t off = slot - page * a.page_size;
      kdst = page * a.k_page_stride + off * a.k_row_stride;
      vdst = page * a.v_page_stride + off * a.v_row_stride;
    }
  }
  const int nk = a.q_heads + a.kv_heads;
  const int heads = nk + (a.slot_map ? a.kv_heads : 0);
#pragma unroll 4
  for (int h = grp; h < heads; h += p.groups) {
    const T* src;
    T* dst;
    if (h < a.q_heads) {
      src = (const T*)a.q + tok * a.q_stride + h * a.q_head_stride;
      dst = (T*)a.q_out + (tok * a.q_heads + h) * a.d;
    } else if (h < nk) {
      const int kh = h - a.q_heads;
      if (!store_kv) continue;
      src = (const T*)a.k + tok * a.k_stride + kh * a.k_head_stride;
      dst = a.slot_map ? (T*)a.k_cache + kdst + kh * a.k_cache_head_stride
                       : (T*)a.k_out + (tok * a.kv_heads + kh) * a.d;
    } else {
      const int vh = h - nk;
      if (!store_kv) continue;
      src = (const T*)a.v + tok * a.v_stride + vh * a.v_head_stride;
      dst = (T*)a.v_cache + vdst + vh * a.v_cache_head_stride;
    }
    P x = *(const P*)(src + o0), y;
    if (turn) {
      y = *(const P*)(src + o1);
      if (h < nk) {
        float e[2 * VEC];  // in pair order for adjacent pairs, else the first members then the second
#pragma unroll
        for (int i = 0; i < VEC; ++i) e[i] = to_f(x.v[i]), e[VEC + i] = to_f(y.v[i]);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const int j0 = a.adjacent ? 2 * i : i, j1 = a.adjacent ? 2 * i + 1 : VEC + i;
          const float f = e[j0], g = e[j1];
          e[j0] = fmaf(f, c[i], -(g * s[i]));
          e[j1] = fmaf(g, c[i], f * s[i]);
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) x.v[i] = from_f<T>(e[i]), y.v[i] = from_f<T>(e[VEC + i]);
      }
      *(P*)(dst + o1) = y;
    }
    *(P*)(dst + o0) = x;
  }
}

template <typename T, int VEC>
int launch(const ea_rope_t& a, cudaStream_t st) {
  Plan p;
  p.turn_units = a.rot / 2 / VEC;
  p.units = p.turn_units + (a.d - a.rot) / VEC;
  const int heads = a.q_heads + a.kv_heads * (a.slot_map ? 2 : 1);
  // Heads a thread: 8 where there are tokens enough to fill the GPU four times over, fewer otherwise.
  const int64_t want = (int64_t)sm_count() * 2048 * 4;
  int per = 8;
  while (per > 1 && a.tokens * p.units * ((heads + per - 1) / per) < want) per >>= 1;
  p.groups = (heads + per - 1) / per;
  p.by_units = fast_div((uint32_t)p.units);
  p.by_groups = fast_div((uint32_t)p.groups);
  p.by_page = fast_div((uint32_t)(a.page_size > 0 ? a.page_size : 1));
  const int64_t items = a.tokens * p.units * p.groups;
  const int64_t blocks = (items + THREADS - 1) / THREADS;
  if (blocks > 0x7FFFFFFF) return fail(-1, "rope: too many tokens");
  rope_kernel<T, VEC><<<(unsigned)blocks, THREADS, 0, st>>>(a, p);
  return cuda_rc(cudaGetLastError());
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
  if (a->d > 8192 || a->q_heads > 65536 || a->kv_heads > 65536) return fail(-9, "rope: d above 8192 or above 65536 heads");
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
