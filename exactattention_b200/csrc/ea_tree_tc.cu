// Launches of the tensor-core tree attention kernel (ea_tree_tc.cuh).
#include <cuda.h>
#include <cudaTypedefs.h>
#include <string.h>

#include <type_traits>

#include "ea_tree_tc.cuh"

namespace ea {
namespace serving {
namespace tree {
namespace {

// Rows of a copy box: the largest power of two that divides the page size, 8 (a swizzle period) to 128; 0: pages
// that no such box tiles, whose tiles are copied piece by piece.
int box_rows(int page_size) {
  const int p2 = page_size & -page_size;
  return p2 < 8 ? 0 : p2 > many::KT ? many::KT : p2;
}

// Tensor map of a cache as (d, page_size, kv_heads, pages), boxes of 64 channels x `box` rows, 128-byte swizzle; what lies
// past d or past the last page reads as zeros. False where the strides allow none.
bool tensor_map(const Args& a, bool value, int box, CUtensorMap* tm) {
  static PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
                   q == cudaDriverEntryPointSuccess
               ? (PFN_cuTensorMapEncodeTiled_v12000)f
               : nullptr;
  }();
  memset(tm, 0, sizeof *tm);
  const int64_t strides[3] = {value ? a.t.v_row_stride : a.t.k_row_stride, value ? a.t.v_head_stride : a.t.k_head_stride,
                              value ? a.t.v_page_stride : a.t.k_page_stride};
  const cuuint64_t dims[4] = {(cuuint64_t)a.t.d, (cuuint64_t)a.t.page_size, (cuuint64_t)a.t.kv_heads, (cuuint64_t)a.t.num_pages};
  cuuint64_t bytes[3];
  for (int i = 0; i < 3; ++i) {
    const int64_t stride = dims[i + 1] > 1 ? strides[i] : a.t.d;  // of an extent of one it may be anything, but not in the map
    if (stride <= 0 || stride >= (1ll << 38)) return false;
    bytes[i] = (cuuint64_t)stride * 2;
  }
  const cuuint32_t tile[4] = {64u, (cuuint32_t)box, 1u, 1u}, step[4] = {1u, 1u, 1u, 1u};
  return encode && a.t.num_pages > 0 && a.t.num_pages < (1ll << 31) &&
         encode(tm, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, (void*)(value ? a.t.v_cache : a.t.k_cache), dims, bytes, tile, step,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DP, bool PAIR>
int launch(const Args& a, cudaStream_t st) {
  using C = many::Cfg<DP, PAIR>;
  // once per device: room for the dynamic shared memory, and whether the block starts with the registers that
  // its groups' later shares add up to
  static int state[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_rc(e);
  const size_t sums = 4 * (size_t)(a.t.batch + 1);
  if (dev >= 64 || !state[dev]) {
    cudaFuncAttributes at;
    e = cudaFuncGetAttributes(&at, many::many_rows_kernel<T, DP, PAIR>);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(many::many_rows_kernel<T, DP, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               C::SMEM + 4 * (MANY_MAX_SEQS + 1));
    if (e != cudaSuccess) return cuda_rc(e);
    if (at.numRegs != many::LAUNCH_REGS) return fail(-4, "tree_attention: the tensor-core kernel was built with another register count");
    if (dev < 64) state[dev] = 1;
  }
  CUtensorMap tk, tv;
  int box = box_rows(a.t.page_size);
  if (box && !(tensor_map(a, false, box, &tk) && tensor_map(a, true, box, &tv))) box = 0;
  e = launch_early(many::many_rows_kernel<T, DP, PAIR>, a.workers, many::THREADS, C::SMEM + sums, st, a, tk, tv, box);
  if (e != cudaSuccess) return cuda_rc(e);
  return launch_combine<T, C::ROWS, many::KT, many::EXTRA>(a, st);
}

}  // namespace

int launch_many(const Args& a, bool pair, cudaStream_t st) {
  if (a.t.dtype == EA_BF16) {
    if (a.dp == 64) return pair ? launch<__nv_bfloat16, 64, true>(a, st) : launch<__nv_bfloat16, 64, false>(a, st);
    return pair ? launch<__nv_bfloat16, 128, true>(a, st) : launch<__nv_bfloat16, 128, false>(a, st);
  }
  if (a.dp == 64) return pair ? launch<__half, 64, true>(a, st) : launch<__half, 64, false>(a, st);
  return pair ? launch<__half, 128, true>(a, st) : launch<__half, 128, false>(a, st);
}

}  // namespace tree
}  // namespace serving
}  // namespace ea
