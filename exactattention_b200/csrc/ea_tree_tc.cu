// Launches of the tensor-core tree attention kernel (ea_tree_tc.cuh).
#include <type_traits>

#include "ea_tree_tc.cuh"

namespace ea {
namespace serving {
namespace tree {
namespace {

template <typename T, int DP, bool PAIR>
int launch(const Args& a, cudaStream_t st) {
  using C = many::Cfg<DP, PAIR>;
  // once per device: room for the dynamic shared memory, and whether the block starts with the 128 registers a
  // thread that its groups' later shares (2 x 192 + 2 x 64) add up to
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
    if (at.numRegs != 128) return fail(-4, "tree_attention: the tensor-core kernel was not built with 128 registers a thread");
    if (dev < 64) state[dev] = 1;
  }
  many::many_rows_kernel<T, DP, PAIR><<<a.workers, many::THREADS, C::SMEM + sums, st>>>(a);
  e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_rc(e);
  if (a.workers > 1) combine_kernel<T, C::ROWS, many::KT, 256><<<dim3(a.workers, C::ROWS / 16), 256, sums, st>>>(a);
  return cuda_rc(cudaGetLastError());
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
