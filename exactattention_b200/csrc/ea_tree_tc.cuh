// Tree attention for many query rows per kv head on the 5th-generation tensor cores (tcgen05): 128-row tiles.
//
// Per block one work item at a time: its query rows (tokens x the heads of a group) in shared memory, key and
// value tiles of 128 keys streamed through a ring of buffers. Two softmax slots of 128 threads (a thread a row)
// take turns on the tensor core:
//   PAIR  = true : the item has 256 rows, slot s owns rows 128 s .. and both use every key tile (half the
//                  traffic from L2 per row);
//   PAIR  = false: the item has 128 rows and slot s takes the key tiles of parity s; the two partial results are
//                  joined at the item's end.
// A slot's cycle: S = Q K^T into tensor memory (SS form, both operands K-major, 128-byte swizzle) -> row maximum,
// weights 2^(alpha s - m) and their sum in registers -> the weights as 16-bit numbers into tensor memory over S ->
// O += P V (A from tensor memory, V with its channels as the MN-major dimension). While one slot computes
// weights the other's products run: at 128 x 128 keys x 128 channels each of the two products takes about 512
// cycles of the tensor pipe and the 16384 exponentials 1024 cycles of the special-function pipe.
// The MMA thread issues PV(t) and then QK of the slot's next tile, so one arrival per cycle tells the slot that its
// scores are there and that O is at rest: the rescale of O needs no wait of its own. It happens only when a row's
// reference moves (Reference in ea_tree.cuh; the sum and O share it).
// Weights are rounded to the cache's type for the product (relative error 2^-9 for bf16; 2^-12 for fp16 down to 2^-24 of the
// row's largest weight, below that 2^-35 of the largest; of random sign, about the rounding of the output itself);
// their sum takes them unrounded.
// Measured on one B200: 16 trees of 17 to 64 nodes over 1K to 15K keys, 16 / 8 heads of 128, 140 us in bursts and 155 us in
// a long loop (545 MB of keys and values: 83 us at the copy rate); four chunks of 256 tokens behind 16K keys, 32 / 4
// heads, 325 us in bursts and 381 us in a long loop (277 GFLOP: 170 us at
// the measured bf16 rate; the tensor pipe is active 43% of the time). A slot's cycle at 128 x 128 x 128 is what bounds it. Clock
// readings in an instrumented copy, whose cycle is 5500 for a tile of either slot: 2000 for the weights, 400 to store them
// and hand them over, 800 until the issuer is done with the other slot, 1850 for the issue of the 16 products beside busy
// softmax warps, 400 to 500 until the scores are seen.
#pragma once
#include <cuda.h>

#include "ea_tcgen05.cuh"
#include "ea_tree.cuh"

namespace ea {
namespace serving {
namespace tree {
namespace many {

using namespace ea::tc;

constexpr int KT = 128, TILE = 128, THREADS = 384;  // warps 0-7 softmax slots, 8 products, 9-11 copies
constexpr int SLOT_THREADS = 128, LOADERS = 64;
// registers a thread: at launch, and after the groups have traded (2 x 128 x 216 + 128 x 72 = 384 x 168)
constexpr int LAUNCH_REGS = 168, SLOT_REGS = 216, OTHER_REGS = 72;
constexpr uint32_t COL_S = 0, COL_O = 256;  // slot s: + 128 s
constexpr int PAGE_RING = 16;
// Units for an item's end: some 15000 cycles (instrumented) from its last weights to the next item's first scores, against
// 5500 of a 256-row item's tile.
constexpr int EXTRA = 3;

template <int DP, bool PAIR>
struct Cfg {
  static constexpr int ROWS = PAIR ? 256 : 128;
  static constexpr int BUF = KT * DP * 2;  // a tile of keys or values
  static constexpr int NBUF = DP == 64 ? 8 : PAIR ? 4 : 5;
  static constexpr int QBYTES = ROWS * DP * 2;
  static constexpr int SMEM = QBYTES + NBUF * BUF + 1024;  // + alignment; the schedule's sums follow
};

struct Shared {
  uint64_t full[8], empty[8], s_full[2], p_ready[2], q_full, q_free, seen, done;
  uint64_t scratch[32];
  uint32_t tmem;
  uint32_t page_ok[PAGE_RING][4];
  int dirty[2][2];  // item parity, slot
  float m[2][TILE], l[2][TILE];
};

template <typename T>
__host__ __device__ constexpr uint32_t idesc(int n, bool b_mn) {
  return (1u << 4) | ((std::is_same<T, __half>::value ? 0u : 1u) << 7) | ((std::is_same<T, __half>::value ? 0u : 1u) << 10) |
         ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(TILE >> 4) << 24);
}

// Low word of a shared-memory descriptor: start address, and for an MN-major operand the distance `lbo` between its
// 64-element blocks. The high word is the same for all: 8-row groups 1024 bytes apart, version 1, 128-byte swizzle.
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t lbo) { return (saddr >> 4) | (lbo >> 4) << 16; }
constexpr uint32_t DESC_HI = (1024u >> 4) | 1u << 14 | 2u << 29;

// One product step, issued by the lane whose `leader` is set; the warp stays together, so that the operands stay in
// uniform registers (a branch to one lane made an issue cost 100-300 cycles instead of the product's 64).
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t acc, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "mov.b64 da, {%1, %6};\n\tmov.b64 db, {%2, %6};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(id), "r"(acc), "r"(leader), "r"(DESC_HI)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t acc, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "mov.b64 db, {%2, %6};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(id), "r"(acc), "r"(leader), "r"(DESC_HI)
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar)),
      "r"(leader)
      : "memory");
}
// Bounded wait that reads the timer only when the phase is late (a read costs some 300 cycles). `debug` (the test hook): the limit
// is 20 ms instead of 2 s. (Asking for it before the loop, at every wait, cost 5 to 11% of a call.)
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, int debug) {
  const uint32_t a = smem_u32(bar);
#pragma unroll 1
  for (int i = 0; i < 256; ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(done)
        : "r"(a), "r"(parity), "r"(10000u)
        : "memory");
    if (done) return true;
  }
  return mbar_wait(bar, parity, debug);
}
__device__ __forceinline__ void arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// 4D tiled tensor load; x times the element size is a multiple of 16 bytes, what lies outside the tensor reads as zeros
__device__ __forceinline__ void tma_load_4d(void* dst, const void* tmap, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(smem_u32(dst)),
      "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ bool try_now(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done;
}

#define EA_R8(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3]), "=r"(v[i + 4]), "=r"(v[i + 5]), "=r"(v[i + 6]), "=r"(v[i + 7])
#define EA_I8(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]), "r"(v[i + 4]), "r"(v[i + 5]), "r"(v[i + 6]), "r"(v[i + 7])
// 32 consecutive columns of this thread's lane
__device__ __forceinline__ void ld32(uint32_t addr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : EA_R8(v, 0), EA_R8(v, 8), EA_R8(v, 16), EA_R8(v, 24)
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void ld16(uint32_t addr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : EA_R8(v, 0), EA_R8(v, 8)
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void st16(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      EA_I8(v, 0), EA_I8(v, 8)
      : "memory");
}
__device__ __forceinline__ void st32(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      EA_I8(v, 0), EA_I8(v, 8), EA_I8(v, 16), EA_I8(v, 24)
      : "memory");
}
#define EA_W8(v, i) "+r"(v[i]), "+r"(v[i + 1]), "+r"(v[i + 2]), "+r"(v[i + 3]), "+r"(v[i + 4]), "+r"(v[i + 5]), "+r"(v[i + 6]), "+r"(v[i + 7])
// waits for this thread's loads; the 16 registers are named so that nothing reads them earlier
__device__ __forceinline__ void wait_ld16(uint32_t* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : EA_W8(v, 0), EA_W8(v, 8)::"memory");
}
// -inf in the places whose bit is clear
__device__ __forceinline__ void hide16(uint32_t* v, uint32_t seen) {
#pragma unroll
  for (int e = 0; e < 16; ++e)
    if (!((seen >> e) & 1)) v[e] = 0xFF800000u;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two binary32 operations in one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint32_t pack2(float x, float y, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *(const uint32_t*)&h;
}
__device__ __forceinline__ uint32_t pack2(float x, float y, __half) {
  const __half2 h = __floats2half2_rn(x, y);
  return *(const uint32_t*)&h;
}
template <int REGS, bool INC>
__device__ __forceinline__ void set_regs() {
  if (INC) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS));
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS));
}

// byte offset of (row, 16-byte piece) in a tile of `rows` rows of 64-channel blocks, 128-byte swizzle
__device__ __forceinline__ uint32_t tile_off(int row, int piece, int rows) {
  return (uint32_t)((piece >> 3) * rows * 128 + row * 128 + (((piece & 7) ^ (row & 7)) << 4));
}

// Bits of keys k0 .. k0 + 31 that token i of the item sees; tile pages aside.
__device__ __forceinline__ uint32_t seen_word(const Args& a, const Item& it, int i, int k0) {
  const int j0 = k0 - it.ctx;
  const auto low = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u; };
  uint32_t bits;
  if (j0 <= -32) {
    bits = 0xFFFFFFFFu;
  } else if (!a.t.tree_mask) {
    bits = low(i + 1 - j0);
  } else {
    const uint32_t* row = (const uint32_t*)a.t.tree_mask + (int64_t)(it.q0 + i) * a.t.mask_words;
    const auto word = [&](int w) { return w >= 0 && w < a.t.mask_words ? row[w] : 0u; };
    if (j0 >= 0) bits = __funnelshift_r(word(j0 >> 5), word((j0 >> 5) + 1), j0 & 31);
    else bits = (word(0) << -j0) | low(-j0);
  }
  return bits & low(it.len - k0);
}

template <typename T>
__device__ __forceinline__ bool pair_not_finite(uint32_t v) {
  constexpr uint32_t EXP = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
  return (v & EXP) == EXP || (v & EXP << 16) == EXP << 16;
}

// Zeroes the infinities and NaN of one row of a value tile; whether there were any.
template <typename T, int DP>
__device__ __noinline__ bool clean_row(uint8_t* buf, int row) {
  constexpr uint32_t EXP = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
  bool any = false;
  for (int p = 0; p < DP / 8; ++p) {
    uint32_t* w = (uint32_t*)(buf + tile_off(row, p, KT));
    for (int e = 0; e < 4; ++e) {
      uint32_t v = w[e];
      if (!pair_not_finite<T>(v)) continue;
      any = true;
      if ((v & EXP) == EXP) v &= 0xFFFF0000u;
      if ((v & EXP << 16) == EXP << 16) v &= 0xFFFFu;
      w[e] = v;
    }
  }
  return any;
}

// Adds to acc (channels c0 ..) the infinities and NaN of the values of keys first .. last - 1 that token i sees, as far as
// their tiles were cleaned: from the tile on that holds the first drafted key.
template <typename T, int N>
__device__ __noinline__ void add_not_finite(const Args& a, const Item& it, int i, int first, int last, int c0, float* acc) {
  for (int k = max(first, max(it.ctx, 0) / KT * KT); k < min(last, it.len); ++k) {
    if (!((seen_word(a, it, i, k)) & 1)) continue;
    const uint32_t col = div_by((uint32_t)k, a.by_page);
    const int page = a.t.page_table[it.b * a.t.table_stride + col];
    if (page < 0 || page >= a.t.num_pages) continue;
    const T* v = (const T*)a.t.v_cache + (int64_t)page * a.t.v_page_stride + it.h * a.t.v_head_stride +
                 (k - (int64_t)col * a.t.page_size) * a.t.v_row_stride;
    for (int c = 0; c < N; ++c) {
      if (c0 + c >= a.t.d) break;
      const float f = to_f(v[c0 + c]);
      if (!isfinite(f)) acc[c] += f;
    }
  }
}

template <typename T, int DP, bool PAIR>
__global__ void __launch_bounds__(THREADS, 1)
    many_rows_kernel(Args a, const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, int box) {
  using C = Cfg<DP, PAIR>;
  constexpr int ROWS = C::ROWS, NBUF = C::NBUF, BUF = C::BUF;
  extern __shared__ uint8_t raw[];
  __shared__ Shared sh;
  uint8_t* base = (uint8_t*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  uint8_t* qbuf = base;
  uint8_t* ring = base + C::QBYTES;
  uint32_t* sums = (uint32_t*)(raw + C::SMEM);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  if (tid == 0) {
    for (int i = 0; i < NBUF; ++i) mbar_init(&sh.full[i], box ? 1 : LOADERS), mbar_init(&sh.empty[i], 1);
    for (int s = 0; s < 2; ++s) mbar_init(&sh.s_full[s], 1), mbar_init(&sh.p_ready[s], SLOT_THREADS);
    mbar_init(&sh.q_full, 32), mbar_init(&sh.q_free, 1), mbar_init(&sh.seen, 2 * SLOT_THREADS);
    mbar_init(&sh.done, 1);
    sh.dirty[0][0] = sh.dirty[0][1] = sh.dirty[1][0] = sh.dirty[1][1] = 0;
  }
  if (warp == 8) tmem_alloc(&sh.tmem, 512);
  begin();
  Schedule<ROWS, KT, EXTRA> sch;
  sch.build(a, sums, sh.scratch);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = sh.tmem;
  uint32_t pos = sch.share(blockIdx.x);
  const uint32_t end = sch.share(blockIdx.x + 1);
  bool alive = true;  // false once a bounded wait gave up: no more waits, products or copies; the rows become NaN

  // order in which the tiles are loaded and used: PAIR K0, then V(t), K(t + 1); else K0, K1, then V(t), K(t + 2)
  constexpr int AHEAD = PAIR ? 1 : 2;
  if (warp >= 8) set_regs<OTHER_REGS, false>();
  if (warp == (box ? 10 : 9)) {
    // ---- query rows of the next item, as soon as the last scores of this one are computed
    uint32_t items = 0;
    while (pos < end && alive) {
      const Item it = sch.item(a, pos, end);
      pos = it.next;
      if (it.kt0 >= it.kt1) continue;
      if (items) alive = __all_sync(0xffffffffu, wait_phase(&sh.q_free, (items - 1) & 1, a.wait_debug));
      if (!alive) break;
      ++items;
      constexpr int PIECES = DP / 8;
      const int rows = min(ROWS, it.new_tokens * a.group - it.m * ROWS);
#pragma unroll 4
      for (int e = lane; e < rows * PIECES; e += 32) {
        const int r = e / PIECES, p = e % PIECES, R = it.m * ROWS + r, tok = (int)div_by((uint32_t)R, a.by_group);
        const T* q = (const T*)a.t.q + (int64_t)(it.q0 + tok) * a.t.q_stride +
                     (int64_t)(it.h * a.group + R - tok * a.group) * a.t.q_head_stride + p * 8;
        const bool in = p * 8 < a.t.d;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(qbuf) + tile_off(r, p, ROWS)),
                     "l"(in ? (const void*)q : a.t.q), "r"(in ? 16 : 0)
                     : "memory");
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      if (a.t.alpha <= 0)  // the slots work with |alpha|, and with 1 for 0
        for (int e = lane; e < rows * PIECES; e += 32) {
          uint32_t* w = (uint32_t*)(qbuf + tile_off(e / PIECES, e % PIECES, ROWS));
          for (int i = 0; i < 4; ++i) w[i] = a.t.alpha < 0 ? w[i] ^ 0x80008000u : 0u;
        }
      fence_async_smem();
      if (!a.wait_debug) arrive(&sh.q_full);  // with the hook what waits for this, and all that waits for that, runs out
    }
  } else if (warp >= 9 && box) {
    // ---- loader warp, tensor copies: a lane issues one box (64 channels x `box` rows of one page) of every tile
    if (warp == 9) {
      constexpr int CB = DP / 64;
      const int sub = lane / CB, cb = lane % CB;
      const bool active = sub * box < KT;
      uint32_t cnt = 0, tile0 = 0;  // tiles loaded; key tiles of earlier items
      while (pos < end && alive) {
        const Item it = sch.item(a, pos, end);
        pos = it.next;
        if (it.kt0 >= it.kt1) continue;
        const int n = it.kt1 - it.kt0;
        const auto page_of = [&](int t) {
          const int key = (it.kt0 + t) * KT + sub * box;
          if (!active || t >= n || key >= it.len) return -1;
          const int p = a.t.page_table[it.b * a.t.table_stride + div_by((uint32_t)key, a.by_page)];
          return p >= 0 && p < a.t.num_pages ? p : -1;
        };
        const auto load = [&](int t, int page, bool value) {
          const uint32_t b = cnt % NBUF;
          if (cnt >= NBUF) alive = __all_sync(0xffffffffu, wait_phase(&sh.empty[b], (cnt / NBUF - 1) & 1, a.wait_debug));
          if (!alive) return;
          if (!value) {  // which of the tile's keys have a page
            const uint32_t bits = page < 0 ? 0u : box >= 32 ? 0xFFFFFFFFu : ((1u << box) - 1) << (sub * box & 31);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const bool here = active && sub * box < (w + 1) * 32 && (sub + 1) * box > w * 32;
              const uint32_t all = __reduce_or_sync(0xffffffffu, here ? bits : 0u);
              if (lane == 0) sh.page_ok[(tile0 + t) % PAGE_RING][w] = all;
            }
          }
          if (lane == 0) mbar_arrive_expect_tx(&sh.full[b], BUF);
          __syncwarp();
          if (active) {
            const int key = (it.kt0 + t) * KT + sub * box;
            const int row = page < 0 ? 0 : key - (int)div_by((uint32_t)key, a.by_page) * a.t.page_size;
            tma_load_4d(ring + b * BUF + cb * KT * 128 + sub * box * 128, value ? &tv : &tk, cb * 64, row, it.h,
                        page < 0 ? (int)a.t.num_pages : page, &sh.full[b]);
          }
          ++cnt;
        };
        int page[AHEAD + 1], next = page_of(AHEAD);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) page[i] = page_of(i);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
          if (i < n && alive) load(i, page[i], false);
        for (int t = 0; t < n && alive; ++t) {
          page[AHEAD] = next;
          next = page_of(t + AHEAD + 1);
          load(t, page[0], true);
          if (t + AHEAD < n && alive) load(t + AHEAD, page[AHEAD], false);
#pragma unroll
          for (int i = 0; i < AHEAD; ++i) page[i] = page[i + 1];
        }
        tile0 += n;
      }
      // copies under way land before the block gives its shared memory back
      for (uint32_t c = cnt > NBUF ? cnt - NBUF : 0; c < cnt; ++c) mbar_wait(&sh.full[c % NBUF], (c / NBUF) & 1);
    }
  } else if (warp >= 10) {
    // ---- loaders, any page size: every thread copies 16-byte pieces of every tile; a lane looks up the pages of two keys
    const int w2 = warp - 10;
    uint32_t cnt = 0, pending = 0, signalled = 0, tile0 = 0;  // tile0: tiles of earlier items
    const auto retire = [&]() {  // waits for the oldest tile in flight and hands it over
      switch (pending) {
        case 1: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
        case 2: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
        case 3: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
        case 4: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
        case 5: asm volatile("cp.async.wait_group 4;" ::: "memory"); break;
        case 6: asm volatile("cp.async.wait_group 5;" ::: "memory"); break;
        case 7: asm volatile("cp.async.wait_group 6;" ::: "memory"); break;
        default: asm volatile("cp.async.wait_group 7;" ::: "memory"); break;
      }
      fence_async_smem();
      arrive(&sh.full[signalled % NBUF]);
      ++signalled, --pending;
    };
    while (pos < end && alive) {
      const Item it = sch.item(a, pos, end);
      pos = it.next;
      if (it.kt0 >= it.kt1) continue;
      const int n = it.kt1 - it.kt0;
      const auto page_of = [&](int t, int half) {
        const int key = (it.kt0 + t) * KT + w2 * 64 + half * 32 + lane;
        if (t >= n || key >= it.len) return -1;
        const int p = a.t.page_table[it.b * a.t.table_stride + div_by((uint32_t)key, a.by_page)];
        return p >= 0 && p < a.t.num_pages ? p : -1;
      };
      const auto load = [&](int t, bool value) {
        const uint32_t b = cnt % NBUF;
        if (cnt >= NBUF) {
          const uint32_t parity = (cnt / NBUF - 1) & 1;
          while (pending && !__all_sync(0xffffffffu, try_now(&sh.empty[b], parity))) retire();
          alive = __all_sync(0xffffffffu, wait_phase(&sh.empty[b], parity, a.wait_debug));
          if (!alive) return;
        }
        if (pending == 7) retire();
        const uint32_t dst = smem_u32(ring + b * BUF);
        const T* src = (const T*)(value ? a.t.v_cache : a.t.k_cache) + it.h * (value ? a.t.v_head_stride : a.t.k_head_stride);
        const int64_t ps = value ? a.t.v_page_stride : a.t.k_page_stride, rs = value ? a.t.v_row_stride : a.t.k_row_stride;
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          const int row0 = w2 * 64 + half * 32, key0 = (it.kt0 + t) * KT + row0;
          const int page = page_of(t, half);
          if (!value) {
            const uint32_t ok = __ballot_sync(0xffffffffu, page >= 0);
            if (lane == 0) sh.page_ok[(tile0 + t) % PAGE_RING][row0 / 32] = ok;
          }
#pragma unroll 2
          for (int q = 0; q < 8; ++q) {
            const int r = q * 4 + lane / 8;
            const int pg = __shfl_sync(0xffffffffu, page, r);
            const int key = key0 + r;
            const int64_t off = pg >= 0 ? key - (int64_t)div_by((uint32_t)key, a.by_page) * a.t.page_size : 0;
            const T* row = src + (pg >= 0 ? pg : 0) * ps + off * rs;
#pragma unroll
            for (int c = 0; c < DP / 64; ++c) {
              const int piece = c * 8 + (lane & 7);
              const bool in = pg >= 0 && piece * 8 < a.t.d;
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + tile_off(row0 + r, piece, KT)),
                           "l"(in ? (const void*)(row + piece * 8) : (value ? a.t.v_cache : a.t.k_cache)), "r"(in ? 16 : 0)
                           : "memory");
            }
          }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        ++cnt, ++pending;
      };
      for (int i = 0; i < AHEAD; ++i)
        if (i < n && alive) load(i, false);
      for (int t = 0; t < n && alive; ++t) {
        load(t, true);
        if (t + AHEAD < n && alive) load(t + AHEAD, false);
      }
      tile0 += n;
    }
    while (pending) retire();
  } else if (warp >= 8) {
    // ---- products, one lane issues them. One issuer for both slots keeps the slots half a cycle apart; with an issuer each
    // they ran in step and waited for the same pipes at the same time (6000 cycles for a pair of tiles against 4600).
    if (warp == 8) {
      constexpr uint32_t QK = idesc<T>(KT, false), PV = idesc<T>(DP, true);
      const uint32_t leader = lane == 0;
      uint32_t cnt = 0, items = 0, phases = 0;  // tiles taken from the ring; items; bit s: parity of slot s's weights
      const uint32_t qd = desc_lo(smem_u32(qbuf), 16), ring_at = smem_u32(ring);
      const auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (alive) alive = __all_sync(0xffffffffu, wait_phase(bar, parity, a.wait_debug));
      };
      while (pos < end && alive) {
        const Item it = sch.item(a, pos, end);
        pos = it.next;
        if (it.kt0 >= it.kt1) continue;
        const int n = it.kt1 - it.kt0;
        const int slots = !PAIR || it.new_tokens * a.group - it.m * ROWS > TILE ? 2 : 1;  // PAIR: slots with rows
        if (items) wait(&sh.seen, (items - 1) & 1);  // the slots have seen the end of the last item
        wait(&sh.q_full, items & 1);
        ++items;
        // A step: the weights of tile t times its values, then the scores of tile t + AHEAD into the same slot, then
        // the word to the slot. PAIR: both slots take every tile; else the slot is the tile's parity.
        const int steps = (n + AHEAD) * (PAIR ? 2 : 1);
#pragma unroll 1
        for (int i = 0; i < steps && alive; ++i) {
          const int t = (PAIR ? i >> 1 : i) - AHEAD, slot = i & 1;
          const bool idle = slot >= slots, first = !PAIR || slot == 0, last = !PAIR || slot == 1;
          const uint32_t s_cols = tmem + COL_S + slot * 128;
          const bool more = t + AHEAD < n;
          const uint32_t cv = cnt, ck = PAIR && t >= 0 ? cnt + 1 : cnt;  // ring positions of V(t) and K(t + AHEAD)
          if (t >= 0) {
            if (first) wait(&sh.full[cv % NBUF], (cv / NBUF) & 1);
            if (!idle) {
              wait(&sh.p_ready[slot], phases >> slot & 1);
              phases ^= 1u << slot;
              fence_after_sync();
            }
            if (!alive) break;
            if (!idle) {
              const uint32_t v = desc_lo(ring_at + (cv % NBUF) * BUF, KT * 128), o = tmem + COL_O + slot * 128;
              const uint32_t acc = t >= AHEAD;
#pragma unroll
              for (int k = 0; k < KT / 16; ++k) mma_ts(o, s_cols + k * 8, v + k * 128, PV, k ? 1u : acc, leader);
            }
            if (last) commit(&sh.empty[cv % NBUF], leader);
            if (!PAIR) ++cnt;
          }
          if (more) {
            const uint32_t c = PAIR ? ck : cnt;
            if (first) wait(&sh.full[c % NBUF], (c / NBUF) & 1);
            if (!alive) break;
            if (!idle) {
              const uint32_t q = qd + (PAIR ? slot * TILE * 8 : 0), kd = desc_lo(ring_at + (c % NBUF) * BUF, 16);
#pragma unroll
              for (int k = 0; k < DP / 16; ++k)
                mma_ss(s_cols, q + (k >> 2) * ROWS * 8 + (k & 3) * 2, kd + (k >> 2) * KT * 8 + (k & 3) * 2, QK, k > 0, leader);
            }
            if (last) commit(&sh.empty[c % NBUF], leader);
            if (last && t + AHEAD == n - 1) commit(&sh.q_free, leader);
            if (!PAIR) ++cnt;
          }
          if (PAIR && slot == 1) cnt += (t >= 0) + more;
          if (!idle || t < 0) commit(&sh.s_full[slot], leader);
        }
      }
      // what has been issued completes before the block frees its tensor memory
      commit(&sh.done, leader);
      mbar_wait(&sh.done, 0);
    }
    __syncwarp();
  } else {
    // ---- softmax slots
    set_regs<SLOT_REGS, true>();
    const int slot = warp >> 2, r = tid & (TILE - 1);
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_addr = lanes + COL_S + slot * 128, o_addr = lanes + COL_O + slot * 128;
    const float scale_s = a.t.alpha == 0 ? 1.0f : fabsf(a.t.alpha);
    uint32_t ns = 0, first = 0, items = 0;  // phases of s_full seen; ring position of the item's first tile; items
    const auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (alive) alive = __all_sync(0xffffffffu, wait_phase(bar, parity, a.wait_debug));
    };
    while (pos < end) {
      const Item it = sch.item(a, pos, end);
      pos = it.next;
      if (it.kt0 >= it.kt1) continue;
      const int n = it.kt1 - it.kt0;
      const int all_rows = it.new_tokens * a.group - it.m * ROWS;
      const int rows = min(TILE, all_rows - (PAIR ? slot * TILE : 0));  // of this slot's tile; may be <= 0 for PAIR
      const int R = it.m * ROWS + (PAIR ? slot * TILE : 0) + min(r, max(rows, 1) - 1);
      const int tok = (int)div_by((uint32_t)R, a.by_group);
      const bool warp_rows = (r & ~31) < rows;
      const int tiles = PAIR ? (rows > 0 ? n : 0) : (n + 1 - slot) / 2;
      float m = -INFINITY, l = 0.0f;
      for (int i = 0; i < tiles; ++i) {
        const int t = PAIR ? i : 2 * i + slot;
        const int key0 = (it.kt0 + t) * KT;
        wait(&sh.s_full[slot], ns++ & 1);
        fence_after_sync();
        const uint32_t* ok = sh.page_ok[(first / 2 + t) % PAGE_RING];
        const bool masked = key0 + KT > it.ctx || (ok[0] & ok[1] & ok[2] & ok[3]) != 0xFFFFFFFFu;
        if (warp_rows && alive) {
          uint32_t vis[KT / 32];
          if (masked) {
#pragma unroll
            for (int c = 0; c < KT / 32; ++c) vis[c] = seen_word(a, it, tok, key0 + c * 32) & ok[c];
          }
          // One pass in the common case (a first pass for the maximum alone cost 500 cycles of a tile's 2650; holding the whole
          // tile's scores in registers spilled): the weights against the maximum so far, while the tile's own is taken.
          // They are stored, over the scores, only if no row's reference moved; else O is rescaled and a second pass
          // computes them anew. A slot's first tile takes its maximum before.
          uint32_t u[2][16], p[KT / 2];
          float2 sum[2];
          float mx[2] = {-INFINITY, -INFINITY};
          // calls f(c, scores of columns 16 c ..), the next columns on their way
          const auto columns = [&](auto f) {
            ld16(s_addr, u[0]);
#pragma unroll
            for (int c = 0; c < KT / 16; ++c) {
              uint32_t* v = u[c & 1];
              wait_ld16(v);
              if (c + 1 < KT / 16) ld16(s_addr + (c + 1) * 16, u[(c + 1) & 1]);
              if (masked) hide16(v, vis[c >> 1] >> (c & 1) * 16);
              f(c, v);
            }
          };
          if (i == 0) {
            columns([&](int, const uint32_t* v) {
#pragma unroll
              for (int e = 0; e < 8; ++e) mx[e & 1] = max3(mx[e & 1], __uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1]));
            });
            m = fmaxf(mx[0], mx[1]) * scale_s - Reference<T>::DOWN;
          }
          for (int pass = 0; pass < 2; ++pass) {
            const float ref = m == -INFINITY ? 0.0f : m;
            const float2 sc = make_float2(scale_s, scale_s), sub = make_float2(-ref, -ref);
            mx[0] = mx[1] = -INFINITY;
            sum[0] = sum[1] = make_float2(0.0f, 0.0f);
            columns([&](int c, const uint32_t* v) {
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                float2 x = make_float2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1]));
                mx[e & 1] = max3(mx[e & 1], x.x, x.y);
                x = fma2(x, sc, sub);
                x.x = ex2(x.x), x.y = ex2(x.y);
                sum[e & 1] = add2(sum[e & 1], x);
                p[c * 8 + e] = pack2(x.x, x.y, T());
              }
            });
            const float top = fmaxf(mx[0], mx[1]) * scale_s;
            const bool grow = Reference<T>::passed(top, m);
            if (!__any_sync(0xffffffffu, grow)) break;
            const float to = top - Reference<T>::DOWN, f = grow ? (m == -INFINITY ? 0.0f : ex2(m - to)) : 1.0f;
            if (grow) m = to;
            l *= f;
            if (i > 0) {
#pragma unroll 1
              for (int c = 0; c < DP / 16; ++c) {
                uint32_t o[16];
                ld16(o_addr + c * 16, o);
                wait_ld16(o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                st16(o_addr + c * 16, o);
              }
            }
          }
          st32(s_addr, p);
          st32(s_addr + 32, p + 32);
          l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
          tmem_wait_st();
        }
        // Drafted keys, and rows behind the last key: their infinities and NaN may not meet the zero weight of a row
        // that does not see them. The tile's whole rows are cleaned, earlier keys' too; rows that see them get them back at the end.
        if (key0 + KT > it.ctx && (!PAIR || slot == 0)) {
          const uint32_t c = first + (PAIR ? 1 + 2 * t : n == 1 ? 1 : 2 + t + min(t, n - 2));
          wait(&sh.full[c % NBUF], (c / NBUF) & 1);
          if (alive && clean_row<T, DP>(ring + (c % NBUF) * BUF, r) && key0 + r < it.len) sh.dirty[items & 1][slot] = 1;
          fence_async_smem();
        }
        fence_before_sync();
        arrive(&sh.p_ready[slot]);
      }
      wait(&sh.s_full[slot], ns++ & 1);  // the slot's products are done
      fence_after_sync();
      arrive(&sh.seen);
      first += 2 * n;

      // join the slots (PAIR: each has rows of its own) and write the rows
      if (!alive) l = NAN;
      const bool whole = it.kt0 == 0 && it.kt1 == it.tiles;
      float ml[2] = {m, m}, ll[2] = {l, 0.0f};
      if (!PAIR) {
        sh.m[slot][r] = m, sh.l[slot][r] = l;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        ml[0] = sh.m[0][r], ml[1] = sh.m[1][r], ll[0] = sh.l[0][r], ll[1] = sh.l[1][r];
      } else {
        asm volatile("bar.sync 1, 256;" ::: "memory");
      }
      const bool dirty = sh.dirty[items & 1][0] || sh.dirty[items & 1][1];
      ++items;
      if (r == 0) sh.dirty[items & 1][slot] = 0;
      const float mm = fmaxf(ml[0], ml[1]), ref = mm == -INFINITY ? 0.0f : mm;
      const float f0 = exp2f(ml[0] - ref), f1 = PAIR || n < 2 ? 0.0f : exp2f(ml[1] - ref);
      const float lsum = ll[0] * f0 + ll[1] * (PAIR ? 0.0f : exp2f(ml[1] - ref));
      const bool mine = r < rows;
      const int64_t head = (int64_t)(it.q0 + tok) * a.t.q_heads + it.h * a.group + (R - tok * a.group);
      const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;
      float* part = slot_of(a, 2 * blockIdx.x + (it.kt0 == 0 ? 1 : 0), ROWS);
      const int pr = (PAIR ? slot * TILE : 0) + r;
      constexpr int COLS = PAIR ? DP : DP / 2;
      const int c0 = PAIR ? 0 : slot * COLS;
      if (warp_rows) {
#pragma unroll
        for (int c = 0; c < COLS / 32; ++c) {
          uint32_t u[32];
          float o[32];
          ld32(lanes + COL_O + (PAIR ? slot * 128 : 0) + c0 + c * 32, u);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __uint_as_float(u[e]) * f0;
          if (!PAIR && n > 1) {
            ld32(lanes + COL_O + 128 + c0 + c * 32, u);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = fmaf(__uint_as_float(u[e]), f1, o[e]);
          }
          const int ch = c0 + c * 32;
          if (mine && dirty) {
            float extra[32];
            for (int e = 0; e < 32; ++e) extra[e] = 0.0f;
            add_not_finite<T, 32>(a, it, tok, it.kt0 * KT, it.kt1 * KT, ch, extra);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] += extra[e];
          }
          if (mine && whole) {
            T* dst = (T*)a.t.out + head * a.t.d + ch;
#pragma unroll
            for (int p = 0; p < 4; ++p) {
              uint4 y;
              uint32_t* yw = (uint32_t*)&y;
#pragma unroll
              for (int e = 0; e < 4; ++e) yw[e] = pack2(o[p * 8 + 2 * e] * inv, o[p * 8 + 2 * e + 1] * inv, T());
              if (ch + p * 8 < a.t.d) *(uint4*)(dst + p * 8) = y;
            }
          } else if (mine) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *(float4*)(part + ((ch + e) * ROWS + pr * 4)) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
          __syncwarp();
        }
      }
      if (mine && (PAIR || slot == 0)) {
        if (whole) {
          if (a.t.lse) a.t.lse[head] = lsum == 0.0f ? -INFINITY : mm + log2f(lsum);
        } else {
          part[ROWS * DP + pr] = mm, part[ROWS * (DP + 1) + pr] = lsum;
        }
      }
      fence_before_sync();
      asm volatile("bar.sync 1, 256;" ::: "memory");  // m, l and dirty are read; O is free
    }
  }
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  if (warp == 8) tmem_free(tmem, 512);
}

}  // namespace many
}  // namespace tree
}  // namespace serving
}  // namespace ea
