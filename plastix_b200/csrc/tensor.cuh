// The tensor cores' instructions (tcgen05), their memory (TMEM) and tensor copies
// (TMA), as far as product_tensor.cu and recurrence.cu use them.
#pragma once

#include <cuda.h>

#include "common.cuh"

namespace plx {

// ---- tensor copies -----------------------------------------------------------
// A map of `outer` rows of `inner` values, `ld` apart (start and stride multiples of
// 16 bytes), for copies of boxes; what is outside reads as 0. swizzle: 16-byte chunks
// of rows of 128 bytes as the products take them.
int tensor_map(CUtensorMap* map, int dtype, const void* p, uint64_t inner, uint64_t outer,
               int64_t ld, uint32_t box_inner, uint32_t box_outer, bool swizzle);

// A box of a two-dimensional array to shared memory; x (values into a row) times
// their size is a multiple of 16 bytes.
__device__ __forceinline__ void tensor_load(void* dst_smem, const CUtensorMap* map, int x, int y,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(smem_addr(dst_smem)),
      "l"(map), "r"(x), "r"(y), "r"(smem_addr(bar))
      : "memory");
}

// The same for a pair of blocks whose products are issued together: `bar` (an
// address as peer_smem gives) may be the other block's.
__device__ __forceinline__ void tensor_load_pair(void* dst_smem, const CUtensorMap* map, int x,
                                                 int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(smem_addr(dst_smem)),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

// A box from shared memory to the array (what is outside stays as it is); bulk_commit
// and bulk_wait_read or bulk_wait_all by the same thread.
__device__ __forceinline__ void tensor_store(const CUtensorMap* map, int x, int y,
                                             const void* src_smem) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   map),
               "r"(x), "r"(y), "r"(smem_addr(src_smem))
               : "memory");
}

// ---- tensor memory -----------------------------------------------------------
// Columns (a power of two from 32) for the block, their address to `to`; by one
// whole warp, which gives them back as well. PAIR: by both blocks of a pair.
template <bool PAIR>
__device__ __forceinline__ void tmem_alloc(uint32_t* to, uint32_t columns) {
  if constexpr (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_addr(to)),
                 "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_addr(to)),
                 "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
}
template <bool PAIR>
__device__ __forceinline__ void tmem_free(uint32_t at, uint32_t columns) {
  if constexpr (PAIR)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns));
  else
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns));
}
__device__ __forceinline__ void tmem_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tmem_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// 32 (16) columns of the warp's 32 lanes: a lane's values to its thread.
__device__ __forceinline__ void tmem_load32(uint32_t at, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
      "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_load16(uint32_t at, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(at));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// ---- products ----------------------------------------------------------------
// An operand in shared memory, in rows of 128 bytes whose 16-byte chunks are
// swizzled as the tensor copy leaves them (eight rows, 1,024 bytes, a group):
// rows over i and a row's values over k, groups 1,024 bytes apart ...
__device__ __forceinline__ uint64_t operand_k_major(const void* at) {
  return (uint64_t)((smem_addr(at) & 0x3FFFF) >> 4) | (uint64_t)1 << 16 |
         (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// ... or rows over k and a row's values over i: 64 of them, the next 64 `apart`
// bytes further on.
__device__ __forceinline__ uint64_t operand_i_major(const void* at, uint32_t apart) {
  return (uint64_t)((smem_addr(at) & 0x3FFFF) >> 4) | (uint64_t)(apart >> 4) << 16 |
         (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// What is multiplied: m (128, or 256 by a pair of blocks) x n values of 16 bits, sums
// in 32 bits. Both operands are of one type.
inline uint32_t product_kind(bool bf16, bool a_i_major, bool b_i_major, uint32_t m, uint32_t n) {
  return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (a_i_major ? 1u << 15 : 0u) |
         (b_i_major ? 1u << 16 : 0u) | (n >> 3) << 17 | (m >> 4) << 24;
}
// Adds the products over 16 values of k to (or, first, puts them in) TMEM. PAIR: each
// block has half of a's rows, of b's and of the sums' rows; one of the two issues.
template <bool PAIR>
__device__ __forceinline__ void tensor_product(uint32_t at, uint64_t a, uint64_t b, uint32_t kind,
                                               bool add) {
  if constexpr (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(at),
        "l"(a), "l"(b), "r"(kind), "r"((uint32_t)add)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(at),
        "l"(a), "l"(b), "r"(kind), "r"((uint32_t)add)
        : "memory");
}
// Arrives at the barrier (PAIR: at both blocks') once the products issued before are
// done.
template <bool PAIR>
__device__ __forceinline__ void products_arrive(uint64_t* bar) {
  if constexpr (PAIR)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
        "[%0], %1;" ::"r"(smem_addr(bar)),
        "h"((uint16_t)3)
        : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
            smem_addr(bar))
        : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}

}  // namespace plx
