// CTA-pair (cta_group::2) building blocks of the dense tcgen05 kernels: cluster addressing, TMA
// into a pair, paired MMAs and their descriptors. Included by files that record no trace stamps.
#pragma once

#include "ptx.cuh"

namespace muse {

constexpr int kWaitFailed = 8;  // device status of an expired wait in a dense product

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// As cluster_sync, without ordering memory: before a CTA's shared and tensor memory go. (A release
// would wait ~1000 clocks for the outputs' stores.)
__device__ __forceinline__ void cluster_sync_relaxed() {
  asm volatile("barrier.cluster.arrive.relaxed;\n\tbarrier.cluster.wait;" ::: "memory");
}
// Address of the same shared-memory object in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t map_rank(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(ptx::smem_u32(p)), "r"(rank));
  return r;
}
// Arrive on a barrier of either CTA. What it announces is ordered by the fence that precedes it
// (fence.proxy.async for operands in shared memory, tcgen05.fence for tensor memory reads); a
// release at cluster scope would also wait ~1300 clocks for this thread's earlier stores.
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// TMA box into this CTA's shared memory, completing on a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void prefetch_l2(const void* p) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}
// A 2-D box into L2 only.
__device__ __forceinline__ void prefetch_tile(const CUtensorMap* map, int c0, int c1) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1)
               : "memory");
}
// Contiguous bytes into L2 only (address and size multiples of 16).
__device__ __forceinline__ void prefetch_bulk(const void* p, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// Store 32 consecutive 32-bit columns of this thread's lane.
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// Arrive on `bar` of both CTAs of the pair (`mask`: their bits in the cluster) once this thread's MMAs
// so far have completed.
__device__ __forceinline__ void commit_pair(uint64_t* bar, uint32_t mask = 3) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          ptx::smem_u32(bar)),
      "h"((uint16_t)mask)
      : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}

// 16 accumulator rows (tensor-memory lanes) x 32 columns, as the fragments of four 16 x 8 blocks:
// v[4 b + i] is row lane / 4 + 8 (i / 2), column 8 b + 2 (lane % 4) + i % 2.
__device__ __forceinline__ void tmem_ld_frag(uint32_t taddr, float (&v)[16]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
// Two 8 x 8 blocks of 16-bit pairs (fragments as above) to and from shared memory, transposed: the
// address of lane l (l < 16) is the 16-byte row that holds column l % 8 of block l / 8.
__device__ __forceinline__ void stmatrix2_t(uint32_t addr, uint32_t a, uint32_t b) {
  asm volatile("stmatrix.sync.aligned.m8n8.x2.trans.shared.b16 [%0], {%1, %2};" ::"r"(addr), "r"(a), "r"(b) : "memory");
}
__device__ __forceinline__ void ldmatrix2_t(uint32_t addr, uint32_t& a, uint32_t& b) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0, %1}, [%2];" : "=r"(a), "=r"(b) : "r"(addr) : "memory");
}

// Shared-memory descriptors, 128-byte swizzle. K-major: rows of 64 k, 8-row groups 1024 B apart.
// MN-major: boxes of 64 (m or n) x 64 k, 8192 B apart (the leading offset); 8-k groups 1024 B
// apart (the stride offset).
template <bool kMn>
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
  uint64_t d = (uint64_t)((addr & 0x3FFFF) >> 4);
  d |= (uint64_t)((kMn ? 8192u : 16u) >> 4) << 16;
  d |= (uint64_t)(1024u >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
// Descriptor step of 16 k (in 16-byte units).
template <bool kMn>
constexpr uint32_t kStepDesc = kMn ? 16 * 128 / 16 : 2;

// What differs between a CTA on its own (kCtas = 1) and a pair (2): tensor-memory allocation, the
// MMAs (A from shared or tensor memory), their commits, TMA boxes, and where barriers live: those
// that a pair shares are its leader's. M is 128 per CTA.
template <int kCtas> struct Group;
#define MUSE_GROUP_OPS(G)                                                                                            \
  static __device__ __forceinline__ void alloc(uint32_t* dst, uint32_t cols) {                                      \
    asm volatile("tcgen05.alloc.cta_group::" G ".sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(ptx::smem_u32(dst)), \
                 "r"(cols) : "memory");                                                                             \
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::" G ".sync.aligned;" ::: "memory");                    \
  }                                                                                                                 \
  static __device__ __forceinline__ void dealloc(uint32_t taddr, uint32_t cols) {                                   \
    asm volatile("tcgen05.dealloc.cta_group::" G ".sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");   \
  }                                                                                                                 \
  static __device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {    \
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"                                                 \
                 "tcgen05.mma.cta_group::" G ".kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),       \
                 "r"(idesc), "r"(acc) : "memory");                                                                  \
  }                                                                                                                 \
  /* A in tensor memory: each CTA's 128 rows, 16 k in eight columns of 16-bit pairs */                              \
  static __device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) { \
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"                                                 \
                 "tcgen05.mma.cta_group::" G ".kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b),     \
                 "r"(idesc), "r"(acc) : "memory");                                                                  \
  }                                                                                                                 \
  static __device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) { \
    asm volatile("cp.async.bulk.tensor.2d.cta_group::" G ".shared::cluster.global.mbarrier::complete_tx::bytes"     \
                 " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), \
                 "r"(bar) : "memory");                                                                              \
  }                                                                                                                 \
  static __device__ __forceinline__ void tma_4d(uint32_t dst, const CUtensorMap* map, int c0, int c3, uint32_t bar) { \
    asm volatile("cp.async.bulk.tensor.4d.cta_group::" G ".shared::cluster.global.mbarrier::complete_tx::bytes"     \
                 " [%0], [%1, {%2, %3, %3, %4}], [%5];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0),  \
                 "r"(0), "r"(c3), "r"(bar) : "memory");                                                             \
  }
template <> struct Group<1> {
  MUSE_GROUP_OPS("1")
  static __device__ __forceinline__ void commit(uint64_t* bar, uint32_t) { ptx::mma_commit(bar); }
  static __device__ __forceinline__ uint32_t shared_bar(uint64_t* bar, uint32_t) { return ptx::smem_u32(bar); }
  static __device__ __forceinline__ void arrive(uint64_t* bar, uint32_t) { ptx::mbar_arrive(bar); }
};
template <> struct Group<2> {
  MUSE_GROUP_OPS("2")
  static __device__ __forceinline__ void commit(uint64_t* bar, uint32_t mask) { commit_pair(bar, mask); }
  static __device__ __forceinline__ uint32_t shared_bar(uint64_t* bar, uint32_t leader) { return map_rank(bar, leader); }
  static __device__ __forceinline__ void arrive(uint64_t* bar, uint32_t leader) { arrive_cluster(map_rank(bar, leader)); }
};
#undef MUSE_GROUP_OPS

// A whole warp waits for a phase. A phase that is over already costs one test by all lanes (~100
// clocks less than one lane's test and the word to the others); else one lane polls, so that the
// polling does not crowd out the arrivals.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  if (__all_sync(0xffffffffu, ptx::mbar_try_wait(bar, parity))) return true;
  int ok = 1;
  if ((threadIdx.x & 31) == 0) ok = ptx::mbar_wait(bar, parity);
  ok = __shfl_sync(0xffffffffu, ok, 0);
  __syncwarp();  // orders the other lanes' reads after the phase
  return ok;
}
__device__ __forceinline__ bool warp_wait_sleep(uint64_t* bar, uint32_t parity) {
  int ok = 1;
  if ((threadIdx.x & 31) == 0) ok = ptx::mbar_wait_sleep(bar, parity);
  ok = __shfl_sync(0xffffffffu, ok, 0);
  __syncwarp();  // orders the other lanes' reads after the phase
  return ok;
}

// After an expired wait: report it, and leave copies and MMAs in flight time to land before the
// shared and tensor memory go.
__device__ __forceinline__ void give_up(int* error_flag) {
  if (error_flag) atomicExch(error_flag, kWaitFailed);
  const long long t0 = clock64();
  while (clock64() - t0 < 20000000LL) __nanosleep(1000);
}

}  // namespace muse
