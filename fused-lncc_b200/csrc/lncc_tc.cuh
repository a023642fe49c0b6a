// Tensor-core plumbing of the feed-forward block: mbarriers with bounded waits, tiled TMA loads, and tcgen05 products of
// a pair of CTAs (cta_group::2) with fp32 accumulators in tensor memory.
//
// Operand tiles lie in shared memory in rows of 128 bytes with the 128-byte swizzle, as a TMA box of 64 16-bit elements
// by R rows leaves them (8 rows make a 1024-byte unit; every tile starts on one). A row holds 64 steps of the inner axis
// of one row of the operand ("K-major"), or 64 rows of the operand at one step ("MN-major", for operands that memory
// holds transposed); 16-bit types take either.
#pragma once

#include "lncc_block.cuh"

#include <cuda.h>

namespace lncc {
namespace tc {

constexpr unsigned long long kWaitLimitNs = 2000000000ull;  // a wait that takes longer is given up

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// the address of the same shared variable in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t peer_addr(uint32_t a, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Arrive on a barrier given by its cluster address, to say that a warp has read its part of tensor memory. What is ordered by it
// are reads before the products that write there next, no data that the other side would read: every lane's loads have
// ended at its wait_ld (their values are in registers), fence_before and __syncwarp put that before lane 0's arrival, and the
// thread that issues the products comes after it by its wait and fence_after. So it may be relaxed: a release would also wait
// for the thread's stores to global memory, a thousand clocks a tile.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred P;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 P, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, P;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ unsigned long long now_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
// Waits for the phase of `parity` to end: true once it has, false when the limit ran out here or at another wait of the
// CTA (whose flag then ends every later wait at once).
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* gave_up) {
  if (mbar_test(bar, parity)) return true;
  const unsigned long long start = now_ns();
  while (!mbar_test(bar, parity)) {
    if (*gave_up) return false;
    if (now_ns() - start > kWaitLimitNs) {
      *gave_up = 1;
      return false;
    }
  }
  return true;
}

// One box of a three-dimensional map into this CTA's shared memory; its bytes are counted on a barrier of the pair.
__device__ __forceinline__ void tma_load(const CUtensorMap* map, uint32_t dst, uint32_t bar_cluster, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4, "
      "%5}], [%2];" ::"r"(dst),
      "l"(map), "r"(bar_cluster), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// Shared-memory matrix descriptors, 128-byte swizzle. K-major: 8-row units 1024 bytes apart, 16 steps of the inner axis
// are 32 bytes. MN-major: 64-row blocks `block_bytes` apart, units of 8 inner steps 1024 bytes apart, 16 steps are 2048.
__device__ __forceinline__ uint64_t desc_common(uint32_t addr) {
  return uint64_t((addr & 0x3FFFF) >> 4) | (uint64_t(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint64_t desc_k(uint32_t addr) { return desc_common(addr) | (1ull << 16); }
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr, uint32_t block_bytes) {
  return desc_common(addr) | (uint64_t(block_bytes >> 4) << 16);
}
// MN-major with the 64-byte swizzle: one block of 32 rows, units of 8 inner steps 512 bytes apart, 16 steps are 1024.
__device__ __forceinline__ uint64_t desc_mn_32(uint32_t addr) {
  return uint64_t((addr & 0x3FFFF) >> 4) | (1ull << 16) | (uint64_t(512 >> 4) << 32) | (1ull << 46) | (4ull << 61);
}
// Instruction descriptor: fp32 accumulators, 256 rows of the pair, n columns.
__device__ __forceinline__ uint32_t instr_desc(bool bf16, bool a_mn, bool b_mn, int n) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) |
         (uint32_t(n >> 3) << 17) | (uint32_t(256 >> 4) << 24);
}
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred P;\n\t"
      "setp.ne.b32 P, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, P;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(add))
      : "memory");
}
// Arrive on this barrier in both CTAs once every product issued so far has ended.
__device__ __forceinline__ void commit_pair(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"(uint16_t(3))
      : "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
template <int COLS> __device__ __forceinline__ void tmem_alloc(uint32_t dst) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(COLS) : "memory");
}
// 16 or 8 columns of the warp's 32 lanes; the values may be read after wait_ld() has named them.
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(addr));
}
__device__ __forceinline__ void wait_ld(uint32_t (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                 "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
               :
               : "memory");
}

__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "r"(addr));
}
__device__ __forceinline__ void wait_ld(uint32_t (&v)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7])
               :
               : "memory");
}

// cuTensorMapEncodeTiled, found through the runtime so that the library links no driver stub; null without a driver.
typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline EncodeTiled encode_tiled() {
  static const EncodeTiled f = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      p = nullptr;
    }
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return f;
}

// A matrix of 16-bit elements: `planes` of `rows` rows of `cols`, ld elements from row to row (a multiple of 8), the
// address on a 16-byte boundary.
struct Matrix {
  void* p;
  int64_t rows, cols, ld, plane;
  int planes;
  bool bf16;
};
// Map of boxes of 64 elements by `box_rows` rows (or of 32, with the 64-byte swizzle); what a box reaches past the matrix reads
// as zero.
inline bool make_map(CUtensorMap* map, const Matrix& m, int box_rows, int box_cols = 64) {
  const EncodeTiled encode = encode_tiled();
  if (!encode) return false;
  const cuuint64_t dims[3] = {cuuint64_t(m.cols), cuuint64_t(m.rows), cuuint64_t(m.planes)};
  const cuuint64_t strides[2] = {cuuint64_t(m.ld) * 2, m.planes > 1 ? cuuint64_t(m.plane) * 2 : cuuint64_t(m.ld) * 2};
  const cuuint32_t box[3] = {cuuint32_t(box_cols), cuuint32_t(box_rows), 1}, steps[3] = {1, 1, 1};
  const auto encoded = [&] {
    return encode(map, m.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, m.p, dims, strides, box,
                  steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  box_cols == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  if (encoded()) return true;
  // The driver encodes for the thread's context, and a thread that has not yet used the device through the runtime (a new
  // thread, or autograd's, whose memory came from a cache) has none.
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess && encoded();
}

}  // namespace tc
}  // namespace lncc
