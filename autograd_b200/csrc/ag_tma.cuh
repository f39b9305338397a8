// What the persistent tensor-core kernels share (ag_flce_tc.cu, ag_muon.cu): tile loads by tensor map, pairs of CTAs, the MMAs of a
// stage, fp16 pairs, wide stores, and the entry point that makes tensor maps.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>

#include <atomic>

#include "ag_tc.cuh"

namespace {

// ---------------------------------------------------------------------------- PTX wrappers
__device__ __forceinline__ void tc_tma_load_2d(const CUtensorMap* tm, void* smem_dst, uint64_t* bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
          ag_smem_u32(smem_dst)),
      "l"(tm), "r"(ag_smem_u32(bar)), "r"(x), "r"(y)
      : "memory");
}

__device__ __forceinline__ void tc_tma_load_3d(const CUtensorMap* tm, void* smem_dst, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          ag_smem_u32(smem_dst)),
      "l"(tm), "r"(ag_smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// ---- CTA pair (thread-block cluster of 2) helpers
__device__ __forceinline__ uint32_t tc_cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// shared::cluster address of the same shared-memory location in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t tc_map_to_cta(uint32_t smem_addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void tc_st_cluster(uint32_t cluster_addr, int v) {
  asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}
__device__ __forceinline__ void tc_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void tc_mbar_arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// commit whose mbarrier may live in either CTA of the pair
__device__ __forceinline__ void tc_commit_pair(uint32_t cluster_addr) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(cluster_addr) : "memory");
}
// tile loads of a CTA of the pair: destination in the own shared memory, completion bytes counted on
// the mbarrier at `mbar_cluster_addr`, which is the leader's
__device__ __forceinline__ void tc_tma_load_2d_pair(const CUtensorMap* tm, void* smem_dst, uint32_t mbar_cluster_addr,
                                                    int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::
          "r"(ag_smem_u32(smem_dst)),
      "l"(tm), "r"(mbar_cluster_addr), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void tc_tma_load_3d_pair(const CUtensorMap* tm, void* smem_dst, uint32_t mbar_cluster_addr,
                                                    int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], "
      "[%2];" ::"r"(ag_smem_u32(smem_dst)),
      "l"(tm), "r"(mbar_cluster_addr), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// two floats -> (hi, lo) fp16 pairs, packed two to a word
__device__ __forceinline__ void split_f16x2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
__device__ __forceinline__ void tc_st_global_v8(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
               "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// All MMAs of one stage: 4 steps of 32 bytes along K, three products each for (hi, lo) operands.
template <bool SPLIT, bool PAIR>
__device__ __forceinline__ void tc_stage_mmas(uint32_t tacc, uint32_t ah, uint32_t al, uint32_t a_step,
                                              uint32_t bh, uint32_t bl, uint32_t b_step, uint32_t idesc,
                                              uint32_t not_first) {
  constexpr uint32_t a_hi = TcDesc::hi, b_hi = TcDesc::hi;
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) {
    const uint32_t ao = (uint32_t)kk * a_step, bo = (uint32_t)kk * b_step;
    if (SPLIT) {
      if (kk == 0)
        tc_mma<2, PAIR>(tacc, ah + ao, a_hi, bl + bo, b_hi, idesc, not_first);
      else
        tc_mma<1, PAIR>(tacc, ah + ao, a_hi, bl + bo, b_hi, idesc, 1u);
      tc_mma<1, PAIR>(tacc, al + ao, a_hi, bh + bo, b_hi, idesc, 1u);
      tc_mma<1, PAIR>(tacc, ah + ao, a_hi, bh + bo, b_hi, idesc, 1u);
    } else {
      if (kk == 0)
        tc_mma<2, PAIR>(tacc, ah + ao, a_hi, bh + bo, b_hi, idesc, not_first);
      else
        tc_mma<1, PAIR>(tacc, ah + ao, a_hi, bh + bo, b_hi, idesc, 1u);
    }
  }
}

// The driver API is reached through the runtime (cudaGetDriverEntryPoint) so that the library has
// no link-time dependency on libcuda and still loads on a machine without a driver.
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn tc_encode_fn(ag_ctx* ctx) {
  static std::atomic<EncodeTiledFn> known{nullptr};
  EncodeTiledFn fn = known.load(std::memory_order_relaxed);
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q);
    if (e != cudaSuccess || q != cudaDriverEntryPointSuccess || !p) {
      snprintf(ctx->err, sizeof ctx->err, "cuTensorMapEncodeTiled is not available from this driver: %s",
               cudaGetErrorString(e));
      return nullptr;
    }
    fn = reinterpret_cast<EncodeTiledFn>(p);
    known.store(fn, std::memory_order_relaxed);
  }
  return fn;
}

}  // namespace
