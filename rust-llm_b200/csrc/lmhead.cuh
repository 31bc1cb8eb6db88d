// Device helpers of the LM-head kernels: TMA, TMEM and MMA instructions, and
// the packed argmax key.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include "common.cuh"

namespace rl {

__device__ __forceinline__ uint64_t lm_policy_first() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ uint64_t lm_policy_last() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(p));
  return p;
}

// 2-D tiled TMA load into this CTA's shared memory (no multicast); x is the
// K coordinate in the map's elements: a multiple of 64 bf16 values (128 bytes), or
// of 64 or 128 one-byte pairs of codes, whatever a box is wide.
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar,
                                            uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4}], [%2], %5;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "l"(policy)
      : "memory");
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Shared-memory matrix descriptor: K-major operand with the 128-byte swizzle
// (8-row groups of 1024 bytes: stride byte offset 1024; the leading byte
// offset is unused for this layout and set to 16 bytes), descriptor version 1.
__device__ __forceinline__ uint64_t sw128_desc(uint32_t saddr) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3fffu) | (static_cast<uint64_t>(1u) << 16) |
         (static_cast<uint64_t>(1024u >> 4) << 32) | (static_cast<uint64_t>(1u) << 46) |
         (static_cast<uint64_t>(2u) << 61);
}

// Instruction descriptor of kind::f16: bf16 A and B (both K-major), f32
// accumulator, M = 128, N = n.
__device__ __forceinline__ uint32_t lm_idesc(int n) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(128 >> 4) << 24);
}

__device__ __forceinline__ void umma_bf16(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, int acc) {
  const uint32_t z = 0u;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc), "r"(z), "r"(z), "r"(z), "r"(z)
      : "memory");
}

// Arrives on `bar` once every tcgen05 operation this thread issued before it
// has completed.
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ void mbar_arrive1(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// 32 TMEM lanes (this warp's quadrant) x 16 columns: register j of lane l is
// column col + j of lane (quadrant base + l).
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// (value, id) packed so that the larger u64 is the later maximum: the
// greedy_sample order (last maximum; -0.0 and +0.0 tie).
__device__ __forceinline__ uint64_t lm_key(float v, int id) {
  return (static_cast<uint64_t>(ord_key(__fadd_rn(v, 0.0f))) << 32) | static_cast<uint32_t>(id);
}
__device__ __forceinline__ uint64_t umax64(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int o) {
  const uint32_t lo = __shfl_xor_sync(0xffffffffu, static_cast<uint32_t>(v), o);
  const uint32_t hi = __shfl_xor_sync(0xffffffffu, static_cast<uint32_t>(v >> 32), o);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}

// Per-column maximum over the warp's 32 lanes for 16 columns, by a
// transposing butterfly (31 exchanges instead of 16 x 5): afterwards lane l
// holds column (l & 15).
__device__ __forceinline__ uint64_t warp_colmax16(uint64_t (&k)[16]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < 16; ++j) k[j] = umax64(k[j], shfl_xor64(k[j], 16));
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const bool up = (lane & 8) != 0;
    const uint64_t send = up ? k[j] : k[j + 8];
    const uint64_t keep = up ? k[j + 8] : k[j];
    k[j] = umax64(keep, shfl_xor64(send, 8));
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool up = (lane & 4) != 0;
    const uint64_t send = up ? k[j] : k[j + 4];
    const uint64_t keep = up ? k[j + 4] : k[j];
    k[j] = umax64(keep, shfl_xor64(send, 4));
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const bool up = (lane & 2) != 0;
    const uint64_t send = up ? k[j] : k[j + 2];
    const uint64_t keep = up ? k[j + 2] : k[j];
    k[j] = umax64(keep, shfl_xor64(send, 2));
  }
  const bool up = (lane & 1) != 0;
  const uint64_t send = up ? k[0] : k[1];
  const uint64_t keep = up ? k[1] : k[0];
  return umax64(keep, shfl_xor64(send, 1));
}

// Host side, in lmhead.cu.
// A [rows, inner] matrix of 2-byte (bf16) or 1-byte elements at row stride
// `stride` bytes, as boxes of box_bytes (128 or 64) x box_rows with the swizzle
// of that many bytes; what lies outside reads as zeros.
bool lm_tensor_map(CUtensorMap* m, const void* ptr, int elem_bytes, int inner, int rows, int64_t stride, int box_rows,
                   int box_bytes = 128);
// Row b's token: the largest packed key of part[b, 0 .. G), or -1 and
// RL_ERR_TIMEOUT where *err is set.
cudaError_t lm_argmax(const uint64_t* part, int B, int G, const int* err, int32_t* out_tok, int32_t* row_status,
                      cudaStream_t stream);
// Token -1 and RL_ERR_TIMEOUT for every row where *err is set.
cudaError_t lm_flag(const int* err, int B, int32_t* out_tok, int32_t* row_status, cudaStream_t stream);

// Makes a device current for the scope of a call.
struct LmDeviceGuard {
  int prev = -1;
  bool ok = true;
  explicit LmDeviceGuard(int dev) {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    if (prev != dev) ok = cudaSetDevice(dev) == cudaSuccess;
  }
  ~LmDeviceGuard() {
    int cur = -1;
    if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev) cudaSetDevice(prev);
  }
};

}  // namespace rl
