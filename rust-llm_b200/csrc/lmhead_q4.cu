// The LM head with 4-bit weights and group scales (rl_lmhead_q4_*; the format
// stands in rl_sampler.h):
//
//   logits[b, v] = sum_g scale[v, g] * sum_{k in g} (code[v, k] - 8) * hidden[b, k]
//
// code - 8 is a whole number in [-8, 7], so code - 8 times a bf16 value is exact
// in f32; a group's sum is multiplied by its scale once, in f32.
//
// On the tensor cores: one persistent CTA per SM walks tiles of 128 vocabulary
// rows (MMA M = 128, N = batch rows padded, K in blocks of 128):
//   warp 0        TMA producer of the codes: [128 rows x 256 codes] a copy, 128
//                 bytes of a row, 128-byte swizzle
//   warp 2        TMA producer of the hidden states: two [N x 64] a block
//   warp 3        copies the scales: [128 rows x 8 groups] a box
//   warps 4-...   turn codes into bf16 (a thread a row, a block at a turn: code | 0x4300
//                 is 128 + code, less 136) and store them into TMEM, from where
//                 the MMA reads them as its A operand: expanded weights never
//                 pass through shared memory, which would take four times the
//                 bytes of the codes in and again out
//   warp 1        tcgen05.mma kind::f16, one accumulator in TMEM for each group.
//                 One thread issues them, eight a block, and at few batch rows
//                 that is what counts: a block's operands (expanded codes and
//                 hidden states) share one full and one free barrier, so that
//                 it waits and commits once for both
//   the last      read a group's accumulator back, times the row's
//                 scale (a thread a row), into f32 sums in registers; at the
//                 tile's end logits are stored along the vocabulary, or the
//                 rows' running maxima kept
// Multiplying the scale in behind the MMA keeps the operands exact (code - 8
// has four bits) for scales of any size, at N / group FMAs a weight.
//
// Up to 16 batch rows (q4_few_kernel) the hand-overs between those roles cost
// more than the work: there each warp multiplies what it loads, on its own. It
// streams the codes of 32 vocabulary rows through a ring of its own and takes
// them, as f16 (the published way of setting codes under the exponent of 1024 and
// subtracting), straight into mma.sync fragments; the hidden states lie in
// shared memory in the order of the fragments. A CTA's warps share its rows'
// codes evenly, cut where they fall, so that none waits for another; the sums of
// rows that two warps share are added at the end.
//
// Bound: HBM, half a byte a weight, up to about 100 batch rows; beside it the
// expansion, 9 (f16) or 11 (bf16) instructions for 8 weights, and for more rows
// the hand-overs and N / group FMAs a weight. H 4096, V 128256: 52 us for one row
// (HBM needs 42), 94 for 12 (43), 147 for 128 (the MMAs need 81). Every wait is
// bounded; where one runs out the error flag is set, copies in flight land and
// TMEM is freed.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <climits>

#include "common.cuh"
#include "internal.h"
#include "lmhead.cuh"

namespace rl {
namespace {

constexpr int kBM = 128;        // vocabulary rows of a tile
constexpr int kQTile = kBM * 128;  // bytes of a copy of codes: 256 codes of each row
constexpr int kSlotCols = 64;   // TMEM columns of a block's expanded codes
constexpr int kSBox = kBM * 16;  // bytes of a box of scales: 8 groups of each row
constexpr int kSSlots = 8;
constexpr int kQMax = 8;

struct Q4Args {
  int B, H, V;
  int ntiles, kstages;  // kstages = H / 64
  int qslots;
  const uint16_t* scale;
  int64_t lds;
  int gran;                // bytes of a copy of scales: 16, 8, 4, or 2 (loads)
  float* out_f32;
  uint16_t* out_bf16;
  int64_t ldo;
  uint64_t* part;          // [B, gridDim.x] packed (value, id) maxima, or null
  int* err;
};

__device__ __forceinline__ float bf16_at(uint32_t w, int hi) { return __uint_as_float(hi ? w & 0xffff0000u : w << 16); }

// D (+)= A B^T with A (bf16, M = 128, K = 16) in TMEM columns and B in shared memory.
__device__ __forceinline__ void umma_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, int acc) {
  const uint32_t z = 0u;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(acc), "r"(z), "r"(z), "r"(z), "r"(z)
      : "memory");
}

// This warp's 32 lanes x 32 columns of TMEM: register j is column j.
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

// a & b | c in one instruction (two immediates would make it two).
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// Eight codes of a word as bf16 code - 8, in element order.
__device__ __forceinline__ void expand(uint32_t w, uint32_t* out) {
  const __nv_bfloat162 c136 = __halves2bfloat162(__ushort_as_bfloat16(0x4308), __ushort_as_bfloat16(0x4308));
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t x = and_or(w >> (4 * j), 0x000f000fu, 0x43004300u);  // 128 + code
    __nv_bfloat162 v;
    *reinterpret_cast<uint32_t*>(&v) = x;
    v = __hsub2(v, c136);
    out[j] = *reinterpret_cast<uint32_t*>(&v);
  }
}

struct Q4Bars {
  uint64_t qfull[kQMax], qempty[kQMax];
  uint64_t full[6], free[6];
  uint64_t dfull[4], dempty[4];
  uint64_t sfull[kSSlots], sempty[kSSlots];
  uint64_t done;
  uint32_t tmem;
};

__device__ __forceinline__ bool q4_try(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done != 0;
}
// A bounded wait as mbar_wait, but without its clock where the phase is over
// already, and asleep between tries: here most warps wait most of the time, and
// their tries would take the issue slots of those that work.
__device__ __forceinline__ bool q4_wait(uint64_t* bar, uint32_t parity) {
  if (q4_try(bar, parity)) return true;
  const long long t0 = clock64();
  while (true) {
    __nanosleep(32);
    if (q4_try(bar, parity)) return true;
    if (clock64() - t0 > kWaitBudget) return false;
  }
}
// The outcome of a converged warp's waits, alike for its lanes: one whose wait
// runs out leaves no others behind at an instruction of the whole warp.
__device__ __forceinline__ bool all_ok(bool ok) { return __all_sync(0xffffffffu, ok) != 0; }
// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}

// A ring position: slot and the parity of its present use.
struct Ring {
  int slot = 0;
  uint32_t par = 0;
  __device__ __forceinline__ void next(int n) {
    if (++slot == n) {
      slot = 0;
      par ^= 1u;
    }
  }
  __device__ __forceinline__ void skip(int d, int n) {
    slot += d;
    while (slot >= n) {
      slot -= n;
      par ^= 1u;
    }
  }
};

// How a launch of N batch rows and groups of 2^GS lays out TMEM: accumulators
// are handed over kSplit times a block, in kDBufs buffers of kDCols columns that
// take at most half of it; the rest holds kSlots blocks of expanded codes (the
// hidden states of as many lie in shared memory).
template <int N, int GS>
struct Q4Plan {
  static constexpr int kSplit = N * (128 >> GS) <= 128 ? 1 : 2;
  static constexpr int kNg = (128 >> GS) / kSplit;  // groups of a hand-over
  static constexpr int kDCols = N * kNg;
  static constexpr int kDBufs = 256 / kDCols < 4 ? 256 / kDCols : 4;
  static constexpr int kRoom = (512 - kDBufs * kDCols) / kSlotCols;
  static constexpr int kSlots = kRoom < 6 ? kRoom : 6;
};

template <int N, int GS, int NDQ, int NEP>  // expanding warps, epilogue warps (multiples of 4)
__global__ void __launch_bounds__((4 + NDQ + NEP) * 32, 1)
    q4_mma_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmX,
                  const __grid_constant__ Q4Args a) {
  extern __shared__ uint8_t q4_smem_raw[];
  __shared__ Q4Bars bars;
  __shared__ unsigned long long best[N];
  using P = Q4Plan<N, GS>;
  constexpr int kSplit = P::kSplit, kNg = P::kNg, kDCols = P::kDCols, kDBufs = P::kDBufs, kSlots = P::kSlots;
  constexpr int NC = N / (NEP / 4);  // columns of an epilogue warp
  constexpr uint32_t kXBytes = N * 128;  // 64 hidden elements of N rows
  uint8_t* qring = q4_smem_raw + ((1024u - (smem_u32(q4_smem_raw) & 1023u)) & 1023u);
  uint8_t* xring = qring + a.qslots * kQTile;
  uint8_t* sring = xring + kSlots * 2 * kXBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < a.qslots; ++i) mbar_init(&bars.qfull[i], 1), mbar_init(&bars.qempty[i], 8);
    for (int i = 0; i < kSlots; ++i) mbar_init(&bars.full[i], 4 + 1), mbar_init(&bars.free[i], 1);
    for (int i = 0; i < kDBufs; ++i) mbar_init(&bars.dfull[i], 1), mbar_init(&bars.dempty[i], NEP);
    for (int i = 0; i < kSSlots; ++i) mbar_init(&bars.sfull[i], 32), mbar_init(&bars.sempty[i], NEP);
    mbar_init(&bars.done, 1);
    fence_mbar_init();
  }
  for (int i = threadIdx.x; i < N; i += blockDim.x) best[i] = 0ull;
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars.tmem, 0);
  const uint32_t tmem_a = tmem + static_cast<uint32_t>(kDBufs * kDCols);  // expanded codes lie behind the accumulators
  const int qtiles = (a.kstages + 3) >> 2;  // copies of codes a tile
  const int blocks = (a.kstages + 1) >> 1;  // the last may be half a block
  const int ngroups = a.H >> GS;
  bool ok = true;

  if (warp == 0) {
    if (lane == 0) {
      // ---- codes ----
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmQ)) : "memory");
      const uint64_t pol = lm_policy_first();  // streamed once
      Ring r;
      uint32_t it = 0;
      for (int tile = blockIdx.x; tile < a.ntiles && ok; tile += gridDim.x) {
        for (int t = 0; t < qtiles; ++t, ++it) {
          if (!q4_wait(&bars.qempty[r.slot], r.par ^ 1u)) {
            ok = false;
            break;
          }
          mbar_expect_tx(&bars.qfull[r.slot], kQTile);
          tma_load_2d(qring + r.slot * kQTile, &tmQ, t * 128, tile * kBM, &bars.qfull[r.slot], pol);
          r.next(a.qslots);
        }
      }
      // every issued copy lands before the CTA may return
      for (int i = 0; i < a.qslots; ++i) {
        const uint32_t n = it / a.qslots + (static_cast<uint32_t>(i) < it % a.qslots ? 1u : 0u);
        if (n > 0 && !q4_wait(&bars.qfull[i], (n - 1u) & 1u)) ok = false;
      }
    }
  } else if (warp == 2) {
    if (lane == 0) {
      // ---- hidden states ----
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmX)) : "memory");
      const uint64_t pol = lm_policy_last();  // read by every CTA, for every tile
      Ring r;
      uint32_t it = 0;
      for (int tile = blockIdx.x; tile < a.ntiles && ok; tile += gridDim.x) {
        for (int kb = 0; kb < blocks; ++kb, ++it) {
          if (!q4_wait(&bars.free[r.slot], r.par ^ 1u)) {
            ok = false;
            break;
          }
          const bool two = 2 * kb + 1 < a.kstages;
          uint8_t* x = xring + r.slot * 2 * kXBytes;
          mbar_expect_tx(&bars.full[r.slot], two ? 2 * kXBytes : kXBytes);
          tma_load_2d(x, &tmX, kb * 128, 0, &bars.full[r.slot], pol);
          if (two) tma_load_2d(x + kXBytes, &tmX, kb * 128 + 64, 0, &bars.full[r.slot], pol);
          r.next(kSlots);
        }
      }
      for (int i = 0; i < kSlots; ++i) {
        const uint32_t n = it / kSlots + (static_cast<uint32_t>(i) < it % kSlots ? 1u : 0u);
        if (n > 0 && !q4_wait(&bars.full[i], (n - 1u) & 1u)) ok = false;
      }
    }
  } else if (warp == 3) {
    // ---- scales: a lane copies rows lane, lane + 32, ... ----
    Ring r;
    for (int tile = blockIdx.x; tile < a.ntiles && ok; tile += gridDim.x) {
      for (int g0 = 0; g0 < ngroups && ok; g0 += 8) {
        if (!all_ok(q4_wait(&bars.sempty[r.slot], r.par ^ 1u))) {
          ok = false;
          break;
        }
        const int bytes = 2 * min(8, ngroups - g0);
        uint8_t* box = sring + r.slot * kSBox;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = 32 * i + lane;
          const int64_t v = static_cast<int64_t>(tile) * kBM + row;
          if (v >= a.V) continue;
          const uint8_t* src = reinterpret_cast<const uint8_t*>(a.scale + v * a.lds + g0);
          const uint32_t dst = smem_u32(box + row * 16);
          if (a.gran == 16) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
          } else if (a.gran == 8) {
            for (int o = 0; o < bytes; o += 8)
              asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst + o), "l"(src + o) : "memory");
          } else if (a.gran == 4) {
            for (int o = 0; o < bytes; o += 4)
              asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst + o), "l"(src + o) : "memory");
          } else {
            for (int o = 0; o < bytes; o += 2)
              *reinterpret_cast<uint16_t*>(box + row * 16 + o) = *reinterpret_cast<const uint16_t*>(src + o);
          }
        }
        // arrives once this lane's copies have landed
        if (a.gran > 2)
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&bars.sfull[r.slot])) : "memory");
        else
          mbar_arrive1(&bars.sfull[r.slot]);
        r.next(kSSlots);
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp == 1) {
    // ---- MMA issuer: the warp goes through the blocks together, so that
    // addresses and descriptors stay uniform; one lane issues ----
    const uint32_t idesc = lm_idesc(N);
    constexpr int gs = GS - 4;  // log2 of a group's steps (K = 16)
    const uint32_t x0 = smem_u32(xring);
    // four MMAs of a stage, `step` steps behind the hand-over's first
    const auto issue = [&](uint32_t d0, uint32_t at, uint64_t bd, int step) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        umma_ta(d0 + static_cast<uint32_t>(((step + k) >> gs) * N), at + 8u * k, bd + 2u * k, idesc,
                ((step + k) & ((1 << gs) - 1)) != 0);
    };
    Ring r, rd;
    for (int tile = blockIdx.x; tile < a.ntiles && ok; tile += gridDim.x) {
      for (int kb = 0; kb < blocks && ok; ++kb) {
        const int nst = min(2, a.kstages - 2 * kb);
        if (!all_ok(q4_wait(&bars.full[r.slot], r.par) && q4_wait(&bars.dempty[rd.slot], rd.par ^ 1u))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint64_t bd = sw128_desc(x0 + r.slot * 2 * kXBytes);
        const uint32_t at = tmem_a + static_cast<uint32_t>(r.slot * kSlotCols);
        const uint32_t d0 = tmem + static_cast<uint32_t>(rd.slot * kDCols);
        if constexpr (kSplit == 1) {
          if (elect_one()) {
            issue(d0, at, bd, 0);
            if (nst == 2) issue(d0, at + 32u, bd + (kXBytes >> 4), 4);
            umma_commit(&bars.free[r.slot]);
            umma_commit(&bars.dfull[rd.slot]);
          }
          rd.next(kDBufs);
        } else {
          if (elect_one()) {
            issue(d0, at, bd, 0);
            umma_commit(&bars.dfull[rd.slot]);
            if (nst == 1) umma_commit(&bars.free[r.slot]);
          }
          rd.next(kDBufs);
          if (nst == 2) {
            if (!all_ok(q4_wait(&bars.dempty[rd.slot], rd.par ^ 1u))) {
              ok = false;
              break;
            }
            tc_fence_after();
            if (elect_one()) {
              issue(tmem + static_cast<uint32_t>(rd.slot * kDCols), at + 32u, bd + (kXBytes >> 4), 0);
              umma_commit(&bars.dfull[rd.slot]);
              umma_commit(&bars.free[r.slot]);
            }
            rd.next(kDBufs);
          }
        }
        __syncwarp();
        r.next(kSlots);
      }
    }
    // every MMA of this CTA completes before its TMEM is freed
    if (elect_one()) umma_commit(&bars.done);
    __syncwarp();
    if (!q4_wait(&bars.done, 0u)) ok = false;
    __syncwarp();
  } else if (warp < 4 + NDQ) {
    // ---- codes into bf16: every so many blocks of this warp's 32 rows ----
    constexpr int kTurns = NDQ / 4;
    const int quad = warp & 3;
    const int row = quad * 32 + lane;
    const uint8_t* qrow = qring + row * 128;
    const uint32_t to0 = tmem_a + (static_cast<uint32_t>(quad * 32) << 16);
    const int swz = row & 7;
    Ring rq, r;
    int tile = blockIdx.x, kb = (warp - 4) >> 2;
    r.skip(kb, kSlots);
    rq.skip(kb >> 1, a.qslots);
    while (kb >= blocks) {  // (few blocks a tile)
      kb -= blocks;
      tile += gridDim.x;
    }
    if (blocks < kTurns) {  // the copies of the tiles passed over
      rq = Ring();
      rq.skip(((tile - static_cast<int>(blockIdx.x)) / static_cast<int>(gridDim.x)) * qtiles + (kb >> 1), a.qslots);
    }
    while (tile < a.ntiles && ok) {
      if (!all_ok(q4_wait(&bars.qfull[rq.slot], rq.par) && q4_wait(&bars.free[r.slot], r.par ^ 1u))) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint8_t* src = qrow + rq.slot * kQTile;
      const uint32_t to = to0 + static_cast<uint32_t>(r.slot * kSlotCols);
      const int nst = min(2, a.kstages - 2 * kb);
      for (int st = 0; st < nst; ++st) {
        const int c0 = (kb & 1) * 4 + st * 2;  // 16-byte piece of the row's 128
        uint32_t e[32];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint4 c = *reinterpret_cast<const uint4*>(src + (((c0 + i) ^ swz) << 4));
          expand(c.x, e + 16 * i);
          expand(c.y, e + 16 * i + 4);
          expand(c.z, e + 16 * i + 8);
          expand(c.w, e + 16 * i + 12);
        }
        tmem_st32(to + 32u * st, e);
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive1(&bars.full[r.slot]);
        // a copy of codes is free once the four quadrants have read both of its
        // blocks (eight arrivals; its only block counts twice)
        mbar_arrive1(&bars.qempty[rq.slot]);
        if ((kb & 1) == 0 && kb == blocks - 1) mbar_arrive1(&bars.qempty[rq.slot]);
      }
      // on to this warp's next block
      r.skip(kTurns, kSlots);
      int copies = -(kb >> 1);
      kb += kTurns;
      while (kb >= blocks) {
        kb -= blocks;
        tile += gridDim.x;
        copies += qtiles;
      }
      rq.skip(copies + (kb >> 1), a.qslots);
    }
  } else {
    // ---- epilogue ----
    const int quad = warp & 3;
    const int col0 = ((warp - 4 - NDQ) >> 2) * NC;
    const int row = quad * 32 + lane;
    const uint32_t from = tmem + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(col0);
    Ring rd, rs;
    for (int tile = blockIdx.x; tile < a.ntiles && ok; tile += gridDim.x) {
      float acc[NC];
#pragma unroll
      for (int j = 0; j < NC; ++j) acc[j] = 0.0f;
      for (int g0 = 0; g0 < ngroups && ok; g0 += 8) {  // a box of scales
        const bool in = q4_wait(&bars.sfull[rs.slot], rs.par);
        const uint4 sc = *reinterpret_cast<const uint4*>(sring + rs.slot * kSBox + row * 16);
        const uint32_t sw[4] = {sc.x, sc.y, sc.z, sc.w};
        __syncwarp();
        if (lane == 0) mbar_arrive1(&bars.sempty[rs.slot]);
        rs.next(kSSlots);
#pragma unroll
        for (int h0 = 0; h0 < 8; h0 += kNg) {  // a hand-over
          if (g0 + h0 >= ngroups) break;
          if (!all_ok(in && q4_wait(&bars.dfull[rd.slot], rd.par))) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t at = from + static_cast<uint32_t>(rd.slot * kDCols);
#pragma unroll
          for (int i = 0; i < kNg; ++i) {
            if (i > 0 && g0 + h0 + i >= ngroups) break;  // half a block, the tile's last
            const float s = bf16_at(sw[(h0 + i) >> 1], (h0 + i) & 1);
            // sixteen columns at a time: wider loads keep the MMAs from TMEM (32
            // columns took 27% longer at 128 batch rows, H 4096, V 128256)
#pragma unroll
            for (int c = 0; c < NC; c += 16) {
              uint32_t r[16];
              tmem_ld16(at + static_cast<uint32_t>(i * N + c), r);
#pragma unroll
              for (int j = 0; j < 16; ++j) acc[c + j] = fmaf(s, __uint_as_float(r[j]), acc[c + j]);
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive1(&bars.dempty[rd.slot]);
          rd.next(kDBufs);
        }
      }
      if (!ok) break;
      const int64_t v = static_cast<int64_t>(tile) * kBM + row;
      const bool vin = v < a.V;
      if (vin && a.out_f32) {
#pragma unroll
        for (int j = 0; j < NC; ++j)
          if (col0 + j < a.B) a.out_f32[static_cast<int64_t>(col0 + j) * a.ldo + v] = acc[j];
      }
      if (vin && a.out_bf16) {
#pragma unroll
        for (int j = 0; j < NC; ++j)
          if (col0 + j < a.B)
            a.out_bf16[static_cast<int64_t>(col0 + j) * a.ldo + v] = __bfloat16_as_ushort(__float2bfloat16_rn(acc[j]));
      }
      if (a.part) {
#pragma unroll
        for (int c = 0; c < NC; c += 16) {
          uint64_t k[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) k[j] = vin ? lm_key(acc[c + j], static_cast<int>(v)) : 0ull;
          const uint64_t m = warp_colmax16(k);
          if (lane < 16 && col0 + c + lane < a.B)
            atomicMax(&best[col0 + c + lane], static_cast<unsigned long long>(m));
        }
      }
    }
  }
  if (!ok) atomicExch(a.err, 1);
  __syncthreads();
  if (a.part)
    for (int b = threadIdx.x; b < a.B; b += blockDim.x) a.part[static_cast<int64_t>(b) * gridDim.x + blockIdx.x] = best[b];
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// ---------------------------------------------------------------------------
// Few batch rows
// ---------------------------------------------------------------------------
constexpr int kFewRows = 32;   // vocabulary rows of a tile (two MMA Ms)
constexpr int kFewWarps = 16;
constexpr int kFewSlots = 4;   // copies in flight a warp, at most
constexpr int kFewHidden = 128 * 1024;   // bytes of the hidden states in shared memory, at most

struct FewArgs {
  const uint16_t* hidden;
  int64_t ldh;
  int B, H, V;
  int ntiles, boxes;  // 32-row tiles; copies (boxes) a tile
  int slots;
  const uint16_t* scale;
  int64_t lds;
  int vec;  // a box's scales of a row may be loaded at once
  float* out_f32;
  uint16_t* out_bf16;
  int64_t ldo;
  uint64_t* part;
  int* err;
};

__device__ __forceinline__ uint32_t h2_bits(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ __half2 bits_h2(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }

// Two pairs of codes (elements 0, 1 and 2, 3 of a word's lower byte lanes) as
// f16 code - 8: 0x6400 | code is 1024 + code, with the code four bits up
// 1024 + 16 code.
__device__ __forceinline__ void expand_h(uint32_t w, uint32_t& lo, uint32_t& hi) {
  lo = h2_bits(__hsub2(bits_h2(and_or(w, 0x000f000fu, 0x64006400u)), bits_h2(0x64086408u)));
  hi = h2_bits(__hfma2(bits_h2(and_or(w, 0x00f000f0u, 0x64006400u)), bits_h2(0x2c002c00u), bits_h2(0xd480d480u)));
}

// D = A B + C: 16 x 8 f32, A 16 x 16 and B 16 x 8 f16.
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

// 2^e, e in [-126, 127].
__device__ __forceinline__ float pow2f(int e) { return __int_as_float((e + 127) << 23); }
// The power of two that brings m (>= 0, finite) to [2^k, 2^(k+1)), as an exponent.
__device__ __forceinline__ int bring_to(float m, int k) {
  const int e = static_cast<int>(__float_as_uint(m) >> 23) - 127;  // -127 for zero and subnormals
  return min(max(k - e, -126), 126);
}
__device__ __forceinline__ float finite_abs(float x) { return fabsf(x) < RL_POS_INF ? fabsf(x) : 0.0f; }

// Fragments. K is summed in another order than it lies in memory, alike for both
// operands, so that a lane's codes lie together and a group is never split over
// a step: of a group of G codes, lane (g, t) = (lane / 4, lane % 4) holds codes
// t G / 4 .. of rows g and g + 8, and the same hidden elements of batch row g;
// step j multiplies 4 j .. 4 j + 3 of those. A group's sum is scaled in f32.
//
// Hidden states are bf16 brought near 2^10 by the power of two of the batch
// row's largest, and so exact in f16 (steps of 2^-24, eight bits a value) but for
// what is below 2^-27 of the largest.
template <int GS>
__device__ __forceinline__ void row_words(const uint8_t* row, int swz, int half, int t, uint32_t (&w)[4]) {
  // the four words of this lane in K = 128 of a row (64 bytes of a box, whose
  // 16-byte pieces are swizzled by the row's number)
  if constexpr (GS == 7) {
    const uint4 c = *reinterpret_cast<const uint4*>(row + (((half * 4 + t) ^ swz) << 4));
    w[0] = c.x, w[1] = c.y, w[2] = c.z, w[3] = c.w;
  } else if constexpr (GS == 6) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint2 c = *reinterpret_cast<const uint2*>(row + (((half * 4 + 2 * i + (t >> 1)) ^ swz) << 4) + 8 * (t & 1));
      w[2 * i] = c.x, w[2 * i + 1] = c.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = *reinterpret_cast<const uint32_t*>(row + (((half * 4 + i) ^ swz) << 4) + 4 * t);
  }
}

// The N scales of a box of four rows, two to a word; sp[i] is row i's first
// scale, at element offset g0 <= ngroups - 1.
template <int N>
__device__ __forceinline__ void box_scales(const uint16_t* const (&sp)[4], int g0, int ngroups, bool vec,
                                           uint32_t (&w)[4][(N + 1) / 2]) {
  if (N > 1 && vec) {  // on 2 N bytes, whole boxes only
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (N == 2) {
        w[i][0] = __ldg(reinterpret_cast<const uint32_t*>(sp[i] + g0));
      } else if constexpr (N == 4) {
        const uint2 c = __ldg(reinterpret_cast<const uint2*>(sp[i] + g0));
        w[i][0] = c.x, w[i][1] = c.y;
      } else if constexpr (N == 8) {
        const uint4 c = __ldg(reinterpret_cast<const uint4*>(sp[i] + g0));
        w[i][0] = c.x, w[i][1] = c.y, w[i][2] = c.z, w[i][3] = c.w;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int k = 0; k < (N + 1) / 2; ++k) {
        const uint32_t lo = g0 + 2 * k < ngroups ? __ldg(sp[i] + g0 + 2 * k) : 0;
        const uint32_t hi = N > 1 && g0 + 2 * k + 1 < ngroups ? __ldg(sp[i] + g0 + 2 * k + 1) : 0;
        w[i][k] = lo | hi << 16;
      }
    }
  }
}

// Batch tiles of 8; log2(group); halves of K = 128 in a box (a box of two needs
// half the copies, of one half the room).
template <int NT, int GS, int HB>
__global__ void __launch_bounds__(kFewWarps * 32, 1)
    q4_few_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ FewArgs a) {
  extern __shared__ uint8_t few_smem_raw[];
  __shared__ uint64_t full[kFewWarps][kFewSlots];
  __shared__ unsigned long long best[NT * 8];
  __shared__ int hexp[NT * 8];  // the batch rows' powers of two
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  uint8_t* base = few_smem_raw + ((1024u - (smem_u32(few_smem_raw) & 1023u)) & 1023u);
  constexpr int kFewBox = kFewRows * 64 * HB;
  const int ring_bytes = a.slots * kFewBox;
  uint8_t* ring = base + static_cast<size_t>(warp) * ring_bytes;  // this warp's
  uint4* hs = reinterpret_cast<uint4*>(base + static_cast<size_t>(kFewWarps) * ring_bytes);  // [half box][NT][4][32]
  if (lane == 0) {
    for (int i = 0; i < a.slots; ++i) mbar_init(&full[warp][i], 1);
    fence_mbar_init();
  }
  if (threadIdx.x < NT * 8) best[threadIdx.x] = 0ull;
  __syncwarp();
  // ---- this warp's boxes: an even share of the CTA's tiles ----
  const int nb = a.boxes;
  const int tfirst = static_cast<int>(static_cast<int64_t>(a.ntiles) * blockIdx.x / gridDim.x);
  const int tlast = static_cast<int>(static_cast<int64_t>(a.ntiles) * (blockIdx.x + 1) / gridDim.x);
  const int64_t units = static_cast<int64_t>(tlast - tfirst) * nb;
  const int u0 = static_cast<int>(units * warp / kFewWarps), u1 = static_cast<int>(units * (warp + 1) / kFewWarps);
  const uint64_t pol = lm_policy_first();
  int cu = u0, cbox = u0 % nb, ctile = tfirst + u0 / nb;  // the next copy
  Ring rc;
  const auto copy = [&] {  // one lane
    mbar_expect_tx(&full[warp][rc.slot], kFewBox);
    tma_load_2d(ring + rc.slot * kFewBox, &tmQ, cbox * (64 * HB), ctile * kFewRows, &full[warp][rc.slot], pol);
    rc.next(a.slots);
    ++cu;
    if (++cbox == nb) {
      cbox = 0;
      ++ctile;
    }
  };
  if (lane == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmQ)) : "memory");
    for (int i = 0; i < a.slots && cu < u1; ++i) copy();
  }
  // ---- the hidden states, as f16 fragments ----
  for (int b = warp; b < NT * 8; b += kFewWarps) {
    float m = 0.0f;
    if (b < a.B) {
      const uint4* x = reinterpret_cast<const uint4*>(a.hidden + static_cast<int64_t>(b) * a.ldh);
      for (int i = lane; i < (a.H >> 3); i += 32) {
        const uint4 v = __ldg(x + i);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) m = fmaxf(m, fmaxf(finite_abs(bf16_at(w[k], 0)), finite_abs(bf16_at(w[k], 1))));
      }
    }
    m = warp_max(m);
    if (lane == 0) hexp[b] = bring_to(m, 10);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nb * HB * NT * 4 * 32; i += kFewWarps * 32) {
    // word w of lane l: eight elements of batch tile n in the hk-th K = 128
    const int l = i & 31, w = (i >> 5) & 3, n = (i >> 7) % NT, hk = (i >> 7) / NT;
    constexpr int kWords = 1 << (GS - 5);  // words of a lane's share of a group
    const int b = n * 8 + (l >> 2), k0 = hk * 128 + (w / kWords << GS) + (l & 3) * (8 * kWords) + 8 * (w % kWords);
    uint4 v = {0u, 0u, 0u, 0u};
    if (b < a.B && k0 < a.H) v = __ldg(reinterpret_cast<const uint4*>(a.hidden + static_cast<int64_t>(b) * a.ldh + k0));
    const float f = pow2f(hexp[b]);
    uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = h2_bits(__floats2half2_rn(bf16_at(x[k], 0) * f, bf16_at(x[k], 1) * f));
    hs[i] = make_uint4(x[0], x[1], x[2], x[3]);
  }
  __syncthreads();

  // ---- tiles ----
  const int ngroups = a.H >> GS;
  constexpr int kNs = (128 * HB) >> GS, kSw = (kNs + 1) / 2;  // scales of a box, in words
  const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  const bool vec = a.vec != 0;
  bool ok = true;
  Ring r;
  float acc[2][NT][4];
  // logits of a tile from the fragments of its sums
  const auto finish = [&](int tile) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int b = n * 8 + 2 * t + k;
        const float back = pow2f(-hexp[b]);
        uint64_t key = 0ull;
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // rows g, g + 8, g + 16, g + 24
          const int64_t v = static_cast<int64_t>(tile) * kFewRows + 8 * i + g;
          const float y = acc[i >> 1][n][2 * (i & 1) + k] * back;
          if (v < a.V) {
            if (b < a.B) {
              if (a.out_f32) a.out_f32[static_cast<int64_t>(b) * a.ldo + v] = y;
              if (a.out_bf16) a.out_bf16[static_cast<int64_t>(b) * a.ldo + v] = __bfloat16_as_ushort(__float2bfloat16_rn(y));
            }
            key = umax64(key, lm_key(y, static_cast<int>(v)));
          }
        }
        if (a.part) {
#pragma unroll
          for (int o = 16; o > 2; o >>= 1) key = umax64(key, shfl_xor64(key, o));  // over g
          if (g == 0 && b < a.B) atomicMax(&best[b], static_cast<unsigned long long>(key));
        }
      }
    }
  };
  // the sums of the end of a tile that began before u0, in the ring once it is read
  float* parts = reinterpret_cast<float*>(ring);  // [2 * NT * 4][32]
  int kept = 0;  // 1: `first` holds those; 2: acc holds a tile that ends behind u1
  float first[2][NT][4];
  int u = u0;
  while (u < u1 && ok) {
    const int tile = tfirst + u / nb;
    const int box0 = u % nb, box1 = min(nb, box0 + (u1 - u));
    const uint16_t* sp[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t v = static_cast<int64_t>(tile) * kFewRows + 8 * i + g;
      sp[i] = a.scale + (v < a.V ? v : 0) * a.lds;
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[m][n][0] = acc[m][n][1] = acc[m][n][2] = acc[m][n][3] = 0.0f;
    uint32_t ahead[4][kSw];
    box_scales<kNs>(sp, box0 * kNs, ngroups, vec, ahead);
    for (int box = box0; box < box1; ++box) {
      uint32_t sc[4][kSw];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < kSw; ++k) sc[i][k] = ahead[i][k];
      if (box + 1 < box1) box_scales<kNs>(sp, (box + 1) * kNs, ngroups, vec, ahead);
      if (!all_ok(q4_wait(&full[warp][r.slot], r.par))) {
        ok = false;
        break;
      }
      const uint8_t* src = ring + r.slot * kFewBox + g * (64 * HB);
      const int swz = HB == 2 ? g : g >> 1;  // of rows g, g + 8, ... alike
#pragma unroll
      for (int half = 0; half < HB; ++half) {
        uint32_t w[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) row_words<GS>(src + i * (8 * 64 * HB), swz, half, t, w[i]);
        if (half == HB - 1) {
          __syncwarp();
          if (lane == 0 && cu < u1) copy();  // the slot is read: the stream goes on in it
          r.next(a.slots);
        }
        const uint4* h = hs + (HB * box + half) * (NT * 4 * 32) + lane;
        constexpr int kWords = 1 << (GS - 5);
        float d[2][NT][4];
#pragma unroll
        for (int jw = 0; jw < 4; ++jw) {
          uint4 hv[NT];
#pragma unroll
          for (int n = 0; n < NT; ++n) hv[n] = h[(n * 4 + jw) * 32];
          const bool begins = jw % kWords == 0, ends = jw % kWords == kWords - 1;
#pragma unroll
          for (int m = 0; m < 2; ++m) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              uint32_t e[4];
              expand_h(w[2 * m][jw] >> (8 * k), e[0], e[2]);
              expand_h(w[2 * m + 1][jw] >> (8 * k), e[1], e[3]);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                if (begins && k == 0) mma_f16(d[m][n], e, hv[n].x, hv[n].y, zero);
                else mma_f16(d[m][n], e, k ? hv[n].z : hv[n].x, k ? hv[n].w : hv[n].y, d[m][n]);
              }
            }
          }
          if (ends) {
            const int gi = (half * 4 + jw) / kWords;  // group of the box
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              const float x = bf16_at(sc[2 * m][gi >> 1], gi & 1), y = bf16_at(sc[2 * m + 1][gi >> 1], gi & 1);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                acc[m][n][0] = fmaf(x, d[m][n][0], acc[m][n][0]);
                acc[m][n][1] = fmaf(x, d[m][n][1], acc[m][n][1]);
                acc[m][n][2] = fmaf(y, d[m][n][2], acc[m][n][2]);
                acc[m][n][3] = fmaf(y, d[m][n][3], acc[m][n][3]);
              }
            }
          }
        }
      }
    }
    if (!ok) break;
    if (box0 == 0 && box1 == nb) {
      finish(tile);
    } else if (box0 > 0) {
      kept |= 1;
#pragma unroll
      for (int i = 0; i < 2 * NT * 4; ++i) first[i / (NT * 4)][(i >> 2) % NT][i & 3] = acc[i / (NT * 4)][(i >> 2) % NT][i & 3];
    } else {
      kept |= 2;
    }
    u += box1 - box0;
  }
  if (!ok) {
    // behind a wait that ran out: every issued copy lands before the CTA returns
    const int issued = __shfl_sync(0xffffffffu, cu, 0) - u0;
    for (int i = 0; i < a.slots; ++i) {
      const int n = issued / a.slots + (i < issued % a.slots ? 1 : 0);
      if (n > 0) mbar_wait(&full[warp][i], (n - 1) & 1, kWaitBudget);
    }
    atomicExch(a.err, 1);
  }
  // ---- tiles that warps share: the one that has the beginning adds the rest ----
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 2 * NT * 4; ++i)
    if (kept & 1) parts[i * 32 + lane] = first[i / (NT * 4)][(i >> 2) % NT][i & 3];
  __syncthreads();
  if ((kept & 2) && ok) {
    const int tile = tfirst + (u1 - 1) / nb;
    const int end = (tile + 1 - tfirst) * nb;
    for (int w = warp + 1; w < kFewWarps; ++w) {
      const int wu0 = static_cast<int>(units * w / kFewWarps), wu1 = static_cast<int>(units * (w + 1) / kFewWarps);
      if (wu0 >= end) break;
      if (wu0 == wu1) continue;
      const float* p = reinterpret_cast<const float*>(base + static_cast<size_t>(w) * ring_bytes);
#pragma unroll
      for (int i = 0; i < 2 * NT * 4; ++i) acc[i / (NT * 4)][(i >> 2) % NT][i & 3] += p[i * 32 + lane];
    }
    finish(tile);
  }
  __syncthreads();
  if (a.part && static_cast<int>(threadIdx.x) < a.B)
    a.part[static_cast<int64_t>(threadIdx.x) * gridDim.x + blockIdx.x] = best[threadIdx.x];
}

// ---------------------------------------------------------------------------
// Quantisation: a thread takes eight elements (a word of codes), the lanes of a
// group find its largest magnitude. 128256 x 4096: 763 us, bound by instructions
// (integer pipe 63% active); HBM needs 203 for the 2.5 bytes an element. It runs
// once for a weight.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256) q4_quantize_kernel(const uint16_t* __restrict__ w, int64_t ldw, int H, int V,
                                                          int group, uint8_t* __restrict__ q, int64_t ldq,
                                                          uint16_t* __restrict__ scale, int64_t lds) {
  const int words = H >> 3, lanes = group >> 3;  // 4, 8 or 16 lanes a group, within a warp
  const int64_t total = static_cast<int64_t>(V) * words;
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * blockDim.x; i0 < total; i0 += step) {
    const int64_t i = i0 + threadIdx.x;
    const bool in = i < total;  // groups are whole: all of a group's lanes, or none
    const int v = in ? static_cast<int>(i / words) : 0, c = in ? static_cast<int>(i % words) : 0;
    uint4 x = {0u, 0u, 0u, 0u};
    if (in) x = __ldg(reinterpret_cast<const uint4*>(w + static_cast<int64_t>(v) * ldw + 8 * c));
    const uint32_t xw[4] = {x.x, x.y, x.z, x.w};
    // |w| as bits, then the earlier element, then its sign
    const int first = (static_cast<int>(threadIdx.x) & (lanes - 1)) * 8;
    uint32_t key = 0u;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t bits = (xw[k >> 1] >> (16 * (k & 1))) & 0xffffu;
      const uint32_t kk = ((bits & 0x7fffu) << 8) | static_cast<uint32_t>((127 - first - k) << 1) | (bits >> 15);
      key = kk > key ? kk : key;
    }
    for (int o = lanes >> 1; o > 0; o >>= 1) {
      const uint32_t t = __shfl_xor_sync(0xffffffffu, key, o);
      key = t > key ? t : key;
    }
    const uint32_t mag = key >> 8;
    const float m = __uint_as_float(mag << 16);
    // scale = -m / 8: the largest element gets code 0
    float sabs = m * 0.125f;
    uint16_t sbits = __bfloat16_as_ushort(__float2bfloat16_rn(sabs));
    sabs = bf16_bits_to_f32(sbits);
    const bool bad = mag >= 0x7f80u;
    if (!(key & 1u)) sbits |= 0x8000u;  // a positive largest element
    if (sabs == 0.0f) sbits = 0;
    if (bad) sbits = 0x7fc0u;
    uint32_t word = 0u;
    if (bad || sabs == 0.0f) {
      word = 0x88888888u;
    } else {
      const bool fast = fixed_div_ok(sabs);
      const float y = __frcp_rn(sabs);
      const float sign = (key & 1u) ? 1.0f : -1.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float e = bf16_at(xw[k >> 1], k & 1);
        int code = __float2int_rn(sign * div_by(e, sabs, y, fast)) + 8;
        code = min(max(code, 0), 15);
        word |= static_cast<uint32_t>(code) << (4 * (k >> 1) + 16 * (k & 1));
      }
    }
    if (in) {
      *reinterpret_cast<uint32_t*>(q + static_cast<int64_t>(v) * ldq + 4 * c) = word;
      if (first == 0) scale[static_cast<int64_t>(v) * lds + c / lanes] = sbits;
    }
  }
}

rl_status q4_check(rl_sampler* h, const uint16_t* hidden, int64_t ldh, const rl_q4_weight* w, int B, int H, int V) {
  clear_error();
  if (!h) return set_error(RL_ERR_INVALID_ARG, "rl_lmhead_q4: handle is NULL");
  if (!w) return set_error(RL_ERR_INVALID_ARG, "rl_lmhead_q4: weight is NULL");
  if (B < 0 || H <= 0 || V <= 0 || ldh < H) return set_error(RL_ERR_INVALID_ARG, "rl_lmhead_q4: bad B / H / V / ld");
  if (w->group != 32 && w->group != 64 && w->group != 128)
    return set_error(RL_ERR_UNSUPPORTED, "rl_lmhead_q4: group must be 32, 64 or 128");
  if (H % 64 != 0 || H % w->group != 0)
    return set_error(RL_ERR_UNSUPPORTED, "rl_lmhead_q4: H must be a multiple of 64 and of the group");
  if (w->ldq < H / 2 || w->lds < H / w->group) return set_error(RL_ERR_INVALID_ARG, "rl_lmhead_q4: ldq or lds too small");
  if (w->ldq % 16) return set_error(RL_ERR_INVALID_ARG, "rl_lmhead_q4: ldq must be a multiple of 16 bytes");
  if (B > 0 && (!hidden || !w->q || !w->scale))
    return set_error(RL_ERR_INVALID_ARG, "rl_lmhead_q4: hidden, codes and scales are required");
  if (((reinterpret_cast<uintptr_t>(hidden) | reinterpret_cast<uintptr_t>(w->q)) & 15u) ||
      (reinterpret_cast<uintptr_t>(w->scale) & 1u))
    return set_error(RL_ERR_INVALID_ARG, "rl_lmhead_q4: hidden and codes must be 16-byte aligned, scales 2-byte");
  if (ldh % 8) return set_error(RL_ERR_INVALID_ARG, "rl_lmhead_q4: hidden's row stride must be a multiple of 8 elements");
  if (B > h->max_batch) return set_error(RL_ERR_SHAPE, "rl_lmhead_q4: B beyond the handle's max_batch");
  return RL_OK;
}

// A launch for at most N batch rows.
template <int N, int GS, int NDQ, int NEP>
cudaError_t q4_run(const CUtensorMap& mq, const CUtensorMap& mx, Q4Args a, int grid, cudaStream_t stream) {
  constexpr int kFixed = 1024 + kSSlots * kSBox + Q4Plan<N, GS>::kSlots * 2 * N * 128;
  constexpr int kRoom = (224 * 1024 - kFixed) / kQTile;
  a.qslots = kRoom < kQMax ? kRoom : kQMax;
  const size_t smem = kFixed + static_cast<size_t>(a.qslots) * kQTile;
  static std::atomic<int> configured[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(q4_mma_kernel<N, GS, NDQ, NEP>, cudaFuncAttributeMaxDynamicSharedMemorySize, 224 * 1024);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) configured[dev].store(1, std::memory_order_release);
  }
  q4_mma_kernel<N, GS, NDQ, NEP><<<grid, (4 + NDQ + NEP) * 32, smem, stream>>>(mq, mx, a);
  return cudaGetLastError();
}
template <int N, int NEP>
cudaError_t q4_run(const CUtensorMap& mq, const CUtensorMap& mx, const Q4Args& a, int group, int grid, cudaStream_t stream) {
  // groups of 32 go up to 64 batch rows a launch: two buffers of two groups
  if constexpr (N <= 64)
    if (group == 32) return q4_run<N, 5, 8, NEP>(mq, mx, a, grid, stream);
  if (group == 64) return q4_run<N, 6, 8, NEP>(mq, mx, a, grid, stream);
  if (group == 128) return q4_run<N, 7, 8, NEP>(mq, mx, a, grid, stream);
  return cudaErrorInvalidValue;
}

template <int NT, int GS, int HB>
cudaError_t few_run(const CUtensorMap& mq, const FewArgs& a, size_t smem, int grid, cudaStream_t stream) {
  static std::atomic<int> configured[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(q4_few_kernel<NT, GS, HB>, cudaFuncAttributeMaxDynamicSharedMemorySize, 224 * 1024);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) configured[dev].store(1, std::memory_order_release);
  }
  q4_few_kernel<NT, GS, HB><<<grid, kFewWarps * 32, smem, stream>>>(mq, a);
  return cudaGetLastError();
}

template <int NT, int HB>
cudaError_t few_run(const CUtensorMap& mq, const FewArgs& a, int group, size_t smem, int grid, cudaStream_t stream) {
  return group == 32   ? few_run<NT, 5, HB>(mq, a, smem, grid, stream)
         : group == 64 ? few_run<NT, 6, HB>(mq, a, smem, grid, stream)
                       : few_run<NT, 7, HB>(mq, a, smem, grid, stream);
}

// Up to 16 batch rows, where the hidden states fit shared memory beside the rings
// (H <= 8192 at 8 batch rows, 4096 at 16). us a call, few rows' kernel / the
// tensor cores' roles: 1 x 4096 x 128256 52 / 94, 12 rows of it 94 / 104, 1 x
// 2048 x 32000 14 / 18; behind 16 rows it would load each code again for every 16.
size_t few_hidden(int B, int H) { return static_cast<size_t>(B <= 8 ? 8 : 16) * ((H + 255) / 256) * 512; }
bool is_few(int B, int H) { return B <= 16 && few_hidden(B, H) <= kFewHidden; }

rl_status few_launch(rl_sampler* h, const uint16_t* hidden, int64_t ldh, const rl_q4_weight& w, int B, int H, int V,
                     float* out_f32, uint16_t* out_bf16, int64_t ldo, uint64_t* part, int* grid_out, cudaStream_t stream) {
  // boxes of K = 256 where two of them a warp fit beside the hidden states
  const size_t hs = few_hidden(B, H), room = 224 * 1024 - 1024 - hs;
  const int hb = room / (kFewWarps * kFewRows * 128) >= 2 ? 2 : 1;
  const size_t box = static_cast<size_t>(kFewRows) * 64 * hb;
  CUtensorMap mq;
  if (!lm_tensor_map(&mq, w.q, 1, H / 2, V, w.ldq, kFewRows, 64 * hb))
    return set_error(RL_ERR_INVALID_ARG, "rl_lmhead_q4: tensor map of the codes rejected (alignment or stride)");
  FewArgs a = {};
  a.hidden = hidden;
  a.ldh = ldh;
  a.B = B;
  a.H = H;
  a.V = V;
  a.ntiles = (V + kFewRows - 1) / kFewRows;
  a.boxes = (H + 128 * hb - 1) / (128 * hb);
  a.scale = w.scale;
  a.lds = w.lds;
  a.out_f32 = out_f32;
  a.out_bf16 = out_bf16;
  a.ldo = ldo;
  a.part = part;
  a.err = h->lm_err;
  const int scales = 128 * hb / w.group;  // of a box
  a.vec = H % (128 * hb) == 0 &&
          (reinterpret_cast<uintptr_t>(w.scale) | static_cast<uint64_t>(w.lds) * 2u) % (2u * static_cast<unsigned>(scales)) == 0;
  a.slots = static_cast<int>(room / (kFewWarps * box));
  if (a.slots > kFewSlots) a.slots = kFewSlots;
  const size_t smem = 1024 + static_cast<size_t>(a.slots) * kFewWarps * box + hs;
  const int grid = a.ntiles < h->num_sms ? a.ntiles : h->num_sms;
  *grid_out = grid;
  const cudaError_t e = B <= 8 ? (hb == 2 ? few_run<1, 2>(mq, a, w.group, smem, grid, stream)
                                          : few_run<1, 1>(mq, a, w.group, smem, grid, stream))
                               : (hb == 2 ? few_run<2, 2>(mq, a, w.group, smem, grid, stream)
                                          : few_run<2, 1>(mq, a, w.group, smem, grid, stream));
  if (e != cudaSuccess) return set_error(RL_ERR_CUDA, cudaGetErrorString(e));
  return RL_OK;
}

rl_status q4_launch(rl_sampler* h, const uint16_t* hidden, int64_t ldh, const rl_q4_weight& w, int B, int H, int V,
                    float* out_f32, uint16_t* out_bf16, int64_t ldo, int32_t* out_tok, int32_t* row_status, bool flagged,
                    cudaStream_t stream) {
  // the flag is read where there are statuses to give
  if (flagged && cudaMemsetAsync(h->lm_err, 0, sizeof(int), stream) != cudaSuccess)
    return set_error(RL_ERR_CUDA, "rl_lmhead_q4: cudaMemsetAsync failed");
  if (is_few(B, H)) {
    int grid = 0;
    rl_status st = few_launch(h, hidden, ldh, w, B, H, V, out_f32, out_bf16, ldo, out_tok ? h->lm_part : nullptr, &grid, stream);
    if (st != RL_OK) return st;
    if (out_tok) {
      const cudaError_t e = lm_argmax(h->lm_part, B, grid, h->lm_err, out_tok, row_status, stream);
      if (e != cudaSuccess) return set_error(RL_ERR_CUDA, cudaGetErrorString(e));
    }
    return RL_OK;
  }
  CUtensorMap mq;
  if (!lm_tensor_map(&mq, w.q, 1, H / 2, V, w.ldq, kBM))
    return set_error(RL_ERR_INVALID_ARG, "rl_lmhead_q4: tensor map of the codes rejected (alignment or stride)");
  Q4Args a = {};
  a.H = H;
  a.V = V;
  a.ntiles = (V + kBM - 1) / kBM;
  a.kstages = H / 64;
  a.scale = w.scale;
  a.lds = w.lds;
  const uint64_t al = reinterpret_cast<uintptr_t>(w.scale) | static_cast<uint64_t>(w.lds) * 2u |
                      static_cast<uint64_t>(H / w.group) * 2u;
  a.gran = al % 16 == 0 ? 16 : al % 8 == 0 ? 8 : al % 4 == 0 ? 4 : 2;
  a.ldo = ldo;
  a.err = h->lm_err;
  const int grid = a.ntiles < h->num_sms ? a.ntiles : h->num_sms;
  // batch rows a launch: two groups of 32 in a stage take 2 N columns, and two
  // buffers of them have to fit
  const int most = w.group == 32 ? 64 : 128;
  const int chunks = (B + most - 1) / most;
  const int per = (B + chunks - 1) / chunks;
  for (int b0 = 0; b0 < B; b0 += per) {
    const int Bc = B - b0 < per ? B - b0 : per;
    a.B = Bc;
    a.out_f32 = out_f32 ? out_f32 + static_cast<int64_t>(b0) * ldo : nullptr;
    a.out_bf16 = out_bf16 ? out_bf16 + static_cast<int64_t>(b0) * ldo : nullptr;
    a.part = out_tok ? h->lm_part : nullptr;
    const int N = Bc <= 16 ? 16 : Bc <= 32 ? 32 : Bc <= 64 ? 64 : Bc <= 96 ? 96 : 128;
    CUtensorMap mx;
    if (!lm_tensor_map(&mx, hidden + static_cast<int64_t>(b0) * ldh, 2, H, Bc, ldh * 2, N))
      return set_error(RL_ERR_INVALID_ARG, "rl_lmhead_q4: hidden tensor map rejected (alignment or stride)");
    cudaError_t e = N == 16   ? q4_run<16, 4>(mq, mx, a, w.group, grid, stream)
                    : N == 32 ? q4_run<32, 8>(mq, mx, a, w.group, grid, stream)
                    : N == 64 ? q4_run<64, 8>(mq, mx, a, w.group, grid, stream)
                    : N == 96 ? q4_run<96, 12>(mq, mx, a, w.group, grid, stream)
                              : q4_run<128, 16>(mq, mx, a, w.group, grid, stream);
    if (e == cudaSuccess && out_tok)
      e = lm_argmax(h->lm_part, Bc, grid, h->lm_err, out_tok + b0, row_status ? row_status + b0 : nullptr, stream);
    if (e != cudaSuccess) return set_error(RL_ERR_CUDA, cudaGetErrorString(e));
  }
  return RL_OK;
}

}  // namespace
}  // namespace rl

extern "C" {
#pragma GCC visibility push(default)

rl_status rl_lmhead_q4_quantize(rl_sampler* h, const uint16_t* weight, int64_t ldw, int H, int V, int group, uint8_t* q,
                                int64_t ldq, uint16_t* scale, int64_t lds, void* stream) {
  rl_q4_weight w = {q, ldq, scale, lds, group};
  rl_status st = rl::q4_check(h, weight, ldw, &w, V > 0 ? 1 : 0, H, V);
  if (st != RL_OK) return st;
  rl::LmDeviceGuard g(h->device);
  if (!g.ok) return rl::set_error(RL_ERR_CUDA, "rl_lmhead_q4_quantize: cudaSetDevice failed");
  const int64_t blocks = (static_cast<int64_t>(V) * (H / 8) + 255) / 256;
  const int64_t most = static_cast<int64_t>(h->num_sms) * 8;
  rl::q4_quantize_kernel<<<static_cast<unsigned>(blocks < most ? blocks : most), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      weight, ldw, H, V, group, q, ldq, scale, lds);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return rl::set_error(RL_ERR_CUDA, cudaGetErrorString(e));
  return RL_OK;
}

rl_status rl_lmhead_q4_logits(rl_sampler* h, const uint16_t* hidden, int64_t ldh, const rl_q4_weight* weight, int B,
                              int H, int V, void* out_logits, rl_dtype out_dtype, int64_t ldo, void* stream) {
  rl_status st = rl::q4_check(h, hidden, ldh, weight, B, H, V);
  if (st != RL_OK) return st;
  if (B > 0 && !out_logits) return rl::set_error(RL_ERR_INVALID_ARG, "rl_lmhead_q4_logits: out_logits is required");
  if (out_dtype != RL_F32 && out_dtype != RL_BF16)
    return rl::set_error(RL_ERR_INVALID_ARG, "rl_lmhead_q4_logits: bad dtype");
  if (ldo < V) return rl::set_error(RL_ERR_INVALID_ARG, "rl_lmhead_q4_logits: ldo < V");
  if (B == 0) return RL_OK;
  rl::LmDeviceGuard g(h->device);
  if (!g.ok) return rl::set_error(RL_ERR_CUDA, "rl_lmhead_q4_logits: cudaSetDevice failed");
  return rl::q4_launch(h, hidden, ldh, *weight, B, H, V, out_dtype == RL_F32 ? static_cast<float*>(out_logits) : nullptr,
                       out_dtype == RL_BF16 ? static_cast<uint16_t*>(out_logits) : nullptr, ldo, nullptr, nullptr, false,
                       static_cast<cudaStream_t>(stream));
}

rl_status rl_lmhead_q4_greedy(rl_sampler* h, const uint16_t* hidden, int64_t ldh, const rl_q4_weight* weight, int B,
                              int H, int V, int32_t* out_tok, int32_t* row_status, float* out_logits, int64_t ldo,
                              void* stream) {
  rl_status st = rl::q4_check(h, hidden, ldh, weight, B, H, V);
  if (st != RL_OK) return st;
  if (B > 0 && !out_tok) return rl::set_error(RL_ERR_INVALID_ARG, "rl_lmhead_q4_greedy: out_tok is required");
  if (out_logits && ldo < V) return rl::set_error(RL_ERR_INVALID_ARG, "rl_lmhead_q4_greedy: ldo < V");
  if (B == 0) return RL_OK;
  rl::LmDeviceGuard g(h->device);
  if (!g.ok) return rl::set_error(RL_ERR_CUDA, "rl_lmhead_q4_greedy: cudaSetDevice failed");
  return rl::q4_launch(h, hidden, ldh, *weight, B, H, V, out_logits, nullptr, ldo, out_tok, row_status, true,
                       static_cast<cudaStream_t>(stream));
}

rl_status rl_lmhead_q4_sample(rl_sampler* h, const uint16_t* hidden, int64_t ldh, const rl_q4_weight* weight, int B,
                              int H, int V, const int32_t* hist, const int32_t* hist_len, int hist_stride,
                              const rl_row_params* params, const float* uniforms, int32_t* out_tok, float* out_prob,
                              int32_t* row_status, void* stream) {
  rl_status st = rl::q4_check(h, hidden, ldh, weight, B, H, V);
  if (st != RL_OK) return st;
  if (V > h->max_vocab) return rl::set_error(RL_ERR_SHAPE, "rl_lmhead_q4_sample: V beyond the handle's max_vocab");
  if (B > 0 && (!params || !uniforms || !out_tok))
    return rl::set_error(RL_ERR_INVALID_ARG, "rl_lmhead_q4_sample: params, uniforms and out_tok are required");
  if (!h->stage_logits) return rl::set_error(RL_ERR_UNSUPPORTED, "rl_lmhead_q4_sample: handle without staging buffers");
  if (B == 0) return RL_OK;
  rl::LmDeviceGuard g(h->device);
  if (!g.ok) return rl::set_error(RL_ERR_CUDA, "rl_lmhead_q4_sample: cudaSetDevice failed");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  st = rl::q4_launch(h, hidden, ldh, *weight, B, H, V, h->stage_logits, nullptr, V, nullptr, nullptr, true, s);
  if (st != RL_OK) return st;
  st = rl_sample_batch(h, h->stage_logits, RL_F32, B, V, V, hist, hist_len, hist_stride, nullptr, 0, params, uniforms,
                       out_tok, out_prob, row_status, stream);
  if (st != RL_OK) return st;
  // a head whose wait ran out leaves its rows' logits undefined
  const cudaError_t e = rl::lm_flag(h->lm_err, B, out_tok, row_status, s);
  if (e != cudaSuccess) return rl::set_error(RL_ERR_CUDA, cudaGetErrorString(e));
  return RL_OK;
}

#pragma GCC visibility pop
}  // extern "C"
