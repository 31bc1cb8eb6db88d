// The LM head with 4-bit weights and group scales (rl_lmhead_q4_*; the format
// stands in rl_sampler.h):
//
//   logits[b, v] = sum_g scale[v, g] * sum_{k in g} (code[v, k] - 8) * hidden[b, k]
//
// code - 8 is a whole number in [-8, 7], so code - 8 times a bf16 value is exact
// in f32; a group's sum is multiplied by its scale once, in f32.
//
// A warp takes a vocabulary row, its lanes the row's words, for up to eight
// batch rows at a time.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <climits>

#include "common.cuh"
#include "internal.h"
#include "lmhead.cuh"

namespace rl {
namespace {

constexpr int kQ4Rows = 256;  // batch rows a launch handles (the size of the argmax workspace)

struct Q4Args {
  const uint16_t* hidden;
  int64_t ldh;
  const uint8_t* q;
  int64_t ldq;
  const uint16_t* scale;
  int64_t lds;
  int gshift;  // log2(group)
  int B, H, V;
  float* out_f32;
  uint16_t* out_bf16;
  int64_t ldo;
  uint64_t* part;  // [B] packed (value, id) maxima, or null
};

__device__ __forceinline__ float bf16_at(uint32_t w, int hi) { return __uint_as_float(hi ? w & 0xffff0000u : w << 16); }

__global__ void __launch_bounds__(256) q4_row_kernel(const __grid_constant__ Q4Args a) {
  const int v = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (v >= a.V) return;
  const uint32_t* q = reinterpret_cast<const uint32_t*>(a.q + static_cast<int64_t>(v) * a.ldq);
  const uint16_t* sc = a.scale + static_cast<int64_t>(v) * a.lds;
  for (int b0 = 0; b0 < a.B; b0 += 8) {
    float acc[8] = {};
    for (int w = lane; w < (a.H >> 3); w += 32) {
      const uint32_t x = q[w];
      const float s = bf16_bits_to_f32(sc[(w << 3) >> a.gshift]);
      float c[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        c[2 * j] = static_cast<float>(static_cast<int>((x >> (4 * j)) & 15u) - 8);
        c[2 * j + 1] = static_cast<float>(static_cast<int>((x >> (16 + 4 * j)) & 15u) - 8);
      }
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        if (b0 + b < a.B) {
          const uint4 h = *reinterpret_cast<const uint4*>(a.hidden + static_cast<int64_t>(b0 + b) * a.ldh + 8 * w);
          const uint32_t hw[4] = {h.x, h.y, h.z, h.w};
          float d = 0.0f;
#pragma unroll
          for (int k = 0; k < 8; ++k) d = fmaf(c[k], bf16_at(hw[k >> 1], k & 1), d);
          acc[b] = fmaf(s, d, acc[b]);
        }
      }
    }
#pragma unroll
    for (int b = 0; b < 8; ++b) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) acc[b] += __shfl_xor_sync(0xffffffffu, acc[b], o);
      if (lane == 0 && b0 + b < a.B) {
        const int64_t at = static_cast<int64_t>(b0 + b) * a.ldo + v;
        if (a.out_f32) a.out_f32[at] = acc[b];
        if (a.out_bf16) a.out_bf16[at] = __bfloat16_as_ushort(__float2bfloat16_rn(acc[b]));
        if (a.part)
          atomicMax(reinterpret_cast<unsigned long long*>(&a.part[b0 + b]), static_cast<unsigned long long>(lm_key(acc[b], v)));
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Quantisation: a thread takes eight elements (a word of codes), the lanes of a
// group find its largest magnitude. Bound by HBM (2.5 bytes an element).
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

rl_status q4_launch(rl_sampler* h, const uint16_t* hidden, int64_t ldh, const rl_q4_weight& w, int B, int H, int V,
                    float* out_f32, uint16_t* out_bf16, int64_t ldo, int32_t* out_tok, int32_t* row_status,
                    cudaStream_t stream) {
  if (cudaMemsetAsync(h->lm_err, 0, sizeof(int), stream) != cudaSuccess)
    return set_error(RL_ERR_CUDA, "rl_lmhead_q4: cudaMemsetAsync failed");
  for (int b0 = 0; b0 < B; b0 += kQ4Rows) {
    const int Bc = B - b0 < kQ4Rows ? B - b0 : kQ4Rows;
    Q4Args a = {};
    a.hidden = hidden + static_cast<int64_t>(b0) * ldh;
    a.ldh = ldh;
    a.q = w.q;
    a.ldq = w.ldq;
    a.scale = w.scale;
    a.lds = w.lds;
    a.gshift = w.group == 32 ? 5 : w.group == 64 ? 6 : 7;
    a.B = Bc;
    a.H = H;
    a.V = V;
    a.out_f32 = out_f32 ? out_f32 + static_cast<int64_t>(b0) * ldo : nullptr;
    a.out_bf16 = out_bf16 ? out_bf16 + static_cast<int64_t>(b0) * ldo : nullptr;
    a.ldo = ldo;
    a.part = out_tok ? h->lm_part : nullptr;
    cudaError_t e = cudaSuccess;
    if (a.part) e = cudaMemsetAsync(a.part, 0, sizeof(uint64_t) * Bc, stream);
    if (e != cudaSuccess) return set_error(RL_ERR_CUDA, cudaGetErrorString(e));
    q4_row_kernel<<<(V + 7) / 8, 256, 0, stream>>>(a);
    e = cudaGetLastError();
    if (e == cudaSuccess && out_tok)
      e = lm_argmax(a.part, Bc, 1, h->lm_err, out_tok + b0, row_status ? row_status + b0 : nullptr, stream);
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
                       out_dtype == RL_BF16 ? static_cast<uint16_t*>(out_logits) : nullptr, ldo, nullptr, nullptr,
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
  return rl::q4_launch(h, hidden, ldh, *weight, B, H, V, out_logits, nullptr, ldo, out_tok, row_status,
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
  st = rl::q4_launch(h, hidden, ldh, *weight, B, H, V, h->stage_logits, nullptr, V, nullptr, nullptr, s);
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
