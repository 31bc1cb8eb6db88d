// Verification of drafted tokens against the target's probabilities
// (rl_specdec_verify_draft, rl_specdec_verify_tree; the semantics stand in
// rl_sampler.h).
//
// Mathematics. p and q are softmaxes over a row's kept ids. A child x drawn
// from q is accepted iff u q(x) S < w(x); w starts as p (S = 1) and every
// refusal makes it max(w - S q, 0). Since max(max(a - b, 0) - c, 0) =
// max(a - b - c, 0) for b, c >= 0, w stays max(p - C q, 0) with one number C,
// the sum of the S so far: no residual row is ever written. The token behind
// the last refusal is the first id whose running sum of w is over u S.
//
// One cluster of CTAs walks one sequence, node by node, so rows behind the
// first refusal are never read (with a draft that is right 70% of the time
// that is half of the rows of a chain of four). Every CTA holds a contiguous
// eighth, quarter, ... of the ids, every warp a contiguous part of that, and
// a lane keeps (max, sum of 2^((x - max) c)) of what it sees: one pass per
// row. The parts' sums are joined through distributed shared memory and give
// Z, the accept tests, and later the part in which the drawn token lies: only
// that part is looked at again. A refusal with a draft row costs a second
// pass over the two rows (from L2) for the sums of w.
//
// Precision: 2^t is ex2.approx (relative error about 2^-22, no bias that
// p and q or two ids would not share); 1 / T is carried as two floats, so
// that no error of 1 / T tilts a distribution; sums are doubles. Draws are
// compared in doubles: a token can differ from the exact one only where the
// draw lies within about 1e-9 of a border.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <climits>

#include "common.cuh"
#include "internal.h"

namespace rl {
namespace {

constexpr int kVT = 512;
constexpr int kVW = kVT / 32;

struct VdSide {
  const void* logits;
  int64_t ld;
  const float* T;
  const uint32_t* mask;
  int64_t mask_stride;
  const int32_t* cut;
  int64_t cut_stride;
  const int32_t* first_row;
  int rows;
  int per_seq;  // rows of a sequence without first_row
};

struct VdArgs {
  VdSide p, q;
  int has_q;
  int V, N;                // N: nodes of the widest sequence (outputs' row stride)
  const int32_t* tokens;   // node i's token and uniform at b * tok_stride + i - tok_off
  const float* accept_u;
  int tok_stride, tok_off;
  const int32_t* parent;   // null: a chain
  const int32_t* count;    // nodes = count[b] + count_add
  int count_add;
  const float* draw_u;
  int32_t* out_accepted;
  int32_t* out_path;
  int32_t* out_tok;
  float* out_prob;
  int32_t* row_status;
};

// 1 / T in base 2, as two floats.
struct Scale {
  float hi, lo;
  double d;
};

__device__ __forceinline__ Scale scale_of(float T) {
  Scale c;
  c.d = fmin(fmax(1.4426950408889634074 / static_cast<double>(T), 1e-30), 3e38);
  c.hi = static_cast<float>(c.d);
  // beyond 1e7 two logits that differ at all are far apart, and lo times a
  // large difference could overflow
  c.lo = c.hi < 1e7f ? static_cast<float>(c.d - static_cast<double>(c.hi)) : 0.0f;
  return c;
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float ex2(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}
// 2^((x - m) c); 0 for x = -inf, NaN for NaN and for x = m = +inf.
__device__ __forceinline__ float weight(float x, float m, const Scale& c) {
  const float d = max_nan(x - m, -3.402823466e38f);
  return ex2(__fmaf_rn(d, c.hi, d * c.lo));
}

// A row of logits with what decides which of its ids are kept.
template <typename T>
struct Row {
  const T* x;
  const uint32_t* mask;  // null: no mask, or one that allows every id
  int V;
  int cut;               // -1: none
  float xcut;
  Scale c;
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ float kept(const Row<T>& r, float x, int j, uint32_t allowed) {
  if (!allowed) return RL_NEG_INF;
  // written so that a NaN stays
  if (r.cut >= 0 && (x < r.xcut || (x == r.xcut && j > r.cut))) return RL_NEG_INF;
  return x;
}

template <typename T>
__device__ __forceinline__ float logit_at(const Row<T>& r, int j) {
  if (static_cast<unsigned>(j) >= static_cast<unsigned>(r.V)) return RL_NEG_INF;
  const uint32_t a = r.mask ? (r.mask[j >> 5] >> (j & 31)) & 1u : 1u;
  return kept(r, to_f(r.x[j]), j, a);
}

// Eight ids of a row, j0 .. j0 + 7, as 16-byte loads where the row's address
// allows and all eight lie in the row.
template <typename T>
__device__ __forceinline__ void load8(const Row<T>& r, int j0, bool aligned, float (&x)[8]);

template <>
__device__ __forceinline__ void load8<float>(const Row<float>& r, int j0, bool aligned, float (&x)[8]) {
  if (aligned && j0 >= 0 && j0 <= r.V - 8) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(r.x + j0));
    const float4 b = __ldg(reinterpret_cast<const float4*>(r.x + j0 + 4));
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      x[k] = static_cast<unsigned>(j0 + k) < static_cast<unsigned>(r.V) ? __ldg(r.x + j0 + k) : RL_NEG_INF;
  }
}

template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const Row<__nv_bfloat16>& r, int j0, bool aligned, float (&x)[8]) {
  if (aligned && j0 >= 0 && j0 <= r.V - 8) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(r.x + j0));
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[2 * k] = __uint_as_float(w[k] << 16);
      x[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      x[k] = static_cast<unsigned>(j0 + k) < static_cast<unsigned>(r.V) ? to_f(r.x[j0 + k]) : RL_NEG_INF;
  }
}

// Puts -inf in the places of the eight that are not kept.
template <typename T>
__device__ __forceinline__ void keep8(const Row<T>& r, int j0, float (&x)[8]) {
  if (r.mask) {
    uint32_t bits = 0;
    if (j0 >= 0) {
      const int w = j0 >> 5, s = j0 & 31;
      if (j0 < r.V) {
        const uint32_t lo = r.mask[w];
        const uint32_t hi = s > 24 && ((w + 1) << 5) < r.V ? r.mask[w + 1] : 0u;
        bits = __funnelshift_r(lo, hi, s);
      }
    } else {
      bits = r.mask[0] << -j0;  // -8 < j0 < 0
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (!((bits >> k) & 1u)) x[k] = RL_NEG_INF;
  }
  if (r.cut >= 0) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (x[k] < r.xcut || (x[k] == r.xcut && j0 + k > r.cut)) x[k] = RL_NEG_INF;
  }
}

// The ids are cut into groups of eight that start on 16-byte boundaries of
// the target row: group g holds ids 8 g - off .. 8 g - off + 7.
template <typename T>
__device__ __forceinline__ int lead(const T* x) {
  return static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
}
template <typename T>
__device__ __forceinline__ bool lines_up(const T* x, int off) {
  return ((reinterpret_cast<uintptr_t>(x) - static_cast<uintptr_t>(off) * sizeof(T)) & 15u) == 0;
}

__device__ __forceinline__ double shfl_d(double v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }

struct Part {
  double s;  // sum of weights, relative to m
  float m;
  int id;    // lowest id at m (rows with T <= 0)
};

struct Ctl {
  Part part[2][2][kVW];  // [parity][side][warp]
  Part cta[2][2];        // [parity][side], read by the other CTAs
  Part all[2];           // [side] joined: s relative to m
  double wsum[kVW];      // this CTA's warps' sums of w, in units of the joined frame
  double scan[kVW];
  double ctaw[2];        // [parity] this CTA's sum of w, read by the other CTAs
  double before, total;  // sums of w in the CTAs before the draw's, and in all
  float cx[RL_VERIFY_MAX_NODES], cq[RL_VERIFY_MAX_NODES];  // children's logits
  float cu[RL_VERIFY_MAX_NODES];
  int child[RL_VERIFY_MAX_NODES], ctok[RL_VERIFY_MAX_NODES];
  int removed[RL_VERIFY_MAX_NODES];
  int nchild, nremoved;
  int next;      // accepted child, -1: none, -2: sums of w wanted
  int at;        // first id found by the draw
  int owner;     // CTA that holds the drawn token, and its warp
  int ownerw;
  int status;
  double rest;   // draw target inside the owner's warp
  double C, S, px;
  int k;         // next child to try
};

// One pass over this warp's groups of a row: (max, sum), or the argmax.
template <typename T>
__device__ Part row_part(const Row<T>& r, int off, bool greedy, int g0, int g1) {
  const int lane = threadIdx.x & 31;
  const bool al = lines_up(r.x, off);
  float m = RL_NEG_INF;
  double s = 0.0;
  int id = INT_MAX;
  constexpr int U = sizeof(T) == 4 ? 2 : 4;
  for (int g = g0 + lane; g < g1; g += 32 * U) {
    float x[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (g + 32 * u < g1) {
        load8<T>(r, 8 * (g + 32 * u) - off, al, x[u]);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[u][k] = RL_NEG_INF;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j0 = 8 * (g + 32 * u) - off;
      if ((r.mask || r.cut >= 0) && g + 32 * u < g1) keep8<T>(r, j0, x[u]);
      float gm = x[u][0];
#pragma unroll
      for (int k = 1; k < 8; ++k) gm = max_nan(gm, x[u][k]);
      if (greedy) {
        if (gm > m) {
          m = gm;
#pragma unroll
          for (int k = 7; k >= 0; --k)
            if (x[u][k] == gm) id = j0 + k;
        }
        if (gm != gm) s = __longlong_as_double(0x7ff8000000000000LL);
        continue;
      }
      if (gm > m) {
        s *= static_cast<double>(weight(m, gm, r.c));
        m = gm;
      }
      if (m == RL_NEG_INF && gm == gm) continue;
      float e = 0.0f;
#pragma unroll
      for (int k = 0; k < 8; k += 2) e += weight(x[u][k], m, r.c) + weight(x[u][k + 1], m, r.c);
      s += static_cast<double>(e);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o);
    const int id2 = __shfl_xor_sync(0xffffffffu, id, o);
    const double s2 = shfl_d(s, o);
    const float mm = fmaxf(m, m2);
    if (greedy) {
      id = m2 > m ? id2 : (m2 == m ? min(id, id2) : id);
      s += s2;  // NaN marks a NaN
    } else {
      const double a = m == mm ? s : s * exp2((static_cast<double>(m) - mm) * r.c.d);
      const double b = m2 == mm ? s2 : s2 * exp2((static_cast<double>(m2) - mm) * r.c.d);
      s = a + b;
    }
    m = mm;
  }
  Part p;
  p.s = s;
  p.m = m;
  p.id = id;
  return p;
}

// Joins the parts held by the lanes of a warp (lanes without one hold
// m = -inf, s = 0). Weights more than 126 binades below the largest drop out.
__device__ __forceinline__ Part join_parts(Part p, bool greedy, double c) {
  float m = p.m;
  int id = p.id;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o);
    const int id2 = __shfl_xor_sync(0xffffffffu, id, o);
    id = m2 > m ? id2 : (m2 == m ? min(id, id2) : id);
    m = fmaxf(m, m2);
  }
  double s = p.s;
  if (!greedy && p.m != m) {
    const double t = (static_cast<double>(p.m) - static_cast<double>(m)) * c;
    s = t >= -126.0 ? s * exp2(t) : (s == s ? 0.0 : s);
  }
  s = warp_sum_d(s);
  Part r;
  r.s = s;
  r.m = m;
  r.id = id;
  return r;
}

// Whether id j is one of the refused given tokens.
__device__ __forceinline__ bool is_removed(const Ctl& sh, int n, int j) {
  for (int k = 0; k < n; ++k)
    if (sh.removed[k] == j) return true;
  return false;
}

// The weights w of eight ids: max(p rho - q, 0) with a draft row (in units of
// q's largest), else p without the refused tokens (in units of p's largest).
template <typename TP, typename TQ>
__device__ __forceinline__ void w8(const Row<TP>& rp, const Row<TQ>& rq, float mp, float mq, float rhi, float rlo,
                                   bool resid, const Ctl& sh, int nrem, int g, int off, bool alp, bool alq,
                                   float (&w)[8]) {
  const int j0 = 8 * g - off;
  float x[8];
  load8<TP>(rp, j0, alp, x);
  if (rp.mask || rp.cut >= 0) keep8<TP>(rp, j0, x);
  if (resid) {
    float y[8];
    load8<TQ>(rq, j0, alq, y);
    if (rq.mask || rq.cut >= 0) keep8<TQ>(rq, j0, y);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float ep = weight(x[k], mp, rp.c), eq = weight(y[k], mq, rq.c);
      w[k] = fmaxf(__fmaf_rn(ep, rhi, __fmaf_rn(ep, rlo, -eq)), 0.0f);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      w[k] = weight(x[k], mp, rp.c);
      if (nrem > 0 && is_removed(sh, nrem, j0 + k)) w[k] = 0.0f;
    }
  }
}

// The CTA that holds the draw's target u * total, from the CTAs' sums (one per
// lane; every CTA finds the same one), the sums before it, and the total. The
// last CTA with any weight where rounding leaves no sum over the target; -1
// where there is no weight.
__device__ __forceinline__ double find_owner(Ctl& sh, double mine, float u) {
  const int lane = threadIdx.x & 31;
  double incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  const double total = __shfl_sync(0xffffffffu, incl, 31);
  const unsigned hit = __ballot_sync(0xffffffffu, mine > 0.0 && incl > static_cast<double>(u) * total);
  const unsigned some = __ballot_sync(0xffffffffu, mine > 0.0);
  const int own = hit ? __ffs(hit) - 1 : 31 - __clz(some);
  const double before = __shfl_sync(0xffffffffu, incl - mine, own & 31);
  if (lane == 0) {
    sh.owner = own;
    sh.before = before;
    sh.total = total;
  }
  return total;
}

template <typename T>
__device__ __forceinline__ Row<T> make_row(const VdSide& a, int64_t row, int V, float T_) {
  Row<T> r;
  r.x = static_cast<const T*>(a.logits) + row * a.ld;
  r.V = V;
  r.mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
  r.cut = a.cut ? a.cut[row * a.cut_stride] : -1;
  if (static_cast<unsigned>(r.cut) >= static_cast<unsigned>(V)) r.cut = -1;
  r.xcut = r.cut >= 0 ? to_f(r.x[r.cut]) : 0.0f;
  r.c = scale_of(T_);
  return r;
}

// A mask row without a bit allows every id (block-wide).
template <typename T>
__device__ __forceinline__ void drop_empty_mask(Row<T>& r) {
  if (!r.mask) return;
  const int words = (r.V + 31) >> 5;
  uint32_t any = 0;
  for (int w = threadIdx.x; w < words; w += kVT) {
    uint32_t m = r.mask[w];
    if (w == words - 1 && (r.V & 31)) m &= (1u << (r.V & 31)) - 1u;
    any |= m;
  }
  if (!__syncthreads_or(any != 0u)) r.mask = nullptr;
}

template <typename TP, typename TQ>
__global__ void __launch_bounds__(kVT, 2) verify_kernel(const __grid_constant__ VdArgs a) {
  __shared__ Ctl sh;
  namespace cgx = cooperative_groups;
  const cgx::cluster_group cl = cgx::this_cluster();
  const int C = static_cast<int>(cl.num_blocks());
  const int rank = static_cast<int>(cl.block_rank());
  const int b = blockIdx.x / C;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int V = a.V, N = a.N;
  int32_t* out_tok = a.out_tok + static_cast<int64_t>(b) * N;
  int32_t* out_path = a.out_path ? a.out_path + static_cast<int64_t>(b) * N : nullptr;
  float* out_prob = a.out_prob ? a.out_prob + static_cast<int64_t>(b) * N : nullptr;
  const int32_t* tokens = a.tokens + static_cast<int64_t>(b) * a.tok_stride - a.tok_off;
  const float* accept_u = a.accept_u + static_cast<int64_t>(b) * a.tok_stride - a.tok_off;
  const int32_t* parent = a.parent ? a.parent + static_cast<int64_t>(b) * a.tok_stride : nullptr;

  // ---- the sequence's numbers, checked ----
  const int n = a.count[b] + a.count_add;
  const float Tp = a.p.T ? a.p.T[b] : 1.0f;
  const float Tq = a.has_q && a.q.T ? a.q.T[b] : 1.0f;
  const bool greedy = Tp <= 0.0f;
  const bool drawn = a.has_q && !(Tq <= 0.0f) && !greedy;  // q comes from draft rows
  const int64_t p0 = a.p.first_row ? a.p.first_row[b] : static_cast<int64_t>(b) * a.p.per_seq;
  const int64_t q0 = a.has_q ? (a.q.first_row ? a.q.first_row[b] : static_cast<int64_t>(b) * a.q.per_seq) : 0;
  int status = RL_OK;
  if (n < 1 || n > N || p0 < 0 || p0 + n > a.p.rows) status = RL_ERR_INVALID_ARG;
  // the last node of a chain has no children, and no draft row
  else if (drawn && n > 1 && (q0 < 0 || q0 + n - (parent ? 0 : 1) > a.q.rows)) status = RL_ERR_INVALID_ARG;
  else if (!(fabsf(Tp) < RL_POS_INF) || !(fabsf(Tq) < RL_POS_INF)) status = RL_ERR_NONFINITE;

  int node = 0, acc = 0, par = 0;
  int token = -1;     // drawn token, in the CTA that finds it (thread 0)
  double tprob = 0.0;
  bool found = false;
  while (status == RL_OK) {
    // ---- the node's children (thread-uniform), their logits ----
    Row<TP> rp = make_row<TP>(a.p, p0 + node, V, greedy ? 1.0f : Tp);
    const int off = lead(rp.x);
    drop_empty_mask(rp);
    if (warp == 0) {
      int c = 0;
      if (parent) {
        for (int i0 = node + 1; i0 < n; i0 += 32) {
          const bool is = i0 + lane < n && parent[i0 + lane] == node;
          const unsigned k = __ballot_sync(0xffffffffu, is);
          if (is) sh.child[c + __popc(k & ((1u << lane) - 1u))] = i0 + lane;
          c += __popc(k);
        }
      } else if (node + 1 < n) {
        if (lane == 0) sh.child[0] = node + 1;
        c = 1;
      }
      if (lane == 0) {
        sh.nchild = c;
        sh.nremoved = 0;
      }
    }
    __syncthreads();
    const int nchild = sh.nchild;
    const bool with_q = drawn && nchild > 0;
    Row<TQ> rq = {};
    if (with_q) {
      rq = make_row<TQ>(a.q, q0 + node, V, Tq);
      drop_empty_mask(rq);
    }
    for (int k = tid; k < nchild; k += kVT) {
      const int t = tokens[sh.child[k]];
      sh.ctok[k] = t;
      sh.cu[k] = accept_u[sh.child[k]];
      sh.cx[k] = logit_at(rp, t);
      sh.cq[k] = with_q ? logit_at(rq, t) : RL_NEG_INF;
    }
    // ---- this warp's part of the ids ----
    const int groups = (off + V + 7) >> 3;
    const int per_cta = (groups + C - 1) / C;
    const int per_warp = (per_cta + kVW - 1) / kVW;
    const int c1 = min((rank + 1) * per_cta, groups);
    const int g0 = min(rank * per_cta + warp * per_warp, c1), g1 = min(g0 + per_warp, c1);
    // ---- sums of both rows, joined over the CTA and the cluster ----
    {
      const Part pp = row_part<TP>(rp, off, greedy, g0, g1);
      if (lane == 0) sh.part[par][0][warp] = pp;
      if (with_q) {
        const Part pq = row_part<TQ>(rq, off, false, g0, g1);
        if (lane == 0) sh.part[par][1][warp] = pq;
      }
    }
    __syncthreads();
    if (warp < (with_q ? 2 : 1)) {
      const double c = warp ? rq.c.d : rp.c.d;
      Part e = {0.0, RL_NEG_INF, INT_MAX};
      if (lane < kVW) e = sh.part[par][warp][lane];
      e = join_parts(e, greedy, c);
      if (lane == 0) sh.cta[par][warp] = e;
    }
    cl.sync();
    if (warp < (with_q ? 2 : 1)) {
      const double c = warp ? rq.c.d : rp.c.d;
      Part e = {0.0, RL_NEG_INF, INT_MAX};
      if (lane < C) e = *cl.map_shared_rank(&sh.cta[par][warp], lane);
      e = join_parts(e, greedy, c);
      if (lane == 0) sh.all[warp] = e;
    }
    par ^= 1;
    __syncthreads();
    const Part P = sh.all[0];
    const Part Q = with_q ? sh.all[1] : Part{1.0, 0.0f, 0};
    if (P.s != P.s || !(fabsf(P.m) < RL_POS_INF) || Q.s != Q.s || !(fabsf(Q.m) < RL_POS_INF)) {
      status = RL_ERR_NONFINITE;
      break;
    }
    const bool alp = lines_up(rp.x, off), alq = with_q && lines_up(rq.x, off);
    // ---- accept tests: thread 0 of every CTA, all alike ----
    bool sums = false;  // sh.wsum / sh.total hold the sums of w
    if (tid == 0) {
      sh.C = 0.0;
      sh.S = 1.0;
      sh.k = 0;
    }
    int next = -1;
    float rhi = 0.0f, rlo = 0.0f;
    while (true) {
      if (tid == 0) {
        int k = sh.k, nx = -1;
        for (; k < nchild; ++k) {
          if (greedy) {
            if (sh.ctok[k] == P.id) {
              nx = sh.child[k];
              sh.px = 1.0;
              break;
            }
            continue;
          }
          const float x = sh.cx[k];
          const double px = x > RL_NEG_INF ? exp2((static_cast<double>(x) - P.m) * rp.c.d) / P.s : 0.0;
          if (with_q) {
            const float y = sh.cq[k];
            const double qx = y > RL_NEG_INF ? exp2((static_cast<double>(y) - Q.m) * rq.c.d) / Q.s : 0.0;
            if (static_cast<double>(sh.cu[k]) * qx * sh.S < px - sh.C * qx) {
              nx = sh.child[k];
              sh.px = px;
              break;
            }
            sh.C += sh.S;  // refused: the sums of the new w are wanted
            nx = -2;
            ++k;
            break;
          }
          const bool gone = is_removed(sh, sh.nremoved, sh.ctok[k]);
          if (!gone && static_cast<double>(sh.cu[k]) * sh.S < px) {
            nx = sh.child[k];
            sh.px = px;
            break;
          }
          if (!gone && px > 0.0) {
            sh.removed[sh.nremoved++] = sh.ctok[k];
            sh.S = fmax(sh.S - px, 0.0);
          }
        }
        sh.k = k;
        sh.next = nx;
      }
      __syncthreads();
      next = sh.next;
      if (next != -2) break;
      // ---- sums of w = max(p - C q, 0) over the parts ----
      const double rho = Q.s / (sh.C * P.s);
      rhi = static_cast<float>(rho);
      rlo = static_cast<float>(rho - static_cast<double>(rhi));
      double s = 0.0;
      for (int g = g0 + lane; g < g1; g += 32) {
        float w[8];
        w8<TP, TQ>(rp, rq, P.m, Q.m, rhi, rlo, true, sh, 0, g, off, alp, alq, w);
        s += static_cast<double>(((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7])));
      }
      s = warp_sum_d(s);
      if (lane == 0) sh.wsum[warp] = s;
      __syncthreads();
      if (warp == 0) {
        const double t = warp_sum_d(lane < kVW ? sh.wsum[lane] : 0.0);
        if (lane == 0) sh.ctaw[par] = t;
      }
      cl.sync();
      if (warp == 0) {
        const double mine = lane < C ? *cl.map_shared_rank(&sh.ctaw[par], lane) : 0.0;
        const double all = find_owner(sh, mine, a.draw_u[b]);
        if (lane == 0) sh.S = all * sh.C / Q.s;  // as a probability
      }
      par ^= 1;
      sums = true;
      __syncthreads();
    }
    if (next >= 0) {
      if (rank == 0 && tid == 0) {
        out_tok[acc] = tokens[next];
        if (out_path) out_path[acc] = next;
        if (out_prob) out_prob[acc] = static_cast<float>(sh.px);
      }
      node = next;
      ++acc;
      __syncthreads();  // sh.child ... are rewritten for the next node
      continue;
    }
    // ---- no child is accepted: the last token ----
    if (greedy) {
      if (rank == 0 && tid == 0) {
        token = P.id;
        tprob = 1.0;
        found = true;
      }
      break;
    }
    const bool resid = sums && sh.total > 0.0;  // all of w rounded away: from p
    const int nrem = sh.nremoved;
    if (!resid) {
      // w = p, without refused given tokens: their warps sum again
      double f = 0.0;
      if (lane == 0) {
        const Part e = sh.part[par ^ 1][0][warp];
        const double t = (static_cast<double>(e.m) - static_cast<double>(P.m)) * rp.c.d;
        f = t >= -126.0 ? e.s * exp2(t) : 0.0;
      }
      if (sums) f = 0.0;
      bool again = sums;  // the parts' buffer may hold a later exchange
      for (int k = 0; k < nrem; ++k) {
        const int g = (sh.removed[k] + off) >> 3;
        again |= g >= g0 && g < g1;
      }
      if (again) {
        double s = 0.0;
        for (int g = g0 + lane; g < g1; g += 32) {
          float w[8];
          w8<TP, TQ>(rp, rq, P.m, Q.m, 0.0f, 0.0f, false, sh, nrem, g, off, alp, false, w);
          s += static_cast<double>(((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7])));
        }
        f = warp_sum_d(s);
      }
      if (lane == 0) sh.wsum[warp] = f;
      __syncthreads();
      if (warp == 0) {
        const double t = warp_sum_d(lane < kVW ? sh.wsum[lane] : 0.0);
        if (lane == 0) sh.ctaw[par] = t;
      }
      cl.sync();
      if (warp == 0) {
        const double mine = lane < C ? *cl.map_shared_rank(&sh.ctaw[par], lane) : 0.0;
        find_owner(sh, mine, a.draw_u[b]);
      }
      par ^= 1;
      __syncthreads();
    }
    // ---- which warp of which CTA holds the drawn token ----
    if (warp == 0) {
      const double t = static_cast<double>(a.draw_u[b]) * sh.total;
      const double w = lane < kVW ? sh.wsum[lane] : 0.0;
      double incl = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      // where rounding leaves no sum over t: the last part with any weight
      const unsigned hit = __ballot_sync(0xffffffffu, w > 0.0 && sh.before + incl > t);
      const unsigned some = __ballot_sync(0xffffffffu, w > 0.0);
      const int pick = hit ? __ffs(hit) - 1 : 31 - __clz(some);
      const double from = __shfl_sync(0xffffffffu, sh.before + incl - w, pick & 31);
      if (lane == 0) {
        sh.ownerw = pick;
        sh.rest = t - from;
        sh.at = INT_MAX;
      }
    }
    __syncthreads();
    if (sh.owner == rank) {
      // ---- the drawn token inside that warp's part, by the whole CTA ----
      const int w0 = min(rank * per_cta + sh.ownerw * per_warp, c1), w1 = min(w0 + per_warp, c1);
      const int per = (w1 - w0 + kVT - 1) / kVT;
      const int a0 = min(w0 + tid * per, w1), a1 = min(a0 + per, w1);
      double s = 0.0;
      int last = -1;
      for (int g = a0; g < a1; ++g) {
        float w[8];
        w8<TP, TQ>(rp, rq, P.m, Q.m, rhi, rlo, resid, sh, nrem, g, off, alp, alq, w);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          s += static_cast<double>(w[k]);
          if (w[k] > 0.0f) last = 8 * g - off + k;
        }
      }
      double incl = s;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      if (lane == 31) sh.scan[warp] = incl;
      __syncthreads();
      double base = 0.0;
      for (int w = 0; w < warp; ++w) base += sh.scan[w];
      double run = base + incl - s;
      if (run + s > sh.rest && s > 0.0) {
        for (int g = a0; g < a1; ++g) {
          float w[8];
          w8<TP, TQ>(rp, rq, P.m, Q.m, rhi, rlo, resid, sh, nrem, g, off, alp, alq, w);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            run += static_cast<double>(w[k]);
            if (w[k] > 0.0f && run > sh.rest) {
              atomicMin(&sh.at, 8 * g - off + k);
              g = a1;
              break;
            }
          }
        }
      }
      __syncthreads();
      if (sh.at == INT_MAX) {
        // the sums reach the target only by their rounding: the last id with weight
        __syncthreads();
        if (tid == 0) sh.at = -1;
        __syncthreads();
        if (last >= 0) atomicMax(&sh.at, last);
        __syncthreads();
      }
      if (tid == 0) {
        token = sh.at;
        if (token >= 0) {
          const float x = logit_at(rp, token);
          tprob = exp2((static_cast<double>(x) - P.m) * rp.c.d) / P.s;
        }
        found = true;
      }
    } else if (sh.owner < 0 && rank == 0 && tid == 0) {
      found = true;  // every id with weight was refused (uniforms of 1): no token
    }
    break;
  }
  // ---- outputs ----
  if (found) {
    out_tok[acc] = token;
    if (out_prob) out_prob[acc] = static_cast<float>(tprob);
  }
  if (rank == 0) {
    const int from = status == RL_OK ? acc + 1 : 0;
    for (int i = from + tid; i < N; i += kVT) {
      out_tok[i] = -1;
      if (out_prob) out_prob[i] = 0.0f;
    }
    if (out_path)
      for (int i = (status == RL_OK ? acc : 0) + tid; i < N; i += kVT) out_path[i] = -1;
    if (tid == 0) {
      a.out_accepted[b] = status == RL_OK ? acc : -1;
      if (a.row_status) a.row_status[b] = status;
    }
  }
  cl.sync();  // no CTA leaves while another may read its shared memory
}

struct VdGuard {
  int prev = -1;
  bool ok = true;
  explicit VdGuard(int dev) {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    if (prev != dev) ok = cudaSetDevice(dev) == cudaSuccess;
  }
  ~VdGuard() {
    int cur = -1;
    if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev) cudaSetDevice(prev);
  }
};

template <typename TP, typename TQ>
cudaError_t launch(const VdArgs& a, int B, int C, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(B) * C);
  cfg.blockDim = dim3(kVT);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, verify_kernel<TP, TQ>, a);
}

rl_status side_of(const rl_dist_rows* d, int V, int per_seq, VdSide* s) {
  if (!d->logits && d->rows != 0) return set_error(RL_ERR_INVALID_ARG, "rl_specdec_verify: a row set has no logits");
  if (d->dtype != RL_F32 && d->dtype != RL_BF16) return set_error(RL_ERR_INVALID_ARG, "rl_specdec_verify: bad dtype");
  if (d->ld < V || d->rows < 0) return set_error(RL_ERR_INVALID_ARG, "rl_specdec_verify: bad ld or rows");
  if (reinterpret_cast<uintptr_t>(d->logits) % (d->dtype == RL_F32 ? 4u : 2u))
    return set_error(RL_ERR_INVALID_ARG, "rl_specdec_verify: logits are not aligned to their type");
  if (d->mask && d->mask_stride < (V + 31) / 32)
    return set_error(RL_ERR_INVALID_ARG, "rl_specdec_verify: mask_stride is less than a row of V bits");
  if (d->cut && d->cut_stride < 0) return set_error(RL_ERR_INVALID_ARG, "rl_specdec_verify: bad cut_stride");
  s->logits = d->logits;
  s->ld = d->ld;
  s->T = d->temperature;
  s->mask = d->mask;
  s->mask_stride = d->mask_stride;
  s->cut = d->cut;
  s->cut_stride = d->cut_stride;
  s->first_row = d->first_row;
  s->rows = d->rows;
  s->per_seq = per_seq;
  return RL_OK;
}

rl_status verify(rl_sampler* h, int B, int V, VdArgs& a, const rl_dist_rows* target, const rl_dist_rows* draft,
                 int q_per_seq, cudaStream_t stream) {
  rl_status st = side_of(target, V, a.N, &a.p);
  if (st != RL_OK) return st;
  if (!target->first_row && static_cast<int64_t>(B) * a.N > target->rows)
    return set_error(RL_ERR_SHAPE, "rl_specdec_verify: fewer target rows than sequences need");
  bool pb = target->dtype == RL_BF16, qb = pb;
  if (draft) {
    st = side_of(draft, V, q_per_seq, &a.q);
    if (st != RL_OK) return st;
    if (!draft->first_row && static_cast<int64_t>(B) * q_per_seq > draft->rows)
      return set_error(RL_ERR_SHAPE, "rl_specdec_verify: fewer draft rows than sequences need");
    qb = draft->dtype == RL_BF16;
  }
  a.has_q = draft != nullptr;
  a.V = V;
  VdGuard g(h->device);
  if (!g.ok) return set_error(RL_ERR_CUDA, "rl_specdec_verify: cudaSetDevice failed");
  const int C = 1;
  using bf = __nv_bfloat16;
  const cudaError_t e = pb ? (qb ? launch<bf, bf>(a, B, C, stream) : launch<bf, float>(a, B, C, stream))
                           : (qb ? launch<float, bf>(a, B, C, stream) : launch<float, float>(a, B, C, stream));
  if (e != cudaSuccess) return set_error(RL_ERR_CUDA, cudaGetErrorString(e));
  return RL_OK;
}

}  // namespace
}  // namespace rl

extern "C" {
#pragma GCC visibility push(default)

rl_status rl_specdec_verify_draft(rl_sampler* h, int B, int V, int max_draft, const rl_dist_rows* target,
                                  const rl_dist_rows* draft, const int32_t* drafts, const int32_t* n_draft,
                                  const float* accept_u, const float* draw_u, int32_t* out_accepted, int32_t* out_tok,
                                  float* out_prob, int32_t* row_status, void* stream) {
  rl::clear_error();
  if (!h) return rl::set_error(RL_ERR_INVALID_ARG, "rl_specdec_verify_draft: handle is NULL");
  if (B < 0 || V <= 0 || max_draft < 0)
    return rl::set_error(RL_ERR_INVALID_ARG, "rl_specdec_verify_draft: bad B, V or max_draft");
  if (max_draft + 1 > RL_VERIFY_MAX_NODES || V > (1 << 30) || B > (1 << 24))
    return rl::set_error(RL_ERR_SHAPE, "rl_specdec_verify_draft: more than 255 drafts, 2^30 ids or 2^24 sequences");
  if (B == 0) return RL_OK;
  if (!target || !n_draft || !draw_u || !out_accepted || !out_tok || (max_draft > 0 && (!drafts || !accept_u)))
    return rl::set_error(RL_ERR_INVALID_ARG, "rl_specdec_verify_draft: a required pointer is NULL");
  rl::VdArgs a = {};
  a.N = max_draft + 1;
  a.tokens = drafts;
  a.accept_u = accept_u;
  a.tok_stride = max_draft;
  a.tok_off = 1;
  a.count = n_draft;
  a.count_add = 1;
  a.draw_u = draw_u;
  a.out_accepted = out_accepted;
  a.out_tok = out_tok;
  a.out_prob = out_prob;
  a.row_status = row_status;
  return rl::verify(h, B, V, a, target, draft, max_draft, static_cast<cudaStream_t>(stream));
}

rl_status rl_specdec_verify_tree(rl_sampler* h, int B, int V, int max_node, const rl_dist_rows* target,
                                 const rl_dist_rows* draft, const int32_t* tokens, const int32_t* parent,
                                 const int32_t* n_node, const float* accept_u, const float* draw_u,
                                 int32_t* out_accepted, int32_t* out_path, int32_t* out_tok, float* out_prob,
                                 int32_t* row_status, void* stream) {
  rl::clear_error();
  if (!h) return rl::set_error(RL_ERR_INVALID_ARG, "rl_specdec_verify_tree: handle is NULL");
  if (B < 0 || V <= 0 || max_node < 1)
    return rl::set_error(RL_ERR_INVALID_ARG, "rl_specdec_verify_tree: bad B, V or max_node");
  if (max_node > RL_VERIFY_MAX_NODES || V > (1 << 30) || B > (1 << 24))
    return rl::set_error(RL_ERR_SHAPE, "rl_specdec_verify_tree: more than 256 nodes, 2^30 ids or 2^24 sequences");
  if (B == 0) return RL_OK;
  if (!target || !tokens || !parent || !n_node || !accept_u || !draw_u || !out_accepted || !out_tok)
    return rl::set_error(RL_ERR_INVALID_ARG, "rl_specdec_verify_tree: a required pointer is NULL");
  rl::VdArgs a = {};
  a.N = max_node;
  a.tokens = tokens;
  a.accept_u = accept_u;
  a.tok_stride = max_node;
  a.tok_off = 0;
  a.parent = parent;
  a.count = n_node;
  a.count_add = 0;
  a.draw_u = draw_u;
  a.out_accepted = out_accepted;
  a.out_path = out_path;
  a.out_tok = out_tok;
  a.out_prob = out_prob;
  a.row_status = row_status;
  return rl::verify(h, B, V, a, target, draft, max_node, static_cast<cudaStream_t>(stream));
}

#pragma GCC visibility pop
}  // extern "C"
