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
// first refusal are not needed (with a draft that is right 70% of the time
// that is half of the rows of a chain of four). Every warp of the cluster
// holds a contiguous part of the ids, and a lane keeps (max, sum of
// 2^((x - max) c)) of what it sees: one pass per row. The parts' sums are
// joined through distributed shared memory and give Z, the accept tests, and
// later the part in which the drawn token lies: only that part is looked at
// again. A refusal with a draft row costs a second pass over the two rows
// (from L2) for the sums of w.
//
// What bounds it is the dependent steps of the walk: loads of a pass, exchange,
// join and accept test follow one another (for 512 ids a warp about 2400, 1000,
// 2300 and 650 cycles), and the longest walk of a batch ends the call. While the
// cluster joins its sums and decides, the rows of the node's first child are
// fetched into L2; a pass then runs on L2, a warp's next chunk loaded as soon as
// the registers of the last are free. 64 chains of 4 x 128256 f32 take 74 us, of
// which HBM needs 27 for the rows that are looked at; one chain of 3 x 32000 12.6.
//
// Precision. A weight is 2^(x c - F): one FMA and ex2.approx, a relative error of
// 2^-22 and the exponent's rounding (2^-24 of it); c = log2(e) / T in single
// precision tilts a row by at most 2^-24 |t| at the exponent t. A lane's F is the
// product max c of the first logits it sees, so that what weighs most has a short
// exponent, and is moved only where a later logit lies 64 binades above: any F
// does, as long as the sums are joined with it. Sums are doubles. The rows' sums,
// and with them the accept tests, the factor of a residual and the probabilities
// that are put out, are within about 1e-6 of 64 bits (1.4e-6 the worst of 20,000
// sequences). A draw is decided on sums of its own: log2(e) / T there is two floats,
// and ids with a 256th of the row or more are weighed in doubles and kept out of
// the sums in floats. What is left is the light ids' ex2, at most 2^-24 of the
// whole, 2e-9 (alike ids) to 5e-9 (one with half of the row) on the average.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <climits>

#include "common.cuh"
#include "internal.h"

namespace rl {
namespace {

constexpr int kVT = 256;
constexpr int kVW = kVT / 32;
constexpr int kChunk = 512;  // ids a warp loads at once
constexpr float kHigh = 18446744073709551616.0f;  // 2^64
constexpr int kMaxCluster = 8;
constexpr int kParts = kMaxCluster * kVW;  // parts of a row, at most
constexpr int kPerLane = kParts / 32;

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
  int part;                // ids of a warp's part (whole chunks)
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

// log2(e) / T.
__device__ __forceinline__ float scale_of(float T) {
  if (T > 1e-30f && T < 1e30f) {  // a quotient and its remainder: nearest but for 2^-30
    constexpr float hi = 1.44269504f, lo = static_cast<float>(1.4426950408889634074 - static_cast<double>(hi));
    const float y = __frcp_rn(T), q = __fmul_rn(hi, y);
    return __fmaf_rn(__fadd_rn(__fmaf_rn(-q, T, hi), lo), y, q);
  }
  return static_cast<float>(fmin(fmax(1.4426950408889634074 / static_cast<double>(T), 1e-30), 3e38));
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max16(const float (&x)[4][4]) {
  float t[5];
#pragma unroll
  for (int k = 0; k < 5; ++k) t[k] = max_nan(x[(3 * k) >> 2][(3 * k) & 3], x[(3 * k + 1) >> 2][(3 * k + 1) & 3], x[(3 * k + 2) >> 2][(3 * k + 2) & 3]);
  return max_nan(max_nan(t[0], t[1], t[2]), max_nan(t[3], t[4], x[3][3]));
}
__device__ __forceinline__ float ex2(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}
// Where a logit m lies in the exponent's domain: F = m c. Far from 0 the product's
// rounding counts in binades (and it can leave the range of floats): such frames
// are marked by NaN, and weights are taken from the difference x - m. From 2^16 on,
// where a row's tilt (Side) is still a small part of a binade.
__device__ __forceinline__ float frame(float m, float c) {
  const float F = m * c;
  return fabsf(F) < 65536.0f ? F : __int_as_float(0x7fc00000);
}
__device__ __forceinline__ bool is_near(float F) { return F == F; }
// The exponent of x relative to the frame of logit m.
__device__ __forceinline__ float exponent(float x, float m, float c, float F) {
  return is_near(F) ? __fmaf_rn(x, c, -F) : (x - m) * c;
}
// The weight of x; 0 for x = -inf, NaN for NaN. Of the first two the one without m
// is for frames that are known to be near, and NaN for others.
__device__ __forceinline__ float weight(float x, float c, float F) { return ex2(__fmaf_rn(x, c, -F)); }
__device__ __forceinline__ float weight(float x, float m, float c, float F) { return ex2(exponent(x, m, c, F)); }
// The same with the exponent in two floats.
__device__ __forceinline__ float weight_2(float x, float m, float c, float F) {
  if (!(x > RL_NEG_INF)) return 0.0f;
  if (!is_near(F)) return weight(x, m, c, F);
  const float p = __fmul_rn(x, c), e = __fmaf_rn(x, c, -p);
  if (!(fabsf(p) < RL_POS_INF)) return ex2(__fmaf_rn(x, c, -F));
  const float t = __fadd_rn(p, -F), v = __fadd_rn(t, -p);
  const float f = __fadd_rn(__fadd_rn(p, -__fadd_rn(t, -v)), __fadd_rn(-F, -v));  // p - F = t + f
  return ex2(t) * ex2(__fadd_rn(e, f));
}
// What a sum relative to frame F (of logit m) is multiplied by to be relative
// to frame G (of logit M >= m); more than 125 binades apart it drops out. What
// stays holds an id, m's, whose own weight in G's frame is not 0, so that a draw
// that falls in it finds an id.
__device__ __forceinline__ float rebase(float m, float F, float M, float G, float c) {
  if (m == M) return 1.0f;
  const float w = exponent(m, M, c, G);
  const float t = !is_near(F) ? w : is_near(G) ? F - G : -__fmaf_rn(M, c, -F);
  return fminf(t, w) >= -125.0f ? ex2(t) : 0.0f;
}

// A row of logits with what decides which of its ids are kept.
template <typename T>
struct Row {
  const T* x;
  const uint32_t* mask;  // null: no mask, or one that allows every id
  int cut;               // -1: none
  float xcut;
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }

// A logit x of id j, -inf where a cutoff leaves it out.
template <typename T>
__device__ __forceinline__ float above_cut(const Row<T>& r, int j, float x) {
  return r.cut >= 0 && (x < r.xcut || (x == r.xcut && j > r.cut)) ? RL_NEG_INF : x;
}

// Four consecutive logits.
__device__ __forceinline__ void unit(const float* s, float (&x)[4]) {
  const float4 v = __ldg(reinterpret_cast<const float4*>(s));
  x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}
__device__ __forceinline__ void unit(const __nv_bfloat16* s, float (&x)[4]) {
  const uint2 v = __ldg(reinterpret_cast<const uint2*>(s));
  x[0] = __uint_as_float(v.x << 16);
  x[1] = __uint_as_float(v.x & 0xffff0000u);
  x[2] = __uint_as_float(v.y << 16);
  x[3] = __uint_as_float(v.y & 0xffff0000u);
}
// The same of ids j0 .. j0 + 3 one by one; -inf from id `end` on.
template <typename T>
__device__ __forceinline__ void unit_guarded(const T* row, int j0, int end, float (&x)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) x[k] = j0 + k < end ? to_f(__ldg(row + j0 + k)) : RL_NEG_INF;
}

// The mask bits of ids j0 .. j0 + 3 (j0 a multiple of 4).
__device__ __forceinline__ uint32_t bits4(const uint32_t* mask, int j0, int end) {
  return j0 < end ? __ldg(mask + (j0 >> 5)) >> (j0 & 31) : 0u;
}
// Puts -inf in the places of the four that are not kept; a NaN that is not
// masked stays.
template <typename T>
__device__ __forceinline__ void keep4(const Row<T>& r, int j0, uint32_t bits, float (&x)[4]) {
  if (r.mask) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (!((bits >> k) & 1u)) x[k] = RL_NEG_INF;
  }
  if (r.cut >= 0) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (x[k] < r.xcut || (x[k] == r.xcut && j0 + k > r.cut)) x[k] = RL_NEG_INF;
  }
}
// The words of a chunk's mask, loaded with its logits.
template <bool Plain>
struct Bits {
  uint32_t w[4];
  template <typename T>
  __device__ __forceinline__ void load(const Row<T>& r, int c0, int end) {
    if (!r.mask) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = c0 + 128 * i + 4 * (static_cast<int>(threadIdx.x) & 31);
      w[i] = j < end ? __ldg(r.mask + (j >> 5)) : 0u;
    }
  }
};
template <>
struct Bits<true> {
  template <typename T>
  __device__ __forceinline__ void load(const Row<T>&, int, int) {}
};

struct __align__(16) Part {
  double s;  // sum of weights relative to m's frame (T <= 0: NaN marks a NaN)
  float m;   // a logit of the part, at most 64 binades below its largest (T <= 0: the largest)
  int id;    // T <= 0: lowest id at m
};

// What is read of a sequence's nodes at the start.
struct Node {
  int tok;
  float u;
  float lp, lq;        // the token's logits in its parent's rows; later its weights
  int cut[2];          // [side] this node's rows' last kept ids
  float xcut[2];
  int first;           // first child (INT_MAX: none)
  int16_t parent;      // -1: none
  uint8_t bit[2];      // the token's mask bits in its parent's rows
};

// What a draw is decided on: the frames and factors of w = max(p rho - q, 0), or
// of p alone. Ids of a 2^-kHeavy of their row and more, 256 at most, are weighed in
// doubles and left out of the sums in floats: most of the error of a running sum
// comes from them, and a flat row has none. Mean error of a running sum next to
// its borders, as a share of the whole, at 32,000 / 128,256 normal logits of
// deviation 3, and where one id has 0.3 to 0.6 of the row beside them:
//   kHeavy 7   2.4e-9 / 2.6e-9, 4.7e-9 / 5.0e-9
//          8   2.2e-9 / 2.4e-9, 4.4e-9 / 5.0e-9
//         10   2.1e-9 / 1.6e-9, 3.6e-9 / 4.4e-9   64 chains of 4 x 128256 2% slower
// (by a share of the row: ids within 3 binades of the frame took 131 us of 64
// chains at T = 5 where this takes 78).
constexpr int kHeavy = 8;
struct Scale {
  double cd, dc;
  float c, crz, lo;
};
struct Side {
  float c, lo, m, F;  // log2(e) / T = c + lo, lo > 0
  float heavy;        // logits from here on
  double cd, r;       // log2(e) / T, and how far m's exponent is from its frame
  double unit;        // what a weight is multiplied by to be as those of the row's sum
};
struct Resid {
  Side p, q;
  double rho;
  float rhi, rlo;
};
struct Ctl {
  Part part[2][2][kParts];  // [parity][side]: every CTA's warps write into every CTA
  double w[2][kParts];      // [parity] the parts' sums of w
  Resid rs;
  Scale scale[2];
  uint64_t bar[2][2];       // [parity][0 parts, 1 sums of w]: what is to come has come
  double scan[kVW];
  double rest;              // draw target inside the draw's part
  double Ps, Qs;            // sums of weights of both rows, relative to Pm, Qm
  double C, S, px;
  double summed;            // S as it was last summed (given drafts: less is taken off it since)
  float Pm, Qm;
  int Pid;
  int status;
  int k;                    // next child to try
  int next;                 // accepted child, or kNone, kSums, kRefresh, kRest
  int owner;                // part that holds the drawn token
  int at;                   // first id found by the draw
  int nchild, nremoved;
  int16_t child[RL_VERIFY_MAX_NODES];    // of the present node
  int16_t removed[RL_VERIFY_MAX_NODES];  // its refused given children
};
constexpr int kNone = -1, kSums = -2, kRefresh = -3, kRest = -4;

// Whether id j is one of the refused given tokens.
__device__ __forceinline__ bool is_removed(const Ctl& sh, const Node* nodes, int n, int j) {
  for (int k = 0; k < n; ++k)
    if (nodes[sh.removed[k]].tok == j) return true;
  return false;
}

// What a lane has seen of a row: a sum relative to F, the frame of logit m
// (T <= 0: the largest logit and its lowest id).
struct Seen {
  float m, F;
  double s;
  int id;
};
__device__ __forceinline__ Seen unseen() {
  return {RL_NEG_INF, 0.0f, 0.0, INT_MAX};
}

__device__ __forceinline__ void see_max(Seen& z, const float (&x)[4][4], int j0) {
  const float gm = max16(x);
  if (gm != gm) z.s = __longlong_as_double(0x7ff8000000000000LL);
  if (gm > z.m) {
    z.m = gm;
#pragma unroll
    for (int k = 15; k >= 0; --k)
      if (x[k >> 2][k & 3] == gm) z.id = j0 + 128 * (k >> 2) + (k & 3);
  }
}

__device__ __forceinline__ void see(Seen& z, const float (&x)[4][4], float c) {
  if (!(z.m > RL_NEG_INF)) {  // nothing seen yet
    z.m = max16(x);
    z.F = frame(z.m, c);
  }
  float e[4];
#pragma unroll
  for (int u = 0; u < 4; ++u)
    e[u] = (weight(x[u][0], c, z.F) + weight(x[u][1], c, z.F)) + (weight(x[u][2], c, z.F) + weight(x[u][3], c, z.F));
  float sum = (e[0] + e[1]) + (e[2] + e[3]);
  if (!(sum < kHigh)) {
    // a frame that is far too low, one that is not near 0, or a NaN
    const float gm = max16(x);
    if (gm != gm) z.s = __longlong_as_double(0x7ff8000000000000LL);
    if (gm > z.m) {
      if (z.m > RL_NEG_INF) z.s *= static_cast<double>(rebase(z.m, z.F, gm, frame(gm, c), c));
      z.m = gm;
      z.F = frame(gm, c);
    }
    sum = 0.0f;
    if (z.m > RL_NEG_INF) {
      if (is_near(z.F)) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
          sum += (weight(x[u][0], c, z.F) + weight(x[u][1], c, z.F)) + (weight(x[u][2], c, z.F) + weight(x[u][3], c, z.F));
      } else {
#pragma unroll
        for (int k = 0; k < 16; ++k) sum += weight(x[k >> 2][k & 3], z.m, c, z.F);
      }
    }
  }
  z.s += static_cast<double>(sum);
}

__device__ __forceinline__ float warp_fmax(float v) { return ord_key_inv(__reduce_max_sync(0xffffffffu, ord_key(v))); }

// Both sides' parts of a warp, from its lanes (an unseen side gives an empty part).
__device__ __forceinline__ void warp_parts(const Seen& a, float ca, const Seen& b, float cb, bool greedy, Part& pa, Part& pb) {
  pa.m = warp_fmax(a.m);
  pb.m = warp_fmax(b.m);
  pa.id = static_cast<int>(__reduce_min_sync(0xffffffffu, static_cast<unsigned>(a.m == pa.m ? a.id : INT_MAX)));
  pb.id = 0;
  const float fa = greedy ? 1.0f : a.m > RL_NEG_INF ? rebase(a.m, a.F, pa.m, frame(pa.m, ca), ca) : 0.0f;
  const float fb = b.m > RL_NEG_INF ? rebase(b.m, b.F, pb.m, frame(pb.m, cb), cb) : 0.0f;
  double sa = a.s == a.s ? a.s * static_cast<double>(fa) : a.s;
  double sb = b.s == b.s ? b.s * static_cast<double>(fb) : b.s;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double ta = __shfl_xor_sync(0xffffffffu, sa, o), tb = __shfl_xor_sync(0xffffffffu, sb, o);
    sa += ta;
    sb += tb;
  }
  pa.s = sa;
  pb.s = sb;
}

// Warp 0 joins the parts of both sides: their sums relative to the largest m.
__device__ __forceinline__ void join_parts(const Part* parts, int np, bool greedy, bool with_q, float cp, float cq, Part& P,
                                           Part& Q) {
  const int lane = threadIdx.x & 31;
  const int per = (np + 31) >> 5;
  Part a[kPerLane], b[kPerLane];
  float ma = RL_NEG_INF, mb = RL_NEG_INF;
#pragma unroll
  for (int k = 0; k < kPerLane; ++k) {
    if (k >= per) continue;
    const int i = lane * per + k;
    a[k].s = b[k].s = 0.0;
    a[k].m = b[k].m = RL_NEG_INF;
    a[k].id = INT_MAX;
    if (i < np) {
      a[k] = parts[i];
      if (with_q) b[k] = parts[kParts + i];
    }
    ma = fmaxf(ma, a[k].m);
    mb = fmaxf(mb, b[k].m);
  }
  P.m = warp_fmax(ma);
  Q.m = warp_fmax(mb);
  const float Ga = frame(P.m, cp), Gb = frame(Q.m, cq);
  double sa = 0.0, sb = 0.0;
  unsigned id = INT_MAX;
#pragma unroll
  for (int k = 0; k < kPerLane; ++k) {
    if (k >= per) continue;
    if (a[k].m == P.m) id = min(id, static_cast<unsigned>(a[k].id));
    const float fa = greedy ? 1.0f : a[k].m > RL_NEG_INF ? rebase(a[k].m, frame(a[k].m, cp), P.m, Ga, cp) : 0.0f;
    const float fb = b[k].m > RL_NEG_INF ? rebase(b[k].m, frame(b[k].m, cq), Q.m, Gb, cq) : 0.0f;
    sa += a[k].s == a[k].s ? a[k].s * static_cast<double>(fa) : a[k].s;
    sb += b[k].s == b[k].s ? b[k].s * static_cast<double>(fb) : b[k].s;
  }
  P.id = static_cast<int>(__reduce_min_sync(0xffffffffu, id));
  Q.id = 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double ta = __shfl_xor_sync(0xffffffffu, sa, o), tb = __shfl_xor_sync(0xffffffffu, sb, o);
    sa += ta;
    sb += tb;
  }
  P.s = sa;
  Q.s = sb;
}

// Loads the ids [c0, c0 + kChunk) into x: unit i of the lane holds ids c0 +
// 128 i + 4 lane ... A row that does not start on a unit's boundary is loaded id
// by id.
template <bool Plain, typename T>
__device__ __forceinline__ void chunk_load(const Row<T>& r, int c0, float (&x)[4][4]) {
  const T* at = r.x + c0 + 4 * (static_cast<int>(threadIdx.x) & 31);
  if (Plain || (reinterpret_cast<uintptr_t>(r.x) & (4 * sizeof(T) - 1)) == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) unit(at + 128 * i, x[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) x[i][k] = to_f(__ldg(at + 128 * i + k));
  }
}
// The same of the last ids of a row or of two, cut at `end`. Parts are whole
// chunks, so this is one warp's, and all others wait for it: all of its loads are
// in flight at once. A function with arrays of its own, which keeps its cases out
// of the other warps' loops.
template <bool Plain, typename T>
__device__ __forceinline__ void load_cut(const T* row, int j0, int end, float (&v)[4][4]) {
  const bool units = Plain || (reinterpret_cast<uintptr_t>(row) & (4 * sizeof(T) - 1)) == 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int j = j0 + 128 * i;
    v[i][0] = v[i][1] = v[i][2] = v[i][3] = RL_NEG_INF;
    if (units && j + 4 <= end) unit(row + j, v[i]);
  }
  if (!units || (end & 3)) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (!units || j0 + 128 * i + 4 > end) unit_guarded(row, j0 + 128 * i, end, v[i]);
  }
}
template <bool Plain, typename T>
__device__ __noinline__ void chunk_cut(const T* row, int c0, int end, float* x) {
  float v[4][4];
  load_cut<Plain>(row, c0 + 4 * (static_cast<int>(threadIdx.x) & 31), end, v);
#pragma unroll
  for (int k = 0; k < 16; ++k) x[k] = v[k >> 2][k & 3];
}
template <bool Plain, typename TP, typename TQ>
__device__ __noinline__ void chunk_cut(const TP* rp, const TQ* rq, int c0, int end, float* x, float* y) {
  float v[4][4], w[4][4];
  const int j0 = c0 + 4 * (static_cast<int>(threadIdx.x) & 31);
  load_cut<Plain>(rp, j0, end, v);
  load_cut<Plain>(rq, j0, end, w);
#pragma unroll
  for (int k = 0; k < 16; ++k) x[k] = v[k >> 2][k & 3];
#pragma unroll
  for (int k = 0; k < 16; ++k) y[k] = w[k >> 2][k & 3];
}
template <bool Plain, typename T>
__device__ __forceinline__ void chunk_keep(const Row<T>& r, int c0, const Bits<Plain>& m, float (&x)[4][4]) {
  if constexpr (!Plain) {
    if (!r.mask && r.cut < 0) return;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      keep4(r, c0 + 128 * i + 4 * (static_cast<int>(threadIdx.x) & 31), m.w[i] >> (4 * (threadIdx.x & 7)), x[i]);
  }
}

// Passes over this warp's part [j0, j1) of one row or of two: f(first id of the
// chunk, logits). The next chunk is loaded as soon as f is done with the last.
template <bool Plain, typename T, typename F>
__device__ __forceinline__ void pass(const Row<T>& r, int j0, int j1, F f) {
  const int whole = j1 - (j1 - j0) % kChunk;
  Bits<Plain> m;
  if (j0 < whole) {
    float x[4][4];
    m.load(r, j0, j1);
    chunk_load<Plain>(r, j0, x);
    for (int c0 = j0; c0 < whole; c0 += kChunk) {
      chunk_keep<Plain>(r, c0, m, x);
      f(c0, x);
      if (c0 + kChunk < whole) {
        m.load(r, c0 + kChunk, j1);
        chunk_load<Plain>(r, c0 + kChunk, x);
      }
    }
  }
  if (whole < j1) {
    float t[4][4];
    m.load(r, whole, j1);
    chunk_cut<Plain>(r.x, whole, j1, &t[0][0]);
    chunk_keep<Plain>(r, whole, m, t);
    f(whole, t);
  }
}
// f on the target's chunk, g on the draft's.
template <bool Plain, typename TP, typename TQ, typename F, typename G>
__device__ __forceinline__ void pass_two(const Row<TP>& rp, const Row<TQ>& rq, int j0, int j1, F f, G g) {
  const int whole = j1 - (j1 - j0) % kChunk;
  Bits<Plain> m, n;
  if (j0 < whole) {
    float x[4][4], y[4][4];
    m.load(rp, j0, j1);
    n.load(rq, j0, j1);
    chunk_load<Plain>(rp, j0, x);
    chunk_load<Plain>(rq, j0, y);
    for (int c0 = j0; c0 < whole; c0 += kChunk) {
      const bool more = c0 + kChunk < whole;
      chunk_keep<Plain>(rp, c0, m, x);
      f(c0, x);
      if (more) {
        m.load(rp, c0 + kChunk, j1);
        chunk_load<Plain>(rp, c0 + kChunk, x);
      }
      chunk_keep<Plain>(rq, c0, n, y);
      g(c0, y);
      if (more) {
        n.load(rq, c0 + kChunk, j1);
        chunk_load<Plain>(rq, c0 + kChunk, y);
      }
    }
  }
  if (whole < j1) {
    float t[4][4], u[4][4];
    m.load(rp, whole, j1);
    n.load(rq, whole, j1);
    chunk_cut<Plain>(rp.x, rq.x, whole, j1, &t[0][0], &u[0][0]);
    chunk_keep<Plain>(rp, whole, m, t);
    f(whole, t);
    chunk_keep<Plain>(rq, whole, n, u);
    g(whole, u);
  }
}
// f on both.
template <bool Plain, typename TP, typename TQ, typename F>
__device__ __forceinline__ void pass_both(const Row<TP>& rp, const Row<TQ>& rq, int j0, int j1, F f) {
  const int whole = j1 - (j1 - j0) % kChunk;
  Bits<Plain> m, n;
  if (j0 < whole) {
    float x[4][4], y[4][4];
    m.load(rp, j0, j1);
    n.load(rq, j0, j1);
    chunk_load<Plain>(rp, j0, x);
    chunk_load<Plain>(rq, j0, y);
    for (int c0 = j0; c0 < whole; c0 += kChunk) {
      chunk_keep<Plain>(rp, c0, m, x);
      chunk_keep<Plain>(rq, c0, n, y);
      f(x, y);
      if (c0 + kChunk < whole) {
        m.load(rp, c0 + kChunk, j1);
        n.load(rq, c0 + kChunk, j1);
        chunk_load<Plain>(rp, c0 + kChunk, x);
        chunk_load<Plain>(rq, c0 + kChunk, y);
      }
    }
  }
  if (whole < j1) {
    float t[4][4], u[4][4];
    m.load(rp, whole, j1);
    n.load(rq, whole, j1);
    chunk_cut<Plain>(rp.x, rq.x, whole, j1, &t[0][0], &u[0][0]);
    chunk_keep<Plain>(rp, whole, m, t);
    chunk_keep<Plain>(rq, whole, n, u);
    f(t, u);
  }
}

// Fetches ids [j0, j1) of a row into L2, a line a lane.
template <typename T>
__device__ __forceinline__ void fetch(const T* row, int j0, int j1) {
  if (j0 >= j1) return;
  const char* a = reinterpret_cast<const char*>(row + j0);
  const char* e = reinterpret_cast<const char*>(row + j1);
  for (a += 128 * (threadIdx.x & 31); a < e; a += 128 * 32) asm volatile("prefetch.global.L2 [%0];" ::"l"(a));
}

// Warp 0: the part that holds the draw's target u * total, and the target
// inside it (every CTA finds the same). The last part with any weight where
// rounding leaves no sum over the target; -1 where there is no weight.
__device__ __forceinline__ void find_owner(Ctl& sh, const double (&w)[kPerLane], int np, float u) {
  const int lane = threadIdx.x & 31;
  const int per = (np + 31) >> 5;
  double own = 0.0;
#pragma unroll
  for (int k = 0; k < kPerLane; ++k) own += w[k];
  double incl = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  const double total = __shfl_sync(0xffffffffu, incl, 31);
  const double t = static_cast<double>(u) * total;
  const unsigned hit = __ballot_sync(0xffffffffu, own > 0.0 && incl > t);
  const unsigned some = __ballot_sync(0xffffffffu, own > 0.0);
  const int pick = hit ? __ffs(hit) - 1 : 31 - __clz(some);
  if (lane == (pick < 0 ? 0 : pick)) {
    // inside the lane's parts, in the same manner
    double run = incl - own;
    int at = -1;
    double before = 0.0;
#pragma unroll
    for (int k = 0; k < kPerLane; ++k) {
      if (w[k] > 0.0 && (at < 0 || !(run > t))) {
        at = k;
        before = run;
      }
      run += w[k];
    }
    sh.owner = pick < 0 ? -1 : lane * per + at;
    sh.rest = t - before;
    sh.at = INT_MAX;
  }
}

// The passes are functions of their own: what the walk keeps stays out of their
// registers, and a warp's loads in flight are what a pass lives on.
template <bool Plain, typename T>
__device__ __noinline__ Seen see_row(Row<T> r, int j0, int j1, float c, bool greedy) {
  Seen z = unseen();
  const int lane = threadIdx.x & 31;
  if (greedy) pass<Plain>(r, j0, j1, [&](int c0, const float (&x)[4][4]) { see_max(z, x, c0 + 4 * lane); });
  else pass<Plain>(r, j0, j1, [&](int, const float (&x)[4][4]) { see(z, x, c); });
  return z;
}
struct Seen2 {
  Seen p, q;
};
template <bool Plain, typename TP, typename TQ>
__device__ __noinline__ Seen2 see_rows(Row<TP> rp, Row<TQ> rq, int j0, int j1, float cp, float cq) {
  Seen zp = unseen(), zq = unseen();
  pass_two<Plain>(rp, rq, j0, j1, [&](int, const float (&x)[4][4]) { see(zp, x, cp); },
                  [&](int, const float (&y)[4][4]) { see(zq, y, cq); });
  return {zp, zq};
}
// A side's log2(e) / T: in doubles, the float c that sums are made with, and as
// crz + lo, rounded towards 0 so that both products of a logit of -inf are -inf.
__device__ __forceinline__ void set_scale(Scale& k, float T, float c) {
  k.cd = fmin(fmax(1.4426950408889634074 / static_cast<double>(T), 1e-30), 3e38);
  k.dc = 0.69314718055994530942 * (static_cast<double>(c) - k.cd);
  k.c = c;
  k.crz = __double2float_rz(k.cd);
  k.lo = fmaxf(static_cast<float>(k.cd - static_cast<double>(k.crz)), 1.17549435e-38f);
}
__device__ __noinline__ double weight_d(float x, float m, double c, double r) {
  return exp2((static_cast<double>(x) - static_cast<double>(m)) * c + r);
}
__device__ __forceinline__ double weight_d(float x, const Side& f) { return weight_d(x, f.m, f.cd, f.r); }
// The weight of x, 2^(x c + x lo - F): c alone would tilt the row by 2^-24 of an exponent.
__device__ __forceinline__ float near_weight(float x, const Side& f) { return ex2(__fmaf_rn(x, f.lo, __fmaf_rn(x, f.c, -f.F))); }
__device__ __forceinline__ float weight(float x, const Side& f) {
  if (is_near(f.F)) return near_weight(x, f);
  const float t = x - f.m;
  return ex2(__fmaf_rn(t, f.lo, t * f.c));
}
// Of a row whose sum is relative to logit m's frame.
__device__ __forceinline__ Side side(const Scale& k, float m, double sum) {
  Side f;
  f.c = k.crz;
  f.lo = k.lo;
  f.m = m;
  f.F = frame(m, k.c);
  f.heavy = m + __fdividef(__log2f(static_cast<float>(sum)) - static_cast<float>(kHeavy), k.c);
  f.cd = k.cd;
  const double md = static_cast<double>(m);
  f.r = is_near(f.F) ? fma(md, k.cd, -static_cast<double>(f.F)) : 0.0;
  const double y = is_near(f.F) ? md * k.dc : 0.0;  // |y| < 2^-8
  f.unit = fma(fma(fma(y, 1.0 / 6.0, 0.5), y, 1.0), y, 1.0);
  return f;
}
__device__ __forceinline__ float resid_w(float ep, float eq, const Resid& f) {
  return fmaxf(__fmaf_rn(ep, f.rhi, __fmaf_rn(ep, f.rlo, -eq)), 0.0f);
}
// The weight of one id.
__device__ __forceinline__ double one_weight(float x, const Side& f) {
  return x >= f.heavy ? weight_d(x, f) : static_cast<double>(weight(x, f));
}
__device__ __forceinline__ double one_weight(float x, float y, const Resid& f) {
  if (x >= f.p.heavy || y >= f.q.heavy) return fmax(weight_d(x, f.p) * f.rho - weight_d(y, f.q), 0.0);
  return static_cast<double>(resid_w(weight(x, f.p), weight(y, f.q), f));
}
__device__ __forceinline__ float pick16(const float (&x)[4][4], int i) {
  float v = x[0][0];
#pragma unroll
  for (int k = 1; k < 16; ++k) v = i == k ? x[k >> 2][k & 3] : v;
  return v;
}
// A lane's sum of w over ids [j0, j1). Heavy ids are left out of the sums in
// floats: added there, what each addition rounds off would stay.
template <bool Plain, typename TP, typename TQ>
__device__ __noinline__ double sum_resid(Row<TP> rp, Row<TQ> rq, int j0, int j1, const Resid* of) {
  const Resid f = *of;
  double s = 0.0;
  pass_both<Plain>(rp, rq, j0, j1, [&](float (&x)[4][4], const float (&y)[4][4]) {
    if (max16(x) >= f.p.heavy || max16(y) >= f.q.heavy) {
      unsigned hv = 0;
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (x[k >> 2][k & 3] >= f.p.heavy || y[k >> 2][k & 3] >= f.q.heavy) hv |= 1u << k;
      for (unsigned h = hv; h; h &= h - 1) s += one_weight(pick16(x, __ffs(h) - 1), pick16(y, __ffs(h) - 1), f);
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (hv >> k & 1u) x[k >> 2][k & 3] = RL_NEG_INF;
    }
    float w = 0.0f;
    if (is_near(f.p.F) && is_near(f.q.F)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = resid_w(near_weight(x[i][k], f.p), near_weight(y[i][k], f.q), f);
        w += (v[0] + v[1]) + (v[2] + v[3]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k) w += resid_w(weight(x[k >> 2][k & 3], f.p), weight(y[k >> 2][k & 3], f.q), f);
    }
    s += static_cast<double>(w);
  });
  return s;
}
// A lane's sum of p over ids [j0, j1) without the refused given tokens.
template <bool Plain, typename T>
__device__ __noinline__ double sum_kept(Row<T> r, int j0, int j1, const Ctl* sh, const Node* nodes, int nrem) {
  const Side f = sh->rs.p;
  double s = 0.0;
  const int lane = threadIdx.x & 31;
  pass<Plain>(r, j0, j1, [&](int c0, float (&x)[4][4]) {
    for (int k = 0; k < nrem; ++k) {
      const int t = nodes[sh->removed[k]].tok - c0;  // its lane takes it out
      if (t >= 0 && t < kChunk && ((t >> 2) & 31) == lane) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (i == ((t >> 7) << 2 | (t & 3))) x[i >> 2][i & 3] = RL_NEG_INF;
      }
    }
    const auto sum = [&] {
      float w = 0.0f;
      if (is_near(f.F)) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w += (near_weight(x[i][0], f) + near_weight(x[i][1], f)) + (near_weight(x[i][2], f) + near_weight(x[i][3], f));
      } else {
#pragma unroll
        for (int k = 0; k < 16; ++k) w += weight(x[k >> 2][k & 3], f);
      }
      return w;
    };
    if (max16(x) >= f.heavy) {
      unsigned hv = 0;
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (x[k >> 2][k & 3] >= f.heavy) hv |= 1u << k;
      for (unsigned h = hv; h; h &= h - 1) s += weight_d(pick16(x, __ffs(h) - 1), f);
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (hv >> k & 1u) x[k >> 2][k & 3] = RL_NEG_INF;
    }
    s += static_cast<double>(sum());
  });
  return s;
}

template <typename T>
__device__ __forceinline__ Row<T> make_row(const VdSide& a, int64_t row, int cut, float xcut) {
  Row<T> r;
  r.x = static_cast<const T*>(a.logits) + row * a.ld;
  r.mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
  r.cut = cut;
  r.xcut = xcut;
  return r;
}

// One side's share of a node's entry: the token's logit (-inf outside the row)
// and mask bit in the parent's row,
template <typename T>
__device__ __forceinline__ void read_token(const VdSide& a, int64_t row0, int V, int parent, int tok, float& logit, uint8_t& bit) {
  logit = RL_NEG_INF;
  bit = 1;
  if (parent >= 0 && static_cast<unsigned>(tok) < static_cast<unsigned>(V)) {
    const int64_t row = row0 + parent;
    logit = to_f(static_cast<const T*>(a.logits)[row * a.ld + tok]);
    if (a.mask) bit = (a.mask[row * a.mask_stride + (tok >> 5)] >> (tok & 31)) & 1u;
  }
}
// and the node's own row's cutoff.
template <typename T>
__device__ __forceinline__ void read_cut(const VdSide& a, int64_t row, int V, int& cut, float& xcut) {
  cut = -1;
  xcut = 0.0f;
  if (a.cut) {
    const int c = a.cut[row * a.cut_stride];
    if (static_cast<unsigned>(c) < static_cast<unsigned>(V)) {
      cut = c;
      xcut = to_f(static_cast<const T*>(a.logits)[row * a.ld + c]);
    }
  }
}

// ---- exchanges: every warp of the cluster writes what it has into every CTA, each
// write counted by that CTA's barrier as it lands. (Plain remote stores behind a
// barrier of the cluster wait for each store's way back first, about 1200 cycles
// of the 1700 that such an exchange took.) ----
__device__ __forceinline__ uint32_t in_cta(const void* p, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void send(const Part* to, const Part& v, const uint64_t* bar, int rank) {
  const long long d = __double_as_longlong(v.s);
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(in_cta(to, rank)),
               "r"(static_cast<uint32_t>(d)), "r"(static_cast<uint32_t>(d >> 32)), "r"(__float_as_uint(v.m)), "r"(v.id), "r"(in_cta(bar, rank))
               : "memory");
}
__device__ __forceinline__ void send(const double* to, double v, const uint64_t* bar, int rank) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(in_cta(to, rank)),
               "l"(__double_as_longlong(v)), "r"(in_cta(bar, rank))
               : "memory");
}
// Warp 0 waits for `bytes` of them; bounded, and alike for its lanes.
__device__ __forceinline__ bool receive(uint64_t* bar, uint32_t parity, uint32_t bytes) {
  if ((threadIdx.x & 31) == 0) mbar_expect_tx(bar, bytes);
  const long long t0 = clock64();
  bool in = false;
  while (!in) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    in = done != 0;
    if (!in && clock64() - t0 > kWaitBudget) break;
  }
  return __all_sync(0xffffffffu, in) != 0;
}

// Whether a mask row has a bit (one without allows every id); block-wide.
__device__ __forceinline__ bool any_bit(const uint32_t* mask, int V) {
  const int words = (V + 31) >> 5;
  uint32_t any = 0;
  for (int w = threadIdx.x; w < words; w += kVT) {
    uint32_t m = mask[w];
    if (w == words - 1 && (V & 31)) m &= (1u << (V & 31)) - 1u;
    any |= m;
  }
  return __syncthreads_or(any != 0u) != 0;
}

// Plain: rows on 16-byte boundaries, without masks and cutoffs.
template <typename TP, typename TQ, bool Plain>
__global__ void __launch_bounds__(kVT, 2) verify_kernel(const __grid_constant__ VdArgs a) {
  extern __shared__ Node nodes[];  // a.N of them
  __shared__ Ctl sh;
  namespace cgx = cooperative_groups;
  const cgx::cluster_group cl = cgx::this_cluster();
  const int C = static_cast<int>(cl.num_blocks());
  const int rank = static_cast<int>(cl.block_rank());
  const int b = blockIdx.x / C;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int V = a.V, N = a.N;
  const bool tree = a.parent != nullptr;
  const int np = C * kVW, mypart = rank * kVW + warp;
  int32_t* out_tok = a.out_tok + static_cast<int64_t>(b) * N;
  int32_t* out_path = a.out_path ? a.out_path + static_cast<int64_t>(b) * N : nullptr;
  float* out_prob = a.out_prob ? a.out_prob + static_cast<int64_t>(b) * N : nullptr;

  // ---- a thread a node ----
  static_assert(RL_VERIFY_MAX_NODES <= kVT, "a thread a node");
  const bool has_entry = tid >= a.tok_off && tid < N;  // a chain's node 0 has none
  const int64_t entry = static_cast<int64_t>(b) * a.tok_stride + tid - a.tok_off;
  const int my_tok = has_entry ? a.tokens[entry] : -1;
  const float my_u = has_entry ? a.accept_u[entry] : 0.0f;
  int my_parent = tid - 1;
  if (tree) my_parent = has_entry ? a.parent[entry] : -1;
  if (my_parent < 0 || my_parent >= tid) my_parent = -1;
  // ---- the sequence's numbers, checked ----
  const int n = a.count[b] + a.count_add;
  const float Tp = a.p.T ? a.p.T[b] : 1.0f;
  const float Tq = a.has_q && a.q.T ? a.q.T[b] : 1.0f;
  const float du = a.draw_u[b];
  const bool greedy = Tp <= 0.0f;
  const bool drawn = a.has_q && !(Tq <= 0.0f) && !greedy;  // q comes from draft rows
  const int64_t p0 = a.p.first_row ? a.p.first_row[b] : static_cast<int64_t>(b) * a.p.per_seq;
  const int64_t q0 = a.has_q ? (a.q.first_row ? a.q.first_row[b] : static_cast<int64_t>(b) * a.q.per_seq) : 0;
  int status = RL_OK;
  if (n < 1 || n > N || p0 < 0 || p0 + n > a.p.rows) status = RL_ERR_INVALID_ARG;
  // the last node of a chain has no children, and no draft row
  else if (drawn && n > 1 && (q0 < 0 || q0 + n - (tree ? 0 : 1) > a.q.rows)) status = RL_ERR_INVALID_ARG;
  else if (!(fabsf(Tp) < RL_POS_INF) || !(fabsf(Tq) < RL_POS_INF)) status = RL_ERR_NONFINITE;
  const float cp = scale_of(greedy ? 1.0f : Tp), cq = scale_of(drawn ? Tq : 1.0f);

  // ---- this warp's part of the ids ----
  const int j0 = static_cast<int>(min(static_cast<int64_t>(mypart) * a.part, static_cast<int64_t>(V)));
  const int j1 = static_cast<int>(min(static_cast<int64_t>(j0) + a.part, static_cast<int64_t>(V)));
  const TP* const px0 = static_cast<const TP*>(a.p.logits) + p0 * a.p.ld;
  const TQ* const qx0 = drawn ? static_cast<const TQ*>(a.q.logits) + q0 * a.q.ld : nullptr;
  if (status == RL_OK) {  // the root's rows are on their way while the nodes are read
    fetch(px0, j0, j1);
    if (drawn && n > 1) fetch(qx0, j0, j1);
  }
  if (tid == 0) {
    for (int i = 0; i < 4; ++i) mbar_init(&sh.bar[i >> 1][i & 1], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid == kVT - 1) set_scale(sh.scale[0], greedy ? 1.0f : Tp, cp);
  if (tid == kVT - 33) set_scale(sh.scale[1], drawn ? Tq : 1.0f, cq);
  __syncwarp();
  cgx::this_cluster().barrier_arrive();
  if (tid < N) {
    Node& nd = nodes[tid];
    nd.tok = my_tok;
    nd.u = my_u;
    nd.parent = static_cast<int16_t>(my_parent);
    nd.first = !tree && tid + 1 < n ? tid + 1 : INT_MAX;
    if (!Plain && status == RL_OK && tid < n) {
      read_cut<TP>(a.p, p0 + tid, V, nd.cut[0], nd.xcut[0]);
      // (a root alone has no use for a draft row, and its place was not checked)
      if (drawn && n > 1 && (tree || tid + 1 < n)) read_cut<TQ>(a.q, q0 + tid, V, nd.cut[1], nd.xcut[1]);
    }
  }
  __syncthreads();
  if (tree && status == RL_OK) {
    if (tid < n && my_parent >= 0) atomicMin(&nodes[my_parent].first, tid);
    __syncthreads();
  }

  int node = 0, acc = 0, par = 0;
  int no_mask = 0;  // the node's rows whose mask has no bit: 1 the target's, 2 the draft's
  int token = -1;  // drawn token, in the CTA that finds it (thread 0)
  float tprob = 0.0f;
  bool found = false, started = false;
  uint32_t phase = 0;  // the barriers' parities, bit 2 par + kind
  while (status == RL_OK) {
    // ---- the node's rows and its children ----
    const Node& nd = nodes[node];
    Row<TP> rp = make_row<TP>(a.p, p0 + node, Plain ? -1 : nd.cut[0], Plain ? 0.0f : nd.xcut[0]);
    const int firstc = nd.first;
    const bool with_q = drawn && firstc != INT_MAX;
    Row<TQ> rq = {};
    if (with_q) rq = make_row<TQ>(a.q, q0 + node, Plain ? -1 : nd.cut[1], Plain ? 0.0f : nd.xcut[1]);
    if (Plain || (no_mask & 1)) rp.mask = nullptr;
    if (Plain || (no_mask & 2)) rq.mask = nullptr;
    // ---- this warp's sums of both rows, into every CTA of the cluster ----
    Seen zp, zq = unseen();
    if (with_q) {
      const Seen2 z = see_rows<Plain>(rp, rq, j0, j1, cp, cq);
      zp = z.p, zq = z.q;
    } else {
      zp = see_row<Plain>(rp, j0, j1, cp, greedy);
    }
    if (firstc != INT_MAX && (drawn || greedy)) {  // likely to be accepted
      fetch(px0 + firstc * a.p.ld, j0, j1);
      if (drawn && nodes[firstc].first != INT_MAX) fetch(qx0 + firstc * a.q.ld, j0, j1);
    }
    {
      Part pp, pq;
      warp_parts(zp, cp, zq, cq, greedy, pp, pq);
      // every CTA of the cluster has started: its shared memory may be written
      if (!started) cgx::this_cluster().barrier_wait();
      if (lane < C) {
        send(&sh.part[par][0][mypart], pp, &sh.bar[par][0], lane);
        if (with_q) send(&sh.part[par][1][mypart], pq, &sh.bar[par][0], lane);
      }
    }
    if (!started) {  // meanwhile: the nodes' logits
      if (tid < n) {
        Node& me = nodes[tid];
        float lp, lq = RL_NEG_INF;  // both loads in flight
        uint8_t bp, bq = 1;
        read_token<TP>(a.p, p0, V, my_parent, my_tok, lp, bp);
        if (drawn) read_token<TQ>(a.q, q0, V, my_parent, my_tok, lq, bq);
        me.lp = lp, me.lq = lq;
        me.bit[0] = bp, me.bit[1] = bq;
      }
      __syncthreads();
      started = true;
    }
    // ---- joined by warp 0 of every CTA ----
    if (warp == 0) {
      Part P, Q;
      const bool in = receive(&sh.bar[par][0], phase >> (2 * par) & 1u, static_cast<uint32_t>(np * sizeof(Part)) << (with_q ? 1 : 0));
      join_parts(sh.part[par][0], np, greedy, with_q, cp, cq, P, Q);
      if (!with_q) Q.s = 1.0, Q.m = 0.0f;
      const float Fp = frame(P.m, cp), Fq = frame(Q.m, cq);
      const bool good = in && P.s == P.s && fabsf(P.m) < RL_POS_INF && Q.s == Q.s && fabsf(Q.m) < RL_POS_INF;
      // the children: their weights
      int nchild = 0;
      for (int i0 = good ? firstc : INT_MAX; i0 < n; i0 += 32) {
        const int i = i0 + lane;
        const bool is = i < n && (tree ? nodes[i].parent == node : i == firstc);
        const unsigned k = __ballot_sync(0xffffffffu, is);
        if (is) {
          Node& c = nodes[i];
          sh.child[nchild + __popc(k & ((1u << lane) - 1u))] = static_cast<int16_t>(i);
          const float x = rp.mask && !c.bit[0] ? RL_NEG_INF : above_cut(rp, c.tok, c.lp);
          c.lp = weight_2(x, P.m, cp, Fp);
          if (with_q) {
            const float y = rq.mask && !c.bit[1] ? RL_NEG_INF : above_cut(rq, c.tok, c.lq);
            c.lq = weight_2(y, Q.m, cq, Fq);
          }
        }
        nchild += __popc(k);
        if (!tree) break;
      }
      if (lane == 0) {
        sh.status = good ? RL_OK : in ? RL_ERR_NONFINITE : RL_ERR_TIMEOUT;
        sh.Ps = P.s;
        sh.Qs = Q.s;
        sh.Pm = P.m;
        sh.Qm = Q.m;
        sh.Pid = P.id;
        sh.C = 0.0;
        sh.S = sh.summed = 1.0;
        sh.k = 0;
        sh.nchild = nchild;
        sh.nremoved = 0;
      }
      __syncwarp();
    }
    phase ^= 1u << (2 * par);
    par ^= 1;
    bool sums = false;  // sh.w holds the parts' sums of w = max(p - C q, 0)
    int next = kNone;
    while (true) {
      // ---- accept tests: thread 0 of every CTA, all alike; both sides of a
      // test are multiplied by the rows' sums ----
      if (tid == 0 && sh.status == RL_OK) {
        int k = sh.k, nx = kNone;
        double S = sh.S;
        for (; k < sh.nchild; ++k) {
          const int c = sh.child[k];
          if (greedy) {
            if (nodes[c].tok == sh.Pid) {
              nx = c;
              sh.px = sh.Ps = 1.0;
              break;
            }
            continue;
          }
          const double ep = nodes[c].lp;
          if (with_q) {
            const double eq = nodes[c].lq * sh.Ps;
            if (static_cast<double>(nodes[c].u) * S * eq < ep * sh.Qs - sh.C * eq) {
              nx = c;
              sh.px = ep;
              break;
            }
            sh.C += S;  // refused: the sums of the new w are wanted
            nx = kSums;
            ++k;
            break;
          }
          const bool gone = is_removed(sh, nodes, sh.nremoved, nodes[c].tok);
          if (!gone && static_cast<double>(nodes[c].u) * S * sh.Ps < ep) {
            nx = c;
            sh.px = ep;
            break;
          }
          if (!gone && ep > 0.0) {
            sh.removed[sh.nremoved++] = static_cast<int16_t>(c);
            S = fmax(S - ep / sh.Ps, 0.0);
            // with most of a sum taken off, what is left is its rounding: where
            // another child asks for it, it is summed again (1 / 4: an error of
            // 1e-6 becomes 4e-6 at most)
            if (S < 0.25 * sh.summed && k + 1 < sh.nchild) {
              nx = kRest;
              ++k;
              break;
            }
          }
        }
        if (nx == kNone && sh.nremoved > 0) nx = kRefresh;
        if (nx < 0 && !greedy) sh.rs.p = side(sh.scale[0], sh.Pm, sh.Ps);
        if (nx == kSums) {
          sh.rs.q = side(sh.scale[1], sh.Qm, sh.Qs);
          const double rho = sh.Qs * sh.rs.p.unit / (sh.C * sh.Ps * sh.rs.q.unit);
          sh.rs.rho = rho;
          sh.rs.rhi = static_cast<float>(rho);
          sh.rs.rlo = static_cast<float>(rho - static_cast<double>(sh.rs.rhi));
        }
        sh.S = S;
        sh.k = k;
        sh.next = nx;
      }
      __syncthreads();
      status = sh.status;
      next = sh.next;
      if (status != RL_OK || (next != kSums && next != kRest)) break;
      // ---- sums of w over the parts: max(p - C q, 0), or p without the refused
      // given tokens ----
      double s = next == kSums ? sum_resid<Plain>(rp, rq, j0, j1, &sh.rs) : sum_kept<Plain>(rp, j0, j1, &sh, nodes, sh.nremoved);
      s = warp_sum_d(s);
      if (lane < C) send(&sh.w[par][mypart], s, &sh.bar[par][1], lane);
      if (warp == 0) {
        const bool in = receive(&sh.bar[par][1], phase >> (2 * par + 1) & 1u, static_cast<uint32_t>(np * sizeof(double)));
        double t = 0.0;
        for (int i = lane; i < np; i += 32) t += sh.w[par][i];
        t = warp_sum_d(t);
        if (lane == 0) {
          sh.S = sh.summed = next == kSums ? t * sh.rs.q.unit * sh.C / sh.Qs : t * sh.rs.p.unit / sh.Ps;  // as a probability
          if (!in) sh.status = RL_ERR_TIMEOUT;
        }
        __syncwarp();
      }
      phase ^= 2u << (2 * par);
      par ^= 1;
      sums = next == kSums;
    }
    if (status != RL_OK) {
      // an empty row: once more without its mask, if that has no bit
      const bool ep = status == RL_ERR_NONFINITE && rp.mask && sh.Pm == RL_NEG_INF && !any_bit(rp.mask, V);
      const bool eq = status == RL_ERR_NONFINITE && with_q && rq.mask && sh.Qm == RL_NEG_INF && !any_bit(rq.mask, V);
      no_mask |= (ep ? 1 : 0) | (eq ? 2 : 0);
      if (!ep && !eq) break;
      status = RL_OK;
      __syncthreads();
      continue;
    }
    if (next >= 0) {
      if (rank == 0 && tid == 0) {
        out_tok[acc] = nodes[next].tok;
        if (out_path) out_path[acc] = next;
        if (out_prob) out_prob[acc] = static_cast<float>(sh.px / sh.Ps);
      }
      node = next;
      ++acc;
      no_mask = 0;
      __syncthreads();  // sh.child ... are rewritten for the next node
      continue;
    }
    // ---- no child is accepted: the last token ----
    if (greedy) {
      if (rank == 0 && tid == 0) {
        token = sh.Pid;
        tprob = 1.0f;
        found = true;
      }
      break;
    }
    const bool resid = sums && sh.S > 0.0;  // else all of w rounded away: from p
    int nrem = sh.nremoved;
    // The weights w of ids j .. j + 3: max(p rho - q, 0) in units of q's frame,
    // or p without the refused given tokens in units of p's.
    const auto w4 = [&](int j, int end, double (&w)[4]) {
      float x[4], y[4];
      unit_guarded(rp.x, j, end, x);
      if (resid) unit_guarded(rq.x, j, end, y);
      keep4(rp, j, rp.mask ? bits4(rp.mask, j, end) : 0u, x);
      if (resid) keep4(rq, j, rq.mask ? bits4(rq.mask, j, end) : 0u, y);
#pragma unroll 1
      for (int k = 0; k < 4; ++k) {
        const float a = k == 0 ? x[0] : k == 1 ? x[1] : k == 2 ? x[2] : x[3];
        double v;
        if (resid) v = one_weight(a, k == 0 ? y[0] : k == 1 ? y[1] : k == 2 ? y[2] : y[3], sh.rs);
        else v = nrem > 0 && is_removed(sh, nodes, nrem, j + k) ? 0.0 : one_weight(a, sh.rs.p);
        if (k == 0) w[0] = v;
        else if (k == 1) w[1] = v;
        else if (k == 2) w[2] = v;
        else w[3] = v;
      }
    };
    while (true) {
      if (!resid) {
        // the parts' sums once more, without refused given tokens (taking a weight
        // off a sum would leave its rounding) and with the heavy ids' exact weights
        double f = 0.0;
        if (j0 < j1) f = warp_sum_d(sum_kept<Plain>(rp, j0, j1, &sh, nodes, nrem));
        if (lane < C) send(&sh.w[par][mypart], f, &sh.bar[par][1], lane);
        if (warp == 0 && !receive(&sh.bar[par][1], phase >> (2 * par + 1) & 1u, static_cast<uint32_t>(np * sizeof(double))) && lane == 0)
          sh.status = RL_ERR_TIMEOUT;
        phase ^= 2u << (2 * par);
        par ^= 1;
      }
      // ---- which part holds the drawn token ----
      if (warp == 0) {
        const int per = (np + 31) >> 5;
        double wp[kPerLane];
#pragma unroll
        for (int k = 0; k < kPerLane; ++k) wp[k] = k < per && lane * per + k < np ? sh.w[par ^ 1][lane * per + k] : 0.0;
        find_owner(sh, wp, np, du);
      }
      __syncthreads();
      status = sh.status;
      if (status != RL_OK || sh.owner >= 0 || nrem == 0) break;
      nrem = 0;  // the refused tokens hold all of the row (uniforms of 1): from p
      __syncthreads();
    }
    if (status != RL_OK) break;
    const int owner = sh.owner;
    if (owner >= 0 && owner / kVW == rank) {  // (a row that passed the join has weight somewhere)
      // ---- the drawn token inside that part, by the whole CTA: down to 4 ids a
      // thread by the sums of the warps' shares ----
      int w0 = static_cast<int>(min(static_cast<int64_t>(owner) * a.part, static_cast<int64_t>(V)));
      int w1 = static_cast<int>(min(static_cast<int64_t>(w0) + a.part, static_cast<int64_t>(V)));
      double rest = sh.rest;
      while (w1 - w0 > 4 * kVT) {
        const int chunks = (w1 - w0 + kChunk - 1) / kChunk;
        const auto share = [&](int w) { return min(w0 + chunks * w / kVW * kChunk, w1); };
        const int s0 = share(warp), s1 = share(warp + 1);
        double s = 0.0;
        if (s0 < s1)
          s = warp_sum_d(resid ? sum_resid<Plain>(rp, rq, s0, s1, &sh.rs) : sum_kept<Plain>(rp, s0, s1, &sh, nodes, nrem));
        if (lane == 0) sh.scan[warp] = s;
        __syncthreads();
        int pick = 0;
        double run = 0.0, before = 0.0;
        for (int w = 0; w < kVW; ++w) {
          const double v = sh.scan[w];
          if (v > 0.0 && !(run > rest)) {
            pick = w;
            before = run;
          }
          run += v;
        }
        rest -= before;
        const int to = share(pick + 1);
        w0 = share(pick);
        w1 = to;
        __syncthreads();
      }
      const int a0 = w0 + 4 * tid;
      double w[4] = {0.0, 0.0, 0.0, 0.0};
      if (a0 < w1) w4(a0, w1, w);
      double s = 0.0;
      int last = -1;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        s += w[k];
        if (w[k] > 0.0) last = a0 + k;
      }
      double incl = s;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      if (lane == 31) sh.scan[warp] = incl;
      __syncthreads();
      double run = incl - s;
      for (int i = 0; i < warp; ++i) run += sh.scan[i];
      if (run + s > rest && s > 0.0) {
        bool hit = false;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          run += w[k];
          if (!hit && w[k] > 0.0 && run > rest) {
            atomicMin(&sh.at, a0 + k);
            hit = true;
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
        if (token >= 0) tprob = static_cast<float>(weight_2(to_f(rp.x[token]), sh.Pm, cp, frame(sh.Pm, cp)) / sh.Ps);
        found = true;
      }
    }
    break;
  }
  if (!started) cgx::this_cluster().barrier_wait();
  // behind a wait that ran out no CTA leaves while others may still write to it
  if (status == RL_ERR_TIMEOUT) {
    cgx::this_cluster().barrier_arrive();
    cgx::this_cluster().barrier_wait();
  }
  // ---- outputs ----
  if (found) {
    out_tok[acc] = token;
    if (out_prob) out_prob[acc] = tprob;
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

template <typename TP, typename TQ, bool Plain>
cudaError_t launch(const VdArgs& a, int B, int C, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.dynamicSmemBytes = static_cast<size_t>(a.N) * sizeof(Node);
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
  return cudaLaunchKernelEx(&cfg, verify_kernel<TP, TQ, Plain>, a);
}

template <typename TP, typename TQ>
cudaError_t launch(const VdArgs& a, int B, int C, bool plain, cudaStream_t stream) {
  return plain ? launch<TP, TQ, true>(a, B, C, stream) : launch<TP, TQ, false>(a, B, C, stream);
}

// Whether every row starts on a 16-byte boundary and keeps all of its ids.
bool is_plain(const rl_dist_rows* d) {
  return reinterpret_cast<uintptr_t>(d->logits) % 16 == 0 && (d->rows <= 1 || d->ld * (d->dtype == RL_F32 ? 4 : 2) % 16 == 0) &&
         !d->mask && !d->cut;
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

// CTAs of a sequence's cluster. A walk's steps follow one another and only its
// rows can be split: eight where they find room on the GPU at once (two CTAs an
// SM), four where there are sequences enough, and at least 2048 ids a CTA,
// below which the join costs more than it saves. us by graph replay at 2 /
// 4 / 8 CTAs: 64 x 4 x 128256 f32 99 / 74 / 82, 128 x 7 x 151936 bf16 193 / 121 /
// 126, 16 trees of 29 nodes x 128256 74 / 48 / 35, 24 masked chains of 5 x 32000
// 71 / 48 / 41, one chain of 3 x 32000 19.2 / 14.2 / 12.8.
int cluster_size(int B, int V) {
  int C = 1;
  while (C < kMaxCluster && (C < 4 || static_cast<int64_t>(B) * C * 2 <= 256) && V / (2 * C) >= 2048) C *= 2;
  return C;
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
  const int C = cluster_size(B, V);
  // parts of whole chunks, so that only the row's end is cut
  const int64_t even = (static_cast<int64_t>(V) + C * kVW - 1) / (C * kVW);
  a.part = static_cast<int>((even + kChunk - 1) / kChunk * kChunk);
  const bool plain = is_plain(target) && (!draft || is_plain(draft));
  using bf = __nv_bfloat16;
  const cudaError_t e = pb ? (qb ? launch<bf, bf>(a, B, C, plain, stream) : launch<bf, float>(a, B, C, plain, stream))
                           : (qb ? launch<float, bf>(a, B, C, plain, stream) : launch<float, float>(a, B, C, plain, stream));
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
