// What the three Newton-Schulz kernels share: arguments, element access, the split of an FP32 value into two binary16 ones.
//
//   X0 = U / max(|U|_F, eps),   X <- a X + (b A + c A^2) X,  A = X X^T   (X the matrix or its transpose, whichever is wider)
//
// Arithmetic: the iteration multiplies a small singular value by up to a^steps (485 with the usual coefficients), so operands of
// eleven bits would put errors of tenths into an orthogonal matrix.  X, A and bA + cA^2 are held as binary16 pairs hi + lo
// (22 bits; X and A, whose entries become small, scaled by 2^10, so that their absolute error stays below 3e-11), every product is
// hi hi + hi lo + lo hi on the tensor cores with FP32 accumulation, and a X is added in FP32, with the diagonals of A, A^2 and P.  On
// Gaussian matrices the result is then nearer to 64-bit arithmetic than an iteration in plain FP32: 8.5e-7 and 1.2e-6 (32 x 72), 8.0e-7 and
// 1.2e-6 (64 x 72), 6.6e-7 and 2.0e-6 (128 x 1152).
#pragma once
#include <type_traits>
#include "frame.cuh"
#include "tc.cuh"

namespace mlpsp {

constexpr float kNsScale = 1024.f;

struct NsArgs {
  const void* g;             // the matrices, or their gradients in a step
  float* m;                  // momentum, or null: orthogonalise g into out
  float* w;                  // weights of a step
  void* out;                 // result, in g's type
  const uint8_t* active;     // [count], or null
  volatile int32_t* gave_up; // page-locked host word that a wait which gives up sets (the cluster kernel), or null
  int32_t withhold;          // this product of the first CTA is not answered (mlpsp_test_withhold_answer), or 0
  int64_t count, stride;     // matrices, elements of each
  int32_t type;              // element type of g and out (MLPSP_PRECISION_*)
  int32_t small, large;      // X is small x large
  int32_t rs, cs;            // X(i, j) lies at i * rs + j * cs
  int32_t steps, nesterov;
  int32_t follows;           // behind another launch of the same step, with which it shares nothing it writes
  int32_t near, far;         // bits by which a step may multiply singular values within 1/2, within 1/16
  int32_t vec;               // elements of a row that may be moved at once: 1, 2 or 4 (large is a multiple, addresses are aligned)
  float a, b, c, eps;
  float momentum, rest;      // rest = 1 - momentum
  float keep, step;          // w <- keep * w - step * X
};

// values beyond 1e19 or far below 1e-13, whose squares FP32 cannot hold, enter the norm multiplied by one of these (exact)
constexpr float kNsShrink = 8.271806125530277e-25f, kNsGrow = 1.2089258196146292e24f;     // 2^-80, 2^80
constexpr float kNsTinySquares = 8.077935669463161e-28f;                                  // 2^-90

__device__ __forceinline__ float ns_exp2i(int k) { return __int_as_float((127 + k) << 23); }      // 2^k, -126 <= k <= 127

// how a matrix enters the iteration: X = (u * pre) * inv is 2^10 2^k X0
struct NsStart { float pre, inv; int k; bool lost; };
// ss: sum of the squares of u * f
__device__ __forceinline__ NsStart ns_start(float eps, float ss, float f) {
  NsStart s;
  s.lost = !(ss < __int_as_float(0x7f800000));
  const float root = sqrtf(ss);
  if (root >= eps * f) {
    s.pre = f;
    s.inv = kNsScale / root;
    s.k = 0;
  } else {
    const float rho = root * (f == 1.f ? 1.f : f < 1.f ? kNsGrow : kNsShrink) / eps;      // |X0| < 1
    s.k = rho > 0.f ? min(116, -ilogbf(rho) - 1) : 0;
    s.pre = ns_exp2i(s.k);
    s.inv = kNsScale / eps;
  }
  return s;
}
// the factors of one step for a matrix at 2^k, which then is at the new k: scaled A = gram * (product of the scaled X), P = b (scaled A)
// + c (scaled A)^2, scaled X <- a X + P X
struct NsStep { float gram, a, b, c; };
template <typename Q>
__device__ __forceinline__ NsStep ns_step(const Q& q, int& k) {
  NsStep s;
  s.gram = k > 50 ? 0.f : ns_exp2i(-10 - 2 * k);
  const int fall = min(k, k >= 4 ? q.far : q.near);
  const float r = ns_exp2i(-fall);
  s.a = q.a * r;
  s.b = q.b * (r / kNsScale);
  s.c = q.c * (r / (kNsScale * kNsScale));
  k -= fall;
  return s;
}

template <int V> using NsTag = std::integral_constant<int, V>;
template <int N> struct NsVec { float v[N]; };

template <bool BF16>
__device__ __forceinline__ float2 ns_unpack(uint32_t v) {
  return BF16 ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v)) : __half22float2(*reinterpret_cast<const __half2*>(&v));
}
// N neighbouring elements at element i, aligned to their size
template <int N>
__device__ __forceinline__ NsVec<N> ns_load(const void* p, int64_t i, int type) {
  NsVec<N> r;
  if (type == MLPSP_PRECISION_F32) {
    const float* f = static_cast<const float*>(p) + i;
    if (N == 4) { const float4 x = *reinterpret_cast<const float4*>(f); r.v[0] = x.x; r.v[1 % N] = x.y; r.v[2 % N] = x.z; r.v[3 % N] = x.w; }
    else if (N == 2) { const float2 x = *reinterpret_cast<const float2*>(f); r.v[0] = x.x; r.v[1 % N] = x.y; }
    else r.v[0] = *f;
  } else {
    const uint16_t* h = static_cast<const uint16_t*>(p) + i;
    uint32_t w[2] = {0u, 0u};
    if (N == 4) { const uint2 x = *reinterpret_cast<const uint2*>(h); w[0] = x.x; w[1] = x.y; }
    else if (N == 2) w[0] = *reinterpret_cast<const uint32_t*>(h);
    else w[0] = *h;
#pragma unroll
    for (int k = 0; k < N; k += 2) {
      const float2 f = type == MLPSP_PRECISION_F16 ? ns_unpack<false>(w[k / 2]) : ns_unpack<true>(w[k / 2]);
      r.v[k] = f.x;
      if (k + 1 < N) r.v[(k + 1) % N] = f.y;
    }
  }
  return r;
}
template <int N>
__device__ __forceinline__ void ns_store(void* p, int64_t i, int type, const NsVec<N>& r) {
  if (type == MLPSP_PRECISION_F32) {
    float* f = static_cast<float*>(p) + i;
    if (N == 4) *reinterpret_cast<float4*>(f) = make_float4(r.v[0], r.v[1 % N], r.v[2 % N], r.v[3 % N]);
    else if (N == 2) *reinterpret_cast<float2*>(f) = make_float2(r.v[0], r.v[1 % N]);
    else *f = r.v[0];
  } else {
    uint16_t* h = static_cast<uint16_t*>(p) + i;
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int k = 0; k < N; k += 2) {
      const float y = k + 1 < N ? r.v[(k + 1) % N] : 0.f;
      w[k / 2] = type == MLPSP_PRECISION_F16 ? pack_h2<false>(r.v[k], y) : pack_h2<true>(r.v[k], y);
    }
    if (N == 4) *reinterpret_cast<uint2*>(h) = make_uint2(w[0], w[1]);
    else if (N == 2) *reinterpret_cast<uint32_t*>(h) = w[0];
    else *h = (uint16_t)w[0];
  }
}
// m <- m + (1 - mu)(g - m)
__device__ __forceinline__ float ns_new_momentum(const NsArgs& q, float g, float m) { return fmaf(q.rest, g - m, m); }
// the update of a step: m, or g + mu (m - g) with the new m
__device__ __forceinline__ float ns_update(const NsArgs& q, float g, float m) { return q.nesterov ? fmaf(q.momentum, m - g, g) : m; }
__device__ __forceinline__ void ns_split(float x0, float x1, uint32_t& hi, uint32_t& lo) {
  hi = pack_h2<false>(x0, x1);
  const float2 f = ns_unpack<false>(hi);
  lo = pack_h2<false>(x0 - f.x, x1 - f.y);
}
__device__ __forceinline__ float2 ns_join(uint32_t hi, uint32_t lo) {
  const float2 h = ns_unpack<false>(hi), l = ns_unpack<false>(lo);
  return make_float2(h.x + l.x, h.y + l.y);
}

// The launches of one step touch different matrices, so each may start while the one before still runs, whose last tiles (or whose few, for
// single large matrices) leave most of the GPU idle.  What came before the step is done when any of them starts: the first waits for it
// before it lets the second be set up, and so on; and since a follower waits for its predecessor before it ends, the last one ends last.
__device__ __forceinline__ void ns_begin(const NsArgs& q) {
  if (!q.follows) chain_wait();
  else __threadfence();
  chain_release();
}
__device__ __forceinline__ void ns_end(const NsArgs& q) {
  if (q.follows) chain_wait();
}

// Which kernel: a warp for matrices of up to 32 rows (muon_warp.cu), two for up to 64 (muon_pair.cu), a CTA or a cluster for the rest
// (muon_tc.cu).  Up to kNsWarpFew or kNsPairFew columns the first two are as fast with a single matrix and much faster with many.  Beyond, a cluster is done sooner
// with few, though its 128 rows are mostly empty (one of 32 x 700 106 us in a warp, 70 in a cluster; of 64 x 300 79 and 62), and behind that
// with many while enough of a warp's or pair's X fit an SM's shared memory: 2,000 of 32 x 700 877 and 974, of 64 x 350 700 and 1,136, but
// of 64 x 400 1,522 and 1,035, 3,000 of 32 x 1,024 3,586 and 2,013.  Many: more than the clusters take at once (200 of 64 x 264 75 and 129).
constexpr int kNsWarpRows = 32, kNsPairRows = 64;
constexpr int kNsWarpFew = 512, kNsPairFew = 256;
constexpr int kNsWarpLong[2] = {1024, 800}, kNsPairLong = 384;       // warp: up to 16 rows, up to 32
// launch false: all that may fail before a launch, and no launch
int launch_ns_warp(const NsArgs& q, cudaStream_t st, bool launch);
int launch_ns_pair(const NsArgs& q, cudaStream_t st, bool launch);
int launch_ns_cluster(const NsArgs& q, cudaStream_t st, bool launch);

}  // namespace mlpsp
