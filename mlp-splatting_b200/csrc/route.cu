// Rows of pixels on their way to the primitives that the pixels' records name, and back.
//
// The records of pixel p are fan * p .. fan * (p + 1) - 1, or pixel_offsets[p] .. pixel_offsets[p + 1] - 1; slots[r] is the place
// of record r among the records grouped by primitive (mlpsp_route_records), *kept how many of these places belong to a
// primitive; a record at *kept or behind is dropped.
//   dispatch            out[slots[r], :] = x[pixel(r), :], rows of dropped records zero
//   combine             out[p, :]        = sum over the records r of p of w[r] y[slots[r], :]
//   combine gradients   dy[slots[r], :]  = w[r] dout[p, :],   dw[r] = <dout[p, :], y[slots[r], :]>
// The gradient of dispatch is combine with weights of one.  Every kernel is pixel-major: a pixel's own row is read (or written)
// once and the rows of its records are visited in their order, so a sum over records is taken in one order whatever the
// launch looks like, in FP32, and rounded once; no atomics.  Bound: memory, one visit of every record's row.
//
// Rows move in pieces of up to 16 bytes (the widest that the row length and all addresses are a multiple of).  dispatch and combine
// give a thread one piece of one pixel, or two where pieces are small: neighbouring threads take neighbouring pieces, so the lines of a
// row are whole whatever its length, and a short row does not idle lanes.  dw is a sum over lanes, whose number is a choice for speed.
// A pixel's records are one chain of rounds of four in dispatch and combine: made for lists of up to hundreds, as images have them; 100,000
// records of one pixel take 5 and 7 ms (their gradients, a record for itself, 0.2).
#include "frame.cuh"
#include <cuda_bf16.h>

namespace mlpsp {

constexpr int kRtThreads = 256;

// where the records of a pixel lie; offsets that descend or leave the records are cut to them
struct RouteView {
  const int64_t* __restrict__ pixel_offsets;
  const int32_t* __restrict__ slots;
  const int64_t* __restrict__ kept;
  int64_t pixels, records;
  int32_t fan;
};
__device__ __forceinline__ void rt_range(const RouteView& v, int64_t p, int64_t& b, int64_t& e) {
  if (v.pixel_offsets) {
    b = min(max(__ldg(v.pixel_offsets + p), (int64_t)0), v.records);
    e = min(max(__ldg(v.pixel_offsets + p + 1), b), v.records);
  } else {
    b = p * v.fan;
    e = b + v.fan;
  }
}
__device__ __forceinline__ uint32_t rt_kept(const RouteView& v) { return (uint32_t)min(max(__ldg(v.kept), (int64_t)0), v.records); }

template <int B> struct RtPiece;
template <> struct RtPiece<16> { using type = uint4; };
template <> struct RtPiece<8> { using type = uint2; };
template <> struct RtPiece<4> { using type = uint32_t; };
template <> struct RtPiece<2> { using type = uint16_t; };

__device__ __forceinline__ float rt_float(float x) { return x; }
__device__ __forceinline__ float rt_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float rt_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T rt_round(float x);
template <> __device__ __forceinline__ float rt_round<float>(float x) { return x; }
template <> __device__ __forceinline__ __half rt_round<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 rt_round<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// the pixel and the first piece of this thread, of K that lie cb apart: `ppb` pixels of `cb` threads each per block, blocks of pieces along y
template <int K>
__device__ __forceinline__ bool rt_place(int pieces, int cb, int ppb, int64_t pixels, int64_t& p, int& c) {
  const int local = threadIdx.x / cb;
  p = (int64_t)blockIdx.x * ppb + local;
  c = blockIdx.y * cb * K + (threadIdx.x - local * cb);
  return local < ppb && p < pixels && c < pieces;
}

template <int B, int K>
__global__ void __launch_bounds__(kRtThreads) k_dispatch(const typename RtPiece<B>::type* __restrict__ x, RouteView v, int pieces,
                                                         int cb, int ppb, typename RtPiece<B>::type* __restrict__ out) {
  chain_wait();
  chain_release();
  using V = typename RtPiece<B>::type;
  int64_t p, b, e;
  int c;
  if (!rt_place<K>(pieces, cb, ppb, v.pixels, p, c)) return;
  rt_range(v, p, b, e);
  if (b >= e) return;
  const uint32_t kept = rt_kept(v), all = (uint32_t)v.records;
  V row[K];
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (c + k * cb < pieces) row[k] = __ldg(x + (size_t)p * pieces + c + k * cb);
  const V zero = {};
  for (int64_t r = b; r < e; r += 4) {
    uint32_t s[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) s[u] = r + u < e ? (uint32_t)__ldg(v.slots + r + u) : all;
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (s[u] < all && c + k * cb < pieces) out[(size_t)s[u] * pieces + c + k * cb] = s[u] < kept ? row[k] : zero;
  }
}

// CTAS: at least so many CTAs per SM.  Six instead of the four that 60 registers leave make the compiler spill (40), which costs where y comes from the L2 and
// pays where it comes from memory in FP32 rows of at least 64 bytes, by the rows that are then on their way: 49,000 and 730,000 rows of 512 bytes
// (25 and 374 MB) 5.4 -> 8.2 and 93 -> 80 us, 1.4 M of 64 bytes (90 MB) 33 -> 30; of 48 (67 MB) 20 -> 25, 7.5 M of 16 45 -> 48.  The
// 16-bit types, with twice the sums, lose everywhere.
constexpr int64_t kRtFromMemory = 80ll << 20;
template <typename T, int B, int K, int CTAS>
__global__ void __launch_bounds__(kRtThreads, CTAS) k_combine(const typename RtPiece<B>::type* __restrict__ y,
                                                              const float* __restrict__ weights, RouteView v, int pieces, int cb,
                                                              int ppb, typename RtPiece<B>::type* __restrict__ out) {
  chain_wait();
  chain_release();
  using V = typename RtPiece<B>::type;
  constexpr int E = B / (int)sizeof(T);
  int64_t p, b, e;
  int c;
  if (!rt_place<K>(pieces, cb, ppb, v.pixels, p, c)) return;
  rt_range(v, p, b, e);
  const uint32_t kept = rt_kept(v);
  float acc[K][E];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < E; ++i) acc[k][i] = 0.f;
  for (int64_t r = b; r < e; r += 4) {
    uint32_t s[4];
    float w[4];
    V row[4][K];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      s[u] = r + u < e ? (uint32_t)__ldg(v.slots + r + u) : 0xffffffffu;
      w[u] = weights && r + u < e ? __ldg(weights + r + u) : 1.f;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (s[u] < kept && c + k * cb < pieces) row[u][k] = __ldg(y + (size_t)s[u] * pieces + c + k * cb);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (s[u] < kept && c + k * cb < pieces) {
          const T* f = reinterpret_cast<const T*>(&row[u][k]);
#pragma unroll
          for (int i = 0; i < E; ++i) acc[k][i] = fmaf(w[u], rt_float(f[i]), acc[k][i]);
        }
  }
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (c + k * cb < pieces) {
      V o;
      T* f = reinterpret_cast<T*>(&o);
#pragma unroll
      for (int i = 0; i < E; ++i) f[i] = rt_round<T>(acc[k][i]);
      out[(size_t)p * pieces + c + k * cb] = o;
    }
}

// Every record for itself: `lanes` (a power of two) neighbouring threads take U consecutive ones a time, whose rows are then on their way
// together.  A block has the records of `ppb` pixels, so slots, weights and dw are read and written in order; the pixel of the first record is
// found by binary search among the block's offsets, those of the others by steps from there.  A group has about as many lanes as rounds: what
// every lane does once a record (slot, weight, sum over the lanes) and idle lanes of the last round cost more than short runs of a row: 570,000
// rows of 256 bytes in four lanes 56 us, in eight 62, in sixteen 67, in two 68; 475,000 of 33 bf16 values in eight 54, in 32 112.  4.6 M records of 16-byte rows: 121 us with a
// thread per pixel (its dw words lie in 32 sectors), 66 so; 950,000 of 128 bytes 90 with a search for each, 73
// with one for four.
// U is four for rows of two to 64 pieces (combine and gradients of 950,000 rows of 128 bytes 107 us, by twos 127; of 475,000 of 66 bytes in
// 2-byte pieces 155 and 208), else two (76,000 of 16 bytes, too few for all SMs, 10 us, by fours 13; 16,000 of 4,096 43 and 47).
constexpr int kRtPixels = 256;
template <typename T, int B, int U>
__global__ void __launch_bounds__(kRtThreads) k_combine_grad(const typename RtPiece<B>::type* __restrict__ dout,
                                                             const typename RtPiece<B>::type* __restrict__ y,
                                                             const float* __restrict__ weights, RouteView v, int pieces, int lanes, int ppb,
                                                             typename RtPiece<B>::type* __restrict__ dy, float* __restrict__ dw) {
  chain_wait();
  chain_release();
  using V = typename RtPiece<B>::type;
  constexpr int E = B / (int)sizeof(T);
  __shared__ int s_first[kRtPixels + 1];
  const int64_t p0 = (int64_t)blockIdx.x * ppb;
  const int here = (int)min((int64_t)ppb, v.pixels - p0);
  int64_t first = p0 * v.fan, last = (p0 + here) * v.fan;
  if (v.pixel_offsets) {
    for (int i = threadIdx.x; i <= here; i += kRtThreads) s_first[i] = (int)min(max(__ldg(v.pixel_offsets + p0 + i), (int64_t)0), v.records);
    __syncthreads();
    first = s_first[0];
    last = s_first[here];
  }
  const uint32_t kept = rt_kept(v), all = (uint32_t)v.records;
  const int sub = threadIdx.x & (lanes - 1), groups = kRtThreads / lanes;
  const uint32_t group = lanes == 32 ? 0xffffffffu : ((1u << lanes) - 1u) << (threadIdx.x & 31 & ~(lanes - 1));
  for (int64_t r0 = first + (int64_t)(threadIdx.x / lanes) * U; r0 < last; r0 += (int64_t)groups * U) {
    uint32_t s[U];
    float w[U], dot[U];
    size_t pixel[U];
    int lo = 0;
    if (v.pixel_offsets) {         // the last of the block's pixels whose first record is not behind r0
      int hi = here;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_first[mid] <= r0) lo = mid; else hi = mid;
      }
    } else {
      lo = (int)(r0 - first) / v.fan;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + u;
      const bool valid = r < last;
      s[u] = valid ? (uint32_t)__ldg(v.slots + r) : 0xffffffffu;
      w[u] = valid && weights ? __ldg(weights + r) : 1.f;
      dot[u] = 0.f;
      if (u > 0 && valid) {
        if (v.pixel_offsets) while (lo + 1 < here && s_first[lo + 1] <= r) ++lo;
        else lo += (lo + 1) * (int64_t)v.fan <= r - first;
      }
      pixel[u] = (size_t)(p0 + lo);
    }
    for (int c = sub; c < pieces; c += lanes) {
      V g[U], row[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (s[u] < kept) {
          g[u] = __ldg(dout + pixel[u] * pieces + c);
          if (dw) row[u] = __ldg(y + (size_t)s[u] * pieces + c);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool live = s[u] < kept;
        const T* gf = reinterpret_cast<const T*>(&g[u]);
        if (dw && live) {
          const T* f = reinterpret_cast<const T*>(&row[u]);
#pragma unroll
          for (int i = 0; i < E; ++i) dot[u] = fmaf(rt_float(gf[i]), rt_float(f[i]), dot[u]);
        }
        if (dy && s[u] < all) {
          V o = {};
          T* of = reinterpret_cast<T*>(&o);
          if (live)
#pragma unroll
            for (int i = 0; i < E; ++i) of[i] = rt_round<T>(w[u] * rt_float(gf[i]));
          dy[(size_t)s[u] * pieces + c] = o;
        }
      }
    }
    if (dw) {
      for (int o = lanes >> 1; o > 0; o >>= 1)
#pragma unroll
        for (int u = 0; u < U; ++u) dot[u] += __shfl_xor_sync(group, dot[u], o);
      if (sub == 0)
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (r0 + u < last) dw[r0 + u] = dot[u];
    }
  }
}

// the widest piece that divides the row and all addresses
static int rt_piece(int64_t row_bytes, std::initializer_list<const void*> ptrs) {
  uintptr_t all = (uintptr_t)row_bytes;
  for (const void* q : ptrs) all |= reinterpret_cast<uintptr_t>(q);
  return all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2;
}

static int rt_check(const char* who, const RouteView& v, int64_t dim, int32_t dtype, std::initializer_list<const void*> rows,
                    std::initializer_list<const void*> floats) {
  MLPSP_REQUIRE(dtype == MLPSP_PRECISION_F32 || dtype == MLPSP_PRECISION_F16 || dtype == MLPSP_PRECISION_BF16, MLPSP_E_ARG,
                "%s: unknown element type %d", who, dtype);
  MLPSP_REQUIRE(v.pixels >= 0 && v.records >= 0 && v.fan >= 0 && dim >= 1, MLPSP_E_ARG, "%s: bad sizes", who);
  MLPSP_REQUIRE(v.pixels < (1ll << 31) && v.records < (1ll << 31) && dim <= MLPSP_ROUTE_MAX_DIM, MLPSP_E_LIMIT,
                "%s: more than 2^31-1 pixels or records, or rows longer than %d", who, MLPSP_ROUTE_MAX_DIM);
  MLPSP_REQUIRE(v.pixel_offsets || v.pixels * v.fan == v.records, MLPSP_E_ARG, "%s: the record count is not pixels x fan", who);
  MLPSP_REQUIRE(v.kept && (v.records == 0 || v.slots), MLPSP_E_ARG, "%s: null pointer", who);
  MLPSP_REQUIRE(aligned_to(dtype == MLPSP_PRECISION_F32 ? 4 : 2, rows) && aligned_to(4, floats) && aligned_to(4, {v.slots}) &&
                aligned_to(8, {v.pixel_offsets, v.kept}), MLPSP_E_ARG, "%s: a pointer is not aligned to its elements", who);
  return MLPSP_OK;
}

// whether so many threads fill the GPU; else each has one piece (2,850 rows of 33 bf16 values: gradients 3.4 us, with the rules for many 5.1)
static bool rt_fills(int64_t threads) { return threads >= (int64_t)sm_count() * 1024; }

struct RtShape { int pieces, cb, ppb; dim3 grid, block; };
static RtShape rt_shape(int64_t row_bytes, int piece, int k, int64_t pixels) {
  RtShape s;
  s.pieces = (int)(row_bytes / piece);
  s.cb = std::min((s.pieces + k - 1) / k, kRtThreads);
  s.ppb = kRtThreads / s.cb;
  s.grid = dim3((unsigned)((pixels + s.ppb - 1) / s.ppb), (unsigned)((s.pieces + s.cb * k - 1) / (s.cb * k)));
  s.block = dim3((unsigned)((s.ppb * s.cb + 31) / 32 * 32));
  return s;
}

template <int B>
static void dispatch_rows(const void* x, const RouteView& v, int64_t row_bytes, void* out, cudaStream_t st) {
  using V = typename RtPiece<B>::type;
  // Two pieces a thread where they are small and many, to share the slots: 190,000 rows of 33 FP32 values 25 -> 21 us, 38,000 of 513 bf16 ones
  // 26 -> 20, but 2 M of 7 FP32 24.6 -> 26, 2.8 M of 3 fp16 26 -> 39, 475,000 of 34 FP32 in 8-byte pieces 15 -> 18.
  const int k = B <= 4 && row_bytes / B >= 12 && rt_fills(v.pixels * (row_bytes / B) / 2) ? 2 : 1;
  const RtShape s = rt_shape(row_bytes, B, k, v.pixels);
  auto* kernel = k_dispatch<B, 1>;
  if constexpr (B <= 4)
    if (k == 2) kernel = k_dispatch<B, 2>;
  launch_chained(kernel, s.grid, s.block, 0, st, static_cast<const V*>(x), v, s.pieces, s.cb, s.ppb, static_cast<V*>(out));
}

template <typename T, int B>
static void combine_rows(const void* y, const float* weights, const RouteView& v, int64_t row_bytes, void* out, cudaStream_t st) {
  using V = typename RtPiece<B>::type;
  // Two pieces a thread where they are one or two values, to share slots and weights: 475,000 rows of 33 FP32 values 32 -> 24 us, 2.8 M of 13 bf16
  // 138 -> 95, 57,000 of 530 29 -> 24, but 2.8 M of 6 bf16 21 -> 23.5, 1.9 M of 12 fp16 (in pieces of four) 18 -> 22.
  constexpr bool few = B / (int)sizeof(T) <= 2;
  const int k = few && row_bytes / B >= 4 && rt_fills(v.pixels * (row_bytes / B) / 2) ? 2 : 1;
  const RtShape s = rt_shape(row_bytes, B, k, v.pixels);
  auto* kernel = k_combine<T, B, 1, 1>;
  if constexpr (few)
    if (k == 2) kernel = k_combine<T, B, 2, 1>;
  if constexpr (sizeof(T) == 4 && B == 16)
    if (row_bytes >= 64 && v.records * row_bytes >= kRtFromMemory) kernel = k_combine<T, B, 1, 6>;
  launch_chained(kernel, s.grid, s.block, 0, st, static_cast<const V*>(y), weights, v,
                 s.pieces, s.cb, s.ppb, static_cast<V*>(out));
}

template <typename T, int B>
static void combine_grad(const void* dout, const void* y, const float* weights, const RouteView& v, int64_t row_bytes, void* dy,
                         float* dw, cudaStream_t st) {
  using V = typename RtPiece<B>::type;
  const int pieces = (int)(row_bytes / B);
  const bool long_row = B == 16 && pieces >= 64;       // 1 KB and more: a warp (78,000 rows of 1 KB 52 us, in eight lanes 58)
  int lanes = 1;
  while (lanes < 32 && lanes < pieces && (lanes * lanes < pieces || long_row || !rt_fills(v.records * lanes))) lanes *= 2;
  const int ppb = (int)std::min<int64_t>(kRtPixels, std::max<int64_t>(1, v.pixels / (sm_count() * 8)));      // eight blocks per SM, if pixels last
  launch_chained(pieces >= 2 && pieces <= 64 ? k_combine_grad<T, B, 4> : k_combine_grad<T, B, 2>,
                 dim3((unsigned)((v.pixels + ppb - 1) / ppb)), dim3(kRtThreads), 0, st, static_cast<const V*>(dout), static_cast<const V*>(y),
                 weights, v, pieces, lanes, ppb, static_cast<V*>(dy), dw);
}

}  // namespace mlpsp

using namespace mlpsp;

#define MLPSP_BY_PIECE(T, call)             \
  switch (piece) {                          \
    case 16: call(T, 16); break;            \
    case 8: call(T, 8); break;              \
    case 4: call(T, 4); break;              \
    default: call(T, 2); break;             \
  }
#define MLPSP_BY_TYPE(call)                                                                                       \
  if (dtype == MLPSP_PRECISION_F32) {                                                                             \
    if (piece == 16) call(float, 16); else if (piece == 8) call(float, 8); else call(float, 4);                   \
  } else if (dtype == MLPSP_PRECISION_F16) { MLPSP_BY_PIECE(__half, call) } else { MLPSP_BY_PIECE(__nv_bfloat16, call) }

extern "C" int mlpsp_dispatch_rows(const void* x, int32_t dtype, int64_t dim, int64_t pixels, int32_t fan, const int64_t* pixel_offsets,
                                   const int32_t* slots, int64_t records, const int64_t* kept, void* out, void* stream) {
  const RouteView v{pixel_offsets, slots, kept, pixels, records, fan};
  const int rc = rt_check("mlpsp_dispatch_rows", v, dim, dtype, {x, out}, {});
  if (rc) return rc;
  if (pixels == 0 || records == 0) return MLPSP_OK;
  MLPSP_REQUIRE(x && out, MLPSP_E_ARG, "mlpsp_dispatch_rows: null pointer");
  cudaStream_t st = (cudaStream_t)stream;
  const int64_t row = dim * (dtype == MLPSP_PRECISION_F32 ? 4 : 2);
  LaunchScope scope(kKMisc, 1, st);
  switch (rt_piece(row, {x, out})) {
    case 16: dispatch_rows<16>(x, v, row, out, st); break;
    case 8: dispatch_rows<8>(x, v, row, out, st); break;
    case 4: dispatch_rows<4>(x, v, row, out, st); break;
    default: dispatch_rows<2>(x, v, row, out, st); break;
  }
  return cuda_check(cudaGetLastError(), "dispatch_rows");
}

extern "C" int mlpsp_combine_rows(const void* y, int32_t dtype, int64_t dim, const float* weights, int64_t pixels, int32_t fan,
                                  const int64_t* pixel_offsets, const int32_t* slots, int64_t records, const int64_t* kept, void* out,
                                  void* stream) {
  const RouteView v{pixel_offsets, slots, kept, pixels, records, fan};
  const int rc = rt_check("mlpsp_combine_rows", v, dim, dtype, {y, out}, {weights});
  if (rc) return rc;
  if (pixels == 0) return MLPSP_OK;
  MLPSP_REQUIRE(out && (y || records == 0), MLPSP_E_ARG, "mlpsp_combine_rows: null pointer");
  cudaStream_t st = (cudaStream_t)stream;
  const int64_t row = dim * (dtype == MLPSP_PRECISION_F32 ? 4 : 2);
  const int piece = rt_piece(row, {y, out});
  LaunchScope scope(kKMisc, 1, st);
#define MLPSP_CALL(T, B) combine_rows<T, B>(y, weights, v, row, out, st)
  MLPSP_BY_TYPE(MLPSP_CALL)
#undef MLPSP_CALL
  return cuda_check(cudaGetLastError(), "combine_rows");
}

extern "C" int mlpsp_combine_rows_gradients(const void* grad_out, const void* y, int32_t dtype, int64_t dim, const float* weights,
                                            int64_t pixels, int32_t fan, const int64_t* pixel_offsets, const int32_t* slots,
                                            int64_t records, const int64_t* kept, void* grad_y, float* grad_weights, void* stream) {
  const RouteView v{pixel_offsets, slots, kept, pixels, records, fan};
  const int rc = rt_check("mlpsp_combine_rows_gradients", v, dim, dtype, {grad_out, y, grad_y}, {weights, grad_weights});
  if (rc) return rc;
  if (pixels == 0 || records == 0) return MLPSP_OK;
  MLPSP_REQUIRE(grad_out && (grad_y || grad_weights) && (y || !grad_weights), MLPSP_E_ARG, "mlpsp_combine_rows_gradients: null pointer");
  cudaStream_t st = (cudaStream_t)stream;
  const int64_t row = dim * (dtype == MLPSP_PRECISION_F32 ? 4 : 2);
  const int piece = rt_piece(row, {grad_out, y, grad_y});
  LaunchScope scope(kKMisc, 1, st);
#define MLPSP_CALL(T, B) combine_grad<T, B>(grad_out, y, weights, v, row, grad_y, grad_weights, st)
  MLPSP_BY_TYPE(MLPSP_CALL)
#undef MLPSP_CALL
  return cuda_check(cudaGetLastError(), "combine_rows_gradients");
}
