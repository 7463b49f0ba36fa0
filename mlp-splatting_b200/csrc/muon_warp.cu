// Newton-Schulz iteration of small matrices (at most 32 x 96: the layers of a primitive), a warp per tile of 16 or 32 rows.
//
// X lies in the warp's shared memory as two binary16 matrices, A and bA + cA^2 in its registers as fragments of m16n8 tiles (lane
// 4 g + t: rows g and g + 8, columns 2 t and 2 t + 1), in which form a symmetric matrix is at once an A and a B operand.  ldmatrix gives X
// as the A operand of X X^T, whose words are also its B operand, and, transposed, as the B operand of (bA + cA^2) X.  Of A and A^2 the
// 16 x 16 blocks on and below the diagonal are computed, the others are their transposes (movmatrix).  Several matrices of few rows
// share a tile (four 4 x 32 ones fill one of 16 rows): blocks of A off their diagonal are cleared, after which everything stays
// block-diagonal.
//
// What bounds it: the tensor cores by way of mma.sync (m16n8k16, 1,024 multiply-adds per SM and cycle on this GPU, 555 TFLOP/s measured; a
// tcgen05 tile of 128 rows would spend three quarters of its products on zeros) and instruction issue, about even.  With X in registers and
// every loop unrolled the code did not fit the instruction caches: 32 ns per 32 x 72 matrix; so the loops over columns are rolled.
// Gradient, momentum and weights are read and written once, in fragments (each lane group of four takes a whole 32-byte sector).
#include "muon.cuh"

namespace mlpsp {

__device__ __forceinline__ void ns_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ns_mma8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5}, {%6}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(b0));
}
__device__ __forceinline__ uint32_t ns_transpose(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// 16 rows by 8 N columns at the lane's address: r[2 n + h] = rows 8 h + g, columns 8 n + 2 t; TRANS: the transposes of these 8 x 8 blocks
template <int N, bool TRANS>
__device__ __forceinline__ void ns_ldmatrix(uint32_t (&r)[4], uint32_t addr) {
  if (N == 2) {
    if (TRANS) asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
    else asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  } else {
    if (TRANS) asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr) : "memory");
    else asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr) : "memory");
    r[2] = r[3] = 0u;
  }
}
template <int N>
__device__ __forceinline__ void ns_stmatrix(uint32_t addr, const uint32_t (&r)[4]) {
  if (N == 2) asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
  else asm volatile("stmatrix.sync.aligned.m8n8.x2.shared.b16 [%0], {%1, %2};" ::"r"(addr), "r"(r[0]), "r"(r[1]) : "memory");
}

// two FP32 operations in one instruction
__device__ __forceinline__ float2 ns_fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<unsigned long long&>(d)) : "l"(reinterpret_cast<const unsigned long long&>(a)),
      "l"(reinterpret_cast<const unsigned long long&>(b)), "l"(reinterpret_cast<const unsigned long long&>(c)));
  return d;
}
__device__ __forceinline__ float2 ns_mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<unsigned long long&>(d)) : "l"(reinterpret_cast<const unsigned long long&>(a)),
      "l"(reinterpret_cast<const unsigned long long&>(b)));
  return d;
}
__device__ __forceinline__ float2 ns_both(float x) { return make_float2(x, x); }
__device__ __forceinline__ void ns_split2(float2 x, uint32_t& hi, uint32_t& lo) {
  hi = pack_h2<false>(x.x, x.y);
  const float2 r = ns_fma2(ns_unpack<false>(hi), ns_both(-1.f), x);
  lo = pack_h2<false>(r.x, r.y);
}

// fragments of a symmetric [16 MB x 16 MB] matrix: f[mb][n][h] = rows 16 mb + 8 h + g, columns 8 n + 2 t and + 1
template <int MB> struct NsFrag { uint32_t hi[MB][2 * MB][2], lo[MB][2 * MB][2]; };

// blocks above the diagonal from those below
template <int MB>
__device__ __forceinline__ void ns_mirror(NsFrag<MB>& s) {
  if (MB == 2)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        s.hi[0][2 * MB - 2 + q][h] = ns_transpose(s.hi[MB - 1][h][q]);
        s.lo[0][2 * MB - 2 + q][h] = ns_transpose(s.lo[MB - 1][h][q]);
      }
}

// d += x x^T over 8 K columns; x.. as ns_ldmatrix<K> gives them; block (mb, n), n <= 2 mb + 1, is d[mb (mb + 1) + n].  The blocks
// advance together, since an MMA takes four times as long to answer as to issue; small products first, so that the tensor core's
// rounding of a sum towards zero meets fewer large ones.
template <int MB, int K>
__device__ __forceinline__ void ns_gram(const uint32_t (&hi)[MB][4], const uint32_t (&lo)[MB][4], float (&d)[MB * (MB + 1)][4]) {
#pragma unroll
  for (int part = 0; part < 3; ++part) {
    const auto& l = part == 1 ? lo : hi;
    const auto& r = part == 0 ? lo : hi;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int n = 0; n < 2 * mb + 2; ++n) {
        if (K == 2) ns_mma(d[mb * (mb + 1) + n], l[mb][0], l[mb][1], l[mb][2], l[mb][3], r[n >> 1][n & 1], r[n >> 1][2 + (n & 1)]);
        else ns_mma8(d[mb * (mb + 1) + n], l[mb][0], l[mb][1], r[n >> 1][n & 1]);
      }
  }
}

template <int MB, int NB> __host__ __device__ constexpr int ns_row_bytes() { return (NB | 1) * 16; }      // an odd number of 16-byte units: no bank conflicts
template <int MB, int NB> __host__ __device__ constexpr int ns_warp_smem() { return 2 * 16 * MB * ns_row_bytes<MB, NB>(); }

template <int MB, int NB, int CTAS>
__global__ void __launch_bounds__(128, CTAS) k_ns_warp(const NsArgs q, const int pack, const int64_t tiles) {
  constexpr int KH = MB == 1 ? 2 : 1;       // with one block of rows, rows h = 0 and 1 of a lane may belong to two matrices
  constexpr int CH = MB == 2 ? (NB % 3 == 0 ? 3 : 4) : (NB % 3 == 0 ? 6 > NB ? NB : NB % 6 == 0 ? 6 : 9 : 4);
  static_assert(NB % CH == 0, "whole chunks");
  constexpr int kRow = ns_row_bytes<MB, NB>(), kLo = 16 * MB * kRow;
  extern __shared__ __align__(128) char smem[];
  chain_wait();
  chain_release();
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  char* const mine = smem + (threadIdx.x >> 5) * ns_warp_smem<MB, NB>();
  const uint32_t xs = smem_u32(mine);
  // this lane's row of the 8 x 8 blocks that ldmatrix and stmatrix name: lanes 0-7 rows 0-7, 8-15 rows 8-15, 16-31 the same, 8 columns on
  const uint32_t xa = xs + (lane & 15) * kRow + (lane >> 4) * 16;
  // the matrix of the tile and its row, for this lane's rows; which columns of A belong to the same matrix
  int sub[KH], row[KH];
  uint32_t same = 0u;      // bit h * 4 + n * 2 + e
#pragma unroll
  for (int h = 0; h < KH; ++h) {
    const int r = h * 8 + g;
    sub[h] = MB == 1 ? (r < pack * q.small ? r / q.small : -1) : 0;
    row[h] = MB == 1 ? (sub[h] >= 0 ? r - sub[h] * q.small : 0) : r;
    if (MB == 1)
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) same |= (sub[h] == (n * 8 + 2 * t + e) / q.small ? 1u : 0u) << (h * 4 + n * 2 + e);
  }
  for (int64_t tile = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5); tile < tiles; tile += (int64_t)gridDim.x * 4) {
    // element of the first column of this lane's rows; rows of block mb and half h are `in`
    int64_t first[KH];
    bool on[KH];
#pragma unroll
    for (int h = 0; h < KH; ++h) {
      const int64_t k = tile * pack + sub[h];
      on[h] = sub[h] >= 0 && k < q.count && (!q.active || q.active[k]);
      first[h] = on[h] ? k * q.stride + (int64_t)row[h] * q.rs : 0;
    }
    if (!__any_sync(0xffffffffu, on[0] || on[KH - 1])) continue;
    auto in = [&](int mb, int h) { return on[h % KH] && (MB == 1 || mb * 16 + h * 8 + g < q.small); };
    auto base = [&](int mb, int h) { return MB == 1 ? first[h % KH] : first[0] + (int64_t)((mb * 16 + h * 8) * q.rs); };
    __syncwarp();
    float2 x[MB][NB][2];
    if (q.vec >= 2) {
      auto fetch = [&](auto tag, auto step) {
        constexpr int TYPE = decltype(tag)::value;
        constexpr bool STEP = decltype(step)::value;
        // a few columns of blocks at a time, so that their loads are under way together
#pragma unroll
        for (int c0 = 0; c0 < NB; c0 += CH) {
          NsVec<2> v[MB][CH][2], m[MB][CH][2];
#pragma unroll
          for (int u = 0; u < CH; ++u)
#pragma unroll
            for (int mb = 0; mb < MB; ++mb)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int col = (c0 + u) * 8 + 2 * t;
                v[mb][u][h] = m[mb][u][h] = NsVec<2>{{0.f, 0.f}};
                if (in(mb, h) && col < q.large) {
                  v[mb][u][h] = ns_load<2>(q.g, base(mb, h) + col, TYPE);
                  if (STEP) m[mb][u][h] = ns_load<2>(q.m, base(mb, h) + col, MLPSP_PRECISION_F32);
                }
              }
#pragma unroll
          for (int u = 0; u < CH; ++u)
#pragma unroll
            for (int mb = 0; mb < MB; ++mb)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int col = (c0 + u) * 8 + 2 * t;
                float y[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  y[e] = v[mb][u][h].v[e];
                  if (STEP) {
                    m[mb][u][h].v[e] = ns_new_momentum(q, y[e], m[mb][u][h].v[e]);
                    y[e] = ns_update(q, y[e], m[mb][u][h].v[e]);
                  }
                }
                x[mb][c0 + u][h] = make_float2(y[0], y[1]);
                if (STEP && in(mb, h) && col < q.large) ns_store<2>(q.m, base(mb, h) + col, MLPSP_PRECISION_F32, m[mb][u][h]);
              }
        }
      };
      if (q.m) {
        if (q.type == MLPSP_PRECISION_F32) fetch(NsTag<MLPSP_PRECISION_F32>{}, NsTag<1>{});
        else if (q.type == MLPSP_PRECISION_F16) fetch(NsTag<MLPSP_PRECISION_F16>{}, NsTag<1>{});
        else fetch(NsTag<MLPSP_PRECISION_BF16>{}, NsTag<1>{});
      } else {
        if (q.type == MLPSP_PRECISION_F32) fetch(NsTag<MLPSP_PRECISION_F32>{}, NsTag<0>{});
        else if (q.type == MLPSP_PRECISION_F16) fetch(NsTag<MLPSP_PRECISION_F16>{}, NsTag<0>{});
        else fetch(NsTag<MLPSP_PRECISION_BF16>{}, NsTag<0>{});
      }
    } else {
      // odd rows, transposed matrices: element by element, through this lane's own places in shared memory so that the loop stays rolled
      float2* const keep = reinterpret_cast<float2*>(mine) + lane;
#pragma unroll 1
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float y[2] = {0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int col = nb * 8 + 2 * t + e;
              if (!in(mb, h) || col >= q.large) continue;
              const int64_t at = base(mb, h) + (int64_t)col * q.cs;
              y[e] = ns_load<1>(q.g, at, q.type).v[0];
              if (q.m) {
                const float m = ns_new_momentum(q, y[e], q.m[at]);
                y[e] = ns_update(q, y[e], m);
                q.m[at] = m;
              }
            }
            keep[((nb * MB + mb) * 2 + h) * 32] = make_float2(y[0], y[1]);
          }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
          for (int h = 0; h < 2; ++h) x[mb][nb][h] = keep[((nb * MB + mb) * 2 + h) * 32];
      __syncwarp();
    }
    // Frobenius norms, per matrix of the tile; once more, scaled, where the squares leave the range of FP32
    float f[KH];
    NsStart start[KH];       // lost: an infinity or a NaN; the result is NaN, and the tile's other matrices must not see it
#pragma unroll
    for (int h = 0; h < KH; ++h) f[h] = 1.f;
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
      float2 s2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 v = ns_mul2(x[mb][nb][h], ns_both(f[h % KH]));
            s2[h] = ns_fma2(v, v, s2[h]);
          }
      float ss[2] = {s2[0].x + s2[0].y, s2[1].x + s2[1].y};
      if (pack == 1) {
        float s = ss[0] + ss[1];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        ss[0] = ss[1] = s;
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          ss[h] += __shfl_xor_sync(0xffffffffu, ss[h], 1);
          ss[h] += __shfl_xor_sync(0xffffffffu, ss[h], 2);
        }
        float s[2] = {0.f, 0.f};
        int of = 0, left = q.small;
#pragma unroll 1
        for (int r = 0; r < 16; ++r) {
          const float v = __shfl_sync(0xffffffffu, r < 8 ? ss[0] : ss[1], (r & 7) * 4);
          if (of == sub[0]) s[0] += v;
          if (of == sub[KH - 1]) s[1] += v;
          if (--left == 0) { ++of; left = q.small; }
        }
        ss[0] = s[0];
        ss[1] = s[1];
      }
      bool again = false;
#pragma unroll
      for (int h = 0; h < KH; ++h) {
        start[h] = ns_start(q.eps, ss[h], f[h]);
        f[h] = start[h].lost ? kNsShrink : ss[h] < kNsTinySquares ? kNsGrow : 1.f;
        again |= f[h] != 1.f;
      }
      if (!__any_sync(0xffffffffu, again)) break;
    }
    int k2[KH];
    bool lost[KH];
#pragma unroll
    for (int h = 0; h < KH; ++h) { k2[h] = start[h].k; lost[h] = start[h].lost; }
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int nb = 0; nb < NB; nb += 2) {
        constexpr int kTail = NB & 1;
        uint32_t hi[4] = {0u, 0u, 0u, 0u}, lo[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (nb + u < NB)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const NsStart& s = start[h % KH];
              float2 v = ns_mul2(ns_mul2(x[mb][(nb + u) % NB][h], ns_both(s.pre)), ns_both(s.inv));
              if (s.lost) v = make_float2(0.f, 0.f);
              ns_split2(v, hi[2 * u + h], lo[2 * u + h]);
            }
        const uint32_t at = xa + mb * 16 * kRow + nb * 16;
        if (kTail && nb + 1 == NB) { ns_stmatrix<1>(at, hi); ns_stmatrix<1>(at + kLo, lo); }
        else { ns_stmatrix<2>(at, hi); ns_stmatrix<2>(at + kLo, lo); }
      }
    __syncwarp();
#pragma unroll 1
    for (int it = 0; it < q.steps; ++it) {
      NsStep by[KH];
#pragma unroll
      for (int h = 0; h < KH; ++h) by[h] = ns_step(q, k2[h]);
      float d[MB * (MB + 1)][4];
      auto clear = [&] {
#pragma unroll
        for (int i = 0; i < MB * (MB + 1); ++i) d[i][0] = d[i][1] = d[i][2] = d[i][3] = 0.f;
      };
      // ---- A = X X^T
      clear();
      auto columns = [&](int nb, auto width) {
        constexpr int K = decltype(width)::value;
        uint32_t hi[MB][4], lo[MB][4];
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          ns_ldmatrix<K, false>(hi[mb], xa + mb * 16 * kRow + nb * 16);
          ns_ldmatrix<K, false>(lo[mb], xa + mb * 16 * kRow + nb * 16 + kLo);
        }
        ns_gram<MB, K>(hi, lo, d);
      };
#pragma unroll 1
      for (int nb = 0; nb + 1 < NB; nb += 2) columns(nb, NsTag<2>{});
      if (NB & 1) columns(NB - 1, NsTag<1>{});
      NsFrag<MB> A;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int n = 0; n < 2 * mb + 2; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float(&o)[4] = d[mb * (mb + 1) + n];
            float2 v = ns_mul2(make_float2(o[2 * h], o[2 * h + 1]), ns_both(by[h % KH].gram));
            if (MB == 1) {
              if (!(same >> (h * 4 + n * 2) & 1u)) v.x = 0.f;
              if (!(same >> (h * 4 + n * 2 + 1) & 1u)) v.y = 0.f;
            }
            ns_split2(v, A.hi[mb][n][h], A.lo[mb][n][h]);
          }
      ns_mirror<MB>(A);
      float diag[MB][2];
      // ---- P = b A + c A^2.  Its diagonal is kept apart and multiplies X in FP32 below: the rest is smaller, and with it what the tensor
      // core's rounding towards zero takes off (4e-6 of the result for 128 rows with the diagonal in, 2e-6 so)
      clear();
#pragma unroll
      for (int k = 0; k < MB; ++k) {
        uint32_t hi[MB][4], lo[MB][4];
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
          for (int i = 0; i < 4; ++i) { hi[mb][i] = A.hi[mb][2 * k + (i >> 1)][i & 1]; lo[mb][i] = A.lo[mb][2 * k + (i >> 1)][i & 1]; }
        ns_gram<MB, 2>(hi, lo, d);
      }
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int n = 0; n < 2 * mb + 2; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float(&o)[4] = d[mb * (mb + 1) + n];
            const NsStep& s = by[h % KH];
            float2 v = ns_mul2(make_float2(o[2 * h], o[2 * h + 1]), ns_both(s.c));
            v = ns_fma2(ns_unpack<false>(A.lo[mb][n][h]), ns_both(s.b), v);
            v = ns_fma2(ns_unpack<false>(A.hi[mb][n][h]), ns_both(s.b), v);
            if (n == 2 * mb + h) {       // the block on the diagonal: lane 4 g + g / 2 has row g's element
              diag[mb][h] = g & 1 ? v.y : v.x;
              if (2 * t == g) v.x = 0.f;
              if (2 * t + 1 == g) v.y = 0.f;
            }
            ns_split2(v, A.hi[mb][n][h], A.lo[mb][n][h]);
          }
      ns_mirror<MB>(A);
      float2 own[MB][2];       // a + P(r, r) of this lane's rows
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int h = 0; h < 2; ++h) own[mb][h] = ns_both(by[h % KH].a + __shfl_sync(0xffffffffu, diag[mb][h], 4 * g + (g >> 1)));
      // ---- X <- a X + P X, two blocks of eight columns at a time
      const bool last = it + 1 == q.steps;
      auto advance = [&](int nb, auto width) {
        constexpr int N = decltype(width)::value;
        uint32_t bh[MB][4], bl[MB][4];
        float e[MB][N][4];
#pragma unroll
        for (int k = 0; k < MB; ++k) {
          ns_ldmatrix<N, true>(bh[k], xa + k * 16 * kRow + nb * 16);
          ns_ldmatrix<N, true>(bl[k], xa + k * 16 * kRow + nb * 16 + kLo);
#pragma unroll
          for (int n = 0; n < N; ++n) e[k][n][0] = e[k][n][1] = e[k][n][2] = e[k][n][3] = 0.f;
        }
#pragma unroll
        for (int part = 0; part < 3; ++part) {
          const auto& l = part == 1 ? A.lo : A.hi;
          const auto& r = part == 0 ? bl : bh;
#pragma unroll
          for (int k = 0; k < MB; ++k)
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
              for (int mb = 0; mb < MB; ++mb)
                ns_mma(e[mb][n], l[mb][2 * k][0], l[mb][2 * k][1], l[mb][2 * k + 1][0], l[mb][2 * k + 1][1], r[k][2 * n], r[k][2 * n + 1]);
        }
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          const uint32_t at = xa + mb * 16 * kRow + nb * 16;
          uint32_t hi[4], lo[4];
          ns_ldmatrix<N, false>(hi, at);
          ns_ldmatrix<N, false>(lo, at + kLo);
          float2 v[N][2];
#pragma unroll
          for (int n = 0; n < N; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              v[n][h] = ns_fma2(ns_unpack<false>(lo[2 * n + h]), own[mb][h], make_float2(e[mb][n][2 * h], e[mb][n][2 * h + 1]));
              v[n][h] = ns_fma2(ns_unpack<false>(hi[2 * n + h]), own[mb][h], v[n][h]);
              ns_split2(v[n][h], hi[2 * n + h], lo[2 * n + h]);
            }
          if (!last) {
            ns_stmatrix<N>(at, hi);
            ns_stmatrix<N>(at + kLo, lo);
            continue;
          }
          const float nan = __int_as_float(0x7fffffff);
#pragma unroll
          for (int n = 0; n < N; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int col = (nb + n) * 8 + 2 * t;
              if (!in(mb, h) || col >= q.large) continue;
              const float fin = ns_exp2i(-10 - k2[h % KH]);
              NsVec<2> y;
              y.v[0] = lost[h % KH] ? nan : v[n][h].x * fin;
              y.v[1] = lost[h % KH] ? nan : v[n][h].y * fin;
              if (q.vec >= 2) {
                const int64_t i = base(mb, h) + col;
                if (q.m) {
                  const NsVec<2> w = ns_load<2>(q.w, i, MLPSP_PRECISION_F32);
#pragma unroll
                  for (int c = 0; c < 2; ++c) y.v[c] = fmaf(-q.step, y.v[c], q.keep * w.v[c]);
                  ns_store<2>(q.w, i, MLPSP_PRECISION_F32, y);
                } else ns_store<2>(q.out, i, q.type, y);
              } else {
#pragma unroll
                for (int c = 0; c < 2; ++c)
                  if (col + c < q.large) {
                    const int64_t i = base(mb, h) + (int64_t)(col + c) * q.cs;
                    if (q.m) q.w[i] = fmaf(-q.step, y.v[c], q.keep * q.w[i]);
                    else ns_store<1>(q.out, i, q.type, NsVec<1>{{y.v[c]}});
                  }
              }
            }
        }
      };
#pragma unroll 1
      for (int nb = 0; nb + 1 < NB; nb += 2) advance(nb, NsTag<2>{});
      if (NB & 1) advance(NB - 1, NsTag<1>{});
      __syncwarp();
    }
  }
}

template <int MB, int NB, int CTAS>
static int ns_warp(const NsArgs& q, cudaStream_t st) {
  constexpr int smem = 4 * ns_warp_smem<MB, NB>();
  static_assert(CTAS * (smem + 1024) <= 227 * 1024, "resident CTAs");
  static DeviceOnce once;
  if (once.first()) MLPSP_CUDA_OK(cudaFuncSetAttribute(k_ns_warp<MB, NB, CTAS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  const int pack = std::max(1, 16 * MB / q.small);
  const int64_t tiles = (q.count + pack - 1) / pack;
  const unsigned grid = (unsigned)std::min<int64_t>((tiles + 3) / 4, (int64_t)sm_count() * CTAS);
  LaunchScope scope(kKMisc, 1, st);
  return cuda_check(launch_chained(k_ns_warp<MB, NB, CTAS>, dim3(grid), dim3(128), smem, st, q, pack, tiles), "orthogonalize");
}

int launch_ns_warp(const NsArgs& q, cudaStream_t st) {
  const int nb = (q.large + 7) / 8;
  if (q.small <= 16) return nb <= 4 ? ns_warp<1, 4, 6>(q, st) : nb <= 6 ? ns_warp<1, 6, 6>(q, st) : nb <= 9 ? ns_warp<1, 9, 5>(q, st) : ns_warp<1, 12, 5>(q, st);
  return nb <= 4 ? ns_warp<2, 4, 4>(q, st) : nb <= 6 ? ns_warp<2, 6, 4>(q, st) : nb <= 9 ? ns_warp<2, 9, 4>(q, st) : ns_warp<2, 12, 3>(q, st);
}

}  // namespace mlpsp
