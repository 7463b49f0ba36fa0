// Newton-Schulz iteration of small matrices (at most 32 x 96: the layers of a primitive), a warp per tile of 16 or 32 rows.
//
// The whole iteration stays in the warp's registers.  X lies there as the accumulator fragments of m16n8 tiles (lane 4 g + t:
// rows g and g + 8, columns 2 t and 2 t + 1), packed to binary16 pairs; in this form it is at once the A operand of X X^T and, read as
// columns, its B operand, so Gram matrices need no data movement.  A and A^2 are symmetric: of the 16 x 16 blocks only those on and
// below the diagonal are computed, the others are their transposes (movmatrix).  For (bA + cA^2) X the B operand is X itself, which
// takes one movmatrix per 8 x 8 block.  Several matrices of few rows share a tile (four 4 x 32 ones fill one of 16 rows): blocks of A
// off their diagonal are cleared, after which everything stays block-diagonal.
//
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

// fragments of a [16 MB x 8 NB] matrix: f[mb][nb][h] = rows 16 mb + 8 h + g, columns 8 nb + 2 t and + 1
template <int MB, int NB> struct NsFrag { uint32_t hi[MB][NB][2], lo[MB][NB][2]; };

// The blocks of x x^T on and below the diagonal: d[mb * (mb + 1) + n] = rows 16 mb.. times rows 8 n.., n <= 2 mb + 1.  All of them
// advance together, since an MMA takes four times as long to answer as to issue; the small products come first, so that the tensor
// core's rounding of a sum towards zero meets the large ones only.
template <int MB, int NB>
__device__ __forceinline__ void ns_gram(const NsFrag<MB, NB>& x, float (&d)[MB * (MB + 1)][4]) {
#pragma unroll
  for (int i = 0; i < MB * (MB + 1); ++i) d[i][0] = d[i][1] = d[i][2] = d[i][3] = 0.f;
#pragma unroll
  for (int part = 0; part < 3; ++part) {
    const auto& l = part == 1 ? x.lo : x.hi;
    const auto& r = part == 0 ? x.lo : x.hi;
#pragma unroll
    for (int k = 0; k < NB; k += 2)
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int n = 0; n < 2 * mb + 2; ++n) {
          float(&o)[4] = d[mb * (mb + 1) + n];
          if (k + 1 < NB) ns_mma(o, l[mb][k][0], l[mb][k][1], l[mb][(k + 1) % NB][0], l[mb][(k + 1) % NB][1], r[n >> 1][k][n & 1], r[n >> 1][(k + 1) % NB][n & 1]);
          else ns_mma8(o, l[mb][k][0], l[mb][k][1], r[n >> 1][k][n & 1]);
        }
  }
}
// blocks above the diagonal from those below
template <int MB>
__device__ __forceinline__ void ns_mirror(NsFrag<MB, 2 * MB>& s) {
  if (MB == 2)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        s.hi[0][2 * MB - 2 + q][h] = ns_transpose(s.hi[MB - 1][h][q]);
        s.lo[0][2 * MB - 2 + q][h] = ns_transpose(s.lo[MB - 1][h][q]);
      }
}

template <int MB, int NB, int CTAS>
__global__ void __launch_bounds__(128, CTAS) k_ns_warp(const NsArgs q, const int pack, const int64_t tiles) {
  constexpr int CH = NB % 3 == 0 ? 3 : 4;
  chain_wait();
  chain_release();
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t warps = (int64_t)gridDim.x * 4;
  // the matrix of the tile and its row, for this lane's rows; -1: no such row.  And which columns of A belong to the same matrix.
  int sub[MB][2], row[MB][2];
  uint32_t same = 0u;      // bit (mb * 2 + h) * 8 + n8 * 2 + e (packs of several matrices have MB = 1)
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = mb * 16 + h * 8 + g;
      const bool in = r < pack * q.small;
      sub[mb][h] = in ? r / q.small : -1;
      row[mb][h] = in ? r - sub[mb][h] * q.small : 0;
      if (MB == 1)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            same |= (sub[mb][h] == (n * 8 + 2 * t + e) / q.small ? 1u : 0u) << (h * 4 + n * 2 + e);
    }
  for (int64_t tile = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5); tile < tiles; tile += warps) {
    int64_t base[MB][2];     // element of the row's first column, -1: none
    bool any = false;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t k = tile * pack + sub[mb][h];
        const bool in = sub[mb][h] >= 0 && k < q.count && (!q.active || q.active[k]);
        base[mb][h] = in ? k * q.stride + (int64_t)row[mb][h] * q.rs : -1;
        any |= in;
      }
    if (!__any_sync(0xffffffffu, any)) continue;
    float x[MB][NB][2][2];
    if (q.vec >= 2) {
      // a few columns of tiles at a time, so that their loads are under way together
#pragma unroll
      for (int c0 = 0; c0 < NB; c0 += CH) {
        NsVec<2> v[MB][CH][2], m[MB][CH][2];
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
          for (int u = 0; u < CH; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int col = (c0 + u) * 8 + 2 * t;
              const bool in = base[mb][h] >= 0 && col < q.large;
              v[mb][u][h] = m[mb][u][h] = NsVec<2>{{0.f, 0.f}};
              if (in) {
                v[mb][u][h] = ns_load<2>(q.g, base[mb][h] + col, q.type);
                if (q.m) m[mb][u][h] = ns_load<2>(q.m, base[mb][h] + col, MLPSP_PRECISION_F32);
              }
            }
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
          for (int u = 0; u < CH; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int col = (c0 + u) * 8 + 2 * t;
              const bool in = base[mb][h] >= 0 && col < q.large;
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float g0 = v[mb][u][h].v[e];
                if (q.m) {
                  m[mb][u][h].v[e] = ns_new_momentum(q, g0, m[mb][u][h].v[e]);
                  g0 = ns_update(q, g0, m[mb][u][h].v[e]);
                }
                x[mb][c0 + u][h][e] = g0;
              }
              if (q.m && in) ns_store<2>(q.m, base[mb][h] + col, MLPSP_PRECISION_F32, m[mb][u][h]);
            }
      }
    } else {
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int col = nb * 8 + 2 * t + e;
              float v = 0.f;
              if (base[mb][h] >= 0 && col < q.large) {
                const int64_t at = base[mb][h] + (int64_t)col * q.cs;
                v = ns_load<1>(q.g, at, q.type).v[0];
                if (q.m) {
                  const float m = ns_new_momentum(q, v, q.m[at]);
                  v = ns_update(q, v, m);
                  q.m[at] = m;
                }
              }
              x[mb][nb][h][e] = v;
            }
    }
    // Frobenius norms, per matrix of the tile; once more, scaled, where the squares leave the range of FP32.  Rows h = 0 and 1 of
    // a lane may belong to two matrices where there is one block of rows, else all rows are those of one.
    constexpr int KH = MB == 1 ? 2 : 1;
    float f[KH];
    NsStart start[KH];       // lost: an infinity or a NaN; the result is NaN, and the tile's other matrices must not see it
#pragma unroll
    for (int h = 0; h < KH; ++h) f[h] = 1.f;
    for (int pass = 0; pass < 2; ++pass) {
      float ss[KH];
#pragma unroll
      for (int h = 0; h < KH; ++h) ss[h] = 0.f;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < 2; ++e) { const float v = x[mb][nb][h][e] * f[h % KH]; ss[h % KH] = fmaf(v, v, ss[h % KH]); }
      if (pack == 1) {
        float s = ss[0] + (KH == 2 ? ss[KH - 1] : 0.f);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
#pragma unroll
        for (int h = 0; h < KH; ++h) ss[h] = s;
      } else {
#pragma unroll
        for (int h = 0; h < KH; ++h) {
          ss[h] += __shfl_xor_sync(0xffffffffu, ss[h], 1);
          ss[h] += __shfl_xor_sync(0xffffffffu, ss[h], 2);
        }
        float s[2] = {0.f, 0.f};
        for (int r = 0; r < 16; ++r) {
          const float v = __shfl_sync(0xffffffffu, r < 8 ? ss[0] : ss[KH - 1], (r & 7) * 4);
          const int of = r / q.small;
          if (of == sub[0][0]) s[0] += v;
          if (of == sub[0][1]) s[1] += v;
        }
#pragma unroll
        for (int h = 0; h < KH; ++h) ss[h] = s[h];
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
    NsFrag<MB, NB> X;
#pragma unroll
    for (int h = 0; h < KH; ++h) { k2[h] = start[h].k; lost[h] = start[h].lost; }
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const NsStart& s = start[h % KH];
          ns_split(s.lost ? 0.f : x[mb][nb][h][0] * s.pre * s.inv, s.lost ? 0.f : x[mb][nb][h][1] * s.pre * s.inv, X.hi[mb][nb][h], X.lo[mb][nb][h]);
        }
    for (int it = 0; it < q.steps; ++it) {
      NsStep by[KH];
#pragma unroll
      for (int h = 0; h < KH; ++h) by[h] = ns_step(q, k2[h]);
      NsFrag<MB, 2 * MB> A;
      {
        float d[MB * (MB + 1)][4];
        ns_gram(X, d);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
          for (int n = 0; n < 2 * mb + 2; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float(&o)[4] = d[mb * (mb + 1) + n];
              float v0 = o[2 * h] * by[h % KH].gram, v1 = o[2 * h + 1] * by[h % KH].gram;
              if (MB == 1) {
                if (!(same >> (h * 4 + n * 2) & 1u)) v0 = 0.f;
                if (!(same >> (h * 4 + n * 2 + 1) & 1u)) v1 = 0.f;
              }
              ns_split(v0, v1, A.hi[mb][n][h], A.lo[mb][n][h]);
            }
      }
      ns_mirror<MB>(A);
      NsFrag<MB, 2 * MB> P;
      {
        float d[MB * (MB + 1)][4];
        ns_gram(A, d);
        const float c = q.c * kNsUnscale;
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
          for (int n = 0; n < 2 * mb + 2; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float(&o)[4] = d[mb * (mb + 1) + n];
              const float2 a = ns_join(A.hi[mb][n][h], A.lo[mb][n][h]);
              ns_split(fmaf(q.b, a.x, c * o[2 * h]), fmaf(q.b, a.y, c * o[2 * h + 1]), P.hi[mb][n][h], P.lo[mb][n][h]);
            }
      }
      ns_mirror<MB>(P);
      const bool last = it + 1 == q.steps;
#pragma unroll
      for (int c0 = 0; c0 < NB; c0 += CH) {
        uint32_t bh[CH][MB][2], bl[CH][MB][2];
        float d[CH][MB][4];
#pragma unroll
        for (int u = 0; u < CH; ++u)
#pragma unroll
          for (int k = 0; k < MB; ++k)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              bh[u][k][h] = ns_transpose(X.hi[k][c0 + u][h]);
              bl[u][k][h] = ns_transpose(X.lo[k][c0 + u][h]);
              d[u][k][2 * h] = d[u][k][2 * h + 1] = 0.f;
            }
#pragma unroll
        for (int part = 0; part < 3; ++part) {
          const auto& l = part == 1 ? P.lo : P.hi;
          const auto& r = part == 0 ? bl : bh;
#pragma unroll
          for (int k = 0; k < MB; ++k)
#pragma unroll
            for (int u = 0; u < CH; ++u)
#pragma unroll
              for (int mb = 0; mb < MB; ++mb)
                ns_mma(d[u][mb], l[mb][2 * k][0], l[mb][2 * k][1], l[mb][2 * k + 1][0], l[mb][2 * k + 1][1], r[u][k][0], r[u][k][1]);
        }
#pragma unroll
        for (int u = 0; u < CH; ++u)
#pragma unroll
          for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t &xh = X.hi[mb][c0 + u][h], &xl = X.lo[mb][c0 + u][h];
              const float2 v = ns_join(xh, xl);
              const NsStep& f1 = by[h % KH];
              const float v0 = fmaf(f1.a, v.x, d[u][mb][2 * h] * f1.unscale), v1 = fmaf(f1.a, v.y, d[u][mb][2 * h + 1] * f1.unscale);
              if (last) {          // the result keeps its FP32 bits in the two words of the pair
                xh = __float_as_uint(v0);
                xl = __float_as_uint(v1);
              } else {
                ns_split(v0, v1, xh, xl);
              }
            }
      }
    }
    const float nan = __int_as_float(0x7fffffff);
    auto result = [&](int mb, int nb, int h) {
      NsVec<2> r;
      const float fin = ns_exp2i(-10 - k2[h % KH]);
      r.v[0] = lost[h % KH] ? nan : __uint_as_float(X.hi[mb][nb][h]) * fin;
      r.v[1] = lost[h % KH] ? nan : __uint_as_float(X.lo[mb][nb][h]) * fin;
      return r;
    };
    if (q.vec >= 2) {
#pragma unroll
      for (int c0 = 0; c0 < NB; c0 += CH) {
        NsVec<2> w[MB][CH][2];
        if (q.m)
#pragma unroll
          for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int u = 0; u < CH; ++u)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int col = (c0 + u) * 8 + 2 * t;
                w[mb][u][h] = NsVec<2>{{0.f, 0.f}};
                if (base[mb][h] >= 0 && col < q.large) w[mb][u][h] = ns_load<2>(q.w, base[mb][h] + col, MLPSP_PRECISION_F32);
              }
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
          for (int u = 0; u < CH; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int col = (c0 + u) * 8 + 2 * t;
              if (base[mb][h] < 0 || col >= q.large) continue;
              NsVec<2> r = result(mb, c0 + u, h);
              if (q.m) {
#pragma unroll
                for (int e = 0; e < 2; ++e) r.v[e] = fmaf(-q.step, r.v[e], q.keep * w[mb][u][h].v[e]);
                ns_store<2>(q.w, base[mb][h] + col, MLPSP_PRECISION_F32, r);
              } else ns_store<2>(q.out, base[mb][h] + col, q.type, r);
            }
      }
    } else {
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const NsVec<2> r = result(mb, nb, h);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int col = nb * 8 + 2 * t + e;
              if (base[mb][h] < 0 || col >= q.large) continue;
              const int64_t at = base[mb][h] + (int64_t)col * q.cs;
              if (q.m) q.w[at] = fmaf(-q.step, r.v[e], q.keep * q.w[at]);
              else ns_store<1>(q.out, at, q.type, NsVec<1>{{r.v[e]}});
            }
          }
    }
  }
}

template <int MB, int NB, int CTAS>
static void ns_warp(const NsArgs& q, cudaStream_t st) {
  const int pack = std::max(1, 16 * MB / q.small);
  const int64_t tiles = (q.count + pack - 1) / pack;
  const unsigned grid = (unsigned)std::min<int64_t>((tiles + 3) / 4, (int64_t)sm_count() * CTAS);
  launch_chained(k_ns_warp<MB, NB, CTAS>, dim3(grid), dim3(128), 0, st, q, pack, tiles);
}

int launch_ns_warp(const NsArgs& q, cudaStream_t st) {
  LaunchScope scope(kKMisc, 1, st);
  const int nb = (q.large + 7) / 8;
  if (q.small <= 16) {
    if (nb <= 4) ns_warp<1, 4, 6>(q, st);
    else if (nb <= 6) ns_warp<1, 6, 5>(q, st);
    else if (nb <= 9) ns_warp<1, 9, 4>(q, st);
    else ns_warp<1, 12, 3>(q, st);
  } else {
    if (nb <= 4) ns_warp<2, 4, 4>(q, st);
    else if (nb <= 6) ns_warp<2, 6, 3>(q, st);
    else if (nb <= 9) ns_warp<2, 9, 3>(q, st);
    else ns_warp<2, 12, 2>(q, st);
  }
  return cuda_check(cudaGetLastError(), "orthogonalize");
}

}  // namespace mlpsp
