// Newton-Schulz iteration of matrices of at most 32 rows (the layers of a primitive among them), a warp per tile of 16 or 32 rows.
//
// X lies in the warp's shared memory as binary16 pairs, in panels of 16 columns, A and bA + cA^2 in its registers as fragments of m16n8 tiles (lane
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
#include "muon_mma.cuh"

namespace mlpsp {

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

// d += x x^T over 8 K columns; block (mb, n), n <= 2 mb + 1, is d[mb (mb + 1) + n].  ah, al: x as ns_ldmatrix<K> gives it; bh, bl: the
// same words with those of a row next to each other, as B operands want them (K = 1: the same).  The blocks
// advance together, since an MMA takes four times as long to answer as to issue; small products first, so that the tensor core's
// rounding of a sum towards zero meets fewer large ones.
template <int MB, int K, bool FIRST, int PART0 = 0, int PARTS = 3>
__device__ __forceinline__ void ns_gram(const uint32_t (&ah)[MB][4], const uint32_t (&al)[MB][4], const uint32_t (&bh)[MB][4],
                                        const uint32_t (&bl)[MB][4], float (&d)[MB * (MB + 1)][4]) {
#pragma unroll
  for (int part = PART0; part < PART0 + PARTS; ++part) {
    const auto& l = part == 1 ? al : ah;
    const auto& r = part == 0 ? bl : bh;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int n = 0; n < 2 * mb + 2; ++n) {
        float(&o)[4] = d[mb * (mb + 1) + n];
        const uint32_t(&w)[4] = r[n >> 1];
        if (K == 1) ns_mma8(o, l[mb][0], l[mb][1], w[n & 1]);
        else if (FIRST && part == 0) ns_mma_first(o, l[mb][0], l[mb][1], l[mb][2], l[mb][3], w[2 * (n & 1)], w[2 * (n & 1) + 1]);
        else ns_mma(o, l[mb][0], l[mb][1], l[mb][2], l[mb][3], w[2 * (n & 1)], w[2 * (n & 1) + 1]);
      }
  }
}

// A panel: hi [16 MB rows][16 columns], then lo; the two 16-byte halves of a row change places every four rows, so that eight rows of
// one half lie in different banks.  It takes the bytes of its values in FP32, as which they arrive.
template <int MB> __host__ __device__ constexpr int ns_panel_bytes() { return 16 * MB * 64; }

// brings the `n` elements at element i of an array of `size`-byte elements into L2 (addresses and sizes are multiples of 16 bytes)
__device__ __forceinline__ void ns_prefetch(const void* p, int64_t i, int n, int size) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(static_cast<const char*>(p) + i * size), "r"(n * size) : "memory");
}

// One tile per warp: which tiles an SM takes is left to the hardware.  With as many CTAs as fit the GPU walking the tiles in turn, the
// slowest SM set the time and its warps fell into step, all loading and then all multiplying: a step of 100,000 matrices of 32 x 72
// 2,540 us, so 1,750 (of which 704 are its bytes).  prefetch: a tile's weights, wanted last, are brought into L2 when it starts (5 percent).  Twenty warps per SM instead of sixteen: 2,160.
template <int MB, int NB, int CTAS>
__global__ void __launch_bounds__(32, CTAS) k_ns_warp(const NsArgs q, const int pack, const bool prefetch) {
  constexpr int KH = MB == 1 ? 2 : 1;       // with one block of rows, rows h = 0 and 1 of a lane may belong to two matrices
  constexpr int kPanel = ns_panel_bytes<MB>(), kLo = kPanel / 2, kBlock = 16 * 32;
  const int kPanels = NB ? (NB + 1) / 2 : (q.large + 15) / 16, kWhole = NB ? NB / 2 : kPanels;      // kWhole: of two columns of blocks
  extern __shared__ __align__(128) char smem[];
  ns_begin(q);
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  char* const mine = smem;
  const uint32_t xs = smem_u32(mine);
  // this lane's row of the 8 x 8 blocks that ldmatrix and stmatrix name: lanes 0-7 rows 0-7, 8-15 rows 8-15, 16-31 the same, 8 columns on
  const uint32_t xa = xs + (lane & 15) * 32 + (((lane >> 4) ^ ((lane >> 2) & 1)) << 4);
  // the same with the two halves of a row one after the other: lanes 0-7 rows 0-7, 8-15 the same, 8 columns on, 16-31 rows 8-15
  const uint32_t xb = xs + ((lane & 7) + ((lane >> 4) << 3)) * 32 + ((((lane >> 3) & 1) ^ ((lane >> 2) & 1)) << 4);
  float2* const keep = reinterpret_cast<float2*>(mine) + lane;      // this lane's values of a panel in FP32: [2 columns of blocks][MB][2]
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
  const int64_t tile = blockIdx.x;
  auto work = [&] {
    // element of the first column of this lane's rows; rows of block mb and half h are `in`
    int64_t first[KH];
    bool on[KH];
#pragma unroll
    for (int h = 0; h < KH; ++h) {
      const int64_t k = tile * pack + sub[h];
      on[h] = sub[h] >= 0 && k < q.count && (!q.active || q.active[k]);
      first[h] = on[h] ? k * q.stride + (int64_t)row[h] * q.rs : 0;
    }
    if (!__any_sync(0xffffffffu, on[0] || on[KH - 1])) return;
    if (prefetch && lane == 0 && q.m && (tile + 1) * pack <= q.count) {
      const int n = pack * (int)q.stride;
      ns_prefetch(q.w, tile * n, n, 4);
    }
    auto in = [&](int mb, int h) { return on[h % KH] && (MB == 1 || mb * 16 + h * 8 + g < q.small); };
    auto base = [&](int mb, int h) { return MB == 1 ? first[h % KH] : first[0] + (int64_t)((mb * 16 + h * 8) * q.rs); };
    __syncwarp();
    // ---- gradient and momentum, a panel at a time, to this lane's places in shared memory; sums of squares on the way
    float squares[2] = {0.f, 0.f};
    auto fetch = [&](auto tag, auto step) {
      constexpr int TYPE = decltype(tag)::value;
      constexpr bool STEP = decltype(step)::value;
#pragma unroll 1
      for (int p = 0; p < kPanels; ++p) {
        NsVec<2> v[2][MB][2], m[2][MB][2];
        float part[2] = {0.f, 0.f};
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int col = p * 16 + u * 8 + 2 * t;
              v[u][mb][h] = m[u][mb][h] = NsVec<2>{{0.f, 0.f}};
              if (in(mb, h) && col < q.large) {
                v[u][mb][h] = ns_load<2>(q.g, base(mb, h) + col, TYPE);
                if (STEP) m[u][mb][h] = ns_load<2>(q.m, base(mb, h) + col, MLPSP_PRECISION_F32);
              }
            }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int col = p * 16 + u * 8 + 2 * t;
              float2 y = make_float2(v[u][mb][h].v[0], v[u][mb][h].v[1]);
              if (STEP) {
                NsVec<2> n = m[u][mb][h];
                n.v[0] = ns_new_momentum(q, y.x, n.v[0]);
                n.v[1] = ns_new_momentum(q, y.y, n.v[1]);
                y = make_float2(ns_update(q, y.x, n.v[0]), ns_update(q, y.y, n.v[1]));
                if (in(mb, h) && col < q.large) ns_store<2>(q.m, base(mb, h) + col, MLPSP_PRECISION_F32, n);
              }
              part[h] = fmaf(y.x, y.x, fmaf(y.y, y.y, part[h]));
              keep[(p * 2 * MB * 2 + (u * MB + mb) * 2 + h) * 32] = y;
            }
        squares[0] += part[0];
        squares[1] += part[1];
      }
    };
    if (q.vec >= 2) {
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
      // odd rows, transposed matrices: element by element
      float part[2] = {0.f, 0.f};
#pragma unroll 1
      for (int i = 0; i < kPanels * 2 * MB; ++i) {
        const int nb = i / MB, mb = i % MB;
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
          part[h] = fmaf(y[0], y[0], fmaf(y[1], y[1], part[h]));
          keep[(i * 2 + h) * 32] = make_float2(y[0], y[1]);
          if (i % (2 * MB) == 2 * MB - 1) { squares[h] += part[h]; part[h] = 0.f; }      // panel by panel, as above
        }
      }
    }
    // Frobenius norms, per matrix of the tile; once more, scaled, where the squares leave the range of FP32
    float f[KH];
    NsStart start[KH];       // lost: an infinity or a NaN; the result is NaN, and the tile's other matrices must not see it
#pragma unroll
    for (int h = 0; h < KH; ++h) f[h] = 1.f;
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
      if (pass == 1) {
        squares[0] = squares[1] = 0.f;
#pragma unroll 1
        for (int i = 0; i < kPanels * 2 * MB; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 v = keep[(i * 2 + h) * 32];
            const float v0 = v.x * f[h % KH], v1 = v.y * f[h % KH];
            squares[h] = fmaf(v0, v0, fmaf(v1, v1, squares[h]));
          }
      }
      float ss[2] = {squares[0], squares[1]};
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
        if (pass == 1 && f[h] == 1.f) continue;       // settled
        start[h] = ns_start(q.eps, ss[h], f[h]);
        f[h] = start[h].lost ? kNsShrink : ss[h] < kNsTinySquares ? kNsGrow : 1.f;
        again |= f[h] != 1.f;
      }
      if (!__any_sync(0xffffffffu, again)) break;
    }
    int k2[KH];
    float done[KH];          // what the scaled result is multiplied by at the end, but for 2^-k
    bool odd = false;
#pragma unroll
    for (int h = 0; h < KH; ++h) {
      k2[h] = start[h].k;
      done[h] = start[h].lost ? __int_as_float(0x7fffffff) : 1.f / kNsScale;
      odd |= start[h].lost || start[h].pre != 1.f;
    }
    if (__any_sync(0xffffffffu, odd))
#pragma unroll 1
      for (int i = 0; i < kPanels * 2 * MB; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float2& v = keep[(i * 2 + h) * 32];
          const NsStart& s = start[h % KH];
          v = s.lost ? make_float2(0.f, 0.f) : make_float2(v.x * s.pre, v.y * s.pre);
        }
    // ---- X0, panel by panel in place
#pragma unroll 1
    for (int p = 0; p < kPanels; ++p) {
      uint32_t hi[MB][4], lo[MB][4];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 v = keep[(p * 2 * MB * 2 + (u * MB + mb) * 2 + h) * 32];
            const float s = start[h % KH].inv;
            ns_split2(v.x * s, v.y * s, hi[mb][2 * u + h], lo[mb][2 * u + h]);
          }
      __syncwarp();
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        ns_stmatrix<2>(xa + p * kPanel + mb * kBlock, hi[mb]);
        ns_stmatrix<2>(xa + p * kPanel + mb * kBlock + kLo, lo[mb]);
      }
    }
    __syncwarp();
#pragma unroll 1
    for (int it = 0; it < q.steps; ++it) {
      NsStep by[KH];
#pragma unroll
      for (int h = 0; h < KH; ++h) by[h] = ns_step(q, k2[h]);
      float d[MB * (MB + 1)][4];
      // ---- A = X X^T
#pragma unroll
      for (int i = 0; i < MB * (MB + 1); ++i) d[i][0] = d[i][1] = d[i][2] = d[i][3] = 0.f;
      auto columns = [&](int p, auto width) {
        constexpr int K = decltype(width)::value;
        uint32_t hi[MB][4], lo[MB][4], bh[MB][4], bl[MB][4];
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          const int at = p * kPanel + mb * kBlock;
          ns_ldmatrix<K, false>(hi[mb], xa + at);
          ns_ldmatrix<K, false>(lo[mb], xa + at + kLo);
          if (K == 2) {
            ns_ldmatrix<K, false>(bh[mb], xb + at);
            ns_ldmatrix<K, false>(bl[mb], xb + at + kLo);
          }
        }
        if (K == 2) ns_gram<MB, K, false>(hi, lo, bh, bl, d);
        else ns_gram<MB, K, false>(hi, lo, hi, lo, d);
      };
      if (NB) {
#pragma unroll 1
        for (int p = 0; p < kWhole; ++p) columns(p, NsTag<2>{});
      } else {
        // Long rows, four panels at a time, whose sums are added in FP32: the tensor core rounds towards zero with every MMA, which came to
        // 6.4e-6 of the result for 16 x 1024 and 6.6e-6 for 32 x 800, so to 4.7e-7 and 9.5e-7
        float sum[MB * (MB + 1)][4];
#pragma unroll
        for (int i = 0; i < MB * (MB + 1); ++i) sum[i][0] = sum[i][1] = sum[i][2] = sum[i][3] = 0.f;
#pragma unroll 1
        for (int p0 = 0; p0 < kWhole; p0 += 4) {
#pragma unroll 1
          for (int p = p0; p < min(p0 + 4, kWhole); ++p) columns(p, NsTag<2>{});
#pragma unroll
          for (int i = 0; i < MB * (MB + 1); ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              sum[i][e] += d[i][e];
              d[i][e] = 0.f;
            }
        }
#pragma unroll
        for (int i = 0; i < MB * (MB + 1); ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) d[i][e] = sum[i][e];
      }
      if (NB & 1) columns(NB / 2, NsTag<1>{});
      NsFrag<MB> A;
      float a32[MB * (MB + 1)][4], diag[MB][2];       // diag: of this lane's rows
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int n = 0; n < 2 * mb + 2; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int i = mb * (mb + 1) + n;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float v = d[i][2 * h + e] * by[h % KH].gram;
              if (MB == 1 && !(same >> (h * 4 + n * 2 + e) & 1u)) v = 0.f;
              a32[i][2 * h + e] = v;
            }
            if (n == 2 * mb + h) {       // the block on the diagonal: lane 4 g + g / 2 has row g's element
              diag[mb][h] = __shfl_sync(0xffffffffu, g & 1 ? a32[i][2 * h + 1] : a32[i][2 * h], 4 * g + (g >> 1));
              if (2 * t == g) a32[i][2 * h] = 0.f;
              if (2 * t + 1 == g) a32[i][2 * h + 1] = 0.f;
            }
            ns_split2(a32[i][2 * h], a32[i][2 * h + 1], A.hi[mb][n][h], A.lo[mb][n][h]);
          }
      ns_mirror<MB>(A);
      float own[MB][2];        // a + P(r, r) of this lane's rows
      float across[2 * MB][2]; // D of this lane's columns
#pragma unroll
      for (int n = 0; n < 2 * MB; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) across[n][e] = __shfl_sync(0xffffffffu, diag[n >> 1][n & 1], 4 * (2 * t + e));
      // ---- P = b A + c A^2, diagonals apart: with A = D + E, A^2 = D^2 + D E + E D + E^2, of which the tensor core forms E^2, and P's
      // diagonal multiplies X in FP32 below.  What is left to the tensor core is smaller, and with it what 22 bits and rounding towards zero take
      // off: 0.9 of a plain FP32 iteration's error instead of 1.3 for matrices of 4 x 32, half of 4e-6 for 128 rows.
#pragma unroll
      for (int round = 0; round < 2; ++round)
#pragma unroll
        for (int k = 0; k < MB; ++k) {
          uint32_t hi[MB][4], lo[MB][4], bh[MB][4], bl[MB][4];
#pragma unroll
          for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              hi[mb][i] = A.hi[mb][2 * k + (i >> 1)][i & 1];
              lo[mb][i] = A.lo[mb][2 * k + (i >> 1)][i & 1];
              bh[mb][i] = A.hi[mb][2 * k + (i & 1)][i >> 1];
              bl[mb][i] = A.lo[mb][2 * k + (i & 1)][i >> 1];
            }
          if (round == 1) ns_gram<MB, 2, false, 2, 1>(hi, lo, bh, bl, d);
          else if (k == 0) ns_gram<MB, 2, true, 0, 2>(hi, lo, bh, bl, d);
          else ns_gram<MB, 2, false, 0, 2>(hi, lo, bh, bl, d);
        }
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int n = 0; n < 2 * mb + 2; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int i = mb * (mb + 1) + n;
            const NsStep& s = by[h % KH];
            const float row_of = fmaf(s.c, diag[mb][h], s.b);
            float v0 = fmaf(s.c, d[i][2 * h], a32[i][2 * h] * fmaf(s.c, across[n][0], row_of));
            float v1 = fmaf(s.c, d[i][2 * h + 1], a32[i][2 * h + 1] * fmaf(s.c, across[n][1], row_of));
            if (n == 2 * mb + h) {
              own[mb][h] = fmaf(diag[mb][h], row_of, s.a) + __shfl_sync(0xffffffffu, g & 1 ? v1 : v0, 4 * g + (g >> 1));
              if (2 * t == g) v0 = 0.f;
              if (2 * t + 1 == g) v1 = 0.f;
            }
            ns_split2(v0, v1, A.hi[mb][n][h], A.lo[mb][n][h]);
          }
      ns_mirror<MB>(A);
      // The diagonal blocks of P's head with a + P(r, r) in binary16 on the diagonal, for the product with X's low half: what that adds
      // of (a + P(r, r)) X is right to 2^-11 of the low half, so only X's head is left to be multiplied below.
      uint32_t mixed[MB][2];
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          mixed[mb][h] = A.hi[mb][2 * mb + h][h] | (2 * t == (g & ~1) ? pack_h2<false>(g & 1 ? 0.f : own[mb][h], g & 1 ? own[mb][h] : 0.f) : 0u);
      // ---- X <- a X + P X, a panel at a time
      auto product = [&](int p, auto width, float (&e)[MB][2][4]) {
        constexpr int N = decltype(width)::value;
        uint32_t bh[MB][4], bl[MB][4];
#pragma unroll
        for (int k = 0; k < MB; ++k) {
          ns_ldmatrix<N, true>(bh[k], xa + p * kPanel + k * kBlock);
          ns_ldmatrix<N, true>(bl[k], xa + p * kPanel + k * kBlock + kLo);
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
              for (int mb = 0; mb < MB; ++mb) {
                const uint32_t a0 = part == 0 && k == mb ? mixed[mb][0] : l[mb][2 * k][0], a3 = part == 0 && k == mb ? mixed[mb][1] : l[mb][2 * k + 1][1];
                if (part == 0 && k == 0) ns_mma_first(e[mb][n], a0, l[mb][0][1], l[mb][1][0], a3, r[0][2 * n], r[0][2 * n + 1]);
                else ns_mma(e[mb][n], a0, l[mb][2 * k][1], l[mb][2 * k + 1][0], a3, r[k][2 * n], r[k][2 * n + 1]);
              }
        }
      };
      auto advance = [&](int mb, int p, auto width, const float (&e)[MB][2][4], float (&v)[2][2][2], uint32_t (&hi)[4]) {
        constexpr int N = decltype(width)::value;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 x = ns_unpack<false>(hi[2 * n + h]);
            v[n][h][0] = fmaf(own[mb][h], x.x, e[mb][n][2 * h]);
            v[n][h][1] = fmaf(own[mb][h], x.y, e[mb][n][2 * h + 1]);
          }
      };
      if (it + 1 < q.steps) {
        // the next panel's products are issued among the splits of this one's: alone, the warps of a scheduler queue for the tensor cores
        // together and then for the other units together, and neither is busy for more than half of the time
        auto heads = [&](int p, auto width, uint32_t (&hi)[MB][4]) {
#pragma unroll
          for (int mb = 0; mb < MB; ++mb) ns_ldmatrix<decltype(width)::value, false>(hi[mb], xa + p * kPanel + mb * kBlock);
        };
        auto store = [&](int p, auto width, const float (&e)[MB][2][4], uint32_t (&hi)[MB][4]) {
          constexpr int N = decltype(width)::value;
          uint32_t lo[MB][4];
#pragma unroll
          for (int mb = 0; mb < MB; ++mb) {
            float v[2][2][2];
            advance(mb, p, width, e, v, hi[mb]);
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
              for (int h = 0; h < 2; ++h) ns_split2(v[n][h][0], v[n][h][1], hi[mb][2 * n + h], lo[mb][2 * n + h]);
          }
#pragma unroll
          for (int mb = 0; mb < MB; ++mb) {
            ns_stmatrix<N>(xa + p * kPanel + mb * kBlock, hi[mb]);
            ns_stmatrix<N>(xa + p * kPanel + mb * kBlock + kLo, lo[mb]);
          }
        };
        float e[MB][2][4], next[MB][2][4];
        uint32_t hi[MB][4];
        product(0, NsTag<2>{}, e);
#pragma unroll 1
        for (int p = 1; p < kWhole; ++p) {
          heads(p - 1, NsTag<2>{}, hi);
          product(p, NsTag<2>{}, next);
          store(p - 1, NsTag<2>{}, e, hi);
#pragma unroll
          for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int i = 0; i < 8; ++i) e[mb][i >> 2][i & 3] = next[mb][i >> 2][i & 3];
        }
        heads(kWhole - 1, NsTag<2>{}, hi);
        if (NB & 1) product(NB / 2, NsTag<1>{}, next);
        store(kWhole - 1, NsTag<2>{}, e, hi);
        if (NB & 1) {
          heads(NB / 2, NsTag<1>{}, hi);
          store(NB / 2, NsTag<1>{}, next, hi);
        }
        __syncwarp();
        continue;
      }
      auto finish = [&](int p, auto width) {
        constexpr int N = decltype(width)::value;
        float e[MB][2][4];
        product(p, width, e);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          uint32_t hi[4];
          ns_ldmatrix<N, false>(hi, xa + p * kPanel + mb * kBlock);
          float v[2][2][2];
          advance(mb, p, width, e, v, hi);
#pragma unroll
          for (int n = 0; n < N; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int col = p * 16 + n * 8 + 2 * t;
              if (!in(mb, h) || col >= q.large) continue;
              const float fin = done[h % KH] * ns_exp2i(-k2[h % KH]);
              NsVec<2> y;
              y.v[0] = v[n][h][0] * fin;
              y.v[1] = v[n][h][1] * fin;
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
      for (int p = 0; p < kWhole; ++p) finish(p, NsTag<2>{});
      if (NB & 1) finish(NB / 2, NsTag<1>{});
    }
  };
  work();
  ns_end(q);
}

template <int MB, int NB, int CTAS>
static int ns_warp(const NsArgs& q, cudaStream_t st, bool launch) {
  constexpr int most = (NB ? (NB + 1) / 2 : kNsWarpLong[MB - 1] / 16) * ns_panel_bytes<MB>();
  static_assert(NB == 0 || CTAS * (most + 1024) <= 227 * 1024, "resident CTAs");
  const int smem = NB ? most : (q.large + 15) / 16 * ns_panel_bytes<MB>();
  MLPSP_SHARED_MEMORY(most, (const void*)k_ns_warp<MB, NB, CTAS>);
  const int pack = std::max(1, 16 * MB / q.small);
  const int64_t tiles = (q.count + pack - 1) / pack;
  MLPSP_REQUIRE(tiles < (1ll << 31), MLPSP_E_LIMIT, "orthogonalize: too many matrices");
  if (!launch) return MLPSP_OK;
  const bool prefetch = reinterpret_cast<uintptr_t>(q.w) % 16 == 0 && pack * q.stride % 4 == 0;
  LaunchScope scope(kKMisc, 1, st);
  return cuda_check(launch_chained(k_ns_warp<MB, NB, CTAS>, dim3((unsigned)tiles), dim3(32), smem, st, q, pack, prefetch), "orthogonalize");
}

int launch_ns_warp(const NsArgs& q, cudaStream_t st, bool launch) {
  const int nb = (q.large + 7) / 8;
  auto* run = q.small <= 16 ? (nb <= 4 ? ns_warp<1, 4, 32> : nb <= 6 ? ns_warp<1, 6, 28> : nb <= 9 ? ns_warp<1, 9, 28> : nb <= 12 ? ns_warp<1, 12, 28> : ns_warp<1, 0, 24>)
                            : (nb <= 4 ? ns_warp<2, 4, 16> : nb <= 6 ? ns_warp<2, 6, 16> : nb <= 9 ? ns_warp<2, 9, 16> : nb <= 12 ? ns_warp<2, 12, 16> : ns_warp<2, 0, 16>);
  return run(q, st, launch);
}

}  // namespace mlpsp
