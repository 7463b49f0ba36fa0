// Newton-Schulz iteration of matrices of 33 to 64 rows (64-wide layers of a primitive among them), two warps per matrix.
//
// The scheme of muon_warp.cu for twice the rows: X and A lie in shared memory as binary16 pairs in panels of 16 columns, warp w has the
// rows 32 w to 32 w + 31.  Of A and A^2 a warp computes the blocks of its own rows on and below the diagonal (six of 16 x 8) and half of the
// 32 x 32 block between the two (rows 0 to 31, columns 32 + 16 w on: four), 20 of 32 in all and ten each, and stores what lies off the
// diagonal a second time transposed.  bA + cA^2 is held as fragments of the warp's rows; X's panels are read by both warps before either
// writes its rows of them back.
//
// A tcgen05 tile holds two such matrices at a time and spends half of its products on the blocks between them: with the passes through
// tensor memory a 64 x 72 matrix took 97 ns of the GPU that way, 57 here (five steps, thousands of matrices), where mma.sync is busy for 55
// percent of the time and shared memory for 60 to 70.
#include "muon_mma.cuh"

namespace mlpsp {

constexpr int kNpThreads = 64, kNpRows = 64, kNpPanel = kNpRows * 64, kNpLo = kNpPanel / 2, kNpBlock = 16 * 32;
__host__ __device__ constexpr int np_smem(int panels) { return (panels + 4) * kNpPanel + 32 + 4 * kNpRows; }

// d: blocks (mb, n), n <= 2 mb + 1, of the warp's own rows at mb (mb + 1) + n; o: blocks (mb, n) of rows 16 mb, columns 32 + 16 w + 8 n at 2 mb + n
struct NpBlocks { float d[6][4], o[4][4]; };

// += x x^T over a panel of 8 K columns at `at`; own, top, off: byte offsets of the warp's rows, of row 0 and of row 32 + 16 w
template <int K>
__device__ __forceinline__ void np_gram(uint32_t xa, uint32_t xb, int own, int off, NpBlocks& b) {
  uint32_t ah[2][4], al[2][4], bh[2][4], bl[2][4];
#pragma unroll
  for (int mb = 0; mb < 2; ++mb) {
    ns_ldmatrix<K, false>(ah[mb], xa + own + mb * kNpBlock);
    ns_ldmatrix<K, false>(al[mb], xa + own + mb * kNpBlock + kNpLo);
    if (K == 2) {
      ns_ldmatrix<K, false>(bh[mb], xb + own + mb * kNpBlock);
      ns_ldmatrix<K, false>(bl[mb], xb + own + mb * kNpBlock + kNpLo);
    }
  }
  // word of rows 8 h of a block as the B operand's first or second
  auto mul = [&](float (&d)[4], const uint32_t (&l)[4], const uint32_t (&r)[4], int h) {
    if (K == 2) ns_mma(d, l[0], l[1], l[2], l[3], r[2 * h], r[2 * h + 1]);
    else ns_mma8(d, l[0], l[1], r[h]);
  };
#pragma unroll
  for (int part = 0; part < 3; ++part)
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int n = 0; n < 2 * mb + 2; ++n) {
        const auto& l = part == 1 ? al : ah;
        const auto& r = K == 2 ? (part == 0 ? bl : bh) : (part == 0 ? al : ah);
        mul(b.d[mb * (mb + 1) + n], l[mb], r[n >> 1], n & 1);
      }
  // the block between the warps: warp 0 has its left operand already, warp 1 its right one
  auto between = [&](const uint32_t (&th)[2][4], const uint32_t (&tl)[2][4], const uint32_t (&oh)[4], const uint32_t (&ol)[4]) {
#pragma unroll
    for (int part = 0; part < 3; ++part)
#pragma unroll
      for (int mb = 0; mb < 2; ++mb)
#pragma unroll
        for (int n = 0; n < 2; ++n) mul(b.o[2 * mb + n], part == 1 ? tl[mb] : th[mb], part == 0 ? ol : oh, n);
  };
  if (own == 0) {
    uint32_t oh[4], ol[4];
    ns_ldmatrix<K, false>(oh, (K == 2 ? xb : xa) + off);
    ns_ldmatrix<K, false>(ol, (K == 2 ? xb : xa) + off + kNpLo);
    between(ah, al, oh, ol);
  } else {
    uint32_t th[2][4], tl[2][4];
#pragma unroll
    for (int mb = 0; mb < 2; ++mb) {
      ns_ldmatrix<K, false>(th[mb], xa + mb * kNpBlock);
      ns_ldmatrix<K, false>(tl[mb], xa + mb * kNpBlock + kNpLo);
    }
    if (K == 2) between(th, tl, bh[1], bl[1]);
    else between(th, tl, ah[1], al[1]);
  }
}

// the 16 x 16 block of a symmetric matrix at (row block i, column block j), and its transpose at (j, i)
__device__ __forceinline__ void np_put(uint32_t sa, int i, int j, const float (&b0)[4], const float (&b1)[4], bool mirror) {
  uint32_t hi[4], lo[4];
  ns_split2(b0[0], b0[1], hi[0], lo[0]);
  ns_split2(b0[2], b0[3], hi[1], lo[1]);
  ns_split2(b1[0], b1[1], hi[2], lo[2]);
  ns_split2(b1[2], b1[3], hi[3], lo[3]);
  ns_stmatrix<2>(sa + j * kNpPanel + i * kNpBlock, hi);
  ns_stmatrix<2>(sa + j * kNpPanel + i * kNpBlock + kNpLo, lo);
  if (!mirror) return;
  const uint32_t th[4] = {hi[0], hi[2], hi[1], hi[3]}, tl[4] = {lo[0], lo[2], lo[1], lo[3]};
  ns_stmatrix<2, true>(sa + i * kNpPanel + j * kNpBlock, th);
  ns_stmatrix<2, true>(sa + i * kNpPanel + j * kNpBlock + kNpLo, tl);
}
__device__ __forceinline__ void np_put(uint32_t sa, int w, const NpBlocks& b) {
  np_put(sa, 2 * w, 2 * w, b.d[0], b.d[1], false);
  np_put(sa, 2 * w + 1, 2 * w, b.d[2], b.d[3], true);
  np_put(sa, 2 * w + 1, 2 * w + 1, b.d[4], b.d[5], false);
  np_put(sa, 0, 2 + w, b.o[0], b.o[1], true);
  np_put(sa, 1, 2 + w, b.o[2], b.o[3], true);
}

template <int NB, int CTAS>
__global__ void __launch_bounds__(kNpThreads, CTAS) k_ns_pair(const NsArgs q, const bool prefetch) {
  const int kPanels = NB ? (NB + 1) / 2 : (q.large + 15) / 16, kWhole = NB ? NB / 2 : kPanels;      // kWhole: of two columns of blocks
  extern __shared__ __align__(128) char smem[];
  ns_begin(q);
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, w = warp_of_cta();
  const int own = 2 * w * kNpBlock, off = (2 + w) * kNpBlock;
  const uint32_t xs = smem_u32(smem);
  // ldmatrix's places as in muon_warp.cu, of the first panel
  const uint32_t xa = xs + (lane & 15) * 32 + (((lane >> 4) ^ ((lane >> 2) & 1)) << 4);
  const uint32_t xb = xs + ((lane & 7) + ((lane >> 4) << 3)) * 32 + ((((lane >> 3) & 1) ^ ((lane >> 2) & 1)) << 4);
  const uint32_t aa = xa + kPanels * kNpPanel, ab = xb + kPanels * kNpPanel;      // A's panels behind X's
  float* const s_sum = reinterpret_cast<float*>(smem + (kPanels + 4) * kNpPanel);   // [2][2] sums of squares, by pass and warp
  float* const s_diag = s_sum + 8;                                                   // [64] the diagonal of A
  // this lane's values of a panel in FP32, [2 columns of blocks][2 blocks of rows][2], in the places of its rows' heads and tails
  auto keep = [&](int p, int u, int mb, int h) -> float2& {
    return *reinterpret_cast<float2*>(smem + p * kNpPanel + u * kNpLo + own + ((mb * 2 + h) * 32 + lane) * 8);
  };
  const int64_t k = blockIdx.x;
  auto work = [&] {
    if (q.active && !q.active[k]) return;
    const int64_t first = k * q.stride + (int64_t)(32 * w + g) * q.rs;
    auto in = [&](int mb, int h) { return 32 * w + mb * 16 + h * 8 + g < q.small; };
    auto base = [&](int mb, int h) { return first + (int64_t)((mb * 16 + h * 8) * q.rs); };
    if (prefetch && threadIdx.x == 0 && q.m)
      asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(q.w + k * q.stride), "r"((int)q.stride * 4) : "memory");
    // ---- gradient and momentum
    float squares = 0.f;
    auto fetch = [&](auto width, auto tag, auto step) {
      constexpr int V = decltype(width)::value, TYPE = decltype(tag)::value;
      constexpr bool STEP = decltype(step)::value;
      const int type = TYPE < 0 ? q.type : TYPE;
      const bool stepping = V == 1 ? q.m != nullptr : STEP;
#pragma unroll 1
      for (int p = 0; p < kPanels; ++p) {
        float v[2][2][2][2], m[2][2][2][2], part = 0.f;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int mb = 0; mb < 2; ++mb)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int e = 0; e < 2; e += V) {
                const int col = p * 16 + u * 8 + 2 * t + e;
#pragma unroll
                for (int i = 0; i < V; ++i) v[u][mb][h][e + i] = m[u][mb][h][e + i] = 0.f;
                if (in(mb, h) && col < q.large) {
                  const int64_t at = base(mb, h) + (V == 2 ? (int64_t)col : (int64_t)col * q.cs);
                  const NsVec<V> x = ns_load<V>(q.g, at, type);
                  NsVec<V> y = {};
                  if (stepping) y = ns_load<V>(q.m, at, MLPSP_PRECISION_F32);
#pragma unroll
                  for (int i = 0; i < V; ++i) { v[u][mb][h][e + i] = x.v[i]; m[u][mb][h][e + i] = y.v[i]; }
                }
              }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int mb = 0; mb < 2; ++mb)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float (&x)[2] = v[u][mb][h];
              if (stepping) {
#pragma unroll
                for (int e = 0; e < 2; e += V) {
                  const int col = p * 16 + u * 8 + 2 * t + e;
                  NsVec<V> n;
#pragma unroll
                  for (int i = 0; i < V; ++i) {
                    n.v[i] = ns_new_momentum(q, x[e + i], m[u][mb][h][e + i]);
                    x[e + i] = ns_update(q, x[e + i], n.v[i]);
                  }
                  if (in(mb, h) && col < q.large)
                    ns_store<V>(q.m, base(mb, h) + (V == 2 ? (int64_t)col : (int64_t)col * q.cs), MLPSP_PRECISION_F32, n);
                }
              }
              part = fmaf(x[0], x[0], fmaf(x[1], x[1], part));
              keep(p, u, mb, h) = make_float2(x[0], x[1]);
            }
        squares += part;
      }
    };
    if (q.vec >= 2) {
      if (q.m) {
        if (q.type == MLPSP_PRECISION_F32) fetch(NsTag<2>{}, NsTag<MLPSP_PRECISION_F32>{}, NsTag<1>{});
        else if (q.type == MLPSP_PRECISION_F16) fetch(NsTag<2>{}, NsTag<MLPSP_PRECISION_F16>{}, NsTag<1>{});
        else fetch(NsTag<2>{}, NsTag<MLPSP_PRECISION_BF16>{}, NsTag<1>{});
      } else {
        if (q.type == MLPSP_PRECISION_F32) fetch(NsTag<2>{}, NsTag<MLPSP_PRECISION_F32>{}, NsTag<0>{});
        else if (q.type == MLPSP_PRECISION_F16) fetch(NsTag<2>{}, NsTag<MLPSP_PRECISION_F16>{}, NsTag<0>{});
        else fetch(NsTag<2>{}, NsTag<MLPSP_PRECISION_BF16>{}, NsTag<0>{});
      }
    } else {
      fetch(NsTag<1>{}, NsTag<-1>{}, NsTag<0>{});
    }
    // ---- the norm; once more, scaled, where the squares leave the range of FP32
    float f = 1.f;
    NsStart start;
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
      if (pass == 1) {
        squares = 0.f;
#pragma unroll 1
        for (int i = 0; i < kPanels * 8; ++i) {
          const float2 v = keep(i >> 3, (i >> 2) & 1, (i >> 1) & 1, i & 1);
          const float v0 = v.x * f, v1 = v.y * f;
          squares = fmaf(v0, v0, fmaf(v1, v1, squares));
        }
      }
      float s = squares;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == 0) s_sum[pass * 2 + w] = s;
      __syncthreads();
      s = s_sum[pass * 2] + s_sum[pass * 2 + 1];
      start = ns_start(q.eps, s, f);
      f = start.lost ? kNsShrink : s < kNsTinySquares ? kNsGrow : 1.f;
      if (f == 1.f) break;           // the same in both warps
    }
    int k2 = start.k;
    const float done = start.lost ? __int_as_float(0x7fffffff) : 1.f / kNsScale;
    // ---- X0, panel by panel in place
#pragma unroll 1
    for (int p = 0; p < kPanels; ++p) {
      uint32_t hi[2][4], lo[2][4];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int mb = 0; mb < 2; ++mb)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 v = keep(p, u, mb, h);
            float x0 = v.x * start.pre * start.inv, x1 = v.y * start.pre * start.inv;
            if (start.lost) x0 = x1 = 0.f;
            ns_split2(x0, x1, hi[mb][2 * u + h], lo[mb][2 * u + h]);
          }
      __syncwarp();
#pragma unroll
      for (int mb = 0; mb < 2; ++mb) {
        ns_stmatrix<2>(xa + p * kNpPanel + own + mb * kNpBlock, hi[mb]);
        ns_stmatrix<2>(xa + p * kNpPanel + own + mb * kNpBlock + kNpLo, lo[mb]);
      }
    }
    __syncthreads();
#pragma unroll 1
    for (int it = 0; it < q.steps; ++it) {
      const NsStep by = ns_step(q, k2);
      NpBlocks A, S;
      // ---- A = X X^T
#pragma unroll
      for (int i = 0; i < 6; ++i) A.d[i][0] = A.d[i][1] = A.d[i][2] = A.d[i][3] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) A.o[i][0] = A.o[i][1] = A.o[i][2] = A.o[i][3] = 0.f;
      if (NB) {
#pragma unroll 1
        for (int p = 0; p < kWhole; ++p) np_gram<2>(xa + p * kNpPanel, xb + p * kNpPanel, own, off, A);
      } else {
        // long rows two panels at a time (muon_warp.cu)
#pragma unroll 1
        for (int p0 = 0; p0 < kWhole; p0 += 2) {
          NpBlocks part = {};
#pragma unroll 1
          for (int p = p0; p < min(p0 + 2, kWhole); ++p) np_gram<2>(xa + p * kNpPanel, xb + p * kNpPanel, own, off, part);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
#pragma unroll
            for (int i = 0; i < 6; ++i) A.d[i][e] += part.d[i][e];
#pragma unroll
            for (int i = 0; i < 4; ++i) A.o[i][e] += part.o[i][e];
          }
        }
      }
      if (NB & 1) np_gram<1>(xa + NB / 2 * kNpPanel, xb + NB / 2 * kNpPanel, own, off, A);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
#pragma unroll
        for (int i = 0; i < 6; ++i) A.d[i][e] *= by.gram;
#pragma unroll
        for (int i = 0; i < 4; ++i) A.o[i][e] *= by.gram;
      }
#pragma unroll
      for (int mb = 0; mb < 2; ++mb)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float (&b)[4] = A.d[mb * (mb + 1) + 2 * mb + h];       // the block on the diagonal: lane 4 g + g / 2 has row g's element
          if (t == g >> 1) s_diag[32 * w + mb * 16 + h * 8 + g] = g & 1 ? b[2 * h + 1] : b[2 * h];
          if (2 * t == g) b[2 * h] = 0.f;
          if (2 * t + 1 == g) b[2 * h + 1] = 0.f;
        }
      np_put(aa, w, A);
      __syncthreads();
      // ---- P = b A + c A^2, diagonals apart (muon_warp.cu)
#pragma unroll
      for (int i = 0; i < 6; ++i) S.d[i][0] = S.d[i][1] = S.d[i][2] = S.d[i][3] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) S.o[i][0] = S.o[i][1] = S.o[i][2] = S.o[i][3] = 0.f;
#pragma unroll 1
      for (int p = 0; p < 4; ++p) np_gram<2>(aa + p * kNpPanel, ab + p * kNpPanel, own, off, S);
      float diag[2][2];        // a + P(r, r) of this lane's rows
      auto form = [&](float (&o)[4], const float (&e)[4], int row0, int col0) {
        const float2 c = *reinterpret_cast<const float2*>(s_diag + col0 + 2 * t);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float row_of = fmaf(by.c, s_diag[row0 + h * 8 + g], by.b);
          o[2 * h] = fmaf(by.c, o[2 * h], e[2 * h] * fmaf(by.c, c.x, row_of));
          o[2 * h + 1] = fmaf(by.c, o[2 * h + 1], e[2 * h + 1] * fmaf(by.c, c.y, row_of));
        }
      };
#pragma unroll
      for (int mb = 0; mb < 2; ++mb) {
#pragma unroll
        for (int n = 0; n < 2 * mb + 2; ++n) form(S.d[mb * (mb + 1) + n], A.d[mb * (mb + 1) + n], 32 * w + 16 * mb, 32 * w + 8 * n);
#pragma unroll
        for (int n = 0; n < 2; ++n) form(S.o[2 * mb + n], A.o[2 * mb + n], 16 * mb, 32 + 16 * w + 8 * n);
      }
#pragma unroll
      for (int mb = 0; mb < 2; ++mb)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float (&b)[4] = S.d[mb * (mb + 1) + 2 * mb + h];
          const float d = s_diag[32 * w + mb * 16 + h * 8 + g];
          diag[mb][h] = fmaf(d, fmaf(by.c, d, by.b), by.a) + __shfl_sync(0xffffffffu, g & 1 ? b[2 * h + 1] : b[2 * h], 4 * g + (g >> 1));
          if (2 * t == g) b[2 * h] = 0.f;
          if (2 * t + 1 == g) b[2 * h + 1] = 0.f;
        }
      __syncthreads();         // A has been read
      np_put(aa, w, S);
      __syncthreads();
      uint32_t ph[2][4][4], pl[2][4][4];
#pragma unroll
      for (int mb = 0; mb < 2; ++mb)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          ns_ldmatrix<2, false>(ph[mb][c], aa + c * kNpPanel + own + mb * kNpBlock);
          ns_ldmatrix<2, false>(pl[mb][c], aa + c * kNpPanel + own + mb * kNpBlock + kNpLo);
        }
      // ---- X <- a X + P X, a panel at a time
      auto product = [&](int p, auto width, float (&e)[2][2][4]) {
        constexpr int N = decltype(width)::value;
        uint32_t bh[4][4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t bl[4];
          ns_ldmatrix<N, true>(bh[c], xa + p * kNpPanel + c * kNpBlock);
          ns_ldmatrix<N, true>(bl, xa + p * kNpPanel + c * kNpBlock + kNpLo);
#pragma unroll
          for (int n = 0; n < N; ++n)
#pragma unroll
            for (int mb = 0; mb < 2; ++mb) {
              const uint32_t(&l)[4] = ph[mb][c];
              if (c == 0) ns_mma_first(e[mb][n], l[0], l[1], l[2], l[3], bl[2 * n], bl[2 * n + 1]);
              else ns_mma(e[mb][n], l[0], l[1], l[2], l[3], bl[2 * n], bl[2 * n + 1]);
            }
#pragma unroll
          for (int n = 0; n < N; ++n)
#pragma unroll
            for (int mb = 0; mb < 2; ++mb)
              ns_mma(e[mb][n], pl[mb][c][0], pl[mb][c][1], pl[mb][c][2], pl[mb][c][3], bh[c][2 * n], bh[c][2 * n + 1]);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int n = 0; n < N; ++n)
#pragma unroll
            for (int mb = 0; mb < 2; ++mb)
              ns_mma(e[mb][n], ph[mb][c][0], ph[mb][c][1], ph[mb][c][2], ph[mb][c][3], bh[c][2 * n], bh[c][2 * n + 1]);
      };
      // rows of block mb: the new values
      auto advance = [&](int mb, int p, auto width, const float (&e)[2][2][4], float (&v)[2][2][2]) {
        constexpr int N = decltype(width)::value;
        uint32_t hi[4], lo[4];
        ns_ldmatrix<N, false>(hi, xa + p * kNpPanel + own + mb * kNpBlock);
        ns_ldmatrix<N, false>(lo, xa + p * kNpPanel + own + mb * kNpBlock + kNpLo);
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 x = ns_unpack<false>(hi[2 * n + h]), y = ns_unpack<false>(lo[2 * n + h]);
            v[n][h][0] = fmaf(diag[mb][h], x.x, fmaf(diag[mb][h], y.x, e[mb][n][2 * h]));
            v[n][h][1] = fmaf(diag[mb][h], x.y, fmaf(diag[mb][h], y.y, e[mb][n][2 * h + 1]));
          }
      };
      if (it + 1 < q.steps) {
        auto store = [&](int p, auto width, const float (&e)[2][2][4]) {
          constexpr int N = decltype(width)::value;
#pragma unroll
          for (int mb = 0; mb < 2; ++mb) {
            float v[2][2][2];
            uint32_t hi[4], lo[4];
            advance(mb, p, width, e, v);
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
              for (int h = 0; h < 2; ++h) ns_split2(v[n][h][0], v[n][h][1], hi[2 * n + h], lo[2 * n + h]);
            ns_stmatrix<N>(xa + p * kNpPanel + own + mb * kNpBlock, hi);
            ns_stmatrix<N>(xa + p * kNpPanel + own + mb * kNpBlock + kNpLo, lo);
          }
        };
        float e[2][2][4], next[2][2][4];
        product(0, NsTag<2>{}, e);
#pragma unroll 1
        for (int p = 1; p < kWhole; ++p) {
          __syncthreads();       // both warps have read panel p - 1
          product(p, NsTag<2>{}, next);
          store(p - 1, NsTag<2>{}, e);
#pragma unroll
          for (int mb = 0; mb < 2; ++mb)
#pragma unroll
            for (int i = 0; i < 8; ++i) e[mb][i >> 2][i & 3] = next[mb][i >> 2][i & 3];
        }
        __syncthreads();
        if (NB & 1) product(NB / 2, NsTag<1>{}, next);
        store(kWhole - 1, NsTag<2>{}, e);
        if (NB & 1) {
          __syncthreads();
          store(NB / 2, NsTag<1>{}, next);
        }
        __syncthreads();
        continue;
      }
      auto finish = [&](int p, auto width) {
        constexpr int N = decltype(width)::value;
        float e[2][2][4];
        product(p, width, e);
#pragma unroll
        for (int mb = 0; mb < 2; ++mb) {
          float v[2][2][2];
          advance(mb, p, width, e, v);
          const float fin = done * ns_exp2i(-k2);
#pragma unroll
          for (int n = 0; n < N; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int col = p * 16 + n * 8 + 2 * t;
              if (!in(mb, h) || col >= q.large) continue;
              NsVec<2> y;
              y.v[0] = v[n][h][0] * fin;
              y.v[1] = v[n][h][1] * fin;
              if (q.vec >= 2) {
                const int64_t i = base(mb, h) + col;
                if (q.m) {
                  const NsVec<2> x = ns_load<2>(q.w, i, MLPSP_PRECISION_F32);
#pragma unroll
                  for (int c = 0; c < 2; ++c) y.v[c] = fmaf(-q.step, y.v[c], q.keep * x.v[c]);
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

template <int NB, int CTAS>
static int ns_pair(const NsArgs& q, cudaStream_t st, bool launch) {
  constexpr int most = np_smem(NB ? (NB + 1) / 2 : kNsPairLong / 16);
  static_assert(most <= 227 * 1024 && (NB == 0 || CTAS * (most + 1024) <= 227 * 1024), "resident CTAs");
  const int smem = NB ? most : np_smem((q.large + 15) / 16);
  MLPSP_SHARED_MEMORY(most, (const void*)k_ns_pair<NB, CTAS>);
  MLPSP_REQUIRE(q.count < (1ll << 31), MLPSP_E_LIMIT, "orthogonalize: too many matrices");
  if (!launch) return MLPSP_OK;
  const bool prefetch = reinterpret_cast<uintptr_t>(q.w) % 16 == 0 && q.stride % 4 == 0;
  LaunchScope scope(kKMisc, 1, st);
  return cuda_check(launch_chained(k_ns_pair<NB, CTAS>, dim3((unsigned)q.count), dim3(kNpThreads), smem, st, q, prefetch), "orthogonalize");
}

int launch_ns_pair(const NsArgs& q, cudaStream_t st, bool launch) {
  const int nb = (q.large + 7) / 8;
  return (nb <= 6 ? ns_pair<6, 6> : nb <= 8 ? ns_pair<8, 6> : nb <= 9 ? ns_pair<9, 6> : nb <= 12 ? ns_pair<12, 5> : ns_pair<0, 6>)(q, st, launch);
}

}  // namespace mlpsp
