// Newton-Schulz iteration of matrices up to 128 x 2048 on the 5th-generation tensor cores (tcgen05), and the C entries.
//
// A CTA holds a slice of X, 128 rows by up to 256 columns, in shared memory as binary16 pairs, in chunks of [128 rows][8 columns].
// The same bytes are the K-major operands of A = X X^T and, read MN-major, the B operand of (bA + cA^2) X.  A matrix of more columns
// than one slice is spread over a cluster of up to eight CTAs, which add their parts of A through distributed shared memory; A^2 is
// computed by each.  Matrices of few rows are stacked (four of 32): the blocks of A off their diagonal are cleared, after which
// everything stays block-diagonal.  Accumulators (A | A^2, later the new slice in the same columns) are in tensor memory.
//
// Every wait on an mbarrier is bounded.  A CTA in which one gives up issues no further products, hands NaN to its cluster, makes its slice of
// the result NaN, waits once more (bounded too) for the products it had issued before it frees their tensor memory, and tells the host.
#include <cmath>
#include "muon.cuh"

namespace mlpsp {

constexpr int kNtThreads = 512, kNtParts = 4;      // four threads per row: the parts of its columns
constexpr int kNtRows = 128, kNtChunk = kNtRows * 16;
constexpr int kNtMaxCols = 256, kNtMaxCluster = 8;
constexpr int kNtTmemCols = 256;
constexpr uint32_t kNtMnB = 1u << 16;      // bit 16 of the instruction descriptor: B is MN-major

// shared memory: X hi | X lo (NP / 8 chunks each) | A hi | A lo (16 chunks each; the FP32 parts of A pass through here too) | small
constexpr int kNtSmall = (kNtParts + 1) * kNtRows * 16 + 64;
__host__ __device__ constexpr int nt_smem(int np) { return np * (2 * kNtChunk / 8) + 32 * kNtChunk + kNtSmall; }
static_assert(nt_smem(kNtMaxCols) <= 227 * 1024, "a CTA's shared memory");

__device__ __forceinline__ uint32_t nt_map(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 nt_peer_load(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void nt_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void nt_put(char* hi, char* lo, const uint32_t (&h)[8], const uint32_t (&l)[8]) {
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    *reinterpret_cast<uint4*>(hi + e * kNtChunk) = make_uint4(h[4 * e], h[4 * e + 1], h[4 * e + 2], h[4 * e + 3]);
    *reinterpret_cast<uint4*>(lo + e * kNtChunk) = make_uint4(l[4 * e], l[4 * e + 1], l[4 * e + 2], l[4 * e + 3]);
  }
}
__device__ __forceinline__ void nt_get(const char* hi, const char* lo, float (&x)[16]) {
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const uint4 h4 = *reinterpret_cast<const uint4*>(hi + e * kNtChunk), l4 = *reinterpret_cast<const uint4*>(lo + e * kNtChunk);
    const uint32_t h[4] = {h4.x, h4.y, h4.z, h4.w}, l[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = ns_join(h[i], l[i]);
      x[e * 8 + 2 * i] = v.x;
      x[e * 8 + 2 * i + 1] = v.y;
    }
  }
}

// `np` columns per CTA, `pack` matrices per tile
__global__ void __launch_bounds__(kNtThreads) k_ns_cluster(const NsArgs q, const int np, const int cluster, const int pack) {
  ns_begin(q);
  extern __shared__ __align__(1024) char smem[];
  const int tid = threadIdx.x, warp = warp_of_cta();
  const int row = tid & (kNtRows - 1), part = tid >> 7;          // the tile's row of this thread; which part of the columns
  const uint32_t sb = smem_u32(smem);
  const uint32_t xh = sb, xl = sb + np * (kNtChunk / 8), ah = xl + np * (kNtChunk / 8), al = ah + 16 * kNtChunk;
  char* const pxh = smem + row * 16;                               // this thread's row in the first chunk
  char* const pxl = pxh + np * (kNtChunk / 8);
  char* const pah = pxl + np * (kNtChunk / 8);
  char* const pal = pah + 16 * kNtChunk;
  // [4][128] squares of a row's parts: plain, shrunk, grown | [128] sums of the tile's matrices, read by the cluster's others too
  float4* const s_part = reinterpret_cast<float4*>(smem + np * (2 * kNtChunk / 8) + 32 * kNtChunk);
  float4* const s_sum = s_part + kNtParts * kNtRows;
  // between the norms: [128] the diagonal of A, and [4][128] each the parts' sums of squares of a row of X and of A
  float* const s_diag = reinterpret_cast<float*>(s_sum);
  float* const s_xsq = reinterpret_cast<float*>(s_part);
  float* const s_asq = s_xsq + kNtParts * kNtRows;
  uint32_t* const s_word = reinterpret_cast<uint32_t*>(s_sum + kNtRows);           // mbarrier (two words) | tensor memory | gave up
  const uint32_t bar = smem_u32(s_word);
  uint32_t rank = 0u;
  if (cluster > 1) asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  if (tid == 0) {
    mbar_init(bar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_word[3] = 0u;
  }
  if (warp == 0) tmem_alloc(smem_u32(s_word + 2), kNtTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_word[2];
  const uint32_t trow = tmem + ((uint32_t)((warp & 3) * 32) << 16);
  const uint32_t idesc_a = instr_desc(kNtRows, kNtRows), idesc_x = instr_desc(kNtRows, np) | kNtMnB;
  const int sub = row / q.small, srow = row - sub * q.small;       // matrix of the tile and row in it (sub >= pack: none)
  const int groups = np / 16;                                      // of 16 columns; a thread has part, part + 4, ...
  const int col0 = (int)rank * np;
  uint32_t phase = 0u;
  bool ok = true, late = false;      // ok: the same in all threads behind ready(); late: this warp's last wait gave up
  int products = 0;

  auto wait = [&] {
    if (ok) {
      ok = __all_sync(0xffffffffu, mbar_wait(bar, phase));
      late = !ok;
      if (late) s_word[3] = 1u;
      if (ok) phase ^= 1u;
    }
    tc_fence_after();
  };
  // everyone's operand writes are in place: make them visible to the tensor cores and let one thread go on; tells the CTA of a wait that
  // gave up
  auto ready = [&] {
    fence_async_smem();
    tc_fence_before();
    __syncthreads();
    ok = ok && *const_cast<volatile uint32_t*>(s_word + 3) == 0u;
    tc_fence_after();
  };
  // `steps` pairs of operands that lie `da` and `db` bytes apart: lo hi and hi lo products, then hi hi (the tensor core rounds a sum towards
  // zero with every MMA, so the small ones come first)
  auto product = [&](uint32_t to, uint64_t a_hi, uint64_t a_lo, uint64_t b_hi, uint64_t b_lo, int steps, int da, int db, uint32_t idesc) {
    ++products;
    if (warp == 0 && ok) {
      if (elect_one()) {
        for (int s = 0; s < steps; ++s) {
          const uint64_t oa = (uint64_t)(s * da >> 4), ob = (uint64_t)(s * db >> 4);
          mma_f16(to, a_hi + oa, b_lo + ob, idesc, s > 0);
          mma_f16(to, a_lo + oa, b_hi + ob, idesc, 1u);
        }
        for (int s = 0; s < steps; ++s) mma_f16(to, a_hi + (uint64_t)(s * da >> 4), b_hi + (uint64_t)(s * db >> 4), idesc, 1u);
        if (products != q.withhold || blockIdx.x != 0) mma_commit(bar);
      }
      __syncwarp();
    }
  };

  auto work = [&] {
    const int64_t k = (int64_t)(blockIdx.x / cluster) * pack + sub;
    const bool in = sub < pack && k < q.count && (!q.active || q.active[k]);
    const int64_t base = in ? k * q.stride + (int64_t)srow * q.rs : 0;
    if (!__syncthreads_or(in)) return;         // the same answer in every CTA of a cluster: they hold slices of the same matrices
    // ---- momentum, and the update's values in FP32 in the places of X's pairs (eight to a pair of 16-byte words); sums of squares
    float4 ss = make_float4(0.f, 0.f, 0.f, 0.f);
    auto load = [&](auto width) {
      constexpr int N = decltype(width)::value;
      for (int gr = part; gr < groups; gr += kNtParts) {
        const int c = col0 + gr * 16;
        float u[16];
        NsVec<N> v[16 / N], m[16 / N];
#pragma unroll
        for (int i = 0; i < 16 / N; ++i)
#pragma unroll
          for (int e = 0; e < N; ++e) v[i].v[e] = m[i].v[e] = 0.f;
        auto at = [&](int i) { return base + (N == 4 ? (int64_t)(c + N * i) : (int64_t)(c + i) * q.cs); };
        if (in) {
#pragma unroll
          for (int i = 0; i < 16 / N; ++i)
            if (c + N * i < q.large) {
              v[i] = ns_load<N>(q.g, at(i), q.type);
              if (q.m) m[i] = ns_load<N>(q.m, at(i), MLPSP_PRECISION_F32);
            }
        }
#pragma unroll
        for (int i = 0; i < 16 / N; ++i) {
#pragma unroll
          for (int e = 0; e < N; ++e) {
            float x = v[i].v[e];
            if (q.m) {
              m[i].v[e] = ns_new_momentum(q, x, m[i].v[e]);
              x = ns_update(q, x, m[i].v[e]);
            }
            u[i * N + e] = x;
            const float s = x * kNsShrink, g = x * kNsGrow;
            ss.x = fmaf(x, x, ss.x);
            ss.y = fmaf(s, s, ss.y);
            ss.z = fmaf(g, g, ss.z);
          }
          if (q.m && in && c + N * i < q.large) ns_store<N>(q.m, at(i), MLPSP_PRECISION_F32, m[i]);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          *reinterpret_cast<float4*>(pxh + (gr * 2 + e) * kNtChunk) = make_float4(u[8 * e], u[8 * e + 1], u[8 * e + 2], u[8 * e + 3]);
          *reinterpret_cast<float4*>(pxl + (gr * 2 + e) * kNtChunk) = make_float4(u[8 * e + 4], u[8 * e + 5], u[8 * e + 6], u[8 * e + 7]);
        }
      }
    };
    if (q.vec == 4) load(NsTag<4>{});
    else load(NsTag<1>{});
    s_part[part * kNtRows + row] = ss;
    __syncthreads();
    // a warp adds up a matrix, or every sixteenth
    for (int p = warp; p < pack; p += kNtThreads / 32) {
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int r = p * q.small + (tid & 31); r < (p + 1) * q.small; r += 32)
#pragma unroll
        for (int w = 0; w < kNtParts; ++w) {
          const float4 o = s_part[w * kNtRows + r];
          sum.x += o.x; sum.y += o.y; sum.z += o.z;
        }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        sum.x += __shfl_xor_sync(0xffffffffu, sum.x, o);
        sum.y += __shfl_xor_sync(0xffffffffu, sum.y, o);
        sum.z += __shfl_xor_sync(0xffffffffu, sum.z, o);
      }
      if ((tid & 31) == 0) s_sum[p] = sum;
    }
    if (cluster > 1) nt_cluster_sync();
    else __syncthreads();
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    if (cluster > 1) {
      float4 o[kNtMaxCluster];
#pragma unroll
      for (int r = 0; r < kNtMaxCluster; ++r)
        if (r < cluster) o[r] = nt_peer_load(nt_map(smem_u32(s_sum + min(sub, pack - 1)), r));
#pragma unroll
      for (int r = 0; r < kNtMaxCluster; ++r)
        if (r < cluster) { sum.x += o[r].x; sum.y += o[r].y; sum.z += o[r].z; }
    } else if (sub < pack) {
      sum = s_sum[sub];
    }
    const bool huge = !(sum.x < __int_as_float(0x7f800000)), tiny = sum.x < kNsTinySquares;
    const NsStart start = ns_start(q.eps, huge ? sum.y : tiny ? sum.z : sum.x, huge ? kNsShrink : tiny ? kNsGrow : 1.f);
    const bool lost = start.lost;
    int k2 = start.k;
    // ---- X0 as binary16 pairs, in place
    float xsq = 0.f;
    for (int gr = part; gr < groups; gr += kNtParts) {
      char* const ph = pxh + gr * 2 * kNtChunk;
      char* const pl = pxl + gr * 2 * kNtChunk;
      uint32_t h[8], l[8];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float4 a = *reinterpret_cast<const float4*>(ph + e * kNtChunk), b = *reinterpret_cast<const float4*>(pl + e * kNtChunk);
        const float u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            x[j] = lost ? 0.f : u[2 * i + j] * start.pre * start.inv;
            xsq = fmaf(x[j], x[j], xsq);
          }
          ns_split(x[0], x[1], h[e * 4 + i], l[e * 4 + i]);
        }
      }
      nt_put(ph, pl, h, l);
    }
    __syncthreads();         // the norms' sums have been read
    s_xsq[part * kNtRows + row] = xsq;
    ready();
    for (int it = 0; it < q.steps; ++it) {
      const NsStep by = ns_step(q, k2);
      // ---- A = X X^T
      {
        const uint64_t dh = smem_desc(xh, kNtChunk, 128), dl = smem_desc(xl, kNtChunk, 128);
        product(tmem, dh, dl, dh, dl, groups, 2 * kNtChunk, 2 * kNtChunk, idesc_a);
      }
      // The diagonals of A and A^2, sums of squares of rows, are taken from FP32 sums: the tensor core's, rounded towards zero with every
      // MMA, are all too small by a few 1e-7, and the iteration carries that on (4e-6 of the result for 128 rows)
      float xx = 0.f;
#pragma unroll
      for (int w = 0; w < kNtParts; ++w) xx += s_xsq[w * kNtRows + row];
      wait();
      if (cluster == 1) {
        for (int gr = part; gr < 8; gr += kNtParts) {
          uint32_t d[16], h[8], l[8];
          tmem_ld16(trow + gr * 16, d);
          const int off = gr * 16 - row;       // column less row
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float v[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int c = 2 * e + i;
              v[i] = (off + c == 0 ? xx : __uint_as_float(d[c])) * by.gram;
              if ((unsigned)(off + c + srow) >= (unsigned)q.small) v[i] = 0.f;
            }
            ns_split(v[0], v[1], h[e], l[e]);
          }
          nt_put(pah + gr * 2 * kNtChunk, pal + gr * 2 * kNtChunk, h, l);
        }
      } else {
        // the slices' parts of A: 32 pieces of [128 rows][4 columns] in FP32, each added up by one CTA and handed to all
        for (int gr = part; gr < 8; gr += kNtParts) {
          uint32_t d[16];
          tmem_ld16(trow + gr * 16, d);
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (gr * 16 + e == row) d[e] = __float_as_uint(xx);
          if (!ok)
#pragma unroll
            for (int e = 0; e < 16; ++e) d[e] = 0x7fffffffu;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *reinterpret_cast<uint4*>(pah + (gr * 4 + e) * kNtChunk) = make_uint4(d[4 * e], d[4 * e + 1], d[4 * e + 2], d[4 * e + 3]);
        }
        nt_cluster_sync();
        // this thread: row `row` of piece `part` of the groups that fall to this CTA, in place (no other reads them here)
        for (int gr = (int)rank; gr < 8; gr += cluster) {
          const uint32_t at = ah + (uint32_t)((gr * 4 + part) * kNtChunk + row * 16);
          float4 o[kNtMaxCluster];
#pragma unroll
          for (int r = 0; r < kNtMaxCluster; ++r)
            if (r < cluster) o[r] = nt_peer_load(nt_map(at, r));
          float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int r = 0; r < kNtMaxCluster; ++r)
            if (r < cluster) { t.x += o[r].x; t.y += o[r].y; t.z += o[r].z; t.w += o[r].w; }
          *reinterpret_cast<float4*>(pah + (gr * 4 + part) * kNtChunk) = t;
        }
        nt_cluster_sync();
        // ... and everyone fetches the sums from their owners.  (Handing them out with remote stores took 12 of 24 us an iteration.)
        float4 t[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int gr = part + j * kNtParts;
          const uint32_t at = nt_map(ah + (uint32_t)(gr * 4 * kNtChunk + row * 16), (uint32_t)(gr % cluster));
#pragma unroll
          for (int e = 0; e < 4; ++e) t[j][e] = nt_peer_load(at + e * kNtChunk);
        }
        nt_cluster_sync();
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int gr = part + j * kNtParts;
          const int first = gr * 16 - row + srow;       // column of the first value in this row's block of A
          uint32_t h[8], l[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float a[4] = {t[j][e].x, t[j][e].y, t[j][e].z, t[j][e].w};
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = (unsigned)(first + 4 * e + i) < (unsigned)q.small ? a[i] * by.gram : 0.f;
            ns_split(v[0], v[1], h[2 * e], l[2 * e]);
            ns_split(v[2], v[3], h[2 * e + 1], l[2 * e + 1]);
          }
          nt_put(pah + gr * 2 * kNtChunk, pal + gr * 2 * kNtChunk, h, l);
        }
      }
      ready();
      // ---- A^2
      {
        const uint64_t dh = smem_desc(ah, kNtChunk, 128), dl = smem_desc(al, kNtChunk, 128);
        product(tmem + kNtRows, dh, dl, dh, dl, 8, 2 * kNtChunk, 2 * kNtChunk, idesc_a);
      }
      wait();
      // ---- P = b A + c A^2 but for its diagonal, which is kept apart (muon_warp.cu)
      float asq = 0.f;
      for (int gr = part; gr < 8; gr += kNtParts) {
        uint32_t d[16], h[8], l[8];
        float a[16];
        tmem_ld16(trow + kNtRows + gr * 16, d);
        nt_get(pah + gr * 2 * kNtChunk, pal + gr * 2 * kNtChunk, a);
        const int off = row - gr * 16;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float p[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int c = 2 * e + i;
            asq = fmaf(a[c], a[c], asq);
            p[i] = fmaf(by.b, a[c], by.c * __uint_as_float(d[c]));
            if (off == c) { s_diag[row] = a[c]; p[i] = 0.f; }
          }
          ns_split(p[0], p[1], h[e], l[e]);
        }
        nt_put(pah + gr * 2 * kNtChunk, pal + gr * 2 * kNtChunk, h, l);
      }
      s_asq[part * kNtRows + row] = asq;
      ready();
      // ---- P X, over the accumulators that have been read
      product(tmem, smem_desc(ah, kNtChunk, 128), smem_desc(al, kNtChunk, 128), smem_desc(xh, 128, kNtChunk), smem_desc(xl, 128, kNtChunk), 8,
              2 * kNtChunk, 256, idesc_x);
      const bool last = it + 1 == q.steps;
      float own = by.b * s_diag[row] + by.a;
#pragma unroll
      for (int w = 0; w < kNtParts; ++w) own = fmaf(by.c, s_asq[w * kNtRows + row], own);
      xsq = 0.f;
      wait();
      if (last) ok = __syncthreads_and(ok) != 0;
      const bool write = last && in;
      for (int gr = part; gr < groups; gr += kNtParts) {
        char* const ph = pxh + gr * 2 * kNtChunk;
        char* const pl = pxl + gr * 2 * kNtChunk;
        uint32_t d[16], h[8], l[8];
        float v[16];
        const int c = col0 + gr * 16;
        NsVec<4> w[4];
        const bool stepping = write && q.m && q.vec == 4;
        if (stepping) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (c + 4 * e < q.large) w[e] = ns_load<4>(q.w, base + c + 4 * e, MLPSP_PRECISION_F32);
        }
        tmem_ld16(trow + gr * 16, d);
        nt_get(ph, pl, v);
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = fmaf(own, v[e], __uint_as_float(d[e]));
        if (!last) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            xsq = fmaf(v[2 * e], v[2 * e], fmaf(v[2 * e + 1], v[2 * e + 1], xsq));
            ns_split(v[2 * e], v[2 * e + 1], h[e], l[e]);
          }
          nt_put(ph, pl, h, l);
        }
        if (!write) continue;
        const float fin = lost || !ok ? __int_as_float(0x7fffffff) : ns_exp2i(-10 - k2);
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] *= fin;
        if (q.vec == 4) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (c + 4 * e < q.large) {
              NsVec<4> r;
#pragma unroll
              for (int i = 0; i < 4; ++i) r.v[i] = q.m ? fmaf(-q.step, v[4 * e + i], q.keep * w[e].v[i]) : v[4 * e + i];
              if (q.m) ns_store<4>(q.w, base + c + 4 * e, MLPSP_PRECISION_F32, r);
              else ns_store<4>(q.out, base + c + 4 * e, q.type, r);
            }
        } else {
          float u[16];
          if (q.m)
#pragma unroll
            for (int e = 0; e < 16; ++e) u[e] = c + e < q.large ? q.w[base + (int64_t)(c + e) * q.cs] : 0.f;
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (c + e < q.large) {
              const int64_t at = base + (int64_t)(c + e) * q.cs;
              if (q.m) q.w[at] = fmaf(-q.step, v[e], q.keep * u[e]);
              else ns_store<1>(q.out, at, q.type, NsVec<1>{{v[e]}});
            }
        }
      }
      s_xsq[part * kNtRows + row] = xsq;
      ready();
    }
  };
  work();
  if (!ok && q.gave_up) *q.gave_up = 1;
  if (late) mbar_wait(bar, phase);
  __syncthreads();
  if (warp == 0) tmem_free(tmem, kNtTmemCols);
  if (cluster > 1) nt_cluster_sync();      // no CTA leaves while another may read its shared memory
  ns_end(q);
}

// CTAs that share a matrix.  With few matrices slices of about 128 columns, since the exchange costs as much as the products it spreads; with
// more than fit the GPU at once, and up to 256 columns, as few CTAs as hold a matrix: one of 128 x 512 66 us in four and 81 in two, forty
// 137 and 84; one of 128 x 144 56 us in two and 45 in one.  (Four fifths of the SMs: clusters of eight leave the odd ones of a GPC, fewer than
// sixteen fit; sixteen of 128 x 1152 152 us in eight CTAs each, eighteen 93 in five.)  A cluster per tile, not a loop over tiles in as many
// clusters as there are SMs for: those that did not fit waited for a whole loop, 400 of 128 x 2048 4,182 us instead of 2,529.
static int nt_cluster(const NsArgs& q) {
  const int64_t pack = kNtRows / q.small, tiles = (q.count + pack - 1) / pack;
  const int narrow = std::min(kNtMaxCluster, (q.large + 127) / 128), wide = (q.large + kNtMaxCols - 1) / kNtMaxCols;
  return wide > 1 && tiles * narrow <= sm_count() * 4 / 5 ? narrow : wide;
}
// the kernel for `count` matrices (the rule: at kNsWarpFew)
enum NsKernel { kNsWarp, kNsPair, kNsCluster };
static NsKernel ns_kernel(int64_t count, int small, int large) {
  const int64_t pack = kNtRows / small;
  // more tiles than clusters on the GPU
  const bool many = (count + pack - 1) / pack * ((large + kNtMaxCols - 1) / kNtMaxCols) > sm_count();
  if (small <= kNsWarpRows) return large <= kNsWarpFew || (large <= kNsWarpLong[small > 16] && many) ? kNsWarp : kNsCluster;
  if (small <= kNsPairRows) return large <= kNsPairFew || (large <= kNsPairLong && many) ? kNsPair : kNsCluster;
  return kNsCluster;
}
// whether the kernel is the one with bounded waits
static bool ns_waits(int64_t count, int rows, int cols) {
  return count > 0 && ns_kernel(count, std::min(rows, cols), std::max(rows, cols)) == kNsCluster;
}

int launch_ns_cluster(const NsArgs& q, cudaStream_t st, bool launch) {
  const int cluster = nt_cluster(q);
  const int np = ((q.large + cluster - 1) / cluster + 15) / 16 * 16;
  const int pack = kNtRows / q.small;
  const int64_t tiles = (q.count + pack - 1) / pack;
  const int smem = nt_smem(np);
  MLPSP_SHARED_MEMORY(nt_smem(kNtMaxCols), (const void*)k_ns_cluster);
  MLPSP_REQUIRE(tiles * cluster < (1ll << 31), MLPSP_E_LIMIT, "orthogonalize: too many matrices");
  if (!launch) return MLPSP_OK;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * cluster));
  cfg.blockDim = dim3(kNtThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  LaunchScope scope(kKMisc, 1, st);
  return cuda_check(cudaLaunchKernelEx(&cfg, k_ns_cluster, q, np, cluster, pack), "orthogonalize");
}

// Whether the iteration stays in the binary16 range of the scaled operands: from singular values in [0, 1], values within [-4, 4] and
// |b s^2 + c s^4| within 32 after every step.  Both polynomials take their extremes over [0, top] at the ends or where their
// derivatives vanish, quadratics in s^2: that of a s + b s^3 + c s^5 has the roots q / (5 c) and a / q, neither a difference of near numbers.
static bool ns_bounded(double a, double b, double c, int steps) {
  double top = 1.0;
  for (int it = 0; it < steps; ++it) {
    double next = 0.0;
    const double disc = 9.0 * b * b - 20.0 * a * c, q = -0.5 * (3.0 * b + std::copysign(disc > 0.0 ? std::sqrt(disc) : 0.0, b));
    const double at[] = {top * top, c != 0.0 ? -b / (2.0 * c) : 0.0, c != 0.0 ? q / (5.0 * c) : 0.0, q != 0.0 ? a / q : 0.0};
    for (double s2 : at) {
      s2 = s2 > 0.0 && s2 < top * top ? s2 : top * top;
      const double p = b * s2 + c * s2 * s2, y = (a + p) * std::sqrt(s2);
      if (!(p >= -32.0 && p <= 32.0 && y >= -4.0 && y <= 4.0)) return false;
      next = std::max(next, std::fabs(y));
    }
    top = std::max(next, 1e-30) * 1.001;
  }
  return true;
}

// what the two entries share; stage: how far to go
enum NsStage { kNsCheck, kNsPrepare, kNsLaunch };
static int ns_launch(const char* who, NsArgs& q, int64_t n, int32_t rows, int32_t cols, int32_t steps, double a, double b, double c,
                     double eps, cudaStream_t st, NsStage stage) {
  MLPSP_REQUIRE(n >= 0 && rows >= 1 && cols >= 1, MLPSP_E_ARG, "%s: bad sizes", who);
  MLPSP_REQUIRE(std::min(rows, cols) <= MLPSP_MUON_MAX_SMALL && std::max(rows, cols) <= MLPSP_MUON_MAX_LARGE, MLPSP_E_LIMIT,
                "%s: %d x %d matrices; at most %d on the smaller and %d on the larger side", who, rows, cols, MLPSP_MUON_MAX_SMALL,
                MLPSP_MUON_MAX_LARGE);
  MLPSP_REQUIRE(q.type == MLPSP_PRECISION_F32 || q.type == MLPSP_PRECISION_F16 || q.type == MLPSP_PRECISION_BF16, MLPSP_E_ARG,
                "%s: unknown element type %d", who, q.type);
  MLPSP_REQUIRE(steps >= 1 && steps <= 32, MLPSP_E_ARG, "%s: steps must be 1..32", who);
  MLPSP_REQUIRE(eps >= 1e-15 && eps <= 1.0, MLPSP_E_ARG, "%s: eps must be within [1e-15, 1]", who);
  MLPSP_REQUIRE(ns_bounded(a, b, c, steps), MLPSP_E_ARG, "%s: singular values leave [0, 4] with these coefficients", who);
  if (n == 0) return MLPSP_OK;
  MLPSP_REQUIRE(q.g && (q.m ? q.w != nullptr : q.out != nullptr), MLPSP_E_ARG, "%s: null pointer", who);
  MLPSP_REQUIRE(aligned_to(q.type == MLPSP_PRECISION_F32 ? 4 : 2, {q.g, q.out}) && aligned_to(4, {q.m, q.w}), MLPSP_E_ARG,
                "%s: a pointer is not aligned to its elements", who);
  if (stage == kNsCheck) return MLPSP_OK;
  const bool tall = rows > cols;
  q.count = n;
  q.stride = (int64_t)rows * cols;
  q.small = tall ? cols : rows;
  q.large = tall ? rows : cols;
  q.rs = tall ? 1 : cols;
  q.cs = tall ? cols : 1;
  q.steps = steps;
  q.a = (float)a; q.b = (float)b; q.c = (float)c; q.eps = (float)eps;
  auto bits = [&](double x) { int k = 0; while (std::ldexp(1.0, k) < x) ++k; return k; };
  q.near = bits(std::fabs(a) + std::fabs(b) / 4 + std::fabs(c) / 16);
  q.far = bits(std::fabs(a) + std::fabs(b) / 256 + std::fabs(c) / 65536);
  q.vec = 1;
  const uintptr_t wide = reinterpret_cast<uintptr_t>(q.m) | reinterpret_cast<uintptr_t>(q.w);
  const uintptr_t typed = reinterpret_cast<uintptr_t>(q.g) | reinterpret_cast<uintptr_t>(q.out);
  const int size = q.type == MLPSP_PRECISION_F32 ? 4 : 2;
  if (!tall)
    for (int v = 2; v <= 4; v *= 2)
      if (cols % v == 0 && wide % (4 * v) == 0 && typed % (size * v) == 0) q.vec = v;
  const NsKernel kernel = ns_kernel(q.count, q.small, q.large);
  return (kernel == kNsWarp ? launch_ns_warp : kernel == kNsPair ? launch_ns_pair : launch_ns_cluster)(q, st, stage == kNsLaunch);
}

}  // namespace mlpsp

using namespace mlpsp;

namespace mlpsp {
static thread_local int32_t g_withhold = 0;

// the answer of a call's waits, for which the call waits, if it has any
struct NsAnswer {
  int32_t* to;
  HostWords& hw;
  cudaEvent_t ev = nullptr;
  explicit NsAnswer(int32_t* host) : to(host), hw(host_words()) {}
  int open(NsArgs& q, bool waits) {
    if (!to) return MLPSP_OK;
    *to = 0;
    if (!waits) return MLPSP_OK;
    const int rc = hw.open(&ev);
    if (rc) return rc;
    hw.word[0] = 0;
    q.gave_up = static_cast<volatile int32_t*>(hw.word);
    return MLPSP_OK;
  }
  // also behind a launch that failed: the kernels before it still write the word
  int read(cudaStream_t st) {
    if (!ev) return MLPSP_OK;
    MLPSP_CUDA_OK(cudaEventRecord(ev, st));
    MLPSP_CUDA_OK(cudaEventSynchronize(ev));
    *to = *static_cast<volatile int32_t*>(hw.word);
    return MLPSP_OK;
  }
};
}  // namespace mlpsp

extern "C" int mlpsp_test_withhold_answer(int32_t product) {
  MLPSP_REQUIRE(product >= 0, MLPSP_E_ARG, "mlpsp_test_withhold_answer: product must not be negative");
  g_withhold = product;
  return MLPSP_OK;
}

extern "C" int mlpsp_orthogonalize_waits(int32_t rows, int32_t cols) {
  const int small = std::min(rows, cols), large = std::max(rows, cols);
  return small > kNsPairRows || large > (small <= kNsWarpRows ? kNsWarpFew : kNsPairFew) ? 1 : 0;
}

extern "C" int mlpsp_orthogonalize_stack_waits(int64_t n, int32_t rows, int32_t cols) {
  const bool sizes = rows >= 1 && cols >= 1 && std::min(rows, cols) <= MLPSP_MUON_MAX_SMALL && std::max(rows, cols) <= MLPSP_MUON_MAX_LARGE;
  return sizes && ns_waits(n, rows, cols) ? 1 : 0;
}

extern "C" int mlpsp_orthogonalize(const void* update, int32_t dtype, int64_t n, int32_t rows, int32_t cols, int32_t steps, double a,
                                   double b, double c, double eps, void* out, int32_t* gave_up_host, void* stream) {
  NsArgs q = {};
  q.g = update;
  q.out = out;
  q.type = dtype;
  q.withhold = g_withhold;
  NsAnswer answer(gave_up_host);
  int rc = ns_launch("mlpsp_orthogonalize", q, n, rows, cols, steps, a, b, c, eps, (cudaStream_t)stream, kNsCheck);
  if (!rc) rc = answer.open(q, ns_waits(n, rows, cols));
  if (!rc) rc = ns_launch("mlpsp_orthogonalize", q, n, rows, cols, steps, a, b, c, eps, (cudaStream_t)stream, kNsLaunch);
  return rc ? rc : answer.read((cudaStream_t)stream);
}

extern "C" int mlpsp_muon_step(const mlpsp_muon_tensor* tensors, int32_t count, const uint8_t* active, double lr, double momentum,
                               int32_t nesterov, double weight_decay, int32_t steps, double a, double b, double c, double eps,
                               int32_t* gave_up_host, void* stream) {
  MLPSP_REQUIRE(count >= 0 && (count == 0 || tensors), MLPSP_E_ARG, "mlpsp_muon_step: null pointer");
  MLPSP_REQUIRE(momentum >= 0.0 && momentum < 1.0, MLPSP_E_ARG, "mlpsp_muon_step: momentum must be within [0, 1)");
  MLPSP_REQUIRE(lr >= 0.0 && lr < 1e30 && weight_decay >= 0.0 && weight_decay < 1e30, MLPSP_E_ARG,
                "mlpsp_muon_step: lr and weight_decay must be finite and not negative");
  NsAnswer answer(gave_up_host);
  // all tensors are checked, and their kernels allowed the shared memory that they take, before the first launch
  bool waits = false;
  for (const NsStage stage : {kNsCheck, kNsPrepare, kNsLaunch}) {
    bool follows = false;
    NsArgs shared = {};
    if (stage == kNsLaunch) {
      const int rc = answer.open(shared, waits);
      if (rc) return rc;
    }
    for (int32_t i = 0; i < count; ++i) {
      const mlpsp_muon_tensor& t = tensors[i];
      MLPSP_REQUIRE(t.n <= 0 || (t.weights && t.grads && t.momenta), MLPSP_E_ARG, "mlpsp_muon_step: null pointer");
      MLPSP_REQUIRE(!active || t.n == tensors[0].n, MLPSP_E_ARG, "mlpsp_muon_step: with active, all tensors must have as many matrices");
      MLPSP_REQUIRE(t.scale > 0.0 && t.scale < 1e30, MLPSP_E_ARG, "mlpsp_muon_step: scale must be finite and positive");
      NsArgs q = shared;
      q.g = t.grads;
      q.m = t.momenta;
      q.w = t.weights;
      q.active = active;
      q.type = t.grad_dtype;
      q.withhold = g_withhold;
      q.nesterov = nesterov != 0;
      q.momentum = (float)momentum;
      q.rest = (float)(1.0 - momentum);
      q.keep = (float)(1.0 - lr * weight_decay);
      q.step = (float)(lr * t.scale);
      q.follows = follows;
      const int rc = ns_launch("mlpsp_muon_step", q, t.n, t.rows, t.cols, steps, a, b, c, eps, (cudaStream_t)stream, stage);
      if (rc) {
        if (follows) answer.read((cudaStream_t)stream);
        return rc;
      }
      waits |= ns_waits(t.n, t.rows, t.cols);
      follows |= t.n > 0;
    }
  }
  return answer.read((cudaStream_t)stream);
}
