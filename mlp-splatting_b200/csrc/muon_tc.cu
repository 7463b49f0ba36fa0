// Newton-Schulz iteration of matrices up to 128 x 2048 on the 5th-generation tensor cores (tcgen05), and the C entries of both kernels.
//
// A CTA holds a slice of X, 128 rows by up to 256 columns, in shared memory as binary16 pairs, in chunks of [128 rows][8 columns].
// The same bytes are the K-major operands of A = X X^T and, read MN-major, the B operand of (bA + cA^2) X.  A matrix of more columns
// than one slice is spread over a cluster of up to eight CTAs, which add their parts of A through distributed shared memory; A^2 is
// computed by each.  Narrow matrices of few rows are stacked (two of 64 rows): the blocks of A off their diagonal are cleared, after
// which everything stays block-diagonal.  Accumulators (A | A^2, later the new slice in the same columns) are in tensor memory.
//
// Every wait on an mbarrier is bounded; one that gives up raises MLPSP_ST_TIMEOUT and this CTA's slice of the result is not written.
#include <cmath>
#include "muon.cuh"

namespace mlpsp {

constexpr int kNtThreads = 256, kNtRows = 128, kNtChunk = kNtRows * 16;
constexpr int kNtMaxCols = 256, kNtMaxCluster = 8;
constexpr int kNtTmemCols = 256;
constexpr uint32_t kNtMnB = 1u << 16;      // bit 16 of the instruction descriptor: B is MN-major

// shared memory: X hi | X lo (NP / 8 chunks each) | A hi | A lo (16 chunks each; the FP32 parts of A pass through here too) | small
constexpr int kNtSmall = 2 * kNtRows * 16 + 16 + 64;
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
__device__ __forceinline__ void nt_peer_store2(uint32_t addr, uint32_t a, uint32_t b) {
  asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(addr), "r"(a), "r"(b) : "memory");
}
__device__ __forceinline__ void nt_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void nt_fence_async() { asm volatile("fence.proxy.async;" ::: "memory"); }

// `np` columns per CTA, `pack` matrices per tile (1 in a cluster)
__global__ void __launch_bounds__(kNtThreads) k_ns_cluster(const NsArgs q, const int np, const int cluster, const int pack, const int64_t tiles) {
  chain_wait();
  chain_release();
  extern __shared__ __align__(1024) char smem[];
  const int tid = threadIdx.x, warp = warp_of_cta();
  const int row = tid & (kNtRows - 1), half = tid >> 7;          // the tile's row of this thread; which half of the columns
  const uint32_t sb = smem_u32(smem);
  const uint32_t xh = sb, xl = sb + np * (kNtChunk / 8), ah = xl + np * (kNtChunk / 8), al = ah + 16 * kNtChunk;
  char* const pxh = smem;
  char* const pxl = smem + np * (kNtChunk / 8);
  char* const pah = pxl + np * (kNtChunk / 8);
  char* const pal = pah + 16 * kNtChunk;
  float4* const s_part = reinterpret_cast<float4*>(pal + 16 * kNtChunk);      // [2][128] squares of a row's halves: plain, shrunk, grown
  // between the norms: [128] the diagonal of bA + cA^2, and [2][128] each the halves' sums of squares of a row of X and of A
  float* const s_diag = reinterpret_cast<float*>(s_part);
  float* const s_xsq = s_diag + kNtRows;
  float* const s_asq = s_xsq + 2 * kNtRows;
  float4* const s_rank = s_part + 2 * kNtRows;                               // this CTA's sums, read by the cluster's others
  uint32_t* const s_word = reinterpret_cast<uint32_t*>(s_rank + 1);           // mbarrier (two words) | tensor memory | gave up
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
  const int groups = np / 16;
  const int col0 = (int)rank * np;
  uint32_t phase = 0u;
  bool ok = true;

  auto wait = [&] {
    if (ok && !mbar_wait(bar, phase)) ok = false;      // after one that gave up the others are not waited for
    phase ^= 1u;
    tc_fence_after();
  };
  // everyone's operand writes are in place: make them visible to the tensor cores and let one thread go on
  auto ready = [&] {
    fence_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
  };

  for (int64_t tile = blockIdx.x / cluster; tile < tiles; tile += gridDim.x / cluster) {
    const int64_t k = tile * pack + sub;
    const bool in = sub < pack && k < q.count && (!q.active || q.active[k]);
    const int64_t base = in ? k * q.stride + (int64_t)srow * q.rs : 0;
    if (!__syncthreads_or(in)) continue;         // the same answer in every CTA of a cluster: it holds one matrix
    // ---- pass one: momentum, sums of squares.  Each thread has the groups of 16 columns half, half + 2, ... of its row.
    float4 ss = make_float4(0.f, 0.f, 0.f, 0.f);
    auto square = [&](float u) {
      const float s = u * kNsShrink, g = u * kNsGrow;
      ss.x = fmaf(u, u, ss.x);
      ss.y = fmaf(s, s, ss.y);
      ss.z = fmaf(g, g, ss.z);
    };
    auto fetch = [&](int64_t at, auto n, bool first) {
      constexpr int N = decltype(n)::value;
      NsVec<N> v = ns_load<N>(q.g, at, q.type);
      if (q.m) {
        NsVec<N> m = ns_load<N>(q.m, at, MLPSP_PRECISION_F32);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          if (first) m.v[e] = ns_new_momentum(q, v.v[e], m.v[e]);
          v.v[e] = ns_update(q, v.v[e], m.v[e]);
        }
        if (first) ns_store<N>(q.m, at, MLPSP_PRECISION_F32, m);
      }
      return v;
    };
    for (int gr = half; gr < groups; gr += 2) {
      const int c = col0 + gr * 16;
      if (!in) break;
      if (q.vec == 4) {
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          if (c + e < q.large) {
            const NsVec<4> v = fetch(base + c + e, NsTag<4>{}, true);
#pragma unroll
            for (int i = 0; i < 4; ++i) square(v.v[i]);
          }
      } else {
        for (int e = 0; e < 16; ++e)
          if (c + e < q.large) square(fetch(base + (int64_t)(c + e) * q.cs, NsTag<1>{}, true).v[0]);
      }
    }
    s_part[half * kNtRows + row] = ss;
    __syncthreads();
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](const float4& o) { sum.x += o.x; sum.y += o.y; sum.z += o.z; };
    if (sub < pack)
      for (int r = sub * q.small; r < (sub + 1) * q.small; ++r) {
        add(s_part[r]);
        add(s_part[kNtRows + r]);
      }
    if (cluster > 1) {
      if (tid == 0) *s_rank = sum;
      nt_cluster_sync();
      sum = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int r = 0; r < cluster; ++r) add(nt_peer_load(nt_map(smem_u32(s_rank), r)));
      nt_cluster_sync();
    }
    const bool huge = !(sum.x < __int_as_float(0x7f800000)), tiny = sum.x < kNsTinySquares;
    const NsStart start = ns_start(q.eps, huge ? sum.y : tiny ? sum.z : sum.x, huge ? kNsShrink : tiny ? kNsGrow : 1.f);
    const bool lost = start.lost;
    int k2 = start.k;
    // ---- pass two: X0 as binary16 pairs
    __syncthreads();         // the norms' sums have been read
    float xsq = 0.f;
    for (int gr = half; gr < groups; gr += 2) {
      const int c = col0 + gr * 16;
      float u[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) u[e] = 0.f;
      if (in && !lost) {
        if (q.vec == 4) {
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            if (c + e < q.large) {
              const NsVec<4> v = fetch(base + c + e, NsTag<4>{}, false);
#pragma unroll
              for (int i = 0; i < 4; ++i) u[e + i] = v.v[i] * start.pre * start.inv;
            }
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (c + e < q.large) u[e] = fetch(base + (int64_t)(c + e) * q.cs, NsTag<1>{}, false).v[0] * start.pre * start.inv;
        }
      }
      uint32_t h[8], l[8];
#pragma unroll
      for (int e = 0; e < 16; ++e) xsq = fmaf(u[e], u[e], xsq);
#pragma unroll
      for (int e = 0; e < 8; ++e) ns_split(u[2 * e], u[2 * e + 1], h[e], l[e]);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        *reinterpret_cast<uint4*>(pxh + (gr * 2 + e) * kNtChunk + row * 16) = make_uint4(h[4 * e], h[4 * e + 1], h[4 * e + 2], h[4 * e + 3]);
        *reinterpret_cast<uint4*>(pxl + (gr * 2 + e) * kNtChunk + row * 16) = make_uint4(l[4 * e], l[4 * e + 1], l[4 * e + 2], l[4 * e + 3]);
      }
    }
    s_xsq[half * kNtRows + row] = xsq;
    ready();
    for (int it = 0; it < q.steps; ++it) {
      const NsStep by = ns_step(q, k2);
      // ---- A = X X^T
      if (warp == 0) {
        if (elect_one()) {
          const uint64_t dh = smem_desc(xh, kNtChunk, 128), dl = smem_desc(xl, kNtChunk, 128);
          // the small products first: the tensor core rounds a sum towards zero with every MMA
          for (int s = 0; s < groups; ++s) {
            const uint64_t o = (uint64_t)(s * 2 * kNtChunk >> 4);
            mma_f16(tmem, dh + o, dl + o, idesc_a, s > 0);
            mma_f16(tmem, dl + o, dh + o, idesc_a, 1u);
          }
          for (int s = 0; s < groups; ++s) {
            const uint64_t o = (uint64_t)(s * 2 * kNtChunk >> 4);
            mma_f16(tmem, dh + o, dh + o, idesc_a, 1u);
          }
          mma_commit(bar);
        }
        __syncwarp();
      }
      wait();
      // The diagonals of A and A^2, sums of squares of rows, are taken from FP32 sums: the tensor core's, rounded towards zero with every
      // MMA, are all too small by a few 1e-7, and the iteration carries that on (4e-6 of the result for 128 rows)
      const float xx = s_xsq[row] + s_xsq[kNtRows + row];
      float asq = 0.f;
      if (cluster == 1) {
        for (int gr = half; gr < 8; gr += 2) {
          uint32_t d[16], h[8], l[8];
          tmem_ld16(trow + gr * 16, d);
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (gr * 16 + e == row) d[e] = __float_as_uint(xx);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float v[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int c = gr * 16 + 2 * e + i;
              v[i] = (unsigned)(c - sub * q.small) < (unsigned)q.small ? __uint_as_float(d[2 * e + i]) * by.gram : 0.f;
            }
            asq = fmaf(v[0], v[0], fmaf(v[1], v[1], asq));
            ns_split(v[0], v[1], h[e], l[e]);
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            *reinterpret_cast<uint4*>(pah + (gr * 2 + e) * kNtChunk + row * 16) = make_uint4(h[4 * e], h[4 * e + 1], h[4 * e + 2], h[4 * e + 3]);
            *reinterpret_cast<uint4*>(pal + (gr * 2 + e) * kNtChunk + row * 16) = make_uint4(l[4 * e], l[4 * e + 1], l[4 * e + 2], l[4 * e + 3]);
          }
        }
      } else {
        // the slices' parts of A: 32 pieces of [128 rows][4 columns] in FP32, each added up by one CTA and handed to all
        for (int gr = half; gr < 8; gr += 2) {
          uint32_t d[16];
          tmem_ld16(trow + gr * 16, d);
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (gr * 16 + e == row) d[e] = __float_as_uint(xx);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *reinterpret_cast<uint4*>(pah + (gr * 4 + e) * kNtChunk + row * 16) = make_uint4(d[4 * e], d[4 * e + 1], d[4 * e + 2], d[4 * e + 3]);
        }
        nt_cluster_sync();
        float4 t[8];
        // unit u = (piece, row): of the 16 rounds of 256 units this CTA takes rank, rank + cluster, ...
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int round = j * cluster + (int)rank;
          t[j] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (round < 16) {
            const uint32_t at = ah + (uint32_t)(round * kNtThreads + tid) * 16;
            for (int r = 0; r < cluster; ++r) {
              const float4 o = nt_peer_load(nt_map(at, r));
              t[j].x += o.x; t[j].y += o.y; t[j].z += o.z; t[j].w += o.w;
            }
          }
        }
        nt_cluster_sync();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int round = j * cluster + (int)rank;
          if (round < 16) {
            const int u = round * kNtThreads + tid, piece = u >> 7, r0 = u & (kNtRows - 1);
            uint32_t h[2], l[2];
            ns_split(t[j].x * by.gram, t[j].y * by.gram, h[0], l[0]);
            ns_split(t[j].z * by.gram, t[j].w * by.gram, h[1], l[1]);
            const uint32_t at = (uint32_t)((piece >> 1) * kNtChunk + r0 * 16 + (piece & 1) * 8);
            for (int r = 0; r < cluster; ++r) {
              nt_peer_store2(nt_map(ah + at, r), h[0], h[1]);
              nt_peer_store2(nt_map(al + at, r), l[0], l[1]);
            }
          }
        }
        nt_fence_async();
        nt_cluster_sync();
        for (int gr = half; gr < 8; gr += 2)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint4 h4 = *reinterpret_cast<const uint4*>(pah + (gr * 2 + e) * kNtChunk + row * 16);
            const uint4 l4 = *reinterpret_cast<const uint4*>(pal + (gr * 2 + e) * kNtChunk + row * 16);
            const uint32_t h[4] = {h4.x, h4.y, h4.z, h4.w}, l[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) { const float2 a = ns_join(h[i], l[i]); asq = fmaf(a.x, a.x, fmaf(a.y, a.y, asq)); }
          }
      }
      s_asq[half * kNtRows + row] = asq;
      ready();
      // ---- A^2
      if (warp == 0) {
        if (elect_one()) {
          const uint64_t dh = smem_desc(ah, kNtChunk, 128), dl = smem_desc(al, kNtChunk, 128);
          for (int s = 0; s < 8; ++s) {
            const uint64_t o = (uint64_t)(s * 2 * kNtChunk >> 4);
            mma_f16(tmem + kNtRows, dh + o, dl + o, idesc_a, s > 0);
            mma_f16(tmem + kNtRows, dl + o, dh + o, idesc_a, 1u);
          }
          for (int s = 0; s < 8; ++s) {
            const uint64_t o = (uint64_t)(s * 2 * kNtChunk >> 4);
            mma_f16(tmem + kNtRows, dh + o, dh + o, idesc_a, 1u);
          }
          mma_commit(bar);
        }
        __syncwarp();
      }
      wait();
      const float aa = s_asq[row] + s_asq[kNtRows + row];
      for (int gr = half; gr < 8; gr += 2) {
        uint32_t d[16];
        tmem_ld16(trow + kNtRows + gr * 16, d);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (gr * 16 + e == row) d[e] = __float_as_uint(aa);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint4* const sh = reinterpret_cast<uint4*>(pah + (gr * 2 + e) * kNtChunk + row * 16);
          uint4* const sl = reinterpret_cast<uint4*>(pal + (gr * 2 + e) * kNtChunk + row * 16);
          const uint4 h4 = *sh, l4 = *sl;
          uint32_t h[4] = {h4.x, h4.y, h4.z, h4.w}, l[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 a = ns_join(h[i], l[i]);
            float p0 = fmaf(by.b, a.x, by.c * __uint_as_float(d[e * 8 + 2 * i])), p1 = fmaf(by.b, a.y, by.c * __uint_as_float(d[e * 8 + 2 * i + 1]));
            const int c = gr * 16 + e * 8 + 2 * i;
            if (c == (row & ~1)) {       // the diagonal is kept apart (muon_warp.cu)
              s_diag[row] = row & 1 ? p1 : p0;
              if (row & 1) p1 = 0.f; else p0 = 0.f;
            }
            ns_split(p0, p1, h[i], l[i]);
          }
          *sh = make_uint4(h[0], h[1], h[2], h[3]);
          *sl = make_uint4(l[0], l[1], l[2], l[3]);
        }
      }
      ready();
      // ---- (bA + cA^2) X, over the accumulators that have been read
      if (warp == 0) {
        if (elect_one()) {
          const uint64_t ph = smem_desc(ah, kNtChunk, 128), pl = smem_desc(al, kNtChunk, 128);
          const uint64_t dh = smem_desc(xh, 128, kNtChunk), dl = smem_desc(xl, 128, kNtChunk);
          for (int s = 0; s < 8; ++s) {
            const uint64_t o = (uint64_t)(s * 2 * kNtChunk >> 4), n = (uint64_t)(s * 256 >> 4);
            mma_f16(tmem, ph + o, dl + n, idesc_x, s > 0);
            mma_f16(tmem, pl + o, dh + n, idesc_x, 1u);
          }
          for (int s = 0; s < 8; ++s) {
            const uint64_t o = (uint64_t)(s * 2 * kNtChunk >> 4), n = (uint64_t)(s * 256 >> 4);
            mma_f16(tmem, ph + o, dh + n, idesc_x, 1u);
          }
          mma_commit(bar);
        }
        __syncwarp();
      }
      wait();
      const bool last = it + 1 == q.steps;
      const float own = by.a + s_diag[row];
      xsq = 0.f;
      if (last && !ok) atomicOr(s_word + 3, 1u);
      if (last) __syncthreads();
      const bool write = last && in && s_word[3] == 0u;
      for (int gr = half; gr < groups; gr += 2) {
        uint32_t d[16];
        tmem_ld16(trow + gr * 16, d);
        float v[16];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint4* const sh = reinterpret_cast<uint4*>(pxh + (gr * 2 + e) * kNtChunk + row * 16);
          uint4* const sl = reinterpret_cast<uint4*>(pxl + (gr * 2 + e) * kNtChunk + row * 16);
          const uint4 h4 = *sh, l4 = *sl;
          uint32_t h[4] = {h4.x, h4.y, h4.z, h4.w}, l[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 x = ns_join(h[i], l[i]);
            v[e * 8 + 2 * i] = fmaf(own, x.x, __uint_as_float(d[e * 8 + 2 * i]));
            v[e * 8 + 2 * i + 1] = fmaf(own, x.y, __uint_as_float(d[e * 8 + 2 * i + 1]));
            xsq = fmaf(v[e * 8 + 2 * i], v[e * 8 + 2 * i], fmaf(v[e * 8 + 2 * i + 1], v[e * 8 + 2 * i + 1], xsq));
            ns_split(v[e * 8 + 2 * i], v[e * 8 + 2 * i + 1], h[i], l[i]);
          }
          if (!last) {
            *sh = make_uint4(h[0], h[1], h[2], h[3]);
            *sl = make_uint4(l[0], l[1], l[2], l[3]);
          }
        }
        if (!write) continue;
        const int c = col0 + gr * 16;
        const float nan = __int_as_float(0x7fffffff), fin = ns_exp2i(-10 - k2);
        if (q.vec == 4) {
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            if (c + e < q.large) {
              NsVec<4> r;
#pragma unroll
              for (int i = 0; i < 4; ++i) r.v[i] = lost ? nan : v[e + i] * fin;
              if (q.m) {
                const NsVec<4> w = ns_load<4>(q.w, base + c + e, MLPSP_PRECISION_F32);
#pragma unroll
                for (int i = 0; i < 4; ++i) r.v[i] = fmaf(-q.step, r.v[i], q.keep * w.v[i]);
                ns_store<4>(q.w, base + c + e, MLPSP_PRECISION_F32, r);
              } else ns_store<4>(q.out, base + c + e, q.type, r);
            }
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (c + e < q.large) {
              const int64_t at = base + (int64_t)(c + e) * q.cs;
              const float r = lost ? nan : v[e] * fin;
              if (q.m) q.w[at] = fmaf(-q.step, r, q.keep * q.w[at]);
              else ns_store<1>(q.out, at, q.type, NsVec<1>{{r}});
            }
        }
      }
      s_xsq[half * kNtRows + row] = xsq;
      ready();
    }
  }
  if (!ok && q.status) atomicOr(q.status + MLPSP_ST_BITS, MLPSP_ST_TIMEOUT);
  __syncthreads();
  if (warp == 0) tmem_free(tmem, kNtTmemCols);
  if (cluster > 1) nt_cluster_sync();      // no CTA leaves while another may read its shared memory
}

int launch_ns_cluster(const NsArgs& q, cudaStream_t st) {
  // columns per CTA: slices of at least 64 (below, the exchange costs more than the products it spreads), at most 256
  const int cluster = std::min(kNtMaxCluster, std::max(1, (q.large + 127) / 128));
  const int np = ((q.large + cluster - 1) / cluster + 15) / 16 * 16;
  const int pack = cluster == 1 ? kNtRows / q.small : 1;
  const int64_t tiles = (q.count + pack - 1) / pack;
  const int smem = nt_smem(np);
  static DeviceOnce once;
  if (once.first()) MLPSP_CUDA_OK(cudaFuncSetAttribute(k_ns_cluster, cudaFuncAttributeMaxDynamicSharedMemorySize, nt_smem(kNtMaxCols)));
  const int resident = std::max(1, std::min(2, 227 * 1024 / (smem + 1024)));
  const int64_t most = std::max<int64_t>(1, (int64_t)sm_count() * resident / cluster);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(std::min(tiles, most) * cluster));
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
  return cuda_check(cudaLaunchKernelEx(&cfg, k_ns_cluster, q, np, cluster, pack, tiles), "orthogonalize");
}

// Whether the iteration stays in the binary16 range of the scaled operands: from singular values in [0, 1], values within [-4, 4] and
// |b s^2 + c s^4| within 32 after every step.  Both polynomials take their extremes over [0, top] at the ends or where their
// derivatives vanish, quadratics in s^2.
static bool ns_bounded(double a, double b, double c, int steps) {
  double top = 1.0;
  for (int it = 0; it < steps; ++it) {
    double next = 0.0;
    const double disc = 9.0 * b * b - 20.0 * a * c, root = disc > 0.0 ? std::sqrt(disc) : 0.0;
    const double at[] = {top * top, c != 0.0 ? -b / (2.0 * c) : 0.0, c != 0.0 ? (-3.0 * b + root) / (10.0 * c) : b != 0.0 ? -a / (3.0 * b) : 0.0,
                         c != 0.0 ? (-3.0 * b - root) / (10.0 * c) : 0.0};
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

// what the two entries share
static int ns_launch(const char* who, NsArgs& q, int64_t n, int32_t rows, int32_t cols, int32_t steps, double a, double b, double c,
                     double eps, cudaStream_t st) {
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
  return q.small <= kNsWarpRows && q.large <= kNsWarpCols ? launch_ns_warp(q, st) : launch_ns_cluster(q, st);
}

}  // namespace mlpsp

using namespace mlpsp;

extern "C" int mlpsp_orthogonalize_waits(int32_t rows, int32_t cols) {
  return std::min(rows, cols) > kNsWarpRows || std::max(rows, cols) > kNsWarpCols ? 1 : 0;
}

extern "C" int mlpsp_orthogonalize(const void* update, int32_t dtype, int64_t n, int32_t rows, int32_t cols, int32_t steps, double a,
                                   double b, double c, double eps, void* out, int32_t* status, void* stream) {
  NsArgs q = {};
  q.g = update;
  q.out = out;
  q.type = dtype;
  q.status = status;
  return ns_launch("mlpsp_orthogonalize", q, n, rows, cols, steps, a, b, c, eps, (cudaStream_t)stream);
}

extern "C" int mlpsp_muon_step(float* weights, const void* grads, int32_t grad_dtype, float* momenta, const uint8_t* active, int64_t n,
                               int32_t rows, int32_t cols, double lr, double momentum, int32_t nesterov, double weight_decay, double scale,
                               int32_t steps, double a, double b, double c, double eps, int32_t* status, void* stream) {
  MLPSP_REQUIRE(n <= 0 || (weights && grads && momenta), MLPSP_E_ARG, "mlpsp_muon_step: null pointer");
  MLPSP_REQUIRE(momentum >= 0.0 && momentum < 1.0, MLPSP_E_ARG, "mlpsp_muon_step: momentum must be within [0, 1)");
  MLPSP_REQUIRE(lr >= 0.0 && lr < 1e30 && weight_decay >= 0.0 && weight_decay < 1e30 && scale > 0.0 && scale < 1e30, MLPSP_E_ARG,
                "mlpsp_muon_step: lr, weight_decay and scale must be finite and not negative");
  NsArgs q = {};
  q.g = grads;
  q.m = momenta;
  q.w = weights;
  q.active = active;
  q.type = grad_dtype;
  q.status = status;
  q.nesterov = nesterov != 0;
  q.momentum = (float)momentum;
  q.rest = (float)(1.0 - momentum);
  q.keep = (float)(1.0 - lr * weight_decay);
  q.step = (float)(lr * scale);
  return ns_launch("mlpsp_muon_step", q, n, rows, cols, steps, a, b, c, eps, (cudaStream_t)stream);
}
