// The places of records among the records grouped by primitive: slots[r], a stable counting sort that moves no rows and whose result is the
// inverse of the usual permutation.
//
// Least significant digit first, nine bits a pass: one pass for up to 511 primitives, two up to 262,143 (mlpsp_group_records takes digits of
// at most eight, evenly split).  A CTA owns 4,096 records in a row, a warp 256 of them.  Per pass: counts of every digit and CTA; their
// exclusive prefix over the CTAs, a CTA per digit; and the placement, in which a warp ranks its records with match.any against its own
// counters.  Passes before the last reorder (key, record) in shared memory and write runs.  The last one only needs each record's place:
// it is written straight from registers (to slots[record]: in order if there was one pass, else scattered), and the sorted keys behind it
// when there is more than one digit, for the offsets, which are found by binary search inside the range of their highest digit.
// Up to 65,536 records of up to 511 primitives take one launch of a cluster of eight CTAs.
//
// Bound: latency of the ranking (sixteen warps a CTA, three CTAs per SM; passes of six bits with sixteen warps per SM took 95 us each for
// 7.8 M records) and, in the last pass of several, the scattered words.  7.8 M records of 100,000 primitives: 330 -> 177 us, of which the
// placements take 59 and 74; 32,764 of 256: 35 -> 10 us.
#include "frame.cuh"

namespace mlpsp {

constexpr int kRsBits = 9, kRsBins = 1 << kRsBits, kRsThreads = kRsBins, kRsWarps = kRsThreads / 32;
constexpr int kRsRounds = 8, kRsItems = kRsThreads * kRsRounds, kRsItemBytes = kRsItems * (int)sizeof(uint2);

// an id outside [0, nprim) sorts behind every primitive, as key nprim
template <bool FIRST>
__device__ __forceinline__ uint32_t rs_key(uint32_t k, int nprim) { return FIRST && k >= (uint32_t)nprim ? (uint32_t)nprim : k; }

// counts[digit * nblocks + block]
template <bool FIRST>
__global__ void __launch_bounds__(kRsThreads) k_rs_count(const uint32_t* __restrict__ keys, int64_t n, int nprim, int shift, uint32_t mask,
                                                         int nblocks, int32_t* __restrict__ counts) {
  chain_wait();
  chain_release();
  __shared__ int h[kRsBins];
  h[threadIdx.x] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kRsItems;
  if ((reinterpret_cast<uintptr_t>(keys) & 15) == 0 && base + kRsItems <= n) {
    uint4 k[kRsRounds / 4];
#pragma unroll
    for (int r = 0; r < kRsRounds / 4; ++r) k[r] = __ldg(reinterpret_cast<const uint4*>(keys + base) + r * kRsThreads + threadIdx.x);
#pragma unroll
    for (int r = 0; r < kRsRounds / 4; ++r) {
      atomicAdd(&h[(rs_key<FIRST>(k[r].x, nprim) >> shift) & mask], 1);
      atomicAdd(&h[(rs_key<FIRST>(k[r].y, nprim) >> shift) & mask], 1);
      atomicAdd(&h[(rs_key<FIRST>(k[r].z, nprim) >> shift) & mask], 1);
      atomicAdd(&h[(rs_key<FIRST>(k[r].w, nprim) >> shift) & mask], 1);
    }
  } else {
    for (int r = 0; r < kRsRounds; ++r) {
      const int64_t i = base + r * kRsThreads + threadIdx.x;
      if (i < n) atomicAdd(&h[(rs_key<FIRST>(__ldg(keys + i), nprim) >> shift) & mask], 1);
    }
  }
  __syncthreads();
  if (threadIdx.x <= mask) counts[(size_t)threadIdx.x * nblocks + blockIdx.x] = h[threadIdx.x];
}

// block = one digit: exclusive prefix of its counts over the blocks, in place, and its total
__global__ void __launch_bounds__(kRsThreads) k_rs_scan(int nblocks, int32_t* __restrict__ counts, int32_t* __restrict__ totals) {
  chain_wait();
  chain_release();
  __shared__ int warp_sums[32];
  int32_t* row = counts + (size_t)blockIdx.x * nblocks;
  int run = 0;
  for (int b0 = 0; b0 < nblocks; b0 += kRsThreads * 4) {
    int v[4], mine = 0, total;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int b = b0 + threadIdx.x * 4 + e;
      v[e] = b < nblocks ? row[b] : 0;
      mine += v[e];
    }
    int ex = run + block_exclusive_scan(mine, warp_sums, total);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int b = b0 + threadIdx.x * 4 + e;
      if (b < nblocks) row[b] = ex;
      ex += v[e];
    }
    run += total;
    __syncthreads();
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = run;
}

// ranks of a warp's records, round by round, among those of the same digit before them; cnt: the warp's counters, zero at first.
// left: records from this lane's first on (a record every 32).
template <int ROUNDS>
__device__ __forceinline__ void rs_rank(const uint32_t (&key)[ROUNDS], int64_t left, int rounds, int shift, uint32_t mask, uint16_t* cnt, uint32_t lt,
                                        int (&rank)[ROUNDS]) {
  uint32_t peers[ROUNDS];      // all of them before the counters' chain begins
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r)
    if (r < rounds) peers[r] = __match_any_sync(0xffffffffu, r * 32 < left ? (key[r] >> shift) & mask : 0x1000u);
  __syncwarp();
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r)
    if (r < rounds) {
      const bool valid = r * 32 < left;
      const uint32_t d = (key[r] >> shift) & mask;
      const int before = valid ? cnt[d] : 0;
      rank[r] = before + __popc(peers[r] & lt);
      __syncwarp();
      if (valid && (peers[r] & lt) == 0u) cnt[d] = (uint16_t)(before + __popc(peers[r]));
      __syncwarp();
    }
}

// FIRST: the values are the positions.  LAST: slots[value] = place, instead of values in their places; offsets (only where a digit is the
// whole key): the first places of all digits, by block 0.
template <bool FIRST, bool LAST>
__global__ void __launch_bounds__(kRsThreads, 3) k_rs_place(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ vals, int64_t n, int nprim,
                                                            int shift, uint32_t mask, int nblocks, const int32_t* __restrict__ counts,
                                                            const int32_t* __restrict__ totals, uint32_t* __restrict__ keys_out,
                                                            uint32_t* __restrict__ vals_out, int32_t* __restrict__ slots,
                                                            int64_t* __restrict__ offsets, int32_t* __restrict__ starts) {
  chain_wait();
  chain_release();
  __shared__ uint16_t s_cnt[kRsWarps][kRsBins];   // running digit counts per warp, then the first position of a warp's items of a digit
  __shared__ int s_dst[kRsBins];                  // global place of the block's first item of a digit, minus its position here
  extern __shared__ __align__(16) uint2 s_item[];  // [kRsItems], not LAST
  __shared__ int warp_sums[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t base = (int64_t)blockIdx.x * kRsItems + warp * (kRsRounds * 32) + lane;
  const uint32_t lt = (1u << lane) - 1u;
  for (int i = lane; i < kRsBins / 2; i += 32) reinterpret_cast<uint32_t*>(s_cnt[warp])[i] = 0u;
  uint32_t key[kRsRounds];
  int rank[kRsRounds];
#pragma unroll
  for (int r = 0; r < kRsRounds; ++r) key[r] = base + r * 32 < n ? rs_key<FIRST>(__ldg(keys + base + r * 32), nprim) : 0xffffffffu;
  // of this thread's digit, on their way while the records are ranked
  const bool live = (uint32_t)tid <= mask;
  const int total_of = live ? __ldg(totals + tid) : 0;
  const int before_us = live ? __ldg(counts + (size_t)tid * nblocks + blockIdx.x) : 0;
  rs_rank<kRsRounds>(key, n - base, kRsRounds, shift, mask, s_cnt[warp], lt, rank);
  __syncthreads();
  // thread = digit: the warps' first positions inside the digit, the digit's first position in the block and its first place of all
  int mine = 0;
#pragma unroll
  for (int w = 0; w < kRsWarps; ++w) { const int c = s_cnt[w][tid]; s_cnt[w][tid] = (uint16_t)mine; mine += c; }
  int total, unused;
  const int global = block_exclusive_scan(total_of, warp_sums, unused);
  __syncthreads();
  if (LAST) {
    s_dst[tid] = global + before_us;
    if (blockIdx.x == 0) {
      if (offsets) for (int i = tid; i <= nprim; i += kRsThreads) offsets[i] = global;       // nprim < kRsBins: one each
      else if (live) starts[tid] = global;
    }
  } else {
    const int local = block_exclusive_scan(mine, warp_sums, total);
    s_dst[tid] = global + before_us - local;
#pragma unroll
    for (int w = 0; w < kRsWarps; ++w) s_cnt[w][tid] = (uint16_t)(s_cnt[w][tid] + local);
  }
  __syncthreads();
  if (LAST) {
#pragma unroll
    for (int r = 0; r < kRsRounds; ++r) {
      const int64_t i = base + r * 32;
      if (i >= n) continue;
      const uint32_t d = (key[r] >> shift) & mask;
      const int dst = s_dst[d] + s_cnt[warp][d] + rank[r];
      slots[FIRST ? (uint32_t)i : __ldg(vals + i)] = dst;
      if (!offsets) keys_out[dst] = key[r];
    }
    return;
  }
#pragma unroll
  for (int r = 0; r < kRsRounds; ++r) {
    const int64_t i = base + r * 32;
    if (i < n) s_item[s_cnt[warp][(key[r] >> shift) & mask] + rank[r]] = make_uint2(key[r], FIRST ? (uint32_t)i : __ldg(vals + i));
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRsRounds; ++r) {
    const int j = r * kRsThreads + tid;
    if (j < total) {
      const uint2 it = s_item[j];
      const int dst = s_dst[(it.x >> shift) & mask] + j;
      keys_out[dst] = it.x;
      vals_out[dst] = it.y;
    }
  }
}

// The whole of it for few records and primitives in one launch of one cluster: the CTAs' counts pass through distributed shared memory.
constexpr int kRsClusterCtas = 8, kRsClusterRounds = 16;
constexpr int64_t kRsClusterRecords = (int64_t)kRsClusterCtas * kRsThreads * kRsClusterRounds;
__global__ void __cluster_dims__(kRsClusterCtas, 1, 1) __launch_bounds__(kRsThreads) k_rs_cluster(const uint32_t* __restrict__ ids, int n, int nprim,
                                                                                              int rounds, int32_t* __restrict__ slots,
                                                                                              int64_t* __restrict__ offsets) {
  chain_wait();
  chain_release();
  __shared__ uint16_t s_cnt[kRsWarps][kRsBins];
  __shared__ int s_total[kRsBins];
  __shared__ int s_dst[kRsBins];
  __shared__ int warp_sums[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank_of = blockIdx.x;
  const int base = (rank_of * kRsWarps + warp) * rounds * 32 + lane;
  for (int i = lane; i < kRsBins / 2; i += 32) reinterpret_cast<uint32_t*>(s_cnt[warp])[i] = 0u;
  uint32_t key[kRsClusterRounds];
  int rank[kRsClusterRounds];
#pragma unroll
  for (int r = 0; r < kRsClusterRounds; ++r)
    if (r < rounds) key[r] = base + r * 32 < n ? rs_key<true>(__ldg(ids + base + r * 32), nprim) : 0xffffffffu;
  rs_rank<kRsClusterRounds>(key, n - base, rounds, 0, kRsBins - 1, s_cnt[warp], (1u << lane) - 1u, rank);
  __syncthreads();
  int mine = 0;
#pragma unroll
  for (int w = 0; w < kRsWarps; ++w) { const int c = s_cnt[w][tid]; s_cnt[w][tid] = (uint16_t)mine; mine += c; }
  s_total[tid] = mine;
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(s_total + tid);
  int others[kRsClusterCtas], all = 0, before_us = 0, unused;
#pragma unroll
  for (int c = 0; c < kRsClusterCtas; ++c) {
    uint32_t peer;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(at), "r"(c));
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(others[c]) : "r"(peer) : "memory");
  }
#pragma unroll
  for (int c = 0; c < kRsClusterCtas; ++c) {
    all += others[c];
    if (c < rank_of) before_us += others[c];
  }
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");      // this CTA has read what it wanted of the others
  const int global = block_exclusive_scan(all, warp_sums, unused);
  s_dst[tid] = global + before_us;
  if (rank_of == 0 && tid <= nprim) offsets[tid] = global;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRsClusterRounds; ++r)
    if (r < rounds && base + r * 32 < n) slots[base + r * 32] = s_dst[key[r]] + s_cnt[warp][key[r]] + rank[r];
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");        // no CTA leaves while another may read its counts
}

// first position of every primitive in the sorted keys; starts: the first positions of the highest digits
__global__ void __launch_bounds__(256) k_rs_offsets(const uint32_t* __restrict__ keys, int64_t n, int nprim, int shift, uint32_t mask,
                                                    const int32_t* __restrict__ starts, int64_t* __restrict__ offsets) {
  chain_wait();
  chain_release();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i > nprim) return;
  const uint32_t d = (uint32_t)i >> shift;
  int64_t lo = __ldg(starts + d), hi = d < mask ? __ldg(starts + d + 1) : n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (__ldg(keys + mid) < (uint32_t)i) lo = mid + 1; else hi = mid;
  }
  offsets[i] = lo;
}

// bit 0: the pixel offsets do not start at zero, end at the record count or ascend
__global__ void k_route_check(const int64_t* __restrict__ offsets, int64_t pixels, int64_t records, volatile int32_t* __restrict__ found) {
  chain_wait();
  chain_release();
  const int64_t stride = (int64_t)gridDim.x * blockDim.x;
  bool bad = false;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i <= pixels; i += stride) {
    const int64_t o = __ldg(offsets + i);
    bad |= i == 0 ? o != 0 : o < __ldg(offsets + i - 1);
    bad |= i == pixels && o != records;
  }
  if (bad) *found = MLPSP_ROUTE_BAD_OFFSETS;
}

struct RsPlan { int passes, bits, nblocks; };
static RsPlan rs_plan(int64_t R, int n) {
  int bits = 1;
  while (bits < 31 && (1ll << bits) <= (int64_t)n) ++bits;      // keys 0 .. n
  RsPlan p;
  p.passes = (bits + kRsBits - 1) / kRsBits;
  p.bits = (bits + p.passes - 1) / p.passes;
  p.nblocks = (int)((R + kRsItems - 1) / kRsItems);
  return p;
}
// scratch: digit totals | first places | block counts | keys and values of the passes before the last, keys of the last
struct RsLayout { int64_t totals, starts, counts, key[2], val[2], bytes; };
static bool rs_in_a_cluster(int64_t R, int n) { return n < kRsBins && R <= kRsClusterRecords; }
static RsLayout rs_layout(int64_t R, int n) {
  const RsPlan p = rs_plan(R, n);
  RsLayout L = {};
  if (rs_in_a_cluster(R, n)) return L;
  int64_t off = 0;
  auto take = [&](int64_t bytes) { const int64_t o = off; off += align_up(bytes, 256); return o; };
  L.totals = take(4 * kRsBins);
  L.starts = take(4 * kRsBins);
  L.counts = take(4ll * kRsBins * std::max(p.nblocks, 1));
  for (int i = 0; i < 2; ++i) L.key[i] = p.passes > 1 ? take(4 * R) : off;
  for (int i = 0; i < 2; ++i) L.val[i] = p.passes > 1 + i ? take(4 * R) : off;
  L.bytes = off;
  return L;
}

}  // namespace mlpsp

using namespace mlpsp;

extern "C" int64_t mlpsp_route_records_scratch_bytes(int64_t num_records, int32_t n) {
  if (num_records < 0 || n < 0) return -1;
  return rs_layout(num_records, n).bytes;
}

extern "C" int mlpsp_route_records(const int32_t* primitive_ids, int64_t num_records, int32_t n, const int64_t* pixel_offsets, int64_t pixels,
                                   int64_t* offsets, int32_t* slots, void* scratch, int64_t scratch_bytes, int32_t* findings_host, void* stream) {
  const char* who = "mlpsp_route_records";
  const int64_t R = num_records;
  MLPSP_REQUIRE(R >= 0 && n >= 0 && offsets, MLPSP_E_ARG, "%s: bad arguments", who);
  MLPSP_REQUIRE(R < (1ll << 31) && n < 2147483647, MLPSP_E_LIMIT, "%s: more than 2^31-1 records or primitives", who);
  MLPSP_REQUIRE(R == 0 || (primitive_ids && slots), MLPSP_E_ARG, "%s: null pointer", who);
  MLPSP_REQUIRE(!findings_host || (pixel_offsets && pixels >= 0), MLPSP_E_ARG, "%s: no pixel offsets to check", who);
  MLPSP_REQUIRE(aligned_to(4, {primitive_ids, slots, scratch}) && aligned_to(8, {offsets, pixel_offsets}), MLPSP_E_ARG,
                "%s: a pointer is not aligned to its elements", who);
  const RsLayout L = rs_layout(R, n);
  MLPSP_REQUIRE(L.bytes == 0 || (scratch && scratch_bytes >= L.bytes), MLPSP_E_SCRATCH, "%s: scratch needs %lld bytes", who, (long long)L.bytes);
  cudaStream_t st = (cudaStream_t)stream;
  MLPSP_SHARED_MEMORY(kRsItemBytes, (const void*)k_rs_place<true, false>, (const void*)k_rs_place<false, false>);
  HostWords& hw = host_words();
  cudaEvent_t ev = nullptr;
  if (findings_host) {
    const int rc = hw.open(&ev);
    if (rc) return rc;
    hw.word[0] = 0;
    LaunchScope scope(kKMisc, 1, st);
    launch_chained(k_route_check, dim3((unsigned)std::min<int64_t>(sm_count() * 8, pixels / 1024 + 1)), dim3(256), 0, st, pixel_offsets, pixels, R,
                   static_cast<volatile int32_t*>(hw.word));
    MLPSP_CUDA_OK(cudaEventRecord(ev, st));
  }
  if (R == 0) {
    MLPSP_CUDA_OK(cudaMemsetAsync(offsets, 0, 8 * ((size_t)n + 1), st));
  } else if (rs_in_a_cluster(R, n)) {
    LaunchScope scope(kKMisc, 1, st);
    constexpr int per_round = kRsClusterCtas * kRsThreads;
    launch_chained(k_rs_cluster, dim3(kRsClusterCtas), dim3(kRsThreads), 0, st, reinterpret_cast<const uint32_t*>(primitive_ids), (int)R, n,
                   (int)((R + per_round - 1) / per_round), slots, offsets);
    MLPSP_CUDA_OK(cudaGetLastError());
  } else {
    const RsPlan p = rs_plan(R, n);
    LaunchScope scope(kKMisc, 3 * p.passes + (p.passes > 1), st);
    char* b = (char*)scratch;
    int32_t* totals = (int32_t*)(b + L.totals);
    int32_t* starts = (int32_t*)(b + L.starts);
    int32_t* counts = (int32_t*)(b + L.counts);
    const uint32_t* k_in = reinterpret_cast<const uint32_t*>(primitive_ids);
    const uint32_t* v_in = nullptr;
    const uint32_t mask = (1u << p.bits) - 1u;
    int shift = 0;
    for (int pass = 0; pass < p.passes; ++pass, shift += p.bits) {
      const bool first = pass == 0, last = pass == p.passes - 1;
      uint32_t* k_out = (uint32_t*)(b + L.key[pass & 1]);
      uint32_t* v_out = (uint32_t*)(b + L.val[pass & 1]);
      launch_chained(first ? k_rs_count<true> : k_rs_count<false>, dim3(p.nblocks), dim3(kRsThreads), 0, st, k_in, R, n, shift, mask, p.nblocks, counts);
      launch_chained(k_rs_scan, dim3(mask + 1), dim3(kRsThreads), 0, st, p.nblocks, counts, totals);
      auto* place = first ? (last ? k_rs_place<true, true> : k_rs_place<true, false>) : (last ? k_rs_place<false, true> : k_rs_place<false, false>);
      const int smem = last ? 0 : kRsItemBytes;
      launch_chained(place, dim3(p.nblocks), dim3(kRsThreads), smem, st, k_in, v_in, R, n, shift, mask, p.nblocks, counts, totals, k_out, v_out, slots,
                     p.passes == 1 ? offsets : nullptr, starts);
      k_in = k_out;
      v_in = v_out;
    }
    if (p.passes > 1)
      launch_chained(k_rs_offsets, dim3((unsigned)(((int64_t)n + 256) / 256)), dim3(256), 0, st, k_in, R, n, shift - p.bits, mask, starts, offsets);
    MLPSP_CUDA_OK(cudaGetLastError());
  }
  if (findings_host) {
    MLPSP_CUDA_OK(cudaEventSynchronize(ev));
    *findings_host = *static_cast<volatile int32_t*>(hw.word);
  }
  return MLPSP_OK;
}
