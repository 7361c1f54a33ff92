// Plan of a batch for the bucketed matrix products: rows grouped by bucket (a stable counting sort), the first place of
// every bucket, and the list of tiles of at most 128 rows of one bucket that the products walk.
//
// Mathematics: place(p) = #{q : b(q) < b(p)} + #{q < p : b(q) = b(p)}.  A warp takes 32 consecutive rows at a time, so
// the second term is a histogram of the rows before its slice plus the lanes below it that hold the same bucket
// (one match instruction).  Work: ids read twice (three times in the form for long batches), order written once; bound by
// latency up to about a million rows.
//
// Three forms, all with a counter per warp and bucket in shared memory, blocks of 1024 threads:
//   up to   2048 rows  one block                                                          (2048 rows, 8 buckets: 10 us)
//   up to  65536 rows  one cluster of eight blocks, which read one another's counters     (16384 rows: 12 us; one block 20)
//   beyond             counters per block of 4096 rows, their scan, the fill: three launches, about 20 us of latency together
//                      (65536 rows of 64 buckets: 24 us either way; 262143 of 256: 34, the cluster 64)
#include "grouped.cuh"
#include "tc.cuh"

namespace nnue {

constexpr int kGpThreads = 1024;
constexpr int kGpWarps = kGpThreads / 32;
constexpr int kAhead = 4;  // ids per lane in flight
constexpr int64_t kSingleRows = 2048;
constexpr int64_t kClusterRows = 65536;
constexpr int kClusterSize = 8;
constexpr int kBlockRows = 4096;  // rows per block of the long form

// bin of a row: its bucket, or E for -1 (padding row) and, with a note in the status word, for an id out of range
template <typename Id>
__device__ __forceinline__ int group_bin(const Id* bucket, int64_t p, int E, unsigned long long* status) {
    const Id b = bucket[p];
    if (b >= 0 && b < (Id)E) return (int)b;
    if (b != (Id)-1 && status) note_bad_index(status);
    return E;
}

// counters of each warp's slice of rows [lo, hi): hist[warp][bin]
template <typename Id>
__device__ __forceinline__ void group_histogram(const Id* bucket, int64_t lo, int64_t hi, int bins, int32_t* hist,
                                                unsigned long long* status) {
    for (int i = threadIdx.x; i < bins * kGpWarps; i += kGpThreads) hist[i] = 0;
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t per = (hi - lo + kGpWarps * 32 - 1) / (kGpWarps * 32) * 32;
    const int64_t a = lo + warp * per, b = min(hi, a + per);
    for (int64_t p0 = a + lane; p0 < b; p0 += 32 * kAhead) {
        int bin[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) bin[u] = p0 + 32 * u < b ? group_bin(bucket, p0 + 32 * u, bins - 1, status) : -1;
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (bin[u] >= 0) atomicAdd(hist + warp * bins + bin[u], 1);
    }
    __syncthreads();
}

// hist[w][bin] becomes the number of rows of `bin` in the slices before w; returns the bin's total
__device__ __forceinline__ int group_scan_warps(int32_t* hist, int bins, int bin) {
    int run = 0;
#pragma unroll 8
    for (int w = 0; w < kGpWarps; ++w) {
        const int v = hist[w * bins + bin];
        hist[w * bins + bin] = run;
        run += v;
    }
    return run;
}

// rows of this block to their places: base[bin] + hist[warp][bin] + rank among the warp's 32
template <typename Id>
__device__ __forceinline__ void group_fill(const Id* bucket, int64_t lo, int64_t hi, int bins, int32_t* hist,
                                           const int32_t* base, int32_t* order) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t per = (hi - lo + kGpWarps * 32 - 1) / (kGpWarps * 32) * 32;
    const int64_t a = lo + warp * per, b = min(hi, a + per);
    int32_t* mine = hist + warp * bins;
    for (int64_t p0 = a; p0 < b; p0 += 32 * kAhead) {
        int bins_of[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int64_t p = p0 + 32 * u + lane;
            bins_of[u] = p < b ? group_bin(bucket, p, bins - 1, nullptr) : -1;
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (p0 + 32 * u >= b) break;
            const int bin = bins_of[u];
            const unsigned same = __match_any_sync(kFullMask, bin);
            const int rank = __popc(same & ((1u << lane) - 1u));
            int at = 0;
            if (bin >= 0) at = mine[bin];
            __syncwarp();
            if (bin >= 0) {
                order[base[bin] + at + rank] = (int32_t)(p0 + 32 * u + lane);
                if (rank == 0) mine[bin] = at + __popc(same);
            }
            __syncwarp();
        }
    }
}

// exclusive scan over the block of four values per thread; the totals go to `total`
__device__ __forceinline__ int4 add4(int4 a, int4 b) { return make_int4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }
__device__ __forceinline__ int4 warp_scan4(int4 v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int4 u = make_int4(__shfl_up_sync(kFullMask, v.x, d), __shfl_up_sync(kFullMask, v.y, d),
                                 __shfl_up_sync(kFullMask, v.z, d), __shfl_up_sync(kFullMask, v.w, d));
        if (lane >= d) v = add4(v, u);
    }
    return v;
}
__device__ __forceinline__ int4 block_scan4(int4 v, int4* s_warp, int4* total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int4 inc = warp_scan4(v);
    __syncthreads();
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    if (warp == 0) s_warp[lane] = warp_scan4(s_warp[lane]);
    __syncthreads();
    const int4 before = warp ? s_warp[warp - 1] : make_int4(0, 0, 0, 0);
    *total = s_warp[kGpWarps - 1];
    return make_int4(before.x + inc.x - v.x, before.y + inc.y - v.y, before.z + inc.z - v.z, before.w + inc.w - v.w);
}

// Totals of the bins (s_total) to the plan's offsets, places and tile lists, shared out over `ranks` CTAs.  s_at[bin] = first place in the order, first
// tile, first pair, first place among rows laid out by bucket.
__device__ __forceinline__ void group_tiles(int64_t T, int E, const int32_t* s_total, int4* s_at, int4* s_warp, int32_t* plan,
                                            int rank = 0, int ranks = 1) {
    const int bins = E + 1;
    int4 carry = make_int4(0, 0, 0, 0);
    for (int b0 = 0; b0 < bins; b0 += kGpThreads) {
        const int b = b0 + threadIdx.x;
        const int n = b < bins ? s_total[b] : 0;
        int4 total;
        const int4 mine = make_int4(n, (n + kGroupRows - 1) / kGroupRows, (n + kGroupPairRows - 1) / kGroupPairRows,
                                    b < E ? (n + kGroupAlign - 1) / kGroupAlign * kGroupAlign : 0);
        const int4 at = add4(carry, block_scan4(mine, s_warp, &total));
        if (b < bins) {
            s_at[b] = at;
            if (rank == 0) {
                plan[group_offsets_at() + b] = at.x;
                plan[group_places_at(T, E) + b] = at.w;
                plan[group_first_at(T, E) + b] = at.y;
            }
        }
        carry = add4(carry, total);
    }
    if (threadIdx.x == 0) {
        s_at[bins] = carry;
        if (rank == 0) {
            plan[0] = carry.y;
            plan[1] = carry.z;
            plan[group_offsets_at() + bins] = (int32_t)T;
        }
    }
    __syncthreads();
    for (int pairs = 0; pairs < 2; ++pairs) {
        int4* tiles = reinterpret_cast<int4*>(plan + (pairs ? group_pairs_at(T, E) : group_tiles_at(T, E)));
        const int rows = pairs ? kGroupPairRows : kGroupRows;
        for (int t = rank * kGpThreads + threadIdx.x; t < (pairs ? carry.z : carry.y); t += ranks * kGpThreads) {
            int lo = 0, hi = bins - 1;  // the last bin whose first tile is not behind t; empty bins share a first tile
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if ((pairs ? s_at[mid].z : s_at[mid].y) <= t) lo = mid;
                else hi = mid - 1;
            }
            const int4 b = s_at[lo];
            const int in = (t - (pairs ? b.z : b.y)) * rows;
            tiles[t] = make_int4(lo, b.x + in, min(rows, s_total[lo] - in), b.w + in);
        }
    }
}

// shared memory: s_at [bins + 1] int4, counters per warp [bins][kGpWarps] (not in the scan), and three
// arrays [bins]
constexpr size_t group_smem_bytes(int bins, bool counters) {
    return sizeof(int4) * (bins + 1) + sizeof(int32_t) * ((counters ? (size_t)bins * kGpWarps : 0) + 3 * (size_t)bins);
}

template <typename Id>
__global__ void __launch_bounds__(kGpThreads)
    k_group_single(const Id* __restrict__ bucket, int64_t T, int E, int32_t* __restrict__ plan, unsigned long long* status) {
    extern __shared__ int4 s_at[];
    const int bins = E + 1;
    int32_t* s_hist = reinterpret_cast<int32_t*>(s_at + bins + 1);
    int32_t* s_total = s_hist + bins * kGpWarps;
    __shared__ int4 s_warp[kGpWarps];
    group_histogram(bucket, 0, T, bins, s_hist, status);
    for (int b = threadIdx.x; b < bins; b += kGpThreads) s_total[b] = group_scan_warps(s_hist, bins, b);
    __syncthreads();
    group_tiles(T, E, s_total, s_at, s_warp, plan);
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += kGpThreads) s_total[b] = s_at[b].x;  // from here on: first places
    __syncthreads();
    group_fill(bucket, 0, T, bins, s_hist, s_total, plan + group_order_at(E));
}

// One cluster: every CTA a run of the rows, the runs' counters read from one another's shared memory.
template <typename Id>
__global__ void __launch_bounds__(kGpThreads)
    k_group_cluster(const Id* __restrict__ bucket, int64_t T, int E, int32_t* __restrict__ plan, unsigned long long* status) {
    extern __shared__ int4 s_at[];
    const int bins = E + 1, rank = (int)cluster_rank();
    int32_t* s_hist = reinterpret_cast<int32_t*>(s_at + bins + 1);
    int32_t* s_total = s_hist + bins * kGpWarps;
    int32_t* s_own = s_total + bins;   // this CTA's counters
    int32_t* s_base = s_own + bins;    // rows of the bin in the CTAs before; from there on first places
    __shared__ int4 s_warp[kGpWarps];
    const int64_t per = (T + kClusterSize * 32 - 1) / (kClusterSize * 32) * 32;
    const int64_t lo = min(T, rank * per), hi = min(T, lo + per);
    group_histogram(bucket, lo, hi, bins, s_hist, status);
    for (int b = threadIdx.x; b < bins; b += kGpThreads) s_own[b] = group_scan_warps(s_hist, bins, b);
    cluster_sync();
    for (int b = threadIdx.x; b < bins; b += kGpThreads) {
        int v[kClusterSize], total = 0, before = 0;
#pragma unroll
        for (int r = 0; r < kClusterSize; ++r) v[r] = ld_cluster_int(s_own + b, (uint32_t)r);
#pragma unroll
        for (int r = 0; r < kClusterSize; ++r) {
            total += v[r];
            if (r < rank) before += v[r];
        }
        s_total[b] = total;
        s_base[b] = before;
    }
    __syncthreads();
    group_tiles(T, E, s_total, s_at, s_warp, plan, rank, kClusterSize);
    for (int b = threadIdx.x; b < bins; b += kGpThreads) s_base[b] += s_at[b].x;
    __syncthreads();
    group_fill(bucket, lo, hi, bins, s_hist, s_base, plan + group_order_at(E));
    cluster_sync();  // nobody leaves while its counters are read
}

// long form, 1: counts[bin][block]
template <typename Id>
__global__ void __launch_bounds__(kGpThreads)
    k_group_count(const Id* __restrict__ bucket, int64_t T, int E, int32_t* __restrict__ counts, unsigned long long* status) {
    extern __shared__ int32_t s_hist[];
    const int bins = E + 1;
    const int64_t lo = (int64_t)blockIdx.x * kBlockRows, hi = min(T, lo + kBlockRows);
    group_histogram(bucket, lo, hi, bins, s_hist, status);
    for (int b = threadIdx.x; b < bins; b += kGpThreads)
        counts[(int64_t)b * gridDim.x + blockIdx.x] = group_scan_warps(s_hist, bins, b);
}

// long form, 2: counts[bin][block] becomes the number of rows of `bin` in the blocks before, and the plan's head
__global__ void __launch_bounds__(kGpThreads)
    k_group_scan(int64_t T, int E, int blocks, int32_t* __restrict__ counts, int32_t* __restrict__ plan) {
    extern __shared__ int4 s_at[];
    const int bins = E + 1;
    int32_t* s_total = reinterpret_cast<int32_t*>(s_at + bins + 1);
    __shared__ int4 s_warp[kGpWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int b = warp; b < bins; b += kGpWarps) {
        int run = 0;
        for (int i0 = 0; i0 < blocks; i0 += 32) {
            const int i = i0 + lane;
            const int v = i < blocks ? counts[(int64_t)b * blocks + i] : 0;
            int inc = v;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int x = __shfl_up_sync(kFullMask, inc, d);
                if (lane >= d) inc += x;
            }
            if (i < blocks) counts[(int64_t)b * blocks + i] = run + inc - v;
            run += __shfl_sync(kFullMask, inc, 31);
        }
        if (lane == 0) s_total[b] = run;
    }
    __syncthreads();
    group_tiles(T, E, s_total, s_at, s_warp, plan);
}

// long form, 3: rows to their places
template <typename Id>
__global__ void __launch_bounds__(kGpThreads)
    k_group_fill(const Id* __restrict__ bucket, int64_t T, int E, const int32_t* __restrict__ counts, int32_t* __restrict__ plan) {
    extern __shared__ int32_t s_hist[];
    const int bins = E + 1;
    int32_t* s_base = s_hist + bins * kGpWarps;
    const int64_t lo = (int64_t)blockIdx.x * kBlockRows, hi = min(T, lo + kBlockRows);
    group_histogram(bucket, lo, hi, bins, s_hist, nullptr);
    for (int b = threadIdx.x; b < bins; b += kGpThreads) {
        group_scan_warps(s_hist, bins, b);
        s_base[b] = plan[group_offsets_at() + b] + counts[(int64_t)b * gridDim.x + blockIdx.x];
    }
    __syncthreads();
    group_fill(bucket, lo, hi, bins, s_hist, s_base, plan + group_order_at(E));
}

inline int64_t group_blocks(int64_t T) { return T <= kClusterRows ? 0 : (T + kBlockRows - 1) / kBlockRows; }

template <typename Id>
int launch_plan(const Id* bucket, int64_t T, int32_t E, int32_t* plan, unsigned long long* status, cudaStream_t s) {
    const int bins = E + 1;
    const size_t smem = group_smem_bytes(bins, true);
    static bool opted[64] = {};  // more than 48 KB of dynamic shared memory needs the opt-in, once per device
    int dev = 0;
    NNUE_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !opted[dev]) {
        const int most = (int)group_smem_bytes(kMaxGroups + 1, true);
        NNUE_CUDA_TRY(cudaFuncSetAttribute(k_group_single<Id>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
        NNUE_CUDA_TRY(cudaFuncSetAttribute(k_group_cluster<Id>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
        NNUE_CUDA_TRY(cudaFuncSetAttribute(k_group_count<Id>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
        NNUE_CUDA_TRY(cudaFuncSetAttribute(k_group_fill<Id>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
        if (dev >= 0 && dev < 64) opted[dev] = true;
    }
    const int64_t blocks = group_blocks(T);
    if (blocks == 0 && T > kSingleRows) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(kClusterSize);
        cfg.blockDim = dim3(kGpThreads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = s;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = kClusterSize;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        NNUE_CUDA_TRY(cudaLaunchKernelEx(&cfg, k_group_cluster<Id>, bucket, T, (int)E, plan, status));
        note_launches(1);
    } else if (blocks == 0) {
        k_group_single<Id><<<1, kGpThreads, smem, s>>>(bucket, T, E, plan, status);
        note_launches(1);
    } else {
        int32_t* counts = plan + group_counts_at(T, E);
        k_group_count<Id><<<(unsigned)blocks, kGpThreads, smem, s>>>(bucket, T, E, counts, status);
        k_group_scan<<<1, kGpThreads, group_smem_bytes(bins, false), s>>>(T, E, (int)blocks, counts, plan);
        k_group_fill<Id><<<(unsigned)blocks, kGpThreads, smem, s>>>(bucket, T, E, counts, plan);
        note_launches(3);
    }
    NNUE_CUDA_TRY(cudaGetLastError());
    return NNUE_OK;
}

}  // namespace nnue

using namespace nnue;

extern "C" size_t nnue_group_plan_bytes(int64_t T, int32_t E) {
    if (T < 0 || T > NNUE_GROUP_MAX_ROWS || E <= 0 || E > kMaxGroups) return 0;
    return sizeof(int32_t) * (size_t)(group_counts_at(T, E) + group_blocks(T) * (E + 1));
}

extern "C" int nnue_group_plan(const void* bucket, int32_t wide_ids, int64_t T, int32_t E, int32_t* plan, size_t plan_bytes,
                               void* stream) {
    NNUE_REQUIRE(T >= 0 && E > 0, NNUE_ERR_ARG, "nnue_group_plan: negative batch or no bucket");
    NNUE_REQUIRE(E <= kMaxGroups && T <= NNUE_GROUP_MAX_ROWS, NNUE_ERR_UNSUPPORTED,
                 "nnue_group_plan: %d buckets (at most %d) of %lld rows (at most %lld)", E, kMaxGroups, (long long)T,
                 (long long)NNUE_GROUP_MAX_ROWS);
    NNUE_REQUIRE(T == 0 || bucket, NNUE_ERR_ARG, "nnue_group_plan: null bucket list");
    NNUE_REQUIRE(plan && plan_bytes >= nnue_group_plan_bytes(T, E) && aligned16(plan), NNUE_ERR_WORKSPACE,
                 "nnue_group_plan: plan buffer too small or unaligned");
    unsigned long long* status = device_status_ptr();
    NNUE_REQUIRE(status, NNUE_ERR_CUDA, "nnue_group_plan: no device status word");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ProfScope prof("group_plan", s);
    return wide_ids ? launch_plan(static_cast<const int64_t*>(bucket), T, E, plan, status, s)
                    : launch_plan(static_cast<const int32_t*>(bucket), T, E, plan, status, s);
}
