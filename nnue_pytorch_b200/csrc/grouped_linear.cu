// Bucketed ("grouped by expert") linear layer on 16-bit operands, on the 5th-generation tensor cores:
//   forward          y[p, n]     = sum_k x[p, k] w[b, n, k] + bias[b, n]        b = bucket of row p
//   input gradient   dx[p, k]    = sum_n dy[p, n] w[b, n, k]
//   weight gradient  dw[b, n, k] = sum_{p of b} dy[p, n] x[p, k],  dbias[b, n] = sum_{p of b} dy[p, n]
//
// One kernel, three ways to read its operands by TMA (128 bytes per row of a stage, swizzled); D accumulates in tensor
// memory in fp32.
//   forward   A = rows of x of one bucket, K-major;    B = rows of w, K-major
//   dx        A = rows of dy, K-major;                 B = columns of w, MN-major (w is read as it lies)
//   dw        A = columns of dy, B = columns of x, both MN-major; the sum runs over the bucket's rows
// Rows laid out by bucket (nnue_group_rows) come as boxes; the zeros between buckets are what dw adds behind a bucket's
// end, and forward and dx never store the rows of a tile behind its count.  Without that layout forward and dx gather
// four rows per copy.  A four-row copy takes an SM about 75 cycles whatever issues it (675 us for the forward of 16384 x
// 4096 x 2048), and rows gathered by 16-byte asynchronous copies came to 36 GB/s per SM with four warps (254 us; 595 for
// dw): laying the rows out first costs 51 us there, and both directions read them.
//
// Roles: warp 0 copies into a ring of stages, warp 1 issues the instructions, warps 4-11 take the accumulators and bring
// finished tiles out while the next run of stages multiplies (two accumulators).  Persistent: a CTA (or pair) per SM walks
// the tiles with a stride of the grid.
// CTAS = 2: a pair of SMs works on 256 rows x BN columns, each holding its half of A and of B: half the bytes of B per
//   SM and flop, through L2 and in shared memory, which is what bounds a single CTA (96 bytes per cycle wanted of L2's
//   64 at 128 x 256).
// SPLIT: few tiles; a cluster of 2 to 8 CTAs splits the sum, the partial tiles meet in distributed shared memory and are
//   added in the order of the ranks.
// Sums in two levels: the tensor core's adder cuts off.  Measured on sums next to 2^23: each of an instruction's 16 terms
//   loses what lies below a quarter of the sum's last bit, the result what lies below that bit, so an addition loses
//   less than 5 x 2^-23 of the sum and a sum of n terms grows off by n / 16 times that.  An accumulator therefore adds up runs
//   of 512 terms; the output warps hold the sums in registers (half a row of the tile per thread) and add the runs rounding
//   to nearest.  Where bf16 results of 16384 x 4096 x 2048 differ from an fp32 product's, 94 % were the farther ones from 64
//   bits in one level, half are in two.
//   Runs of 8 stages against one for the whole sum, us at that size over 8 buckets: forward 198 (183), dx 202 (197), dw 219
//   (217); of 4 stages 213, 212, 221; of 16 193, 198, 218: a change of accumulator costs the issuing warp about 400
//   cycles.  dw in fp32 227 (353 with the total in tensor memory, which leaves room for 128 columns only).
// Measured at that size, bf16: forward 198 us (1.39 PFLOP/s), dx 202, dw 219 after 51 for laying x out and 28 for dy; bound by the
// issuing warp's way from stage to stage (about 800 cycles for 512 of multiplying) and the operands' way through L2 and
// shared memory (32 KB per SM and stage).
// All orders are fixed by the sizes: results are reproducible.  Every wait is bounded; one that runs out raises the
// device status word and the CTA leaves, its tensor memory freed; copies in flight are then as old as that wait.
#include "grouped_tc.cuh"

namespace nnue {

enum { kModeFwd = 0, kModeDx = 1, kModeDw = 2 };

constexpr int kGlK = 64;                     // reduction elements per stage: one 128-byte swizzle row
constexpr int kGlABytes = kGroupRows * 128;  // 16 KiB
constexpr int kGlBoxBytes = kGlK * 128;      // MN-major block: 64 rows of the reduction x 128 bytes
constexpr int kGlThreads = 384;  // copies, instructions, two warps without work, eight output warps
constexpr int kGlOutWarp = 4;    // the first output warp
// An output thread of the widest tile holds 128 sums and two reads of 32 columns: the first warpgroup gives registers up
// (at 72 and 216 the sums spill: dx 210 us for 202).
constexpr int kGlFewRegs = 56, kGlManyRegs = 224, kGlLaunchRegs = 168;
static_assert(128 * kGlFewRegs + 256 * kGlManyRegs <= kGlThreads * kGlLaunchRegs, "more registers than the launch brings");
constexpr int kGlRun = 8;                    // stages that one accumulator adds up: 512 terms

constexpr int gl_stage_bytes(int bn, int ctas) { return kGlABytes + bn / ctas * 128; }
constexpr int gl_stages(int bn, int ctas) { return gl_stage_bytes(bn, ctas) > 32768 ? 4 : gl_stage_bytes(bn, ctas) > 24576 ? 6 : 8; }
constexpr int gl_smem(int bn, int ctas) {  // alignment, ring, staging, barriers
    return 1024 + gl_stages(bn, ctas) * gl_stage_bytes(bn, ctas) + 8 * kStagingBytes + 256;
}
constexpr int gl_warp_cols(int bn) { return bn >= 64 ? bn / 2 : bn; }  // columns of an output warp

struct GlArgs {
    GroupPlanView plan;
    RowsOut o;
    void* sums;              // dw: dbias, or null
    const float* tile_sums;  // dw: sums of dy's columns per tile of 128 rows [tiles][N]
    const void* bias;        // forward, or null
    int32_t sums_type, bias_type;
    int32_t T, E, N;         // N: rows of w per bucket
    int32_t red;             // length of the reduction (forward, dx)
    int32_t col_tiles;       // ceil(cols / BN)
    int32_t row_tiles;       // dw: tiles along N
    int32_t gather;          // forward, dx: A's rows are gathered by the plan's order
    uint32_t idesc;
    unsigned long long* status;
};

// One tile of the output and the part of its sum that this CTA adds up.
struct GlTile {
    int32_t bucket, first, count, place;  // rows order[first .. first + count), laid out from `place` on: the tile's or (dw) the bucket's
    int32_t row0, col0;                   // dw: first row inside the bucket's matrix; first column
    int32_t c0, c1;                       // chunks of the reduction
    bool live;                            // false: rows without a bucket
};

template <int MODE, int BN, int CTAS, bool SPLIT>
__device__ __forceinline__ GlTile gl_tile(const GlArgs& a, int t, int rank, int ranks) {
    GlTile x;
    const int rt = t / a.col_tiles, ct = t - rt * a.col_tiles;
    x.col0 = ct * BN;
    int chunks;
    if (MODE == kModeDw) {
        x.bucket = rt / a.row_tiles;
        x.row0 = (rt - x.bucket * a.row_tiles) * (kGroupRows * CTAS);
        x.first = __ldg(a.plan.offsets + x.bucket);
        x.count = __ldg(a.plan.offsets + x.bucket + 1) - x.first;
        x.place = __ldg(a.plan.places + x.bucket);
        chunks = (x.count + kGlK - 1) / kGlK;
        x.live = true;
    } else {
        const int4 g = __ldg(reinterpret_cast<const int4*>(CTAS == 2 ? a.plan.pairs : a.plan.tiles) + rt);
        x.bucket = g.x;
        x.first = g.y;
        x.count = g.z;
        x.place = g.w;
        x.row0 = 0;
        x.live = x.bucket < a.E;
        chunks = x.live ? (a.red + kGlK - 1) / kGlK : 0;
    }
    x.c0 = SPLIT ? (int)((int64_t)chunks * rank / ranks) : 0;
    x.c1 = SPLIT ? (int)((int64_t)chunks * (rank + 1) / ranks) : chunks;
    return x;
}

// instructions of 16 reduction elements that chunk c needs
template <int MODE>
__device__ __forceinline__ int gl_steps(const GlArgs& a, const GlTile& x, int c) {
    const int left = (MODE == kModeDw ? x.count : a.red) - c * kGlK;
    return left >= kGlK ? 4 : (left + 15) >> 4;
}

// a0 += v0, a1 += v1, each rounded to nearest
__device__ __forceinline__ void add2(float& a0, float& a1, uint32_t v0, uint32_t v1) {
    unsigned long long a, v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(a) : "f"(a0), "f"(a1));
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(v0), "r"(v1));
    asm("add.rn.f32x2 %0, %0, %1;" : "+l"(a) : "l"(v));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a0), "=f"(a1) : "l"(a));
}

// One output warp: sum (FIRST: =, else +=, rounding to nearest) accumulator, its 32 lanes and COLS columns.
template <int COLS, bool FIRST>
__device__ __forceinline__ void gl_add(uint32_t taddr, float (&sum)[COLS]) {
    constexpr int kReads = COLS / 32, kAtOnce = kReads < 2 ? kReads : 2;
#pragma unroll
    for (int c = 0; c < kReads; c += kAtOnce) {
        uint32_t v[kAtOnce][32];  // the reads under way before the wait
#pragma unroll
        for (int h = 0; h < kAtOnce; ++h) tmem_ld32(taddr + 32 * (c + h), v[h]);
#pragma unroll
        for (int h = 0; h < kAtOnce; ++h) tmem_wait_ld(v[h]);
#pragma unroll
        for (int h = 0; h < kAtOnce; ++h)
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
                float& s0 = sum[32 * (c + h) + j];
                float& s1 = sum[32 * (c + h) + j + 1];
                if (FIRST) s0 = __uint_as_float(v[h][j]), s1 = __uint_as_float(v[h][j + 1]);
                else add2(s0, s1, v[h][j], v[h][j + 1]);
            }
    }
}

// ---- warp 0: copies ---------------------------------------------------------------------------------------------------
template <int MODE, int BN, int CTAS, bool SPLIT>
__device__ __forceinline__ bool gl_copy_role(const GlArgs& a, const CUtensorMap* map_a, const CUtensorMap* map_b, uint32_t ring,
                                             uint64_t* full, uint64_t* empty, int t0, int stride, int tiles, int rank, int ranks) {
    constexpr bool PAIR = CTAS == 2;
    constexpr int S = gl_stages(BN, CTAS), kBn = BN / CTAS;  // kBn: this CTA's columns of B
    const int lane = threadIdx.x & 31;
    StageRing<S> at;
    bool ok = true;
    for (int t = t0; t < tiles && ok; t += stride) {
        const GlTile x = gl_tile<MODE, BN, CTAS, SPLIT>(a, t, rank, ranks);
        if (x.c0 == x.c1) continue;
        const int side = PAIR ? rank : 0;
        // blocks of 64 columns wholly outside the operand are not read: their rows or columns of D are never stored
        const int a_row0 = x.row0 + side * kGroupRows, b_col0 = x.col0 + side * kBn;
        const int a_boxes = MODE == kModeDw ? max(0, min(2, (a.N - a_row0 + 63) >> 6)) : 0;
        const int b_boxes = MODE == kModeFwd ? 0 : max(0, min(kBn / 64, (a.o.cols - b_col0 + 63) >> 6));
        const bool a_rows = MODE != kModeDw && x.count > side * kGroupRows;
        const bool gather = MODE != kModeDw && !PAIR && a.gather;
        // the bytes that complete the stage: both CTAs' of a pair, announced by the first
        int bytes;
        if (MODE == kModeDw) {
            bytes = (min(2 * CTAS, (a.N - x.row0 + 63) >> 6) + min(BN / 64, (a.o.cols - x.col0 + 63) >> 6)) * kGlBoxBytes;
        } else {
            bytes = gather ? ((x.count + 3) >> 2) * 512 : (PAIR && x.count > kGroupRows ? 2 : 1) * kGlABytes;
            bytes += MODE == kModeFwd ? BN * 128 : min(BN / 64, (a.o.cols - x.col0 + 63) >> 6) * kGlBoxBytes;
        }
        int rows[4];
        if (gather) {
#pragma unroll
            for (int j = 0; j < 4; ++j) rows[j] = 4 * lane + j < x.count ? __ldg(a.plan.order + x.first + 4 * lane + j) : a.T;
        }
        for (int c = x.c0; c < x.c1; ++c) {
            if (lane == 0) ok = mbar_wait_timed(empty + at.stage, at.phase ^ 1u);
            if (MODE != kModeDw && !PAIR) ok = __shfl_sync(kFullMask, (int)ok, 0) != 0;
            if (!ok) break;
            const uint32_t sa = ring + at.stage * gl_stage_bytes(BN, CTAS), sb = sa + kGlABytes;
            const uint32_t bar = PAIR ? map_rank(full + at.stage, 0) : smem_u32(full + at.stage);
            if (lane == 0) {
                if (!PAIR || rank == 0) mbar_expect_tx(full + at.stage, bytes);
                if (MODE == kModeDw) {
                    const int y = x.place + c * kGlK;
                    for (int i = 0; i < a_boxes; ++i) tma_tile_2d<PAIR>(sa + i * kGlBoxBytes, map_a, a_row0 + i * 64, y, bar);
                    for (int i = 0; i < b_boxes; ++i) tma_tile_2d<PAIR>(sb + i * kGlBoxBytes, map_b, b_col0 + i * 64, y, bar);
                } else {
                    if (!gather && a_rows) tma_tile_2d<PAIR>(sa, map_a, c * kGlK, x.place + side * kGroupRows, bar);
                    if (MODE == kModeFwd) tma_tile_3d<PAIR>(sb, map_b, c * kGlK, b_col0, x.bucket, bar);
                    else
                        for (int i = 0; i < b_boxes; ++i) tma_tile_3d<PAIR>(sb + i * kGlBoxBytes, map_b, b_col0 + i * 64, c * kGlK, x.bucket, bar);
                }
            }
            if (gather) {
                __syncwarp();
                if (4 * lane < x.count) tma_gather4(sa + lane * 512, map_a, c * kGlK, rows[0], rows[1], rows[2], rows[3], bar);
            }
            at.next();
        }
        if (MODE == kModeDw || PAIR) ok = __shfl_sync(kFullMask, (int)ok, 0) != 0;
    }
    return ok;
}

// ---- warp 1: the instructions -------------------------------------------------------------------------------------
template <int MODE, int BN, int CTAS, bool SPLIT>
__device__ __forceinline__ bool gl_issue_role(const GlArgs& a, uint32_t tmem, uint32_t ring, uint64_t* full, uint64_t* empty,
                                              uint64_t* done, uint64_t* taken, uint64_t* drained, int t0, int stride, int tiles,
                                              int rank, int ranks) {
    constexpr bool PAIR = CTAS == 2;
    constexpr bool kAMn = MODE == kModeDw, kBMn = MODE != kModeFwd;
    constexpr uint32_t kAStep = kAMn ? 2048 >> 4 : 32 >> 4, kBStep = kBMn ? 2048 >> 4 : 32 >> 4;  // 16 reduction elements
    StageRing<gl_stages(BN, CTAS)> at;
    StageRing<2> acc;
    bool ok = true;
    for (int t = t0; t < tiles && ok; t += stride) {
        const GlTile x = gl_tile<MODE, BN, CTAS, SPLIT>(a, t, rank, ranks);
        for (int g = x.c0; g < x.c1 && ok; g += kGlRun) {  // one accumulator's chunks
            const int end = min(x.c1, g + kGlRun);
            ok = mbar_wait_warp(taken + acc.stage, acc.phase ^ 1u);
            if (!ok) break;
            tc_fence_after();
            const uint32_t d = tmem + acc.stage * BN;
            for (int c = g; c < end; ++c) {
                ok = mbar_wait_warp(full + at.stage, at.phase);
                if (!ok) break;
                tc_fence_after();
                const uint32_t sa = ring + at.stage * gl_stage_bytes(BN, CTAS);
                const uint64_t da = umma_desc_sw128(sa, kGlBoxBytes), db = umma_desc_sw128(sa + kGlABytes, kGlBoxBytes);
                const int steps = gl_steps<MODE>(a, x, c);
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (k < steps) umma_f16<PAIR>(d, da + k * kAStep, db + k * kBStep, a.idesc, c != g || k != 0);
                    umma_commit_to<PAIR>(empty + at.stage);
                    if (c + 1 == end) umma_commit_to<PAIR>(done + acc.stage);
                }
                __syncwarp();
                at.next();
            }
            if (!ok) break;
            acc.next();
        }
    }
    if (!ok) {  // instructions in flight finish before the tensor memory is freed
        if (elect_one()) umma_commit_to<PAIR>(drained);
        __syncwarp();
        mbar_wait_warp(drained, 0);
    }
    return ok;
}

// dw: dbias of this thread's row, from the sums of the bucket's tiles in order
__device__ __forceinline__ void gl_bias_gradient(const GlArgs& a, const GlTile& x, int n) {
    float total = 0.f;
    const int t1 = __ldg(a.plan.first + x.bucket + 1);
#pragma unroll 8
    for (int t = __ldg(a.plan.first + x.bucket); t < t1; ++t) total += __ldg(a.tile_sums + (int64_t)t * a.N + n);
    store_from_float(a.sums, a.sums_type, (int64_t)x.bucket * a.N + n, total);
}

template <int MODE, int BN, int CTAS, bool SPLIT>
__global__ void __launch_bounds__(kGlThreads, 1)
    k_grouped(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ GlArgs a) {
    constexpr bool PAIR = CTAS == 2;
    constexpr int S = gl_stages(BN, CTAS);
    constexpr uint32_t kTmemCols = 2 * BN;
    constexpr int kPartPitch = BN + 4;  // floats per row of a partial tile
    static_assert(!(PAIR && SPLIT), "no such variant");
    extern __shared__ unsigned char smem_raw[];
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
    unsigned char* ring_ptr = smem_raw + (ring - smem_u32(smem_raw));
    unsigned char* staging = ring_ptr + S * gl_stage_bytes(BN, CTAS);
    uint64_t* full = reinterpret_cast<uint64_t*>(staging + 8 * kStagingBytes);  // [S] a stage's copies are in (pair: the first CTA's)
    uint64_t* empty = full + S;                                            // [S] a stage may be overwritten
    uint64_t* done = empty + S;                                            // [2] an accumulator is complete
    uint64_t* taken = done + 2;                                            // [2] an accumulator has been read
    uint64_t* drained = taken + 2;                                         // [1]
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(drained + 1);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int rank = 0, ranks = 1;
    if (SPLIT || PAIR) {
        rank = (int)cluster_rank();
        uint32_t n;
        asm volatile("mov.u32 %0, %cluster_nctaid.x;" : "=r"(n));
        ranks = (int)n;
    }
    const int tiles = (MODE == kModeDw ? a.E * a.row_tiles : __ldg(a.plan.n_tiles + (PAIR ? 1 : 0))) * a.col_tiles;
    const int t0 = (int)blockIdx.x / ranks, stride = (int)gridDim.x / ranks;  // split: at most one tile per cluster
    if (t0 >= tiles) return;                                                  // (the whole cluster)

    if (tid == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(full + s, 1);
            mbar_init(empty + s, 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(done + s, 1);
            mbar_init(taken + s, 8 * CTAS);
        }
        mbar_init(drained, 1);
        fence_barrier_init();
        prefetch_map(&map_a);
        prefetch_map(&map_b);
    }
    if (warp == 1) tmem_alloc<PAIR>(s_tmem, kTmemCols);
    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();  // the other CTA's barriers are there
    tc_fence_after();
    const uint32_t tmem = *s_tmem;

    bool ok = true;
    if (warp < kGlOutWarp) {
        if (BN == 256) fewer_registers<kGlFewRegs>();
        if (warp == 0)
            ok = gl_copy_role<MODE, BN, CTAS, SPLIT>(a, &map_a, &map_b, ring, full, empty, t0, stride, tiles, rank, ranks);
        else if (warp == 1 && !(PAIR && rank != 0))
            ok = gl_issue_role<MODE, BN, CTAS, SPLIT>(a, tmem, ring, full, empty, done, taken, drained, t0, stride, tiles, rank, ranks);
    } else {
        if (BN == 256) more_registers<kGlManyRegs>();
        constexpr int kCols = gl_warp_cols(BN);
        const int q = warp & 3, half = (warp - kGlOutWarp) >> 2;  // the quarter of tensor memory's lanes, the half of the columns
        const bool works = BN >= 64 || half == 0;                 // 32 columns are one half
        const uint32_t lanes = ((uint32_t)(q * 32) << 16) + half * kCols;
        StageRing<2> acc;
        for (int t = t0; t < tiles && ok; t += stride) {
            const GlTile x = gl_tile<MODE, BN, CTAS, SPLIT>(a, t, rank, ranks);
            const int r = (PAIR ? rank * kGroupRows : 0) + q * 32 + lane;
            int32_t my_row;
            int64_t row_base = 0;
            if (MODE == kModeDw) {
                my_row = x.row0 + r < a.N ? x.row0 + r : -1;
                row_base = (int64_t)x.bucket * a.N;
                if (!SPLIT && a.sums && x.col0 == 0 && half == 0 && my_row >= 0) gl_bias_gradient(a, x, my_row);
            } else {
                my_row = r < x.count ? __ldg(a.plan.order + x.first + r) : -1;
            }
            const int col = x.col0 + half * kCols;
            const bool biased = MODE == kModeFwd && !SPLIT && a.bias && x.live;
            float bias[kCols / 32];  // of columns lane, 32 + lane, ..: on its way while the tile multiplies
            if (biased) {
#pragma unroll
                for (int i = 0; i < kCols / 32; ++i) {
                    const int j = 32 * i + lane;
                    bias[i] = works && col + j < a.o.cols ? load_as_float(a.bias, a.bias_type, (int64_t)x.bucket * a.N + col + j) : 0.f;
                }
            }
            float sum[kCols];
            auto taken_in = [&] {  // the accumulator is in registers
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (PAIR) mbar_arrive_cluster(map_rank(taken + acc.stage, 0));
                    else mbar_arrive(taken + acc.stage);
                }
                acc.next();
            };
            if (x.c0 < x.c1) {
                ok = mbar_wait_warp(done + acc.stage, acc.phase);
                if (!ok) break;
                tc_fence_after();
                if (works) gl_add<kCols, true>(tmem + lanes + acc.stage * BN, sum);
                taken_in();
#pragma unroll 1
                for (int g = x.c0 + kGlRun; g < x.c1; g += kGlRun) {
                    ok = mbar_wait_warp(done + acc.stage, acc.phase);
                    if (!ok) break;
                    tc_fence_after();
                    if (works) gl_add<kCols, false>(tmem + lanes + acc.stage * BN, sum);
                    taken_in();
                }
                if (!ok) break;
            } else {
#pragma unroll
                for (int j = 0; j < kCols; ++j) sum[j] = 0.f;
            }
            if (SPLIT) {
                // the last accumulator is complete, so nothing reads the ring any more: it takes the partial tile
                float* part = reinterpret_cast<float*>(ring_ptr) + (q * 32 + lane) * kPartPitch + half * kCols;
                if (works) {
#pragma unroll
                    for (int j = 0; j < kCols; j += 4) *reinterpret_cast<float4*>(part + j) = make_float4(sum[j], sum[j + 1], sum[j + 2], sum[j + 3]);
                }
                break;
            }
            if (!works || col >= a.o.cols || !__any_sync(kFullMask, my_row >= 0)) continue;
            unsigned char* stg = staging + (warp - kGlOutWarp) * kStagingBytes;
            if (biased) {
                float* s_bias = reinterpret_cast<float*>(stg);
#pragma unroll
                for (int i = 0; i < kCols / 32; ++i) s_bias[32 * i + lane] = bias[i];
                __syncwarp();
#pragma unroll
                for (int j = 0; j < kCols; j += 4) {
                    const float4 b = *reinterpret_cast<const float4*>(s_bias + j);
                    sum[j] += b.x;
                    sum[j + 1] += b.y;
                    sum[j + 2] += b.z;
                    sum[j + 3] += b.w;
                }
                __syncwarp();
            }
            bring_out<0, kCols>(a.o, sum, stg, my_row, row_base, col);
        }
    }
    __syncwarp();
    if (!ok && lane == 0) note_timeout(a.status);

    if (SPLIT) {
        const GlTile x = gl_tile<MODE, BN, CTAS, SPLIT>(a, t0, rank, ranks);
        cluster_sync();
        // row r of the tile is finished by rank r mod ranks: partial sums in the order of the ranks
        const int rows = MODE == kModeDw ? min(kGroupRows, a.N - x.row0) : x.count;
        const int mine = (rows - rank + ranks - 1) / ranks;
        const int es = a.o.type == NNUE_T_F32 ? 4 : 2;
        for (int i = tid; i < mine * (BN / 4); i += kGlThreads) {
            const int r = rank + i / (BN / 4) * ranks, c = i % (BN / 4) * 4, col = x.col0 + c;
            if (col >= a.o.cols) continue;
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            if (x.live) {
                const uint32_t addr = ring + (uint32_t)(r * kPartPitch + c) * 4;
                for (int s = 0; s < ranks; ++s) {
                    const float4 p = ld_cluster4(addr, (uint32_t)s);
                    v[0] += p.x;
                    v[1] += p.y;
                    v[2] += p.z;
                    v[3] += p.w;
                }
            }
            if (MODE == kModeFwd && a.bias && x.live) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (col + j < a.o.cols) v[j] += load_as_float(a.bias, a.bias_type, (int64_t)x.bucket * a.N + col + j);
            }
            const int64_t row = MODE == kModeDw ? (int64_t)x.bucket * a.N + x.row0 + r : (int64_t)__ldg(a.plan.order + x.first + r);
            const int64_t at = row * a.o.ld + col;
            if (a.o.vec && es == 4) {
                *reinterpret_cast<float4*>(static_cast<float*>(a.o.out) + at) = make_float4(v[0], v[1], v[2], v[3]);
            } else if (a.o.vec) {
                *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o.out) + at) =
                    make_uint2(pack_half(v[0], v[1], a.o.type), pack_half(v[2], v[3], a.o.type));
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (col + j < a.o.cols) store_from_float(a.o.out, a.o.type, at + j, v[j]);
            }
        }
        if (MODE == kModeDw && a.sums && x.col0 == 0 && rank == 0 && tid < rows) gl_bias_gradient(a, x, x.row0 + tid);
        cluster_sync();  // nobody leaves while its shared memory is read
    }
    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();  // both have read their tensor memory, and nobody's barriers are arrived on any more
    if (warp == 1) tmem_free<PAIR>(tmem, kTmemCols);
}

// ---- host ---------------------------------------------------------------------------------------------------------------
template <int MODE, int BN, int CTAS, bool SPLIT>
int gl_launch(const CUtensorMap& ma, const CUtensorMap& mb, const GlArgs& a, int64_t tiles, int ranks, cudaStream_t s) {
    auto kernel = k_grouped<MODE, BN, CTAS, SPLIT>;
    static bool opted[64] = {};  // more than 48 KB of dynamic shared memory needs the opt-in, once per device
    int dev = 0;
    NNUE_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !opted[dev]) {
        NNUE_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, gl_smem(BN, CTAS)));
        cudaFuncAttributes attr;
        NNUE_CUDA_TRY(cudaFuncGetAttributes(&attr, kernel));
        NNUE_REQUIRE(BN != 256 || attr.numRegs >= kGlLaunchRegs, NNUE_ERR_UNSUPPORTED, "grouped linear: built with %d registers per thread",
                     attr.numRegs);
        if (dev >= 0 && dev < 64) opted[dev] = true;
    }
    const int64_t at_once = sm_count() / CTAS;
    const int64_t ctas = SPLIT ? tiles * ranks : (tiles < at_once ? tiles : at_once) * CTAS;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(kGlThreads);
    cfg.dynamicSmemBytes = gl_smem(BN, CTAS);
    cfg.stream = s;
    cudaLaunchAttribute attr;
    if (SPLIT || CTAS > 1) {
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = (unsigned)(SPLIT ? ranks : CTAS);
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
    }
    NNUE_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, ma, mb, a));
    note_launches(1);
    return NNUE_OK;
}

template <int MODE>
int gl_run(const CUtensorMap& ma, const CUtensorMap& mb, GlArgs& a, int64_t tile_rows, TileShape shape, cudaStream_t s) {
    constexpr int kNarrowest = MODE == kModeFwd ? 32 : 64, kWidest = 256;
    a.col_tiles = (a.o.cols + shape.bn - 1) / shape.bn;
    a.idesc = umma_idesc(a.idesc, (uint32_t)(kGroupRows * shape.ctas), (uint32_t)shape.bn, MODE == kModeDw, MODE != kModeFwd);
    const int64_t tiles = tile_rows * a.col_tiles;
    NNUE_REQUIRE(tiles * 8 < 0x7fffffffLL, NNUE_ERR_UNSUPPORTED, "grouped linear: too many tiles");
    if (shape.ctas == 2) return gl_launch<MODE, kWidest, 2, false>(ma, mb, a, tiles, 1, s);
    if (shape.ranks > 1) return gl_launch<MODE, kNarrowest, 1, true>(ma, mb, a, tiles, shape.ranks, s);
    if (shape.bn == 32) return gl_launch<MODE, kNarrowest, 1, false>(ma, mb, a, tiles, 1, s);
    if (shape.bn == 64) return gl_launch<MODE, 64, 1, false>(ma, mb, a, tiles, 1, s);
    if (shape.bn == 128) return gl_launch<MODE, 128, 1, false>(ma, mb, a, tiles, 1, s);
    return gl_launch<MODE, kWidest, 1, false>(ma, mb, a, tiles, 1, s);
}

static CUtensorMapDataType map_type(int32_t type) {
    return type == NNUE_T_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}
// [rows, cols] read in boxes of 64 columns and `high` rows
static int rows_map(CUtensorMap* map, const void* p, int64_t ld, int64_t rows, int64_t cols, int high, int32_t type) {
    const uint64_t dims[2] = {(uint64_t)cols, (uint64_t)rows}, strides[1] = {(uint64_t)ld * 2};
    const uint32_t box[2] = {64, (uint32_t)high};
    return encode_map(map, map_type(type), 2, p, dims, strides, box);
}
// [E, N, K] read in boxes of 64 columns and `high` rows of one bucket
static int weight_map(CUtensorMap* map, const void* p, int64_t ld, int64_t E, int64_t N, int64_t K, int high, int32_t type) {
    const uint64_t dims[3] = {(uint64_t)K, (uint64_t)N, (uint64_t)E}, strides[2] = {(uint64_t)ld * 2, (uint64_t)(N * ld) * 2};
    const uint32_t box[3] = {64, (uint32_t)high, 1};
    return encode_map(map, map_type(type), 3, p, dims, strides, box);
}
// x or dy: in the batch's order (gathered) or laid out by bucket
static int operand_map(CUtensorMap* map, GlArgs* a, bool laid, const void* p, int64_t ld, int64_t T, int64_t cols, int32_t E, int32_t type) {
    a->gather = !laid;
    return laid ? rows_map(map, p, (cols + 7) / 8 * 8, group_laid_rows(T, E), cols, kGroupRows, type) : rows_map(map, p, ld, T, cols, 1, type);
}

static int check_grouped(const char* what, const void* plan, int64_t T, int64_t K, int64_t N, int32_t E, int32_t type) {
    NNUE_REQUIRE(T >= 0 && K > 0 && N > 0 && E > 0, NNUE_ERR_ARG, "%s: sizes T=%lld K=%lld N=%lld E=%d", what, (long long)T,
                 (long long)K, (long long)N, E);
    NNUE_REQUIRE(E <= kMaxGroups && T <= NNUE_GROUP_MAX_ROWS && K < (1 << 24) && N < (1 << 24), NNUE_ERR_UNSUPPORTED,
                 "%s: sizes T=%lld K=%lld N=%lld E=%d beyond the kernels' range", what, (long long)T, (long long)K, (long long)N, E);
    NNUE_REQUIRE(is_half_type(type), NNUE_ERR_UNSUPPORTED, "%s: operand type %d is neither bf16 nor fp16", what, type);
    NNUE_REQUIRE(plan && aligned16(plan), NNUE_ERR_ARG, "%s: null or unaligned plan", what);
    return NNUE_OK;
}

static int check_operand(const char* what, const char* name, const void* p, int64_t ld, int64_t cols, int32_t type) {
    NNUE_REQUIRE(p, NNUE_ERR_ARG, "%s: null %s", what, name);
    NNUE_REQUIRE(ld >= cols, NNUE_ERR_ARG, "%s: pitch %lld of %s below its %lld columns", what, (long long)ld, name, (long long)cols);
    NNUE_REQUIRE(aligned16(p) && ld * type_bytes(type) % 16 == 0, NNUE_ERR_ALIGN,
                 "%s: rows of %s must start at multiples of 16 bytes", what, name);
    return NNUE_OK;
}

static int common_args(const char* what, GlArgs* a, const void* plan, int64_t T, int64_t N, int32_t E, int32_t type, void* out,
                       int32_t out_type, int64_t cols) {
    *a = GlArgs{};
    a->plan = group_view(plan, T, E);
    a->o = rows_out(out, out_type, cols);
    a->T = (int32_t)T;
    a->E = E;
    a->N = (int32_t)N;
    a->row_tiles = 1;
    a->idesc = type == NNUE_T_BF16 ? 1u : 0u;  // the operands' format; the rest of the descriptor follows the tile
    a->status = device_status_ptr();
    NNUE_REQUIRE(a->status, NNUE_ERR_CUDA, "%s: no device status word", what);
    return NNUE_OK;
}

}  // namespace nnue

using namespace nnue;

extern "C" int nnue_grouped_linear_fwd(const void* x, int64_t ldx, int32_t laid, const void* w, int64_t ldw, const void* bias,
                                       int32_t bias_type, const void* plan, void* y, int32_t y_type, int64_t T, int64_t K,
                                       int64_t N, int32_t E, int32_t type, void* stream) {
    const char* what = "nnue_grouped_linear_fwd";
    if (int st = check_grouped(what, plan, T, K, N, E, type)) return st;
    NNUE_REQUIRE(y_type == NNUE_T_F32 || y_type == type, NNUE_ERR_UNSUPPORTED, "%s: output type %d", what, y_type);
    NNUE_REQUIRE(!bias || is_float_type(bias_type), NNUE_ERR_UNSUPPORTED, "%s: bias type %d", what, bias_type);
    if (T == 0) return NNUE_OK;
    if (int st = check_operand(what, "x", x, laid ? (K + 7) / 8 * 8 : ldx, K, type)) return st;
    if (int st = check_operand(what, "weight", w, ldw, K, type)) return st;
    NNUE_REQUIRE(y && aligned16(y), NNUE_ERR_ALIGN, "%s: null or unaligned output", what);
    GlArgs a;
    if (int st = common_args(what, &a, plan, T, N, E, type, y, y_type, N)) return st;
    a.bias = bias;
    a.bias_type = bias_type;
    a.red = (int32_t)K;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ProfScope prof("grouped_fwd", s);
    const int64_t runs = E < T ? E : T;
    const TileShape shape = tile_shape(runs, (T + runs - 1) / runs, N, (K + kGlK - 1) / kGlK, 32, 256, laid);
    CUtensorMap ma, mb;
    if (int st = operand_map(&ma, &a, laid, x, ldx, T, K, E, type)) return st;
    if (int st = weight_map(&mb, w, ldw, E, N, K, shape.bn / shape.ctas, type)) return st;
    return gl_run<kModeFwd>(ma, mb, a, group_max_tiles(T, E), shape, s);
}

extern "C" int nnue_grouped_linear_bwd_input(const void* dy, int64_t lddy, int32_t laid, const void* w, int64_t ldw, const void* plan,
                                             void* dx, int64_t T, int64_t K, int64_t N, int32_t E, int32_t type, void* stream) {
    const char* what = "nnue_grouped_linear_bwd_input";
    if (int st = check_grouped(what, plan, T, K, N, E, type)) return st;
    if (T == 0) return NNUE_OK;
    if (int st = check_operand(what, "dy", dy, laid ? (N + 7) / 8 * 8 : lddy, N, type)) return st;
    if (int st = check_operand(what, "weight", w, ldw, K, type)) return st;
    NNUE_REQUIRE(dx && aligned16(dx), NNUE_ERR_ALIGN, "%s: null or unaligned output", what);
    GlArgs a;
    if (int st = common_args(what, &a, plan, T, N, E, type, dx, type, K)) return st;
    a.red = (int32_t)N;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ProfScope prof("grouped_dx", s);
    const int64_t runs = E < T ? E : T;
    const TileShape shape = tile_shape(runs, (T + runs - 1) / runs, K, (N + kGlK - 1) / kGlK, 64, 256, laid);
    CUtensorMap ma, mb;
    if (int st = operand_map(&ma, &a, laid, dy, lddy, T, N, E, type)) return st;
    if (int st = weight_map(&mb, w, ldw, E, N, K, 64, type)) return st;
    return gl_run<kModeDx>(ma, mb, a, group_max_tiles(T, E), shape, s);
}

extern "C" int nnue_grouped_linear_bwd_weight(const void* dy, const float* dy_sums, const void* x, const void* plan, void* dw,
                                              int32_t dw_type, void* dbias, int32_t dbias_type, int64_t T, int64_t K, int64_t N,
                                              int32_t E, int32_t type, void* stream) {
    const char* what = "nnue_grouped_linear_bwd_weight";
    if (int st = check_grouped(what, plan, T, K, N, E, type)) return st;
    NNUE_REQUIRE(dw_type == NNUE_T_F32 || dw_type == type, NNUE_ERR_UNSUPPORTED, "%s: type %d", what, dw_type);
    NNUE_REQUIRE(!dbias || is_float_type(dbias_type), NNUE_ERR_UNSUPPORTED, "%s: bias type %d", what, dbias_type);
    if (T > 0) {
        if (int st = check_operand(what, "dy", dy, (N + 7) / 8 * 8, N, type)) return st;
        if (int st = check_operand(what, "x", x, (K + 7) / 8 * 8, K, type)) return st;
        NNUE_REQUIRE(!dbias || dy_sums, NNUE_ERR_ARG, "%s: the bias gradient needs dy's sums", what);
    }
    NNUE_REQUIRE(dw && aligned16(dw), NNUE_ERR_ALIGN, "%s: null or unaligned output", what);
    GlArgs a;
    if (int st = common_args(what, &a, plan, T, N, E, type, dw, dw_type, K)) return st;
    a.sums = dbias;
    a.sums_type = dbias_type;
    a.tile_sums = dy_sums;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ProfScope prof("grouped_dw", s);
    const int64_t mean = (T + E - 1) / E;
    const TileShape shape = tile_shape(E, N, K, (mean + kGlK - 1) / kGlK, 64, 256, true);
    a.row_tiles = (int32_t)((N + kGroupRows * shape.ctas - 1) / (kGroupRows * shape.ctas));
    CUtensorMap ma, mb;
    if (T > 0) {
        if (int st = rows_map(&ma, dy, (N + 7) / 8 * 8, group_laid_rows(T, E), N, kGlK, type)) return st;
        if (int st = rows_map(&mb, x, (K + 7) / 8 * 8, group_laid_rows(T, E), K, kGlK, type)) return st;
    } else {  // no row is read: any valid map
        if (int st = rows_map(&ma, dw, 64, 1, 1, 1, type)) return st;
        mb = ma;
    }
    return gl_run<kModeDw>(ma, mb, a, (int64_t)E * a.row_tiles, shape, s);
}
