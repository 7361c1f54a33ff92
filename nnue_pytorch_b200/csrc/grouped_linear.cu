// Bucketed ("grouped by expert") linear layer on 16-bit operands, on the 5th-generation tensor cores:
//   forward          y[p, n]     = sum_k x[p, k] w[b, n, k] + bias[b, n]        b = bucket of row p
//   input gradient   dx[p, k]    = sum_n dy[p, n] w[b, n, k]
//   weight gradient  dw[b, n, k] = sum_{p of b} dy[p, n] x[p, k],  dbias[b, n] = sum_{p of b} dy[p, n]
//
// One kernel, three ways to read its operands; D (128 rows x BN columns) accumulates in tensor memory in fp32.
//   forward   A = 128 rows of x of one bucket, gathered by the plan, K-major;   B = rows of w, K-major
//   dx        A = 128 rows of dy, gathered, K-major;                       B = columns of w, MN-major (w is read as it lies)
//   dw        A = columns of dy, B = columns of x, both MN-major; the sum runs over the bucket's rows, gathered
// Rows behind the end of a bucket are zeros where the sum runs over rows and never read elsewhere; no row of another bucket
// is ever multiplied.  (Gathering with TMA, four rows per copy, was measured first: about 75 cycles per copy and SM whatever
// issues it, 675 us for the forward of 16384 x 4096 x 2048 and 1700 for its dw.)
//
// Roles: warps 0-3 copy into a ring of shared-memory stages (128 bytes of K or of M/N per row, swizzled; gathered rows 16
// bytes per thread, w as TMA boxes), one thread of warp 4 issues the instructions, warps 5-8 bring finished tiles out while
// the next tile multiplies (two accumulators), and in dw warps 9-12 add up the bias gradient from the same stages.  Persistent: a CTA per SM walks the tiles with a
// stride of the grid.  With few tiles the sum is split over a cluster of 2 to 8 CTAs, whose partial tiles meet in
// distributed shared memory and are added in the order of their ranks.  All orders are fixed by the sizes: results are
// reproducible.  Every wait is bounded; one that runs out raises the device status word and the CTA leaves, its tensor
// memory freed and its copies in.
#include "grouped.cuh"
#include "tc.cuh"

namespace nnue {

enum { kModeFwd = 0, kModeDx = 1, kModeDw = 2 };

constexpr int kGlK = 64;                     // reduction elements per stage: one 128-byte swizzle row
constexpr int kGlABytes = kGroupRows * 128;  // 16 KiB
constexpr int kGlBoxBytes = kGlK * 128;      // MN-major block: 64 rows of the reduction x 128 bytes
constexpr int kGlStageWarp = 4096;           // staging of one output warp: 32 rows x 128 bytes

constexpr int gl_stages(int bn) { return bn == 256 ? 4 : bn == 128 ? 6 : 8; }
constexpr int gl_stage_bytes(int bn) { return kGlABytes + bn * 128; }
constexpr int gl_threads(int mode) { return mode == kModeDw ? 416 : 288; }
constexpr int gl_smem(int bn) {  // alignment, ring, staging, bias per output warp, bias gradient, barriers
    return 1024 + gl_stages(bn) * gl_stage_bytes(bn) + 4 * kGlStageWarp + 4 * bn * 4 + kGroupRows * 4 + 256;
}

struct GlArgs {
    GroupPlanView plan;
    const unsigned char *rows_a, *rows_b;  // gathered operands: x (forward), dy (dx), dy and x (dw)
    int64_t pitch_a, pitch_b;              // bytes
    void* out;
    void* sums;              // dw: dbias, or null
    const void* bias;        // forward, or null
    int64_t ld_out;          // elements
    int32_t out_type, sums_type, bias_type;
    int32_t T, E, N;         // N: rows of w per bucket
    int32_t red, cols;       // length of the reduction (forward, dx); columns of the output
    int32_t col_tiles;       // ceil(cols / BN)
    int32_t row_tiles;       // dw: ceil(N / 128)
    int32_t vec;             // rows of `out` start at multiples of 16 bytes
    uint32_t idesc;
    unsigned long long* status;
};

// One tile of the output and the part of its sum that this CTA adds up.
struct GlTile {
    int32_t bucket, first, count;  // rows order[first .. first + count): the tile's rows or (dw) the bucket's
    int32_t row0, col0;            // dw: first row inside the bucket's matrix; first column
    int32_t c0, c1;                // chunks of the reduction
    bool live;                     // false: rows without a bucket
};

template <int MODE, int BN, bool SPLIT>
__device__ __forceinline__ GlTile gl_tile(const GlArgs& a, int t, int rank, int ranks) {
    GlTile x;
    const int rt = t / a.col_tiles, ct = t - rt * a.col_tiles;
    x.col0 = ct * BN;
    int chunks;
    if (MODE == kModeDw) {
        x.bucket = rt / a.row_tiles;
        x.row0 = (rt - x.bucket * a.row_tiles) * kGroupRows;
        x.first = __ldg(a.plan.offsets + x.bucket);
        x.count = __ldg(a.plan.offsets + x.bucket + 1) - x.first;
        chunks = (x.count + kGlK - 1) / kGlK;
        x.live = true;
    } else {
        const int4 g = __ldg(reinterpret_cast<const int4*>(a.plan.tiles) + rt);
        x.bucket = g.x;
        x.first = g.y;
        x.count = g.z;
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

// Position in the ring of stages.
template <int S>
struct GlRing {
    int stage = 0;
    unsigned phase = 0;
    __device__ __forceinline__ void next() {
        if (++stage == S) {
            stage = 0;
            phase ^= 1u;
        }
    }
};

// A pass of columns (`bytes` per row in the warp's staging, 16-byte pieces swizzled) to the rows of the output, in whole
// 128- or 64-byte pieces of rows.  Lane r holds row r's place in the output, or -1.
__device__ __forceinline__ void gl_copy_out(const GlArgs& a, const unsigned char* stg, int bytes, int32_t my_row, int64_t row_base,
                                            int col) {
    const int lane = threadIdx.x & 31;
    const int es = a.out_type == NNUE_T_F32 ? 4 : 2;
    unsigned char* out = static_cast<unsigned char*>(a.out);
    __syncwarp();
    if (a.vec) {
        const int shift = bytes == 128 ? 3 : 2, piece = lane & ((1 << shift) - 1);
        const bool inside = col + piece * (16 / es) < a.cols;  // cols is a multiple of a piece
#pragma unroll
        for (int it = 0; it < 8; ++it) {
            const int r = (it << (5 - shift)) + (lane >> shift);
            const int32_t row = __shfl_sync(kFullMask, my_row, r & 31);
            if (r >= 32 || row < 0 || !inside) continue;
            const uint4 v = *reinterpret_cast<const uint4*>(stg + r * 128 + ((piece ^ (r & 7)) << 4));
            *reinterpret_cast<uint4*>(out + ((row_base + row) * a.ld_out + col) * es + piece * 16) = v;
        }
    } else {
#pragma unroll 1
        for (int r = 0; r < 32; ++r) {
            const int32_t row = __shfl_sync(kFullMask, my_row, r);
            if (row < 0) continue;
            for (int j = lane; j < bytes / es && col + j < a.cols; j += 32) {
                const unsigned char* src = stg + r * 128 + (((j * es / 16) ^ (r & 7)) << 4) + j * es % 16;
                unsigned char* dst = out + ((row_base + row) * a.ld_out + col + j) * es;
                if (es == 4) *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(src);
                else *reinterpret_cast<uint16_t*>(dst) = *reinterpret_cast<const uint16_t*>(src);
            }
        }
    }
    __syncwarp();
}

__device__ __forceinline__ uint32_t pack_half(float a, float b, int32_t type) {
    if (type == NNUE_T_BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// One output warp: its 32 rows of the tile, from tensor memory (or zeros) to the output.
template <int BN>
__device__ __forceinline__ void gl_bring_out(const GlArgs& a, uint32_t taddr, bool zeros, const float* s_bias, unsigned char* stg,
                                             int32_t my_row, int64_t row_base, int col0) {
    const int lane = threadIdx.x & 31;
    const bool f32 = a.out_type == NNUE_T_F32;
    const bool wide = !f32 && BN >= 64;  // two reads of 32 columns make one 128-byte piece of a row
#pragma unroll 1
    for (int c = 0; c < BN && col0 + c < a.cols; c += wide ? 64 : 32) {
#pragma unroll 1
        for (int h = 0; h < (wide ? 2 : 1); ++h) {
            uint32_t v[32];
            if (zeros) {
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = 0u;
            } else {
                tmem_ld32(taddr + c + 32 * h, v);
                tmem_wait_ld();
                if (s_bias) {
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const float4 b = *reinterpret_cast<const float4*>(s_bias + c + 32 * h + j);
                        v[j] = __float_as_uint(__uint_as_float(v[j]) + b.x);
                        v[j + 1] = __float_as_uint(__uint_as_float(v[j + 1]) + b.y);
                        v[j + 2] = __float_as_uint(__uint_as_float(v[j + 2]) + b.z);
                        v[j + 3] = __float_as_uint(__uint_as_float(v[j + 3]) + b.w);
                    }
                }
            }
            if (f32) {
#pragma unroll
                for (int p = 0; p < 8; ++p)
                    *reinterpret_cast<uint4*>(stg + lane * 128 + ((p ^ (lane & 7)) << 4)) =
                        make_uint4(v[4 * p], v[4 * p + 1], v[4 * p + 2], v[4 * p + 3]);
            } else {
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    uint32_t w[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        w[j] = pack_half(__uint_as_float(v[8 * p + 2 * j]), __uint_as_float(v[8 * p + 2 * j + 1]), a.out_type);
                    *reinterpret_cast<uint4*>(stg + lane * 128 + (((4 * h + p) ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
        gl_copy_out(a, stg, f32 || wide ? 128 : 64, my_row, row_base, col0 + c);
    }
}

// ---- warps 0-3: copies ------------------------------------------------------------------------------------------------
// Gathered rows come 16 bytes per thread and copy: eight neighbouring threads read 128 bytes of one row, a thread serves
// rows j / 8 + 16 i.  Copies announce themselves on the stage's barrier when they land; the thread does not wait.
template <int MODE, int BN, bool SPLIT>
__device__ __forceinline__ bool gl_copy_role(const GlArgs& a, const CUtensorMap* map_b, uint32_t ring, uint64_t* full,
                                             uint64_t* empty, int t0, int stride, int tiles, int rank, int ranks) {
    constexpr int S = gl_stages(BN);
    const int j = threadIdx.x, lane = j & 31, piece = j & 7, r0 = j >> 3;
    const uint32_t dst0 = r0 * 128 + ((piece ^ (r0 & 7)) << 4);
    GlRing<S> at;
    bool ok = true;
    for (int t = t0; t < tiles && ok; t += stride) {
        const GlTile x = gl_tile<MODE, BN, SPLIT>(a, t, rank, ranks);
        if (x.c0 == x.c1) continue;
        constexpr int kRows = MODE == kModeDw ? 4 : 8;
        int rows[kRows];
        auto rows_of = [&](int i0, int(&r)[kRows]) {  // rows i0 + r0 + 16 i of the tile's or bucket's list; -1 behind its end
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                const int k = i0 + r0 + 16 * i;
                r[i] = k < x.count ? __ldg(a.plan.order + x.first + k) : -1;
            }
        };
        rows_of(MODE == kModeDw ? x.c0 * kGlK : 0, rows);
        for (int c = x.c0; c < x.c1; ++c) {
            int ahead[kRows];
            if (MODE == kModeDw) rows_of((c + 1) * kGlK, ahead);  // on their way while this stage is awaited
            if (lane == 0) ok = mbar_wait_timed(empty + at.stage, at.phase ^ 1u);
            ok = __shfl_sync(kFullMask, ok, 0);
            if (!ok) break;
            const uint32_t sa = ring + at.stage * gl_stage_bytes(BN), sb = sa + kGlABytes;
            uint64_t* bar = full + at.stage;
            if (MODE == kModeDw) {
                const int n = 16 * gl_steps<MODE>(a, x, c);
#pragma unroll
                for (int i = 0; i < kRows; ++i) {
                    if (16 * i >= n) break;
                    const bool live = rows[i] >= 0;
                    const unsigned char* pa = a.rows_a + (live ? rows[i] * a.pitch_a : 0);
                    const unsigned char* pb = a.rows_b + (live ? rows[i] * a.pitch_b : 0);
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const int col = x.row0 + b * 64 + piece * 8;
                        if (x.row0 + b * 64 < a.N) cp_async16_n(sa + b * kGlBoxBytes + dst0 + i * 2048, pa, col, live ? a.N - col : 0);
                    }
#pragma unroll
                    for (int b = 0; b < BN / 64; ++b) {
                        const int col = x.col0 + b * 64 + piece * 8;
                        if (x.col0 + b * 64 < a.cols) cp_async16_n(sb + b * kGlBoxBytes + dst0 + i * 2048, pb, col, live ? a.cols - col : 0);
                    }
                }
#pragma unroll
                for (int i = 0; i < kRows; ++i) rows[i] = ahead[i];
            } else {
                if (j < (MODE == kModeFwd ? 1 : BN / 64)) {  // w comes as whole boxes
                    if (MODE == kModeFwd) {
                        mbar_expect_tx(bar, BN * 128);
                        tma_tile_3d(sb, map_b, c * kGlK, x.col0, x.bucket, bar);
                    } else {
                        const int boxes = min(BN / 64, (a.cols - x.col0 + 63) >> 6);
                        if (j == 0) mbar_expect_tx(bar, boxes * kGlBoxBytes);
                        if (j < boxes) tma_tile_3d(sb + j * kGlBoxBytes, map_b, x.col0 + j * 64, c * kGlK, x.bucket, bar);
                    }
                }
                const int col = c * kGlK + piece * 8;
#pragma unroll
                for (int i = 0; i < kRows; ++i)
                    if (rows[i] >= 0) cp_async16_n(sa + dst0 + i * 2048, a.rows_a + rows[i] * a.pitch_a, col, a.red - col);
            }
            cp_async_arrive(bar);
            at.next();
        }
    }
    if (!ok) cp_async_wait<0>();  // copies in flight land before the CTA leaves; w's boxes are older than the wait that ran out
    return ok;
}

// ---- one thread: the instructions -------------------------------------------------------------------------------------
template <int MODE, int BN, bool SPLIT>
__device__ __forceinline__ bool gl_issue_role(const GlArgs& a, uint32_t tmem, uint32_t ring, uint64_t* full, uint64_t* empty,
                                              uint64_t* done, uint64_t* taken, uint64_t* drained, int t0, int stride, int tiles,
                                              int rank, int ranks) {
    constexpr bool kAMn = MODE == kModeDw, kBMn = MODE != kModeFwd;
    constexpr uint32_t kAStep = kAMn ? 2048 >> 4 : 32 >> 4, kBStep = kBMn ? 2048 >> 4 : 32 >> 4;  // 16 reduction elements
    GlRing<gl_stages(BN)> at;
    int acc = 0;
    unsigned acc_phase = 0;
    bool ok = true;
    for (int t = t0; t < tiles && ok; t += stride) {
        const GlTile x = gl_tile<MODE, BN, SPLIT>(a, t, rank, ranks);
        if (x.c0 == x.c1) continue;
        ok = mbar_wait_timed(taken + acc, acc_phase ^ 1u);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem + acc * BN;
        for (int c = x.c0; c < x.c1; ++c) {
            ok = mbar_wait_timed(full + at.stage, at.phase);
            if (!ok) break;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the gathered rows were written by ordinary copies
            tc_fence_after();
            const uint32_t sa = ring + at.stage * gl_stage_bytes(BN);
            const uint64_t da = umma_desc_sw128(sa, kGlBoxBytes), db = umma_desc_sw128(sa + kGlABytes, kGlBoxBytes);
            const int steps = gl_steps<MODE>(a, x, c);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (k < steps) umma_f16(d, da + k * kAStep, db + k * kBStep, a.idesc, c != x.c0 || k != 0);
            umma_commit_to(empty + at.stage);
            at.next();
        }
        if (!ok) break;
        umma_commit_to(done + acc);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
    }
    if (!ok) {  // instructions in flight finish before the tensor memory is freed
        umma_commit_to(drained);
        mbar_wait_timed(drained, 0);
    }
    return ok;
}

// ---- dw: sums of the columns of dy --------------------------------------------------------------------------------------
// Thread n adds column n of the A stages: the bucket's rows in order, 64 at a time (two levels, so that long buckets lose no
// precision).  Reads beside the tensor core's, no byte of dy more.
template <int BN, bool SPLIT>
__device__ __forceinline__ bool gl_sums_role(const GlArgs& a, const unsigned char* ring, uint64_t* full, uint64_t* empty,
                                             float* s_sums, int t0, int stride, int tiles, int rank, int ranks) {
    const int n = threadIdx.x - 288, lane = threadIdx.x & 31;
    GlRing<gl_stages(BN)> at;
    bool ok = true;
    for (int t = t0; t < tiles && ok; t += stride) {
        const GlTile x = gl_tile<kModeDw, BN, SPLIT>(a, t, rank, ranks);
        const bool wanted = a.sums && x.col0 == 0;
        float total = 0.f;
        for (int c = x.c0; c < x.c1; ++c) {
            ok = mbar_wait_timed(full + at.stage, at.phase);
            if (__any_sync(kFullMask, !ok)) {
                ok = false;
                break;
            }
            if (wanted) {
                const unsigned char* col = ring + at.stage * gl_stage_bytes(BN) + (n >> 6) * kGlBoxBytes;
                const int piece = (n & 63) >> 3, in = (n & 7) * 2, rows = 16 * gl_steps<kModeDw>(a, x, c);
                float sum = 0.f;
#pragma unroll 8
                for (int r = 0; r < rows; ++r) {
                    const uint16_t v = *reinterpret_cast<const uint16_t*>(col + r * 128 + ((piece ^ (r & 7)) << 4) + in);
                    sum += a.idesc >> 7 & 1 ? __uint_as_float((uint32_t)v << 16) : __half2float(__ushort_as_half(v));
                }
                total += sum;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + at.stage);
            at.next();
        }
        if (SPLIT) s_sums[n] = total;
        else if (ok && wanted && x.row0 + n < a.N) store_from_float(a.sums, a.sums_type, (int64_t)x.bucket * a.N + x.row0 + n, total);
    }
    return ok;
}

template <int MODE, int BN, bool SPLIT>
__global__ void __launch_bounds__(gl_threads(MODE), 1)
    k_grouped(const __grid_constant__ CUtensorMap map_b, const __grid_constant__ GlArgs a) {
    constexpr int S = gl_stages(BN);
    constexpr uint32_t kTmemCols = 2 * BN;
    constexpr int kPartPitch = BN + 4;  // floats per row of a partial tile
    extern __shared__ unsigned char smem_raw[];
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
    unsigned char* ring_ptr = smem_raw + (ring - smem_u32(smem_raw));
    unsigned char* staging = ring_ptr + S * gl_stage_bytes(BN);
    float* s_bias = reinterpret_cast<float*>(staging + 4 * kGlStageWarp);  // [4][BN], one copy per output warp
    float* s_sums = s_bias + 4 * BN;                                       // [128] dw, split: this CTA's bias gradient
    uint64_t* full = reinterpret_cast<uint64_t*>(s_sums + kGroupRows);     // [S] a stage's copies are in
    uint64_t* empty = full + S;                                            // [S] a stage may be overwritten
    uint64_t* done = empty + S;                                            // [2] an accumulator is complete
    uint64_t* taken = done + 2;                                            // [2] an accumulator has been read
    uint64_t* drained = taken + 2;                                         // [1]
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(drained + 1);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int rank = 0, ranks = 1;
    if (SPLIT) {
        rank = (int)cluster_rank();
        uint32_t n;
        asm volatile("mov.u32 %0, %cluster_nctaid.x;" : "=r"(n));
        ranks = (int)n;
    }
    const int tiles = (MODE == kModeDw ? a.E * a.row_tiles : __ldg(a.plan.n_tiles)) * a.col_tiles;
    const int t0 = (int)blockIdx.x / ranks, stride = (int)gridDim.x / ranks;  // split: at most one tile per cluster
    if (t0 >= tiles) return;                                                  // (the whole cluster)

    if (tid == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(full + s, MODE == kModeDw ? 128 : 129);  // the copying threads, and the boxes of w
            mbar_init(empty + s, MODE == kModeDw ? 5 : 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(done + s, 1);
            mbar_init(taken + s, 4);
        }
        mbar_init(drained, 1);
        fence_barrier_init();
        if (MODE != kModeDw) prefetch_map(&map_b);
    }
    if (warp == 4) tmem_alloc(s_tmem, kTmemCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;

    bool ok = true;
    if (warp < 4) {
        ok = gl_copy_role<MODE, BN, SPLIT>(a, &map_b, ring, full, empty, t0, stride, tiles, rank, ranks);
    } else if (warp == 4) {
        if (lane == 0) ok = gl_issue_role<MODE, BN, SPLIT>(a, tmem, ring, full, empty, done, taken, drained, t0, stride, tiles, rank, ranks);
    } else if (warp < 9) {
        const int q = warp & 3;  // the quarter of tensor memory's lanes that this warp may read
        float* my_bias = s_bias + q * BN;
        int acc = 0;
        unsigned acc_phase = 0;
        for (int t = t0; t < tiles && ok; t += stride) {
            const GlTile x = gl_tile<MODE, BN, SPLIT>(a, t, rank, ranks);
            const bool some = x.c1 > x.c0;
            if (SPLIT) {
                if (some) {
                    ok = mbar_wait_timed(done, 0);
                    if (__any_sync(kFullMask, !ok)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                }
                break;
            }
            const int r = q * 32 + lane;
            int32_t my_row;
            int64_t row_base = 0;
            if (MODE == kModeDw) {
                my_row = x.row0 + r < a.N ? x.row0 + r : -1;
                row_base = (int64_t)x.bucket * a.N;
            } else {
                my_row = r < x.count ? __ldg(a.plan.order + x.first + r) : -1;
            }
            const bool biased = MODE == kModeFwd && a.bias && x.live;
            if (biased) {
                for (int j = lane; j < BN; j += 32)
                    my_bias[j] = x.col0 + j < a.cols ? load_as_float(a.bias, a.bias_type, (int64_t)x.bucket * a.N + x.col0 + j) : 0.f;
                __syncwarp();
            }
            if (some) {
                ok = mbar_wait_timed(done + acc, acc_phase);
                if (__any_sync(kFullMask, !ok)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
            }
            if (q * 32 < x.count || MODE == kModeDw)
                gl_bring_out<BN>(a, tmem + ((uint32_t)(q * 32) << 16) + acc * BN, !some, biased ? my_bias : nullptr,
                                 staging + q * kGlStageWarp, my_row, row_base, x.col0);
            if (some) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(taken + acc);
                acc ^= 1;
                if (acc == 0) acc_phase ^= 1u;
            }
        }
    } else {
        ok = gl_sums_role<BN, SPLIT>(a, ring_ptr, full, empty, s_sums, t0, stride, tiles, rank, ranks);
    }
    __syncwarp();
    if (!ok && lane == 0) note_timeout(a.status);

    if (SPLIT) {
        __syncthreads();  // nobody reads the ring any more: the partial tile takes its place
        const GlTile x = gl_tile<MODE, BN, SPLIT>(a, t0, rank, ranks);
        if (warp >= 5 && warp < 9) {
            const int q = warp & 3;
            float* part = reinterpret_cast<float*>(ring_ptr) + (q * 32 + lane) * kPartPitch;
#pragma unroll 1
            for (int c = 0; c < BN; c += 32) {
                uint32_t v[32];
                if (x.c1 > x.c0) {
                    tmem_ld32(tmem + ((uint32_t)(q * 32) << 16) + c, v);
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = 0u;
                }
#pragma unroll
                for (int j = 0; j < 32; j += 4)
                    *reinterpret_cast<uint4*>(part + c + j) = make_uint4(v[j], v[j + 1], v[j + 2], v[j + 3]);
            }
        }
        cluster_sync();
        // row r of the tile is finished by rank r mod ranks: partial sums in the order of the ranks
        const int rows = MODE == kModeDw ? min(kGroupRows, a.N - x.row0) : x.count;
        const int mine = (rows - rank + ranks - 1) / ranks;
        const int es = a.out_type == NNUE_T_F32 ? 4 : 2;
        for (int i = tid; i < mine * (BN / 4); i += gl_threads(MODE)) {
            const int r = rank + i / (BN / 4) * ranks, c = i % (BN / 4) * 4, col = x.col0 + c;
            if (col >= a.cols) continue;
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
                    if (col + j < a.cols) v[j] += load_as_float(a.bias, a.bias_type, (int64_t)x.bucket * a.N + col + j);
            }
            const int64_t row = MODE == kModeDw ? (int64_t)x.bucket * a.N + x.row0 + r : (int64_t)__ldg(a.plan.order + x.first + r);
            const int64_t at = row * a.ld_out + col;
            if (a.vec && es == 4) {
                *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = make_float4(v[0], v[1], v[2], v[3]);
            } else if (a.vec) {
                *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) =
                    make_uint2(pack_half(v[0], v[1], a.out_type), pack_half(v[2], v[3], a.out_type));
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (col + j < a.cols) store_from_float(a.out, a.out_type, at + j, v[j]);
            }
        }
        if (MODE == kModeDw && a.sums && x.col0 == 0 && rank == 0 && tid < rows) {
            float total = 0.f;
            for (int s = 0; s < ranks; ++s) {
                float v;
                asm volatile(
                    "{\n\t.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.f32 %0, [a];\n\t}"
                    : "=f"(v)
                    : "r"(smem_u32(s_sums + tid)), "r"(s)
                    : "memory");
                total += v;
            }
            store_from_float(a.sums, a.sums_type, (int64_t)x.bucket * a.N + x.row0 + tid, total);
        }
        cluster_sync();  // nobody leaves while its shared memory is read
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 4) tmem_free(tmem, kTmemCols);
}

// ---- host ---------------------------------------------------------------------------------------------------------------
template <int MODE, int BN, bool SPLIT>
int gl_launch(const CUtensorMap& mb, const GlArgs& a, int64_t tiles, int ranks, cudaStream_t s) {
    auto kernel = k_grouped<MODE, BN, SPLIT>;
    static bool opted[64] = {};  // more than 48 KB of dynamic shared memory needs the opt-in, once per device
    int dev = 0;
    NNUE_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !opted[dev]) {
        NNUE_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, gl_smem(BN)));
        if (dev >= 0 && dev < 64) opted[dev] = true;
    }
    const int64_t ctas = SPLIT ? tiles * ranks : (tiles < sm_count() ? tiles : sm_count());
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(gl_threads(MODE));
    cfg.dynamicSmemBytes = gl_smem(BN);
    cfg.stream = s;
    cudaLaunchAttribute attr;
    if (SPLIT) {
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = (unsigned)ranks;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
    }
    NNUE_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, mb, a));
    note_launches(1);
    return NNUE_OK;
}

// Width of a tile and parts of its sum.  `row_tiles` is an estimate of the tiles along the rows (exact in dw), `chunks` the
// length of the reduction in stages.  The widest tile that still gives every SM one; where even the narrowest leaves SMs
// idle, the sum is split while every part keeps two stages.
struct GlShape {
    int bn, ranks;
};
static GlShape gl_shape(int64_t row_tiles, int64_t cols, int64_t chunks, int narrowest) {
    const int64_t sms = sm_count();
    int bn = 256;
    while (bn > narrowest && (row_tiles * ((cols + bn - 1) / bn) < sms || cols <= bn / 2)) bn /= 2;
    const int64_t tiles = row_tiles * ((cols + bn - 1) / bn);
    int ranks = 1;
    while (ranks < 8 && tiles * ranks * 2 <= sms && chunks >= ranks * 4) ranks *= 2;
    return {bn, ranks};
}

template <int MODE>
int gl_run(const CUtensorMap& mb, GlArgs& a, int64_t tile_rows, GlShape shape, cudaStream_t s) {
    a.col_tiles = (a.cols + shape.bn - 1) / shape.bn;
    a.idesc = umma_idesc(a.idesc, (uint32_t)shape.bn, MODE == kModeDw, MODE != kModeFwd);
    const int64_t tiles = tile_rows * a.col_tiles;
    NNUE_REQUIRE(tiles * 8 < 0x7fffffffLL, NNUE_ERR_UNSUPPORTED, "grouped linear: too many tiles");
    if (MODE == kModeFwd && shape.bn == 32)
        return shape.ranks > 1 ? gl_launch<MODE, MODE == kModeFwd ? 32 : 64, true>(mb, a, tiles, shape.ranks, s)
                               : gl_launch<MODE, MODE == kModeFwd ? 32 : 64, false>(mb, a, tiles, 1, s);
    if (shape.bn == 64)
        return shape.ranks > 1 ? gl_launch<MODE, 64, true>(mb, a, tiles, shape.ranks, s)
                               : gl_launch<MODE, 64, false>(mb, a, tiles, 1, s);
    if (shape.bn == 128)
        return shape.ranks > 1 ? gl_launch<MODE, 128, true>(mb, a, tiles, shape.ranks, s)
                               : gl_launch<MODE, 128, false>(mb, a, tiles, 1, s);
    return shape.ranks > 1 ? gl_launch<MODE, 256, true>(mb, a, tiles, shape.ranks, s)
                           : gl_launch<MODE, 256, false>(mb, a, tiles, 1, s);
}

static CUtensorMapDataType map_type(int32_t type) {
    return type == NNUE_T_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}
// [E, N, K] read in boxes of 64 columns and `high` rows of one bucket
static int weight_map(CUtensorMap* map, const void* p, int64_t ld, int64_t E, int64_t N, int64_t K, int high, int32_t type) {
    const uint64_t dims[3] = {(uint64_t)K, (uint64_t)N, (uint64_t)E}, strides[2] = {(uint64_t)ld * 2, (uint64_t)(N * ld) * 2};
    const uint32_t box[3] = {64, (uint32_t)high, 1};
    return encode_map(map, map_type(type), 3, p, dims, strides, box);
}

// tiles along the rows to expect: full ones, and one more per bucket in use
static int64_t expected_row_tiles(int64_t T, int64_t E) {
    const int64_t n = T / kGroupRows + E;
    return n < T ? n : T;
}

// dst[r, c] = src[r, c], rows of another type or pitch; columns [cols, ldd) of dst become zero
__global__ void __launch_bounds__(kThreads)
    k_pack_rows(const void* __restrict__ src, int src_type, int64_t lds, void* __restrict__ dst, int dst_type, int64_t ldd,
                int64_t rows, int64_t cols) {
    const int64_t per = (ldd + kThreads - 1) / kThreads;
    for (int64_t i = blockIdx.x; i < rows * per; i += gridDim.x) {
        const int64_t r = i / per, c = (i % per) * kThreads + threadIdx.x;
        if (c >= ldd) continue;
        if (type_is_byte(src_type)) {
            static_cast<uint8_t*>(dst)[r * ldd + c] = c < cols ? static_cast<const uint8_t*>(src)[r * lds + c] : 0;
            continue;
        }
        store_from_float(dst, dst_type, r * ldd + c, c < cols ? load_as_float(src, src_type, r * lds + c) : 0.f);
    }
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
    a->out = out;
    a->ld_out = cols;
    a->out_type = out_type;
    a->T = (int32_t)T;
    a->E = E;
    a->N = (int32_t)N;
    a->cols = (int32_t)cols;
    a->row_tiles = 1;
    a->vec = cols * type_bytes(out_type) % 16 == 0;
    a->idesc = type == NNUE_T_BF16 ? 1u : 0u;  // the operands' format; the rest of the descriptor follows the tile
    a->status = device_status_ptr();
    NNUE_REQUIRE(a->status, NNUE_ERR_CUDA, "%s: no device status word", what);
    return NNUE_OK;
}

}  // namespace nnue

using namespace nnue;

extern "C" int nnue_pack_rows(const void* src, int32_t src_type, int64_t lds, void* dst, int32_t dst_type, int64_t ldd,
                              int64_t rows, int64_t cols, void* stream) {
    NNUE_REQUIRE(rows >= 0 && cols >= 0 && lds >= cols && ldd >= cols, NNUE_ERR_ARG, "nnue_pack_rows: bad sizes");
    NNUE_REQUIRE((is_float_type(src_type) && is_float_type(dst_type)) || (type_bytes(src_type) == 1 && src_type == dst_type),
                 NNUE_ERR_UNSUPPORTED, "nnue_pack_rows: no conversion from type %d to %d", src_type, dst_type);
    if (rows == 0 || ldd == 0) return NNUE_OK;
    NNUE_REQUIRE(src && dst, NNUE_ERR_ARG, "nnue_pack_rows: null pointer");
    const int64_t blocks = rows * ((ldd + kThreads - 1) / kThreads);
    k_pack_rows<<<(unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)), kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        src, src_type, lds, dst, dst_type, ldd, rows, cols);
    note_launches(1);
    NNUE_CUDA_TRY(cudaGetLastError());
    return NNUE_OK;
}

extern "C" int nnue_grouped_linear_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias,
                                       int32_t bias_type, const void* plan, void* y, int32_t y_type, int64_t T, int64_t K,
                                       int64_t N, int32_t E, int32_t type, void* stream) {
    if (int st = check_grouped("nnue_grouped_linear_fwd", plan, T, K, N, E, type)) return st;
    NNUE_REQUIRE(y_type == NNUE_T_F32 || y_type == type, NNUE_ERR_UNSUPPORTED, "nnue_grouped_linear_fwd: output type %d", y_type);
    NNUE_REQUIRE(!bias || is_float_type(bias_type), NNUE_ERR_UNSUPPORTED, "nnue_grouped_linear_fwd: bias type %d", bias_type);
    if (T == 0) return NNUE_OK;
    if (int st = check_operand("nnue_grouped_linear_fwd", "x", x, ldx, K, type)) return st;
    if (int st = check_operand("nnue_grouped_linear_fwd", "weight", w, ldw, K, type)) return st;
    NNUE_REQUIRE(y && aligned16(y), NNUE_ERR_ALIGN, "nnue_grouped_linear_fwd: null or unaligned output");
    GlArgs a;
    if (int st = common_args("nnue_grouped_linear_fwd", &a, plan, T, N, E, type, y, y_type, N)) return st;
    a.bias = bias;
    a.bias_type = bias_type;
    a.red = (int32_t)K;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ProfScope prof("grouped_fwd", s);
    const GlShape shape = gl_shape(expected_row_tiles(T, E), N, (K + kGlK - 1) / kGlK, 32);
    a.rows_a = static_cast<const unsigned char*>(x);
    a.pitch_a = ldx * 2;
    CUtensorMap mb;
    if (int st = weight_map(&mb, w, ldw, E, N, K, shape.bn, type)) return st;
    return gl_run<kModeFwd>(mb, a, group_max_tiles(T, E), shape, s);
}

extern "C" int nnue_grouped_linear_bwd_input(const void* dy, int64_t lddy, const void* w, int64_t ldw, const void* plan, void* dx,
                                             int64_t T, int64_t K, int64_t N, int32_t E, int32_t type, void* stream) {
    if (int st = check_grouped("nnue_grouped_linear_bwd_input", plan, T, K, N, E, type)) return st;
    if (T == 0) return NNUE_OK;
    if (int st = check_operand("nnue_grouped_linear_bwd_input", "dy", dy, lddy, N, type)) return st;
    if (int st = check_operand("nnue_grouped_linear_bwd_input", "weight", w, ldw, K, type)) return st;
    NNUE_REQUIRE(dx && aligned16(dx), NNUE_ERR_ALIGN, "nnue_grouped_linear_bwd_input: null or unaligned output");
    GlArgs a;
    if (int st = common_args("nnue_grouped_linear_bwd_input", &a, plan, T, N, E, type, dx, type, K)) return st;
    a.red = (int32_t)N;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ProfScope prof("grouped_dx", s);
    const GlShape shape = gl_shape(expected_row_tiles(T, E), K, (N + kGlK - 1) / kGlK, 64);
    a.rows_a = static_cast<const unsigned char*>(dy);
    a.pitch_a = lddy * 2;
    CUtensorMap mb;
    if (int st = weight_map(&mb, w, ldw, E, N, K, 64, type)) return st;
    return gl_run<kModeDx>(mb, a, group_max_tiles(T, E), shape, s);
}

extern "C" int nnue_grouped_linear_bwd_weight(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* plan, void* dw,
                                              int32_t dw_type, void* dbias, int32_t dbias_type, int64_t T, int64_t K, int64_t N,
                                              int32_t E, int32_t type, void* stream) {
    if (int st = check_grouped("nnue_grouped_linear_bwd_weight", plan, T, K, N, E, type)) return st;
    NNUE_REQUIRE(dw_type == NNUE_T_F32 || dw_type == type, NNUE_ERR_UNSUPPORTED, "nnue_grouped_linear_bwd_weight: type %d", dw_type);
    NNUE_REQUIRE(!dbias || is_float_type(dbias_type), NNUE_ERR_UNSUPPORTED, "nnue_grouped_linear_bwd_weight: bias type %d", dbias_type);
    if (T > 0) {
        if (int st = check_operand("nnue_grouped_linear_bwd_weight", "dy", dy, lddy, N, type)) return st;
        if (int st = check_operand("nnue_grouped_linear_bwd_weight", "x", x, ldx, K, type)) return st;
    }
    NNUE_REQUIRE(dw && aligned16(dw), NNUE_ERR_ALIGN, "nnue_grouped_linear_bwd_weight: null or unaligned output");
    GlArgs a;
    if (int st = common_args("nnue_grouped_linear_bwd_weight", &a, plan, T, N, E, type, dw, dw_type, K)) return st;
    a.sums = dbias;
    a.sums_type = dbias_type;
    a.row_tiles = (int32_t)((N + kGroupRows - 1) / kGroupRows);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ProfScope prof("grouped_dw", s);
    const int64_t row_tiles = (int64_t)E * a.row_tiles, mean = (T + E - 1) / E;
    const GlShape shape = gl_shape(row_tiles, K, (mean + kGlK - 1) / kGlK, 64);
    a.rows_a = static_cast<const unsigned char*>(dy);
    a.pitch_a = lddy * 2;
    a.rows_b = static_cast<const unsigned char*>(x);
    a.pitch_b = ldx * 2;
    const CUtensorMap none = {};  // both operands are gathered
    return gl_run<kModeDw>(none, a, row_tiles, shape, s);
}
