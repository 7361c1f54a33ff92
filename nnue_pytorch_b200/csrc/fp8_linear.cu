// Linear layer on 8-bit operands with a scale per 128 inputs of a row and per 128 x 128 tile of the weights, dense or
// bucketed, on the 5th-generation tensor cores:
//   y[p, n] = sum_c sx[p, c] sw[b, n / 128, c] sum_{k in block c} x[p, k] w[b, n, k] + bias[b, n]
//
// A stage is one block of 128 inputs (a 128-byte swizzle row per operand row), four tcgen05.mma of 32 inputs each, whose
// sum goes to an accumulator of its own in tensor memory.  Eight warps take the accumulators one after the other, multiply
// them by sx * sw and add them up in fp32 registers (a thread holds half a row of the tile; its row's scale is one number,
// and so is the weights' on its columns); another warp fetches the scales, which may be any fp32 numbers.
// Bound by the way of an accumulator, not by the tensor core: a stage of a pair of SMs on 256 x 256 multiplies in 390 cycles,
// but its first result is there after 900, is read and scaled in 700 to 900 and given back in 240, and tensor memory holds
// two: about 1000 cycles per stage (16384 x 4096 x 2048 over 8 buckets: 180 us, 1.53 PFLOP/s; 135 us of it are stages at
// work, 20 to 40 the bringing out of eight tiles per pair).  Four accumulators of 128 columns halve the way but double the
// stages (223 us, when 256 columns took 178), and two products of 128 columns per stage came to 219.
// Copies, pairs of SMs, split sums and bounded waits as in the 16-bit kernel (grouped_linear.cu).  Rows come laid out by
// bucket (the quantiser leaves them so), in their own order where there is one matrix, or are gathered by TMA, four per
// copy, where a bucket has few.
#include "grouped_tc.cuh"

#include <type_traits>

namespace nnue {

constexpr int kF8K = 128;
constexpr int kF8ABytes = kGroupRows * 128;
constexpr int kF8Threads = 384;  // copies, instructions, scales, a warp without work, eight output warps
constexpr int kF8OutWarp = 4;    // the first output warp
// An output thread of the widest tile holds 128 sums and two reads of 32 columns: the first warpgroup gives registers up.
constexpr int kF8FewRegs = 72, kF8ManyRegs = 216, kF8LaunchRegs = 168;
static_assert(128 * kF8FewRegs + 256 * kF8ManyRegs <= kF8Threads * kF8LaunchRegs, "more registers than the launch brings");

constexpr int f8_stage_bytes(int bn, int ctas) { return kF8ABytes + bn / ctas * 128; }
constexpr int f8_accs(int bn) { return bn == 256 ? 2 : 4; }
constexpr int kF8Groups = 2;  // groups of scales of four stages each
constexpr int kF8Slots = 4 * kF8Groups;
constexpr int f8_slot_floats(int bn) { return kGroupRows * (bn == 256 ? 2 : 1); }
constexpr int f8_rest(int bn) { return 1024 + 8 * kStagingBytes + kF8Slots * f8_slot_floats(bn) * 4 + 512; }  // alignment, staging, scales, barriers
constexpr int f8_stages(int bn, int ctas) { return (232448 - f8_rest(bn)) / f8_stage_bytes(bn, ctas); }  // what 227 KB hold
constexpr int f8_smem(int bn, int ctas) { return f8_rest(bn) + f8_stages(bn, ctas) * f8_stage_bytes(bn, ctas); }

struct F8Args {
    GroupPlanView plan;
    RowsOut o;
    const float *x_scale, *w_scale, *bias;
    int64_t scale_ld;    // 0: x_scale [T, C] by rows of the batch; else [C, scale_ld] by the rows' places in x
    int32_t scale_vec;   // the latter, four rows at a time
    int32_t T, E, N, K;
    int32_t C, R;        // blocks along K and along N
    int32_t col_tiles;
    int32_t dense;       // one matrix, rows in their own order
    int32_t gather;
    uint32_t idesc;
    unsigned long long* status;
};

struct F8Tile {
    int32_t bucket, first, count, place, col0, c0, c1;
    bool live;
};

template <int BN, int CTAS, bool SPLIT>
__device__ __forceinline__ F8Tile f8_tile(const F8Args& a, int t, int rank, int ranks) {
    F8Tile x;
    const int rt = t / a.col_tiles;
    x.col0 = (t - rt * a.col_tiles) * BN;
    if (a.dense) {
        x.bucket = 0;
        x.first = x.place = rt * (kGroupRows * CTAS);
        x.count = min(kGroupRows * CTAS, a.T - x.first);
    } else {
        const int4 g = __ldg(reinterpret_cast<const int4*>(CTAS == 2 ? a.plan.pairs : a.plan.tiles) + rt);
        x.bucket = g.x;
        x.first = g.y;
        x.count = g.z;
        x.place = g.w;
    }
    x.live = x.bucket < a.E;
    const int chunks = x.live ? a.C : 0;
    x.c0 = SPLIT ? chunks * rank / ranks : 0;
    x.c1 = SPLIT ? chunks * (rank + 1) / ranks : chunks;
    return x;
}

template <int BN, int CTAS, bool SPLIT>
__device__ __forceinline__ bool f8_copy_role(const F8Args& a, const CUtensorMap* map_x, const CUtensorMap* map_w, uint32_t ring,
                                             uint64_t* full, uint64_t* empty, int t0, int stride, int tiles, int rank, int ranks) {
    constexpr bool PAIR = CTAS == 2;
    const int lane = threadIdx.x & 31, side = PAIR ? rank : 0;
    StageRing<f8_stages(BN, CTAS)> at;
    bool ok = true;
    for (int t = t0; t < tiles && ok; t += stride) {
        const F8Tile x = f8_tile<BN, CTAS, SPLIT>(a, t, rank, ranks);
        if (x.c0 == x.c1) continue;
        const bool gather = !PAIR && a.gather;
        // the bytes that complete a stage: both CTAs' of a pair, announced by the first
        const int bytes = BN * 128 + (gather ? ((x.count + 3) >> 2) * 512 : (PAIR && x.count > kGroupRows ? 2 : 1) * kF8ABytes);
        int rows[4];
        if (gather) {
#pragma unroll
            for (int j = 0; j < 4; ++j) rows[j] = 4 * lane + j < x.count ? __ldg(a.plan.order + x.first + 4 * lane + j) : a.T;
        }
        for (int c = x.c0; c < x.c1; ++c) {
            if (lane == 0) ok = mbar_wait_timed(empty + at.stage, at.phase ^ 1u);
            ok = __shfl_sync(kFullMask, (int)ok, 0) != 0;
            if (!ok) break;
            const uint32_t sa = ring + at.stage * f8_stage_bytes(BN, CTAS), sb = sa + kF8ABytes;
            const uint32_t bar = PAIR ? map_rank(full + at.stage, 0) : smem_u32(full + at.stage);
            if (lane == 0) {
                if (!PAIR || rank == 0) mbar_expect_tx(full + at.stage, bytes);
                if (!gather && x.count > side * kGroupRows) tma_tile_2d<PAIR>(sa, map_x, c * kF8K, x.place + side * kGroupRows, bar);
                tma_tile_3d<PAIR>(sb, map_w, c * kF8K, x.col0 + side * (BN / CTAS), x.bucket, bar);
            }
            if (gather) {
                __syncwarp();
                if (4 * lane < x.count) tma_gather4(sa + lane * 512, map_x, c * kF8K, rows[0], rows[1], rows[2], rows[3], bar);
            }
            at.next();
        }
    }
    return ok;
}

template <int BN, int CTAS, bool SPLIT>
__device__ __forceinline__ bool f8_issue_role(const F8Args& a, uint32_t tmem, uint32_t ring, uint64_t* full, uint64_t* empty,
                                              uint64_t* done, uint64_t* taken, uint64_t* drained, int t0, int stride, int tiles,
                                              int rank, int ranks) {
    constexpr bool PAIR = CTAS == 2;
    StageRing<f8_stages(BN, CTAS)> at;
    StageRing<f8_accs(BN)> acc;
    bool ok = true;
    for (int t = t0; t < tiles && ok; t += stride) {
        const F8Tile x = f8_tile<BN, CTAS, SPLIT>(a, t, rank, ranks);
        for (int c = x.c0; c < x.c1; ++c) {
            ok = mbar_wait_warp(taken + acc.stage, acc.phase ^ 1u) && mbar_wait_warp(full + at.stage, at.phase);
            if (!ok) break;
            tc_fence_after();
            const uint32_t sa = ring + at.stage * f8_stage_bytes(BN, CTAS);
            const uint64_t da = umma_desc_sw128(sa, 16), db = umma_desc_sw128(sa + kF8ABytes, 16);
            const int steps = min(4, (a.K - c * kF8K + 31) >> 5);  // instructions of 32 inputs
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (k < steps) umma_f8<PAIR>(tmem + acc.stage * BN, da + 2 * k, db + 2 * k, a.idesc, k != 0);
                umma_commit_to<PAIR>(empty + at.stage);
                umma_commit_to<PAIR>(done + acc.stage);
            }
            __syncwarp();
            at.next();
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

// s * v + acc, two numbers at once, each product-sum rounded once
__device__ __forceinline__ void fma2(float& a0, float& a1, uint32_t v0, uint32_t v1, float s) {
    unsigned long long a, v, ss;
    asm("mov.b64 %0, {%1, %2};" : "=l"(a) : "f"(a0), "f"(a1));
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(v0), "r"(v1));
    asm("mov.b64 %0, {%1, %1};" : "=l"(ss) : "f"(s));
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(a) : "l"(v), "l"(ss));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a0), "=f"(a1) : "l"(a));
}

// A block's sum is multiplied by sx * sw at once where that product is a normal number.  Else an output warp multiplies by the
// larger scale first: what comes out in range then meets neither an overflow nor a loss of digits on the way (the smaller
// one only takes it down where the product is too small, up where it is too large).  A second loop does that from the first
// such group of a tile on: the first loop pays one test per group (16384 x 4096 x 2048 over 8 buckets: 180 us for 175;
// with the test in every stage of one loop 213).
__device__ __forceinline__ bool is_normal(float p) { return fabsf(p) >= 1.17549435e-38f && fabsf(p) <= 3.40282347e38f; }

// One warp: sx * sw of every row and half of the columns, four stages at a time, into the ring that the output warps read.
// (As loads of the output warps themselves they were waited for in every stage: their registers hold the sums.)
template <int BN, int CTAS, bool SPLIT>
__device__ __forceinline__ bool f8_scale_role(const F8Args& a, float* slots, int* apart, uint64_t* sfull, uint64_t* sfree, int t0, int stride,
                                              int tiles, int rank, int ranks) {
    constexpr int kHalves = f8_slot_floats(BN) / kGroupRows;
    const int lane = threadIdx.x & 31, r0 = 4 * lane + (CTAS == 2 ? rank * kGroupRows : 0);
    StageRing<kF8Groups> at;
    for (int t = t0; t < tiles; t += stride) {
        const F8Tile x = f8_tile<BN, CTAS, SPLIT>(a, t, rank, ranks);
        const int left = x.count - r0;  // rows of the lane's four that there are
        const float* sx[4];
        const int64_t step = a.scale_ld ? a.scale_ld : 1;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = j < left ? r0 + j : 0;
            sx[j] = a.x_scale + (a.scale_ld ? x.place + r : (int64_t)(a.dense ? x.first + r : x.live ? __ldg(a.plan.order + x.first + r) : 0) * a.C);
        }
        const float* sw[kHalves];
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
            sw[h] = a.w_scale + ((int64_t)(x.live ? x.bucket : 0) * a.R + min(x.col0 / kF8K + h, a.R - 1)) * a.C;
        for (int c4 = x.c0; c4 < x.c1; c4 += 4) {
            float v[4][4], w[4][kHalves];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = min(c4 + i, x.c1 - 1);
                if (a.scale_vec && left >= 4) {
                    const float4 f = __ldg(reinterpret_cast<const float4*>(sx[0] + c * step));
                    v[i][0] = f.x;
                    v[i][1] = f.y;
                    v[i][2] = f.z;
                    v[i][3] = f.w;
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[i][j] = j < left ? __ldg(sx[j] + c * step) : 1.f;  // 1: rows that there are not
                }
#pragma unroll
                for (int h = 0; h < kHalves; ++h) w[i][h] = __ldg(sw[h] + c);
            }
            if (!mbar_wait_warp(sfree + at.stage, at.phase ^ 1u)) return false;
            float* to = slots + at.stage * 4 * f8_slot_floats(BN) + 4 * lane;
            float least = 1.f, most = 1.f;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int h = 0; h < kHalves; ++h) {
                    const float4 p = make_float4(v[i][0] * w[i][h], v[i][1] * w[i][h], v[i][2] * w[i][h], v[i][3] * w[i][h]);
                    *reinterpret_cast<float4*>(to + i * f8_slot_floats(BN) + h * kGroupRows) = p;
                    least = fminf(fminf(least, fminf(fabsf(p.x), fabsf(p.y))), fminf(fabsf(p.z), fabsf(p.w)));
                    most = fmaxf(fmaxf(most, fmaxf(fabsf(p.x), fabsf(p.y))), fmaxf(fabsf(p.z), fabsf(p.w)));
                }
            const bool odd = __any_sync(kFullMask, !is_normal(least) || !is_normal(most));
            if (lane == 0) apart[at.stage] = odd;
            __syncwarp();
            if (lane == 0) mbar_arrive(sfull + at.stage);
            at.next();
        }
    }
    return true;
}

// An output warp's 32 rows and half of the columns, from registers to the output.
template <int HALF>
__device__ __forceinline__ void f8_bring_out(const F8Args& a, const F8Tile& x, float (&acc)[HALF], unsigned char* stg, int32_t my_row,
                                             int col) {
    const int lane = threadIdx.x & 31;
    if (a.bias && x.live) {
        float* b = reinterpret_cast<float*>(stg);
        for (int j = lane; j < HALF; j += 32) b[j] = col + j < a.o.cols ? __ldg(a.bias + (int64_t)x.bucket * a.N + col + j) : 0.f;
        __syncwarp();
#pragma unroll
        for (int j = 0; j < HALF; j += 4) {
            const float4 v = *reinterpret_cast<const float4*>(b + j);
            acc[j] += v.x;
            acc[j + 1] += v.y;
            acc[j + 2] += v.z;
            acc[j + 3] += v.w;
        }
        __syncwarp();
    }
    bring_out<0, HALF>(a.o, acc, stg, my_row, 0, col);
}

template <int BN, int CTAS, bool SPLIT>
__device__ __forceinline__ bool f8_output_role(const F8Args& a, uint32_t tmem, uint64_t* done, uint64_t* taken, const float* slots,
                                               const int* s_apart, uint64_t* sfull, uint64_t* sfree, unsigned char* ring_ptr, unsigned char* staging,
                                               int t0, int stride, int tiles, int rank, int ranks) {
    constexpr bool PAIR = CTAS == 2;
    constexpr int A = f8_accs(BN), HALF = BN / 2;  // HALF: columns of an output warp
    const int warp = (threadIdx.x >> 5) - kF8OutWarp, lane = threadIdx.x & 31;
    const int q = warp & 3, half = warp >> 2;  // the quarter of tensor memory's lanes, the half of the columns
    const int r = (PAIR ? rank * kGroupRows : 0) + q * 32 + lane;
    const uint32_t from = tmem + ((uint32_t)(q * 32) << 16) + half * HALF;
    const float* my_scale = slots + (BN == 256 ? half * kGroupRows : 0) + q * 32 + lane;
    unsigned char* stg = staging + warp * kStagingBytes;
    StageRing<A> at;
    StageRing<kF8Groups> sat;
    F8Tile x = f8_tile<BN, CTAS, SPLIT>(a, t0, rank, ranks);
    for (int t = t0; t < tiles; t += stride) {
        // the next tile is looked up while this one multiplies
        const F8Tile next = f8_tile<BN, CTAS, SPLIT>(a, t + stride < tiles ? t + stride : t, rank, ranks);
        const int32_t my_row = r >= x.count ? -1 : a.dense ? x.first + r : __ldg(a.plan.order + x.first + r);
        const int col = x.col0 + half * HALF;
        float acc[HALF];
#pragma unroll
        for (int j = 0; j < HALF; ++j) acc[j] = 0.f;
        // Two reads of 32 columns are under way at any time, the first two of the next stage during this one's last products.
        constexpr int kReads = HALF / 32;
        uint32_t v[2][32];
        if (x.c0 < x.c1) {
            if (!mbar_wait_warp(done + at.stage, at.phase)) return false;
            tc_fence_after();
#pragma unroll
            for (int h = 0; h < 2 && h < kReads; ++h) tmem_ld32(from + at.stage * BN + 32 * h, v[h]);
        }
        // One stage; APART: some row's two scales may have to be multiplied one after the other.
        auto stage = [&](auto odd, int c) {
            constexpr bool APART = decltype(odd)::value;
            const int in_group = (c - x.c0) & 3;
            float scale = my_scale[(sat.stage * 4 + in_group) * f8_slot_floats(BN)], before = 1.f;
            if (APART && !is_normal(scale)) {
                const int tile = min(x.col0 / kF8K + (BN == 256 ? half : 0), a.R - 1);
                const float sx = my_row < 0 ? 1.f : __ldg(a.x_scale + (a.scale_ld ? x.place + r + c * a.scale_ld : (int64_t)my_row * a.C + c));
                const float sw = my_row < 0 ? 1.f : __ldg(a.w_scale + ((int64_t)x.bucket * a.R + tile) * a.C + c);
                before = fabsf(sx) < fabsf(sw) ? sw : sx;
                scale = fabsf(sx) < fabsf(sw) ? sx : sw;
            }
            const bool more = c + 1 < x.c1;
            const int now = at.stage;
            at.next();
            tmem_wait_ld(v[0]);
            if (kReads > 1) tmem_wait_ld(v[1]);
#pragma unroll
            for (int h = 0; h < kReads; ++h) {
                if (h + 2 == kReads || kReads == 1) {  // all of it is in registers: the accumulator goes back
                    if (h > 0) {
                        tmem_wait_ld(v[0]);
                        tmem_wait_ld(v[1]);
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if (PAIR) mbar_arrive_cluster(map_rank(taken + now, 0));
                        else mbar_arrive(taken + now);
                        if (in_group == 3 || !more) mbar_arrive(sfree + sat.stage);
                    }
                }
                if (APART) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[h & 1][j] = __float_as_uint(__uint_as_float(v[h & 1][j]) * before);
                }
#pragma unroll
                for (int j = 0; j < 32; j += 2) fma2(acc[32 * h + j], acc[32 * h + j + 1], v[h & 1][j], v[h & 1][j + 1], scale);
                if (h + 2 < kReads) {
                    tmem_ld32(from + now * BN + 32 * (h + 2), v[h & 1]);
                } else if (more) {
                    if (h + 2 == kReads || kReads == 1) {
                        if (!mbar_wait_warp(done + at.stage, at.phase)) return false;
                        tc_fence_after();
                    }
                    tmem_ld32(from + at.stage * BN + 32 * (h & 1), v[h & 1]);
                }
            }
            if (in_group == 3 || !more) sat.next();
            return true;
        };
        int c = x.c0;
#pragma unroll 1
        for (; c < x.c1; ++c) {
            if (((c - x.c0) & 3) == 0) {
                if (!mbar_wait_warp(sfull + sat.stage, sat.phase)) return false;
                if (s_apart[sat.stage]) break;
            }
            if (!stage(std::false_type(), c)) return false;
        }
#pragma unroll 1
        for (; c < x.c1; ++c) {  // from the first group with such scales on
            if (((c - x.c0) & 3) == 0 && !mbar_wait_warp(sfull + sat.stage, sat.phase)) return false;
            if (!stage(std::true_type(), c)) return false;
        }
        if (SPLIT) {
            // the last accumulator is complete, so nothing reads the ring any more: it takes the partial tile
            float* part = reinterpret_cast<float*>(ring_ptr) + (q * 32 + lane) * (BN + 4) + half * HALF;
#pragma unroll
            for (int j = 0; j < HALF; j += 4) *reinterpret_cast<float4*>(part + j) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
            break;
        }
        if (__any_sync(kFullMask, my_row >= 0) && col < a.o.cols) f8_bring_out<HALF>(a, x, acc, stg, my_row, col);
        x = next;
    }
    return true;
}

// Split sums: row r of the tile is finished by rank r mod ranks, partial sums in the order of the ranks.
template <int BN>
__device__ __forceinline__ void f8_join(const F8Args& a, const F8Tile& x, uint32_t ring, int rank, int ranks) {
    const int mine = (x.count - rank + ranks - 1) / ranks;
    for (int i = threadIdx.x - kF8OutWarp * 32; i < mine * (BN / 4); i += kF8Threads - kF8OutWarp * 32) {
        const int r = rank + i / (BN / 4) * ranks, c = i % (BN / 4) * 4, col = x.col0 + c;
        if (col >= a.o.cols) continue;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (x.live) {
            const uint32_t addr = ring + (uint32_t)(r * (BN + 4) + c) * 4;
            for (int s = 0; s < ranks; ++s) {
                const float4 p = ld_cluster4(addr, (uint32_t)s);
                v[0] += p.x;
                v[1] += p.y;
                v[2] += p.z;
                v[3] += p.w;
            }
            if (a.bias) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (col + j < a.o.cols) v[j] += __ldg(a.bias + (int64_t)x.bucket * a.N + col + j);
            }
        }
        const int64_t row = a.dense ? x.first + r : __ldg(a.plan.order + x.first + r), at = row * a.o.ld + col;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (col + j < a.o.cols) store_from_float(a.o.out, a.o.type, at + j, v[j]);
    }
}

template <int BN, int CTAS, bool SPLIT>
__global__ void __launch_bounds__(kF8Threads, 1)
    k_fp8_linear(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ F8Args a) {
    constexpr bool PAIR = CTAS == 2;
    constexpr int S = f8_stages(BN, CTAS), A = f8_accs(BN);
    constexpr uint32_t kTmemCols = A * BN;
    static_assert(!(PAIR && SPLIT), "no such variant");
    extern __shared__ unsigned char smem_raw[];
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
    unsigned char* ring_ptr = smem_raw + (ring - smem_u32(smem_raw));
    unsigned char* staging = ring_ptr + S * f8_stage_bytes(BN, CTAS);
    float* slots = reinterpret_cast<float*>(staging + 8 * kStagingBytes);
    uint64_t* full = reinterpret_cast<uint64_t*>(slots + kF8Slots * f8_slot_floats(BN));  // [S] a stage's copies are in (pair: the first CTA's)
    uint64_t* empty = full + S;                                                 // [S] a stage may be overwritten
    uint64_t* done = empty + S;                                                 // [A] an accumulator is complete
    uint64_t* taken = done + A;                                                 // [A] an accumulator has been read
    uint64_t* sfull = taken + A;                                                // [kF8Groups] a group of scales is there
    uint64_t* sfree = sfull + kF8Groups;                                        // [kF8Groups] and has been read
    uint64_t* drained = sfree + kF8Groups;                                      // [1]
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(drained + 1);
    int* s_apart = reinterpret_cast<int*>(s_tmem + 1);                          // [kF8Groups] a product of two scales of the group is not normal

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int rank = 0, ranks = 1;
    if (SPLIT || PAIR) {
        rank = (int)cluster_rank();
        uint32_t n;
        asm volatile("mov.u32 %0, %cluster_nctaid.x;" : "=r"(n));
        ranks = (int)n;
    }
    const int row_tiles = a.dense ? (a.T + kGroupRows * CTAS - 1) / (kGroupRows * CTAS) : __ldg(a.plan.n_tiles + (PAIR ? 1 : 0));
    const int tiles = row_tiles * a.col_tiles;
    const int t0 = (int)blockIdx.x / ranks, stride = (int)gridDim.x / ranks;  // split: at most one tile per cluster
    if (t0 >= tiles) return;                                                  // (the whole cluster)

    if (tid == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(full + s, 1);
            mbar_init(empty + s, 1);
        }
        for (int s = 0; s < A; ++s) {
            mbar_init(done + s, 1);
            mbar_init(taken + s, 8 * CTAS);
        }
        for (int s = 0; s < kF8Groups; ++s) {
            mbar_init(sfull + s, 1);
            mbar_init(sfree + s, 8);
        }
        mbar_init(drained, 1);
        fence_barrier_init();
        prefetch_map(&map_x);
        prefetch_map(&map_w);
    }
    if (warp == 1) tmem_alloc<PAIR>(s_tmem, kTmemCols);
    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();  // the other CTA's barriers are there
    tc_fence_after();
    const uint32_t tmem = *s_tmem;

    if (warp < kF8OutWarp) {
        if (BN == 256) fewer_registers<kF8FewRegs>();
        bool ok = true;
        if (warp == 0) {
            ok = f8_copy_role<BN, CTAS, SPLIT>(a, &map_x, &map_w, ring, full, empty, t0, stride, tiles, rank, ranks);
        } else if (warp == 1) {
            if (!(PAIR && rank != 0))
                ok = f8_issue_role<BN, CTAS, SPLIT>(a, tmem, ring, full, empty, done, taken, drained, t0, stride, tiles, rank, ranks);
        } else if (warp == 2) {
            ok = f8_scale_role<BN, CTAS, SPLIT>(a, slots, s_apart, sfull, sfree, t0, stride, tiles, rank, ranks);
        }
        __syncwarp();
        if (!ok && lane == 0) note_timeout(a.status);
        if (SPLIT) {
            cluster_sync();
            cluster_sync();
        }
    } else {
        if (BN == 256) more_registers<kF8ManyRegs>();
        const bool ok = f8_output_role<BN, CTAS, SPLIT>(a, tmem, done, taken, slots, s_apart, sfull, sfree, ring_ptr, staging, t0, stride, tiles, rank, ranks);
        if (!ok && lane == 0) note_timeout(a.status);
        if (SPLIT) {
            __syncwarp();
            cluster_sync();
            f8_join<BN>(a, f8_tile<BN, CTAS, SPLIT>(a, t0, rank, ranks), ring, rank, ranks);
            __syncwarp();
            cluster_sync();  // nobody leaves while its shared memory is read
        }
    }
    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();  // both have read their tensor memory, and nobody's barriers are arrived on any more
    if (warp == 1) tmem_free<PAIR>(tmem, kTmemCols);
}

template <int BN, int CTAS, bool SPLIT>
int f8_launch(const CUtensorMap& mx, const CUtensorMap& mw, const F8Args& a, int64_t tiles, int ranks, cudaStream_t s) {
    auto kernel = k_fp8_linear<BN, CTAS, SPLIT>;
    static bool opted[64] = {};  // more than 48 KB of dynamic shared memory needs the opt-in, once per device
    int dev = 0;
    NNUE_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !opted[dev]) {
        NNUE_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, f8_smem(BN, CTAS)));
        cudaFuncAttributes attr;
        NNUE_CUDA_TRY(cudaFuncGetAttributes(&attr, kernel));
        NNUE_REQUIRE(BN != 256 || attr.numRegs >= kF8LaunchRegs, NNUE_ERR_UNSUPPORTED, "fp8 linear: built with %d registers per thread", attr.numRegs);
        if (dev >= 0 && dev < 64) opted[dev] = true;
    }
    const int64_t at_once = sm_count() / CTAS;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(SPLIT ? tiles * ranks : (tiles < at_once ? tiles : at_once) * CTAS));
    cfg.blockDim = dim3(kF8Threads);
    cfg.dynamicSmemBytes = f8_smem(BN, CTAS);
    cfg.stream = s;
    cudaLaunchAttribute attr;
    if (SPLIT || CTAS > 1) {
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = (unsigned)(SPLIT ? ranks : CTAS);
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
    }
    NNUE_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, mx, mw, a));
    note_launches(1);
    return NNUE_OK;
}

// Pairs on 256 columns or CTAs on up to 128.  A round of the latter takes about 5/8 of a pair's round for half the work.
// Pairs and single CTAs, us, the kept one first:
//   pairs   2048 x 4096 x 2048 28, 35      4096 x 4096 x 4096 89, 102      16384 x 4096 x 2048 over 8 even buckets 157, 203
//           8192 x 2048 x 512 over 8 21, 23      16384 x 512 x 512 over 8 18.5 to 19.5, 17.8 (the rule's one miss of these)
//   single  4099 x 2000 x 1500 49, 54      20000 x 1000 x 520 over 3 34, 38      6000 x 1024 x 1000 over 2 21, 24
// Pairs on 128 columns took 223 for 180 at 16384 x 4096 x 2048 over 8 uneven buckets.
static TileShape f8_shape(int64_t runs, int64_t T, int64_t N, int64_t chunks, bool pairs) {
    const int64_t rows = (T + runs - 1) / runs, sms = sm_count();
    auto rounds = [&](int64_t high, int64_t wide, int64_t at_once) {
        return (runs * ((rows + high - 1) / high) * ((N + wide - 1) / wide) + at_once - 1) / at_once;
    };
    const TileShape narrow = tile_shape(runs, rows, N, chunks, 64, 128, false);
    if (pairs && narrow.bn == 128 && rows > kGroupRows && rounds(kGroupPairRows, 256, sms / 2) * 8 <= rounds(kGroupRows, 128, sms) * 5)
        return {256, 2, 1};
    return narrow;
}

}  // namespace nnue

using namespace nnue;

extern "C" int nnue_fp8_linear_fwd(const void* x, int64_t ldx, int32_t laid, const float* x_scale, int64_t scale_ld, const void* w, int64_t ldw,
                                   const float* w_scale, const float* bias, const void* plan, void* y, int32_t y_type, int64_t T,
                                   int64_t K, int64_t N, int32_t E, int32_t format, void* stream) {
    const char* what = "nnue_fp8_linear_fwd";
    NNUE_REQUIRE(T >= 0 && K > 0 && N > 0 && E > 0, NNUE_ERR_ARG, "%s: sizes T=%lld K=%lld N=%lld E=%d", what, (long long)T,
                 (long long)K, (long long)N, E);
    NNUE_REQUIRE(E <= kMaxGroups && T <= NNUE_GROUP_MAX_ROWS && K < (1 << 24) && N < (1 << 24), NNUE_ERR_UNSUPPORTED,
                 "%s: sizes T=%lld K=%lld N=%lld E=%d beyond the kernel's range", what, (long long)T, (long long)K, (long long)N, E);
    NNUE_REQUIRE(format == NNUE_T_E4M3 || format == NNUE_T_E5M2, NNUE_ERR_UNSUPPORTED, "%s: format %d", what, format);
    NNUE_REQUIRE(is_float_type(y_type), NNUE_ERR_UNSUPPORTED, "%s: output type %d", what, y_type);
    NNUE_REQUIRE(plan || E == 1, NNUE_ERR_ARG, "%s: %d buckets need a plan", what, E);
    NNUE_REQUIRE(plan || !laid, NNUE_ERR_ARG, "%s: rows laid out by bucket need their plan", what);
    if (T == 0) return NNUE_OK;
    NNUE_REQUIRE(x && w && x_scale && w_scale && y, NNUE_ERR_ARG, "%s: null pointer", what);
    if (laid) ldx = (K + 15) / 16 * 16;
    NNUE_REQUIRE(scale_ld == 0 || (!plan && scale_ld >= T) || (laid && scale_ld >= group_laid_rows(T, E)), NNUE_ERR_ARG,
                 "%s: scales by place need rows laid out by bucket, or one matrix, and room for every row", what);
    NNUE_REQUIRE(ldx >= K && ldw >= K, NNUE_ERR_ARG, "%s: pitch below the row length", what);
    NNUE_REQUIRE(aligned16(x) && aligned16(w) && ldx % 16 == 0 && ldw % 16 == 0, NNUE_ERR_ALIGN,
                 "%s: rows of x and w must start at multiples of 16 bytes", what);
    NNUE_REQUIRE(aligned16(y) && aligned16(plan), NNUE_ERR_ALIGN, "%s: unaligned output or plan", what);
    F8Args a = {};
    if (plan) a.plan = group_view(plan, T, E);
    a.o = rows_out(y, y_type, N);
    a.x_scale = x_scale;
    a.scale_ld = scale_ld;
    a.scale_vec = scale_ld > 0 && scale_ld % 4 == 0 && aligned16(x_scale);
    a.w_scale = w_scale;
    a.bias = bias;
    a.T = (int32_t)T;
    a.E = E;
    a.N = (int32_t)N;
    a.K = (int32_t)K;
    a.C = (int32_t)((K + kF8K - 1) / kF8K);
    a.R = (int32_t)((N + kF8K - 1) / kF8K);
    a.dense = !plan;
    a.gather = plan && !laid;
    a.status = device_status_ptr();
    NNUE_REQUIRE(a.status, NNUE_ERR_CUDA, "%s: no device status word", what);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ProfScope prof("fp8_linear", s);
    const TileShape shape = f8_shape(E < T ? E : T, T, N, a.C, !a.gather);
    a.col_tiles = (int32_t)((N + shape.bn - 1) / shape.bn);
    a.idesc = umma_idesc(format == NNUE_T_E5M2 ? 1u : 0u, (uint32_t)(kGroupRows * shape.ctas), (uint32_t)shape.bn, 0, 0);
    CUtensorMap mx, mw;
    {
        const uint64_t dims[2] = {(uint64_t)K, (uint64_t)(laid ? group_laid_rows(T, E) : T)}, strides[1] = {(uint64_t)ldx};
        const uint32_t box[2] = {kF8K, a.gather ? 1u : (uint32_t)kGroupRows};
        if (int st = encode_map(&mx, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, x, dims, strides, box)) return st;
    }
    {
        const uint64_t dims[3] = {(uint64_t)K, (uint64_t)N, (uint64_t)E}, strides[2] = {(uint64_t)ldw, (uint64_t)(N * ldw)};
        const uint32_t box[3] = {kF8K, (uint32_t)(shape.bn / shape.ctas), 1};
        if (int st = encode_map(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, w, dims, strides, box)) return st;
    }
    const int64_t tiles = (plan ? group_max_tiles(T, E) : (T + kGroupRows - 1) / kGroupRows) * a.col_tiles;
    NNUE_REQUIRE(tiles * 8 < 0x7fffffffLL, NNUE_ERR_UNSUPPORTED, "%s: too many tiles", what);
    if (shape.ctas == 2) return f8_launch<256, 2, false>(mx, mw, a, tiles, 1, s);
    if (shape.ranks > 1) return f8_launch<64, 1, true>(mx, mw, a, tiles, shape.ranks, s);
    if (shape.bn == 64) return f8_launch<64, 1, false>(mx, mw, a, tiles, 1, s);
    return f8_launch<128, 1, false>(mx, mw, a, tiles, 1, s);
}
