// Quantisation to 8-bit floating point with one scale per block: 128 consecutive numbers of a row (activations) or a
// 128 x 128 tile of a matrix (weights).
//
// Mathematics: a = max |v| over the block's finite numbers; scale = 2^ceil(log2(a / MAX)), 1 for a = 0, at least 2^-126;
// q = v / scale rounded to the nearest number of the format, ties to even.  MAX (448 for e4m3, 57344 for e5m2) is 7/8 of
// a power of two, so with a = m 2^e, 1/2 <= m < 1, the exponent is e - 9 or e - 16, one more where m > 7/8: whole-number
// arithmetic on the bits of a.  A power of two makes the division exact: the one rounding is that to 8 bits, and it does
// not depend on the precision the formula is evaluated in.  Numbers that are not finite become NaN in e4m3, which has no
// infinity, and keep their value in e5m2; they leave the block's scale alone.
#include "grouped.cuh"

#include <cuda_fp8.h>

namespace nnue {

constexpr int kFp8Block = 128;

// |v| where it is finite, else 0, as bits (ordered like the numbers)
__device__ __forceinline__ uint32_t finite_abs_bits(float v) {
    const uint32_t u = __float_as_uint(v) & 0x7fffffffu;
    return u < 0x7f800000u ? u : 0u;
}

// exponent of the block's scale from the bits of its largest number
__device__ __forceinline__ int fp8_scale_exponent(uint32_t bits, int format) {
    if (bits == 0) return 0;
    int shift = 0;
    if (bits < 0x00800000u) {  // subnormal: normalise
        shift = __clz(bits) - 8;
        bits <<= shift;
        bits = (bits & 0x007fffffu) | 0x00800000u;
    }
    const int e = (int)(bits >> 23) - 126 - shift;             // a = m 2^e with 1/2 <= m < 1
    const bool above = (bits & 0x007fffffu) > 0x00600000u;     // m > 7/8
    const int x = e + (above ? 1 : 0) - (format == NNUE_T_E4M3 ? 9 : 16);
    return x < -126 ? -126 : x;
}

__device__ __forceinline__ float power_of_two(int x) { return __uint_as_float((uint32_t)(x + 127) << 23); }  // -126 <= x <= 127

__device__ __forceinline__ uint8_t to_fp8(float v, int format) {
    const uint32_t u = __float_as_uint(v);
    if ((u & 0x7fffffffu) >= 0x7f800000u) {
        const bool nan = (u & 0x7fffffffu) > 0x7f800000u;
        if (format == NNUE_T_E4M3 || nan) return 0x7f;
        return (uint8_t)(0x7c | (u >> 31 << 7));
    }
    return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, format == NNUE_T_E4M3 ? __NV_E4M3 : __NV_E5M2);
}

constexpr int kLaneNumbers = 16;                                 // consecutive numbers of a lane: 16 bytes of q
constexpr int kWarpNumbers = 32 * kLaneNumbers;                  // four blocks of a row
constexpr int kBlockLanes = kFp8Block / kLaneNumbers;            // 8

// ROWS times sixteen numbers, v[u][i] = p[at[u] + i], zeros from i = left on and for u from n on.  All loads before any use.
template <int TYPE, int ROWS>
__device__ __forceinline__ void load_sixteen(const void* p, const int64_t (&at)[ROWS], int n, int left, bool vec,
                                             float (&v)[ROWS][kLaneNumbers]) {
    if (vec && left >= kLaneNumbers) {
        constexpr int kPieces = TYPE == NNUE_T_F32 ? 4 : 2;  // of 16 bytes
        uint4 raw[ROWS][kPieces];
#pragma unroll
        for (int u = 0; u < ROWS; ++u)
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                raw[u][i] = make_uint4(0, 0, 0, 0);
                if (u < n) raw[u][i] = __ldcs(reinterpret_cast<const uint4*>(static_cast<const char*>(p) + at[u] * (TYPE == NNUE_T_F32 ? 4 : 2)) + i);
            }
#pragma unroll
        for (int u = 0; u < ROWS; ++u)
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const uint32_t w[4] = {raw[u][i].x, raw[u][i].y, raw[u][i].z, raw[u][i].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (TYPE == NNUE_T_F32) {
                        v[u][4 * i + j] = __uint_as_float(w[j]);
                    } else if (TYPE == NNUE_T_BF16) {
                        v[u][(8 * i + 2 * j) & 15] = __uint_as_float(w[j] << 16);
                        v[u][(8 * i + 2 * j + 1) & 15] = __uint_as_float(w[j] & 0xffff0000u);
                    } else {
                        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
                        v[u][(8 * i + 2 * j) & 15] = f.x;
                        v[u][(8 * i + 2 * j + 1) & 15] = f.y;
                    }
                }
            }
        return;
    }
#pragma unroll
    for (int u = 0; u < ROWS; ++u)
#pragma unroll
        for (int i = 0; i < kLaneNumbers; ++i) v[u][i] = u < n && i < left ? load_as_float(p, TYPE, at[u] + i) : 0.f;
}

// bits of the largest finite |v|
__device__ __forceinline__ uint32_t largest_bits(const float (&v)[kLaneNumbers]) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < kLaneNumbers; ++i) most = max(most, __float_as_uint(v[i]) & 0x7fffffffu);
    if (most < 0x7f800000u) return most;
    most = 0;
#pragma unroll
    for (int i = 0; i < kLaneNumbers; ++i) most = max(most, finite_abs_bits(v[i]));
    return most;
}

// q[at + i] = v[i] * inverse in 8 bits, `room` of them
__device__ __forceinline__ void store_sixteen(uint8_t* q, int64_t at, int room, bool vec, const float (&v)[kLaneNumbers], float inverse,
                                              int format) {
    uint32_t raw = 0;
#pragma unroll
    for (int i = 0; i < kLaneNumbers; ++i) raw = max(raw, __float_as_uint(v[i]) & 0x7fffffffu);
    uint32_t w[4];
    if (raw < 0x7f800000u) {
        const __nv_fp8_interpretation_t kind = format == NNUE_T_E4M3 ? __NV_E4M3 : __NV_E5M2;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i] * inverse, v[4 * i + 1] * inverse), __NV_SATFINITE, kind);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i + 2] * inverse, v[4 * i + 3] * inverse), __NV_SATFINITE, kind);
            w[i] = lo | hi << 16;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[i] |= (uint32_t)to_fp8(v[4 * i + j] * inverse, format) << (8 * j);
        }
    }
    if (vec && room >= kLaneNumbers) {
        *reinterpret_cast<uint4*>(q + at) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int i = 0; i < kLaneNumbers; ++i)
            if (i < room) q[at + i] = (uint8_t)(w[i / 4] >> (8 * (i % 4)));
    }
}

struct Fp8Args {
    GroupPlanView plan;
    const void* x;
    uint8_t* q;
    float* scale;
    int64_t ldx, ldq, T;
    int64_t scale_ld;     // 0: scale [T, C]; else [C, scale_ld] by places in q
    int32_t K, format, E;
    int32_t parts;        // of a row: four blocks each
    int32_t vec_x, vec_q;
};

// A warp quantises four blocks of two neighbouring rows: a lane holds 16 consecutive numbers of each (one 16-byte store),
// eight lanes a block.  A CTA takes 16 rows; the scales go out together, 16 neighbours of a block where they lie by place.
// Bound by HBM: 16384 x 4096 bf16 in 41 us, 4.9 TB/s (four rows per warp 54 us, too few warps; one 46).  LAID: the rows are
// walked by the plan's tiles.
constexpr int kFp8Rows = 2;
template <int TYPE, bool LAID>
__global__ void __launch_bounds__(kThreads, 5) k_fp8_rows(const __grid_constant__ Fp8Args a) {
    constexpr int kCtaRows = kWarpsPerCta * kFp8Rows;
    __shared__ float s_scale[kWarpNumbers / kFp8Block][kCtaRows + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t group = blockIdx.x / a.parts;
    const int part = (int)(blockIdx.x - group * a.parts);
    int64_t to = group * kCtaRows;  // the CTA's first row in q
    int rows, start = 0;
    if (LAID) {
        const int64_t t = group / (kGroupRows / kCtaRows);
        if (t >= __ldg(a.plan.n_tiles)) return;
        const int4 tile = __ldg(reinterpret_cast<const int4*>(a.plan.tiles) + t);
        const int in = (int)(group % (kGroupRows / kCtaRows)) * kCtaRows;
        if (tile.x >= a.E || in >= tile.z) return;
        rows = min(kCtaRows, tile.z - in);
        start = tile.y + in;
        to = tile.w + in;
    } else {
        rows = (int)min((int64_t)kCtaRows, a.T - to);
    }
    const int r0 = warp * kFp8Rows, n = min(kFp8Rows, rows - r0);
    const int k = part * kWarpNumbers + lane * kLaneNumbers, C = (a.K + kFp8Block - 1) / kFp8Block, c = k / kFp8Block;
    if (n > 0) {
        int64_t from[kFp8Rows], at[kFp8Rows];
#pragma unroll
        for (int u = 0; u < kFp8Rows; ++u) {
            from[u] = u >= n ? 0 : LAID ? (int64_t)__ldg(a.plan.order + start + r0 + u) : to + r0 + u;
            at[u] = from[u] * a.ldx + k;
        }
        float v[kFp8Rows][kLaneNumbers];
        load_sixteen<TYPE, kFp8Rows>(a.x, at, n, a.K - k, a.vec_x, v);
#pragma unroll
        for (int u = 0; u < kFp8Rows; ++u) {
            uint32_t most = largest_bits(v[u]);
#pragma unroll
            for (int d = 1; d < kBlockLanes; d <<= 1) most = max(most, __shfl_xor_sync(kFullMask, most, d));
            if (u >= n) continue;
            const int e = fp8_scale_exponent(most, a.format);
            store_sixteen(a.q, (to + r0 + u) * a.ldq + k, (int)min((int64_t)kLaneNumbers, a.ldq - k), a.vec_q, v[u], power_of_two(-e), a.format);
            if (lane % kBlockLanes == 0 && c < C) {
                if (a.scale_ld) s_scale[lane / kBlockLanes][r0 + u] = power_of_two(e);
                else a.scale[from[u] * C + c] = power_of_two(e);
            }
        }
    }
    if (!a.scale_ld) return;
    __syncthreads();
    const int sc = part * (kWarpNumbers / kFp8Block) + warp;
    if (warp < kWarpNumbers / kFp8Block && sc < C && lane < rows) a.scale[sc * a.scale_ld + to + lane] = s_scale[warp][lane];
}

// One CTA per 128 x 128 tile: every number is read once and held in registers, 64 per thread, until the scale is known.
// Bound by HBM with too little in flight: 8 x 1000 x 2040 fp32 in 23 us with a cold L2, 3.6 TB/s.
template <int TYPE>
__global__ void __launch_bounds__(kThreads, 2)
    k_fp8_tiles(const void* __restrict__ w, int64_t ldw, uint8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale,
                int64_t N, int64_t K, int format, int vec_w, int vec_q) {
    const int64_t C = (K + kFp8Block - 1) / kFp8Block, R = (N + kFp8Block - 1) / kFp8Block;
    const int64_t tile = blockIdx.x, c = tile % C, r = tile / C % R, e = tile / (C * R);
    const int64_t k = c * kFp8Block + (threadIdx.x % kBlockLanes) * kLaneNumbers;
    const int64_t n0 = r * kFp8Block + threadIdx.x / kBlockLanes;
    constexpr int kRows = kThreads / kBlockLanes;  // 32 rows at once
    float v[4][kLaneNumbers];
    int64_t at[4];
    const int there = (int)max((int64_t)0, min((int64_t)4, (N - n0 + kRows - 1) / kRows));
#pragma unroll
    for (int j = 0; j < 4; ++j) at[j] = (e * N + n0 + j * kRows) * ldw + k;
    load_sixteen<TYPE, 4>(w, at, there, (int)(K - k), vec_w, v);
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) most = max(most, largest_bits(v[j]));
    __shared__ uint32_t s_most[kWarpsPerCta];
    most = __reduce_max_sync(kFullMask, most);
    if ((threadIdx.x & 31) == 0) s_most[threadIdx.x >> 5] = most;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kWarpsPerCta; ++j) most = max(most, s_most[j]);
    const int x = fp8_scale_exponent(most, format);
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j < there)
            store_sixteen(q, (e * N + n0 + j * kRows) * ldq + k, (int)min((int64_t)kLaneNumbers, ldq - k), vec_q, v[j], power_of_two(-x), format);
    if (threadIdx.x == 0) scale[tile] = power_of_two(x);
}

template <int TYPE>
void launch_fp8_rows(const Fp8Args& a, bool laid, unsigned blocks, cudaStream_t s) {
    if (laid) k_fp8_rows<TYPE, true><<<blocks, kThreads, 0, s>>>(a);
    else k_fp8_rows<TYPE, false><<<blocks, kThreads, 0, s>>>(a);
}

}  // namespace nnue

using namespace nnue;

static int check_fp8(const char* what, const void* x, int32_t type, int64_t ldx, const void* q, int64_t ldq, const void* scale,
                     int64_t rows, int64_t K, int32_t format) {
    NNUE_REQUIRE(rows >= 0 && K > 0 && ldx >= K && ldq >= K, NNUE_ERR_ARG, "%s: bad sizes", what);
    NNUE_REQUIRE(is_float_type(type), NNUE_ERR_UNSUPPORTED, "%s: input type %d", what, type);
    NNUE_REQUIRE(format == NNUE_T_E4M3 || format == NNUE_T_E5M2, NNUE_ERR_UNSUPPORTED, "%s: format %d", what, format);
    NNUE_REQUIRE(ldq < (K + kFp8Block - 1) / kFp8Block * kFp8Block + 1, NNUE_ERR_ARG, "%s: pitch of q beyond its last block", what);
    NNUE_REQUIRE(rows == 0 || (x && q && scale), NNUE_ERR_ARG, "%s: null pointer", what);
    return NNUE_OK;
}

extern "C" int nnue_fp8_quantize_rows(const void* x, int32_t type, int64_t ldx, void* q, int64_t ldq, float* scale, int64_t scale_ld, int64_t T,
                                      int64_t K, int32_t format, const void* plan, int32_t E, void* stream) {
    const char* what = "nnue_fp8_quantize_rows";
    if (plan) {
        NNUE_REQUIRE(E > 0 && E <= kMaxGroups && T <= NNUE_GROUP_MAX_ROWS && aligned16(plan), NNUE_ERR_ARG, "%s: bad plan", what);
        ldq = (K + 15) / 16 * 16;
    }
    if (int st = check_fp8(what, x, type, ldx, q, ldq, scale, T, K, format)) return st;
    NNUE_REQUIRE(K < (1 << 24), NNUE_ERR_UNSUPPORTED, "%s: rows of %lld numbers", what, (long long)K);
    NNUE_REQUIRE(scale_ld == 0 || scale_ld >= (plan ? group_laid_rows(T, E) : T), NNUE_ERR_ARG, "%s: no room for every row's scales", what);
    if (T == 0) return NNUE_OK;
    Fp8Args a = {};
    if (plan) a.plan = group_view(plan, T, E);
    a.x = x;
    a.q = static_cast<uint8_t*>(q);
    a.scale = scale;
    a.ldx = ldx;
    a.ldq = ldq;
    a.scale_ld = scale_ld;
    a.T = T;
    a.K = (int32_t)K;
    a.format = format;
    a.E = E;
    a.parts = (int32_t)((K + kWarpNumbers - 1) / kWarpNumbers);
    a.vec_x = aligned16(x) && ldx * type_bytes(type) % 16 == 0;
    a.vec_q = aligned16(q) && ldq % 16 == 0;
    const int64_t rows = plan ? group_max_tiles(T, E) * kGroupRows : T;
    constexpr int kCtaRows = kWarpsPerCta * kFp8Rows;
    const int64_t blocks = (rows + kCtaRows - 1) / kCtaRows * a.parts;
    NNUE_REQUIRE(blocks <= 0x7fffffffLL, NNUE_ERR_UNSUPPORTED, "%s: too many blocks", what);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ProfScope prof("fp8_rows", s);
    if (type == NNUE_T_F32) launch_fp8_rows<NNUE_T_F32>(a, plan, (unsigned)blocks, s);
    else if (type == NNUE_T_BF16) launch_fp8_rows<NNUE_T_BF16>(a, plan, (unsigned)blocks, s);
    else launch_fp8_rows<NNUE_T_F16>(a, plan, (unsigned)blocks, s);
    note_launches(1);
    NNUE_CUDA_TRY(cudaGetLastError());
    return NNUE_OK;
}

extern "C" int nnue_fp8_quantize_tiles(const void* w, int32_t type, int64_t ldw, void* q, int64_t ldq, float* scale, int32_t E,
                                       int64_t N, int64_t K, int32_t format, void* stream) {
    NNUE_REQUIRE(E > 0 && N >= 0, NNUE_ERR_ARG, "nnue_fp8_quantize_tiles: bad sizes");
    if (int st = check_fp8("nnue_fp8_quantize_tiles", w, type, ldw, q, ldq, scale, N, K, format)) return st;
    if (N == 0) return NNUE_OK;
    const int64_t tiles = E * ((N + kFp8Block - 1) / kFp8Block) * ((K + kFp8Block - 1) / kFp8Block);
    NNUE_REQUIRE(tiles <= 0x7fffffffLL, NNUE_ERR_UNSUPPORTED, "nnue_fp8_quantize_tiles: too many tiles");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ProfScope prof("fp8_tiles", s);
    auto kernel = type == NNUE_T_F32 ? k_fp8_tiles<NNUE_T_F32> : type == NNUE_T_BF16 ? k_fp8_tiles<NNUE_T_BF16> : k_fp8_tiles<NNUE_T_F16>;
    kernel<<<(unsigned)tiles, kThreads, 0, s>>>(w, ldw, static_cast<uint8_t*>(q), ldq, scale, N, K, format,
                                                aligned16(w) && ldw * type_bytes(type) % 16 == 0, aligned16(q) && ldq % 16 == 0);
    note_launches(1);
    NNUE_CUDA_TRY(cudaGetLastError());
    return NNUE_OK;
}
