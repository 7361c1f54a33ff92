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

// One warp per row block.  q's columns [K, ldq) become zero.
__global__ void __launch_bounds__(kThreads)
    k_fp8_rows(const void* __restrict__ x, int type, int64_t ldx, uint8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale,
               int64_t T, int64_t K, int format) {
    const int64_t C = (K + kFp8Block - 1) / kFp8Block;
    const int lane = threadIdx.x & 31;
    const int64_t i = (int64_t)blockIdx.x * kWarpsPerCta + (threadIdx.x >> 5);
    if (i >= T * C) return;
    const int64_t t = i / C, c = i % C;
    float v[4];
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t k = c * kFp8Block + j * 32 + lane;
        v[j] = k < K ? load_as_float(x, type, t * ldx + k) : 0.f;
        most = max(most, finite_abs_bits(v[j]));
    }
    most = __reduce_max_sync(kFullMask, most);
    const int e = fp8_scale_exponent(most, format);
    const float inverse = power_of_two(-e);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t k = c * kFp8Block + j * 32 + lane;
        if (k < ldq) q[t * ldq + k] = to_fp8(v[j] * inverse, format);
    }
    if (lane == 0) scale[i] = power_of_two(e);
}

// One CTA per 128 x 128 tile.
__global__ void __launch_bounds__(kThreads)
    k_fp8_tiles(const void* __restrict__ w, int type, int64_t ldw, uint8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale,
                int64_t N, int64_t K, int format) {
    const int64_t C = (K + kFp8Block - 1) / kFp8Block, R = (N + kFp8Block - 1) / kFp8Block;
    const int64_t tile = blockIdx.x, c = tile % C, r = tile / C % R, e = tile / (C * R);
    const int col = threadIdx.x & 127, sub = threadIdx.x >> 7;
    const int64_t k = c * kFp8Block + col;
    __shared__ uint32_t s_most;
    if (threadIdx.x == 0) s_most = 0;
    __syncthreads();
    uint32_t most = 0;
    for (int j = sub; j < kFp8Block; j += 2) {
        const int64_t n = r * kFp8Block + j;
        if (n < N && k < K) most = max(most, finite_abs_bits(load_as_float(w, type, (e * N + n) * ldw + k)));
    }
    most = __reduce_max_sync(kFullMask, most);
    if ((threadIdx.x & 31) == 0) atomicMax(&s_most, most);
    __syncthreads();
    const int x = fp8_scale_exponent(s_most, format);
    const float inverse = power_of_two(-x);
    for (int j = sub; j < kFp8Block; j += 2) {
        const int64_t n = r * kFp8Block + j;
        if (n < N && k < ldq)
            q[(e * N + n) * ldq + k] = k < K ? to_fp8(load_as_float(w, type, (e * N + n) * ldw + k) * inverse, format) : 0;
    }
    if (threadIdx.x == 0) scale[tile] = power_of_two(x);
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

extern "C" int nnue_fp8_quantize_rows(const void* x, int32_t type, int64_t ldx, void* q, int64_t ldq, float* scale, int64_t T,
                                      int64_t K, int32_t format, void* stream) {
    if (int st = check_fp8("nnue_fp8_quantize_rows", x, type, ldx, q, ldq, scale, T, K, format)) return st;
    if (T == 0) return NNUE_OK;
    const int64_t blocks = (T * ((K + kFp8Block - 1) / kFp8Block) + kWarpsPerCta - 1) / kWarpsPerCta;
    NNUE_REQUIRE(blocks <= 0x7fffffffLL, NNUE_ERR_UNSUPPORTED, "nnue_fp8_quantize_rows: too many blocks");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ProfScope prof("fp8_rows", s);
    k_fp8_rows<<<(unsigned)blocks, kThreads, 0, s>>>(x, type, ldx, static_cast<uint8_t*>(q), ldq, scale, T, K, format);
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
    k_fp8_tiles<<<(unsigned)tiles, kThreads, 0, s>>>(w, type, ldw, static_cast<uint8_t*>(q), ldq, scale, N, K, format);
    note_launches(1);
    NNUE_CUDA_TRY(cudaGetLastError());
    return NNUE_OK;
}
