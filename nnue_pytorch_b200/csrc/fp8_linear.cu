// Linear layer on 8-bit operands with a scale per 128 inputs of a row and per 128 x 128 tile of the weights:
//   y[p, n] = sum_c sx[p, c] sw[b, n / 128, c] sum_{k in block c} x[p, k] w[b, n, k] + bias[b, n]
// First form: one thread per output element, fp32 sums.
#include "grouped.cuh"

#include <cuda_fp8.h>

namespace nnue {

constexpr int kF = 32;
constexpr int kFp8Block = 128;

__device__ __forceinline__ float from_fp8(uint8_t v, int format) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(v, format == NNUE_T_E4M3 ? __NV_E4M3 : __NV_E5M2)));
}

__global__ void __launch_bounds__(kF* kF)
    k_fp8_linear(const uint8_t* x, int64_t ldx, const float* sx, const uint8_t* w, int64_t ldw, const float* sw, const float* bias,
                 const int32_t* plan, void* y, int y_type, int64_t T, int64_t K, int64_t N, int E, int format) {
    const int64_t t = blockIdx.y / (kGroupRows / kF);
    GroupTile tile{0, (int32_t)(t * kGroupRows), (int32_t)min((int64_t)kGroupRows, T - t * kGroupRows), 0};
    const GroupPlanView view = group_view(plan, T, E);
    if (plan) {
        if (t >= *view.n_tiles) return;
        tile = view.tiles[t];
    }
    __shared__ float sa[kF][kF + 1], sb[kF][kF + 1];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int row = blockIdx.y % (kGroupRows / kF) * kF + ty;
    const int64_t p = row < tile.count ? (plan ? view.order[tile.start + row] : tile.start + row) : -1;
    const int64_t C = (K + kFp8Block - 1) / kFp8Block, R = (N + kFp8Block - 1) / kFp8Block;
    for (int64_t n0 = (int64_t)blockIdx.x * kF; n0 < N; n0 += (int64_t)gridDim.x * kF) {
        float acc = 0.f;
        if (tile.bucket < E) {
            const int64_t wrow = (int64_t)tile.bucket * N;
            for (int64_t c = 0; c < C; ++c) {
                float part = 0.f;
                for (int64_t k0 = c * kFp8Block; k0 < min(K, (c + 1) * kFp8Block); k0 += kF) {
                    sa[ty][tx] = p >= 0 && k0 + tx < K ? from_fp8(x[p * ldx + k0 + tx], format) : 0.f;
                    sb[tx][ty] = n0 + ty < N && k0 + tx < K ? from_fp8(w[(wrow + n0 + ty) * ldw + k0 + tx], format) : 0.f;
                    __syncthreads();
                    for (int i = 0; i < kF; ++i) part = fmaf(sa[ty][i], sb[i][tx], part);
                    __syncthreads();
                }
                if (p >= 0) acc = fmaf(part, sx[p * C + c] * sw[((int64_t)tile.bucket * R + n0 / kFp8Block) * C + c], acc);
            }
            if (bias && n0 + tx < N) acc += bias[wrow + n0 + tx];
        }
        if (p >= 0 && n0 + tx < N) store_from_float(y, y_type, p * N + n0 + tx, acc);
    }
}

}  // namespace nnue

using namespace nnue;

extern "C" int nnue_fp8_linear_fwd(const void* x, int64_t ldx, const float* x_scale, const void* w, int64_t ldw,
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
    if (T == 0) return NNUE_OK;
    NNUE_REQUIRE(x && w && x_scale && w_scale && y, NNUE_ERR_ARG, "%s: null pointer", what);
    NNUE_REQUIRE(ldx >= K && ldw >= K, NNUE_ERR_ARG, "%s: pitch below the row length", what);
    NNUE_REQUIRE(aligned16(x) && aligned16(w) && ldx % 16 == 0 && ldw % 16 == 0, NNUE_ERR_ALIGN,
                 "%s: rows of x and w must start at multiples of 16 bytes", what);
    NNUE_REQUIRE(aligned16(y) && aligned16(plan), NNUE_ERR_ALIGN, "%s: unaligned output or plan", what);
    const int64_t tiles = plan ? group_max_tiles(T, E) : (T + kGroupRows - 1) / kGroupRows;
    const dim3 grid((unsigned)((N + kF - 1) / kF), (unsigned)(tiles * (kGroupRows / kF)));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ProfScope prof("fp8_linear", s);
    k_fp8_linear<<<grid, kF * kF, 0, s>>>(static_cast<const uint8_t*>(x), ldx, x_scale, static_cast<const uint8_t*>(w), ldw, w_scale,
                                          bias, static_cast<const int32_t*>(plan), y, y_type, T, K, N, E, format);
    note_launches(1);
    NNUE_CUDA_TRY(cudaGetLastError());
    return NNUE_OK;
}
