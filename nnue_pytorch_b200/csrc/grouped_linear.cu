// Bucketed linear layer on 16-bit operands: forward, input gradient, weight and bias gradient.  First form: one thread
// per output element, 32 x 32 tiles in shared memory, fp32 sums.
#include "grouped.cuh"

namespace nnue {

constexpr int kS = 32;

// y[p, n] = sum_k x[p, k] w[b, n, k] + bias[b, n]        (transposed == 0; red = K, cols = N)
// dx[p, k] = sum_n dy[p, n] w[b, n, k]                   (transposed == 1; red = N, cols = K)
__global__ void __launch_bounds__(kS* kS)
    k_grouped_rows(const void* a, int64_t lda, const void* w, int64_t ldw, const void* bias, GroupPlanView plan, void* out,
                   int64_t red, int64_t cols, int64_t N, int E, int type, int bias_type, int out_type, int transposed) {
    const int t = blockIdx.y / (kGroupRows / kS), part = blockIdx.y % (kGroupRows / kS);
    if (t >= *plan.n_tiles) return;
    const GroupTile tile = plan.tiles[t];
    __shared__ float sa[kS][kS + 1], sb[kS][kS + 1];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int row = part * kS + ty;
    const int64_t p = row < tile.count ? plan.order[tile.start + row] : -1;
    for (int64_t c0 = (int64_t)blockIdx.x * kS; c0 < cols; c0 += (int64_t)gridDim.x * kS) {
        float acc = 0.f;
        if (tile.bucket < E) {
            const int64_t wrow = (int64_t)tile.bucket * N;
            for (int64_t r0 = 0; r0 < red; r0 += kS) {
                sa[ty][tx] = p >= 0 && r0 + tx < red ? load_as_float(a, type, p * lda + r0 + tx) : 0.f;
                const int64_t n = transposed ? r0 + ty : c0 + ty, k = transposed ? c0 + tx : r0 + tx;
                const float v = n < N && k < (transposed ? cols : red) ? load_as_float(w, type, (wrow + n) * ldw + k) : 0.f;
                if (transposed) sb[ty][tx] = v;
                else sb[tx][ty] = v;
                __syncthreads();
                for (int i = 0; i < kS; ++i) acc = fmaf(sa[ty][i], sb[i][tx], acc);
                __syncthreads();
            }
            if (bias && c0 + tx < cols) acc += load_as_float(bias, bias_type, wrow + c0 + tx);
        }
        if (p >= 0 && c0 + tx < cols) store_from_float(out, out_type, p * cols + c0 + tx, acc);
    }
}

// dw[b, n, k] = sum_p dy[p, n] x[p, k];  dbias[b, n] = sum_p dy[p, n]
__global__ void __launch_bounds__(kS* kS)
    k_grouped_dw(const void* dy, int64_t lddy, const void* x, int64_t ldx, GroupPlanView plan, void* dw, void* dbias,
                 int64_t K, int64_t N, int type, int dw_type, int dbias_type) {
    __shared__ float sa[kS][kS + 1], sb[kS][kS + 1];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, e = blockIdx.z;
    const int first = plan.offsets[e], last = plan.offsets[e + 1];
    for (int64_t n0 = (int64_t)blockIdx.y * kS; n0 < N; n0 += (int64_t)gridDim.y * kS)
        for (int64_t k0 = (int64_t)blockIdx.x * kS; k0 < K; k0 += (int64_t)gridDim.x * kS) {
            float acc = 0.f, sum = 0.f;
            for (int q0 = first; q0 < last; q0 += kS) {
                const int64_t p = q0 + ty < last ? plan.order[q0 + ty] : -1;
                sa[ty][tx] = p >= 0 && n0 + tx < N ? load_as_float(dy, type, p * lddy + n0 + tx) : 0.f;
                sb[ty][tx] = p >= 0 && k0 + tx < K ? load_as_float(x, type, p * ldx + k0 + tx) : 0.f;
                __syncthreads();
                for (int i = 0; i < kS; ++i) {
                    acc = fmaf(sa[i][ty], sb[i][tx], acc);
                    sum += sa[i][ty];
                }
                __syncthreads();
            }
            const int64_t n = n0 + ty;
            if (n < N && k0 + tx < K) store_from_float(dw, dw_type, ((int64_t)e * N + n) * K + k0 + tx, acc);
            if (dbias && n < N && k0 == 0 && tx == 0) store_from_float(dbias, dbias_type, (int64_t)e * N + n, sum);
        }
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
    const dim3 grid((unsigned)((N + kS - 1) / kS), (unsigned)(group_max_tiles(T, E) * (kGroupRows / kS)));
    k_grouped_rows<<<grid, kS * kS, 0, static_cast<cudaStream_t>(stream)>>>(x, ldx, w, ldw, bias, group_view(plan, T, E), y, K, N,
                                                                            N, E, type, bias_type, y_type, 0);
    note_launches(1);
    NNUE_CUDA_TRY(cudaGetLastError());
    return NNUE_OK;
}

extern "C" int nnue_grouped_linear_bwd_input(const void* dy, int64_t lddy, const void* w, int64_t ldw, const void* plan, void* dx,
                                             int64_t T, int64_t K, int64_t N, int32_t E, int32_t type, void* stream) {
    if (int st = check_grouped("nnue_grouped_linear_bwd_input", plan, T, K, N, E, type)) return st;
    if (T == 0) return NNUE_OK;
    if (int st = check_operand("nnue_grouped_linear_bwd_input", "dy", dy, lddy, N, type)) return st;
    if (int st = check_operand("nnue_grouped_linear_bwd_input", "weight", w, ldw, K, type)) return st;
    NNUE_REQUIRE(dx && aligned16(dx), NNUE_ERR_ALIGN, "nnue_grouped_linear_bwd_input: null or unaligned output");
    const dim3 grid((unsigned)((K + kS - 1) / kS), (unsigned)(group_max_tiles(T, E) * (kGroupRows / kS)));
    k_grouped_rows<<<grid, kS * kS, 0, static_cast<cudaStream_t>(stream)>>>(dy, lddy, w, ldw, nullptr, group_view(plan, T, E), dx,
                                                                            N, K, N, E, type, 0, type, 1);
    note_launches(1);
    NNUE_CUDA_TRY(cudaGetLastError());
    return NNUE_OK;
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
    const dim3 grid((unsigned)((K + kS - 1) / kS), (unsigned)((N + kS - 1) / kS < 65535 ? (N + kS - 1) / kS : 65535), (unsigned)E);
    k_grouped_dw<<<grid, kS * kS, 0, static_cast<cudaStream_t>(stream)>>>(dy, lddy, x, ldx, group_view(plan, T, E), dw, dbias, K, N,
                                                                          type, dw_type, dbias_type);
    note_launches(1);
    NNUE_CUDA_TRY(cudaGetLastError());
    return NNUE_OK;
}
