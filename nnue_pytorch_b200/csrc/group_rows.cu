// Rows of a batch laid out by bucket, in the form the products' copy engine reads: 16-bit numbers, rows at multiples of 16
// bytes, every bucket from a multiple of 64 rows on and filled up with rows of zeros.  On the way the columns' sums of
// every tile of 128 rows can be taken (the bias gradient of a linear layer: dbias[b] = sum of its rows of dy).
//
// Bound by HBM: every row is read and written once; a warp moves rows of up to 512 bytes, four at a time in flight.
// 16384 x 4096 bf16 51 us, 81 % of the measured copy rate; 16384 x 2048 with sums 28 us, 74 %; short rows less (8192 x 1024
// with sums 13 us, 40 %), and rows off 16 bytes are read number by number.
#include "grouped.cuh"

namespace nnue {

struct RowsArgs {
    GroupPlanView plan;
    const void* src;
    int64_t ld, ldd;      // elements
    uint16_t* dst;
    float* sums;          // [tiles][cols] or null
    int32_t src_type, type, cols, E;
    int32_t shift;        // lanes per row: 1 << shift, eight columns each
    int32_t col_blocks;
    int32_t vec;          // src: the same type, rows at multiples of 16 bytes, cols a multiple of 8
};

__device__ __forceinline__ uint16_t to_half_bits(float v, int32_t type) {
    return type == NNUE_T_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}
__device__ __forceinline__ float from_half_bits(uint32_t v, int32_t type) {
    return type == NNUE_T_BF16 ? __uint_as_float(v << 16) : __half2float(__ushort_as_half((uint16_t)v));
}

// eight numbers from column c of a row on; zeros from column `cols` on
__device__ __forceinline__ uint4 load_eight(const RowsArgs& a, int64_t row, int c) {
    if (a.vec) return __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.src) + row * a.ld + c));
    uint16_t h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t at = row * a.ld + c + i;
        if (c + i >= a.cols) h[i] = 0;
        else if (a.src_type == a.type) h[i] = __ldg(static_cast<const uint16_t*>(a.src) + at);
        else h[i] = to_half_bits(load_as_float(a.src, a.src_type, at), a.type);
    }
    return make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16, h[6] | (uint32_t)h[7] << 16);
}

template <bool SUMS>
__global__ void __launch_bounds__(kThreads) k_group_rows(const __grid_constant__ RowsArgs a) {
    const int t = blockIdx.x / a.col_blocks, cb = blockIdx.x - t * a.col_blocks;
    if (t >= __ldg(a.plan.n_tiles)) return;
    const int4 tile = __ldg(reinterpret_cast<const int4*>(a.plan.tiles) + t);
    if (tile.x >= a.E) return;  // rows without a bucket have no place
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per = 32 >> a.shift;                       // rows a warp moves at once
    const int in = lane & ((1 << a.shift) - 1), sub = warp * per + (lane >> a.shift);
    const int c = (cb << a.shift) * 8 + in * 8;
    const int rows = (tile.z + kGroupAlign - 1) / kGroupAlign * kGroupAlign, step = kWarpsPerCta * per;
    float acc[8] = {};
    if (c < a.ldd) {
        for (int r0 = sub; r0 < rows; r0 += 4 * step) {
            uint4 v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int r = r0 + u * step;
                v[u] = make_uint4(0, 0, 0, 0);
                if (r < tile.z) v[u] = load_eight(a, __ldg(a.plan.order + tile.y + r), c);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int r = r0 + u * step;
                if (r >= rows) break;
                *reinterpret_cast<uint4*>(a.dst + (int64_t)(tile.w + r) * a.ldd + c) = v[u];
                if (SUMS) {
                    const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        acc[2 * i] += from_half_bits(w[i] & 0xffffu, a.type);
                        acc[2 * i + 1] += from_half_bits(w[i] >> 16, a.type);
                    }
                }
            }
        }
    }
    if (SUMS) {  // the row lanes' sums in order: [row lane][column]
        __shared__ float s[kWarpsPerCta * 32 * 8];
        const int width = 8 << a.shift;
#pragma unroll
        for (int i = 0; i < 8; ++i) s[sub * width + in * 8 + i] = acc[i];
        __syncthreads();
        for (int i = threadIdx.x; i < width; i += kThreads) {
            const int col = cb * width + i;
            if (col >= a.cols) continue;
            float sum = 0.f;
            for (int r = 0; r < step; ++r) sum += s[r * width + i];
            a.sums[(int64_t)t * a.cols + col] = sum;
        }
    }
}

// out[b, c] = sum over the bucket's tiles, in order
__global__ void __launch_bounds__(kThreads)
    k_group_sums(const float* __restrict__ sums, GroupPlanView plan, void* __restrict__ out, int type, int64_t cols, int64_t total) {
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
        const int64_t e = i / cols, c = i - e * cols;
        float v = 0.f;
        for (int t = plan.first[e]; t < plan.first[e + 1]; ++t) v += sums[t * cols + c];
        store_from_float(out, type, i, v);
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
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ProfScope prof("pack_rows", s);
    k_pack_rows<<<(unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)), kThreads, 0, s>>>(src, src_type, lds, dst, dst_type, ldd, rows,
                                                                                        cols);
    note_launches(1);
    NNUE_CUDA_TRY(cudaGetLastError());
    return NNUE_OK;
}

extern "C" size_t nnue_group_rows_bytes(int64_t T, int64_t cols, int32_t E) {
    if (T < 0 || T > NNUE_GROUP_MAX_ROWS || cols <= 0 || E <= 0 || E > kMaxGroups) return 0;
    return (size_t)group_laid_rows(T, E) * (size_t)((cols + 7) / 8 * 8) * 2;
}

extern "C" size_t nnue_group_sums_bytes(int64_t T, int64_t cols, int32_t E) {
    if (T < 0 || T > NNUE_GROUP_MAX_ROWS || cols <= 0 || E <= 0 || E > kMaxGroups) return 0;
    return (size_t)group_max_tiles(T, E) * (size_t)cols * sizeof(float);
}

extern "C" int nnue_group_rows(const void* src, int32_t src_type, int64_t ld, const void* plan, void* dst, int32_t type, float* sums,
                               int64_t T, int64_t cols, int32_t E, void* stream) {
    NNUE_REQUIRE(T >= 0 && cols > 0 && E > 0 && ld >= cols, NNUE_ERR_ARG, "nnue_group_rows: bad sizes");
    NNUE_REQUIRE(E <= kMaxGroups && T <= NNUE_GROUP_MAX_ROWS && cols < (1 << 24), NNUE_ERR_UNSUPPORTED,
                 "nnue_group_rows: sizes T=%lld cols=%lld E=%d beyond the kernel's range", (long long)T, (long long)cols, E);
    NNUE_REQUIRE(is_float_type(src_type) && is_half_type(type), NNUE_ERR_UNSUPPORTED, "nnue_group_rows: types %d to %d", src_type, type);
    if (T == 0) return NNUE_OK;
    NNUE_REQUIRE(src && plan && dst, NNUE_ERR_ARG, "nnue_group_rows: null pointer");
    NNUE_REQUIRE(aligned16(plan) && aligned16(dst), NNUE_ERR_ALIGN, "nnue_group_rows: unaligned plan or destination");
    RowsArgs a;
    a.plan = group_view(plan, T, E);
    a.src = src;
    a.ld = ld;
    a.ldd = (cols + 7) / 8 * 8;
    a.dst = static_cast<uint16_t*>(dst);
    a.sums = sums;
    a.src_type = src_type;
    a.type = type;
    a.cols = (int32_t)cols;
    a.E = E;
    a.shift = 0;
    while (a.shift < 5 && (8 << a.shift) < cols) ++a.shift;
    a.col_blocks = (int32_t)((a.ldd + (8 << a.shift) - 1) / (8 << a.shift));
    a.vec = src_type == type && aligned16(src) && ld % 8 == 0 && cols % 8 == 0;
    const int64_t blocks = group_max_tiles(T, E) * a.col_blocks;
    NNUE_REQUIRE(blocks <= 0x7fffffffLL, NNUE_ERR_UNSUPPORTED, "nnue_group_rows: too many blocks");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ProfScope prof("group_rows", s);
    if (sums) k_group_rows<true><<<(unsigned)blocks, kThreads, 0, s>>>(a);
    else k_group_rows<false><<<(unsigned)blocks, kThreads, 0, s>>>(a);
    note_launches(1);
    NNUE_CUDA_TRY(cudaGetLastError());
    return NNUE_OK;
}

extern "C" int nnue_group_sums(const float* sums, const void* plan, void* out, int32_t type, int64_t T, int64_t cols, int32_t E,
                               void* stream) {
    NNUE_REQUIRE(T >= 0 && cols > 0 && E > 0, NNUE_ERR_ARG, "nnue_group_sums: bad sizes");
    NNUE_REQUIRE(is_float_type(type), NNUE_ERR_UNSUPPORTED, "nnue_group_sums: type %d", type);
    NNUE_REQUIRE(plan && out && (sums || T == 0), NNUE_ERR_ARG, "nnue_group_sums: null pointer");
    const int64_t blocks = (E * cols + kThreads - 1) / kThreads;
    k_group_sums<<<(unsigned)(blocks < 65536 ? blocks : 65536), kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        sums, group_view(plan, T, E), out, type, cols, E * cols);
    note_launches(1);
    NNUE_CUDA_TRY(cudaGetLastError());
    return NNUE_OK;
}
