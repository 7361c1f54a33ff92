// What the tensor-core products of 16-bit and 8-bit operands share: the ring of stages, bringing rows of a tile out, and
// the choice of a tile.
#pragma once

#include "grouped.cuh"
#include "tc.cuh"

namespace nnue {

constexpr int kStagingBytes = 4096;  // of one output warp: 32 rows x 128 bytes

// The contiguous output [.., cols] that tiles are brought out to.
struct RowsOut {
    void* out;
    int64_t ld;    // elements
    int32_t type, cols;
    int32_t vec;   // rows start at multiples of 16 bytes
};
inline RowsOut rows_out(void* out, int32_t type, int64_t cols) {
    return {out, cols, type, (int32_t)cols, cols * type_bytes(type) % 16 == 0};
}

struct TileShape {
    int bn, ctas, ranks;
};

// Width of a tile, CTAs on it and parts of its sum.  `rows` per bucket in use and the number of such runs of rows are
// estimates in forward and dx (the host does not know the plan), exact in dw; `chunks` is the length of the reduction in
// stages.  Pairs where they fill the GPU.  Else the widest tile that still gives every SM one; where even the narrowest
// leaves SMs idle, the sum is split while every part keeps two stages.
inline TileShape tile_shape(int64_t runs, int64_t rows, int64_t cols, int64_t chunks, int narrowest, int widest, bool pairs) {
    const int64_t sms = sm_count();
    auto tiles = [&](int64_t high, int64_t wide) { return runs * ((rows + high - 1) / high) * ((cols + wide - 1) / wide); };
    if (pairs && rows > kGroupRows && tiles(kGroupPairRows, widest) * 2 >= sms) return {widest, 2, 1};
    int bn = widest;
    while (bn > narrowest && (tiles(kGroupRows, bn) < sms || cols <= bn / 2)) bn /= 2;
    int ranks = 1;  // more only at the narrowest: a wider tile was kept because every SM has one
    while (bn == narrowest && ranks < 8 && tiles(kGroupRows, bn) * ranks * 2 <= sms && chunks >= ranks * 4) ranks *= 2;
    return {bn, 1, ranks};
}

#ifdef __CUDACC__
// Position in the ring of stages.
template <int S>
struct StageRing {
    int stage = 0;
    unsigned phase = 0;
    __device__ __forceinline__ void next() {
        if (++stage == S) {
            stage = 0;
            phase ^= 1u;
        }
    }
};

// A pass of columns (BYTES per row in the warp's staging, 16-byte pieces swizzled) to the rows of the output, in whole
// 128- or 64-byte pieces of rows.  Lane r holds row r's place in the output, or -1.  The places and the pieces are fetched
// before the first store: one after the other they cost a warp 800 cycles per pass, more than reading the accumulator.
template <int BYTES>
__device__ __forceinline__ void copy_rows_out(const RowsOut& o, const unsigned char* stg, int32_t my_row, int64_t row_base, int col) {
    const int lane = threadIdx.x & 31;
    const int es = o.type == NNUE_T_F32 ? 4 : 2;
    unsigned char* out = static_cast<unsigned char*>(o.out);
    __syncwarp();
    if (o.vec) {
        constexpr int kShift = BYTES == 128 ? 3 : 2, kRows = 32 >> kShift, kPasses = 32 / kRows;  // kRows: rows at once
        const int piece = lane & ((1 << kShift) - 1);
        const bool inside = col + piece * (16 / es) < o.cols;  // cols is a multiple of a piece
        int32_t row[kPasses];
        uint4 v[kPasses];
#pragma unroll
        for (int it = 0; it < kPasses; ++it) row[it] = __shfl_sync(kFullMask, my_row, it * kRows + (lane >> kShift));
#pragma unroll
        for (int it = 0; it < kPasses; ++it) {
            const int r = it * kRows + (lane >> kShift);
            v[it] = *reinterpret_cast<const uint4*>(stg + r * 128 + ((piece ^ (r & 7)) << 4));
        }
#pragma unroll
        for (int it = 0; it < kPasses; ++it)
            if (row[it] >= 0 && inside) *reinterpret_cast<uint4*>(out + ((row_base + row[it]) * o.ld + col) * es + piece * 16) = v[it];
    } else {
#pragma unroll 1
        for (int r = 0; r < 32; ++r) {
            const int32_t row = __shfl_sync(kFullMask, my_row, r);
            if (row < 0) continue;
            for (int j = lane; j < BYTES / es && col + j < o.cols; j += 32) {
                const unsigned char* src = stg + r * 128 + (((j * es / 16) ^ (r & 7)) << 4) + j * es % 16;
                unsigned char* dst = out + ((row_base + row) * o.ld + col + j) * es;
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

// An output warp's 32 rows and the sums [FROM, FROM + COUNT) of each, to the output from column `col` on: one rounding.
template <int FROM, int COUNT, int COLS>
__device__ __forceinline__ void bring_out(const RowsOut& o, const float (&sum)[COLS], unsigned char* stg, int32_t my_row, int64_t row_base,
                                          int col) {
    const int lane = threadIdx.x & 31;
    if (o.type == NNUE_T_F32) {
#pragma unroll
        for (int h = 0; h < COUNT; h += 32) {
            if (col + h >= o.cols) break;
            const float* v = sum + FROM + h;
#pragma unroll
            for (int p = 0; p < 8; ++p)
                *reinterpret_cast<float4*>(stg + lane * 128 + ((p ^ (lane & 7)) << 4)) = make_float4(v[4 * p], v[4 * p + 1], v[4 * p + 2], v[4 * p + 3]);
            copy_rows_out<128>(o, stg, my_row, row_base, col + h);
        }
    } else {
        constexpr int kPass = COUNT < 64 ? COUNT : 64;
#pragma unroll
        for (int h = 0; h < COUNT; h += kPass) {
            if (col + h >= o.cols) break;
            const float* v = sum + FROM + h;
#pragma unroll
            for (int p = 0; p < kPass / 8; ++p) {
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = pack_half(v[8 * p + 2 * j], v[8 * p + 2 * j + 1], o.type);
                *reinterpret_cast<uint4*>(stg + lane * 128 + ((p ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            copy_rows_out<kPass * 2>(o, stg, my_row, row_base, col + h);
        }
    }
}

#endif  // __CUDACC__

}  // namespace nnue
