// Shared declarations of the bucketed ("grouped by expert") matrix products: the plan of a batch, the element types of
// the C ABI and conversions between them.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace nnue {

constexpr int kGroupRows = 128;       // rows per tile of the plan: M of one CTA's tensor-core instructions
constexpr int kGroupPairRows = 256;   // rows per tile of a pair of CTAs
constexpr int kGroupAlign = 64;       // rows laid out by bucket: every bucket starts at a multiple of this, zeros between
constexpr int kMaxGroups = 1024;

__host__ __device__ inline int64_t pad4(int64_t n) { return (n + 3) / 4 * 4; }

// A tile of the plan: `count` rows of one bucket, at order[start]; `place` is the first row's place among rows laid out by
// bucket.  bucket == groups: rows of no bucket (no place).
struct GroupTile {
    int32_t bucket, start, count, place;
};

struct GroupPlanView {
    const int32_t* n_tiles;   // [2]: tiles of 128 rows, of 256 rows
    const int32_t* offsets;   // [E + 2]: first place of each bucket in `order`, of the rows without one, T
    const int32_t* order;     // [T] rows by bucket, in their own order inside a bucket
    const int32_t* places;    // [E + 1]: first place of each bucket among rows laid out by bucket, and their number
    const int32_t* first;     // [E + 1]: first tile of 128 rows of each bucket
    const GroupTile* tiles;   // [<= group_max_tiles]
    const GroupTile* pairs;   // [<= group_max_tiles]
};

__host__ __device__ inline int64_t group_max_tiles(int64_t T, int32_t E) {
    const int64_t by_rows = (T + kGroupRows - 1) / kGroupRows + E + 1;
    return by_rows < T ? by_rows : T;  // every tile holds a row
}

// Rows of a buffer that holds a batch laid out by bucket: it ends with the last bucket's multiple of kGroupAlign rows, at the
// most.  A tile's box of 128 rows may reach behind it: the tensor map has this number of rows, and what lies behind reads as
// zeros.  Plain loads have to stay below the tile's count, rounded up to kGroupAlign.
__host__ __device__ inline int64_t group_laid_rows(int64_t T, int32_t E) {
    return T + (int64_t)(kGroupAlign - 1) * (E < T ? E : T);
}

// int32 words: [0], [1] tiles, [4..] offsets, order, places, first tiles, tiles, pairs, then the counters of the launches
// for long batches
__host__ __device__ inline int64_t group_offsets_at() { return 4; }
__host__ __device__ inline int64_t group_order_at(int32_t E) { return 4 + pad4(E + 2); }
__host__ __device__ inline int64_t group_places_at(int64_t T, int32_t E) { return group_order_at(E) + pad4(T); }
__host__ __device__ inline int64_t group_first_at(int64_t T, int32_t E) { return group_places_at(T, E) + pad4(E + 1); }
__host__ __device__ inline int64_t group_tiles_at(int64_t T, int32_t E) { return group_first_at(T, E) + pad4(E + 1); }
__host__ __device__ inline int64_t group_pairs_at(int64_t T, int32_t E) { return group_tiles_at(T, E) + 4 * group_max_tiles(T, E); }
__host__ __device__ inline int64_t group_counts_at(int64_t T, int32_t E) { return group_pairs_at(T, E) + 4 * group_max_tiles(T, E); }

__host__ __device__ inline GroupPlanView group_view(const void* plan, int64_t T, int32_t E) {
    const int32_t* p = static_cast<const int32_t*>(plan);
    GroupPlanView v;
    v.n_tiles = p;
    v.offsets = p + group_offsets_at();
    v.order = p + group_order_at(E);
    v.places = p + group_places_at(T, E);
    v.first = p + group_first_at(T, E);
    v.tiles = reinterpret_cast<const GroupTile*>(p + group_tiles_at(T, E));
    v.pairs = reinterpret_cast<const GroupTile*>(p + group_pairs_at(T, E));
    return v;
}

inline int type_bytes(int32_t t) { return t == NNUE_T_F32 ? 4 : (t == NNUE_T_BF16 || t == NNUE_T_F16) ? 2 : 1; }
inline bool is_float_type(int32_t t) { return t == NNUE_T_F32 || t == NNUE_T_BF16 || t == NNUE_T_F16; }
inline bool is_half_type(int32_t t) { return t == NNUE_T_BF16 || t == NNUE_T_F16; }

#ifdef __CUDACC__
__device__ __forceinline__ bool type_is_byte(int32_t t) { return t == NNUE_T_E4M3 || t == NNUE_T_E5M2; }

// element `i` of an array of type `t` (F32, BF16 or F16) as fp32; exact
__device__ __forceinline__ float load_as_float(const void* p, int32_t t, int64_t i) {
    if (t == NNUE_T_F32) return __ldg(static_cast<const float*>(p) + i);
    if (t == NNUE_T_BF16) return __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(p) + i));
    return __half2float(__ldg(static_cast<const __half*>(p) + i));
}
// one rounding (to nearest, ties to even), none for F32
__device__ __forceinline__ void store_from_float(void* p, int32_t t, int64_t i, float v) {
    if (t == NNUE_T_F32) static_cast<float*>(p)[i] = v;
    else if (t == NNUE_T_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    else static_cast<__half*>(p)[i] = __float2half_rn(v);
}
#endif

}  // namespace nnue
