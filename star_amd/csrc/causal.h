// What the kernels on 16-bit tiles share (causal.hip, kv8.hip): the two input types, their MFMAs and the LDS tile.
#pragma once
#include "common.h"

namespace star {

constexpr float A_LOG2E = 1.4426950408889634f;
constexpr float A_LN2 = 0.6931471805599453f;
constexpr float M_NONE = -1.0e30f;       // running maximum before the first visible key (finite: no inf - inf)
constexpr float M_SLACK = 8.0f;          // log2 units: the running maximum follows only when a tile exceeds it by 2^8

template <typename T> struct Vec;
template <> struct Vec<__bf16> { typedef bf16x8 x8; typedef bf16x4 x4; };
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;
template <> struct Vec<_Float16> { typedef f16x8 x8; typedef f16x4 x4; };
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;

// D[row 4g+i][col r16] += sum_k A[row][k] B[k][col]; lane (g = lane / 16, r16 = lane % 16) holds A[r16][8g..8g+7],
// B[8g..8g+7][r16] and D[4g..4g+3][r16]
__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// two accumulator blocks (rows 4g+i of two 16-row tiles) -> the 8 contraction slots of a B operand.  The contraction
// order is then (tile 0 rows 4g..4g+3, tile 1 rows 4g..4g+3); tile_tr8 reads the A side in the same order.
template <typename T>
__device__ __forceinline__ typename Vec<T>::x8 pack_b(const f32x4& t0, const f32x4& t1) {
    typename Vec<T>::x8 r;
#pragma unroll
    for (int j = 0; j < 4; ++j) { r[j] = (T)t0[j]; r[4 + j] = (T)t1[j]; }
    return r;
}

// An LDS tile of ROWS rows of HD 16-bit values.  Rows are 128 or 256 bytes (HD = 96 leaves the last 64 bytes unused)
// and their 16-byte chunks are permuted by the row, so that both ways of reading it are free of bank conflicts:
//   row8   16 rows x 4 chunks of one wave, for operands that contract over HD
//   tr8    ds_read_b64_tr_b16: 4 rows x 16 columns per 16 lanes, transposed, for operands that contract over rows
template <typename T, int HD>
struct Tile {
    static constexpr int ROWB = HD == 64 ? 128 : 256;
    static constexpr int CHUNKS = HD / 8;
    __device__ static __forceinline__ int swz(int r) {
        if constexpr (HD == 64) return (((r >> 1) & 1) << 2) | (((r >> 2) & 1) << 1) | ((r >> 2) & 1);
        else return (r & 7) << 1;
    }
    // rows row0 + r16, values 32 ks + 8 g ..
    __device__ static __forceinline__ typename Vec<T>::x8 row8(const uint8_t* tile, int row0, int ks, int lane) {
        const int r = lane & 15, g = lane >> 4;
        return *(const typename Vec<T>::x8*)(tile + (row0 + r) * ROWB + (((4 * ks + g) ^ swz(r)) << 4));
    }
    // column 16 nt + r16 of rows row0 + 4g .. + 3 and row0 + 16 + 4g .. + 3
    __device__ static __forceinline__ typename Vec<T>::x8 tr8(const uint8_t* tile, int row0, int nt, int lane) {
        const int r = lane & 15, g = lane >> 4;
        const int row = 4 * g + (r >> 2);
        const uint8_t* p = tile + (row0 + row) * ROWB + (((2 * nt + ((r >> 1) & 1)) ^ swz(row)) << 4) + 8 * (r & 1);
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(LDS_PTR(s16x4, p));
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(LDS_PTR(s16x4, p + 16 * ROWB));
        return __builtin_bit_cast(typename Vec<T>::x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
};

// A tile on its way from global memory through registers: load() asks for it, store() puts it into LDS after the
// tile before it has been used.  Rows at or past `limit` read row limit - 1 (their weights are exact zeros).
template <typename T, int HD, int ROWS, int NTH>
struct TileLoad {
    static constexpr int CHUNKS = HD / 8, TOTAL = ROWS * CHUNKS, N = (TOTAL + NTH - 1) / NTH;
    u32x4 v[N];
    __device__ __forceinline__ void load(const T* __restrict__ g, int64_t sr, int row0, int limit, int tid) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = tid + i * NTH;
            const int row = min(row0 + c / CHUNKS, limit - 1);
            v[i] = *(const u32x4*)(g + (int64_t)row * sr + (c % CHUNKS) * 8);
        }
    }
    __device__ __forceinline__ void store(uint8_t* tile, int tid) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = tid + i * NTH, row = c / CHUNKS;
            if (TOTAL % NTH == 0 || c < TOTAL)
                *(u32x4*)(tile + row * Tile<T, HD>::ROWB + (((c % CHUNKS) ^ Tile<T, HD>::swz(row & 15)) << 4)) = v[i];
        }
    }
};

}  // namespace star
