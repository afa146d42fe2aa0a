// What the kernels on 16-bit tiles share (causal.hip, kv8.hip): the two input types, their MFMAs and the LDS tile.
#pragma once
#include "common.h"

namespace star {

constexpr float A_LOG2E = 1.4426950408889634f;
constexpr float A_LN2 = 0.6931471805599453f;
// Running maximum before the first visible key: the lowest finite value (no inf - inf), so that no finite logit is below it
constexpr float M_NONE = -3.402823466e38f;
constexpr float M_SLACK = 8.0f;          // log2 units: the running maximum follows only when a tile exceeds it by 2^8

constexpr float M_MOST = 4096.0f;        // largest sum of a lane's weights of a tile against an earlier tile's maximum

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
__device__ __forceinline__ typename Vec<T>::x4 pack4(const f32x4& t) {
    return (typename Vec<T>::x4){(T)t[0], (T)t[1], (T)t[2], (T)t[3]};
}
template <typename X4>
__device__ __forceinline__ auto join8(const X4& a, const X4& b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }
template <typename T>
__device__ __forceinline__ typename Vec<T>::x8 pack_b(const f32x4& t0, const f32x4& t1) {
    return join8(pack4<T>(t0), pack4<T>(t1));
}

// An LDS tile of rows of HD 16-bit values, read in two ways, each from one address per lane plus constants:
//   row8   16 rows x 4 chunks of 16 bytes of one wave, for operands that contract over HD
//   tr8    ds_read_b64_tr_b16: 8 rows x 32 bytes of one half wave, transposed, for operands that contract over rows
// A row is HD * 2 + 32 bytes, twice an odd number of 16-byte chunks, so 8 neighbouring rows begin 32 bytes apart or more
// in the 256-byte bank cycle, which is what tr8 reads at once, and rows r and r + 8 begin alike, which row8 never meets:
// a wave's 16-byte reads go 16 lanes at a time, 8 rows of one chunk with the other 8 of its neighbour.
template <typename T, int HD>
struct Tile {
    static constexpr int ROWB = HD * 2 + 32;
    static constexpr int CHUNKS = HD / 8;
    // rows row0 + r16, values 32 ks + 8 g ..
    __device__ static __forceinline__ typename Vec<T>::x8 row8(const uint8_t* tile, int row0, int ks, int lane) {
        const int r = lane & 15, g = lane >> 4;
        return *(const typename Vec<T>::x8*)(tile + r * ROWB + 16 * g + row0 * ROWB + 64 * ks);
    }
    // column 16 nt + r16 of rows row0 + 4g .. + 3 and row0 + 16 + 4g .. + 3
    __device__ static __forceinline__ typename Vec<T>::x8 tr8(const uint8_t* tile, int row0, int nt, int lane) {
        const int r = lane & 15, g = lane >> 4;
        const uint8_t* p = tile + (4 * g + (r >> 2)) * ROWB + 8 * (r & 3) + row0 * ROWB + 32 * nt;
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(LDS_PTR(s16x4, p));
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(LDS_PTR(s16x4, p + 16 * ROWB));
        return __builtin_bit_cast(typename Vec<T>::x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
};

// A tile on its way from global memory through registers: load() asks for it, store() puts it into LDS after the
// tile before it has been used.  Rows at or past `limit` read row limit - 1 (their weights are exact zeros).  A thread's
// place in a whole tile is a 32-bit byte offset (ROWS * sr * 2 < 2^32, checked on the host) from the tile's scalar
// address, found once.
template <typename T, int HD, int ROWS, int NTH>
struct TileLoad {
    static constexpr int CHUNKS = HD / 8, TOTAL = ROWS * CHUNKS, N = (TOTAL + NTH - 1) / NTH;
    static constexpr bool EVEN = NTH % CHUNKS == 0;                // chunk i then lies i * NTH / CHUNKS whole rows further
    u32x4 v[N];
    uint32_t at[EVEN ? 1 : N];
    __device__ __forceinline__ void place(int64_t sr, int tid) {
#pragma unroll
        for (int i = 0; i < (EVEN ? 1 : N); ++i) {
            const int c = min(tid + i * NTH, TOTAL - 1);
            at[i] = (uint32_t)(c / CHUNKS) * (uint32_t)(sr * 2) + (uint32_t)(c % CHUNKS) * 16;
        }
    }
    __device__ __forceinline__ void load(const T* __restrict__ g, int64_t sr, int row0, int limit, int tid) {
        const char* p = (const char*)(g + (int64_t)row0 * sr);
        if (row0 + ROWS <= limit) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if constexpr (EVEN) v[i] = *(const u32x4*)(p + i * (NTH / CHUNKS) * (sr * 2) + at[0]);
                else v[i] = *(const u32x4*)(p + at[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int c = min(tid + i * NTH, TOTAL - 1);
                v[i] = *(const u32x4*)(p + (int64_t)min(c / CHUNKS, limit - 1 - row0) * (sr * 2) + (c % CHUNKS) * 16);
            }
        }
    }
    __device__ __forceinline__ void store(uint8_t* tile, int tid) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = tid + i * NTH, row = c / CHUNKS;
            if (TOTAL % NTH == 0 || c < TOTAL)
                *(u32x4*)(tile + row * Tile<T, HD>::ROWB + (c % CHUNKS) * 16) = v[i];
        }
    }
};

// A row's softmax state in parts: part p's maximum and sum at ml[2 p stride], its HD weighted sums at o[p stride HD].  One
// wave adds them up, HD / 4 lanes a part, two or four parts side by side, eight of each on their way at once.  What the
// first trip to memory can hold is asked for in ask(), before anything is waited for; sum() then leaves the whole's
// maximum and sum of weights in every lane and four of the sums in each lane below HD / 4.
template <int HD>
struct PartSum {
    static constexpr int D4 = HD / 4, G = 64 / D4, U = 8;
    const float *o, *ml;
    int64_t stride;
    int np, at, d4;
    f32x4 x[U];
    float m0, l0;
    __device__ __forceinline__ void load(int i) {
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = *(const f32x4*)(o + min(i + u * G + at, np - 1) * stride * HD + 4 * d4);
    }
    __device__ __forceinline__ void ask(const float* o_, const float* ml_, int64_t stride_, int np_, int lane) {
        o = o_, ml = ml_, stride = stride_, np = np_;
        at = min(lane / D4, G - 1), d4 = lane % D4;                // (96: the last 16 lanes repeat and are not added)
        const float* p = ml + 2 * min(lane, np - 1) * stride;
        m0 = p[0], l0 = p[1];
        load(0);
    }
    __device__ __forceinline__ void sum(int lane, float& mm, float& ll, f32x4& r) {
        mm = m0;
        for (int p = 64 + lane; p < np; p += 64) mm = fmaxf(mm, ml[2 * p * stride]);
#pragma unroll
        for (int k = 32; k > 0; k >>= 1) mm = fmaxf(mm, __shfl_xor(mm, k, 64));
        ll = 0.f;
        r = (f32x4){0.f, 0.f, 0.f, 0.f};
        for (int c0 = 0; c0 < np; c0 += 64) {
            const int cnt = min(np - c0, 64);
            if (c0 > 0) {
                const float* p = ml + 2 * (c0 + min(lane, cnt - 1)) * stride;
                m0 = p[0], l0 = p[1];
            }
            const float f = lane < cnt ? __builtin_amdgcn_exp2f(m0 - mm) : 0.f;
            if (lane < cnt) ll += f * l0;
            for (int i = 0; i < cnt; i += G * U) {
                if (c0 + i > 0) load(c0 + i);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int p = i + u * G + at;
                    const float w = __shfl(f, min(p, 63), 64);
                    if (p < cnt) r += w * x[u];
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float t = r[e];
            if constexpr (HD == 64) t += __shfl_xor(t, 16, 64);
            t += __shfl(t, HD == 96 ? min(lane + 24, 63) : lane ^ 32, 64);
            r[e] = t;
        }
        ll = wave_sum(ll);
    }
};

// A tile on its way through buffer loads, one 16-byte piece of a thread at a time and without a branch, so that the pieces
// can be asked for between other instructions: a load holds its wave for 64 clocks when the four waves of a workgroup
// ask at once, and eight in a row hold it longer than the products of a tile take.  Rows at or past `limit` are zeros
// by the range check (their weights are exact zeros as well), so a tile behind the last one is asked for like any other.
template <typename T, int HD, int ROWS, int NTH>
struct TileBuf {
    static constexpr int CHUNKS = HD / 8, TOTAL = ROWS * CHUNKS, N = (TOTAL + NTH - 1) / NTH;
    static constexpr bool EVEN = NTH % CHUNKS == 0 && TOTAL % NTH == 0;
    u32x4 v[N];
    uint32_t at[EVEN ? 1 : N];
    __device__ __forceinline__ void place(int64_t sr, int tid) {
#pragma unroll
        for (int i = 0; i < (EVEN ? 1 : N); ++i) {
            const int c = min(tid + i * NTH, TOTAL - 1);
            at[i] = (uint32_t)(c / CHUNKS) * (uint32_t)(sr * 2) + (uint32_t)(c % CHUNKS) * 16;
        }
    }
    // the rows from row0 on (at most (ROWS - 1) * 2^24 + HD * 2 bytes: row strides are below 2^23 values)
    __device__ static __forceinline__ auto rows(const T* g, int64_t sr, int row0, int limit) {
        const int n = max(0, min(ROWS, limit - row0)), bytes = ((n - 1) * (int)(sr * 2) + HD * 2) & (-n >> 31);   // (no branch)
        return __builtin_amdgcn_make_buffer_rsrc((void*)(g + (int64_t)row0 * sr), 0, bytes, 0x00020000);
    }
    template <typename R>
    __device__ __forceinline__ void load(R rows, int64_t sr) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t off = EVEN ? at[0] + i * (NTH / CHUNKS) * (uint32_t)(sr * 2) : at[i];
            v[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rows, off, 0, 0));
        }
    }
    __device__ __forceinline__ void store(uint8_t* tile, int tid) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = tid + i * NTH;
            if (TOTAL % NTH == 0 || c < TOTAL) *(u32x4*)(tile + c / CHUNKS * Tile<T, HD>::ROWB + (c % CHUNKS) * 16) = v[i];
        }
    }
};

// what __builtin_amdgcn_sched_group_barrier(kind, how many, 0) puts in order, one call after another, within a block of code
constexpr int SG_VALU = 0x2, SG_MFMA = 0x8, SG_VMEM_READ = 0x20, SG_DS_READ = 0x100, SG_DS_WRITE = 0x200;

}  // namespace star
