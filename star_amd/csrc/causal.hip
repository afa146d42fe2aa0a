// Causal self-attention of packed sequences, forward and backward (star_causal_* in star_nugget.h).
//
//   S = scale Q K^T over the keys j <= i + nk - nq,  P = softmax(S),  O = P V
//   dV = P^T dO,  dP = dO V^T,  dS = P (dP - rowsum(dO O)),  dQ = scale dS K,  dK = scale dS^T Q
//
// Both directions walk tiles of 64 rows of the other side with a running maximum and sum (forward) or the stored
// log-sum-exp (backward); no [nq, nk] tensor exists.  Two products per pair of rows forward, seven backward (the
// gradients of the queries and of the keys are two kernels, each recomputing P and dP in the order it needs: no
// atomics, the result does not depend on the order in which workgroups run).
//
// One operand of every product stays in registers, the other is read from LDS, where a 16-bit tile is read by rows or
// transposed from the same copy (Tile in causal.h).  The softmax side has the query on the MFMA column, so maximum and
// sum of a row are in-lane but for two shuffles, and the accumulator of S^T is, packed to 16 bits, the next operand.
#include "causal.h"
#include <type_traits>

namespace star {

constexpr int CT = STAR_CAUSAL_TILE;     // rows of one workgroup: 4 waves x 32
constexpr int CK = 64;                   // rows of the tiles it walks

struct Work { int q0, nq, k0, nk, first; };      // a tile's sequence (first query row, queries, first key row, keys), its first row
__device__ __forceinline__ Work work_of(const int32_t* tiles, int t) {
    const int32_t* w = tiles + 8 * (int64_t)t;
    return Work{w[0], w[1], w[2], w[3], w[4]};
}

// keys that the queries of a tile see
__device__ __forceinline__ int keys_seen(const Work& w) { return max(0, min(w.nk, min(w.first + CT, w.nq) + w.nk - w.nq)); }
// tiles of CQ queries that see keys of a tile, per head, and the first of them
constexpr int CQ = 32;
struct Walk { int first, n; };
__device__ __forceinline__ Walk queries_of(const Work& w) {
    const int first = max(0, w.first - (w.nk - w.nq)) / CQ;
    return Walk{first, max(0, (w.nq + CQ - 1) / CQ - first)};
}

// Few query tiles over long keys are cut along the keys: part p of `parts` walks its share of a tile's key tiles and
// leaves its softmax state, sums[tile][head][part][row][HD], then maximum and sum [tile][head][part][row][2].
struct KeyTiles { int first, end; };
__device__ __forceinline__ KeyTiles key_tiles(int keys, int part, int parts) {
    const int n = (keys + CK - 1) / CK, per = (n + parts - 1) / parts, first = min(n, part * per);
    return KeyTiles{first, min(n, first + per)};
}
struct Partial { float *o, *ml; };
template <int HD>
__device__ __forceinline__ Partial partial(float* sums, const star_causal_shape& s, int parts, int rows, int t, int part, int h, int row) {
    const int64_t at = (((int64_t)t * s.H + h) * parts + part) * rows + row, all = (int64_t)s.n_q_tiles * s.H * parts * rows;
    return Partial{sums + at * HD, sums + all * HD + at * 2};
}

// ------------------------------------------------------------------------------------------------------ forward
template <typename T, int HD>
__global__ __launch_bounds__(256, 2) void causal_fwd_kernel(const T* __restrict__ Q, const T* __restrict__ K,
                                                           const T* __restrict__ V, const int32_t* __restrict__ tiles, star_causal_shape s,
                                                           int parts, float* __restrict__ sums, T* __restrict__ O,
                                                           float* __restrict__ lse) {
    typedef typename Vec<T>::x8 x8;
    typedef typename Vec<T>::x4 x4;
    using Ti = Tile<T, HD>;
    constexpr int KS = HD / 32, NT = HD / 16;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    constexpr int TB = CK * Ti::ROWB;

    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    // consecutive workgroups go to consecutive XCDs: key heads first, so that the tiles and query heads that share a
    // key head meet in one L2 when Hkv is a multiple of 8
    const int hi = blockIdx.x % s.H, part = blockIdx.x / s.H % parts, t = blockIdx.x / s.H / parts;
    const int hk = hi % s.Hkv, h = hk * (s.H / s.Hkv) + hi / s.Hkv;
    const Work sq = work_of(tiles, t);
    const int i0 = sq.first;                               // first query of the workgroup
    const int off = sq.nk - sq.nq;
    const T* Qh = Q + (int64_t)sq.q0 * s.q_sr + (int64_t)h * s.q_sh;
    const T* Kh = K + (int64_t)sq.k0 * s.k_sr + (int64_t)hk * s.k_sh;
    const T* Vh = V + (int64_t)sq.k0 * s.v_sr + (int64_t)hk * s.v_sh;

    const int w0 = i0 + 32 * wid;                                  // first query of the wave
    int lim[2];                                                    // keys that this lane's query of block qb sees
    x8 qf[2][KS];
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
        const int i = w0 + 16 * qb + r16;
        lim[qb] = i < sq.nq ? max(0, min(sq.nk, i + off + 1)) : 0;
        const T* row = Qh + (int64_t)min(i, sq.nq - 1) * s.q_sr + 8 * g;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qf[qb][ks] = *(const x8*)(row + 32 * ks);
    }
    const int all_see = w0 + 32 <= sq.nq ? max(0, min(sq.nk, w0 + off + 1)) : 0;   // keys that every query of the wave sees
    const int wave_end = w0 < sq.nq ? max(0, min(sq.nk, min(w0 + 32, sq.nq) + off)) : 0;
    const int end = max(0, min(sq.nk, min(i0 + CT, sq.nq) + off)); // keys that any query of the workgroup sees
    const float c2 = s.scale * A_LOG2E;

    f32x4 oacc[2][NT];
    float m[2], l[2];
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) oacc[qb][nt] = (f32x4){0.f, 0.f, 0.f, 0.f};
        m[qb] = M_NONE;
        l[qb] = 0.f;
    }

    using Load = TileBuf<T, HD, CK, 256>;
    Load kl, vl;
    const KeyTiles kt_ = key_tiles(end, part, parts);
    const int ntile = kt_.end, mine = min(ntile, (wave_end + CK - 1) / CK);    // (tiles that the wave's queries see)
    kl.place(s.k_sr, tid);
    vl.place(s.v_sr, tid);
    auto ask = [&](int tile) {
        const int limit = tile < ntile ? sq.nk : 0;
        kl.load(Load::rows(Kh, s.k_sr, tile * CK, limit), s.k_sr);
        vl.load(Load::rows(Vh, s.v_sr, tile * CK, limit), s.v_sr);
    };
    auto put = [&](int tile) {
        uint8_t* kt = smem + (tile & 1) * 2 * TB;
        kl.store(kt, tid);
        vl.store(kt + TB, tid);
    };
    // A step multiplies S, forms the weights while the next tile goes from registers to LDS, and multiplies O while the one
    // after it is asked for.  The order of the instructions is given: with loads and stores in front of the step
    // 12001 tokens took 562 us, 523 so.
    int tile = kt_.first;
    ask(tile);
    put(tile);
    ask(tile + 1);
#pragma unroll 1
    for (; tile < mine; ++tile) {
        const uint8_t *kt = smem + (tile & 1) * 2 * TB, *vt = kt + TB;
        __syncthreads();                                           // the tile is there, the one before is done with
        const int key0 = tile * CK;

        f32x4 sc[2][4];
#pragma unroll
        for (int kt4 = 0; kt4 < 4; ++kt4) {
            x8 kf[KS];
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) kf[ks] = Ti::row8(kt, 16 * kt4, ks, lane);
#pragma unroll
            for (int qb = 0; qb < 2; ++qb) {
                sc[qb][kt4] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) sc[qb][kt4] = mfma16(kf[ks], qf[qb][ks], sc[qb][kt4]);
            }
        }
        __builtin_amdgcn_sched_group_barrier(SG_DS_READ, 4, 0);
#pragma unroll
        for (int j = 0; j < 4 * KS; ++j) {
            __builtin_amdgcn_sched_group_barrier(SG_MFMA, 2, 0);
            if (j + 4 < 4 * KS) __builtin_amdgcn_sched_group_barrier(SG_DS_READ, 1, 0);
        }
        if (key0 + CK > all_see) {                                 // (wave-uniform) some query does not see the whole tile
#pragma unroll
            for (int qb = 0; qb < 2; ++qb)
#pragma unroll
                for (int kt4 = 0; kt4 < 4; ++kt4)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        sc[qb][kt4][i] = key0 + 16 * kt4 + 4 * g + i < lim[qb] ? sc[qb][kt4][i] : -INFINITY;
        }
        // The weights are formed against the maximum of an earlier tile and only their sum is looked at: while it stays
        // under M_MOST no weight can have overflowed 16 bits, and the tile needs no maximum of its own.  The first visible
        // tile (M_NONE makes the sum infinite) and a rise of the logits by 12 in log2 take the other way once.
        x8 pf[2][2];
        float sum[2];
        auto weights = [&](int qb) {
            sum[qb] = 0.f;
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                f32x4 p[2];
#pragma unroll
                for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        p[k2][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[qb][2 * hf + k2][i], c2, -m[qb]));
                        sum[qb] += p[k2][i];
                    }
                pf[qb][hf] = pack_b<T>(p[0], p[1]);
            }
        };
        put(tile + 1);
        weights(0);
        weights(1);
#pragma unroll
        for (int i = 0; i < 2 * Load::N; ++i) {
            __builtin_amdgcn_sched_group_barrier(SG_VALU, 16, 0);
            __builtin_amdgcn_sched_group_barrier(SG_DS_WRITE, 1, 0);
        }
        if (!__all(sum[0] < M_MOST && sum[1] < M_MOST)) {
#pragma unroll
            for (int qb = 0; qb < 2; ++qb) {
                float mx = sc[qb][0][0];                           // of the raw products: the scale is positive
#pragma unroll
                for (int kt4 = 0; kt4 < 4; ++kt4)
#pragma unroll
                    for (int i = 0; i < 4; ++i) mx = fmaxf(mx, sc[qb][kt4][i]);
                mx *= c2;
                mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
                mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
                int over = !(sum[qb] < M_MOST);                    // of this row: no other row of the wave changes its bits
                over |= __shfl_xor(over, 16, 64);
                over |= __shfl_xor(over, 32, 64);
                const float mn = over ? fmaxf(m[qb], mx) : m[qb], a = __builtin_amdgcn_exp2f(m[qb] - mn);
                m[qb] = mn;
                l[qb] *= a;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) oacc[qb][nt][i] *= a;
                weights(qb);
            }
        }
        l[0] += sum[0];
        l[1] += sum[1];
        ask(tile + 2);
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const x8 vf = Ti::tr8(vt, 32 * hf, nt, lane);
#pragma unroll
                for (int qb = 0; qb < 2; ++qb) oacc[qb][nt] = mfma16(vf, pf[qb][hf], oacc[qb][nt]);
            }
        __builtin_amdgcn_sched_group_barrier(SG_DS_READ, 8, 0);    // (two reads a fragment)
#pragma unroll
        for (int j = 0; j < 2 * NT; ++j) {
            __builtin_amdgcn_sched_group_barrier(SG_MFMA, 2, 0);
            if (j + 4 < 2 * NT) __builtin_amdgcn_sched_group_barrier(SG_DS_READ, 2, 0);
            if (j % (NT / Load::N) == 0) __builtin_amdgcn_sched_group_barrier(SG_VMEM_READ, 1, 0);
        }
    }
#pragma unroll 1
    for (; tile < ntile; ++tile) {                                 // tiles for other waves
        __syncthreads();
        put(tile + 1);
        ask(tile + 2);
    }

#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
        float sum = l[qb];
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        const int i = w0 + 16 * qb + r16;
        if (i >= sq.nq) continue;
        if (parts > 1) {
            const Partial p = partial<HD>(sums, s, parts, CT, t, part, h, i - i0);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) *(f32x4*)(p.o + 16 * nt + 4 * g) = oacc[qb][nt];
            if (g == 0) { p.ml[0] = m[qb]; p.ml[1] = sum; }
            continue;
        }
        const float inv = sum > 0.f ? 1.0f / sum : (sum == 0.f ? 0.f : sum);   // no visible key: 0; NaN stays NaN
        T* orow = O + (int64_t)(sq.q0 + i) * s.o_sr + (int64_t)h * s.o_sh + 4 * g;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            x4 o4;
#pragma unroll
            for (int e = 0; e < 4; ++e) o4[e] = (T)(oacc[qb][nt][e] * inv);
            *(x4*)(orow + 16 * nt) = o4;
        }
        if (g == 0 && lse) lse[(int64_t)h * s.lse_stride + sq.q0 + i] = sum == 0.f ? -INFINITY : m[qb] * A_LN2 + logf(sum);
    }
}

// The same for sequences of at most 16 * QB queries each (a chunk of a stream, a speculated run of tokens): the waves of
// a workgroup share the queries and take the 64-key tiles in turn, each with K straight from memory in registers (its
// rows are the operand) and V through an LDS tile of its own, so no wave waits for another before the four softmax states
// are joined at the end.  Bound by the latency of two dependent trips to memory per 256 keys: one utterance of 375 frames,
// 16 queries, 8 heads of 128 takes 8.4 us, 13.1 with the kernel above, whose waves would share keys and leave three of
// four without a query.
template <typename T, int HD, int QB>
__global__ __launch_bounds__(256, 1) void causal_few_kernel(const T* __restrict__ Q, const T* __restrict__ K,
                                                           const T* __restrict__ V, const int32_t* __restrict__ tiles, star_causal_shape s,
                                                           int parts, float* __restrict__ sums, T* __restrict__ O,
                                                           float* __restrict__ lse) {
    typedef typename Vec<T>::x8 x8;
    using Ti = Tile<T, HD>;
    constexpr int KS = HD / 32, NT = HD / 16, OP = HD + 4;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    __shared__ float msh[4 * 16 * QB], lsh[4 * 16 * QB];

    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    const int hi = blockIdx.x % s.H, part = blockIdx.x / s.H % parts, t = blockIdx.x / s.H / parts;
    const int hk = hi % s.Hkv, h = hk * (s.H / s.Hkv) + hi / s.Hkv;
    const Work sq = work_of(tiles, t);
    const int off = sq.nk - sq.nq;                                 // (the last query sees every key)
    const KeyTiles kt_ = key_tiles(sq.nk, part, parts);
    const int end = min(sq.nk, kt_.end * CK);
    const T* Kh = K + (int64_t)sq.k0 * s.k_sr + (int64_t)hk * s.k_sh;
    const T* Vh = V + (int64_t)sq.k0 * s.v_sr + (int64_t)hk * s.v_sh;
    int lim[QB];
    x8 qf[QB][KS];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        const int i = 16 * qb + r16;
        lim[qb] = i < sq.nq ? max(0, min(sq.nk, i + off + 1)) : 0;
        const T* row = Q + (int64_t)(sq.q0 + min(i, sq.nq - 1)) * s.q_sr + (int64_t)h * s.q_sh + 8 * g;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qf[qb][ks] = *(const x8*)(row + 32 * ks);
    }
    const int all_see = sq.nq == 16 * QB ? max(0, off + 1) : 0;
    const float c2 = s.scale * A_LOG2E;
    f32x4 acc[QB][NT];
    float m[QB], l[QB];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[qb][nt] = (f32x4){0.f, 0.f, 0.f, 0.f};
        m[qb] = M_NONE;
        l[qb] = 0.f;
    }
    uint8_t* vt = smem + wid * CK * Ti::ROWB;
#pragma unroll 1
    for (int key0 = (kt_.first + wid) * CK; key0 < end; key0 += 4 * CK) {
        TileLoad<T, HD, CK, 64> vl;
        vl.place(s.v_sr, lane);
        vl.load(Vh, s.v_sr, key0, sq.nk, lane);
        f32x4 sc[QB][4];
#pragma unroll
        for (int kt4 = 0; kt4 < 4; ++kt4) {
            const T* row = Kh + (int64_t)min(key0 + 16 * kt4 + r16, sq.nk - 1) * s.k_sr + 8 * g;
            x8 kf[KS];
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) kf[ks] = *(const x8*)(row + 32 * ks);
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) {
                sc[qb][kt4] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) sc[qb][kt4] = mfma16(kf[ks], qf[qb][ks], sc[qb][kt4]);
            }
        }
        __builtin_amdgcn_wave_barrier();                           // (the reads of the tile before are behind: LDS is in order)
        vl.store(vt, lane);
        __builtin_amdgcn_wave_barrier();
        if (key0 + CK > all_see) {
#pragma unroll
            for (int qb = 0; qb < QB; ++qb)
#pragma unroll
                for (int kt4 = 0; kt4 < 4; ++kt4)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        sc[qb][kt4][i] = key0 + 16 * kt4 + 4 * g + i < lim[qb] ? sc[qb][kt4][i] : -INFINITY;
        }
        x8 pf[QB][2];
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
            float mx = sc[qb][0][0];
#pragma unroll
            for (int kt4 = 0; kt4 < 4; ++kt4)
#pragma unroll
                for (int i = 0; i < 4; ++i) mx = fmaxf(mx, sc[qb][kt4][i]);
            mx *= c2;
            if (!__all(mx <= m[qb] + M_SLACK)) {
                mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
                mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
                const float mn = fmaxf(m[qb], mx), a = __builtin_amdgcn_exp2f(m[qb] - mn);
                m[qb] = mn;
                l[qb] *= a;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[qb][nt][i] *= a;
            }
            float sum = 0.f;
#pragma unroll
            for (int kt4 = 0; kt4 < 4; ++kt4)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[qb][kt4][i], c2, -m[qb]));
                    sum += p;
                    sc[qb][kt4][i] = p;
                }
            l[qb] += sum;
            pf[qb][0] = pack_b<T>(sc[qb][0], sc[qb][1]);
            pf[qb][1] = pack_b<T>(sc[qb][2], sc[qb][3]);
        }
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const x8 vf = Ti::tr8(vt, 32 * hf, nt, lane);
#pragma unroll
                for (int qb = 0; qb < QB; ++qb) acc[qb][nt] = mfma16(vf, pf[qb][hf], acc[qb][nt]);
            }
    }
    // join the four waves
    float* osh = (float*)smem;                                     // [4][16 * QB][OP], over the tiles
    __syncthreads();
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        float sum = l[qb];
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        const int row = (wid * QB + qb) * 16 + r16;
        if (g == 0) {
            msh[row] = m[qb];
            lsh[row] = sum;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) *(f32x4*)(osh + row * OP + 16 * nt + 4 * g) = acc[qb][nt];
    }
    __syncthreads();
    constexpr int PER = HD / 16;
    for (int row = tid >> 4; row < min(sq.nq, 16 * QB); row += 16) {
        const int d0 = (tid & 15) * PER;
        float mm = M_NONE, ll = 0.f, o[PER];
#pragma unroll
        for (int w = 0; w < 4; ++w) mm = fmaxf(mm, msh[w * 16 * QB + row]);
#pragma unroll
        for (int e = 0; e < PER; ++e) o[e] = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = __builtin_amdgcn_exp2f(msh[w * 16 * QB + row] - mm);
            ll += f * lsh[w * 16 * QB + row];
#pragma unroll
            for (int e = 0; e < PER; ++e) o[e] += f * osh[(w * 16 * QB + row) * OP + d0 + e];
        }
        if (parts > 1) {
            const Partial p = partial<HD>(sums, s, parts, 16 * QB, t, part, h, row);
#pragma unroll
            for (int e = 0; e < PER; ++e) p.o[d0 + e] = o[e];
            if ((tid & 15) == 0) { p.ml[0] = mm; p.ml[1] = ll; }
            continue;
        }
        const float inv = ll > 0.f ? 1.0f / ll : ll;               // no visible key: 0; NaN stays NaN
        T* orow = O + (int64_t)(sq.q0 + row) * s.o_sr + (int64_t)h * s.o_sh + d0;
#pragma unroll
        for (int e = 0; e < PER; ++e) orow[e] = (T)(o[e] * inv);
        if ((tid & 15) == 0 && lse) lse[(int64_t)h * s.lse_stride + sq.q0 + row] = ll == 0.f ? -INFINITY : mm * A_LN2 + logf(ll);
    }
}

// The states that the parts of a row's keys left, joined: W waves a row, each adding up its share of the parts.
template <typename T, int HD, int W>
__global__ __launch_bounds__(256) void causal_join_kernel(const int32_t* __restrict__ tiles,
                                                         star_causal_shape s, int parts, int rows, const float* __restrict__ sums,
                                                         T* __restrict__ O, float* __restrict__ lse) {
    __shared__ __attribute__((aligned(16))) float osh[W > 1 ? W * HD : 4];
    __shared__ float msh[4], lsh[4];
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = blockIdx.y * (4 / W) + wid / W;
    const int h = blockIdx.x % s.H, t = blockIdx.x / s.H;
    const int per = (parts + W - 1) / W, p0 = min(wid % W * per, parts - 1);
    const Partial x = partial<HD>((float*)sums, s, parts, rows, t, p0, h, row);
    PartSum<HD> ps;
    ps.ask(x.o, x.ml, rows, min(per, parts - p0), lane);           // (rows that the tile lacks have room as well)
    const Work sq = work_of(tiles, t);
    const int i = sq.first + row;
    if (i >= sq.nq) return;                                        // (a row's waves alike)
    float mm, ll;
    f32x4 o;
    ps.sum(lane, mm, ll, o);
    if constexpr (W > 1) {
        if (lane < HD / 4) *(f32x4*)(osh + wid * HD + 4 * lane) = o;
        if (lane == 0) msh[wid] = mm, lsh[wid] = ll;
        __syncthreads();
        if (wid > 0 || lane >= HD / 4) return;
        mm = fmaxf(fmaxf(msh[0], msh[1]), fmaxf(msh[2], msh[3]));
        ll = 0.f;
        o = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < W; ++w) {
            if (w * per >= parts) break;
            const float f = __builtin_amdgcn_exp2f(msh[w] - mm);
            o += f * *(const f32x4*)(osh + w * HD + 4 * lane);
            ll += f * lsh[w];
        }
    }
    if (lane >= HD / 4) return;
    const float inv = ll > 0.f ? 1.0f / ll : ll;                   // no visible key: 0; NaN stays NaN
    *(typename Vec<T>::x4*)(O + (int64_t)(sq.q0 + i) * s.o_sr + (int64_t)h * s.o_sh + 4 * lane) = pack4<T>(o * inv);
    if (lane == 0 && lse) lse[(int64_t)h * s.lse_stride + sq.q0 + i] = ll == 0.f ? -INFINITY : mm * A_LN2 + logf(ll);
}

// ------------------------------------------------------------------------------------------------------ gradient of Q
// The forward's walk with dP^T = V dO^T beside S^T = K Q^T; dQ^T += K^T dS^T with K read transposed from the same tile.
// Also writes delta = rowsum(dO O) for the kernel below.  o has been rounded to 16 bits, which weighs most where a row
// sees few keys and |o| is not small against |V|: with o's delta the error of dQ and dK was 1.55 times that of rounding
// the exact gradients once.  A workgroup that sees at most two tiles of keys therefore walks them twice, first for
// delta = sum_j P dP in 32 bits; its walk is the shortest there is.
// A launch of few workgroups or very unequal ones is cut: part p takes tiles p * per .. of a walk, and a walk of more than
// one part leaves fp32 sums, which causal_dq_sum_kernel adds up in order.
template <typename T, int HD>
__global__ __launch_bounds__(256, 2) void causal_dq_kernel(const T* __restrict__ Q, const T* __restrict__ K,
                                                          const T* __restrict__ V, const T* __restrict__ O,
                                                          const T* __restrict__ dO, const float* __restrict__ lse,
                                                          const int32_t* __restrict__ tiles, star_causal_shape s, int parts, int per,
                                                          float* __restrict__ sums, T* __restrict__ dQ, float* __restrict__ delta) {
    typedef typename Vec<T>::x8 x8;
    typedef typename Vec<T>::x4 x4;
    using Ti = Tile<T, HD>;
    constexpr int KS = HD / 32, NT = HD / 16;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    constexpr int TB = CK * Ti::ROWB;

    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    const int hi = blockIdx.x % s.H, part = blockIdx.x / s.H % parts, t = blockIdx.x / s.H / parts;
    const int hk = hi % s.Hkv, h = hk * (s.H / s.Hkv) + hi / s.Hkv;
    const Work sq = work_of(tiles, t);
    const int i0 = sq.first;
    const int off = sq.nk - sq.nq;
    const int end = keys_seen(sq), ntile = (end + CK - 1) / CK, t0 = part * per, t1 = min(ntile, t0 + per);
    if (part > 0 && t0 >= ntile) return;
    const T* Kh = K + (int64_t)sq.k0 * s.k_sr + (int64_t)hk * s.k_sh;
    const T* Vh = V + (int64_t)sq.k0 * s.v_sr + (int64_t)hk * s.v_sh;

    const int w0 = i0 + 32 * wid;
    int lim[2];
    float l2[2], dl[2];
    x8 qf[2][KS], gf[2][KS];
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
        const int i = w0 + 16 * qb + r16;
        const int64_t row = sq.q0 + min(i, sq.nq - 1);
        lim[qb] = i < sq.nq ? max(0, min(sq.nk, i + off + 1)) : 0;
        const T* qr = Q + row * s.q_sr + (int64_t)h * s.q_sh + 8 * g;
        const T* gr = dO + row * s.o_sr + (int64_t)h * s.o_sh + 8 * g;
        const T* orow = O + row * s.o_sr + (int64_t)h * s.o_sh + 8 * g;
        float sum = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            qf[qb][ks] = *(const x8*)(qr + 32 * ks);
            gf[qb][ks] = *(const x8*)(gr + 32 * ks);
            const x8 of = *(const x8*)(orow + 32 * ks);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum += (float)gf[qb][ks][e] * (float)of[e];
        }
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        dl[qb] = sum;
        l2[qb] = lse[(int64_t)h * s.lse_stride + row] * A_LOG2E;
    }
    const int all_see = w0 + 32 <= sq.nq ? max(0, min(sq.nk, w0 + off + 1)) : 0;
    const int wave_end = w0 < sq.nq ? max(0, min(sq.nk, min(w0 + 32, sq.nq) + off)) : 0;
    const float c2 = s.scale * A_LOG2E;

    f32x4 acc[2][NT];
#pragma unroll
    for (int qb = 0; qb < 2; ++qb)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[qb][nt] = (f32x4){0.f, 0.f, 0.f, 0.f};

    using Load = TileBuf<T, HD, CK, 256>;
    Load kl, vl;
    kl.place(s.k_sr, tid);
    vl.place(s.v_sr, tid);
    auto ask_k = [&](int tile) { kl.load(Load::rows(Kh, s.k_sr, tile * CK, tile < t1 ? sq.nk : 0), s.k_sr); };
    auto ask_v = [&](int tile) { vl.load(Load::rows(Vh, s.v_sr, tile * CK, tile < t1 ? sq.nk : 0), s.v_sr); };
    auto k_tile = [&](int tile) { return smem + (tile & 1) * 2 * TB; };
    ask_k(t0);
    ask_v(t0);
    if (ntile <= 2) {                                              // both tiles stay in LDS, each in its own half
        float d[2] = {0.f, 0.f};
#pragma unroll 1
        for (int tile = 0; tile < ntile; ++tile) {
            uint8_t *kt = k_tile(tile), *vt = kt + TB;
            kl.store(kt, tid);
            vl.store(vt, tid);
            __syncthreads();
            ask_k(tile + 1);
            ask_v(tile + 1);
#pragma unroll 1
            for (int k4 = 0; k4 < 4; ++k4) {
                f32x4 sc[2], dp[2];
#pragma unroll
                for (int qb = 0; qb < 2; ++qb) sc[qb] = dp[qb] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const x8 kf = Ti::row8(kt, 16 * k4, ks, lane);
                    const x8 vf = Ti::row8(vt, 16 * k4, ks, lane);
#pragma unroll
                    for (int qb = 0; qb < 2; ++qb) {
                        sc[qb] = mfma16(kf, qf[qb][ks], sc[qb]);
                        dp[qb] = mfma16(vf, gf[qb][ks], dp[qb]);
                    }
                }
#pragma unroll
                for (int qb = 0; qb < 2; ++qb)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[qb][i], c2, -l2[qb])) * dp[qb][i];
                        d[qb] += tile * CK + 16 * k4 + 4 * g + i < lim[qb] ? p : 0.f;
                    }
            }
        }
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) {
            d[qb] += __shfl_xor(d[qb], 16, 64);
            d[qb] += __shfl_xor(d[qb], 32, 64);
            dl[qb] = d[qb];
        }
    }
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
        const int i = w0 + 16 * qb + r16;
        if (g == 0 && i < sq.nq && part == 0) delta[(int64_t)h * s.lse_stride + sq.q0 + i] = dl[qb];
    }
    // one tile; `on`: the next one goes from registers to LDS and the one after it is asked for among the instructions
    auto step = [&](int tile, auto masked, auto on) {
        uint8_t *kt = k_tile(tile), *vt = kt + TB;
        const int key0 = tile * CK;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {                           // 32 keys at a time
            x4 ds[2][2];
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2) {
                f32x4 sc[2], dp[2];
#pragma unroll
                for (int qb = 0; qb < 2; ++qb) sc[qb] = dp[qb] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const x8 kf = Ti::row8(kt, 32 * hf + 16 * k2, ks, lane);
                    const x8 vf = Ti::row8(vt, 32 * hf + 16 * k2, ks, lane);
#pragma unroll
                    for (int qb = 0; qb < 2; ++qb) {
                        sc[qb] = mfma16(kf, qf[qb][ks], sc[qb]);
                        dp[qb] = mfma16(vf, gf[qb][ks], dp[qb]);
                    }
                }
                if constexpr (on.value) {
                    if (hf == 0 && k2 == 0) kl.store(k_tile(tile + 1), tid);
                    if (hf == 0 && k2 == 1) vl.store(k_tile(tile + 1) + TB, tid);
                }
#pragma unroll
                for (int qb = 0; qb < 2; ++qb) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        sc[qb][i] = __builtin_fmaf(sc[qb][i], c2, -l2[qb]);
                        dp[qb][i] -= dl[qb];
                        if constexpr (masked.value) {
                            const bool vis = key0 + 32 * hf + 16 * k2 + 4 * g + i < lim[qb];
                            sc[qb][i] = vis ? sc[qb][i] : -INFINITY;
                            dp[qb][i] = vis ? dp[qb][i] : 0.f;
                        }
                        dp[qb][i] *= __builtin_amdgcn_exp2f(sc[qb][i]);
                    }
                    ds[qb][k2] = pack4<T>(dp[qb]);
                }
            }
            if constexpr (on.value) {
                if (hf == 0) ask_k(tile + 2);
                else ask_v(tile + 2);
            }
            x8 df[2];
#pragma unroll
            for (int qb = 0; qb < 2; ++qb) df[qb] = join8(ds[qb][0], ds[qb][1]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const x8 kf = Ti::tr8(kt, 32 * hf, nt, lane);
#pragma unroll
                for (int qb = 0; qb < 2; ++qb) acc[qb][nt] = mfma16(kf, df[qb], acc[qb][nt]);
            }
            if (hf == 0) __builtin_amdgcn_sched_barrier(0);        // (the halves mixed: 1219 us for 8191 grouped tokens, 1176 so)
        }
    };
    constexpr std::true_type yes{};
    constexpr std::false_type no{};
    if (ntile <= 2) {
#pragma unroll 1
        for (int tile = 0; tile < min(ntile, (wave_end + CK - 1) / CK); ++tile) step(tile, yes, no);
    } else {
        int tile = t0;
        kl.store(k_tile(tile), tid);
        vl.store(k_tile(tile) + TB, tid);
        ask_k(tile + 1);
        ask_v(tile + 1);
        const int mine = min(t1, (wave_end + CK - 1) / CK), clear = min(mine, all_see / CK);   // tiles that the wave sees, sees whole
#pragma unroll 1
        for (; tile < clear; ++tile) {
            __syncthreads();
            step(tile, no, yes);
        }
#pragma unroll 1
        for (; tile < mine; ++tile) {
            __syncthreads();
            step(tile, yes, yes);
        }
#pragma unroll 1
        for (; tile < t1; ++tile) {                                // tiles for other waves
            __syncthreads();
            kl.store(k_tile(tile + 1), tid);
            vl.store(k_tile(tile + 1) + TB, tid);
            ask_k(tile + 2);
            ask_v(tile + 2);
        }
    }
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
        const int i = w0 + 16 * qb + r16;
        if (i >= sq.nq) continue;
        if (ntile > per) {
            float* row = sums + (((int64_t)part * s.lse_stride + sq.q0 + i) * s.H + h) * HD + 4 * g;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) *(f32x4*)(row + 16 * nt) = acc[qb][nt];
            continue;
        }
        T* row = dQ + (int64_t)(sq.q0 + i) * s.dq_sr + h * HD + 4 * g;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            x4 o4;
#pragma unroll
            for (int e = 0; e < 4; ++e) o4[e] = (T)(acc[qb][nt][e] * s.scale);
            *(x4*)(row + 16 * nt) = o4;
        }
    }
}

// the fp32 sums of 16 rows -> dQ
template <typename T, int HD>
__global__ __launch_bounds__(256) void causal_dq_sum_kernel(const float* __restrict__ sums, const int32_t* __restrict__ tiles, star_causal_shape s, int per,
                                                           T* __restrict__ dQ) {
    const int h = blockIdx.x % s.H, t = blockIdx.x / s.H;
    const Work sq = work_of(tiles, t);
    const int np = ((keys_seen(sq) + CK - 1) / CK + per - 1) / per, i0 = sq.first + 16 * blockIdx.y, rows = min(16, sq.nq - i0);
    if (np <= 1) return;
    const int64_t one = s.lse_stride * s.H * HD;
    for (int c = threadIdx.x; c < rows * (HD / 4); c += 256) {
        const int64_t row = sq.q0 + i0 + c / (HD / 4), d = h * HD + 4 * (c % (HD / 4));
        f32x4 sum = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
        for (int p = 0; p < np; ++p) sum += *(const f32x4*)(sums + p * one + row * s.H * HD + d);
        *(typename Vec<T>::x4*)(dQ + row * s.dq_sr + d) = pack4<T>(sum * s.scale);
    }
}

// ------------------------------------------------------------------------------------------------------ gradients of K, V
// One workgroup: 128 keys of one key head, 32 per wave with K, dK^T and dV^T in registers and V in LDS (with V in
// registers too only one wave would fit a SIMD, and nothing would cover its LDS and exponential latencies); it walks the
// queries of its query heads in tiles of 32.  The key is on the MFMA column, so P and dS come out as the operands of
// dV^T += dO^T P and dK^T += Q^T dS.
// A launch of few workgroups is cut, first by query heads: part p of hp takes heads p * grp / hp .. of the group (an XCD
// then reads few heads); if that is not enough, each of these walks by its steps, `per` to a piece.  Where a tile
// has more than one part or piece they leave fp32 sums, which causal_dkv_sum_kernel adds up in order.
template <typename T, int HD>
__global__ __launch_bounds__(256, 2) void causal_dkv_kernel(const T* __restrict__ Q, const T* __restrict__ K,
                                                           const T* __restrict__ V, const T* __restrict__ dO,
                                                           const float* __restrict__ lse, const float* __restrict__ delta,
                                                           const int32_t* __restrict__ tiles, star_causal_shape s,
                                                           int hp, int pieces, int per, float* __restrict__ sums,
                                                           T* __restrict__ dK, T* __restrict__ dV) {
    typedef typename Vec<T>::x8 x8;
    typedef typename Vec<T>::x4 x4;
    using Ti = Tile<T, HD>;
    constexpr int KS = HD / 32, NT = HD / 16;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    constexpr int VB = CT * Ti::ROWB, TB = CQ * Ti::ROWB, SB = 2 * TB + 2 * CQ * 4;   // V | 2 x (Q | dO | lse | delta)

    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    const int hk = blockIdx.x % s.Hkv, part = blockIdx.x / s.Hkv % (hp * pieces), t = blockIdx.x / s.Hkv / (hp * pieces);
    const int piece = part / hp, heads = s.H / s.Hkv / hp;
    const Work sq = work_of(tiles, t);
    const Walk walk = queries_of(sq);
    const int total = walk.n * heads, n0 = piece * per, ntile = min(per, total - n0);
    if (piece > 0 && ntile <= 0) return;
    const int j0 = sq.first, w0 = j0 + 32 * wid;           // first key of the workgroup, of the wave
    const int off = sq.nk - sq.nq;
    uint8_t* vt = smem + 32 * wid * Ti::ROWB;                      // the wave's rows of V

    x8 kf[2][KS];
    const int see = w0 + r16 - off;                                // first query that sees this lane's key of block 0
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
        const int j = w0 + 16 * kb + r16;
        const T* kr = K + (int64_t)(sq.k0 + min(j, sq.nk - 1)) * s.k_sr + (int64_t)hk * s.k_sh + 8 * g;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) kf[kb][ks] = *(const x8*)(kr + 32 * ks);
    }
    {
        TileLoad<T, HD, CT, 256> vl;
        vl.place(s.v_sr, tid);
        vl.load(V + (int64_t)sq.k0 * s.v_sr + (int64_t)hk * s.v_sh, s.v_sr, j0, sq.nk, tid);
        vl.store(smem, tid);
    }
    f32x4 dk[2][NT], dv[2][NT];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) dk[kb][nt] = dv[kb][nt] = (f32x4){0.f, 0.f, 0.f, 0.f};
    const float c2 = s.scale * A_LOG2E;
    const int first = walk.first;
    const int all_see = w0 + 31 - off;                             // from this query on every key of the wave is visible

    TileLoad<T, HD, CQ, 256> ql, gl;
    float lr = 0.f;
    // head and first query of the next tile to load
    int lh = hk * (s.H / s.Hkv) + part % hp * heads, lq = first * CQ;
    if (n0 > 0) {
        const int skip = __builtin_amdgcn_readfirstlane(n0 / walk.n);
        lh += skip;
        lq += (n0 - skip * walk.n) * CQ;
    }
    auto load = [&]() {
        ql.load(Q + (int64_t)sq.q0 * s.q_sr + (int64_t)lh * s.q_sh, s.q_sr, lq, sq.nq, tid);
        gl.load(dO + (int64_t)sq.q0 * s.o_sr + (int64_t)lh * s.o_sh, s.o_sr, lq, sq.nq, tid);
        if (wid < 2 && lane < CQ) {
            const float* p = (wid == 0 ? lse : delta) + (int64_t)lh * s.lse_stride + sq.q0 + lq;
            lr = p[min(lane, sq.nq - 1 - lq)];
        }
        lq += CQ;
        if (lq >= sq.nq) { lq = first * CQ; ++lh; }
    };
    ql.place(s.q_sr, tid);
    gl.place(s.o_sr, tid);
    int q0 = lq;
    if (ntile > 0) load();
#pragma unroll 1
    for (int n = 0; n < ntile; ++n) {
        uint8_t* qt = smem + VB + (n & 1) * SB;
        uint8_t* gt = qt + TB;
        float* lt = (float*)(gt + TB);
        ql.store(qt, tid);
        gl.store(gt, tid);
        if (wid < 2 && lane < CQ) lt[wid * CQ + lane] = wid == 0 ? lr * A_LOG2E : lr;
        __syncthreads();
        if (n + 1 < ntile) load();
        const int qa0 = q0;
        q0 += CQ;
        if (q0 >= sq.nq) q0 = first * CQ;
        if (qa0 + CQ <= w0 - off) continue;                        // (wave-uniform) no query of the tile sees a key of the wave
        const bool masked = qa0 < all_see || qa0 + CQ > sq.nq;
        // both 16-query halves at once: the fragments of V are read once for them
        x4 pp[2][2], ds[2][2];
        f32x4 sc[2][2], dp[2][2];
#pragma unroll
        for (int q2 = 0; q2 < 2; ++q2)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) sc[q2][kb] = dp[q2][kb] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            // (head dim 96: the reads of all steps at once would not fit the registers)
            if constexpr (HD == 96) __builtin_amdgcn_sched_barrier(0);
            x8 vf[2];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) vf[kb] = Ti::row8(vt, 16 * kb, ks, lane);
#pragma unroll
            for (int q2 = 0; q2 < 2; ++q2) {
                const x8 qa = Ti::row8(qt, 16 * q2, ks, lane);
                const x8 ga = Ti::row8(gt, 16 * q2, ks, lane);
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    sc[q2][kb] = mfma16(qa, kf[kb][ks], sc[q2][kb]);
                    dp[q2][kb] = mfma16(ga, vf[kb], dp[q2][kb]);
                }
            }
        }
#pragma unroll
        for (int q2 = 0; q2 < 2; ++q2) {
            const f32x4 ls = *(const f32x4*)(lt + 16 * q2 + 4 * g);
            const f32x4 de = *(const f32x4*)(lt + CQ + 16 * q2 + 4 * g);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sc[q2][kb][i] = __builtin_fmaf(sc[q2][kb][i], c2, -ls[i]);
                    dp[q2][kb][i] -= de[i];
                }
        }
        if (masked) {
#pragma unroll
            for (int q2 = 0; q2 < 2; ++q2)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int qi = qa0 + 16 * q2 + 4 * g + i;
                        const bool vis = qi >= see + 16 * kb && qi < sq.nq;
                        sc[q2][kb][i] = vis ? sc[q2][kb][i] : -INFINITY;
                        dp[q2][kb][i] = vis ? dp[q2][kb][i] : 0.f;
                    }
        }
#pragma unroll
        for (int q2 = 0; q2 < 2; ++q2)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sc[q2][kb][i] = __builtin_amdgcn_exp2f(sc[q2][kb][i]);
                    dp[q2][kb][i] *= sc[q2][kb][i];
                }
                pp[kb][q2] = pack4<T>(sc[q2][kb]);
                ds[kb][q2] = pack4<T>(dp[q2][kb]);
            }
        __builtin_amdgcn_sched_barrier(0);
        x8 pf[2], df[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            pf[kb] = join8(pp[kb][0], pp[kb][1]);
            df[kb] = join8(ds[kb][0], ds[kb][1]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const x8 ga = Ti::tr8(gt, 0, nt, lane);
            const x8 qa = Ti::tr8(qt, 0, nt, lane);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                dv[kb][nt] = mfma16(ga, pf[kb], dv[kb][nt]);
                dk[kb][nt] = mfma16(qa, df[kb], dk[kb][nt]);
            }
        }
    }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
        const int j = w0 + 16 * kb + r16;
        if (j >= sq.nk) continue;
        const int64_t at = (int64_t)(sq.k0 + j) * s.dkv_sr + hk * HD + 4 * g;
        if (hp > 1 || total > per) {
            float* sk = sums + ((int64_t)part * 2 * s.k_rows + sq.k0 + j) * s.Hkv * HD + hk * HD + 4 * g;
            float* sv = sk + s.k_rows * s.Hkv * HD;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                *(f32x4*)(sk + 16 * nt) = dk[kb][nt];
                *(f32x4*)(sv + 16 * nt) = dv[kb][nt];
            }
            continue;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            x4 a, b;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                a[e] = (T)(dk[kb][nt][e] * s.scale);
                b[e] = (T)dv[kb][nt][e];
            }
            *(x4*)(dK + at + 16 * nt) = a;
            *(x4*)(dV + at + 16 * nt) = b;
        }
    }
}

// the fp32 sums of 16 keys -> dK, dV
template <typename T, int HD>
__global__ __launch_bounds__(256) void causal_dkv_sum_kernel(const float* __restrict__ sums, const int32_t* __restrict__ tiles, star_causal_shape s, int hp, int per,
                                                            T* __restrict__ dK, T* __restrict__ dV) {
    const int hk = blockIdx.x % s.Hkv, t = blockIdx.x / s.Hkv;
    const Work sq = work_of(tiles, t);
    const int np = hp * max(1, (queries_of(sq).n * (s.H / s.Hkv / hp) + per - 1) / per), j0 = sq.first + 16 * blockIdx.y, rows = min(16, sq.nk - j0);
    if (np <= 1) return;
    const int64_t one = s.k_rows * s.Hkv * HD;
    for (int c = threadIdx.x; c < 2 * 16 * (HD / 4); c += 256) {
        const int which = c / (16 * (HD / 4)), cc = c % (16 * (HD / 4));
        if (cc / (HD / 4) >= rows) continue;
        const int64_t row = sq.k0 + j0 + cc / (HD / 4), d = hk * HD + 4 * (cc % (HD / 4)), at = row * s.Hkv * HD + d;
        f32x4 sum = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int p = 0; p < np; ++p) sum += *(const f32x4*)(sums + (2 * p + which) * one + at);
        *(typename Vec<T>::x4*)((which ? dV : dK) + row * s.dkv_sr + d) = pack4<T>(which ? sum : sum * s.scale);
    }
}

// Pieces of the walks of a launch of wgs workgroups, `longest` steps at most and `mean` on average (a causal walk is
// anything up to the longest): steps of `per`, so that wgs * (mean / per + 1/2) pieces, which is what such walks come to, fill
// the 512 places (two a CU) once.  From 320 workgroups on, and from 256 with walks of middle length, a walk in one piece
// is as good or better: two rounds of pieces and the sums' way through memory cost what the idle CUs did.  Forward
// and backward, 8 heads of 128: one sequence of 1500 tokens 143 -> 98 us, 3000 tokens 266 -> 178, 5000 tokens (320 workgroups)
// 467 -> 361; 6 of 800 to 1300 (400) 147 -> 186.
struct Pieces { int hp, pieces, per; };                            // parts by heads, pieces of the longest walk, steps of a piece
static Pieces pieces(int hp, int64_t wgs, int64_t longest, int64_t mean, int least) {
    const int64_t room = 512 - wgs / 2;
    if (wgs < 1 || wgs > 320 || 2 * longest <= (wgs > 256 ? 12 : 3) * least) return Pieces{hp, 1, 0x3fffffff};
    const int64_t per = max((int64_t)least, (wgs * mean + room - 1) / room);
    if (per >= longest) return Pieces{hp, 1, 0x3fffffff};
    return Pieces{hp, (int)((longest + per - 1) / per), (int)per};
}
static Pieces dq_pieces(const star_causal_shape* s) {
    const int64_t n = cdiv(s->max_k, CK);
    return pieces(1, (int64_t)s->n_q_tiles * s->H, n, max((int64_t)1, n - cdiv(min(s->max_q, s->max_k), CT)), 4);
}
// By query heads: into 1 when the longest walk is short (under 16 tiles of 32 queries over all heads), or the key tiles
// alone give every CU a workgroup -- two from walks of 16 tiles a head on, four from 32, which go from 1 tile to 32 and more
// and leave no balance to a single round; otherwise into the fewest that do.  Forward and backward of 8191 tokens, 16
// heads on 4 of 128: 1144 us for 1024 workgroups, 1346 for 512 by heads, 1223 by steps alone; 4 sequences of 500 to 900, 32 on
// 4 of 128: 155 for 512, 183 for 256; 53 of 200 to 210, 8 on 2 of 128: 126 and 113; 2 of up to 622, 16 on 2 of 96: 68, 217 in
// one part.
static Pieces dkv_pieces(const star_causal_shape* s) {
    const int grp = s->H / s->Hkv, walk = cdiv(s->max_q, CQ);
    const int64_t wgs = (int64_t)s->n_k_tiles * s->Hkv, want = walk >= 32 ? 1024 : walk >= 16 ? 512 : 256;
    int hp = 1;
    if ((int64_t)grp * walk >= 16)
        while (hp < grp && wgs * hp < want) {
            do ++hp; while (grp % hp);
        }
    const int64_t heads = grp / hp, mean = max(1, walk - cdiv(min(s->max_q, s->max_k), 2 * CQ));
    return pieces(hp, wgs * hp, heads * walk, heads * mean, 8);
}

// ------------------------------------------------------------------------------------------------------ host side
static int check_causal(const star_causal_shape* s, const char* who) {
    STAR_REQUIRE(s, "%s: null shape", who);
    STAR_REQUIRE(s->hd == 64 || s->hd == 96 || s->hd == 128, "%s: head dim %d not in {64, 96, 128}", who, s->hd);
    STAR_REQUIRE(s->dtype == STAR_DT_BF16 || s->dtype == STAR_DT_F16, "%s: dtype %d is neither bf16 nor fp16", who, s->dtype);
    STAR_REQUIRE(s->Hkv >= 1 && s->H >= s->Hkv && s->H % s->Hkv == 0, "%s: %d query heads do not divide into %d key heads", who, s->H, s->Hkv);
    STAR_REQUIRE(s->max_q >= 0 && s->max_k >= 0 && s->n_q_tiles >= 0 && s->n_k_tiles >= 0 && s->lse_stride >= 0 && s->k_rows >= 0,
                 "%s: negative size", who);
    // (a launch has less than 2^32 threads in x)
    STAR_REQUIRE((int64_t)s->n_q_tiles * s->H < (1ll << 24) && (int64_t)s->n_k_tiles * s->H < (1ll << 24), "%s: %d and %d tiles x %d heads",
                 who, s->n_q_tiles, s->n_k_tiles, s->H);
    const int64_t st[8] = {s->q_sr, s->q_sh, s->k_sr, s->k_sh, s->v_sr, s->v_sh, s->o_sr, s->o_sh};
    for (int i = 0; i < 8; ++i) STAR_REQUIRE(st[i] % 8 == 0, "%s: strides must be multiples of 8 elements", who);
    for (int i = 0; i < 8; i += 2)
        STAR_REQUIRE(st[i] >= 0 && st[i] < (1ll << 23), "%s: row stride %lld not in [0, 2^23)", who, (long long)st[i]);
    STAR_REQUIRE(s->scale > 0.f && s->scale < INFINITY, "%s: scale must be positive and finite", who);
    return STAR_OK;
}
static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Rows of a workgroup of the forward, and the parts that its keys are cut into.  A tile of keys takes a workgroup about
// 1 us whoever else runs (each CU fetches it for itself), a second launch that joins the parts 3, so few workgroups over
// keys that are not quite short are cut until there is one for every CU, or two where the parts would still be long.
// The few-query kernel takes four tiles at once; its break-even is by bytes.  Us in one part and in parts, hd 128, 8 heads,
// 16 queries: 8.0 and 7.8 over 375 keys, 14.0 and 7.9 over 1000, 80 and 12 over 8000; 64 queries: 11.1 and 9.0 over
// 320, 26 and 9.2 over 1000, 167 and 17 over 8000.
static int fwd_rows(const star_causal_shape* s) { return s->max_q <= 16 ? 16 : s->max_q <= 32 ? 32 : CT; }
static int fwd_parts(const star_causal_shape* s) {
    const int64_t wgs = (int64_t)s->n_q_tiles * s->H;
    const int n = cdiv(s->max_k, CK);
    const bool few_keys = fwd_rows(s) == CT ? n < 6 : n * s->hd < 7 * 128;
    if (wgs < 1 || wgs >= 256 || few_keys) return 1;
    int per = cdiv(n, 256 / wgs);
    // (two a CU: 200 queries of 16 sequences with 2 heads over 8000 keys 46 -> 35 us; 16 queries, 144 workgroups over 8000
    // keys 77 -> 59, over 2000 18 -> 20)
    if (per >= (2 * wgs > 256 ? 40 : 12)) per = cdiv(n, 512 / wgs);
    return cdiv(n, per);
}
static int64_t causal_fwd_bytes(const star_causal_shape* s) {
    const int parts = fwd_parts(s);
    return parts == 1 ? 0 : (int64_t)s->n_q_tiles * s->H * parts * fwd_rows(s) * (s->hd + 2) * 4;
}

template <typename T, int HD>
static int launch_causal_fwd(const void* q, const void* k, const void* v, const int32_t* tiles,
                             const star_causal_shape* s, void* o, float* lse, float* sums, hipStream_t st) {
    constexpr int tile = 4 * CK * Tile<T, HD>::ROWB, join2 = 4 * 32 * (HD + 4) * 4;
    constexpr int smem_few = tile > join2 ? tile : join2;
    const int rows = fwd_rows(s), parts = fwd_parts(s);
    const void* fn = rows == 16 ? (const void*)causal_few_kernel<T, HD, 1> : rows == 32 ? (const void*)causal_few_kernel<T, HD, 2>
                                                                                       : (const void*)causal_fwd_kernel<T, HD>;
    const int smem = rows == CT ? tile : smem_few;
    static DevOnce once[3];
    if (!reserve_lds_once(once[rows == 16 ? 0 : rows == 32 ? 1 : 2], fn, smem)) {
        set_error("star_causal_fwd: cannot reserve %d bytes of LDS", smem);
        return STAR_ERR_LAUNCH;
    }
    const dim3 grid((unsigned)((int64_t)s->n_q_tiles * s->H * parts));
#define CAUSAL_FWD_ARGS grid, dim3(256), smem, st, (const T*)q, (const T*)k, (const T*)v, tiles, *s, parts, sums, (T*)o, lse
    if (rows == 16) hipLaunchKernelGGL((causal_few_kernel<T, HD, 1>), CAUSAL_FWD_ARGS);
    else if (rows == 32) hipLaunchKernelGGL((causal_few_kernel<T, HD, 2>), CAUSAL_FWD_ARGS);
    else hipLaunchKernelGGL((causal_fwd_kernel<T, HD>), CAUSAL_FWD_ARGS);
#undef CAUSAL_FWD_ARGS
#define CAUSAL_JOIN_ARGS dim3(256), 0, st, tiles, *s, parts, rows, (const float*)sums, (T*)o, lse
    const unsigned tiles_h = (unsigned)((int64_t)s->n_q_tiles * s->H);
    if (parts > 16) hipLaunchKernelGGL((causal_join_kernel<T, HD, 4>), dim3(tiles_h, rows), CAUSAL_JOIN_ARGS);
    else if (parts > 1) hipLaunchKernelGGL((causal_join_kernel<T, HD, 1>), dim3(tiles_h, rows / 4), CAUSAL_JOIN_ARGS);
#undef CAUSAL_JOIN_ARGS
    return STAR_OK;
}

static int64_t causal_bwd_bytes(const star_causal_shape* s) {
    const Pieces k = dkv_pieces(s);
    const int64_t pq = dq_pieces(s).pieces, pk = (int64_t)k.hp * k.pieces;
    return max(pq == 1 ? 0 : pq * s->lse_stride * s->H, pk == 1 ? 0 : pk * 2 * s->k_rows * s->Hkv) * s->hd * 4;
}

template <typename T, int HD>
static int launch_causal_bwd(const void* q, const void* k, const void* v, const void* o, const void* do_, const float* lse,
                             const int32_t* q_tiles, const int32_t* k_tiles,
                             const star_causal_shape* s, void* dq, void* dk, void* dv, float* delta,
                             float* sums, hipStream_t st) {
    constexpr int smem_q = 4 * CK * Tile<T, HD>::ROWB;
    constexpr int smem_k = CT * Tile<T, HD>::ROWB + 2 * (2 * CQ * Tile<T, HD>::ROWB + 2 * CQ * 4);
    static DevOnce once_q, once_k;
    if (!reserve_lds_once(once_q, (const void*)causal_dq_kernel<T, HD>, smem_q) ||
        !reserve_lds_once(once_k, (const void*)causal_dkv_kernel<T, HD>, smem_k)) {
        set_error("star_causal_bwd: cannot reserve %d bytes of LDS", smem_k);
        return STAR_ERR_LAUNCH;
    }
    if (s->n_q_tiles > 0) {
        const Pieces p = dq_pieces(s);
        const unsigned wgs = (unsigned)s->n_q_tiles * s->H;
        hipLaunchKernelGGL((causal_dq_kernel<T, HD>), dim3(wgs * p.pieces), dim3(256), smem_q, st, (const T*)q,
                           (const T*)k, (const T*)v, (const T*)o, (const T*)do_, lse, q_tiles, *s, p.pieces, p.per, sums, (T*)dq, delta);
        if (p.pieces > 1)
            hipLaunchKernelGGL((causal_dq_sum_kernel<T, HD>), dim3(wgs, CT / 16), dim3(256), 0, st, (const float*)sums, q_tiles, *s, p.per, (T*)dq);
    }
    if (s->n_k_tiles > 0) {
        const Pieces p = dkv_pieces(s);
        const unsigned wgs = (unsigned)s->n_k_tiles * s->Hkv;
        hipLaunchKernelGGL((causal_dkv_kernel<T, HD>), dim3(wgs * p.hp * p.pieces), dim3(256), smem_k, st,
                           (const T*)q, (const T*)k, (const T*)v, (const T*)do_, lse, (const float*)delta, k_tiles, *s,
                           p.hp, p.pieces, p.per, sums, (T*)dk, (T*)dv);
        if (p.hp * p.pieces > 1)
            hipLaunchKernelGGL((causal_dkv_sum_kernel<T, HD>), dim3(wgs, CT / 16), dim3(256), 0, st,
                               (const float*)sums, k_tiles, *s, p.hp, p.per, (T*)dk, (T*)dv);
    }
    return STAR_OK;
}

#define CAUSAL_BY_TYPE(CALL)                                         \
    do {                                                             \
        if (s->dtype == STAR_DT_BF16) {                              \
            if (s->hd == 64) { using T = __bf16; constexpr int HD = 64; rc = CALL; }       \
            else if (s->hd == 96) { using T = __bf16; constexpr int HD = 96; rc = CALL; }  \
            else { using T = __bf16; constexpr int HD = 128; rc = CALL; }                  \
        } else {                                                     \
            if (s->hd == 64) { using T = _Float16; constexpr int HD = 64; rc = CALL; }      \
            else if (s->hd == 96) { using T = _Float16; constexpr int HD = 96; rc = CALL; } \
            else { using T = _Float16; constexpr int HD = 128; rc = CALL; }                 \
        }                                                            \
    } while (0)

}  // namespace star

extern "C" size_t star_causal_fwd_workspace(const star_causal_shape* s) {
    using namespace star;
    return check_causal(s, "star_causal_fwd_workspace") ? 0 : (size_t)causal_fwd_bytes(s);
}

extern "C" int star_causal_fwd(const void* q, const void* k, const void* v, const int32_t* tiles,
                               const star_causal_shape* s, void* o, float* lse, void* workspace, size_t workspace_bytes,
                               void* stream) {
    using namespace star;
    int rc = check_causal(s, "star_causal_fwd");
    if (rc) return rc;
    if (s->n_q_tiles == 0) return STAR_OK;
    STAR_REQUIRE(q && k && v && tiles && o, "star_causal_fwd: null pointer");
    STAR_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(o), "star_causal_fwd: tensors must be 16-byte aligned");
    const int64_t need = causal_fwd_bytes(s);
    if (need > 0 && (!workspace || (int64_t)workspace_bytes < need || !aligned16(workspace))) {
        set_error("star_causal_fwd: workspace of %zu bytes, %lld needed", workspace_bytes, (long long)need);
        return STAR_ERR_WORKSPACE;
    }
    CAUSAL_BY_TYPE((launch_causal_fwd<T, HD>(q, k, v, tiles, s, o, lse, (float*)workspace, (hipStream_t)stream)));
    if (rc) return rc;
    STAR_LAUNCH_CHECK("star_causal_fwd");
    return STAR_OK;
}

extern "C" size_t star_causal_bwd_workspace(const star_causal_shape* s) {
    using namespace star;
    return check_causal(s, "star_causal_bwd_workspace") ? 0 : (size_t)causal_bwd_bytes(s);
}

extern "C" int star_causal_bwd(const void* q, const void* k, const void* v, const void* o, const void* do_,
                               const float* lse, const int32_t* q_tiles, const int32_t* k_tiles,
                               const star_causal_shape* s, void* dq, void* dk, void* dv, float* delta, void* workspace,
                               size_t workspace_bytes, void* stream) {
    using namespace star;
    int rc = check_causal(s, "star_causal_bwd");
    if (rc) return rc;
    if (s->n_q_tiles == 0 && s->n_k_tiles == 0) return STAR_OK;
    STAR_REQUIRE(q && k && v && o && do_ && lse && (q_tiles || !s->n_q_tiles) && (k_tiles || !s->n_k_tiles) && dq && dk && dv && delta,
                 "star_causal_bwd: null pointer");
    STAR_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(o) && aligned16(do_) && aligned16(dq) && aligned16(dk) && aligned16(dv),
                 "star_causal_bwd: tensors must be 16-byte aligned");
    STAR_REQUIRE(s->dq_sr % 8 == 0 && s->dkv_sr % 8 == 0 && s->dq_sr >= (int64_t)s->H * s->hd && s->dkv_sr >= (int64_t)s->Hkv * s->hd,
                 "star_causal_bwd: gradient row strides %lld, %lld", (long long)s->dq_sr, (long long)s->dkv_sr);
    const int64_t need = causal_bwd_bytes(s);
    if (need > 0 && (!workspace || (int64_t)workspace_bytes < need || !aligned16(workspace))) {
        set_error("star_causal_bwd: workspace of %zu bytes, %lld needed", workspace_bytes, (long long)need);
        return STAR_ERR_WORKSPACE;
    }
    CAUSAL_BY_TYPE((launch_causal_bwd<T, HD>(q, k, v, o, do_, lse, q_tiles, k_tiles, s, dq, dk, dv, delta, (float*)workspace,
                                             (hipStream_t)stream)));
    if (rc) return rc;
    STAR_LAUNCH_CHECK("star_causal_bwd");
    return STAR_OK;
}
