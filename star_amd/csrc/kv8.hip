// 8-bit key/value cache: append and attention (star_kv8_* in star_nugget.h, which states the format).
//
// A power of two as the scale of a block makes its division exact and lets it commute with every later rounding: the
// K scale multiplies the logits of its 64 tokens, the V scale rides in the conversion of the codes to 16 bits (both
// exact), so the attention computes with the very values that the cache stands for, on 16-bit MFMAs with fp32 sums.
// The layouts are the MFMA's: K by rows, V transposed inside its block, so every operand goes from HBM to a register
// with 16-byte loads and no LDS.
#include "causal.h"

namespace star {

constexpr int KB = STAR_KV8_BLOCK;

// ------------------------------------------------------------------------------------------------------ append
// e4m3 scale of a block with finite maximum m >= 0
__device__ __forceinline__ float block_scale(float m) {
    if (!(m > 0.f)) return 1.f;
    const int e = (int)((__float_as_uint(m) >> 23) & 0xff) - 127;              // floor(log2 m), -127 for a denormal
    const bool up = (__float_as_uint(m) & 0x7fffff) > 0x600000;                // mantissa over 1.75 = 448 / 256
    const int s = max(e - 8 + (up ? 1 : 0), -126);
    return __uint_as_float((uint32_t)(s + 127) << 23);
}
__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a < INFINITY ? a : 0.f;                                             // (false for NaN too)
}
__device__ __forceinline__ float code_in(float x, float inv) { return fabsf(x) < INFINITY ? x * inv : __uint_as_float(0x7fc00000u); }
// 8 values -> 8 codes, round to nearest even (|x * inv| <= 448)
template <typename X8>
__device__ __forceinline__ u32x2 codes8(const X8& x, float inv) {
    u32x2 r;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(code_in((float)x[4 * j], inv), code_in((float)x[4 * j + 1], inv), 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(code_in((float)x[4 * j + 2], inv), code_in((float)x[4 * j + 3], inv), w, true);
        r[j] = (uint32_t)w;
    }
    return r;
}

__device__ __forceinline__ int count(int32_t* p) { return __hip_atomic_fetch_add(p, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

struct AppendArgs {
    star_kv8_cache c;
    const void *k, *v;
    int64_t k_sb, k_sh, k_sr, v_sb, v_sh, v_sr;
    const int32_t *starts, *counts, *at;
    int idx_stride, max_rows;
};

// Workgroup (x, 2 * head + {K, V}, b): the blocks x, x + gridDim.x, ... that this call completes; x = 0, which holds the
// first of them (the only one that reads the open block), afterwards writes the rows of the new open block.
// A block goes through registers once: a thread has N chunks of 8 values of one token, the largest magnitude is found
// over the workgroup, the codes of K leave as they are and those of V are turned by 4 x 4 bytes through an LDS tile
// whose pitch (HD + 4) spreads both its rows and its columns over all banks.
template <typename T, int HD>
__global__ __launch_bounds__(256) void kv8_append_kernel(AppendArgs a) {
    typedef typename Vec<T>::x8 x8;
    constexpr int CH = HD / 8, N = KB * CH / 256;                   // 16-byte chunks of a row, chunks per thread
    constexpr int VP = HD + 4;
    __shared__ __attribute__((aligned(16))) uint8_t vt[KB * VP];
    __shared__ float wmax[4];
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    const int b = blockIdx.z, h = blockIdx.y >> 1;
    const bool is_v = blockIdx.y & 1;
    const star_kv8_cache& c = a.c;

    const int at = min(max((a.at ? a.at : c.lens)[b], 0), c.T);
    const int want = a.counts ? min(max(a.counts[(int64_t)b * a.idx_stride], 0), a.max_rows) : a.max_rows;
    const int n = min(want, c.T - at), end = at + n;
    const int first = at / KB, last = end / KB;                     // the open block before and after the call
    const int row0 = a.starts ? a.starts[(int64_t)b * a.idx_stride] : 0;
    const int64_t sr = is_v ? a.v_sr : a.k_sr;
    // row of token `pos` is src + (pos - at) * sr
    const T* src = (const T*)(is_v ? a.v : a.k) + (int64_t)b * (is_v ? a.v_sb : a.k_sb) + (int64_t)h * (is_v ? a.v_sh : a.k_sh) +
                   (int64_t)row0 * sr;
    const int64_t bh = (int64_t)b * c.Hkv + h;
    T* tail = (T*)(is_v ? c.v_tail : c.k_tail) + bh * KB * HD;
    uint8_t* codes = (is_v ? c.v_codes : c.k_codes) + bh * c.T * HD;
    float* scales = (is_v ? c.v_scales : c.k_scales) + bh * (c.T / KB);

    // chunk i of this thread: a row's chunks across the lanes, or (turned) the rows of a chunk
    auto row_of = [&](int i, bool turned) { return turned ? (tid + 256 * i) % KB : (tid + 256 * i) / CH; };
    auto ch_of = [&](int i, bool turned) { return turned ? (tid + 256 * i) / KB : (tid + 256 * i) % CH; };
    // (32-bit byte offsets from a scalar address: 63 rows of sr < 2^23 values)
    auto load = [&](x8 (&x)[N], int blk) {
        const char* from = (const char*)(src + (int64_t)(blk * KB - at) * sr);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = *(const x8*)(from + ((uint32_t)row_of(i, false) * (uint32_t)sr + 8 * ch_of(i, false)) * 2);
    };
    // the block that was open: its first `held` tokens lie in the open block's rows, V transposed
    auto load_opened = [&](x8 (&x)[N], int blk) {
        const int held = at - blk * KB;
        const char* from = (const char*)src - (int64_t)held * sr * 2;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int row = row_of(i, is_v), ch = ch_of(i, is_v);
            if (row >= held) x[i] = *(const x8*)(from + ((uint32_t)row * (uint32_t)sr + 8 * ch) * 2);
            else if (!is_v) x[i] = *(const x8*)((const char*)tail + (uint32_t)(row * HD + 8 * ch) * 2);
            else {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[i][e] = *(const T*)((const char*)tail + (uint32_t)((8 * ch + e) * KB + row) * 2);
            }
        }
    };
    auto write = [&](const x8 (&x)[N], int blk, bool turned) {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) m = fmaxf(m, finite_abs((float)x[i][e]));
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
        __syncthreads();                                            // wmax and vt are free
        if (lane == 0) wmax[wid] = m;
        __syncthreads();                                            // (also: every read of the open block's rows is done)
        m = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
        const float sc = block_scale(m), inv = 1.0f / sc;           // (exact: powers of two between 2^-126 and 2^120)
        uint8_t* out = codes + (int64_t)blk * KB * HD;
        if (tid == 0) scales[blk] = sc;
        if (!is_v) {
#pragma unroll
            for (int i = 0; i < N; ++i) *(u32x2*)(out + row_of(i, false) * HD + 8 * ch_of(i, false)) = codes8(x[i], inv);
            return;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const u32x2 w = codes8(x[i], inv);
            uint8_t* to = vt + row_of(i, turned) * VP + 8 * ch_of(i, turned);
            *(uint32_t*)to = w[0];
            *(uint32_t*)(to + 4) = w[1];
        }
        __syncthreads();
#pragma unroll 1
        for (int q = tid; q < 2 * HD; q += 256) {                   // 8 tokens x 4 dimensions each
            const int t8 = q & 7, d4 = q >> 3;
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = *(const uint32_t*)(vt + (8 * t8 + i) * VP + 4 * d4);
            uint8_t* to = out + 4 * d4 * KB + 8 * t8;
            u32x2 o0, o1, o2, o3;
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const uint32_t lo01 = __builtin_amdgcn_perm(w[4 * p + 1], w[4 * p], 0x05010400), lo23 = __builtin_amdgcn_perm(w[4 * p + 3], w[4 * p + 2], 0x05010400);
                const uint32_t hi01 = __builtin_amdgcn_perm(w[4 * p + 1], w[4 * p], 0x07030602), hi23 = __builtin_amdgcn_perm(w[4 * p + 3], w[4 * p + 2], 0x07030602);
                o0[p] = __builtin_amdgcn_perm(lo23, lo01, 0x05040100);
                o1[p] = __builtin_amdgcn_perm(lo23, lo01, 0x07060302);
                o2[p] = __builtin_amdgcn_perm(hi23, hi01, 0x05040100);
                o3[p] = __builtin_amdgcn_perm(hi23, hi01, 0x07060302);
            }
            *(u32x2*)to = o0;
            *(u32x2*)(to + KB) = o1;
            *(u32x2*)(to + 2 * KB) = o2;
            *(u32x2*)(to + 3 * KB) = o3;
        }
    };
    int blk = first + blockIdx.x;
    if (blk < last && blk * KB < at) {
        x8 x[N];
        load_opened(x, blk);
        write(x, blk, is_v);
        blk += gridDim.x;
    }
    if (blk < last) {
        x8 x[N], next[N];
        load(x, blk);
        for (; blk < last; blk += gridDim.x) {
            if (blk + (int)gridDim.x < last) load(next, blk + gridDim.x);
            write(x, blk, false);
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = next[i];
        }
    }
    if (blockIdx.x == 0) {
        const int from = max(at, last * KB), cnt = end - from, r0 = from - last * KB;   // new rows of the open block
        const bool turned = is_v && cnt > 8;
        for (int q = tid; q < (turned ? KB : cnt) * CH; q += 256) {
            const int row = turned ? q % KB : q / CH, ch = turned ? q / KB : q % CH;
            if (row >= cnt) continue;
            const x8 y = *(const x8*)(src + (int64_t)(from + row - at) * sr + 8 * ch);
            if (!is_v) *(x8*)(tail + (r0 + row) * HD + 8 * ch) = y;
            else {
#pragma unroll
                for (int e = 0; e < 8; ++e) tail[(8 * ch + e) * KB + r0 + row] = y[e];
            }
        }
    }
    // lens is read by every workgroup of the sequence and changed by the last of them to get here: a workgroup's count
    // goes out after its own read has come back (the value has steered everything above), so no fence is needed.  Counted
    // in two steps, first among the workgroups of one head's K or V, each counter in a cache line of its own: one counter
    // for all of 3432 workgroups took longer than their work.
    __syncthreads();
    if (tid == 0) {
        int32_t* ticket = c.tickets + (int64_t)b * (1 + 2 * c.Hkv) * STAR_KV8_TICKET_STRIDE;
        int32_t* mine = ticket + (1 + blockIdx.y) * STAR_KV8_TICKET_STRIDE;
        if (gridDim.x == 1 || count(mine) == (int)gridDim.x - 1) {
            if (gridDim.x > 1) *mine = 0;
            if (count(ticket) == (int)gridDim.y - 1) {
                c.lens[b] = end;
                // (with `at` the sequence is at + want tokens long, whatever was missing before)
                if (a.at) c.dropped[b] = (int)min((int64_t)max(a.at[b], 0) + want - end, (int64_t)0x7fffffff);
                else if (want > n) c.dropped[b] += want - n;
                *ticket = 0;
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------------ attention
struct AttnArgs {
    star_kv8_cache c;
    star_kv8_query s;
    const void* q;
    void* o;
    const float* bias;
    const int32_t* q_len;
    int slots;                 // (sequence, part) pairs that the grid has room for, >= B
    int min_part;              // blocks of a part at least
    int even;                  // 1: sequences of much the same length stay whole
    int nrg;                   // groups of 16 * RT rows
    float* part;               // [slots][Hkv][rows][HD] partial sums, [slots][Hkv][rows][2] maximum and sum behind them
};


__device__ __forceinline__ int held_by(const AttnArgs& a, int b) { return min(max(a.c.lens[b], 0), a.c.T); }
__device__ __forceinline__ int queries_of(const AttnArgs& a, int b) { return a.q_len ? min(max(a.q_len[b], 0), a.s.L) : a.s.L; }
// blocks of sequence b that any of its queries sees
__device__ __forceinline__ int blocks_of(const AttnArgs& a, int b) {
    const int n = held_by(a, b), nq = queries_of(a, b);
    int see = nq > 0 ? n : 0;
    if (a.s.ilk_diag >= 0) see = (int)min((int64_t)see, (int64_t)nq + a.s.ilk_diag);
    return (see + KB - 1) / KB;
}

// The work is cut on the device, where the lengths are: parts of `per` blocks, as few as fill the slots, counted off
// sequence by sequence.  sum_b max(1, ceil(nb_b / per)) <= B + sum_b nb_b / per <= slots for per >= sum nb / (slots - B).
struct Parts { int per; };
__device__ __forceinline__ Parts cut(const AttnArgs& a, int lane) {
    if (a.slots == a.c.B) return Parts{0x7fffffff};
    int64_t total = 0;
    int top = 0;
    for (int b0 = 0; b0 < a.c.B; b0 += 64) {
        const int b = b0 + lane, nb = b < a.c.B ? blocks_of(a, b) : 0;
        total += nb;
        top = max(top, nb);
    }
    total = wave_sum(total);
    if (a.even) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) top = max(top, __shfl_xor(top, o, 64));
        if (2 * (int64_t)top * a.c.B <= 3 * total) return Parts{0x7fffffff};
    }
    const int64_t room = a.slots - a.c.B;
    return Parts{(int)max((int64_t)a.min_part, (total + room - 1) / room)};
}
__device__ __forceinline__ int parts_of(int nb, int per) { return nb <= per ? 1 : (nb - 1) / per + 1; }

template <typename T>
__device__ __forceinline__ typename Vec<T>::x8 widen(uint32_t lo, uint32_t hi, float scale);
template <>
__device__ __forceinline__ bf16x8 widen<__bf16>(uint32_t lo, uint32_t hi, float scale) {
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    const auto c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    return (bf16x8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
template <>
__device__ __forceinline__ f16x8 widen<_Float16>(uint32_t lo, uint32_t hi, float scale) {
    typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
    const f16x2 a = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, false));
    const f16x2 b = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, true));
    const f16x2 c = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, false));
    const f16x2 d = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, true));
    return (f16x8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// V in fp16 is used at half its value (and the sum doubled): the largest code of a block may stand for 65536
template <typename T> struct VHalf { static constexpr float by = 1.f; };
template <> struct VHalf<_Float16> { static constexpr float by = 0.5f; };

// Codes that one workgroup alone reads pass the caches by (four sequences of up to 131072 tokens, 1.0 GB: 178 -> 161 us)
template <bool ONCE, typename V>
__device__ __forceinline__ V codes(const V* p) {
    if constexpr (ONCE) return __builtin_nontemporal_load(p);
    else return *p;
}

// Wave w of a workgroup takes the blocks w, w + 4, ... of its part for RT * 16 rows (a row is one query of one head of
// the group); the four softmax states are joined through LDS at the end.  Token of the MFMA: row rho of K tile t is
// token 16 * (rho / 4) + 4 t + rho % 4, so lane group g ends up with the weights of the tokens 16 g .. 16 g + 15, which
// are the 16 bytes it loads from each row of V.
template <typename T, int HD, int RT, bool ONCE>
__global__ __launch_bounds__(256) void kv8_attn_kernel(AttnArgs a) {
    typedef typename Vec<T>::x8 x8;
    constexpr int KS = HD / 32, NT = HD / 16, C64 = HD / 64;
    constexpr bool ODD = HD % 64 != 0;                              // head dim 96: 64 + 32
    constexpr int OP = HD + 4;
    // 32 rows of 128: V is widened only where it is used and the next block's V asked for after that, 60 registers fewer, so that
    // two waves fit a SIMD (four sequences of up to 131072 tokens, 64 rows: 210 -> 189 us; 16 rows, 161 -> 163, are not)
    constexpr bool LATE = RT * HD > 192;
    __shared__ __attribute__((aligned(16))) float osh[4 * 16 * OP];
    __shared__ float msh[4 * 16], lsh[4 * 16];

    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    const star_kv8_cache& c = a.c;
    const int grp = a.s.H / c.Hkv, rows = grp * a.s.L;
    const int hk = blockIdx.x % c.Hkv, rg = (blockIdx.x / c.Hkv) % a.nrg, slot = blockIdx.x / (c.Hkv * a.nrg);

    // which part of which sequence
    int b = slot, part = 0, np = 1;
    const int per = cut(a, lane).per;
    if (a.slots != c.B) {
        int base = 0;
        b = -1;
        for (int b0 = 0; b0 < c.B; b0 += 64) {
            const int bb = b0 + lane;
            const int mine = bb < c.B ? parts_of(blocks_of(a, bb), per) : 0;
            int incl = mine;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int y = __shfl_up(incl, o, 64);
                if (lane >= o) incl += y;
            }
            const unsigned long long over = __ballot(base + incl > slot);
            if (over) {
                const int f = __builtin_ctzll(over);
                np = __shfl(mine, f, 64);
                part = slot - (base + __shfl(incl, f, 64) - np);
                b = b0 + f;
                break;
            }
            base += __shfl(incl, 63, 64);
        }
        if (b < 0) return;
        b = __builtin_amdgcn_readfirstlane(b);
        np = __builtin_amdgcn_readfirstlane(np);
        part = __builtin_amdgcn_readfirstlane(part);
    }
    const int n = held_by(a, b), nq = queries_of(a, b), nb = blocks_of(a, b);
    const int each = (nb + np - 1) / np, blk0 = part * each, blk1 = min(nb, blk0 + each);
    const int open = n / KB;                                        // the incomplete block (n % 64 tokens)

    int lim[RT];
    x8 qf[RT][KS];
    const int64_t came = a.s.causal ? (int64_t)n + max(c.dropped[b], 0) : 0;    // tokens of the sequence, those without room too
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int rho = (rg * RT + rt) * 16 + r16, i = rho / grp, hh = rho % grp;
        const bool real = rho < rows && i < nq;
        int see = n;
        if (a.s.causal) see = (int)min((int64_t)see, came - nq + i + 1);
        if (a.s.ilk_diag >= 0) see = (int)min((int64_t)see, (int64_t)i + a.s.ilk_diag + 1);
        lim[rt] = real ? max(see, 0) : 0;
        const T* qr = (const T*)a.q + (int64_t)b * a.s.q_sb + (int64_t)(hk * grp + (rho < rows ? hh : 0)) * a.s.q_sh +
                      (int64_t)(rho < rows ? i : 0) * a.s.q_sr;
#pragma unroll
        for (int cc = 0; cc < C64; ++cc) {
            qf[rt][2 * cc] = *(const x8*)(qr + 64 * cc + 16 * g);
            qf[rt][2 * cc + 1] = *(const x8*)(qr + 64 * cc + 16 * g + 8);
        }
        if constexpr (ODD) qf[rt][KS - 1] = *(const x8*)(qr + 64 * C64 + 8 * g);
    }
    const float c2 = a.s.scale * A_LOG2E;
    const int64_t bh = (int64_t)b * c.Hkv + hk;
    const uint8_t* kc = c.k_codes + bh * c.T * HD;
    const uint8_t* vc = c.v_codes + bh * c.T * HD;
    const float* ksc = c.k_scales + bh * (c.T / KB);
    const float* vsc = c.v_scales + bh * (c.T / KB);
    const float* brow = a.bias ? a.bias + (int64_t)b * a.s.bias_len : nullptr;

    f32x4 acc[RT][NT];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[rt][nt] = (f32x4){0.f, 0.f, 0.f, 0.f};
        m[rt] = M_NONE;
        l[rt] = 0.f;
    }

    const int krow = 16 * (r16 >> 2) + (r16 & 3);                   // token of this lane's K row, + 4 t
    // logits of one block -> weights as operands of the product with V; kscale includes the softmax scale
    auto softmax = [&](f32x4 (&sc)[RT][4], float kscale, int blk, x8 (&pf)[RT][2]) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float mx = M_NONE;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = blk * KB + 16 * g + 4 * t + i;
                    float x = sc[rt][t][i] * kscale;
                    if (brow) x += key < a.s.bias_len ? brow[key] * A_LOG2E : 0.f;
                    x = key < lim[rt] ? x : -INFINITY;
                    sc[rt][t][i] = x;
                    mx = fmaxf(mx, x);
                }
            if (!__all(mx <= m[rt] + M_SLACK)) {
                mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
                mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
                const float mn = fmaxf(m[rt], mx), al = __builtin_amdgcn_exp2f(m[rt] - mn);
                m[rt] = mn;
                l[rt] *= al;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[rt][nt][i] *= al;
            }
            float sum = 0.f;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = __builtin_amdgcn_exp2f(sc[rt][t][i] - m[rt]);
                    sum += p;
                    sc[rt][t][i] = p;
                }
            l[rt] += sum;
            pf[rt][0] = pack_b<T>(sc[rt][0], sc[rt][1]);
            pf[rt][1] = pack_b<T>(sc[rt][2], sc[rt][3]);
        }
    };

    u32x4 kr[4][C64], vr[NT];
    u32x2 ko[4];
    float ks_ = 0.f, vs_ = 0.f;
    auto load_k = [&](int blk) {
        const uint8_t* kb = kc + (int64_t)blk * KB * HD;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int cc = 0; cc < C64; ++cc) kr[t][cc] = codes<ONCE>((const u32x4*)(kb + (krow + 4 * t) * HD + 64 * cc + 16 * g));
            if constexpr (ODD) ko[t] = codes<ONCE>((const u32x2*)(kb + (krow + 4 * t) * HD + 64 * C64 + 8 * g));
        }
        ks_ = ksc[blk];
    };
    auto load_v = [&](int blk) {
        const uint8_t* vb = vc + (int64_t)blk * KB * HD;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) vr[nt] = codes<ONCE>((const u32x4*)(vb + (16 * nt + r16) * KB + 16 * g));
        vs_ = vsc[blk];
    };
    const int full1 = min(blk1, open);                              // complete blocks end here
    if (blk0 + wid < full1) {
        load_k(blk0 + wid);
        load_v(blk0 + wid);
    }
#pragma unroll 1
    for (int blk = blk0 + wid; blk < full1; blk += 4) {
        f32x4 sc[RT][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            x8 kf[KS];
#pragma unroll
            for (int cc = 0; cc < C64; ++cc) {
                kf[2 * cc] = widen<T>(kr[t][cc][0], kr[t][cc][1], 1.f);
                kf[2 * cc + 1] = widen<T>(kr[t][cc][2], kr[t][cc][3], 1.f);
            }
            if constexpr (ODD) kf[KS - 1] = widen<T>(ko[t][0], ko[t][1], 1.f);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                sc[rt][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) sc[rt][t] = mfma16(kf[ks], qf[rt][ks], sc[rt][t]);
            }
        }
        const float kscale = ks_ * c2, vs = vs_ * VHalf<T>::by;
        auto v_half = [&](int nt, int hf) { return widen<T>(vr[nt][2 * hf], vr[nt][2 * hf + 1], vs); };
        x8 vf[LATE ? 1 : NT][2];
        if constexpr (!LATE) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) vf[nt][0] = v_half(nt, 0), vf[nt][1] = v_half(nt, 1);
        }
        if (blk + 4 < full1) {                                      // in flight during the softmax and the product with V
            load_k(blk + 4);
            if constexpr (!LATE) load_v(blk + 4);
        }
        x8 pf[RT][2];
        softmax(sc, kscale, blk, pf);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const x8 v = LATE ? v_half(nt, hf) : vf[LATE ? 0 : nt][hf];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) acc[rt][nt] = mfma16(v, pf[rt][hf], acc[rt][nt]);
            }
        if constexpr (LATE) {
            if (blk + 4 < full1) load_v(blk + 4);
        }
    }
    if (open < blk1 && open >= blk0 && (open - blk0) % 4 == wid) {  // the open block, in 16 bits
        const T* kt = (const T*)c.k_tail + bh * KB * HD;
        const T* vt = (const T*)c.v_tail + bh * KB * HD;
        const int cnt = n - open * KB;
        f32x4 sc[RT][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            x8 kf[KS];
            const T* row = kt + (krow + 4 * t) * HD;
#pragma unroll
            for (int cc = 0; cc < C64; ++cc) {
                kf[2 * cc] = *(const x8*)(row + 64 * cc + 16 * g);
                kf[2 * cc + 1] = *(const x8*)(row + 64 * cc + 16 * g + 8);
            }
            if constexpr (ODD) kf[KS - 1] = *(const x8*)(row + 64 * C64 + 8 * g);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                sc[rt][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) sc[rt][t] = mfma16(kf[ks], qf[rt][ks], sc[rt][t]);
            }
        }
        x8 pf[RT][2];
        softmax(sc, c2, open, pf);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                x8 vf = *(const x8*)(vt + (16 * nt + r16) * KB + 16 * g + 8 * hf);
#pragma unroll
                for (int e = 0; e < 8; ++e)                         // (rows behind the last token may hold anything)
                    vf[e] = 16 * g + 8 * hf + e < cnt ? (T)((float)vf[e] * VHalf<T>::by) : (T)0.f;
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) acc[rt][nt] = mfma16(vf, pf[rt][hf], acc[rt][nt]);
            }
        }
    }

    // join the four waves, 16 rows at a time
    constexpr int PER = HD / 16;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        float sum = l[rt];
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        if (rt) __syncthreads();
        if (g == 0) {
            msh[wid * 16 + r16] = m[rt];
            lsh[wid * 16 + r16] = sum;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) *(f32x4*)(osh + (wid * 16 + r16) * OP + 16 * nt + 4 * g) = acc[rt][nt];
        __syncthreads();
        const int row = tid >> 4, d0 = (tid & 15) * PER;
        const int rho = (rg * RT + rt) * 16 + row;
        float mm = msh[row];
#pragma unroll
        for (int w = 1; w < 4; ++w) mm = fmaxf(mm, msh[w * 16 + row]);
        float ll = 0.f, o[PER];
#pragma unroll
        for (int e = 0; e < PER; ++e) o[e] = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = __builtin_amdgcn_exp2f(msh[w * 16 + row] - mm);
            ll += f * lsh[w * 16 + row];
#pragma unroll
            for (int e = 0; e < PER; ++e) o[e] += f * osh[(w * 16 + row) * OP + d0 + e];
        }
        if (rho >= rows) continue;
        if (np == 1) {
            const float inv = (ll > 0.f ? 1.0f / ll : ll) / VHalf<T>::by;       // ll = 0: nothing seen; NaN stays NaN
            T* orow = (T*)a.o + (int64_t)b * a.s.o_sb + (int64_t)(hk * grp + rho % grp) * a.s.o_sh + (int64_t)(rho / grp) * a.s.o_sr;
#pragma unroll
            for (int e = 0; e < PER; ++e) orow[d0 + e] = (T)(o[e] * inv);
        } else {
            const int64_t at = ((int64_t)slot * c.Hkv + hk) * rows + rho;
#pragma unroll
            for (int e = 0; e < PER; ++e) a.part[at * HD + d0 + e] = o[e];
            if ((tid & 15) == 0) {
                float* ml = a.part + (int64_t)a.slots * c.Hkv * rows * HD + 2 * at;
                ml[0] = mm;
                ml[1] = ll;
            }
        }
    }
}

// A row that was cut into few parts: one wave adds them up.
template <typename T, int HD>
__global__ __launch_bounds__(256) void kv8_join_few_kernel(AttnArgs a) {
    const int lane = threadIdx.x & 63;
    const star_kv8_cache& c = a.c;
    const int grp = a.s.H / c.Hkv, rows = grp * a.s.L;
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int b = (int)(item / ((int64_t)c.Hkv * rows));
    if (b >= c.B) return;
    const int hk = (int)(item / rows % c.Hkv), rho = (int)(item % rows);
    const int per = cut(a, lane).per;
    const int np = parts_of(blocks_of(a, b), per);
    if (np == 1) return;
    int base = 0;
    for (int b0 = 0; b0 < b; b0 += 64) base += b0 + lane < b ? parts_of(blocks_of(a, b0 + lane), per) : 0;
    base = wave_sum(base);
    const float* ml = a.part + (int64_t)a.slots * c.Hkv * rows * HD;
    const int64_t stride = (int64_t)c.Hkv * rows, at0 = (int64_t)base * stride + (int64_t)hk * rows + rho;
    PartSum<HD> ps;
    ps.ask(a.part + at0 * HD, ml + 2 * at0, stride, np, lane);
    float mm, ll;
    f32x4 o;
    ps.sum(lane, mm, ll, o);
    if (lane >= HD / 4) return;
    const float inv = (ll > 0.f ? 1.0f / ll : ll) / VHalf<T>::by;
    T* orow = (T*)a.o + (int64_t)b * a.s.o_sb + (int64_t)(hk * grp + rho % grp) * a.s.o_sh + (int64_t)(rho / grp) * a.s.o_sr;
    *(typename Vec<T>::x4*)(orow + 4 * lane) = pack4<T>(o * inv);
}

// Many parts: one workgroup a row, the parts' factors first, one per thread, then every thread adds the
// parts of four values, PG of them at a time with all loads in flight.
template <typename T, int HD>
__global__ __launch_bounds__(256) void kv8_join_kernel(AttnArgs a) {
    constexpr int D4 = HD / 4, PG = 256 / D4;                       // threads of a part, parts at a time
    constexpr int MOST = 256;
    __shared__ float fsh[MOST], red[8];
    __shared__ __attribute__((aligned(16))) float osh[PG * HD];
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    const star_kv8_cache& c = a.c;
    const int grp = a.s.H / c.Hkv, rows = grp * a.s.L;
    const int64_t item = blockIdx.x;
    const int b = (int)(item / ((int64_t)c.Hkv * rows)), hk = (int)(item / rows % c.Hkv), rho = (int)(item % rows);
    const int per = cut(a, lane).per;
    const int np = parts_of(blocks_of(a, b), per);
    if (np == 1) return;
    int base = 0;
    for (int b0 = 0; b0 < b; b0 += 64) base += b0 + lane < b ? parts_of(blocks_of(a, b0 + lane), per) : 0;
    base = wave_sum(base);
    const float* ml = a.part + (int64_t)a.slots * c.Hkv * rows * HD;
    const int64_t stride = (int64_t)c.Hkv * rows, at0 = (int64_t)base * stride + (int64_t)hk * rows + rho;
    float mm = M_NONE;
    for (int p = tid; p < np; p += 256) mm = fmaxf(mm, ml[2 * (at0 + p * stride)]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor(mm, o, 64));
    if (lane == 0) red[wid] = mm;
    __syncthreads();
    mm = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const int d4 = tid % D4, pg = tid / D4;
    f32x4 o = (f32x4){0.f, 0.f, 0.f, 0.f};
    float ll = 0.f;
    for (int p0 = 0; p0 < np; p0 += MOST) {
        const int cnt = min(np - p0, MOST);
        __syncthreads();
        if (tid < cnt) {
            const int64_t at = at0 + (p0 + tid) * stride;
            const float f = __builtin_amdgcn_exp2f(ml[2 * at] - mm);
            fsh[tid] = f;
            ll += f * ml[2 * at + 1];
        }
        __syncthreads();
        if (pg < PG) {
#pragma unroll 4
            for (int p = pg; p < cnt; p += PG) o += fsh[p] * *(const f32x4*)(a.part + (at0 + (p0 + p) * stride) * HD + 4 * d4);
        }
    }
    ll = wave_sum(ll);
    if (lane == 0) red[4 + wid] = ll;
    if (pg < PG) *(f32x4*)(osh + pg * HD + 4 * d4) = o;
    __syncthreads();
    if (tid >= HD) return;
    ll = (red[4] + red[5]) + (red[6] + red[7]);
    float sum = 0.f;
#pragma unroll
    for (int p = 0; p < PG; ++p) sum += osh[p * HD + tid];
    const float inv = (ll > 0.f ? 1.0f / ll : ll) / VHalf<T>::by;
    T* orow = (T*)a.o + (int64_t)b * a.s.o_sb + (int64_t)(hk * grp + rho % grp) * a.s.o_sh + (int64_t)(rho / grp) * a.s.o_sr;
    orow[tid] = (T)(sum * inv);
}

// ------------------------------------------------------------------------------------------------------ host side
static int check_cache(const star_kv8_cache* c, const char* who) {
    STAR_REQUIRE(c, "%s: null cache", who);
    STAR_REQUIRE(c->hd == 64 || c->hd == 96 || c->hd == 128, "%s: head dim %d not in {64, 96, 128}", who, c->hd);
    STAR_REQUIRE(c->dtype == STAR_DT_BF16 || c->dtype == STAR_DT_F16, "%s: dtype %d is neither bf16 nor fp16", who, c->dtype);
    STAR_REQUIRE(c->B >= 1 && c->B <= 65535 && c->Hkv >= 1 && c->Hkv <= 32767, "%s: %d sequences x %d heads", who, c->B, c->Hkv);
    STAR_REQUIRE(c->T >= KB && c->T % KB == 0, "%s: capacity %d is not a multiple of %d tokens", who, c->T, KB);
    STAR_REQUIRE(c->k_codes && c->k_scales && c->v_codes && c->v_scales && c->k_tail && c->v_tail && c->lens && c->dropped && c->tickets,
                 "%s: null pointer in the cache", who);
    const void* p[4] = {c->k_codes, c->v_codes, c->k_tail, c->v_tail};
    for (int i = 0; i < 4; ++i) STAR_REQUIRE(((uintptr_t)p[i] & 15) == 0, "%s: the cache must be 16-byte aligned", who);
    return STAR_OK;
}

// tiles of 16 rows of one workgroup.  Four would read and convert the codes half as often, with one wave a SIMD and, at head
// dim 128, half of the state in accumulation registers: 25 sequences of up to 15442 tokens, 40 rows a key head of 64, 177 us
// with four and 131 with two; 16 of 2000, 64 rows of 128, 43 and 26; four of up to 131072, 64 rows of 128, 199 and 189.
static int row_tiles(int rows) { return rows <= 16 ? 1 : 2; }
// (sequence, part) pairs that the grid has room for.  512 workgroups (two a CU) run at once: few sequences are cut into
// parts that fill these places once; where the sequences alone make half of them or more, there is room for three times
// as many parts besides, so that a sequence much longer than the others does not run alone at the end.  32 rows of 128 keep a
// CU busy almost alone, so that for them half of the places counts as all (40 sequences of 2000 tokens, 64 rows: 26 us
// whole, 30 in parts).
// Sequences that fill three quarters of the places and of which none is longer than 1.5 times their mean stay whole (53
// of 2590 to 2908 tokens, 8 key heads of 128, 5 queries: 97 us in parts, 73 whole).
// A part has 4 blocks (256 tokens) at least, one per wave, or 24 where the card is full without it.  The join is a launch of
// its own, 3.4 us, which a short cache does not repay (one query, 8 heads of 128: 10.1 us whole and 12.5 in parts for 1024
// tokens, 15.0 and 12.9 for 1536, 204 and 21 for 32000; 64 rows a key head of 64: 12.1 and 13.4
// for 1280, 16.8 and 13.5 for 2048).
struct Cut { int slots, min_part, even; };
static Cut attn_cut(const star_kv8_cache* c, int H, int L) {
    const int rows = H / c->Hkv * L, rt = row_tiles(rows), nrg = cdiv(rows, 16 * rt), blocks = c->T / KB;
    const int64_t places = 512 / ((int64_t)c->Hkv * nrg), fill = rt * c->hd > 192 ? places / 2 : places;
    const bool full = fill < 2 * c->B;
    const int min_part = full ? 24 : 4;
    if (full ? blocks <= 32 : rt == 1 ? blocks * c->hd <= 18 * 128 : blocks <= 22) return Cut{c->B, min_part, 0};
    const int64_t most = (int64_t)c->B * cdiv(blocks, min_part), s = full ? c->B + 3 * (places > 1 ? places : 1) : places;
    return Cut{(int)(s < most ? s : most), min_part, 4 * c->B >= 3 * fill};
}

#define KV8_BY_TYPE(DT, HDIM, CALL)                                                        \
    do {                                                                                   \
        if ((DT) == STAR_DT_BF16) {                                                        \
            if ((HDIM) == 64) { using T = __bf16; constexpr int HD = 64; CALL; }           \
            else if ((HDIM) == 96) { using T = __bf16; constexpr int HD = 96; CALL; }      \
            else { using T = __bf16; constexpr int HD = 128; CALL; }                       \
        } else {                                                                           \
            if ((HDIM) == 64) { using T = _Float16; constexpr int HD = 64; CALL; }         \
            else if ((HDIM) == 96) { using T = _Float16; constexpr int HD = 96; CALL; }    \
            else { using T = _Float16; constexpr int HD = 128; CALL; }                     \
        }                                                                                  \
    } while (0)

template <typename T, int HD>
static void launch_attn(const AttnArgs& a, int rt, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)a.slots * a.c.Hkv * a.nrg));
    if (rt == 1) hipLaunchKernelGGL((kv8_attn_kernel<T, HD, 1, true>), grid, dim3(256), 0, st, a);
    else if (a.nrg == 1) hipLaunchKernelGGL((kv8_attn_kernel<T, HD, 2, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((kv8_attn_kernel<T, HD, 2, false>), grid, dim3(256), 0, st, a);
    if (a.slots == a.c.B) return;
    // (one wave has 16 parts, 32 at hd 64, on their way at once: up to 32 the two take the same time, beyond it 64 parts 1 us more)
    const int64_t rows = (int64_t)a.c.B * a.s.H * a.s.L;
    if (a.slots <= 32 * a.c.B) hipLaunchKernelGGL((kv8_join_few_kernel<T, HD>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((kv8_join_kernel<T, HD>), dim3((unsigned)rows), dim3(256), 0, st, a);
}

}  // namespace star

extern "C" int star_kv8_append(const star_kv8_cache* c, const void* k, const void* v, int64_t k_sb, int64_t k_sh, int64_t k_sr,
                               int64_t v_sb, int64_t v_sh, int64_t v_sr, const int32_t* starts, const int32_t* counts,
                               int idx_stride, const int32_t* at, int max_rows, void* stream) {
    using namespace star;
    int rc = check_cache(c, "star_kv8_append");
    if (rc) return rc;
    STAR_REQUIRE(max_rows >= 0, "star_kv8_append: max_rows = %d", max_rows);
    STAR_REQUIRE((k && v) || max_rows == 0, "star_kv8_append: null pointer");
    STAR_REQUIRE((((uintptr_t)k | (uintptr_t)v) & 15) == 0, "star_kv8_append: k and v must be 16-byte aligned");
    const int64_t sd[6] = {k_sb, k_sh, k_sr, v_sb, v_sh, v_sr};
    for (int i = 0; i < 6; ++i) STAR_REQUIRE(sd[i] % 8 == 0, "star_kv8_append: strides must be multiples of 8 elements");
    AppendArgs a{*c, k, v, k_sb, k_sh, k_sr, v_sb, v_sh, v_sr, starts, counts, at, idx_stride, max_rows};
    STAR_REQUIRE(k_sr >= 0 && k_sr < (1ll << 23) && v_sr >= 0 && v_sr < (1ll << 23), "star_kv8_append: row strides %lld, %lld not in [0, 2^23)",
                 (long long)k_sr, (long long)v_sr);
    // A call of n rows completes at most (n + 63) / 64 blocks, and never more than the cache has.  4096 workgroups in all
    // (16 a CU) take them in turn, the next block's rows on their way while one is written: 32 prompts of up to 4000
    // tokens 168 us with a workgroup for every block, 110 with these
    const int gx = max(1, min(min(cdiv((int64_t)max_rows + KB - 1, KB), c->T / KB), 4096 / (2 * c->Hkv * c->B)));
    const dim3 grid(gx, 2 * c->Hkv, c->B);
    KV8_BY_TYPE(c->dtype, c->hd, hipLaunchKernelGGL((kv8_append_kernel<T, HD>), grid, dim3(256), 0, (hipStream_t)stream, a));
    STAR_LAUNCH_CHECK("star_kv8_append");
    return STAR_OK;
}

extern "C" size_t star_kv8_attn_workspace(const star_kv8_cache* c, int H, int L) {
    using namespace star;
    if (check_cache(c, "star_kv8_attn_workspace") || H < c->Hkv || H % c->Hkv || L < 1 || (int64_t)H * L >= (1ll << 24)) return 0;
    const int slots = attn_cut(c, H, L).slots;
    return slots == c->B ? 0 : (size_t)slots * H * L * (c->hd + 2) * sizeof(float);
}

extern "C" int star_kv8_attn(const star_kv8_cache* c, const void* q, const float* bias, const int32_t* q_len,
                             const star_kv8_query* s, void* o, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace star;
    int rc = check_cache(c, "star_kv8_attn");
    if (rc) return rc;
    STAR_REQUIRE(s && q && o, "star_kv8_attn: null pointer");
    STAR_REQUIRE(s->H >= c->Hkv && s->H % c->Hkv == 0, "star_kv8_attn: %d query heads do not divide into %d key heads", s->H, c->Hkv);
    STAR_REQUIRE(s->L >= 1 && s->bias_len >= 0, "star_kv8_attn: L = %d, bias_len = %d", s->L, s->bias_len);
    STAR_REQUIRE((((uintptr_t)q | (uintptr_t)o) & 15) == 0, "star_kv8_attn: q and o must be 16-byte aligned");
    const int64_t sd[6] = {s->q_sb, s->q_sh, s->q_sr, s->o_sb, s->o_sh, s->o_sr};
    for (int i = 0; i < 6; ++i) STAR_REQUIRE(sd[i] % 8 == 0, "star_kv8_attn: strides must be multiples of 8 elements");
    // (a launch has less than 2^32 threads in x)
    STAR_REQUIRE((int64_t)c->B * s->H * s->L < (1ll << 24), "star_kv8_attn: %d sequences x %d heads x %d queries", c->B, s->H, s->L);
    const int rows = s->H / c->Hkv * s->L, rt = row_tiles(rows);
    const Cut cut = attn_cut(c, s->H, s->L);
    AttnArgs a{*c, *s, q, o, s->bias_len > 0 ? bias : nullptr, q_len, cut.slots, cut.min_part, cut.even, cdiv(rows, 16 * rt), (float*)workspace};
    STAR_REQUIRE((int64_t)a.slots * c->Hkv * a.nrg < (1ll << 24), "star_kv8_attn: %d parts x %d heads x %d groups of rows", a.slots, c->Hkv, a.nrg);
    STAR_REQUIRE(!(s->bias_len > 0 && !bias), "star_kv8_attn: bias_len > 0 but bias is null");
    if (workspace_bytes < star_kv8_attn_workspace(c, s->H, s->L) || (a.slots > c->B && !workspace)) {
        set_error("star_kv8_attn: workspace of %zu bytes, %zu needed", workspace_bytes, star_kv8_attn_workspace(c, s->H, s->L));
        return STAR_ERR_WORKSPACE;
    }
    KV8_BY_TYPE(c->dtype, c->hd, (launch_attn<T, HD>(a, rt, (hipStream_t)stream)));
    STAR_LAUNCH_CHECK("star_kv8_attn");
    return STAR_OK;
}
