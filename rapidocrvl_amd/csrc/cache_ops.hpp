// cache_ops.hpp — kernels of the cache operators: masked prompt attention,
// attention of drafted trees, accumulated weights, row selection and
// compaction, over fp32 caches the caller owns.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "kernels.hpp"

namespace pocr {

// One call of the attention family.  Prompt form: seqs = 1, spans from
// begin/end; tree form: lens, counts and parents per sequence.
struct CacheAttn {
    const float *q, *k, *v;
    float *out, *lse;
    const int32_t *begin, *end;                // prompt spans, or null
    const int32_t *lens, *counts, *parents;    // tree
    const int32_t *pos;                        // tree: [seq][kv head][side], or null
    const float *slopes;
    float *weights;                            // [seq][kv head][side]
    const uint64_t *take;
    int64_t q_ss, q_st, k_ss, k_st, v_ss, v_st, o_ss, o_st, side;
    int n, rows0, rows, heads, kvh, group;     // rows: prompt rows0 + n, tree max_rows
    int key0;                                  // weights: first key of the grid
    float scale, cap, inv_group;
};

constexpr float kLog2e = 1.4426950408889634f;

// |a - b| of any two positions, up to 2^32: one instruction in the order of the
// unsigned (selects for it: 64 biased tokens' weights of 8,256 rows 22.9 us for 22.3)
__device__ __forceinline__ float distance(int a, int b) {
    uint32_t d;
    asm("v_sad_u32 %0, %1, %2, 0" : "=v"(d) : "v"((uint32_t)a ^ 0x80000000u), "v"((uint32_t)b ^ 0x80000000u));
    return (float)d;
}

// slope[h] to the base 2; the largest ones stay finite, so that distance 0 costs nothing
__device__ __forceinline__ float slope_of(const CacheAttn &p, int h) {
    const float x = p.slopes ? p.slopes[h] * kLog2e : 0.0f;
    return fabsf(x) == INFINITY ? copysignf(3.4028235e38f, x) : x;
}

// lane t of a full wave: token t of a drafted tree, the bits of itself and its
// ancestors (pointer doubling: after k rounds the bits cover 2^k generations)
__device__ __forceinline__ uint64_t tree_bits(const int32_t *parents, int n, int lane) {
    int par = -1;
    if (lane < n) {
        par = parents ? parents[lane] : lane - 1;
        if (par < 0 || par >= lane) par = -1;
    }
    uint64_t bits = 1ull << lane;
#pragma unroll
    for (int r = 0; r < 6; ++r) {
        const uint64_t up = __shfl((unsigned long long)bits, par & 63);
        const int next = __shfl(par, par & 63);
        if (par >= 0) {
            bits |= up;
            par = next;
        }
    }
    return bits;
}

// rows and tokens of a sequence, forced into range
struct SeqRows {
    int len, count;
};
__device__ __forceinline__ SeqRows seq_rows(const CacheAttn &p, int s) {
    const int count = p.counts ? min(max(p.counts[s], 0), p.n) : p.n;
    return {min(max(p.lens[s], 0), p.rows - count), count};
}

// ---------------------------------------------------------------------------
// attention on the matrix cores
// ---------------------------------------------------------------------------
// Products of fp32 operands as products of their fp16 halves x = hi + lo (11
// bits each, so 22 of the operand's 24): hi·hi + hi·lo + lo·hi, three
// v_mfma_f32_16x16x32_f16 where the fp32 matrix instruction takes eight times
// one's time.  Exponents are taken out first, by a power of two per query row,
// key row, value row and row of weights, so that no size of an operand leaves
// fp16's range and none costs another its bits.
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));

// the halves of a·f and b·f: the conversions and the remainders a·f - hi are
// each one mixed-precision multiply-add (hi's halves are read where they lie;
// without the empty asm the compiler makes each of them twice)
__device__ __forceinline__ v2h whole_v2h(v2h x) {
    uint32_t u = __builtin_bit_cast(uint32_t, x);
    asm("" : "+v"(u));
    return __builtin_bit_cast(v2h, u);
}
__device__ __forceinline__ void split_h(float a, float b, float f, v2h &hi, v2h &lo) {
    hi = whole_v2h((v2h){(_Float16)__builtin_fmaf(a, f, 0.0f), (_Float16)__builtin_fmaf(b, f, 0.0f)});
    lo = (v2h){(_Float16)__builtin_fmaf(a, f, -(float)hi[0]), (_Float16)__builtin_fmaf(b, f, -(float)hi[1])};
}
// likewise of a and b; one: 1, where the compiler does not see it
__device__ __forceinline__ void split_one(float a, float b, float one, v2h &hi, v2h &lo) {
    hi = whole_v2h(__builtin_convertvector((v2f){a, b}, v2h));
    lo = (v2h){(_Float16)__builtin_fmaf(a, one, -(float)hi[0]), (_Float16)__builtin_fmaf(b, one, -(float)hi[1])};
}

// x as rounded: no part of a multiply-add (a score less its row's rounded maximum is then at most 0)
__device__ __forceinline__ float rounded(float x) {
    asm("" : "+v"(x));
    return x;
}

constexpr int kTop = 14;        // operand rows are scaled to sizes below 2^kTop
constexpr int kSpread = 4;      // key (value) rows of one exponent's scale lie within 2^kSpread
constexpr int kMaxExp = 110;    // rows of larger exponents count as infinite
constexpr float kLowest = -3.0e38f;
// Up to here a score's last bit is 1/4 and whole numbers are exact: a weight's
// argument may be one multiply-add of the unrounded product and carry a power
// of two with the maximum.  Beyond, what that rounds away is more than the
// weights' room in fp16 (2^14 of 2^16), and each operation rounds for itself.
constexpr float kFarScore = 4194304.0f;
constexpr int kBlock = 32;      // keys per step
constexpr int kAttnThreads = 256;

// exponent e of a row from the bits of its largest size: |x| < 2^e
__device__ __forceinline__ int row_exp(uint32_t bits) { return max((int)(bits >> 23) - 126, -kMaxExp); }
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
__device__ __forceinline__ uint32_t umax3(uint32_t a, uint32_t b, uint32_t c) { return max(max(a, b), c); }

// a lane's share of a row, scaled by its exponent, as halves
template <int C>
__device__ __forceinline__ void split_row(const float (&x)[C][8], int e, v8h (&hi)[C], v8h (&lo)[C]) {
    const float f = pow2(kTop - e);
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            v2h h, l;
            split_h(x[c][i], x[c][i + 1], f, h, l);
            hi[c][i] = h[0];
            hi[c][i + 1] = h[1];
            lo[c][i] = l[0];
            lo[c][i + 1] = l[1];
        }
}

// lds_load from a uniform address and a lane's offset to a uniform LDS address
__device__ __forceinline__ void lds_load_at(const void *base, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "s"(lds) : "m0");
}

// max over the lanes l, l^16, l^32, l^48 (an MFMA column's four lane groups)
__device__ __forceinline__ uint32_t groups_umax(uint32_t v) {
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max((uint32_t)a[0], (uint32_t)a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max((uint32_t)b[0], (uint32_t)b[1]);
}
__device__ __forceinline__ float groups_max(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float groups_sum(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// tanh of N numbers, to 2.5 · 2^-24 of its value; NaN stays NaN.  Up to 0.85, x +
// x³·P(x²) with a P fitted to (tanh(x)/x − 1)/x² there (least largest error,
// 2^-27 of tanh); above, 1 − 2/(e^2x + 1), where the difference no longer
// cancels.  Scores are mostly far below their cap: a wave whose numbers all are
// takes the polynomial alone, 9 instructions a number instead of 22.
template <int N>
__device__ __forceinline__ void tanh_all(float (&x)[N]) {
    float top = fabsf(x[0]);
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, fabsf(x[i]));
    const bool some_high = __any(top > 0.85f);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float z = x[i] * x[i];
        float q = fmaf(z, 0.00144017930142581463f, -0.00714282691478729248f);
        q = fmaf(z, q, 0.0211210921406745911f);
        q = fmaf(z, q, -0.0537964627146720886f);
        q = fmaf(z, q, 0.133314788341522217f);
        q = fmaf(z, q, -0.333332657814025879f);
        const float low = fmaf(x[i] * z, q, x[i]);
        if (some_high) {
            const float a = fabsf(x[i]);
            const float d = __builtin_amdgcn_exp2f((a > 20.0f ? 20.0f : a) * (2.0f * kLog2e)) + 1.0f;
            float r = __builtin_amdgcn_rcpf(d);
            r = fmaf(fmaf(-d, r, 1.0f), r, r);
            x[i] = a > 0.85f ? copysignf(fmaf(-2.0f, r, 1.0f), x[i]) : low;
        } else {
            x[i] = low;
        }
    }
}

// x / p.group for x below 2^20 (the quotient is at least 1/2 group away from the next)
__device__ __forceinline__ int by_group(const CacheAttn &p, int x) { return (int)(((float)x + 0.5f) * p.inv_group); }

// the rows of one tile and its share of the keys
struct AttnTile {
    int lo, hi;        // keys some row of the tile sees: [lo, hi)
    int parts;         // shares they are cut into
    int from, to;      // this share's steps, from lo rounded down to a multiple of kBlock
};

// a tile's steps of `keys` keys cut into at most `splits` shares of at least `least` steps
// 32, 64 or 128 shares, us: one token over 6,400 rows and one KV head 14.6, 12.6,
// 14.1; 20,000 rows 23.6, 17.6, 17.0; 64,000 rows 53.5, 33.8, 24.9; one tree of 12
// over 8,192 rows and two KV heads 30.5, 26.1, 29.7; 30,000 rows 71.2, 47.1, 41.1.
// 64 do best up to about 20,000 rows; from four KV heads on the 256 workgroups of
// a call are the bound instead.
constexpr int kMaxShares = 64;
__device__ __forceinline__ void share_tile(AttnTile &t, int keys, int parts, int part) {
    const int steps = max(0, (t.hi - t.lo + keys - 1) / keys);
    t.parts = parts;
    t.from = (int)((uint32_t)steps * (uint32_t)part / (uint32_t)parts);  // at most 2^25 steps, 64 shares
    t.to = (int)((uint32_t)steps * (uint32_t)(part + 1) / (uint32_t)parts);
}
__device__ __forceinline__ void cut_tile(AttnTile &t, int keys, int splits, int least, int part) {
    t.lo &= ~(kBlock - 1);
    const int steps = max(0, (t.hi - t.lo + keys - 1) / keys);
    share_tile(t, keys, min(splits, max(1, steps / least)), part);
}

// what the launch adds to a call's arguments
struct TileCut {
    int lo, hi, all_lo, all_hi;  // keys some row of the tile sees, and all its rows see
    int first, parts;            // its jobs
};
struct AttnPlan {
    int tiles;        // row tiles per (sequence, KV head)
    int splits;       // shares a tile's keys may be cut into; 1: no partial sums
    int least;        // steps of a share
    float *part;      // sums of a share [128 or 16 rows][HD]: [tile][split], with images [KV head][job]
    float2 *stat;     // their rows' maxima and denominators
    int32_t *parts;   // [tile] shares in use
    // with images
    const uint8_t *img;  // [kv head][step] images of all rows
    int steps;        // images per KV head
    TileCut *cuts;    // [tile]
    int32_t *jobs;    // [max_jobs] a job's tile, long rows first, or -1
    int max_jobs;     // workgroups per KV head; tiles: their keys are not cut
};

// A step's 32 key and value rows as the matrix instructions take them, in LDS
// and, for prompts of many tiles, in memory:
//   K  [16-key tile][32-dim chunk][half] lane l = 16·q + r: key r, dims 32c + 8q .. +7
//   V  [32-dim chunk][t][half] lane l = 16·q + j: keys 4q .. +3 and 16+4q .. +3, dim 32c + 2j + t
//   the keys' factors kf (key row = stored · kf) and vf (value row = stored · 2^-kTop · vf).
// Scores come out with lane group q on keys 4q .. +3 and 16+4q .. +3; where the
// exponents of these eight rows allow it, for all four groups (`even`), a
// group's rows have one factor: a lane then needs one of each.
template <int HD>
struct StepImage {
    static constexpr int C = HD / 32, kK = 2 * C * 2 * 1024, kV = C * 2 * 2 * 1024, kSide = kK + kV, kBytes = kSide + 1024;
    uint8_t k[kK], v[kV];
    float kf[kBlock], vf[kBlock];
    float kf_group[4];
    int ve_group[4];  // exponents of vf
    int even[4];
    uint8_t pad[1024 - 8 * kBlock - 48];
};
static_assert(sizeof(StepImage<128>) == StepImage<128>::kBytes && sizeof(StepImage<64>) == StepImage<64>::kBytes, "whole KB");

// Lays eight rows of each of K and V into a step's image, those of lane group
// `group`, by one wave that waits for no other.  K: lane kk + 8·part holds key
// kk's floats 4·part + 32c .. +3 (whole 128-byte lines); V: lane l dims 2l,
// 2l + 1 of all eight keys (heads of 64: lanes l and l + 32 four keys each).
template <int HD>
struct StepLayer {
    static constexpr int C = HD / 32, kVKeys = HD == 128 ? 8 : 4;
    v4f kx[C];
    v2f vx[kVKeys];
    __device__ __forceinline__ static int key_of(int group, int i) { return 4 * group + (i & 3) + 4 * (i & 4); }
    __device__ __forceinline__ static int v_first(int lane) { return HD == 128 ? 0 : (lane >> 5) * 4; }
    // k, v: row 0 of the KV head; keys k0 .. k0+31, those past `last` as it
    __device__ __forceinline__ void load(const float *k, int64_t k_st, const float *v, int64_t v_st, int k0, int last, int group, int lane) {
        const float *ks = k + min(k0 + key_of(group, lane & 7), last) * k_st + 4 * (lane >> 3);
#pragma unroll
        for (int c = 0; c < C; ++c) kx[c] = *reinterpret_cast<const v4f *>(ks + 32 * c);
        const float *vs = v + 2 * (lane % (HD / 2));
#pragma unroll
        for (int i = 0; i < kVKeys; ++i)
            vx[i] = *reinterpret_cast<const v2f *>(vs + min(k0 + key_of(group, v_first(lane) + i), last) * v_st);
    }
    template <int N, int X>
    __device__ __forceinline__ static void halve(uint32_t (&m)[8], bool upper) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t keep = upper ? m[i + N] : m[i], give = upper ? m[i] : m[i + N];
            m[i] = max(keep, __float_as_uint(xchg<X>(__uint_as_float(give))));
        }
    }
    __device__ __forceinline__ void put(StepImage<HD> *im, int group, int lane) const {
        // sizes: lane's K key kk = lane & 7, and V key i
        uint32_t kt = 0;
#pragma unroll
        for (int c = 0; c < C; ++c)
            kt = umax3(kt, max(abs_bits(kx[c][0]), abs_bits(kx[c][1])), max(abs_bits(kx[c][2]), abs_bits(kx[c][3])));
        kt = max(kt, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)kt, 0x128, 0xF, 0xF, false));  // lane ^ 8
        const int ke = row_exp(groups_umax(kt));
        uint32_t m[8];
#pragma unroll
        for (int i = 0; i < kVKeys; ++i) m[i] = max(abs_bits(vx[i][0]), abs_bits(vx[i][1]));
        if (kVKeys == 8) halve<4, XM16>(m, lane & 8);
        else
#pragma unroll
            for (int i = 0; i < 4; ++i) m[i] = max(m[i], __float_as_uint(xchg<XM16>(__uint_as_float(m[i]))));
        halve<2, XM8>(m, lane & 4);
        halve<1, XQ2>(m, lane & 2);
        m[0] = max(m[0], __float_as_uint(xchg<XQ1>(__uint_as_float(m[0]))));
        const int at = (kVKeys == 8 ? (lane & 8) >> 1 : (lane >> 5) * 4) + ((lane & 4) >> 1) + ((lane & 2) >> 1);  // the key of m[0]
        {
            const auto a = __builtin_amdgcn_permlane16_swap(m[0], m[0], false, false);
            m[0] = max((uint32_t)a[0], (uint32_t)a[1]);
        }
        if (HD == 128) {
            const auto a = __builtin_amdgcn_permlane32_swap(m[0], m[0], false, false);
            m[0] = max((uint32_t)a[0], (uint32_t)a[1]);
        }
        const int ve = row_exp(m[0]);
        // all eight of each: the wave's largest
        const int k_hi = max8lanes(ke);
        int v_hi = max8lanes(ve);  // over lanes of a row of 16
        v_hi = max(v_hi, __float_as_int(xchg<XM16>(__int_as_float(v_hi))));
        {
            const auto a = __builtin_amdgcn_permlane32_swap((uint32_t)v_hi, (uint32_t)v_hi, false, false);
            v_hi = max((int)a[0], (int)a[1]);
        }
        const bool even = __all(ke >= k_hi - kSpread && ve >= v_hi - kSpread && k_hi <= kMaxExp && v_hi <= kMaxExp);
        const int kk = even ? k_hi : ke;
        {
            const int key = key_of(group, lane & 7), part = lane >> 3;
            const float f = pow2(kTop - kk);
            uint8_t *dst = im->k + (key >> 4) * C * 2048 + (16 * (part >> 1) + (key & 15)) * 16 + (part & 1) * 8;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                v2h h0, l0, h1, l1;
                split_h(kx[c][0], kx[c][1], f, h0, l0);
                split_h(kx[c][2], kx[c][3], f, h1, l1);
                *reinterpret_cast<v4h *>(dst + c * 2048) = (v4h){h0[0], h0[1], h1[0], h1[1]};
                *reinterpret_cast<v4h *>(dst + c * 2048 + 1024) = (v4h){l0[0], l0[1], l1[0], l1[1]};
            }
            if (part == 0) im->kf[key] = pow2(kk - kTop);
        }
        const int ee = even ? v_hi : ve;
        if ((lane & 1) == 0 && (HD == 64 || lane < 16)) im->vf[key_of(group, at)] = ee > kMaxExp ? __uint_as_float(0x7fc00000u) : pow2(ee);
        // rows that count as infinite are stored as zeros
        const float mine = ee > kMaxExp ? 0.0f : pow2(kTop - ee);
        uint8_t *dst = im->v + (lane % (HD / 2)) / 16 * 4096 + (16 * group + (lane & 15)) * 16 + v_first(lane) * 2;
#pragma unroll
        for (int i = 0; i < kVKeys; i += 4) {
            float f[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) f[x] = even ? mine : __shfl(mine, key_lane(v_first(lane) + i + x));
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                v2h h0, l0, h1, l1;
                if (even) {
                    split_h(vx[i][t], vx[i + 1][t], mine, h0, l0);
                    split_h(vx[i + 2][t], vx[i + 3][t], mine, h1, l1);
                } else {
                    float y[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) y[x] = f[x] != 0.0f ? vx[i + x][t] * f[x] : 0.0f;
                    split_h(y[0], y[1], 1.0f, h0, l0);
                    split_h(y[2], y[3], 1.0f, h1, l1);
                }
                *reinterpret_cast<v4h *>(dst + 2 * i + 2048 * t) = (v4h){h0[0], h0[1], h1[0], h1[1]};
                *reinterpret_cast<v4h *>(dst + 2 * i + 2048 * t + 1024) = (v4h){l0[0], l0[1], l1[0], l1[1]};
            }
        }
        if (lane == 0) {
            im->kf_group[group] = pow2(min(k_hi, kMaxExp) - kTop);
            im->ve_group[group] = v_hi;
            im->even[group] = even;
        }
    }
    // a lane that holds V key i's size (of a half of the lanes for heads of 64)
    __device__ __forceinline__ static int key_lane(int i) {
        return HD == 128 ? ((i & 4) << 1) + ((i & 2) << 1) + ((i & 1) << 1) : ((i & 4) << 3) + ((i & 2) << 1) + ((i & 1) << 1);
    }
    __device__ __forceinline__ static int max8lanes(int v) {
        v = max(v, __float_as_int(xchg<XQ1>(__int_as_float(v))));
        v = max(v, __float_as_int(xchg<XQ2>(__int_as_float(v))));
        return max(v, __float_as_int(xchg<XM8>(__int_as_float(v))));
    }
};

// The jobs of a prompt's tiles: the spans of each, and shares as even as
// max_jobs workgroups allow, by bisecting the length of a share.  One workgroup,
// done before the images beside it are (5 to 6 us).  Shares cut by each tile's
// own workgroups, a fixed number of them, left most of these without work where
// prompts are packed: seven in 2,403 rows took 56 us, cut here 42.
constexpr int kCutTiles = 512;  // tiles that may be cut
constexpr int kTileRows = 128;
__device__ __forceinline__ void cut_prompt(const CacheAttn &p, const AttnPlan &pl) {
    __shared__ int s_steps[kCutTiles], s_wave[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, rows = p.n * p.group;
    const bool cut = pl.max_jobs > pl.tiles;
    int most = 1;
    for (int tile = tid; tile < pl.tiles; tile += kAttnThreads) {
        const int tok0 = tile * kTileRows / p.group, tok1 = (min((tile + 1) * kTileRows, rows) - 1) / p.group;
        TileCut c{0, p.rows0 + tok1 + 1, 0, p.rows0 + tok0 + 1, pl.tiles - 1 - tile, 1};
        if (p.begin) {
            c.lo = c.all_hi = p.rows;
            c.hi = c.all_lo = 0;
#pragma unroll 8
            for (int tok = tok0; tok <= tok1; ++tok) {
                const int b = min(max(p.begin[tok], 0), p.rows), e = min(max(p.end[tok], 0), p.rows);
                c.lo = b < e ? min(c.lo, b) : c.lo;
                c.hi = b < e ? max(c.hi, e) : c.hi;
                c.all_lo = max(c.all_lo, b);
                c.all_hi = min(c.all_hi, e);
            }
            c.lo = c.lo < c.hi ? c.lo & ~(kBlock - 1) : c.hi;
        }
        pl.cuts[tile] = c;
        if (!cut) pl.jobs[c.first] = tile;
        const int steps = (c.hi - c.lo + kBlock - 1) / kBlock;
        if (cut) s_steps[tile] = steps;
        most = max(most, steps);
    }
    if (!cut) return;
    __syncthreads();
    auto parts_of = [&](int steps, int length) {  // steps / length rounded up, 1 to kMaxShares; both at most 2^25
        const uint32_t n = steps + length - 1;
        if (n >= (uint32_t)kMaxShares * length) return kMaxShares;
        int parts = (int)((float)n * __builtin_amdgcn_rcpf((float)length));
        parts -= parts * length > (int)n;
        parts += (parts + 1) * length <= (int)n;
        return max(parts, 1);
    };
    // every wave by itself, eight tiles a lane
    int own[kCutTiles / 64];
#pragma unroll
    for (int i = 0; i < kCutTiles / 64; ++i) {
        const int tile = 64 * i + lane;
        own[i] = tile < pl.tiles ? s_steps[tile] : -1;
        most = max(most, own[i]);
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) most = max(most, __shfl_xor(most, o));
    int lo = pl.least, hi = max(lo, most);
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        float jobs = 0.0f;
#pragma unroll
        for (int i = 0; i < kCutTiles / 64; ++i) jobs += own[i] < 0 ? 0.0f : (float)parts_of(own[i], mid);
        if (wave_sum(jobs) <= (float)pl.max_jobs) hi = mid;
        else lo = mid + 1;
    }
    // jobs in order, the last tile's first: two tiles a thread
    const int at = pl.tiles - 1 - 2 * tid;
    const int n0 = at >= 0 ? parts_of(s_steps[at], lo) : 0, n1 = at >= 1 ? parts_of(s_steps[at - 1], lo) : 0;
    int before = n0 + n1;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(before, o);
        if (lane >= o) before += y;
    }
    if (lane == 63) s_wave[wave] = before;
    __syncthreads();
    for (int w = 0; w < wave; ++w) before += s_wave[w];
    before -= n0 + n1;
    for (int i = 0; i < n0 + n1; ++i) pl.jobs[before + i] = i < n0 ? at : at - 1;
    if (at >= 0) {
        pl.cuts[at].first = before;
        pl.cuts[at].parts = n0;
    }
    if (at >= 1) {
        pl.cuts[at - 1].first = before + n0;
        pl.cuts[at - 1].parts = n1;
    }
    const int jobs = s_wave[0] + s_wave[1] + s_wave[2] + s_wave[3];
    for (int i = jobs + tid; i < pl.max_jobs; i += kAttnThreads) pl.jobs[i] = -1;
}

// Images of all of a prompt's rows, for prompts of so many tiles that laying
// every step out in each of them would cost more, and the tiles' jobs.
// Workgroup: the jobs, or one step of one KV head.  16.8 MB of rows in 8.6 us,
// 3.9 TB/s of reads and writes.
template <int HD>
__global__ void __launch_bounds__(kAttnThreads) k_cache_images(CacheAttn p, AttnPlan pl, uint8_t *img) {
    using Im = StepImage<HD>;
    __shared__ __attribute__((aligned(16))) Im im;
    const int tid = threadIdx.x, g = blockIdx.y, step = (int)blockIdx.x - 1;
    if (step < 0) {
        if (g == 0) cut_prompt(p, pl);
        return;
    }
    StepLayer<HD> st;
    st.load(p.k + g * HD, p.k_st, p.v + g * HD, p.v_st, step * kBlock, p.rows - 1, tid >> 6, tid & 63);
    st.put(&im, tid >> 6, tid & 63);
    __syncthreads();
    const uint4 *src = reinterpret_cast<const uint4 *>(&im);
    uint4 *dst = reinterpret_cast<uint4 *>(img + ((size_t)g * pl.steps + step) * Im::kBytes);
    for (int i = tid; i < Im::kBytes / 16; i += kAttnThreads) dst[i] = src[i];
}

// Workgroup: 128 rows (token, head of the KV head's group) of one sequence and
// KV head; one share of the keys, 32 a step.  Scores come out transposed (lane
// l: query row l%16, keys 4·(l/16) + i of each 16), so a row's maximum,
// denominator and weights stay with its four lanes and the weights are the
// second product's operand as they are; the sums come out transposed too (lane:
// the same query row, 8 consecutive dims of each 32).  Two LDS buffers: a step's
// products run on one while the next step's image arrives in the other.
//
// IMG: images come ready from memory by direct loads; four waves of 32 rows (a
// value read from LDS serves two products), two workgroups a CU, so one's
// softmax runs beside the other's products.  8,192 causal rows of 16 heads:
// 825 GFLOP of fp16 products in 0.75 ms, 1,103 TFLOP/s where a large matrix
// product of the library reaches 1,159.  Its products alone, with no softmax and
// no LDS reads between them, take 0.57 ms: the clock falls under them.
// (256 rows in eight waves, whose halves take turns at products and softmax
// behind barriers, were no faster there and took 80 us for 61 at 1,345 rows.)
// Otherwise one workgroup a CU: four waves do nothing but lay rows out, eight of
// 16 rows multiply.  What the ones spend on vector instructions runs beside the
// others' matrix instructions; eight waves that did both in turn took 65 us for
// one tree of 64 over 8,192 rows, four of each 38, four and eight 33.
//
// A row's weights are e = 2^(x - m), m an integer above its maximum so far; the
// products take e·vf·2^(14-a) with 2^a above the row's largest e·vf so far, so
// the halves hold the products that count whatever the sizes of V's rows.  All
// rescales are by powers of two.  Steps that every row of the tile sees, with
// even factors, need neither masks nor factors per key.
template <int HD, bool TREE, bool SHAPED, bool IMG>
__global__ void __launch_bounds__(IMG ? 256 : 768, IMG ? 2 : 3) k_cache_attn(CacheAttn p, AttnPlan pl) {
    using Im = StepImage<HD>;
    constexpr int C = HD / 32;              // 32-dim chunks
    constexpr int QT = IMG ? 2 : 1, W = IMG ? 4 : 8, kRows = 16 * W * QT;
    __shared__ __attribute__((aligned(16))) Im ims[2];
    __shared__ uint64_t s_bits[64];
    __shared__ int s_depth[64], s_lo, s_hi, s_lo_max, s_hi_min;
    __shared__ int2 s_row[kRows];  // the cache rows that each row sees: [x, y)

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r16 = lane & 15, kg = lane >> 4;
    const int g = blockIdx.y, s = blockIdx.z;
    int tile, part;
    if (IMG) {
        tile = pl.jobs[blockIdx.x];
        if (tile < 0) return;
        part = (int)blockIdx.x - pl.cuts[tile].first;
    } else {
        tile = pl.tiles - 1 - (int)(blockIdx.x / pl.splits), part = blockIdx.x % pl.splits;  // long rows first
    }
    const int first_row = tile * kRows;
    int len = 0, count = p.n;
    if (TREE) {
        const SeqRows q = seq_rows(p, s);
        len = q.len;
        count = q.count;
    }
    const int rows = count * p.group;
    const size_t slot = ((size_t)s * p.kvh + g) * pl.tiles + tile;
    if (first_row >= rows) {
        if (pl.parts && part == 0 && tid == 0) pl.parts[slot] = 0;
        return;
    }
    // the keys of the tile, and those that all its rows see
    AttnTile t{0, 0, 1, 0, 0};
    int all_lo = 0, all_hi;
    const int tok0 = first_row / p.group, tok1 = (min(first_row + kRows, rows) - 1) / p.group;
    if (IMG) {
        const TileCut c = pl.cuts[tile];
        t.lo = c.lo;
        t.hi = c.hi;
        all_lo = c.all_lo;
        all_hi = c.all_hi;
        share_tile(t, kBlock, c.parts, part);
    } else {
        if (TREE) {
            t.hi = len + count;
            all_hi = len;
            if (wave == 0) {
                const uint64_t b = tree_bits(p.parents ? p.parents + (size_t)s * p.n : nullptr, p.n, lane);
                s_bits[lane] = b;
                s_depth[lane] = __popcll(b) - 1;
            }
            __syncthreads();
        } else if (p.begin) {
            if (tid == 0) {
                s_lo = s_hi_min = p.rows;
                s_hi = s_lo_max = 0;
            }
            __syncthreads();
            const int tok = tok0 + tid;
            if (tok <= tok1) {  // at most kRows tokens
                const int b = min(max(p.begin[tok], 0), p.rows), e = min(max(p.end[tok], 0), p.rows);
                if (b < e) {
                    atomicMin(&s_lo, b);
                    atomicMax(&s_hi, e);
                }
                atomicMax(&s_lo_max, b);
                atomicMin(&s_hi_min, e);
            }
            __syncthreads();
            t.lo = s_lo & ~(kBlock - 1);
            t.hi = s_hi;
            all_lo = s_lo_max;
            all_hi = s_hi_min;
        } else {
            t.hi = p.rows0 + tok1 + 1;
            all_hi = p.rows0 + tok0 + 1;
        }
        cut_tile(t, kBlock, pl.splits, pl.least, part);
        if (part >= t.parts) return;
        if (pl.parts && part == 0 && tid == 0) pl.parts[slot] = t.parts;
    }
    const size_t share = IMG ? (size_t)g * pl.max_jobs + blockIdx.x : slot * pl.splits + part;

    // the first step's rows are on their way before the query rows
    const uint8_t *images = IMG ? pl.img + ((size_t)g * pl.steps + t.lo / kBlock) * Im::kBytes : nullptr;
    const uint32_t ims_at = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void *)ims;
    const int wave_u = __builtin_amdgcn_readfirstlane(wave);
    auto fetch = [&](int step, int b) {
        constexpr int kChunks = Im::kBytes / 1024;
        const uint8_t *src = images + (size_t)step * Im::kBytes + wave_u * 1024;
        const uint32_t dst = ims_at + b * Im::kBytes + wave_u * 1024;
#pragma unroll
        for (int i = 0; i < (kChunks + W - 1) / W; ++i)
            if (W * i + wave_u < kChunks) lds_load_at(src + i * W * 1024, 16 * lane, dst + i * W * 1024);
    };
    if (IMG && t.from < t.to) fetch(t.from, 0);
    if (!IMG && wave_u >= W) {  // a producer: its group's rows of every step, two steps ahead of their use
        const float *kbase = p.k + s * p.k_ss + g * HD, *vbase = p.v + s * p.v_ss + g * HD;
        StepLayer<HD> x[2];
        if (t.from < t.to) x[0].load(kbase, p.k_st, vbase, p.v_st, t.lo + t.from * kBlock, t.hi - 1, wave_u - W, lane);
        if (t.from + 1 < t.to) x[1].load(kbase, p.k_st, vbase, p.v_st, t.lo + (t.from + 1) * kBlock, t.hi - 1, wave_u - W, lane);
        for (int step = t.from; step < t.to; step += 2) {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                if (step + b >= t.to) break;
                x[b].put(&ims[b], wave_u - W, lane);
                if (step + b + 2 < t.to)
                    x[b].load(kbase, p.k_st, vbase, p.v_st, t.lo + (step + b + 2) * kBlock, t.hi - 1, wave_u - W, lane);
                __syncthreads();  // the step is there, and the one before it done with
            }
        }
        return;
    }
    const int last = t.hi - 1;

    // query rows: halves, scale, what they see
    v8h qh[QT][C], ql[QT][C];
    float qf[QT], slope[QT];
    int row_pos[QT];
    uint64_t bits[QT];
#pragma unroll
    for (int u = 0; u < QT; ++u) {
        const int row = first_row + (wave * QT + u) * 16 + r16;
        const bool live = row < rows;
        const int in = row - tok0 * p.group, tok = live ? tok0 + by_group(p, in) : tok0;
        const int h = g * p.group + (live ? row - tok * p.group : 0);
        const float *src = p.q + s * p.q_ss + tok * p.q_st + h * HD + 8 * kg;
        float x[C][8];
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const v4f a = *reinterpret_cast<const v4f *>(src + 32 * c), b = *reinterpret_cast<const v4f *>(src + 32 * c + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[c][i] = a[i];
                x[c][4 + i] = b[i];
                top = umax3(top, abs_bits(a[i]), abs_bits(b[i]));
            }
        }
        const int e = row_exp(groups_umax(top));
        split_row<C>(x, e, qh[u], ql[u]);
        qf[u] = pow2(e - kTop) * (SHAPED ? p.scale : p.scale * kLog2e);
        slope[u] = SHAPED ? slope_of(p, h) : 0.0f;
        row_pos[u] = 0;
        bits[u] = 0;
        int2 sees = {0, 0};
        if (TREE) {
            if (live) {
                sees.y = len;
                bits[u] = s_bits[tok];
                if (SHAPED) row_pos[u] = p.pos ? p.pos[((size_t)s * p.kvh + g) * p.side + len + tok] : len + s_depth[tok];
            }
        } else if (live) {
            sees.x = p.begin ? min(max(p.begin[tok], 0), p.rows) : 0;
            sees.y = p.end ? min(max(p.end[tok], 0), p.rows) : p.rows0 + tok + 1;
            row_pos[u] = p.rows0 + tok;
        }
        if (kg == 0) s_row[row - first_row] = sees;  // for this wave alone
    }
    const float inv_cap = SHAPED && p.cap > 0.0f ? 1.0f / p.cap : 0.0f, cap2 = SHAPED && p.cap > 0.0f ? p.cap * kLog2e : kLog2e;
    const int32_t *pos = TREE && SHAPED && p.pos ? p.pos + ((size_t)s * p.kvh + g) * p.side : nullptr;

    v4f o[QT][2 * C];
    float m[QT], l[QT];
    int a[QT];  // o holds the weighted sums, relative to 2^m, times 2^(14 + kTop - a)
#pragma unroll
    for (int u = 0; u < QT; ++u) {
        m[u] = kLowest;
        l[u] = 0.0f;
        a[u] = -16384;
#pragma unroll
        for (int d = 0; d < 2 * C; ++d) o[u][d] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
    }
    // a row's maximum (in its four lanes), and the largest exponent of its
    // weighted values: the power of two that its sums are due for it
    auto raise_m = [&](int u, float top) {
        const float mn = top > m[u] ? ceilf(top) + 2.0f : m[u];
        l[u] *= __builtin_amdgcn_exp2f(m[u] - mn);
        a[u] = max(a[u] - (int)fminf(mn - m[u], 16384.0f), -16384);
        m[u] = mn;
    };
    auto raise_a = [&](int u, int need) {
        const int an = need > a[u] ? need + 3 : a[u], by = max(a[u] - an, -200);
        a[u] = an;
        return by;
    };
    auto max8 = [](const float (&x)[8]) {
        return fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
    };
    float one = 1.0f;
    asm("" : "+s"(one));
    const bool live_wave = first_row + wave * QT * 16 < rows;

    v4f sc[QT][2];
    v8h ph[QT], pL[QT];
    // Products of a step in pieces of 12·QT: pieces 0 .. C-1 its sums, C .. 2C-1 its
    // scores.  A piece's operands are on their way two pieces before (by itself the
    // compiler asks for them right before their use: 61 us for 58 at 1,345 rows that
    // see each other, 8,192 causal rows 3% more); neighbouring products go to
    // different sums.
    auto products = [&](auto first, auto end, const Im &im) {
        constexpr int kFirst = decltype(first)::value, kEnd = decltype(end)::value;
        v8h f[2 * C][4];
        auto load = [&](int i) {
#pragma unroll
            for (int y = 0; y < 4; ++y)
                f[i][y] = *reinterpret_cast<const v8h *>((i < C ? im.v + (2 * i + (y >> 1)) * 2048 : im.k + ((y >> 1) * C + i - C) * 2048) +
                                                         (y & 1) * 1024 + lane * 16);
        };
        load(kFirst);
        load(kFirst + 1);
        if (kFirst == C)
#pragma unroll
            for (int u = 0; u < QT; ++u) sc[u][0] = sc[u][1] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = kFirst; i < kEnd; ++i) {
            if (i + 2 < kEnd) load(i + 2);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int x = 0; x < 3; ++x)
#pragma unroll
                for (int y = 0; y < 2; ++y)
#pragma unroll
                    for (int u = 0; u < QT; ++u) {
                        const v8h op = f[i][2 * y + (x == 0)];
                        if (i < C)
                            o[u][2 * i + y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(op, x == 1 ? pL[u] : ph[u], o[u][2 * i + y], 0, 0, 0);
                        else
                            sc[u][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(op, x == 1 ? ql[u][i - C] : qh[u][i - C], sc[u][y], 0, 0, 0);
                    }
        }
    };
    constexpr std::integral_constant<int, 0> kSums;
    constexpr std::integral_constant<int, C> kScores;
    constexpr std::integral_constant<int, 2 * C> kAll;
    // a step's weights; false: no row of the wave sees it
    auto softmax = [&](int k0, const Im &im) {
        const bool whole = k0 >= all_lo && k0 + kBlock <= all_hi;
        // what each row sees of the step's keys, as bits
        uint32_t see[QT];
        if (!whole) {
            bool any = false;
#pragma unroll
            for (int u = 0; u < QT; ++u) {
                const int2 sees = s_row[(wave * QT + u) * 16 + r16];
                const int n1 = min(max(sees.y - k0, 0), 32), n0 = min(max(sees.x - k0, 0), 32);
                see[u] = (uint32_t)((1ull << n1) - 1) & ~(uint32_t)((1ull << n0) - 1);
                if (TREE) {
                    const int off = k0 - len;  // the step's first key among the drafted ones
                    if (off > -32 && off < 64) see[u] |= (uint32_t)(off >= 0 ? bits[u] >> off : bits[u] << -off);
                }
                any = any || see[u];
            }
            if (!__any(any)) return false;
        }
        // capped and biased scores, to the base 2, of keys k0 + 16(e/4) + 4kg + e%4
        auto shape = [&](int u, float (&x)[8]) {
            if (p.cap > 0.0f) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] *= inv_cap;
                tanh_all(x);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= cap2;
            if (!p.slopes) return;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int in = 16 * (e >> 2) + (e & 3);
                float dist = (float)(row_pos[u] - k0 - 4 * kg) - (float)in;
                if (TREE) {
                    if (e == 4) __builtin_amdgcn_sched_barrier(0);  // not all eight loads at once: registers
                    const int key = k0 + 4 * kg + in;
                    const int at = pos ? pos[min(key, last)] : (key < len ? key : len + s_depth[min(key - len, 63)]);
                    dist = distance(row_pos[u], at);
                }
                x[e] = fmaf(-slope[u], fabsf(dist), x[e]);
            }
        };
        int by[QT];
        auto weights = [&](int u, const float (&w)[8]) {
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                v2h hi, lo;
                split_one(w[e], w[e + 1], one, hi, lo);
                ph[u][e] = hi[0];
                ph[u][e + 1] = hi[1];
                pL[u][e] = lo[0];
                pL[u][e + 1] = lo[1];
            }
        };
        if (whole && __all(im.even[kg])) {  // all rows see all keys, the lane's keys have one factor
            const float kf = im.kf_group[kg];
            const int ve = im.ve_group[kg];
#pragma unroll
            for (int u = 0; u < QT; ++u) {
                const float f = kf * qf[u];
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = sc[u][e >> 2][e & 3] * (SHAPED ? f : 1.0f);
                if (SHAPED) shape(u, x);
                const float mine = rounded(SHAPED ? max8(x) : max8(x) * f);
                raise_m(u, groups_max(mine));
                by[u] = raise_a(u, (int)groups_max(ceilf(fmaxf(mine - m[u], -16000.0f)) + (float)ve));
                // weights below 2^-60 of the largest come out 0 either way
                const int sh = max(14 + ve - a[u], -60);
                const float mm = m[u] - (float)sh;
                float w[8], sum = 0.0f;
                if (__any(fabsf(m[u]) > kFarScore)) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[e] = rounded(SHAPED ? x[e] : x[e] * f) - m[u] + (float)sh;
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[e] = SHAPED ? x[e] - mm : __builtin_fmaf(x[e], f, -mm);
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    w[e] = __builtin_amdgcn_exp2f(w[e]);
                    sum += w[e];
                }
                l[u] += __builtin_ldexpf(sum, -sh);
                weights(u, w);
            }
        } else {
#pragma unroll
            for (int u = 0; u < QT; ++u) {
                const uint32_t mine = whole ? ~0u : see[u] >> (4 * kg);
                float x[8], vf[8];
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) {
                    const v4f fk = *reinterpret_cast<const v4f *>(&im.kf[16 * kt + 4 * kg]);
                    const v4f fv = *reinterpret_cast<const v4f *>(&im.vf[16 * kt + 4 * kg]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int e = 4 * kt + i;
                        x[e] = sc[u][kt][i] * (fk[i] * qf[u]);
                        vf[e] = fv[i];
                    }
                }
                if (SHAPED) shape(u, x);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = rounded(mine >> (16 * (e >> 2) + (e & 3)) & 1 ? x[e] : -INFINITY);
                raise_m(u, groups_max(max8(x)));
                float w[8], sum = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    w[e] = __builtin_amdgcn_exp2f(x[e] - m[u]);
                    sum += w[e];
                    // a bad value row is NaN, for the rows that see it only
                    w[e] = mine >> (16 * (e >> 2) + (e & 3)) & 1 ? w[e] * vf[e] : 0.0f;
                }
                l[u] += sum;
                const float big = groups_max(max8(w));
                by[u] = raise_a(u, big > 0.0f ? __builtin_amdgcn_frexp_expf(big) : -16384);  // big < 2^that
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = __builtin_ldexpf(w[e], 14 - a[u]);
                weights(u, w);
            }
        }
#pragma unroll
        for (int u = 0; u < QT; ++u)
            if (__any(by[u] < 0)) {
                const float f = __builtin_ldexpf(1.0f, by[u]);
#pragma unroll
                for (int d = 0; d < 2 * C; ++d) o[u][d] *= f;
            }
        return true;
    };
    for (int step = t.from; step < t.to; ++step) {
        const int b = (step - t.from) & 1;
        if (IMG) {
            wait_vm<0>();   // this wave's part of the step's image is in LDS,
            lds_barrier();  // now everybody's is, and nobody reads the other buffer any more
            if (step + 1 < t.to) fetch(step + 1, b ^ 1);
        } else {
            __syncthreads();  // the producers' image likewise
        }
        if (!live_wave) continue;
        products(kScores, kAll, ims[b]);
        if (softmax(t.lo + step * kBlock, ims[b])) products(kSums, kScores, ims[b]);
    }

#pragma unroll
    for (int u = 0; u < QT; ++u) {
        const int local = (wave * QT + u) * 16 + r16, row = first_row + local;
        const float total = groups_sum(l[u]);
        if (row >= rows) continue;
        const bool whole_row = t.parts == 1;
        const int tok = tok0 + by_group(p, row - tok0 * p.group), h = g * p.group + row - tok * p.group;
        const float f = whole_row ? (total == 0.0f ? 0.0f : 1.0f / total) : 1.0f;
        float *dst = whole_row ? p.out + s * p.o_ss + tok * p.o_st + h * HD + 8 * kg
                               : pl.part + (share * kRows + local) * HD + 8 * kg;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                v4f x;
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = __builtin_ldexpf(o[u][2 * c + (i & 1)][2 * y + (i >> 1)] * f, a[u] - 14 - kTop);
                *reinterpret_cast<v4f *>(dst + 32 * c + 4 * y) = x;
            }
        if (kg != 0) continue;
        if (!whole_row) {
            pl.stat[share * kRows + local] = make_float2(m[u], total);
        } else if (p.lse) {
            p.lse[((size_t)s * p.n + tok) * p.heads + h] = (m[u] + __builtin_amdgcn_logf(total)) * 0.6931471805599453f;
        }
    }
}

// Few rows (at most 16 per sequence and KV head: one token, small trees).  What
// counts is how soon the cache is read: no wave waits for another, and K and V
// go from memory to the fp32 matrix instruction as they are loaded.
// Workgroup: 16 rows, four waves that take the share's blocks of 16 keys in
// turn, the next block's rows requested before this one's products:
//   K  lane 16·q + r: key r, dims 16c + 4q .. +3; product e of chunk c sums over
//      the dims 16c + 4q + e, as the query rows are held
//   V  lane 16·q + j: keys 4q .. 4q+3, dims 64d + 4j .. +3
// Scores and sums come out transposed, as in k_cache_attn; the waves' sums are
// joined in LDS.  Products, weights and sums are fp32 throughout.
// One token of 16 heads and 2 KV heads over 1,609 rows of 128: 8.4 us and 3.8 of
// the join, 3.3 MB; of 16 sequences 15 us, of 64 41 us (5.1 TB/s), of 256 143 us
// (5.9 TB/s).
constexpr int kFewKeys = 16;
constexpr int kFewWaves = 4;
template <int HD, bool TREE, bool SHAPED>
__global__ void __launch_bounds__(64 * kFewWaves, 2) k_cache_attn_few(CacheAttn p, AttnPlan pl) {
    constexpr int KC = HD / 16, D = HD / 64, kRows = 16, kPad = HD + 4, W = kFewWaves, kFewStep = W * kFewKeys;
    __shared__ __attribute__((aligned(16))) float s_o[W][kRows][kPad];
    __shared__ float s_m[W][kRows], s_l[W][kRows];
    __shared__ uint64_t s_bits[64];
    __shared__ int s_depth[64], s_lo, s_hi, s_lo_max, s_hi_min;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r16 = lane & 15, kg = lane >> 4;
    const int part = blockIdx.x, g = blockIdx.y, s = blockIdx.z;
    const size_t slot = (size_t)s * p.kvh + g;
    // nothing here waits for the lengths: the query rows, also of tokens that are not there
    v4f q[KC];
    const int in = min(r16, p.n * p.group - 1), row_tok = by_group(p, in), row_head = g * p.group + in - row_tok * p.group;
    const float *src = p.q + s * p.q_ss + row_tok * p.q_st + row_head * HD + 4 * kg;
#pragma unroll
    for (int c = 0; c < KC; ++c) q[c] = *reinterpret_cast<const v4f *>(src + 16 * c);
    int len = 0, count = p.n;
    if (TREE) {
        const SeqRows q = seq_rows(p, s);
        len = q.len;
        count = q.count;
    }
    const int rows = count * p.group;
    if (rows == 0) {
        if (pl.parts && part == 0 && tid == 0) pl.parts[slot] = 0;
        return;
    }
    AttnTile t{0, 0, 1, 0, 0};
    int all_lo = 0, all_hi;
    if (TREE) {
        t.hi = len + count;
        all_hi = len;
        if (wave == 0) {
            const uint64_t b = tree_bits(p.parents ? p.parents + (size_t)s * p.n : nullptr, p.n, lane);
            s_bits[lane] = b;
            s_depth[lane] = __popcll(b) - 1;
        }
        __syncthreads();
    } else if (p.begin) {
        if (tid == 0) {
            s_lo = s_hi_min = p.rows;
            s_hi = s_lo_max = 0;
        }
        __syncthreads();
        if (tid < count) {  // at most 16 tokens
            const int b = min(max(p.begin[tid], 0), p.rows), e = min(max(p.end[tid], 0), p.rows);
            if (b < e) {
                atomicMin(&s_lo, b);
                atomicMax(&s_hi, e);
            }
            atomicMax(&s_lo_max, b);
            atomicMin(&s_hi_min, e);
        }
        __syncthreads();
        t.lo = s_lo;
        t.hi = s_hi;
        all_lo = s_lo_max;
        all_hi = s_hi_min;
    } else {
        t.hi = p.rows0 + count;
        all_hi = p.rows0 + 1;
    }
    cut_tile(t, kFewStep, pl.splits, pl.least, part);
    if (part >= t.parts) return;
    if (pl.parts && part == 0 && tid == 0) pl.parts[slot] = t.parts;

    const float *kbase = p.k + s * p.k_ss + g * HD + 4 * kg, *vbase = p.v + s * p.v_ss + g * HD + 4 * r16;
    const int last = t.hi - 1;
    v4f kx[KC], vx[4][D];
    auto load = [&](int k0) {
        const float *ks = kbase + min(k0 + r16, last) * p.k_st;
#pragma unroll
        for (int c = 0; c < KC; ++c) kx[c] = *reinterpret_cast<const v4f *>(ks + 16 * c);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int d = 0; d < D; ++d)
                vx[i][d] = *reinterpret_cast<const v4f *>(vbase + min(k0 + 4 * kg + i, last) * p.v_st + 64 * d);
    };
    if (t.from < t.to) load(t.lo + t.from * kFewStep + wave * kFewKeys);

    const bool live = r16 < rows;
    const float slope = SHAPED ? slope_of(p, row_head) : 0.0f;
    int row_lo = 0, row_hi = 0, row_pos = 0;
    uint64_t bits = 0;
    if (TREE) {
        if (live) {
            row_hi = len;
            bits = s_bits[row_tok];
            if (SHAPED) row_pos = p.pos ? p.pos[slot * p.side + len + row_tok] : len + s_depth[row_tok];
        }
    } else if (live) {
        row_lo = p.begin ? min(max(p.begin[row_tok], 0), p.rows) : 0;
        row_hi = p.end ? min(max(p.end[row_tok], 0), p.rows) : p.rows0 + row_tok + 1;
        row_pos = p.rows0 + row_tok;
    }
    // the scale's power of two goes into the query rows (no bit changes): a score
    // that fp32 holds has products that it holds
    const uint32_t scale_bits = __float_as_uint(p.scale);
    const float power = __uint_as_float(scale_bits & 0x7f800000u), rest = __uint_as_float((scale_bits & 0x7fffffu) | 0x3f800000u);
#pragma unroll
    for (int c = 0; c < KC; ++c) q[c] *= power;
    const float scale = SHAPED ? rest : rest * kLog2e;
    const float inv_cap = SHAPED && p.cap > 0.0f ? 1.0f / p.cap : 0.0f, cap2 = SHAPED && p.cap > 0.0f ? p.cap * kLog2e : kLog2e;
    const int32_t *pos = TREE && SHAPED && p.pos ? p.pos + slot * p.side : nullptr;

    v4f o[D][4];  // [..][x][i]: dim 64d + 16·kg + 4i + x
    float m = kLowest, l = 0.0f;
    uint32_t sees_bad = 0;
#pragma unroll
    for (int d = 0; d < D; ++d)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[d][x] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
    for (int step = t.from; step < t.to; ++step) {
        const int k0 = t.lo + step * kFewStep + wave * kFewKeys;
        v4f a[4] = {};
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) a[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(kx[c][e], q[c][e], a[e], 0, 0, 0);
        const v4f sc = (a[0] + a[1]) + (a[2] + a[3]);
        v4f v[4][D];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int d = 0; d < D; ++d) v[i][d] = vx[i][d];
        if (step + 1 < t.to) load(k0 + kFewStep);
        const bool whole = k0 >= all_lo && k0 + kFewKeys <= all_hi;
        uint32_t bad = 0;  // keys whose value row is not finite, where not every row sees all keys
        if (!whole) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t top = 0;
#pragma unroll
                for (int d = 0; d < D; ++d)
                    top = umax3(top, max(abs_bits(v[i][d][0]), abs_bits(v[i][d][1])), max(abs_bits(v[i][d][2]), abs_bits(v[i][d][3])));
                const uint64_t b = __ballot(top >= 0x7f800000u);
                const bool here = b >> (16 * kg) & 0xffff;
                if (here)
#pragma unroll
                    for (int d = 0; d < D; ++d) v[i][d] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
                bad |= here ? 1u << i : 0u;
            }
        }
        uint32_t see = 0xf;  // of the lane's four keys
        if (!whole) {
            const int n1 = min(max(row_hi - k0, 0), 16), n0 = min(max(row_lo - k0, 0), 16);
            uint32_t w = ((1u << n1) - 1) & ~((1u << n0) - 1);
            if (TREE) {
                const int off = k0 - len;  // the block's first key among the drafted ones
                if (off > -16 && off < 64) w |= (uint32_t)(off >= 0 ? bits >> off : bits << -off);
            }
            see = w >> (4 * kg) & 0xf;
        }
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = sc[i] * scale;
        if (SHAPED) {
            if (p.cap > 0.0f) {
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] *= inv_cap;
                tanh_all(x);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = k0 + 4 * kg + i;
                int at = key;
                if (TREE) at = pos ? pos[min(key, last)] : (key < len ? key : len + s_depth[min(key - len, 63)]);
                x[i] = fmaf(x[i], cap2, -slope * distance(row_pos, at));
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = rounded(see >> i & 1 ? x[i] : -INFINITY);
        const float top = groups_max(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
        if (__any(top > m)) {
            const float mn = top > m ? top : m;
            const float f = __builtin_amdgcn_exp2f(m - mn);
            l *= f;
#pragma unroll
            for (int d = 0; d < D; ++d)
#pragma unroll
                for (int y = 0; y < 4; ++y) o[d][y] *= f;
            m = mn;
        }
        sees_bad |= bad & see;
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = __builtin_amdgcn_exp2f(x[i] - m);
            l += w[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int d = 0; d < D; ++d)
#pragma unroll
                for (int y = 0; y < 4; ++y)
                    o[d][y] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[i][d][y], w[i], o[d][y], 0, 0, 0);
    }

    if (groups_umax(sees_bad))  // the sums alone: the denominator is of the scores
#pragma unroll
        for (int d = 0; d < D; ++d)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[d][x] = (v4f){NAN, NAN, NAN, NAN};
    const float total = groups_sum(l);
    if (kg == 0) {
        s_m[wave][r16] = m;
        s_l[wave][r16] = total;
    }
#pragma unroll
    for (int d = 0; d < D; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<v4f *>(&s_o[wave][r16][64 * d + 16 * kg + 4 * i]) = (v4f){o[d][0][i], o[d][1][i], o[d][2][i], o[d][3][i]};
    __syncthreads();
    for (int i = tid; i < rows * (HD / 4); i += 64 * W) {
        const int row = i / (HD / 4), at = i % (HD / 4) * 4;
        float mm = s_m[0][row], total = 0.0f;
#pragma unroll
        for (int w = 1; w < W; ++w) mm = fmaxf(mm, s_m[w][row]);
        v4f x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float f = __builtin_amdgcn_exp2f(s_m[w][row] - mm);
            total = fmaf(s_l[w][row], f, total);
            x += *reinterpret_cast<const v4f *>(&s_o[w][row][at]) * f;
        }
        if (t.parts > 1) {
            *reinterpret_cast<v4f *>(pl.part + ((slot * pl.splits + part) * kRows + row) * HD + at) = x;
            if (at == 0) pl.stat[(slot * pl.splits + part) * kRows + row] = make_float2(mm, total);
            continue;
        }
        const int tok = by_group(p, row), h = g * p.group + row - tok * p.group;
        *reinterpret_cast<v4f *>(p.out + s * p.o_ss + tok * p.o_st + h * HD + at) = x * (total == 0.0f ? 0.0f : 1.0f / total);
        if (p.lse && at == 0)
            p.lse[((size_t)s * p.n + tok) * p.heads + h] = (mm + __builtin_amdgcn_logf(total)) * 0.6931471805599453f;
    }
}

// Joins the shares of the tiles that were cut: HD / 4 lanes of float4 per row;
// rows of uncut tiles are done already.  The lanes first take the shares'
// maxima and denominators, one or a few each, then all walk the shares with
// the factors that those give, kJoin loads in flight.
// kSub groups of lanes share a row's sums where rows are few (one token over
// 6,400 rows, 64 shares: 8.9 us by one group, 5.3 by four; of 128 rows a tile
// 9.6 by one, 19.4 by four).
constexpr int kJoin = 8;
template <int HD, int kRows, int kSub>
__global__ void __launch_bounds__(256) k_cache_attn_join(CacheAttn p, AttnPlan pl) {
    constexpr int kLanes = HD / 4, kPer = 256 / kLanes / kSub, kOwn = kMaxShares / kLanes;
    const int per_tile = kRows / kPer;
    const int tile = blockIdx.x / per_tile, local = blockIdx.x % per_tile * kPer + threadIdx.x / kLanes / kSub;
    const int sub = threadIdx.x / kLanes % kSub;
    const int g = blockIdx.y, s = blockIdx.z, lane = threadIdx.x % kLanes;
    const size_t slot = ((size_t)s * p.kvh + g) * pl.tiles + tile;
    const int parts = pl.cuts ? pl.cuts[tile].parts : pl.parts[slot];
    const size_t first = pl.cuts ? (size_t)g * pl.max_jobs + pl.cuts[tile].first : slot * pl.splits;
    const int rows = (p.lens ? seq_rows(p, s).count : p.n) * p.group, row = tile * kRows + local;
    if (parts < 2 || (kSub == 1 && row >= rows)) return;  // the same for a row's lanes, or for the workgroup
    const float2 *st = pl.stat + first * kRows + local;
    const float *src = pl.part + (first * kRows + local) * HD + 4 * lane;
    float2 mine[kOwn];
    float m = kLowest;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
        const int x = i * kLanes + lane;
        mine[i] = x < parts ? st[(size_t)x * kRows] : make_float2(kLowest, 0.0f);
        m = fmaxf(m, mine[i].x);
    }
#pragma unroll
    for (int o = kLanes / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, kLanes));
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
        mine[i].x = __builtin_amdgcn_exp2f(mine[i].x - m);
        total = fmaf(mine[i].y, mine[i].x, total);
    }
#pragma unroll
    for (int o = kLanes / 2; o; o >>= 1) total += __shfl_xor(total, o, kLanes);
    v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i0 = sub; i0 < parts; i0 += kJoin * kSub) {
        v4f x[kJoin];
#pragma unroll
        for (int i = 0; i < kJoin; ++i) x[i] = *reinterpret_cast<const v4f *>(src + (size_t)min(i0 + i * kSub, parts - 1) * kRows * HD);
#pragma unroll
        for (int i = 0; i < kJoin; ++i) {
            const int at = i0 + i * kSub;
            float f = mine[0].x;
#pragma unroll
            for (int y = 1; y < kOwn; ++y) f = at / kLanes == y ? mine[y].x : f;
            f = __shfl(f, at % kLanes, kLanes);
            if (at < parts)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[c] = fmaf(x[i][c], f, acc[c]);
        }
    }
    if (kSub > 1) {
        __shared__ v4f s_acc[256];
        s_acc[threadIdx.x] = acc;
        __syncthreads();
        if (sub) return;
#pragma unroll
        for (int i = 1; i < kSub; ++i) acc += s_acc[threadIdx.x + i * kLanes];
    }
    if (row >= rows) return;
    const int tok = row / p.group, h = g * p.group + row % p.group;
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    *reinterpret_cast<v4f *>(p.out + s * p.o_ss + tok * p.o_st + h * HD + 4 * lane) = acc * inv;
    if (p.lse && lane == 0)
        p.lse[((size_t)s * p.n + tok) * p.heads + h] = (m + __builtin_amdgcn_logf(total)) * 0.6931471805599453f;
}

// The weights of cache rows.  Workgroup: 64 rows (MANY·32) of one sequence and
// KV head, their halves in four waves' registers throughout; the query rows
// (token, head) pass through LDS 64 at a time, laid out as the matrix
// instructions take them.  A lane sums its query row of each 16 for four keys;
// the sum over a key's 16 lanes ends the kernel, so the order of every sum is
// fixed.
//
// Up to 64 query rows there is one step, and four waves of 16 keys lay the rows
// out themselves (16 single tokens of 16 heads over 1,610 rows: 11 us, the keys
// at 2.4 TB/s).  For more (MANY), four more waves do so in two buffers, two
// steps ahead of their use; the others hold 16·MANY keys each and take every
// other 32 query rows.
constexpr int kWRows = 64;
template <int HD>
struct WeightRows {
    uint8_t q[4 * (HD / 32) * 2 * 1024];  // [16-row tile][32-dim chunk][half] lane l = 16·q + r: row r, dims 32c + 8q .. +7
    float qf[kWRows], lse[kWRows];        // scale; log2 of the denominator, +inf for rows that do not count
    float slope[kWRows];
    int pos[kWRows];
    uint64_t see[kWRows];
};
template <int HD, bool SHAPED, int MANY>
__global__ void __launch_bounds__(MANY ? 512 : 256, 2) k_cache_weights(CacheAttn p) {
    constexpr int C = HD / 32, KT = MANY ? MANY : 1, kKeys = MANY ? 32 * MANY : 64;
    __shared__ __attribute__((aligned(16))) WeightRows<HD> steps[MANY ? 2 : 1];
    __shared__ float s_sum[kKeys];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, kg = lane >> 4;
    const int g = blockIdx.y, s = blockIdx.z, key0 = p.key0 + blockIdx.x * kKeys;
    const SeqRows q = seq_rows(p, s);
    const int end = q.len + q.count, rows = q.count * p.group;
    if (key0 >= end || q.count == 0) return;
    const uint64_t take = p.take ? p.take[s] : ~0ull;
    const int32_t *pos = SHAPED && p.pos ? p.pos + ((size_t)s * p.kvh + g) * p.side : nullptr;
    uint64_t mine = 0;

    // 16 query rows as a wave loads and lays them out
    struct Row {
        float x[C][8], lse;
        int pos;
    };
    auto load = [&](Row &r, int first) {
        const int row = min(first + r16, rows - 1), tok = by_group(p, row), h = g * p.group + row - tok * p.group;
        const float *src = p.q + s * p.q_ss + tok * p.q_st + h * HD + 8 * kg;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const v4f a = *reinterpret_cast<const v4f *>(src + 32 * c), b = *reinterpret_cast<const v4f *>(src + 32 * c + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                r.x[c][i] = a[i];
                r.x[c][4 + i] = b[i];
            }
        }
        r.lse = p.lse[((size_t)s * p.n + tok) * p.heads + h];
        if (SHAPED) r.pos = pos ? pos[q.len + tok] : 0;
    };
    auto put = [&](const Row &r, WeightRows<HD> &to, int first, int tile) {
        const int row = min(first + r16, rows - 1), tok = by_group(p, row), local = 16 * tile + r16;
        if (first < rows) {
            uint32_t top = 0;
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < 8; i += 2) top = umax3(top, abs_bits(r.x[c][i]), abs_bits(r.x[c][i + 1]));
            const int e = row_exp(groups_umax(top));
            v8h hi[C], lo[C];
            split_row<C>(r.x, e, hi, lo);
#pragma unroll
            for (int c = 0; c < C; ++c) {
                *reinterpret_cast<v8h *>(to.q + ((tile * C + c) * 2) * 1024 + lane * 16) = hi[c];
                *reinterpret_cast<v8h *>(to.q + ((tile * C + c) * 2 + 1) * 1024 + lane * 16) = lo[c];
            }
            const uint64_t b = __shfl((unsigned long long)mine, tok);
            if (kg == 0) {
                to.qf[local] = pow2(e - kTop) * (SHAPED ? p.scale : p.scale * kLog2e);
                to.see[local] = b;
                if (SHAPED) {
                    to.slope[local] = slope_of(p, g * p.group + row - tok * p.group);
                    to.pos[local] = pos ? r.pos : q.len + __popcll(b) - 1;
                }
            }
        }
        const bool live = first + r16 < rows && (take >> tok & 1) && r.lse != -INFINITY;
        if (kg == 0) to.lse[local] = live ? r.lse * kLog2e : INFINITY;
    };
    if (MANY && wave >= 4) {
        const int mine16 = 16 * (wave - 4);
        Row r[2];
        load(r[0], mine16);
        load(r[1], kWRows + mine16);
        mine = tree_bits(p.parents ? p.parents + (size_t)s * p.n : nullptr, p.n, lane);
        for (int row0 = 0; row0 < rows; row0 += 2 * kWRows) {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int at = row0 + b * kWRows;
                if (at >= rows) break;
                put(r[b], steps[b], at + mine16, wave - 4);
                if (at + 2 * kWRows < rows) load(r[b], at + 2 * kWRows + mine16);
                __syncthreads();  // the step is there, and the one before it done with
            }
        }
        __syncthreads();  // the others' last
        return;
    }

    Row own;
    if (!MANY) load(own, 16 * wave);
    const int first_key = key0 + 16 * KT * (MANY ? wave & 1 : wave), half = MANY ? wave >> 1 : 0;
    // a lane writes at most one sum; what it adds to is on its way
    const int out_key = first_key + (r16 < 4 * KT ? 16 * (r16 >> 2) + 4 * kg + (r16 & 3) : kKeys);
    float *out = p.weights + ((size_t)s * p.kvh + g) * p.side + out_key;
    const bool writes = half == 0 && out_key < min(first_key + 16 * KT, end);
    const float before = writes ? *out : 0.0f;
    v8h kh[KT][C], kl[KT][C];
    float kf[KT][4], x[KT][C][8];
    int kpos[KT][4];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
        const float *src = p.k + s * p.k_ss + min(first_key + 16 * kt + r16, end - 1) * p.k_st + g * HD + 8 * kg;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const v4f a = *reinterpret_cast<const v4f *>(src + 32 * c), b = *reinterpret_cast<const v4f *>(src + 32 * c + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[kt][c][i] = a[i];
                x[kt][c][4 + i] = b[i];
            }
        }
    }
    mine = tree_bits(p.parents ? p.parents + (size_t)s * p.n : nullptr, p.n, lane);
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 8; i += 2) top = umax3(top, abs_bits(x[kt][c][i]), abs_bits(x[kt][c][i + 1]));
        const int e = row_exp(groups_umax(top));
        split_row<C>(x[kt], e, kh[kt], kl[kt]);
        const float f = pow2(e - kTop);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int key = first_key + 16 * kt + 4 * kg + i;
            kf[kt][i] = __shfl(f, 4 * kg + i);
            kpos[kt][i] = key;
            if (SHAPED) {
                const int depth = __popcll(__shfl((unsigned long long)mine, min(max(key - q.len, 0), 63))) - 1;
                if (pos) kpos[kt][i] = pos[min(key, end - 1)];
                else if (key >= q.len) kpos[kt][i] = q.len + depth;
            }
        }
    }
    const float inv_cap = SHAPED && p.cap > 0.0f ? 1.0f / p.cap : 0.0f, cap2 = SHAPED && p.cap > 0.0f ? p.cap * kLog2e : kLog2e;
    const bool drafts = key0 + kKeys > q.len;  // some key is a drafted token's
    float acc[KT][4] = {};
    for (int row0 = 0; row0 < rows; row0 += kWRows) {
        if (!MANY) put(own, steps[0], 16 * wave, wave);
        __syncthreads();
        const WeightRows<HD> &in = steps[MANY ? row0 / kWRows & 1 : 0];
        for (int pair = half; row0 + 32 * pair < rows && pair < 2; pair += MANY ? 2 : 1) {
            v4f sc[2][KT];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) sc[t][kt] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < C; ++c) {
                v8h qh[2], ql[2];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    qh[t] = *reinterpret_cast<const v8h *>(in.q + (((2 * pair + t) * C + c) * 2) * 1024 + lane * 16);
                    ql[t] = *reinterpret_cast<const v8h *>(in.q + (((2 * pair + t) * C + c) * 2 + 1) * 1024 + lane * 16);
                }
#pragma unroll
                for (int x = 0; x < 3; ++x)
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int kt = 0; kt < KT; ++kt)
                            sc[t][kt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x == 0 ? kl[kt][c] : kh[kt][c], x == 1 ? ql[t] : qh[t],
                                                                               sc[t][kt], 0, 0, 0);
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int local = 32 * pair + 16 * t + r16;
                const float qf = in.qf[local], lse = in.lse[local];
                const uint64_t see = drafts ? in.see[local] : 0;
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    float y[4];
                    if (SHAPED) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) y[i] = sc[t][kt][i] * (kf[kt][i] * qf);
                        if (p.cap > 0.0f) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) y[i] *= inv_cap;
                            tanh_all(y);
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            y[i] = fmaf(y[i], cap2, -in.slope[local] * distance(in.pos[local], kpos[kt][i])) - lse;
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) y[i] = fmaf(sc[t][kt][i], kf[kt][i] * qf, -lse);
                    }
                    uint32_t take4 = lse != INFINITY ? 0xf : 0;  // which of the lane's keys the row sees
                    if (drafts) {
                        const int off = first_key + 16 * kt + 4 * kg - q.len, up = min(max(off, 0), 63), down = min(max(-off, 0), 4);
                        take4 &= (off < 64 ? (uint32_t)(see >> up) << down : 0u) | ((1u << down) - 1);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[kt][i] += __builtin_amdgcn_exp2f(take4 >> i & 1 ? y[i] : -INFINITY);
                }
            }
        }
    }
    float sum = 0.0f;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float a = acc[kt][i];
            a += xchg<XQ1>(a);
            a += xchg<XQ2>(a);
            a += xchg<XM8>(a);
            a += xchg<XM16>(a);
            sum = r16 == 4 * kt + i ? a : sum;
        }
    if (MANY) {
        if (half && r16 < 4 * KT) s_sum[out_key - key0] = sum;
        __syncthreads();
        if (writes) sum += s_sum[out_key - key0];
    }
    if (writes) *out = before + sum;
}

// ---------------------------------------------------------------------------
// selection and compaction
// ---------------------------------------------------------------------------
struct CacheSelect {
    const float *weights;
    const int32_t *lens;
    int32_t *kept, *counts;
    int64_t side;
    int kvh, max_rows, budget, sinks, recent;
};

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;

// weights in the order of their floats; NaN below everything, -0 with 0
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0u;
    const uint32_t b = __float_as_uint(w + 0.0f);
    return (b & 0x80000000u ? ~b : b | 0x80000000u);
}

// One workgroup per (KV head, cache).  The need-th largest key of the rows
// between sinks and recent by three histogram passes over 11, 11 and 10 of its
// bits (integer counts: the order of the atomics does not matter; eleven bits
// hold two of the mantissa, which spreads weights of few exponents over the
// bins; a pass whose bin is taken whole is the last, as the second mostly is
// among weights that differ), then one pass that writes the kept rows in order:
// a wave owns 64·KPT consecutive rows of a tile, so a row's place is a count of
// ballots.  KPT rows per thread and tile; a cache of one tile is read once, its
// keys stay in registers (8,192 rows in a buffer of 32,768: 15.3 us, 18.1 read by
// each pass).  36 selections, one workgroup each: 6.5 us of 1,609 rows, 10.6 of
// 8,192, nearly all of it the chain of load, passes and barriers.
template <int KPT>
__global__ void __launch_bounds__(kSelThreads) k_cache_select(CacheSelect p) {
    constexpr int kTile = kSelThreads * KPT, kBins = 2048;
    __shared__ int hist[kBins];
    __shared__ int s_bin, s_need, s_all;
    __shared__ int s_eq[kSelWaves], s_gt[kSelWaves];
    const int g = blockIdx.x, c = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float *w = p.weights + ((size_t)c * p.kvh + g) * p.side;
    const bool early = p.max_rows <= kTile;  // one tile holds any cache: its weights wait for no length
    float x[KPT];
    auto load = [&](int tile) {
#pragma unroll
        for (int i = 0; i < KPT; ++i)  // all on their way at once
            x[i] = w[min(tile * kTile + (wave * KPT + i) * 64 + lane, p.max_rows - 1)];
    };
    if (early) load(0);
    const int len = min(max(p.lens[c], 0), p.max_rows);
    int32_t *kept = p.kept + ((size_t)c * p.kvh + g) * p.budget;
    if (g == 0 && tid == 0) p.counts[c] = min(len, p.budget);
    if (len <= p.budget) {
        for (int j = tid; j < len; j += kSelThreads) kept[j] = j;
        return;
    }
    const int first = p.sinks, last = len - p.recent;  // candidates [first, last): more than `need` of them
    int need = p.budget - p.sinks - p.recent;
    const int tiles = (len + kTile - 1) / kTile;
    uint32_t key[KPT];
    auto keys = [&] {
#pragma unroll
        for (int i = 0; i < KPT; ++i) key[i] = weight_key(x[i]);
    };
    const bool one = tiles == 1;  // this cache's keys stay in registers
    if (one && !early) load(0);
    if (one) keys();
    uint32_t prefix = 0, mask = 0;
    if (need > 0)
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bins = pass == 2 ? 1024 : kBins;
            hist[tid] = 0;
            hist[tid + kSelThreads] = 0;
            __syncthreads();
            for (int tile = 0; tile < tiles; ++tile) {
                if (!one) {
                    load(tile);
                    keys();
                }
#pragma unroll
                for (int i = 0; i < KPT; ++i) {
                    const int j = tile * kTile + (wave * KPT + i) * 64 + lane;
                    if ((j >= first) & (j < last) & ((key[i] & mask) == prefix)) atomicAdd(&hist[key[i] >> shift & (bins - 1)], 1);
                }
            }
            __syncthreads();
            // thread t: bins 2047 - 2t and 2046 - 2t, counts above them by a scan
            const int n0 = hist[kBins - 1 - 2 * tid], n1 = hist[kBins - 2 - 2 * tid];
            int upto = n0 + n1;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int x = __shfl_up(upto, o);
                if (lane >= o) upto += x;
            }
            if (lane == 63) s_gt[wave] = upto;
            __syncthreads();
            int above = upto - n0 - n1;
            for (int x = 0; x < kSelWaves; ++x) above += x < wave ? s_gt[x] : 0;
            if (above < need && above + n0 + n1 >= need) {  // one thread
                const bool lower = above + n0 < need;
                s_bin = kBins - 1 - 2 * tid - (lower ? 1 : 0);
                s_need = need - above - (lower ? n0 : 0);
                s_all = s_need == (lower ? n1 : n0);
            }
            __syncthreads();
            prefix |= (uint32_t)s_bin << shift;
            mask |= (uint32_t)(bins - 1) << shift;
            need = s_need;  // how many keys equal to prefix are taken, after the last pass
            if (s_all && prefix) {  // the whole bin is taken: every key above the one below it
                prefix -= 1;
                need = 0;
                break;
            }
        }
    const bool some = p.budget > p.sinks + p.recent;
    int done = 0, eq_done = 0;  // rows written, equal keys met
    for (int tile = 0; tile < tiles; ++tile) {
        if (!one) {
            load(tile);
            keys();
        }
        int gt = 0, eq = 0;
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            const int j = tile * kTile + (wave * KPT + i) * 64 + lane;
            const bool cand = (j >= first) & (j < last);  // selects, not branches: 8,192 rows 12.0 -> 10.7 us
            gt += __popcll(__ballot((j < len) & (!cand | (some & (key[i] > prefix)))));
            eq += __popcll(__ballot(cand & some & (key[i] == prefix)));
        }
        if (lane == 0) {
            s_gt[wave] = gt;
            s_eq[wave] = eq;
        }
        __syncthreads();
        int at = done, eqs = eq_done, all_gt = 0, all_eq = 0;
        for (int x = 0; x < kSelWaves; ++x) {
            if (x < wave) {
                at += s_gt[x];
                eqs += s_eq[x];
            }
            all_gt += s_gt[x];
            all_eq += s_eq[x];
        }
        at += min(eqs, need) - min(eq_done, need);
        done += all_gt + min(eq_done + all_eq, need) - min(eq_done, need);
        eq_done += all_eq;
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            const int j = tile * kTile + (wave * KPT + i) * 64 + lane;
            const bool cand = (j >= first) & (j < last);
            const bool is_eq = cand & some & (key[i] == prefix);
            const uint64_t below = (1ull << lane) - 1, be = __ballot(is_eq);
            const bool keep = ((j < len) & (!cand | (some & (key[i] > prefix)))) |
                              (is_eq & (eqs + __popcll(be & below) < need));
            const uint64_t bk = __ballot(keep);
            if (keep) kept[at + __popcll(bk & below)] = j;
            at += __popcll(bk);
            eqs += __popcll(be);
        }
        __syncthreads();
    }
}

struct CacheKeep {
    const float *src[2];  // K, V
    float *dst[2];
    const float *weights;
    float *weights_out;
    const int32_t *pos, *rows, *counts, *first;
    int32_t *pos_out;
    int64_t src_cs[2], src_st[2], dst_cs[2], dst_st[2], side, side_out;
    int kvh, max_keep, per_head, max_rows, max_rows_out;
};

constexpr int kKeepThreads = 256;
constexpr int kKeepRows = 64;  // rows that a workgroup of k_cache_keep moves
constexpr int kKeepSlab = 16;  // floats of a row that a workgroup of k_cache_keep_slabs moves

// every wave's loads have arrived
__device__ __forceinline__ void loads_done() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

struct KeepRange {
    int first, count;
    const int32_t *rows;
};
__device__ __forceinline__ KeepRange keep_range(const CacheKeep &p, int c, int g) {
    KeepRange r;
    r.first = p.first ? min(max(p.first[c], 0), p.max_rows_out) : 0;
    r.count = min(max(p.counts[c], 0), min(p.max_keep, p.max_rows_out - r.first));
    r.rows = p.rows + (p.per_head ? (size_t)c * p.kvh + g : (size_t)c) * p.max_keep;
    return r;
}
// the source row of list entry i, read whatever the count is (i < max_keep)
template <bool INPLACE>
__device__ __forceinline__ int keep_source(const CacheKeep &p, int listed, int first, int i) {
    return min(max(listed, INPLACE ? min(first + i, p.max_rows - 1) : 0), p.max_rows - 1);
}

// weights and positions of list entries from, from + step, ... chunks of 256
// (their numbers pass 31 bits behind the longest lists)
template <bool INPLACE>
__device__ __forceinline__ void keep_side(const CacheKeep &p, const KeepRange &r, int c, int g, int from, int step) {
    const size_t in = ((size_t)c * p.kvh + g) * p.side, out = ((size_t)c * p.kvh + g) * p.side_out + r.first;
    const int64_t stride = (int64_t)step * kKeepThreads;
    for (int64_t b = (int64_t)from * kKeepThreads; b < r.count; b += stride) {
        const int64_t i = b + threadIdx.x;
        float w = 0.0f;
        int32_t at = 0;
        if (i < r.count) {
            const int j = keep_source<INPLACE>(p, r.rows[i], r.first, (int)i);
            if (p.weights) w = p.weights[in + j];
            if (p.pos) at = p.pos[in + j];
        }
        if (INPLACE) loads_done();
        if (i < r.count) {
            if (p.weights) p.weights_out[out + i] = w;
            if (p.pos) p.pos_out[out + i] = at;
        }
    }
    if (INPLACE) __syncthreads();
    if (p.weights)
        for (int64_t i = r.count + (int64_t)from * kKeepThreads + threadIdx.x; r.first + i < p.max_rows_out; i += stride)
            p.weights_out[out + i] = 0.0f;
}

// Workgroup: 64 listed rows of K or V of one KV head and cache (x even, odd),
// HD / 4 lanes a row, all loads before the first store; or (the last x's) their
// weights and positions.  In place for lists of at most 64 rows, which one
// workgroup holds whole.  A grid has `chunks` of a list's all_chunks, from chunk0
// on.  2,048 rows of 18 caches with two KV heads into others:
// 151 MB read and written in 35.7 us, 4.2 TB/s of a large copy's 4.8; 768 rows,
// 57 MB, in 11.6 us, 4.9 TB/s.
template <int HD, bool INPLACE>
__global__ void __launch_bounds__(kKeepThreads) k_cache_keep(CacheKeep p, int chunk0, int chunks, int all_chunks) {
    constexpr int kLanes = HD / 4, kStep = kKeepThreads / kLanes, kUnroll = kKeepRows / kStep;
    const int g = blockIdx.y, c = blockIdx.z, tid = threadIdx.x, x = blockIdx.x;
    const KeepRange r = keep_range(p, c, g);
    if (x >= 2 * chunks) {
        keep_side<INPLACE>(p, r, c, g, chunk0 + x - 2 * chunks, all_chunks);
        return;
    }
    const int which = x & 1, i0 = (chunk0 + (x >> 1)) * kKeepRows + tid / kLanes;
    int j[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) j[u] = r.rows[min(i0 + u * kStep, p.max_keep - 1)];
    const float *src = p.src[which] + c * p.src_cs[which] + g * HD + tid % kLanes * 4;
    float *dst = p.dst[which] + c * p.dst_cs[which] + g * HD + tid % kLanes * 4;
    v4f v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)  // entries behind the count: a row that is there, not stored
        v[u] = *reinterpret_cast<const v4f *>(src + keep_source<INPLACE>(p, j[u], r.first, min(i0 + u * kStep, p.max_keep - 1)) * p.src_st[which]);
    if (INPLACE) loads_done();
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
        if (i0 + u * kStep < r.count) *reinterpret_cast<v4f *>(dst + (r.first + i0 + u * kStep) * p.dst_st[which]) = v[u];
}

// Longer lists in place.  Workgroup: one slab of 16 columns of K or V of one KV
// head and cache, or (the last x) its weights and positions; it walks the list
// in chunks: all loads of a chunk, then its stores.  The list ascends with
// rows[i] >= first + i, so what a later chunk reads lies at or behind its own
// places, past everything written before it, and only the chunk's own loads
// have to end (the barrier) before its stores.  18 caches with two KV heads,
// 8,192 -> 2,048 rows: 48 us, 3.1 TB/s read and written (elsewhere, by
// k_cache_keep, 36 us); 1,609 -> 768 rows 16.7 us, 3.4 TB/s (11.2).
template <int HD>
__global__ void __launch_bounds__(kKeepThreads) k_cache_keep_slabs(CacheKeep p) {
    constexpr int kSlabs = HD / kKeepSlab, kLanes = kKeepSlab / 4, kStep = kKeepThreads / kLanes, kUnroll = 8;
    const int g = blockIdx.y, c = blockIdx.z, tid = threadIdx.x, x = blockIdx.x;
    const KeepRange r = keep_range(p, c, g);
    if (x == 2 * kSlabs) {
        keep_side<true>(p, r, c, g, 0, 1);
        return;
    }
    const int which = x / kSlabs, at = x % kSlabs * kKeepSlab + tid % kLanes * 4;
    const float *src = p.src[which] + c * p.src_cs[which] + g * HD + at;
    float *dst = p.dst[which] + c * p.dst_cs[which] + g * HD + at;
    for (int b = tid / kLanes; b - tid / kLanes < r.count; b += kStep * kUnroll) {
        v4f v[kUnroll];
        int j[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) j[u] = r.rows[min(b + u * kStep, p.max_keep - 1)];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            v[u] = *reinterpret_cast<const v4f *>(src + keep_source<true>(p, j[u], r.first, min(b + u * kStep, p.max_keep - 1)) * p.src_st[which]);
        loads_done();
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            if (b + u * kStep < r.count) *reinterpret_cast<v4f *>(dst + (r.first + b + u * kStep) * p.dst_st[which]) = v[u];
    }
}

}  // namespace pocr
