// qcache.hpp — kernels of the K/V caches held in 4 or 8 bits: rows normed,
// rotated and appended, quantised as they are written, read back, and the
// attention over them.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "cache_ops.hpp"

namespace pocr {

// ---------------------------------------------------------------------------
// rows of a cache
// ---------------------------------------------------------------------------

// One cache: rows of a (sequence, KV head) lie together.
struct QRows {
    uint8_t *codes[2];    // K, V
    _Float16 *params[2];
    int64_t seq_rows;     // rows from sequence to sequence
    int kvh, capacity;
};

template <int HD, int BITS>
struct QFormat {
    static constexpr int kGroups = HD / 64;           // of 64 elements
    static constexpr int kCodes = HD * BITS / 8;      // bytes of a row's codes
    static constexpr int kParams = 2 * kGroups;       // fp16 numbers: steps, midpoints
    static constexpr int kHalf = 1 << (BITS - 1);     // codes from -kHalf to kHalf - 1, stored as code + kHalf
    static constexpr int kLanes = HD / 8;             // lanes of 8 neighbouring elements
};

// A lane's elements: HD / 8 lanes hold a row of a head, lane i elements 4i .. +3 and
// HD / 2 + 4i .. +3.  A wave's loads and stores are then whole lines, the pairs of a
// rotation of the whole head lie in one lane, and so does V's word of eight codes.

// where the codes of elements 8b .. 8b+7 of a K row begin
template <int HD, int BITS>
__device__ __forceinline__ int k_place(int b) {
    const int c = b >> 2, u = b & 3;  // elements 32c + 8u
    return BITS == 4 ? 4 * (u * (HD / 32) + c) : 64 * (c >> 1) + 16 * u + 8 * (c & 1);
}

// lane i's elements of a K (V) row: mid + step * code, one rounding
template <int HD, int BITS, bool V>
__device__ __forceinline__ void q_values(const uint8_t *codes, const _Float16 *params, int i, float (&x)[8]) {
    using F = QFormat<HD, BITS>;
    float step[2], mid[2];
    if constexpr (HD == 128) {
        const v4h y = *reinterpret_cast<const v4h *>(params);
        step[0] = y[0], step[1] = y[1], mid[0] = y[2], mid[1] = y[3];
    } else {
        const v2h y = *reinterpret_cast<const v2h *>(params);
        step[0] = step[1] = y[0], mid[0] = mid[1] = y[1];
    }
    const int odd = i & 1;
    int c[8];
    if constexpr (V && HD == 128) {
        uint32_t w[BITS / 4];
        if constexpr (BITS == 4) w[0] = *reinterpret_cast<const uint32_t *>(codes + 4 * i);
        else *reinterpret_cast<uint2 *>(w) = *reinterpret_cast<const uint2 *>(codes + 8 * i);
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e] = BITS == 4 ? w[0] >> 4 * e & 15 : w[e >> 2] >> 8 * (e & 3) & 255;
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // half a word of eight (half of 8 bytes)
            const int b = h * (HD / 16) + (i >> 1);
            if constexpr (BITS == 4) {
                const uint32_t w = *reinterpret_cast<const uint32_t *>(codes + (V ? 4 * b : k_place<HD, BITS>(b))) >> (V ? 16 * odd : 8 * odd);
#pragma unroll
                for (int e = 0; e < 4; ++e) c[4 * h + e] = w >> 4 * (V ? e : (e >> 1) + 4 * (e & 1)) & 15;
            } else {
                const uint32_t w = *reinterpret_cast<const uint32_t *>(codes + (V ? 8 * b : k_place<HD, BITS>(b)) + 4 * odd);
#pragma unroll
                for (int e = 0; e < 4; ++e) c[4 * h + e] = w >> 8 * e & 255;
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmaf((float)(c[e] - F::kHalf), step[e >> 2], mid[e >> 2]);
}

// midpoint and step of a group whose elements are lo to hi, and 1 / step
template <int BITS>
__device__ __forceinline__ void q_grid(float lo, float hi, _Float16 &step, _Float16 &mid, double &inv) {
    constexpr double kUp = (1 << (BITS - 1)) - 1, kDown = 1 << (BITS - 1);
    // `rounded`: to fp32 first, which the compiler would skip
    mid = (_Float16)rounded((float)((kUp * (double)lo + kDown * (double)hi) * (1.0 / (kUp + kDown))));
    const double need = fmax(((double)hi - (double)mid) * (1.0 / kUp), ((double)mid - (double)lo) * (1.0 / kDown));
    step = (_Float16)rounded((float)need);
    if ((double)step < need) step = __builtin_bit_cast(_Float16, (uint16_t)(__builtin_bit_cast(uint16_t, step) + 1));
    inv = step > (_Float16)0 ? 1.0 / (double)step : 0.0;
}

// Lane i's elements into a row's codes, with the parameters of its groups.
// 64-bit arithmetic, so that a code next to a border is the one of the definition
// whatever computed it.  K and V rows side by side in a wave take one instruction
// stream (`v`: this lane's is a V row): they differ in the order of what is packed.
template <int HD, int BITS>
__device__ __forceinline__ void q_store(const float (&x)[8], uint8_t *codes, _Float16 *params, int i, bool v) {
    using F = QFormat<HD, BITS>;
    constexpr int G = F::kGroups;
    float y[8], lo, hi, odd_sum = 0.0f;  // of the lane's group: HD 128: lanes 0-7 the first, 8-15 the second
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = __builtin_amdgcn_fmed3f(x[e], -65504.0f, 65504.0f);
    // NaN where an element is NaN or infinite
    float bad_sum[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        bad_sum[h] = x[4 * h] * 0.0f;
#pragma unroll
        for (int e = 1; e < 4; ++e) bad_sum[h] = fmaf(x[4 * h + e], 0.0f, bad_sum[h]);
    }
    auto lowest = [&](int h) { return fminf(fminf(y[4 * h], y[4 * h + 1]), fminf(y[4 * h + 2], y[4 * h + 3])); };
    auto highest = [&](int h) { return fmaxf(fmaxf(y[4 * h], y[4 * h + 1]), fmaxf(y[4 * h + 2], y[4 * h + 3])); };
    const float l0 = lowest(0), l1 = lowest(1), h0 = highest(0), h1 = highest(1);
    const bool upper = HD == 128 && i >= 8;
    auto swap8 = [](float a) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(a), 0x128, 0xF, 0xF, false)); };  // lane ^ 8
    if constexpr (G == 2) {
        lo = fminf(upper ? l1 : l0, swap8(upper ? l0 : l1));
        hi = fmaxf(upper ? h1 : h0, swap8(upper ? h0 : h1));
        odd_sum = (upper ? bad_sum[1] : bad_sum[0]) + swap8(upper ? bad_sum[0] : bad_sum[1]);
    } else {
        lo = fminf(l0, l1);
        hi = fmaxf(h0, h1);
        odd_sum = bad_sum[0] + bad_sum[1];
    }
    auto over = [&](auto which) {
        constexpr int S = decltype(which)::value;
        lo = fminf(lo, xchg<S>(lo));
        hi = fmaxf(hi, xchg<S>(hi));
        odd_sum += xchg<S>(odd_sum);
    };
    over(std::integral_constant<int, XQ1>{});
    over(std::integral_constant<int, XQ2>{});
    over(std::integral_constant<int, XM8>{});
    _Float16 own_step, own_mid;
    double own_inv;
    q_grid<BITS>(lo, hi, own_step, own_mid, own_inv);
    v2h grid[2];  // step and midpoint of each half's group
    double inv[2];
    bool bad[2];
    const bool own_bad = odd_sum != odd_sum;
    const v2h nan = __builtin_bit_cast(v2h, 0x7e007e00u);
    grid[0] = grid[1] = own_bad ? nan : (v2h){own_step, own_mid};
    inv[0] = inv[1] = own_inv;
    bad[0] = bad[1] = own_bad;
    if constexpr (G == 2) {
        const v2h other = __builtin_bit_cast(v2h, swap8(__builtin_bit_cast(float, grid[0])));
        const uint64_t w = __builtin_bit_cast(uint64_t, own_inv);
        const uint32_t w0 = __float_as_uint(swap8(__uint_as_float((uint32_t)w))), w1 = __float_as_uint(swap8(__uint_as_float((uint32_t)(w >> 32))));
        const double other_inv = __builtin_bit_cast(double, (uint64_t)w1 << 32 | w0);
        grid[0] = upper ? other : grid[0];
        grid[1] = upper ? grid[1] : other;
        inv[0] = upper ? other_inv : own_inv;
        inv[1] = upper ? own_inv : other_inv;
        bad[0] = grid[0][1] != grid[0][1];
        bad[1] = grid[1][1] != grid[1][1];
    }
    // Step and reciprocal are exact to 2^-52, so no quotient rounds past the outermost
    // codes.  Adding 3 · 2^51 rounds to a whole number, ties to even, into the low bits.
    uint32_t c[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        double t = ((double)y[e] - (double)grid[e >> 2][1]) * inv[e >> 2];
        asm("" : "+v"(t));  // rounded by itself: no multiply-add with what follows
        c[e] = (uint32_t)__builtin_bit_cast(uint64_t, t + (6755399441055744.0 + F::kHalf));
    }
    if (i == 0) {
        if constexpr (G == 2) *reinterpret_cast<v4h *>(params) = (v4h){grid[0][0], grid[1][0], grid[0][1], grid[1][1]};
        else *reinterpret_cast<v2h *>(params) = grid[0];
    }
    uint32_t kw[2], vw[2];  // the halves' codes as K and as V packs them
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t *d = c + 4 * h;
        if constexpr (BITS == 8) {
            kw[h] = vw[h] = bad[h] ? 0u : d[0] | d[1] << 8 | d[2] << 16 | d[3] << 24;
        } else {
            kw[h] = bad[h] ? 0u : d[0] | d[1] << 16 | d[2] << 4 | d[3] << 20;
            vw[h] = bad[h] ? 0u : d[0] | d[1] << 4 | d[2] << 8 | d[3] << 12;
        }
    }
    // Lanes i and i ^ 1 have halves of two pieces of eight neighbours: the even lane
    // writes the lower elements' one.  V's pieces for heads of 128 are the lane's own.
    const int odd = i & 1, b = odd * (HD / 16) + (i >> 1);
    auto pieces = [&](const uint32_t (&w)[2], uint32_t &first, uint32_t &second) {
        const uint32_t got = __float_as_uint(xchg<XQ1>(__uint_as_float(odd ? w[0] : w[1])));
        first = odd ? got : w[0];
        second = odd ? w[1] : got;
    };
    uint32_t first, second;
    pieces(kw, first, second);
    int at = k_place<HD, BITS>(b);
    if constexpr (HD == 128) {
        first = v ? vw[0] : first;
        second = v ? vw[1] : second;
        at = v ? BITS * i : at;
    } else {
        uint32_t vf, vs;
        pieces(vw, vf, vs);
        first = v ? vf : first;
        second = v ? vs : second;
        at = v ? BITS * b : at;
    }
    if constexpr (BITS == 4) *reinterpret_cast<uint32_t *>(codes + at) = first | second << (v ? 16 : 8);
    else *reinterpret_cast<uint2 *>(codes + at) = make_uint2(first, second);
}

// ---------------------------------------------------------------------------
// rows normed, rotated and written
// ---------------------------------------------------------------------------

struct RowsCall {
    const float *src[3];  // q, k, v
    float *dst[3];
    int64_t src_ss[3], src_st[3], dst_ss[3], dst_st[3];
    int end[3];           // heads of q; of q and k; of q, k and v
    const float *norm[2];
    const int32_t *positions, *counts, *first;
    const double *freqs;
    QRows cache;
    int n, half, axes, sections[4], interleaved, adjacent;
    int rows;             // of a destination
    int per, chunks;      // heads of a wave, waves of a token
    int tokens;           // of a wave, one after the other
    float eps;
};

// cos and sin of x, |x| up to 2^31 or so, to 2^-52: x less a multiple of pi/2 in
// two parts (each product is exact inside its multiply-add), then Taylor's series
// up to pi/4, whose next terms are below 2^-54.
__device__ __forceinline__ double2 turn(double x) {
    const double k = rint(x * 0.63661977236758134308);
    double r = fma(-k, 1.57079632679489655800, x);
    r = fma(-k, 6.12323399573676603587e-17, r);
    const double z = r * r;
    double c = 1.0 / 20922789888000.0, s = 1.0 / 355687428096000.0;
    c = fma(c, -z, 1.0 / 87178291200.0);
    c = fma(c, -z, 1.0 / 479001600.0);
    c = fma(c, -z, 1.0 / 3628800.0);
    c = fma(c, -z, 1.0 / 40320.0);
    c = fma(c, -z, 1.0 / 720.0);
    c = fma(c, -z, 1.0 / 24.0);
    c = fma(c, -z, 0.5);
    c = fma(c, -z, 1.0);
    s = fma(s, -z, 1.0 / 1307674368000.0);
    s = fma(s, -z, 1.0 / 6227020800.0);
    s = fma(s, -z, 1.0 / 39916800.0);
    s = fma(s, -z, 1.0 / 362880.0);
    s = fma(s, -z, 1.0 / 5040.0);
    s = fma(s, -z, 1.0 / 120.0);
    s = fma(s, -z, 1.0 / 6.0);
    s = fma(s * z, -r, r);
    const int quarter = (int)(long long)k;
    const double a = quarter & 1 ? s : c, b = quarter & 1 ? c : s;
    return make_double2((quarter + 1) & 2 ? -a : a, quarter & 2 ? -b : b);
}

// what the wave's lanes wrote to LDS is there for its other lanes
__device__ __forceinline__ void wave_lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// the axis that turns pair i
__device__ __forceinline__ int axis_of(const RowsCall &p, int i) {
    if (p.interleaved) {
        const int a = i % p.axes;
        return a && i < p.axes * p.sections[a] ? a : 0;
    }
    int a = 0;
    for (int end = p.sections[0]; a < p.axes - 1 && i >= end;) end += p.sections[++a];
    return a;
}

template <int S>
__device__ __forceinline__ double xchg(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __float_as_uint(xchg<S>(__uint_as_float((uint32_t)u))), hi = __float_as_uint(xchg<S>(__uint_as_float((uint32_t)(u >> 32))));
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// 1 / sqrt(x): the instruction's estimate, then a step of third and one of second order
__device__ __forceinline__ double inverse_root(double x) {
    double r = __builtin_amdgcn_rsq(x);
    double e = fma(-x * r, r, 1.0);
    r = fma(r * e, fma(e, 0.375, 0.5), r);
    e = fma(-x * r, r, 1.0);
    return fma(r * e, 0.5, r);
}

// how a head's pairs lie: (i, H + i) over the whole of it, (2i, 2i + 1), or over part of it by halves
enum : int { kPairsWhole = 0, kPairsAdjacent = 1, kPairsPart = 2 };

// Wave: `tokens` tokens one after the other, `per` heads of each, HD / 8 lanes a
// head; the next heads are on their way meanwhile.  A token's angles are computed
// once, one a lane, and go through LDS to the lanes of every head.
template <int HD, int BITS, int PAIRS>  // BITS 0: fp32 destinations
__global__ void __launch_bounds__(256) k_rows(RowsCall p) {
    constexpr int L = HD / 8, U = 64 / L, H = HD / 2;
    __shared__ double2 s_turn[4][H];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), s = blockIdx.y, i = lane % L;
    const uint32_t job = blockIdx.x * 4 + wave;  // at most 2^22 tokens, 2^9 chunks
    const int step = job / (uint32_t)p.chunks, chunk = job - step * p.chunks;
    const int count = p.counts ? min(max(p.counts[s], 0), p.n) : p.n;
    int tok = step * p.tokens;
    const int end = min(count, tok + p.tokens), begin = chunk * p.per, last = min(p.end[2], begin + p.per);
    if (tok >= end) return;
    const int64_t row0 = p.first ? min(max(p.first[s], 0), p.rows - count) : 0;
    // of a token's unit u0 + lane / L: 0 q, 1 k, 2 v, and the head
    auto kind_of = [&](int u) { return u < p.end[0] ? 0 : (u < p.end[1] ? 1 : 2); };
    auto pick = [](int kind, auto a, auto b, auto c) { return kind == 0 ? a : (kind == 1 ? b : c); };
    auto fetch = [&](int t, int u0, v4f (&x)[2]) {
        const int u = u0 + lane / L, kind = kind_of(u);
        x[0] = x[1] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
        if (u < last) {
            const float *at[3];
#pragma unroll
            for (int k = 0; k < 3; ++k) at[k] = p.src[k] + s * p.src_ss[k] + t * p.src_st[k];
            const float *src = pick(kind, at[0], at[1], at[2]) + (u - pick(kind, 0, p.end[0], p.end[1])) * HD + 4 * i;
            x[0] = *reinterpret_cast<const v4f *>(src);
            x[1] = *reinterpret_cast<const v4f *>(src + H);
        }
    };
    const bool turned = p.positions && lane < p.half;
    const int32_t *place = p.positions + (int64_t)s * p.n * p.axes + (turned ? axis_of(p, lane) : 0);
    double freq = 0.0;
    int position = 0;
    if (turned) {
        freq = p.freqs[lane];
        position = place[(int64_t)tok * p.axes];
    }
    v4f next[2];
    fetch(tok, begin, next);
    for (; tok < end; ++tok) {
        double2 t4[4];  // the turns of this lane's pairs
        bool turns[2] = {true, true};
        if (p.positions) {
            if (turned) {
                s_turn[wave][lane] = turn((double)position * freq);
                if (tok + 1 < end) position = place[(int64_t)(tok + 1) * p.axes];
            }
            wave_lds_order();
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int at = PAIRS == kPairsAdjacent ? (e < 2 ? 2 * i + e : H / 2 + 2 * i + e - 2) : 4 * i + e;
                if (PAIRS != kPairsPart) t4[e] = s_turn[wave][at];
            }
            if (PAIRS == kPairsAdjacent) {
                turns[0] = 2 * i < p.half;
                turns[1] = H / 2 + 2 * i < p.half;
            }
        }
        for (int u0 = begin; u0 < last; u0 += U) {
            const int u = u0 + lane / L, kind = kind_of(u), head = u - pick(kind, 0, p.end[0], p.end[1]);
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = next[e >> 2][e & 3];
            if (u0 + U < last) fetch(tok, u0 + U, next);
            else if (tok + 1 < end) fetch(tok + 1, begin, next);
            const float *w = kind == 0 ? p.norm[0] : p.norm[1];
            if (kind < 2 && (w || p.positions)) {
                double y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = x[e];
                if (w) {
                    double sum = 0.0;
#pragma unroll
                    for (int e = 0; e < 8; ++e) sum = fma(y[e], y[e], sum);
                    sum += xchg<XQ1>(sum);
                    sum += xchg<XQ2>(sum);
                    sum += xchg<XM8>(sum);
                    if (HD == 128) sum += xchg<XM16>(sum);
                    const double r = inverse_root(fma(sum, 1.0 / HD, (double)p.eps));
                    const v4f w0 = *reinterpret_cast<const v4f *>(w + 4 * i), w1 = *reinterpret_cast<const v4f *>(w + H + 4 * i);
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] = y[e] * r * (double)(e < 4 ? w0 : w1)[e & 3];
                }
                if (!p.positions) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = (float)y[e];
                } else if (PAIRS == kPairsWhole) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[e] = (float)(y[e] * t4[e].x - y[4 + e] * t4[e].y);
                        x[4 + e] = (float)(y[4 + e] * t4[e].x + y[e] * t4[e].y);
                    }
                } else if (PAIRS == kPairsAdjacent) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const double a = y[2 * e], b = y[2 * e + 1];
                        x[2 * e] = (float)(turns[e >> 1] ? a * t4[e].x - b * t4[e].y : a);
                        x[2 * e + 1] = (float)(turns[e >> 1] ? b * t4[e].x + a * t4[e].y : b);
                    }
                } else {
                    // elements d and d + half, half a multiple of 8: chunks of four `far` chunks apart
                    const int far = p.half / 4;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int q = h * L + i, mate = q < far ? q + far : q - far;
                        const int from = (lane & ~(L - 1)) + (mate & (L - 1));
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const double lower = __shfl(y[e], from & 63), upper = __shfl(y[4 + e], from & 63);
                            const double own = y[4 * h + e], z = mate & L ? upper : lower;
                            const double2 tr = s_turn[wave][min(4 * (q < far ? q : q - far) + e, H - 1)];
                            x[4 * h + e] = (float)(q < far ? own * tr.x - z * tr.y : (q < 2 * far ? own * tr.x + z * tr.y : own));
                        }
                    }
                }
            }
            if (u >= last) continue;
            const int64_t row = row0 + tok;
            if (BITS && kind) {
                constexpr int B = BITS ? BITS : 4;
                using F = QFormat<HD, B>;
                const int64_t at = s * p.cache.seq_rows + (int64_t)head * p.cache.capacity + row;
                const bool v = kind == 2;
                q_store<HD, B>(x, (v ? p.cache.codes[1] : p.cache.codes[0]) + at * F::kCodes,
                               (v ? p.cache.params[1] : p.cache.params[0]) + at * F::kParams, i, v);
            } else {
                float *at[3];
#pragma unroll
                for (int k = 0; k < 3; ++k) at[k] = p.dst[k] + s * p.dst_ss[k] + (k ? row : tok) * p.dst_st[k];
                float *dst = pick(kind, at[0], at[1], at[2]) + head * HD + 4 * i;
                *reinterpret_cast<v4f *>(dst) = (v4f){x[0], x[1], x[2], x[3]};
                *reinterpret_cast<v4f *>(dst + H) = (v4f){x[4], x[5], x[6], x[7]};
            }
        }
        if (p.positions) wave_lds_order();  // all lanes have read this token's turns
    }
}

// ---------------------------------------------------------------------------
// rows read back
// ---------------------------------------------------------------------------

struct QReadCall {
    float *dst[2];
    int64_t dst_ss[2], dst_st[2];
    const int32_t *rows, *counts, *first;
    QRows cache;
    int n, per_head;
    int row0;  // first row of the grid
};

// HD / 8 lanes a row of a head, K and V one after the other
template <int HD, int BITS>
__global__ void __launch_bounds__(256) k_qcache_read(QReadCall p) {
    using F = QFormat<HD, BITS>;
    constexpr int L = HD / 8;
    const int i = threadIdx.x % L, g = blockIdx.y, s = blockIdx.z;
    const int most = p.rows ? p.n : min(p.n, p.cache.capacity);
    const int count = p.counts ? min(max(p.counts[s], 0), most) : most;
    const int t = p.row0 + (int)blockIdx.x * (256 / L) + (int)threadIdx.x / L;
    if (t >= count) return;
    int row;
    if (p.rows) {
        row = p.rows[(p.per_head ? (int64_t)s * p.cache.kvh + g : s) * p.n + t];
        row = min(max(row, 0), p.cache.capacity - 1);
    } else {
        row = (p.first ? min(max(p.first[s], 0), p.cache.capacity - count) : 0) + t;
    }
    const int64_t at = s * p.cache.seq_rows + (int64_t)g * p.cache.capacity + row;
    auto one = [&](auto v) {
        constexpr int V = decltype(v)::value;
        if (!p.dst[V]) return;
        float x[8];
        q_values<HD, BITS, V == 1>(p.cache.codes[V] + at * F::kCodes, p.cache.params[V] + at * F::kParams, i, x);
        float *dst = p.dst[V] + s * p.dst_ss[V] + t * p.dst_st[V] + g * HD + 4 * i;
        *reinterpret_cast<v4f *>(dst) = (v4f){x[0], x[1], x[2], x[3]};
        *reinterpret_cast<v4f *>(dst + HD / 2) = (v4f){x[4], x[5], x[6], x[7]};
    };
    one(std::integral_constant<int, 0>{});
    one(std::integral_constant<int, 1>{});
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------

struct QAttnCall {
    const float *q;
    float *out, *lse;
    const int32_t *lens, *counts;
    const float *slopes;
    int64_t q_ss, q_st, o_ss, o_st;
    QRows cache;
    int n, heads, group, max_rows, window;
    float scale, cap;
};

// Row tiles and key shares of a call.
struct QAttnPlan {
    int tiles, splits;  // of a (sequence, KV head); shares a tile's keys may be cut into
    int least;          // blocks of a share
    float *part;        // [sequence][KV head][tile][split][rows][HD] sums
    float2 *stat;       // their rows' reference exponents and denominators
};

constexpr int kQBlock = 32;      // keys per step of a wave
constexpr int kQTop = 13;        // weights times steps stay below 2^(kQTop + kQSlack)
constexpr int kQSlack = 2;       // a score may pass its row's reference by this before that moves
constexpr float kQFar = 4194304.0f;  // up to here whole numbers and their differences are exact

// the query rows of a tile: [first, last] and what they see
struct QTile {
    int count, len;
    int lo, hi;          // keys some row sees
    int all_lo, all_hi;  // keys all rows see
};
__device__ __forceinline__ QTile q_tile(const QAttnCall &p, int s, int first, int rows) {
    QTile t;
    t.count = p.counts ? min(max(p.counts[s], 0), p.n) : p.n;
    t.len = min(max(p.lens[s], 0), p.max_rows);
    const int all = t.count * p.group;
    if (first >= all) {
        t.lo = t.hi = t.all_lo = t.all_hi = 0;
        t.count = 0;
        return t;
    }
    const int tok0 = first / p.group, tok1 = (min(first + rows, all) - 1) / p.group, pos = t.len - t.count;
    t.hi = max(0, pos + tok1 + 1);
    t.all_hi = max(0, pos + tok0 + 1);
    t.lo = p.window ? min(t.hi, max(0, pos + tok0 - p.window + 1)) : 0;
    t.all_lo = p.window ? max(0, pos + tok1 - p.window + 1) : 0;
    return t;
}

// the blocks of one share of a tile's keys
struct QShare {
    int parts, from, to;
};
__device__ __forceinline__ QShare q_share(const QAttnPlan &pl, const QTile &t, int part) {
    const int first = t.lo / kQBlock, blocks = max(0, (t.hi + kQBlock - 1) / kQBlock - first);
    QShare h;
    h.parts = min(pl.splits, max(1, blocks / pl.least));
    h.from = first + (int)((int64_t)blocks * part / h.parts);
    h.to = first + (int)((int64_t)blocks * (part + 1) / h.parts);
    return h;
}

// Codes as fp16 numbers: 1024 + n is a bit pattern away from n < 1024, and taking
// 1024 off again exact.  `magic` holds the pattern in a vector register, where one
// instruction can both mask and set bits (it may name a single scalar one).
__device__ __forceinline__ uint32_t code_magic() {
    uint32_t m = 0x64006400u;
    asm("" : "+v"(m));
    return m;
}
template <int LESS>  // 1024 + what the codes are stored with
__device__ __forceinline__ v2h code_pair(uint32_t bits, uint32_t mask, uint32_t magic) {
    return __builtin_bit_cast(v2h, (bits & mask) | magic) - (v2h){(_Float16)LESS, (_Float16)LESS};
}

// Codes of 32 keys as a lane loads and uses them.  Lane l = 16u + i.  K: keys i and
// 16 + i, elements 32c + 8u .. +7 of each 32 (a matrix instruction's operand); V: keys
// 4u .. +3 and 16 + 4u .. +3, elements 4i .. +3 of each 64.  Of two codes of 4 bits
// in a byte the upper one stays where it is, 16 times too large: the query row's
// elements and the sums that meet it are that much smaller.
template <int HD, int BITS>
struct QCodes {
    using F = QFormat<HD, BITS>;
    static constexpr int C = HD / 32;
    static constexpr int kKWords = C * BITS / 4;           // of a key's codes in a lane
    static constexpr int kVWords = HD == 64 && BITS == 4 ? 1 : HD * BITS / 512;  // (16 bits for heads of 64 in 4 bits)
    uint32_t k[2][kKWords], v[8][kVWords];

    template <int W>
    __device__ __forceinline__ static void words(const uint8_t *at, uint32_t *to) {
        if constexpr (W == 8) {
            words<4>(at, to);
            words<4>(at + 64, to + 4);
        } else if constexpr (W == 4) {
            const uint4 x = *reinterpret_cast<const uint4 *>(at);
            to[0] = x.x;
            to[1] = x.y;
            to[2] = x.z;
            to[3] = x.w;
        } else if constexpr (W == 2) {
            const uint2 x = *reinterpret_cast<const uint2 *>(at);
            to[0] = x.x;
            to[1] = x.y;
        } else {
            to[0] = *reinterpret_cast<const uint32_t *>(at);
        }
    }
    // rows k0 .. k0 + 31 of a cache of `rows` rows, its last in place of those behind it
    __device__ __forceinline__ void load_k(const uint8_t *codes, int k0, int rows, int lane) {
        const uint8_t *at = codes + (int64_t)k0 * F::kCodes;
        const uint32_t i = lane & 15, part = (lane >> 4) * (kKWords == 2 ? 8 : 16), last = rows - 1 - k0;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint32_t row = 16 * t + i;
            words<kKWords>(at + ((k0 + kQBlock <= rows ? row : min(row, last)) * F::kCodes + part), k[t]);
        }
    }
    __device__ __forceinline__ void load_v(const uint8_t *codes, int k0, int rows, int lane) {
        const uint8_t *at = codes + (int64_t)k0 * F::kCodes;
        const uint32_t u = lane >> 4, part = (lane & 15) * (HD == 64 && BITS == 4 ? 2 : 4 * kVWords), last = rows - 1 - k0;
        auto one = [&](int j, uint32_t row) {
            if constexpr (HD == 64 && BITS == 4) v[j][0] = *reinterpret_cast<const uint16_t *>(at + (row * F::kCodes + part));
            else words<kVWords>(at + (row * F::kCodes + part), v[j]);
        };
        if (k0 + kQBlock <= rows) {
#pragma unroll
            for (int j = 0; j < 8; ++j) one(j, 16 * (j >> 2) + 4 * u + (j & 3));
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) one(j, min(16 * (j >> 2) + 4 * u + (j & 3), last));
        }
    }
    // what elements of key chunks are to be taken times: of eight, 0 .. 7
    __device__ __forceinline__ static constexpr bool k_upper(int e) { return BITS == 4 && (e >> 1 & 1); }
    __device__ __forceinline__ static constexpr bool v_upper(int t) { return BITS == 4 && (t & 1); }
    // K's operand of chunk c, key tile t
    __device__ __forceinline__ v8h key(int t, int c, uint32_t magic) const {
        v8h r;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v2h x;
            if constexpr (BITS == 4) {
                const uint32_t w = k[t][c] >> (e & 2 ? 8 : 0);
                x = e & 1 ? code_pair<1024 + 128>(w, 0x00f000f0u, magic) : code_pair<1024 + 8>(w, 0x000f000fu, magic);
            } else {
                x = code_pair<1024 + 128>(__builtin_amdgcn_perm(magic, k[t][2 * c + e / 2], e & 1 ? 0x05030502u : 0x05010500u), ~0u, 0u);
            }
            r[2 * e] = x[0];
            r[2 * e + 1] = x[1];
        }
        return r;
    }
    // V's operand of dim tile t: element 64 (t / 4) + 4i + t % 4 of eight keys
    __device__ __forceinline__ v8h value(int t, uint32_t magic) const {
        v8h r;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const uint32_t b = BITS == 4 ? t >> 1 : t & 3;  // the byte that holds it
            const int w = BITS == 4 ? 0 : t >> 2;
            const uint32_t two = __builtin_amdgcn_perm(v[j + 1][w], v[j][w], 0x0c040c00u + 0x00010001u * b);
            v2h x;
            if constexpr (BITS == 4) x = t & 1 ? code_pair<1024 + 128>(two, 0x00f000f0u, magic) : code_pair<1024 + 8>(two, 0x000f000fu, magic);
            else x = code_pair<1024 + 128>(two, ~0u, magic);
            r[j] = x[0];
            r[j + 1] = x[1];
        }
        return r;
    }
};

// a weight times a step as halves
__device__ __forceinline__ void split_steps(float a, _Float16 sa, float b, _Float16 sb, v2h &hi, v2h &lo) {
    hi = whole_v2h((v2h){(_Float16)__builtin_fmaf(a, (float)sa, 0.0f), (_Float16)__builtin_fmaf(b, (float)sb, 0.0f)});
    lo = (v2h){(_Float16)__builtin_fmaf(a, (float)sa, -(float)hi[0]), (_Float16)__builtin_fmaf(b, (float)sb, -(float)hi[1])};
}

// Attention over codes.  Workgroup: a tile of query rows (token, head of the KV
// head's group) of one sequence and KV head, and a share of its keys.  KEYS: 16 ·
// RT rows, the four waves take its blocks of 32 keys in turn and join; otherwise
// 16 · RT rows a wave, all of the share's blocks.
//
// Codes go to the matrix instructions as they are, exact in fp16, and meet query
// rows and weights as two fp16 halves each.  Scores come out transposed (lane l:
// query row l % 16, keys 4 (l / 16) + r of each 16), so a row's statistics stay
// with its four lanes and its weights are the second product's operand:
//   q . k = sum over groups of step (q . c) + mid (sum of q),
//   out = sum over keys of (p step) . c + sum of p mid.
// p = 2^(s - ref), ref a whole number near the row's largest score, lowered by the
// exponent that brings V's largest step so far to 2^kQTop, so that the halves of p
// step hold the products that count whatever V's size.  All rescales are by powers
// of two.  A block's codes are requested as soon as the registers of the block
// before are free.
template <int HD, int BITS, int RT, bool SHAPED, bool KEYS>
__global__ void __launch_bounds__(256, RT == 1 ? 3 : 2) k_qcache_attn(QAttnCall p, QAttnPlan pl) {
    using F = QFormat<HD, BITS>;
    using Codes = QCodes<HD, BITS>;
    constexpr int C = HD / 32, G = HD / 64, T = HD / 16;
    constexpr int kRows = 16 * RT * (KEYS ? 1 : 4);
    constexpr int kPar = 32 * 4 * G;  // bytes of a block's parameters of K or V
    __shared__ __attribute__((aligned(16))) uint8_t s_par[4][2 * kPar];
    __shared__ v4f s_acc[KEYS ? 2 : 1][KEYS ? RT * T : 1][64];
    __shared__ float s_ref[KEYS ? 4 : 1][16 * RT], s_sum[KEYS ? 4 : 1][16 * RT];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = lane & 15, u = lane >> 4;
    const int g = blockIdx.y, s = blockIdx.z;
    const int tile = pl.tiles - 1 - (int)(blockIdx.x / pl.splits), part = blockIdx.x % pl.splits;  // long rows first
    const QTile wt = q_tile(p, s, tile * kRows, kRows);
    if (!wt.count) return;
    const QShare share = q_share(pl, wt, part);
    if (part >= share.parts) return;
    const int first = tile * kRows + (KEYS ? 0 : wave * 16 * RT), all = wt.count * p.group;
    if (first >= all) return;  // no barriers without KEYS
    const QTile t = KEYS ? wt : q_tile(p, s, first, 16 * RT);

    const int64_t base = s * p.cache.seq_rows + (int64_t)g * p.cache.capacity;
    const uint8_t *kc = p.cache.codes[0] + base * F::kCodes, *vc = p.cache.codes[1] + base * F::kCodes;
    const uint8_t *kp = reinterpret_cast<const uint8_t *>(p.cache.params[0] + base * F::kParams);
    const uint8_t *vp = reinterpret_cast<const uint8_t *>(p.cache.params[1] + base * F::kParams);
    const int cap = p.cache.capacity;
    int block = share.from, end = share.to;
    if (KEYS) {
        block += wave;
    } else {
        block = max(block, t.lo / kQBlock);
        end = min(end, (t.hi + kQBlock - 1) / kQBlock);
    }
    constexpr int kStep = KEYS ? 4 : 1;
    // parameters: a word a lane, spread over the lanes through LDS
    uint32_t kw = 0, vw = 0;
    const uint32_t par_key = HD == 128 ? lane >> 1 : lane & 31, par_word = HD == 128 ? 4 * (lane & 1) : 0;
    auto load_par = [&](int k0) {
        const uint32_t row = min(par_key, (uint32_t)(cap - 1 - k0)) * (4 * G) + par_word;
        kw = *reinterpret_cast<const uint32_t *>(kp + (int64_t)k0 * (4 * G) + row);
        vw = *reinterpret_cast<const uint32_t *>(vp + (int64_t)k0 * (4 * G) + row);
    };
    Codes codes;
    if (block < end) {
        codes.load_k(kc, block * kQBlock, cap, lane);
        load_par(block * kQBlock);
        codes.load_v(vc, block * kQBlock, cap, lane);
    }

    // query rows as halves below 2^kTop, their sums of each group
    v8h qh[RT][C], ql[RT][C];
    float qs[RT][G], f[RT], slope[RT];
    int pos[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = first + 16 * rt + i;
        const bool live = r < all;
        const int tok = live ? r / p.group : 0, head = g * p.group + (live ? r - tok * p.group : 0);
        pos[rt] = live ? wt.len - wt.count + tok : -1;
        float x[C][8];
        const float *src = p.q + s * p.q_ss + tok * p.q_st + head * HD + 8 * u;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const v4f y = *reinterpret_cast<const v4f *>(src + 32 * c + e);
#pragma unroll
                for (int k = 0; k < 4; ++k) x[c][e + k] = live ? y[k] : 0.0f;
            }
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max(top, abs_bits(x[c][e]));
        const int e = row_exp(groups_umax(top));
        const float up = pow2(kTop - e);
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
            float sum = 0.0f;
#pragma unroll
            for (int c = 2 * gr; c < 2 * gr + 2; ++c)
#pragma unroll
                for (int k = 0; k < 8; ++k) sum += x[c][k] * up;
            qs[rt][gr] = groups_sum(sum);
        }
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (Codes::k_upper(k)) x[c][k] *= 0.0625f;
        split_row<C>(x, e, qh[rt], ql[rt]);
        // score = product · f; with a cap: tanh(product · f) · cap
        const float size = pow2(e - kTop);
        f[rt] = SHAPED && p.cap > 0.0f ? fminf(p.scale * size * (1.0f / p.cap), 3.0e38f) : p.scale * kLog2e * size;
        slope[rt] = 0.0f;
        if (SHAPED && p.slopes) {
            const float y = p.slopes[head] * kLog2e;
            slope[rt] = fabsf(y) == INFINITY ? copysignf(3.4028235e38f, y) : y;
        }
    }

    v4f acc[RT][T];
    float ref[RT], m[RT], sum[RT], mids[RT][G];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int k = 0; k < T; ++k) acc[rt][k] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
        m[rt] = ref[rt] = kLowest;
        sum[rt] = 0.0f;
#pragma unroll
        for (int gr = 0; gr < G; ++gr) mids[rt][gr] = 0.0f;
    }
    uint32_t step_top = 0;  // bits of V's largest step so far
    int raise = kQTop + 14;  // exponent that brings it below 2^kQTop
    const uint32_t magic = code_magic();
    uint32_t *par = reinterpret_cast<uint32_t *>(s_par[wave]);

    for (; block < end; block += kStep) {
        const int k0 = block * kQBlock, next0 = k0 + kStep * kQBlock;
        const bool more = block + kStep < end;
        const bool masked = k0 < t.all_lo || k0 + kQBlock > t.all_hi;
        if (masked) {  // parameters of keys outside the tile's are zero
            const int key = k0 + (int)par_key;
            if (key < t.lo || key >= t.hi) kw = vw = 0;
        }
        // V's largest step.  Numbers that are none stay out of products: they would
        // meet the zero weights of rows that do not see them.  Rows that do get them below.
        uint64_t bad[2] = {0, 0};
        bool moved = false;
        {
            const bool b0 = (vw & 0x7c00u) == 0x7c00u, b1 = (vw & 0x7c000000u) == 0x7c000000u;
            const uint32_t s0 = vw & 0x7fffu, s1 = HD == 128 ? vw >> 16 : 0u;
            const uint32_t lane_top = HD == 128 && (lane & 1) ? 0u : max(s0, s1);
            if (__any((b0 || b1 || lane_top > step_top) && (HD == 128 || lane < 32))) {
                if (b0) vw &= 0xffff0000u;
                if (b1) vw &= 0x0000ffffu;
                bad[0] = __ballot(HD == 128 ? b0 : b0 || b1);
                bad[1] = __ballot(b1);
                uint32_t y = HD == 128 && (lane & 1) ? 0u : max(vw & 0x7fffu, HD == 128 ? vw >> 16 : 0u);
                y = groups_umax(y);
#pragma unroll
                for (int o = 8; o; o >>= 1) y = max(y, (uint32_t)__shfl_xor((int)y, o));
                if (y > step_top) {
                    step_top = y;
                    // step < 2^(exponent - 14), subnormal ones < 2^-14
                    const int now = kQTop + 14 - (int)(y >> 10);
                    moved = now != raise;
                    raise = now;
                }
            }
        }
        if (HD == 128 || lane < 32) {
            par[lane] = kw;
            par[kPar / 4 + lane] = vw;
        }
        wave_lds_order();
        if (more) load_par(next0);

        // scores: row i, keys 16 · kt + 4u + k
        float sc[RT][8];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            v8h pars[G];
#pragma unroll
            for (int k = 0; k < G; ++k) pars[k] = *reinterpret_cast<const v8h *>(s_par[wave] + (16 * kt + 4 * u) * 4 * G + 16 * k);
            v4f d[RT][G];
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const v8h key = codes.key(kt, c, magic);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    const v4f from = c % 2 ? d[rt][c / 2] : (v4f){0.0f, 0.0f, 0.0f, 0.0f};
                    const v4f x = __builtin_amdgcn_mfma_f32_16x16x32_f16(key, qh[rt][c], from, 0, 0, 0);
                    d[rt][c / 2] = __builtin_amdgcn_mfma_f32_16x16x32_f16(key, ql[rt][c], x, 0, 0, 0);
                }
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float x = 0.0f;
#pragma unroll
                    for (int gr = 0; gr < G; ++gr) {
                        const int at = k * 2 * G + gr;
                        const float step = (float)pars[at >> 3][at & 7], mid = (float)pars[(at + G) >> 3][(at + G) & 7];
                        x = gr ? fmaf(mid, qs[rt][gr], x) : mid * qs[rt][gr];
                        x = fmaf(step, d[rt][gr][k], x);
                    }
                    sc[rt][4 * kt + k] = rounded(x * f[rt]);
                }
        }
        if (more) codes.load_k(kc, next0, cap, lane);

        v8h wh[RT][G], wl[RT][G];
        v8h vpar[2][G];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int k = 0; k < G; ++k) vpar[kt][k] = *reinterpret_cast<const v8h *>(s_par[wave] + kPar + (16 * kt + 4 * u) * 4 * G + 16 * k);
        auto v_par = [&](int j, int gr, int which) {  // step (which 0) or midpoint of the lane's key j
            const int at = (j & 3) * 2 * G + which * G + gr;
            return vpar[j >> 2][at >> 3][at & 7];
        };
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float (&x)[8] = sc[rt];
            if (SHAPED) {
                if (p.cap > 0.0f) {
                    tanh_all<8>(x);
                    const float up = p.cap * kLog2e;
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] *= up;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    x[j] = rounded(fmaf(-slope[rt], (float)(pos[rt] - (k0 + 16 * (j >> 2) + 4 * u + (j & 3))), x[j]));
            }
            if (masked) {
                const int from = p.window ? max(0, pos[rt] - p.window + 1) : 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int key = k0 + 16 * (j >> 2) + 4 * u + (j & 3);
                    const bool sees = key >= from && key <= pos[rt];
                    x[j] = sees ? x[j] : -INFINITY;
                }
            }
            if (bad[0] | bad[1]) {  // NaN for the rows that see it, in its group
                const int from = p.window ? max(0, pos[rt] - p.window + 1) : 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int at = 16 * (j >> 2) + 4 * u + (j & 3), key = k0 + at;
                    const bool sees = key >= from && key <= pos[rt];
#pragma unroll
                    for (int gr = 0; gr < G; ++gr)
                        if (sees && (bad[gr] >> (HD == 128 ? 2 * at : at) & (HD == 128 ? 3 : 1))) mids[rt][gr] = __builtin_nanf("");
                }
            }
            float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
            if (moved || __any(top > m[rt] + kQSlack)) {
                top = groups_max(top);
                if (top > m[rt]) m[rt] = fminf(ceilf(top), 3.0e38f);
                const float now = fabsf(m[rt]) < kQFar ? m[rt] - (float)raise : m[rt];
                const float by = __builtin_amdgcn_exp2f(ref[rt] - now);
                ref[rt] = now;
                sum[rt] *= by;
#pragma unroll
                for (int gr = 0; gr < G; ++gr) mids[rt][gr] *= by;
#pragma unroll
                for (int k = 0; k < T; ++k) acc[rt][k] *= by;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[j] = __builtin_amdgcn_exp2f(x[j] - ref[rt]);
                sum[rt] += x[j];
            }
#pragma unroll
            for (int gr = 0; gr < G; ++gr)
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    v2h h, l;
                    split_steps(x[j], v_par(j, gr, 0), x[j + 1], v_par(j + 1, gr, 0), h, l);
                    wh[rt][gr][j] = h[0];
                    wh[rt][gr][j + 1] = h[1];
                    wl[rt][gr][j] = l[0];
                    wl[rt][gr][j + 1] = l[1];
                    mids[rt][gr] = fmaf((float)v_par(j, gr, 1), x[j], mids[rt][gr]);
                    mids[rt][gr] = fmaf((float)v_par(j + 1, gr, 1), x[j + 1], mids[rt][gr]);
                }
        }
#pragma unroll
        for (int k = 0; k < T; ++k) {
            const v8h v = codes.value(k, magic);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                acc[rt][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, wh[rt][k / 4], acc[rt][k], 0, 0, 0);
                acc[rt][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, wl[rt][k / 4], acc[rt][k], 0, 0, 0);
            }
        }
        if (more) codes.load_v(vc, next0, cap, lane);
        wave_lds_order();
    }

    // denominators and midpoints over a row's four lanes
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        sum[rt] = groups_sum(sum[rt]);
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
            mids[rt][gr] = groups_sum(mids[rt][gr]);
#pragma unroll
            for (int k = 4 * gr; k < 4 * gr + 4; ++k) acc[rt][k] = acc[rt][k] * (Codes::v_upper(k) ? 0.0625f : 1.0f) + mids[rt][gr];
        }
    }
    if (KEYS) {  // four waves' sums: 2 and 3 to 0 and 1, then 1 to 0
        if (u == 0)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                s_ref[wave][16 * rt + i] = sum[rt] == 0.0f ? kLowest : ref[rt];
                s_sum[wave][16 * rt + i] = sum[rt];
            }
        __syncthreads();
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float top = kLowest, total = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) top = fmaxf(top, s_ref[w][16 * rt + i]);
#pragma unroll
            for (int w = 0; w < 4; ++w) total += s_sum[w][16 * rt + i] * __builtin_amdgcn_exp2f(s_ref[w][16 * rt + i] - top);
            const float by = __builtin_amdgcn_exp2f((sum[rt] == 0.0f ? kLowest : ref[rt]) - top);
#pragma unroll
            for (int k = 0; k < T; ++k) acc[rt][k] *= by;
            sum[rt] = total;
            ref[rt] = top;
        }
#pragma unroll
        for (int half = 2; half; half >>= 1) {
            if (wave >= half && wave < 2 * half)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int k = 0; k < T; ++k) s_acc[wave - half][rt * T + k][lane] = acc[rt][k];
            __syncthreads();
            if (wave < half)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int k = 0; k < T; ++k) acc[rt][k] += s_acc[wave][rt * T + k][lane];
            __syncthreads();
        }
        if (wave) return;
    }
    const int64_t slot = (((int64_t)s * p.cache.kvh + g) * pl.tiles + tile) * pl.splits + part;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = first + 16 * rt + i;
        if (r >= all) continue;
        float *dst;
        float by = 1.0f;
        if (share.parts > 1) {
            const int64_t at = slot * kRows + (r - tile * kRows);
            dst = pl.part + at * HD;
            if (u == 0) pl.stat[at] = make_float2(sum[rt] == 0.0f ? kLowest : ref[rt], sum[rt]);
        } else {
            const int tok = r / p.group, head = g * p.group + r - tok * p.group;
            dst = p.out + s * p.o_ss + tok * p.o_st + head * HD;
            by = sum[rt] == 0.0f ? 0.0f : 1.0f / sum[rt];
            if (p.lse && u == 0)
                p.lse[((int64_t)s * p.n + tok) * p.heads + head] =
                    sum[rt] == 0.0f ? -INFINITY : (ref[rt] + __builtin_amdgcn_logf(sum[rt])) * 0.69314718055994531f;
        }
#pragma unroll
        for (int gr = 0; gr < G; ++gr)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                *reinterpret_cast<v4f *>(dst + 64 * gr + 16 * u + 4 * k) =
                    (v4f){acc[rt][4 * gr][k] * by, acc[rt][4 * gr + 1][k] * by, acc[rt][4 * gr + 2][k] * by, acc[rt][4 * gr + 3][k] * by};
    }
}

// A tile's shares joined: HD / 4 lanes a row.
template <int HD, int ROWS>
__global__ void __launch_bounds__(256) k_qcache_join(QAttnCall p, QAttnPlan pl) {
    constexpr int L = HD / 4, U = 256 / L;
    const int i = threadIdx.x % L, g = blockIdx.y, s = blockIdx.z;
    const int tile = blockIdx.x / (ROWS / U), row = (int)(blockIdx.x % (ROWS / U)) * U + (int)threadIdx.x / L;
    const QTile t = q_tile(p, s, tile * ROWS, ROWS);
    const int r = tile * ROWS + row;
    if (r >= t.count * p.group) return;
    const int parts = q_share(pl, t, 0).parts;
    if (parts == 1) return;
    const int64_t at = ((((int64_t)s * p.cache.kvh + g) * pl.tiles + tile) * pl.splits) * ROWS + row;
    const float2 *stat = pl.stat + at;
    const float *part = pl.part + at * HD + 4 * i;
    float top = kLowest, total = 0.0f;
    for (int k = 0; k < parts; ++k) top = fmaxf(top, stat[(int64_t)k * ROWS].x);
    v4f sum = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int k = 0; k < parts; ++k) {
        const float2 st = stat[(int64_t)k * ROWS];
        const float by = __builtin_amdgcn_exp2f(st.x - top);
        total += st.y * by;
        sum += *reinterpret_cast<const v4f *>(part + (int64_t)k * ROWS * HD) * by;
    }
    const int tok = r / p.group, head = g * p.group + r - tok * p.group;
    *reinterpret_cast<v4f *>(p.out + s * p.o_ss + tok * p.o_st + head * HD + 4 * i) = sum * (total == 0.0f ? 0.0f : 1.0f / total);
    if (p.lse && i == 0)
        p.lse[((int64_t)s * p.n + tok) * p.heads + head] =
            total == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * 0.69314718055994531f;
}

}  // namespace pocr
