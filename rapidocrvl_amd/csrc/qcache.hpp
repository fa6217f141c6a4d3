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

// 1 / sqrt(x): the instruction's estimate, then a step of third and one of second order;
// 0 of an infinity, where the steps would multiply it by its estimate
__device__ __forceinline__ double inverse_root(double x) {
    const double first = __builtin_amdgcn_rsq(x);
    double e = fma(-x * first, first, 1.0);
    double r = fma(first * e, fma(e, 0.375, 0.5), first);
    e = fma(-x * r, r, 1.0);
    r = fma(r * e, 0.5, r);
    return first == 0.0 ? 0.0 : r;
}

// how a head's pairs lie: (i, H + i) over the whole of it, (2i, 2i + 1), or over part of it by halves
enum : int { kPairsWhole = 0, kPairsAdjacent = 1, kPairsPart = 2 };

// Wave: `tokens` tokens one after the other, `per` heads of each, HD / 8 lanes a
// head; the next heads are on their way meanwhile.  A token's angles are computed
// once, one a lane, and go through LDS to the lanes of every head; an angle's product,
// its turn and the norm's sum are in 64 bits, so that a row is the same to its last
// bit, and its code with it, whichever call makes it.
//
// Memory bounds it: 8,192 normed tokens of 16 + 2 + 2 heads of 128 rotated 37 us (168 MB,
// 4.5 TB/s), with K and V into 4 bits 37 too (151 MB: the quantising shows), 18 layers of
// 1,345 K and V rows of 2 heads into 8 bits 17.7 to 20 (62 MB).  1,345 tokens of 16 + 2 heads
// take 8.5 us (27 MB), where the launch and the first loads' way count.  The simplest
// form, a lane with eight neighbouring elements and a wave a head, took 118 us for the
// first: its loads and stores were halves of lines, and a rotation fetched its other
// half from eight lanes away.
template <int HD, int BITS, int PAIRS>  // BITS 0: fp32 destinations
__global__ void __launch_bounds__(256) k_rows(RowsCall p) {
    constexpr int L = HD / 8, U = 64 / L, H = HD / 2;
    __shared__ double2 s_turn[4][H];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), s = blockIdx.y, i = lane % L;
    const uint32_t job = blockIdx.x * 4 + wave;  // at most 2^22 tokens, and 768 chunks below 2,048 of them
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

// HD / 8 lanes a row of a head, K and V one after the other: mid + step * code, a
// multiply-add.  Stores bound it: 18 caches of 1,609 rows of 2 heads of 128 in 4 bits
// (60 MB) 11.4 to 12.3 us, 4.8 to 5.2 TB/s; 2,048 listed rows of each in 8 bits (84 MB)
// 19.3, 4.4 TB/s.  Loads of codes and parameters are short pieces of lines, which the
// neighbours' loads find in the cache.
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
    uint32_t group_inv;  // 2^32 / group, rounded up (group 1: 0)
    float scale, cap, cap_inverse, cap_log2;  // 1 / cap, cap · log2(e)
    // the token of query row r < 2^24: the quotient, at most one too large before its correction
    __device__ __forceinline__ int token(int r) const {
        const uint32_t q = group == 1 ? (uint32_t)r : __umulhi((uint32_t)r, group_inv);
        return (int)(q - (q * (uint32_t)group > (uint32_t)r));
    }
};

// Row tiles and key shares of a call.
struct QAttnPlan {
    int tiles, splits;  // of a (sequence, KV head); shares of a tile's keys
    float *part;        // [sequence][KV head][tile][split][rows][HD] sums
    float2 *stat;       // their rows' reference exponents and denominators
};

constexpr int kQBlock = 32;      // keys per step of a wave
constexpr int kQTop = 9;         // weights times steps stay below 2^(kQTop + kQSlack)
constexpr int kQSlack = 6;       // a score may pass its row's reference by this before that moves
// From here on a reference's exponent stands apart from its whole number: fp32's steps there
// are 1/2 and more, and further up more than an exponent.  Nor may scores pass such a
// reference, since one step of theirs may be more than kQSlack.
constexpr float kQFar = 4194304.0f;

// the query rows of a tile: [first, last] and what they see
struct QTile {
    int count, len;
    int lo, hi;          // keys some row sees
    int all_lo, all_hi;  // keys all rows see
    __device__ __forceinline__ bool partly(int k0) const { return k0 < all_lo || k0 + kQBlock > all_hi; }  // some row, of the block from k0 on
    __device__ __forceinline__ bool mixed() const { return lo != all_lo || hi != all_hi; }
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
    const int tok0 = p.token(first), tok1 = p.token(min(first + rows, all) - 1), pos = t.len - t.count;
    t.hi = max(0, pos + tok1 + 1);
    t.all_hi = max(0, pos + tok0 + 1);
    t.lo = p.window ? min(t.hi, max(0, pos + tok0 - p.window + 1)) : 0;
    t.all_lo = p.window ? max(0, pos + tok1 - p.window + 1) : 0;
    return t;
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

// Rows k0 .. k0 + 31, W bytes each, of a cache of `rows` rows: what lies behind its
// last row is not read, and comes as zeros.
template <int W>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t q_block(const uint8_t *at, int k0, int rows) {
    const int count = min(rows - min(k0, rows), kQBlock);
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(at) + (int64_t)k0 * W, 0, count * W, 0x00027000);
}
template <int N>
__device__ __forceinline__ void q_words(__amdgpu_buffer_rsrc_t from, uint32_t at, uint32_t *to) {
    if constexpr (N == 8) {
        q_words<4>(from, at, to);
        q_words<4>(from, at + 64, to + 4);
    } else if constexpr (N == 4) {
        const auto x = __builtin_amdgcn_raw_buffer_load_b128(from, at, 0, 0);
        to[0] = x[0];
        to[1] = x[1];
        to[2] = x[2];
        to[3] = x[3];
    } else if constexpr (N == 2) {
        const auto x = __builtin_amdgcn_raw_buffer_load_b64(from, at, 0, 0);
        to[0] = x[0];
        to[1] = x[1];
    } else {
        to[0] = __builtin_amdgcn_raw_buffer_load_b32(from, at, 0, 0);
    }
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

    // rows k0 .. k0 + 31 of a cache of `rows` rows
    __device__ __forceinline__ void load_k(const uint8_t *codes, int k0, int rows, int lane) {
        const auto from = q_block<F::kCodes>(codes, k0, rows);
        const uint32_t at = (lane & 15) * F::kCodes + (lane >> 4) * (kKWords == 2 ? 8 : 16);
#pragma unroll
        for (int t = 0; t < 2; ++t) q_words<kKWords>(from, at + 16 * t * F::kCodes, k[t]);
    }
    __device__ __forceinline__ void load_v(const uint8_t *codes, int k0, int rows, int lane) {
        const auto from = q_block<F::kCodes>(codes, k0, rows);
        const uint32_t at = (lane >> 4) * 4 * F::kCodes + (lane & 15) * (HD == 64 && BITS == 4 ? 2 : 4 * kVWords);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t row = at + (16 * (j >> 2) + (j & 3)) * F::kCodes;
            if constexpr (HD == 64 && BITS == 4) v[j][0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(from, row, 0, 0);
            else q_words<kVWords>(from, row, v[j]);
        }
    }
    // what elements of key chunks are to be taken times: of eight, 0 .. 7
    __device__ __forceinline__ static constexpr bool k_upper(int e) { return BITS == 4 && (e >> 1 & 1); }
    __device__ __forceinline__ static constexpr bool v_upper(int t) { return BITS == 4 && (t & 1); }
    // K's operand of chunk c, key tile t
    __device__ __forceinline__ v8h key(int t, int c, uint32_t magic) const { return key_of(k[t], c, magic); }
    __device__ __forceinline__ static v8h key_of(const uint32_t *k, int c, uint32_t magic) {
        v8h r;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v2h x;
            if constexpr (BITS == 4) {
                const uint32_t w = k[c] >> (e & 2 ? 8 : 0);
                x = e & 1 ? code_pair<1024 + 128>(w, 0x00f000f0u, magic) : code_pair<1024 + 8>(w, 0x000f000fu, magic);
            } else {
                x = code_pair<1024 + 128>(__builtin_amdgcn_perm(magic, k[2 * c + e / 2], e & 1 ? 0x05030502u : 0x05010500u), ~0u, 0u);
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
            const v2h x = value_pair(v[j], v[j + 1], t, magic);
            r[j] = x[0];
            r[j + 1] = x[1];
        }
        return r;
    }
    // code t of two keys' words
    __device__ __forceinline__ static v2h value_pair(const uint32_t *a, const uint32_t *b, int t, uint32_t magic) {
        const uint32_t at = BITS == 4 ? t >> 1 : t & 3;  // the byte that holds it
        const int w = BITS == 4 ? 0 : t >> 2;
        const uint32_t two = __builtin_amdgcn_perm(b[w], a[w], 0x0c040c00u + 0x00010001u * at);
        if constexpr (BITS == 4) return t & 1 ? code_pair<1024 + 128>(two, 0x00f000f0u, magic) : code_pair<1024 + 8>(two, 0x000f000fu, magic);
        else return code_pair<1024 + 128>(two, ~0u, magic);
    }
};

// a weight times a step as halves
__device__ __forceinline__ void split_steps(float a, _Float16 sa, float b, _Float16 sb, v2h &hi, v2h &lo) {
    hi = whole_v2h((v2h){(_Float16)__builtin_fmaf(a, (float)sa, 0.0f), (_Float16)__builtin_fmaf(b, (float)sb, 0.0f)});
    lo = (v2h){(_Float16)__builtin_fmaf(a, (float)sa, -(float)hi[0]), (_Float16)__builtin_fmaf(b, (float)sb, -(float)hi[1])};
}

// One query row's part of a score, in a lane of its tile.
struct QQuery {
    float sum;      // of the row's elements of group u, in lane 16u + i (zero where there is none)
    float size;     // a power of two: score = size · product
    float slope;
    int pos;        // the last key it sees
};

// A lane's share of query row r (token, head of the KV head's group), elements 32c +
// 8u .. +7 of it.  Rows behind the last hold the last one's.
template <int HD>
__device__ __forceinline__ void q_fetch(const QAttnCall &p, int s, int g, int r, int u, v4f (&x)[HD / 16]) {
    r = min(r, p.n * p.group - 1);
    const int tok = p.token(r), head = g * p.group + r - tok * p.group;
    const float *src = p.q + s * p.q_ss + tok * p.q_st + head * HD + 8 * u;
#pragma unroll
    for (int c = 0; c < HD / 32; ++c)
#pragma unroll
        for (int e = 0; e < 2; ++e) x[2 * c + e] = *reinterpret_cast<const v4f *>(src + 32 * c + 4 * e);
}

// The same times the scale, as halves below 2^kTop, smaller where they meet the
// upper codes of bytes.
template <int HD, int BITS, bool SHAPED>
__device__ __forceinline__ void q_query(const QAttnCall &p, const QTile &t, int g, int r, int u, const v4f (&y)[HD / 16], v8h (&hi)[HD / 32],
                                        v8h (&lo)[HD / 32], QQuery &q) {
    constexpr int C = HD / 32, G = HD / 64;
    const bool live = r < t.count * p.group;
    const int tok = p.token(live ? r : 0), head = g * p.group + (live ? r - tok * p.group : 0);
    q.pos = live ? t.len - t.count + tok : -1;
    const float scale = SHAPED && p.cap > 0.0f ? p.scale : p.scale * kLog2e;  // a cap takes scores as they are
    float x[C][8];
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[c][e] = live ? y[2 * c + e / 4][e & 3] * scale : 0.0f;
            top = max(top, abs_bits(x[c][e]));
        }
    const int e = row_exp(groups_umax(top));
    const float up = pow2(kTop - e);
    q.sum = 0.0f;
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
        float sum = 0.0f;
#pragma unroll
        for (int c = 2 * gr; c < 2 * gr + 2; ++c)
#pragma unroll
            for (int k = 0; k < 8; ++k) sum += x[c][k] * up;
        sum = groups_sum(sum);
        if (u == gr) q.sum = sum;
    }
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (QCodes<HD, BITS>::k_upper(k)) x[c][k] *= 0.0625f;
    split_row<C>(x, e, hi, lo);
    q.size = pow2(e - kTop);
    q.slope = 0.0f;
    if (SHAPED && p.slopes) {
        const float y = p.slopes[head] * kLog2e;
        q.slope = fabsf(y) == INFINITY ? copysignf(3.4028235e38f, y) : y;
    }
}

// The parameters of a block's 32 keys: a word of K's and of V's a lane, spread over
// the wave's lanes through LDS.
template <int HD>
struct QParams {
    static constexpr int G = HD / 64, kBytes = 32 * 4 * G;  // of K or V
    uint32_t k, v;
    __device__ __forceinline__ static int key_of(int lane) { return HD == 128 ? lane >> 1 : lane & 31; }
    __device__ __forceinline__ static uint32_t word(const uint8_t *par, int k0, int rows, int lane) {
        return __builtin_amdgcn_raw_buffer_load_b32(q_block<4 * G>(par, k0, rows), HD == 128 ? 4 * lane : 4 * (lane & 31), 0, 0);
    }
    __device__ __forceinline__ void load(const uint8_t *kp, const uint8_t *vp, int k0, int rows, int lane) {
        k = word(kp, k0, rows, lane);
        v = word(vp, k0, rows, lane);
    }
    // of the lane's keys 16 · kt + 4u .. +3
    __device__ __forceinline__ static void get(const uint8_t *par, int kt, int u, v8h (&x)[G]) {
#pragma unroll
        for (int i = 0; i < G; ++i) x[i] = *reinterpret_cast<const v8h *>(par + (16 * kt + 4 * u) * 4 * G + 16 * i);
    }
    // of the group gr of key k of those: the step (which 0) or the midpoint
    __device__ __forceinline__ static _Float16 of(const v8h (&x)[G], int k, int gr, int which) {
        const int at = k * 2 * G + which * G + gr;
        return x[at >> 3][at & 7];
    }
};

// Products of a row's halves with keys' codes, d of each group → of the row with the
// keys 16 · kt + 4u .. +3, by the keys' parameters: step · d, and midpoint · sum of the
// row's elements, a matrix product in 32 bits that leaves half of the multiply-adds.
template <int HD>
__device__ __forceinline__ void q_scores(float sum, const uint8_t *par, int kt, int i, int u, const v4f (&d)[HD / 64], float *x) {
    constexpr int G = HD / 64;
    const float mid = (float)reinterpret_cast<const _Float16 *>(par)[(16 * kt + i) * 2 * G + G + (u & (G - 1))];
    const v4f y = __builtin_amdgcn_mfma_f32_16x16x4f32(mid, sum, (v4f){0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
    v8h steps[G];
    QParams<HD>::get(par, kt, u, steps);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        x[k] = y[k];
#pragma unroll
        for (int gr = 0; gr < G; ++gr) x[k] = fmaf((float)QParams<HD>::of(steps, k, gr, 0), d[gr][k], x[k]);
    }
}

// The exponent that brings V's step of these bits below 2^kQTop: step < 2^(exponent - 14),
// subnormal ones < 2^-14.
__device__ __forceinline__ int q_raise(uint32_t step) { return kQTop + 14 - (int)(step >> 10); }

// V's largest step so far in blocks of which all rows see the same, its exponent, and
// whether the present block has parameters that are no numbers.
constexpr uint16_t kQBad = 0x8000;  // in place of such a group's step: no step is a negative zero
struct QScale {
    uint32_t top = 0;  // its bits
    int raise = q_raise(0);
    bool moved = false, bad = false;
    // `v`: a lane's word of V's parameters.  What is no number stays out of products,
    // where it would meet the zero weights of rows that do not see it.  alone: rows see
    // different keys of the block, and each looks for itself (QSums::shape).
    template <int HD>
    __device__ __forceinline__ void look(uint32_t &v, int lane, bool alone) {
        const uint32_t most_seen = alone ? 0x7bffu : top;
        const bool mine = HD == 128 || lane < 32, steps = HD == 64 || !(lane & 1);
        const uint32_t low = v & 0x7fffu, high = v >> 16 & 0x7fffu, none = 0x7bffu;  // none: the largest number
        moved = bad = false;
        if constexpr (HD == 128) {
            if (!__any(max(low, high) > (steps ? most_seen : none))) return;
        } else {
            if (!__any(mine && (low > most_seen || high > none))) return;
        }
        bool b0 = low > none, b1 = high > none;
        bad = __any(mine && (b0 || b1));
        if (bad) {
            if constexpr (HD == 128) {  // the steps of both groups, the midpoints of both: two lanes
                const uint32_t other = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false);
                b0 = b0 || (other & 0x7fffu) > none;
                b1 = b1 || (other >> 16 & 0x7fffu) > none;
                const uint32_t mark = steps ? kQBad : 0u;
                if (b0) v = (v & 0xffff0000u) | mark;
                if (b1) v = (v & 0x0000ffffu) | mark << 16;
            } else {
                if (b0 || b1) v = kQBad;
            }
        }
        if (alone) return;
        uint32_t most = groups_umax(steps ? max(v & 0x7fffu, HD == 128 ? v >> 16 & 0x7fffu : 0u) : 0u);
#pragma unroll
        for (int o = 8; o; o >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o));
        most = (uint32_t)__builtin_amdgcn_readfirstlane((int)most);
        if (most <= top) return;
        top = most;
        const int now = q_raise(most);
        moved = now != raise;
        raise = now;
    }
};

// A row's running sums, in a lane of its tile.  Weights are 2^(score - m + raise), m a
// whole number near the row's largest score, raise the exponent of the largest step of V
// that it has seen: ref is m - raise, and of a row whose m is far from zero -raise, where
// `shape` takes m from its scores.
template <int HD>
struct QSums {
    static constexpr int G = HD / 64, T = HD / 16;
    v4f acc[T];
    float ref = -(kQTop + 14), m = kLowest, total = 0.0f, mids[G];
    bool far = false;  // some row of the wave's
    // what of m its scores lose beforehand
    __device__ __forceinline__ static float apart(float m) { return fabsf(m) >= kQFar ? m : 0.0f; }
    __device__ __forceinline__ float down() const { return ref - (m - apart(m)); }  // -raise
    __device__ __forceinline__ void rescale(float by) {
        total *= by;
#pragma unroll
        for (int gr = 0; gr < G; ++gr) mids[gr] *= by;
#pragma unroll
        for (int k = 0; k < T; ++k) acc[k] *= by;
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int k = 0; k < T; ++k) acc[k] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int gr = 0; gr < G; ++gr) mids[gr] = 0.0f;
    }
    // products x of a block from key k0 on (lane: keys 16 (j / 4) + 4u + j % 4) → scores,
    // but for q.size, and the row's reference.  masked: some row does not see all keys;
    // alone: nor do all see the same, or some of V's parameters are no numbers; raise and
    // moved: of blocks of which all rows see the same.
    template <bool SHAPED>
    __device__ __forceinline__ void shape(const QAttnCall &p, const QQuery &q, int raise, bool moved, float (&x)[8], int k0, int u, bool masked,
                                          bool alone, const v8h (&v)[2][G]) {
        auto key_of = [&](int j) { return k0 + 16 * (j >> 2) + 4 * u + (j & 3); };
        const float size = SHAPED ? 1.0f : q.size;  // exact, so a score may round with its reference
        if (SHAPED) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] *= q.size;
            if (p.cap > 0.0f) {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] *= p.cap_inverse;
                tanh_all<8>(x);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] *= p.cap_log2;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = rounded(fmaf(-q.slope, (float)(q.pos - key_of(j)), x[j]));
        }
        // of key_of(j), as bits of a vector register: eight lane masks are more than the
        // scalar ones hold beside the round's own numbers
        auto sees = [&](int j) {
            const int from = p.window ? max(0, q.pos - p.window + 1) : 0;
            uint32_t bits = (uint32_t)(key_of(j) - from) < (uint32_t)max(0, q.pos + 1 - from) ? ~0u : 0u;
            asm("" : "+v"(bits));
            return bits;
        };
        float least = -(float)raise;  // of -raise
        if (__builtin_expect(masked || alone, 0)) {
            if (masked) {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = __uint_as_float((__float_as_uint(x[j]) & sees(j)) | (0xff800000u & ~sees(j)));
            }
            if (alone) {
                uint32_t most = 0, worst[G] = {};
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int gr = 0; gr < G; ++gr) {
                        const uint32_t step = sees(j) & __builtin_bit_cast(uint16_t, QParams<HD>::of(v[j >> 2], j & 3, gr, 0));
                        worst[gr] = max(worst[gr], step);
                        most = max(most, step & 0x7fffu);
                    }
#pragma unroll
                for (int gr = 0; gr < G; ++gr)  // NaN for the rows that see one, in its group
                    if (worst[gr] == kQBad) mids[gr] = __builtin_nanf("");
                least = fmaxf(least, -(float)q_raise(groups_umax(most)));
                moved = moved || __any(least > down());
            }
        }
        float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7]))) * size;
        if (__any(moved || far || top > m + kQSlack)) {
            top = groups_max(top);
            const float before = apart(m), own = fmaxf(down(), least);
            if (top > m) m = fminf(ceilf(top), 3.0e38f);
            const float less = apart(m), now = m - less + own, by = __builtin_amdgcn_exp2f((before - less) + (ref - now));
            ref = now;
            far = __any(fabsf(m) >= kQFar && m > kLowest);
            rescale(by);
            if (far) {  // `split` multiplies by size again: a power of two
                const float inverse = __uint_as_float(0x7f000000u - __float_as_uint(size));
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = less != 0.0f ? fmaf(x[j], size, -less) * inverse : x[j];
            }
        }
    }
    // scores → weights times V's steps, as halves
    template <bool SHAPED>
    __device__ __forceinline__ void split(const QQuery &q, float (&x)[8], const v8h (&v)[2][G], v8h (&hi)[G], v8h (&lo)[G]) {
        const float size = SHAPED ? 1.0f : q.size;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[j] = __builtin_amdgcn_exp2f(fmaf(x[j], size, -ref));
            total += x[j];
        }
#pragma unroll
        for (int gr = 0; gr < G; ++gr)
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const v8h(&par)[G] = v[j >> 2];
                v2h h, l;
                split_steps(x[j], QParams<HD>::of(par, j & 3, gr, 0), x[j + 1], QParams<HD>::of(par, (j & 3) + 1, gr, 0), h, l);
                hi[gr][j] = h[0];
                hi[gr][j + 1] = h[1];
                lo[gr][j] = l[0];
                lo[gr][j + 1] = l[1];
                mids[gr] = fmaf((float)QParams<HD>::of(par, j & 3, gr, 1), x[j], mids[gr]);
                mids[gr] = fmaf((float)QParams<HD>::of(par, (j & 3) + 1, gr, 1), x[j + 1], mids[gr]);
            }
    }
    // the row's sums over its four lanes; acc in whole
    template <int BITS>
    __device__ __forceinline__ void finish() {
        total = groups_sum(total);
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
            mids[gr] = groups_sum(mids[gr]);
#pragma unroll
            for (int k = 4 * gr; k < 4 * gr + 4; ++k) acc[k] = acc[k] * (QCodes<HD, BITS>::v_upper(k) ? 0.0625f : 1.0f) + mids[gr];
        }
        if (far && apart(m) != 0.0f) {  // the exponent into the sums
            const float by = __builtin_amdgcn_exp2f(ref);
            ref = m;
            total *= by;
#pragma unroll
            for (int k = 0; k < T; ++k) acc[k] *= by;
        }
        if (total == 0.0f) ref = kLowest;
    }
};

// what a tile's row r leaves behind: its part of a share, or its result
__device__ __forceinline__ float *q_out_row(const QAttnCall &p, int s, int g, int r, int hd) {
    const int tok = p.token(r), head = g * p.group + r - tok * p.group;
    return p.out + s * p.o_ss + tok * p.o_st + head * hd;
}
__device__ __forceinline__ void q_out_lse(const QAttnCall &p, int s, int g, int r, float ref, float total) {
    const int tok = p.token(r), head = g * p.group + r - tok * p.group;
    p.lse[((int64_t)s * p.n + tok) * p.heads + head] = total == 0.0f ? -INFINITY : (ref + __builtin_amdgcn_logf(total)) * 0.69314718055994531f;
}

// Attention over codes.  Workgroup: 16 · RT query rows (token, head of the KV head's
// group) of one sequence and KV head; its W waves take the share's blocks of 32 keys
// in turn and join.
//
// Codes go to the matrix instructions as they are, exact in fp16, and meet query
// rows and weights as two fp16 halves each, 22 bits together.  Scores come out
// transposed (lane l: query row l % 16, keys 4 (l / 16) + r of each 16), so a row's
// statistics stay with its four lanes, in 32 bits, and its weights are the second
// product's operand:
//   q . k = sum over groups of step (q . c) + mid (sum of q),
//   out = sum over keys of (p step) . c + sum of p mid.
// p = 2^(s - ref), ref a whole number near the row's largest score, lowered by the
// exponent that brings the largest step of V that the row has seen so far to 2^kQTop, so
// that the halves of p step hold the products that count whatever V's size, and a row's
// precision does not hang on keys that other rows of its tile see.  All rescales are by
// powers of two.  A wave's first block and its query rows do not depend on the sequence's
// length, and are requested with it; a later block's codes as soon as the registers
// of the one before are free.
//
// Few rows are bound by the chain of one wave: launch, lengths and first codes (5 us),
// then 0.7 us a block, sums joined in LDS.  One token of 16 heads on 2 KV heads of 128 in
// 4 bits behind 1,609 rows 9.0 to 9.7 us with the join (two launches over 17 blocks of keys
// 8.9, one over a single block 6.5), in 8 bits 8.9 to 9.8; 16 of them behind up to 8,192
// rows (33 MB) 17.1, without arithmetic 12.8, the join's 3 in both.  Two blocks of a wave
// on their way: 18.0, registers for two workgroups a CU in place of three; two blocks a
// round: one token 10.7.
template <int HD, int BITS, int RT, int W, bool SHAPED>
__global__ void __launch_bounds__(64 * W, RT == 1 && W == 4 ? 3 : 2) k_qcache_attn(QAttnCall p, QAttnPlan pl) {
    using F = QFormat<HD, BITS>;
    using Codes = QCodes<HD, BITS>;
    using Params = QParams<HD>;
    constexpr int C = HD / 32, G = HD / 64, T = HD / 16, kRows = 16 * RT;
    union Shared {
        struct {
            v8h q[RT][C][2][64];
            uint8_t par[W][2][Params::kBytes];
        } in;
        v4f acc[W][RT][T][64];
    };
    __shared__ Shared sh;
    __shared__ QQuery s_query[RT][16];
    __shared__ float s_qsum[RT][64];
    __shared__ float s_ref[W][kRows], s_sum[W][kRows];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = lane & 15, u = lane >> 4;
    const int g = blockIdx.y, s = blockIdx.z;
    const int tile = pl.tiles - 1 - (int)(blockIdx.x / pl.splits), part = blockIdx.x % pl.splits;  // long rows first
    const int64_t base = s * p.cache.seq_rows + (int64_t)g * p.cache.capacity;
    const uint8_t *kc = p.cache.codes[0] + base * F::kCodes, *vc = p.cache.codes[1] + base * F::kCodes;
    const uint8_t *kp = reinterpret_cast<const uint8_t *>(p.cache.params[0] + base * F::kParams);
    const uint8_t *vp = reinterpret_cast<const uint8_t *>(p.cache.params[1] + base * F::kParams);
    const int cap = p.cache.capacity, step = pl.splits * W, first = tile * kRows;
    int block = part * W + wave;
    Codes codes;
    Params par;
    auto load = [&](int at) {
        codes.load_k(kc, at * kQBlock, cap, lane);
        par.load(kp, vp, at * kQBlock, cap, lane);
        codes.load_v(vc, at * kQBlock, cap, lane);
    };
    if (!p.window && block <= (cap - 1) / kQBlock) load(block);
    v4f y[HD / 16];
    if (wave < RT) q_fetch<HD>(p, s, g, first + 16 * wave + i, u, y);
    const QTile t = q_tile(p, s, first, kRows);
    if (!t.count) return;
    const int end = (t.hi + kQBlock - 1) / kQBlock, all = t.count * p.group;
    if (p.window) {
        block += t.lo / kQBlock;
        if (block < end) load(block);
    }
    if (wave < RT) {
        v8h hi[C], lo[C];
        QQuery q;
        q_query<HD, BITS, SHAPED>(p, t, g, first + 16 * wave + i, u, y, hi, lo, q);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            sh.in.q[wave][c][0][lane] = hi[c];
            sh.in.q[wave][c][1][lane] = lo[c];
        }
        if (u == 0) s_query[wave][i] = q;
        s_qsum[wave][lane] = q.sum;
    }
    __syncthreads();
    QQuery query[RT];
    QSums<HD> sums[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        query[rt] = s_query[rt][i];
        query[rt].sum = s_qsum[rt][lane];
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) sums[rt].clear();
    QScale scale;
    const uint32_t magic = code_magic();
    uint8_t *kpar = sh.in.par[wave][0], *vpar = sh.in.par[wave][1];

    for (; block < end; block += step) {
        const int k0 = block * kQBlock, next0 = k0 + step * kQBlock;
        const bool more = block + step < end, masked = t.partly(k0), mixed = masked && t.mixed();
        if (masked) {  // parameters of keys outside the tile's are zero
            const int key = k0 + Params::key_of(lane);
            if (key < t.lo || key >= t.hi) par.k = par.v = 0;
        }
        scale.look<HD>(par.v, lane, mixed);
        if (HD == 128 || lane < 32) {
            reinterpret_cast<uint32_t *>(kpar)[lane] = par.k;
            reinterpret_cast<uint32_t *>(vpar)[lane] = par.v;
        }
        wave_lds_order();
        if (more) par.load(kp, vp, next0, cap, lane);

        float x[RT][8];  // row i, keys 16 · kt + 4u + k
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            v4f d[RT][G];
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const v8h key = codes.key(kt, c, magic);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    const v4f from = c % 2 ? d[rt][c / 2] : (v4f){0.0f, 0.0f, 0.0f, 0.0f};
                    const v4f y = __builtin_amdgcn_mfma_f32_16x16x32_f16(key, sh.in.q[rt][c][0][lane], from, 0, 0, 0);
                    d[rt][c / 2] = __builtin_amdgcn_mfma_f32_16x16x32_f16(key, sh.in.q[rt][c][1][lane], y, 0, 0, 0);
                }
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) q_scores<HD>(query[rt].sum, kpar, kt, i, u, d[rt], x[rt] + 4 * kt);
        }
        if (more) codes.load_k(kc, next0, cap, lane);
        v8h pv[2][G], hi[RT][G], lo[RT][G];
        Params::get(vpar, 0, u, pv[0]);
        Params::get(vpar, 1, u, pv[1]);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            sums[rt].template shape<SHAPED>(p, query[rt], scale.raise, scale.moved, x[rt], k0, u, masked, mixed || scale.bad, pv);
            sums[rt].template split<SHAPED>(query[rt], x[rt], pv, hi[rt], lo[rt]);
        }
#pragma unroll
        for (int k = 0; k < T; ++k) {
            const v8h v = codes.value(k, magic);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                v4f &a = sums[rt].acc[k];
                a = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, hi[rt][k / 4], a, 0, 0, 0);
                a = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, lo[rt][k / 4], a, 0, 0, 0);
            }
        }
        if (more) codes.load_v(vc, next0, cap, lane);
        wave_lds_order();
    }

    // The waves' sums, to the rows' largest reference.  A lane's four numbers of LDS are
    // neighbours: elements 64 (k / 4) + 16u + 4r + k % 4 of dim tiles k, registers r.
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        sums[rt].template finish<BITS>();
        if (u == 0) {
            s_ref[wave][16 * rt + i] = sums[rt].ref;
            s_sum[wave][16 * rt + i] = sums[rt].total;
        }
    }
    __syncthreads();
    float ref[RT], total[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        ref[rt] = kLowest;
        total[rt] = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) ref[rt] = fmaxf(ref[rt], s_ref[w][16 * rt + i]);
#pragma unroll
        for (int w = 0; w < W; ++w) total[rt] += s_sum[w][16 * rt + i] * __builtin_amdgcn_exp2f(s_ref[w][16 * rt + i] - ref[rt]);
    }
    const int64_t slot = ((((int64_t)s * p.cache.kvh + g) * pl.tiles + tile) * pl.splits + part) * kRows;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const float by = __builtin_amdgcn_exp2f(sums[rt].ref - ref[rt]);
#pragma unroll
        for (int k = 0; k < T; ++k) {
            const int gr = k / 4, r = k % 4;
            sh.acc[wave][rt][k][lane] = (v4f){sums[rt].acc[4 * gr][r], sums[rt].acc[4 * gr + 1][r], sums[rt].acc[4 * gr + 2][r], sums[rt].acc[4 * gr + 3][r]} * by;
        }
    }
    __syncthreads();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int row = 16 * rt + i, r = first + row;
        if (r >= all) continue;
        float *dst = pl.splits > 1 ? pl.part + (slot + row) * HD : q_out_row(p, s, g, r, HD);
        const float by = pl.splits > 1 ? 1.0f : (total[rt] == 0.0f ? 0.0f : 1.0f / total[rt]);
#pragma unroll
        for (int k = wave; k < T; k += W) {
            v4f sum = sh.acc[0][rt][k][lane];
#pragma unroll
            for (int w = 1; w < W; ++w) sum += sh.acc[w][rt][k][lane];
            *reinterpret_cast<v4f *>(dst + 64 * (k / 4) + 16 * u + 4 * (k % 4)) = sum * by;
        }
        if (wave == 0 && u == 0) {
            if (pl.splits > 1) pl.stat[slot + row] = make_float2(ref[rt], total[rt]);
            else if (p.lse) q_out_lse(p, s, g, r, ref[rt], total[rt]);
        }
    }
}

// One wave's part of a block's codes on their way into LDS, as the matrix
// instructions take them, for the four waves of a workgroup: 16 bytes a lane for each
// of K's [key tile][chunk] and V's [dim tile].  Of K a wave has whole pieces, of V a
// pair of keys in all dim tiles, so that its loads are words of codes and not their
// bytes; another pair in each of its lane groups, so that its words lie in different
// banks.
template <int HD, int BITS>
struct QLayer {
    using F = QFormat<HD, BITS>;
    static constexpr int C = HD / 32, T = HD / 16, kK = C / 2;  // K's pieces of a wave
    static constexpr int kKBytes = 2 * C * 1024, kVBytes = T * 1024, kWords = BITS / 4;
    static constexpr int kVWords = (T * BITS + 31) / 32;  // of a key's codes in a lane
    uint32_t k[kK * kWords], v[2][kVWords];
    // rows k0 .. k0 + 31 of a cache of `rows` rows
    __device__ __forceinline__ void load_k(const uint8_t *codes, int k0, int rows, int wave, int lane) {
        const uint32_t i = lane & 15, u = lane >> 4, f = wave * kK, c = f % C;  // pieces f, f + 1: neighbours
        const uint32_t part = BITS == 4 ? 4 * (u * C + c) : 64 * (c >> 1) + 16 * u + 8 * (c & 1);
        q_words<kK * kWords>(q_block<F::kCodes>(codes, k0, rows), (16 * (f / C) + i) * F::kCodes + part, k);
    }
    __device__ __forceinline__ void load_v(const uint8_t *codes, int k0, int rows, int wave, int lane) {
        const auto from = q_block<F::kCodes>(codes, k0, rows);
        const uint32_t i = lane & 15, u = lane >> 4, j = 2 * (wave ^ u);  // keys of slots j and j + 1
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const uint32_t at = (16 * (j >> 2) + 4 * u + (j & 3) + n) * F::kCodes + T * BITS / 8 * i;
            if constexpr (T * BITS == 16) v[n][0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(from, at, 0, 0);
            else q_words<kVWords>(from, at, v[n]);
        }
    }
    __device__ __forceinline__ void put_k(uint8_t *to, int wave, int lane, uint32_t magic) const {
#pragma unroll
        for (int n = 0; n < kK; ++n) reinterpret_cast<v8h *>(to)[(wave * kK + n) * 64 + lane] = QCodes<HD, BITS>::key_of(k, n, magic);
    }
    __device__ __forceinline__ void put_v(uint8_t *to, int wave, int lane, uint32_t magic) const {
        v2h *at = reinterpret_cast<v2h *>(to) + 4 * lane + (wave ^ lane >> 4);
#pragma unroll
        for (int t = 0; t < T; ++t) at[256 * t] = QCodes<HD, BITS>::value_pair(v[0], v[1], t, magic);
    }
};

// The same attention for many query rows: four waves of 16 rows take the share's blocks
// together, each unpacking its part of a block's codes into LDS for all of them.
//
// A round of a wave (32 keys, heads of 128) has 34 matrix instructions of 16 cycles or 32
// and about 169 vector instructions of 4, which run beside them only where they lie
// between them: the next block's scores are multiplied among this block's exponentials,
// this block's sums among the unpacking of later codes.  So a round needs the next
// block's keys and this block's values, both in two buffers, and one barrier; codes are
// requested two blocks ahead.  Rounds come in pairs, so that buffers and registers are
// fixed numbers of the code.  From its scores to its sums a wave goes before those of
// other workgroups that unpack or wait, which keeps them apart in their rounds.
//
// 600 tokens of 16 heads on 2 KV heads of 128 in 4 bits behind 8,192 rows: 112 to 125 us
// with the join, 0.31 to 0.35 PFLOP/s and, with two halves each, 0.66 to 0.74 of products
// (1.16 for a large fp16 product); with cap and slopes 162, in 8 bits 122.  Instructions
// bound it, at three waves to a SIMD: vector ones take 46 % of the cycles, matrix ones 39 %,
// LDS 41 %; a wave waits for its turn to issue for 36 % of its time.  With cap or slopes, in
// 4 bits, seven registers spill.
// At least and at most so many waves to a SIMD: told the least alone, the compiler spares
// registers for more than fit, and the 8-bit kernel's vector instructions end up in one
// piece behind its matrix ones (540 tokens 128 us for 136).
// Eight waves a workgroup took 143 us where four took 138; codes one round ahead 135
// where this takes 129; 32 rows a wave spilled 22 registers and took 177 where 16 took
// 136; four sums of scores at a time in place of two, spilled too, 143 where two took
// 126; without the priorities 117 where this takes 112.
template <int HD, int BITS, bool SHAPED>
__global__ void __launch_bounds__(256)
    __attribute__((amdgpu_waves_per_eu(HD == 128 && BITS == 4 ? 3 : 2, HD == 64 ? 4 : BITS == 8 ? 2 : 3))) k_qcache_attn_rows(QAttnCall p, QAttnPlan pl) {
    using F = QFormat<HD, BITS>;
    using Layer = QLayer<HD, BITS>;
    using Params = QParams<HD>;
    constexpr int C = HD / 32, G = HD / 64, T = HD / 16, kRows = 64;
    __shared__ __attribute__((aligned(16))) uint8_t s_k[2][Layer::kKBytes], s_v[2][Layer::kVBytes];
    __shared__ __attribute__((aligned(16))) uint8_t s_kpar[2][Params::kBytes], s_vpar[2][Params::kBytes];
    __shared__ int2 s_raise[2];  // what V's parameters ask for: QScale's raise and bad

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = lane & 15, u = lane >> 4;
    const int g = blockIdx.y, s = blockIdx.z;
    const int tile = pl.tiles - 1 - (int)(blockIdx.x / pl.splits), part = blockIdx.x % pl.splits;  // long rows first
    const int64_t base = s * p.cache.seq_rows + (int64_t)g * p.cache.capacity;
    const uint8_t *kc = p.cache.codes[0] + base * F::kCodes, *vc = p.cache.codes[1] + base * F::kCodes;
    const uint8_t *kp = reinterpret_cast<const uint8_t *>(p.cache.params[0] + base * F::kParams);
    const uint8_t *vp = reinterpret_cast<const uint8_t *>(p.cache.params[1] + base * F::kParams);
    const int cap = p.cache.capacity, step = pl.splits * kQBlock, first = tile * kRows + 16 * wave;
    int k0 = part * kQBlock;  // of this round's block

    Layer layer[2];  // of blocks of even and of odd number
    const uint32_t magic = code_magic();
    uint32_t par[2];  // a word of their parameters: wave 0 K's, the others V's
    auto load_par = [&](int from) { return Params::word(wave ? vp : kp, from, cap, lane); };
    auto load_first = [&] {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            layer[n].load_k(kc, k0 + n * step, cap, wave, lane);
            par[n] = load_par(k0 + n * step);
            layer[n].load_v(vc, k0 + n * step, cap, wave, lane);
        }
    };
    if (!p.window) load_first();
    v4f y[HD / 16];
    q_fetch<HD>(p, s, g, first + i, u, y);
    const QTile wt = q_tile(p, s, tile * kRows, kRows);
    if (!wt.count) return;
    const int all = wt.count * p.group;
    if (p.window) {
        k0 += wt.lo / kQBlock * kQBlock;
        load_first();
    }
    v8h qh[C], ql[C];
    QQuery query;
    QSums<HD> sums;
    q_query<HD, BITS, SHAPED>(p, wt, g, first + i, u, y, qh, ql, query);
    sums.clear();
    // parameters of the block from key `from` on for the waves, those of keys outside
    // the tile's as zeros, and the load of those two blocks later
    QScale scale;  // wave 1's
    auto put_par = [&](auto number, int from) {
        constexpr int N = decltype(number)::value;
        if (wave < 2) {
            const int key = from + Params::key_of(lane);
            uint32_t w = par[N];
            const bool masked = wt.partly(from);
            if (masked && (key < wt.lo || key >= wt.hi)) w = 0;
            if (wave) {
                scale.look<HD>(w, lane, masked);
                if (lane == 0) s_raise[N] = make_int2(scale.raise, scale.bad);
            }
            if (HD == 128 || lane < 32) reinterpret_cast<uint32_t *>(wave ? s_vpar[N] : s_kpar[N])[lane] = w;
        }
        par[N] = load_par(from + 2 * step);
    };
    layer[0].put_k(s_k[0], wave, lane, magic);
    put_par(std::integral_constant<int, 0>{}, k0);
    layer[0].load_k(kc, k0 + 2 * step, cap, wave, lane);
    __syncthreads();
    v4f d[2][G];
    // two sums at a time: one product does not wait for the one before
    auto multiply = [&](const uint8_t *codes) {
        const v8h *kf = reinterpret_cast<const v8h *>(codes) + lane;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                v8h key[G];
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int gr = 0; gr < G; ++gr) {
                        if (half == 0) key[gr] = kf[(kt * C + 2 * gr + c) * 64];
                        const v4f from = c || half ? d[kt][gr] : (v4f){0.0f, 0.0f, 0.0f, 0.0f};
                        d[kt][gr] = __builtin_amdgcn_mfma_f32_16x16x32_f16(key[gr], half ? ql[2 * gr + c] : qh[2 * gr + c], from, 0, 0, 0);
                    }
            }
    };
    multiply(s_k[0]);
    layer[1].put_k(s_k[1], wave, lane, magic);
    layer[0].put_v(s_v[0], wave, lane, magic);
    layer[1].load_k(kc, k0 + 3 * step, cap, wave, lane);
    layer[0].load_v(vc, k0 + 2 * step, cap, wave, lane);
    int raise = q_raise(0);  // as QScale begins
    // the round of a block of even (N 0) or odd number; k0 moves on
    auto round = [&](auto number) {
        constexpr int N = decltype(number)::value;
        __syncthreads();
        put_par(std::integral_constant<int, 1 - N>{}, k0 + step);
        const int2 ask = s_raise[N];  // into scalar registers where they are used (at once: a chunk 113.6 us for 112.4)
        float x[8];  // row i, keys 16 · kt + 4u + k
        v8h pv[2][G];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            q_scores<HD>(query.sum, s_kpar[N], kt, i, u, d[kt], x + 4 * kt);
            Params::get(s_vpar[N], kt, u, pv[kt]);
        }
        __builtin_amdgcn_s_setprio(1);
        const int asked = __builtin_amdgcn_readfirstlane(ask.x);
        const bool rare = wt.partly(k0) || __builtin_amdgcn_readfirstlane(ask.y);
        sums.template shape<SHAPED>(p, query, asked, asked != raise, x, k0, u, rare, rare, pv);
        raise = asked;
        v8h hi[G], lo[G];
        multiply(s_k[1 - N]);
        sums.template split<SHAPED>(query, x, pv, hi, lo);
        const v8h *vf = reinterpret_cast<const v8h *>(s_v[N]) + lane;
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
            v8h v[4];
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (half == 0) v[k] = vf[(4 * gr + k) * 64];
                    v4f &a = sums.acc[4 * gr + k];
                    a = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[k], half ? lo[gr] : hi[gr], a, 0, 0, 0);
                }
        }
        __builtin_amdgcn_s_setprio(0);
        layer[N].put_k(s_k[N], wave, lane, magic);
        layer[1 - N].put_v(s_v[1 - N], wave, lane, magic);
        layer[N].load_k(kc, k0 + 4 * step, cap, wave, lane);
        layer[1 - N].load_v(vc, k0 + 3 * step, cap, wave, lane);
        k0 += step;
    };
    for (int left = (wt.hi - k0 + step - 1) / step; left > 0; left -= 2) {
        round(std::integral_constant<int, 0>{});
        if (left > 1) round(std::integral_constant<int, 1>{});
    }
    const int64_t slot = ((((int64_t)s * p.cache.kvh + g) * pl.tiles + tile) * pl.splits + part) * kRows;
    sums.template finish<BITS>();
    const int r = first + i, row = r - tile * kRows;
    if (r >= all) return;
    float *dst = pl.splits > 1 ? pl.part + (slot + row) * HD : q_out_row(p, s, g, r, HD);
    const float by = pl.splits > 1 ? 1.0f : (sums.total == 0.0f ? 0.0f : 1.0f / sums.total);
#pragma unroll
    for (int k = 0; k < T; ++k) {
        const int gr = k / 4, e = k % 4;
        *reinterpret_cast<v4f *>(dst + 64 * gr + 16 * u + 4 * e) =
            (v4f){sums.acc[4 * gr][e], sums.acc[4 * gr + 1][e], sums.acc[4 * gr + 2][e], sums.acc[4 * gr + 3][e]} * by;
    }
    if (u == 0) {
        if (pl.splits > 1) pl.stat[slot + row] = make_float2(sums.ref, sums.total);
        else if (p.lse) q_out_lse(p, s, g, r, sums.ref, sums.total);
    }
}

// A tile's shares joined: HD / 4 lanes a row and share, N shares at a time, the sums of
// each to the largest reference.  3 to 4 us under a trace, launch and one round of loads.
template <int HD, int ROWS, int N>
__global__ void __launch_bounds__(256) k_qcache_join(QAttnCall p, QAttnPlan pl) {
    constexpr int L = HD / 4, U = 256 / L, R = U / N;  // rows of a workgroup
    __shared__ float s_ref[U], s_sum[U];
    __shared__ v4f s_acc[U][L];
    const int i = threadIdx.x % L, unit = threadIdx.x / L, g = blockIdx.y, s = blockIdx.z;
    const int tile = blockIdx.x / (ROWS / R), row = (int)(blockIdx.x % (ROWS / R)) * R + unit / N, from = unit % N;
    const int r = tile * ROWS + row;
    const int64_t at = ((((int64_t)s * p.cache.kvh + g) * pl.tiles + tile) * pl.splits) * ROWS + row;
    const int count = p.counts ? min(max(p.counts[s], 0), p.n) : p.n;
    const bool live = r < count * p.group;  // other rows' slots hold nothing
    float ref = kLowest, total = 0.0f;
    v4f sum = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
    if (live) {
#pragma unroll 4
        for (int k = from; k < pl.splits; k += N) {
            const float2 st = pl.stat[at + (int64_t)k * ROWS];
            const v4f x = *reinterpret_cast<const v4f *>(pl.part + (at + (int64_t)k * ROWS) * HD + 4 * i);
            const float top = fmaxf(ref, st.x), a = __builtin_amdgcn_exp2f(ref - top), b = __builtin_amdgcn_exp2f(st.x - top);
            sum = sum * a + x * b;
            total = total * a + st.y * b;
            ref = top;
        }
    }
    if (N > 1) {
        if (i == 0) {
            s_ref[unit] = ref;
            s_sum[unit] = total;
        }
        s_acc[unit][i] = sum;
        __syncthreads();
        if (from) return;
        float top = ref;
#pragma unroll
        for (int k = 1; k < N; ++k) top = fmaxf(top, s_ref[unit + k]);
        const float a = __builtin_amdgcn_exp2f(ref - top);
        sum *= a;
        total *= a;
#pragma unroll
        for (int k = 1; k < N; ++k) {
            const float b = __builtin_amdgcn_exp2f(s_ref[unit + k] - top);
            sum += s_acc[unit + k][i] * b;
            total += s_sum[unit + k] * b;
        }
        ref = top;
    }
    if (!live) return;
    *reinterpret_cast<v4f *>(q_out_row(p, s, g, r, HD) + 4 * i) = sum * (total == 0.0f ? 0.0f : 1.0f / total);
    if (p.lse && i == 0) q_out_lse(p, s, g, r, ref, total);
}

}  // namespace pocr
