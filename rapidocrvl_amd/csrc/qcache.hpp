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

// Where lane i's elements 8i .. 8i+7 of a row lie among its codes: K's in one
// piece of BITS bytes; V's, for heads of 128, as halves of two pieces, which lane
// i ^ 8 shares.
template <int HD, int BITS>
__device__ __forceinline__ int k_place(int i) {
    const int c = i >> 2, u = i & 3;  // elements 32c + 8u
    return BITS == 4 ? 4 * (u * (HD / 32) + c) : 64 * (c >> 1) + 16 * u + 8 * (c & 1);
}

// lane i's 8 elements of a K (V) row: mid + step * code, one rounding
template <int HD, int BITS, bool V>
__device__ __forceinline__ void q_values(const uint8_t *codes, const _Float16 *params, int i, float (&x)[8]) {
    using F = QFormat<HD, BITS>;
    const float step = params[i >> 3], mid = params[F::kGroups + (i >> 3)];
    int c[8];
    if constexpr (BITS == 4) {
        uint32_t w;
        if (V && HD == 128) {
            const uint32_t sh = 16 * (i >> 3);
            const uint2 d = *reinterpret_cast<const uint2 *>(codes + 8 * (i & 7));
            w = (d.x >> sh & 0xffffu) | (d.y >> sh) << 16;
        } else {
            w = *reinterpret_cast<const uint32_t *>(codes + (V ? 4 * i : k_place<HD, BITS>(i)));
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e] = w >> 4 * (V ? e : (e >> 1) + 4 * (e & 1)) & 15;
    } else {
        uint2 d;
        if (V && HD == 128) {
            const uint8_t *at = codes + 16 * (i & 7) + 4 * (i >> 3);
            d = make_uint2(*reinterpret_cast<const uint32_t *>(at), *reinterpret_cast<const uint32_t *>(at + 8));
        } else {
            d = *reinterpret_cast<const uint2 *>(codes + (V ? 8 * i : k_place<HD, BITS>(i)));
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e] = (e < 4 ? d.x : d.y) >> 8 * (e & 3) & 255;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmaf((float)(c[e] - F::kHalf), step, mid);
}

// Eight lanes hold a group's 64 elements; writes lane i's codes and the group's
// parameters.  64-bit arithmetic, so that a code next to a border is the one of
// the definition whatever computed it.
template <int HD, int BITS, bool V>
__device__ __forceinline__ void q_store(float (&x)[8], uint8_t *codes, _Float16 *params, int i) {
    using F = QFormat<HD, BITS>;
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, abs_bits(x[e]));
    float lo = INFINITY, hi = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        x[e] = fminf(fmaxf(x[e], -65504.0f), 65504.0f);
        lo = fminf(lo, x[e]);
        hi = fmaxf(hi, x[e]);
    }
    auto over = [&](auto step) {
        constexpr int S = decltype(step)::value;
        top = max(top, __float_as_uint(xchg<S>(__uint_as_float(top))));
        lo = fminf(lo, xchg<S>(lo));
        hi = fmaxf(hi, xchg<S>(hi));
    };
    over(std::integral_constant<int, XQ1>{});
    over(std::integral_constant<int, XQ2>{});
    over(std::integral_constant<int, XM8>{});
    const bool bad = top >= 0x7f800000u;  // a NaN or an infinity
    constexpr double kUp = F::kHalf - 1, kDown = F::kHalf;
    // `rounded`: to fp32 first, which the compiler would skip
    _Float16 mid = (_Float16)rounded((float)((kUp * (double)lo + kDown * (double)hi) * (1.0 / (kUp + kDown))));
    const double need = fmax(((double)hi - (double)mid) * (1.0 / kUp), ((double)mid - (double)lo) * (1.0 / kDown));
    _Float16 step = (_Float16)rounded((float)need);
    if ((double)step < need) step = __builtin_bit_cast(_Float16, (uint16_t)(__builtin_bit_cast(uint16_t, step) + 1));
    const double inv = step > (_Float16)0 ? 1.0 / (double)step : 0.0;
    if (bad) step = mid = __builtin_bit_cast(_Float16, (uint16_t)0x7e00);
    uint32_t c[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const double t = fmin(fmax(rint(((double)x[e] - (double)mid) * inv), -kDown), kUp);
        c[e] = bad ? 0u : (uint32_t)((int)t + F::kHalf);
    }
    if ((i & 7) == 0) {
        params[i >> 3] = step;
        params[F::kGroups + (i >> 3)] = mid;
    }
    if constexpr (BITS == 4) {
        uint32_t w = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) w |= c[e] << 4 * (V ? e : (e >> 1) + 4 * (e & 1));
        if (V && HD == 128) {  // words 2i' and 2i'+1 of lanes i' and i' + 8: each writes one
            const uint32_t other = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0x128, 0xF, 0xF, false);  // lane ^ 8
            w = i < 8 ? (w & 0xffffu) | other << 16 : (other >> 16) | (w & 0xffff0000u);
            *reinterpret_cast<uint32_t *>(codes + 8 * (i & 7) + 4 * (i >> 3)) = w;
        } else {
            *reinterpret_cast<uint32_t *>(codes + (V ? 4 * i : k_place<HD, BITS>(i))) = w;
        }
    } else {
        const uint2 d = make_uint2(c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24, c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24);
        if (V && HD == 128) {
            uint8_t *at = codes + 16 * (i & 7) + 4 * (i >> 3);
            *reinterpret_cast<uint32_t *>(at) = d.x;
            *reinterpret_cast<uint32_t *>(at + 8) = d.y;
        } else {
            *reinterpret_cast<uint2 *>(codes + (V ? 8 * i : k_place<HD, BITS>(i))) = d;
        }
    }
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

// Wave: one token, `per` of its heads.  A lane has 8 neighbouring elements of a
// head (a head of 128: 16 lanes); the token's angles are computed once, one a
// lane, and go through LDS to the lanes of every head.
template <int HD, int BITS>  // BITS 0: fp32 destinations
__global__ void __launch_bounds__(256) k_rows(RowsCall p) {
    constexpr int L = HD / 8, U = 64 / L;
    __shared__ double2 s_turn[4][HD / 2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, s = blockIdx.y, i = lane % L;
    const int64_t job = (int64_t)blockIdx.x * 4 + wave;
    const int tok = (int)(job / p.chunks), chunk = (int)(job % p.chunks);
    const int count = p.counts ? min(max(p.counts[s], 0), p.n) : p.n;
    if (tok >= count) return;
    const int64_t row = (p.first ? min(max(p.first[s], 0), p.rows - count) : 0) + tok;
    if (p.positions) {
        if (lane < p.half)
            s_turn[wave][lane] = turn((double)p.positions[((int64_t)s * p.n + tok) * p.axes + axis_of(p, lane)] * p.freqs[lane]);
        wave_lds_order();
    }
    const int last = min(p.end[2], (chunk + 1) * p.per);
    for (int u0 = chunk * p.per; u0 < last; u0 += U) {
        const int u = u0 + lane / L;
        const bool live = u < last;
        const int kind = u < p.end[0] ? 0 : (u < p.end[1] ? 1 : 2), head = !live ? 0 : u - (kind ? p.end[kind - 1] : 0);
        float x[8];
        if (live) {
            const float *src = p.src[kind] + s * p.src_ss[kind] + tok * p.src_st[kind] + head * HD + 8 * i;
#pragma unroll
            for (int e = 0; e < 8; e += 4) *reinterpret_cast<v4f *>(x + e) = *reinterpret_cast<const v4f *>(src + e);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = 0.0f;
        }
        if (kind < 2) {
            const float *w = p.norm[kind];
            double r = 1.0, y[8];
            if (w) {
                double sum = 0.0;
#pragma unroll
                for (int e = 0; e < 8; ++e) sum = fma((double)x[e], (double)x[e], sum);
                sum += xchg<XQ1>(sum);
                sum += xchg<XQ2>(sum);
                sum += xchg<XM8>(sum);
                if (HD == 128) sum += xchg<XM16>(sum);
                r = 1.0 / sqrt(sum / HD + (double)p.eps);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = w ? (double)x[e] * r * (double)w[8 * i + e] : (double)x[e];
            if (p.positions) {
                if (p.adjacent) {
                    if (8 * i < 2 * p.half)
#pragma unroll
                        for (int e = 0; e < 8; e += 2) {
                            const double2 t = s_turn[wave][4 * i + e / 2];
                            const double a = y[e], b = y[e + 1];
                            y[e] = a * t.x - b * t.y;
                            y[e + 1] = b * t.x + a * t.y;
                        }
                } else {
                    const int far = p.half / 8;  // lanes to a pair's other element
                    const bool low = i < far;
                    const int from = (lane & ~(L - 1)) + (low ? i + far : i - far);
                    float o[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) o[e] = __shfl(x[e], from & 63);
                    if (i < 2 * far)
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int at = 8 * (low ? i + far : i - far) + e;
                            const double2 t = s_turn[wave][8 * (low ? i : i - far) + e];
                            const double b = w ? (double)o[e] * r * (double)w[at] : (double)o[e];
                            y[e] = low ? y[e] * t.x - b * t.y : y[e] * t.x + b * t.y;
                        }
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = (float)y[e];
        }
        if (!live) continue;
        if (BITS && kind) {
            constexpr int B = BITS ? BITS : 4;
            using F = QFormat<HD, B>;
            const int64_t at = s * p.cache.seq_rows + (int64_t)head * p.cache.capacity + row;
            if (kind == 1) q_store<HD, B, false>(x, p.cache.codes[0] + at * F::kCodes, p.cache.params[0] + at * F::kParams, i);
            else q_store<HD, B, true>(x, p.cache.codes[1] + at * F::kCodes, p.cache.params[1] + at * F::kParams, i);
        } else {
            float *dst = p.dst[kind] + s * p.dst_ss[kind] + (kind ? row : tok) * p.dst_st[kind] + head * HD + 8 * i;
#pragma unroll
            for (int e = 0; e < 8; e += 4) *reinterpret_cast<v4f *>(dst + e) = *reinterpret_cast<const v4f *>(x + e);
        }
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
        float *dst = p.dst[V] + s * p.dst_ss[V] + t * p.dst_st[V] + g * HD + 8 * i;
#pragma unroll
        for (int e = 0; e < 8; e += 4) *reinterpret_cast<v4f *>(dst + e) = *reinterpret_cast<const v4f *>(x + e);
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

// One query row (token, head) a workgroup, HD / 8 lanes a key: products, softmax
// and sums in fp32, one pass.
template <int HD, int BITS>
__global__ void __launch_bounds__(256) k_qcache_attn(QAttnCall p) {
    using F = QFormat<HD, BITS>;
    constexpr int L = HD / 8, U = 256 / L;
    __shared__ float s_m[U], s_l[U], s_acc[U][HD];
    const int i = threadIdx.x % L, unit = threadIdx.x / L, tok = blockIdx.x, h = blockIdx.y, s = blockIdx.z;
    const int count = p.counts ? min(max(p.counts[s], 0), p.n) : p.n;
    if (tok >= count) return;
    const int len = min(max(p.lens[s], 0), p.max_rows), pos = len - count + tok;
    const int from = p.window ? max(0, pos - p.window + 1) : 0;
    const float slope = p.slopes ? p.slopes[h] : 0.0f;
    float q[8], acc[8] = {};
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = p.q[s * p.q_ss + tok * p.q_st + h * HD + 8 * i + e];
    float m = -INFINITY, l = 0.0f;
    const int64_t base = s * p.cache.seq_rows + (int64_t)(h / p.group) * p.cache.capacity;
    for (int j = from + unit; j <= pos; j += U) {
        const int64_t at = base + j;
        float x[8];
        q_values<HD, BITS, false>(p.cache.codes[0] + at * F::kCodes, p.cache.params[0] + at * F::kParams, i, x);
        float d = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) d = fmaf(q[e], x[e], d);
        d += xchg<XQ1>(d);
        d += xchg<XQ2>(d);
        d += xchg<XM8>(d);
        if (HD == 128) d += xchg<XM16>(d);
        d *= p.scale;
        if (p.cap > 0.0f) d = p.cap * tanhf(d / p.cap);
        d -= slope * (float)(pos - j);
        const float top = fmaxf(m, d);
        const float keep = m == top ? 1.0f : expf(m - top), w = expf(d - top);
        l = l * keep + w;
        m = top;
        q_values<HD, BITS, true>(p.cache.codes[1] + at * F::kCodes, p.cache.params[1] + at * F::kParams, i, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = fmaf(w, x[e], acc[e] * keep);
    }
    if (i == 0) {
        s_m[unit] = m;
        s_l[unit] = l;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) s_acc[unit][8 * i + e] = acc[e];
    __syncthreads();
    const int d = threadIdx.x;
    if (d >= HD) return;
    float top = -INFINITY, total = 0.0f, sum = 0.0f;
    for (int k = 0; k < U; ++k) top = fmaxf(top, s_m[k]);
    for (int k = 0; k < U; ++k) {
        if (s_l[k] == 0.0f) continue;
        const float f = s_m[k] == top ? 1.0f : expf(s_m[k] - top);
        total += s_l[k] * f;
        sum += s_acc[k][d] * f;
    }
    p.out[s * p.o_ss + tok * p.o_st + h * HD + d] = total == 0.0f ? 0.0f : sum / total;
    if (p.lse && d == 0) p.lse[((int64_t)s * p.n + tok) * p.heads + h] = total == 0.0f ? -INFINITY : top + logf(total);
}

}  // namespace pocr
