// cache_ops.hpp — kernels of the cache operators: masked prompt attention,
// attention of drafted trees, accumulated weights, row selection and
// compaction, over fp32 caches the caller owns.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

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
    float scale, cap;
};

constexpr float kLog2e = 1.4426950408889634f;

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

// s = scale·q·k with the cap and the distance bias applied
__device__ __forceinline__ float shape_score(float dot, float scale, float cap, float slope, int dist) {
    float s = dot * scale;
    if (cap > 0.0f) s = cap * tanhf(s / cap);
    return s - slope * fabsf((float)dist);
}

// One workgroup per (token, head, sequence), one key per wave and step: each
// lane holds head_dim / 64 dims, an online softmax per wave, joined at the end.
template <int HD, bool TREE>
__global__ void __launch_bounds__(256) k_cache_attn_rows(CacheAttn p) {
    constexpr int D = HD / 64;
    __shared__ float sm[4], sl[4], sacc[4][HD];
    __shared__ uint64_t sbits[64];
    __shared__ int sdepth[64];
    const int t = blockIdx.x, h = blockIdx.y, s = blockIdx.z, g = h / p.group;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int lo = 0, hi = 0, len = p.rows, count = p.n, own = p.rows0 + t;
    if (TREE) {
        const SeqRows r = seq_rows(p, s);
        len = r.len;
        count = r.count;
        if (t >= count) return;
        if (wave == 0) {
            const uint64_t b = tree_bits(p.parents ? p.parents + (size_t)s * p.n : nullptr, p.n, lane);
            sbits[lane] = b;
            sdepth[lane] = __popcll(b) - 1;
        }
        __syncthreads();
        hi = len + count;
    } else {
        hi = p.end ? min(max(p.end[t], 0), p.rows) : p.rows0 + t + 1;
        lo = p.begin ? min(max(p.begin[t], 0), p.rows) : 0;
    }
    const int32_t *pos = TREE && p.pos ? p.pos + ((size_t)s * p.kvh + g) * p.side : nullptr;
    const uint64_t bits = TREE ? sbits[t] : 0;
    if (TREE) own = pos ? pos[len + t] : len + sdepth[t];
    const float slope = p.slopes ? p.slopes[h] : 0.0f;
    float q[D], acc[D];
#pragma unroll
    for (int d = 0; d < D; ++d) {
        q[d] = p.q[s * p.q_ss + t * p.q_st + h * HD + 64 * d + lane];
        acc[d] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    for (int j = lo + wave; j < hi; j += 4) {
        if (TREE && j >= len && !(bits >> (j - len) & 1)) continue;
        float dot = 0.0f;
#pragma unroll
        for (int d = 0; d < D; ++d) dot = fmaf(q[d], p.k[s * p.k_ss + j * p.k_st + g * HD + 64 * d + lane], dot);
        const int at = TREE ? (pos ? pos[j] : (j < len ? j : len + sdepth[j - len])) : j;
        const float x = shape_score(wave_sum(dot), p.scale, p.cap, slope, own - at);
        const float mn = fmaxf(m, x);
        const float old = m == -INFINITY ? 0.0f : expf(m - mn), e = expf(x - mn);
        l = l * old + e;
#pragma unroll
        for (int d = 0; d < D; ++d) acc[d] = acc[d] * old + e * p.v[s * p.v_ss + j * p.v_st + g * HD + 64 * d + lane];
        m = mn;
    }
    if (lane == 0) {
        sm[wave] = m;
        sl[wave] = l;
    }
#pragma unroll
    for (int d = 0; d < D; ++d) sacc[wave][64 * d + lane] = acc[d];
    __syncthreads();
    if (wave) return;
    float mm = -INFINITY, ll = 0.0f;
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, sm[w]);
    float o[D] = {};
    for (int w = 0; w < 4; ++w) {
        const float e = sm[w] == -INFINITY ? 0.0f : expf(sm[w] - mm);
        ll += sl[w] * e;
#pragma unroll
        for (int d = 0; d < D; ++d) o[d] += sacc[w][64 * d + lane] * e;
    }
    const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
#pragma unroll
    for (int d = 0; d < D; ++d) p.out[s * p.o_ss + t * p.o_st + h * HD + 64 * d + lane] = o[d] * inv;
    if (p.lse && lane == 0) p.lse[((size_t)s * p.n + t) * p.heads + h] = mm + logf(ll);
}

// One wave per (row, KV head, sequence): the weights of its tokens and heads, in order.
template <int HD>
__global__ void __launch_bounds__(64) k_cache_weights_rows(CacheAttn p) {
    constexpr int D = HD / 64;
    const int j = blockIdx.x, g = blockIdx.y, s = blockIdx.z, lane = threadIdx.x;
    const SeqRows r = seq_rows(p, s);
    if (j >= r.len + r.count) return;
    const uint64_t bits = tree_bits(p.parents ? p.parents + (size_t)s * p.n : nullptr, p.n, lane);
    const int32_t *pos = p.pos ? p.pos + ((size_t)s * p.kvh + g) * p.side : nullptr;
    const int depth_j = j < r.len ? 0 : __popcll(__shfl((unsigned long long)bits, j - r.len)) - 1;
    const int at = pos ? pos[j] : (j < r.len ? j : r.len + depth_j);
    float k[D];
#pragma unroll
    for (int d = 0; d < D; ++d) k[d] = p.k[s * p.k_ss + j * p.k_st + g * HD + 64 * d + lane];
    float w = 0.0f;
    for (int t = 0; t < r.count; ++t) {
        const uint64_t b = __shfl((unsigned long long)bits, t);
        if (p.take && !(p.take[s] >> t & 1)) continue;
        if (j >= r.len && !(b >> (j - r.len) & 1)) continue;
        const int own = pos ? pos[r.len + t] : r.len + __popcll(b) - 1;
        for (int h = g * p.group; h < (g + 1) * p.group; ++h) {
            float dot = 0.0f;
#pragma unroll
            for (int d = 0; d < D; ++d) dot = fmaf(p.q[s * p.q_ss + t * p.q_st + h * HD + 64 * d + lane], k[d], dot);
            const float x = shape_score(wave_sum(dot), p.scale, p.cap, p.slopes ? p.slopes[h] : 0.0f, own - at);
            const float lse = p.lse[((size_t)s * p.n + t) * p.heads + h];
            if (lse != -INFINITY) w += expf(x - lse);
        }
    }
    if (lane == 0) p.weights[((size_t)s * p.kvh + g) * p.side + j] += w;
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
// between sinks and recent by four histogram passes over its bytes (integer
// counts: the order of the atomics does not matter), then one pass that writes
// the kept rows in order: a wave owns 64·KPT consecutive rows of a tile, so a
// row's place is a count of ballots.  KPT rows per thread and tile; where one
// tile holds the cache its keys are read once and stay in registers.
template <int KPT>
__global__ void __launch_bounds__(kSelThreads) k_cache_select(CacheSelect p) {
    constexpr int kTile = kSelThreads * KPT;
    __shared__ int hist[256];
    __shared__ int s_bin, s_need;
    __shared__ int s_eq[kSelWaves], s_gt[kSelWaves];
    const int g = blockIdx.x, c = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int len = min(max(p.lens[c], 0), p.max_rows);
    int32_t *kept = p.kept + ((size_t)c * p.kvh + g) * p.budget;
    if (g == 0 && tid == 0) p.counts[c] = min(len, p.budget);
    if (len <= p.budget) {
        for (int j = tid; j < len; j += kSelThreads) kept[j] = j;
        return;
    }
    const float *w = p.weights + ((size_t)c * p.kvh + g) * p.side;
    const int first = p.sinks, last = len - p.recent;  // candidates [first, last): more than `need` of them
    int need = p.budget - p.sinks - p.recent;
    const int tiles = (len + kTile - 1) / kTile;
    uint32_t key[KPT];
    auto load = [&](int tile) {
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            const int j = tile * kTile + (wave * KPT + i) * 64 + lane;
            key[i] = j >= first && j < last ? weight_key(w[j]) : 0u;
        }
    };
    uint32_t prefix = 0, mask = 0;
    if (need > 0)
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256; i += kSelThreads) hist[i] = 0;
            __syncthreads();
            for (int tile = 0; tile < tiles; ++tile) {
                if (tiles > 1 || shift == 24) load(tile);
#pragma unroll
                for (int i = 0; i < KPT; ++i) {
                    const int j = tile * kTile + (wave * KPT + i) * 64 + lane;
                    if (j >= first && j < last && (key[i] & mask) == prefix) atomicAdd(&hist[key[i] >> shift & 255], 1);
                }
            }
            __syncthreads();
            if (wave == 0) {  // lane l: bins 255 - 4l .. 252 - 4l, from the top
                int n[4], sum = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    n[i] = hist[255 - 4 * lane - i];
                    sum += n[i];
                }
                int above = sum;
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) {
                    const int x = __shfl_up(above, o);
                    if (lane >= o) above += x;
                }
                above -= sum;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (above < need && above + n[i] >= need) {
                        s_bin = 255 - 4 * lane - i;
                        s_need = need - above;
                    }
                    above += n[i];
                }
            }
            __syncthreads();
            prefix |= (uint32_t)s_bin << shift;
            mask |= 255u << shift;
            need = s_need;  // how many keys equal to prefix are taken, after the last pass
        }
    const bool none = p.budget == p.sinks + p.recent;
    int done = 0, eq_done = 0;  // rows written, equal keys met
    for (int tile = 0; tile < tiles; ++tile) {
        if (tiles > 1 || none) load(tile);
        int gt = 0, eq = 0;
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            const int j = tile * kTile + (wave * KPT + i) * 64 + lane;
            const bool cand = j >= first && j < last;
            gt += __popcll(__ballot(j < len && (!cand || (!none && key[i] > prefix))));
            eq += __popcll(__ballot(cand && !none && key[i] == prefix));
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
            const bool cand = j >= first && j < last;
            const bool is_eq = cand && !none && key[i] == prefix;
            const uint64_t below = (1ull << lane) - 1, be = __ballot(is_eq);
            const bool keep = (j < len && (!cand || (!none && key[i] > prefix))) ||
                              (is_eq && eqs + __popcll(be & below) < need);
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
constexpr int kKeepSlab = 16;  // floats of a row that a workgroup moves
constexpr int kKeepUnroll = 4;

// every wave's loads have arrived
__device__ __forceinline__ void loads_done() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// Workgroup: one slab of 16 columns of K or V of one KV head and cache, or (the
// last x) its weights and positions.  Chunks of rows: all loads of a chunk,
// then its stores.  In place one workgroup walks a slab's chunks in order: a
// list ascends with rows[i] >= first + i, so what a later chunk reads lies at
// or behind its own places, past everything written before it, and only the
// chunk's own loads have to end (the barrier) before its stores.
template <int HD, bool INPLACE>
__global__ void __launch_bounds__(kKeepThreads) k_cache_keep(CacheKeep p) {
    constexpr int kSlabs = HD / kKeepSlab;
    const int g = blockIdx.y, c = blockIdx.z, tid = threadIdx.x, x = blockIdx.x;
    const int first = p.first ? min(max(p.first[c], 0), p.max_rows_out) : 0;
    const int count = min(max(p.counts[c], 0), min(p.max_keep, p.max_rows_out - first));
    const int32_t *rows = p.rows + (p.per_head ? (size_t)c * p.kvh + g : (size_t)c) * p.max_keep;
    auto source = [&](int i) {
        return min(max(rows[i], INPLACE ? min(first + i, p.max_rows - 1) : 0), p.max_rows - 1);
    };
    const int part = INPLACE ? x : x % (2 * kSlabs + 1);
    const int from = INPLACE ? 0 : x / (2 * kSlabs + 1), step = INPLACE ? 1 : gridDim.x / (2 * kSlabs + 1);
    if (part == 2 * kSlabs) {
        if (!p.weights && !p.pos) return;
        const size_t in = ((size_t)c * p.kvh + g) * p.side, out = ((size_t)c * p.kvh + g) * p.side_out + first;
        constexpr int kChunk = kKeepThreads;
        for (int b = from; b * kChunk < count; b += step) {
            const int i = b * kChunk + tid;
            float w = 0.0f;
            int32_t at = 0;
            if (i < count) {
                const int j = source(i);
                if (p.weights) w = p.weights[in + j];
                if (p.pos) at = p.pos[in + j];
            }
            if (INPLACE) loads_done();
            if (i < count) {
                if (p.weights) p.weights_out[out + i] = w;
                if (p.pos) p.pos_out[out + i] = at;
            }
        }
        if (INPLACE) __syncthreads();
        if (p.weights)
            for (int i = count + from * kChunk + tid; first + i < p.max_rows_out; i += step * kChunk)
                p.weights_out[out + i] = 0.0f;
        return;
    }
    const int which = part / kSlabs, slab = part % kSlabs;
    constexpr int kLanes = kKeepSlab / 4, kRows = kKeepThreads / kLanes, kChunk = kRows * kKeepUnroll;
    const float *src = p.src[which] + c * p.src_cs[which] + g * HD + slab * kKeepSlab + tid % kLanes * 4;
    float *dst = p.dst[which] + c * p.dst_cs[which] + g * HD + slab * kKeepSlab + tid % kLanes * 4;
    for (int b = from; b * kChunk < count; b += step) {
        float4 v[kKeepUnroll];
#pragma unroll
        for (int u = 0; u < kKeepUnroll; ++u) {
            const int i = b * kChunk + u * kRows + tid / kLanes;
            if (i < count) v[u] = *reinterpret_cast<const float4 *>(src + source(i) * p.src_st[which]);
        }
        if (INPLACE) loads_done();
#pragma unroll
        for (int u = 0; u < kKeepUnroll; ++u) {
            const int i = b * kChunk + u * kRows + tid / kLanes;
            if (i < count) *reinterpret_cast<float4 *>(dst + (first + i) * p.dst_st[which]) = v[u];
        }
    }
}

}  // namespace pocr
