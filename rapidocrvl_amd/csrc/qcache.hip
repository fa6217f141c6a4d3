// qcache.hip — the entry points of the K/V caches in 4 or 8 bits (qcache.hpp):
// argument checks, launch shapes, and the device and stream they run on.
#include "cache_host.hpp"
#include "qcache.hpp"

using namespace pocr;

namespace {

constexpr int kMaxTokens = 1 << 22;
constexpr int kMaxQRows = 1 << 24;                 // query rows of a KV head
constexpr int64_t kMaxStride = (int64_t)1 << 40;  // floats, or rows of a cache

int check_stride(int64_t stride, const char *what, const char *op) {
    if (stride > kMaxStride) return fail(POCR_ERR_ARG, "%s: %s stride %lld is more than 2^40", op, what, (long long)stride);
    return POCR_OK;
}

// a buffer of `seqs` blocks of rows
int check_blocks(const void *p, int64_t seq_stride, int64_t stride, int seqs, int64_t width, const char *what, const char *op) {
    RC(check_rows(p, stride, width, what, op));
    RC(check_outer(seq_stride, seqs, what, op));
    RC(check_stride(stride, what, op));
    return check_stride(seq_stride, what, op);
}

int cache_shape(const pocr_qcache *c, const char *op) {
    if (!c) return fail(POCR_ERR_ARG, "%s: null cache", op);
    if (c->bits != 4 && c->bits != 8) return fail(POCR_ERR_UNSUPPORTED, "%s: %d bits (4 or 8)", op, c->bits);
    if (c->head_dim != 64 && c->head_dim != 128) return fail(POCR_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", op, c->head_dim);
    if (c->seqs < 1 || c->seqs > kMaxGridYZ) return fail(POCR_ERR_ARG, "%s: %d sequences", op, c->seqs);
    if (c->kv_heads < 1 || c->kv_heads > kMaxQueryHeads) return fail(POCR_ERR_ARG, "%s: %d KV heads", op, c->kv_heads);
    if (c->capacity < 1 || c->capacity > kMaxCacheRows) return fail(POCR_ERR_ARG, "%s: capacity %d", op, c->capacity);
    if (c->seq_stride && c->seq_stride < (int64_t)c->kv_heads * c->capacity)
        return fail(POCR_ERR_ARG, "%s: sequences %lld rows apart", op, (long long)c->seq_stride);
    return check_stride(c->seq_stride, "cache", op);
}

int64_t seq_rows(const pocr_qcache *c) { return c->seq_stride ? c->seq_stride : (int64_t)c->kv_heads * c->capacity; }

// the cache's four buffers, as floats
void cache_areas(const pocr_qcache *c, Area (&a)[4]) {
    const int64_t codes = c->head_dim * c->bits / 32, params = c->head_dim / 64, rows = (int64_t)c->kv_heads * c->capacity;
    const void *at[4] = {c->k_codes, c->v_codes, c->k_params, c->v_params};
    for (int i = 0; i < 4; ++i) {
        const int64_t w = i < 2 ? codes : params;
        a[i] = {at[i], seq_rows(c) * w, 0, c->seqs, 1, rows * w};
    }
}

int check_cache(const pocr_qcache *c, const char *op) {
    RC(cache_shape(c, op));
    for (const void *x : {(const void *)c->k_codes, (const void *)c->v_codes, (const void *)c->k_params, (const void *)c->v_params})
        if (!x || !aligned(x, 16)) return fail(POCR_ERR_ARG, "%s: a buffer of the cache is null or not 16-byte aligned", op);
    return POCR_OK;
}

QRows cache_rows(const pocr_qcache *c) {
    QRows r{};
    r.codes[0] = c->k_codes;
    r.codes[1] = c->v_codes;
    r.params[0] = reinterpret_cast<_Float16 *>(c->k_params);
    r.params[1] = reinterpret_cast<_Float16 *>(c->v_params);
    r.seq_rows = seq_rows(c);
    r.kvh = c->kv_heads;
    r.capacity = c->capacity;
    return r;
}

const char *const kRowNames[3] = {"q", "k", "v"}, *const kOutNames[3] = {"q_out", "k_out", "v_out"};

// Rows on their way: shapes, sources, destinations (those of k and v a cache's, or their own).
int rows_call(const pocr_rows_args *a, const pocr_qcache *c, const char *op, RowsCall *p) {
    if (!a) return fail(POCR_ERR_ARG, "%s: null arguments", op);
    if (a->seqs < 1 || a->seqs > kMaxGridYZ) return fail(POCR_ERR_ARG, "%s: %d sequences", op, a->seqs);
    if (a->n < 1 || a->n > kMaxTokens) return fail(POCR_ERR_ARG, "%s: %d tokens", op, a->n);
    if (a->head_dim != 64 && a->head_dim != 128) return fail(POCR_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", op, a->head_dim);
    const float *src[3] = {a->q, a->k, a->v};
    float *dst[3] = {a->q_out, a->k_out, a->v_out};
    const int64_t src_ss[3] = {a->q_seq_stride, a->k_seq_stride, a->v_seq_stride}, src_st[3] = {a->q_stride, a->k_stride, a->v_stride};
    const int64_t dst_ss[3] = {a->q_out_seq_stride, a->k_out_seq_stride, a->v_out_seq_stride},
                  dst_st[3] = {a->q_out_stride, a->k_out_stride, a->v_out_stride};
    if (c) {
        RC(check_cache(c, op));
        if (c->seqs != a->seqs || c->kv_heads != a->kv_heads || c->head_dim != a->head_dim)
            return fail(POCR_ERR_ARG, "%s: rows of %d sequences, %d KV heads of %d, a cache of %d, %d of %d", op, a->seqs, a->kv_heads,
                        a->head_dim, c->seqs, c->kv_heads, c->head_dim);
        if (!a->k || !a->v) return fail(POCR_ERR_ARG, "%s: null k or v", op);
        if (a->k_out || a->v_out) return fail(POCR_ERR_ARG, "%s: k_out and v_out are null, rows go to the cache", op);
        if (a->n > c->capacity) return fail(POCR_ERR_ARG, "%s: %d tokens in %d rows", op, a->n, c->capacity);
    } else {
        if (!a->q && !a->k && !a->v) return fail(POCR_ERR_ARG, "%s: null q, k and v", op);
        if ((a->k || a->v) && (a->max_rows < a->n || a->max_rows > kMaxCacheRows)) return fail(POCR_ERR_ARG, "%s: max_rows %d", op, a->max_rows);
    }
    p->rows = c ? c->capacity : a->max_rows;
    int heads = 0;
    Area from[3] = {}, to[7] = {};
    for (int i = 0; i < 3; ++i) {
        const int own = i ? a->kv_heads : a->heads;
        if (src[i]) {
            if (own < 1 || own > kMaxQueryHeads) return fail(POCR_ERR_ARG, "%s: %d heads of %s", op, own, kRowNames[i]);
            const int64_t width = (int64_t)own * a->head_dim;
            RC(check_blocks(src[i], src_ss[i], src_st[i], a->seqs, width, kRowNames[i], op));
            from[i] = {src[i], src_ss[i], src_st[i], a->seqs, a->n, width};
            if (!i || !c) {
                RC(check_blocks(dst[i], dst_ss[i], dst_st[i], a->seqs, width, kOutNames[i], op));
                to[i] = {dst[i], dst_ss[i], dst_st[i], a->seqs, i ? a->max_rows : a->n, width};
            }
            heads += own;
        } else if (dst[i]) {
            return fail(POCR_ERR_ARG, "%s: %s without %s", op, kOutNames[i], kRowNames[i]);
        }
        p->src[i] = src[i];
        p->dst[i] = dst[i];
        p->src_ss[i] = src_ss[i];
        p->src_st[i] = src_st[i];
        p->dst_ss[i] = dst_ss[i];
        p->dst_st[i] = dst_st[i];
        p->end[i] = heads;
    }
    if (a->rotary_dim) {
        if (a->rotary_dim < 0 || a->rotary_dim > a->head_dim || a->rotary_dim % 16)
            return fail(POCR_ERR_ARG, "%s: rotary_dim %d (a multiple of 16 up to head_dim)", op, a->rotary_dim);
        if (a->axes < 1 || a->axes > 4) return fail(POCR_ERR_ARG, "%s: %d axes", op, a->axes);
        int64_t sum = 0;
        for (int i = 0; i < a->axes; ++i) {
            const int64_t own = a->sections[i];
            if (own < 0 || own > a->rotary_dim / 2) return fail(POCR_ERR_ARG, "%s: section %d of %lld pairs", op, i, (long long)own);
            if (a->interleaved && i && own && a->axes * (own - 1) + i >= a->rotary_dim / 2)
                return fail(POCR_ERR_ARG, "%s: section %d of %lld pairs, %d apart", op, i, (long long)own, a->axes);
            sum += own;
        }
        if (sum != a->rotary_dim / 2) return fail(POCR_ERR_ARG, "%s: sections of %lld pairs, rotary_dim %d", op, (long long)sum, a->rotary_dim);
        if (!a->positions || !a->freqs) return fail(POCR_ERR_ARG, "%s: null positions or freqs", op);
    } else if (a->positions) {
        return fail(POCR_ERR_ARG, "%s: positions without rotary_dim", op);
    }
    if (!(a->eps >= 0.0f && a->eps <= 1.0f)) return fail(POCR_ERR_ARG, "%s: eps must be 0 to 1", op);
    RC(check_index(a->freqs, "freqs", op, 8));
    for (const void *x : {(const void *)a->positions, (const void *)a->counts, (const void *)a->first, (const void *)a->q_norm, (const void *)a->k_norm})
        RC(check_index(x, "an index or side buffer", op));
    // what a call writes meets nothing else of it, but a row its own source
    if (c) {
        Area at[4];
        cache_areas(c, at);
        std::copy(at, at + 4, to + 3);
    }
    const int64_t tokens = (int64_t)a->seqs * a->n;
    const Area side[6] = {{a->positions, 0, 0, 1, 1, tokens * (a->rotary_dim ? a->axes : 0)}, {a->counts, 0, 0, 1, 1, a->seqs},
                          {a->first, 0, 0, 1, 1, a->seqs}, {a->freqs, 0, 0, 1, 1, a->rotary_dim},
                          {a->q_norm, 0, 0, 1, 1, a->head_dim}, {a->k_norm, 0, 0, 1, 1, a->head_dim}};
    for (int i = 0; i < 7; ++i) {
        if (!to[i].at) continue;
        const char *name = i < 3 ? kOutNames[i] : "the cache";
        if (overlap(to[i], to[i], true)) return fail(POCR_ERR_ARG, "%s: sequences of %s overlap", op, name);
        for (int j = 0; j < i; ++j)
            if (to[j].at && overlap(to[i], to[j])) return fail(POCR_ERR_ARG, "%s: %s overlaps another destination", op, name);
        for (int j = 0; j < 3; ++j) {
            if (!from[j].at) continue;
            const bool own = i == j && dst[i] == src[j];  // in place: the same rows
            if (own && dst_st[i] == src_st[j] && (a->seqs == 1 || dst_ss[i] == src_ss[j]) && (!i || !a->first)) continue;
            if (overlap(to[i], from[j])) return fail(POCR_ERR_ARG, "%s: %s overlaps %s", op, name, kRowNames[j]);
        }
        for (const Area &x : side)
            if (x.at && x.width && overlap(to[i], x)) return fail(POCR_ERR_ARG, "%s: %s overlaps an index or side buffer", op, name);
    }
    p->norm[0] = a->q_norm;
    p->norm[1] = a->k_norm;
    p->positions = a->rotary_dim ? a->positions : nullptr;
    p->freqs = a->freqs;
    p->counts = a->counts;
    p->first = a->first;
    if (c) p->cache = cache_rows(c);
    p->n = a->n;
    p->half = a->rotary_dim / 2;
    p->axes = a->axes;
    std::copy(a->sections, a->sections + 4, p->sections);
    p->interleaved = a->interleaved;
    p->adjacent = a->adjacent;
    p->eps = a->eps;
    return POCR_OK;
}

int launch_rows(hipStream_t s, RowsCall p, int head_dim, int bits, int seqs) {
    const int own = 512 / head_dim;  // heads of a wave at a time
    const int64_t total = (int64_t)p.n * seqs;
    // Few tokens: a wave for each four heads (1,345 tokens of 20 heads 8.74 us in one
    // wave a token, 8.50 in five; 8,192 tokens 48.6 : 49.6).  Many: several tokens a
    // wave, as long as 8,192 waves are left (18 x 1,345 tokens of 4 heads in 2,048,
    // 4,096, 8,192 and 16,384 waves 28, 24, 19 and 20 us).
    p.chunks = total < 2048 ? round_up_div(p.end[2], own) : 1;
    p.per = round_up_div(round_up_div(p.end[2], own), p.chunks) * own;
    p.tokens = (int)std::min<int64_t>(p.n, std::max<int64_t>(1, total * p.chunks / 8192));
    const dim3 grid(round_up_div((int64_t)round_up_div(p.n, p.tokens) * p.chunks, 4), seqs);
    const int pairs = p.adjacent ? kPairsAdjacent : (!p.positions || 2 * p.half == head_dim ? kPairsWhole : kPairsPart);
    auto with = [&](auto hd, auto b) {
        constexpr int HD = decltype(hd)::value, B = decltype(b)::value;
        auto *kernel = pairs == kPairsWhole ? k_rows<HD, B, kPairsWhole> : (pairs == kPairsAdjacent ? k_rows<HD, B, kPairsAdjacent> : k_rows<HD, B, kPairsPart>);
        return launch(s, grid, 256, kernel, p);
    };
    auto of = [&](auto hd) {
        if (bits == 4) return with(hd, std::integral_constant<int, 4>{});
        return bits == 8 ? with(hd, std::integral_constant<int, 8>{}) : with(hd, std::integral_constant<int, 0>{});
    };
    return head_dim == 128 ? of(std::integral_constant<int, 128>{}) : of(std::integral_constant<int, 64>{});
}

int attention_shape(const pocr_qattention_args *a, const pocr_qcache *c, const char *op) {
    if (!a) return fail(POCR_ERR_ARG, "%s: null arguments", op);
    RC(cache_shape(c, op));
    RC(check_heads(a->heads, c->kv_heads, c->head_dim, op));
    RC(check_scores(a->scale, a->cap, op));
    if (a->n < 1 || a->n > kMaxTokens || (int64_t)a->n * (a->heads / c->kv_heads) > kMaxQRows)
        return fail(POCR_ERR_ARG, "%s: %d tokens of %d heads", op, a->n, a->heads);
    if (a->max_rows < 1 || a->max_rows > c->capacity) return fail(POCR_ERR_ARG, "%s: max_rows %d of %d", op, a->max_rows, c->capacity);
    if (a->window < 0) return fail(POCR_ERR_ARG, "%s: window %d", op, a->window);
    return POCR_OK;
}

// A window that holds every row is none, which keeps positions less it in 32 bits.
int window_of(const pocr_qattention_args *a) { return a->window < a->max_rows ? a->window : 0; }

// Row tiles and key shares of one attention call.
struct QShape {
    bool many;   // k_qcache_attn_rows
    int rt;      // else: row tiles of 16 a workgroup
    int rows;    // of a workgroup
    bool brief;  // one launch, however few its workgroups
    int tiles, splits;
    int64_t slots, bytes;
};
// The choices were measured at heads of 128 in 4 bits unless stated, 16 heads on 2 KV
// heads, both sides in us.
// Rows of a (sequence, KV head).  Up to 32 a wave takes blocks of its own for all of
// them, more come in tiles of 64 whose waves take blocks together: 24 rows behind 500
// keys 10.7 : 11.9, of 16 sequences behind 8,192 keys 26.3 : 36.8, 32 rows 26.5 : 37.5.
// 48 rows in three row tiles of a wave spilled registers.
// One launch without a join, up to the keys where shares and their join take no longer:
// 16 rows 512 keys 8.7 : 9.1, 768 keys 10.5 : 9.2; 32 rows 256 keys 9.8 : 10.3, 384 keys
// 11.4 : 10.7; 48 rows 128 keys 10.1 : 10.5, 160 keys 11.3 : 10.9.  Heads of 64: 16 rows
// 1,024 keys 8.8 : 9.0, 1,280 keys 9.9 : 9.0; 32 rows 512 keys 9.5 : 9.3; 48 rows 192 keys
// 8.8 : 9.8, 256 keys 10.2 : 9.1.
// Eight waves a workgroup, up to 16 rows: for short caches (8 tokens of 4 heads of 64 behind
// 700 rows 7.9 us, four waves 9.6), and for heads of 64 where there are so many workgroups
// that long ones have one share too (64 sequences of 8 KV heads, 2,048 and 8,192 rows, 22.7
// and 71 us, four waves 25.3 and 91).  Long ones of heads of 128 then take four: 38.4 and
// 127.5 us, eight 42.7 and 133; 160 sequences of 2 KV heads in 8 bits 41 and 137, eight 46
// and 152.
// Shares: few rows 512 workgroups (16 sequences of 8 rows, 8,192 keys, in 256, 512 and
// 768: 19.7, 18.3, 18.9) of 4 blocks or more, one for each wave (8 rows, 8,192 keys, 2, 4
// and 8: 10.4, 9.3, 10.0).  Many rows: one workgroup a CU first, of 2 blocks or more (64
// rows, 2,048 keys, 2, 3 and 6: 12.0, 13.2, 15.7), then as many as a CU holds, of 6 or more
// (64 rows of 16 sequences, 2,048 keys, 2, 3 and 6: 27.5, 27.2, 24.4).  Those are three of
// heads of 128 in 4 bits (600 tokens behind 8,192 rows in 512, 768 and 1,024 workgroups:
// 130, 106, 130), and three of heads of 64 too, of which a CU holds four (88, 70, 73).  In
// 8 bits they are two (122, 142, 127; 16 sequences of 40: 120, 160, 126), or two after one
// another where that leaves 8 blocks less in a row: 540 tokens 119, 126, 112; 700: 168,
// 155, 145.
QShape qattn_shape(const pocr_qattention_args *a, const pocr_qcache *c) {
    QShape q;
    const int64_t rows = (int64_t)a->n * (a->heads / c->kv_heads), groups = (int64_t)c->kv_heads * c->seqs;
    const bool small = c->head_dim == 64;
    q.many = rows > 32;
    q.rt = rows <= 16 ? 1 : 2;
    q.rows = q.many ? 64 : 16 * q.rt;
    q.tiles = round_up_div(rows, q.rows);
    const int64_t work = q.tiles * groups;
    const int window = window_of(a);
    const int64_t keys = window ? std::min<int64_t>(a->max_rows, (int64_t)window + q.rows) : a->max_rows;
    const int64_t blocks = round_up_div(keys, kQBlock);
    const int whole = q.many ? (small ? 6 : 4) : (q.rt == 2 ? 8 : 16) * (small ? 2 : 1);
    // so many shares that at most `wgs` workgroups result, of `least` blocks or more
    auto shares = [&](int64_t wgs, int64_t least) { return std::max<int64_t>(1, std::min<int64_t>(wgs / work, round_up_div(blocks, least))); };
    int64_t most = shares(512, 4);
    if (q.many && !small && c->bits == 8) {
        const int64_t once = std::max(shares(256, 2), shares(512, 6)), twice = shares(1024, 6);
        most = 2 * round_up_div(blocks, twice) + 8 < round_up_div(blocks, once) ? twice : once;
    } else if (q.many) {
        most = std::max(shares(256, 2), shares(768, 6));
    }
    q.brief = blocks <= whole;
    q.splits = q.brief ? 1 : (int)std::min<int64_t>(most, 128);
    q.slots = q.splits > 1 ? work * q.splits : 0;
    q.bytes = q.slots * q.rows * (c->head_dim + 2) * 4;
    return q;
}

template <int HD, int BITS, int ROWS>  // rows of a workgroup
int launch_qattn(hipStream_t s, const QAttnCall &p, const QShape &q, void *work, int seqs) {
    QAttnPlan pl{};
    pl.tiles = q.tiles;
    pl.splits = q.splits;
    pl.part = static_cast<float *>(work);
    pl.stat = reinterpret_cast<float2 *>(pl.part + q.slots * ROWS * HD);
    const dim3 grid(q.tiles * q.splits, p.cache.kvh, seqs);
    const bool shaped = p.cap > 0.0f || p.slopes;
    if constexpr (ROWS == 64) {
        RC(launch(s, grid, 256, shaped ? k_qcache_attn_rows<HD, BITS, true> : k_qcache_attn_rows<HD, BITS, false>, p, pl));
    } else {
        if (ROWS == 16 && q.splits == 1 && (HD == 64 || q.brief)) return launch(s, grid, 512, shaped ? k_qcache_attn<HD, BITS, 1, 8, true> : k_qcache_attn<HD, BITS, 1, 8, false>, p, pl);
        RC(launch(s, grid, 256, shaped ? k_qcache_attn<HD, BITS, ROWS / 16, 4, true> : k_qcache_attn<HD, BITS, ROWS / 16, 4, false>, p, pl));
    }
    if (q.splits == 1) return POCR_OK;
    // 13 shares of 8 rows, eight at a time and two: 8.9, 9.5 us; 5 shares of 4,800 rows: 117, 115.
    constexpr int U = 1024 / HD;
    if (q.splits >= 8) return launch(s, dim3(q.tiles * ROWS / (U / 8), p.cache.kvh, seqs), 256, k_qcache_join<HD, ROWS, 8>, p, pl);
    return launch(s, dim3(q.tiles * ROWS / (U / 2), p.cache.kvh, seqs), 256, k_qcache_join<HD, ROWS, 2>, p, pl);
}

template <int HD, int BITS>
int launch_qattn_t(hipStream_t s, const QAttnCall &p, const QShape &q, void *work, int seqs) {
    if (q.many) return launch_qattn<HD, BITS, 64>(s, p, q, work, seqs);
    return q.rt == 1 ? launch_qattn<HD, BITS, 16>(s, p, q, work, seqs) : launch_qattn<HD, BITS, 32>(s, p, q, work, seqs);
}

}  // namespace

extern "C" int pocr_rotate_rows(pocr_ctx *ctx, const pocr_rows_args *a, void *stream) {
    const char *op = "pocr_rotate_rows";
    RowsCall p{};
    RC(rows_call(a, nullptr, op, &p));
    CACHE_OP_ENTER(ctx, stream, op);
    return launch_rows((hipStream_t)stream, p, a->head_dim, 0, a->seqs);
}

extern "C" int pocr_qcache_write(pocr_ctx *ctx, const pocr_rows_args *a, const pocr_qcache *c, void *stream) {
    const char *op = "pocr_qcache_write";
    if (!c) return fail(POCR_ERR_ARG, "%s: null cache", op);
    RowsCall p{};
    RC(rows_call(a, c, op, &p));
    CACHE_OP_ENTER(ctx, stream, op);
    return launch_rows((hipStream_t)stream, p, a->head_dim, c->bits, a->seqs);
}

extern "C" int pocr_qcache_read(pocr_ctx *ctx, const pocr_qread_args *a, const pocr_qcache *c, void *stream) {
    const char *op = "pocr_qcache_read";
    if (!a) return fail(POCR_ERR_ARG, "%s: null arguments", op);
    RC(check_cache(c, op));
    if (a->n < 1 || a->n > kMaxCacheRows) return fail(POCR_ERR_ARG, "%s: %d rows", op, a->n);
    if (!a->k_out && !a->v_out) return fail(POCR_ERR_ARG, "%s: null k_out and v_out", op);
    if (a->rows && a->first) return fail(POCR_ERR_ARG, "%s: rows and first", op);
    for (const void *x : {(const void *)a->rows, (const void *)a->counts, (const void *)a->first}) RC(check_index(x, "an index buffer", op));
    const int64_t width = (int64_t)c->kv_heads * c->head_dim;
    float *dst[2] = {a->k_out, a->v_out};
    const int64_t ss[2] = {a->k_out_seq_stride, a->v_out_seq_stride}, st[2] = {a->k_out_stride, a->v_out_stride};
    Area at[4], to[2] = {};
    cache_areas(c, at);
    const int64_t lists = (int64_t)c->seqs * (a->per_head ? c->kv_heads : 1) * a->n;
    const Area side[3] = {{a->rows, 0, 0, 1, 1, lists}, {a->counts, 0, 0, 1, 1, c->seqs}, {a->first, 0, 0, 1, 1, c->seqs}};
    QReadCall p{};
    for (int i = 0; i < 2; ++i) {
        if (!dst[i]) continue;
        const char *name = kOutNames[i + 1];
        RC(check_blocks(dst[i], ss[i], st[i], c->seqs, width, name, op));
        to[i] = {dst[i], ss[i], st[i], c->seqs, a->n, width};
        if (overlap(to[i], to[i], true)) return fail(POCR_ERR_ARG, "%s: sequences of %s overlap", op, name);
        if (i && to[0].at && overlap(to[0], to[1])) return fail(POCR_ERR_ARG, "%s: k_out overlaps v_out", op);
        for (const Area &x : at)
            if (overlap(to[i], x)) return fail(POCR_ERR_ARG, "%s: %s overlaps the cache", op, name);
        for (const Area &x : side)
            if (x.at && overlap(to[i], x)) return fail(POCR_ERR_ARG, "%s: %s overlaps an index buffer", op, name);
        p.dst[i] = dst[i];
        p.dst_ss[i] = ss[i];
        p.dst_st[i] = st[i];
    }
    CACHE_OP_ENTER(ctx, stream, op);
    p.rows = a->rows;
    p.counts = a->counts;
    p.first = a->first;
    p.cache = cache_rows(c);
    p.n = a->n;
    p.per_head = a->per_head != 0;
    hipStream_t s = (hipStream_t)stream;
    auto run = [&](auto kernel) {
        const int rows = 256 / (c->head_dim / 8), blocks = round_up_div(a->rows ? a->n : std::min(a->n, c->capacity), rows);
        const int most = (int)(kMaxGrid / 256);
        for (int b = 0; b < blocks; b += most) {
            p.row0 = b * rows;
            RC(launch(s, dim3(std::min(most, blocks - b), c->kv_heads, c->seqs), 256, kernel, p));
        }
        return (int)POCR_OK;
    };
    if (c->head_dim == 128) return c->bits == 4 ? run(k_qcache_read<128, 4>) : run(k_qcache_read<128, 8>);
    return c->bits == 4 ? run(k_qcache_read<64, 4>) : run(k_qcache_read<64, 8>);
}

extern "C" int64_t pocr_qcache_attention_workspace(const pocr_qattention_args *a, const pocr_qcache *c) {
    RC(attention_shape(a, c, "pocr_qcache_attention_workspace"));
    return qattn_shape(a, c).bytes;
}

extern "C" int pocr_qcache_attention(pocr_ctx *ctx, const pocr_qattention_args *a, const pocr_qcache *c, void *stream) {
    const char *op = "pocr_qcache_attention";
    RC(attention_shape(a, c, op));
    RC(check_cache(c, op));
    const int64_t width = (int64_t)a->heads * c->head_dim;
    RC(check_blocks(a->q, a->q_seq_stride, a->q_stride, c->seqs, width, "q", op));
    RC(check_blocks(a->out, a->out_seq_stride, a->out_stride, c->seqs, width, "out", op));
    if (!a->lens) return fail(POCR_ERR_ARG, "%s: null lens", op);
    for (const void *x : {(const void *)a->lens, (const void *)a->counts, (const void *)a->slopes, (const void *)a->lse})
        RC(check_index(x, "an index or side buffer", op));
    const Area out{a->out, a->out_seq_stride, a->out_stride, c->seqs, a->n, width};
    if (overlap(out, out, true)) return fail(POCR_ERR_ARG, "%s: out rows of two sequences overlap", op);
    const QShape shape = qattn_shape(a, c);
    RC(check_workspace(a->workspace, a->workspace_bytes, shape.bytes, op));
    CACHE_OP_ENTER(ctx, stream, op);
    QAttnCall p{};
    p.q = a->q;
    p.out = a->out;
    p.lse = a->lse;
    p.lens = a->lens;
    p.counts = a->counts;
    p.slopes = a->slopes;
    p.q_ss = a->q_seq_stride;
    p.q_st = a->q_stride;
    p.o_ss = a->out_seq_stride;
    p.o_st = a->out_stride;
    p.cache = cache_rows(c);
    p.n = a->n;
    p.heads = a->heads;
    p.group = a->heads / c->kv_heads;
    p.group_inv = p.group == 1 ? 0u : (uint32_t)((((uint64_t)1 << 32) + p.group - 1) / p.group);
    p.max_rows = a->max_rows;
    p.window = window_of(a);
    p.scale = default_scale(a->scale, c->head_dim);
    p.cap = a->cap;
    p.cap_inverse = a->cap > 0.0f ? 1.0f / a->cap : 0.0f;
    p.cap_log2 = a->cap * kLog2e;
    hipStream_t s = (hipStream_t)stream;
    if (c->head_dim == 128)
        return c->bits == 4 ? launch_qattn_t<128, 4>(s, p, shape, a->workspace, c->seqs) : launch_qattn_t<128, 8>(s, p, shape, a->workspace, c->seqs);
    return c->bits == 4 ? launch_qattn_t<64, 4>(s, p, shape, a->workspace, c->seqs) : launch_qattn_t<64, 8>(s, p, shape, a->workspace, c->seqs);
}
