// cache_ops.hip — the cache operators' entry points (cache_ops.hpp): argument
// checks, launch shapes, and the device and stream they run on.
#include "cache_host.hpp"
#include "cache_ops.hpp"

using namespace pocr;

namespace {

constexpr int kMaxPromptRows = 1 << 22;
constexpr int kMaxQueryRows = 1 << 29;  // of a KV head: 2^22 tiles, 768 threads each
constexpr int kMaxTreeTokens = 64;  // a token's ancestors are the bits of one 64-bit word
// Images cost a launch and a pass over the rows, and pay by the steps that all
// tiles take (of 128 rows and 32 keys): images, attention and join against
// attention and join took, 16 heads over 2 KV heads of 128, causal, in us:
//   600 rows                   1,444 steps at most   32 : 30
//   256 rows behind 2,000      2,272                 43 : 37
//   800 rows                   2,500                 36 : 42
//   128 rows behind 8,000      4,064                 56 : 54
//   1,200 rows                 5,700                 49 : 88
//   256 rows behind 8,000      8,256                 82 : 94
// (what counts is steps; 128 rows behind 8,000, few tiles with long shares, lose 2 us)
constexpr int kImageTiles = 8, kImageSteps = 2400;

int prompt_shape(const pocr_prompt_args *a, const char *op) {
    if (!a) return fail(POCR_ERR_ARG, "%s: null arguments", op);
    RC(check_heads(a->heads, a->kv_heads, a->head_dim, op));
    RC(check_scores(a->scale, a->cap, op));
    if (a->n < 1 || a->n > kMaxPromptRows || (int64_t)a->n * (a->heads / a->kv_heads) > kMaxQueryRows)
        return fail(POCR_ERR_ARG, "%s: %d rows of %d heads", op, a->n, a->heads);
    if (a->rows_before < 0 || a->rows_before > kMaxCacheRows - a->n) return fail(POCR_ERR_ARG, "%s: %d rows before", op, a->rows_before);
    return POCR_OK;
}

int tree_shape(const pocr_tree_args *a, const char *op) {
    if (!a) return fail(POCR_ERR_ARG, "%s: null arguments", op);
    RC(check_heads(a->heads, a->kv_heads, a->head_dim, op));
    RC(check_scores(a->scale, a->cap, op));
    if (a->seqs < 1 || a->seqs > kMaxGridYZ) return fail(POCR_ERR_ARG, "%s: %d sequences", op, a->seqs);
    if (a->n < 1 || a->n > kMaxTreeTokens) return fail(POCR_ERR_ARG, "%s: %d tokens (1 to %d)", op, a->n, kMaxTreeTokens);
    if (a->max_rows < a->n || a->max_rows > kMaxCacheRows) return fail(POCR_ERR_ARG, "%s: max_rows %d", op, a->max_rows);
    return POCR_OK;
}

// what pocr_tree_attention and pocr_cache_weights share
int tree_params(const pocr_tree_args *a, const char *op, CacheAttn *p) {
    RC(tree_shape(a, op));
    const int64_t kvd = (int64_t)a->kv_heads * a->head_dim, qd = (int64_t)a->heads * a->head_dim;
    RC(check_rows(a->q, a->q_stride, qd, "q", op));
    RC(check_rows(a->k, a->k_stride, kvd, "k", op));
    RC(check_outer(a->q_seq_stride, a->seqs, "q", op));
    RC(check_outer(a->k_seq_stride, a->seqs, "k", op));
    if (!a->lens) return fail(POCR_ERR_ARG, "%s: null lens", op);
    RC(check_side(a->side_stride, a->max_rows, "side_stride", op));
    for (const void *x : {(const void *)a->lens, (const void *)a->counts, (const void *)a->parents, (const void *)a->slopes,
                          (const void *)a->positions, (const void *)a->lse})
        RC(check_index(x, "an index or side buffer", op));
    p->q = a->q;
    p->k = a->k;
    p->lens = a->lens;
    p->counts = a->counts;
    p->parents = a->parents;
    p->slopes = a->slopes;
    p->pos = a->positions;
    p->lse = a->lse;
    p->q_ss = a->q_seq_stride;
    p->q_st = a->q_stride;
    p->k_ss = a->k_seq_stride;
    p->k_st = a->k_stride;
    p->side = a->side_stride ? a->side_stride : a->max_rows;
    p->n = a->n;
    p->rows = a->max_rows;
    p->heads = a->heads;
    p->kvh = a->kv_heads;
    p->group = a->heads / a->kv_heads;
    p->inv_group = 1.0f / (float)p->group;
    p->scale = default_scale(a->scale, a->head_dim);
    p->cap = a->cap;
    return POCR_OK;
}

// Row tiles and key shares of one attention call: `rows` query rows (token,
// head) per sequence and KV head over at most `keys` keys.
struct AttnShape {
    bool few;                       // k_cache_attn_few
    int wg_rows, tiles, splits, least;
    int steps;                      // images of a prompt's rows, or 0
    int jobs;                       // with images: workgroups per KV head
    int64_t slots;                  // shares with partial sums, or 0
    int64_t part_bytes, cut_bytes, bytes;  // of the workspace: partial sums and their counts or jobs, images
};
template <int HD>
constexpr int64_t image_bytes = StepImage<HD>::kBytes;
AttnShape attn_shape(int64_t rows, int64_t keys, int64_t groups, int head_dim, bool images) {
    AttnShape a;
    // 16 rows by either form, 16 sequences of 2 tokens over 1,609 rows: 16 us in
    // fp32 straight from the cache, 19 laid out; beyond, the fp32 products of two
    // tiles took 29 us where laying out takes 20
    a.few = rows <= 16;
    a.wg_rows = a.few ? 16 : kTileRows;
    a.tiles = round_up_div(rows, a.wg_rows);
    const int64_t work = a.tiles * groups;
    const int steps = round_up_div(keys, kBlock);
    a.steps = images && a.tiles >= kImageTiles && work * steps >= kImageSteps ? steps : 0;
    const int step = a.few ? kFewKeys * kFewWaves : kBlock;
    if (a.steps) {
        // Two workgroups a CU run at once; the device cuts the tiles into shares of
        // at least two steps that fill them once (480 or 768 workgroups for the
        // same prompts: 15 to 25% more time).  More tiles than that stay whole.
        a.least = 2;
        a.splits = 1;
        a.jobs = work <= kCutTiles ? (int)(kCutTiles / groups) : a.tiles;
        a.slots = a.jobs > a.tiles ? a.jobs * groups : 0;
        a.cut_bytes = (a.tiles * (int64_t)sizeof(TileCut) + a.jobs * 4 + 15) / 16 * 16;
    } else {
        // One workgroup a CU at a time (512 for 16 trees of 12 over 1,609 rows: 41
        // us, 256: 32, by the form that both were measured with; 256 and 512 are
        // alike for few rows).  From 256 tiles on, whose lengths may differ, shares
        // for four rounds.  Shares of fewer steps than `least` cost more in sums
        // than they save where the tiles fill half of the chip anyway (least 2 and
        // 6, us: 16 trees of 12 over 250 rows, 32 tiles, 17.5 and 24.0, over 800 rows
        // 22.9 and 25.8; 64 trees, 128 tiles, over 250 rows 25.9 and 24.8; 128 trees
        // over 250 rows 68 and 29, over 500 rows 82 and 63; 1,609 rows alike).
        const int64_t want = std::max<int64_t>(1, (work >= 256 ? 1024 : 256) / work);
        a.least = a.few ? 1 : (work < 128 ? 2 : 6);
        a.splits = (int)std::min<int64_t>({want, kMaxShares, std::max<int64_t>(1, keys / (step * a.least))});
        a.jobs = 0;
        a.slots = a.splits > 1 ? work * a.splits : 0;
        a.cut_bytes = a.slots ? (work * 4 + 15) / 16 * 16 : 0;
    }
    a.part_bytes = a.slots * a.wg_rows * (head_dim + 2) * 4;
    a.bytes = a.part_bytes + a.cut_bytes + a.steps * groups * (head_dim == 128 ? image_bytes<128> : image_bytes<64>);
    return a;
}

AttnPlan attn_plan(const AttnShape &sh, void *work, int head_dim) {
    AttnPlan pl{};
    pl.tiles = sh.tiles;
    pl.splits = sh.splits;
    pl.least = sh.least;
    pl.steps = sh.steps;
    pl.max_jobs = sh.jobs;
    if (sh.slots) {
        pl.part = static_cast<float *>(work);
        pl.stat = reinterpret_cast<float2 *>(pl.part + sh.slots * sh.wg_rows * head_dim);
    }
    char *at = static_cast<char *>(work) + sh.part_bytes;
    if (sh.steps) {
        pl.cuts = reinterpret_cast<TileCut *>(at);
        pl.jobs = reinterpret_cast<int32_t *>(pl.cuts + sh.tiles);
        pl.img = reinterpret_cast<uint8_t *>(at + sh.cut_bytes);
    } else if (sh.slots) {
        pl.parts = reinterpret_cast<int32_t *>(at);
    }
    return pl;
}

template <int HD, int kRows, int kSub>
int launch_join(hipStream_t s, const CacheAttn &p, const AttnPlan &pl, int seqs) {
    if (!pl.part) return POCR_OK;
    return launch(s, dim3(pl.tiles * (kRows * kSub / (1024 / HD)), p.kvh, seqs), 256, k_cache_attn_join<HD, kRows, kSub>, p, pl);
}

template <int HD, bool TREE, bool SHAPED>
int launch_few(hipStream_t s, const CacheAttn &p, const AttnShape &sh, void *work, int seqs) {
    const AttnPlan pl = attn_plan(sh, work, HD);
    RC(launch(s, dim3(sh.splits, p.kvh, seqs), 64 * kFewWaves, k_cache_attn_few<HD, TREE, SHAPED>, p, pl));
    return launch_join<HD, 16, 4>(s, p, pl, seqs);
}

template <int HD, bool TREE, bool SHAPED, bool IMG>
int launch_attn_t(hipStream_t s, const CacheAttn &p, const AttnShape &sh, void *work, int seqs) {
    const AttnPlan pl = attn_plan(sh, work, HD);
    if (IMG) RC(launch(s, dim3(sh.steps + 1, p.kvh), kAttnThreads, k_cache_images<HD>, p, pl, const_cast<uint8_t *>(pl.img)));
    const int x = IMG ? sh.jobs : sh.tiles * sh.splits;
    RC(launch(s, dim3(x, p.kvh, seqs), IMG ? 256 : 768, k_cache_attn<HD, TREE, SHAPED, IMG>, p, pl));
    return launch_join<HD, 128, 1>(s, p, pl, seqs);
}

template <int HD, bool TREE, bool SHAPED>
int launch_attn_s(hipStream_t s, const CacheAttn &p, const AttnShape &sh, void *work, int seqs) {
    if constexpr (!TREE)
        if (sh.steps) return launch_attn_t<HD, TREE, SHAPED, true>(s, p, sh, work, seqs);
    if (sh.few) return launch_few<HD, TREE, SHAPED>(s, p, sh, work, seqs);
    return launch_attn_t<HD, TREE, SHAPED, false>(s, p, sh, work, seqs);
}

template <int HD, bool SHAPED>
int launch_weights(hipStream_t s, CacheAttn p, int seqs) {
    const int64_t groups = (int64_t)p.kvh * seqs;
    auto run = [&](auto kernel, int keys, int threads) {
        const int blocks = round_up_div(p.rows, keys), most = kMaxGrid / threads;  // max_rows is a bound, lengths are on the device
        for (int at = 0; at < blocks; at += most) {
            p.key0 = at * keys;
            RC(launch(s, dim3(std::min(most, blocks - at), p.kvh, seqs), threads, kernel, p));
        }
        return (int)POCR_OK;
    };
    // A workgroup lays all query rows out by itself and takes about as long for
    // 32, 64 or 96 keys (512 query rows: 15, 17, 19 us), so one round on 256 CUs
    // is what counts: 64 tokens of 16 heads over 8,256 rows took 35 us as 516
    // workgroups of 32 keys, 33 as 258 of 64, 21 as 172 of 96; over 4,064 rows 16, 18, 19.
    if (p.n * p.group <= kWRows) return run(k_cache_weights<HD, SHAPED, 0>, 64, 256);
    if (round_up_div(p.rows, 32) * groups <= 256) return run(k_cache_weights<HD, SHAPED, 1>, 32, 512);
    if (round_up_div(p.rows, 64) * groups <= 256) return run(k_cache_weights<HD, SHAPED, 2>, 64, 512);
    return run(k_cache_weights<HD, SHAPED, 3>, 96, 512);
}

template <bool TREE>
int launch_attn(hipStream_t s, const CacheAttn &p, int head_dim, int seqs, const AttnShape &sh, void *work) {
    const bool shaped = p.cap > 0.0f || p.slopes;
    if (head_dim == 128)
        return shaped ? launch_attn_s<128, TREE, true>(s, p, sh, work, seqs) : launch_attn_s<128, TREE, false>(s, p, sh, work, seqs);
    return shaped ? launch_attn_s<64, TREE, true>(s, p, sh, work, seqs) : launch_attn_s<64, TREE, false>(s, p, sh, work, seqs);
}

AttnShape prompt_attn(const pocr_prompt_args *a, bool spans) {
    const int64_t rows = (int64_t)a->rows_before + a->n;
    // Spans may leave out most of a long cache, whose images are made all the
    // same: worth it where all rows are seen, or not many more than the prompt's
    // own.  Images against none, us, spans that see all rows, the latter half or
    // the prompt's own alone:
    //   600 rows behind 1,200      50 : 58    43 : 45    33 : 31
    //   600 rows behind 9,600     167 : 245  102 : 139   36 : 31
    //   300 rows behind 4,800      65 : 75    49 : 47    28 : 21
    // The spans are on the device: far behind, where images may cost a third, none
    // are made, which costs up to half as much again where spans see everything.
    const bool images = !spans || a->rows_before <= 4 * (int64_t)a->n;
    return attn_shape((int64_t)a->n * (a->heads / a->kv_heads), rows, a->kv_heads, a->head_dim, images);
}
AttnShape tree_attn(const pocr_tree_args *a) {
    return attn_shape((int64_t)a->n * (a->heads / a->kv_heads), a->max_rows, (int64_t)a->kv_heads * a->seqs, a->head_dim, false);
}

}  // namespace

extern "C" int64_t pocr_prompt_attention_workspace(const pocr_prompt_args *a) {
    RC(prompt_shape(a, "pocr_prompt_attention_workspace"));
    return std::max(prompt_attn(a, false).bytes, prompt_attn(a, true).bytes);  // shapes alone: with spans or without
}

extern "C" int64_t pocr_tree_attention_workspace(const pocr_tree_args *a) {
    RC(tree_shape(a, "pocr_tree_attention_workspace"));
    return tree_attn(a).bytes;
}

extern "C" int pocr_prompt_attention(pocr_ctx *ctx, const pocr_prompt_args *a, void *stream) {
    const char *op = "pocr_prompt_attention";
    RC(prompt_shape(a, op));
    const int64_t kvd = (int64_t)a->kv_heads * a->head_dim, qd = (int64_t)a->heads * a->head_dim;
    RC(check_rows(a->q, a->q_stride, qd, "q", op));
    RC(check_rows(a->k, a->k_stride, kvd, "k", op));
    RC(check_rows(a->v, a->v_stride, kvd, "v", op));
    RC(check_rows(a->out, a->out_stride, qd, "out", op));
    if (!a->row_begin != !a->row_end) return fail(POCR_ERR_ARG, "%s: row_begin and row_end come together", op);
    for (const void *x : {(const void *)a->row_begin, (const void *)a->row_end, (const void *)a->slopes, (const void *)a->lse})
        RC(check_index(x, "an index or side buffer", op));
    const AttnShape shape = prompt_attn(a, a->row_begin);
    RC(check_workspace(a->workspace, a->workspace_bytes, shape.bytes, op));
    CACHE_OP_ENTER(ctx, stream, op);
    CacheAttn p{};
    p.q = a->q;
    p.k = a->k;
    p.v = a->v;
    p.out = a->out;
    p.lse = a->lse;
    p.begin = a->row_begin;
    p.end = a->row_end;
    p.slopes = a->slopes;
    p.q_st = a->q_stride;
    p.k_st = a->k_stride;
    p.v_st = a->v_stride;
    p.o_st = a->out_stride;
    p.n = a->n;
    p.rows0 = a->rows_before;
    p.rows = a->rows_before + a->n;
    p.heads = a->heads;
    p.kvh = a->kv_heads;
    p.group = a->heads / a->kv_heads;
    p.inv_group = 1.0f / (float)p.group;
    p.scale = default_scale(a->scale, a->head_dim);
    p.cap = a->cap;
    return launch_attn<false>((hipStream_t)stream, p, a->head_dim, 1, shape, a->workspace);
}

extern "C" int pocr_tree_attention(pocr_ctx *ctx, const pocr_tree_args *a, void *stream) {
    const char *op = "pocr_tree_attention";
    CacheAttn p{};
    RC(tree_params(a, op, &p));
    RC(check_rows(a->v, a->v_stride, (int64_t)a->kv_heads * a->head_dim, "v", op));
    RC(check_rows(a->out, a->out_stride, (int64_t)a->heads * a->head_dim, "out", op));
    RC(check_outer(a->v_seq_stride, a->seqs, "v", op));
    RC(check_outer(a->out_seq_stride, a->seqs, "out", op));
    const Area out{a->out, a->out_seq_stride, a->out_stride, a->seqs, a->n, (int64_t)a->heads * a->head_dim};
    if (overlap(out, out, true)) return fail(POCR_ERR_ARG, "%s: out rows of two sequences overlap", op);
    const AttnShape shape = tree_attn(a);
    RC(check_workspace(a->workspace, a->workspace_bytes, shape.bytes, op));
    CACHE_OP_ENTER(ctx, stream, op);
    p.v = a->v;
    p.out = a->out;
    p.v_ss = a->v_seq_stride;
    p.v_st = a->v_stride;
    p.o_ss = a->out_seq_stride;
    p.o_st = a->out_stride;
    return launch_attn<true>((hipStream_t)stream, p, a->head_dim, a->seqs, shape, a->workspace);
}

extern "C" int pocr_cache_weights(pocr_ctx *ctx, const pocr_tree_args *a, void *stream) {
    const char *op = "pocr_cache_weights";
    CacheAttn p{};
    RC(tree_params(a, op, &p));
    if (!a->lse || !a->weights) return fail(POCR_ERR_ARG, "%s: null lse or weights", op);
    RC(check_index(a->weights, "weights", op));
    RC(check_index(a->take, "take", op, 8));
    CACHE_OP_ENTER(ctx, stream, op);
    p.weights = a->weights;
    p.take = a->take;
    hipStream_t s = (hipStream_t)stream;
    const bool shaped = p.cap > 0.0f || p.slopes;
    if (a->head_dim == 128) return shaped ? launch_weights<128, true>(s, p, a->seqs) : launch_weights<128, false>(s, p, a->seqs);
    return shaped ? launch_weights<64, true>(s, p, a->seqs) : launch_weights<64, false>(s, p, a->seqs);
}

extern "C" int pocr_cache_select(pocr_ctx *ctx, const pocr_select_args *a, void *stream) {
    const char *op = "pocr_cache_select";
    if (!a) return fail(POCR_ERR_ARG, "%s: null arguments", op);
    if (a->caches < 1 || a->caches > kMaxGridYZ || a->kv_heads < 1 || a->kv_heads > kMaxGridYZ)
        return fail(POCR_ERR_ARG, "%s: %d caches of %d KV heads", op, a->caches, a->kv_heads);
    if (a->max_rows < 1 || a->max_rows > kMaxCacheRows) return fail(POCR_ERR_ARG, "%s: max_rows %d", op, a->max_rows);
    if (a->budget < 1 || a->budget > kMaxCacheRows) return fail(POCR_ERR_ARG, "%s: budget %d", op, a->budget);
    if (a->sinks < 0 || a->recent < 0 || (int64_t)a->sinks + a->recent > a->budget)
        return fail(POCR_ERR_ARG, "%s: %d first and %d last rows in a budget of %d", op, a->sinks, a->recent, a->budget);
    RC(check_side(a->side_stride, a->max_rows, "side_stride", op));
    if (!a->weights || !a->lens || !a->kept || !a->counts) return fail(POCR_ERR_ARG, "%s: null buffer", op);
    if (a->counts == a->lens) return fail(POCR_ERR_ARG, "%s: counts is lens", op);
    for (const void *x : {(const void *)a->weights, (const void *)a->lens, (const void *)a->kept, (const void *)a->counts})
        RC(check_index(x, "a buffer", op));
    CACHE_OP_ENTER(ctx, stream, op);
    CacheSelect p{};
    p.weights = a->weights;
    p.lens = a->lens;
    p.kept = a->kept;
    p.counts = a->counts;
    p.side = a->side_stride ? a->side_stride : a->max_rows;
    p.kvh = a->kv_heads;
    p.max_rows = a->max_rows;
    p.budget = a->budget;
    p.sinks = a->sinks;
    p.recent = a->recent;
    // rows per thread: the fewest that hold the cache in registers (1,609 rows: 2)
    const dim3 grid(a->kv_heads, a->caches);
    hipStream_t s = (hipStream_t)stream;
    if (a->max_rows <= 2 * kSelThreads) return launch(s, grid, kSelThreads, k_cache_select<2>, p);
    if (a->max_rows <= 8 * kSelThreads) return launch(s, grid, kSelThreads, k_cache_select<8>, p);
    return launch(s, grid, kSelThreads, k_cache_select<16>, p);
}

extern "C" int pocr_cache_keep(pocr_ctx *ctx, const pocr_keep_args *a, void *stream) {
    const char *op = "pocr_cache_keep";
    if (!a) return fail(POCR_ERR_ARG, "%s: null arguments", op);
    if (a->caches < 1 || a->caches > kMaxGridYZ || a->kv_heads < 1 || a->kv_heads > kMaxGridYZ)
        return fail(POCR_ERR_ARG, "%s: %d caches of %d KV heads", op, a->caches, a->kv_heads);
    if (a->head_dim != 64 && a->head_dim != 128) return fail(POCR_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", op, a->head_dim);
    for (const int32_t n : {a->max_keep, a->max_rows, a->max_rows_out})
        if (n < 1 || n > kMaxCacheRows) return fail(POCR_ERR_ARG, "%s: max_keep, max_rows and max_rows_out are 1 to 2^30", op);
    const int64_t kvd = (int64_t)a->kv_heads * a->head_dim;
    RC(check_rows(a->k, a->k_stride, kvd, "k", op));
    RC(check_rows(a->v, a->v_stride, kvd, "v", op));
    RC(check_rows(a->k_out, a->k_out_stride, kvd, "k_out", op));
    RC(check_rows(a->v_out, a->v_out_stride, kvd, "v_out", op));
    RC(check_outer(a->k_cache_stride, a->caches, "k", op));
    RC(check_outer(a->v_cache_stride, a->caches, "v", op));
    RC(check_outer(a->k_out_cache_stride, a->caches, "k_out", op));
    RC(check_outer(a->v_out_cache_stride, a->caches, "v_out", op));
    if (!a->rows || !a->counts) return fail(POCR_ERR_ARG, "%s: null rows or counts", op);
    if (!a->weights != !a->weights_out || !a->positions != !a->positions_out)
        return fail(POCR_ERR_ARG, "%s: weights and positions come with their destinations", op);
    for (const void *x : {(const void *)a->weights, (const void *)a->weights_out, (const void *)a->positions,
                          (const void *)a->positions_out, (const void *)a->rows, (const void *)a->counts, (const void *)a->first})
        RC(check_index(x, "an index or side buffer", op));
    RC(check_side(a->side_stride, a->max_rows, "side_stride", op));
    RC(check_side(a->side_out_stride, a->max_rows_out, "side_out_stride", op));
    CacheKeep p{};
    p.side = a->side_stride ? a->side_stride : a->max_rows;
    p.side_out = a->side_out_stride ? a->side_out_stride : a->max_rows_out;
    const bool inplace = a->k_out == a->k;
    if (inplace != (a->v_out == a->v) || (a->weights && inplace != (a->weights_out == a->weights)) ||
        (a->positions && inplace != (a->positions_out == a->positions)))
        return fail(POCR_ERR_ARG, "%s: K, V, weights and positions move in place together or not at all", op);
    if (inplace) {
        if (a->k_stride != a->k_out_stride || a->v_stride != a->v_out_stride ||
            (a->caches > 1 && (a->k_cache_stride != a->k_out_cache_stride || a->v_cache_stride != a->v_out_cache_stride)) ||
            a->max_rows != a->max_rows_out || ((a->weights || a->positions) && p.side != p.side_out))
            return fail(POCR_ERR_ARG, "%s: in place, the strides and row counts of source and destination are equal", op);
    }
    const int64_t sides = (int64_t)a->caches * a->kv_heads;
    const Area src[4] = {{a->k, a->k_cache_stride, a->k_stride, a->caches, a->max_rows, kvd},
                         {a->v, a->v_cache_stride, a->v_stride, a->caches, a->max_rows, kvd},
                         {a->weights, 0, p.side, 1, sides, a->max_rows},
                         {a->positions, 0, p.side, 1, sides, a->max_rows}};
    const Area dst[4] = {{a->k_out, a->k_out_cache_stride, a->k_out_stride, a->caches, a->max_rows_out, kvd},
                         {a->v_out, a->v_out_cache_stride, a->v_out_stride, a->caches, a->max_rows_out, kvd},
                         {a->weights_out, 0, p.side_out, 1, sides, a->max_rows_out},
                         {a->positions_out, 0, p.side_out, 1, sides, a->max_rows_out}};
    if (!inplace)
        for (int i = 0; i < 4; ++i)
            if (dst[i].at && overlap(src[i], dst[i])) return fail(POCR_ERR_ARG, "%s: a destination overlaps its source", op);
    CACHE_OP_CONTEXT(ctx, op);
    for (int i = 0; i < 2; ++i)
        if (overlap(dst[i], dst[i], true)) return fail(POCR_ERR_ARG, "%s: caches of the destination overlap", op);
    // What one workgroup writes no other reads, or writes otherwise: one buffer as
    // K and V goes to one destination elsewhere (the same values twice), not in place.
    const Area lists[3] = {{a->rows, 0, 0, 1, 1, (a->per_head ? sides : a->caches) * a->max_keep},
                           {a->counts, 0, 0, 1, 1, a->caches},
                           {a->first, 0, 0, 1, 1, a->caches}};
    const char *names[7] = {"K", "V", "weights", "positions", "rows", "counts", "first"};
    const bool twice = !inplace && a->k == a->v && a->k_out == a->v_out && a->k_stride == a->v_stride && a->k_out_stride == a->v_out_stride &&
                       (a->caches == 1 || (a->k_cache_stride == a->v_cache_stride && a->k_out_cache_stride == a->v_out_cache_stride));
    for (int i = 0; i < 4; ++i)
        for (int j = 0; dst[i].at && j < 7; ++j) {
            const Area &read = j < 4 ? src[j] : lists[j - 4];
            if (j == i || !read.at || (twice && i + j == 1)) continue;
            if (overlap(dst[i], read) || (j < i && overlap(dst[i], dst[j])))
                return fail(POCR_ERR_ARG, "%s: the destination of %s overlaps %s", op, names[i], names[j]);
        }
    CACHE_OP_DEVICE(ctx, stream, op);
    p.src[0] = a->k;
    p.src[1] = a->v;
    p.dst[0] = a->k_out;
    p.dst[1] = a->v_out;
    p.weights = a->weights;
    p.weights_out = a->weights_out;
    p.pos = a->positions;
    p.pos_out = a->positions_out;
    p.rows = a->rows;
    p.counts = a->counts;
    p.first = a->first;
    p.src_cs[0] = a->k_cache_stride;
    p.src_cs[1] = a->v_cache_stride;
    p.src_st[0] = a->k_stride;
    p.src_st[1] = a->v_stride;
    p.dst_cs[0] = a->k_out_cache_stride;
    p.dst_cs[1] = a->v_out_cache_stride;
    p.dst_st[0] = a->k_out_stride;
    p.dst_st[1] = a->v_out_stride;
    p.kvh = a->kv_heads;
    p.max_keep = a->max_keep;
    p.per_head = a->per_head != 0;
    p.max_rows = a->max_rows;
    p.max_rows_out = a->max_rows_out;
    hipStream_t s = (hipStream_t)stream;
    const int side = a->weights || a->positions ? 1 : 0;
    if (inplace && a->max_keep > kKeepRows) {
        const dim3 grid(2 * a->head_dim / kKeepSlab + side, a->kv_heads, a->caches);
        return launch(s, grid, kKeepThreads, a->head_dim == 128 ? k_cache_keep_slabs<128> : k_cache_keep_slabs<64>, p);
    }
    // no list is longer than its destination; lists of more workgroups than a grid holds take several
    const int chunks = round_up_div(std::min(a->max_keep, a->max_rows_out), kKeepRows), most = kMaxGrid / ((2 + side) * kKeepThreads);
    auto run = [&](auto kernel) {
        for (int at = 0; at < chunks; at += most)
            RC(launch(s, dim3((2 + side) * std::min(most, chunks - at), a->kv_heads, a->caches), kKeepThreads, kernel, p, at,
                      std::min(most, chunks - at), chunks));
        return (int)POCR_OK;
    };
    if (a->head_dim == 128) return run(inplace ? k_cache_keep<128, true> : k_cache_keep<128, false>);
    return run(inplace ? k_cache_keep<64, true> : k_cache_keep<64, false>);
}
