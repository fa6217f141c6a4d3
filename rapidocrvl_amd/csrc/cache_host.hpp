// cache_host.hpp — what the entry points of the cache operators share: argument
// checks, the device and stream of a call, launches, memory of buffers.
#pragma once

#include <cfloat>
#include <cmath>
#include <type_traits>

#include "internal.hpp"

namespace {

using namespace pocr;

constexpr int kMaxGridYZ = 65535;
constexpr int64_t kMaxGrid = 0xffffffff;  // threads along x
constexpr int kMaxCacheRows = 1 << 30;
constexpr int kMaxQueryHeads = 1024;
constexpr float kLeast = FLT_MIN, kMost = 0x1p126f;  // of scale and cap

// The calling thread's device becomes the context's for one call.
struct DeviceScope {
    int was = -1;
    int enter(int device) {
        int now = 0;
        HIP_TRY(hipGetDevice(&now));
        if (now == device) return POCR_OK;
        HIP_TRY(hipSetDevice(device));
        was = now;
        return POCR_OK;
    }
    ~DeviceScope() {
        if (was >= 0) (void)hipSetDevice(was);
    }
};

int check_stream(const pocr_ctx *ctx, hipStream_t s, const char *op) {
    if (!s) return POCR_OK;
    hipDevice_t dev = 0;
    if (hipStreamGetDevice(s, &dev) != hipSuccess) {
        (void)hipGetLastError();  // answered here: no later check finds it
        return fail(POCR_ERR_ARG, "%s: not a stream of the HIP runtime that this library runs on", op);
    }
    if (dev != ctx->device) return fail(POCR_ERR_ARG, "%s: a stream of device %d, the context is on %d", op, dev, ctx->device);
    return POCR_OK;
}

#define CACHE_OP_CONTEXT(ctx, op)                                  \
    if (!(ctx)) return fail(POCR_ERR_ARG, "%s: null context", op); \
    CHECK_INJECT((op) + 5) /* the name without pocr_ */

#define CACHE_OP_DEVICE(ctx, stream, op) \
    DeviceScope scope_;                  \
    RC(scope_.enter((ctx)->device));     \
    RC(check_stream(ctx, (hipStream_t)(stream), op))

#define CACHE_OP_ENTER(ctx, stream, op) \
    CACHE_OP_CONTEXT(ctx, op);          \
    CACHE_OP_DEVICE(ctx, stream, op)

// Queues a kernel and answers for that alone: the thread's last error may be
// anyone's, an application's handled one or another call's.
template <class... P, class... A>
int launch(hipStream_t s, dim3 grid, int threads, void (*kernel)(P...), A... args) {
    static_assert((std::is_same_v<P, A> && ...), "arguments are passed by address");
    void *at[] = {&args...};
    HIP_TRY(hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, dim3(threads), at, 0, s));
    return POCR_OK;
}

bool aligned(const void *p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

int check_heads(int heads, int kv_heads, int head_dim, const char *op) {
    if (heads < 1 || kv_heads < 1 || heads % kv_heads || heads > kMaxQueryHeads)
        return fail(POCR_ERR_ARG, "%s: %d heads over %d KV heads", op, heads, kv_heads);
    if (head_dim != 64 && head_dim != 128) return fail(POCR_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", op, head_dim);
    return POCR_OK;
}

// Both meet log2(e), and a cap its reciprocal, as factors in fp32.
int check_scores(float scale, float cap, const char *op) {
    if (!(scale == 0.0f || (scale >= kLeast && scale <= kMost))) return fail(POCR_ERR_ARG, "%s: scale must be 0 or 2^-126 to 2^126", op);
    if (!(cap == 0.0f || (cap >= kLeast && cap <= kMost))) return fail(POCR_ERR_ARG, "%s: cap must be 0 or 2^-126 to 2^126", op);
    return POCR_OK;
}

// rows of `width` floats, `stride` apart
int check_rows(const void *p, int64_t stride, int64_t width, const char *what, const char *op) {
    if (!p) return fail(POCR_ERR_ARG, "%s: null %s", op, what);
    if (!aligned(p, 16)) return fail(POCR_ERR_ARG, "%s: %s is not 16-byte aligned", op, what);
    if (stride < width || stride % 4) return fail(POCR_ERR_ARG, "%s: %s rows %lld floats apart: at least %lld, a multiple of 4", op, what, (long long)stride, (long long)width);
    return POCR_OK;
}

// `count` blocks of rows, `stride` apart (any multiple of 4 where there is one)
int check_outer(int64_t stride, int count, const char *what, const char *op) {
    if (count > 1 && (stride < 1 || stride % 4)) return fail(POCR_ERR_ARG, "%s: %s blocks %lld floats apart", op, what, (long long)stride);
    return POCR_OK;
}

int check_index(const void *p, const char *what, const char *op, size_t a = 4) {
    return aligned(p, a) ? POCR_OK : fail(POCR_ERR_ARG, "%s: %s is not %zu-byte aligned", op, what, a);
}

int check_workspace(const void *p, int64_t have, int64_t need, const char *op) {
    if (need && (!p || !aligned(p, 16) || have < need))
        return fail(POCR_ERR_ARG, "%s: needs a 16-byte aligned workspace of %lld bytes, has %lld", op, (long long)need, (long long)(p ? have : 0));
    return POCR_OK;
}

int check_side(int64_t stride, int rows, const char *what, const char *op) {
    if (stride && stride < rows) return fail(POCR_ERR_ARG, "%s: %s %lld for %d rows", op, what, (long long)stride, rows);
    return POCR_OK;
}

float default_scale(float scale, int head_dim) { return scale > 0.0f ? scale : (float)(1.0 / std::sqrt((double)head_dim)); }

int round_up_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// Memory of one buffer: `blocks` blocks of `rows` rows of `width` floats.
struct Area {
    const void *at;
    int64_t outer, inner;  // floats from block to block and from row to row
    int64_t blocks, rows, width;
    int64_t block() const { return (rows - 1) * inner + width; }
};

// The numbers k in [least, most] for which a span of `a` floats and one of `b`
// floats, d - k * step behind its start, share some: [*from, *to] (step > 0).
bool meeting(int64_t d, int64_t step, int64_t least, int64_t most, int64_t a, int64_t b, int64_t *from, int64_t *to) {
    auto floor_div = [](int64_t x, int64_t y) { return x / y - (x % y < 0); };
    *from = std::max(least, floor_div(d - a, step) + 1);  // d - k * step < a
    *to = std::min(most, -floor_div(-d - b, step) - 1);   // d - k * step > -b
    return *from <= *to;
}

// Rows of a block of x and of one of y, d floats behind it, share memory.
// Rows of two strides count as meeting where their blocks do.
bool rows_meet(const Area &x, const Area &y, int64_t d) {
    if (d >= x.block() || d <= -y.block()) return false;
    if (x.rows > 1 && y.rows > 1 && x.inner != y.inner) return true;
    const int64_t step = x.rows > 1 ? x.inner : (y.rows > 1 ? y.inner : 1);
    int64_t from, to;
    return x.rows == 1 && y.rows == 1 ? true : meeting(d, step, 1 - y.rows, x.rows - 1, x.width, y.width, &from, &to);
}

// x and y share memory (other: of two different blocks, x and y being one
// buffer).  Interleaved blocks and rows do not meet, as where several caches lie
// in one pool; blocks of two strides count as meeting where their ranges do.
bool overlap(const Area &x, const Area &y, bool other = false) {
    const int64_t bytes = (int64_t)(reinterpret_cast<uintptr_t>(y.at) - reinterpret_cast<uintptr_t>(x.at));
    const int64_t d = bytes / 4 - (bytes % 4 < 0);  // addresses are multiples of 4
    if (d >= (x.blocks - 1) * x.outer + x.block() || d <= -((y.blocks - 1) * y.outer + y.block())) return false;
    if (x.blocks > 1 && y.blocks > 1 && x.outer != y.outer) return true;
    if (x.blocks == 1 && y.blocks == 1) return !other && rows_meet(x, y, d);
    const int64_t step = x.blocks > 1 ? x.outer : y.outer;
    int64_t from, to;
    if (!meeting(d, step, 1 - y.blocks, x.blocks - 1, x.block(), y.block(), &from, &to)) return false;
    for (int64_t k = from; k <= to; ++k)
        if (!(other && k == 0) && rows_meet(x, y, d - k * step)) return true;
    return false;
}

}  // namespace
