// rope.hip -- the rotation of queries and keys by positions of several axes, and the
// appending of keys and values to a paged cache with that rotation on the way.
//
//   y = R x: pair j of the first `rot` entries, (j, j + rot/2) or, interleaved, (2j, 2j+1),
//   turns by the angle whose cosine and sine stand in entry j of the tables' row
//   positions[axis of j][batch][token]; the other entries pass.
// R is orthogonal, so its gradient is the rotation by the negative angles: the same call
// on the upstream gradient.
//
// Memory bounds it: 4 bytes read an entry and 4 written (2 to bfloat16 pages), with the
// tables' rows shared by a token's heads.
#include <hip/hip_runtime.h>

#include "paged.h"

namespace trs {

namespace {

constexpr int kMaxDim = 1024, kMostAxes = 4, kMaxPairs = kMaxDim / 2;
// Eights from which a lane has several heads of a token: 2 x 4096 tokens, 40 heads of 128, three axes, us with
// one, two and four heads a lane: 74, 63, 61; gradients of 4 x 2047 tokens, 20 heads of 64: 41, 43, 39; two prompts
// of 4096 tokens appended to float32 pages, 8 key heads of 128 and 32 of queries: 86, 73, 77.
constexpr int64_t kManyEights = 1 << 19;

// A tensor to be turned, or moved as it is: [batch, head, token, dim].
struct RopeJob {
    const float *x;
    void *y;  // the output, or a pool
    int64_t xs[4], ys[4];
    SmallDivisor by_chunk, by_inner;
    int32_t heads, units, batch_blocks;  // units of a sequence, and the blocks that they take
    int64_t first;                                    // first block
    int32_t turns, paged, heads_inner;  // rows walked with the heads innermost, else the tokens
};

struct RopeArgs {
    RopeJob job[3];
    int32_t jobs, tokens, batch, dim, rot, interleaved, axes;
    float sign;
    int64_t blocks;
    const float *cos, *sin;
    int64_t table_rows, table_stride, start;
    const int32_t *positions;  // [axis, batch, token]; null: start + token, or the place in the cache
    int32_t appends, bf16;
    Pages pages;
    uint32_t pair_axis[kMaxPairs / 16];  // two bits a pair
};

// A lane's token: where it stands in its sequence and in the pools.
struct Token {
    int place;     // below 0: padding; from the table's tokens on: no place
    int id, slot;  // its page; id < 0: nothing is to be written
};

__device__ __forceinline__ Token token_of(const RopeArgs &a, int b, int t) {
    Token k = {t, -1, 0};
    if (!a.appends) return k;
    k.place = max(a.pages.lengths[b], 0) - a.tokens + t;
    if (k.place < 0 || k.place >= a.pages.capacity) return k;
    const int id = a.pages.page_of(b, k.place);
    k.id = a.pages.holds(id) ? id : -1;
    k.slot = a.pages.slot_of(k.place);
    return k;
}

__device__ __forceinline__ int axis_of(const RopeArgs &a, int pair) { return (int)(a.pair_axis[pair >> 4] >> (pair & 15) * 2 & 3); }

// The row of the tables that an axis of a token reads; one outside [0, table_rows) is not read.
__device__ __forceinline__ int64_t row_of(const RopeArgs &a, int axis, int b, int t, const Token &k) {
    if (a.positions) return a.positions[((int64_t)axis * a.batch + b) * a.tokens + t];
    return a.appends ? max(k.place, 0) : a.start + t;
}

struct Angle {
    float co, si;
};
__device__ __forceinline__ Angle angle_of(const RopeArgs &a, int64_t row, int pair) {
    const bool known = row >= 0 && row < a.table_rows;
    const int64_t at = (known ? row : 0) * a.table_stride + pair;
    if (a.table_rows == 0) return {__builtin_nanf(""), __builtin_nanf("")};
    const float c = a.cos[at], s = a.sin[at] * a.sign;
    return known ? Angle{c, s} : Angle{__builtin_nanf(""), __builtin_nanf("")};
}

// (u, w) by an angle.
__device__ __forceinline__ void turn(float &u, float &w, float co, float si) {
    const float x = u * co - w * si;
    w = w * co + u * si;
    u = x;
}

// The angles of a lane's four pairs: p to p + 3, or, of neighbours, p and p + 1 and the two that lie
// rot/4 behind them.
struct Angles {
    float co[4], si[4];
};
__device__ __forceinline__ Angles angles_of(const RopeArgs &a, int b, int t, const Token &k, int p) {
    typedef float f2u __attribute__((ext_vector_type(2), aligned(4)));
    Angles g;
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const int pair = i == 0 ? p : a.interleaved ? p + a.rot / 4 : p + 2, axis = axis_of(a, pair);
        const int64_t row = row_of(a, axis, b, t, k);
        if (axis == axis_of(a, pair + 1) && a.table_rows) {
            const bool known = row >= 0 && row < a.table_rows;
            const int64_t at = (known ? row : 0) * a.table_stride + pair;
            const f2u c = *(const f2u *)(a.cos + at), s = *(const f2u *)(a.sin + at);
            const float nan = __builtin_nanf("");
#pragma unroll
            for (int e = 0; e < 2; e++) g.co[i + e] = known ? c[e] : nan, g.si[i + e] = known ? s[e] * a.sign : nan;
        } else {
            const Angle x = angle_of(a, row, pair), y = angle_of(a, row_of(a, axis_of(a, pair + 1), b, t, k), pair + 1);
            g.co[i] = x.co, g.si[i] = x.si, g.co[i + 1] = y.co, g.si[i + 1] = y.si;
        }
    }
    return g;
}

// The one rounding on the way to bfloat16 pages, of the turned fp32 value, to the nearest, ties to even.
typedef uint32_t u2u __attribute__((ext_vector_type(2), aligned(2)));
__device__ __forceinline__ uint32_t to_bf16(float x, float y) {
    typedef float F2 __attribute__((ext_vector_type(2)));
    typedef __bf16 B2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((F2{x, y}), B2));
}
__device__ __forceinline__ uint16_t to_bf16(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }

// Entries of any number, strides and rotation: a lane has a pair, or an entry that passes.
__device__ __forceinline__ void rope_pair(const RopeArgs &a, int64_t at_block) {
    int which = 0;
    while (which + 1 < a.jobs && at_block >= a.job[which + 1].first) which++;
    const RopeJob &j = a.job[which];
    const int64_t block = at_block - j.first;
    const int b = (int)(block / j.batch_blocks), u = (int)(block - (int64_t)b * j.batch_blocks) * 256 + (int)threadIdx.x;
    if (u >= j.units) return;
    const int r = (int)j.by_chunk.divide((uint32_t)u), c = u - r * (int)j.by_chunk.d;
    const int outer = (int)j.by_inner.divide((uint32_t)r), inner = r - outer * (int)j.by_inner.d;
    const int h = j.heads_inner ? inner : outer, t = j.heads_inner ? outer : inner;
    const int rot = j.turns ? a.rot : 0, half = rot / 2;
    const bool pair = c < half;
    const int e0 = pair ? (a.interleaved ? 2 * c : c) : half + c, e1 = pair ? (a.interleaved ? e0 + 1 : e0 + half) : e0;
    const Token k = token_of(a, b, t);
    const float *x = j.x + b * j.xs[0] + h * j.xs[1] + t * j.xs[2];
    float u0 = x[e0 * j.xs[3]], u1 = x[e1 * j.xs[3]];
    if (pair) {
        const Angle g = angle_of(a, row_of(a, axis_of(a, c), b, t, k), c);
        turn(u0, u1, g.co, g.si);
    }
    if (!j.paged) {
        float *y = (float *)j.y + b * j.ys[0] + h * j.ys[1] + t * j.ys[2];
        y[e0 * j.ys[3]] = u0;
        if (pair) y[e1 * j.ys[3]] = u1;
    } else if (k.id >= 0) {
        const int64_t at = k.id * j.ys[0] + h * j.ys[1] + k.slot * j.ys[2];
        if (a.bf16) {
            uint16_t *y = (uint16_t *)j.y + at;
            y[e0] = to_bf16(u0);
            if (pair) y[e1] = to_bf16(u1);
        } else {
            float *y = (float *)j.y + at;
            y[e0] = u0;
            if (pair) y[e1] = u1;
        }
    }
}
__global__ void __launch_bounds__(256) rope_pairs(RopeArgs a) {
    for (int64_t at = blockIdx.x; at < a.blocks; at += gridDim.x) rope_pair(a, at);
}

// Rows of whole eights (dim and rot multiples of 8, unit strides): a lane has four entries of the
// first half of what is turned and the four that lie rot/2 on, so that both partners of every pair
// are in it, or the like of what passes (eight in a row, read as two fours 32 bytes apart from lane
// to lane, are slower); of HEADS heads of a token, whose angles are the same.
template <int HEADS>
__device__ __forceinline__ void rope_eight(const RopeArgs &a, int64_t at_block) {
    int which = 0;
    while (which + 1 < a.jobs && at_block >= a.job[which + 1].first) which++;
    const RopeJob &j = a.job[which];
    const int64_t block = at_block - j.first;
    const int b = (int)(block / j.batch_blocks), u = (int)(block - (int64_t)b * j.batch_blocks) * 256 + (int)threadIdx.x;
    if (u >= j.units) return;
    const int r = (int)j.by_chunk.divide((uint32_t)u), c = u - r * (int)j.by_chunk.d;
    const int outer = (int)j.by_inner.divide((uint32_t)r), inner = r - outer * (int)j.by_inner.d;
    const int h0 = (j.heads_inner ? inner : outer) * HEADS, t = j.heads_inner ? outer : inner;
    const int rot = j.turns ? a.rot : 0;
    const bool turns = c * 8 < rot;
    const int at = turns ? c * 4 : rot + (c - rot / 8) * 4, half = (turns ? rot : a.dim - rot) / 2;
    const float *x = j.x + b * j.xs[0] + h0 * j.xs[1] + t * j.xs[2] + at;
    float v[HEADS][8];
#pragma unroll
    for (int n = 0; n < HEADS; n++) {
        const float *p = x + (h0 + n < j.heads ? n : 0) * j.xs[1];
        const f4u y = __builtin_nontemporal_load((const f4u *)p), z = __builtin_nontemporal_load((const f4u *)(p + half));
#pragma unroll
        for (int e = 0; e < 4; e++) v[n][e] = y[e], v[n][4 + e] = z[e];
    }
    const Token k = token_of(a, b, t);
    if (turns) {
        const Angles g = angles_of(a, b, t, k, a.interleaved ? at / 2 : at);
#pragma unroll
        for (int n = 0; n < HEADS; n++) {
            if (a.interleaved) {
#pragma unroll
                for (int e = 0; e < 4; e++) turn(v[n][2 * e], v[n][2 * e + 1], g.co[e], g.si[e]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) turn(v[n][e], v[n][4 + e], g.co[e], g.si[e]);
            }
        }
    }
    if (j.paged && k.id < 0) return;
    const int64_t to = (j.paged ? k.id * j.ys[0] + k.slot * j.ys[2] : b * j.ys[0] + t * j.ys[2]) + h0 * j.ys[1] + at;
#pragma unroll
    for (int n = 0; n < HEADS; n++) {
        if (h0 + n >= j.heads) break;
        const int64_t y = to + n * j.ys[1];
        if (j.paged && a.bf16) {
            uint16_t *p = (uint16_t *)j.y + y;
            *(u2u *)p = u2u{to_bf16(v[n][0], v[n][1]), to_bf16(v[n][2], v[n][3])};
            *(u2u *)(p + half) = u2u{to_bf16(v[n][4], v[n][5]), to_bf16(v[n][6], v[n][7])};
        } else {
            __builtin_nontemporal_store((f4u{v[n][0], v[n][1], v[n][2], v[n][3]}), (f4u *)((float *)j.y + y));
            __builtin_nontemporal_store((f4u{v[n][4], v[n][5], v[n][6], v[n][7]}), (f4u *)((float *)j.y + y + half));
        }
    }
}
template <int HEADS>
__global__ void __launch_bounds__(256) rope_eights(RopeArgs a) {
    for (int64_t at = blockIdx.x; at < a.blocks; at += gridDim.x) rope_eight<HEADS>(a, at);
}

// The rotation's arguments, as both entry points have them.
struct Rotation {
    const float *cos, *sin;
    const trs_layout *ltab;
    int interleaved, axes;
    const uint8_t *pair_axis;
    const int32_t *positions;
};

int take_rotation(const Rotation &r, int64_t dim, RopeArgs &a) {
    if (!r.ltab && !r.cos && !r.sin) return TRS_OK;  // nothing is turned
    TRS_CHECK(check_layout(r.ltab, "rotation table"));
    if (r.ltab->rank != 2) return set_error(TRS_E_INVALID_ARGUMENT, "rotation tables have rank 2, got %d", r.ltab->rank);
    const int64_t pairs = r.ltab->shape[1];
    if (pairs > dim / 2)
        return set_error(TRS_E_SHAPE_MISMATCH, "rotation tables of %lld pairs need a head dim of at least %lld, got %lld", (long long)pairs,
                         (long long)pairs * 2, (long long)dim);
    if (pairs > 1 && r.ltab->stride[1] != 1) return set_error(TRS_E_INVALID_ARGUMENT, "rotation tables need a unit stride along their rows");
    if (r.axes < 1 || r.axes > kMostAxes) return set_error(TRS_E_INVALID_ARGUMENT, "a rotation has 1 to %d axes, got %d", kMostAxes, r.axes);
    for (int64_t i = 0; r.pair_axis && i < pairs; i++) {
        if (r.pair_axis[i] >= r.axes)
            return set_error(TRS_E_INVALID_ARGUMENT, "pair %lld turns by axis %d of %d", (long long)i, r.pair_axis[i], r.axes);
        a.pair_axis[i / 16] |= (uint32_t)r.pair_axis[i] << (i % 16) * 2;
    }
    a.rot = (int32_t)(2 * pairs);
    a.interleaved = r.interleaved != 0;
    a.axes = r.axes;
    a.table_rows = r.ltab->shape[0], a.table_stride = r.ltab->stride[0];
    a.cos = r.cos ? r.cos + r.ltab->offset : nullptr;
    a.sin = r.sin ? r.sin + r.ltab->offset : nullptr;
    a.positions = r.positions;
    return TRS_OK;
}

int check_rows(const trs_layout *l, const char *what, const int64_t (&want)[4]) {
    TRS_CHECK(check_layout(l, what));
    if (l->rank != 4) return set_error(TRS_E_INVALID_ARGUMENT, "%s has rank %d, not 4 (batch, head, token, dim)", what, l->rank);
    for (int d = 0; d < 4; d++)
        if (want[d] >= 0 && l->shape[d] != want[d])
            return set_error(TRS_E_SHAPE_MISMATCH, "%s has size %lld in dim %d, expected %lld", what, (long long)l->shape[d], d, (long long)want[d]);
    if (l->shape[3] < 1 || l->shape[3] > kMaxDim) return set_error(TRS_E_INVALID_ARGUMENT, "head dim %lld outside [1, %d]", (long long)l->shape[3], kMaxDim);
    return TRS_OK;
}

RopeJob job_of(const float *x, const trs_layout *lx, bool turns) {
    RopeJob j{};
    j.x = x ? x + lx->offset : nullptr;
    for (int d = 0; d < 4; d++) j.xs[d] = lx->stride[d];
    j.heads = (int32_t)lx->shape[1];
    j.turns = turns;
    return j;
}
void to_rows(RopeJob &j, float *y, const trs_layout *lo) {
    j.y = y ? y + lo->offset : nullptr;
    for (int d = 0; d < 4; d++) j.ys[d] = lo->stride[d];
}
void to_pages(RopeJob &j, void *pool, const PoolView &v) {
    j.y = pool, j.paged = 1;
    j.ys[0] = (int64_t)v.p, j.ys[1] = v.h, j.ys[2] = (int64_t)v.s, j.ys[3] = 1;
}

// Launches the jobs that have elements.
int launch(RopeArgs &a) {
    int32_t n = 0;
    int64_t blocks = 0, eights = 0;
    bool whole = a.rot % 8 == 0 && a.dim % 8 == 0;
    for (int i = 0; i < a.jobs; i++) {
        const RopeJob &j = a.job[i];
        whole = whole && j.xs[3] == 1 && j.ys[3] == 1;
        eights += (int64_t)a.batch * j.heads * a.tokens * (a.dim / 8);
    }
    const int heads = !whole || eights < kManyEights ? 1 : a.appends ? 2 : 4;
    for (int i = 0; i < a.jobs; i++) {
        RopeJob j = a.job[i];
        const int64_t chunks = whole ? a.dim / 8 : j.turns ? a.dim - a.rot / 2 : a.dim, groups = (j.heads + heads - 1) / heads;
        const int64_t units = chunks * groups * a.tokens;
        if (units == 0 || a.batch == 0) continue;
        if (units >> 31) return set_error(TRS_E_INDEX_OVERFLOW, "rotation of more than 2^31 entries a sequence");
        j.units = (int32_t)units;
        j.heads_inner = j.xs[1] <= j.xs[2];
        j.by_chunk = SmallDivisor((uint32_t)chunks);
        j.by_inner = SmallDivisor((uint32_t)(j.heads_inner ? groups : a.tokens));
        j.batch_blocks = (int32_t)((units + 255) / 256);
        j.first = blocks;
        blocks += (int64_t)j.batch_blocks * a.batch;
        a.job[n++] = j;
    }
    a.jobs = n, a.blocks = blocks;
    if (n == 0) return TRS_OK;
    DeviceState *dev = device_state();
    if (!dev) return TRS_E_NO_DEVICE;
    const dim3 grid((unsigned)std::min<int64_t>(blocks, 1 << 22));
    if (!whole) hipLaunchKernelGGL(rope_pairs, grid, dim3(256), 0, dev->stream, a);
    else if (heads == 4) hipLaunchKernelGGL(rope_eights<4>, grid, dim3(256), 0, dev->stream, a);
    else if (heads == 2) hipLaunchKernelGGL(rope_eights<2>, grid, dim3(256), 0, dev->stream, a);
    else hipLaunchKernelGGL(rope_eights<1>, grid, dim3(256), 0, dev->stream, a);
    TRS_LAUNCH_CHECK("rotation launch");
    return TRS_OK;
}

// An input whose output is its own view is no other operand.
bool in_place(const float *x, const trs_layout *lx, const float *y, const trs_layout *ly) {
    return x && y && x + lx->offset == y + ly->offset && same_view_shape(lx, ly);
}

int run_rope(int n, const float *const *x, const trs_layout *lx, const Rotation &r, int64_t start, int inverse, float *const *out,
             const trs_layout *lo) {
    if (n < 1 || n > 2) return set_error(TRS_E_INVALID_ARGUMENT, "rotation takes 1 or 2 tensors, got %d", n);
    if (!x || !lx || !out || !lo) return set_error(TRS_E_INVALID_ARGUMENT, "null rotation argument");
    if (!r.ltab) return set_error(TRS_E_INVALID_ARGUMENT, "rotation table layout is null");
    RopeArgs a{};
    a.jobs = n, a.sign = inverse ? -1.f : 1.f, a.start = start;
    for (int i = 0; i < n; i++) {
        TRS_CHECK(check_rows(&lx[i], "rotation input", {-1, -1, -1, -1}));
        if (i && (lx[i].shape[0] != lx[0].shape[0] || lx[i].shape[2] != lx[0].shape[2] || lx[i].shape[3] != lx[0].shape[3]))
            return set_error(TRS_E_SHAPE_MISMATCH, "queries and keys differ in batch, tokens or head dim");
        TRS_CHECK(check_rows(&lo[i], "rotation output", {lx[i].shape[0], lx[i].shape[1], lx[i].shape[2], lx[i].shape[3]}));
        TRS_CHECK(check_written_once(&lo[i], "rotation output"));
    }
    const int64_t batch = lx[0].shape[0], tokens = lx[0].shape[2];
    if (batch > INT32_MAX || tokens > kMaxPagedTokens || lx[0].shape[1] > INT32_MAX || lx[n - 1].shape[1] > INT32_MAX)
        return set_error(TRS_E_INDEX_OVERFLOW, "rotation of more than 2^29 tokens, or of 2^31 sequences or heads");
    a.batch = (int32_t)batch, a.tokens = (int32_t)tokens, a.dim = (int32_t)lx[0].shape[3];
    TRS_CHECK(take_rotation(r, a.dim, a));
    if (!r.positions && batch > 0 && tokens > 0 && (start < 0 || start > a.table_rows - tokens))
        return set_error(TRS_E_INVALID_ARGUMENT, "positions %lld to %lld outside the rotation tables' %lld rows", (long long)start,
                         (long long)(start + tokens - 1), (long long)a.table_rows);
    const auto input = [&](int i) { return in_place(x[i], &lx[i], out[i], &lo[i]) ? Operand{"input", nullptr, nullptr, false, 0} : Operand{"input", x[i], &lx[i], false}; };
    const Operand none{"", nullptr, nullptr, false, 0};
    const Operand ops[] = {
        input(0), n > 1 ? input(1) : none, {"output", out[0], &lo[0], true}, n > 1 ? Operand{"output", out[1], &lo[1], true} : none,
        {"cosines", r.cos, r.ltab, false}, {"sines", r.sin, r.ltab, false},
        {"positions", r.positions, nullptr, false, r.positions ? a.axes * batch * tokens : 0},
    };
    TRS_CHECK(check_memory(ops));
    for (int i = 0; i < n; i++) {
        a.job[i] = job_of(x[i], &lx[i], true);
        to_rows(a.job[i], out[i], &lo[i]);
    }
    return launch(a);
}

int run_append(const trs_paged_cache *cache, const float *k, const trs_layout *lk, const float *v, const trs_layout *lv, const float *q,
               const trs_layout *lq, float *q_out, const trs_layout *lqo, const Rotation &r) {
    RopeArgs a{};
    if (!cache) return set_error(TRS_E_INVALID_ARGUMENT, "paged cache is null");
    TRS_CHECK(check_rows(lk, "key", {-1, cache->lk.rank == 4 ? cache->lk.shape[1] : -1, -1, cache->lk.rank == 4 ? cache->lk.shape[3] : -1}));
    const int64_t batch = lk->shape[0], tokens = lk->shape[2];
    TRS_CHECK(check_rows(lv, "value", {batch, lk->shape[1], tokens, lk->shape[3]}));
    const bool query = lq != nullptr;
    if (query) {
        TRS_CHECK(check_rows(lq, "query", {batch, -1, tokens, lk->shape[3]}));
        TRS_CHECK(check_rows(lqo, "turned query", {batch, lq->shape[1], tokens, lk->shape[3]}));
        TRS_CHECK(check_written_once(lqo, "turned query"));
    } else if (q || q_out || lqo) {
        return set_error(TRS_E_INVALID_ARGUMENT, "a query or its output without the query's layout");
    }
    if (batch > INT32_MAX || tokens > kMaxPagedTokens || lk->shape[1] > INT32_MAX || (query && lq->shape[1] > INT32_MAX))
        return set_error(TRS_E_INDEX_OVERFLOW, "appending more than 2^29 tokens, or to 2^31 sequences or heads");
    TRS_CHECK(check_cache(cache, batch, &a.pages));
    a.batch = (int32_t)batch, a.tokens = (int32_t)tokens, a.dim = (int32_t)lk->shape[3];
    a.appends = 1, a.bf16 = cache->type == TRS_PAGES_BF16, a.sign = 1.f;
    TRS_CHECK(take_rotation(r, a.dim, a));
    const Operand none{"", nullptr, nullptr, false, 0};
    const Operand ops[] = {
        {"key", k, lk, false},
        {"value", v, lv, false},
        query && !in_place(q, lq, q_out, lqo) ? Operand{"query", q, lq, false} : none,
        query ? Operand{"turned query", q_out, lqo, true} : none,
        r.ltab ? Operand{"cosines", r.cos, r.ltab, false} : none,
        r.ltab ? Operand{"sines", r.sin, r.ltab, false} : none,
        {"positions", r.positions, nullptr, false, r.ltab && r.positions ? a.axes * batch * tokens : 0},
        {"page table", cache->table, nullptr, false, batch * cache->table_width},
        {"lengths", cache->lengths, nullptr, false, batch},
    };
    TRS_CHECK(check_memory(ops));
    TRS_CHECK(check_pools(cache, true, ops));
    a.job[0] = job_of(k, lk, true);
    to_pages(a.job[0], a.pages.k, a.pages.ks);
    a.job[1] = job_of(v, lv, false);
    to_pages(a.job[1], a.pages.v, a.pages.vs);
    a.jobs = 2;
    if (query) {
        a.job[2] = job_of(q, lq, true);
        to_rows(a.job[2], q_out, lqo);
        a.jobs = 3;
    }
    return launch(a);
}

}  // namespace

}  // namespace trs

extern "C" int trs_rope_axes_f32(int n, const float *const *x, const trs_layout *lx, const float *cos, const float *sin,
                                 const trs_layout *ltab, int interleaved, int axes, const uint8_t *pair_axis,
                                 const int32_t *positions, int64_t start, int inverse, float *const *out,
                                 const trs_layout *lo) {
    return trs::abi_guard([&]() -> int {
        return trs::run_rope(n, x, lx, {cos, sin, ltab, interleaved, axes, pair_axis, positions}, start, inverse, out, lo);
    });
}

extern "C" int trs_paged_append_f32(const trs_paged_cache *cache, const float *k, const trs_layout *lk, const float *v,
                                    const trs_layout *lv, const float *q, const trs_layout *lq, float *q_out,
                                    const trs_layout *lqo, const float *cos, const float *sin, const trs_layout *ltab,
                                    int interleaved, int axes, const uint8_t *pair_axis, const int32_t *positions) {
    return trs::abi_guard([&]() -> int {
        return trs::run_append(cache, k, lk, v, lv, q, lq, q_out, lqo, {cos, sin, ltab, interleaved, axes, pair_axis, positions});
    });
}
