// paged_attention.hip -- attention.h's attention over a cache in pages (paged.h): its
// entry point, checks and kernels.
#include <hip/hip_runtime.h>

#include <cmath>

#include "paged_attention.h"

namespace trs {

namespace {

constexpr int64_t kMaxHeadDim = 256;
constexpr int kFewTile = 16;  // rows of a tile of paged_few
constexpr int kFewRows = 32;

// The parts of a row, joined: four columns a lane.  Every part is read before the first is
// added, up to eight.
__global__ void __launch_bounds__(256) paged_join(PagedArgs a) {
    const int64_t rows = (int64_t)a.batch * a.kv_heads * a.seq_rows;
    const uint32_t quads = (uint32_t)a.part_width / 4;
    const int64_t lane = (int64_t)blockIdx.x * 256 + threadIdx.x, at = lane / quads;
    if (at >= rows) return;
    const int d = (int)(lane - at * quads) * 4;
    const int64_t head = at / a.seq_rows;
    const int r = (int)(at - head * a.seq_rows), b = (int)(head / a.kv_heads), hk = (int)(head - (int64_t)b * a.kv_heads);
    float most = -__builtin_inff(), sum = 0.f;
    at_f4 o = (at_f4)(0.f);
    for (int n = 0; n < a.stages; n++) {
        const PagedStage &s = a.stage[n];
        const int one = s.together ? b * a.seq_rows + r : r, tile = one / s.tile_rows;
        const int entry = s.together ? tile : b * s.row_tiles + tile;
        const int2 blocks = s.found[(int64_t)hk * s.entries + entry];
        if (a.stages == 1 && blocks.x == blocks.y) return;  // its block wrote it
        const int parts = blocks.y - blocks.x + 1;
        for (int p0 = 0; p0 < parts; p0 += 8) {
            float m[8], l[8];
            at_f4 x[8];
#pragma unroll
            for (int p = 0; p < 8; p++) {
                const int w = min(blocks.x + p0 + p, blocks.y);
                const int64_t part = ((int64_t)hk * s.slots + slot_of_part(a, s, w, entry, w == blocks.x)) * s.tile_rows + one - tile * s.tile_rows;
                m[p] = s.part_ml[2 * part], l[p] = s.part_ml[2 * part + 1];
                x[p] = *(const at_f4 *)(s.part_o + part * a.part_width + d);
            }
            float now = most;
#pragma unroll
            for (int p = 0; p < 8; p++) now = __builtin_fmaxf(now, m[p]);
            const float base = now == -__builtin_inff() ? 0.f : now, keep = __builtin_amdgcn_exp2f(most - base);
            sum *= keep, o *= keep, most = now;
#pragma unroll
            for (int p = 0; p < 8; p++) {
                if (p0 + p >= parts) break;
                const float f = __builtin_amdgcn_exp2f(m[p] - base);
                sum += l[p] * f, o += x[p] * f;
            }
        }
    }
    const int i = (int)a.by_group.divide((uint32_t)r);
    const int64_t h = (int64_t)hk * a.group + r - i * a.group;
    o *= a.pages.keys_of(b) - a.Sq + i < 0 ? 0.f : 1.f / sum;
    float *out = a.out + b * a.os.b + h * a.os.h + (int64_t)i * a.os.s + d;
#pragma unroll
    for (int q = 0; q < 4; q++)
        if (d + q < a.D) out[q] = o[q];
    if (a.lse && d == 0) a.lse[((int64_t)b * a.heads + h) * a.Sq + i] = log_sum(most, sum);
}

// A stage of keys [from, to): its tiles of rows, and the blocks that share them.
PagedStage plan_stage(const PagedArgs &a, bool together, int from, int to, int cu_count, bool bf16) {
    PagedStage s{};
    s.together = together, s.from = from, s.to = to;
    const int64_t rows = together ? (int64_t)a.batch * a.seq_rows : a.seq_rows;
    s.tile_rows = rows <= kFewRows || a.D > kPiecesDim ? kFewTile : rows <= 128 && bf16 ? 128 : 256;
    s.row_tiles = (int32_t)((rows + s.tile_rows - 1) / s.tile_rows);
    s.entries = (int32_t)(together ? s.row_tiles : (int64_t)s.row_tiles * a.batch);
    if (s.tile_rows == kFewTile) {
        s.least = bf16 ? 4 : 8;
        s.blocks = std::max(1, 2 * cu_count / a.kv_heads);
    } else {
        s.least = 2;
        s.blocks = std::max(1, cu_count * (256 / s.tile_rows) / a.kv_heads);
    }
    return s;
}

// Whether the stages have memory for parts; the parts are for speed alone.
int take_parts(PagedArgs &a, void **ws) {
    size_t floats = 0, found = 0;
    for (int i = 0; i < a.stages; i++) {
        PagedStage &s = a.stage[i];
        s.slots = a.stages > 1 ? (int64_t)s.blocks + s.entries : 2 * (int64_t)s.blocks;
        floats += (size_t)(a.kv_heads * s.slots * s.tile_rows) * (size_t)(a.part_width + 2);
        found += (size_t)a.kv_heads * (size_t)s.entries;
    }
    TRS_CHECK(trs_alloc(floats * sizeof(float) + found * sizeof(int2), ws));
    float *p = (float *)*ws;
    for (int i = 0; i < a.stages; i++) {
        PagedStage &s = a.stage[i];
        const size_t parts = (size_t)(a.kv_heads * s.slots * s.tile_rows);
        s.part_o = p, s.part_ml = p + parts * (size_t)a.part_width;
        p += parts * (size_t)(a.part_width + 2);
    }
    for (int i = 0; i < a.stages; i++) {
        PagedStage &s = a.stage[i];
        s.found = (int2 *)p;
        p += 2 * (size_t)a.kv_heads * (size_t)s.entries;
    }
    return TRS_OK;
}

int paged_forward(PagedArgs &a, bool bf16, DeviceState *dev) {
    a.part_width = (a.D + 3) / 4 * 4;
    a.stages = 0;
    if (a.shared > 0 && a.batch > 1 && (int64_t)a.batch * a.seq_rows < (int64_t)1 << 31) {
        a.all_rows = a.batch * a.seq_rows, a.by_seq_rows = SmallDivisor((uint32_t)a.seq_rows);
        a.stage[a.stages++] = plan_stage(a, true, 0, a.shared, dev->cu_count, bf16);
    }
    const int from = a.stages ? a.shared : 0;
    if (from < a.pages.capacity || a.stages == 0) a.stage[a.stages++] = plan_stage(a, false, from, a.pages.capacity, dev->cu_count, bf16);
    void *ws = nullptr;
    const int rc0 = take_parts(a, &ws);
    if (rc0 == TRS_E_ALLOCATION_FAILED) {
        a.stages = 1;
        a.stage[0] = plan_stage(a, false, 0, a.pages.capacity, dev->cu_count, bf16);
        a.stage[0].blocks = 0;
    } else if (rc0) {
        return rc0;
    }
    const auto launch = [&]() -> int {
        const auto few = [&](int i) { return a.stage[i].tile_rows == kFewTile; };
        if (a.stages == 2 && few(0) && few(1)) {
            TRS_CHECK(launch_paged_few(a, 0, 2, bf16, dev->stream));
        } else {
            for (int i = 0; i < a.stages; i++) TRS_CHECK(few(i) ? launch_paged_few(a, i, 1, bf16, dev->stream) : launch_paged_rows(a, i, bf16, dev->stream));
        }
        if (!ws) return TRS_OK;
        const int64_t lanes = (int64_t)a.batch * a.kv_heads * a.seq_rows * (a.part_width / 4);
        if ((lanes + 255) / 256 >> 24) return set_error(TRS_E_INVALID_ARGUMENT, "attention over %lld rows", (long long)a.batch * a.seq_rows);
        hipLaunchKernelGGL(paged_join, dim3((unsigned)((lanes + 255) / 256)), dim3(256), 0, dev->stream, a);
        TRS_LAUNCH_CHECK("paged attention join launch");
        return TRS_OK;
    };
    const int rc = launch(), frc = ws ? trs_free(ws) : TRS_OK;
    return rc ? rc : frc;
}

int run_paged(const float *q, const trs_layout *lq, const trs_paged_cache *cache, int64_t shared, int64_t window, int64_t sinks, float scale,
              float *out, const trs_layout *lo, float *lse) {
    if (!cache) return set_error(TRS_E_INVALID_ARGUMENT, "paged cache is null");
    TRS_CHECK(check_layout(lq, "query"));
    TRS_CHECK(check_layout(lo, "output"));
    if (lq->rank != 4) return set_error(TRS_E_INVALID_ARGUMENT, "query has rank %d, not 4 (batch, head, token, dim)", lq->rank);
    if (lo->rank != 4) return set_error(TRS_E_SHAPE_MISMATCH, "output has rank %d, not 4 (batch, head, token, dim)", lo->rank);
    for (int d = 0; d < 4; d++)
        if (lo->shape[d] != lq->shape[d]) return set_error(TRS_E_SHAPE_MISMATCH, "query and output differ in dim %d", d);
    const int64_t B = lq->shape[0], H = lq->shape[1], Sq = lq->shape[2], D = lq->shape[3];
    PagedArgs a{};
    TRS_CHECK(check_cache(cache, B, &a.pages));
    const int64_t HK = cache->lk.shape[1];
    if (D < 1 || D > kMaxHeadDim) return set_error(TRS_E_INVALID_ARGUMENT, "head dim %lld outside [1, %lld]", (long long)D, (long long)kMaxHeadDim);
    if (cache->lk.shape[3] != D) return set_error(TRS_E_SHAPE_MISMATCH, "pages have a head dim of %lld, queries %lld", (long long)cache->lk.shape[3], (long long)D);
    if (HK < 1 ? H != 0 : H % HK != 0)
        return set_error(TRS_E_SHAPE_MISMATCH, "%lld query heads cannot share %lld key heads", (long long)H, (long long)HK);
    if (window < 1) return set_error(TRS_E_INVALID_ARGUMENT, "attention window has to be at least 1, got %lld", (long long)window);
    if (sinks < 0) return set_error(TRS_E_INVALID_ARGUMENT, "attention sinks have to be at least 0, got %lld", (long long)sinks);
    if (shared < 0) return set_error(TRS_E_INVALID_ARGUMENT, "shared keys have to be at least 0, got %lld", (long long)shared);
    if (!std::isfinite(scale)) return set_error(TRS_E_INVALID_ARGUMENT, "attention scale has to be finite");
    if (Sq > kMaxPagedTokens || B > INT32_MAX || H > INT32_MAX || (HK > 0 && (H / HK) * Sq > kMaxPagedTokens) ||
        (HK > 0 && B * (((H / HK) * Sq + kFewTile - 1) / kFewTile) > INT32_MAX))
        return set_error(TRS_E_INDEX_OVERFLOW, "attention over more than 2^30 tokens, or rows that share a key head");
    TRS_CHECK(check_written_once(lo, "output"));
    if (D > 1 && lo->stride[3] != 1) return set_error(TRS_E_INVALID_ARGUMENT, "output needs a unit stride along its last dim");
    const int64_t rows = B * H * Sq;
    const Operand ops[] = {
        {"query", q, lq, false},
        {"output", out, lo, true},
        {"lse", lse, nullptr, true, lse ? rows : 0},
        {"page table", cache->table, nullptr, false, B * cache->table_width},
        {"lengths", cache->lengths, nullptr, false, B},
    };
    TRS_CHECK(check_memory(ops));
    TRS_CHECK(check_pools(cache, false, ops));
    if (rows == 0) return TRS_OK;
    DeviceState *dev = device_state();
    if (!dev) return TRS_E_NO_DEVICE;
    Dense dense;
    TRS_CHECK(dense.take(q, lq));
    a.q = dense.at, a.qs = dense.view;
    a.out = out + lo->offset, a.os = {lo->stride[0], lo->stride[1], lo->stride[2]};
    a.lse = lse;
    a.batch = (int32_t)B, a.heads = (int32_t)H, a.kv_heads = (int32_t)HK, a.group = (int32_t)(H / HK), a.Sq = (int32_t)Sq, a.D = (int32_t)D;
    const int64_t most = std::max(a.pages.capacity, 1);
    a.window = (int32_t)std::min(window, most), a.sinks = (int32_t)std::min(sinks, most), a.shared = (int32_t)std::min<int64_t>(shared, a.pages.capacity);
    a.scale2 = scale * kLog2e;
    a.seq_rows = a.group * a.Sq;
    a.by_group = SmallDivisor((uint32_t)a.group);
    return paged_forward(a, cache->type == TRS_PAGES_BF16, dev);
}

}  // namespace

}  // namespace trs

extern "C" int trs_paged_attention_f32(const float *q, const trs_layout *lq, const trs_paged_cache *cache, int64_t shared,
                                       int64_t window, int64_t sinks, float scale, float *out, const trs_layout *lo,
                                       float *lse) {
    return trs::abi_guard([&]() -> int { return trs::run_paged(q, lq, cache, shared, window, sinks, scale, out, lo, lse); });
}
