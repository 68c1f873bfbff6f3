// paged_attention.hip -- attention.h's attention over a cache in pages (paged.h): its
// entry point, checks and kernels.
#include <hip/hip_runtime.h>

#include <cmath>

#include "paged_attention.h"

namespace trs {

namespace {

constexpr int64_t kMaxHeadDim = 256;
constexpr int kFewTile = 16;  // rows of a tile of paged_few
// paged_few takes up to so many rows, and any number with fewer pairs of a row and a key in all, us in it / in
// paged_rows: one token or a few over 4096 keys, 8 key heads of 128, bfloat16, 64 rows of 1, 4 and 16 sequences
// 32 / 40, 46 / 50, 128 / 126, 128 rows 36 / 44, 66 / 56, 231 / 140; float32, 64 rows 36 / 44, 70 / 91, 218 / 292, 96 rows 45 / 46,
// 98 / 93, 378 / 296; rows of a batch over shared keys, bfloat16, 128 rows over 8192 keys 52 / 57 and 32768 126 / 99, 256 over 1024
// 38 / 43, 4096 54 / 52 and 8192 74 / 62, 512 over 1024 49 / 53 and 4096 81 / 68.
constexpr int kFewRows = 64;
constexpr int64_t kFewPairs = 1 << 23;
// Shared keys are worked on together where that saves so much reading, us apart / together, 8 key heads of 128: bfloat16,
// 2 sequences over 1024 keys (4 MiB) 17.2 / 17.9 and 4096 (16 MiB) 25.7 / 22.9, 4 over 1024 (12 MiB) 17.8 / 17.9, 8 over 256 (7 MiB)
// 16.3 / 17.3 and 1024 (28 MiB) 21.3 / 18.5; float32, 4 over 1024 (24 MiB) 24.0 / 20.5, 8 over 256 (14 MiB) 19.1 / 19.0.  Of shared keys
// a sequence reads at most what window, first tokens and new tokens leave: 64 tokens behind 8192 and 200 of their own, 32 heads,
// bfloat16, window 16 (4 MiB) 14.4 / 18.4, 512 (126 MiB) 28.2 / 32.6, 2048 (505 MiB) 63.0 / 48.0, float32, window 64 (32 MiB)
// 21.9 / 24.5: how many own keys a window has first stands on the device, and 512 and 64 count as more than they are.
constexpr int64_t kTogetherBytes = 16 << 20;
// A row's parts are joined by 16 waves of a block where as many have a lane's four each and rows are at most two a CU, by
// 4 where 2 do and rows are at most four a CU; us in all with 1, 4 and 16: one token over 14170 keys, one head of 256
// 52.7, 27.4 and 23.9, 2 over 15168, 2 heads of 200, float32 108, 50.5 and 40.4, one over 16384, 8 heads of 128 42.3, 27.2 and 25.3 and over
// 4000 19.6, 16.0 and 16.6, over 1000, 8 of 64, float32 12.9, 12.6 and 13.3, 8 tokens over 1024 keys (256 rows) 25.3, 24.6 and 25.6,
// 16 over 1000 (512 rows) 23.2, 23.1 and 26.1; 640 rows over 288 shared keys 32.8, 32.5 and 38.4, 1024 over 2048 35.0, 34.7 and -, 2048 over
// 8192 71.9, 73.6 and 92.8.

// The parts of rows, joined: a lane has four columns of a row's every `groups`-th part, `quads` lanes a part
// (a power of two), four of its parts on their way at once; a wave 64 / (quads groups) rows.  WAVES above 1: so
// many waves, a block, have every WAVES-th such share of one row's parts, and the first of them joins these.
template <int WAVES>
__global__ void __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) paged_join(PagedArgs a, int quads, int groups) {
    constexpr bool BLOCK = WAVES > 1;
    __shared__ at_f4 wave_o[WAVES][64];
    __shared__ float2 wave_ml[WAVES][64];
    const int64_t rows = (int64_t)a.batch * a.kv_heads * a.seq_rows;
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, quad = lane & (quads - 1), per = 64 / (quads * groups);
    const int group = (lane / quads & (groups - 1)) + (BLOCK ? wave * groups : 0), apart_by = groups * WAVES;
    const int64_t first = BLOCK ? (int64_t)blockIdx.x : (blockIdx.x * 4ll + wave) * per + lane / (quads * groups);
    const int64_t step = BLOCK ? (int64_t)gridDim.x : gridDim.x * 4ll * per;
    for (int64_t at = first; at < rows; at += step) {
        const int64_t head = at / a.seq_rows;
        const int r = (int)(at - head * a.seq_rows), b = (int)(head / a.kv_heads), hk = (int)(head - (int64_t)b * a.kv_heads);
        const int d = min(quad * 4, a.part_width - 4);
        float most = -__builtin_inff(), sum = 0.f;
        at_f4 o = (at_f4)(0.f);
        // Another maximum, sum and output of the row.
        const auto add = [&](float m, float l, const at_f4 &x) {
            const float now = __builtin_fmaxf(most, m), base = now == -__builtin_inff() ? 0.f : now;
            const float keep = __builtin_amdgcn_exp2f(most - base), f = __builtin_amdgcn_exp2f(m - base);
            sum = sum * keep + l * f, o = o * keep + x * f, most = now;
        };
        bool whole = false;
        for (int n = 0; n < a.stages; n++) {
            const PagedStage &s = a.stage[n];
            const int one = s.together ? b * a.seq_rows + r : r, tile = one / s.tile_rows;
            const int entry = s.together ? tile : b * s.row_tiles + tile;
            const int2 workers = s.found[(int64_t)hk * s.entries + entry];
            whole = a.stages == 1 && workers.x == workers.y;  // its worker wrote it
            if (whole) break;
            for (int w0 = workers.x + group; w0 <= workers.y; w0 += 4 * apart_by) {
                float m[4], l[4];
                at_f4 x[4];
#pragma unroll
                for (int p = 0; p < 4; p++) {
                    const int w = min(w0 + p * apart_by, workers.y);
                    const int64_t part = ((int64_t)hk * s.slots + slot_of_part(a, s, w, entry, w == workers.x)) * s.tile_rows + one - tile * s.tile_rows;
                    m[p] = s.part_ml[2 * part], l[p] = s.part_ml[2 * part + 1];
                    x[p] = *(const at_f4 *)(s.part_o + part * a.part_width + d);
                }
#pragma unroll
                for (int p = 0; p < 4; p++)
                    if (w0 + p * apart_by <= workers.y) add(m[p], l[p], x[p]);
            }
        }
        if (whole) continue;  // (the same in a whole block)
        for (int apart = quads; apart < quads * groups; apart *= 2) {
            const float m = __shfl_xor(most, apart), l = __shfl_xor(sum, apart);
            at_f4 x;
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = __shfl_xor(o[e], apart);
            add(m, l, x);
        }
        if constexpr (BLOCK) {
            __syncthreads();  // the last row's have been read
            wave_o[wave][lane] = o, wave_ml[wave][lane] = make_float2(most, sum);
            __syncthreads();
            if (wave != 0) continue;
#pragma unroll 5
            for (int w = 1; w < WAVES; w++) add(wave_ml[w][lane].x, wave_ml[w][lane].y, wave_o[w][lane]);
        }
        if (group != 0) continue;
        const int i = (int)a.by_group.divide((uint32_t)r);
        const int64_t h = (int64_t)hk * a.group + r - i * a.group;
        o *= a.pages.keys_of(b) - a.Sq + i < 0 ? 0.f : 1.f / sum;
        float *out = a.out + b * a.os.b + h * a.os.h + (int64_t)i * a.os.s + quad * 4;
#pragma unroll
        for (int q = 0; q < 4; q++)
            if (quad * 4 + q < a.D) out[q] = o[q];
        if (a.lse && quad == 0) a.lse[((int64_t)b * a.heads + h) * a.Sq + i] = log_sum(most, sum);
    }
}

// A stage of keys [from, to): its tiles of rows, and the blocks that share them.
PagedStage plan_stage(const PagedArgs &a, bool together, int from, int to, int cu_count, bool bf16) {
    PagedStage s{};
    s.together = together, s.from = from, s.to = to;
    const int64_t rows = together ? (int64_t)a.batch * a.seq_rows : a.seq_rows;
    const int64_t keys = std::min<int64_t>(to - from, (int64_t)a.window + a.sinks + a.Sq);
    const bool pairs = rows * (together ? 1 : a.batch) * a.kv_heads * keys < kFewPairs, few = rows <= kFewRows || a.D > kPiecesDim || pairs;
    s.tile_rows = few ? kFewTile : rows <= 128 && bf16 ? 128 : 256;
    s.row_tiles = (int32_t)((rows + s.tile_rows - 1) / s.tile_rows);
    s.entries = (int32_t)(together ? s.row_tiles : (int64_t)s.row_tiles * a.batch);
    const int shift = bf16 || s.tile_rows != kFewTile ? 5 : 4;
    s.least = 2;
    if (s.tile_rows == kFewTile) {
        // Two waves a SIMD, one of wide heads, which fill its registers: 64 rows over 6240 shared keys, heads of 256, bfloat16,
        // 30.1 us with 4 waves a CU and 33.6 with 8, 7 x 32 over 1838 33.8 and 41.0; the shares of many rows are evener with 8: 2 x 1024
        // tokens of 4096, 16 heads of 256 over 4 787 and 739.
        s.workers = std::max(1, (a.D > kPiecesDim && pairs ? 4 : 8) * cu_count / a.kv_heads);
        // A tile a wave where that gives every SIMD one at most and a row not too many parts, else two, us with 1 and 2: 500 keys,
        // 8 heads of 64, bfloat16 11.6 and 12.8, 1000, float32 11.6 and 12.6, 7 x 4 tokens of 432, 24 heads of 200 over 3 19.8 and 25.1; 3 x 4 of
        // 3000, 16 heads of 128 over 2 23.3 and 18.6, 14 of 7172 shared ones, 8 heads of 128, float32 33.3 and 28.8, 16384 keys, one head of 128
        // 19.1 and 17.6.
        const int64_t seen = (keys >> shift) + 1;
        if (seen <= 128 && seen * s.entries * a.kv_heads <= 4 * cu_count) s.least = 1;
    } else {
        s.workers = std::max(1, cu_count * (256 / s.tile_rows) / a.kv_heads);
    }
    s.by_row_tiles = SmallDivisor((uint32_t)s.row_tiles);
    const int64_t most = ((to - from) >> shift) + 2;  // key tiles of an entry
    s.most = (int32_t)most;
    if (most * s.entries >> 31) s.workers = 0;
    return s;
}

// A workspace that captured calls share: their replays follow one another on the library's stream.  A
// larger one leaves the smaller to the graphs that have it.
int graph_workspace(DeviceState *dev, size_t bytes, void **ws) {
    std::lock_guard<std::mutex> lock(dev->graph_mu);
    if (bytes > dev->graph_parts_bytes) {
        void *more = nullptr;
        TRS_CHECK(trs_alloc(bytes, &more));
        dev->graph_parts = more, dev->graph_parts_bytes = bytes;
    }
    *ws = dev->graph_parts;
    return TRS_OK;
}

// Memory for the stages' parts.
int take_parts(PagedArgs &a, DeviceState *dev, bool captured, void **ws) {
    size_t floats = 0, found = 0;
    for (int i = 0; i < a.stages; i++) {
        PagedStage &s = a.stage[i];
        s.slots = a.stages > 1 ? (int64_t)s.workers + s.entries : 2 * (int64_t)s.workers;
        floats += (size_t)(a.kv_heads * s.slots * s.tile_rows) * (size_t)(a.part_width + 2);
        found += (size_t)a.kv_heads * (size_t)s.entries;
    }
    const size_t bytes = floats * sizeof(float) + found * sizeof(int2);
    TRS_CHECK(captured ? graph_workspace(dev, bytes, ws) : trs_alloc(bytes, ws));
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

int paged_forward(PagedArgs &a, bool bf16, DeviceState *dev, bool captured) {
    a.part_width = (a.D + 3) / 4 * 4;
    a.stages = 0;
    const int64_t seen = std::min<int64_t>(a.shared, (int64_t)a.window + a.sinks + a.Sq);  // of the shared keys, by a sequence, at most
    const int64_t saved = (int64_t)(a.batch - 1) * seen * a.kv_heads * a.D * (bf16 ? 4 : 8);
    if (saved >= kTogetherBytes && (int64_t)a.batch * a.seq_rows < (int64_t)1 << 31) {
        a.all_rows = a.batch * a.seq_rows, a.by_seq_rows = SmallDivisor((uint32_t)a.seq_rows);
        a.stage[a.stages++] = plan_stage(a, true, 0, a.shared, dev->cu_count, bf16);
    }
    const int from = a.stages ? a.shared : 0;
    if (from < a.pages.capacity || a.stages == 0) a.stage[a.stages++] = plan_stage(a, false, from, a.pages.capacity, dev->cu_count, bf16);
    if (a.pages.capacity == 0) a.stages = 0;  // nobody sees anything
    // One stage with a worker for every entry: no parts, and nothing to join.
    const auto entry_each = [&]() {
        a.stages = 1, a.stage[1] = PagedStage{};
        a.stage[0] = plan_stage(a, false, 0, a.pages.capacity, dev->cu_count, bf16);
        a.stage[0].workers = 0;
    };
    if (a.stages == 2 && (a.stage[0].workers == 0 || a.stage[1].workers == 0)) entry_each();
    void *ws = nullptr;
    if (a.stages && a.stage[0].workers) {
        const int rc = take_parts(a, dev, captured, &ws);
        if (rc == TRS_E_ALLOCATION_FAILED) entry_each();  // the parts are for speed alone
        else if (rc) return rc;
    }
    const bool joins = a.stages == 0 || a.stage[0].workers;
    const auto launch = [&]() -> int {
        const auto few = [&](int i) { return a.stage[i].tile_rows == kFewTile; };
        if (a.stages == 2 && few(0) && few(1)) {
            TRS_CHECK(launch_paged_few(a, 0, 2, bf16, dev->stream));
        } else {
            for (int i = 0; i < a.stages; i++) TRS_CHECK(few(i) ? launch_paged_few(a, i, 1, bf16, dev->stream) : launch_paged_rows(a, i, bf16, dev->stream));
        }
        if (!joins) return TRS_OK;
        int quads = 1;
        while (quads * 4 < a.part_width) quads *= 2;
        // Waves have parts of few rows each, blocks two or three of many.
        const int64_t rows = (int64_t)a.batch * a.kv_heads * a.seq_rows;
        int64_t parts = 0;  // of a row, at most or so
        for (int i = 0; i < a.stages; i++) parts = std::max<int64_t>(parts, std::min(a.stage[i].workers / a.stage[i].entries, a.stage[i].most / a.stage[i].least));
        const int64_t waves = parts * quads / (4 * 64);  // of four parts a lane
        if (rows <= 2 * dev->cu_count && waves >= 16) {
            hipLaunchKernelGGL(paged_join<16>, dim3((unsigned)rows), dim3(1024), 0, dev->stream, a, quads, 64 / quads);
        } else if (rows <= 4 * dev->cu_count && waves >= 2) {
            hipLaunchKernelGGL(paged_join<4>, dim3((unsigned)rows), dim3(256), 0, dev->stream, a, quads, 64 / quads);
        } else {
            const int groups = a.stages && few(a.stages - 1) ? 64 / quads : 1;
            const int64_t lanes = rows * quads * groups;
            hipLaunchKernelGGL(paged_join<1>, dim3((unsigned)std::min<int64_t>((lanes + 255) / 256, 1 << 22)), dim3(256), 0, dev->stream, a, quads, groups);
        }
        TRS_LAUNCH_CHECK("paged attention join launch");
        return TRS_OK;
    };
    const int rc = launch(), frc = ws && !captured ? trs_free(ws) : TRS_OK;
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
        return set_error(TRS_E_INDEX_OVERFLOW, "attention over more than 2^29 tokens, or rows that share a key head");
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
    bool captured = false;
    TRS_CHECK(is_captured(dev, &captured));
    if (captured && D > 1 && lq->stride[3] != 1)
        return set_error(TRS_E_INVALID_ARGUMENT, "query needs a unit stride along its last dim in a captured call");
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
    return paged_forward(a, cache->type == TRS_PAGES_BF16, dev, captured);
}

}  // namespace

}  // namespace trs

extern "C" int trs_paged_attention_f32(const float *q, const trs_layout *lq, const trs_paged_cache *cache, int64_t shared,
                                       int64_t window, int64_t sinks, float scale, float *out, const trs_layout *lo,
                                       float *lse) {
    return trs::abi_guard([&]() -> int { return trs::run_paged(q, lq, cache, shared, window, sinks, scale, out, lo, lse); });
}
