// paged_attention.hip -- attention.h's attention over a cache in pages (paged.h): its
// entry point, checks and kernels.
#include <hip/hip_runtime.h>

#include <cmath>

#include "attention.h"
#include "paged.h"

namespace trs {

namespace {

constexpr int64_t kMaxHeadDim = 256;

struct PagedArgs {
    Pages pages;
    const float *q;
    float *out, *lse;
    AttnView qs, os;
    int32_t batch, heads, kv_heads, group, Sq, D;
    int32_t window, sinks, shared;
    float scale2;
};

// A wave a query: a key at a time, its entries dealt to the lanes.
template <class E>
__global__ void __launch_bounds__(64) paged_each(PagedArgs a) {
    const int lane = (int)threadIdx.x;
    const int64_t id = blockIdx.x;
    const int i = (int)(id % a.Sq), h = (int)(id / a.Sq % a.heads), b = (int)(id / a.Sq / a.heads), hk = h / a.group;
    const int place = a.pages.keys_of(b) - a.Sq + i;
    const float *qp = a.q + b * a.qs.b + h * a.qs.h + i * a.qs.s;
    float q[4], acc[4] = {0.f, 0.f, 0.f, 0.f}, most = -__builtin_inff(), sum = 0.f;
    for (int e = 0; e < 4; e++) q[e] = lane + 64 * e < a.D ? qp[lane + 64 * e] * a.scale2 : 0.f;
    const auto key = [&](int j) {
        const int at = a.pages.page_of(j < a.shared ? 0 : b, j), slot = a.pages.slot_of(j);
        const bool held = a.pages.holds(at);
        const int64_t page = held ? at : 0;
        const E *k = (const E *)a.pages.k + page * a.pages.ks.p + hk * a.pages.ks.h + slot * a.pages.ks.s;
        const E *v = (const E *)a.pages.v + page * a.pages.vs.p + hk * a.pages.vs.h + slot * a.pages.vs.s;
        float s = 0.f;
        for (int e = 0; e < 4; e++)
            if (lane + 64 * e < a.D) s += q[e] * (float)k[lane + 64 * e];
        for (int d = 1; d < 64; d *= 2) s += __shfl_xor(s, d);
        if (!held) s = __builtin_nanf("");
        const float now = __builtin_fmaxf(most, s), base = now == -__builtin_inff() ? 0.f : now;
        const float keep = __builtin_amdgcn_exp2f(most - base), p = __builtin_amdgcn_exp2f(s - base);
        sum = sum * keep + p;
        most = now;
        for (int e = 0; e < 4; e++)
            if (lane + 64 * e < a.D) acc[e] = acc[e] * keep + p * (float)v[lane + 64 * e];
    };
    const int first = max(place - a.window + 1, 0);
    for (int j = 0; j < min(a.sinks, first); j++) key(j);
    for (int j = first; j <= place; j++) key(j);
    float *op = a.out + b * a.os.b + h * a.os.h + i * a.os.s;
    for (int e = 0; e < 4; e++)
        if (lane + 64 * e < a.D) op[lane + 64 * e] = place < 0 ? 0.f : acc[e] / sum;
    if (a.lse && lane == 0) a.lse[((int64_t)b * a.heads + h) * a.Sq + i] = log_sum(most, sum);
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
    if (Sq > kMaxPagedTokens || B > INT32_MAX || H > INT32_MAX || (HK > 0 && (H / HK) * Sq > kMaxPagedTokens))
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
    a.window = (int32_t)std::min(window, most), a.sinks = (int32_t)std::min(sinks, most), a.shared = (int32_t)std::min(shared, most);
    a.scale2 = scale * kLog2e;
    if (rows >> 26) return set_error(TRS_E_INDEX_OVERFLOW, "attention over %lld rows", (long long)rows);
    if (cache->type == TRS_PAGES_BF16) hipLaunchKernelGGL(paged_each<__bf16>, dim3((unsigned)rows), dim3(64), 0, dev->stream, a);
    else hipLaunchKernelGGL(paged_each<float>, dim3((unsigned)rows), dim3(64), 0, dev->stream, a);
    TRS_LAUNCH_CHECK("paged attention launch");
    return TRS_OK;
}

}  // namespace

}  // namespace trs

extern "C" int trs_paged_attention_f32(const float *q, const trs_layout *lq, const trs_paged_cache *cache, int64_t shared,
                                       int64_t window, int64_t sinks, float scale, float *out, const trs_layout *lo,
                                       float *lse) {
    return trs::abi_guard([&]() -> int { return trs::run_paged(q, lq, cache, shared, window, sinks, scale, out, lo, lse); });
}
