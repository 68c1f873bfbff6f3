// attention.hip -- the entry points of attention.h's attention: checks,
// workspaces and launches.
#include <hip/hip_runtime.h>

#include <cmath>

#include "attention.h"

namespace trs {

namespace {

constexpr int64_t kMaxHeadDim = 256, kMaxTokens = (int64_t)1 << 30;

// The operands of a call, in the order of the entry points' arguments.
struct AttnCall {
    const float *q, *k, *v;
    const trs_layout *lq, *lk, *lv;
    const int32_t *lengths;
    int64_t window, sinks;
    float scale;
    float *out;
    const trs_layout *lo;
    float *lse;
    const float *up = nullptr;
    const trs_layout *lup = nullptr;
    float *dq = nullptr, *dk = nullptr, *dv = nullptr;
    const trs_layout *ldq = nullptr, *ldk = nullptr, *ldv = nullptr;
};

int check_shape(const trs_layout *l, const char *what, const int64_t (&want)[4]) {
    TRS_CHECK(check_layout(l, what));
    if (l->rank != 4) return set_error(TRS_E_INVALID_ARGUMENT, "%s has rank %d, not 4 (batch, head, token, dim)", what, l->rank);
    for (int d = 0; d < 4; d++)
        if (want[d] >= 0 && l->shape[d] != want[d])
            return set_error(TRS_E_SHAPE_MISMATCH, "%s has size %lld in dim %d, expected %lld", what, (long long)l->shape[d], d, (long long)want[d]);
    return TRS_OK;
}

int check_output(const trs_layout *l, const char *what) {
    TRS_CHECK(check_written_once(l, what));
    if (l->shape[3] > 1 && l->stride[3] != 1) return set_error(TRS_E_INVALID_ARGUMENT, "%s needs a unit stride along its last dim", what);
    return TRS_OK;
}

AttnView view_of(const trs_layout *l) { return {l->stride[0], l->stride[1], l->stride[2]}; }

int run(const AttnCall &c) {
    const bool grad = c.up != nullptr || c.lup != nullptr;
    TRS_CHECK(check_shape(c.lq, "query", {-1, -1, -1, -1}));
    const int64_t B = c.lq->shape[0], H = c.lq->shape[1], Sq = c.lq->shape[2], D = c.lq->shape[3];
    TRS_CHECK(check_shape(c.lk, "key", {B, -1, -1, D}));
    const int64_t HK = c.lk->shape[1], Sk = c.lk->shape[2];
    TRS_CHECK(check_shape(c.lv, "value", {B, HK, Sk, D}));
    TRS_CHECK(check_shape(c.lo, "output", {B, H, Sq, D}));
    if (grad) {
        TRS_CHECK(check_shape(c.lup, "upstream gradient", {B, H, Sq, D}));
        TRS_CHECK(check_shape(c.ldq, "query gradient", {B, H, Sq, D}));
        TRS_CHECK(check_shape(c.ldk, "key gradient", {B, HK, Sk, D}));
        TRS_CHECK(check_shape(c.ldv, "value gradient", {B, HK, Sk, D}));
    }
    if (D < 1 || D > kMaxHeadDim) return set_error(TRS_E_INVALID_ARGUMENT, "head dim %lld outside [1, %lld]", (long long)D, (long long)kMaxHeadDim);
    if (HK < 1 ? H != 0 : H % HK != 0)
        return set_error(TRS_E_SHAPE_MISMATCH, "%lld query heads cannot share %lld key heads", (long long)H, (long long)HK);
    if (c.window < 1) return set_error(TRS_E_INVALID_ARGUMENT, "attention window has to be at least 1, got %lld", (long long)c.window);
    if (c.sinks < 0) return set_error(TRS_E_INVALID_ARGUMENT, "attention sinks have to be at least 0, got %lld", (long long)c.sinks);
    if (!std::isfinite(c.scale)) return set_error(TRS_E_INVALID_ARGUMENT, "attention scale has to be finite");
    if (Sq > kMaxTokens || Sk > kMaxTokens || (HK > 0 && (H / HK) * Sq > kMaxTokens) || B > INT32_MAX || H > INT32_MAX)
        return set_error(TRS_E_INDEX_OVERFLOW, "attention over more than 2^30 tokens, or rows that share a key head");
    TRS_CHECK(check_output(c.lo, "output"));
    if (grad) {
        TRS_CHECK(check_output(c.ldq, "query gradient"));
        TRS_CHECK(check_output(c.ldk, "key gradient"));
        TRS_CHECK(check_output(c.ldv, "value gradient"));
    }
    const int64_t rows = B * H * Sq;
    if (grad && rows > 0 && !c.lse) return set_error(TRS_E_INVALID_ARGUMENT, "lse is null");
    {
        const trs_layout *const none = nullptr;
        const Operand ops[] = {
            {"query", c.q, c.lq, false},
            {"key", c.k, c.lk, false},
            {"value", c.v, c.lv, false},
            {"lengths", c.lengths, none, false, c.lengths ? B : 0},
            {"output", c.out, c.lo, !grad},
            {"lse", c.lse, none, !grad, c.lse ? rows : 0},
            {"upstream gradient", grad ? c.up : c.q, grad ? c.lup : c.lq, false},
            {"query gradient", grad ? c.dq : nullptr, grad ? c.ldq : none, grad},
            {"key gradient", grad ? c.dk : nullptr, grad ? c.ldk : none, grad},
            {"value gradient", grad ? c.dv : nullptr, grad ? c.ldv : none, grad},
        };
        TRS_CHECK(check_memory(ops));
    }
    if (B == 0 || (grad ? H * Sq == 0 && HK * Sk == 0 : H * Sq == 0)) return TRS_OK;
    DeviceState *dev = device_state();
    if (!dev) return TRS_E_NO_DEVICE;
    AttnArgs a{};
    Dense q, k, v, o, u;
    TRS_CHECK(q.take(c.q, c.lq));
    TRS_CHECK(k.take(c.k, c.lk));
    TRS_CHECK(v.take(c.v, c.lv));
    a.q = q.at, a.k = k.at, a.v = v.at, a.qs = q.view, a.ks = k.view, a.vs = v.view;
    a.lengths = c.lengths;
    a.batch = (int32_t)B, a.heads = (int32_t)H, a.kv_heads = (int32_t)HK;
    a.group = HK ? (int32_t)(H / HK) : 0;
    a.Sq = (int32_t)Sq, a.Sk = (int32_t)Sk, a.D = (int32_t)D;
    a.rows = a.group * a.Sq;
    a.window = (int32_t)std::min<int64_t>(c.window, std::max<int64_t>(Sk, 1));
    a.sinks = (int32_t)std::min<int64_t>(c.sinks, Sk);
    a.scale = c.scale, a.scale2 = c.scale * kLog2e;
    a.by_group = SmallDivisor((uint32_t)std::max(a.group, 1));
    a.out = c.out ? c.out + c.lo->offset : nullptr, a.os = view_of(c.lo);
    a.lse = c.lse;
    if (!grad) return attention_forward(a, dev->stream, dev->cu_count);
    TRS_CHECK(o.take(c.out, c.lo));
    TRS_CHECK(u.take(c.up, c.lup));
    a.up = u.at, a.us = u.view;
    a.dq = c.dq ? c.dq + c.ldq->offset : nullptr, a.dqs = view_of(c.ldq);
    a.dk = c.dk ? c.dk + c.ldk->offset : nullptr, a.dks = view_of(c.ldk);
    a.dv = c.dv ? c.dv + c.ldv->offset : nullptr, a.dvs = view_of(c.ldv);
    return attention_backward(a, dev->stream, dev->cu_count);
}

}  // namespace

}  // namespace trs

extern "C" int trs_window_attention_f32(const float *q, const trs_layout *lq, const float *k, const trs_layout *lk,
                                        const float *v, const trs_layout *lv, const int32_t *lengths, int64_t window,
                                        int64_t sinks, float scale, float *out, const trs_layout *lo, float *lse) {
    return trs::abi_guard([&]() -> int {
        return trs::run(trs::AttnCall{q, k, v, lq, lk, lv, lengths, window, sinks, scale, out, lo, lse});
    });
}

extern "C" int trs_window_attention_backward_f32(const float *q, const trs_layout *lq, const float *k,
                                                 const trs_layout *lk, const float *v, const trs_layout *lv,
                                                 const int32_t *lengths, int64_t window, int64_t sinks, float scale,
                                                 const float *out, const trs_layout *lo, const float *lse,
                                                 const float *up, const trs_layout *lup, float *dq,
                                                 const trs_layout *ldq, float *dk, const trs_layout *ldk, float *dv,
                                                 const trs_layout *ldv) {
    return trs::abi_guard([&]() -> int {
        if (!lup) return trs::set_error(TRS_E_INVALID_ARGUMENT, "upstream gradient layout is null");
        return trs::run(trs::AttnCall{q, k, v, lq, lk, lv, lengths, window, sinks, scale, const_cast<float *>(out), lo,
                                      const_cast<float *>(lse), up, lup, dq, dk, dv, ldq, ldk, ldv});
    });
}
