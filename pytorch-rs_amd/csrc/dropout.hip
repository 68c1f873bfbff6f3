// dropout.hip -- dropout whose mask comes from a counter and is never stored.
//
// Element i of x in row-major order keeps its value, scaled, where word i % 4
// of Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as
// easy as 1, 2, 3", SC'11) at counter offset + i/4 and key `seed` is at least
// round(p * 2^32):
//     y[i] = keep(i) ? x[i] * f32(1/(1-p)) : +0
// The gradient is the same function of the upstream gradient, so the backward
// pass works the words out again and no mask is kept.
#include <hip/hip_runtime.h>

#include <cmath>

#include "op_checks.h"

namespace trs {

namespace {

struct Words {
    uint32_t w[4];
};

__device__ __forceinline__ Words philox(uint64_t counter, uint64_t seed) {
    uint32_t x0 = (uint32_t)counter, x1 = (uint32_t)(counter >> 32), x2 = 0, x3 = 0;
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; r++) {
        const uint64_t a = (uint64_t)x0 * 0xD2511F53u, b = (uint64_t)x2 * 0xCD9E8D57u;
        x0 = (uint32_t)(b >> 32) ^ x1 ^ k0, x1 = (uint32_t)b;
        x2 = (uint32_t)(a >> 32) ^ x3 ^ k1, x3 = (uint32_t)a;
        k0 += 0x9E3779B9u, k1 += 0xBB67AE85u;
    }
    return Words{{x0, x1, x2, x3}};
}

struct DropoutArgs {
    const float *x;
    float *y;
    int64_t n;
    uint64_t seed, offset;
    uint32_t least;  // the least word that keeps
    bool any;        // false: nothing is kept (p rounds to 1)
    float scale;
    int32_t rank;
    // Dims after size-1 dims are dropped and those contiguous for both merged.
    int64_t size[TRS_MAX_RANK], xs[TRS_MAX_RANK], ys[TRS_MAX_RANK];
    int64_t ls[TRS_MAX_RANK];  // row-major strides: an index tuple's element number
};

__device__ __forceinline__ float kept(float x, uint32_t word, const DropoutArgs &a) {
    return a.any && word >= a.least ? x * a.scale : 0.f;
}

// Blocks of one wave, a group of four a lane, in one go over the tensor: the DRAM pages in
// use stay few.  Bound by memory: forward and gradient of 8192 x 4096 83.2 us (6.5 TB/s; a copy's rate is 6.7),
// 87.0 with blocks of 256 lanes, 94.5 with four groups a lane and through the caches.  The
// words take most of 101 vector instructions a group, which run under the loads.
constexpr int kGroupLanes = 64;

// Unit strides along the last dim, whose length is a multiple of four unless it
// is the only one: a lane's four elements share a generator block and are 16
// bytes of a row.
template <bool FLAT>
__global__ void __launch_bounds__(kGroupLanes) dropout_groups(DropoutArgs a) {
    const int64_t groups = (a.n + 3) / 4;
    for (int64_t g = (int64_t)blockIdx.x * kGroupLanes + threadIdx.x; g < groups; g += (int64_t)gridDim.x * kGroupLanes) {
        int64_t i = g * 4, xo = i, yo = i;
        if constexpr (!FLAT) {
            xo = yo = 0;
            for (int d = 0; d < a.rank; d++) {
                const int64_t at = (a.n >> 32) ? i / a.ls[d] : (int64_t)((uint32_t)i / (uint32_t)a.ls[d]);
                i -= at * a.ls[d];
                xo += at * a.xs[d], yo += at * a.ys[d];
            }
        }
        const bool whole = g * 4 + 4 <= a.n;
        f4u v;
        if (whole) v = __builtin_nontemporal_load((const f4u *)(a.x + xo));
        else
            for (int e = 0; e < 4; e++) v[e] = g * 4 + e < a.n ? a.x[xo + e] : 0.f;
        const Words w = philox(a.offset + (uint64_t)g, a.seed);
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = kept(v[e], w.w[e], a);
        if (whole) __builtin_nontemporal_store(v, (f4u *)(a.y + yo));
        else
            for (int e = 0; e < 4; e++)
                if (g * 4 + e < a.n) a.y[yo + e] = v[e];
    }
}

// Any strides: elements in the order of the output's memory, a generator block
// each (one word of it is used).  8192 x 4096 transposed in both 139 us, where rows take 41.
__global__ void __launch_bounds__(256) dropout_elements(DropoutArgs a) {
    const int64_t step = (int64_t)gridDim.x * 256;
    for (int64_t m = (int64_t)blockIdx.x * 256 + threadIdx.x; m < a.n; m += step) {
        int64_t rest = m, xo = 0, yo = 0, i = 0;
        for (int d = a.rank - 1; d >= 0; d--) {
            const int64_t n = a.size[d];
            const int64_t q = (a.n >> 32) ? rest / n : (int64_t)((uint32_t)rest / (uint32_t)n);
            const int64_t at = rest - q * n;
            rest = q;
            xo += at * a.xs[d], yo += at * a.ys[d], i += at * a.ls[d];
        }
        const Words w = philox(a.offset + (uint64_t)(i >> 2), a.seed);
        const int e = (int)(i & 3);
        const uint32_t word = e < 2 ? (e == 0 ? w.w[0] : w.w[1]) : (e == 2 ? w.w[2] : w.w[3]);
        a.y[yo] = kept(a.x[xo], word, a);
    }
}

int run_dropout(const float *x, const trs_layout *lx, double p, uint64_t seed, uint64_t offset, float *out,
                const trs_layout *lo) {
    TRS_CHECK(check_layout(lx, "input"));
    TRS_CHECK(check_layout(lo, "output"));
    if (!(p >= 0.0 && p <= 1.0))
        return set_error(TRS_E_INVALID_ARGUMENT, "dropout probability has to be between 0 and 1, but got %g", p);
    if (lx->rank != lo->rank) return set_error(TRS_E_SHAPE_MISMATCH, "dropout input and output ranks differ");
    for (int d = 0; d < lx->rank; d++)
        if (lx->shape[d] != lo->shape[d]) return set_error(TRS_E_SHAPE_MISMATCH, "dropout input and output shapes differ");
    DropoutArgs a{};
    a.n = layout_numel(lx);
    if (a.n == 0) return TRS_OK;
    TRS_CHECK(check_written_once(lo, "output"));
    if (!x || !out) return set_error(TRS_E_INVALID_ARGUMENT, "null dropout operand");
    a.x = x + lx->offset, a.y = out + lo->offset;
    if (ranges_overlap(byte_range(x, lx, 4), byte_range(out, lo, 4)) && !(a.x == a.y && same_view_shape(lx, lo)))
        return set_error(TRS_E_INVALID_ARGUMENT, "dropout output overlaps its input other than as the same view");
    DeviceState *dev = device_state();
    if (!dev) return TRS_E_NO_DEVICE;
    const double least = std::floor(p * 4294967296.0 + 0.5);
    a.any = least < 4294967296.0;
    if (a.any) a.least = (uint32_t)least, a.scale = (float)(1.0 / (1.0 - p));
    a.seed = seed, a.offset = offset;
    // Innermost first, then turned round.
    int r = 0;
    int64_t size[TRS_MAX_RANK], xs[TRS_MAX_RANK], ys[TRS_MAX_RANK], ls[TRS_MAX_RANK], inner = 1;
    for (int d = lx->rank - 1; d >= 0; d--) {
        const int64_t n = lx->shape[d];
        if (n == 1) continue;
        if (r > 0 && lx->stride[d] == xs[r - 1] * size[r - 1] && lo->stride[d] == ys[r - 1] * size[r - 1]) {
            size[r - 1] *= n;
        } else {
            size[r] = n, xs[r] = lx->stride[d], ys[r] = lo->stride[d], ls[r] = inner;
            r++;
        }
        inner *= n;
    }
    if (r == 0) size[0] = 1, xs[0] = ys[0] = ls[0] = 1, r = 1;
    const bool groups = xs[0] == 1 && ys[0] == 1 && (r == 1 || size[0] % 4 == 0);
    int order[TRS_MAX_RANK];
    for (int i = 0; i < r; i++) order[i] = i;
    if (!groups) std::stable_sort(order, order + r, [&](int i, int j) { return ys[i] < ys[j]; });
    a.rank = r;
    for (int i = 0; i < r; i++) {
        const int d = r - 1 - i;
        a.size[d] = size[order[i]], a.xs[d] = xs[order[i]], a.ys[d] = ys[order[i]], a.ls[d] = ls[order[i]];
    }
    const int64_t lanes = groups ? (a.n + 3) / 4 : a.n, block = groups ? kGroupLanes : 256;
    const dim3 grid((unsigned)std::min<int64_t>((lanes + block - 1) / block, 1 << 22));
    if (groups && r == 1) hipLaunchKernelGGL(dropout_groups<true>, grid, dim3(kGroupLanes), 0, dev->stream, a);
    else if (groups) hipLaunchKernelGGL(dropout_groups<false>, grid, dim3(kGroupLanes), 0, dev->stream, a);
    else hipLaunchKernelGGL(dropout_elements, grid, dim3(256), 0, dev->stream, a);
    TRS_LAUNCH_CHECK("dropout launch");
    return TRS_OK;
}

}  // namespace

}  // namespace trs

extern "C" int trs_dropout_f32(const float *x, const trs_layout *lx, double p, uint64_t seed, uint64_t offset,
                               float *out, const trs_layout *lo) {
    return trs::abi_guard([&]() -> int { return trs::run_dropout(x, lx, p, seed, offset, out, lo); });
}
