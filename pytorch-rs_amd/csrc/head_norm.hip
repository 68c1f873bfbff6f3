// head_norm.hip -- the norm of every head's vector and the rotation by its
// position, in one pass, for queries and keys in one launch; and its gradient.
//
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r w,  y = R n
// R turns the pairs of the first `rot` entries, (i, i + rot/2) or, interleaved,
// (2i, 2i+1), by the angle whose cosine and sine stand in row `position` of the
// tables; the other entries pass.  With g = R^T dy
//   dw = sum over rows of g x r,  dx = r (w g - x r^2 mean(w g x)).
//
// Memory bounds it: 4 bytes read and 4 written an entry (8 and 4 in the
// gradient), with the tables' rows shared by a position's heads.
#include <hip/hip_runtime.h>

#include <cmath>

#include "op_checks.h"

namespace trs {

namespace {

constexpr int kMaxDim = 1024;
// Blocks per CU of the gradient: more give the sum of dw more to add (4 x 2047 tokens, 20 heads
// of 64: 28.9 us with 2, 30.5 with 4, 37.0 with 8).
constexpr int kGradBlocks = 2;

struct NormTensor {  // [batch, head, token, dim]
    const float *x, *w, *up;
    float *y, *dw;  // the output, or the gradient of x
    int64_t xs[4], us[4], ys[4];
    int64_t heads, rows;
    SmallDivisor inner, outer;  // by the dims that the rows are walked over, below 2^31 rows
    int32_t heads_inner;  // rows walked with the heads innermost, else the tokens
    int32_t first;        // first block
    int32_t blocks;
    float *parts;  // [blocks][dim]: each block's share of dw
};

struct NormArgs {
    NormTensor t[2];
    int32_t count;
    int64_t tokens, dim, rot, table_rows, table_stride, start;
    const float *cos, *sin;
    const int32_t *positions;  // [batch, token]; null: start + token
    float eps, inv_dim;
    int32_t interleaved;
};

struct Row {
    int64_t b, h, s, position;
};

__device__ __forceinline__ Row row_at(const NormArgs &a, const NormTensor &t, int64_t r) {
    int64_t i0, i1, b;
    if (t.rows >> 31) {
        const int64_t n0 = t.heads_inner ? t.heads : a.tokens, n1 = t.heads_inner ? a.tokens : t.heads;
        i0 = r % n0, i1 = r / n0 % n1, b = r / n0 / n1;
    } else {
        const uint32_t q = t.inner.divide((uint32_t)r), q2 = t.outer.divide(q);
        i0 = (uint32_t)r - q * t.inner.d, i1 = q - q2 * t.outer.d, b = q2;
    }
    Row o;
    o.b = b;
    o.h = t.heads_inner ? i0 : i1;
    o.s = t.heads_inner ? i1 : i0;
    o.position = a.positions ? (int64_t)a.positions[b * a.tokens + o.s] : a.start + o.s;
    return o;
}

__device__ __forceinline__ int64_t at_row(const int64_t (&st)[4], const Row &r) { return r.b * st[0] + r.h * st[1] + r.s * st[2]; }

// The reciprocal root, within a unit in the last place; the instruction takes subnormals for 0,
// so what is that small (rows of nothing above 2^-50, without eps) goes in 2^64 times as large.
__device__ __forceinline__ float inv_rms(const NormArgs &a, float sum) {
    const float mean = sum * a.inv_dim + a.eps;
    const bool small = mean < 0x1p-100f;
    return __builtin_amdgcn_rsqf(mean * (small ? 0x1p64f : 1.f)) * (small ? 0x1p32f : 1.f);
}

// The sum over groups of LPR consecutive lanes.
template <int LPR>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int d = 1; d < LPR; d *= 2) v += __shfl_xor(v, d);
    return v;
}

// Eight entries of a row: four of the first half of what is turned and the four that lie
// rot/2 on, so that both partners of every pair are in the lane; or eight that pass.
struct Eight {
    f4u a, b;
};

// Turns the lane's pairs by +angle (SIGN 1) or -angle (SIGN -1).
template <int SIGN>
__device__ __forceinline__ void turn(Eight &v, const NormArgs &a, int64_t position, int at) {
    const float *c = a.cos + position * a.table_stride, *s = a.sin + position * a.table_stride;
    if (a.interleaved) {
        const int64_t half = a.rot / 2;
#pragma unroll
        for (int p = 0; p < 2; p++) {
            f4u &x = p ? v.b : v.a;
            const int64_t i = ((int64_t)at + p * half) / 2;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float co = c[i + e], si = SIGN * s[i + e], u = x[2 * e], w = x[2 * e + 1];
                x[2 * e] = u * co - w * si;
                x[2 * e + 1] = w * co + u * si;
            }
        }
    } else {
        const f4u co = *(const f4u *)(c + at), si = *(const f4u *)(s + at);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float u = v.a[e], w = v.b[e], t = SIGN * si[e];
            v.a[e] = u * co[e] - w * t;
            v.b[e] = w * co[e] + u * t;
        }
    }
}

__device__ __forceinline__ Eight load8(const float *p, int64_t half) { return Eight{*(const f4u *)p, *(const f4u *)(p + half)}; }
// Read and written once: past the caches.
__device__ __forceinline__ Eight stream8(const float *p, int64_t half) {
    return Eight{__builtin_nontemporal_load((const f4u *)p), __builtin_nontemporal_load((const f4u *)(p + half))};
}
__device__ __forceinline__ void store8(float *p, int64_t half, const Eight &v) {
    __builtin_nontemporal_store(v.a, (f4u *)p);
    __builtin_nontemporal_store(v.b, (f4u *)(p + half));
}

__device__ __forceinline__ int which(const NormArgs &a) { return a.count > 1 && (int)blockIdx.x >= a.t[1].first ? 1 : 0; }

// Rows of whole eights (dim and rot multiples of 8, unit strides): LPR lanes a row,
// 256 / LPR rows a block, one block for each such group.  2 x 4096 tokens, 40 heads of 128:
// 57.5 us, 5.9 TB/s; 63 with loads and stores through the caches, 64 and 68 with two and four rows
// a lane on their way at once.  The gradients 91 us, 5.5 TB/s.
template <int LPR, bool GRAD>
__global__ void __launch_bounds__(256) norm_rows(NormArgs a) {
    const NormTensor &t = a.t[which(a)];
    const int sub = (int)threadIdx.x % LPR;
    const bool in = sub * 8 < a.dim, turns = sub * 8 < a.rot;
    const int at = turns ? sub * 4 : sub * 8;
    const int64_t half = turns ? a.rot / 2 : 4;  // from the lane's first four to its others
    Eight w = {(f4u)(1.f), (f4u)(1.f)}, dw = {(f4u)(0.f), (f4u)(0.f)};
    if (in && t.w) w = load8(t.w + at, half);
    constexpr int RPB = 256 / LPR;
    const int64_t block = (int)blockIdx.x - t.first;
    for (int64_t r0 = block * RPB; r0 < t.rows; r0 += (int64_t)t.blocks * RPB) {
        const int64_t r = r0 + (int)threadIdx.x / LPR;
        const bool on = in && r < t.rows;
        Row row = {};
        Eight x = {(f4u)(0.f), (f4u)(0.f)}, g = x;
        if (on) {
            row = row_at(a, t, r);
            x = stream8(t.x + at_row(t.xs, row) + at, half);
            if constexpr (GRAD) g = stream8(t.up + at_row(t.us, row) + at, half);
        }
        // A position that the tables do not hold gives NaN, and no read past them.
        const bool known = row.position >= 0 && row.position < a.table_rows;
        if constexpr (GRAD) {
            if (on && known && turns) turn<-1>(g, a, row.position, at);
        }
        float sum = 0.f, dot = 0.f;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            sum += x.a[e] * x.a[e] + x.b[e] * x.b[e];
            if constexpr (GRAD) dot += w.a[e] * g.a[e] * x.a[e] + w.b[e] * g.b[e] * x.b[e];
        }
        const float rms = inv_rms(a, group_sum<LPR>(sum));
        if constexpr (GRAD) dot = group_sum<LPR>(dot) * a.inv_dim * rms * rms;
        if (!on) continue;
        Eight y;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if constexpr (GRAD) {
                dw.a[e] += known ? g.a[e] * (x.a[e] * rms) : __builtin_nanf("");
                dw.b[e] += known ? g.b[e] * (x.b[e] * rms) : __builtin_nanf("");
                y.a[e] = rms * (w.a[e] * g.a[e] - x.a[e] * dot);
                y.b[e] = rms * (w.b[e] * g.b[e] - x.b[e] * dot);
            } else {
                y.a[e] = x.a[e] * rms * w.a[e];
                y.b[e] = x.b[e] * rms * w.b[e];
            }
        }
        if constexpr (!GRAD) {
            if (known && turns) turn<1>(y, a, row.position, at);
        }
        if (!known) y = {(f4u)(__builtin_nanf("")), (f4u)(__builtin_nanf(""))};
        store8(t.y + at_row(t.ys, row) + at, half, y);
    }
    if constexpr (GRAD) {
        if (!t.dw) return;
        // The block's rows' shares of dw, added in row order.
        __shared__ float part[RPB][LPR * 8];
        const int g = (int)threadIdx.x / LPR;
#pragma unroll
        for (int e = 0; e < 4; e++) part[g][sub * 8 + e] = dw.a[e], part[g][sub * 8 + 4 + e] = dw.b[e];
        __syncthreads();
        for (int d = (int)threadIdx.x; d < a.dim; d += 256) {
            const int second = (int)a.rot / 2;
            const int col = d >= a.rot ? d : d < second ? d / 4 * 8 + d % 4 : (d - second) / 4 * 8 + 4 + d % 4;
            float s = part[0][col];
            for (int i = 1; i < RPB; i++) s += part[i][col];
            t.parts[block * a.dim + d] = s;
        }
    }
}

// Any dim up to kMaxDim, any part of it rotated, any strides: a wave a row, the
// entries dealt to its lanes, partners read again from the cache (2 x 4096 tokens, 40
// heads of 80, 36 of them turned: 151 to 176 us by card; 40 of them, in eights, 46.  The
// gradients 340 and 76).
template <bool GRAD>
__global__ void __launch_bounds__(256) norm_any(NormArgs a) {
    const NormTensor &t = a.t[which(a)];
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const int dim = (int)a.dim, rot = (int)a.rot;
    constexpr int J = kMaxDim / 64;
    float dw[GRAD ? J : 1] = {};
    const int64_t block = (int)blockIdx.x - t.first;
    for (int64_t r = block * 4 + wave; r < t.rows; r += (int64_t)t.blocks * 4) {
        const Row row = row_at(a, t, r);
        const bool known = row.position >= 0 && row.position < a.table_rows;
        const float *c = a.cos + (known ? row.position * a.table_stride : 0);
        const float *s = a.sin + (known ? row.position * a.table_stride : 0);
        const float *x = t.x + at_row(t.xs, row), *up = GRAD ? t.up + at_row(t.us, row) : nullptr;
        float *y = t.y + at_row(t.ys, row);
        const auto weight = [&](int e) { return t.w ? t.w[e] : 1.f; };
        // The partner of entry e, its angle's number, and whether e is the pair's second.
        const auto pair = [&](int e, int &partner, int &angle, bool &second) {
            second = a.interleaved ? (e & 1) : e >= rot / 2;
            angle = a.interleaved ? e >> 1 : second ? e - rot / 2 : e;
            partner = a.interleaved ? e ^ 1 : second ? e - rot / 2 : e + rot / 2;
        };
        const auto back = [&](int e) {  // entry e of R^T up
            const float u = up[e * t.us[3]];
            if (e >= rot || !known) return u;
            int p, i;
            bool second;
            pair(e, p, i, second);
            const float v = up[p * t.us[3]];
            return second ? u * c[i] - v * s[i] : u * c[i] + v * s[i];
        };
        float sum = 0.f, dot = 0.f;
        for (int e = lane; e < dim; e += 64) {
            const float v = x[e * t.xs[3]];
            sum += v * v;
            if constexpr (GRAD) dot += weight(e) * back(e) * v;
        }
        const float rms = inv_rms(a, group_sum<64>(sum));
        if constexpr (GRAD) {
            dot = group_sum<64>(dot) * a.inv_dim * rms * rms;
#pragma unroll
            for (int j = 0; j < J; j++) {
                const int e = lane + 64 * j;
                if (e >= dim) break;
                const float v = x[e * t.xs[3]], g = back(e);
                dw[j] += known ? g * (v * rms) : __builtin_nanf("");
                y[e * t.ys[3]] = known ? rms * (weight(e) * g - v * dot) : __builtin_nanf("");
            }
        } else {
            for (int e = lane; e < dim; e += 64) {
                float n = x[e * t.xs[3]] * rms * weight(e);
                if (e < rot && known) {
                    int p, i;
                    bool second;
                    pair(e, p, i, second);
                    const float m = x[p * t.xs[3]] * rms * weight(p);
                    n = second ? n * c[i] + m * s[i] : n * c[i] - m * s[i];
                }
                y[e * t.ys[3]] = known ? n : __builtin_nanf("");
            }
        }
    }
    if constexpr (GRAD) {
        if (!t.dw) return;
        __shared__ float part[4][kMaxDim];
#pragma unroll
        for (int j = 0; j < J; j++)
            if (lane + 64 * j < dim) part[wave][lane + 64 * j] = dw[j];
        __syncthreads();
        for (int d = (int)threadIdx.x; d < dim; d += 256)
            t.parts[block * dim + d] = ((part[0][d] + part[1][d]) + part[2][d]) + part[3][d];
    }
}

// dw: the blocks' shares added in a fixed order, 16 runs of blocks an entry, eight shares
// read at a time (one memory latency for all of them).
__global__ void __launch_bounds__(1024) norm_weight_sum(NormArgs a) {
    const NormTensor &t = a.t[blockIdx.y];
    if (!t.dw) return;
    __shared__ float part[16][64];
    const int lane = (int)threadIdx.x & 63, run = (int)threadIdx.x >> 6;
    const int64_t d = (int64_t)blockIdx.x * 64 + lane;
    float s = 0.f;
    if (d < a.dim) {
        const int from = (int)((int64_t)t.blocks * run / 16), to = (int)((int64_t)t.blocks * (run + 1) / 16);
        for (int b = from; b < to; b += 8) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = t.parts[(int64_t)min(b + e, to - 1) * a.dim + d];
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (b + e < to) s += x[e];
        }
    }
    part[run][lane] = s;
    __syncthreads();
    if (run == 0 && d < a.dim) {
        for (int r = 1; r < 16; r++) s += part[r][lane];
        t.dw[d] = s;
    }
}

template <bool GRAD>
void launch_rows(int lpr, dim3 grid, hipStream_t s, const NormArgs &a) {
    switch (lpr) {
    case 1: hipLaunchKernelGGL((norm_rows<1, GRAD>), grid, dim3(256), 0, s, a); break;
    case 2: hipLaunchKernelGGL((norm_rows<2, GRAD>), grid, dim3(256), 0, s, a); break;
    case 4: hipLaunchKernelGGL((norm_rows<4, GRAD>), grid, dim3(256), 0, s, a); break;
    case 8: hipLaunchKernelGGL((norm_rows<8, GRAD>), grid, dim3(256), 0, s, a); break;
    case 16: hipLaunchKernelGGL((norm_rows<16, GRAD>), grid, dim3(256), 0, s, a); break;
    case 32: hipLaunchKernelGGL((norm_rows<32, GRAD>), grid, dim3(256), 0, s, a); break;
    default: hipLaunchKernelGGL((norm_rows<64, GRAD>), grid, dim3(256), 0, s, a); break;
    }
}

struct NormCall {
    int n;
    const float *const *x;
    const trs_layout *lx;
    const float *const *weight;
    float eps;
    const float *cos, *sin;
    const trs_layout *ltab;
    int interleaved;
    const int32_t *positions;
    int64_t start;
    const float *const *up;
    const trs_layout *lup;
    float *const *out;
    const trs_layout *lo;
    float *const *dweight;
};

template <bool GRAD>
int run_norm(const NormCall &c) {
    if (c.n < 1 || c.n > 2) return set_error(TRS_E_INVALID_ARGUMENT, "head norm takes 1 or 2 tensors, got %d", c.n);
    if (!c.x || !c.lx || !c.out || !c.lo || (GRAD && (!c.up || !c.lup)))
        return set_error(TRS_E_INVALID_ARGUMENT, "null head norm argument");
    if (!(c.eps >= 0.f) || std::isinf(c.eps)) return set_error(TRS_E_INVALID_ARGUMENT, "head norm eps has to be finite and not negative");
    TRS_CHECK(check_layout(c.ltab, "rotation table"));
    if (c.ltab->rank != 2) return set_error(TRS_E_INVALID_ARGUMENT, "rotation tables have rank 2, got %d", c.ltab->rank);
    NormArgs a{};
    a.count = c.n;
    a.eps = c.eps;
    a.interleaved = c.interleaved != 0;
    a.table_rows = c.ltab->shape[0];
    a.rot = c.ltab->shape[1] * 2;
    a.table_stride = c.ltab->stride[0];
    a.start = c.start;
    bool whole = true;
    int64_t batch = 0;
    for (int i = 0; i < c.n; i++) {
        const trs_layout *lx = &c.lx[i], *lo = &c.lo[i], *lu = GRAD ? &c.lup[i] : lx;
        TRS_CHECK(check_layout(lx, "head norm input"));
        TRS_CHECK(check_layout(lo, "head norm output"));
        TRS_CHECK(check_layout(lu, "head norm upstream gradient"));
        if (lx->rank != 4) return set_error(TRS_E_INVALID_ARGUMENT, "head norm inputs have rank 4 (batch, head, token, dim), got %d", lx->rank);
        if (lo->rank != 4 || lu->rank != 4) return set_error(TRS_E_SHAPE_MISMATCH, "head norm input and output ranks differ");
        for (int d = 0; d < 4; d++)
            if (lo->shape[d] != lx->shape[d] || lu->shape[d] != lx->shape[d])
                return set_error(TRS_E_SHAPE_MISMATCH, "head norm input and output shapes differ");
        if (i == 0) {
            batch = lx->shape[0], a.tokens = lx->shape[2], a.dim = lx->shape[3];
        } else if (lx->shape[0] != batch || lx->shape[2] != a.tokens || lx->shape[3] != a.dim) {
            return set_error(TRS_E_SHAPE_MISMATCH, "queries and keys differ in batch, tokens or head dim");
        }
        TRS_CHECK(check_written_once(lo, "head norm output"));
    }
    if (a.dim < 1 || a.dim > kMaxDim) return set_error(TRS_E_INVALID_ARGUMENT, "head dim %lld outside [1, %d]", (long long)a.dim, kMaxDim);
    if (a.rot > a.dim)
        return set_error(TRS_E_SHAPE_MISMATCH, "rotation tables of %lld pairs need a head dim of at least %lld, got %lld",
                         (long long)a.rot / 2, (long long)a.rot, (long long)a.dim);
    if (a.rot > 2 && c.ltab->stride[1] != 1) return set_error(TRS_E_INVALID_ARGUMENT, "rotation tables need a unit stride along their rows");
    if (!c.positions && batch > 0 && a.tokens > 0 && (c.start < 0 || c.start > a.table_rows - a.tokens))
        return set_error(TRS_E_INVALID_ARGUMENT, "positions %lld to %lld outside the rotation tables' %lld rows", (long long)c.start,
                         (long long)(c.start + a.tokens - 1), (long long)a.table_rows);
    // What is read and written.
    {
        Operand ops[13];
        int n = 0;
        for (int i = 0; i < 2; i++) {
            const int q = i < c.n ? i : 0;  // the first one's again: the same operand is no overlap
            const bool mine = i < c.n;
            ops[n++] = {"input", c.x[q], &c.lx[q], false};
            ops[n++] = {"upstream gradient", GRAD ? c.up[q] : c.x[q], GRAD ? &c.lup[q] : &c.lx[q], false};
            ops[n++] = {"weight", c.weight ? c.weight[q] : nullptr, nullptr, false, c.weight && c.weight[q] ? a.dim : 0};
            ops[n++] = {"output", mine ? c.out[q] : nullptr, nullptr, false, 0};
            if (mine) ops[n - 1].layout = &c.lo[q], ops[n - 1].written = true;
            float *dw = mine && GRAD && c.dweight ? c.dweight[q] : nullptr;
            ops[n++] = {"weight gradient", dw, nullptr, dw != nullptr, dw ? a.dim : 0};
        }
        ops[n++] = {"cosines", c.cos, c.ltab, false};
        ops[n++] = {"sines", c.sin, c.ltab, false};
        ops[n++] = {"positions", c.positions, nullptr, false, c.positions ? batch * a.tokens : 0};
        TRS_CHECK(check_memory(ops));
    }
    a.cos = c.cos ? c.cos + c.ltab->offset : nullptr;
    a.sin = c.sin ? c.sin + c.ltab->offset : nullptr;
    a.positions = c.positions;
    a.inv_dim = 1.0f / (float)a.dim;
    DeviceState *dev = device_state();
    if (!dev) return TRS_E_NO_DEVICE;
    whole = a.rot % 8 == 0 && a.dim % 8 == 0 && a.dim <= 512;
    for (int i = 0; i < c.n; i++) {
        NormTensor &t = a.t[i];
        const trs_layout *lx = &c.lx[i], *lo = &c.lo[i], *lu = GRAD ? &c.lup[i] : lx;
        t.heads = lx->shape[1];
        t.rows = batch * t.heads * a.tokens;
        t.x = c.x[i] ? c.x[i] + lx->offset : nullptr;
        t.y = c.out[i] ? c.out[i] + lo->offset : nullptr;
        t.up = GRAD && c.up[i] ? c.up[i] + lu->offset : nullptr;
        t.w = c.weight ? c.weight[i] : nullptr;
        t.dw = GRAD && c.dweight ? c.dweight[i] : nullptr;
        for (int d = 0; d < 4; d++) t.xs[d] = lx->stride[d], t.ys[d] = lo->stride[d], t.us[d] = lu->stride[d];
        t.heads_inner = lx->stride[1] <= lx->stride[2];
        if (t.rows > 0 && !(t.rows >> 31)) {
            t.inner = SmallDivisor((uint32_t)(t.heads_inner ? t.heads : a.tokens));
            t.outer = SmallDivisor((uint32_t)(t.heads_inner ? a.tokens : t.heads));
        }
        whole = whole && (t.rows == 0 || (t.xs[3] == 1 && t.ys[3] == 1 && t.us[3] == 1));
    }
    int lpr = 1;
    while (lpr * 8 < a.dim) lpr *= 2;
    const int64_t rows_per_block = whole ? 256 / lpr : 4;
    int32_t blocks = 0;
    size_t parts = 0;
    for (int i = 0; i < c.n; i++) {
        NormTensor &t = a.t[i];
        const int64_t want = (t.rows + rows_per_block - 1) / rows_per_block;
        const bool grad_w = GRAD && t.dw;
        t.first = blocks;
        t.blocks = (int32_t)std::min<int64_t>(want, GRAD ? (int64_t)dev->cu_count * kGradBlocks : 1 << 22);
        if (grad_w && t.blocks == 0) t.blocks = 1;  // no rows: dw is 0
        if (grad_w) parts += (size_t)t.blocks * (size_t)a.dim;
        blocks += t.blocks;
    }
    if (blocks == 0) return TRS_OK;
    void *ws = nullptr;
    if (parts) {
        TRS_CHECK(trs_alloc(parts * sizeof(float), &ws));
        float *p = (float *)ws;
        for (int i = 0; i < c.n; i++)
            if (a.t[i].dw) a.t[i].parts = p, p += (size_t)a.t[i].blocks * (size_t)a.dim;
    }
    const dim3 grid((unsigned)blocks);
    if (whole) launch_rows<GRAD>(lpr, grid, dev->stream, a);
    else hipLaunchKernelGGL(norm_any<GRAD>, grid, dim3(256), 0, dev->stream, a);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && parts) {
        hipLaunchKernelGGL(norm_weight_sum, dim3((unsigned)((a.dim + 63) / 64), (unsigned)c.n), dim3(1024), 0, dev->stream, a);
        e = hipGetLastError();
    }
    const int frc = ws ? trs_free(ws) : TRS_OK;
    if (e != hipSuccess) return hip_fail(e, "head norm launch");
    return frc;
}

}  // namespace

}  // namespace trs

extern "C" int trs_head_norm_rope_f32(int n, const float *const *x, const trs_layout *lx, const float *const *weight,
                                      float eps, const float *cos, const float *sin, const trs_layout *ltab,
                                      int interleaved, const int32_t *positions, int64_t start, float *const *out,
                                      const trs_layout *lo) {
    return trs::abi_guard([&]() -> int {
        return trs::run_norm<false>({n, x, lx, weight, eps, cos, sin, ltab, interleaved, positions, start, nullptr, nullptr, out, lo, nullptr});
    });
}

extern "C" int trs_head_norm_rope_backward_f32(int n, const float *const *x, const trs_layout *lx,
                                               const float *const *weight, float eps, const float *cos,
                                               const float *sin, const trs_layout *ltab, int interleaved,
                                               const int32_t *positions, int64_t start, const float *const *up,
                                               const trs_layout *lup, float *const *dx, const trs_layout *ldx,
                                               float *const *dweight) {
    return trs::abi_guard([&]() -> int {
        return trs::run_norm<true>({n, x, lx, weight, eps, cos, sin, ltab, interleaved, positions, start, up, lup, dx, ldx, dweight});
    });
}
