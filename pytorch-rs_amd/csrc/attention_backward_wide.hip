// attention_backward_wide.hip -- the gradients of attention_backward.hip for heads of
// more than 128 dims.
//
// A tile's pieces and the operands held for it would not fit a CU's LDS and a lane's 512
// registers there, nor would fp32 tiles staged in LDS without spilling (a training step of 2048
// tokens, 16 heads of 256, window 512: 4066 us so, 1340 now).  So every wave works alone, on 16 keys or 16 rows, with its operands
// straight from memory (attention_wide.h): the next operand is asked for while the one
// before is multiplied, and the four waves of a block take neighbours, whose rows
// they find in the L1.  Bound by the fp32 matrix instruction's rate and the L2's.
#include <hip/hip_runtime.h>

#include "attention_wide.h"

namespace trs {

namespace {

// dQ of 16 rows of a key head.
template <int DP, int MODE>
__device__ __forceinline__ void rows_unit(const AttnArgs &a, int head, int tile) {
    using T = Wide<DP, MODE>;
    const int lane = (int)threadIdx.x & 63, col = lane & 15, quarter = lane >> 4;
    const int hk = head % a.kv_heads, b = head / a.kv_heads;
    const Sequence seq = sequence_of(a, b);
    const int r0 = tile * 16, r1 = min(r0 + 16, a.rows), row = min(r0 + col, a.rows - 1);
    const int i = (int)a.by_group.divide((uint32_t)row), g = row - i * a.group;
    const int64_t h = (int64_t)hk * a.group + g, at = ((int64_t)b * a.heads + h) * a.Sq + i;
    const bool live = r0 + col < a.rows && seq.first + i >= 0;
    const int place = live ? seq.first + i : -1;
    const KeyTiles<4> keys(a, seq, r0, r1);
    const int tiles = keys.tiles;
    at_f4 acc[T::TO];
#pragma unroll
    for (int t = 0; t < T::TO; t++) acc[t] = (at_f4)(0.f);
    if (tiles > 0) {
        const float *kb = a.k + b * a.ks.b + hk * a.ks.h, *vb = a.v + b * a.vs.b + hk * a.vs.h;
        // Past the last key, and past the last tile: that one.
        const auto key = [&](int t, int n) { return (int64_t)min(keys.first_key(min(t, tiles - 1)) + n, keys.key_hi); };
        typename T::Along q, u, k, v;
        typename T::Across k2;
        T::load(k, kb + key(0, col) * a.ks.s, a.D, quarter);
        T::load(q, a.q + b * a.qs.b + h * a.qs.h + (int64_t)i * a.qs.s, a.D, quarter);
        T::load(u, a.up + b * a.us.b + h * a.us.h + (int64_t)i * a.us.s, a.D, quarter);
        const float base = live ? a.facts.fp32.base[at] : 0.f, share = live ? a.facts.fp32.share[at] : 0.f;
        const float delta = live ? a.facts.delta[at] * share : 0.f;
#pragma unroll
        for (int j = 0; j < T::KJ; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) q[j][e] = live ? q[j][e] * a.scale2 : 0.f, u[j][e] = live ? u[j][e] * share : 0.f;
#pragma unroll 1
        for (int t = 0; t < tiles; t++) {
            const int j0 = keys.first_key(t);
            const auto row2 = [&](int n) { return kb + key(t, n) * a.ks.s; };
            at_f4 s = (at_f4)(0.f), d = (at_f4)(0.f);
            T::load(v, vb + key(t, col) * a.vs.s, a.D, quarter);
            T::product(s, k, q);
            T::load(k2, [&](int n) { return row2(4 * quarter + n); }, a.D, col);
            T::product(d, v, u);
            T::load(k, kb + key(t + 1, col) * a.ks.s, a.D, quarter);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                s[e] = __builtin_exp2f(s[e] - base) * (d[e] - delta) * a.scale;  // its sums might leave the range
                s[e] = sees(a, place, j0 + 4 * quarter + e) ? s[e] : 0.f;
            }
            if (__builtin_expect(!T::bad(k2), 1)) T::add(acc, k2, s);
            else T::add_seen(acc, s, a.D, col, quarter, row2, [&](int n) { return sees(a, place, j0 + n); });
        }
    }
    if (r0 + col < a.rows) T::write(acc, a.dq + b * a.dqs.b + h * a.dqs.h + (int64_t)i * a.dqs.s, 1.f, a.D, quarter);
}

// dK and dV of 16 keys, over the rows whose window holds them, or (far) over the rows
// beyond it, which the sinks alone see.
template <int DP, int MODE>
__device__ __forceinline__ void keys_unit(const AttnArgs &a, int head, int tile, int part, bool far) {
    using T = Wide<DP, MODE>;
    const int lane = (int)threadIdx.x & 63, col = lane & 15, quarter = lane >> 4;
    const int hk = head % a.kv_heads, b = head / a.kv_heads;
    const Sequence seq = sequence_of(a, b);
    const int keys = far ? min(a.sinks, seq.keys) : seq.keys, parts = far ? a.sink_splits : a.row_splits;
    const int j0 = tile * 16, j1 = min(j0 + 16, keys), key = j0 + col;
    const int place_lo = max(far ? j0 + a.window : j0, max(seq.first, 0));
    const int place_hi = far ? seq.keys - 1 : min(seq.keys - 1, j1 - 1 + a.window - 1);
    int rlo = 0, rhi = 0, tiles = 0;
    if (j0 < j1 && place_lo <= place_hi) {
        rlo = (place_lo - seq.first) * a.group, rhi = (place_hi - seq.first + 1) * a.group;
        tiles = (rhi - rlo + 15) / 16;
    }
    const int t0 = (int)((int64_t)tiles * part / parts), t1 = (int)((int64_t)tiles * (part + 1) / parts);
    at_f4 dk[T::TO], dv[T::TO];
#pragma unroll
    for (int t = 0; t < T::TO; t++) dk[t] = dv[t] = (at_f4)(0.f);
    if (t0 < t1) {
        const float *qb = a.q + b * a.qs.b + (int64_t)hk * a.group * a.qs.h, *ub = a.up + b * a.us.b + (int64_t)hk * a.group * a.us.h;
        const int64_t facts = ((int64_t)b * a.heads + hk * a.group) * a.Sq;
        // Past the last row, and past the last tile: that one.
        const auto row_of = [&](int t, int n, int &i, int &g) {
            const int row = min(rlo + min(t, t1 - 1) * 16 + n, rhi - 1);
            i = (int)a.by_group.divide((uint32_t)row), g = row - i * a.group;
        };
        const auto row_at = [&](const float *p, const AttnView &v, int t, int n) {
            int i, g;
            row_of(t, n, i, g);
            return p + (g * v.h + i * v.s);
        };
        typename T::Along k, v, q;
        typename T::Across x;
        T::load(q, row_at(qb, a.qs, t0, col), a.D, quarter);
        const bool live = key < keys;
        const int64_t kat = live ? key : 0;
        T::load(k, a.k + b * a.ks.b + hk * a.ks.h + kat * a.ks.s, a.D, quarter);
        T::load(v, a.v + b * a.vs.b + hk * a.vs.h + kat * a.vs.s, a.D, quarter);
#pragma unroll
        for (int j = 0; j < T::KJ; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) k[j][e] = live ? k[j][e] : 0.f, v[j][e] = live ? v[j][e] : 0.f;
#pragma unroll 1
        for (int t = t0; t < t1; t++) {
            float base[4], share[4], delta[4];
            int place[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                int i, g;
                row_of(t, 4 * quarter + e, i, g);
                const int64_t at = facts + (int64_t)g * a.Sq + i;
                base[e] = a.facts.fp32.base[at], share[e] = a.facts.fp32.share[at], delta[e] = a.facts.delta[at] * share[e];
                place[e] = rlo + t * 16 + 4 * quarter + e < rhi ? seq.first + i : -1;
            }
            const auto pair = [&](int place) { return (key < keys) & (key <= place) & ((place - key < a.window) != far); };
            const auto seen = [&](int n) {
                int i, g;
                row_of(t, n, i, g);
                return rlo + t * 16 + n < rhi && pair(seq.first + i);
            };
            const auto q2 = [&](int n) { return row_at(qb, a.qs, t, n); };
            const auto u2 = [&](int n) { return row_at(ub, a.us, t, n); };
            typename T::Along u;
            at_f4 p = (at_f4)(0.f), d = (at_f4)(0.f);
            T::load(u, row_at(ub, a.us, t, col), a.D, quarter);
            T::product(p, q, k, a.scale2);  // as rows_unit takes it: queries are scaled
            T::load(x, [&](int n) { return u2(4 * quarter + n); }, a.D, col);
            T::product(d, u, v);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                // Subnormals too: a key may have no larger weight.
                const float w = __builtin_exp2f(p[e] - base[e]);
                p[e] = pair(place[e]) ? w * share[e] : 0.f;
                d[e] = pair(place[e]) ? w * (d[e] * share[e] - delta[e]) * a.scale : 0.f;
            }
            typename T::Across y;
            T::load(y, [&](int n) { return q2(4 * quarter + n); }, a.D, col);
            if (__builtin_expect(!T::bad(x), 1)) T::add(dv, x, p);
            else T::add_seen(dv, p, a.D, col, quarter, u2, seen);
            T::load(q, row_at(qb, a.qs, t + 1, col), a.D, quarter);
            if (__builtin_expect(!T::bad(y), 1)) T::add(dk, y, d);
            else T::add_seen(dk, d, a.D, col, quarter, q2, seen);
        }
    }
    if (key >= (far ? a.sinks : a.Sk)) return;
    float *pk, *pv;
    if (far) {
        const int64_t at = ((int64_t)head * a.sink_splits + part) * a.sinks + key;
        pk = a.sink_k + at * a.D, pv = a.sink_v + at * a.D;
    } else if (a.row_splits > 1) {
        const int64_t at = ((int64_t)part * a.batch * a.kv_heads + head) * a.Sk + key;
        pk = a.part_k + at * a.D, pv = a.part_v + at * a.D;
    } else {
        pk = a.dk + b * a.dks.b + hk * a.dks.h + (int64_t)key * a.dks.s;
        pv = a.dv + b * a.dvs.b + hk * a.dvs.h + (int64_t)key * a.dvs.s;
    }
    T::write(dk, pk, 1.f, a.D, quarter);
    T::write(dv, pv, 1.f, a.D, quarter);
}

// Units of a wave each: the sinks' keys, all keys, then the rows.
template <int DP, int MODE>
__global__ void __launch_bounds__(256, 1) attn_grad_wide(AttnArgs a, uint32_t key_units, uint32_t row_units) {
    const uint32_t unit = blockIdx.x * 4 + (uint32_t)__builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    if (unit < key_units) {
        const uint32_t far_units = (uint32_t)(a.sink_tiles * a.sink_splits), units = far_units + (uint32_t)(a.key_tiles * a.row_splits);
        const uint32_t head = unit / units, id = unit - head * units;
        const bool far = id < far_units;
        const uint32_t n = far ? id : id - far_units, tiles = (uint32_t)(far ? a.sink_tiles : a.key_tiles);
        keys_unit<DP, MODE>(a, (int)head, (int)(n % tiles), (int)(n / tiles), far);
    } else if (unit < key_units + row_units) {
        const uint32_t n = unit - key_units;
        rows_unit<DP, MODE>(a, (int)(n / (uint32_t)a.row_tiles), (int)(n % (uint32_t)a.row_tiles));
    }
}

template <int DP>
void launch(const AttnArgs &a, uint32_t key_units, uint32_t row_units, hipStream_t s) {
    const dim3 grid((key_units + row_units + 3) / 4);
    if (a.D == DP) hipLaunchKernelGGL((attn_grad_wide<DP, 0>), grid, dim3(256), 0, s, a, key_units, row_units);
    else if (a.D % 4 == 0) hipLaunchKernelGGL((attn_grad_wide<DP, 1>), grid, dim3(256), 0, s, a, key_units, row_units);
    else hipLaunchKernelGGL((attn_grad_wide<DP, 2>), grid, dim3(256), 0, s, a, key_units, row_units);
}

}  // namespace

void launch_attention_grad_wide(const AttnArgs &a, uint32_t key_units, uint32_t row_units, hipStream_t s) {
    if (a.D <= 192) launch<192>(a, key_units, row_units, s);
    else launch<256>(a, key_units, row_units, s);
}

}  // namespace trs
