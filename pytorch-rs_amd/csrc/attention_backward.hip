// attention_backward.hip -- the gradients of attention.h's attention: their host part,
// and what comes before and after the products.
//
// With P = exp(scale Q K^T - lse) (of a row: RowFacts) over the pairs that see each other and
// delta = rowsum(dO o):
//   dS = P (dO V^T - delta),  dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO.
// P and dO V^T are worked out twice, over rows for dQ and over keys for dK and dV (seven
// products where one walk would take five), so that every sum has one owner and a fixed
// order: no atomic adds, the same bits each time.
//
// Pairs that only the sinks make visible (first keys, far rows) go to blocks of their
// own: their keys are seen by every later row, the other keys by a window of rows.  What
// these blocks sum, in parts, is added by attn_reduce.
#include <hip/hip_runtime.h>

#include "attention.h"

namespace trs {

namespace {

// The least row tiles of a part: 333 tokens, 4 heads of 32 57.8 us with 8, 34.5 with 4, 33.2 with 2
// (2 x 2048 tokens, whose parts are longer, alike).
constexpr int kPartTiles = 2;

// Maximum and sum of the lane's row, over the keys that it sees: R rows a wave, lane l has row
// l % R and a tile's keys key(register, l / R) of the scores that tile(key's row) gives, in `unit`s.
// Straight from memory, few rows need it.
template <int R, class Key, class Tile>
__device__ __forceinline__ void statistics(const AttnArgs &a, const Sequence &seq, int b, int hk, int r0, int r1, int place, float unit,
                                           Key &&key, Tile &&tile, float &base, float &share) {
    constexpr int E = R * R / 64;
    const int lane = (int)threadIdx.x & 63;
    const KeyTiles<R == 32 ? 5 : 4> keys(a, seq, r0, r1);
    const float *kb = a.k + b * a.ks.b + hk * a.ks.h;
    float most = -__builtin_inff(), sum = 0.f;
#pragma unroll 1
    for (int t = 0; t < keys.tiles; t++) {
        const int j0 = keys.first_key(t);
        auto s = tile(kb + (int64_t)min(j0 + lane % R, keys.key_hi) * a.ks.s);
        float m = -__builtin_inff();
#pragma unroll
        for (int e = 0; e < E; e++) {
            s[e] = sees(a, place, j0 + key(e, lane / R)) ? s[e] : -__builtin_inff();
            m = __builtin_fmaxf(m, s[e]);
        }
#pragma unroll
        for (int d = R; d < 64; d *= 2) m = __builtin_fmaxf(m, __shfl_xor(m, d));
        const float now = __builtin_fmaxf(most, m), from = now == -__builtin_inff() ? 0.f : now;
        sum *= __builtin_amdgcn_exp2f((most - from) * unit);
#pragma unroll
        for (int e = 0; e < E; e++) sum += __builtin_amdgcn_exp2f((s[e] - from) * unit);
        most = now;
    }
#pragma unroll
    for (int d = R; d < 64; d *= 2) sum += __shfl_xor(sum, d);
    base = most * unit, share = 1.f / sum;
}

// The facts of 16 rows of a key head a wave (333 tokens, 4 heads of 32 3.7 us, with 32 rows 4.6; 4096
// tokens, 32 heads of 128 22.4 and 24.5).
template <bool WIDE>
__global__ void __launch_bounds__(64) attn_facts(AttnArgs a) {
    constexpr int R = 16, COLS = WIDE ? 16 : 32;  // of a product
    const int lane = (int)threadIdx.x, sub = lane & 15;
    const uint32_t tiles = (uint32_t)(a.rows + R - 1) / R, rest = blockIdx.x / (uint32_t)a.kv_heads;
    const int hk = (int)(blockIdx.x % (uint32_t)a.kv_heads), tile = (int)(rest % tiles), b = (int)(rest / tiles);
    const int r0 = tile * R, r1 = min(r0 + R, a.rows);
    // Query, head and [batch, head, token] of a row of the wave.
    const auto find = [&](int n, int &i, int &h) {
        const int row = min(r0 + n, r1 - 1);
        i = (int)a.by_group.divide((uint32_t)row), h = hk * a.group + row - i * a.group;
        return ((int64_t)b * a.heads + h) * a.Sq + i;
    };
    int i, h;
    const int64_t at = find(lane % COLS, i, h);
    const Sequence seq = sequence_of(a, b);
    const int place = seq.first + i;
    const float lse = a.lse[at];
    // delta: 16 lanes a row, the rows' loads together.
    float delta[R / 4] = {};
    const float *out[R / 4], *up[R / 4];
#pragma unroll
    for (int n = 0; n < R / 4; n++) {
        int i, h;
        find(4 * n + lane / 16, i, h);
        out[n] = a.out + b * a.os.b + h * a.os.h + i * a.os.s, up[n] = a.up + b * a.us.b + h * a.us.h + i * a.us.s;
    }
    const auto add = [&](auto &&chunk) {
        for (int d = sub * 4; d < a.D; d += 64)
#pragma unroll
            for (int n = 0; n < R / 4; n++) {
                const at_f4 x = chunk(out[n], d), y = chunk(up[n], d);
#pragma unroll
                for (int e = 0; e < 4; e++) delta[n] += x[e] * y[e];
            }
    };
    if (a.D % 4 == 0) add([](const float *p, int d) { return __builtin_bit_cast(at_f4, *(const f4u *)(p + d)); });
    else add([&](const float *p, int d) { return row_chunk(p, d, a.D); });
    float base = lse * kLog2e, base32 = base;
    float share = __builtin_amdgcn_exp2f(-(__builtin_fmaf(lse, kLog2e, -base) + lse * kLog2eLow)), share32 = share;
    const bool again = place >= 0 && !(__builtin_fabsf(lse) <= kMostLse);
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(again) != 0, 0)) {
        const float *q = a.q + b * a.qs.b + h * a.qs.h + i * a.qs.s;
        const auto row = [&](int c) { return row_chunk(q, c, a.D) * a.scale2; };
        const int mine = r0 + lane % COLS < r1 ? place : -1;
        float x, y;
        if constexpr (WIDE) {
            statistics<16>(
                a, seq, b, hk, r0, r1, mine, 1.f, [](int e, int quarter) { return 4 * quarter + e; },
                [&](const float *k) {
                    at_f4 c = (at_f4)(0.f);
#pragma unroll 1
                    for (int j = 0; j < a.D; j += 16) {
                        const at_f4 u = row_chunk(k, j + 4 * (lane >> 4), a.D), w = row(j + 4 * (lane >> 4));
#pragma unroll
                        for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(u[e], w[e], c, 0, 0, 0);
                    }
                    return c;
                },
                x, y);
        } else {
            const auto key = [](int e, int half) { return result_row(e, half); };
            Lowest lowest;
            statistics<32>(
                a, seq, b, hk, r0, r1, mine, kDown2, key,
                [&](const float *k) {
                    at_f16 c = (at_f16)(0.f);
#pragma unroll 1
                    for (int u = 0; 16 * u < a.D; u++) {
                        Unit<1> n, m;
#pragma unroll
                        for (int e = 0; e < 8; e += 4) {
                            const int d = 16 * u + 8 * (lane >> 5) + e;
                            const at_f4 x = row_chunk(k, d, a.D), y = row_chunk(q, d, a.D);
#pragma unroll
                            for (int i = 0; i < 4; i++) n.v[e + i] = x[i], m.v[e + i] = y[i];
                        }
                        mfma_pieces<true>(c, n.split(kUp), m.split(a.scale2 * kUp));
                    }
                    lowest.add(c);
                    return c;
                },
                x, y);
            // A score beyond the pieces' range may be in one block of keys: NaN sends all to the fp32 form.
            if (again) base = lowest.infinite() ? __builtin_nanf("") : x, share = y;
            statistics<32>(
                a, seq, b, hk, r0, r1, mine, 1.f, key,
                [&](const float *k) { return product_fp32(a.D, lane >> 5, [&](int c) { return row_chunk(k, c, a.D); }, row); }, x, y);
        }
        if (again) base32 = x, share32 = y;
    }
    if (lane < r1 - r0) {
        a.facts.pieces.base[at] = base, a.facts.pieces.share[at] = share * kUp;
        a.facts.fp32.base[at] = base32, a.facts.fp32.share[at] = share32;
    }
#pragma unroll
    for (int n = 0; n < R / 4; n++) {
#pragma unroll
        for (int d = 1; d < 16; d *= 2) delta[n] += __shfl_xor(delta[n], d);
        const int row = 4 * n + lane / 16;
        if (sub == 0 && row < r1 - r0) a.facts.delta[find(row, i, h)] = delta[n];
    }
}

// dk and dv of the first `count` keys: the parts over the rows, or what the one part
// wrote, and the sinks' `far` parts, in a fixed order.  Eight parts are read at a time: one
// memory latency for all of them.
__global__ void __launch_bounds__(256) attn_reduce(AttnArgs a, int count, int far) {
    const int64_t heads = (int64_t)a.batch * a.kv_heads, n = heads * count * a.D;
    const auto add = [](float &x, float &y, const float *px, const float *py, int64_t step, int parts) {
        for (int p = 0; p < parts; p += 8) {
            float u[8], w[8];
#pragma unroll
            for (int q = 0; q < 8; q++) {
                const int64_t at = min(p + q, parts - 1) * step;
                u[q] = px[at], w[q] = py[at];
            }
#pragma unroll
            for (int q = 0; q < 8; q++)
                if (p + q < parts) x += u[q], y += w[q];
        }
    };
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < n; e += (int64_t)gridDim.x * 256) {
        const int64_t row = e / a.D, head = row / count;
        const int d = (int)(e - row * a.D), key = (int)(row - head * count), hk = (int)(head % a.kv_heads);
        const int64_t b = head / a.kv_heads;
        float *dk = a.dk + b * a.dks.b + hk * a.dks.h + (int64_t)key * a.dks.s + d;
        float *dv = a.dv + b * a.dvs.b + hk * a.dvs.h + (int64_t)key * a.dvs.s + d;
        float x = 0.f, y = 0.f;
        if (a.row_splits > 1) {
            const int64_t at = (head * a.Sk + key) * a.D + d;
            add(x, y, a.part_k + at, a.part_v + at, heads * a.Sk * a.D, a.row_splits);
        } else {
            x = *dk, y = *dv;
        }
        if (far && key < a.sinks) {
            const int64_t at = (head * far * a.sinks + key) * a.D + d;
            add(x, y, a.sink_k + at, a.sink_v + at, (int64_t)a.sinks * a.D, far);
        }
        *dk = x, *dv = y;
    }
}

}  // namespace

int attention_backward(AttnArgs a, hipStream_t s, int cu_count) {
    const int64_t heads = (int64_t)a.batch * a.kv_heads;
    // In pieces: blocks of 128 rows or keys, tiles of 32.  Wide heads: waves of 16, tiles of 16,
    // four waves a block.
    const bool wide = a.D > kPiecesDim;
    const int block = wide ? 16 : kRowsBlock, tile = wide ? 16 : kTile;
    const int64_t room = (wide ? 8 : 2) * (int64_t)cu_count;  // blocks or waves that the device is to have
    a.row_tiles = (a.rows + block - 1) / block;
    a.key_tiles = (a.Sk + block - 1) / block;
    // The rows that see a key tile in parts where the tiles are few for the CUs.
    const int64_t near_tiles = std::max<int64_t>(1, std::min<int64_t>(a.rows, ((int64_t)a.window + block) * a.group) / tile);
    a.row_splits = 1;
    if (a.key_tiles)
        a.row_splits = (int32_t)std::max<int64_t>(1, std::min<int64_t>({room / (heads * a.key_tiles), near_tiles / kPartTiles, 16}));
    // Rows beyond a window see sinks alone: in parts of about as many row tiles as the others.
    a.sink_tiles = a.window < a.Sk ? (std::min(a.sinks, a.Sk) + block - 1) / block : 0;
    a.sink_splits = 1;
    if (a.sink_tiles)
        a.sink_splits = (int32_t)std::max<int64_t>(1, std::min<int64_t>(64, std::max<int64_t>(1, a.rows / tile) * a.row_splits / near_tiles));
    const int64_t row_blocks = heads * a.row_tiles;
    const int64_t most_blocks = row_blocks + heads * (a.sink_tiles * a.sink_splits + (int64_t)a.key_tiles * a.row_splits);
    const int64_t fact_units = heads * ((a.rows + 15) / 16);
    if (most_blocks >> 24 || fact_units >> 25)  // a launch has fewer than 2^32 lanes
        return set_error(TRS_E_INVALID_ARGUMENT, "attention gradient over too many blocks");
    const int64_t facts = ((int64_t)a.batch * a.heads * a.Sq + 63) / 64 * 64;
    const auto sink_floats = [&] { return a.sink_tiles ? heads * a.sink_splits * a.sinks * a.D : 0; };
    const auto part_floats = [&] { return a.row_splits > 1 ? heads * a.row_splits * a.Sk * a.D : 0; };
    void *ws = nullptr;
    const auto take = [&] { return trs_alloc((size_t)(5 * facts + 2 * sink_floats() + 2 * part_floats()) * sizeof(float), &ws); };
    int got = take();
    if (got == TRS_E_ALLOCATION_FAILED && (a.row_splits > 1 || a.sink_splits > 1)) {  // the parts are for speed alone
        a.row_splits = a.sink_splits = 1;
        got = take();
    }
    TRS_CHECK(got);
    const int far = a.sink_tiles ? a.sink_splits : 0;
    const int64_t key_blocks = heads * (a.sink_tiles * a.sink_splits + (int64_t)a.key_tiles * a.row_splits);
    float *const f = (float *)ws;
    a.facts = RowFacts{f, {f + facts, f + 2 * facts}, {f + 3 * facts, f + 4 * facts}};
    a.sink_k = f + 5 * facts, a.sink_v = a.sink_k + sink_floats();
    a.part_k = a.sink_v + sink_floats(), a.part_v = a.part_k + part_floats();
    const auto launch = [&]() -> int {
        // No rows: the keys' gradients are 0.  No keys: the rows' are.
        const dim3 fact_blocks((unsigned)fact_units);
        if (fact_units && wide) hipLaunchKernelGGL(attn_facts<true>, fact_blocks, dim3(64), 0, s, a);
        else if (fact_units) hipLaunchKernelGGL(attn_facts<false>, fact_blocks, dim3(64), 0, s, a);
        TRS_LAUNCH_CHECK("attention gradient launch");
        if (key_blocks + row_blocks) {
            if (wide) launch_attention_grad_wide(a, (uint32_t)key_blocks, (uint32_t)row_blocks, s);
            else launch_attention_grad(a, (uint32_t)key_blocks, (uint32_t)row_blocks, s);
            TRS_LAUNCH_CHECK("attention gradient launch");
        }
        const int count = a.row_splits > 1 ? a.Sk : a.sink_tiles ? std::min(a.sinks, a.Sk) : 0;
        if (count) {
            const int64_t n = heads * count * a.D;
            hipLaunchKernelGGL(attn_reduce, dim3((unsigned)std::min<int64_t>((n + 255) / 256, 1 << 20)), dim3(256), 0, s, a, count, far);
            TRS_LAUNCH_CHECK("attention gradient launch");
        }
        return TRS_OK;
    };
    const int rc = launch(), frc = trs_free(ws);
    return rc ? rc : frc;
}

}  // namespace trs
