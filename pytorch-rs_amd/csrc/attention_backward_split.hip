// attention_backward_split.hip -- the gradients of attention_backward.hip on the
// bf16 matrix cores, in pieces (attention.h), for dims up to 128.
//
// A tile in LDS serves twice: along its columns for the scores and dO V^T, across its
// rows for the gradients.  It is split into one of two buffers while the block
// computes from the other, the loads from memory a tile further ahead: one barrier a
// tile.  Bound by the card's power and by issue: 4096 tokens, 32 heads of 128 over 8, window
// 2048 1.9 to 2.1 ms by card, up to 1.2 PFLOP/s of bf16 products, the matrix cores busy for 53% of
// the cycles and the other vector instructions' issue 28%; 2 x 2048 tokens, 16 heads of 64 200 us, 47%
// and 34%.  The block has a CU to itself (512 registers a lane) above dims of 64, and a wave
// a SIMD nothing to run beside but its own instructions: so splitting and exponentials stand
// among the matrix instructions (steps()).
//
// Queries, keys, values and upstream rows are taken times 2^40, and P as 2^40 P, so
// that no piece of a value or weight is lost.  A block whose sums are not finite does
// its work again on the fp32 instruction, pair by pair where a tile holds infinities or
// NaN.
#include <hip/hip_runtime.h>

#include "attention.h"

namespace trs {

namespace {

// 2^40 2^x.  The exponential gives 0 for subnormal results, and a key may have no
// larger weight: below 2^-126 it is taken of x + 64.  (Adding 40 to x would cost the
// low bits of x.)
__device__ __forceinline__ float up_exp2(float x) {
    const bool low = x < -126.f;
    return __builtin_amdgcn_exp2f(x + (low ? 64.f : 0.f)) * (low ? 0x1p-24f : kUp);
}

// ---- dQ -----------------------------------------------------------------------

// The block's rows on the fp32 instruction, whatever the values.  dS is scaled, not its sums, which
// would leave the range ahead of the gradients.
template <int NT, int NW>
__device__ __forceinline__ void grad_rows_fp32(const AttnArgs &a, const RowBlock<NW> &r, float delta, float *lds,
                                               at_f16 (&acc)[NT]) {
    using T = Tile<NT, 64 * NW>;
    const float *kb = a.k + r.b * a.ks.b + r.hk * a.ks.h, *vb = a.v + r.b * a.vs.b + r.hk * a.vs.h;
    const float *q = r.place >= 0 ? a.q + r.at(a, a.qs) : nullptr, *u = r.place >= 0 ? a.up + r.at(a, a.us) : nullptr;
    const float base = r.place >= 0 ? a.facts.fp32.base[r.index(a)] : 0.f, share = r.place >= 0 ? a.facts.fp32.share[r.index(a)] : 0.f;
#pragma unroll
    for (int t = 0; t < NT; t++) acc[t] = (at_f16)(0.f);
#pragma unroll 1
    for (int t = 0; t < r.tiles; t++) {
        const int j0 = r.first_key(t);
        T::stage(lds, a.D, [&](int k) { return r.read(j0 + k) ? kb + (int64_t)(j0 + k) * a.ks.s : nullptr; });
        T::stage(lds + T::kFloats, a.D, [&](int k) { return r.read(j0 + k) ? vb + (int64_t)(j0 + k) * a.vs.s : nullptr; });
        __syncthreads();
        if (r.any(a, j0)) {
            at_f16 s = T::times_row(lds, q, a.D, a.scale2, r.lane);
            const at_f16 d = T::times_row(lds + T::kFloats, u, a.D, 1.f, r.lane);
#pragma unroll
            for (int e = 0; e < 16; e++) {
                s[e] = __builtin_exp2f(s[e] - base) * share * (d[e] - delta) * a.scale;
                if (!sees(a, r.place, j0 + result_row(e, r.half))) s[e] = 0.f;
            }
            T::add_product_seen(acc, lds, s, r.lane, [&](int k) { return sees(a, r.place, j0 + k); });
        }
        __syncthreads();
    }
}

// A block of 128 rows over their key tiles.
template <int NT, int WIDTH>
__device__ __forceinline__ void rows_block(const AttnArgs &a, uint32_t id, char *lds, Notices<4> &notices) {
    constexpr int NW = 4;
    using T = Tile<NT, 64 * NW>;
    constexpr int UNITS = 4 * NT, OWN = NT;  // of keys and values; of a wave
    constexpr int kBuffer = 3 * UNITS * 1024;
    const uint32_t rest = id / (uint32_t)a.kv_heads;
    const RowBlock<NW> r(a, (int)(id % (uint32_t)a.kv_heads), a.row_tiles - 1 - (int)(rest % (uint32_t)a.row_tiles), (int)(rest / (uint32_t)a.row_tiles));
    const float *kb = a.k + r.b * a.ks.b + r.hk * a.ks.h, *vb = a.v + r.b * a.vs.b + r.hk * a.vs.h;
    Unit<WIDTH> in[OWN];
    const auto load = [&](int t) {  // past the last tile: that one
        const int j = min(r.first_key(min(t, r.tiles - 1)) + (r.lane & 31), r.key_hi);
        const float *kp = kb + (int64_t)j * a.ks.s, *vp = vb + (int64_t)j * a.vs.s;
#pragma unroll
        for (int q = 0; q < OWN; q++) {
            const int u = r.wave + q * NW;
            in[q].load(u < UNITS / 2 ? kp : vp, u < UNITS / 2 ? u : u - UNITS / 2, a.D, r.lane);
        }
    };
    const bool live = r.place >= 0;
    const int64_t at = r.index(a);
    const float base = live ? a.facts.pieces.base[at] : 0.f, share = live ? a.facts.pieces.share[at] : 0.f, delta = live ? a.facts.delta[at] : 0.f;
    at_f16 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) acc[t] = (at_f16)(0.f);
    if (r.tiles > 0) {
        Lowest lowest;
        load(0);
        Pieces qp[2 * NT], up[2 * NT];
#pragma unroll
        for (int s = 0; s < 2 * NT; s++) {
            Unit<WIDTH> x;
            x.load(a.q + r.at(a, a.qs), s, a.D, r.lane, s < 2 * NT - 2);
            qp[s] = x.split(live ? a.scale2 * kUp : 0.f);
            x.load(a.up + r.at(a, a.us), s, a.D, r.lane, s < 2 * NT - 2);
            up[s] = x.split(share);
        }
#pragma unroll
        for (int n = 0; n < OWN; n++) in[n].template store<UNITS>(lds, r.wave + n * NW, r.lane);
        load(1);
#pragma unroll 1
        for (int t = 0; t < r.tiles; t++) {
            const int j0 = r.first_key(t);
            char *const buf = lds + (t & 1) * kBuffer, *const other = lds + (t & 1 ? 0 : kBuffer);
            __syncthreads();
            // share (dO V^T - delta), times 2^80: the sum starts from delta's part.  (The scores' does
            // not start from -base: it is the larger part, and every product would be rounded to it.)
            at_f16 s = (at_f16)(0.f), d = (at_f16)(-delta * (share * kUp));
            Splitting x;
            {
                const auto read = [&](int n) { return along<UNITS>(buf, (n & 1) * 2 * NT + n / 2, r.lane); };
                Pieces f = read(0);
                steps<4 * NT>(
                    f, read,
                    [&](int n, const Pieces &now) {
                        if (n & 1) mfma_pieces(d, now, up[n / 2]);
                        else mfma_pieces<true>(s, now, qp[n / 2]);  // the scores of keys_block, bit for bit
                    },
                    [&](int n) {
                        dealt(4 * OWN, n, 4 * NT, [&](int i) { in[i / 4].template store_pair<UNITS>(x, i % 4, other, r.wave + i / 4 * NW, r.lane); });
                    },
                    [](Pieces &) {});
            }
            load(t + 2);
            lowest.add(s);
            if (!r.all(a, j0)) {
#pragma unroll
                for (int e = 0; e < 16; e++) s[e] = sees(a, r.place, j0 + result_row(e, r.half)) ? s[e] : -__builtin_inff();
            }
            const auto weigh = [&](int e) {  // 2^40 dS; the weight's root is not subnormal where the weight is
                const float root = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], kDown2 / 2, -base / 2));
                return root * (root * (d[e] * kDown));
            };
            const auto read = [&](int n) { return across<UNITS>(buf, 2 * (n % NT), n / NT, r.lane); };
            Pieces f = read(0);
            Splitting w;
#pragma unroll
            for (int i = 0; i < 4; i++) w.pair(i, weigh(2 * i), weigh(2 * i + 1));
            const Pieces p0 = w.done();
            steps<NT>(
                f, read, [&](int n, const Pieces &now) { mfma_pieces(acc[n], now, p0); },
                [&](int n) { dealt(4, n, NT, [&](int i) { w.pair(i, weigh(8 + 2 * i), weigh(9 + 2 * i)); }); },
                [&](Pieces &y) { y = read(NT); });
            const Pieces p1 = w.done();
            steps<NT>(
                f, [&](int n) { return read(NT + n); }, [&](int n, const Pieces &now) { mfma_pieces(acc[n], now, p1); }, [](int) {},
                [](Pieces &) {});
        }
        __syncthreads();
        notices.word[1][r.wave] = not_finite(acc, 0.f) || lowest.infinite();
        __syncthreads();
        if (__builtin_expect(notices.any(1), 0)) {
            grad_rows_fp32<NT, NW>(a, r, delta, (float *)lds, acc);
            if (r.row < a.rows) T::write(acc, a.dq + r.at(a, a.dqs), 1.f, a.D, r.half);
            return;
        }
    }
    if (r.row < a.rows) write_row<WIDTH>(acc, a.dq + r.at(a, a.dqs), kDown2, a.scale, a.D, r.half);
}

// ---- dK and dV ------------------------------------------------------------------

// What a block of 128 keys works on: its keys, 32 a wave, and the rows whose window
// holds them; or, of the first keys, the rows beyond it, which the sinks alone see.
struct KeyBlock {
    bool far;
    int lane, half, wave;
    int hk, b, head, key, keys;  // the lane's key; past the last key
    int j0, j1;                  // the wave's keys
    int tile, part;
    int first;          // place of query 0
    int rlo, rhi;       // rows
    int t0, t1;         // row tiles of the part, from rlo on
    __device__ __forceinline__ KeyBlock(const AttnArgs &a, uint32_t id) {
        lane = (int)threadIdx.x & 63, half = lane >> 5;
        wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
        const uint32_t far_units = (uint32_t)(a.sink_tiles * a.sink_splits), units = far_units + (uint32_t)(a.key_tiles * a.row_splits);
        head = (int)(id / units);
        id -= (uint32_t)head * units;
        far = id < far_units;
        const int parts = far ? a.sink_splits : a.row_splits;
        if (!far) id -= far_units;
        tile = (int)(id / (uint32_t)parts), part = (int)(id % (uint32_t)parts);
        hk = head % a.kv_heads, b = head / a.kv_heads;
        const Sequence seq = sequence_of(a, b);
        first = seq.first, keys = far ? min(a.sinks, seq.keys) : seq.keys;
        const int block_j0 = tile * kRowsBlock, block_j1 = min(block_j0 + kRowsBlock, keys);
        j0 = block_j0 + wave * 32, j1 = min(j0 + 32, keys);
        key = j0 + (lane & 31);
        const int place_lo = max(far ? block_j0 + a.window : block_j0, max(first, 0));
        const int place_hi = far ? seq.keys - 1 : min(seq.keys - 1, block_j1 - 1 + a.window - 1);
        rlo = rhi = 0;
        int tiles = 0;
        if (block_j0 < block_j1 && place_lo <= place_hi) {
            rlo = (place_lo - first) * a.group, rhi = (place_hi - first + 1) * a.group;
            tiles = (rhi - rlo + kTile - 1) / kTile;
        }
        t0 = (int)((int64_t)tiles * part / parts), t1 = (int)((int64_t)tiles * (part + 1) / parts);
    }
    // Whether every key of the wave makes a pair with every row of tile t.
    __device__ __forceinline__ bool all(const AttnArgs &a, int t) const {
        const int r0 = rlo + t * kTile, r1 = min(r0 + kTile, rhi);
        const int lo = first + (int)a.by_group.divide((uint32_t)r0), hi = first + (int)a.by_group.divide((uint32_t)(r1 - 1));
        return r1 - r0 == kTile && j1 - j0 == 32 && (far ? lo - (j1 - 1) >= a.window : j1 - 1 <= lo && hi - j0 < a.window);
    }
    __device__ __forceinline__ bool pair(const AttnArgs &a, int place) const {
        return (key < keys) & (key <= place) & ((place - key < a.window) != far);
    }
};

// A tile's rows, as the waves of a block share them; two tiles in turn.
struct TileFacts {
    float base[2][kTile];
    float delta[2][kTile];  // -2^80 share delta, what the sum of share dO V^T starts from
    int place[2][kTile];    // -1: past the last row
    float share[kTile];     // for the fp32 form, whose delta is delta
};

template <int NT>
__device__ __forceinline__ void grad_keys_fp32(const AttnArgs &a, const KeyBlock &k, float *lds, TileFacts &facts,
                                               at_f16 (&dk)[NT], at_f16 (&dv)[NT]) {
    using T = Tile<NT, 256>;
    const bool live = k.key < k.keys;
    const float *kp = live ? a.k + k.b * a.ks.b + k.hk * a.ks.h + (int64_t)k.key * a.ks.s : nullptr;
    const float *vp = live ? a.v + k.b * a.vs.b + k.hk * a.vs.h + (int64_t)k.key * a.vs.s : nullptr;
#pragma unroll
    for (int t = 0; t < NT; t++) dk[t] = dv[t] = (at_f16)(0.f);
#pragma unroll 1
    for (int t = k.t0; t < k.t1; t++) {
        const int r0 = k.rlo + t * kTile;
        const auto row_at = [&](const float *p, const AttnView &v, int r) -> const float * {
            const int row = r0 + r;
            if (row >= k.rhi) return nullptr;
            const int i = (int)a.by_group.divide((uint32_t)row), g = row - i * a.group;
            return p + k.b * v.b + (int64_t)(k.hk * a.group + g) * v.h + (int64_t)i * v.s;
        };
        T::stage(lds, a.D, [&](int r) { return row_at(a.q, a.qs, r); });
        T::stage(lds + T::kFloats, a.D, [&](int r) { return row_at(a.up, a.us, r); });
        if (threadIdx.x < kTile) {
            const int row = r0 + (int)threadIdx.x;
            float base = 0.f, delta = 0.f, share = 0.f;
            int place = -1;
            if (row < k.rhi) {
                const int i = (int)a.by_group.divide((uint32_t)row), g = row - i * a.group;
                const int64_t at = ((int64_t)k.b * a.heads + k.hk * a.group + g) * a.Sq + i;
                base = a.facts.fp32.base[at], share = a.facts.fp32.share[at], delta = a.facts.delta[at], place = k.first + i;
            }
            facts.base[0][threadIdx.x] = base, facts.delta[0][threadIdx.x] = delta, facts.place[0][threadIdx.x] = place, facts.share[threadIdx.x] = share;
        }
        __syncthreads();
        {
            at_f16 p = T::times_row(lds, kp, a.D, 1.f, k.lane, a.scale2);
            at_f16 d = T::times_row(lds + T::kFloats, vp, a.D, 1.f, k.lane);
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int r = result_row(e, k.half);
                p[e] = __builtin_exp2f(p[e] - facts.base[0][r]) * facts.share[r];
                d[e] = p[e] * (d[e] - facts.delta[0][r]) * a.scale;
                if (!k.pair(a, facts.place[0][r])) p[e] = d[e] = 0.f;
            }
            const auto seen = [&](int r) { return k.pair(a, facts.place[0][r]); };
            T::add_product_seen(dv, lds + T::kFloats, p, k.lane, seen);
            T::add_product_seen(dk, lds, d, k.lane, seen);
        }
        __syncthreads();
    }
}

// A block of 128 keys over the row tiles that make pairs with them.
template <int NT, int WIDTH>
__device__ __forceinline__ void keys_block(const AttnArgs &a, uint32_t id, char *lds, TileFacts &facts, Notices<4> &notices) {
    using T = Tile<NT, 256>;
    constexpr int UNITS = 4 * NT, kBuffer = 3 * UNITS * 1024;  // of queries and upstream rows
    const KeyBlock k(a, id);
    const float *qb = a.q + k.b * a.qs.b + (int64_t)k.hk * a.group * a.qs.h, *ub = a.up + k.b * a.us.b + (int64_t)k.hk * a.group * a.us.h;

    // A lane's row of a tile, and what the waves share of it.  Past the part's last tile
    // that one is loaded, past the last row that one.
    Unit<WIDTH> in[NT];
    float base = 0.f, delta = 0.f, share = 0.f;
    int place = -1;
    const auto load = [&](int t) {
        const int at = k.rlo + min(t, k.t1 - 1) * kTile + (k.lane & 31), row = min(at, k.rhi - 1);
        const int i = (int)a.by_group.divide((uint32_t)row), g = row - i * a.group;
        const float *q = qb + (g * a.qs.h + i * a.qs.s), *u = ub + (g * a.us.h + i * a.us.s);
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const int unit = k.wave + 4 * n;
            in[n].load(unit < 2 * NT ? q : u, unit < 2 * NT ? unit : unit - 2 * NT, a.D, k.lane);
        }
        const int64_t fact = ((int64_t)k.b * a.heads + k.hk * a.group + g) * a.Sq + i;
        base = a.facts.pieces.base[fact], share = a.facts.pieces.share[fact], delta = a.facts.delta[fact];
        place = at < k.rhi ? k.first + i : -1;
    };
    // Queries are scaled, as rows_block has them, and upstream rows taken times their share.
    const float up_q = kUp * a.scale2;
    const auto up_to = [&](int n) { return 4 * n + 4 <= 2 * NT || (4 * n < 2 * NT && k.wave + 4 * n < 2 * NT) ? up_q : share; };
    const auto store_facts = [&](int n) {
        if (threadIdx.x < kTile) facts.base[n][threadIdx.x] = base, facts.delta[n][threadIdx.x] = delta * (share * -kUp), facts.place[n][threadIdx.x] = place;
    };
    at_f16 dk[NT], dv[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) dk[t] = dv[t] = (at_f16)(0.f);
    bool again = false;
    if (k.t0 < k.t1) {
        Lowest lowest;
        load(k.t0);
        const bool live = k.key < k.keys;
        const int key = live ? k.key : 0;
        Pieces kp[2 * NT], vp[2 * NT];
#pragma unroll
        for (int s = 0; s < 2 * NT; s++) {
            Unit<WIDTH> x;
            x.load(a.k + k.b * a.ks.b + k.hk * a.ks.h + (int64_t)key * a.ks.s, s, a.D, k.lane, s < 2 * NT - 2);
            kp[s] = x.split(live ? kUp : 0.f);
            x.load(a.v + k.b * a.vs.b + k.hk * a.vs.h + (int64_t)key * a.vs.s, s, a.D, k.lane, s < 2 * NT - 2);
            vp[s] = x.split(live ? kUp : 0.f);
        }
#pragma unroll
        for (int n = 0; n < NT; n++) in[n].template store<UNITS>(lds, k.wave + 4 * n, k.lane, up_to(n));
        store_facts(0);
        load(k.t0 + 1);
#pragma unroll 1
        for (int t = k.t0; t < k.t1; t++) {
            const int n2 = (t - k.t0) & 1;
            char *const buf = lds + n2 * kBuffer, *const other = lds + (n2 ? 0 : kBuffer);
            __syncthreads();
            at_f16 p, d;
#pragma unroll
            for (int e = 0; e < 16; e++) p[e] = 0.f, d[e] = facts.delta[n2][result_row(e, k.half)];
            Splitting x, w;
            {
                const auto read = [&](int n) { return along<UNITS>(buf, (n & 1) * 2 * NT + n / 2, k.lane); };
                Pieces f = read(0);
                steps<4 * NT>(
                    f, read, [&](int n, const Pieces &now) { mfma_pieces(n & 1 ? d : p, now, n & 1 ? vp[n / 2] : kp[n / 2]); },
                    [&](int n) { in[n / 4].template store_pair<UNITS>(x, n % 4, other, k.wave + n / 4 * 4, k.lane, up_to(n / 4)); }, [](Pieces &) {});
            }
            at_f16 base16;
#pragma unroll
            for (int e = 0; e < 16; e++) base16[e] = facts.base[n2][result_row(e, k.half)];
            store_facts(n2 ^ 1);
            lowest.add(p);
            if (!k.all(a, t)) {
#pragma unroll
                for (int e = 0; e < 16; e++) p[e] = k.pair(a, facts.place[n2][result_row(e, k.half)]) ? p[e] : -__builtin_inff();
            }
            // 2^40 P and 2^40 dS come pair by pair, each eight of them ahead of the products that take them.
            const auto pair_p = [&](int e) { return p[e] = up_exp2(__builtin_fmaf(p[e], kDown2, -base16[e])); };
            const auto pair_d = [&](int e) { return p[e] * (d[e] * kDown2); };
            // dV's first 16 rows, its others, dK's first, its others.
            const auto read = [&](int n) { return across<UNITS>(buf, (n < 2 * NT ? 2 * NT : 0) + 2 * (n % NT), n / NT % 2, k.lane); };
            Pieces f = read(0);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float w0 = pair_p(2 * i), w1 = pair_p(2 * i + 1);
                w.pair(i, w0, w1);
            }
            Pieces weights = w.done();
#pragma unroll
            for (int g = 0; g < 4; g++) {
                steps<NT>(
                    f, [&](int n) { return read(g * NT + n); }, [&](int n, const Pieces &now) { mfma_pieces(g < 2 ? dv[n] : dk[n], now, weights); },
                    [&](int n) {
                        dealt(4, n, NT, [&](int i) {
                            if (g == 3) return;
                            const int e = (g == 1 ? 0 : 8) + 2 * i;
                            const float w0 = g == 0 ? pair_p(e) : pair_d(e), w1 = g == 0 ? pair_p(e + 1) : pair_d(e + 1);
                            w.pair(i, w0, w1);
                        });
                    },
                    [&](Pieces &y) {
                        if (g < 3) y = read((g + 1) * NT);
                    });
                if (g < 3) weights = w.done();
                // Late, for few registers at a time: the first is wanted in the next tile's first step.
                if (g == 2) load(t + 2);
            }
        }
        __syncthreads();
        notices.word[0][k.wave] = not_finite(dk, 0.f) || not_finite(dv, 0.f) || lowest.infinite();
        __syncthreads();
        again = notices.any(0);
        if (__builtin_expect(again, 0)) {
            __syncthreads();
            grad_keys_fp32<NT>(a, k, (float *)lds, facts, dk, dv);
        }
    }
    if (k.key >= (k.far ? a.sinks : a.Sk)) return;
    float *pk, *pv;
    if (k.far) {
        const int64_t at = ((int64_t)k.head * a.sink_splits + k.part) * a.sinks + k.key;
        pk = a.sink_k + at * a.D, pv = a.sink_v + at * a.D;
    } else if (a.row_splits > 1) {
        const int64_t at = ((int64_t)k.part * a.batch * a.kv_heads + k.head) * a.Sk + k.key;
        pk = a.part_k + at * a.D, pv = a.part_v + at * a.D;
    } else {
        pk = a.dk + k.b * a.dks.b + k.hk * a.dks.h + (int64_t)k.key * a.dks.s;
        pv = a.dv + k.b * a.dvs.b + k.hk * a.dvs.h + (int64_t)k.key * a.dvs.s;
    }
    if (again) {
        T::write(dk, pk, 1.f, a.D, k.half);
        T::write(dv, pv, 1.f, a.D, k.half);
    } else {
        write_row<WIDTH>(dk, pk, kDown2, kLn2, a.D, k.half);  // scale / scale2
        write_row<WIDTH>(dv, pv, kDown2, 1.f, a.D, k.half);
    }
}

// Both kinds of block in one launch, so that neither waits for the other's last: those
// of the keys first, whose tiles take longer.
template <int NT, int WIDTH>
__global__ void __launch_bounds__(256, NT <= 2 ? 2 : 1) attn_grad(AttnArgs a, uint32_t key_blocks) {
    using T = Tile<NT, 256>;
    constexpr int kBytes = 2 * 3 * 4 * NT * 1024;
    static_assert(kBytes >= 8 * T::kFloats, "the fp32 tiles fit the pieces' LDS");
    __shared__ __attribute__((aligned(1024))) char lds[kBytes];
    __shared__ TileFacts facts;
    __shared__ Notices<4> notices;
    if (blockIdx.x < key_blocks) keys_block<NT, WIDTH>(a, blockIdx.x, lds, facts, notices);
    else rows_block<NT, WIDTH>(a, blockIdx.x - key_blocks, lds, notices);
}

template <int NT>
void launch(const AttnArgs &a, uint32_t key_blocks, uint32_t row_blocks, hipStream_t s) {
    const dim3 grid(key_blocks + row_blocks);
    if (a.D == 32 * NT) hipLaunchKernelGGL((attn_grad<NT, 4>), grid, dim3(256), 0, s, a, key_blocks);
    else if (a.D % 4 == 0) hipLaunchKernelGGL((attn_grad<NT, 2>), grid, dim3(256), 0, s, a, key_blocks);
    else hipLaunchKernelGGL((attn_grad<NT, 1>), grid, dim3(256), 0, s, a, key_blocks);
}

}  // namespace

void launch_attention_grad(const AttnArgs &a, uint32_t key_blocks, uint32_t row_blocks, hipStream_t s) {
    if (a.D <= 32) launch<1>(a, key_blocks, row_blocks, s);
    else if (a.D <= 64) launch<2>(a, key_blocks, row_blocks, s);
    else if (a.D <= 96) launch<3>(a, key_blocks, row_blocks, s);
    else launch<4>(a, key_blocks, row_blocks, s);
}

}  // namespace trs
