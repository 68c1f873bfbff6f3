// attention_backward.hip -- the gradients of attention.h's attention.
//
// With P = exp(scale Q K^T - lse) over the pairs that see each other and
// delta = rowsum(dO o):
//   dS = P (dO V^T - delta),  dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO.
// P and dO V^T are worked out twice, in a kernel over rows for dQ and in one over
// keys for dK and dV (seven products where one kernel would take five), so that
// every sum has one owner and a fixed order: no atomic adds, the same bits each
// time.
//
// Pairs that only the sinks make visible (first keys, far rows) go to blocks of
// their own: their 32 keys are seen by every later row, the other keys by a
// window of rows.  Such a block's waves take different row tiles for the same
// keys, and what each sums is added by attn_reduce.
#include <hip/hip_runtime.h>

#include "attention.h"

namespace trs {

namespace {

// The least row tiles of a part: 333 tokens, 4 heads of 32 57.8 us with 8, 34.5 with 4, 33.2 with 2
// (2 x 2048 tokens, whose parts are longer, alike).
constexpr int kPartTiles = 2;

// delta of every row: 16 lanes a row.
__global__ void __launch_bounds__(256) attn_delta(AttnArgs a, float *delta) {
    const int64_t rows = (int64_t)a.batch * a.heads * a.Sq;
    const int sub = (int)threadIdx.x & 15;
    const int64_t r = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    float s = 0.f;
    if (r < rows) {
        const int64_t bh = r / a.Sq, i = r - bh * a.Sq, b = bh / a.heads, h = bh - b * a.heads;
        const float *o = a.out + b * a.os.b + h * a.os.h + i * a.os.s, *u = a.up + b * a.us.b + h * a.us.h + i * a.us.s;
        for (int d = sub * 4; d < a.D; d += 64) {
            const at_f4 x = row_chunk(o, d, a.D), y = row_chunk(u, d, a.D);
#pragma unroll
            for (int e = 0; e < 4; e++) s += x[e] * y[e];
        }
    }
#pragma unroll
    for (int d = 1; d < 16; d *= 2) s += __shfl_xor(s, d);
    if (r < rows && sub == 0) delta[r] = s;
}

// dQ: 128 rows of one key head, 32 a wave, over the key tiles, as in attn_rows.
// NA result tiles a block: those of one half of the columns where all would not
// fit the registers.
template <int NT, int NA>
__global__ void __launch_bounds__(256, NT <= 2 ? 2 : 1) attn_grad_rows_fp32(AttnArgs a) {
    using T = Tile<NT>;
    __shared__ __attribute__((aligned(16))) float lds[2][2][T::kFloats];
    __shared__ Notices<4> notices;
    const int lane = (int)threadIdx.x & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    uint32_t id = blockIdx.x;
    const int c0 = (int)(id % (NT / NA)) * 32 * NA;
    id /= NT / NA;
    const int tile = (int)(id % (uint32_t)a.row_tiles);
    id /= (uint32_t)a.row_tiles;
    const int hk = (int)(id % (uint32_t)a.kv_heads), b = (int)(id / (uint32_t)a.kv_heads);

    const Sequence seq = sequence_of(a, b);
    const int r0 = tile * kRowsBlock, r1 = min(r0 + kRowsBlock, a.rows);
    const int row = r0 + wave * 32 + (lane & 31);
    const int i = (int)a.by_group.divide((uint32_t)min(row, a.rows - 1)), g = min(row, a.rows - 1) - i * a.group;
    // A row that sees nothing reads nothing: its gradient is 0.
    const bool live = row < a.rows && seq.first + i >= 0;
    const int place = live ? seq.first + i : -1;
    const int block_lo = seq.first + (int)a.by_group.divide((uint32_t)r0);
    const int block_hi = seq.first + (int)a.by_group.divide((uint32_t)(r1 - 1));
    const int w0 = r0 + wave * 32, w1 = min(w0 + 32, a.rows);
    const int wave_lo = seq.first + (int)a.by_group.divide((uint32_t)min(w0, a.rows - 1));
    const int wave_hi = w0 < w1 ? seq.first + (int)a.by_group.divide((uint32_t)(w1 - 1)) : -1;
    const int key_hi = block_hi, key_lo = max(0, block_lo - a.window + 1);
    const int sinks = min(a.sinks, key_hi + 1);
    const int first = key_lo / kTile;
    const int nsink = key_hi < 0 ? 0 : min((sinks + kTile - 1) / kTile, first);
    const int tiles = key_hi < 0 ? 0 : nsink + key_hi / kTile - first + 1;
    const auto first_key = [&](int t) { return (t < nsink ? t : first + t - nsink) * kTile; };

    const float *kb = a.k + b * a.ks.b + hk * a.ks.h, *vb = a.v + b * a.vs.b + hk * a.vs.h;
    typename T::Regs kr, vr;
    const auto load = [&](int t) {
        const int j0 = first_key(t);
        const auto seen = [&](int r) { return j0 + r <= key_hi && (j0 + r >= key_lo || j0 + r < sinks); };
        T::load(kr, a.D, [&](int r) { return seen(r) ? kb + (int64_t)(j0 + r) * a.ks.s : nullptr; });
        T::load(vr, a.D, [&](int r) { return seen(r) ? vb + (int64_t)(j0 + r) * a.vs.s : nullptr; });
    };
    const auto store = [&](int buf) {
        const bool bad = T::store(kr, lds[buf][0]);
        T::store(vr, lds[buf][1]);
        notices.word[buf][wave] = __builtin_amdgcn_ballot_w64(bad) != 0;
    };
    if (tiles > 0) load(0);
    const int64_t h = (int64_t)hk * a.group + g, at = ((int64_t)b * a.heads + h) * a.Sq + i;
    at_f4 qf[NT * 4], uf[NT * 4];
    T::hold(qf, live ? a.q + b * a.qs.b + h * a.qs.h + (int64_t)i * a.qs.s : nullptr, a.D, half, a.scale2);
    T::hold(uf, live ? a.up + b * a.us.b + h * a.us.h + (int64_t)i * a.us.s : nullptr, a.D, half, 1.f);
    const float lse = live ? a.lse[at] * kLog2e : 0.f, delta = live ? a.delta[at] : 0.f;
    at_f16 acc[NA];
#pragma unroll
    for (int t = 0; t < NA; t++) acc[t] = (at_f16)(0.f);
    if (tiles > 0) store(0);
    __syncthreads();
    for (int t = 0; t < tiles; t++) {
        const int buf = t & 1, j0 = first_key(t);
        if (t + 1 < tiles) load(t + 1);
        if (j0 <= wave_hi && (wave_lo - (j0 + kTile - 1) < a.window || j0 < a.sinks)) {
            at_f16 s = T::times_held(lds[buf][0], qf, lane);
            const at_f16 d = T::times_held(lds[buf][1], uf, lane);
#pragma unroll
            for (int e = 0; e < 16; e++) s[e] = __builtin_amdgcn_exp2f(s[e] - lse) * (d[e] - delta);
            const bool all = j0 + kTile - 1 <= wave_lo && (wave_hi - j0 < a.window || j0 + kTile <= a.sinks) && w1 - w0 == 32;
            if (!all) {
#pragma unroll
                for (int e = 0; e < 16; e++)
                    if (!sees(a, place, j0 + result_row(e, half))) s[e] = 0.f;
            }
            const uint32_t bad = notices.word[buf][0] | notices.word[buf][1] | notices.word[buf][2] | notices.word[buf][3];
            if (__builtin_expect(__builtin_amdgcn_readfirstlane(bad) == 0, 1))
                T::add_product(acc, c0, lds[buf][0], s, lane);
            else
                T::add_product_seen(acc, c0, lds[buf][0], s, lane, [&](int k) { return sees(a, place, j0 + k); });
        }
        if (t + 1 < tiles) store(buf ^ 1);
        __syncthreads();
    }
    if (row < a.rows) T::write(acc, c0, a.dq + b * a.dqs.b + h * a.dqs.h + (int64_t)i * a.dqs.s, a.scale, a.D, half);
}

// dK and dV.  A block of the window's pairs holds 128 keys, 32 a wave, and walks
// the row tiles that see them; S = Q K^T puts a key in a lane, so that P and dS
// are the operands of dV^T += dO^T P and dK^T += Q^T dS as they stand.  A block
// of the sinks' pairs holds 32 keys and walks groups of SLOTS row tiles, one a
// wave.
template <int NT, int NA>
__global__ void __launch_bounds__(256, NT <= 2 ? 2 : 1) attn_grad_keys_fp32(AttnArgs a) {
    using T = Tile<NT>;
    constexpr int SLOTS = NT <= 4 ? 4 : 2;
    __shared__ __attribute__((aligned(16))) float lds[SLOTS][2][T::kFloats];
    __shared__ __attribute__((aligned(16))) float row_lse[SLOTS][kTile], row_delta[SLOTS][kTile];
    __shared__ __attribute__((aligned(16))) int row_place[SLOTS][kTile];
    __shared__ uint32_t bad_q[SLOTS][4], bad_u[SLOTS][4];
    const int tid = (int)threadIdx.x, lane = tid & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    uint32_t id = blockIdx.x;
    const int c0 = (int)(id % (NT / NA)) * 32 * NA;
    id /= NT / NA;
    const int sink_blocks = a.sink_tiles * a.sink_splits, per_head = sink_blocks + a.key_tiles * a.row_splits;
    const int head = (int)(id / (uint32_t)per_head), hk = head % a.kv_heads, b = head / a.kv_heads;
    int unit = (int)(id % (uint32_t)per_head);
    const bool far = unit < sink_blocks;  // of the sinks' pairs
    int tile, part, parts;
    if (far) {
        parts = a.sink_splits;
    } else {
        unit -= sink_blocks;
        parts = a.row_splits;
    }
    tile = unit / parts, part = unit - tile * parts;

    const Sequence seq = sequence_of(a, b);
    const int j0 = far ? tile * kTile : tile * kRowsBlock + wave * 32, key = j0 + (lane & 31);
    const int block_j0 = far ? j0 : tile * kRowsBlock;
    const int keys = far ? min(a.sinks, seq.keys) : seq.keys;
    const int block_j1 = min(block_j0 + (far ? kTile : kRowsBlock), keys);  // past the block's last key
    // The rows that see them: by their places, then by their numbers.
    int place_lo = max(far ? block_j0 + a.window : block_j0, max(seq.first, 0)), place_hi = seq.keys - 1;
    if (!far) place_hi = min(place_hi, block_j1 - 1 + a.window - 1);
    int rlo = 0, tiles = 0, rhi = 0;
    if (block_j0 < block_j1 && place_lo <= place_hi) {
        rlo = (place_lo - seq.first) * a.group;
        rhi = (place_hi - seq.first + 1) * a.group;
        tiles = (rhi - rlo + kTile - 1) / kTile;
    }
    const int t0 = (int)((int64_t)tiles * part / parts), t1 = (int)((int64_t)tiles * (part + 1) / parts);

    const bool live = key < keys;
    at_f4 kf[NT * 4], vf[NT * 4];
    T::hold(kf, live ? a.k + b * a.ks.b + hk * a.ks.h + (int64_t)key * a.ks.s : nullptr, a.D, half, a.scale2);
    T::hold(vf, live ? a.v + b * a.vs.b + hk * a.vs.h + (int64_t)key * a.vs.s : nullptr, a.D, half, 1.f);
    at_f16 dk[NA], dv[NA];
#pragma unroll
    for (int t = 0; t < NA; t++) dk[t] = dv[t] = (at_f16)(0.f);

    typename T::Regs qr, ur;
    float lse_r = 0.f, delta_r = 0.f;
    int place_r = -1;
    const auto load = [&](int t) {
        const int r0 = rlo + t * kTile;
        const auto row_at = [&](const float *p, const AttnView &s, int r) -> const float * {
            const int row = r0 + r;
            if (row >= rhi) return nullptr;
            const int i = (int)a.by_group.divide((uint32_t)row), g = row - i * a.group;
            return p + b * s.b + (int64_t)(hk * a.group + g) * s.h + (int64_t)i * s.s;
        };
        T::load(qr, a.D, [&](int r) { return row_at(a.q, a.qs, r); });
        T::load(ur, a.D, [&](int r) { return row_at(a.up, a.us, r); });
        if (tid < kTile) {
            const int row = r0 + tid;
            lse_r = delta_r = 0.f, place_r = -1;
            if (row < rhi) {
                const int i = (int)a.by_group.divide((uint32_t)row), g = row - i * a.group;
                const int64_t at = ((int64_t)b * a.heads + hk * a.group + g) * a.Sq + i;
                lse_r = a.lse[at] * kLog2e, delta_r = a.delta[at], place_r = seq.first + i;
            }
        }
    };
    const auto store = [&](int slot) {
        const bool bq = T::store(qr, lds[slot][0]), bu = T::store(ur, lds[slot][1]);
        bad_q[slot][wave] = __builtin_amdgcn_ballot_w64(bq) != 0;
        bad_u[slot][wave] = __builtin_amdgcn_ballot_w64(bu) != 0;
        if (tid < kTile) row_lse[slot][tid] = lse_r, row_delta[slot][tid] = delta_r, row_place[slot][tid] = place_r;
    };
    const auto pair_of = [&](int place) {
        if (far) return live && place - key >= a.window;
        return live && key <= place && place - key < a.window;
    };
    const auto compute = [&](int slot, int t) {
        // Places of the tile's rows (the last row's may be of the last tile: rhi).
        const int r0 = rlo + t * kTile, r1 = min(r0 + kTile, rhi);
        const int lo = seq.first + (int)a.by_group.divide((uint32_t)r0), hi = seq.first + (int)a.by_group.divide((uint32_t)(r1 - 1));
        const int j1 = min(j0 + 32, keys);  // past the wave's last key
        if (j0 >= j1) return;
        if (far ? hi - j0 < a.window : (j0 > hi || lo - (j1 - 1) >= a.window)) return;
        const bool all = r1 - r0 == kTile && j1 - j0 == 32 && (far ? lo - (j1 - 1) >= a.window : j1 - 1 <= lo && hi - j0 < a.window);
        at_f16 p = T::times_held(lds[slot][0], kf, lane);
        at_f16 d = T::times_held(lds[slot][1], vf, lane);
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const int r = result_row(e, half);
            // Subnormals too (the instruction alone gives 0): a key may have no larger weight.
            p[e] = __builtin_exp2f(p[e] - row_lse[slot][r]);
            d[e] = p[e] * (d[e] - row_delta[slot][r]);
        }
        if (!all) {
#pragma unroll
            for (int e = 0; e < 16; e++)
                if (!pair_of(row_place[slot][result_row(e, half)])) p[e] = d[e] = 0.f;
        }
        const auto seen = [&](int k) { return pair_of(row_place[slot][k]); };
        const uint32_t bu = bad_u[slot][0] | bad_u[slot][1] | bad_u[slot][2] | bad_u[slot][3];
        if (__builtin_expect(__builtin_amdgcn_readfirstlane(bu) == 0, 1)) T::add_product(dv, c0, lds[slot][1], p, lane);
        else T::add_product_seen(dv, c0, lds[slot][1], p, lane, seen);
        const uint32_t bq = bad_q[slot][0] | bad_q[slot][1] | bad_q[slot][2] | bad_q[slot][3];
        if (__builtin_expect(__builtin_amdgcn_readfirstlane(bq) == 0, 1)) T::add_product(dk, c0, lds[slot][0], d, lane);
        else T::add_product_seen(dk, c0, lds[slot][0], d, lane, seen);
    };
    if (far) {
        for (int t = t0; t < t1; t += SLOTS) {
#pragma unroll 1
            for (int u = 0; u < SLOTS && t + u < t1; u++) {
                load(t + u);
                store(u);
            }
            __syncthreads();
            if (wave < SLOTS && t + wave < t1) compute(wave < SLOTS ? wave : 0, t + wave);
            __syncthreads();
        }
    } else {
        if (t0 < t1) load(t0), store(0);
        __syncthreads();
        for (int t = t0; t < t1; t++) {
            const int slot = (t - t0) & 1;
            if (t + 1 < t1) load(t + 1);
            compute(slot, t);
            if (t + 1 < t1) store(slot ^ 1);
            __syncthreads();
        }
    }
    if (far) {
        if (wave >= SLOTS) return;
        const int64_t at = ((((int64_t)head * a.sink_tiles + tile) * a.sink_splits + part) * SLOTS + wave) * kTile + (lane & 31);
        T::write(dk, c0, a.sink_k + at * a.D, a.scale, a.D, half);
        T::write(dv, c0, a.sink_v + at * a.D, 1.f, a.D, half);
    } else if (a.row_splits > 1) {
        if (key >= a.Sk) return;
        const int64_t at = ((int64_t)part * a.batch * a.kv_heads + head) * a.Sk + key;
        T::write(dk, c0, a.part_k + at * a.D, a.scale, a.D, half);
        T::write(dv, c0, a.part_v + at * a.D, 1.f, a.D, half);
    } else {
        if (key >= a.Sk) return;
        T::write(dk, c0, a.dk + b * a.dks.b + hk * a.dks.h + (int64_t)key * a.dks.s, a.scale, a.D, half);
        T::write(dv, c0, a.dv + b * a.dvs.b + hk * a.dvs.h + (int64_t)key * a.dvs.s, 1.f, a.D, half);
    }
}

// dk and dv of the first `count` keys: the parts over the rows, or what the one part
// wrote, and the sinks' `far` parts of tiles of `tile` keys, in a fixed order.  Eight parts
// are read at a time: one memory latency for all of them.
__global__ void __launch_bounds__(256) attn_reduce(AttnArgs a, int count, int tile, int far) {
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
            const int64_t at = (((head * a.sink_tiles + key / tile) * far) * tile + key % tile) * a.D + d;
            add(x, y, a.sink_k + at, a.sink_v + at, (int64_t)tile * a.D, far);
        }
        *dk = x, *dv = y;
    }
}

template <int NT, int NA>
int run(AttnArgs a, hipStream_t s, int cu_count) {
    constexpr bool pieces = NT <= 4;
    const int64_t heads = (int64_t)a.batch * a.kv_heads;
    const int slots = NT <= 4 ? 4 : 2, sink_tile = pieces ? kRowsBlock : kTile;
    a.row_tiles = (a.rows + kRowsBlock - 1) / kRowsBlock;
    a.key_tiles = (a.Sk + kRowsBlock - 1) / kRowsBlock;
    // The rows that see a key tile in parts where the tiles are few for the CUs.
    const int64_t near_tiles = std::max<int64_t>(1, std::min<int64_t>(a.rows, ((int64_t)a.window + kRowsBlock) * a.group) / kTile);
    a.row_splits = 1;
    if (pieces && a.key_tiles)
        a.row_splits = (int32_t)std::max<int64_t>(1, std::min<int64_t>({2 * (int64_t)cu_count / (heads * a.key_tiles), near_tiles / kPartTiles, 16}));
    // Rows beyond a window see sinks alone: in parts of about as many row tiles as the others,
    // or that fill the device.
    a.sink_tiles = a.window < a.Sk ? (std::min(a.sinks, a.Sk) + sink_tile - 1) / sink_tile : 0;
    a.sink_splits = 1;
    if (a.sink_tiles) {
        const int64_t far_tiles = std::max<int64_t>(1, a.rows / kTile);
        const int64_t want = pieces ? far_tiles * a.row_splits / near_tiles : 2 * (int64_t)cu_count / (heads * a.sink_tiles);
        a.sink_splits = (int32_t)std::max<int64_t>(1, std::min<int64_t>({64, (far_tiles + slots - 1) / slots, want}));
    }
    const int far = a.sink_tiles ? a.sink_splits * (pieces ? 1 : slots) : 0;
    const int64_t row_blocks = heads * a.row_tiles * (NT / NA);
    const int64_t key_blocks = heads * (a.sink_tiles * a.sink_splits + (int64_t)a.key_tiles * a.row_splits) * (NT / NA);
    const int64_t delta_blocks = ((int64_t)a.batch * a.heads * a.Sq + 15) / 16;
    if ((row_blocks + key_blocks) >> 31 || delta_blocks >> 31)
        return set_error(TRS_E_INVALID_ARGUMENT, "attention gradient over too many blocks");
    const int64_t deltas = ((int64_t)a.batch * a.heads * a.Sq + 63) / 64 * 64;
    const int64_t sink_floats = heads * a.sink_tiles * far * sink_tile * a.D;
    const int64_t part_floats = a.row_splits > 1 ? heads * a.row_splits * a.Sk * a.D : 0;
    void *ws = nullptr;
    TRS_CHECK(trs_alloc((size_t)(deltas + 2 * sink_floats + 2 * part_floats) * sizeof(float), &ws));
    float *delta = (float *)ws;
    a.delta = delta;
    a.sink_k = delta + deltas, a.sink_v = a.sink_k + sink_floats;
    a.part_k = a.sink_v + sink_floats, a.part_v = a.part_k + part_floats;
    const auto launch = [&]() -> int {
        // No rows: the keys' gradients are 0.  No keys: the rows' are.
        if (delta_blocks) hipLaunchKernelGGL(attn_delta, dim3((unsigned)delta_blocks), dim3(256), 0, s, a, delta);
        TRS_LAUNCH_CHECK("attention gradient launch");
        if constexpr (pieces) {
            if (key_blocks + row_blocks) launch_attention_grad(a, (uint32_t)key_blocks, (uint32_t)row_blocks, s);
            TRS_LAUNCH_CHECK("attention gradient launch");
        } else {
            if (key_blocks) hipLaunchKernelGGL((attn_grad_keys_fp32<NT, NA>), dim3((unsigned)key_blocks), dim3(256), 0, s, a);
            TRS_LAUNCH_CHECK("attention gradient launch");
            if (row_blocks) hipLaunchKernelGGL((attn_grad_rows_fp32<NT, NA>), dim3((unsigned)row_blocks), dim3(256), 0, s, a);
            TRS_LAUNCH_CHECK("attention gradient launch");
        }
        const int count = a.row_splits > 1 ? a.Sk : a.sink_tiles ? std::min(a.sinks, a.Sk) : 0;
        if (count) {
            const int64_t n = heads * count * a.D;
            hipLaunchKernelGGL(attn_reduce, dim3((unsigned)std::min<int64_t>((n + 255) / 256, 1 << 20)), dim3(256), 0, s, a, count, sink_tile, far);
            TRS_LAUNCH_CHECK("attention gradient launch");
        }
        return TRS_OK;
    };
    const int rc = launch(), frc = trs_free(ws);
    return rc ? rc : frc;
}

}  // namespace

int attention_backward(AttnArgs a, hipStream_t s, int cu_count) {
    if (a.D <= 32) return run<1, 1>(a, s, cu_count);
    if (a.D <= 64) return run<2, 2>(a, s, cu_count);
    if (a.D <= 96) return run<3, 3>(a, s, cu_count);
    if (a.D <= 128) return run<4, 4>(a, s, cu_count);
    return run<8, 4>(a, s, cu_count);
}

}  // namespace trs
