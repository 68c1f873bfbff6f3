// attention.h -- causal attention with a sliding window and first tokens that
// stay visible: what its host part (attention.hip) and its kernels
// (attention_forward.hip, attention_backward.hip) share.
//
// Query i of a sequence that has n keys stands at place p = n - Sq + i and sees
//   key j  where  j <= p  and  (p - j < window  or  j < sinks).
// The query heads that share a key head are taken together: their rows are
// numbered r = i * group + (head within the group), so that a tile of rows
// reads its keys and values once for all of them and spans few places.
//
// Products run on the bf16 matrix cores, in pieces, for heads of up to 128 dims, and on
// the fp32 instruction for wider ones and for few rows (attention_wide.h).  Lane l of a
// wave holds of the operands of a 32x32 product row (or column) l % 32, at 1 or 8 k in its
// half l / 32, and of the result column l % 32, register i row 8 (i/4) + 4 (l/32) + i%4.
// Which k a step takes is free as long as both operands agree, which saves every
// transposition of a result: a product whose k runs over the rows of an earlier result
// takes that result's registers as its operand as they stand, with the other operand read
// at those rows.
#pragma once

#include "gemm_tile.h"
#include "op_checks.h"

namespace trs {

typedef float at_f16 __attribute__((ext_vector_type(16)));
typedef float at_f4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 32;        // keys or rows per tile in LDS
constexpr int kRowsBlock = 128;  // rows (or keys) per block of the gradients: 32 a wave
constexpr int kPiecesDim = 128;  // the widest heads that run in pieces
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLog2eLow = 1.925963033500e-8f, kLn2Low = -1.904654299958e-9f;  // what the floats above leave out

struct AttnView {  // [batch, head, token, dim], unit stride along dim
    int64_t b, h, s;
};

// What the gradients take of every row, [batch, head, token] each: a pair's weight is
// exp2(score - base) * share, the score in base 2.
//
// A row's lse is one float, off by up to half a unit in its last place, and so is every weight
// from it, by |lse| 2^-24 of itself.  Up to kMostLse (2^-17 of a weight) it serves, its product
// with log2(e) in two floats, base and log2(1/share).  Of other rows maximum and sum are worked
// out again, in the order in which the gradients add a score up: the same bits, or the largest
// would be off by its last place, however much that is.  The forms in pieces have one order, the
// fp32 forms another.  (All rows again: training step of 4096 tokens, 32 heads of 128, window 2048
// 2.7 -> 5.4 ms, of 2 x 2048 tokens, 16 heads of 64 0.30 -> 0.59.)
constexpr float kMostLse = 256.f;
struct RowFacts {
    float *delta;  // rowsum(dO o)
    struct Weights {
        float *base, *share;  // pieces': times 2^40
    } pieces, fp32;
};

struct AttnArgs {
    const float *q, *k, *v;
    float *out, *lse;
    const float *up;
    RowFacts facts;
    float *dq, *dk, *dv;
    const int32_t *lengths;  // keys of each sequence; null: Sk
    AttnView qs, ks, vs, os, us, dqs, dks, dvs;
    int32_t batch, heads, kv_heads, group, Sq, Sk, D;
    int32_t rows;  // Sq * group
    int32_t window, sinks;
    float scale, scale2;  // scale2 = scale * log2(e)
    SmallDivisor by_group;
    // Work split over the keys (forward): a block of rows has up to `splits` parts, in
    // attn_rows one for every part_tiles of its key tiles; the parts' unnormalised
    // outputs [part][batch, key head, row][part_width], and (maximum, sum).
    int32_t splits, part_tiles, row_tiles, part_width;
    int32_t few_waves;  // waves of a block of attn_few
    float *part_o, *part_ml;
    // Work split over the rows (backward).
    int32_t key_tiles, row_splits, sink_tiles, sink_splits;
    float *part_k, *part_v, *sink_k, *sink_v;
};

// A sequence's keys, and the place of its first query (below 0 where the
// queries are more than the keys).
struct Sequence {
    int32_t keys, first;
};
__device__ __forceinline__ Sequence sequence_of(const AttnArgs &a, int b) {
    int n = a.Sk;
    if (a.lengths) n = min(max(a.lengths[b], 0), a.Sk);
    return Sequence{n, n - a.Sq};
}

__device__ __forceinline__ bool sees(const AttnArgs &a, int place, int key) {
    return (key <= place) & ((place - key < a.window) | (key < a.sinks));
}

// log(sum of exponentials) of a row from the base-2 maximum and the sum: rounded once.
__device__ __forceinline__ float log_sum(float most, float sum) {
    const float l = __builtin_amdgcn_logf(sum), t = most + l;
    const float b = t - most, low = (most - (t - b)) + (l - b);  // t + low is most + l
    return __builtin_isfinite(t) ? __builtin_fmaf(t, kLn2, __builtin_fmaf(t, kLn2Low, low * kLn2)) : t;
}

// Four floats of a row from column c on, zero from the row's end on.
__device__ __forceinline__ at_f4 row_chunk(const float *row, int c, int D) {
    if (c + 4 <= D) {
        const f4u v = *(const f4u *)(row + c);
        return at_f4{v[0], v[1], v[2], v[3]};
    }
    at_f4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (c + e < D) v[e] = row[c + e];
    return v;
}

// The row (of M or N) or k that register i of a result holds in this lane.
__device__ __forceinline__ int result_row(int i, int half) { return 8 * (i >> 2) + 4 * half + (i & 3); }

// 32 rows x times 32 rows y over their columns on the fp32 instruction: x(c) and y(c) are four
// floats of the lane's rows from column c on.  One order of the sum for all that need a score.
template <class X, class Y>
__device__ __forceinline__ at_f16 product_fp32(int D, int half, X &&x, Y &&y) {
    at_f16 c = (at_f16)(0.f);
#pragma unroll 1
    for (int j = 0; j < D; j += 8) {
        const at_f4 u = x(j + 4 * half), w = y(j + 4 * half);
#pragma unroll
        for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(u[e], w[e], c, 0, 0, 0);
    }
    return c;
}

// A tile of kTile rows by 32 NT floats in LDS, for blocks whose values the pieces below
// do not hold.  The pitch puts rows 4 banks apart, so that 8 lanes reading 16 bytes each at
// one column cover 32 banks.
template <int NT, int LANES>
struct Tile {
    static constexpr int kCols = 32 * NT, kPitch = kCols + 4, kFloats = kTile * kPitch;

    // row(r): the tile's row r in memory, or null for a row of zeros.
    template <class Row>
    __device__ __forceinline__ static void stage(float *lds, int D, Row &&row) {
#pragma unroll 1
        for (int n = (int)threadIdx.x; n < kTile * kCols / 4; n += LANES) {
            const int r = n / (kCols / 4), c = n % (kCols / 4) * 4;
            const float *p = row(r);
            *(at_f4 *)(lds + r * kPitch + c) = p ? row_chunk(p, c, D) : at_f4{0.f, 0.f, 0.f, 0.f};
        }
    }
    // (tile_scale times the tile's rows) x (scale times the lane's row; null: zeros), over the columns.
    __device__ __forceinline__ static at_f16 times_row(const float *lds, const float *row, int D, float scale, int lane, float tile_scale = 1.f) {
        const float *p = lds + (lane & 31) * kPitch;
        return product_fp32(
            D, lane >> 5, [&](int c) { return *(const at_f4 *)(p + c) * tile_scale; },
            [&](int c) { return row ? row_chunk(row, c, D) * scale : at_f4{0.f, 0.f, 0.f, 0.f}; });
    }
    // acc^T += w^T tile over its rows.  A pair of a row (of the tile) and a column (of the
    // lane) that seen(row) leaves out adds nothing, where the matrix instruction would
    // add 0 * NaN.
    template <class Seen>
    __device__ __forceinline__ static void add_product_seen(at_f16 (&acc)[NT], const float *lds, const at_f16 &w, int lane, Seen &&seen) {
#pragma unroll 1
        for (int k = 0; k < kTile; k++) {
            const int i = (k >> 3) * 4 + (k & 3), from = (lane & 31) + 32 * ((k >> 2) & 1);
            float x = 0.f;
#pragma unroll
            for (int q = 0; q < 16; q++) x = q == i ? w[q] : x;
            x = __shfl(x, from);
            if (!seen(k)) continue;
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int r = 0; r < 16; r++) acc[t][r] += x * lds[k * kPitch + 32 * t + result_row(r, lane >> 5)];
        }
    }
    // Writes f * acc^T: the lane's column of acc is the row at p.
    __device__ __forceinline__ static void write(const at_f16 (&acc)[NT], float *p, float f, int D, int half) {
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int c = 32 * t + result_row(r, half);
                if (c < D) p[c] = acc[t][r] * f;
            }
    }
};

// The same products on the bf16 matrix cores: every float as the exact sum of
// three bf16 pieces and six of their nine products, as in gemm_tile.h, at 3/8 of
// the fp32 instruction's time.  Values are taken times 2^40 and results times the
// inverse, powers of two that cost no rounding: so the third piece of any float,
// subnormals included, stands above bf16's least value and nothing is lost.
// An infinity, a NaN or a value (or sum) beyond what is left of the range, 2^87 and
// 2^47, shows as a result that is not finite; the block then does its rows again on
// the fp32 instruction.  A score of -inf alone would show in no result, it weighs nothing:
// scores are looked at before any is hidden (Lowest).
constexpr float kUp = 0x1p40f, kDown = 0x1p-40f, kUp2 = 0x1p80f, kDown2 = 0x1p-80f;

struct Pieces {
    gt_bf8 p[3];  // h, m, l of eight values
};
// Eight values split pair by pair, among matrix instructions.
struct Splitting {
    uint32_t h[4], m[4], l[4];
    __device__ __forceinline__ void pair(int i, float a, float b) {
        uint32_t lost = 0;
        split_pair(a, b, h[i], m[i], l[i], lost);
    }
    __device__ __forceinline__ Pieces done() const {
        typedef uint32_t U4 __attribute__((ext_vector_type(4)));
        const U4 x = {h[0], h[1], h[2], h[3]}, y = {m[0], m[1], m[2], m[3]}, z = {l[0], l[1], l[2], l[3]};
        return Pieces{{__builtin_bit_cast(gt_bf8, x), __builtin_bit_cast(gt_bf8, y), __builtin_bit_cast(gt_bf8, z)}};
    }
};
// TURNED: the same sum, bit for bit, as of (b, a), whose result is this one's transpose.
template <bool TURNED = false>
__device__ __forceinline__ void mfma_pieces(at_f16 &c, const Pieces &a, const Pieces &b) {
    constexpr int PA[6] = {2, 1, 1, 0, 0, 0}, PB[6] = {0, 0, 1, 1, 2, 0};
#pragma unroll
    for (int i = 0; i < 6; i++)
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[TURNED ? PB[i] : PA[i]], b.p[TURNED ? PA[i] : PB[i]], c, 0, 0, 0);
}

// A lane's 16 bytes of a unit (the next comment): row lane % 32 at columns 8 (lane/32) on.
__device__ __forceinline__ int unit_place(int lane) { return (lane ^ lane >> 5 << 2) * 16; }

// A tile of kTile rows by 32 NT columns of one tensor or of two, as pieces in LDS.  A
// unit is 16 columns, 1 KiB of each piece, loaded, split and stored by one wave: (row,
// column) at 512 (column/8) + 16 (row ^ 4 (column/8)) + 2 (column%8), which is the order of a
// fragment whose k runs along the columns (lane l: row l % 32 at columns 8 (l/32) on).  A
// fragment whose k runs across the rows is read from the same bytes by the transposing
// load: 16 lanes ask for 4 rows by 16 columns, four columns of a row each, and each gets
// its own column's four rows; the exchange of rows puts their two halves on different
// banks (prompt of 4096 tokens, 32 heads of 128: a third of the conflicts, 327 -> 326 us; rows
// exchanged by the unit too leave none, but cost two registers, 331).
//
// Columns from D on are 0.  No branch stands around a load, which would wait for all of
// them: what must not be read is read elsewhere in the row and then 0.  WIDTH 4: D is the
// tile's width; 2: D is a multiple of 4, read 16 bytes at a time; 1: any D, read float by
// float (3 prompts of 1000 tokens with heads of 80: 68 us so, 44 in fours).
template <int WIDTH>
struct Unit {
    float v[8];
    // `sure`: the unit's columns are all below D.
    __device__ __forceinline__ void load(const float *row, int u, int D, int lane, bool sure = false) {
        const int c = 16 * u + 8 * (lane >> 5);
        if constexpr (WIDTH > 1) {
            const bool in0 = WIDTH == 4 || sure || c < D, in1 = WIDTH == 4 || sure || c + 4 < D;
            const f4u x = *(const f4u *)(row + (in0 ? c : 0)), y = *(const f4u *)(row + (in1 ? c + 4 : 0));
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = in0 ? x[e] : 0.f, v[4 + e] = in1 ? y[e] : 0.f;
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const bool in = sure || c + e < D;
                const float x = row[in ? c + e : 0];
                v[e] = in ? x : 0.f;
            }
        }
    }
    __device__ __forceinline__ Pieces split(float scale) const {
        Splitting x;
#pragma unroll
        for (int i = 0; i < 4; i++) x.pair(i, v[2 * i] * scale, v[2 * i + 1] * scale);
        return x.done();
    }
    // Pair i of four; the last one stores the unit.  UNITS: units of a piece in the buffer.
    template <int UNITS>
    __device__ __forceinline__ void store_pair(Splitting &x, int i, char *lds, int u, int lane, float up = kUp) const {
        x.pair(i, v[2 * i] * up, v[2 * i + 1] * up);
        if (i == 3) {
            const Pieces y = x.done();
#pragma unroll
            for (int p = 0; p < 3; p++) *(gt_bf8 *)(lds + (p * UNITS + u) * 1024 + unit_place(lane)) = y.p[p];
        }
    }
    template <int UNITS>
    __device__ __forceinline__ void store(char *lds, int u, int lane, float up = kUp) const {
        Splitting x;
#pragma unroll
        for (int i = 0; i < 4; i++) store_pair<UNITS>(x, i, lds, u, lane, up);
    }
};
// Unit u: k runs along its columns.
template <int UNITS>
__device__ __forceinline__ Pieces along(const char *lds, int u, int lane) {
    Pieces x;
#pragma unroll
    for (int p = 0; p < 3; p++) x.p[p] = *(const gt_bf8 *)(lds + (p * UNITS + u) * 1024 + unit_place(lane));
    return x;
}
// Units u and u + 1 as 32 columns: k runs across rows 16 slot to 16 slot + 15, in the
// order in which a result holds them: place 8 h + e is row 8 (e/4) + 4 h + e%4.
template <int UNITS>
__device__ __forceinline__ Pieces across(const char *lds, int u, int slot, int lane) {
    typedef short S4 __attribute__((ext_vector_type(4)));
    typedef short S8 __attribute__((ext_vector_type(8)));
    typedef S4 __attribute__((address_space(3))) *Lds;
    const int second = lane >> 1 & 1;
    const char *at = lds + (lane >> 4 & 1) * 1024 + second * 512 + (4 * (lane >> 5 ^ second) + (lane >> 2 & 3)) * 16 + (lane & 1) * 8;
    Pieces x;
#pragma unroll
    for (int p = 0; p < 3; p++) {
        const char *q = at + (p * UNITS + u) * 1024 + slot * 256;
        const S4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)q), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(q + 128));
        x.p[p] = __builtin_bit_cast(gt_bf8, (S8){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
    }
    return x;
}
// STEPS steps of six matrix instructions, in the order written: multiply(s, f) takes the
// fragment that read(s) asked for a step earlier, and work(s) is other work for the
// step's matrix instructions to run under (a wave issues in order, so it has to stand
// among them).  `f` holds step 0's fragment; next(f) reads the one that follows the last
// step's, with that step.
template <int STEPS, class Read, class Multiply, class Work, class Next>
__device__ __forceinline__ void steps(Pieces &f, Read &&read, Multiply &&multiply, Work &&work, Next &&next) {
#pragma unroll
    for (int s = 0; s < STEPS; s++) {
        const Pieces now = f;
        if (s + 1 < STEPS) f = read(s + 1);
        else next(f);
        multiply(s, now);
        work(s);
        __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);  // LDS reads
#pragma unroll
        for (int i = 0; i < 6; i++) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a matrix instruction
            __builtin_amdgcn_sched_group_barrier(0x002, 8, 0);  // vector instructions (3 and 6 measured alike)
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}
// Items first to last of `items` dealt evenly to `of` steps: those of step s.
template <class F>
__device__ __forceinline__ void dealt(int items, int s, int of, F &&item) {
#pragma unroll
    for (int i = s * items / of; i < (s + 1) * items / of; i++) item(i);
}
// Writes unit * f * acc^T: the lane's column of acc is the row at p.  Registers 4 i to 4 i + 3 are
// consecutive columns, 16 bytes; two halves of a wave write 32 of a row.
template <int WIDTH, int NT>
__device__ __forceinline__ void write_row(const at_f16 (&acc)[NT], float *p, float unit, float f, int D, int half) {
#pragma unroll
    for (int c = 0; c < NT; c++)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const int d = 32 * c + result_row(e, half);
            const f4u x = {acc[c][e] * unit * f, acc[c][e + 1] * unit * f, acc[c][e + 2] * unit * f, acc[c][e + 3] * unit * f};
            if (WIDTH == 4 || (WIDTH == 2 && d < D)) {
                *(f4u *)(p + d) = x;
            } else if (WIDTH == 1) {
#pragma unroll
                for (int q = 0; q < 4; q++)
                    if (d + q < D) p[d + q] = x[q];
            }
        }
}

// Whether any score so far was -inf.  As unsigned numbers its bits are above those of every
// score that is not NaN: a maximum of three takes two scores at a time, and no comparison.
struct Lowest {
    uint32_t bits = 0;
    __device__ __forceinline__ void add(const at_f16 &s) {
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const uint32_t x = __builtin_bit_cast(uint32_t, s[e]);
            bits = bits > x ? bits : x;
        }
    }
    // Whether one is, in any lane of the wave.
    __device__ __forceinline__ bool infinite() const { return __builtin_amdgcn_ballot_w64(bits >= 0xff800000u) != 0; }
};

// Whether a value is an infinity or NaN in any lane of the wave.
template <int N>
__device__ __forceinline__ bool not_finite(const at_f16 (&acc)[N], float more) {
    float s = more * 0.f;
#pragma unroll
    for (int t = 0; t < N; t++)
#pragma unroll
        for (int r = 0; r < 16; r++) s += acc[t][r] * 0.f;
    return __builtin_amdgcn_ballot_w64(s != 0.f) != 0;
}

// The tiles of 1 << SHIFT keys that rows r0 to r1 of a key head see, the sinks' first and
// then the window's.
template <int SHIFT>
struct KeyTiles {
    int key_lo, key_hi, sinks, first, nsink, tiles;

    KeyTiles() = default;
    __host__ __device__ __forceinline__ KeyTiles(const AttnArgs &a, const Sequence &seq, int r0, int r1) {
        const int lo = seq.first + (int)a.by_group.divide((uint32_t)r0) - a.window + 1;
        key_lo = lo > 0 ? lo : 0, key_hi = seq.first + (int)a.by_group.divide((uint32_t)(r1 - 1));
        sinks = a.sinks < key_hi + 1 ? a.sinks : key_hi + 1;
        first = key_lo >> SHIFT;
        const int before = (sinks + (1 << SHIFT) - 1) >> SHIFT;
        nsink = key_hi < 0 ? 0 : before < first ? before : first;
        tiles = key_hi < 0 ? 0 : nsink + (key_hi >> SHIFT) - first + 1;
    }
    __host__ __device__ __forceinline__ int parts(const AttnArgs &a) const {
        const int n = tiles > a.part_tiles ? (tiles + a.part_tiles - 1) / a.part_tiles : 1;
        return n < a.splits ? n : a.splits;
    }
    __device__ __forceinline__ int first_key(int t) const { return (t < nsink ? t : first + t - nsink) << SHIFT; }
    // Whether a row sees key j.
    __device__ __forceinline__ bool read(int j) const { return j <= key_hi && (j >= key_lo || j < sinks); }
};

// What a block of 32 rows a wave works on: its rows, their places, and their key tiles.
template <int NW>
struct RowBlock : KeyTiles<5> {
    int lane, half, wave;
    int hk, b, row, i, g;  // the lane's row: query i of head hk * group + g
    int place;             // below 0: sees nothing
    int wave_lo, wave_hi;  // places of the wave's rows
    bool whole;            // the wave has 32 rows

    __device__ __forceinline__ RowBlock(const AttnArgs &a, int kv_head, int tile, int batch) : hk(kv_head), b(batch) {
        lane = (int)threadIdx.x & 63, half = lane >> 5;
        wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
        const Sequence seq = sequence_of(a, b);
        const auto place_of = [&](int r) { return seq.first + (int)a.by_group.divide((uint32_t)r); };
        const int r0 = tile * 32 * NW, r1 = min(r0 + 32 * NW, a.rows), last = a.rows - 1;
        const int w0 = r0 + wave * 32, w1 = min(w0 + 32, a.rows);
        row = w0 + (lane & 31);
        i = (int)a.by_group.divide((uint32_t)min(row, last)), g = min(row, last) - i * a.group;
        place = row < a.rows ? max(seq.first + i, -1) : -1;
        wave_lo = place_of(min(w0, last));
        wave_hi = w0 < w1 ? place_of(w1 - 1) : -1;
        whole = w1 - w0 == 32;
        (KeyTiles<5> &)*this = KeyTiles<5>(a, seq, r0, r1);
    }
    // Whether a row of the wave sees a key of the tile at j0, and whether all see all.
    __device__ __forceinline__ bool any(const AttnArgs &a, int j0) const {
        return j0 <= wave_hi && (wave_lo - (j0 + kTile - 1) < a.window || j0 < a.sinks);
    }
    __device__ __forceinline__ bool all(const AttnArgs &a, int j0) const {
        return whole && j0 + kTile - 1 <= wave_lo && (wave_hi - j0 < a.window || j0 + kTile <= a.sinks);
    }
    // The row's place in a [batch, head, token, dim] view.
    __device__ __forceinline__ int64_t at(const AttnArgs &a, const AttnView &v) const {
        return b * v.b + (int64_t)(hk * a.group + g) * v.h + (int64_t)i * v.s;
    }
    // And in [batch, head, token].
    __device__ __forceinline__ int64_t index(const AttnArgs &a) const {
        return ((int64_t)b * a.heads + hk * a.group + g) * a.Sq + i;
    }
};

// Words that the waves of a block tell one another ahead of a barrier.
template <int NW>
struct Notices {
    uint32_t word[2][NW];
    __device__ __forceinline__ bool any(int n) const {
        uint32_t x = 0;
#pragma unroll
        for (int w = 0; w < NW; w++) x |= word[n][w];
        return __builtin_amdgcn_readfirstlane(x) != 0;
    }
};

// An input whose last dim has a unit stride: itself, or a contiguous copy in the
// block cache.
struct Dense {
    const float *at = nullptr;
    AttnView view{};
    void *copy = nullptr;
    int take(const float *p, const trs_layout *l) {
        if (layout_numel(l) == 0) return TRS_OK;
        if (l->stride[3] == 1 || l->shape[3] == 1) {
            at = p + l->offset;
            view = {l->stride[0], l->stride[1], l->stride[2]};
            return TRS_OK;
        }
        const trs_layout c = contiguous_like(l);
        TRS_CHECK(trs_alloc((size_t)layout_numel(l) * sizeof(float), &copy));
        at = (const float *)copy;
        view = {c.stride[0], c.stride[1], c.stride[2]};
        return trs_unary_f32(TRS_COPY, p, l, (float *)copy, &c);
    }
    ~Dense() {
        if (copy) (void)trs_free(copy);
    }
};

// Few rows a key head (attention_few.hip): row_tiles of 16 rows, `splits` parts.
int launch_attention_few(const AttnArgs &a, dim3 grid, hipStream_t s);
// The gradients in pieces, for D up to kPiecesDim: blocks of 128 keys over their windows'
// rows, or over the rows beyond the window of the sinks (sink_tiles of 128 keys), and of 128
// rows.
void launch_attention_grad(const AttnArgs &a, uint32_t key_blocks, uint32_t row_blocks, hipStream_t s);
// And of wider heads: waves of 16 keys, of 16 of the sinks' keys, and of 16 rows.
void launch_attention_grad_wide(const AttnArgs &a, uint32_t key_units, uint32_t row_units, hipStream_t s);
int attention_forward(AttnArgs a, hipStream_t s, int cu_count);
int attention_backward(AttnArgs a, hipStream_t s, int cu_count);

}  // namespace trs
