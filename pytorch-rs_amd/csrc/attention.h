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
// Products run on the fp32 matrix instruction v_mfma_f32_32x32x2_f32.  Lane l of
// a wave holds of its operands row (or column) l % 32 at k = l / 32, and of
// its result column l % 32, register i row  8 (i/4) + 4 (l/32) + i%4.  Which k
// a step takes is free as long as both operands agree, which saves every
// transposition here: a product whose k runs over the rows of an earlier
// result takes that result's register i as its operand as it stands, with the
// other operand read at row 8 (i/4) + 4 (l/32) + i%4.
#pragma once

#include "op_checks.h"

namespace trs {

typedef float at_f16 __attribute__((ext_vector_type(16)));
typedef float at_f4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 32;      // keys or rows per tile in LDS
constexpr int kRowsBlock = 128;  // rows (or keys) per block: 32 a wave
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttnView {  // [batch, head, token, dim], unit stride along dim
    int64_t b, h, s;
};

struct AttnArgs {
    const float *q, *k, *v;
    float *out, *lse;
    const float *up, *delta;
    float *dq, *dk, *dv;
    const int32_t *lengths;  // keys of each sequence; null: Sk
    AttnView qs, ks, vs, os, us, dqs, dks, dvs;
    int32_t batch, heads, kv_heads, group, Sq, Sk, D;
    int32_t rows;  // Sq * group
    int32_t window, sinks;
    float scale, scale2;  // scale2 = scale * log2(e)
    SmallDivisor by_group;
    // Work split over the keys (forward): the parts, their unnormalised
    // outputs [part][batch, key head, row][D], and (maximum, sum).
    int32_t splits, row_tiles;
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
    return key <= place && (place - key < a.window || key < a.sinks);
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

// A tile of kTile rows by 32 NT floats in LDS.  The pitch puts rows 4 banks
// apart, so that 8 lanes reading 16 bytes each at one column cover 32 banks.
template <int NT>
struct Tile {
    static constexpr int kCols = 32 * NT, kPitch = kCols + 4, kFloats = kTile * kPitch;
    static constexpr int kChunks = kTile * kCols / 4 / 256;  // 16-byte chunks a lane of 256 moves
    // Columns a lane reads at once in a product over the tile's rows, and so the
    // result tiles whose rows interleave: result tile u * W + w holds in its row
    // rho the tile's column 32 W u + W rho + w.
    static constexpr int W = NT % 4 == 0 ? 4 : NT % 2 == 0 ? 2 : 1;
    typedef at_f4 Regs[kChunks];

    __device__ __forceinline__ static int row_of(int q) { return ((int)threadIdx.x + q * 256) / (kCols / 4); }
    __device__ __forceinline__ static int col_of(int q) { return ((int)threadIdx.x + q * 256) % (kCols / 4) * 4; }
    // row(r): the tile's row r in memory, or null for a row of zeros.
    template <class Row>
    __device__ __forceinline__ static void load(Regs &v, int D, Row &&row) {
#pragma unroll
        for (int q = 0; q < kChunks; q++) {
            const float *p = row(row_of(q));
            v[q] = p ? row_chunk(p, col_of(q), D) : at_f4{0.f, 0.f, 0.f, 0.f};
        }
    }
    // Whether a value of the lane's chunks is infinite or NaN.
    __device__ __forceinline__ static bool store(const Regs &v, float *lds) {
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < kChunks; q++) {
            *(at_f4 *)(lds + row_of(q) * kPitch + col_of(q)) = v[q];
            s += v[q][0] * 0.f + v[q][1] * 0.f + v[q][2] * 0.f + v[q][3] * 0.f;
        }
        return s != 0.f;
    }
    // A lane's operand of 32 rows held in registers: row `p` (null: zeros), at
    // the k that load_frag reads.
    __device__ __forceinline__ static void hold(at_f4 (&f)[NT * 4], const float *p, int D, int half, float scale) {
#pragma unroll
        for (int j = 0; j < NT * 4; j++) {
            f[j] = p ? row_chunk(p, 8 * j + 4 * half, D) : at_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 4; e++) f[j][e] *= scale;
        }
    }
    // c += (the tile's rows) x (held rows), over the columns.
    __device__ __forceinline__ static at_f16 times_held(const float *lds, const at_f4 (&f)[NT * 4], int lane) {
        at_f16 c = (at_f16)(0.f);
        const float *p = lds + (lane & 31) * kPitch + 4 * (lane >> 5);
#pragma unroll
        for (int j = 0; j < NT * 4; j++) {
            const at_f4 x = *(const at_f4 *)(p + 8 * j);
#pragma unroll
            for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], f[j][e], c, 0, 0, 0);
        }
        return c;
    }
    // acc[t] += (the tile's columns) x w over its rows: acc^T += w^T tile, for the
    // NA result tiles from column c0 on (whole groups of W tiles).
    template <int NA>
    __device__ __forceinline__ static void add_product(at_f16 (&acc)[NA], int c0, const float *lds, const at_f16 &w, int lane) {
        static_assert(NA % W == 0);
        typedef float Vec __attribute__((ext_vector_type(W)));
        const float *p = lds + 4 * (lane >> 5) * kPitch + c0 + W * (lane & 31);
#pragma unroll
        for (int i = 0; i < 16; i++)
#pragma unroll
            for (int u = 0; u < NA / W; u++) {
                const float *at = p + (8 * (i >> 2) + (i & 3)) * kPitch + 32 * W * u;
                if constexpr (W == 1) {
                    acc[u] = __builtin_amdgcn_mfma_f32_32x32x2f32(*at, w[i], acc[u], 0, 0, 0);
                } else {
                    const Vec x = *(const Vec *)at;
#pragma unroll
                    for (int e = 0; e < W; e++)
                        acc[u * W + e] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], w[i], acc[u * W + e], 0, 0, 0);
                }
            }
    }
    // The same where the tile holds infinities or NaN: a pair whose row (of the
    // tile) and column (of the lane) do not see each other adds nothing, where
    // the matrix instruction would add 0 * NaN.
    template <int NA, class Sees>
    __device__ __forceinline__ static void add_product_seen(at_f16 (&acc)[NA], int c0, const float *lds, const at_f16 &w,
                                                            int lane, Sees &&seen) {
#pragma unroll 1
        for (int k = 0; k < kTile; k++) {
            const int i = (k >> 3) * 4 + (k & 3), from = (lane & 31) + 32 * ((k >> 2) & 1);
            float x = 0.f;
#pragma unroll
            for (int q = 0; q < 16; q++) x = q == i ? w[q] : x;
            x = __shfl(x, from);
            if (!seen(k)) continue;
#pragma unroll
            for (int t = 0; t < NA; t++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    acc[t][r] += x * lds[k * kPitch + c0 + column(t, r, lane >> 5)];
        }
    }
    // The tile's column that register r of result tile t holds.
    __device__ __forceinline__ static int column(int t, int r, int half) {
        return 32 * W * (t / W) + W * result_row(r, half) + t % W;
    }
    // Writes f * acc^T from column c0 on: the lane's column of acc is the row at p.
    template <int NA>
    __device__ __forceinline__ static void write(const at_f16 (&acc)[NA], int c0, float *p, float f, int D, int half) {
#pragma unroll
        for (int u = 0; u < NA / W; u++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int c = c0 + column(u * W, r, half);
#pragma unroll
                for (int e = 0; e < W; e++)
                    if (c + e < D) p[c + e] = acc[u * W + e][r] * f;
            }
    }
};

// Words that the waves of a block tell one another ahead of a barrier.
struct Notices {
    uint32_t word[2][4];
};

// Few rows a key head (attention_few.hip): row_tiles of 16 rows, `splits` parts.
int launch_attention_few(const AttnArgs &a, hipStream_t s);
int attention_forward(AttnArgs a, hipStream_t s, int cu_count);
int attention_backward(AttnArgs a, hipStream_t s, int cu_count);

}  // namespace trs
