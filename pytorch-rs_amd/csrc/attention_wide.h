// attention_wide.h -- operands of v_mfma_f32_16x16x4_f32 straight from memory, for
// the attention kernels that stage nothing in LDS: few rows (attention_few.hip) and
// the gradients of wide heads (attention_backward_wide.hip).
//
// Lane l holds of an operand row (column) l % 16 at k = l / 16, of a result column
// l % 16, register i row 4 (l/16) + i.  Two forms of 16 rows of a tensor, DP floats wide:
//   along: k runs over the columns, 16 j + 4 (l/16) + e in step (j, e), so that a lane's
//     four steps are 16 bytes of its row l % 16.
//   across: k runs over the rows, 4 (l/16) + i in step i, where the lane has an earlier
//     result's register i; it reads W consecutive columns of that row at once, which go to
//     W result tiles: tile u W + w holds in its row rho column 16 W u + W rho + w.
#pragma once

#include "attention.h"

namespace trs {

// N floats of a row from column c on; columns from D on are 0.  MODE 0: D is the
// padded width; 1: D is a multiple of 4; 2: any D.  No branch around a load:
// what lies past the row's end is read at its start.  `sure`, known at compile time: the
// columns are below any D that takes this width.
template <int N, int MODE>
__device__ __forceinline__ void take(float *v, const float *row, int c, int D, bool sure) {
    typedef float Vec __attribute__((ext_vector_type(N), aligned(4)));
    if constexpr (MODE == 2) {
#pragma unroll
        for (int e = 0; e < N; e++) {
            const bool in = sure || c + e < D;
            const float x = row[in ? c + e : 0];
            v[e] = in ? x : 0.f;
        }
    } else {
        const bool in = MODE == 0 || sure || c < D;
        const Vec x = *(const Vec *)(row + (in ? c : 0));
#pragma unroll
        for (int e = 0; e < N; e++) v[e] = in ? x[e] : 0.f;
    }
}

template <int DP, int MODE>
struct Wide {
    static constexpr int kLeast = DP <= 128 ? DP - 32 : DP - 64;  // D is more: the next width down
    static constexpr int KJ = DP / 16, W = DP % 64 == 0 ? 4 : 2, VU = DP / (16 * W), TO = DP / 16;
    typedef float Along[KJ][4];
    typedef float Across[4][VU][W];

    // The lane's row.
    __device__ __forceinline__ static void load(Along &v, const float *row, int D, int quarter) {
#pragma unroll
        for (int j = 0; j < KJ; j++) take<4, MODE>(v[j], row, 16 * j + 4 * quarter, D, 16 * j + 16 <= kLeast);
    }
    // The lane's four rows: row(i) is row 4 quarter + i.
    template <class Row>
    __device__ __forceinline__ static void load(Across &v, Row &&row, int D, int col) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float *p = row(i);
#pragma unroll
            for (int u = 0; u < VU; u++) take<W, MODE>(v[i][u], p, 16 * W * u + W * col, D, 16 * W * (u + 1) <= kLeast);
        }
    }
    // c += (scale x) y^T over the columns.
    __device__ __forceinline__ static void product(at_f4 &c, const Along &x, const Along &y, float scale = 1.f) {
#pragma unroll
        for (int j = 0; j < KJ; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j][e] * scale, y[j][e], c, 0, 0, 0);
    }
    // acc^T += w^T x over the rows.
    __device__ __forceinline__ static void add(at_f4 (&acc)[TO], const Across &x, const at_f4 &w) {
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int u = 0; u < VU; u++)
#pragma unroll
                for (int e = 0; e < W; e++)
                    acc[u * W + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i][u][e], w[i], acc[u * W + e], 0, 0, 0);
    }
    // Whether a value is an infinity or NaN, in any lane.
    __device__ __forceinline__ static bool bad(const Across &x) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int u = 0; u < VU; u++)
#pragma unroll
                for (int e = 0; e < W; e++) s += x[i][u][e] * 0.f;
        return __builtin_amdgcn_ballot_w64(s != 0.f) != 0;
    }
    // add() where a value is: a pair of row n (at row(n) in memory) and the lane's column
    // that seen(n) leaves out adds nothing, where the matrix instruction would add 0 * NaN.
    template <class Row, class Seen>
    __device__ __forceinline__ static void add_seen(at_f4 (&acc)[TO], const at_f4 &w, int D, int col, int quarter, Row &&row, Seen &&seen) {
#pragma unroll 1
        for (int n = 0; n < 16; n++) {
            float p = 0.f;
#pragma unroll
            for (int i = 0; i < 4; i++) p = (n & 3) == i ? w[i] : p;
            p = __shfl(p, col + 16 * (n >> 2));
            if (!seen(n)) continue;
            const float *x = row(n);
#pragma unroll
            for (int t = 0; t < TO; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int d = column(t, i, quarter);
                    if (d < D) acc[t][i] += p * x[d];
                }
        }
    }
    // The column that register i of result tile t holds.
    __device__ __forceinline__ static int column(int t, int i, int quarter) {
        return 16 * W * (t / W) + W * (4 * quarter + i) + t % W;
    }
    // Writes f * acc^T: the lane's column of acc is the row at p.
    __device__ __forceinline__ static void write(const at_f4 (&acc)[TO], float *p, float f, int D, int quarter) {
#pragma unroll
        for (int u = 0; u < VU; u++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int d = column(u * W, i, quarter);
#pragma unroll
                for (int e = 0; e < W; e++)
                    if (MODE == 0 || d + e < D) p[d + e] = acc[u * W + e][i] * f;
            }
    }
};

}  // namespace trs
