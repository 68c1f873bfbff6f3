// attention_few.hip -- attention.h's attention for few rows a key head: single
// tokens over a cache.
//
// Bound by reading the keys and values once: 16 sequences of 1600 to 8192 keys, 8 key heads
// of 128, window 4096 (470 MB) 90-93 us, 5.1-5.2 TB/s; a sum over 1 GiB reads 5.9.  A wave takes 16 rows (the query
// heads that share the key head, and the few tokens) and streams its share of
// the keys 16 at a time, straight from memory into the registers that
// v_mfma_f32_16x16x4_f32 takes them from: no LDS, no barrier, nothing that waits
// for another wave.  Lane l holds of an operand row (column) l % 16 at k = l / 16,
// of a result column l % 16, register i row 4 (l/16) + i.
// The waves of a block join their maxima and sums in LDS, blocks, if several have a row, in a second
// pass.
#include <hip/hip_runtime.h>

#include "attention_wide.h"

namespace trs {

namespace {

// DP: the width, a multiple of 32.  NW waves a block (16 or 8, the CU to itself: dims that are multiples of four).
template <int DP, int NW, int MODE>
__global__ void __launch_bounds__(64 * NW, NW > 8 ? 4 : DP <= 128 ? 2 : 1) attn_few(AttnArgs a) {
    using T = Wide<DP, MODE>;
    __shared__ __attribute__((aligned(16))) float out_o[NW][16][DP + 4];
    __shared__ float out_ml[NW][16][2];
    const int lane = (int)threadIdx.x & 63, col = lane & 15, quarter = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    uint32_t id = blockIdx.x;
    const int hk = (int)(id % (uint32_t)a.kv_heads);
    id /= (uint32_t)a.kv_heads;
    const int tile = (int)(id % (uint32_t)a.row_tiles);
    id /= (uint32_t)a.row_tiles;
    const int b = (int)(id % (uint32_t)a.batch), part = (int)(id / (uint32_t)a.batch);

    const Sequence seq = sequence_of(a, b);
    const int r0 = tile * 16, r1 = min(r0 + 16, a.rows), row = min(r0 + col, a.rows - 1);
    const int i = (int)a.by_group.divide((uint32_t)row), g = row - i * a.group;
    const int place = r0 + col < a.rows ? seq.first + i : -1;
    const KeyTiles<4> keys(a, seq, r0, r1);
    const int tiles = keys.tiles, waves = a.splits * NW, mine = part * NW + wave;
    const int t0 = (int)((int64_t)tiles * mine / waves), t1 = (int)((int64_t)tiles * (mine + 1) / waves);
    const auto first_key = [&](int t) { return keys.first_key(t); };
    // A key that no row of the block sees is not read: the last one that is seen stands for it.
    const auto read_key = [&](int j) { return keys.read(j) ? j : keys.key_hi; };

    const float *kb = a.k + b * a.ks.b + hk * a.ks.h, *vb = a.v + b * a.vs.b + hk * a.vs.h;
    const float *qrow = a.q + b * a.qs.b + (int64_t)(hk * a.group + g) * a.qs.h + (int64_t)i * a.qs.s;
    typename T::Along q, k;
    typename T::Across v;
    const auto load_k = [&](int t) { T::load(k, kb + (int64_t)read_key(first_key(t) + col) * a.ks.s, a.D, quarter); };
    const auto load_v = [&](int t) {
        T::load(v, [&](int n) { return vb + (int64_t)read_key(first_key(t) + 4 * quarter + n) * a.vs.s; }, a.D, col);
    };
    at_f4 acc[T::TO];
#pragma unroll
    for (int t = 0; t < T::TO; t++) acc[t] = (at_f4)(0.f);
    float most = -__builtin_inff(), sum = 0.f;
    if (t0 < t1) {
        load_k(t0);
        load_v(t0);
        T::load(q, qrow, a.D, quarter);
#pragma unroll
        for (int j = 0; j < T::KJ; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) q[j][e] *= a.scale2;
    }
    for (int t = t0; t < t1; t++) {
        const int j0 = first_key(t), next = t + 1 < t1 ? t + 1 : t;  // the last tile's loads repeat it
        at_f4 s = (at_f4)(0.f);
        T::product(s, k, q);
        load_k(next);
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (!sees(a, place, j0 + 4 * quarter + e)) s[e] = -__builtin_inff();
        float m = __builtin_fmaxf(__builtin_fmaxf(s[0], s[1]), __builtin_fmaxf(s[2], s[3]));
        m = __builtin_fmaxf(m, __shfl_xor(m, 16));
        m = __builtin_fmaxf(m, __shfl_xor(m, 32));
        const float now = __builtin_fmaxf(most, m), base = now == -__builtin_inff() ? 0.f : now;
        const float keep = __builtin_amdgcn_exp2f(most - base);
#pragma unroll
        for (int e = 0; e < 4; e++) s[e] = __builtin_amdgcn_exp2f(s[e] - base);
        sum = sum * keep + ((s[0] + s[1]) + (s[2] + s[3]));
        most = now;
        if (__builtin_amdgcn_ballot_w64(keep != 1.f)) {
#pragma unroll
            for (int c = 0; c < T::TO; c++) acc[c] *= keep;
        }
        if (__builtin_expect(!T::bad(v), 1)) T::add(acc, v, s);
        else
            T::add_seen(acc, s, a.D, col, quarter, [&](int n) { return vb + (int64_t)(j0 + n) * a.vs.s; }, [&](int n) { return sees(a, place, j0 + n); });
        load_v(next);
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
#pragma unroll
    for (int c = 0; c < T::TO; c++)
#pragma unroll
        for (int e = 0; e < 4; e++) out_o[wave][col][T::column(c, e, quarter)] = acc[c][e];
    if (quarter == 0) out_ml[wave][col][0] = most, out_ml[wave][col][1] = sum;
    __syncthreads();
    // The waves' shares of row r, and the row's place in the output.
    for (int x = (int)threadIdx.x; x < 16 * (DP / 4); x += 64 * NW) {
        const int r = x / (DP / 4), d = x % (DP / 4) * 4, at_row = r0 + r;
        if (at_row >= a.rows || d >= a.D) continue;
        float top = -__builtin_inff(), total = 0.f;
#pragma unroll
        for (int w = 0; w < NW; w++) top = __builtin_fmaxf(top, out_ml[w][r][0]);
        const float base = top == -__builtin_inff() ? 0.f : top;
        at_f4 o = (at_f4)(0.f);
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float f = __builtin_amdgcn_exp2f(out_ml[w][r][0] - base);
            total += out_ml[w][r][1] * f;
            o += *(const at_f4 *)&out_o[w][r][d] * f;
        }
        const int at_i = (int)a.by_group.divide((uint32_t)at_row);
        const int64_t h = (int64_t)hk * a.group + at_row - at_i * a.group;
        const int64_t head = (int64_t)b * a.kv_heads + hk;
        float *p;
        if (a.splits > 1) {
            const int64_t at = ((int64_t)part * a.batch * a.kv_heads + head) * a.rows + at_row;
            p = a.part_o + at * a.part_width + d;
            if (d == 0) a.part_ml[2 * at] = top, a.part_ml[2 * at + 1] = total;
        } else {
            o *= seq.first + at_i < 0 ? 0.f : 1.f / total;
            p = a.out + b * a.os.b + h * a.os.h + (int64_t)at_i * a.os.s + d;
            if (a.lse && d == 0) a.lse[((int64_t)b * a.heads + h) * a.Sq + at_i] = log_sum(top, total);
        }
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (d + e < a.D) p[e] = o[e];
    }
}

template <int DP, int NW>
void launch(const AttnArgs &a, dim3 grid, hipStream_t s) {
    if (a.D == DP) hipLaunchKernelGGL((attn_few<DP, NW, 0>), grid, dim3(64 * NW), 0, s, a);
    else if (a.D % 4 == 0) hipLaunchKernelGGL((attn_few<DP, NW, 1>), grid, dim3(64 * NW), 0, s, a);
    else if constexpr (NW == 4) hipLaunchKernelGGL((attn_few<DP, NW, 2>), grid, dim3(64 * NW), 0, s, a);
}

}  // namespace

int launch_attention_few(const AttnArgs &a, dim3 grid, hipStream_t s) {
    if (a.few_waves == 16 && a.D <= 32) launch<32, 16>(a, grid, s);
    else if (a.few_waves == 16) launch<64, 16>(a, grid, s);
    else if (a.few_waves == 8 && a.D <= 96) launch<96, 8>(a, grid, s);
    else if (a.few_waves == 8) launch<128, 8>(a, grid, s);
    else if (a.D <= 32) launch<32, 4>(a, grid, s);
    else if (a.D <= 64) launch<64, 4>(a, grid, s);
    else if (a.D <= 96) launch<96, 4>(a, grid, s);
    else if (a.D <= 128) launch<128, 4>(a, grid, s);
    else if (a.D <= 192) launch<192, 4>(a, grid, s);
    else launch<256, 4>(a, grid, s);
    TRS_LAUNCH_CHECK("attention launch");
    return TRS_OK;
}

}  // namespace trs
