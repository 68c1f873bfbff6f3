// attention_forward.hip -- the output of attention.h's attention.
#include <hip/hip_runtime.h>

#include "attention.h"

namespace trs {

namespace {

constexpr int kFewRows = 32;   // rows a key head that attn_few takes
constexpr int kPartTiles = 2;  // the least key tiles of a part, a wave

// 128 rows of one key head, 32 a wave, over key tiles that the block stages in
// LDS, two buffers in turn.  S^T = K Q^T puts a row of the softmax in a lane
// (and its other half): the running maximum and sum are per lane, and P^T is
// the operand of O^T += V^T P^T as it stands.  The maximum and sum are of
// base-2 exponents, log2(e) going into the queries with the scale.
template <int NT>
__global__ void __launch_bounds__(256, NT <= 4 ? 2 : 1) attn_rows(AttnArgs a) {
    using T = Tile<NT>;
    __shared__ __attribute__((aligned(16))) float lds[2][2][T::kFloats];
    __shared__ Notices notices;
    const int lane = (int)threadIdx.x & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    uint32_t id = blockIdx.x;
    const int part = (int)(id % (uint32_t)a.splits);
    id /= (uint32_t)a.splits;
    const int tile = (int)(id % (uint32_t)a.row_tiles);
    id /= (uint32_t)a.row_tiles;
    const int hk = (int)(id % (uint32_t)a.kv_heads), b = (int)(id / (uint32_t)a.kv_heads);

    const Sequence seq = sequence_of(a, b);
    const int r0 = tile * kRowsBlock, r1 = min(r0 + kRowsBlock, a.rows);
    const int row = r0 + wave * 32 + (lane & 31);
    const bool live = row < a.rows;
    const int i = (int)a.by_group.divide((uint32_t)min(row, a.rows - 1)), g = min(row, a.rows - 1) - i * a.group;
    const int place = live ? seq.first + i : -1;
    // Places of the block's and of the wave's rows.
    const int block_lo = seq.first + (int)a.by_group.divide((uint32_t)r0);
    const int block_hi = seq.first + (int)a.by_group.divide((uint32_t)(r1 - 1));
    const int w0 = r0 + wave * 32, w1 = min(w0 + 32, a.rows);
    const int wave_lo = seq.first + (int)a.by_group.divide((uint32_t)min(w0, a.rows - 1));
    const int wave_hi = w0 < w1 ? seq.first + (int)a.by_group.divide((uint32_t)(w1 - 1)) : -1;
    // Key tiles: those of the sinks, then the window's.
    const int key_hi = block_hi, key_lo = max(0, block_lo - a.window + 1);
    const int sinks = min(a.sinks, key_hi + 1);
    const int first = key_lo / kTile;
    const int nsink = key_hi < 0 ? 0 : min((sinks + kTile - 1) / kTile, first);
    const int tiles = key_hi < 0 ? 0 : nsink + key_hi / kTile - first + 1;
    const int t0 = (int)((int64_t)tiles * part / a.splits), t1 = (int)((int64_t)tiles * (part + 1) / a.splits);
    const auto first_key = [&](int t) { return (t < nsink ? t : first + t - nsink) * kTile; };

    const float *kb = a.k + b * a.ks.b + hk * a.ks.h, *vb = a.v + b * a.vs.b + hk * a.vs.h;
    typename T::Regs kr, vr;
    const auto load = [&](int t) {
        const int j0 = first_key(t);
        // A key that no row of the block sees is not read.
        const auto seen = [&](int r) { return j0 + r <= key_hi && (j0 + r >= key_lo || j0 + r < sinks); };
        T::load(kr, a.D, [&](int r) { return seen(r) ? kb + (int64_t)(j0 + r) * a.ks.s : nullptr; });
        T::load(vr, a.D, [&](int r) { return seen(r) ? vb + (int64_t)(j0 + r) * a.vs.s : nullptr; });
    };
    const auto store = [&](int buf) {
        T::store(kr, lds[buf][0]);
        const bool bad = T::store(vr, lds[buf][1]);
        notices.word[buf][wave] = __builtin_amdgcn_ballot_w64(bad) != 0;
    };

    if (t0 < t1) load(t0);
    at_f4 qf[NT * 4];
    T::hold(qf, live ? a.q + b * a.qs.b + (int64_t)(hk * a.group + g) * a.qs.h + (int64_t)i * a.qs.s : nullptr, a.D, half, a.scale2);
    at_f16 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) acc[t] = (at_f16)(0.f);
    float most = -__builtin_inff(), sum = 0.f;
    if (t0 < t1) store(0);
    __syncthreads();
    for (int t = t0; t < t1; t++) {
        const int buf = (t - t0) & 1, j0 = first_key(t);
        if (t + 1 < t1) load(t + 1);
        // Whether a row of the wave sees a key of the tile, and whether all see all.
        const bool any = j0 <= wave_hi && (wave_lo - (j0 + kTile - 1) < a.window || j0 < a.sinks);
        if (any) {
            at_f16 s = T::times_held(lds[buf][0], qf, lane);
            const bool all = j0 + kTile - 1 <= wave_lo && (wave_hi - j0 < a.window || j0 + kTile <= a.sinks) && w1 - w0 == 32;
            if (!all) {
#pragma unroll
                for (int e = 0; e < 16; e++)
                    if (!sees(a, place, j0 + result_row(e, half))) s[e] = -__builtin_inff();
            }
            float m = s[0];
#pragma unroll
            for (int e = 1; e < 16; e++) m = __builtin_fmaxf(m, s[e]);
            m = __builtin_fmaxf(m, __shfl_xor(m, 32));
            const float now = __builtin_fmaxf(most, m);
            const float base = now == -__builtin_inff() ? 0.f : now;  // a row that sees nothing so far
            const float keep = __builtin_amdgcn_exp2f(most - base);
            float add = 0.f;
#pragma unroll
            for (int e = 0; e < 16; e++) {
                s[e] = __builtin_amdgcn_exp2f(s[e] - base);
                add += s[e];
            }
            sum = sum * keep + add;
            most = now;
            if (__builtin_amdgcn_ballot_w64(keep != 1.f)) {
#pragma unroll
                for (int c = 0; c < NT; c++) acc[c] *= keep;
            }
            const uint32_t bad = notices.word[buf][0] | notices.word[buf][1] | notices.word[buf][2] | notices.word[buf][3];
            if (__builtin_expect(__builtin_amdgcn_readfirstlane(bad) == 0, 1))
                T::add_product(acc, 0, lds[buf][1], s, lane);
            else
                T::add_product_seen(acc, 0, lds[buf][1], s, lane, [&](int k) { return sees(a, place, j0 + k); });
        }
        if (t + 1 < t1) store(buf ^ 1);
        __syncthreads();
    }
    sum += __shfl_xor(sum, 32);
    if (!live) return;
    const int64_t head = (int64_t)b * a.kv_heads + hk;
    if (a.splits > 1) {
        const int64_t at = ((int64_t)part * a.batch * a.kv_heads + head) * a.rows + row;
        T::write(acc, 0, a.part_o + at * a.D, 1.f, a.D, half);
        if (half == 0) a.part_ml[2 * at] = most, a.part_ml[2 * at + 1] = sum;
        return;
    }
    // A row that sees nothing gives 0 and a logarithm of -inf.
    const float f = sum == 0.f ? 0.f : 1.f / sum;
    const int64_t h = (int64_t)hk * a.group + g;
    T::write(acc, 0, a.out + b * a.os.b + h * a.os.h + (int64_t)i * a.os.s, f, a.D, half);
    if (a.lse && half == 0) a.lse[((int64_t)b * a.heads + h) * a.Sq + i] = (most + __builtin_amdgcn_logf(sum)) * kLn2;
}

// The parts of a row, joined: a wave a row.
__global__ void __launch_bounds__(256) attn_join(AttnArgs a) {
    const int lane = (int)threadIdx.x & 63;
    const int64_t rows = (int64_t)a.batch * a.kv_heads * a.rows;
    const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= rows) return;
    const int64_t head = r / a.rows;
    const int row = (int)(r - head * a.rows), b = (int)(head / a.kv_heads), hk = (int)(head - (int64_t)b * a.kv_heads);
    const int i = (int)a.by_group.divide((uint32_t)row);
    const int64_t h = (int64_t)hk * a.group + row - i * a.group;
    float most = -__builtin_inff(), sum = 0.f;
    for (int p = 0; p < a.splits; p++) most = __builtin_fmaxf(most, a.part_ml[2 * (p * rows + r)]);
    const float base = most == -__builtin_inff() ? 0.f : most;
    for (int p = 0; p < a.splits; p++) {
        const float *ml = a.part_ml + 2 * (p * rows + r);
        sum += ml[1] * __builtin_amdgcn_exp2f(ml[0] - base);
    }
    const float f = sum == 0.f ? 0.f : 1.f / sum;
    float *o = a.out + b * a.os.b + h * a.os.h + (int64_t)i * a.os.s;
    for (int d = lane; d < a.D; d += 64) {
        float v = 0.f;
        for (int p = 0; p < a.splits; p++) {
            const int64_t at = p * rows + r;
            v += a.part_o[at * a.D + d] * __builtin_amdgcn_exp2f(a.part_ml[2 * at] - base);
        }
        o[d] = v * f;
    }
    if (a.lse && lane == 0) a.lse[((int64_t)b * a.heads + h) * a.Sq + i] = (most + __builtin_amdgcn_logf(sum)) * kLn2;
}

}  // namespace

int attention_forward(AttnArgs a, hipStream_t s, int cu_count) {
    const int64_t heads = (int64_t)a.batch * a.kv_heads;
    const bool few = a.rows <= kFewRows;
    const int rows_block = few ? 16 : kRowsBlock, tile = few ? 16 : kTile, waves = few ? 4 : 1;
    a.row_tiles = (a.rows + rows_block - 1) / rows_block;
    // The keys in parts where the rows' blocks are fewer than the device takes.
    const int64_t blocks = heads * a.row_tiles, keys = std::min<int64_t>(a.Sk, (int64_t)a.window + a.sinks + rows_block / std::max(a.group, 1));
    const int64_t most = std::max<int64_t>(1, keys / tile / waves / kPartTiles);
    a.splits = (int32_t)std::max<int64_t>(1, std::min<int64_t>({most, (4 * (int64_t)cu_count + blocks - 1) / blocks, 64}));
    if ((blocks * a.splits) >> 31) return set_error(TRS_E_INVALID_ARGUMENT, "attention over %lld blocks of rows", (long long)blocks);
    void *ws = nullptr;
    if (a.splits > 1) {
        const int64_t parts = a.splits * heads * a.rows;
        const int rc = trs_alloc((size_t)(parts * (a.D + 2)) * sizeof(float), &ws);
        if (rc == TRS_E_ALLOCATION_FAILED) a.splits = 1;  // the parts are for speed alone
        else if (rc) return rc;
        a.part_ml = (float *)ws, a.part_o = a.part_ml + 2 * parts;
    }
    const auto launch = [&]() -> int {
        const dim3 grid((unsigned)(blocks * a.splits));
        if (few) TRS_CHECK(launch_attention_few(a, s));
        else if (a.D <= 32) hipLaunchKernelGGL(attn_rows<1>, grid, dim3(256), 0, s, a);
        else if (a.D <= 64) hipLaunchKernelGGL(attn_rows<2>, grid, dim3(256), 0, s, a);
        else if (a.D <= 96) hipLaunchKernelGGL(attn_rows<3>, grid, dim3(256), 0, s, a);
        else if (a.D <= 128) hipLaunchKernelGGL(attn_rows<4>, grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL(attn_rows<8>, grid, dim3(256), 0, s, a);
        TRS_LAUNCH_CHECK("attention launch");
        if (a.splits > 1) {
            hipLaunchKernelGGL(attn_join, dim3((unsigned)((heads * a.rows + 3) / 4)), dim3(256), 0, s, a);
            TRS_LAUNCH_CHECK("attention join launch");
        }
        return TRS_OK;
    };
    const int rc = launch(), frc = ws ? trs_free(ws) : TRS_OK;
    return rc ? rc : frc;
}

}  // namespace trs
