// attention_forward.hip -- the output of attention.h's attention.
#include <hip/hip_runtime.h>

#include "attention.h"

namespace trs {

namespace {

// Rows a key head that attn_few takes; of more than 128 dims it takes any.  4000 keys, few / this
// kernel, us: 1 head of 128, 64 rows 24 / 42, 512 39 / 48; 8 heads 32 rows 30 / 36, 64 42 / 38;
// 64 heads 32 rows 69 / 140, 64 116 / 143, 96 176 / 149.
constexpr int kFewRows = 64;
constexpr int kPartTiles = 2, kMostParts = 64;  // the least key tiles of a part, a wave; the most parts
constexpr int kForwardRows = 256;               // rows of a block, 32 a wave

// A row of the softmax so far: maximum and sum are of base-2 exponents, log2(e)
// going into the queries with the scale.  A lane holds its row's sum over half of
// the keys (its other half the rest).
template <int NT>
struct RowState {
    at_f16 acc[NT];
    float most, sum;
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int t = 0; t < NT; t++) acc[t] = (at_f16)(0.f);
        most = -__builtin_inff(), sum = 0.f;
    }
    // A tile's scores become its weights: s is S^T / unit, -inf where hidden.  The
    // maximum is kept in the units of s.
    __device__ __forceinline__ void weigh(at_f16 &s, float unit) {
        float m = s[0];
#pragma unroll
        for (int e = 1; e < 16; e++) m = __builtin_fmaxf(m, s[e]);
        m = __builtin_fmaxf(m, __shfl_xor(m, 32));
        const float now = __builtin_fmaxf(most, m);
        const float base = now == -__builtin_inff() ? 0.f : now;  // a row that sees nothing so far
        const float keep = __builtin_amdgcn_exp2f((most - base) * unit);
        float add[2] = {0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 16; e++) {
            s[e] = __builtin_amdgcn_exp2f((s[e] - base) * unit);
            add[e & 1] += s[e];
        }
        sum = sum * keep + (add[0] + add[1]);
        most = now;
        if (__builtin_amdgcn_ballot_w64(keep != 1.f)) {
#pragma unroll
            for (int c = 0; c < NT; c++) acc[c] *= keep;
        }
    }
};

// The rows of a block over its key tiles t0 to t1 on the fp32 matrix instruction,
// whatever the values: a tile at a time staged in LDS, few registers.  S^T = K Q^T puts a
// row of the softmax in a lane (and its other half), and P^T is the operand of
// O^T += V^T P^T as it stands.
template <int NT, int NW>
__device__ __forceinline__ void rows_fp32(const AttnArgs &a, const RowBlock<NW> &r, int t0, int t1, float *lds, RowState<NT> &state) {
    using T = Tile<NT, 64 * NW>;
    const float *kb = a.k + r.b * a.ks.b + r.hk * a.ks.h, *vb = a.v + r.b * a.vs.b + r.hk * a.vs.h;
    const float *q = r.place >= 0 ? a.q + r.at(a, a.qs) : nullptr;
    state.clear();
#pragma unroll 1
    for (int t = t0; t < t1; t++) {
        const int j0 = r.first_key(t);
        // A key that no row of the block sees is not read.
        T::stage(lds, a.D, [&](int k) { return r.read(j0 + k) ? kb + (int64_t)(j0 + k) * a.ks.s : nullptr; });
        T::stage(lds + T::kFloats, a.D, [&](int k) { return r.read(j0 + k) ? vb + (int64_t)(j0 + k) * a.vs.s : nullptr; });
        __syncthreads();
        if (r.any(a, j0)) {
            at_f16 s = T::times_row(lds, q, a.D, a.scale2, r.lane);
#pragma unroll
            for (int e = 0; e < 16; e++) s[e] = sees(a, r.place, j0 + result_row(e, r.half)) ? s[e] : -__builtin_inff();
            state.weigh(s, 1.f);
            T::add_product_seen(state.acc, lds + T::kFloats, s, r.lane, [&](int k) { return sees(a, r.place, j0 + k); });
        }
        __syncthreads();
    }
}

// The rows' outputs, or the part's (of several), through write(row, factor).  `unit`: of
// the maximum.
template <int NT, int NW, class Write>
__device__ __forceinline__ void write_rows(const AttnArgs &a, const RowBlock<NW> &r, int part, int parts, RowState<NT> &state, float unit,
                                           Write &&write) {
    const float sum = state.sum + __shfl_xor(state.sum, 32), most = state.most * unit;
    if (r.row >= a.rows) return;
    if (parts > 1) {
        const int64_t at = (((int64_t)part * a.batch + r.b) * a.kv_heads + r.hk) * a.rows + r.row;
        write(a.part_o + at * a.part_width, 1.f);
        if (r.half == 0) a.part_ml[2 * at] = most, a.part_ml[2 * at + 1] = sum;
        return;
    }
    // A row that sees nothing gives 0 and a logarithm of -inf; one whose scores are all -inf,
    // NaN, as the formula does.
    write(a.out + r.at(a, a.os), r.place < 0 ? 0.f : 1.f / sum);
    if (a.lse && r.half == 0) a.lse[r.index(a)] = log_sum(most, sum);
}

// The key tiles of tile t of kForwardRows rows in the longest sequence that may be.
__host__ __device__ __forceinline__ KeyTiles<5> longest(const AttnArgs &a, int t) {
    const int r0 = t * kForwardRows, r1 = r0 + kForwardRows;
    return KeyTiles<5>(a, Sequence{a.Sk, a.Sk - a.Sq}, r0, r1 < a.rows ? r1 : a.rows);
}

// The parts of tile t of a sequence's rows, which see the tiles `keys`.  Where a shorter
// sequence's window begins elsewhere in a tile it may touch one tile more than the longest's:
// it still has no more parts than the longest has, for which blocks are launched.
__device__ __forceinline__ int parts_of(const AttnArgs &a, const KeyTiles<5> &keys, int t) {
    return min(keys.parts(a), longest(a, t).parts(a));
}

// Of the parts of a key head's tiles of rows, in that order, number n: every lane counts a
// tile's.
__device__ __forceinline__ void find_part(const AttnArgs &a, int n, int lane, int &tile, int &part) {
    tile = part = 0;
    for (int t0 = 0; t0 < a.row_tiles; t0 += 64) {
        int sum = t0 + lane < a.row_tiles ? longest(a, t0 + lane).parts(a) : 0;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int before = __shfl_up(sum, d);
            sum += lane >= d ? before : 0;
        }
        const int all = __builtin_amdgcn_readlane(sum, 63);
        if (n < all) {
            const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(sum > n));
            tile = t0 + l, part = l ? n - __builtin_amdgcn_readlane(sum, l - 1) : n;
            return;
        }
        n -= all;
    }
}

// 32 NW rows of a key head on the bf16 matrix cores, in pieces: the block splits a key tile once for
// its waves, into one of two LDS buffers while it computes from the other; the loads from
// memory are a tile further ahead.  Bound by the card's power and, behind it, by issue: prompt
// of 4096 tokens, 32 heads of 128 over 8, window 1024, 328-342 us by card, up to 1.16 PFLOP/s
// of bf16 products (of a large product 1.24): the matrix cores are busy for 51% of the cycles, at a
// clock of 2.0 GHz of 2.4, and the other vector instructions, 4.4 a matrix instruction, issue in 28%.
// Blocks of four waves, which split every tile for half the rows, take 427.
template <int NT, int NW, int WIDTH>
__global__ void __launch_bounds__(64 * NW, 2) attn_rows(AttnArgs a) {
    using T = Tile<NT, 64 * NW>;
    constexpr int UNITS = 4 * NT, OWN = (UNITS + NW - 1) / NW;  // of keys and values; of a wave (some twice)
    constexpr int kBuffer = 3 * UNITS * 1024, kBytes = 2 * kBuffer;
    static_assert(kBytes >= 8 * T::kFloats, "the fp32 tiles fit the pieces' LDS");
    __shared__ __attribute__((aligned(1024))) char lds[kBytes];
    __shared__ Notices<NW> notices;
    // Heads first: the chip's parts with an L2 each take them in turn, and so read the fewer
    // keys twice (prompt of 4096 tokens, 32 heads of 128, 8 key heads, window 1024: 339 us with
    // the tiles first, 333 so).  Then the rows' tiles, the last ones, which see the most keys,
    // first; then batches.
    const uint32_t heads = (uint32_t)a.kv_heads * (a.splits > 1 ? (uint32_t)a.batch : 1u);
    const uint32_t head = blockIdx.x % heads, rest = blockIdx.x / heads;
    int part = 0, tile, batch;
    if (a.splits > 1) {
        batch = (int)(head / (uint32_t)a.kv_heads);
        find_part(a, (int)rest, (int)threadIdx.x & 63, tile, part);
    } else {
        tile = a.row_tiles - 1 - (int)(rest % (uint32_t)a.row_tiles), batch = (int)(rest / (uint32_t)a.row_tiles);
    }
    const RowBlock<NW> r(a, (int)(head % (uint32_t)a.kv_heads), tile, batch);
    const int parts = parts_of(a, r, tile);
    if (part >= parts) return;
    const int t0 = (int)((int64_t)r.tiles * part / parts), t1 = (int)((int64_t)r.tiles * (part + 1) / parts);
    const float *kb = a.k + r.b * a.ks.b + r.hk * a.ks.h, *vb = a.v + r.b * a.vs.b + r.hk * a.vs.h;
    Unit<WIDTH> in[OWN];
    const auto unit = [&](int q) { return min(r.wave + q * NW, UNITS - 1); };
    const auto load = [&](int t) {  // past the part's last tile: that one
        const int j = min(r.first_key(min(t, t1 - 1)) + (r.lane & 31), r.key_hi);
        const float *kp = kb + (int64_t)j * a.ks.s, *vp = vb + (int64_t)j * a.vs.s;
#pragma unroll
        for (int q = 0; q < OWN; q++) {
            const bool key = unit(q) < UNITS / 2;
            in[q].load(key ? kp : vp, key ? unit(q) : unit(q) - UNITS / 2, a.D, r.lane);
        }
    };
    RowState<NT> state;
    state.clear();
    if (t0 < t1) {
        Lowest lowest;
        load(t0);
        Pieces q[2 * NT];
#pragma unroll
        for (int s = 0; s < 2 * NT; s++) {
            Unit<WIDTH> x;
            x.load(a.q + r.at(a, a.qs), s, a.D, r.lane, s < 2 * NT - 2);
            q[s] = x.split(r.place >= 0 ? a.scale2 * kUp : 0.f);
        }
#pragma unroll
        for (int n = 0; n < OWN; n++) in[n].template store<UNITS>(lds, unit(n), r.lane);
        load(t0 + 1);
#pragma unroll 1
        for (int t = t0; t < t1; t++) {
            const int j0 = r.first_key(t);
            char *const buf = lds + ((t - t0) & 1) * kBuffer, *const other = lds + ((t - t0) & 1 ? 0 : kBuffer);
            __syncthreads();
            Splitting x;
            const auto stage = [&](int i) { in[i / 4].template store_pair<UNITS>(x, i % 4, other, unit(i / 4), r.lane); };
            if (!r.any(a, j0)) {  // no row of the wave sees the tile
#pragma unroll
                for (int i = 0; i < 4 * OWN; i++) stage(i);
                load(t + 2);
                continue;
            }
            at_f16 s = (at_f16)(0.f);
            {
                const auto read = [&](int n) { return along<UNITS>(buf, n, r.lane); };
                Pieces f = read(0);
                steps<2 * NT>(
                    f, read, [&](int n, const Pieces &now) { mfma_pieces(s, now, q[n]); }, [&](int n) { dealt(4 * OWN, n, 2 * NT, stage); },
                    [](Pieces &) {});
            }
            load(t + 2);
            lowest.add(s);
            if (!r.all(a, j0)) {
#pragma unroll
                for (int e = 0; e < 16; e++) s[e] = sees(a, r.place, j0 + result_row(e, r.half)) ? s[e] : -__builtin_inff();
            }
            state.weigh(s, kDown2);
            {
                const auto read = [&](int n) { return across<UNITS>(buf, 2 * NT + 2 * (n % NT), n / NT, r.lane); };
                Pieces f = read(0);
                Splitting w;
#pragma unroll
                for (int i = 0; i < 4; i++) w.pair(i, s[2 * i], s[2 * i + 1]);
                const Pieces p0 = w.done();
                steps<NT>(
                    f, read, [&](int n, const Pieces &now) { mfma_pieces(state.acc[n], now, p0); },
                    [&](int n) { dealt(4, n, NT, [&](int i) { w.pair(i, s[8 + 2 * i], s[9 + 2 * i]); }); },
                    [&](Pieces &y) { y = read(NT); });
                const Pieces p1 = w.done();
                steps<NT>(
                    f, [&](int n) { return read(NT + n); }, [&](int n, const Pieces &now) { mfma_pieces(state.acc[n], now, p1); }, [](int) {},
                    [](Pieces &) {});
            }
        }
        __syncthreads();
        notices.word[0][r.wave] = not_finite(state.acc, state.sum) || lowest.infinite();
        __syncthreads();
        if (__builtin_expect(notices.any(0), 0)) {
            __syncthreads();
            rows_fp32<NT, NW>(a, r, t0, t1, (float *)lds, state);
            write_rows(a, r, part, parts, state, 1.f, [&](float *p, float f) { T::write(state.acc, p, f, a.D, r.half); });
            return;
        }
    }
    write_rows(a, r, part, parts, state, kDown2, [&](float *p, float f) { write_row<WIDTH>(state.acc, p, kDown, f, a.D, r.half); });
}

// The parts of a row, joined: four columns a lane.  Every part is read before the
// first is added, up to eight: one memory latency, not one a part.  3 to 6 us, of which most is
// the launch behind another.
template <bool FEW>
__global__ void __launch_bounds__(256) attn_join(AttnArgs a) {
    const int64_t rows = (int64_t)a.batch * a.kv_heads * a.rows;
    const uint32_t quads = (uint32_t)a.part_width / 4;
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x, r = e / quads;
    if (r >= rows) return;
    const int d = (int)(e - r * quads) * 4;
    const int64_t head = r / a.rows;
    const int row = (int)(r - head * a.rows), b = (int)(head / a.kv_heads), hk = (int)(head - (int64_t)b * a.kv_heads);
    const int i = (int)a.by_group.divide((uint32_t)row);
    const int64_t h = (int64_t)hk * a.group + row - i * a.group;
    int parts = a.splits;
    if constexpr (!FEW) {
        const int t = row / kForwardRows, r0 = t * kForwardRows;
        parts = parts_of(a, KeyTiles<5>(a, sequence_of(a, b), r0, min(r0 + kForwardRows, a.rows)), t);
        if (parts == 1) return;  // its block wrote it
    }
    float most = -__builtin_inff(), sum = 0.f;
    at_f4 o = (at_f4)(0.f);
    for (int p0 = 0; p0 < parts; p0 += 8) {
        float m[8], l[8];
        at_f4 x[8];
#pragma unroll
        for (int p = 0; p < 8; p++) {
            const int64_t at = min(p0 + p, parts - 1) * rows + r;
            m[p] = a.part_ml[2 * at], l[p] = a.part_ml[2 * at + 1];
            x[p] = *(const at_f4 *)(a.part_o + at * a.part_width + d);
        }
        float now = most;
#pragma unroll
        for (int p = 0; p < 8; p++) now = __builtin_fmaxf(now, m[p]);
        const float base = now == -__builtin_inff() ? 0.f : now, keep = __builtin_amdgcn_exp2f(most - base);
        sum *= keep, o *= keep, most = now;
#pragma unroll
        for (int p = 0; p < 8; p++) {
            if (p0 + p >= parts) break;
            const float f = __builtin_amdgcn_exp2f(m[p] - base);
            sum += l[p] * f, o += x[p] * f;
        }
    }
    o *= sequence_of(a, b).first + i < 0 ? 0.f : 1.f / sum;
    float *out = a.out + b * a.os.b + h * a.os.h + (int64_t)i * a.os.s + d;
#pragma unroll
    for (int q = 0; q < 4; q++)
        if (d + q < a.D) out[q] = o[q];
    if (a.lse && d == 0) a.lse[((int64_t)b * a.heads + h) * a.Sq + i] = log_sum(most, sum);
}

template <int NT>
void launch_rows(const AttnArgs &a, dim3 grid, hipStream_t s) {
    constexpr int NW = kForwardRows / 32;
    const dim3 block(64 * NW);
    if (a.D == 32 * NT) hipLaunchKernelGGL((attn_rows<NT, NW, 4>), grid, block, 0, s, a);
    else if (a.D % 4 == 0) hipLaunchKernelGGL((attn_rows<NT, NW, 2>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((attn_rows<NT, NW, 1>), grid, block, 0, s, a);
}

// Parts of about as many key tiles in all blocks of rows, which see from few keys to all: the
// shortest of which there are at most `want`, so that the chip holds all of them at once.
// Returns how many a key head has.  Lengths are not known here: every sequence counts as the
// longest, and in shorter ones a block's last parts have nothing to do.  (As many parts in
// every block, us / so, causal: 32 heads of 128 over 8, 768 tokens 69 / 50, 1024 88 / 71; 8 heads of
// 128, 2048 tokens 86 / 68; 32 heads, 300 tokens 30 / 34; 3 x 1000 tokens, 6 heads of 80, window
// 200 35 / 31.)
int64_t choose_parts(AttnArgs &a, int64_t heads, int64_t want) {
    a.splits = 1, a.part_tiles = INT32_MAX;
    want /= heads;
    if (a.row_tiles >= want) return a.row_tiles;
    int most = 0;
    for (int t = 0; t < a.row_tiles; t++) most = std::max(most, longest(a, t).tiles);
    const auto parts = [&](int length) {
        a.part_tiles = length, a.splits = std::max(1, (most + length - 1) / length);
        int64_t n = 0;
        for (int t = 0; t < a.row_tiles; t++) n += longest(a, t).parts(a);
        return n;
    };
    int lo = std::max(kPartTiles, (most + kMostParts - 1) / kMostParts), hi = std::max(most, lo);  // parts as long as `hi` are few enough
    while (lo < hi) {
        const int mid = lo + (hi - lo) / 2;
        if (parts(mid) <= want) hi = mid;
        else lo = mid + 1;
    }
    return parts(lo);
}

}  // namespace

int attention_forward(AttnArgs a, hipStream_t s, int cu_count) {
    const int64_t heads = (int64_t)a.batch * a.kv_heads;
    const bool few = a.rows <= kFewRows || a.D > kPiecesDim;
    // The keys in parts where the rows' blocks leave CUs without one.
    int64_t blocks;
    if (few) {
        a.row_tiles = (a.rows + 15) / 16;
        const int64_t rows = heads * a.row_tiles, keys = std::min<int64_t>(a.Sk, (int64_t)a.window + a.sinks + 16 / std::max(a.group, 1));
        a.splits = (int32_t)std::max<int64_t>(1, std::min<int64_t>({keys / 16 / 4 / kPartTiles, 4 * (int64_t)cu_count / rows, kMostParts}));
        // Where blocks of 16 waves (8 above 64 dims, for their registers) do what the parts would, the
        // second launch is saved.  One of them fills a CU: so where one round of them takes all CUs and the
        // sequences are alike, or where the keys are few.  us in parts / so: 8 heads of 64, 260 keys
        // 12.2 / 9.3, 383 11.9 / 11.0, 520 10.8 / 11.9; 8 of 128, 300 keys 12.4 / 13.4; 256 of 64, 1000 keys
        // 26.7 / 23.0; 256 of 128, 300 20.5 / 16.3, 4000 182 / 178; 128 of 128, 2000 55 / 60; 384 of
        // 128, 1000 72 / 77.
        const bool full = 8 * rows >= 7 * (int64_t)cu_count && a.D <= kPiecesDim && !a.lengths;
        const bool whole = a.splits > 1 && rows <= cu_count && a.D % 4 == 0 && (full || (a.splits == 2 && a.D <= 64));
        a.few_waves = !whole ? 4 : a.D <= 64 ? 16 : 8;
        if (whole) a.splits = 1;
        blocks = rows * a.splits;
    } else {
        a.row_tiles = (a.rows + kForwardRows - 1) / kForwardRows;
        blocks = heads * choose_parts(a, heads, cu_count);
    }
    if (blocks * (few ? 64 * a.few_waves : 2 * kForwardRows) >> 32)  // a launch has fewer lanes
        return set_error(TRS_E_INVALID_ARGUMENT, "attention over %lld blocks of rows", (long long)blocks);
    a.part_width = (a.D + 3) / 4 * 4;
    const int64_t parts = a.splits * heads * a.rows, join_blocks = (heads * a.rows * (a.part_width / 4) + 255) / 256;
    void *ws = nullptr;
    if (a.splits > 1) {
        const int rc = trs_alloc((size_t)(parts * (a.part_width + 2)) * sizeof(float), &ws);
        if (rc == TRS_E_ALLOCATION_FAILED) a.splits = 1, blocks = heads * a.row_tiles;  // the parts are for speed alone
        else if (rc) return rc;
        a.part_o = (float *)ws, a.part_ml = a.part_o + parts * a.part_width;
    }
    const auto launch = [&]() -> int {
        const dim3 grid((unsigned)blocks);
        if (few) TRS_CHECK(launch_attention_few(a, grid, s));
        else if (a.D <= 32) launch_rows<1>(a, grid, s);
        else if (a.D <= 64) launch_rows<2>(a, grid, s);
        else if (a.D <= 96) launch_rows<3>(a, grid, s);
        else launch_rows<4>(a, grid, s);
        TRS_LAUNCH_CHECK("attention launch");
        if (a.splits > 1) {
            const dim3 joins((unsigned)join_blocks);
            if (few) hipLaunchKernelGGL(attn_join<true>, joins, dim3(256), 0, s, a);
            else hipLaunchKernelGGL(attn_join<false>, joins, dim3(256), 0, s, a);
            TRS_LAUNCH_CHECK("attention join launch");
        }
        return TRS_OK;
    };
    const int rc = launch(), frc = ws ? trs_free(ws) : TRS_OK;
    return rc ? rc : frc;
}

}  // namespace trs
