// paged_few.hip -- attention over a cache in pages for few rows: single tokens of a batch.
//
// Bound by reading the keys and values once.  A wave takes 16 rows and streams its share
// of the keys straight from the pages into the registers that the matrix instructions take
// them from: no LDS, no barrier, nothing that waits for another wave.  The waves of a block
// join their maxima and sums in LDS; what several blocks have of an entry is joined by a second
// launch.
//
// float32 pages: tiles of 16 keys on v_mfma_f32_16x16x4_f32, as attention_wide.h has them.
// bfloat16 pages: tiles of 32 keys on v_mfma_f32_16x16x32_bf16.  A key is an operand as it
// stands in memory; queries and weights go in as the exact sums of three bf16 pieces, three
// products where float32 pages would take six.  Lane l holds of an operand row (column)
// l % 16 at k = 8 (l/16) + e, of a result column l % 16, register i row 4 (l/16) + i.  The
// scores' registers are the operand of the second product as they stand: its k in lane
// quarter q are keys 4 q + e of the tile's first half and of its second, and of these eight
// keys a lane reads W consecutive columns each, which v_perm_b32 turns into W columns of
// eight keys.
#include <hip/hip_runtime.h>

#include "attention_wide.h"
#include "paged_attention.h"

namespace trs {

namespace {

typedef uint32_t U2 __attribute__((ext_vector_type(2)));
typedef uint32_t U4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4, kTileRows = 16;

// DP: the width, padded.  MODE 0: D is DP; 1: rows are read in vectors; 2: entry by entry.
template <int DP, int MODE>
struct FloatPages {
    using E = float;
    using T = Wide<DP, MODE>;
    static constexpr int kShift = 4, kHalves = 1, kTiles = T::TO;
    static constexpr float kDownScale = 1.f;
    typename T::Along q, k;
    typename T::Across v;

    __device__ __forceinline__ void load_q(const float *row, int D, int quarter, float scale) {
        T::load(q, row, D, quarter);
#pragma unroll
        for (int j = 0; j < T::KJ; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) q[j][e] *= scale;
    }
    // row(h, n): key n of half h.
    template <class Row>
    __device__ __forceinline__ void load_k(Row &&row, int D, int col, int quarter) {
        T::load(k, row(0, col), D, quarter);
    }
    template <class Row>
    __device__ __forceinline__ void load_v(Row &&row, int D, int col, int quarter) {
        T::load(v, [&](int n) { return row(0, 4 * quarter + n); }, D, col);
    }
    __device__ __forceinline__ void scores(at_f4 (&s)[1]) const {
        s[0] = (at_f4)(0.f);
        T::product(s[0], k, q);
    }
    __device__ __forceinline__ void add(at_f4 (&acc)[kTiles], const at_f4 (&p)[1]) const { T::add(acc, v, p[0]); }
    __device__ __forceinline__ static int column(int t, int i, int quarter) { return T::column(t, i, quarter); }
};

template <int DP, int MODE>
struct Bf16Pages {
    using E = uint16_t;
    static constexpr int kShift = 5, kHalves = 2, KJ = DP / 32, W = DP >= 128 ? 8 : DP / 16, VU = DP / (16 * W), kTiles = DP / 16;
    static constexpr float kDownScale = kDown;
    gt_bf8 q[3][KJ];
    U4 k[2][KJ];
    uint32_t v[8][VU][W / 2];

    // N entries of a row from column c on, in words; columns from D on are 0.
    template <int N>
    __device__ __forceinline__ static void take(uint32_t *o, const E *row, int c, int D) {
        if constexpr (MODE == 2) {
#pragma unroll
            for (int e = 0; e < N; e += 2) {
                const bool in0 = c + e < D, in1 = c + e + 1 < D;
                const uint32_t x = row[in0 ? c + e : 0], y = row[in1 ? c + e + 1 : 0];
                o[e / 2] = (in0 ? x : 0) | (in1 ? y << 16 : 0);
            }
        } else {
            typedef uint32_t Vec __attribute__((ext_vector_type(N / 2)));
            const bool in = MODE == 0 || c < D;
            const Vec x = *(const Vec *)(row + (in ? c : 0));
#pragma unroll
            for (int e = 0; e < N / 2; e++) o[e] = in ? x[e] : 0;
        }
    }
    __device__ __forceinline__ void load_q(const float *row, int D, int quarter, float scale) {
#pragma unroll
        for (int j = 0; j < KJ; j++) {
            Unit<1> x;
            const int c = 32 * j + 8 * quarter;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const bool in = MODE == 0 || c + e < D;
                const float y = row[in ? c + e : 0];
                x.v[e] = in ? y : 0.f;
            }
            const Pieces p = x.split(scale * kUp);
#pragma unroll
            for (int i = 0; i < 3; i++) q[i][j] = p.p[i];
        }
    }
    template <class Row>
    __device__ __forceinline__ void load_k(Row &&row, int D, int col, int quarter) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const E *p = row(h, col);
#pragma unroll
            for (int j = 0; j < KJ; j++) {
                uint32_t x[4];
                take<8>(x, p, 32 * j + 8 * quarter, D);
                k[h][j] = U4{x[0], x[1], x[2], x[3]};
            }
        }
    }
    template <class Row>
    __device__ __forceinline__ void load_v(Row &&row, int D, int col, int quarter) {
#pragma unroll
        for (int n = 0; n < 8; n++) {
            const E *p = row(n >> 2, 4 * quarter + (n & 3));
#pragma unroll
            for (int u = 0; u < VU; u++) take<W>(v[n][u], p, 16 * W * u + W * col, D);
        }
    }
    __device__ __forceinline__ void scores(at_f4 (&s)[2]) const {
#pragma unroll
        for (int h = 0; h < 2; h++) s[h] = (at_f4)(0.f);
#pragma unroll
        for (int i = 2; i >= 0; i--)
#pragma unroll
            for (int j = 0; j < KJ; j++)
#pragma unroll
                for (int h = 0; h < 2; h++) s[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(gt_bf8, k[h][j]), q[i][j], s[h], 0, 0, 0);
    }
    __device__ __forceinline__ void add(at_f4 (&acc)[kTiles], const at_f4 (&p)[2]) const {
        Splitting w;
#pragma unroll
        for (int i = 0; i < 4; i++) w.pair(i, p[i >> 1][2 * (i & 1)], p[i >> 1][2 * (i & 1) + 1]);
        const Pieces x = w.done();
#pragma unroll
        for (int u = 0; u < VU; u++)
#pragma unroll
            for (int e = 0; e < W; e++) {
                // Column e of the lane's W, of eight keys.
                U4 c;
#pragma unroll
                for (int n = 0; n < 4; n++)
                    c[n] = __builtin_amdgcn_perm(v[2 * n + 1][u][e >> 1], v[2 * n][u][e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
                for (int i = 2; i >= 0; i--)
                    acc[u * W + e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(gt_bf8, c), x.p[i], acc[u * W + e], 0, 0, 0);
            }
    }
    __device__ __forceinline__ static int column(int t, int i, int quarter) { return 16 * W * (t / W) + W * (4 * quarter + i) + t % W; }
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }

// Of a tile's keys: where they stand.
template <class E, int HALVES, bool ONE>
struct Places {
    const E *k[HALVES], *v[HALVES];  // ONE: of the half's first key
    int last[HALVES];                // ONE: its last key that is read
    bool held[HALVES];
};

// ONE: pages hold a multiple of 16 tokens, and no 16 keys are the first sequence's in part, so that a
// half's keys stand in one page, and its entry of the table is read by the scalar unit.
template <class T, bool ONE>
__device__ __forceinline__ void few_rows(const PagedArgs &a, const PagedStage &s, int hk, int w, float (&out_o)[kWaves][kTileRows][T::kTiles * 16 + 4],
                                         float (&out_ml)[kWaves][kTileRows][2]) {
    using E = typename T::E;
    constexpr int H = T::kHalves;
    const int lane = (int)threadIdx.x & 63, col = lane & 15, quarter = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const E *const kb = (const E *)a.pages.k + hk * a.pages.ks.h, *const vb = (const E *)a.pages.v + hk * a.pages.vs.h;
    for (PagedShare<T::kShift> share(a, s, w, lane); share.more();) {
        const int entry = share.entry;
        const PagedKeys<T::kShift> keys = share.keys(entry);
        const int tiles = max(keys.tiles, 1);
        const int ta = (int)(share.pos - share.before), tb = (int)min((int64_t)tiles, share.end - share.before);
        const int64_t before = share.before;
        const PagedRow row(a, s, entry, hk, col);
        const int owner = s.together ? 0 : entry / s.row_tiles;  // the sequence whose keys these are
        const int n = keys.tiles ? tb - ta : 0;
        const int t0 = ta + n * wave / kWaves, t1 = ta + n * (wave + 1) / kWaves;

        const int first_row_to = s.from < a.shared ? a.shared : 0;  // keys below it are the first sequence's
        const auto page_at = [&](int j) { return a.pages.page_of(j < first_row_to ? 0 : owner, j); };
        // A key that is not read: the last one that is seen stands for it.
        const auto places = [&](int t, Places<E, H, ONE> &p) {
            const int j0 = keys.first_key(min(t, t1 - 1));
#pragma unroll
            for (int h = 0; h < H; h++) {
                if constexpr (ONE) {
                    const int at = min(j0 + 16 * h, keys.last & ~15), id = page_at(at), slot = a.pages.slot_of(at);
                    p.held[h] = a.pages.holds(id);
                    const int64_t page = p.held[h] ? id : 0;
                    p.k[h] = kb + page * a.pages.ks.p + slot * a.pages.ks.s;
                    p.v[h] = vb + page * a.pages.vs.p + slot * a.pages.vs.s;
                    p.last[h] = min(keys.last - at, 15);
                }
            }
        };
        const auto any_place = [&](int j, bool &held, int64_t &page, int &slot) {
            const int at = min(j, keys.last), id = page_at(at);
            held = a.pages.holds(id);
            page = held ? id : 0, slot = a.pages.slot_of(at);
        };
        const auto k_row = [&](int t, const Places<E, H, ONE> &p, int h, int x) -> const E * {
            if constexpr (ONE) return p.k[h] + (int64_t)min(x, p.last[h]) * a.pages.ks.s;
            bool held;
            int64_t page;
            int slot;
            any_place(keys.first_key(min(t, t1 - 1)) + 16 * h + x, held, page, slot);
            return kb + page * a.pages.ks.p + slot * a.pages.ks.s;
        };
        const auto v_row = [&](int t, const Places<E, H, ONE> &p, int h, int x) -> const E * {
            if constexpr (ONE) return p.v[h] + (int64_t)min(x, p.last[h]) * a.pages.vs.s;
            bool held;
            int64_t page;
            int slot;
            any_place(keys.first_key(min(t, t1 - 1)) + 16 * h + x, held, page, slot);
            return vb + page * a.pages.vs.p + slot * a.pages.vs.s;
        };

        at_f4 acc[T::kTiles];
#pragma unroll
        for (int t = 0; t < T::kTiles; t++) acc[t] = (at_f4)(0.f);
        float most = -__builtin_inff(), sum = 0.f;
        if (t0 < t1) {
            T ops;
            Places<E, H, ONE> now, next;
            places(t0, now);
            ops.load_k([&](int h, int x) { return k_row(t0, now, h, x); }, a.D, col, quarter);
            ops.load_v([&](int h, int x) { return v_row(t0, now, h, x); }, a.D, col, quarter);
            ops.load_q(a.q + row.at(a.qs), a.D, quarter, a.scale2);
            places(t0 + 1, next);
            uint32_t lowest = 0;
            for (int t = t0; t < t1; t++) {
                const int j0 = keys.first_key(t);
                at_f4 x[H];
                ops.scores(x);
                ops.load_k([&](int h, int y) { return k_row(t + 1, next, h, y); }, a.D, col, quarter);
                float m = -__builtin_inff();
#pragma unroll
                for (int h = 0; h < H; h++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int j = j0 + 16 * h + 4 * quarter + e;
                        const uint32_t bits = __float_as_uint(x[h][e]);
                        lowest = lowest > bits ? lowest : bits;
                        bool held = true;
                        if constexpr (ONE) held = now.held[h];
                        else held = a.pages.holds(page_at(min(j, keys.last)));
                        const float y = held ? x[h][e] * T::kDownScale : __builtin_nanf("");
                        x[h][e] = row.sees(a, s, j) ? y : -__builtin_inff();
                        m = __builtin_fmaxf(m, x[h][e]);
                    }
                m = __builtin_fmaxf(m, __shfl_xor(m, 16));
                m = __builtin_fmaxf(m, __shfl_xor(m, 32));
                const float top = __builtin_fmaxf(most, m), base = top == -__builtin_inff() ? 0.f : top;
                const float keep = __builtin_amdgcn_exp2f(most - base);
                float add = 0.f;
#pragma unroll
                for (int h = 0; h < H; h++) {
#pragma unroll
                    for (int e = 0; e < 4; e++) x[h][e] = __builtin_amdgcn_exp2f(x[h][e] - base);
                    add += (x[h][0] + x[h][1]) + (x[h][2] + x[h][3]);
                }
                sum = sum * keep + add;
                most = top;
                if (__builtin_amdgcn_ballot_w64(keep != 1.f)) {
#pragma unroll
                    for (int c = 0; c < T::kTiles; c++) acc[c] *= keep;
                }
                ops.add(acc, x);
                ops.load_v([&](int h, int y) { return v_row(t + 1, next, h, y); }, a.D, col, quarter);
                now = next;
                places(t + 2, next);
            }
            // A sum that is not finite, or a score of -inf, which shows in no result: what a query
            // sees may hold that, or what it does not see; a key at a time then.
            float odd = sum * 0.f;
#pragma unroll
            for (int c = 0; c < T::kTiles; c++)
#pragma unroll
                for (int e = 0; e < 4; e++) odd += acc[c][e] * 0.f;
            if (__builtin_expect(__builtin_amdgcn_ballot_w64(odd != 0.f || lowest >= 0xff800000u) != 0, 0)) {
#pragma unroll
                for (int c = 0; c < T::kTiles; c++) acc[c] = (at_f4)(0.f);
                most = -__builtin_inff(), sum = 0.f;
                const float *q = a.q + row.at(a.qs);
#pragma unroll 1
                for (int t = t0; t < t1; t++)
#pragma unroll 1
                    for (int x = 0; x < 16 * H; x++) {
                        const int j = keys.first_key(t) + x;
                        bool held;
                        int64_t page;
                        int slot;
                        any_place(j, held, page, slot);
                        const E *kp = kb + page * a.pages.ks.p + slot * a.pages.ks.s, *vp = vb + page * a.pages.vs.p + slot * a.pages.vs.s;
                        float y = 0.f;
                        for (int c = quarter; c < a.D; c += 4) y += q[c] * a.scale2 * to_float(kp[c]);
                        y += __shfl_xor(y, 16);
                        y += __shfl_xor(y, 32);
                        if (!row.sees(a, s, j)) continue;
                        if (!held) y = __builtin_nanf("");
                        const float top = __builtin_fmaxf(most, y), base = top == -__builtin_inff() ? 0.f : top;
                        const float keep = __builtin_amdgcn_exp2f(most - base), p = __builtin_amdgcn_exp2f(y - base);
                        sum = sum * keep + (quarter == 0 ? p : 0.f);
                        most = top;
#pragma unroll
                        for (int c = 0; c < T::kTiles; c++)
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const int d = T::column(c, e, quarter);
                                acc[c][e] = acc[c][e] * keep + (d < a.D ? p * to_float(vp[d]) : 0.f);
                            }
                    }
            }
        }
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        __syncthreads();  // the last entry's have been read
#pragma unroll
        for (int c = 0; c < T::kTiles; c++)
#pragma unroll
            for (int e = 0; e < 4; e++) out_o[wave][col][T::column(c, e, quarter)] = acc[c][e];
        if (quarter == 0) out_ml[wave][col][0] = most, out_ml[wave][col][1] = sum;
        __syncthreads();
        const bool whole = ta == 0 && tb == tiles && a.stages == 1;
        const int64_t slot = slot_of_part(a, s, w, entry, ta == 0), part0 = ((int64_t)hk * s.slots + slot) * kTileRows;
        constexpr int kQuads = T::kTiles * 4;
        for (int x = (int)threadIdx.x; x < kTileRows * kQuads; x += 64 * kWaves) {
            const int r = x / kQuads, d = x % kQuads * 4;
            const PagedRow o(a, s, entry, hk, r);
            if (!o.is || d >= a.D) continue;
            float top = -__builtin_inff(), total = 0.f;
#pragma unroll
            for (int v = 0; v < kWaves; v++) top = __builtin_fmaxf(top, out_ml[v][r][0]);
            const float base = top == -__builtin_inff() ? 0.f : top;
            at_f4 y = (at_f4)(0.f);
#pragma unroll
            for (int v = 0; v < kWaves; v++) {
                const float f = __builtin_amdgcn_exp2f(out_ml[v][r][0] - base);
                total += out_ml[v][r][1] * f;
                y += *(const at_f4 *)&out_o[v][r][d] * f;
            }
            float *p;
            if (whole) {
                y *= o.place < 0 ? 0.f : 1.f / total;
                p = a.out + o.at(a.os) + d;
                if (a.lse && d == 0) a.lse[o.index(a)] = log_sum(top, total);
            } else {
                p = s.part_o + (part0 + r) * a.part_width + d;
                if (d == 0) s.part_ml[2 * (part0 + r)] = top, s.part_ml[2 * (part0 + r) + 1] = total;
            }
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (d + e < a.D) p[e] = y[e];
        }
        if (ta == 0 && s.found && threadIdx.x == 0)
            s.found[(int64_t)hk * s.entries + entry] = make_int2(share.block_of(before), share.block_of(before + tiles - 1));
        share.next(tiles);
    }
}

template <class T, bool ONE>
__global__ void __launch_bounds__(64 * kWaves, T::kTiles <= 8 ? 2 : 1) paged_few(PagedArgs a, int from) {
    __shared__ __attribute__((aligned(16))) float out_o[kWaves][kTileRows][T::kTiles * 16 + 4];
    __shared__ float out_ml[kWaves][kTileRows][2];
    int id = (int)blockIdx.x;
    const bool second = id >= a.few_blocks;
    const PagedStage &s = a.stage[from + second];
    if (second) id -= a.few_blocks;
    few_rows<T, ONE>(a, s, id % a.kv_heads, id / a.kv_heads, out_o, out_ml);
}

template <class T>
void launch_few(const PagedArgs &a, int from, dim3 grid, hipStream_t s) {
    bool mixed = false;
    for (int i = from; i < a.stages; i++) mixed |= a.stage[i].from < a.shared && a.stage[i].to > a.shared;
    if (a.pages.page % 16 == 0 && !(mixed && a.shared % 16)) hipLaunchKernelGGL((paged_few<T, true>), grid, dim3(64 * kWaves), 0, s, a, from);
    else hipLaunchKernelGGL((paged_few<T, false>), grid, dim3(64 * kWaves), 0, s, a, from);
}

template <template <int, int> class Ops, int DP>
void launch_width(const PagedArgs &a, int from, bool vectors, dim3 grid, hipStream_t s) {
    if (vectors && a.D == DP) launch_few<Ops<DP, 0>>(a, from, grid, s);
    else if (vectors) launch_few<Ops<DP, 1>>(a, from, grid, s);
    else launch_few<Ops<DP, 2>>(a, from, grid, s);
}

}  // namespace

int launch_paged_few(const PagedArgs &args, int from, int count, bool bf16, hipStream_t s) {
    PagedArgs a = args;
    int64_t blocks[2] = {0, 0};
    for (int i = 0; i < count; i++) {
        const PagedStage &st = a.stage[from + i];
        blocks[i] = (int64_t)a.kv_heads * (st.blocks ? st.blocks : st.entries);
    }
    if ((blocks[0] + blocks[1]) * 64 * kWaves >> 32)
        return set_error(TRS_E_INVALID_ARGUMENT, "attention over %lld blocks of rows", (long long)(blocks[0] + blocks[1]));
    a.few_blocks = (int32_t)blocks[0];
    const dim3 grid((unsigned)(blocks[0] + blocks[1]));
    const bool vectors = paged_vectors(a, bf16);
    if (bf16) {
        if (a.D <= 64) launch_width<Bf16Pages, 64>(a, from, vectors, grid, s);
        else if (a.D <= 128) launch_width<Bf16Pages, 128>(a, from, vectors, grid, s);
        else launch_width<Bf16Pages, 256>(a, from, vectors, grid, s);
    } else {
        if (a.D <= 32) launch_width<FloatPages, 32>(a, from, vectors, grid, s);
        else if (a.D <= 64) launch_width<FloatPages, 64>(a, from, vectors, grid, s);
        else if (a.D <= 96) launch_width<FloatPages, 96>(a, from, vectors, grid, s);
        else if (a.D <= 128) launch_width<FloatPages, 128>(a, from, vectors, grid, s);
        else if (a.D <= 192) launch_width<FloatPages, 192>(a, from, vectors, grid, s);
        else launch_width<FloatPages, 256>(a, from, vectors, grid, s);
    }
    TRS_LAUNCH_CHECK("paged attention launch");
    return TRS_OK;
}

}  // namespace trs
