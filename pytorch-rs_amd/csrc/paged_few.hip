// paged_few.hip -- attention over a cache in pages for few rows: single tokens of a batch.
//
// Bound by reading the keys and values once: 32 sequences of 1640 to 8192 tokens, 8 key heads of 128,
// bfloat16 (645 MB) 120-125 us; of calls over 4096, 8192 and 16384 keys each (104, 187 and 358 us) the keys added are
// read at 6.3-6.4 TB/s, and 17 to 20 us are the way in and out, joining's 5 among them; 7 to 9 us for one sequence of 1000 tokens, 8 heads of 64, float32.  A wave takes 16 rows and streams its
// share of the keys straight from the pages into the registers that the matrix instructions take
// them from: no LDS, no barrier, nothing that waits for another wave.  (Blocks of four waves that join
// in LDS, two blocks a CU: a batch of 64 with 60 to 512 tokens of its own 38 us, 24 so.)  What several
// waves have of an entry is joined by a second launch, 5 us of which most is the launch.
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
    __device__ __forceinline__ static void write(const at_f4 (&acc)[kTiles], float *p, int D, int quarter) { T::write(acc, p, 1.f, D, quarter); }
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
            if constexpr (MODE == 2) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const bool in = c + e < D;
                    const float y = row[in ? c + e : 0];
                    x.v[e] = in ? y : 0.f;
                }
            } else {
                const bool in = MODE == 0 || c < D;
                const f4u y = *(const f4u *)(row + (in ? c : 0)), z = *(const f4u *)(row + (in ? c + 4 : 0));
#pragma unroll
                for (int e = 0; e < 4; e++) x.v[e] = in ? y[e] : 0.f, x.v[4 + e] = in ? z[e] : 0.f;
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
        for (int i = 0; i < 4; i++) split_weights(w, i, p[i >> 1][2 * (i & 1)], p[i >> 1][2 * (i & 1) + 1]);
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
    // acc^T: the lane's column of acc is the row at p.
    __device__ __forceinline__ static void write(const at_f4 (&acc)[kTiles], float *p, int D, int quarter) {
#pragma unroll
        for (int u = 0; u < VU; u++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int e = 0; e < W; e += 4) {
                    const int d = column(u * W + e, i, quarter);
                    const f4u x = {acc[u * W + e][i], acc[u * W + e + 1][i], acc[u * W + e + 2][i], acc[u * W + e + 3][i]};
                    if (MODE == 0 || (MODE == 1 && d < D)) {
                        *(f4u *)(p + d) = x;
                    } else if (MODE == 2) {
#pragma unroll
                        for (int n = 0; n < 4; n++)
                            if (d + n < D) p[d + n] = x[n];
                    }
                }
    }
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }

// A wave's way along its share of the list: a tile of an entry.
template <int SHIFT>
struct Step {
    PagedKeys<SHIFT> keys;
    int entry, owner;  // owner: the sequence whose pages are read
    int tiles;         // of the entry
    int from, t, to;   // the entry's tiles that are the wave's, and the one that this is
    uint32_t before;   // tiles ahead of the entry

    __device__ __forceinline__ Step(const PagedShare<SHIFT> &share)
        : keys(share.keys(share.entry)), entry(share.entry), owner(share.s.together ? 0 : share.sequence_of(share.entry)) {
        tiles = max(keys.tiles, 1), before = share.before;
        from = t = (int)(share.pos - share.before), to = min(tiles, (int)(share.end - share.before));
    }
};

// Where a tile's keys stand.  ONE: pages hold a multiple of 16 tokens, and no 16 keys are the first
// sequence's in part, so that a half's keys stand in one page, and its entry of the table is read by the
// scalar unit.  Else every lane looks one key up and the others ask it (32 sequences of 2000 tokens, 8 key
// heads of 128, bfloat16: pages of 16 so 54.2 us, of 8 the other way 56.0; a look-up of its own for every row a
// lane reads takes 83).
template <class T, bool ONE>
struct Places {
    using E = typename T::E;
    const E *k[T::kHalves], *v[T::kHalves];  // ONE: of the half's first key
    int last[T::kHalves];                    // ONE: its last key that is read
    uint32_t absent;                         // ONE: halves whose page the pool does not have

    int id, slot;  // else: the page and the token of it of key `lane` of the tile (of 16 or 32)

    // The page and the token of it that a key stands in; past the last key that is read, that one's.  (An
    // entry that sees nothing has a tile none of whose keys is seen: any key that there is will do.)
    __device__ __forceinline__ static int find(const PagedArgs &a, int first_row_to, int owner, int j, int last, int &slot) {
        const int at = max(min(j, last), 0);
        slot = a.pages.slot_of(at);
        return a.pages.page_of(at < first_row_to ? 0 : owner, at);
    }
    __device__ __forceinline__ Places(const PagedArgs &a, int first_row_to, const E *kb, const E *vb, const Step<T::kShift> &x, int lane) {
        const int j0 = x.keys.first_key(x.t), end = x.keys.last;
        if constexpr (ONE) {
            absent = 0;
#pragma unroll
            for (int h = 0; h < T::kHalves; h++) {
                const int at = max(min(j0 + 16 * h, end & ~15), 0), there = find(a, first_row_to, x.owner, at, end, slot);
                if (!a.pages.holds(there)) absent |= 1u << h;
                const int page = a.pages.holds(there) ? there : 0;
                k[h] = kb + a.pages.ks.at(page, slot);
                v[h] = vb + a.pages.vs.at(page, slot);
                last[h] = max(min(end - at, 15), 0);
            }
        } else {
            id = find(a, first_row_to, x.owner, j0 + (lane & (16 * T::kHalves - 1)), end, slot);
        }
    }
    __device__ __forceinline__ const E *k_row(const PagedArgs &a, const E *kb, int h, int n) const {
        if constexpr (ONE) return k[h] + (uint64_t)(uint32_t)min(n, last[h]) * a.pages.ks.s;
        const int page = __shfl(id, 16 * h + n);
        return kb + a.pages.ks.at(a.pages.holds(page) ? page : 0, __shfl(slot, 16 * h + n));
    }
    __device__ __forceinline__ const E *v_row(const PagedArgs &a, const E *vb, int h, int n) const {
        if constexpr (ONE) return v[h] + (uint64_t)(uint32_t)min(n, last[h]) * a.pages.vs.s;
        const int page = __shfl(id, 16 * h + n);
        return vb + a.pages.vs.at(a.pages.holds(page) ? page : 0, __shfl(slot, 16 * h + n));
    }
    // Whether the pool has the page of key n of half h.
    __device__ __forceinline__ bool held(const PagedArgs &a, int h, int n) const {
        if constexpr (ONE) return !(absent >> h & 1);
        return a.pages.holds(__shfl(id, 16 * h + n));
    }
};

// A wave's share of a key head's tiles, one behind another whatever entries they belong to: the
// next tile's loads are on their way while one is worked on, and the page after that looked up.
template <class T, bool ONE>
__device__ __forceinline__ void few_rows(const PagedArgs &a, const PagedStage &s, int hk, int w) {
    using E = typename T::E;
    constexpr int H = T::kHalves;
    const int lane = (int)threadIdx.x & 63, col = lane & 15, quarter = lane >> 4;
    PagedShare<T::kShift> share(a, s, w, lane);
    if (share.pos >= share.end) return;
    const E *const kb = (const E *)a.pages.k + hk * a.pages.ks.h, *const vb = (const E *)a.pages.v + hk * a.pages.vs.h;
    const int first_row_to = s.from < a.shared ? a.shared : 0;  // keys below it are the first sequence's
    Step<T::kShift> now(share), ahead = now;
    const uint32_t count = share.end - share.pos;
    // `ahead` to the tile behind it; past the wave's last tile it stays.
    const auto advance = [&]() {
        if (ahead.t + 1 < ahead.to) {
            ahead.t++;
        } else if (share.before + ahead.tiles < share.end) {
            share.next(ahead.tiles);
            ahead = Step<T::kShift>(share);
        }
    };
    using P = Places<T, ONE>;
    T ops;
    P here(a, first_row_to, kb, vb, now, lane);
    const auto load_k = [&](const P &p) { ops.load_k([&](int h, int n) { return p.k_row(a, kb, h, n); }, a.D, col, quarter); };
    const auto load_v = [&](const P &p) { ops.load_v([&](int h, int n) { return p.v_row(a, vb, h, n); }, a.D, col, quarter); };
    load_k(here);
    load_v(here);
    int place = 0;
    const auto load_q = [&]() {
        const PagedRow row(a, s, now.entry, hk, col);
        place = row.place;
        ops.load_q(a.q + row.at(a.qs), a.D, quarter, a.scale2);
    };
    load_q();
    advance();
    P next(a, first_row_to, kb, vb, ahead, lane);

    at_f4 acc[T::kTiles];
    float most, sum;
    uint32_t lowest;
    const auto clear = [&]() {
#pragma unroll
        for (int c = 0; c < T::kTiles; c++) acc[c] = (at_f4)(0.f);
        most = -__builtin_inff(), sum = 0.f, lowest = 0;
    };
    // A key at a time, for what a query sees, or does not, of infinities and NaN.
    const auto each_key = [&]() {
        const PagedRow row(a, s, now.entry, hk, col);
        const float *q = a.q + row.at(a.qs);
#pragma unroll 1
        for (int t = now.from; t < now.to; t++)
#pragma unroll 1
            for (int x = 0; x < 16 * H; x++) {
                const int j = now.keys.first_key(t) + x;
                int slot;
                const int id = P::find(a, first_row_to, now.owner, j, now.keys.last, slot);
                const bool held = a.pages.holds(id);
                const int page = held ? id : 0;
                const E *kp = kb + a.pages.ks.at(page, slot), *vp = vb + a.pages.vs.at(page, slot);
                float y = 0.f;
                for (int c = quarter; c < a.D; c += 4) y += q[c] * a.scale2 * to_float(kp[c]);
                y += __shfl_xor(y, 16);
                y += __shfl_xor(y, 32);
                if (!paged_sees(a, s, place, j)) continue;
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
    };
    // The entry's rows, or the wave's part of them.
    const auto write = [&]() {
        // A sum that is not finite, or a score of -inf, which shows in no result.
        float odd = sum * 0.f;
#pragma unroll
        for (int c = 0; c < T::kTiles; c++)
#pragma unroll
            for (int e = 0; e < 4; e++) odd += acc[c][e] * 0.f;
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(odd != 0.f || lowest >= 0xff800000u) != 0, 0)) {
            clear();
            each_key();
        }
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        const PagedRow row(a, s, now.entry, hk, col);
        const bool whole = now.from == 0 && now.to == now.tiles && a.stages == 1;
        if (row.is) {
            float *p;
            if (whole) {
                const float f = row.place < 0 ? 0.f : 1.f / sum;
#pragma unroll
                for (int c = 0; c < T::kTiles; c++) acc[c] *= f;
                p = a.out + row.at(a.os);
                if (a.lse && quarter == 0) a.lse[row.index(a)] = log_sum(most, sum);
            } else {
                const int64_t part = ((int64_t)hk * s.slots + slot_of_part(a, s, w, now.entry, now.from == 0)) * kTileRows + col;
                p = s.part_o + part * a.part_width;
                if (quarter == 0) s.part_ml[2 * part] = most, s.part_ml[2 * part + 1] = sum;
            }
            T::write(acc, p, a.D, quarter);
        }
        if (now.from == 0 && s.found && lane == 0)
            s.found[(int64_t)hk * s.entries + now.entry] = make_int2(w, share.worker_of(now.before + now.tiles - 1));
    };

    clear();
    for (uint32_t left = count; left > 0; left--) {
        const int j0 = now.keys.first_key(now.t);
        at_f4 x[H];
        ops.scores(x);
        load_k(next);
        float m = -__builtin_inff();
#pragma unroll
        for (int h = 0; h < H; h++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int n = 4 * quarter + e;
                const uint32_t bits = __float_as_uint(x[h][e]);
                lowest = lowest > bits ? lowest : bits;
                const float y = here.held(a, h, n) ? x[h][e] * T::kDownScale : __builtin_nanf("");
                x[h][e] = paged_sees(a, s, place, j0 + 16 * h + n) ? y : -__builtin_inff();
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
        load_v(next);
        if (now.t + 1 == now.to) {
            write();
            now = ahead;
            if (left > 1) load_q();
            clear();
        } else {
            now.t++;
        }
        here = next;
        advance();
        next = P(a, first_row_to, kb, vb, ahead, lane);
    }
}

template <class T, bool ONE>
__global__ void __launch_bounds__(64 * kWaves, T::kTiles <= 8 ? 2 : 1) paged_few(PagedArgs a, int from) {
    int id = (int)blockIdx.x * kWaves + uniform((int)threadIdx.x >> 6);
    if (id >= a.few_all) return;  // the last block's waves without work
    const bool second = id >= a.few_workers;
    const PagedStage &s = a.stage[from + second];
    if (second) id -= a.few_workers;
    few_rows<T, ONE>(a, s, id % a.kv_heads, id / a.kv_heads);
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
    int64_t waves[2] = {0, 0};
    for (int i = 0; i < count; i++) {
        const PagedStage &st = a.stage[from + i];
        waves[i] = (int64_t)a.kv_heads * (st.workers ? st.workers : st.entries);
    }
    const int64_t all = waves[0] + waves[1];
    if ((all + kWaves) * 64 >> 32) return set_error(TRS_E_INVALID_ARGUMENT, "attention over %lld tiles of rows", (long long)all);
    a.few_workers = (int32_t)waves[0], a.few_all = (int32_t)all;
    const dim3 grid((unsigned)((all + kWaves - 1) / kWaves));
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
