// paged_rows.hip -- attention over a cache in pages for many rows: prompts, and the rows
// of a batch over the keys that it shares.
//
// 32 NW rows of a key head on the bf16 matrix cores.  A block brings a tile of 32 keys and
// values into one of two LDS buffers once for its waves while it computes from the other;
// the loads from the pages are a tile further ahead, and their entries of the table one more.
// S^T = K Q^T puts a row of the softmax in a lane (and its other half), and P^T is the operand of
// O^T += V^T P^T as it stands.
//
// Bound by the card's power and by issue: 1024 tokens of two prompts over 4096, 32 heads of 128 over 8,
// bfloat16, 313-327 us back to back, 1.10-1.16 PFLOP/s of bf16 products (a library product of 8192^3 reaches 1.31 on
// the same card): the matrix cores are busy for half the cycles at a clock of 2.0 GHz of 2.4, and 5.5 other vector
// instructions a matrix instruction take 35%.  Fragments read one step ahead of their products gave 376 -> 355.
// Waves of a SIMD held in opposite phases, one multiplying while the other works out weights, took 373, blocks
// of 128 rows, one for every tile of rows and no parts, 351 (a block brings every tile for half the rows).  The
// same for float32 pages 600.
//
// float32 pages: three bf16 pieces a float on both sides, six
// products (attention.h).  bfloat16 pages: keys and values as they are, queries and weights in
// three pieces, three products.
#include <hip/hip_runtime.h>

#include "paged_attention.h"

namespace trs {

namespace {

// A tile of keys and values in LDS: 2 NT units of 16 columns each, a KiB a piece (attention.h's Unit).
// One unit of a lane on its way there: 8 columns of row lane % 32.
template <class E, int WIDTH>
struct Staged;

template <int WIDTH>
struct Staged<float, WIDTH> {
    static constexpr int kPieces = 3;
    Unit<WIDTH> x;
    __device__ __forceinline__ void load(const float *row, int u, int D, int lane) { x.load(row, u, D, lane); }
    template <int UNITS>
    __device__ __forceinline__ void store(char *lds, int u, int lane) const { x.template store<UNITS>(lds, u, lane); }
};

template <int WIDTH>
struct Staged<uint16_t, WIDTH> {
    static constexpr int kPieces = 1;
    typedef uint32_t U4 __attribute__((ext_vector_type(4)));
    U4 x;
    __device__ __forceinline__ void load(const uint16_t *row, int u, int D, int lane) {
        const int c = 16 * u + 8 * (lane >> 5);
        if constexpr (WIDTH > 1) {
            const bool in = WIDTH == 4 || c < D;
            const U4 y = *(const U4 *)(row + (in ? c : 0));
            x = in ? y : (U4)(0u);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const bool in0 = c + 2 * e < D, in1 = c + 2 * e + 1 < D;
                const uint32_t y = row[in0 ? c + 2 * e : 0], z = row[in1 ? c + 2 * e + 1 : 0];
                x[e] = (in0 ? y : 0) | (in1 ? z << 16 : 0);
            }
        }
    }
    template <int UNITS>
    __device__ __forceinline__ void store(char *lds, int u, int lane) const { *(U4 *)(lds + u * 1024 + unit_place(lane)) = x; }
};

// A fragment of the tile's pieces, and its product with one of three pieces a value.
template <int PIECES>
struct Fragment {
    gt_bf8 p[PIECES];
    template <int UNITS>
    __device__ __forceinline__ static Fragment along(const char *lds, int u, int lane) {
        Fragment f;
        if constexpr (PIECES == 3) {
            const Pieces x = trs::along<UNITS>(lds, u, lane);
#pragma unroll
            for (int i = 0; i < 3; i++) f.p[i] = x.p[i];
        } else {
            f.p[0] = *(const gt_bf8 *)(lds + u * 1024 + unit_place(lane));
        }
        return f;
    }
    template <int UNITS>
    __device__ __forceinline__ static Fragment across(const char *lds, int u, int slot, int lane) {
        Fragment f;
        if constexpr (PIECES == 3) {
            const Pieces x = trs::across<UNITS>(lds, u, slot, lane);
#pragma unroll
            for (int i = 0; i < 3; i++) f.p[i] = x.p[i];
        } else {
            typedef short S4 __attribute__((ext_vector_type(4)));
            typedef short S8 __attribute__((ext_vector_type(8)));
            typedef S4 __attribute__((address_space(3))) *Lds;
            const int second = lane >> 1 & 1;
            const char *q = lds + (lane >> 4 & 1) * 1024 + second * 512 + (4 * (lane >> 5 ^ second) + (lane >> 2 & 3)) * 16 + (lane & 1) * 8 + u * 1024 + slot * 256;
            const S4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)q), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(q + 128));
            f.p[0] = __builtin_bit_cast(gt_bf8, (S8){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
        }
        return f;
    }
    // What was written so far: the reads, then the products.
    __device__ __forceinline__ static void in_order() {
        __builtin_amdgcn_sched_group_barrier(0x100, 2 * PIECES, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, PIECES == 3 ? 6 : 3, 0);
        __builtin_amdgcn_sched_barrier(0);
    }
    __device__ __forceinline__ void multiply(at_f16 &c, const Pieces &b) const {
        if constexpr (PIECES == 3) {
            const Pieces x{{p[0], p[1], p[2]}};
            mfma_pieces(c, x, b);
        } else {
#pragma unroll
            for (int i = 2; i >= 0; i--) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(p[0], b.p[i], c, 0, 0, 0);
        }
    }
};

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }

// WIDTH 4: D is 32 NT; 2: rows are read in vectors; 1: entry by entry.
template <class E, int NT, int NW, int WIDTH>
__global__ void __launch_bounds__(64 * NW, 2) paged_rows(PagedArgs a, int stage) {
    using In = Staged<E, WIDTH>;
    using F = Fragment<In::kPieces>;
    constexpr int UNITS = 4 * NT, OWN = (UNITS + NW - 1) / NW, kBuffer = In::kPieces * UNITS * 1024;
    constexpr float kUnit = In::kPieces == 3 ? kDown2 : kDown, kOut = In::kPieces == 3 ? kDown : 1.f;  // of scores, of outputs
    __shared__ __attribute__((aligned(1024))) char lds[2 * kBuffer];
    const PagedStage &s = a.stage[stage];
    const int lane = (int)threadIdx.x & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int hk = (int)(blockIdx.x % (uint32_t)a.kv_heads), w = (int)(blockIdx.x / (uint32_t)a.kv_heads);
    const E *const kb = (const E *)a.pages.k + hk * a.pages.ks.h, *const vb = (const E *)a.pages.v + hk * a.pages.vs.h;
    const auto unit = [&](int q) { return min(wave + q * NW, UNITS - 1); };
    for (PagedShare<5> share(a, s, w, lane); share.pos < share.end;) {
        const int entry = uniform(share.entry);
        const PagedKeys<5> keys = share.keys(entry);
        const int tiles = max(keys.tiles, 1);
        const int t0 = (int)(share.pos - share.before), end = min(tiles, (int)(share.end - share.before));
        const int t1 = keys.tiles ? end : t0;
        // The lane's row, worked out where it is used: its parts are not held in registers over the tiles.
        const auto row = [&]() {
            int e = entry;
            asm volatile("" : "+s"(e));
            return PagedRow(a, s, e, hk, wave * 32 + (lane & 31));
        };
        const auto [place, is] = [&]() {
            const PagedRow r = row();
            return int2{r.place, r.is};
        }();
        int lo = is ? place : INT32_MAX, hi = place;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) lo = min(lo, __shfl_xor(lo, d)), hi = max(hi, __shfl_xor(hi, d));
        const int wave_lo = __builtin_amdgcn_readfirstlane(lo), wave_hi = __builtin_amdgcn_readfirstlane(hi);
        const bool whole = __builtin_amdgcn_ballot_w64(!is) == 0;
        const int owner = s.together ? 0 : share.sequence_of(entry), first_row_to = s.from < a.shared ? a.shared : 0;
        at_f16 acc[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) acc[t] = (at_f16)(0.f);
        float most = -__builtin_inff(), sum = 0.f, unit_out = kOut;
        if (t0 < t1) {
            // The lane's key of a tile, past the last that is read that one, and past the share's last tile that one's.
            const auto key_at = [&](int t) { return min(keys.first_key(min(t, t1 - 1)) + (lane & 31), keys.last); };
            const auto page_at = [&](int j) { return a.pages.page_of(j < first_row_to ? 0 : owner, j); };
            In in[OWN];
            uint32_t missing;  // keys of the tile being loaded whose pages the pool does not have
            const auto load = [&](int t, int id) {
                const bool held = a.pages.holds(id);
                missing = (uint32_t)__builtin_amdgcn_ballot_w64(!held);
                const int page = held ? id : 0, slot = a.pages.slot_of(key_at(t));
                const E *kp = kb + a.pages.ks.at(page, slot), *vp = vb + a.pages.vs.at(page, slot);
#pragma unroll
                for (int q = 0; q < OWN; q++) {
                    const bool key = unit(q) < UNITS / 2;
                    in[q].load(key ? kp : vp, key ? unit(q) : unit(q) - UNITS / 2, a.D, lane);
                }
            };
            load(t0, page_at(key_at(t0)));
            int id = page_at(key_at(t0 + 1));
            Pieces q[2 * NT];
            const float *const q0 = a.q + row().at(a.qs);
#pragma unroll
            for (int n = 0; n < 2 * NT; n++) {
                Unit<WIDTH> x;
                x.load(q0, n, a.D, lane);
                if (place < 0) {  // nothing of a query that sees nothing
#pragma unroll
                    for (int e = 0; e < 8; e++) x.v[e] = 0.f;
                }
                q[n] = x.split(a.scale2 * kUp);
            }
            uint32_t missing0 = missing, missing1;
            __syncthreads();  // the last entry's tiles have been read
#pragma unroll
            for (int n = 0; n < OWN; n++) in[n].template store<UNITS>(lds, unit(n), lane);
            load(t0 + 1, id);
            missing1 = missing;
            id = page_at(key_at(t0 + 2));
            Lowest lowest;
#pragma unroll 1
            for (int t = t0; t < t1; t++) {
                const int j0 = keys.first_key(t);
                char *const buf = lds + ((t - t0) & 1) * kBuffer, *const other = lds + ((t - t0) & 1 ? 0 : kBuffer);
                __syncthreads();
#pragma unroll
                for (int n = 0; n < OWN; n++) in[n].template store<UNITS>(other, unit(n), lane);
                load(t + 2, id);
                id = page_at(key_at(t + 3));
                const uint32_t absent = missing0;
                missing0 = missing1, missing1 = missing;
                // Whether a row of the wave sees a key of the tile.
                if (j0 <= wave_hi && (wave_lo - (j0 + 31) < a.window || j0 < a.sinks)) {
                    // Fragments are read a step ahead of their products.
                    const auto value = [&](int n) { return F::template across<UNITS>(buf, 2 * NT + 2 * (n % NT), n / NT, lane); };
                    at_f16 x = (at_f16)(0.f);
                    F f = F::template along<UNITS>(buf, 0, lane);
#pragma unroll
                    for (int n = 0; n < 2 * NT; n++) {
                        const F now = f;
                        f = n + 1 < 2 * NT ? F::template along<UNITS>(buf, n + 1, lane) : value(0);
                        now.multiply(x, q[n]);
                        F::in_order();
                    }
                    lowest.add(x);
                    const bool all = whole && j0 >= s.from && j0 + 31 < s.to && j0 + 31 <= wave_lo && (wave_hi - j0 < a.window || j0 + 32 <= a.sinks);
                    if (!all || absent) {
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            const int k = result_row(e, half);
                            if (absent >> k & 1) x[e] = __builtin_nanf("");
                            x[e] = paged_sees(a, s, place, j0 + k) ? x[e] : -__builtin_inff();
                        }
                    }
                    float m = x[0];
#pragma unroll
                    for (int e = 1; e < 16; e++) m = __builtin_fmaxf(m, x[e]);
                    m = __builtin_fmaxf(m, __shfl_xor(m, 32));
                    // (The unit is a power of two: the sum is rounded once.)
                    const float top = __builtin_fmaxf(most, m), base = (top == -__builtin_inff() ? 0.f : top) * kUnit;
                    const float keep = __builtin_amdgcn_exp2f(__builtin_fmaf(most, kUnit, -base));
                    float add[2] = {0.f, 0.f};
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], kUnit, -base));
                        add[e & 1] += x[e];
                    }
                    sum = sum * keep + (add[0] + add[1]);
                    most = top;
                    if (__builtin_amdgcn_ballot_w64(keep != 1.f)) {
#pragma unroll
                        for (int c = 0; c < NT; c++) acc[c] *= keep;
                    }
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        Splitting p;
#pragma unroll
                        for (int i = 0; i < 4; i++) split_weights(p, i, x[8 * n + 2 * i], x[8 * n + 2 * i + 1]);
                        const Pieces y = p.done();
#pragma unroll
                        for (int c = 0; c < NT; c++) {
                            const F now = f;
                            if (n * NT + c + 1 < 2 * NT) f = value(n * NT + c + 1);
                            now.multiply(acc[c], y);
                            F::in_order();
                        }
                    }
                }
            }
            most *= kUnit;
            // What the pieces do not hold, and infinities and NaN, seen or hidden: a key at a time.
            if (__builtin_expect(not_finite(acc, sum) || lowest.infinite(), 0)) {
#pragma unroll
                for (int t = 0; t < NT; t++) acc[t] = (at_f16)(0.f);
                most = -__builtin_inff(), sum = 0.f, unit_out = 1.f;
                const float *qp = a.q + row().at(a.qs);
#pragma unroll 1
                for (int t = t0; t < t1; t++)
#pragma unroll 1
                    for (int k = 0; k < 32; k++) {
                        const int j = keys.first_key(t) + k, at = min(j, keys.last), page_id = page_at(at);
                        const bool held = a.pages.holds(page_id);
                        const int page = held ? page_id : 0, slot = a.pages.slot_of(at);
                        const E *kp = kb + a.pages.ks.at(page, slot), *vp = vb + a.pages.vs.at(page, slot);
                        float y = 0.f;
                        for (int c = half; c < a.D; c += 2) y += qp[c] * a.scale2 * as_float(kp[c]);
                        y += __shfl_xor(y, 32);
                        if (!paged_sees(a, s, place, j)) continue;
                        if (!held) y = __builtin_nanf("");
                        const float top = __builtin_fmaxf(most, y), base = top == -__builtin_inff() ? 0.f : top;
                        const float keep = __builtin_amdgcn_exp2f(most - base), p = __builtin_amdgcn_exp2f(y - base);
                        sum = sum * keep + (half == 0 ? p : 0.f);
                        most = top;
#pragma unroll
                        for (int c = 0; c < NT; c++)
#pragma unroll
                            for (int e = 0; e < 16; e++) {
                                const int d = 32 * c + result_row(e, half);
                                acc[c][e] = acc[c][e] * keep + (d < a.D ? p * as_float(vp[d]) : 0.f);
                            }
                    }
            }
        }
        sum += __shfl_xor(sum, 32);
        if (is) {
            const PagedRow r = row();
            if (t0 == 0 && end == tiles && a.stages == 1) {
                write_row<WIDTH>(acc, a.out + r.at(a.os), unit_out, r.place < 0 ? 0.f : 1.f / sum, a.D, half);
                if (a.lse && half == 0) a.lse[r.index(a)] = log_sum(most, sum);
            } else {
                const int64_t part = ((int64_t)hk * s.slots + slot_of_part(a, s, w, entry, t0 == 0)) * s.tile_rows + wave * 32 + (lane & 31);
                write_row<WIDTH>(acc, s.part_o + part * a.part_width, unit_out, 1.f, a.D, half);
                if (half == 0) s.part_ml[2 * part] = most, s.part_ml[2 * part + 1] = sum;
            }
        }
        if (t0 == 0 && s.found && threadIdx.x == 0)
            s.found[(int64_t)hk * s.entries + entry] = make_int2(share.worker_of(share.before), share.worker_of(share.before + tiles - 1));
        share.next(tiles);
    }
}

template <class E, int NT, int NW>
void launch_width(const PagedArgs &a, int stage, bool vectors, dim3 grid, hipStream_t s) {
    const dim3 block(64 * NW);
    if (vectors && a.D == 32 * NT) hipLaunchKernelGGL((paged_rows<E, NT, NW, 4>), grid, block, 0, s, a, stage);
    else if (vectors) hipLaunchKernelGGL((paged_rows<E, NT, NW, 2>), grid, block, 0, s, a, stage);
    else hipLaunchKernelGGL((paged_rows<E, NT, NW, 1>), grid, block, 0, s, a, stage);
}
template <class E, int NT>
void launch_rows(const PagedArgs &a, int stage, bool vectors, dim3 grid, hipStream_t s) {
    if constexpr (sizeof(E) == 2) {
        if (a.stage[stage].tile_rows == 128) return launch_width<E, NT, 4>(a, stage, vectors, grid, s);
    }
    launch_width<E, NT, 8>(a, stage, vectors, grid, s);
}
template <class E>
void launch_type(const PagedArgs &a, int stage, bool vectors, dim3 grid, hipStream_t s) {
    if (a.D <= 32) launch_rows<E, 1>(a, stage, vectors, grid, s);
    else if (a.D <= 64) launch_rows<E, 2>(a, stage, vectors, grid, s);
    else if (a.D <= 96) launch_rows<E, 3>(a, stage, vectors, grid, s);
    else launch_rows<E, 4>(a, stage, vectors, grid, s);
}

}  // namespace

int launch_paged_rows(const PagedArgs &a, int stage, bool bf16, hipStream_t s) {
    const PagedStage &st = a.stage[stage];
    const int64_t blocks = (int64_t)a.kv_heads * (st.workers ? st.workers : st.entries);
    if (blocks * 2 * st.tile_rows >> 32) return set_error(TRS_E_INVALID_ARGUMENT, "attention over %lld blocks of rows", (long long)blocks);
    const dim3 grid((unsigned)blocks);
    if (bf16) launch_type<uint16_t>(a, stage, paged_vectors(a, bf16), grid, s);
    else launch_type<float>(a, stage, paged_vectors(a, bf16), grid, s);
    TRS_LAUNCH_CHECK("paged attention launch");
    return TRS_OK;
}

}  // namespace trs
