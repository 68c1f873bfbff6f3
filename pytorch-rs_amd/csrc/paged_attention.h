// paged_attention.h -- attention over a cache in pages: what its host part
// (paged_attention.hip) and its kernels (paged_few.hip, paged_rows.hip) share.
//
// Query i of a sequence of n tokens stands at place p = n - Sq + i and sees
//   key j  where  j <= p  and  (p - j < window  or  j < sinks).
// The query heads that share a key head are taken together: row r = i * group + (head
// within the group) of a sequence.  A stage is a range of keys for rows: of a sequence
// each, or, for the prefix that a batch shares, of all its sequences one behind another.
//
// Lengths are on the device, so the work is divided there.  A stage's tiles of rows (its
// entries) have as many key tiles as their rows see; all of them in a list, the workers of a key
// head (waves of paged_few, blocks of paged_rows) take equal shares of it: an entry's end, some
// whole entries and the next one's start.  What a worker has of an entry that others have too is
// a part, joined by a second launch.
#pragma once

#include "attention.h"
#include "paged.h"

namespace trs {

struct PagedStage {
    int32_t together;   // rows of all sequences, one behind another
    int32_t from, to;   // keys [from, to)
    int32_t row_tiles;  // of a sequence, or of all
    int32_t entries;
    int32_t tile_rows;
    int32_t workers;     // of a key head; 0: one for every entry
    int32_t least;       // the least key tiles of a worker that has others beside it
    int32_t most;        // the most key tiles of an entry
    SmallDivisor by_row_tiles;
    int64_t slots;       // of parts, a key head
    float *part_o, *part_ml;  // [key head][slot][row of the tile]: part_width floats, and (maximum, sum)
    int2 *found;              // [key head][entry]: the first and the last worker that have tiles of it
};

struct PagedArgs {
    Pages pages;
    const float *q;
    float *out, *lse;
    AttnView qs, os;
    int32_t batch, heads, kv_heads, group, Sq, D;
    int32_t window, sinks, shared;
    int32_t part_width;
    float scale2;
    int32_t seq_rows;  // Sq * group
    int32_t all_rows;  // batch * seq_rows; only where rows are together
    SmallDivisor by_group, by_seq_rows;
    int32_t stages;
    int32_t few_workers, few_all;  // of paged_few's launch: of the first of its stages, and of all
    PagedStage stage[2];
};

// The tiles of 1 << SHIFT keys of a stage that rows at places lo to hi see, the sinks' first and
// then the window's.
template <int SHIFT>
struct PagedKeys {
    int last;  // the last key that any row sees; below `from`: none does
    int first, sink_first, sink_tiles, tiles;

    __device__ __forceinline__ PagedKeys(const PagedArgs &a, const PagedStage &s, int lo, int hi) {
        last = min(hi, s.to - 1);
        const int near = max(lo - a.window + 1, s.from);  // the first key of a window
        const bool some = last >= s.from;
        first = near <= last ? near >> SHIFT : (last >> SHIFT) + 1;
        sink_first = s.from >> SHIFT;
        const int end = (min(a.sinks, last + 1) + (1 << SHIFT) - 1) >> SHIFT;
        sink_tiles = some ? max(min(end, first) - sink_first, 0) : 0;
        tiles = some ? sink_tiles + max((last >> SHIFT) - first + 1, 0) : 0;
    }
    __device__ __forceinline__ int first_key(int t) const { return (t < sink_tiles ? sink_first + t : first + t - sink_tiles) << SHIFT; }
};

// Pair i of a fragment's four, finite values: split_pair's pieces, the remainder behind each rounding by
// one dot product with (-1, 0) or (0, -1), which is exact (compared bit for bit with the subtraction on
// 2^22 pairs each of close, distant, subnormal, large and zero values), where the subtraction has to
// widen the piece first: 7 instructions a pair, not 11.  The constants come from registers: as literals the
// compiler takes them for the inline constant -1, which stands in both halves.
__device__ __forceinline__ void split_weights(Splitting &x, int i, float a, float b) {
    uint32_t low, high;
    asm("s_mov_b32 %0, 0xbf80" : "=s"(low));
    asm("s_mov_b32 %0, 0xbf800000" : "=s"(high));
    const auto pack = [](float u, float v) { return __builtin_convertvector((gt_f2){u, v}, gt_bf2); };
    const gt_bf2 first = __builtin_bit_cast(gt_bf2, low), second = __builtin_bit_cast(gt_bf2, high);
    const gt_bf2 h = pack(a, b);
    a = __builtin_amdgcn_fdot2_f32_bf16(h, first, a, false);
    b = __builtin_amdgcn_fdot2_f32_bf16(h, second, b, false);
    const gt_bf2 m = pack(a, b);
    a = __builtin_amdgcn_fdot2_f32_bf16(m, first, a, false);
    b = __builtin_amdgcn_fdot2_f32_bf16(m, second, b, false);
    x.h[i] = __builtin_bit_cast(uint32_t, h), x.m[i] = __builtin_bit_cast(uint32_t, m), x.l[i] = __builtin_bit_cast(uint32_t, pack(a, b));
}

// What is the same in all lanes, where the compiler cannot tell: to scalar registers.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) { return (int64_t)(uint32_t)uniform((int)x) | (int64_t)uniform((int)(x >> 32)) << 32; }

// The least and the most keys of a sequence of the batch (every lane of the wave calls it).
__device__ __forceinline__ int2 keys_of_all(const PagedArgs &a, int lane) {
    int lo = a.pages.capacity, hi = 0;
    for (int b = lane; b < a.batch; b += 64) {
        const int n = a.pages.keys_of(b);
        lo = min(lo, n), hi = max(hi, n);
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) lo = min(lo, __shfl_xor(lo, d)), hi = max(hi, __shfl_xor(hi, d));
    return make_int2(uniform(lo), uniform(hi));
}

// A stage's list of tiles, and worker w's share of it: tiles `pos` to `end`.  (Below 2^31 tiles,
// which the host sees to.)  Every lane of the wave calls it.
template <int SHIFT>
struct PagedShare {
    const PagedArgs &a;
    const PagedStage &s;
    int2 all;                // together: the batch's least and most keys
    uint32_t base, extra;    // the tiles of a worker; the first `extra` have one more
    uint32_t pos, end;
    int entry;               // the entry of tile `pos`
    uint32_t before;         // tiles ahead of that entry

    __device__ __forceinline__ int sequence_of(int e) const { return (int)s.by_row_tiles.divide((uint32_t)e); }
    // What entry e of a sequence of n tokens sees.
    __device__ __forceinline__ PagedKeys<SHIFT> keys(int e, int n) const {
        const int r0 = (e - sequence_of(e) * s.row_tiles) * s.tile_rows, r1 = min(r0 + s.tile_rows, a.seq_rows) - 1;
        return PagedKeys<SHIFT>(a, s, n - a.Sq + (int)a.by_group.divide((uint32_t)r0), n - a.Sq + (int)a.by_group.divide((uint32_t)r1));
    }
    __device__ __forceinline__ PagedKeys<SHIFT> keys(int e) const {
        return s.together ? PagedKeys<SHIFT>(a, s, all.x - a.Sq, all.y - 1) : keys(e, a.pages.keys_of(sequence_of(e)));
    }
    // At least one tile, so that every row is written by some worker.
    __device__ __forceinline__ int tiles_of(int e) const { return max(keys(e).tiles, 1); }
    __device__ __forceinline__ uint32_t start_of(uint32_t w) const { return w * base + min(w, extra); }
    // The worker that has tile x of the list.
    __device__ __forceinline__ int worker_of(uint32_t x) const {
        const uint32_t longer = extra * (base + 1);
        return (int)(x < longer ? x / (base + 1) : extra + (x - longer) / base);
    }
    __device__ __forceinline__ void divide(uint32_t total, uint32_t w) {
        const uint32_t workers = min((uint32_t)s.workers, (total + s.least - 1) / s.least);
        base = total / workers, extra = total - base * workers;
        pos = w < workers ? start_of(w) : 0, end = w < workers ? start_of(w + 1) : 0;
    }
    __device__ __forceinline__ PagedShare(const PagedArgs &args, const PagedStage &stage, int w, int lane) : a(args), s(stage) {
        all = s.together ? keys_of_all(a, lane) : make_int2(0, 0);
        entry = 0, before = 0;
        if (s.workers == 0) {  // an entry each
            entry = w, base = extra = pos = 0, end = w < s.entries ? uniform(tiles_of(entry)) : 0;
        } else if (s.together) {
            const uint32_t each = tiles_of(0);
            divide(s.entries * each, w);
            if (pos < end) entry = (int)(pos / each), before = entry * each;
        } else {
            // The tiles up to each entry, 64 of them at a time, and the last one that begins at or ahead of `pos`.
            const auto up_to = [&](int e0) {
                uint32_t sum = e0 + lane < s.entries ? tiles_of(e0 + lane) : 0;
#pragma unroll
                for (int d = 1; d < 64; d *= 2) {
                    const uint32_t more = __shfl_up(sum, d);
                    sum += lane >= d ? more : 0;
                }
                return sum;
            };
            const auto last = [](uint32_t sum) { return (uint32_t)__builtin_amdgcn_readlane(sum, 63); };
            const uint32_t first = up_to(0);
            uint32_t total = last(first), sum = first;
            for (int e0 = 64; e0 < s.entries; e0 += 64) total += last(up_to(e0));
            divide(total, w);
            if (pos >= end) return;
            int e0 = 0;
            while (pos >= before + last(sum)) before += last(sum), e0 += 64, sum = up_to(e0);
            const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(before + sum > pos));
            if (l) before += (uint32_t)__builtin_amdgcn_readlane(sum, l - 1);
            entry = e0 + l;
        }
    }
    // To the next entry, behind one of so many tiles.
    __device__ __forceinline__ void next(int tiles) { pos = before = before + tiles, entry++; }
};

// Whether a row at `place` sees key j of the stage.
__device__ __forceinline__ bool paged_sees(const PagedArgs &a, const PagedStage &s, int place, int j) {
    return (j <= min(place, s.to - 1)) & (j >= s.from) & ((place - j < a.window) | (j < a.sinks));
}

// A lane's row of an entry.
struct PagedRow {
    int b, i, g;
    int place;  // -1: no such row, or one that sees nothing
    int64_t h;

    __device__ __forceinline__ PagedRow(const PagedArgs &a, const PagedStage &s, int entry, int hk, int at) {
        int r, rows;
        if (s.together) {
            const int all = entry * s.tile_rows + at, in = min(all, a.all_rows - 1);
            b = (int)a.by_seq_rows.divide((uint32_t)in);
            r = in - b * a.seq_rows;
            rows = all < a.all_rows;
        } else {
            b = (int)s.by_row_tiles.divide((uint32_t)entry);
            const int one = (entry - b * s.row_tiles) * s.tile_rows + at;
            r = min(one, a.seq_rows - 1);
            rows = one < a.seq_rows;
        }
        i = (int)a.by_group.divide((uint32_t)r), g = r - i * a.group;
        h = (int64_t)hk * a.group + g;
        place = rows ? max(a.pages.keys_of(b) - a.Sq + i, -1) : -1;
        is = rows;
    }
    bool is;  // there is such a row
    __device__ __forceinline__ int64_t at(const AttnView &v) const { return b * v.b + h * v.h + i * v.s; }
    __device__ __forceinline__ int64_t index(const PagedArgs &a) const { return ((int64_t)b * a.heads + h) * a.Sq + i; }
};

// A part's place, and where an entry's parts are.
__device__ __forceinline__ int64_t slot_of_part(const PagedArgs &a, const PagedStage &s, int w, int entry, bool starts) {
    return a.stages > 1 ? (int64_t)w + entry : 2 * (int64_t)w + starts;
}

// Whether rows of the pages are read in vectors: ones of 16 bytes need that alignment in bfloat16 pages; float32's need none.
inline bool paged_vectors(const PagedArgs &a, bool bf16) {
    const auto aligned = [](const void *p, const PoolView &v) { return (uintptr_t)p % 16 == 0 && v.p % 8 == 0 && v.h % 8 == 0 && v.s % 8 == 0; };
    return bf16 ? a.D % 8 == 0 && aligned(a.pages.k, a.pages.ks) && aligned(a.pages.v, a.pages.vs) : a.D % 4 == 0;
}

// Many rows (paged_rows.hip): one stage, tiles of 128 or 256 rows, heads of up to kPiecesDim.
int launch_paged_rows(const PagedArgs &a, int stage, bool bf16, hipStream_t s);
// Few rows a sequence, or of all (paged_few.hip): stages [from, from + count).
int launch_paged_few(const PagedArgs &a, int from, int count, bool bf16, hipStream_t s);

}  // namespace trs
