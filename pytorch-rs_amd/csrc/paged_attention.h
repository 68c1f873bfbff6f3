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
// entries) have as many key tiles as their rows see; all of them in a list, the W blocks
// of a key head take equal shares of it: block w the tiles from T w / W on, of an entry's
// end, some whole entries and the next one's start.  What a block has of an entry that
// others have too is a part, joined by a second launch.
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
    int32_t blocks;      // W; 0: a block for every entry
    int32_t least;       // the least key tiles of a block that has others beside it
    int64_t slots;       // of parts, a key head
    float *part_o, *part_ml;  // [key head][slot][row of the tile]: part_width floats, and (maximum, sum)
    int2 *found;              // [key head][entry]: the first and the last block that have tiles of it
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
    int32_t stages, few_blocks;  // few_blocks: of the first of two stages that one launch has
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

// The least and the most keys of a sequence of the batch (every lane of the wave calls it).
__device__ __forceinline__ int2 keys_of_all(const PagedArgs &a, int lane) {
    int lo = a.pages.capacity, hi = 0;
    for (int b = lane; b < a.batch; b += 64) {
        const int n = a.pages.keys_of(b);
        lo = min(lo, n), hi = max(hi, n);
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) lo = min(lo, __shfl_xor(lo, d)), hi = max(hi, __shfl_xor(hi, d));
    return make_int2(lo, hi);
}

// A stage's list of tiles, and a block's share of it.
template <int SHIFT>
struct PagedShare {
    const PagedArgs &a;
    const PagedStage &s;
    int2 all;        // together: the batch's least and most keys
    int blocks;      // that have a share
    int64_t total, pos, end;  // tiles: of the list, of the share
    int entry;       // the entry of tile `pos`
    int64_t before;  // tiles ahead of that entry

    // Entry e: at least one tile, so that every row is written by some block.
    __device__ __forceinline__ PagedKeys<SHIFT> keys(int e) const {
        if (s.together) return PagedKeys<SHIFT>(a, s, all.x - a.Sq, all.y - 1);
        const int b = e / s.row_tiles, t = e - b * s.row_tiles, n = a.pages.keys_of(b);
        const int r0 = t * s.tile_rows, r1 = min(r0 + s.tile_rows, a.seq_rows) - 1;
        return PagedKeys<SHIFT>(a, s, n - a.Sq + (int)a.by_group.divide((uint32_t)r0), n - a.Sq + (int)a.by_group.divide((uint32_t)r1));
    }
    __device__ __forceinline__ int tiles_of(int e) const { return max(keys(e).tiles, 1); }

    __device__ __forceinline__ PagedShare(const PagedArgs &args, const PagedStage &stage, int w, int lane) : a(args), s(stage) {
        all = s.together ? keys_of_all(a, lane) : make_int2(0, 0);
        if (s.blocks == 0) {  // an entry each
            blocks = s.entries, entry = w, before = pos = 0, end = total = w < s.entries ? tiles_of(w) : 0;
            return;
        }
        if (s.together) {
            total = (int64_t)s.entries * tiles_of(0);
        } else {
            int64_t sum = 0;
            for (int e = lane; e < s.entries; e += 64) sum += tiles_of(e);
#pragma unroll
            for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
            total = sum;
        }
        blocks = (int)min((int64_t)s.blocks, (total + s.least - 1) / s.least);
        pos = w < blocks ? total * w / blocks : 0, end = w < blocks ? total * (w + 1) / blocks : 0;
        entry = 0, before = 0;
        if (pos >= end) return;
        if (s.together) {
            const int each = tiles_of(0);
            entry = (int)(pos / each), before = (int64_t)entry * each;
            return;
        }
        // The last entry that begins at or ahead of `pos`.
        for (int e0 = 0; e0 < s.entries; e0 += 64) {
            const int mine = e0 + lane < s.entries ? tiles_of(e0 + lane) : 0;
            int64_t sum = mine;
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {
                const int64_t more = __shfl_up(sum, d);
                sum += lane >= d ? more : 0;
            }
            const int64_t group = __shfl(sum, 63);
            if (pos < before + group) {
                const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(before + sum > pos));
                before += __shfl(sum - mine, l);
                entry = e0 + l;
                break;
            }
            before += group;
        }
        entry = __builtin_amdgcn_readfirstlane(entry);
    }
    __device__ __forceinline__ bool more() const { return pos < end; }
    __device__ __forceinline__ void next(int tiles) { pos = before = before + tiles, entry++; }
    // The block that has tile x of the list.
    __device__ __forceinline__ int block_of(int64_t x) const { return (int)(((x + 1) * blocks - 1) / total); }
};

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
            b = entry / s.row_tiles;
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
    __device__ __forceinline__ bool sees(const PagedArgs &a, const PagedStage &s, int j) const {
        return (j <= min(place, s.to - 1)) & (j >= s.from) & ((place - j < a.window) | (j < a.sinks));
    }
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
