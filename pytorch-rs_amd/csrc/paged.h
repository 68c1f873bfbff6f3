// paged.h -- a cache of keys and values in pages: what its operators
// (rope.hip, paged_attention.hip) share.
//
// A pool holds pages of `page` tokens; row b of the table gives the pages of sequence
// b's tokens in order, and lengths[b] the tokens that it has.
#pragma once

#include "op_checks.h"

namespace trs {

constexpr int64_t kMaxPagedTokens = (int64_t)1 << 29;  // of a sequence

struct PoolView {  // [page, key head, token of the page], unit stride along dim
    int64_t h;
    uint32_t p, s;
    __device__ __forceinline__ uint64_t at(int page, int slot) const { return (uint64_t)(uint32_t)page * p + (uint64_t)(uint32_t)slot * s; }
};

// The cache as kernels see it.
struct Pages {
    void *k, *v;
    PoolView ks, vs;
    const int32_t *table, *lengths;
    int32_t pages, page, width, capacity;  // capacity: tokens that a row of the table holds
    SmallDivisor by_page;

    __device__ __forceinline__ int keys_of(int b) const { return min(max(lengths[b], 0), capacity); }
    // The page of a sequence's token at `place`, in [0, capacity): outside [0, pages) if the table holds no page for it.
    __device__ __forceinline__ int page_of(int b, int place) const { return table[(int64_t)b * width + (int)by_page.divide((uint32_t)place)]; }
    __device__ __forceinline__ int slot_of(int place) const { return place - (int)by_page.divide((uint32_t)place) * page; }
    __device__ __forceinline__ bool holds(int id) const { return (uint32_t)id < (uint32_t)pages; }
};

inline int page_bytes(const trs_paged_cache *c) { return c->type == TRS_PAGES_BF16 ? 2 : 4; }

// Checks a cache for `batch` sequences and fills in what kernels need of it.
inline int check_cache(const trs_paged_cache *c, int64_t batch, Pages *out) {
    if (!c) return set_error(TRS_E_INVALID_ARGUMENT, "paged cache is null");
    if (c->type != TRS_PAGES_F32 && c->type != TRS_PAGES_BF16) return set_error(TRS_E_INVALID_ARGUMENT, "paged cache has pages of type %d", c->type);
    const char *const names[2] = {"key pages", "value pages"};
    const trs_layout *const layouts[2] = {&c->lk, &c->lv};
    for (int i = 0; i < 2; i++) {
        const trs_layout *l = layouts[i];
        TRS_CHECK(check_layout(l, names[i]));
        if (l->rank != 4) return set_error(TRS_E_INVALID_ARGUMENT, "%s have rank %d, not 4 (page, key head, token, dim)", names[i], l->rank);
        for (int d = 0; d < 4; d++)
            if (l->shape[d] != c->lk.shape[d]) return set_error(TRS_E_SHAPE_MISMATCH, "key pages and value pages differ in dim %d", d);
        if (l->shape[3] > 1 && l->stride[3] != 1) return set_error(TRS_E_INVALID_ARGUMENT, "%s need a unit stride along their last dim", names[i]);
        if (l->stride[0] > INT32_MAX || l->stride[2] > INT32_MAX)
            return set_error(TRS_E_INDEX_OVERFLOW, "%s have a stride of 2^31 entries or more from page to page or token to token", names[i]);
        if (layout_numel(l) > 0 && !(i ? c->v : c->k)) return set_error(TRS_E_INVALID_ARGUMENT, "%s are null", names[i]);
    }
    const int64_t pages = c->lk.shape[0], page = c->lk.shape[2];
    if (c->table_width < 0) return set_error(TRS_E_INVALID_ARGUMENT, "page table has a width of %lld", (long long)c->table_width);
    if (page < 1) return set_error(TRS_E_INVALID_ARGUMENT, "pages hold no token");
    if (pages > INT32_MAX || page > kMaxPagedTokens || c->table_width > kMaxPagedTokens / page)
        return set_error(TRS_E_INDEX_OVERFLOW, "a paged cache of more than 2^31 pages, or of more than 2^29 tokens a sequence");
    if (pages == 0 && c->table_width > 0) return set_error(TRS_E_INVALID_ARGUMENT, "paged cache has no pages");
    if (batch > 0 && !c->lengths) return set_error(TRS_E_INVALID_ARGUMENT, "lengths are null");
    if (batch > 0 && c->table_width > 0 && !c->table) return set_error(TRS_E_INVALID_ARGUMENT, "page table is null");
    const int size = page_bytes(c);
    out->k = c->k ? (char *)c->k + c->lk.offset * size : nullptr;
    out->v = c->v ? (char *)c->v + c->lv.offset * size : nullptr;
    out->ks = {c->lk.stride[1], (uint32_t)c->lk.stride[0], (uint32_t)c->lk.stride[2]};
    out->vs = {c->lv.stride[1], (uint32_t)c->lv.stride[0], (uint32_t)c->lv.stride[2]};
    out->table = c->table, out->lengths = c->lengths;
    out->pages = (int32_t)pages, out->page = (int32_t)page, out->width = (int32_t)c->table_width;
    out->capacity = (int32_t)(page * c->table_width);
    out->by_page = SmallDivisor((uint32_t)page);
    return TRS_OK;
}

// The pools share no memory with another operand of a call (which counts as a whole range here), nor, where
// they are written, with each other or themselves.
template <int N>
int check_pools(const trs_paged_cache *c, bool written, const Operand (&ops)[N]) {
    if (layout_numel(&c->lk) == 0) return TRS_OK;
    const int size = page_bytes(c);
    const ByteRange pools[2] = {byte_range(c->k, &c->lk, size), byte_range(c->v, &c->lv, size)};
    if (written) {
        TRS_CHECK(check_written_once(&c->lk, "key pages"));
        TRS_CHECK(check_written_once(&c->lv, "value pages"));
        if (ranges_overlap(pools[0], pools[1]) && may_share(pools[0].begin, &c->lk, pools[1].begin, &c->lv, size))
            return set_error(TRS_E_INVALID_ARGUMENT, "key pages overlap value pages");
    }
    for (const Operand &o : ops) {
        if (!(written || o.written) || (o.layout ? layout_numel(o.layout) : o.count) == 0) continue;
        const uintptr_t at = (uintptr_t)o.ptr;
        const ByteRange r = o.layout ? byte_range(o.ptr, o.layout, 4) : ByteRange{at, at + (uintptr_t)o.count * 4};
        for (int i = 0; i < 2; i++)
            if (ranges_overlap(r, pools[i])) return set_error(TRS_E_INVALID_ARGUMENT, "%s overlaps %s pages", o.name, i ? "value" : "key");
    }
    return TRS_OK;
}

}  // namespace trs
