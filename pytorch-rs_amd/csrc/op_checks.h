// op_checks.h -- argument checks and device helpers shared by the attention
// block's operators (dropout.hip, head_norm.hip, attention*.hip).
#pragma once

#include <algorithm>

#include "trs_internal.h"

namespace trs {

typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));  // 16 bytes at any float

// Checks that an output layout writes each of its elements once.
inline int check_written_once(const trs_layout *l, const char *what) {
    int order[TRS_MAX_RANK], n = 0;
    for (int d = 0; d < l->rank; d++) {
        if (l->shape[d] == 0) return TRS_OK;
        if (l->shape[d] > 1) order[n++] = d;
    }
    std::sort(order, order + n, [&](int x, int y) { return l->stride[x] < l->stride[y]; });
    int64_t reach = 0;  // the last offset of the dims so far
    for (int i = 0; i < n; i++) {
        const int d = order[i];
        if (l->stride[d] <= reach) return set_error(TRS_E_INVALID_ARGUMENT, "%s layout overlaps itself", what);
        reach += (l->shape[d] - 1) * l->stride[d];
    }
    return TRS_OK;
}

// Whether two views of elements of `size` bytes, whose first are at a and b, may share a byte.  Where both
// have their largest stride in common, what lies within a step of one is compared with what lies
// within the steps of the other that are beside it, as far as the strides agree (slices of one
// buffer); from there on views count as whole ranges.
inline bool may_share(uintptr_t a, const trs_layout *la, uintptr_t b, const trs_layout *lb, int64_t size = 4) {
    struct Dims {
        int64_t count[TRS_MAX_RANK], stride[TRS_MAX_RANK], reach[TRS_MAX_RANK + 1];  // largest first; reach: of the dims from here on
        int n = 0;
        explicit Dims(const trs_layout *l) {
            for (int d = 0; d < l->rank; d++) {
                if (l->shape[d] <= 1 || l->stride[d] == 0) continue;
                int i = n++;
                for (; i > 0 && stride[i - 1] < l->stride[d]; i--) count[i] = count[i - 1], stride[i] = stride[i - 1];
                count[i] = l->shape[d], stride[i] = l->stride[d];
            }
            reach[n] = 0;
            for (int i = n; i-- > 0;) reach[i] = reach[i + 1] + (count[i] - 1) * stride[i];
        }
    };
    const Dims x(la), y(lb);
    // b's dims from j on against a's from i on, b's first element `apart` bytes behind a's.
    const auto meet = [&](auto &&self, int i, int j, int64_t apart) -> bool {
        if (apart >= (x.reach[i] + 1) * size || -apart >= (y.reach[j] + 1) * size) return false;
        if (i == x.n || j == y.n || x.stride[i] != y.stride[j]) return true;
        // Step s of a's dim and t of b's, for every k = s - t at which what lies within them may meet.
        const int64_t pitch = x.stride[i] * size;
        const int64_t first = std::max((apart - (x.reach[i + 1] + 1) * size) / pitch - 1, 1 - y.count[j]);
        const int64_t last = std::min((apart + (y.reach[j + 1] + 1) * size) / pitch + 1, x.count[i] - 1);
        if (last - first > 8) return true;  // neither holds its steps apart
        for (int64_t k = first; k <= last; k++)
            if (self(self, i + 1, j + 1, apart - k * pitch)) return true;
        return false;
    };
    return meet(meet, 0, 0, (int64_t)(b - a));
}

// An operand of a call, as the overlap check sees it.
struct Operand {
    const char *name;
    const void *ptr;
    const trs_layout *layout;  // null: `count` contiguous elements
    bool written;
    int64_t count = 0;
};

// Every operand with elements has memory, and what is written shares none with
// another operand.
template <int N>
int check_memory(const Operand (&ops)[N]) {
    ByteRange r[N];
    trs_layout counted{};
    counted.rank = 1, counted.stride[0] = 1;
    for (int i = 0; i < N; i++) {
        const Operand &o = ops[i];
        if ((o.layout ? layout_numel(o.layout) : o.count) == 0) continue;
        if (!o.ptr) return set_error(TRS_E_INVALID_ARGUMENT, "%s is null", o.name);
        counted.shape[0] = o.count;
        r[i] = byte_range(o.ptr, o.layout ? o.layout : &counted, 4);
    }
    const auto share = [&](int i, int j) {
        trs_layout of_i = counted, of_j = counted;
        of_i.shape[0] = ops[i].count, of_j.shape[0] = ops[j].count;
        return may_share(r[i].begin, ops[i].layout ? ops[i].layout : &of_i, r[j].begin, ops[j].layout ? ops[j].layout : &of_j);
    };
    for (int i = 0; i < N; i++)
        for (int j = 0; j < N; j++)
            if (i != j && ops[i].written && r[i].begin < r[i].end && r[j].begin < r[j].end && ranges_overlap(r[i], r[j]) && share(i, j))
                return set_error(TRS_E_INVALID_ARGUMENT, "%s overlaps %s", ops[i].name, ops[j].name);
    return TRS_OK;
}

// r / d for r below 2^31 by a multiplication: with s = ceil(log2 d) and
// m = ceil(2^(31+s) / d), m d exceeds 2^(31+s) by less than 2^s, so r m is off
// by less than one part in 2^(31+s) of a whole.
struct SmallDivisor {
    uint32_t d = 1, m = 1u << 31, s = 31;
    SmallDivisor() = default;
    explicit SmallDivisor(uint32_t divisor) : d(divisor) {
        uint32_t l = 0;
        while ((1ull << l) < d) l++;
        s = 31 + l;
        m = (uint32_t)(((1ull << s) + d - 1) / d);
    }
    __host__ __device__ __forceinline__ uint32_t divide(uint32_t r) const { return (uint32_t)((uint64_t)r * m >> s); }
};

}  // namespace trs
