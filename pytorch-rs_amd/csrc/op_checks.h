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
    for (int i = 0; i < N; i++) {
        const Operand &o = ops[i];
        if ((o.layout ? layout_numel(o.layout) : o.count) == 0) continue;
        if (!o.ptr) return set_error(TRS_E_INVALID_ARGUMENT, "%s is null", o.name);
        r[i] = o.layout ? byte_range(o.ptr, o.layout, 4)
                        : ByteRange{(uintptr_t)o.ptr, (uintptr_t)o.ptr + (uintptr_t)o.count * 4};
    }
    for (int i = 0; i < N; i++)
        for (int j = 0; j < N; j++)
            if (i != j && ops[i].written && r[i].begin < r[i].end && r[j].begin < r[j].end && ranges_overlap(r[i], r[j]))
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
