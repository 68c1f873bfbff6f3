// attention_backward.hip -- the gradients of attention.h's attention: their host part,
// and what comes before and after the products.
//
// With P = exp(scale Q K^T - lse) over the pairs that see each other and
// delta = rowsum(dO o):
//   dS = P (dO V^T - delta),  dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO.
// P and dO V^T are worked out twice, over rows for dQ and over keys for dK and dV (seven
// products where one walk would take five), so that every sum has one owner and a fixed
// order: no atomic adds, the same bits each time.
//
// Pairs that only the sinks make visible (first keys, far rows) go to blocks of their
// own: their keys are seen by every later row, the other keys by a window of rows.  What
// these blocks sum, in parts, is added by attn_reduce.
#include <hip/hip_runtime.h>

#include "attention.h"

namespace trs {

namespace {

// The least row tiles of a part: 333 tokens, 4 heads of 32 57.8 us with 8, 34.5 with 4, 33.2 with 2
// (2 x 2048 tokens, whose parts are longer, alike).
constexpr int kPartTiles = 2;

// delta of every row: 16 lanes a row.
__global__ void __launch_bounds__(256) attn_delta(AttnArgs a, float *delta) {
    const int64_t rows = (int64_t)a.batch * a.heads * a.Sq;
    const int sub = (int)threadIdx.x & 15;
    const int64_t r = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    float s = 0.f;
    if (r < rows) {
        const int64_t bh = r / a.Sq, i = r - bh * a.Sq, b = bh / a.heads, h = bh - b * a.heads;
        const float *o = a.out + b * a.os.b + h * a.os.h + i * a.os.s, *u = a.up + b * a.us.b + h * a.us.h + i * a.us.s;
        for (int d = sub * 4; d < a.D; d += 64) {
            const at_f4 x = row_chunk(o, d, a.D), y = row_chunk(u, d, a.D);
#pragma unroll
            for (int e = 0; e < 4; e++) s += x[e] * y[e];
        }
    }
#pragma unroll
    for (int d = 1; d < 16; d *= 2) s += __shfl_xor(s, d);
    if (r < rows && sub == 0) delta[r] = s;
}

// dk and dv of the first `count` keys: the parts over the rows, or what the one part
// wrote, and the sinks' `far` parts of tiles of `tile` keys, in a fixed order.  Eight parts
// are read at a time: one memory latency for all of them.
__global__ void __launch_bounds__(256) attn_reduce(AttnArgs a, int count, int tile, int far) {
    const int64_t heads = (int64_t)a.batch * a.kv_heads, n = heads * count * a.D;
    const auto add = [](float &x, float &y, const float *px, const float *py, int64_t step, int parts) {
        for (int p = 0; p < parts; p += 8) {
            float u[8], w[8];
#pragma unroll
            for (int q = 0; q < 8; q++) {
                const int64_t at = min(p + q, parts - 1) * step;
                u[q] = px[at], w[q] = py[at];
            }
#pragma unroll
            for (int q = 0; q < 8; q++)
                if (p + q < parts) x += u[q], y += w[q];
        }
    };
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < n; e += (int64_t)gridDim.x * 256) {
        const int64_t row = e / a.D, head = row / count;
        const int d = (int)(e - row * a.D), key = (int)(row - head * count), hk = (int)(head % a.kv_heads);
        const int64_t b = head / a.kv_heads;
        float *dk = a.dk + b * a.dks.b + hk * a.dks.h + (int64_t)key * a.dks.s + d;
        float *dv = a.dv + b * a.dvs.b + hk * a.dvs.h + (int64_t)key * a.dvs.s + d;
        float x = 0.f, y = 0.f;
        if (a.row_splits > 1) {
            const int64_t at = (head * a.Sk + key) * a.D + d;
            add(x, y, a.part_k + at, a.part_v + at, heads * a.Sk * a.D, a.row_splits);
        } else {
            x = *dk, y = *dv;
        }
        if (far && key < a.sinks) {
            const int64_t at = (((head * a.sink_tiles + key / tile) * far) * tile + key % tile) * a.D + d;
            add(x, y, a.sink_k + at, a.sink_v + at, (int64_t)tile * a.D, far);
        }
        *dk = x, *dv = y;
    }
}

}  // namespace

int attention_backward(AttnArgs a, hipStream_t s, int cu_count) {
    const int64_t heads = (int64_t)a.batch * a.kv_heads;
    // In pieces: blocks of 128 rows or keys, tiles of 32.  Wide heads: waves of 16, tiles of 16,
    // four waves a block.
    const bool wide = a.D > kPiecesDim;
    const int block = wide ? 16 : kRowsBlock, tile = wide ? 16 : kTile;
    const int64_t room = (wide ? 8 : 2) * (int64_t)cu_count;  // blocks or waves that the device is to have
    a.row_tiles = (a.rows + block - 1) / block;
    a.key_tiles = (a.Sk + block - 1) / block;
    // The rows that see a key tile in parts where the tiles are few for the CUs.
    const int64_t near_tiles = std::max<int64_t>(1, std::min<int64_t>(a.rows, ((int64_t)a.window + block) * a.group) / tile);
    a.row_splits = 1;
    if (a.key_tiles)
        a.row_splits = (int32_t)std::max<int64_t>(1, std::min<int64_t>({room / (heads * a.key_tiles), near_tiles / kPartTiles, 16}));
    // Rows beyond a window see sinks alone: in parts of about as many row tiles as the others.
    a.sink_tiles = a.window < a.Sk ? (std::min(a.sinks, a.Sk) + block - 1) / block : 0;
    a.sink_splits = 1;
    if (a.sink_tiles)
        a.sink_splits = (int32_t)std::max<int64_t>(1, std::min<int64_t>(64, std::max<int64_t>(1, a.rows / tile) * a.row_splits / near_tiles));
    const int far = a.sink_tiles ? a.sink_splits : 0;
    const int64_t row_blocks = heads * a.row_tiles;
    const int64_t key_blocks = heads * (a.sink_tiles * a.sink_splits + (int64_t)a.key_tiles * a.row_splits);
    const int64_t delta_blocks = ((int64_t)a.batch * a.heads * a.Sq + 15) / 16;
    if ((row_blocks + key_blocks) >> 24 || delta_blocks >> 24)  // a launch has fewer than 2^32 lanes
        return set_error(TRS_E_INVALID_ARGUMENT, "attention gradient over too many blocks");
    const int64_t deltas = ((int64_t)a.batch * a.heads * a.Sq + 63) / 64 * 64;
    const int64_t sink_floats = heads * a.sink_tiles * far * block * a.D;
    const int64_t part_floats = a.row_splits > 1 ? heads * a.row_splits * a.Sk * a.D : 0;
    void *ws = nullptr;
    TRS_CHECK(trs_alloc((size_t)(deltas + 2 * sink_floats + 2 * part_floats) * sizeof(float), &ws));
    float *delta = (float *)ws;
    a.delta = delta;
    a.sink_k = delta + deltas, a.sink_v = a.sink_k + sink_floats;
    a.part_k = a.sink_v + sink_floats, a.part_v = a.part_k + part_floats;
    const auto launch = [&]() -> int {
        // No rows: the keys' gradients are 0.  No keys: the rows' are.
        if (delta_blocks) hipLaunchKernelGGL(attn_delta, dim3((unsigned)delta_blocks), dim3(256), 0, s, a, delta);
        TRS_LAUNCH_CHECK("attention gradient launch");
        if (key_blocks + row_blocks) {
            if (wide) launch_attention_grad_wide(a, (uint32_t)key_blocks, (uint32_t)row_blocks, s);
            else launch_attention_grad(a, (uint32_t)key_blocks, (uint32_t)row_blocks, s);
            TRS_LAUNCH_CHECK("attention gradient launch");
        }
        const int count = a.row_splits > 1 ? a.Sk : a.sink_tiles ? std::min(a.sinks, a.Sk) : 0;
        if (count) {
            const int64_t n = heads * count * a.D;
            hipLaunchKernelGGL(attn_reduce, dim3((unsigned)std::min<int64_t>((n + 255) / 256, 1 << 20)), dim3(256), 0, s, a, count, block, far);
            TRS_LAUNCH_CHECK("attention gradient launch");
        }
        return TRS_OK;
    };
    const int rc = launch(), frc = trs_free(ws);
    return rc ? rc : frc;
}

}  // namespace trs
