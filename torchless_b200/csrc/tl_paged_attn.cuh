// tl_paged_attn.cuh -- arguments and device pieces of the paged attention
// kernels (tl_paged_attn.cu, tl_paged_attn_tc.cu).
#pragma once

#include <math.h>

#include "tl_paged.cuh"
#include "tl_tc.cuh"

namespace tl {
namespace paged {

struct AttendArgs {
    void* out;           // [n_tokens][H][hd]
    const void* q;       // rows q_stride elements apart
    const void* k;       // pages, block_stride elements apart
    const void* v;
    const int32_t* table;     // [n_seq][max_blocks]
    const int32_t* q_start;   // [n_seq + 1]
    const int32_t* seq_lens;  // [n_seq]
    size_t q_stride, block_stride;
    int n_seq, n_tokens, H, KV, group, max_blocks, n_blocks, shift;  // block size 1 << shift
    int window;   // 0: none
    float scale;
};

// 2^x (hardware approximation, 2 ulp; 2^-inf = +0)
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The query rows of sequence b, cut to the rows that exist.
__device__ __forceinline__ void rows_of(const AttendArgs& a, int b, int& first, int& n) {
    first = min(max(a.q_start[b], 0), a.n_tokens);
    n = max(0, min(a.q_start[b + 1], a.n_tokens) - first);
}

// Positions [lo, hi) that the query at position p of a sequence may attend to
// (pages that do not exist are left out later, key by key).
__device__ __forceinline__ void attended(const AttendArgs& a, long long p, int& lo, int& hi) {
    hi = static_cast<int>(min(p + 1, static_cast<long long>(a.max_blocks) << a.shift));
    lo = a.window > 0 ? static_cast<int>(max(0ll, p + 1 - a.window)) : 0;
}

// The page of position key of sequence b; -1 if there is none.
__device__ __forceinline__ int page_of(const AttendArgs& a, int b, int key) {
    const int j = key >> a.shift;
    if (key < 0 || j >= a.max_blocks) return -1;
    const int id = a.table[static_cast<size_t>(b) * a.max_blocks + j];
    return id >= 0 && id < a.n_blocks ? id : -1;
}

// A tile of `rows` query rows of one kv head: row r of sequence b is its token
// r / group, q head g * group + r % group, so that all heads that share a kv
// head lie in one tile with their tokens, whatever the group.
struct Tile {
    int first, n;        // the sequence's token rows
    int r0, nrows;       // rows of the tile
    long long p0;        // position of the sequence's first token row
    int lo, lo_last;     // first attended position of the tile's first and last token
    int hi, hi_first;    // end of the attended positions of the last and first token
};
__device__ __forceinline__ Tile tile_of(const AttendArgs& a, int b, int rt, int rows) {
    Tile t;
    rows_of(a, b, t.first, t.n);
    t.r0 = rt * rows;
    t.nrows = min(rows, t.n * a.group - t.r0);
    t.p0 = static_cast<long long>(a.seq_lens[b]) - t.n;
    attended(a, t.p0 + t.r0 / a.group, t.lo, t.hi_first);
    attended(a, t.p0 + (t.r0 + t.nrows - 1) / a.group, t.lo_last, t.hi);
    return t;
}

// One (token, head) by one warp, straight from the pages in fp32: lane l holds
// dims l * HD / 32 ...  Reads the attended keys only.
template <typename T, int HD>
__device__ __noinline__ void attend_row(const AttendArgs& a, int b, int t, int h, int lane) {
    constexpr int D = HD / 32;
    int first, n;
    rows_of(a, b, first, n);
    const long long p = static_cast<long long>(a.seq_lens[b]) - n + (t - first);
    int lo, hi;
    attended(a, p, lo, hi);
    const int g = h / a.group;
    const T* qp = static_cast<const T*>(a.q) + static_cast<size_t>(t) * a.q_stride + static_cast<size_t>(h) * HD + lane * D;
    float q[D], acc[D];
#pragma unroll
    for (int d = 0; d < D; d++) {
        q[d] = to_f32<T>(qp[d]);
        acc[d] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int j = lo; j < hi; j++) {
        const int id = page_of(a, b, j);
        if (id < 0) continue;
        const size_t at = static_cast<size_t>(id) * a.block_stride +
                          ((static_cast<size_t>(g) << a.shift) + (j & ((1 << a.shift) - 1))) * HD + lane * D;
        const T* kp = static_cast<const T*>(a.k) + at;
        const T* vp = static_cast<const T*>(a.v) + at;
        float s = 0.f;
#pragma unroll
        for (int d = 0; d < D; d++) s += q[d] * to_f32<T>(kp[d]);
        s = warp_sum(s) * a.scale;
        const float mn = fmaxf(m, s);
        const float f = m == -INFINITY ? 1.f : expf(m - mn);
        const float e = s == -INFINITY ? 0.f : expf(s - mn);  // NaN stays NaN
        m = mn;
        l = l * f + e;
#pragma unroll
        for (int d = 0; d < D; d++) acc[d] = acc[d] * f + e * to_f32<T>(vp[d]);
    }
    T* op = static_cast<T*>(a.out) + (static_cast<size_t>(t) * a.H + h) * HD + lane * D;
#pragma unroll
    for (int d = 0; d < D; d++) op[d] = from_f32<T>(l != 0.f ? acc[d] / l : 0.f);
}

// Map of one side (K or V) of the pages: {64 or hd columns, rows of all kv heads, column
// panels, pages}; a box is `rows` rows of every panel of one page, zero where the page does not exist.
// 16-bit types: panels of 64 columns, SWIZZLE_128B; fp32: one panel, no swizzle.
tl_status encode_pages(CUtensorMap* map, const void* base, const tl_paged_cache* c, int rows);

// Work of few query rows per sequence (tl_paged_attn.cu) and of many (tl_paged_attn_tc.cu).
size_t split_workspace(int hd);
tl_status attend_split(const AttendArgs& a, const tl_paged_cache* c, void* workspace, cudaStream_t s);

}  // namespace paged
}  // namespace tl
