// tl_paged_attn.cuh -- arguments and device pieces of the paged attention
// kernels (tl_paged_attn.cu, tl_paged_attn_tc.cu).
#pragma once

#include <math.h>

#include "tl_paged.cuh"

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

// The query rows of sequence b, cut to the rows that exist.
__device__ __forceinline__ void rows_of(const AttendArgs& a, int b, int& first, int& n) {
    first = min(max(a.q_start[b], 0), a.n_tokens);
    n = max(0, min(a.q_start[b + 1], a.n_tokens) - first);
}

// The sequence that row t belongs to, -1 if none.
__device__ __forceinline__ int sequence_of(const AttendArgs& a, int t) {
    int lo = 0, hi = a.n_seq;  // largest b with q_start[b] <= t
    if (t < a.q_start[0]) return -1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.q_start[mid] <= t) lo = mid;
        else hi = mid;
    }
    return t < a.q_start[lo + 1] ? lo : -1;
}

// Positions [lo, hi) that the query at position p of sequence b may attend to
// (pages that do not exist are left out later, key by key).
__device__ __forceinline__ void attended(const AttendArgs& a, long long p, int& lo, int& hi) {
    hi = static_cast<int>(min(p + 1, static_cast<long long>(a.max_blocks) << a.shift));
    lo = a.window > 0 ? static_cast<int>(max(0ll, p + 1 - a.window)) : 0;
}

// One (token, head) by one warp, straight from the pages in fp32: lane l holds
// dims l * HD / 32 ...  Reads the attended keys only.
template <typename T, int HD>
__device__ void attend_row(const AttendArgs& a, int b, int t, int h, int lane) {
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
        const int id = a.table[static_cast<size_t>(b) * a.max_blocks + (j >> a.shift)];
        if (id < 0 || id >= a.n_blocks) continue;
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

}  // namespace paged
}  // namespace tl
