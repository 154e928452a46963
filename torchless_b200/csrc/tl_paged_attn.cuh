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

// ---- division of a call's work among the blocks -----------------------------
// The steps of all tiles lie in one line: sequence by sequence, row tile by row
// tile, kv head by kv head.  Block i takes the steps [i * per, (i + 1) * per).
// `Plan` says how many rows a tile has (R) and how many steps.

// What a block leaves behind of a tile that it begins and others end.
struct Head {
    int parts, slot, b, rt, g;
};
constexpr int kMaxBlocks = 512;
constexpr size_t kHeadBytes = 16384;  // heads of up to kMaxBlocks blocks
static_assert(sizeof(Head) * kMaxBlocks <= kHeadBytes, "heads");

// Place in the line: tile (b, rt, g) and the steps [s, end) of it that belong to this block.
struct Cursor {
    int b, rt, g;
    int s, end, steps;
    long long left;  // steps of the block from this tile's step s on
    Tile t;
};

template <class Plan>
__device__ __forceinline__ void enter(const AttendArgs& a, Cursor& c) {
    c.t = tile_of(a, c.b, c.rt, Plan::R);
    c.steps = Plan::steps(c.t);
    c.end = static_cast<int>(min(static_cast<long long>(c.steps), c.s + c.left));
}
// To the next tile that has rows; false when the block's share is done.
template <class Plan>
__device__ __forceinline__ bool next_tile(const AttendArgs& a, Cursor& c) {
    c.left -= c.end - c.s;
    if (c.left <= 0) return false;
    c.s = 0;
    if (++c.g == a.KV) {
        c.g = 0;
        c.rt++;
        while (c.rt * Plan::R >= c.t.n * a.group) {  // sequences without rows have no steps
            if (++c.b >= a.n_seq) return false;
            c.rt = 0;
            rows_of(a, c.b, c.t.first, c.t.n);
        }
    }
    enter<Plan>(a, c);
    return true;
}

// Exclusive running sum over the block's NW warps; `total` gets the sum.
template <int NW>
__device__ __forceinline__ long long scan_block(long long v, long long* ws, long long& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(FULL, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) ws[warp] = x;
    __syncthreads();
    long long before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < NW; w++) {
        if (w < warp) before += ws[w];
        sum += ws[w];
    }
    total = sum;
    return x - v + before;
}

template <class Plan>
__device__ __forceinline__ long long steps_of_sequence(const AttendArgs& a, int b) {
    if (b >= a.n_seq) return 0;
    int first, n;
    rows_of(a, b, first, n);
    long long u = 0;
    for (int rt = 0; rt * Plan::R < n * a.group; rt++) u += Plan::steps(tile_of(a, b, rt, Plan::R));
    return u * a.KV;
}

// This block's share: `c` at its first tile; returns the steps of a full share, 0 if there is nothing
// for this block.  All NW warps call it.  ws: [NW], found: [1], in shared memory.
template <class Plan, int NW>
__device__ long long find_share(const AttendArgs& a, Cursor& c, long long* ws, int* found, int least) {
    constexpr int NT = NW * 32;
    long long total = 0;
    const long long mine = steps_of_sequence<Plan>(a, threadIdx.x);
    const long long at0 = scan_block<NW>(mine, ws, total);
    const long long chunk0 = total;
    if (a.n_seq > NT) {  // the rest of the sequences: their sum first
        long long rest = 0, sum;
        for (int b = NT + threadIdx.x; b < a.n_seq; b += NT) rest += steps_of_sequence<Plan>(a, b);
        scan_block<NW>(rest, ws, sum);
        total += sum;
    }
    const long long per = max((total + gridDim.x - 1) / gridDim.x, static_cast<long long>(least));
    const long long u0 = per * blockIdx.x;
    if (u0 >= total) return 0;
    if (threadIdx.x == 0) *found = -1;
    __syncthreads();
    auto place = [&](int b, long long at, long long n) {
        if (u0 >= at && u0 < at + n) {
            *found = b;
            ws[0] = u0 - at;
        }
    };
    if (u0 < chunk0) {
        place(threadIdx.x, at0, mine);
    } else {
        long long before = chunk0;
        for (int b0 = NT; b0 < a.n_seq; b0 += NT) {
            const long long n = steps_of_sequence<Plan>(a, b0 + threadIdx.x);
            long long sum;
            const long long at = before + scan_block<NW>(n, ws, sum);
            __syncthreads();
            if (u0 < before + sum) {
                place(b0 + threadIdx.x, at, n);
                break;
            }
            before += sum;
        }
    }
    __syncthreads();
    if (*found < 0) return 0;  // (the lengths changed under the call)
    c.b = *found;
    c.rt = 0;
    c.left = min(per, total - u0);
    long long u = ws[0];
    for (;; c.rt++) {
        c.t = tile_of(a, c.b, c.rt, Plan::R);
        c.steps = Plan::steps(c.t);
        if (u < static_cast<long long>(c.steps) * a.KV) break;
        u -= static_cast<long long>(c.steps) * a.KV;
    }
    c.g = static_cast<int>(u / c.steps);
    c.s = static_cast<int>(u % c.steps);
    c.end = static_cast<int>(min(static_cast<long long>(c.steps), c.s + c.left));
    return per;
}
// The number of blocks that share a tile whose first block ends at step `end` of `steps`.
__device__ __forceinline__ int parts_of(int steps, int end, long long per) {
    return 1 + static_cast<int>((steps - end + per - 1) / per);
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
// panels, pages}; a box is `rows` rows of `panels` panels of one page, zero where the page does not
// exist.  16-bit types: panels of 64 columns, SWIZZLE_128B; fp32: one panel, no swizzle.
tl_status encode_pages(CUtensorMap* map, const void* base, const tl_paged_cache* c, int rows, int panels);

// Few query rows per sequence (tl_paged_attn.cu), and many (tl_paged_attn_tc.cu; not fp32).
size_t split_workspace(int hd);
tl_status attend_split(const AttendArgs& a, const tl_paged_cache* c, void* workspace, cudaStream_t s);
size_t chunk_workspace(int hd);
tl_status attend_chunk(const AttendArgs& a, const tl_paged_cache* c, void* workspace, cudaStream_t s);

}  // namespace paged
}  // namespace tl
