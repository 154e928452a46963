// tl_paged_attn.cuh -- arguments and device pieces of the paged attention
// kernels (tl_paged_attn.cu, tl_paged_attn_tc.cu).
#pragma once

#include <math.h>

#include "tl_paged.cuh"
#include "tl_tc.cuh"

namespace tl {
namespace paged {

constexpr int kMaxLen = 0x7fff0000;  // longer lengths count as this one

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
    int cap;      // positions that a table can name, at most kMaxLen
    int window;   // 0: none; below 2^30, so that no difference of it and a position passes 32 bits
    float scale;
    unsigned long long group_inv;  // ceil(2^64 / group)
    unsigned fail_one_in;  // 0; for tests: about one in so many waits gives up at once, as all do after about 2 s
};
__device__ __forceinline__ bool told_to_fail(unsigned one_in) {
    return ((static_cast<unsigned>(clock()) + 977u * blockIdx.x) * 2654435761u >> 8) % one_in == 0;
}

// r / group, r >= 0 (exact: r < 2^32, and the inverse is off by less than 2^-32 relative)
__device__ __forceinline__ int div_group(const AttendArgs& a, int r) {
    return a.group == 1 ? r : static_cast<int>(__umul64hi(static_cast<unsigned long long>(r), a.group_inv));
}

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

// Position of the first query row of a sequence with n of them.  (A length below 0 leaves all of them before position 0, as
// 0 does, and less n it could pass the smallest whole number.)
__device__ __forceinline__ int first_pos(const AttendArgs& a, int b, int n) { return min(max(a.seq_lens[b], 0), kMaxLen) - n; }

// Positions [lo, hi) that the query at position p of a sequence may attend to
// (pages that do not exist are left out later, key by key).
__device__ __forceinline__ void attended(const AttendArgs& a, int p, int& lo, int& hi) {
    hi = min(p + 1, a.cap);
    lo = a.window > 0 ? max(0, p + 1 - a.window) : 0;
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
    int p0;              // position of the sequence's first token row
    int lo, lo_last;     // first attended position of the tile's first and last token
    int hi, hi_first;    // end of the attended positions of the last and first token
};
__device__ __forceinline__ Tile tile_of(const AttendArgs& a, int b, int rt, int rows) {
    Tile t;
    rows_of(a, b, t.first, t.n);
    t.r0 = rt * rows;
    t.nrows = min(rows, t.n * a.group - t.r0);
    t.p0 = first_pos(a, b, t.n);
    attended(a, t.p0 + div_group(a, t.r0), t.lo, t.hi_first);
    attended(a, t.p0 + div_group(a, max(0, t.r0 + t.nrows - 1)), t.lo_last, t.hi);
    return t;
}

// ---- division of a call's work among the blocks -----------------------------
// The steps of all tiles lie in one line: sequence by sequence, row tile by row
// tile, kv head by kv head.  Block i takes the steps [i * per, (i + 1) * per).
// `Plan` says how many rows a tile has (R) and how many steps, and (kLookAgain) whether a tile's lengths are looked up
// again for the next kv head.  That only costs time (8192 tokens bf16: 614 us against 602, 130 short sequences 42.4 against
// 41.3), but some kernels' registers come out better with it (2048 tokens of 4096 fp32 2.47 ms against 2.61, decode 64 x
// 4096 bf16 hd 64 94.2 us against 96.2; decode fp32 333 us both ways).

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
    int left;  // steps of the block from this tile's step s on
    Tile t;
};

// To the next tile that has rows; false when the block's share is done.
template <class Plan>
__device__ __forceinline__ bool next_tile(const AttendArgs& a, Cursor& c) {
    c.left -= c.end - c.s;
    if (c.left <= 0) return false;
    c.s = 0;
    const bool same = ++c.g < a.KV;  // the same rows of the next kv head
    if (!same) {
        c.g = 0;
        c.rt++;
        while (c.rt * Plan::R >= c.t.n * a.group) {  // sequences without rows have no steps
            if (++c.b >= a.n_seq) return false;
            c.rt = 0;
            rows_of(a, c.b, c.t.first, c.t.n);
        }
    }
    if (!same || Plan::kLookAgain) {
        c.t = tile_of(a, c.b, c.rt, Plan::R);
        c.steps = Plan::steps(c.t);
    }
    c.end = min(c.steps, c.left);
    return true;
}

// Exclusive running sum over the block's NW warps; `total` gets the sum.  (Loops are not unrolled in what a block
// does once: every instruction's first execution waits for its code.)
template <int NW>
__device__ __noinline__ long long scan_block(long long v, long long* ws, long long& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long mine = v, base = 0, sum = 0;
#pragma unroll 1
    for (int turn = 0; turn < 2; turn++) {  // over the lanes, then over the warps
        long long c = mine;
#pragma unroll 1
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(FULL, c, o);
            if (lane >= o) c += y;
        }
        if (turn == 0) {
            base = c - mine;
            __syncthreads();
            if (lane == 31) ws[warp] = c;
            __syncthreads();
            mine = lane < NW ? ws[lane] : 0;
        } else {
            sum = c;
        }
    }
    total = __shfl_sync(FULL, sum, 31);
    const long long up = __shfl_sync(FULL, sum, warp ? warp - 1 : 0);
    return base + (warp ? up : 0);
}

template <class Plan>
__device__ __noinline__ long long steps_of_sequence(const AttendArgs& a, int b, int rt0, int stride) {
    if (b >= a.n_seq) return 0;
    int first, n;
    rows_of(a, b, first, n);
    long long u = 0;
#pragma unroll 1
    for (int rt = rt0; rt * Plan::R < n * a.group; rt += stride) u += Plan::steps(tile_of(a, b, rt, Plan::R));
    return u;
}
__device__ __forceinline__ long long warp_sum_ll(long long v) {
#pragma unroll 1
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
    return v;
}

// This block's share: `c` at its first tile; returns the steps of a full share, 0 if there is nothing
// for this block.  All NW warps call it.  ws: [NW + 2] in shared memory.
template <class Plan, int NW>
__device__ __forceinline__ int find_share(const AttendArgs& a, Cursor& c, long long* ws, int least) {
    constexpr int NT = NW * 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // a thread (few tiles each) or a warp (few sequences) adds up a sequence
    const bool wide = a.n_seq <= NW;
    const int unit = wide ? warp : threadIdx.x;
    auto steps_at = [&](int b) -> long long {  // of sequence b; wide: lane 0 has it
        if (!wide) return steps_of_sequence<Plan>(a, b, 0, 1) * a.KV;
        const long long s = warp_sum_ll(steps_of_sequence<Plan>(a, b, lane, 32)) * a.KV;
        return lane == 0 ? s : 0;
    };
    long long total = 0;
    const long long mine = steps_at(unit);
    const long long at0 = scan_block<NW>(mine, ws, total);
    const long long chunk0 = total;
    if (a.n_seq > NT) {  // the rest of the sequences: their sum first
        long long rest = 0, sum;
        for (int b = NT + threadIdx.x; b < a.n_seq; b += NT) rest += steps_at(b);
        scan_block<NW>(rest, ws, sum);
        total += sum;
    }
    const unsigned t32 = static_cast<unsigned>(min(total, 0xffff0000ll));  // (32-bit division where it is enough)
    const long long per = max(total <= 0xffff0000ll ? static_cast<long long>((t32 + gridDim.x - 1) / gridDim.x)
                                                    : (total + gridDim.x - 1) / gridDim.x,
                              static_cast<long long>(least));
    if (per > 0x40000000ll) return 0;  // (days of work: no such memory)
    const long long u0 = per * blockIdx.x;
    if (u0 >= total) return 0;
    if (threadIdx.x == 0) ws[NW + 1] = -1;
    __syncthreads();
    auto place = [&](int b, long long at, long long n) {
        if (u0 >= at && u0 < at + n) {
            ws[NW] = u0 - at;
            ws[NW + 1] = b;
        }
    };
    if (u0 < chunk0) {
        place(unit, at0, mine);
    } else {
        long long before = chunk0;
        for (int b0 = NT; b0 < a.n_seq; b0 += NT) {
            const long long n = steps_at(b0 + threadIdx.x);
            long long sum;
            const long long at = before + scan_block<NW>(n, ws, sum);
            if (u0 < before + sum) {
                place(b0 + threadIdx.x, at, n);
                break;
            }
            before += sum;
        }
    }
    __syncthreads();
    if (ws[NW + 1] < 0) return 0;  // (the lengths changed under the call)
    c.b = static_cast<int>(ws[NW + 1]);
    c.left = static_cast<int>(min(per, total - u0));
    // the row tile: 32 of them at a time, every warp for itself
    long long u = ws[NW];
    int first, n;
    rows_of(a, c.b, first, n);
    for (c.rt = 0;; c.rt += 32) {
        const int rt = c.rt + lane;
        const long long s = rt * Plan::R < n * a.group ? static_cast<long long>(Plan::steps(tile_of(a, c.b, rt, Plan::R))) * a.KV : 0;
        long long x = s;
#pragma unroll 1
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(FULL, x, o);
            if (lane >= o) x += y;
        }
        const unsigned past = __ballot_sync(FULL, x > u);  // tiles that end behind u
        if (past) {
            const int k = __ffs(past) - 1;
            u -= __shfl_sync(FULL, x - s, k);
            c.rt += k;
            break;
        }
        u -= __shfl_sync(FULL, x, 31);
        if ((c.rt + 32) * Plan::R >= n * a.group) return 0;  // (as above)
    }
    c.t = tile_of(a, c.b, c.rt, Plan::R);
    c.steps = Plan::steps(c.t);
    c.g = u < 0x100000000ll ? static_cast<int>(static_cast<unsigned>(u) / static_cast<unsigned>(c.steps))
                            : static_cast<int>(u / c.steps);
    c.s = static_cast<int>(u - static_cast<long long>(c.g) * c.steps);
    c.end = min(c.steps, c.s + c.left);
    return static_cast<int>(per);
}
// The number of blocks that share a tile whose first block ends at step `end` of `steps`.
__device__ __forceinline__ int parts_of(int steps, int end, int per) {
    return 1 + (steps - end + per - 1) / per;
}

// Row r0 + r of a tile: its token row and its q head (rows that do not exist: the tile's first).
__device__ __forceinline__ void row_of(const AttendArgs& a, const Cursor& c, int r, int& tok, int& h) {
    const int fr = c.t.r0 + (r < c.t.nrows ? r : 0), i = div_group(a, fr);
    tok = c.t.first + i;
    h = c.g * a.group + fr - i * a.group;
}

// One (token, head) by one warp, straight from the pages: lane l holds dims l * HD / 32 ...  Reads the attended keys only.
// What the kernels' fp32 cannot hold comes here (scores beyond its range, rows whose weights all vanish, values that are
// not finite), so scores and sums are 64-bit: products of three 32-bit numbers stay in range.  Two columns a lane at a
// time, so that the kernels that call this keep their registers (with all of them at once 2048 tokens of 4096 bf16 took 1 %
// longer).  Columns [cols & 0xffff, cols >> 16) are written (multiples of HD / 32).
template <typename T, int HD>
__device__ __noinline__ void attend_row(const AttendArgs& a, int b, int t, int h, int lane, int cols = HD << 16) {
    constexpr int D = HD / 32;
    int first, n;
    rows_of(a, b, first, n);
    const int p = first_pos(a, b, n) + (t - first);
    int lo, hi;
    attended(a, p, lo, hi);
    const int g = div_group(a, h);
    const T* qp = static_cast<const T*>(a.q) + static_cast<size_t>(t) * a.q_stride + static_cast<size_t>(h) * HD + lane * D;
#pragma unroll 1
    for (int c = 0; c < D; c += 2) {
        double acc[2] = {0.0, 0.0}, m = -INFINITY, l = 0.0;
#pragma unroll 1
        for (int j = lo; j < hi; j++) {
            const int id = page_of(a, b, j);
            if (id < 0) {  // to the last position of the page
                j |= (1 << a.shift) - 1;
                continue;
            }
            const size_t at = static_cast<size_t>(id) * a.block_stride +
                              ((static_cast<size_t>(g) << a.shift) + (j & ((1 << a.shift) - 1))) * HD + lane * D;
            const T* kp = static_cast<const T*>(a.k) + at;
            const T* vp = static_cast<const T*>(a.v) + at + c;
            double s = 0.0;
#pragma unroll
            for (int d = 0; d < D; d++) s += static_cast<double>(to_f32<T>(qp[d])) * to_f32<T>(kp[d]);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(FULL, s, o);
            s *= a.scale;
            const double mn = fmax(m, s);
            const float f = m == -INFINITY ? 1.f : expf(static_cast<float>(m - mn));
            const float e = s == -INFINITY ? 0.f : expf(static_cast<float>(s - mn));  // NaN stays NaN
            m = mn;
            l = l * f + e;
#pragma unroll
            for (int d = 0; d < 2; d++) acc[d] = acc[d] * f + static_cast<double>(e) * to_f32<T>(vp[d]);
        }
        if (lane * D < (cols & 0xffff) || lane * D >= (cols >> 16)) continue;
        T* op = static_cast<T*>(a.out) + (static_cast<size_t>(t) * a.H + h) * HD + lane * D + c;
#pragma unroll
        for (int d = 0; d < 2; d++) op[d] = from_f32<T>(static_cast<float>(l != 0.0 ? acc[d] / l : 0.0));
    }
}

constexpr int kJoinWarps = 8;
// Joins the parts (fp32 rows of hd + 4: maximum, sum, whether to do it over, -, values) of the tile that block blockIdx.x began: part i > 0 is the first tile of block blockIdx.x + i.
// Two warps a row (one for its
// even parts, one for the odd); lane = 4 or 2 dims; the rows are spread over gridDim.y blocks.
template <typename T, int HD, int R>
__global__ void __launch_bounds__(kJoinWarps * 32) k_attend_join(const __grid_constant__ AttendArgs a, const Head* heads,
                                                          const float* parts) {
    constexpr int D = HD / 32;
    __shared__ float half[kJoinWarps / 2][32 * D + 2];
    pdl_wait();
    const Head h = heads[blockIdx.x];
    if (h.parts == 0) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, odd = warp & 1;
    Cursor c;
    c.g = h.g;
    c.t = tile_of(a, h.b, h.rt, R);
    constexpr size_t rec = static_cast<size_t>(R) * (HD + 4);
    const float* p0 = parts + (static_cast<size_t>(blockIdx.x) * 2 + h.slot) * rec;
    const float* p1 = parts + (static_cast<size_t>(blockIdx.x) + 1) * 2 * rec;  // parts 1 .. are 2 * rec apart
    auto part = [&](int i, int row) { return (i == 0 ? p0 : p1 + static_cast<size_t>(i - 1) * 2 * rec) + row * (HD + 4); };
#pragma unroll 1
    for (int row0 = blockIdx.y * (kJoinWarps / 2); row0 < c.t.nrows; row0 += gridDim.y * (kJoinWarps / 2)) {
        const int row = row0 + (warp >> 1);
        float M = -INFINITY, bad = 0.f, L = 0.f, acc[D];
#pragma unroll
        for (int d = 0; d < D; d++) acc[d] = 0.f;
        if (row < c.t.nrows) {
#pragma unroll 1
            for (int i0 = odd; i0 < h.parts; i0 += 16) {  // 8 parts at a time
                float m[8], l[8], v[8][D], mx = M;
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const int i = i0 + 2 * k;
                    m[k] = -INFINITY;
                    l[k] = 0.f;
#pragma unroll
                    for (int d = 0; d < D; d++) v[k][d] = 0.f;
                    if (i < h.parts) {
                        const float* p = part(i, row);
                        const float4 q = *reinterpret_cast<const float4*>(p);
                        m[k] = q.x;
                        l[k] = q.y;
                        bad = fmaxf(bad, q.z);
#pragma unroll
                        for (int d = 0; d < D; d++) v[k][d] = p[4 + lane + 32 * d];
                    }
                }
#pragma unroll
                for (int k = 0; k < 8; k++) mx = fmaxf(mx, m[k]);
                const float f0 = mx == -INFINITY ? 1.f : ex2(M - mx);
                L *= f0;
#pragma unroll
                for (int d = 0; d < D; d++) acc[d] *= f0;
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const float f = mx == -INFINITY ? 1.f : ex2(m[k] - mx);
                    L += l[k] * f;
#pragma unroll
                    for (int d = 0; d < D; d++) acc[d] += v[k][d] * f;
                }
                M = mx;
            }
        }
        if (odd) {
            float* x = half[warp >> 1];
            if (lane == 0) {
                x[0] = M;
                x[1] = bad > 0.f ? NAN : L;  // (NaN: to be done over)
            }
#pragma unroll
            for (int d = 0; d < D; d++) x[2 + lane + 32 * d] = acc[d];
        }
        __syncthreads();
        if (!odd && row < c.t.nrows) {
            const float* x = half[warp >> 1];
            int tok, hh;
            row_of(a, c, row, tok, hh);
            const float mx = fmaxf(M, x[0]), f0 = mx == -INFINITY ? 1.f : ex2(M - mx), f1 = mx == -INFINITY ? 1.f : ex2(x[0] - mx);
            const float sum = L * f0 + x[1] * f1;
            float o[D], z = 0.f;  // NaN once a sum is not finite
#pragma unroll
            for (int d = 0; d < D; d++) {
                o[d] = acc[d] * f0 + x[2 + lane + 32 * d] * f1;
                z = fmaf(o[d], 0.f, z);
            }
            if (bad > 0.f || x[1] != x[1] || sum == 0.f || __any_sync(FULL, z != z)) {
                attend_row<T, HD>(a, h.b, tok, hh, lane);
            } else {
                T* out = static_cast<T*>(a.out) + (static_cast<size_t>(tok) * a.H + hh) * HD;
#pragma unroll
                for (int d = 0; d < D; d++) out[lane + 32 * d] = from_f32<T>(o[d] / sum);
            }
        }
        __syncthreads();
    }
}

template <typename T, int HD, int R>
tl_status launch_join(const AttendArgs& a, const Head* heads, const float* parts, int blocks, int slices, cudaStream_t s) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(blocks, slices);
    cfg.blockDim = dim3(kJoinWarps * 32);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    TL_CUDA_TRY(cudaLaunchKernelEx(&cfg, k_attend_join<T, HD, R>, a, heads, parts));
    return TL_OK;
}

// Map of one side (K or V) of the pages: {64 or hd columns, rows of all kv heads, column
// panels, pages}; a box is `rows` rows of `panels` panels of one page, zero where the page does not
// exist.  16-bit types: panels of 64 columns, SWIZZLE_128B; fp32: one panel, no swizzle.
tl_status encode_pages(CUtensorMap* map, const void* base, const tl_paged_cache* c, int rows, int panels);

// Few query rows per sequence (tl_paged_attn.cu), and many (tl_paged_attn_tc.cu; fp32: tl_paged_attn_f32.cu).
size_t split_workspace(int hd);
tl_status attend_split(const AttendArgs& a, const tl_paged_cache* c, void* workspace, cudaStream_t s);
size_t chunk_workspace(int hd);
tl_status attend_chunk(const AttendArgs& a, const tl_paged_cache* c, void* workspace, cudaStream_t s);
size_t chunk_f32_workspace(int hd);
tl_status attend_chunk_f32(const AttendArgs& a, const tl_paged_cache* c, void* workspace, cudaStream_t s);

}  // namespace paged
}  // namespace tl
