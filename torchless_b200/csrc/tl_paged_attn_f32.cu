// tl_paged_attn_f32.cu -- paged attention of many query rows over an fp32 cache.
//
// No matrix instruction keeps fp32's 24 bits, so this is FMA work: 2 * hd FMAs
// a row and key, 128 a cycle and SM.  What the kernel has to do is to keep the
// FMA pipes fed from shared memory:
//   - A block of 128 threads works on 64 rows of one kv head, 64 keys at a time;
//     thread (ty, tx) of 8 x 16 has rows ty + 8 i (8 of them), keys tx + 16 j of
//     the scores and 4 columns of every 64 of the values.  A load of 16 bytes
//     feeds 11 (scores) or 16 (values) FMAs a thread.
//   - Packed FMAs (fma.rn.f32x2) take half the issue slots, which the loads use.
//   - A row belongs to half a warp: its maximum and its weights never leave the
//     warp, and a tile of keys takes two barriers (K is there, V is there).
//   - K and V come by cp.async (8 keys lie in one page; rows that no query of the
//     tile attends to and pages that do not exist are zeros).  One buffer each: K
//     of the next tile arrives while the values are summed, V while the scores
//     are.
//   - Two blocks an SM: one takes exponentials while the other multiplies.
// Blocks have equal shares of the key tiles (tl_paged_attn.cuh).
// Bound by the FMA pipes and by what two warps a scheduler can hide: 2048 tokens of 4096, 32 heads, 8 kv heads, hd 128:
// 2.47 ms, 41.7 TFLOP/s of 72 that the pipes have (plain FMAs: 2.99 ms); 512 of 1024: 192 us (in 16-row tiles of the
// decode kernel 395 us).  128 rows in one block of 256 threads: the same where rows abound, and 229 instead of 130 us
// for 16 sequences of 20 rows.
#include <math.h>

#include <algorithm>

#include "tl_paged_attn.cuh"

namespace tl {
namespace paged {
namespace {

constexpr int kRows = 64, kKeys = 64, kWarps = 4, kThreads = kWarps * 32, kGroups = kKeys / 8;

template <int HD>
struct Shape {
    static constexpr size_t SMEM = 4 * (static_cast<size_t>(kRows) * HD + 2 * kKeys * HD + kRows * kKeys) + 8 * (kWarps + 2) +
                                   4 * kGroups + 4 * kRows / 32;
    static_assert(2 * (SMEM + 1024) <= 228 * 1024, "two blocks' shared memory");
};

// Steps of 64 keys; a tile without keys counts as one, so that its zeros get written.  (A step takes as long as beginning and
// ending a tile: counting those as a step of their own made no difference above 3 %, either way.)
struct Plan {
    static constexpr int R = kRows;
    static constexpr bool kLookAgain = true;
    static __device__ __forceinline__ int steps(const Tile& t) { return t.hi <= t.lo ? 1 : (t.hi - 1) / kKeys - t.lo / kKeys + 1; }
};

using pair = unsigned long long;  // two floats
__device__ __forceinline__ void fma2(pair& c, pair a, pair b) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(c) : "l"(a), "l"(b));
}
__device__ __forceinline__ void mul2(pair& c, pair a) { asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(c) : "l"(a)); }
__device__ __forceinline__ pair both(float x) {
    pair y;
    asm("mov.b64 %0, {%1, %1};" : "=l"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float2 halves(pair x) {
    float2 y;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(y.x), "=f"(y.y) : "l"(x));
    return y;
}
__device__ __forceinline__ void copy16(float* dst, const float* src, bool there) {  // 16 bytes, or zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(tc::su32(dst)), "l"(src), "r"(there ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

template <int HD>
__global__ void __launch_bounds__(kThreads, 2)
    k_attend_chunk_f32(const __grid_constant__ AttendArgs a, Head* heads, float* parts) {
    using S = Shape<HD>;
    constexpr int NC = HD / 64;  // 4-column groups of a thread
    extern __shared__ __align__(16) uint8_t raw[];
    float* sq = reinterpret_cast<float*>(raw);
    float* sk = sq + kRows * HD;
    float* sv = sk + kKeys * HD;
    float* sp = sv + kKeys * HD;
    long long* ws = reinterpret_cast<long long*>(sp + kRows * kKeys);  // [kWarps + 2]
    int* exists = reinterpret_cast<int*>(ws + kWarps + 2);             // [kGroups]: whether a group of 8 keys has a page
    unsigned* redo = reinterpret_cast<unsigned*>(exists + kGroups);    // [kRows / 32]: rows to be done over
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;

    if (threadIdx.x == 0) heads[blockIdx.x].parts = 0;
    Cursor c;
    const int per = find_share<Plan, kWarps>(a, c, ws, 2);
    if (per == 0) return;

    // 8 rows of K or V; `key`: of the first.  K's pieces of 16 bytes are swapped within a row (piece x of row r lies at
    // x ^ (r & 7)), so that 8 rows' pieces x lie in different banks.
    auto fetch = [&](float* dst, const void* src, int key, int id, int swap) {
        const float* from = static_cast<const float*>(src);
        if (id >= 0)
            from += static_cast<size_t>(id) * a.block_stride +
                    ((static_cast<size_t>(c.g) << a.shift) + (key & ((1 << a.shift) - 1))) * HD;
        constexpr int PR = HD / 4;  // pieces of a row
#pragma unroll
        for (int x = lane; x < 8 * PR; x += 32) {
            const int r = x / PR, d = x % PR;
            const bool there = id >= 0 && key + r >= c.t.lo && key + r < c.t.hi;
            copy16(dst + r * HD + 4 * (d ^ (swap & r)), from + (there ? r * HD + 4 * d : 0), there);
        }
    };
    const float sl = a.scale * 1.4426950408889634f;  // log2 units
    bool first_tile = true;
#pragma unroll 1
    for (bool go = true; go; go = next_tile<Plan>(a, c), first_tile = false) {
        const int s0 = c.s, s1 = c.t.hi <= c.t.lo ? 0 : c.end;
        int id[2] = {-1, -1};
        auto next_keys = [&](int s) {  // K of step s on its way: two groups of 8 a warp
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const int group = 2 * warp + x, key = (c.t.lo / kKeys + s) * kKeys + 8 * group;
                id[x] = page_of(a, c.b, key);
                if (lane == 0) exists[group] = id[x] >= 0;
                fetch(sk + 8 * group * HD, a.k, key, id[x], 7);
            }
        };
        if (s0 < s1) next_keys(s0);
#pragma unroll 1
        for (int r = warp; r < kRows; r += kWarps) {  // Q; rows that do not exist are zeros
            int tok, h;
            row_of(a, c, r, tok, h);
            const float* src = static_cast<const float*>(a.q) + static_cast<size_t>(tok) * a.q_stride + static_cast<size_t>(h) * HD;
            if (lane < HD / 4) copy16(sq + r * HD + 4 * lane, src + 4 * lane, r < c.t.nrows);
        }
        pair o[8][NC][2];
        float m[8], l[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            m[i] = -INFINITY;
            l[i] = 0.f;
#pragma unroll
            for (int j = 0; j < NC; j++) o[i][j][0] = o[i][j][1] = 0;
        }
#pragma unroll 1
        for (int s = s0; s < s1; s++) {
            const int key0 = (c.t.lo / kKeys + s) * kKeys;
            copies_done();
            __syncthreads();  // K is there, and everyone is done with the last V
#pragma unroll
            for (int x = 0; x < 2; x++) fetch(sv + 8 * (2 * warp + x) * HD, a.v, key0 + 8 * (2 * warp + x), id[x], 0);
            // ---- scores: pairs of dims ----
            pair acc[8][4];
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = 0;
#pragma unroll 2
            for (int d = 0; d < HD; d += 4) {
                ulonglong2 k[4];
#pragma unroll
                for (int j = 0; j < 4; j++) k[j] = *reinterpret_cast<const ulonglong2*>(sk + (tx + 16 * j) * HD + (d ^ (4 * (tx & 7))));
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(sq + (ty + 8 * i) * HD + d);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        fma2(acc[i][j], q.x, k[j].x);
                        fma2(acc[i][j], q.y, k[j].y);
                    }
                }
            }
            // ---- weights ----
            int pages = 0;  // bit k: the page of keys 8 k .. exists
#pragma unroll
            for (int w = 0; w < kGroups; w++) pages |= exists[w] << w;
            const bool edge = pages != (1 << kGroups) - 1 || key0 < c.t.lo_last || key0 > c.t.hi_first - kKeys;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                float w[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float2 x = halves(acc[i][j]);
                    w[j] = (x.x + x.y) * sl;
                }
                if (edge) {
                    int lo, hi;
                    attended(a, c.t.p0 + div_group(a, c.t.r0 + ty + 8 * i), lo, hi);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int kk = tx + 16 * j;
                        if (!(key0 + kk >= lo && key0 + kk < hi && ((pages >> (kk >> 3)) & 1))) w[j] = -INFINITY;
                    }
                }
                float mx = fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3]));
#pragma unroll
                for (int x = 1; x < 16; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, x));
                const float mn = fmaxf(m[i], mx), base = mn == -INFINITY ? 0.f : mn, f = ex2(m[i] - base);
                m[i] = mn;
                float* p = sp + (ty + 8 * i) * kKeys + tx;
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float e = ex2(w[j] - base);
                    sum += e;
                    p[(16 * j) ^ (16 * (ty & 1))] = e;  // (a warp's two rows in different banks)
                }
                l[i] = l[i] * f + sum;
                if (f != 1.f) {
                    const pair ff = both(f);
#pragma unroll
                    for (int j = 0; j < NC; j++) {
                        mul2(o[i][j][0], ff);
                        mul2(o[i][j][1], ff);
                    }
                }
            }
            copies_done();
            __syncthreads();  // V is there, and everyone is done with K
            if (s + 1 < s1) next_keys(s + 1);
            // ---- values: pairs of columns ----
#pragma unroll 2
            for (int k = 0; k < kKeys; k += 4) {
                float4 p[8];
#pragma unroll
                for (int i = 0; i < 8; i++) p[i] = *reinterpret_cast<const float4*>(sp + (ty + 8 * i) * kKeys + (k ^ (16 * (ty & 1))));
#pragma unroll
                for (int e = 0; e < 4; e++)
#pragma unroll
                    for (int j = 0; j < NC; j++) {
                        const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(sv + (k + e) * HD + 64 * j + 4 * tx);
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const pair w = both(e == 0 ? p[i].x : e == 1 ? p[i].y : e == 2 ? p[i].z : p[i].w);
                            fma2(o[i][j][0], w, v.x);
                            fma2(o[i][j][1], w, v.y);
                        }
                    }
            }
        }
        // ---- results: to their place, or as a part to the workspace ----
        const bool whole = c.s == 0 && c.end == c.steps;
        float* part = parts + (static_cast<size_t>(blockIdx.x) * 2 + (first_tile ? 0 : 1)) * kRows * (HD + 4);
        copies_done();  // (a tile without keys: Q's)
        if (threadIdx.x < kRows / 32) redo[threadIdx.x] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int r = ty + 8 * i;
#pragma unroll
            for (int x = 1; x < 16; x <<= 1) l[i] += __shfl_xor_sync(FULL, l[i], x);
            if (r < c.t.nrows) {
                float4 v[NC];
                // NaN once a value is not finite, or a whole row's weights are all 0: the row is done over
                float z = whole && l[i] == 0.f ? NAN : l[i] * 0.f;
#pragma unroll
                for (int j = 0; j < NC; j++) {
                    const float2 x = halves(o[i][j][0]), y = halves(o[i][j][1]);
                    v[j] = make_float4(x.x, x.y, y.x, y.y);
                    z = fmaf(x.x, 0.f, fmaf(x.y, 0.f, fmaf(y.x, 0.f, fmaf(y.y, 0.f, z))));
                }
                if (z != z) atomicOr(&redo[r >> 5], 1u << (r & 31));
                int tok, h;
                row_of(a, c, r, tok, h);
                float* dst = whole ? static_cast<float*>(a.out) + (static_cast<size_t>(tok) * a.H + h) * HD
                                   : part + r * (HD + 4) + 4;
#pragma unroll
                for (int j = 0; j < NC; j++) {
                    if (whole) v[j] = make_float4(v[j].x / l[i], v[j].y / l[i], v[j].z / l[i], v[j].w / l[i]);
                    *reinterpret_cast<float4*>(dst + 64 * j + 4 * tx) = v[j];
                }
                if (!whole && tx == 0) *reinterpret_cast<float2*>(dst - 4) = make_float2(m[i], l[i]);
            }
        }
        __syncthreads();
        for (int r = warp; r < c.t.nrows; r += kWarps) {
            const bool bad = (redo[r >> 5] >> (r & 31)) & 1;
            if (!whole) {
                if (lane == 0) part[r * (HD + 4) + 2] = bad ? 1.f : 0.f;
            } else if (bad) {
                int tok, h;
                row_of(a, c, r, tok, h);
                attend_row<float, HD>(a, c.b, tok, h, lane);
            }
        }
        if (!whole && c.s == 0 && threadIdx.x == 0) {  // this block begins the tile: it says who has the rest
            Head h;
            h.parts = parts_of(c.steps, c.end, per);
            h.slot = first_tile ? 0 : 1;
            h.b = c.b;
            h.rt = c.rt;
            h.g = c.g;
            heads[blockIdx.x] = h;
        }
        __syncthreads();
    }
}

template <int HD>
tl_status run_chunk_f32(const AttendArgs& a, void* workspace, cudaStream_t s) {
    using S = Shape<HD>;
    TL_CUDA_TRY(cudaFuncSetAttribute(k_attend_chunk_f32<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     static_cast<int>(S::SMEM)));
    const int grid = std::min(2 * sm_count(), kMaxBlocks);
    Head* heads = static_cast<Head*>(workspace);
    float* parts = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kHeadBytes);
    k_attend_chunk_f32<HD><<<grid, kThreads, S::SMEM, s>>>(a, heads, parts);
    TL_TRY(check_launch("paged_attention"));
    return launch_join<float, HD, kRows>(a, heads, parts, grid, kRows / 8, s);
}

}  // namespace

size_t chunk_f32_workspace(int hd) {
    return kHeadBytes + static_cast<size_t>(std::min(2 * sm_count(), kMaxBlocks)) * 2 * kRows * (hd + 4) * 4;
}

tl_status attend_chunk_f32(const AttendArgs& a, const tl_paged_cache* c, void* workspace, cudaStream_t s) {
    return c->head_dim == 128 ? run_chunk_f32<128>(a, workspace, s) : run_chunk_f32<64>(a, workspace, s);
}

}  // namespace paged
}  // namespace tl
