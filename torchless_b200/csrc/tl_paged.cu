// tl_paged.cu -- tl_paged_plan (block tables and slot maps from request
// lengths) and tl_qk_norm_rope (per-head norm, rotation, write into the pages).
#include <algorithm>

#include "tl_paged.cuh"

namespace tl {
namespace paged {

tl_status check_cache(const char* who, const tl_paged_cache* c) {
    TL_REQUIRE(c && c->k && c->v, "%s: no cache", who);
    TL_REQUIRE(dtype_ok(c->dtype), "%s: cache dtype %d", who, static_cast<int>(c->dtype));
    if (c->head_dim != 64 && c->head_dim != 128)
        return set_error(TL_ERR_UNSUPPORTED, "%s: head_dim %zu (64 or 128)", who, c->head_dim);
    if (c->block_size < 8 || c->block_size > 256 || (c->block_size & (c->block_size - 1)))
        return set_error(TL_ERR_UNSUPPORTED, "%s: block_size %zu (a power of two from 8 to 256)", who, c->block_size);
    TL_REQUIRE(c->n_blocks > 0 && c->n_blocks <= 0x7fffffffull / c->block_size, "%s: n_blocks %zu", who, c->n_blocks);
    TL_REQUIRE(c->n_kv_heads > 0 && c->n_kv_heads <= 1024, "%s: n_kv_heads %zu", who, c->n_kv_heads);
    TL_REQUIRE(c->block_stride >= c->n_kv_heads * c->block_size * c->head_dim &&
                   c->block_stride <= (1ull << 36) && c->block_stride * dtype_size(c->dtype) % 16 == 0,
               "%s: block_stride %zu", who, c->block_stride);
    TL_REQUIRE(aligned16(c->k) && aligned16(c->v), "%s: k and v must be 16-byte aligned", who);
    return TL_OK;
}

namespace {

// ---- plan -----------------------------------------------------------------
// Every block scans all requests (chunks of kPlanThreads, running sums in
// carries) and then takes its share of the flat lists that the scan lays out:
// ids taken (entry f of the free list) and tokens.  Both find their request by
// a binary search in the chunk's running sums, so one long request spreads
// over all threads as well as many short ones.  Bound by latency: one load of
// the lengths, one block scan, one dependent load for a token's page.  509
// requests, 15656 tokens: 7.8 us (cold); one call after the other 12.8 us, the
// host's part of a launch.
constexpr int kPlanThreads = 1024;

struct PlanArgs {
    int32_t *table, *q_start, *seq_lens, *positions, *slots, *counts;
    const int32_t *cached, *fresh, *free_blocks;
    int n_free, n_req, max_blocks, shift, n_tokens;  // block_size = 1 << shift
};

// Largest i in [0, n) with a[i] <= v (a not decreasing, a[0] <= v).
__device__ __forceinline__ int last_le(const int* a, int n, int v) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= v) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Exclusive running sum over the block; `total` gets the sum.
__device__ __forceinline__ long long block_scan(long long v, long long* warp_sums, long long& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(FULL, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    if (warp == 0) {
        long long w = warp_sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(FULL, w, o);
            if (lane >= o) w += y;
        }
        warp_sums[lane] = w;
    }
    __syncthreads();
    total = warp_sums[31];
    return x - v + (warp ? warp_sums[warp - 1] : 0);
}

__global__ void __launch_bounds__(kPlanThreads) k_plan(PlanArgs a) {
    __shared__ long long ws[32];
    __shared__ int s_start[kPlanThreads + 1], s_first[kPlanThreads + 1], s_cached[kPlanThreads];
    const int tid = threadIdx.x;
    const int bs = 1 << a.shift;
    long long tok0 = 0, blk0 = 0;  // tokens and ids of the chunks before
    for (int c0 = 0; c0 < a.n_req; c0 += kPlanThreads) {
        const int b = c0 + tid;
        const int m = min(kPlanThreads, a.n_req - c0);
        const int cached = b < a.n_req ? max(0, a.cached[b]) : 0;
        const int fresh = b < a.n_req ? max(0, a.fresh[b]) : 0;
        long long ntok, nblk;
        const long long at = tok0 + block_scan(fresh, ws, ntok);
        const int s0 = static_cast<int>(min(at, static_cast<long long>(a.n_tokens)));
        const int s1 = static_cast<int>(min(at + fresh, static_cast<long long>(a.n_tokens)));
        const long long len = min(static_cast<long long>(cached) + (s1 - s0), 0x7fffffffll);
        const int have = static_cast<int>((static_cast<long long>(cached) + bs - 1) >> a.shift);
        const int want = static_cast<int>(min((len + bs - 1) >> a.shift, static_cast<long long>(a.max_blocks)));
        const int need = max(0, want - have);
        const int f0 = static_cast<int>(blk0 + block_scan(need, ws, nblk));
        if (tid < m) {
            s_start[tid] = s0;
            s_first[tid] = f0;
            s_cached[tid] = cached;
            if (tid == m - 1) {
                s_start[m] = s1;
                s_first[m] = f0 + need;
            }
            if (blockIdx.x == 0) {
                a.q_start[b] = s0;
                if (b == a.n_req - 1) a.q_start[a.n_req] = s1;
                a.seq_lens[b] = static_cast<int>(len);
            }
        }
        __syncthreads();
        const int step = gridDim.x * kPlanThreads;
        for (int f = s_first[0] + blockIdx.x * kPlanThreads + tid; f < s_first[m]; f += step) {
            const int i = last_le(s_first, m, f);
            const int j = static_cast<int>((static_cast<long long>(s_cached[i]) + bs - 1) >> a.shift) + f - s_first[i];
            a.table[static_cast<size_t>(c0 + i) * a.max_blocks + j] = f < a.n_free ? a.free_blocks[f] : -1;
        }
        for (int t = s_start[0] + blockIdx.x * kPlanThreads + tid; t < s_start[m]; t += step) {
            const int i = last_le(s_start, m, t);
            const int p = static_cast<int>(min(static_cast<long long>(s_cached[i]) + (t - s_start[i]), 0x7fffffffll));
            const int blk = p >> a.shift, have_i = static_cast<int>((static_cast<long long>(s_cached[i]) + bs - 1) >> a.shift);
            int id = -1;
            if (blk < a.max_blocks) {
                if (blk < have_i) {
                    id = a.table[static_cast<size_t>(c0 + i) * a.max_blocks + blk];
                } else {  // an id that this step takes: from the list, not from the table being written
                    const int f = s_first[i] + blk - have_i;
                    if (f < a.n_free) id = a.free_blocks[f];
                }
            }
            const long long slot = (static_cast<long long>(id) << a.shift) + (p & (bs - 1));
            a.positions[t] = p;
            a.slots[t] = (id >= 0 && slot <= 0x7fffffffll) ? static_cast<int>(slot) : -1;
        }
        tok0 += ntok;
        blk0 += nblk;
        __syncthreads();
    }
    for (long long t = min(tok0, static_cast<long long>(a.n_tokens)) + blockIdx.x * kPlanThreads + tid; t < a.n_tokens;
         t += gridDim.x * kPlanThreads) {
        a.positions[t] = -1;
        a.slots[t] = -1;
    }
    if (blockIdx.x == 0 && tid == 0) {
        if (a.n_req == 0) a.q_start[0] = 0;
        a.counts[0] = static_cast<int>(min(blk0, static_cast<long long>(a.n_free)));
        a.counts[1] = static_cast<int>(max(0ll, blk0 - a.n_free));
    }
}

// ---- norm, rotation, cache write -------------------------------------------
// A warp takes a share of one token's heads, 32 / L of them at a time, L = hd / 8 lanes a head and 8 dims a lane:
// 16-byte accesses, and the token's angles and the norm's weights stay in registers over its heads.  The rotation's
// partner dims lie half / 8 lanes away; their raw bits come by shuffles (for 16-bit types half as many as of the
// fp32 values).  The next turns' heads are fetched before these are worked on, the first before the angles.  One read
// and one write of every element: bound by HBM for many tokens (32 heads, 8 kv heads, hd 128, 16381 tokens: bf16 with
// both norms 85.6 us, 4.7 TB/s, where the norm's and the conversions' instructions take as long as the memory; fp32 to
// fp16 95 us, 6.4 TB/s), by latency for few (one token 2.1 us); then a token's heads are spread over more warps.
struct RopeArgs {
    const int32_t *positions, *slots;
    const float *cos_, *sin_, *wq, *wk;
    size_t row_stride, block_stride;
    float eps;
    int n_tokens, H, KV, n_pos, rot, shift, n_slots;
    int parts;  // warps a token
};

// 8 elements as raw words, and as fp32.
template <typename T>
struct Raw8 {
    static constexpr int W = sizeof(T) == 4 ? 8 : 4;
    uint32_t w[W];
    __device__ __forceinline__ void load(const T* p) {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
        if (W == 8) {
            const uint4 b = reinterpret_cast<const uint4*>(p)[1];
            w[W - 4] = b.x; w[W - 3] = b.y; w[W - 2] = b.z; w[W - 1] = b.w;
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const;
};
template <>
__device__ __forceinline__ void Raw8<float>::get(float (&v)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = __uint_as_float(w[j]);
}
template <>
__device__ __forceinline__ void Raw8<__half>::get(float (&v)[8]) const {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        v[2 * j] = f.x;
        v[2 * j + 1] = f.y;
    }
}
template <>
__device__ __forceinline__ void Raw8<__nv_bfloat16>::get(float (&v)[8]) const {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
}

constexpr int kRopeWarps = 4;

template <typename TI, typename TO, int HD>
__global__ void __launch_bounds__(kRopeWarps * 32) k_qk_norm_rope(TO* q_out, TO* kc, TO* vc, const TI* qkv,
                                                                  const __grid_constant__ RopeArgs a) {
    constexpr int L = HD / 8, PER = 32 / L, AHEAD = sizeof(TI) == 2 ? 6 : 3;  // lanes a head, heads at a time, turns fetched ahead
    const int lane = threadIdx.x & 31, l = lane % L, sub = lane / L;
    const unsigned w = blockIdx.x * kRopeWarps + (threadIdx.x >> 5);
    const int t = static_cast<int>(w / static_cast<unsigned>(a.parts)), part = static_cast<int>(w % static_cast<unsigned>(a.parts));
    if (t >= a.n_tokens) return;
    const int rows = a.H + 2 * a.KV, turns = (rows + PER - 1) / PER, per = (turns + a.parts - 1) / a.parts;
    const int u0 = part * per, u1 = min(turns, u0 + per);
    const TI* src = qkv + static_cast<size_t>(t) * a.row_stride + 8 * l;
    Raw8<TI> next[AHEAD];
    auto fetch = [&](int u) {
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const int hh = (u + i) * PER + sub;
            if (u + i < u1 && hh < rows) next[i].load(src + static_cast<size_t>(hh) * HD);
            else {
#pragma unroll
                for (int j = 0; j < Raw8<TI>::W; j++) next[i].w[j] = 0u;
            }
        }
    };
    fetch(u0);
    const int pos = a.positions[t];
    if (pos < 0 || pos >= a.n_pos) return;  // a row of no sequence
    const int slot = a.slots[t];

    const int half = a.rot / 2, off = half / 8;
    const bool lower = l < off, turned = l < 2 * off;
    const int from = lane + (lower ? off : turned ? -off : 0), pl = l + (from - lane);  // the partner's lane, and within its head
    float c[8], s[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        c[j] = 1.f;
        s[j] = 0.f;
    }
    if (turned) {
        const size_t ang = static_cast<size_t>(pos) * half + 8 * (lower ? l : l - off);
        Vec8<float>::load(c, a.cos_ + ang);
        Vec8<float>::load(s, a.sin_ + ang);
        if (lower) {
#pragma unroll
            for (int j = 0; j < 8; j++) s[j] = -s[j];
        }
    }
    const bool cached = slot >= 0 && slot < a.n_slots;
    const size_t at = cached ? static_cast<size_t>(slot >> a.shift) * a.block_stride +
                                   static_cast<size_t>(slot & ((1 << a.shift) - 1)) * HD + 8 * l
                             : 0;
    float fa[8], fb[8];  // x' = (x fa + partner fb) / rms
    int cur = -1;
    const float* wt = nullptr;
    for (int u = u0; u < u1; u += AHEAD) {
        Raw8<TI> raw[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) raw[i] = next[i];
        fetch(u + AHEAD);
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            if (u + i >= u1) break;
            const int hh = (u + i) * PER + sub;
            const int kind = hh < a.H ? 0 : hh < a.H + a.KV ? 1 : 2;  // q, k, v
            if (kind != cur && kind < 2) {  // the section's factors
                wt = kind ? a.wk : a.wq;
                float g[8], gy[8];
#pragma unroll
                for (int j = 0; j < 8; j++) g[j] = gy[j] = 1.f;
                if (wt != nullptr) {
                    Vec8<float>::load(g, wt + 8 * l);
                    Vec8<float>::load(gy, wt + 8 * pl);
                }
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    fa[j] = g[j] * c[j];
                    fb[j] = gy[j] * s[j];
                }
            }
            cur = kind;
            float x[8], y[8];
            raw[i].get(x);
            Raw8<TI> other;
#pragma unroll
            for (int j = 0; j < Raw8<TI>::W; j++) other.w[j] = __shfl_sync(FULL, raw[i].w[j], from);
            float inv = 1.f;
            if (a.wq != nullptr || a.wk != nullptr) {
                float ss = 0.f;
#pragma unroll
                for (int j = 0; j < 8; j++) ss += x[j] * x[j];
#pragma unroll
                for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(FULL, ss, o);
                if (wt != nullptr) inv = rsqrtf(ss * (1.f / HD) + a.eps);  // (2 ulp)
            }
            if (hh >= rows) continue;  // (a last turn of fewer heads; the shuffles are behind)
            if (kind < 2) {
                if (turned) {
                    other.get(y);
#pragma unroll
                    for (int j = 0; j < 8; j++) x[j] = (x[j] * fa[j] + y[j] * fb[j]) * inv;
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j++) x[j] = x[j] * fa[j] * inv;
                }
            }
            if (hh < a.H) {
                Vec8<TO>::store(q_out + (static_cast<size_t>(t) * a.H + hh) * HD + 8 * l, x);
            } else if (cached) {
                const int g = kind == 2 ? hh - a.H - a.KV : hh - a.H;
                Vec8<TO>::store((kind == 2 ? vc : kc) + at + (static_cast<size_t>(g) << a.shift) * HD, x);
            }
        }
    }
}

template <typename TI, typename TO>
void launch_rope(void* q_out, const tl_paged_cache* c, const void* qkv, RopeArgs a, cudaStream_t s) {
    const int per = 32 / (static_cast<int>(c->head_dim) / 8), turns = (a.H + 2 * a.KV + per - 1) / per;
    // Few tokens: as many warps a token as fill the device (16 an SM), down to one turn each.  bf16 with norms, 1 / 64 /
    // 200 / 1000 tokens: 2.1 / 2.8 / 3.7 / 7.5 us, and with one warp a token 8.8 / 9.2 / 9.5 / 10.4 us; with 8 warps an
    // SM 200 and 1000 tokens take 4.1 and 10.4 us, with 32 5.0 and 8.5 us.
    const long long want = 16ll * sm_count();
    a.parts = static_cast<int>(std::max<long long>(1, std::min<long long>(turns, want / std::max(1, a.n_tokens))));
    const long long warps = static_cast<long long>(a.n_tokens) * a.parts;
    const unsigned grid = static_cast<unsigned>((warps + kRopeWarps - 1) / kRopeWarps);
    if (c->head_dim == 128)
        k_qk_norm_rope<TI, TO, 128><<<grid, kRopeWarps * 32, 0, s>>>(
            static_cast<TO*>(q_out), static_cast<TO*>(c->k), static_cast<TO*>(c->v), static_cast<const TI*>(qkv), a);
    else
        k_qk_norm_rope<TI, TO, 64><<<grid, kRopeWarps * 32, 0, s>>>(
            static_cast<TO*>(q_out), static_cast<TO*>(c->k), static_cast<TO*>(c->v), static_cast<const TI*>(qkv), a);
}

template <typename TI>
void launch_rope_to(void* q_out, const tl_paged_cache* c, const void* qkv, const RopeArgs& a, cudaStream_t s) {
    if (c->dtype == TL_F32) launch_rope<TI, float>(q_out, c, qkv, a, s);
    else if (c->dtype == TL_F16) launch_rope<TI, __half>(q_out, c, qkv, a, s);
    else launch_rope<TI, __nv_bfloat16>(q_out, c, qkv, a, s);
}

}  // namespace
}  // namespace paged
}  // namespace tl

using namespace tl;
using namespace tl::paged;

extern "C" {

tl_status tl_paged_plan(int32_t* block_table, int32_t* q_start, int32_t* seq_lens, int32_t* positions, int32_t* slots,
                        int32_t* counts, const int32_t* cached, const int32_t* new_tokens, const int32_t* free_blocks,
                        size_t n_free, size_t n_req, size_t max_blocks, size_t block_size, size_t n_tokens,
                        void* stream) {
    clear_error();
    TL_REQUIRE(q_start && counts, "tl_paged_plan: no q_start or counts");
    TL_REQUIRE(n_req == 0 || (block_table && seq_lens && cached && new_tokens && max_blocks > 0),
               "tl_paged_plan: %zu requests without their arrays", n_req);
    TL_REQUIRE(n_tokens == 0 || (positions && slots), "tl_paged_plan: %zu tokens without their arrays", n_tokens);
    TL_REQUIRE(n_free == 0 || free_blocks, "tl_paged_plan: no free_blocks");
    if (block_size < 8 || block_size > 256 || (block_size & (block_size - 1)))
        return set_error(TL_ERR_UNSUPPORTED, "tl_paged_plan: block_size %zu (a power of two from 8 to 256)", block_size);
    TL_REQUIRE(n_req < (1u << 31) - 1 && n_free < (1u << 31) && n_tokens < (1u << 31) - (1u << 20) &&
                   (n_req == 0 || max_blocks <= ((1ull << 31) - (1u << 20)) / n_req),
               "tl_paged_plan: %zu requests x %zu blocks, %zu tokens", n_req, max_blocks, n_tokens);
    PlanArgs a{block_table, q_start, seq_lens, positions, slots, counts, cached, new_tokens, free_blocks,
               static_cast<int>(n_free), static_cast<int>(n_req), static_cast<int>(max_blocks),
               __builtin_ctzll(block_size), static_cast<int>(n_tokens)};
    const size_t want = (std::max(n_tokens, n_req) + kPlanThreads - 1) / kPlanThreads;
    const int grid = static_cast<int>(std::min<size_t>(std::max<size_t>(want, 1), static_cast<size_t>(sm_count())));
    k_plan<<<grid, kPlanThreads, 0, as_stream(stream)>>>(a);
    return check_launch("paged_plan");
}

tl_status tl_qk_norm_rope(void* q_out, const tl_paged_cache* cache, const void* qkv, tl_dtype dtype, size_t row_stride,
                          const int32_t* positions, const int32_t* slots, const float* cos_, const float* sin_,
                          size_t n_pos, size_t rot_dim, const float* q_weight, const float* k_weight, float eps,
                          size_t n_tokens, size_t n_heads, void* stream) {
    clear_error();
    TL_TRY(check_cache("tl_qk_norm_rope", cache));
    TL_REQUIRE(dtype_ok(dtype), "tl_qk_norm_rope: dtype %d", static_cast<int>(dtype));
    TL_REQUIRE(n_heads > 0 && n_heads <= 65536, "tl_qk_norm_rope: n_heads %zu", n_heads);
    if (rot_dim < 16 || rot_dim % 16 || rot_dim > cache->head_dim)
        return set_error(TL_ERR_UNSUPPORTED, "tl_qk_norm_rope: rot_dim %zu (a multiple of 16 up to head_dim %zu)",
                         rot_dim, cache->head_dim);
    if (n_tokens == 0) return TL_OK;
    TL_REQUIRE(q_out && qkv && positions && slots && cos_ && sin_, "tl_qk_norm_rope: null pointer");
    TL_REQUIRE(n_tokens < (1ull << 31) && n_pos > 0 && n_pos < (1ull << 31), "tl_qk_norm_rope: %zu tokens, %zu positions",
               n_tokens, n_pos);
    TL_REQUIRE(row_stride >= (n_heads + 2 * cache->n_kv_heads) * cache->head_dim && row_stride <= (1ull << 36),
               "tl_qk_norm_rope: row_stride %zu", row_stride);
    TL_REQUIRE(aligned16(q_out) && aligned16(qkv) && aligned16(cos_) && aligned16(sin_) && aligned16(q_weight) &&
                   aligned16(k_weight) && row_stride * dtype_size(dtype) % 16 == 0,
               "tl_qk_norm_rope: pointers and row_stride must be 16-byte aligned");
    RopeArgs a{positions, slots, cos_, sin_, q_weight, k_weight, row_stride, cache->block_stride, eps,
               static_cast<int>(n_tokens), static_cast<int>(n_heads), static_cast<int>(cache->n_kv_heads),
               static_cast<int>(n_pos), static_cast<int>(rot_dim), __builtin_ctzll(cache->block_size),
               static_cast<int>(cache->n_blocks * cache->block_size), 1};
    const cudaStream_t s = as_stream(stream);
    if (dtype == TL_F32) launch_rope_to<float>(q_out, cache, qkv, a, s);
    else if (dtype == TL_F16) launch_rope_to<__half>(q_out, cache, qkv, a, s);
    else launch_rope_to<__nv_bfloat16>(q_out, cache, qkv, a, s);
    return check_launch("qk_norm_rope");
}

}  // extern "C"
