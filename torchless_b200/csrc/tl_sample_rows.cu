// tl_sample_rows.cu -- tl_sample_rows: temperature, top-k, top-p and min-p for
// many rows, each with its own settings.
#include <math.h>

#include <algorithm>

#include "tl_paged.cuh"

namespace tl {
namespace {

using namespace paged;

constexpr int kThreads = 1024;
constexpr double kOne = 1099511627776.0;  // 2^40: weights are multiples of its inverse

struct SampleRowsArgs {
    uint32_t* out;
    const void* logits;
    size_t row_stride;
    int n;
    const float *r, *temperature, *top_p, *min_p;
    const int32_t* top_k;
};

// Order-preserving key of a logit: larger logit, larger key; -0 and +0 the same.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// The weight of a logit as a multiple of 2^-40.
__device__ __forceinline__ unsigned long long weight_of(float x, float top, double inv_t) {
    return __double2ull_rn(exp((static_cast<double>(x) - static_cast<double>(top)) * inv_t) * kOne);
}

__device__ __forceinline__ unsigned long long block_sum_u64(unsigned long long v, unsigned long long* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    unsigned long long t = red[threadIdx.x & 31];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(FULL, t, o);
    return t;
}

// Block = one row.  The kept set is a threshold: every logit whose key is above
// `key`, and of those equal to it the first `ties` by index.
template <typename T>
__global__ void __launch_bounds__(kThreads) k_sample_rows(SampleRowsArgs a) {
    __shared__ unsigned long long red[32], bins[256];
    __shared__ uint32_t sk[32], si[32], s_sel[4];
    __shared__ unsigned long long s_above;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T* x = static_cast<const T*>(a.logits) + static_cast<size_t>(row) * a.row_stride;
    const int n = a.n;
    const float temp = a.temperature[row];

    // largest logit, lowest index; NaN or +inf anywhere
    uint32_t bk = 0, bi = 0xffffffffu;
    int bad = 0;
    for (int i = tid; i < n; i += kThreads) {
        const float v = to_f32<T>(x[i]);
        if (!(v < INFINITY)) bad = 1;
        if (v == v) {
            const uint32_t k = key_of(v);
            if (k > bk || (k == bk && static_cast<uint32_t>(i) < bi)) {
                bk = k;
                bi = static_cast<uint32_t>(i);
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const uint32_t k = __shfl_xor_sync(FULL, bk, o), i = __shfl_xor_sync(FULL, bi, o);
        if (k > bk || (k == bk && i < bi)) {
            bk = k;
            bi = i;
        }
    }
    if (lane == 0) {
        sk[warp] = bk;
        si[warp] = bi;
    }
    bad = __syncthreads_or(bad);
    bk = sk[lane];
    bi = si[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const uint32_t k = __shfl_xor_sync(FULL, bk, o), i = __shfl_xor_sync(FULL, bi, o);
        if (k > bk || (k == bk && i < bi)) {
            bk = k;
            bi = i;
        }
    }
    const float top = bi == 0xffffffffu ? -INFINITY : logit_of(bk);
    if (!(temp > 0.f)) {  // sample_max: first strict maximum above -inf; NaN at index 0 keeps 0
        if (tid == 0) {
            const float x0 = to_f32<T>(x[0]);
            a.out[row] = (x0 != x0 || top == -INFINITY) ? 0u : bi;
        }
        return;
    }
    if (bad || top == -INFINITY) {
        if (tid == 0) a.out[row] = static_cast<uint32_t>(n - 1);
        return;
    }
    const double inv_t = 1.0 / static_cast<double>(temp);
    uint32_t key = 0;            // keep keys > key ...
    unsigned long long ties = ~0ull;  // ... and the first `ties` equal to it

    // top-k: the k-th largest key, 8 bits at a time
    const int k = a.top_k ? a.top_k[row] : 0;
    if (k > 0 && k < n) {
        uint32_t prefix = 0, left = static_cast<uint32_t>(k);
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) bins[tid] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += kThreads) {
                const uint32_t u = key_of(to_f32<T>(x[i]));
                if (shift == 24 || (u >> (shift + 8)) == (prefix >> (shift + 8)))
                    atomicAdd(reinterpret_cast<unsigned*>(&bins[(u >> shift) & 255]), 1u);
            }
            __syncthreads();
            if (tid == 0) {
                uint32_t rest = left;
                int d = 255;
                for (; d > 0 && bins[d] < rest; d--) rest -= static_cast<uint32_t>(bins[d]);
                s_sel[0] = static_cast<uint32_t>(d);
                s_sel[1] = rest;
            }
            __syncthreads();
            prefix |= s_sel[0] << shift;
            left = s_sel[1];
            __syncthreads();
        }
        key = prefix;
        ties = left;
    }
    const uint32_t kkey = key;
    const unsigned long long kties = ties;

    // top-p: the same by sums of weights over what top-k keeps
    const float p = a.top_p ? a.top_p[row] : 1.f;
    if (p < 1.f) {
        unsigned long long sum = 0;
        for (int i = tid; i < n; i += kThreads) {
            const float v = to_f32<T>(x[i]);
            if (key_of(v) > kkey) sum += weight_of(v, top, inv_t);
        }
        sum = block_sum_u64(sum, red);
        if (kties != ~0ull) sum += kties * weight_of(logit_of(kkey), top, inv_t);
        const double want = static_cast<double>(p) * static_cast<double>(sum);  // stop at the first prefix that reaches it
        uint32_t prefix = 0;
        unsigned long long above = 0;  // weight of the keys above the prefix's range
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) bins[tid] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += kThreads) {
                const float v = to_f32<T>(x[i]);
                const uint32_t u = key_of(v);
                if (u > kkey && (shift == 24 || (u >> (shift + 8)) == (prefix >> (shift + 8))))
                    atomicAdd(&bins[(u >> shift) & 255], weight_of(v, top, inv_t));
            }
            __syncthreads();
            if (tid == 0 && kties != ~0ull && (shift == 24 || (kkey >> (shift + 8)) == (prefix >> (shift + 8))))
                bins[(kkey >> shift) & 255] += kties * weight_of(logit_of(kkey), top, inv_t);
            __syncthreads();
            if (tid == 0) {
                unsigned long long at = above;
                int d = 255;
                // the largest key's digit is always entered: its own weight may be what reaches `want`
                const int least = shift == 24 || (bk >> (shift + 8)) == (prefix >> (shift + 8))
                                      ? static_cast<int>((bk >> shift) & 255) : 255;
                for (; d > 0 && (d > least || static_cast<double>(at + bins[d]) < want); d--) at += bins[d];
                s_sel[0] = static_cast<uint32_t>(d);
                s_above = at;
            }
            __syncthreads();
            prefix |= s_sel[0] << shift;
            above = s_above;
            __syncthreads();
        }
        const unsigned long long w = weight_of(logit_of(prefix), top, inv_t);
        // ties of equal weight: as many as the sum still lacks, at least one
        unsigned long long m = 1;
        if (w > 0 && static_cast<double>(above) < want) {
            m = static_cast<unsigned long long>(ceil((want - static_cast<double>(above)) / static_cast<double>(w)));
            if (m < 1) m = 1;
        }
        if (prefix > kkey || (prefix == kkey && m < kties)) {
            key = prefix;
            ties = m;
        }
    }
    const float mp = a.min_p ? a.min_p[row] : 0.f;

    // kept weights in index order: thread t owns a run of consecutive indexes
    const int per = (n + kThreads - 1) / kThreads;
    const int i0 = min(n, tid * per), i1 = min(n, i0 + per);
    unsigned long long eq = 0;
    for (int i = i0; i < i1; i++) eq += key_of(to_f32<T>(x[i])) == key;
    // exclusive running count of ties
    __syncthreads();
    unsigned long long c = eq;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(FULL, c, o);
        if (lane >= o) c += y;
    }
    if (lane == 31) red[warp] = c;
    __syncthreads();
    unsigned long long before = c - eq;
    for (int w = 0; w < warp; w++) before += red[w];
    __syncthreads();
    auto kept = [&](int i, unsigned long long& rank) -> unsigned long long {
        const float v = to_f32<T>(x[i]);
        const uint32_t u = key_of(v);
        bool in = u > key;
        if (u == key) in = rank++ < ties;
        if (!in) return 0;
        if (mp > 0.f && exp((static_cast<double>(v) - static_cast<double>(top)) * inv_t) < static_cast<double>(mp) && u != bk) return 0;
        return weight_of(v, top, inv_t);
    };
    unsigned long long mine = 0, rank = before;
    for (int i = i0; i < i1; i++) mine += kept(i, rank);
    c = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(FULL, c, o);
        if (lane >= o) c += y;
    }
    if (lane == 31) red[warp] = c;
    __syncthreads();
    unsigned long long at = c - mine, total = 0;
    for (int w = 0; w < 32; w++) {
        if (w < warp) at += red[w];
        total += red[w];
    }
    const double goal = static_cast<double>(a.r[row]) * static_cast<double>(total);
    uint32_t found = 0xffffffffu, last = 0;
    rank = before;
    for (int i = i0; i < i1; i++) {
        const unsigned long long w = kept(i, rank);
        if (!w) continue;
        at += w;
        last = static_cast<uint32_t>(i);
        if (found == 0xffffffffu && static_cast<double>(at) >= goal) found = static_cast<uint32_t>(i);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        found = min(found, __shfl_xor_sync(FULL, found, o));
        last = max(last, __shfl_xor_sync(FULL, last, o));
    }
    __syncthreads();
    if (lane == 0) {
        sk[warp] = found;
        si[warp] = last;
    }
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < 32; w++) {
            found = min(found, sk[w]);
            last = max(last, si[w]);
        }
        a.out[row] = found != 0xffffffffu ? found : last;
    }
}

}  // namespace
}  // namespace tl

using namespace tl;

extern "C" tl_status tl_sample_rows(uint32_t* out, const void* logits, tl_dtype dtype, size_t row_stride, size_t n_rows,
                                    size_t n, const float* r, const float* temperature, const int32_t* top_k,
                                    const float* top_p, const float* min_p, void* stream) {
    clear_error();
    TL_REQUIRE(paged::dtype_ok(dtype), "tl_sample_rows: dtype %d", static_cast<int>(dtype));
    TL_REQUIRE(n > 0 && n < (1u << 22), "tl_sample_rows: n = %zu", n);
    TL_REQUIRE(row_stride >= n && row_stride <= (1ull << 36), "tl_sample_rows: row_stride %zu", row_stride);
    if (n_rows == 0) return TL_OK;
    TL_REQUIRE(n_rows <= 0x7fffffffull, "tl_sample_rows: n_rows = %zu", n_rows);
    TL_REQUIRE(out && logits && r && temperature, "tl_sample_rows: null pointer");
    TL_REQUIRE(reinterpret_cast<uintptr_t>(logits) % paged::dtype_size(dtype) == 0, "tl_sample_rows: logits misaligned");
    SampleRowsArgs a{out, logits, row_stride, static_cast<int>(n), r, temperature, top_p, min_p, top_k};
    const unsigned grid = static_cast<unsigned>(n_rows);
    const cudaStream_t s = as_stream(stream);
    if (dtype == TL_F32) k_sample_rows<float><<<grid, kThreads, 0, s>>>(a);
    else if (dtype == TL_F16) k_sample_rows<__half><<<grid, kThreads, 0, s>>>(a);
    else k_sample_rows<__nv_bfloat16><<<grid, kThreads, 0, s>>>(a);
    return check_launch("sample_rows");
}
