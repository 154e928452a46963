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
    int fits;  // the row fits shared memory
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

struct Scratch {
    unsigned long long red[32], bins[256];
    uint32_t sk[32], si[32], sel[4];
    unsigned long long above;
};

// Any row: cuts by radix selection, 8 bits of the keys at a time, straight from global memory.  The rows that the
// ways below give up on come here (thousands of equal logits at a cut, cuts far down a row).  The kept set is a
// threshold: every logit whose key is above `key`, and of those equal to it the first `ties` by index.
template <typename T>
__device__ __noinline__ uint32_t sample_by_radix(const T* x, int n, int k, float p, float mp, float r, double inv_t, float top,
                                                 uint32_t bk, Scratch& sc) {
    unsigned long long *red = sc.red, *bins = sc.bins;
    uint32_t *sk = sc.sk, *si = sc.si, *s_sel = sc.sel;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t key = 0;            // keep keys > key ...
    unsigned long long ties = ~0ull;  // ... and the first `ties` equal to it

    // top-k: the k-th largest key, 8 bits at a time
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
                sc.above = at;
            }
            __syncthreads();
            prefix |= s_sel[0] << shift;
            above = sc.above;
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
    const double goal = static_cast<double>(r) * static_cast<double>(total);
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
    for (int w = 0; w < 32; w++) {
        found = min(found, sk[w]);
        last = max(last, si[w]);
    }
    return found != 0xffffffffu ? found : last;
}

// ---- the fast ways -----------------------------------------------------------
// A row is read from global memory once and stays in shared memory where it fits.  A logit and its index make one
// 64-bit number whose order is the row's order (larger logit first, lower index first), so that every cut is one
// such number.  Weights are computed in 64 bits and summed as integers: a result does not depend on the order of
// sums, and a running sum that passes close to a border is on the right side of it.
//   k <= kSmallK  The k-th largest of the threads' maxima bounds the k-th largest logit from below: the few
//                 logits that reach it are sorted, and everything after that happens on the list.
//   otherwise     Logits are counted in 2048 bins of equal width below the largest.  The count gives the bin of
//                 the k-th exactly, and the bins around the top-p cut nearly (mass = count x weight of the bin's
//                 middle); the logits of those bins are sorted, the weights above them summed exactly, and the
//                 cut read off.  If it is not inside, or there are too many, sample_by_radix takes the row.
//   draw          sums of kept weights of 4096 consecutive logits at a time, then the warp, lane and logit in
//                 which the running sum crosses.
// A block per row: bound by the 64-bit exponentials of the rows that keep thousands of logits and by
// barriers, not by reading.
constexpr int kSmallK = 256, kBins = 2048, kList = 4096, kSegs = 16;
constexpr int kWarps = kThreads / 32;
constexpr float kDepth = 20.f;  // the bins reach to weights of e^-20

struct Row {
    const float* v;  // in shared memory
    int n;
    float top;
    double inv_t;
    float bin_scale;
    __device__ __forceinline__ int bin(float x) const { return min(kBins - 1, static_cast<int>((top - x) * bin_scale)); }
};

__device__ __forceinline__ unsigned long long place_of(float x, uint32_t i) {
    return (static_cast<unsigned long long>(key_of(x)) << 32) | (0xffffffffu - i);
}
__device__ __forceinline__ uint32_t index_of(unsigned long long place) { return 0xffffffffu - static_cast<uint32_t>(place); }

// Sorts list[0, n) in descending order; n <= kList, the list has room up to the next power of two.
__device__ void sort_list(unsigned long long* list, int n) {
    int size = 32;
    while (size < n) size <<= 1;
    for (int i = n + threadIdx.x; i < size; i += kThreads) list[i] = 0;
    __syncthreads();
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int t = threadIdx.x; t < size / 2; t += kThreads) {
                const int a = 2 * t - (t & (j - 1)), b = a + j;  // (t with a 0 bit put in at j)
                const unsigned long long x = list[a], y = list[b];
                if ((x < y) == ((a & k) == 0)) {
                    list[a] = y;
                    list[b] = x;
                }
            }
            __syncthreads();
        }
}

// Exclusive running sum over the block; `total` gets the sum.
__device__ unsigned long long scan_u64(unsigned long long v, unsigned long long* red, unsigned long long& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned long long c = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(FULL, c, o);
        if (lane >= o) c += y;
    }
    __syncthreads();
    if (lane == 31) red[warp] = c;
    __syncthreads();
    unsigned long long w = red[lane], sum = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(FULL, sum, o);
        if (lane >= o) sum += y;
    }
    total = __shfl_sync(FULL, sum, 31);
    return c - v + (warp ? __shfl_sync(FULL, sum, warp - 1) : 0ull);
}

// In a descending list: how many elements it takes until the weights, on top of `above`, reach `want`
// (n + 1 if they do not); `reached` gets the sum up to there.  n <= kList.
__device__ int prefix_reaching(const Row& R, const unsigned long long* list, int n, unsigned long long above, double want,
                               Scratch& sc, unsigned long long& reached) {
    constexpr int PER = kList / kThreads;
    unsigned long long w[PER], mine = 0;
#pragma unroll
    for (int e = 0; e < PER; e++) {
        const int i = threadIdx.x * PER + e;
        w[e] = i < n ? weight_of(logit_of(static_cast<uint32_t>(list[i] >> 32)), R.top, R.inv_t) : 0;
        mine += w[e];
    }
    unsigned long long total;
    unsigned long long at = above + scan_u64(mine, sc.red, total);
    if (threadIdx.x == 0) {
        sc.sel[0] = static_cast<uint32_t>(n + 1);
        sc.above = above + total;
    }
    __syncthreads();
    int hit = 0x7fffffff;
    unsigned long long sum = 0;
#pragma unroll
    for (int e = 0; e < PER; e++) {
        const int i = threadIdx.x * PER + e;
        at += w[e];
        if (i < n && hit == 0x7fffffff && static_cast<double>(at) >= want) {
            hit = i + 1;
            sum = at;
        }
    }
    if (hit != 0x7fffffff) atomicMin(&sc.sel[0], static_cast<uint32_t>(hit));
    __syncthreads();
    if (hit == static_cast<int>(sc.sel[0])) sc.above = sum;
    __syncthreads();
    reached = sc.above;
    return static_cast<int>(sc.sel[0]);
}

// The row's logits that `keep` holds for, into the list; their number (which may be more than fit).
template <class F>
__device__ int collect(const Row& R, unsigned long long* list, uint32_t* count, F keep) {
    if (threadIdx.x == 0) *count = 0;
    __syncthreads();
    for (int i0 = 0; i0 < R.n; i0 += kThreads) {
        const int i = i0 + threadIdx.x;
        const float x = i < R.n ? R.v[i] : -INFINITY;
        const bool in = i < R.n && keep(x, i);
        const unsigned who = __ballot_sync(FULL, in);
        if (who) {
            uint32_t at = 0;
            if ((threadIdx.x & 31) == 0) at = atomicAdd(count, __popc(who));
            at = __shfl_sync(FULL, at, 0) + __popc(who & ((1u << (threadIdx.x & 31)) - 1));
            if (in && at < kList) list[at] = place_of(x, i);
        }
    }
    __syncthreads();
    return static_cast<int>(*count);
}

// A short list in descending order holds everything that top-k left: the rest of the settings and the draw.
__device__ uint32_t draw_from_list(const Row& R, unsigned long long* list, int m, float p, float mp, float r, Scratch& sc) {
    unsigned long long* w = sc.bins;  // kSmallK weights
    static_assert(kSmallK <= 256 && kSmallK <= kThreads, "one thread a weight");
    const int t = threadIdx.x;
    const unsigned long long mine = t < m ? weight_of(logit_of(static_cast<uint32_t>(list[t] >> 32)), R.top, R.inv_t) : 0;
    if (t < kSmallK) w[t] = mine;
    unsigned long long total;
    const unsigned long long before = scan_u64(mine, sc.red, total);
    bool in = t < m;
    if (p < 1.f) in = in && (t == 0 || static_cast<double>(before) < static_cast<double>(p) * static_cast<double>(total));
    if (mp > 0.f && in && t > 0) {
        const double d = static_cast<double>(logit_of(static_cast<uint32_t>(list[t] >> 32))) - static_cast<double>(R.top);
        in = d == 0.0 || exp(d * R.inv_t) >= static_cast<double>(mp);
    }
    const int keep = __syncthreads_count(in);  // a prefix
    unsigned long long kept_sum;
    scan_u64(t < keep ? mine : 0, sc.red, kept_sum);
    const double goal = static_cast<double>(r) * static_cast<double>(kept_sum);
    uint32_t found = 0xffffffffu, last = 0;
    if (t < keep && mine > 0) {  // the running sum at this element, in index order
        const uint32_t idx = index_of(list[t]);
        unsigned long long s = 0;
        for (int j = 0; j < keep; j++)
            if (index_of(list[j]) <= idx) s += w[j];
        last = idx;
        if (static_cast<double>(s) >= goal) found = idx;
    }
    found = __reduce_min_sync(FULL, found);
    last = __reduce_max_sync(FULL, last);
    __syncthreads();
    if ((t & 31) == 0) {
        sc.sk[t >> 5] = found;
        sc.si[t >> 5] = last;
    }
    __syncthreads();
    found = __reduce_min_sync(FULL, sc.sk[t & 31]);
    last = __reduce_max_sync(FULL, sc.si[t & 31]);
    return found != 0xffffffffu ? found : last;
}

// Draw over the whole row among the logits not below `cut` whose weight reaches mp.
__device__ uint32_t draw_from_row(const Row& R, unsigned long long cut, float mp, float r, Scratch& sc, unsigned long long* segs) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per = 4 * ((R.n + kSegs * 4 * kThreads - 1) / (kSegs * 4 * kThreads));  // consecutive logits of a thread
    const int seg = per * kThreads, nseg = (R.n + seg - 1) / seg;
    auto weight = [&](int i) -> unsigned long long {
        const float x = R.v[i];
        if (place_of(x, i) < cut) return 0;
        const double d = static_cast<double>(x) - static_cast<double>(R.top), e = exp(d * R.inv_t);
        if (mp > 0.f && d != 0.0 && e < static_cast<double>(mp)) return 0;
        return __double2ull_rn(e * kOne);
    };
    auto mine_of = [&](int s) {
        unsigned long long m = 0;
        const int i0 = s * seg + threadIdx.x * per;
        for (int i = i0; i < min(R.n, i0 + per); i++) m += weight(i);
        return m;
    };
    for (int s = 0; s < nseg; s++) {
        unsigned long long m = mine_of(s);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(FULL, m, o);
        if (lane == 0) segs[s * kWarps + warp] = m;
    }
    for (int i = nseg * kWarps + threadIdx.x; i < kSegs * kWarps; i += kThreads) segs[i] = 0;
    __syncthreads();
    const unsigned long long own = threadIdx.x < kSegs * kWarps ? segs[threadIdx.x] : 0;
    unsigned long long total;
    const unsigned long long at = scan_u64(own, sc.red, total);
    const double goal = static_cast<double>(r) * static_cast<double>(total);
    // the first entry whose running sum reaches the goal and which holds weight
    if (threadIdx.x == 0) {
        sc.sel[0] = 0xffffffffu;
        sc.sel[1] = 0;
    }
    __syncthreads();
    if (own) {
        if (static_cast<double>(at + own) >= goal) atomicMin(&sc.sel[0], static_cast<uint32_t>(threadIdx.x));
        atomicMax(&sc.sel[1], static_cast<uint32_t>(threadIdx.x));
    }
    __syncthreads();
    const bool crossed = sc.sel[0] != 0xffffffffu;
    const int e = static_cast<int>(crossed ? sc.sel[0] : sc.sel[1]);  // (no crossing: the last logit with weight)
    if (threadIdx.x == static_cast<unsigned>(e)) sc.above = at;
    __syncthreads();
    if (warp == e % kWarps) {
        const int s = e / kWarps;
        const unsigned long long m = mine_of(s);
        unsigned long long c = m;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long y = __shfl_up_sync(FULL, c, o);
            if (lane >= o) c += y;
        }
        const unsigned long long before = sc.above + c - m;
        const unsigned hit = __ballot_sync(FULL, m && static_cast<double>(before + m) >= goal), any = __ballot_sync(FULL, m != 0);
        const int who = hit ? __ffs(hit) - 1 : 31 - __clz(any);
        if (lane == who) {
            unsigned long long sum = before;
            const int i0 = s * seg + threadIdx.x * per;
            uint32_t last = 0, found = 0xffffffffu;
            for (int i = i0; i < min(R.n, i0 + per); i++) {
                const unsigned long long w = weight(i);
                if (!w) continue;
                sum += w;
                last = i;
                if (found == 0xffffffffu && static_cast<double>(sum) >= goal) found = i;
            }
            sc.sel[2] = found != 0xffffffffu ? found : last;
        }
    }
    __syncthreads();
    return sc.sel[2];
}

// Block = one row, all of it in shared memory.
template <typename T>
__global__ void __launch_bounds__(kThreads) k_sample_rows(SampleRowsArgs a) {
    extern __shared__ __align__(16) unsigned long long smem_rows[];
    __shared__ Scratch sc;
    __shared__ unsigned long long segs[kSegs * kWarps];
    unsigned long long* list = smem_rows;                                 // kList
    uint32_t* hist = reinterpret_cast<uint32_t*>(list + kList);           // kBins
    float* v = reinterpret_cast<float*>(hist + kBins);                    // the row, when it fits
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T* x = static_cast<const T*>(a.logits) + static_cast<size_t>(row) * a.row_stride;
    const int n = a.n;
    const float temp = a.temperature[row];
    const int k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.f, mp = a.min_p ? a.min_p[row] : 0.f, r = a.r[row];

    // the largest logit, lowest index; NaN or +inf anywhere; the row into shared memory
    uint32_t bk = 0, bi = 0xffffffffu;
    int bad = 0;
    auto see = [&](float f, int i) {
        if (!(f < INFINITY)) bad = 1;
        if (f == f) {
            const uint32_t u = key_of(f);
            if (u > bk) {  // (a thread's indexes rise)
                bk = u;
                bi = static_cast<uint32_t>(i);
            }
        }
    };
    constexpr int VE = 16 / sizeof(T);
    const int head = a.fits ? min(n, static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T))) : n;
    for (int i = tid; i < head; i += kThreads) {
        const float f = to_f32<T>(x[i]);
        see(f, i);
        if (a.fits) v[i] = f;
    }
    if (a.fits) {
        const int nv = (n - head) / VE;
#pragma unroll 4
        for (int q = tid; q < nv; q += kThreads) {
            const uint4 raw = *reinterpret_cast<const uint4*>(x + head + q * VE);
            const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
            for (int c = 0; c < VE; c++) {
                const float f = to_f32<T>(e[c]);
                see(f, head + q * VE + c);
                v[head + q * VE + c] = f;
            }
        }
        for (int i = head + nv * VE + tid; i < n; i += kThreads) {
            const float f = to_f32<T>(x[i]);
            see(f, i);
            v[i] = f;
        }
    }
    const uint32_t own_best = bk;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const uint32_t u = __shfl_xor_sync(FULL, bk, o), i = __shfl_xor_sync(FULL, bi, o);
        if (u > bk || (u == bk && i < bi)) {
            bk = u;
            bi = i;
        }
    }
    if (lane == 0) {
        sc.sk[warp] = bk;
        sc.si[warp] = bi;
    }
    bad = __syncthreads_or(bad);
    bk = sc.sk[lane];
    bi = sc.si[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const uint32_t u = __shfl_xor_sync(FULL, bk, o), i = __shfl_xor_sync(FULL, bi, o);
        if (u > bk || (u == bk && i < bi)) {
            bk = u;
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
    __syncthreads();  // sk and si have been read
    Row R{v, n, top, inv_t, static_cast<float>(kBins / (kDepth * static_cast<double>(temp)))};
    uint32_t answer = 0xffffffffu;
    bool done = false;
    if (a.fits) {
        const bool by_k = k > 0 && k < n;
        if (by_k && k <= kSmallK) {
            // the k-th largest of the threads' best keys, by bisection
            uint32_t lo = 0, hi = bk;  // count(best >= lo) >= k or lo = 0
            while (lo < hi) {
                const uint32_t mid = lo + (hi - lo) / 2 + ((hi - lo) & 1);
                if (__syncthreads_count(own_best >= mid) >= k) lo = mid;
                else hi = mid - 1;
            }
            const int m = collect(R, list, &sc.sel[3], [&](float f, int) { return key_of(f) >= lo; });
            if (m <= kList) {
                sort_list(list, m);
                answer = draw_from_list(R, list, min(k, m), p, mp, r, sc);
                done = true;
            }
        } else {
            unsigned long long cut = 0;
            done = true;
            if (by_k || p < 1.f) {
                for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
                __syncthreads();
                for (int i = tid; i < n; i += kThreads) atomicAdd(&hist[R.bin(v[i])], 1u);
                __syncthreads();
            }
            uint32_t room = 0xffffffffu;  // logits left by top-k
            if (by_k) {
                // the bin of the k-th
                const uint32_t c0 = hist[2 * tid], c1 = hist[2 * tid + 1];
                unsigned long long all;
                const uint32_t before = static_cast<uint32_t>(scan_u64(c0 + c1, sc.red, all));
                const uint32_t uk = static_cast<uint32_t>(k);
                if (before < uk && uk <= before + c0 + c1) {
                    const bool second = uk > before + c0;
                    sc.sel[0] = 2 * tid + second;
                    sc.sel[1] = uk - before - (second ? c0 : 0);  // which of the bin's, from 1
                }
                __syncthreads();
                const int b = static_cast<int>(sc.sel[0]), at = static_cast<int>(sc.sel[1]);
                const int m = collect(R, list, &sc.sel[3], [&](float f, int) { return R.bin(f) == b; });
                if (m <= kList) {
                    sort_list(list, m);
                    cut = list[at - 1];
                    room = uk;
                } else {
                    done = false;
                }
                __syncthreads();
            }
            if (done && p < 1.f) {
                if (!(p > 0.f)) {
                    cut = place_of(top, bi);
                } else {
                    // masses of the bins, from their counts and middles; those that top-k cut off are left out
                    const float step = 20.f / kBins;
                    const uint32_t c0 = hist[2 * tid], c1 = hist[2 * tid + 1];
                    unsigned long long all;
                    const uint32_t nb = static_cast<uint32_t>(scan_u64(c0 + c1, sc.red, all));
                    const uint32_t k0 = min(c0, room > nb ? room - nb : 0u), k1 = min(c1, room > nb + c0 ? room - nb - c0 : 0u);
                    const float m0 = k0 * expf(-(2 * tid + 0.5f) * step), m1 = k1 * expf(-(2 * tid + 1.5f) * step);
                    constexpr double kMass = 1073741824.0;  // 2^30: sums of 2^22 logits fit
                    const unsigned long long w0 = __double2ull_rn(m0 * kMass), w1 = __double2ull_rn(m1 * kMass);
                    unsigned long long mass;
                    const unsigned long long mb = scan_u64(w0 + w1, sc.red, mass);
                    // the bins in which the cut may lie: its mass 0.2 % up and down
                    const double goal = static_cast<double>(p) * static_cast<double>(mass), slack = 0.002 * static_cast<double>(mass);
                    if (tid == 0) {
                        sc.sel[0] = kBins - 1;
                        sc.sel[1] = kBins - 1;
                    }
                    __syncthreads();
                    if (static_cast<double>(mb + w0) >= goal - slack) atomicMin(&sc.sel[0], static_cast<uint32_t>(2 * tid));
                    else if (static_cast<double>(mb + w0 + w1) >= goal - slack) atomicMin(&sc.sel[0], static_cast<uint32_t>(2 * tid + 1));
                    if (static_cast<double>(mb + w0) >= goal + slack) atomicMin(&sc.sel[1], static_cast<uint32_t>(2 * tid));
                    else if (static_cast<double>(mb + w0 + w1) >= goal + slack) atomicMin(&sc.sel[1], static_cast<uint32_t>(2 * tid + 1));
                    __syncthreads();
                    const int ba = static_cast<int>(sc.sel[0]), bb = static_cast<int>(sc.sel[1]);
                    __syncthreads();
                    // exact: the weights above those bins and of everything; the list of the bins between
                    unsigned long long over = 0, sum = 0;
                    const int m = collect(R, list, &sc.sel[3], [&](float f, int i) {
                        if (place_of(f, i) < cut) return false;
                        const unsigned long long w = weight_of(f, top, inv_t);
                        const int b = R.bin(f);
                        sum += w;
                        if (b < ba) over += w;
                        return b >= ba && b <= bb;
                    });
                    unsigned long long over_all, sum_all, reached;
                    scan_u64(over, sc.red, over_all);
                    scan_u64(sum, sc.red, sum_all);
                    const double want = static_cast<double>(p) * static_cast<double>(sum_all);
                    if (m <= kList && (static_cast<double>(over_all) < want || ba == 0)) {
                        sort_list(list, m);
                        const int t = prefix_reaching(R, list, m, over_all, want, sc, reached);
                        if (t <= m) cut = max(cut, list[t - 1]);
                        else done = false;
                        __syncthreads();
                    } else {
                        done = false;
                    }
                }
            }
            if (done) answer = draw_from_row(R, cut, mp, r, sc, segs);
        }
    }
    __syncthreads();
    if (!done) answer = sample_by_radix<T>(x, n, k, p, mp, r, inv_t, top, bk, sc);
    if (tid == 0) a.out[row] = answer;
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
    const size_t base = kList * 8 + kBins * 4, most = 227 * 1024 - sizeof(Scratch) - kSegs * kWarps * 8 - 1024;
    const bool fits = base + n * 4 <= most;
    SampleRowsArgs a{out, logits, row_stride, static_cast<int>(n), r, temperature, top_p, min_p, top_k, fits};
    const int smem = static_cast<int>(fits ? base + n * 4 : base);
    const unsigned grid = static_cast<unsigned>(n_rows);
    const cudaStream_t s = as_stream(stream);
    auto run = [&](auto kernel) -> tl_status {
        TL_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        kernel<<<grid, kThreads, smem, s>>>(a);
        return TL_OK;
    };
    if (dtype == TL_F32) TL_TRY(run(k_sample_rows<float>));
    else if (dtype == TL_F16) TL_TRY(run(k_sample_rows<__half>));
    else TL_TRY(run(k_sample_rows<__nv_bfloat16>));
    return check_launch("sample_rows");
}
