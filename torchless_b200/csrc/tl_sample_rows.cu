// tl_sample_rows.cu -- tl_sample_rows: temperature, top-k, top-p and min-p for
// many rows, each with its own settings.
#include <limits.h>
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
    int segs;  // segments of kSeg logits
    int rows;  // the grid is as large, or twice (see tl_sample_rows)
};

// Order-preserving key of a logit: larger logit, larger key; -0 and +0 the same.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// 32-bit to 64-bit floating point by integer operations (the conversion instruction runs at a quarter of the rate of
// the 64-bit arithmetic).  Zero and subnormals become about 2^-127: no weight changes by 2^-40.  Infinity becomes about
// 2^128, which a large temperature brings near the other logits: the weight of -inf is 0 and never comes from here.
__device__ __forceinline__ double widen(float x) {
    const uint32_t u = __float_as_uint(x);
    return __hiloint2double(static_cast<int>((u & 0x80000000u) | (((u & 0x7fffffffu) >> 3) + (896u << 20))), static_cast<int>(u << 29));
}

__constant__ double kPow2[32] = {  // 2^(j / 32)
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237, 1.0905077326652577, 1.1143867425958924,
    1.1387886347566916, 1.1637248587775775, 1.189207115002721, 1.215247359980469, 1.241857812073484,
    1.2690509571917332, 1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228, 1.5422108254079407,
    1.5759808451078865, 1.6104903319492543, 1.645755478153965, 1.681792830507429, 1.718619298122478,
    1.7562521603732995, 1.7947090750031072, 1.8340080864093424, 1.8741676341103, 1.9152065613971474,
    1.9571441241754002};

// A row's scale: weights are 2^((x - top) * c / 32), c = 32 log2(e) / temperature.
struct Scale {
    double top, c;
    const double* pow2;  // kPow2 in shared memory
};

// The weight of a logit as a multiple of 2^-40.  2^(t / 32) = 2^(k >> 5) 2^((k & 31) / 32) 2^(f / 32) with t = k + f,
// |f| <= 1/2; the last factor by its series to the 5th power of f ln2 / 32 (what is left out is below 2^-48), all in
// 64 bits, then rounded to a multiple of 2^-40 by adding 2^52.  x is finite.
__device__ __forceinline__ unsigned long long weight_of(float x, const Scale& s) {
    const double t = fmax((widen(x) - s.top) * s.c, -1400.0);  // 2^(-1400 / 32) rounds to 0
    const double magic = 6755399441055744.0;                   // 1.5 * 2^52: k in the low bits
    const double r = t + magic;
    const int k = __double2loint(r);
    const double f = t - (r - magic);
    double q = 3.9737099845494154e-11;
    q = fma(q, f, 9.172562701824643e-09);
    q = fma(q, f, 1.6938509724371819e-06);
    q = fma(q, f, 0.00023459619820224677);
    q = fma(q, f, 0.02166084939249829);
    q = fma(q, f, 1.0);
    q *= s.pow2[k & 31];
    const double v = __hiloint2double(__double2hiint(q) + (((k >> 5) + 40) << 20), __double2loint(q));
    return static_cast<unsigned long long>(__double_as_longlong(v + 4503599627370496.0)) & 0xfffffffffffffull;
}

// The same for any logit up to the largest: none of -inf, whatever the temperature.
__device__ __forceinline__ unsigned long long weight_of_any(float x, const Scale& s) {
    return x > -INFINITY ? weight_of(x, s) : 0ull;
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
__device__ __noinline__ uint32_t sample_by_radix(const T* x, int n, int k, float p, float mp, float r, const Scale& ws, uint32_t bk,
                                                 Scratch& sc) {
    unsigned long long *red = sc.red, *bins = sc.bins;
    uint32_t *sk = sc.sk, *si = sc.si, *s_sel = sc.sel;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t key = 0;            // keep keys > key ...
    unsigned long long ties = ~0ull;  // ... and the first `ties` equal to it

    // top-k: the k-th largest key, 8 bits at a time
    if (k > 0 && k < n) {
        uint32_t prefix = 0, left = static_cast<uint32_t>(k);
#pragma unroll 1
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) bins[tid] = 0;
            __syncthreads();
#pragma unroll 1
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
#pragma unroll 1
        for (int i = tid; i < n; i += kThreads) {
            const float v = to_f32<T>(x[i]);
            if (key_of(v) > kkey) sum += weight_of_any(v, ws);
        }
        sum = block_sum_u64(sum, red);
        if (kties != ~0ull) sum += kties * weight_of_any(logit_of(kkey), ws);
        const double want = static_cast<double>(p) * static_cast<double>(sum);  // stop at the first prefix that reaches it
        uint32_t prefix = 0;
        unsigned long long above = 0;  // weight of the keys above the prefix's range
#pragma unroll 1
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) bins[tid] = 0;
            __syncthreads();
#pragma unroll 1
            for (int i = tid; i < n; i += kThreads) {
                const float v = to_f32<T>(x[i]);
                const uint32_t u = key_of(v);
                if (u > kkey && (shift == 24 || (u >> (shift + 8)) == (prefix >> (shift + 8))))
                    atomicAdd(&bins[(u >> shift) & 255], weight_of_any(v, ws));
            }
            __syncthreads();
            if (tid == 0 && kties != ~0ull && (shift == 24 || (kkey >> (shift + 8)) == (prefix >> (shift + 8))))
                bins[(kkey >> shift) & 255] += kties * weight_of_any(logit_of(kkey), ws);
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
        const unsigned long long w = weight_of_any(logit_of(prefix), ws);
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
        const unsigned long long w = weight_of_any(v, ws);
        return mp > 0.f && u != bk && static_cast<double>(w) < static_cast<double>(mp) * kOne ? 0 : w;
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
#pragma unroll 1
    for (int w = 0; w < 32; w++) {
        if (w < warp) at += red[w];
        total += red[w];
    }
    const double goal = static_cast<double>(r) * static_cast<double>(total);
    uint32_t found = 0xffffffffu, last = 0;
    rank = before;
#pragma unroll 1
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
#pragma unroll 1
    for (int w = 0; w < 32; w++) {
        found = min(found, sk[w]);
        last = max(last, si[w]);
    }
    return found != 0xffffffffu ? found : last;
}

// ---- the fast ways -----------------------------------------------------------
// A row is read from global memory once and stays in shared memory where it fits (else it is read again from L2).
// A logit and its index make one 64-bit number whose order is the row's order (larger logit first, lower index
// first), so that every cut is one such number.  Weights are computed in 64 bits and summed as integers: a result
// does not depend on the order of sums, and a running sum that passes close to a border is on the right side of it.
//   k <= kSmallK  The k-th largest of the threads' maxima bounds the k-th largest logit from below: the few
//                 logits that reach it are sorted, and everything after that happens on the list.
//   otherwise     Logits are counted in 2048 bins of equal width below the largest.  The count gives the bin of
//                 the k-th exactly, and the bins around the top-p cut nearly (mass = count x weight of the bin's
//                 middle); the logits of those bins are sorted, the weights above them summed exactly, and the
//                 cut read off.  If it is not inside, or there are too many, sample_by_radix takes the row.
//   draw          sums of kept weights of 128 consecutive logits (one a warp, 4 a lane), then the lane and logit
//                 in which the running sum crosses.
// A block per row.  An instruction that is executed once costs some 35 cycles (its line of code comes from L2), so
// for one row the length of the path counts as much as the work on it; with many rows the 64-bit arithmetic of the
// rows that keep thousands of logits does.  32000 logits of fp32, 1 row / 256 rows: top-k below 257 with top-p and
// min-p 13 / 31 us, no cut 20 / 43 us, top-p alone 31 / 74 us, mixed rows 54 us (0.6 TB/s); by radix selection 156 /
// 343, 76 / 156, 465 / 1142 us.  With the row read again from L2 in place of shared memory 14 / 37, 23 / 53, 35 / 88 us.
// 512 threads a row, two rows an SM, are no faster.
constexpr int kSmallK = 256, kBins = 2048, kList = 4096, kSeg = 4 * kThreads, kMaxSegs = 64;
constexpr int kWarps = kThreads / 32;
constexpr float kDepth = 20.f;  // the bins reach to weights of e^-20

struct Row {
    const float* v;  // positions [0, segs * kSeg) in shared memory; logit i is position i + pad, the others are -inf
    const void* x;   // the row in global memory
    int n, pad, segs;
    float top;
    float bin_scale;
    unsigned long long* cells;  // sums of the weights of 128 positions: [segs][kWarps]
    __device__ __forceinline__ int bin(float f) const { return min(kBins - 1, static_cast<int>((top - f) * bin_scale)); }
};

// The 4 positions of this thread in segment s.
template <typename T, bool SMEM>
__device__ __forceinline__ void four(const Row& R, int s, float (&f)[4]) {
    const int j = s * kSeg + 4 * threadIdx.x;
    if (SMEM) {
        const float4 q = *reinterpret_cast<const float4*>(R.v + j);
        f[0] = q.x; f[1] = q.y; f[2] = q.z; f[3] = q.w;
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) f[e] = j + e < R.n ? to_f32<T>(static_cast<const T*>(R.x)[j + e]) : -INFINITY;
    }
}

__device__ __forceinline__ unsigned long long place_of(float x, uint32_t i) {
    return (static_cast<unsigned long long>(key_of(x)) << 32) | (0xffffffffu - i);
}
__device__ __forceinline__ uint32_t index_of(unsigned long long place) { return 0xffffffffu - static_cast<uint32_t>(place); }
__device__ __forceinline__ float logit_at(unsigned long long place) { return logit_of(static_cast<uint32_t>(place >> 32)); }

// Sorts list[0, n) in descending order; the list has room up to the next power of two.
__device__ __noinline__ void sort_list(unsigned long long* list, int n, Scratch& sc) {
    if (n <= kSmallK) {  // the place of each is the number of larger ones: 4 threads count for each
        const int t = threadIdx.x >> 2;
        const unsigned long long mine = t < n ? list[t] : 0;
        int rank = 0;
        for (int j = threadIdx.x & 3; j < n; j += 4) rank += list[j] > mine;
        rank += __shfl_xor_sync(FULL, rank, 1);
        rank += __shfl_xor_sync(FULL, rank, 2);
        __syncthreads();
        if (t < n && (threadIdx.x & 3) == 0) list[rank] = mine;
        __syncthreads();
        return;
    }
    int size = 512;
    while (size < n) size <<= 1;
    for (int i = n + threadIdx.x; i < size; i += kThreads) list[i] = 0;
    __syncthreads();
#pragma unroll 1
    for (int k = 2; k <= size; k <<= 1)
#pragma unroll 1
        for (int j = k >> 1; j > 0; j >>= 1) {
            if (j >= 32) __syncthreads();  // (up to 32 apart, a warp's pairs lie in its own 64 elements)
            else __syncwarp();
#pragma unroll 1
            for (int t = threadIdx.x; t < size / 2; t += kThreads) {
                const int a = 2 * t - (t & (j - 1)), b = a + j;  // (t with a 0 bit put in at j)
                const unsigned long long x = list[a], y = list[b];
                if ((x < y) == ((a & k) == 0)) {
                    list[a] = y;
                    list[b] = x;
                }
            }
        }
    __syncthreads();
}

// Exclusive running sum over the block; `total` gets the sum.
__device__ __noinline__ unsigned long long scan_u64(unsigned long long v, unsigned long long* red, unsigned long long& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned long long mine = v, base = 0, sum = 0;
#pragma unroll 1
    for (int turn = 0; turn < 2; turn++) {  // over the lanes, then over the warps
        unsigned long long c = mine;
#pragma unroll 1
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long y = __shfl_up_sync(FULL, c, o);
            if (lane >= o) c += y;
        }
        if (turn == 0) {
            base = c - mine;
            __syncthreads();
            if (lane == 31) red[warp] = c;
            __syncthreads();
            mine = red[lane];
        } else {
            sum = c;
        }
    }
    total = __shfl_sync(FULL, sum, 31);
    const unsigned long long up = __shfl_sync(FULL, sum, max(0, warp - 1));
    return base + (warp ? up : 0ull);
}

// In a descending list: how many elements it takes until the weights, on top of `above`, reach `want`; n + 1 if
// they do not.  n <= kList.
__device__ __noinline__ int prefix_reaching(const Row& R, const Scale& ws, const unsigned long long* list, int n,
                                            unsigned long long above, double want, Scratch& sc) {
    const int per = (n + kThreads - 1) / kThreads, i0 = threadIdx.x * per, i1 = min(n, i0 + per);
    unsigned long long mine = 0, total;
#pragma unroll 1
    for (int i = i0; i < i1; i++) mine += weight_of(logit_at(list[i]), ws);
    unsigned long long at = above + scan_u64(mine, sc.red, total);
    if (threadIdx.x == 0) sc.sel[0] = static_cast<uint32_t>(n + 1);
    __syncthreads();
    if (static_cast<double>(at + mine) >= want) {
#pragma unroll 1
        for (int i = i0; i < i1; i++) {
            at += weight_of(logit_at(list[i]), ws);
            if (static_cast<double>(at) >= want) {
                atomicMin(&sc.sel[0], static_cast<uint32_t>(i + 1));
                break;
            }
        }
    }
    __syncthreads();
    return static_cast<int>(sc.sel[0]);
}

// The logits (above -inf) that `keep(x, position)` holds for, into the list; their number (which may be more than
// fit).  `done(segment)` follows each segment, with the whole warp.
template <typename T, bool SMEM, class F, class G>
__device__ __forceinline__ int collect(const Row& R, unsigned long long* list, uint32_t* count, F keep, G done) {
    if (threadIdx.x == 0) *count = 0;
    __syncthreads();
#pragma unroll 1
    for (int s = 0; s < R.segs; s++) {
        float f[4];
        four<T, SMEM>(R, s, f);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int j = s * kSeg + 4 * threadIdx.x + e;
            if (keep(f[e], j - R.pad) && f[e] > -INFINITY) {
                const uint32_t at = atomicAdd(count, 1u);
                if (at < kList) list[at] = place_of(f[e], j - R.pad);
            }
        }
        done(s);
    }
    __syncthreads();
    return static_cast<int>(*count);
}

// A short list in descending order holds everything that top-k left: the rest of the settings and the draw.
__device__ __noinline__ uint32_t draw_from_list(const Scale& ws, const unsigned long long* list, int m, float p, float mp,
                                                float r, Scratch& sc) {
    unsigned long long* w = sc.bins;  // kSmallK weights
    static_assert(kSmallK <= 256 && 4 * kSmallK <= kThreads, "four threads an element");
    const int t = threadIdx.x;
    const unsigned long long mine = t < m ? weight_of(logit_at(list[t]), ws) : 0;
    if (t < kSmallK) w[t] = mine;
    unsigned long long total, kept_sum;
    const unsigned long long before = scan_u64(mine, sc.red, total);
    bool in = t < m;
    if (p < 1.f) in = in && (t == 0 || static_cast<double>(before) < static_cast<double>(p) * static_cast<double>(total));
    if (mp > 0.f && in && (list[t] >> 32) != (list[0] >> 32)) in = static_cast<double>(mine) >= static_cast<double>(mp) * kOne;
    const int keep = __syncthreads_count(in);  // a prefix
    scan_u64(t < keep ? mine : 0, sc.red, kept_sum);
    const double goal = static_cast<double>(r) * static_cast<double>(kept_sum);
    // the running sum at each kept element, in index order: 4 threads add for each
    const int e = t >> 2;
    const uint32_t idx = e < keep ? index_of(list[e]) : 0u;
    unsigned long long s = 0;
#pragma unroll 1
    for (int j = t & 3; j < keep; j += 4)
        if (index_of(list[j]) <= idx) s += w[j];
    s += __shfl_xor_sync(FULL, s, 1);
    s += __shfl_xor_sync(FULL, s, 2);
    uint32_t found = 0xffffffffu, last = 0;
    if (e < keep && w[e] > 0) {
        last = idx;
        if (static_cast<double>(s) >= goal) found = idx;
    }
    if (t == 0) {
        sc.sel[0] = 0xffffffffu;
        sc.sel[1] = 0;
    }
    __syncthreads();
    found = __reduce_min_sync(FULL, found);
    last = __reduce_max_sync(FULL, last);
    if ((t & 31) == 0) {
        atomicMin(&sc.sel[0], found);
        atomicMax(&sc.sel[1], last);
    }
    __syncthreads();
    return sc.sel[0] != 0xffffffffu ? sc.sel[0] : sc.sel[1];
}

// This thread's 4 weights of segment s: of the logits not below `cut` whose weight reaches `least`.
template <typename T, bool SMEM>
__device__ __forceinline__ unsigned long long kept_weights(const Row& R, const Scale& ws, unsigned long long cut, double least, int s,
                                                           unsigned long long (&w)[4]) {
    float f[4];
    four<T, SMEM>(R, s, f);
    const float cut_x = cut ? logit_at(cut) : -INFINITY;  // (no cut: above -inf, which the padding holds too)
    const int cut_i = cut ? static_cast<int>(index_of(cut)) : INT_MIN;
    unsigned long long sum = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const int i = s * kSeg + 4 * threadIdx.x + e - R.pad;
        w[e] = 0;
        if (f[e] > cut_x || (f[e] == cut_x && i <= cut_i)) {
            w[e] = weight_of(f[e], ws);
            if (static_cast<double>(w[e]) < least && f[e] != R.top) w[e] = 0;
        }
        sum += w[e];
    }
    return sum;
}
__device__ __forceinline__ unsigned long long warp_total(unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
    return v;
}

// The draw over the whole row, from the cells' sums.
template <typename T, bool SMEM>
__device__ __noinline__ uint32_t draw_from_cells(const Row& R, const Scale& ws, unsigned long long cut, double least, float r,
                                                 Scratch& sc) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, cells = R.segs * kWarps;
    const int per = (cells + kThreads - 1) / kThreads, c0 = threadIdx.x * per, c1 = min(cells, c0 + per);
    unsigned long long own = 0, total;
#pragma unroll 1
    for (int c = c0; c < c1; c++) own += R.cells[c];
    unsigned long long at = scan_u64(own, sc.red, total);
    const double goal = static_cast<double>(r) * static_cast<double>(total);
    // the first cell whose running sum reaches the goal and which holds weight; if none does, the last with weight
    if (threadIdx.x == 0) {
        sc.sel[0] = 0xffffffffu;
        sc.sel[1] = 0;
    }
    __syncthreads();
#pragma unroll 1
    for (int c = c0; c < c1; c++) {
        const unsigned long long w = R.cells[c];
        if (!w) continue;
        at += w;
        if (static_cast<double>(at) >= goal) atomicMin(&sc.sel[0], static_cast<uint32_t>(c));
        atomicMax(&sc.sel[1], static_cast<uint32_t>(c));
        if (static_cast<double>(at) >= goal) break;
    }
    __syncthreads();
    const int cell = static_cast<int>(sc.sel[0] != 0xffffffffu ? sc.sel[0] : sc.sel[1]);
    if (cell >= c0 && cell < c1) {  // (if this thread went on behind the cell, `at` is too large: add up again)
        unsigned long long b = 0;
#pragma unroll 1
        for (int c = c0; c < cell; c++) b += R.cells[c];
        sc.above = b;
        sc.sel[3] = threadIdx.x;
    }
    at = scan_u64(own, sc.red, total);
    if (threadIdx.x == sc.sel[3]) sc.above += at;
    __syncthreads();
    if (warp == cell % kWarps) {
        unsigned long long w[4];
        const unsigned long long m = kept_weights<T, SMEM>(R, ws, cut, least, cell / kWarps, w);
        unsigned long long c = m;
#pragma unroll 1
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long y = __shfl_up_sync(FULL, c, o);
            if (lane >= o) c += y;
        }
        unsigned long long sum = sc.above + c - m;
        const unsigned hit = __ballot_sync(FULL, m && static_cast<double>(sum + m) >= goal), any = __ballot_sync(FULL, m != 0);
        if (lane == (hit ? __ffs(hit) - 1 : 31 - __clz(any))) {
            int last = 0, found = -1;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (!w[e]) continue;
                sum += w[e];
                last = e;
                if (found < 0 && static_cast<double>(sum) >= goal) found = e;
            }
            sc.sel[2] = static_cast<uint32_t>(cell / kWarps * kSeg + 4 * threadIdx.x + (found >= 0 ? found : last) - R.pad);
        }
    }
    __syncthreads();
    return sc.sel[2];
}

// sample_max: first strict maximum above -inf; NaN at index 0 keeps 0.
template <typename T>
__device__ __noinline__ uint32_t first_max(const T* x, int n, Scratch& sc) {
    if (threadIdx.x == 0) sc.above = 0;
    __syncthreads();
    unsigned long long best = 0;
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const float f = to_f32<T>(x[i]);
        if (f == f) best = max(best, place_of(f, i));
    }
#pragma unroll 1
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(FULL, best, o));
    if ((threadIdx.x & 31) == 0) atomicMax(&sc.above, best);
    __syncthreads();
    const float x0 = to_f32<T>(x[0]);
    return x0 != x0 || !sc.above || logit_at(sc.above) == -INFINITY ? 0u : index_of(sc.above);
}

// The larger of two; NaN (the positive one) if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// Everything but greedy rows.
template <typename T, bool SMEM>
__device__ __forceinline__ uint32_t sample_row(const Row& R, const Scale& ws, uint32_t best, uint32_t bk, uint32_t lk, int k, float p,
                                               float mp, float r, unsigned long long* list, uint32_t* hist, Scratch& sc) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const double least = mp > 0.f ? static_cast<double>(mp) * kOne : 0.0;
    const bool by_k = k > 0 && k < R.n;
    auto nothing = [](int) {};
    if (by_k && k <= kSmallK) {
        // the k-th largest of the threads' best keys, from below: bisection, to 2^-12 of where they lie
        uint32_t lo = 0, hi = bk;
        if (__syncthreads_count(best >= lk) >= k) lo = lk;
        const uint32_t fine = (hi - lo) >> 12;
#pragma unroll 1
        while (hi - lo > fine) {
            const uint32_t mid = lo + (hi - lo) / 2 + ((hi - lo) & 1);
            if (__syncthreads_count(best >= mid) >= k) lo = mid;
            else hi = mid - 1;
        }
        const float bound = lo <= key_of(-INFINITY) ? -INFINITY : logit_of(lo);
        const int m = collect<T, SMEM>(R, list, &sc.sel[3], [&](float f, int) { return f >= bound; }, nothing);
        if (m > kList) return 0xffffffffu;
        sort_list(list, m, sc);
        return draw_from_list(ws, list, min(k, m), p, mp, r, sc);
    }
    unsigned long long cut = 0;
    bool summed = false;  // the cells hold the kept weights
    if (by_k || p < 1.f) {
        for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
        __syncthreads();
#pragma unroll 1
        for (int s = 0; s < R.segs; s++) {
            float f[4];
            four<T, SMEM>(R, s, f);
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (f[e] > -INFINITY) atomicAdd(&hist[R.bin(f[e])], 1u);
        }
        __syncthreads();
        const uint32_t c0 = hist[2 * tid], c1 = hist[2 * tid + 1];
        unsigned long long all;
        const uint32_t before = static_cast<uint32_t>(scan_u64(c0 + c1, sc.red, all));
        uint32_t room = 0xffffffffu;  // logits left by top-k
        if (by_k && static_cast<unsigned long long>(k) < all) {
            const uint32_t uk = static_cast<uint32_t>(k);
            if (before < uk && uk <= before + c0 + c1) {
                const bool second = uk > before + c0;
                sc.sel[0] = 2 * tid + second;
                sc.sel[1] = uk - before - (second ? c0 : 0);  // which of its bin, from 1
            }
            __syncthreads();
            const int b = static_cast<int>(sc.sel[0]), at = static_cast<int>(sc.sel[1]);
            const int m = collect<T, SMEM>(R, list, &sc.sel[3], [&](float f, int) { return R.bin(f) == b; }, nothing);
            if (m > kList) return 0xffffffffu;
            sort_list(list, m, sc);
            cut = list[at - 1];
            room = uk;
            __syncthreads();
        }
        if (p < 1.f && !(p > 0.f)) {  // the first of the order alone
            const int m = collect<T, SMEM>(R, list, &sc.sel[3], [&](float f, int) { return f == R.top; }, nothing);
            if (m > kList) return 0xffffffffu;
            sort_list(list, m, sc);
            return index_of(list[0]);
        }
        if (p < 1.f) {
            // masses of the bins, from their counts and middles; those that top-k cut off are left out
            const float step = kDepth / kBins;
            const uint32_t k0 = min(c0, room > before ? room - before : 0u), k1 = min(c1, room > before + c0 ? room - before - c0 : 0u);
            const float m0 = k0 * expf(-(2 * tid + 0.5f) * step), m1 = k1 * expf(-(2 * tid + 1.5f) * step);
            const unsigned long long w0 = __float2ull_rn(m0 * 1073741824.f), w1 = __float2ull_rn(m1 * 1073741824.f);  // of 2^-30
            unsigned long long mass;
            const unsigned long long mb = scan_u64(w0 + w1, sc.red, mass);
            // The bins in which the cut may lie.  A logit's weight is off by up to half a bin's width (step / 2), as
            // good as independently: four standard deviations, and 0.01 % of the mass.
            unsigned long long squares;
            scan_u64(__float2ull_rn((m0 * expf(-(2 * tid + 0.5f) * step) + m1 * expf(-(2 * tid + 1.5f) * step)) * 1073741824.f), sc.red,
                     squares);
            const double goal = static_cast<double>(p) * static_cast<double>(mass);
            const double slack = 1e-4 * static_cast<double>(mass) +
                                 4.0 * 0.289 * step * 32768.0 * sqrt(static_cast<double>(squares));  // (both are counted in 2^-30)
            if (tid == 0) sc.sel[0] = sc.sel[1] = kBins - 1;
            __syncthreads();
#pragma unroll
            for (int q = 0; q < 2; q++) {
                const double edge = q ? goal + slack : goal - slack;
                if (static_cast<double>(mb + w0 + w1) >= edge)
                    atomicMin(&sc.sel[q], static_cast<uint32_t>(2 * tid + (static_cast<double>(mb + w0) < edge)));
            }
            __syncthreads();
            const int ba = static_cast<int>(sc.sel[0]), bb = static_cast<int>(sc.sel[1]);
            __syncthreads();
            // exact: the weights above those bins, by cells, and of everything; the list of the bins between
            const float cut_x = cut ? logit_at(cut) : -INFINITY;
            const int cut_i = cut ? static_cast<int>(index_of(cut)) : INT_MIN;
            unsigned long long over = 0, sum = 0, over_all, sum_all;
            const int m = collect<T, SMEM>(
                R, list, &sc.sel[3],
                [&](float f, int i) {
                    if (!(f > cut_x || (f == cut_x && i <= cut_i))) return false;
                    const unsigned long long w = weight_of(f, ws);
                    const int b = R.bin(f);
                    sum += w;
                    if (b < ba) over += w;
                    return b >= ba && b <= bb;
                },
                [&](int s) {
                    const unsigned long long w = warp_total(over);
                    if (lane == 0) R.cells[s * kWarps + warp] = w;
                    over_all = s ? over_all + w : w;
                    over = 0;
                });
            unsigned long long t1;
            scan_u64(lane == 0 ? over_all : 0, sc.red, t1);
            over_all = t1;
            scan_u64(sum, sc.red, sum_all);
            const double want = static_cast<double>(p) * static_cast<double>(sum_all);
            if (m > kList || !(static_cast<double>(over_all) < want || ba == 0)) return 0xffffffffu;
            sort_list(list, m, sc);
            const int t = prefix_reaching(R, ws, list, m, over_all, want, sc);
            if (t > m) return 0xffffffffu;
            cut = list[t - 1];
            // the kept ones of the list join the cells, unless min-p takes some away again
            summed = least == 0.0 || static_cast<double>(weight_of(logit_at(cut), ws)) >= least;
            if (summed)
                for (int i = tid; i < t; i += kThreads) {
                    const int j = static_cast<int>(index_of(list[i])) + R.pad;
                    atomicAdd(&R.cells[j / kSeg * kWarps + j % kSeg / 128], weight_of(logit_at(list[i]), ws));
                }
        }
    }
    if (!summed) {
#pragma unroll 1
        for (int s = 0; s < R.segs; s++) {
            unsigned long long w[4];
            const unsigned long long m = warp_total(kept_weights<T, SMEM>(R, ws, cut, least, s, w));
            if (lane == 0) R.cells[s * kWarps + warp] = m;
        }
    }
    __syncthreads();
    return draw_from_cells<T, SMEM>(R, ws, cut, least, r, sc);
}

// Block = one row.
template <typename T, bool SMEM>
__global__ void __launch_bounds__(kThreads) k_sample_rows(SampleRowsArgs a) {
    extern __shared__ __align__(16) unsigned long long smem_rows[];
    __shared__ Scratch sc;
    __shared__ double pow2[32];
    unsigned long long* list = smem_rows;                                  // kList
    uint32_t* hist = reinterpret_cast<uint32_t*>(list + kList);            // kBins
    unsigned long long* cells = reinterpret_cast<unsigned long long*>(hist + kBins);
    float* v = reinterpret_cast<float*>(cells + a.segs * kWarps);          // SMEM: the row
    const bool again = blockIdx.x >= static_cast<unsigned>(a.rows);  // the second half of a grid of twice the rows
    const int row = blockIdx.x - (again ? a.rows : 0), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T* x = static_cast<const T*>(a.logits) + static_cast<size_t>(row) * a.row_stride;
    const int n = a.n;
    const float temp = a.temperature[row];
    const int k = a.top_k ? a.top_k[row] : 0;
    if (gridDim.x > static_cast<unsigned>(a.rows) && (!(temp > 0.f) || (k > 0 && k < n && k <= kSmallK)) != again) return;
    if (!(temp > 0.f)) {
        const uint32_t best = first_max<T>(x, n, sc);
        if (tid == 0) a.out[row] = best;
        return;
    }
    if (tid < 32) pow2[tid] = kPow2[tid];

    // each thread's largest logit (NaN if there is one); the row into shared memory, 16 bytes of it at a time
    float own = -INFINITY;
    int pad = 0;
    constexpr int VE = 16 / sizeof(T);
    if (SMEM) {
        const int head = min(n, static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)));
        pad = (4 - (head & 3)) & 3;  // the first whole 16 bytes begin at a multiple of 4 positions
        const int nv = (n - head) / VE, tail = head + nv * VE;
        for (int j = tid; j < pad + head; j += kThreads) {
            const float f = j < pad ? -INFINITY : to_f32<T>(x[j - pad]);
            own = max_nan(own, f);
            v[j] = f;
        }
#pragma unroll 4
        for (int q = tid; q < nv; q += kThreads) {
            const uint4 raw = *reinterpret_cast<const uint4*>(x + head + q * VE);
            const T* e = reinterpret_cast<const T*>(&raw);
            float f[VE];
#pragma unroll
            for (int c = 0; c < VE; c++) {
                f[c] = to_f32<T>(e[c]);
                own = max_nan(own, f[c]);
            }
#pragma unroll
            for (int c = 0; c < VE; c += 4)
                *reinterpret_cast<float4*>(v + pad + head + q * VE + c) = make_float4(f[c], f[c + 1], f[c + 2], f[c + 3]);
        }
        for (int j = pad + tail + tid; j < a.segs * kSeg; j += kThreads) {
            const float f = j - pad < n ? to_f32<T>(x[j - pad]) : -INFINITY;
            own = max_nan(own, f);
            v[j] = f;
        }
    } else {
#pragma unroll 4
        for (int i = tid; i < n; i += kThreads) own = max_nan(own, to_f32<T>(x[i]));
    }
    // the largest and the smallest of the threads' keys (of those that saw more than -inf)
    const uint32_t best = key_of(own);
    uint32_t bk = __reduce_max_sync(FULL, best), lk = __reduce_min_sync(FULL, own == -INFINITY ? 0xffffffffu : best);
    if (lane == 0) {
        sc.sk[warp] = bk;
        sc.si[warp] = lk;
    }
    __syncthreads();
    bk = __reduce_max_sync(FULL, sc.sk[lane]);
    lk = __reduce_min_sync(FULL, sc.si[lane]);
    uint32_t answer = static_cast<uint32_t>(n - 1);
    if (bk < 0xff800000u && bk > key_of(-INFINITY)) {  // neither NaN nor +inf, and something above -inf
        const float top = logit_of(bk);
        float p = a.top_p ? a.top_p[row] : 1.f, mp = a.min_p ? a.min_p[row] : 0.f;
        const float r = a.r[row];
        if (mp > 1.f) p = mp = 0.f;  // no weight reaches it: the first of the order, as for a top-p of 0
        const Scale ws{widen(top), 46.16624130844683 / static_cast<double>(temp), pow2};  // 32 / ln 2
        const Row R{v, x, n, pad, a.segs, top, kBins / (kDepth * temp), cells};
        answer = 0xffffffffu;
        if (a.segs <= kMaxSegs) answer = sample_row<T, SMEM>(R, ws, best, bk, lk, k, p, mp, r, list, hist, sc);
        if (answer == 0xffffffffu) {
            __syncthreads();
            answer = sample_by_radix<T>(x, n, k, p, mp, r, ws, bk, sc);
        }
    }
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
    // up to 3 positions before the first logit align it; a segment more than shared memory holds: read from L2
    const int segs = static_cast<int>((n + 3 + kSeg - 1) / kSeg);
    const size_t base = kList * 8 + kBins * 4 + static_cast<size_t>(std::min(segs, kMaxSegs)) * kWarps * 8;
    constexpr size_t most = 227 * 1024 - sizeof(Scratch) - 32 * 8 - 1024;
    const bool fits = base + static_cast<size_t>(segs) * kSeg * 4 <= most;
    SampleRowsArgs a{out, logits, row_stride, static_cast<int>(n), r, temperature, top_p, min_p, top_k, segs, static_cast<int>(n_rows)};
    const int smem = static_cast<int>(fits ? base + static_cast<size_t>(segs) * kSeg * 4 : base);
    // More rows than run at once: a block for each row that takes long, then one for each that does not (greedy or a short
    // list); the others of a grid of twice the rows leave at once.  256 rows of 32000, mixed: 54 us, in the rows' order 70;
    // 1000 rows 232 and 253 us; rows that are all alike 31.1 and 29.5 us (short lists), 74 and 74 us (top-p).
    const size_t at_once = static_cast<size_t>(sm_count()) * (2 * (smem + sizeof(Scratch) + 2048) <= 227 * 1024 ? 2 : 1);
    const unsigned grid = static_cast<unsigned>(n_rows > at_once && n_rows <= 0x3fffffff ? 2 * n_rows : n_rows);
    const cudaStream_t s = as_stream(stream);
    auto run = [&](auto kernel) -> tl_status {
        // (the limit is the kernel's, not the launch's: another thread may be about to launch a longer row)
        TL_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most)));
        kernel<<<grid, kThreads, smem, s>>>(a);
        return TL_OK;
    };
    if (dtype == TL_F32) TL_TRY(fits ? run(k_sample_rows<float, true>) : run(k_sample_rows<float, false>));
    else if (dtype == TL_F16) TL_TRY(fits ? run(k_sample_rows<__half, true>) : run(k_sample_rows<__half, false>));
    else TL_TRY(fits ? run(k_sample_rows<__nv_bfloat16, true>) : run(k_sample_rows<__nv_bfloat16, false>));
    return check_launch("sample_rows");
}
