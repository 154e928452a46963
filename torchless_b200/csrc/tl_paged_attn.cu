// tl_paged_attn.cu -- tl_paged_attention: entry points, and the kernel for few
// query rows per sequence (decode steps).
//
// Every key is read once for all query rows that share its kv head, and with so
// few rows the reading is what takes the time: 2 * size * hd bytes a key and kv
// head against at most 16 rows of arithmetic.  So the kernel is built to keep
// HBM busy whatever the lengths are:
//   - The work of the whole call, counted in steps of 16 keys (8 for fp32), is
//     cut into one equal share per SM, across sequences, kv heads and the middle
//     of a sequence.  Each block finds its share by a scan over the lengths on
//     the device: no length is known to the host, and a batch of unlike lengths
//     is as balanced as one of equal ones.
//   - In a block, 8 warps take the steps of a tile in turn.  Each has its own
//     ring of stages that lane 0 fills by TMA (a page's rows, both panels, one
//     instruction for K and one for V), running ahead into the next tiles; no
//     barrier is shared in the loop.
//   - fp16 / bf16: scores and values on mma.sync m16n8k16 (16 rows fill the
//     instruction's height; tcgen05's 128 would be nearly empty, and its rate is
//     not what bounds).  The weights enter as a sum of two 16-bit numbers, so
//     that only the result's own rounding remains.  fp32: FMA.
//   - At a tile's end the warps join (max, sum, accumulator) in shared memory;
//     a tile that continues in another block leaves its part in the workspace,
//     and a second small kernel joins the parts in order.
// 32 heads, 8 kv heads, hd 128, one token a sequence: 64 x 4096 keys bf16 177 us (6.1 TB/s of 6.55 that a copy reaches),
// hd 64 94 us, fp32 333 us (6.45 TB/s; 24 us more where 512 MB were written before it, whose last part leaves L2
// meanwhile), 64 ragged lengths of at most 4096 fp16 69 us (5.4 TB/s); 1 x 8192 bf16 15.1 us, where finding the shares
// (2.7 us), the first copies, the join and the launches count more than the 5.1 us of reading.  A tile costs about 3 us
// beside its keys: 200 x 300 keys 73 us (3.4 TB/s).
#include <math.h>

#include <algorithm>
#include <cstdlib>
#include <type_traits>

#include "tl_paged_attn.cuh"

namespace tl {
namespace paged {

using namespace tc;

tl_status encode_pages(CUtensorMap* map, const void* base, const tl_paged_cache* c, int rows, int box_panels) {
    auto fn = encode_fn();
    if (!fn) return set_error(TL_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const bool wide = c->dtype == TL_F32;
    const size_t es = dtype_size(c->dtype);
    const cuuint32_t cols = wide ? static_cast<cuuint32_t>(c->head_dim) : 64u;
    const cuuint32_t panels = static_cast<cuuint32_t>(c->head_dim) / cols;
    const cuuint64_t dims[4] = {cols, c->n_kv_heads * c->block_size, panels, c->n_blocks};
    const cuuint64_t strides[3] = {c->head_dim * es, cols * es, c->block_stride * es};
    const cuuint32_t box[4] = {cols, static_cast<cuuint32_t>(rows), static_cast<cuuint32_t>(box_panels), 1};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    const CUresult r = fn(map,
                          wide ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                               : c->dtype == TL_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                          4, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          wide ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(TL_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
    return TL_OK;
}

namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32;

__device__ __forceinline__ void tma_page(void* dst, const CUtensorMap* map, int row, int page, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %2, %4}], [%5];" ::
            "r"(su32(dst)), "l"(map), "r"(0), "r"(row), "r"(page), "r"(su32(bar))
        : "memory");
}

// Waits by polling (the copies are short, and a suspended wait may wake late); false after ~2 s.
__device__ __noinline__ bool spin_slow(uint64_t* b, uint32_t parity, unsigned fail_one_in) {
    if (fail_one_in != 0 && told_to_fail(fail_one_in)) return false;
    const unsigned long long t0 = gtime();
    for (unsigned i = 1;; i++) {
        if (bar_test_now(b, parity)) return true;
        if ((i & 255) == 0 && gtime() - t0 > kTimeoutNs) return false;
    }
}
__device__ __forceinline__ bool spin(uint64_t* b, uint32_t parity, unsigned fail_one_in) {
    return (bar_test_now(b, parity) && fail_one_in == 0) || spin_slow(b, parity, fail_one_in);
}

// Waits for the copies of `n` stages from st on.
template <int NST>
__device__ __noinline__ void drain(uint64_t* bars, int st, uint32_t parity, int n) {
    for (; n > 0; n--) {
        bar_wait(&bars[st], (parity >> st) & 1);
        st = st + 1 == NST ? 0 : st + 1;
    }
}

// Keys per step, stages per warp, and the bytes of one side of a stage.
template <typename T, int HD>
struct Shape {
    static constexpr int KS = std::is_same<T, float>::value ? 8 : HD == 64 ? 32 : 16;
    static constexpr int SIDE = KS * HD * static_cast<int>(sizeof(T));
    static constexpr int NST = SIDE >= 4096 ? 3 : 5;
    static constexpr int JOIN = 8 * (HD + 4);  // floats of one warp's 8 rows: {max, sum, flag, -, values}
    static constexpr size_t SMEM = 1024 + static_cast<size_t>(kWarps) * NST * 2 * SIDE + kWarps * JOIN * 4 + 512;
};

// Steps of KS keys, tiles of R rows.  Beginning and ending a tile takes about as long as kTileCost steps, which count
// as steps before its first key, so that a batch of short sequences is shared as evenly as one of long ones.  64 ragged
// lengths of at most 4096, 12 / 16 / 24 / 32 steps: fp16 (steps of 16 keys) 78 / 73 / 68 / 69 us, bf16 hd 64 (32 keys)
// 54.1 / 51.1 / 49.5 / 52.2, fp32 (8 keys) 125.8 / 122.5 / 120.6 / 122; where all are alike (200 x 300) it makes no
// difference.  A tile without keys counts one step more, so that its zeros get written.
template <int R_, int KS>
struct SplitPlan {
    static constexpr int R = R_;
    static constexpr int kTileCost = 24;
    static constexpr bool kLookAgain = KS != 16;  // fp32, and head_dim 64
    static __device__ __forceinline__ int steps(const Tile& t) {
        return kTileCost + (t.hi <= t.lo ? 1 : (t.hi - 1) / KS - t.lo / KS + 1);
    }
};

// ---- arithmetic of one warp -------------------------------------------------

// One step: keys [key0, key0 + KS); bit k of valid: the page of its keys 8 k .. exists.
struct StepInfo {
    int key0;
    uint32_t valid;
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two floats as 16-bit halves of a word, and what the rounding left of them.
__device__ __forceinline__ uint32_t split2(float x, float y, uint32_t& lo, __half*) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 r = __floats2half2_rn(x - f.x, y - f.y);
    lo = *reinterpret_cast<const uint32_t*>(&r);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t split2(float x, float y, uint32_t& lo, __nv_bfloat16*) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    const float2 f = __bfloat1622float2(h);
    const __nv_bfloat162 r = __floats2bfloat162_rn(x - f.x, y - f.y);
    lo = *reinterpret_cast<const uint32_t*>(&r);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// 16 rows on the matrix instruction: lane l holds rows l / 4 and l / 4 + 8.
template <typename T, int HD, int R>
struct Core {
    static_assert(R == 16, "the instruction's height");
    static constexpr int NO = HD / 8;
    // fp16 ends at 2^-24, and many weights below that may add up to a result: they are formed, and summed, 2^15 times as
    // large, which the largest of 1 has room for.  (Where scores beyond 2^24 round that to 2^16, an infinity, the rows are
    // done over.)  bf16 has fp32's range.
    static constexpr float kLift = std::is_same<T, __half>::value ? 15.f : 0.f;
    uint32_t q[HD / 16][4];
    float o[NO][4];
    float m[2], l[2];
    int lo[2], hi[2];  // this lane's rows' attended positions
    int hs, ps;        // bytes between the 8-key halves and between the panels of a side

    __device__ void begin(const AttendArgs& a, const Cursor& c, int lane) {
        const T* qb = static_cast<const T*>(a.q);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int r = lane / 4 + 8 * i;
            const bool in = r < c.t.nrows;
            int tok, h;
            row_of(a, c, r, tok, h);
            attended(a, c.t.p0 + (tok - c.t.first), lo[i], hi[i]);
            if (!in) hi[i] = 0;
            const uint32_t* src = reinterpret_cast<const uint32_t*>(
                qb + static_cast<size_t>(tok) * a.q_stride + static_cast<size_t>(h) * HD) + (lane & 3);
#pragma unroll
            for (int k = 0; k < HD / 16; k++) {
                q[k][i] = in ? src[8 * k] : 0u;
                q[k][2 + i] = in ? src[8 * k + 4] : 0u;
            }
            m[i] = -INFINITY;
            l[i] = 0.f;
        }
#pragma unroll
        for (int n = 0; n < NO; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
        hs = 1024;
        ps = 2048;
        if (a.shift == 3) {
            hs = 1024 * (HD / 64);
            ps = 1024;
        }
    }

    __device__ __forceinline__ uint32_t at(int key, int chunk) const {  // byte offset of 8 dims of a key
        return static_cast<uint32_t>((key >> 3) * hs + (chunk >> 3) * ps + (key & 7) * 128 +
                                     (((chunk & 7) ^ (key & 7)) << 4));
    }

    __device__ void step(const AttendArgs& a, const Cursor& c, StepInfo si, const uint8_t* sk, const uint8_t* sv,
                         int lane) {
        constexpr int KS = Shape<T, HD>::KS, G = KS / 16, NT = KS / 8;
        const uint32_t kb = su32(sk), vb = su32(sv);
        uint32_t kr[G][HD / 16][4], vr[G][HD / 16][4];
        const int kk = (lane >> 4) * 8 + (lane & 7), kc0 = (lane >> 3) & 1;
#pragma unroll
        for (int g = 0; g < G; g++)
#pragma unroll
            for (int k = 0; k < HD / 16; k++) ldsm4(kr[g][k], kb + at(16 * g + kk, 2 * k + kc0));
        // the scores in two chains of sums, and the values on their way while they are worked on
        float s[NT][4], s2[NT][4];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) s[n][e] = s2[n][e] = 0.f;
#pragma unroll
        for (int k = 0; k < HD / 16; k += 2)
#pragma unroll
            for (int g = 0; g < G; g++) {
                mma16<T>(s[2 * g], q[k], kr[g][k][0], kr[g][k][1]);
                mma16<T>(s[2 * g + 1], q[k], kr[g][k][2], kr[g][k][3]);
                mma16<T>(s2[2 * g], q[k + 1], kr[g][k + 1][0], kr[g][k + 1][1]);
                mma16<T>(s2[2 * g + 1], q[k + 1], kr[g][k + 1][2], kr[g][k + 1][3]);
            }
        const int vkey = ((lane >> 3) & 1) * 8 + (lane & 7), vc = lane >> 4;
#pragma unroll
        for (int g = 0; g < G; g++)
#pragma unroll
            for (int j = 0; j < HD / 16; j++) ldsm4t(vr[g][j], vb + at(16 * g + vkey, 2 * j + vc));
        const float sl = a.scale * 1.4426950408889634f;  // log2 units
        // every row attends to every key of an inner step
        const bool edge = si.valid != (1u << NT) - 1 || si.key0 < c.t.lo_last || si.key0 > c.t.hi_first - KS;
        const int kc = si.key0 + 2 * (lane & 3);
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) s[n][e] = (s[n][e] + s2[n][e]) * sl;
        if (edge) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int key = kc + 8 * n + (e & 1), i = e >> 1;
                    if (!(key >= lo[i] && key < hi[i] && ((si.valid >> n) & 1))) s[n][e] = -INFINITY;
                }
            // keys that no row attends to must not reach the products (0 x NaN)
#pragma unroll
            for (int n = 0; n < NT; n++) {
                uint32_t keep = ~0u;
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int key = kc + 8 * n + e;
                    if (!(key >= c.t.lo && key < c.t.hi && ((si.valid >> n) & 1))) keep &= e ? 0xffffu : 0xffff0000u;
                }
#pragma unroll
                for (int j = 0; j < HD / 16; j++) {
                    vr[n / 2][j][n & 1] &= keep;
                    vr[n / 2][j][2 + (n & 1)] &= keep;
                }
            }
        }
        float f[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            float mx = fmaxf(s[0][2 * i], s[0][2 * i + 1]);
#pragma unroll
            for (int n = 1; n < NT; n++) mx = fmaxf(mx, fmaxf(s[n][2 * i], s[n][2 * i + 1]));
            mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, 2));
            const float mn = fmaxf(m[i], mx);
            float base = mn == -INFINITY ? 0.f : mn;
            f[i] = ex2(m[i] - base);
            m[i] = mn;
            if (kLift != 0.f) base -= kLift;
            float sum = 0.f;
#pragma unroll
            for (int n = 0; n < NT; n++) {
#pragma unroll
                for (int e = 0; e < 2; e++) s[n][2 * i + e] = ex2(s[n][2 * i + e] - base);
                sum += s[n][2 * i] + s[n][2 * i + 1];
            }
            l[i] = l[i] * f[i] + sum;
        }
        if (__any_sync(FULL, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
            for (int n = 0; n < NO; n++) {
                o[n][0] *= f[0];
                o[n][1] *= f[0];
                o[n][2] *= f[1];
                o[n][3] *= f[1];
            }
        }
#pragma unroll
        for (int g = 0; g < G; g++) {
            uint32_t ph[4], pl[4];
#pragma unroll
            for (int e = 0; e < 4; e++)
                ph[e] = split2(s[2 * g + e / 2][2 * (e & 1)], s[2 * g + e / 2][2 * (e & 1) + 1], pl[e], static_cast<T*>(nullptr));
#pragma unroll
            for (int j = 0; j < HD / 16; j++) {
                mma16<T>(o[2 * j], ph, vr[g][j][0], vr[g][j][1]);
                mma16<T>(o[2 * j + 1], ph, vr[g][j][2], vr[g][j][3]);
            }
#pragma unroll
            for (int j = 0; j < HD / 16; j++) {
                mma16<T>(o[2 * j], pl, vr[g][j][0], vr[g][j][1]);
                mma16<T>(o[2 * j + 1], pl, vr[g][j][2], vr[g][j][3]);
            }
        }
    }

    // Sums over the lanes; whether a result of this lane is not finite.
    __device__ bool finish(int nrows, int lane) {
        float z = 0.f;  // NaN once a value is not finite
#pragma unroll
        for (int i = 0; i < 2; i++) {
            l[i] += __shfl_xor_sync(FULL, l[i], 1);
            l[i] += __shfl_xor_sync(FULL, l[i], 2);
            if (lane / 4 + 8 * i < nrows) {
                z = fmaf(l[i], 0.f, z);
#pragma unroll
                for (int n = 0; n < NO; n++) z = fmaf(o[n][2 * i], 0.f, fmaf(o[n][2 * i + 1], 0.f, z));
            }
        }
        return z != z;
    }
    // rows 8 * pass .. of this warp into its part of the join buffer
    __device__ void dump(float* j, int pass, int lane) const {
        float* row = j + (lane >> 2) * (HD + 4);
        if ((lane & 3) == 0) {
            row[0] = pass ? m[1] : m[0];
            row[1] = pass ? l[1] : l[0];
        }
#pragma unroll
        for (int n = 0; n < NO; n++)
            *reinterpret_cast<float2*>(row + 4 + 8 * n + 2 * (lane & 3)) =
                pass ? make_float2(o[n][2], o[n][3]) : make_float2(o[n][0], o[n][1]);
    }
};

// fp32: lane l holds dims l * HD / 32 ... of R rows; the R x 8 partial dot
// products of a step are reduced together (transposed reduction), after which
// lane l has the score of row 4 * rg + l / 8 and key l % 8.
template <int HD, int R>
struct Core<float, HD, R> {
    static constexpr int D = HD / 32, RG = R / 4;
    float q[R][D], o[R][D], m[R];
    float l[RG];
    int lo[RG], hi[RG];

    __device__ __forceinline__ static void load(float (&v)[D], const float* p) {
        if constexpr (D == 4) {
            const float4 f = *reinterpret_cast<const float4*>(p);
            v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
        } else {
            const float2 f = *reinterpret_cast<const float2*>(p);
            v[0] = f.x; v[1] = f.y;
        }
    }

    __device__ void begin(const AttendArgs& a, const Cursor& c, int lane) {
        const float* qb = static_cast<const float*>(a.q);
#pragma unroll
        for (int r = 0; r < R; r++) {
            const bool in = r < c.t.nrows;
            int tok, h;
            row_of(a, c, r, tok, h);
            load(q[r], qb + static_cast<size_t>(tok) * a.q_stride + static_cast<size_t>(h) * HD + lane * D);
#pragma unroll
            for (int d = 0; d < D; d++) {
                if (!in) q[r][d] = 0.f;
                o[r][d] = 0.f;
            }
            m[r] = -INFINITY;
        }
#pragma unroll
        for (int g = 0; g < RG; g++) {
            const int r = 4 * g + lane / 8;
            attended(a, c.t.p0 + div_group(a, c.t.r0 + r), lo[g], hi[g]);
            if (r >= c.t.nrows) hi[g] = 0;
            l[g] = 0.f;
        }
    }

    __device__ void step(const AttendArgs& a, const Cursor& c, StepInfo si, const uint8_t* sk, const uint8_t* sv,
                         int lane) {
        const float* K = reinterpret_cast<const float*>(sk) + lane * D;
        const float* V = reinterpret_cast<const float*>(sv) + lane * D;
        const float sl = a.scale * 1.4426950408889634f;
        const int key = si.key0 + (lane & 7);
        float p[RG];
        float k[8][D];
#pragma unroll
        for (int f = 0; f < 8; f++) load(k[f], K + f * HD);
#pragma unroll
        for (int g = 0; g < RG; g++) {
            float v[32];
#pragma unroll
            for (int h = 0; h < 4; h++)
#pragma unroll
                for (int f = 0; f < 8; f++) {
                    float t = q[4 * g + h][0] * k[f][0];
#pragma unroll
                    for (int d = 1; d < D; d++) t = fmaf(q[4 * g + h][d], k[f][d], t);
                    v[8 * h + f] = t;
                }
            warp_reduce_multi<32>(v);
            const bool in = key >= lo[g] && key < hi[g] && (si.valid & 1);
            const float s = in ? v[0] * sl : -INFINITY;
            float mx = s;
            mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, 2));
            mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, 4));
            float mine = 0.f, fm = 1.f;  // base and factor of this lane's row
#pragma unroll
            for (int h = 0; h < 4; h++) {
                const int r = 4 * g + h;
                const float mn = fmaxf(m[r], __shfl_sync(FULL, mx, 8 * h));
                const float base = mn == -INFINITY ? 0.f : mn;
                const float f = ex2(m[r] - base);
                m[r] = mn;
#pragma unroll
                for (int d = 0; d < D; d++) o[r][d] *= f;
                if ((lane >> 3) == h) {
                    mine = base;
                    fm = f;
                }
            }
            p[g] = ex2(s - mine);
            l[g] = l[g] * fm + p[g];
        }
#pragma unroll
        for (int f = 0; f < 8; f++) {
            float v[D];
            load(v, V + f * HD);
            const int kf = si.key0 + f;
            if (!(kf >= c.t.lo && kf < c.t.hi && (si.valid & 1))) {  // keys that no row attends to: no 0 x NaN
#pragma unroll
                for (int d = 0; d < D; d++) v[d] = 0.f;
            }
#pragma unroll
            for (int g = 0; g < RG; g++)
#pragma unroll
                for (int h = 0; h < 4; h++) {
                    const float w = __shfl_sync(FULL, p[g], 8 * h + f);
#pragma unroll
                    for (int d = 0; d < D; d++) o[4 * g + h][d] = fmaf(w, v[d], o[4 * g + h][d]);
                }
        }
    }

    __device__ bool finish(int nrows, int lane) {
        float z = 0.f;
#pragma unroll
        for (int g = 0; g < RG; g++) {
#pragma unroll
            for (int x = 1; x < 8; x <<= 1) l[g] += __shfl_xor_sync(FULL, l[g], x);
            if (4 * g + lane / 8 < nrows) z = fmaf(l[g], 0.f, z);
        }
#pragma unroll
        for (int r = 0; r < R; r++)
            if (r < nrows) {
#pragma unroll
                for (int d = 0; d < D; d++) z = fmaf(o[r][d], 0.f, z);
            }
        return z != z;
    }
    __device__ void dump(float* j, int pass, int lane) const {
#pragma unroll
        for (int r = 0; r < R; r++) {
            if (r / 8 != pass) continue;
            float* row = j + (r & 7) * (HD + 4);
            const float lr = __shfl_sync(FULL, l[r / 4], 8 * (r & 3));
            if (lane == 0) {
                row[0] = m[r];
                row[1] = lr;
            }
#pragma unroll
            for (int d = 0; d < D; d++) row[4 + lane * D + d] = o[r][d];
        }
    }
};

template <typename T, int HD, int R>
__global__ void __launch_bounds__(kThreads, 1)
    k_attend_split(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                   const __grid_constant__ AttendArgs a,
                   Head* heads, float* parts) {
    using S = Shape<T, HD>;
    constexpr int KS = S::KS, NST = S::NST;
    extern __shared__ uint8_t raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint8_t* ring = base + static_cast<size_t>(warp) * NST * 2 * S::SIDE;
    float* join = reinterpret_cast<float*>(base + static_cast<size_t>(kWarps) * NST * 2 * S::SIDE);
    uint64_t* bars = reinterpret_cast<uint64_t*>(join + kWarps * S::JOIN) + warp * NST;
    long long* ws = reinterpret_cast<long long*>(join + kWarps * S::JOIN) + kWarps * NST;  // [kWarps + 2]

    if (lane == 0) {
        for (int i = 0; i < NST; i++) bar_init(&bars[i], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x == 0) heads[blockIdx.x].parts = 0;

    using P = SplitPlan<R, KS>;
    Cursor c;
    // at least one step a warp beside the tile's cost, so that a small call is not cut into crumbs
    const int per = find_share<P, kWarps>(a, c, ws, kWarps + P::kTileCost);
    if (per == 0) return;

    // producer: a second cursor that runs up to NST steps ahead; ids of this warp's next 32 steps in the lanes
    Cursor pc = c;
    auto first_step = [&](const Cursor& x) { return max(0, x.s - P::kTileCost) + warp; };
    constexpr int NT = KS / 8;          // most pages of a step
    const int rows = min(KS, 1 << a.shift);  // rows of a copy
    int ps = first_step(pc), pid_at = 32, pid[NT];
    bool more = true;
    int put_st = 0, got_st = 0, ahead = 0;
    uint32_t got_parity = 0;
    uint32_t valid_bits = 0;  // NT bits for each stage
    int stage_key[NST];
#pragma unroll
    for (int i = 0; i < NST; i++) stage_key[i] = 0;
    __syncwarp();

    Core<T, HD, R> core;
    bool first_tile = true, dead = false;
#pragma unroll 1
    for (bool go = true; go; go = next_tile<P>(a, c), first_tile = false) {
        bool begun = false;
#pragma unroll 1
        for (int s = first_step(c);; s += kWarps) {
#pragma unroll 1
            while (more && !dead && ahead < NST) {  // one step into the ring
                if (ps >= pc.end - P::kTileCost) {
                    more = next_tile<P>(a, pc);
                    ps = first_step(pc);
                    pid_at = 32;
                    continue;
                }
                if (pid_at == 32) {
                    const int blk = (pc.t.lo / KS + ps) + kWarps * lane;  // below 2^31 / KS + 256
                    const int key = blk < kMaxLen / KS ? blk * KS : -1;
#pragma unroll
                    for (int k = 0; k < NT; k++)
                        pid[k] = k == 0 || 8 * k % rows == 0 ? page_of(a, pc.b, key < 0 ? -1 : key + 8 * k) : pid[k - 1];
                    pid_at = 0;
                }
                const int key0 = (pc.t.lo / KS + ps) * KS;
                int id[NT];
                uint32_t v = 0;
#pragma unroll
                for (int k = 0; k < NT; k++) {
                    id[k] = __shfl_sync(FULL, pid[k], pid_at);
                    v |= (id[k] >= 0 ? 1u : 0u) << k;
                }
                pid_at++;
                valid_bits = (valid_bits & ~(((1u << NT) - 1) << (NT * put_st))) | (v << (NT * put_st));
#pragma unroll
                for (int i = 0; i < NST; i++)
                    if (i == put_st) stage_key[i] = key0;
                if (lane == 0) {
                    uint8_t* k = ring + put_st * 2 * S::SIDE;
                    bar_expect_tx(&bars[put_st], 2 * S::SIDE);
#pragma unroll
                    for (int x = 0; x < NT; x++)
                        if (8 * x % rows == 0) {
                            const int row = (pc.g << a.shift) + ((key0 + 8 * x) & ((1 << a.shift) - 1));
                            tma_page(k + x * (S::SIDE / NT), &map_k, row, id[x], &bars[put_st]);
                            tma_page(k + S::SIDE + x * (S::SIDE / NT), &map_v, row, id[x], &bars[put_st]);
                        }
                }
                put_st = put_st + 1 == NST ? 0 : put_st + 1;
                ahead++;
                ps += kWarps;
            }
            if (!begun) {
                core.begin(a, c, lane);
                begun = true;
            }
            if (s >= c.end - P::kTileCost) break;
            if (ahead == 0) continue;  // (a copy never came: no further ones)
            // (the outcome is the whole warp's: what follows exchanges values between its lanes)
            if (!__all_sync(FULL, spin(&bars[got_st], (got_parity >> got_st) & 1, a.fail_one_in))) {
                dead = true;  // and the copies on their way land before the block ends
                drain<NST>(bars, got_st, got_parity, ahead);
                ahead = 0;
                continue;
            }
            got_parity ^= 1u << got_st;
            StepInfo si;
            si.valid = (valid_bits >> (NT * got_st)) & ((1u << NT) - 1);
            si.key0 = 0;
#pragma unroll
            for (int i = 0; i < NST; i++)
                if (i == got_st) si.key0 = stage_key[i];
            const uint8_t* k = ring + got_st * 2 * S::SIDE;
            core.step(a, c, si, k, k + S::SIDE, lane);
            got_st = got_st + 1 == NST ? 0 : got_st + 1;
            ahead--;
            __syncwarp();  // every lane has read the stage
        }
        // A result that is not finite: a value that one row must not see may have met it as 0 x infinity, or an infinite
        // value the split weights, or values near the type's largest add up to more.  Such a tile is done over row by
        // row, which gives the formula's result to each.  The same where a score passed fp32's range or a copy never
        // came, and for a row whose weights are all 0: it attends to nothing, or all its scores lie below that range.
        const bool redo = core.finish(c.t.nrows, lane) || dead;
        const bool whole = c.s == 0 && c.end == c.steps;
        float* part = parts + (static_cast<size_t>(blockIdx.x) * 2 + (first_tile ? 0 : 1)) * R * (HD + 4);
        const int any_redo = __syncthreads_or(redo);
#pragma unroll 1
        for (int pass = 0; pass * 8 < c.t.nrows; pass++) {
            if (pass) __syncthreads();
            core.dump(join + warp * S::JOIN, pass, lane);
            __syncthreads();
            const int row = 8 * pass + warp;  // one warp a row
            if (row < c.t.nrows) {
                const float* j = join + warp * (HD + 4);
                float M = -INFINITY;
#pragma unroll
                for (int w = 0; w < kWarps; w++) M = fmaxf(M, j[w * S::JOIN]);
                float L = 0.f, acc[HD / 32];
#pragma unroll
                for (int d = 0; d < HD / 32; d++) acc[d] = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; w++) {
                    const float mw = j[w * S::JOIN];
                    const float f = M == -INFINITY ? 1.f : ex2(mw - M);  // (all empty: sums are 0 or NaN)
                    L += j[w * S::JOIN + 1] * f;
#pragma unroll
                    for (int d = 0; d < HD / 32; d++) acc[d] += j[w * S::JOIN + 4 + lane + 32 * d] * f;
                }
                float z = L * 0.f;  // NaN once the sum over the warps is not finite
#pragma unroll
                for (int d = 0; d < HD / 32; d++) z = fmaf(acc[d], 0.f, z);
                const bool over = any_redo || __any_sync(FULL, z != z);
                int tok, h;
                row_of(a, c, row, tok, h);
                if (whole) {
                    if (over || L == 0.f) {
                        attend_row<T, HD>(a, c.b, tok, h, lane);
                    } else {
                        T* out = static_cast<T*>(a.out) + (static_cast<size_t>(tok) * a.H + h) * HD;
#pragma unroll
                        for (int d = 0; d < HD / 32; d++) out[lane + 32 * d] = from_f32<T>(acc[d] / L);
                    }
                } else {
                    float* pr = part + row * (HD + 4);
                    if (lane == 0) {
                        pr[0] = M;
                        pr[1] = L;
                        pr[2] = over ? 1.f : 0.f;
                    }
#pragma unroll
                    for (int d = 0; d < HD / 32; d++) pr[4 + lane + 32 * d] = acc[d];
                }
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

template <typename T, int HD, int R>
tl_status run_split(const AttendArgs& a, const tl_paged_cache* c, void* workspace, cudaStream_t s) {
    using S = Shape<T, HD>;
    static_assert(S::SMEM <= 232448, "shared memory of a block");
    CUtensorMap mk, mv;
    const int rows = std::min(S::KS, 1 << a.shift);
    const int panels = std::is_same<T, float>::value ? 1 : HD / 64;
    TL_TRY(encode_pages(&mk, c->k, c, rows, panels));
    TL_TRY(encode_pages(&mv, c->v, c, rows, panels));
    TL_CUDA_TRY(cudaFuncSetAttribute(k_attend_split<T, HD, R>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     static_cast<int>(S::SMEM)));
    const int grid = std::min(sm_count(), kMaxBlocks);
    Head* heads = static_cast<Head*>(workspace);
    float* parts = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kHeadBytes);
    k_attend_split<T, HD, R><<<grid, kThreads, S::SMEM, s>>>(mk, mv, a, heads, parts);
    TL_TRY(check_launch("paged_attention"));
    return launch_join<T, HD, R>(a, heads, parts, grid, 1, s);
}

template <int HD>
tl_status run_split_hd(const AttendArgs& a, const tl_paged_cache* c, void* workspace, cudaStream_t s) {
    if (c->dtype == TL_F16) return run_split<__half, HD, 16>(a, c, workspace, s);
    if (c->dtype == TL_BF16) return run_split<__nv_bfloat16, HD, 16>(a, c, workspace, s);
    // fp32: rows are paid for one by one, so no more of them than a decode step has (64 x 4096 keys: 4 rows 339 us,
    // as 16 882 us; 8 rows 244 us, as 16 454 us)
    const long long rows = static_cast<long long>(a.n_tokens) * a.group;
    if (a.group <= 4 && rows <= 4ll * a.n_seq) return run_split<float, HD, 4>(a, c, workspace, s);
    if (a.group <= 8 && rows <= 8ll * a.n_seq) return run_split<float, HD, 8>(a, c, workspace, s);
    return run_split<float, HD, 16>(a, c, workspace, s);
}

}  // namespace

size_t split_workspace(int hd) {
    return kHeadBytes + static_cast<size_t>(std::min(sm_count(), kMaxBlocks)) * 2 * 16 * (hd + 4) * 4;
}

tl_status attend_split(const AttendArgs& a, const tl_paged_cache* c, void* workspace, cudaStream_t s) {
    return c->head_dim == 128 ? run_split_hd<128>(a, c, workspace, s) : run_split_hd<64>(a, c, workspace, s);
}

}  // namespace paged
}  // namespace tl

using namespace tl;
using namespace tl::paged;

namespace {
// TL_PAGED_FAIL_WAITS=n: about one in n waits of the kernels gives up at once, for tests of what follows.
unsigned fail_one_in() {
    static const unsigned n = [] {
        const char* e = std::getenv("TL_PAGED_FAIL_WAITS");
        return e ? static_cast<unsigned>(std::max(0, std::atoi(e))) : 0u;
    }();
    return n;
}

// Rows per sequence and kv head, on average, from which the kernels for chunks pay: this file's kernel reads all keys
// once for every 16 rows, theirs for every 256 (fp32: 64).  32 heads, 8 kv heads, hd 128, 64 x 4096 keys, bf16 / fp32:
// 16 rows 180 / 905 us here and 205 / 1630 us there, 20 rows 343 / 1763 and 212 / 1631; 16 x 1000 keys: 16 rows
// 30 / 85 and 28 / 130, 20 rows 43 / 139 and 28 / 130.
bool many_rows(const tl_paged_cache* c, size_t n_tokens, size_t n_heads, size_t n_seq) {
    return n_tokens * (n_heads / c->n_kv_heads) > 16 * n_seq;
}
}  // namespace

extern "C" {

tl_status tl_paged_attention_workspace(const tl_paged_cache* cache, size_t n_tokens, size_t n_heads, size_t n_seq,
                                       size_t max_blocks, size_t* bytes) {
    clear_error();
    TL_TRY(check_cache("tl_paged_attention_workspace", cache));
    TL_REQUIRE(bytes, "tl_paged_attention_workspace: no result");
    TL_REQUIRE(n_heads > 0 && n_heads % cache->n_kv_heads == 0, "tl_paged_attention_workspace: %zu heads, %zu kv heads",
               n_heads, cache->n_kv_heads);
    (void)max_blocks;
    const int hd = static_cast<int>(cache->head_dim);
    *bytes = !many_rows(cache, n_tokens, n_heads, n_seq) ? split_workspace(hd)
             : cache->dtype == TL_F32                    ? chunk_f32_workspace(hd)
                                                         : chunk_workspace(hd);
    return TL_OK;
}

tl_status tl_paged_attention(void* out, const void* q, size_t q_stride, const tl_paged_cache* cache,
                             const int32_t* block_table, size_t max_blocks, const int32_t* q_start,
                             const int32_t* seq_lens, size_t n_seq, size_t n_tokens, size_t n_heads, float scale,
                             size_t window, void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    TL_TRY(check_cache("tl_paged_attention", cache));
    TL_REQUIRE(n_heads > 0 && n_heads % cache->n_kv_heads == 0 && n_heads <= 65536,
               "tl_paged_attention: %zu heads, %zu kv heads", n_heads, cache->n_kv_heads);
    if (n_tokens == 0 || n_seq == 0) return TL_OK;
    TL_REQUIRE(out && q && block_table && q_start && seq_lens, "tl_paged_attention: null pointer");
    TL_REQUIRE(max_blocks > 0 && n_seq <= 0x7fffffffull && max_blocks <= 0x7fffffffull / n_seq,
               "tl_paged_attention: %zu sequences x %zu blocks", n_seq, max_blocks);
    TL_REQUIRE(n_tokens <= 0x3fffffffull / n_heads, "tl_paged_attention: %zu tokens x %zu heads", n_tokens, n_heads);
    TL_REQUIRE(q_stride >= n_heads * cache->head_dim && q_stride <= (1ull << 36), "tl_paged_attention: q_stride %zu",
               q_stride);
    TL_REQUIRE(aligned16(out) && aligned16(q) && q_stride * dtype_size(cache->dtype) % 16 == 0,
               "tl_paged_attention: out, q and q_stride must be 16-byte aligned");
    TL_REQUIRE(scale == scale && fabsf(scale) <= 2.0e38f, "tl_paged_attention: scale %g", static_cast<double>(scale));
    size_t need = 0;
    TL_TRY(tl_paged_attention_workspace(cache, n_tokens, n_heads, n_seq, max_blocks, &need));
    TL_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= need,
               "tl_paged_attention: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    AttendArgs a{};
    a.out = out;
    a.q = q;
    a.k = cache->k;
    a.v = cache->v;
    a.table = block_table;
    a.q_start = q_start;
    a.seq_lens = seq_lens;
    a.q_stride = q_stride;
    a.block_stride = cache->block_stride;
    a.n_seq = static_cast<int>(n_seq);
    a.n_tokens = static_cast<int>(n_tokens);
    a.H = static_cast<int>(n_heads);
    a.KV = static_cast<int>(cache->n_kv_heads);
    a.group = a.H / a.KV;
    a.group_inv = ~0ull / static_cast<unsigned long long>(a.group) + 1;
    a.max_blocks = static_cast<int>(max_blocks);
    a.n_blocks = static_cast<int>(cache->n_blocks);
    a.shift = __builtin_ctzll(cache->block_size);
    a.cap = static_cast<int>(std::min<size_t>(max_blocks << a.shift, kMaxLen));
    a.window = window >= 1ull << 30 ? 0 : static_cast<int>(window);
    a.scale = scale == 0.f ? 1e-45f : scale;  // (a masked score is -inf, which no factor may turn into NaN)
    a.fail_one_in = fail_one_in();
    if (!many_rows(cache, n_tokens, n_heads, n_seq)) return attend_split(a, cache, workspace, as_stream(stream));
    return cache->dtype == TL_F32 ? attend_chunk_f32(a, cache, workspace, as_stream(stream))
                                  : attend_chunk(a, cache, workspace, as_stream(stream));
}

}  // extern "C"
