// tl_paged_attn_tc.cu -- paged attention of many query rows (chunks of a
// prompt) on the 5th-generation tensor cores; fp16 and bf16 caches.
//
// With 128 rows a K / V tile of 128 keys costs 512 cycles of the matrix unit a
// product pair and 64 KB of reading; at full rate 128-row tiles would ask L2
// for 128 bytes a cycle and SM, more than it gives.  So a block works on 256
// rows of one kv head at a time, as two streams of 128 rows that share every
// K / V tile:
//   S_i[128 x 128] = Q_i K^T      tcgen05.mma, tensor memory
//   P_i            = 2^(S_i scale - m_i)   two threads a row, 16-bit, over S_i (fp16: 2^11 times as large)
//   O_i[128 x hd] += P_i V        tcgen05.mma, P_i from tensor memory
// While the threads of one stream take exponentials, the matrix unit works for
// the other.  A tile of at most 128 rows (the tail of a chunk, a single token
// beside chunks) has its rows in both streams, which then take the key tiles in
// turn and are added at the end.
//   - V comes as [keys][hd] from its pages and is the N-major operand as it
//     lies: nothing is transposed.
//   - The row maximum moves only when it grows by more than 2^8 (then O is
//     rescaled in tensor memory); exponents up to 2^8 stay in 16 bits' range and
//     the final O / l is exact all the same.  fp16 ends at 2^-24, and many weights
//     below that may add up to a result: there it moves from 2^4 on, and weights
//     and sums are 2^11 times as large.
//   - Persistent blocks with equal shares of the key tiles (tl_paged_attn.cuh);
//     a row tile that two blocks share is joined by a second kernel.
// Warps: 0-7 stream 0, 8-15 stream 1 (softmax and epilogue: a row's first 64 keys and first columns by warps 0-3
// of a stream, the rest by 4-7, which agree on the row's maximum through shared memory), 16 TMA, 17 MMA, 18 and 19
// Q of stream 0 and 1: the next tile's, as soon as the last scores of this one are done.
// Every mbarrier wait is bounded (~2 s): on expiry the roles stop, copies and MMAs in flight drain, the block's rows
// are done over by attend_row, tensor memory is freed.
//
// What bounds it: a step of 256 rows x 128 keys is 2048 cycles of the matrix unit and as many of the special function
// units (one exponential a score at 8 cycles a warp); it takes about 4100, since a stream's scores wait for its last
// product and its exponentials for the scores, and two streams cover that only in part.  32 heads, 8 kv heads, hd 128,
// bf16: 2048 tokens of 4096 123 us (840 TFLOP/s, of 1675 that a large product reaches), 2048 of 2048 71 us, a prompt of
// 8192 602 us (913 TFLOP/s), 256 of 4096 36 us; hd 64, 2048 of 4096 111 us.  Some 20 us of a call are its
// beginning (finding the shares 3.3 us, first copies 2 us), the tiles' epilogues and the join.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "tl_paged_attn.cuh"

namespace tl {
namespace paged {
namespace {

using namespace tc;

constexpr int kRows = 256, kHalf = 128, kKB = 128;
constexpr int kWarps = 20, kThreads = kWarps * 32;
template <typename T>
struct Range {  // log2 units
    static constexpr float kRescale = std::is_same<T, __half>::value ? 4.f : 8.f;
    static constexpr float kLift = std::is_same<T, __half>::value ? 11.f : 0.f;
    static constexpr float kLeast = std::is_same<T, __half>::value ? 1024.f : 0.5f;  // half of the largest weight's least
};

// One step: 256 rows x 128 keys, or (tiles of at most 128 rows) 128 rows x 256 keys.  Beginning and ending a
// tile takes about as long as kTileCost steps, which count as steps before its first key tile.  0 / 2 / 4 steps: 2048
// tokens of 4096 bf16 128 / 124 / 127 us, 2048 of 2048 138 / 71 / 66, 9 ragged chunks of at most 389 tokens fp16 146 / 108 /
// 110, 9 x 200 tokens of 2000 117 / 109 / 105.
struct ChunkPlan {
    static constexpr int R = kRows;
    static constexpr int kTileCost = 2;
    static constexpr bool kLookAgain = false;
    static __device__ __forceinline__ int key_tiles(const Tile& t) {
        return t.hi <= t.lo ? 1 : (t.hi - 1) / kKB - t.lo / kKB + 1;
    }
    static __device__ __forceinline__ int steps(const Tile& t) {
        const int n = key_tiles(t);
        return kTileCost + (t.nrows > kHalf ? n : (n + 1) / 2);
    }
};

template <int HD>
struct Shape {
    static constexpr int PANELS = HD / 64;
    static constexpr int PANEL = kKB * 128;       // bytes of 64 columns of 128 rows
    static constexpr int STAGE = PANELS * PANEL;  // K or V of 128 keys
    static constexpr int NST = HD == 128 ? 5 : 10;
    static constexpr size_t SMEM = 2 * static_cast<size_t>(STAGE) + static_cast<size_t>(NST) * STAGE + 512 +
                                   4 * kHalf * 4 + 16;
};

// K-major operand: rows of 64 columns (128 bytes), SWIZZLE_128B: sdesc_k128.
// N-major operand of 16-bit values, SWIZZLE_128B: rows are k, 64 columns each;
// 8-row atoms 1024 bytes apart (stride offset), column panels `panel` bytes
// apart (leading offset).
__device__ __forceinline__ uint64_t sdesc_n128(uint32_t addr, uint32_t panel) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((addr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>(panel >> 4) << 16;
    d |= static_cast<uint64_t>(1024 >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}
// Instruction descriptor, kind::f16: D fp32, A and B of one 16-bit type, M 128; B K-major or N-major.
template <typename T>
__device__ __forceinline__ constexpr uint32_t idesc(int n, bool b_n_major) {
    const uint32_t f = std::is_same<T, __half>::value ? 0u : 1u;
    return (1u << 4) | (f << 7) | (f << 10) | ((b_n_major ? 1u : 0u) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
           (static_cast<uint32_t>(128 >> 4) << 24);
}

// One lane of a converged warp, the same one every time.
__device__ __forceinline__ bool elect_one() {
    uint32_t y;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(y));
    return y != 0;
}
// Four products of 16 keys (or dims) each.  Addresses in tensor memory, the instruction descriptor and the upper
// halves of the operand descriptors are constants, so that what an instruction takes from registers is the lower
// half of one or two descriptors: moving all of them cost more time than the products.
template <uint32_t D, uint32_t ID, uint32_t HI>
__device__ __forceinline__ void mma4_ss(uint32_t a, uint32_t b, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b32 x, y;\n\t.reg .b64 da, db;\n\t"
        "setp.ne.b32 p, %2, 0;\n\tsetp.eq.b32 q, 0, 0;\n\t"
        "mov.b64 da, {%0, %5};\n\tmov.b64 db, {%1, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%3], da, db, %4, p;\n\t"
        "add.u32 x, %0, 2;\n\tadd.u32 y, %1, 2;\n\tmov.b64 da, {x, %5};\n\tmov.b64 db, {y, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%3], da, db, %4, q;\n\t"
        "add.u32 x, %0, 4;\n\tadd.u32 y, %1, 4;\n\tmov.b64 da, {x, %5};\n\tmov.b64 db, {y, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%3], da, db, %4, q;\n\t"
        "add.u32 x, %0, 6;\n\tadd.u32 y, %1, 6;\n\tmov.b64 da, {x, %5};\n\tmov.b64 db, {y, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%3], da, db, %4, q;\n\t}" ::"r"(a),
        "r"(b), "r"(acc), "r"(D), "r"(ID), "r"(HI));
}
template <uint32_t D, uint32_t A, uint32_t ID, uint32_t HI>
__device__ __forceinline__ void mma4_ts(uint32_t b, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b32 y;\n\t.reg .b64 db;\n\t"
        "setp.ne.b32 p, %1, 0;\n\tsetp.eq.b32 q, 0, 0;\n\t"
        "mov.b64 db, {%0, %4};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%2], [%5], db, %3, p;\n\t"
        "add.u32 y, %0, 128;\n\tmov.b64 db, {y, %4};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%2], [%6], db, %3, q;\n\t"
        "add.u32 y, %0, 256;\n\tmov.b64 db, {y, %4};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%2], [%7], db, %3, q;\n\t"
        "add.u32 y, %0, 384;\n\tmov.b64 db, {y, %4};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%2], [%8], db, %3, q;\n\t}" ::"r"(b),
        "r"(acc), "r"(D), "r"(ID), "r"(HI), "r"(A), "r"(A + 8), "r"(A + 16), "r"(A + 24));
}

__device__ __noinline__ bool fails(unsigned one_in) { return told_to_fail(one_in); }

__device__ __noinline__ bool wait_slow(uint64_t* b, uint32_t parity, volatile int* abort_flag, unsigned fail_one_in) {
    return !(fail_one_in != 0 && fails(fail_one_in)) && bar_spin_ab(b, parity, abort_flag);
}

__device__ __noinline__ bool doze_slow(uint64_t* b, uint32_t parity, volatile int* abort_flag, unsigned fail_one_in) {
    return !(fail_one_in != 0 && fails(fail_one_in)) && bar_wait_ab(b, parity, abort_flag);
}

// All threads of a stream meet; whether `good` holds for all of them.
__device__ __forceinline__ bool stream_sync(int i, bool good) {
    uint32_t y;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, %2, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(y)
        : "r"(static_cast<uint32_t>(good)), "r"(1 + i)
        : "memory");
    return y != 0;
}

// The larger of three.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ void tma_panel(void* dst, const CUtensorMap* map, int row, int panel, int page, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::
            "r"(su32(dst)), "l"(map), "r"(0), "r"(row), "r"(panel), "r"(page), "r"(su32(bar))
        : "memory");
}
__device__ __forceinline__ uint32_t sw128(int r, int c) {
    return static_cast<uint32_t>(r * 128 + ((c ^ (r & 7)) << 4));
}
// 32 columns, without waiting for them.
__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld16_async(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16_async(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
            taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ uint32_t pack2(float x, float y, __half*) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float x, float y, __nv_bfloat16*) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// The key tiles [jb, je) of a cursor's part of a row tile, and which of them each stream takes.
struct Part {
    int jb, je, kb0;  // key tile j covers positions (kb0 + j) * 128 ..
    bool two;         // two streams of rows (else the streams take key tiles in turn)
    int end0;         // two: stream 0's last key tile + 1 (its tokens end earlier)
    __device__ __forceinline__ bool active(int i) const { return begin(i) < end(i); }
    __device__ __forceinline__ int begin(int i) const { return two ? jb : jb + i; }
    __device__ __forceinline__ int end(int i) const { return two && i == 0 ? end0 : je; }
    __device__ __forceinline__ int stride() const { return two ? 1 : 2; }
};
__device__ __forceinline__ Part part_of(const AttendArgs& a, const Cursor& c) {
    Part p;
    const int n = ChunkPlan::key_tiles(c.t);
    p.two = c.t.nrows > kHalf;
    const int s = max(0, c.s - ChunkPlan::kTileCost), e = max(0, c.end - ChunkPlan::kTileCost);
    p.jb = p.two ? s : 2 * s;
    p.je = min(n, p.two ? e : 2 * e);
    p.kb0 = c.t.lo / kKB;
    p.end0 = p.je;
    if (p.two) {
        int lo, hi;
        attended(a, c.t.p0 + div_group(a, c.t.r0 + kHalf - 1), lo, hi);
        p.end0 = hi <= 0 ? 0 : max(0, min(p.je, (hi - 1) / kKB - p.kb0 + 1));
    }
    return p;
}

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, 1)
    k_attend_chunk(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                   const __grid_constant__ CUtensorMap map_q, const __grid_constant__ AttendArgs a,
                   Head* heads, float* parts) {
    using S = Shape<HD>;
    constexpr int NST = S::NST;
    extern __shared__ __align__(1024) uint8_t smem_chunk[];
    uint8_t* sQ = smem_chunk;  // [2 streams]
    uint8_t* ring = sQ + 2 * S::STAGE;
    uint64_t* full = reinterpret_cast<uint64_t*>(ring + NST * S::STAGE);
    uint64_t* empty = full + NST;
    uint64_t* s_full = empty + NST;  // [2] S_i written (and every MMA before it done)
    uint64_t* p_full = s_full + 2;   // [2][2] halves of P_i (64 keys) written: 4 warps
    uint64_t* q_full = p_full + 4;   // [2] Q_i written
    uint64_t* o_full = q_full + 2;   // [2] the stream's last product done
    uint64_t* xbar = o_full + 2;     // both streams' 16 warps
    uint64_t* drain = xbar + 1;
    uint64_t* q_free = drain + 1;    // [2] the tile's last scores of stream i done
    static_assert((2 * 10 + 14) * 8 <= 512, "barriers");
    uint8_t* xch = reinterpret_cast<uint8_t*>(full) + 512;  // what the halves and streams of a row exchange
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(xch + 2048);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    long long* ws = reinterpret_cast<long long*>(ring);  // the scan runs before the ring is used

    const int warp = __shfl_sync(FULL, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // (uniform for the compiler)
    if (threadIdx.x == 0) heads[blockIdx.x].parts = 0;
    Cursor c;
    const int per = find_share<ChunkPlan, kWarps>(a, c, ws, ChunkPlan::kTileCost + 1);
    if (per == 0) return;

    if (threadIdx.x == 0) {
        for (int i = 0; i < NST; i++) {
            bar_init(&full[i], 1);
            bar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            bar_init(&s_full[i], 1);
            bar_init(&p_full[2 * i], 4);
            bar_init(&p_full[2 * i + 1], 4);
            bar_init(&q_full[i], 1);
            bar_init(&q_free[i], 1);
            bar_init(&o_full[i], 1);
        }
        bar_init(xbar, 16);
        bar_init(drain, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 17) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(tmem_slot)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_proxy_async();  // the scan's writes to the ring precede the copies into it
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // All 512 columns are this block's, so they begin at 0.  S_i at 128 i, O_i at 256 + 128 i.
    constexpr uint32_t tmem = 0, tS = 0, kTO = 256, tO = kTO;
    if (*tmem_slot != tmem) *abort_flag = 1;

    auto fail = [&] { *abort_flag = 1; };
    // waits poll: the hand-offs here are short and frequent
    auto wait = [&](uint64_t* b, uint32_t parity) { return bar_test_now(b, parity) || wait_slow(b, parity, abort_flag, a.fail_one_in); };
    auto doze = [&](uint64_t* b, uint32_t parity) { return bar_test_now(b, parity) || doze_slow(b, parity, abort_flag, a.fail_one_in); };

    if (warp == 16) {
        // ---- TMA: K_j, V_j of each key tile; lane = one page's rows of one panel ----
        const int rows = min(kKB, 1 << a.shift);  // rows of a copy
        const int pages = kKB / rows;
        const int pg = lane / S::PANELS, panel = lane % S::PANELS;
        uint32_t n = 0;  // loads issued
        bool ok = true;
        for (bool go = true; ok && go; go = next_tile<ChunkPlan>(a, c)) {
            const Part p = part_of(a, c);
            const int off = pg * rows;
            auto id_of = [&](int j) { return pg < pages && j < p.je ? page_of(a, c.b, (p.kb0 + j) * kKB + off) : -1; };
            int id = id_of(p.jb);
            for (int j = p.jb; ok && j < p.je; j++) {
                const int id_next = id_of(j + 1);
                const int key0 = (p.kb0 + j) * kKB + off;
                const int row = (c.g << a.shift) + (key0 & ((1 << a.shift) - 1));
#pragma unroll
                for (int kv = 0; kv < 2; kv++) {
                    const uint32_t st = n % NST;
                    if (!__all_sync(FULL, n < NST || doze(&empty[st], (n / NST - 1) & 1))) {
                        ok = false;
                        break;
                    }
                    if (lane == 0) bar_expect_tx(&full[st], S::STAGE);
                    __syncwarp();
                    if (pg < pages)
                        tma_panel(ring + st * S::STAGE + panel * S::PANEL + off * 128, kv ? &map_v : &map_k, row, panel, id,
                                  &full[st]);
                    n++;
                }
                id = id_next;
            }
        }
        if (!ok) fail();
        // every copy issued lands before the block ends
        for (uint32_t k = n > NST ? n - NST : 0; k < n; k++) bar_wait(&full[k % NST], (k / NST) & 1);
    } else if (warp == 17) {
        if (elect_one()) {
            // ---- MMA: one thread for both streams, so that they stay half a step apart and do not take the
            // exponentials at the same time.  It has to be quick between its waits: what it queues in the matrix
            // unit lasts for two or three products. ----
            constexpr uint32_t id_s = idesc<T>(kKB, false), id_o = idesc<T>(HD, true);
            constexpr uint32_t kHi = (1024 >> 4) | (1u << 14) | (2u << 29);  // stride offset, version, SWIZZLE_128B
            constexpr uint32_t STEP = S::STAGE >> 4, PSTEP = S::PANEL >> 4;
            const uint32_t lq = static_cast<uint32_t>(sdesc_k128(su32(sQ))), lk = static_cast<uint32_t>(sdesc_k128(su32(ring))),
                           lv = static_cast<uint32_t>(sdesc_n128(su32(ring), S::PANEL));
            uint32_t n0 = 0;                         // loads before this tile
            uint32_t nq[2] = {0, 0}, np[2] = {0, 0}; // phases of q_full and p_full
            bool ok = true;
#pragma unroll 1
            for (bool go = true; ok && go; go = next_tile<ChunkPlan>(a, c)) {
                const Part p = part_of(a, c);
                const uint32_t step = 2 * p.stride();
                // the stages and phases of each stream's next K and V
                uint32_t ks[2], kp[2], vs[2], vp[2];
                int nb[2];  // key tiles of the streams
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const uint32_t k = n0 + 2 * (p.begin(i) - p.jb);
                    ks[i] = k % NST;
                    kp[i] = (k / NST) & 1;
                    vs[i] = (k + 1) % NST;
                    vp[i] = ((k + 1) / NST) & 1;
                    nb[i] = max(0, p.two ? p.end(i) - p.jb : (p.je - p.jb + 1 - i) / 2);
                }
                auto advance = [&](uint32_t& st, uint32_t& ph) {
                    st += step;
                    if (st >= NST) {
                        st -= NST;
                        ph ^= 1;
                    }
                };
                const bool both = p.two;  // stream 0 has waited for what stream 1 reads; stream 1 frees it
                auto scores = [&](auto stream, bool known, bool last) -> bool {  // S_i = Q_i K^T
                    constexpr int i = decltype(stream)::value;
                    if (!known && !doze(&full[ks[i]], kp[i])) return false;
                    tc_fence_after();
                    const uint32_t x = lq + i * STEP, y = lk + ks[i] * STEP;
#pragma unroll
                    for (int d = 0; d < S::PANELS; d++) mma4_ss<128 * i, id_s, kHi>(x + d * PSTEP, y + d * PSTEP, d);
                    umma_commit(&s_full[i]);
                    if (last) umma_commit(&q_free[i]);
                    if (!both || i == 1) umma_commit(&empty[ks[i]]);
                    advance(ks[i], kp[i]);
                    return true;
                };
                auto values = [&](auto stream, bool known, uint32_t acc) -> bool {  // O_i (+)= P_i V
                    constexpr int i = decltype(stream)::value;
                    if (!known && !doze(&full[vs[i]], vp[i])) return false;
                    const uint32_t y = lv + vs[i] * STEP;
                    if (!doze(&p_full[2 * i], np[i])) return false;
                    tc_fence_after();
                    mma4_ts<kTO + 128 * i, 128 * i, id_o, kHi>(y, acc);
                    if (!doze(&p_full[2 * i + 1], np[i])) return false;
                    tc_fence_after();
                    mma4_ts<kTO + 128 * i, 128 * i + 64, id_o, kHi>(y + 512, 1);
                    np[i] ^= 1;
                    if (!both || i == 1) umma_commit(&empty[vs[i]]);
                    advance(vs[i], vp[i]);
                    return true;
                };
                auto begin = [&](auto stream) {
                    constexpr int i = decltype(stream)::value;
                    if (!ok || nb[i] == 0) return;
                    ok = wait(&q_full[i], nq[i]);
                    nq[i] ^= 1;
                    ok = ok && scores(stream, both && i == 1 && nb[0] > 0, nb[i] == 1);
                };
                auto turn = [&](auto stream, int j) {
                    constexpr int i = decltype(stream)::value;
                    if (!ok || j >= nb[i]) return;
                    ok = values(stream, both && i == 1 && j < nb[0], j != 0);
                    if (!ok) return;
                    if (j + 1 < nb[i]) ok = scores(stream, both && i == 1 && j + 1 < nb[0], j + 2 == nb[i]);
                    else umma_commit(&o_full[i]);
                };
                constexpr std::integral_constant<int, 0> s0{};
                constexpr std::integral_constant<int, 1> s1{};
                begin(s0);
                begin(s1);
                const int nt = max(nb[0], nb[1]);
#pragma unroll 1
                for (int j = 0; ok && j < nt; j++) {
                    turn(s0, j);
                    turn(s1, j);
                }
                n0 += 2 * (p.je - p.jb);
            }
            if (!ok) fail();
            umma_commit(drain);  // completes once every MMA issued above has
            bar_wait(drain, 0);
        }
    } else if (warp >= 18) {
        // ---- Q rows of stream i into the swizzled K-major panels.  Where the group divides 128 they are whole tokens,
        // a box of the map for each panel (rows behind the tile are other tokens', and nobody's results); else a row
        // is CH pieces of 16 bytes, one a lane.  A prompt of 8192 with groups of 4: 604 us by the boxes, 612 by lanes.
        // ----
        const int i = warp - 18;
        constexpr int CH = HD / 8, RPI = 32 / CH;
        const int d = lane % CH;
        uint8_t* dst = sQ + i * S::STAGE + (d / 8) * S::PANEL;
        uint32_t loaded = 0;
        bool ok = true;
#pragma unroll 1
        for (bool go = true; ok && go; go = next_tile<ChunkPlan>(a, c)) {
            const Part p = part_of(a, c);
            if (!p.active(i)) continue;
            if (loaded && !__all_sync(FULL, doze(&q_free[i], (loaded - 1) & 1))) {
                ok = false;
                break;
            }
            const int row0 = p.two ? i * kHalf : 0;
            loaded++;
            if (kHalf % a.group == 0) {
                if (lane == 0) {
                    bar_expect_tx(&q_full[i], S::STAGE);
                    for (int x = 0; x < S::PANELS; x++)
                        tma_panel(sQ + i * S::STAGE + x * S::PANEL, &map_q, x, c.g * a.group, c.t.first + div_group(a, c.t.r0 + row0),
                                  &q_full[i]);
                }
                __syncwarp();
                continue;
            }
#pragma unroll 1
            for (int r0 = 0; r0 < kHalf; r0 += 32) {  // a lane finds one row's place, the others get it from there
                int tok, h;
                row_of(a, c, row0 + r0 + lane, tok, h);
                const unsigned long long at = static_cast<size_t>(tok) * a.q_stride + static_cast<size_t>(h) * HD;
#pragma unroll 2
                for (int k = 0; k < 32; k += RPI) {
                    const int kk = k + lane / CH, rr = r0 + kk;
                    const T* src = static_cast<const T*>(a.q) + __shfl_sync(FULL, at, kk) + 8 * d;
                    const uint32_t bytes = row0 + rr < c.t.nrows ? 16u : 0u;  // (a row that does not exist: zeros)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(su32(dst + sw128(rr, d & 7))), "l"(src), "r"(bytes)
                                 : "memory");
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) bar_arrive(&q_full[i]);
        }
        if (!ok) fail();
        if (loaded) bar_wait(&q_full[i], (loaded - 1) & 1);  // a copy lands before the block ends
    } else {
        // ---- softmax and epilogue: thread = half hf of row r of stream i.  A thread whose wait fails goes on
        // through the loops' barriers, doing no work, so that the others find it there ----
        const int i = warp >> 3, hf = (warp >> 2) & 1, quad = (warp & 3) * 32, r = quad + lane;
        const uint32_t lane_off = static_cast<uint32_t>(quad) << 16;
        const uint32_t ts = tS + 128 * i + 64 * hf + lane_off, to = tO + 128 * i + lane_off;
        const float scale = a.scale * 1.4426950408889634f;  // log2 units
        const float sl = fabsf(scale);
        // [stream][half][row]: the maxima of a block (read before its weights, which the next block's scores wait
        // for: one buffer is enough), at a tile's end the sums
        float* xl = reinterpret_cast<float*>(xch);
        uint32_t n0 = 0, ns = 0, no = 0, nx = 0;
        bool ok = true, first_tile = true, go = true;
        auto give_up = [&] {
            ok = false;
            fail();
        };
#pragma unroll 1
        for (; go; go = next_tile<ChunkPlan>(a, c), first_tile = false) {
            const Part p = part_of(a, c);
            const int row = p.two ? i * kHalf + r : r;  // of the tile
            const bool in = row < c.t.nrows;
            int tok, h;
            row_of(a, c, row, tok, h);
            const bool act = p.active(i);
            int lo, hi;
            attended(a, c.t.p0 + (tok - c.t.first), lo, hi);
            float m = -INFINITY, l = 0.f;
            if (act) {
                const int stride = p.stride();
                auto page_at = [&](int j) { return lane < 8 ? page_of(a, c.b, (p.kb0 + j) * kKB + 64 * hf + 8 * lane) : 0; };
                int pid_next = page_at(p.begin(i));
#pragma unroll 1
                for (int j = p.begin(i); j < p.end(i); j += stride, ns++) {
                    const int key0 = (p.kb0 + j) * kKB + 64 * hf;  // of this half
                    const int pid = pid_next;
                    pid_next = j + stride < p.end(i) ? page_at(j + stride) : 0;
                    // every lane waits; the outcome is warp-uniform (tensor-memory access is warp-wide)
                    bool good = ok && __all_sync(FULL, doze(&s_full[i], ns & 1));
                    if (ok && !good) give_up();
                    uint32_t u[32];
                    float mx[2] = {-INFINITY, -INFINITY};
                    if (good) {
                        tc_fence_after();
                        const uint32_t pages = __ballot_sync(FULL, pid >= 0);  // bit k: keys 8 k .. 8 k + 7 exist
                        // Masked columns, and the sign of a negative scale, go into the scores in tensor memory first;
                        // only the border tiles of a row need that, and the loops below stay short.
                        if (!__all_sync(FULL, !in || (key0 >= lo && key0 <= hi - 64)) || pages != FULL || scale < 0.f) {
                            const uint32_t sign = scale < 0.f ? 0x80000000u : 0u;
#pragma unroll 1
                            for (int q = 0; q < 2; q++) {
                                const int k0 = key0 + 32 * q;
                                const int x0 = max(0, min(32, lo - k0)), x1 = max(0, min(32, hi - k0));
                                uint32_t keep = x1 > x0 ? (x1 == 32 ? ~0u : (1u << x1) - 1) & ~(x0 == 32 ? ~0u : (1u << x0) - 1) : 0u;
                                const uint32_t pq = pages >> (4 * q);
                                keep &= ((pq & 1) ? 0xffu : 0u) | ((pq & 2) ? 0xff00u : 0u) | ((pq & 4) ? 0xff0000u : 0u) |
                                        ((pq & 8) ? 0xff000000u : 0u);
                                tmem_ld32_async(ts + 32 * q, u);
                                tmem_wait_ld();
#pragma unroll
                                for (int e = 0; e < 32; e++) u[e] = ((keep >> e) & 1) ? u[e] ^ sign : 0xff800000u;
                                tmem_st16_async(ts + 32 * q, u);
                                tmem_st16_async(ts + 32 * q + 16, u + 16);
                            }
                            tmem_wait_st();
                        }
                        // the maximum, the first 32 columns last: they stay in registers for the weights
#pragma unroll
                        for (int q = 1; q >= 0; q--) {
                            tmem_ld32_async(ts + 32 * q, u);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; e += 2)
                                mx[(e / 2) & 1] = max3(mx[(e / 2) & 1], __uint_as_float(u[e]), __uint_as_float(u[e + 1]));
                        }
                    }
                    const float own = fmaxf(mx[0], mx[1]) * sl;
                    xl[(2 * i + hf) * 128 + r] = own;
                    good = stream_sync(i, good);
                    if (!good) continue;
                    const float top = fmaxf(own, xl[(2 * i + (hf ^ 1)) * 128 + r]);
                    float f = 1.f;
                    if (top > m + Range<T>::kRescale || (m == -INFINITY && top > -INFINITY)) {
                        if (m != -INFINITY) f = ex2(m - top);
                        m = top;
                    }
                    if (__any_sync(FULL, f != 1.f)) {  // S of this tile is done, so the products before it are
                        l *= f;
#pragma unroll 1
                        for (int q = 0; q < HD / 32; q++) {  // this half's columns
                            uint32_t o[16];
                            const uint32_t ta = to + hf * (HD / 2) + 16 * q;
                            tmem_ld16_async(ta, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            tmem_st16_async(ta, o);
                        }
                        tmem_wait_st();
                        tc_fence_before();
                        // the first half's weights start the products: not before the other half's columns are scaled
                        asm volatile("bar.sync %0, 64;" ::"r"(3 + 4 * i + (warp & 3)) : "memory");
                    }
                    // masked scores and rows that see nothing: 2^(-inf) = 0
                    const float base = m == -INFINITY ? 0.f : Range<T>::kLift == 0.f ? -m : Range<T>::kLift - m;
                    if (key0 < c.t.lo || key0 > c.t.hi - 64) {
                        // rows of V that no query attends to may hold anything: no 0 x NaN.  (Both streams
                        // write the same zeros; each before its own product.)
                        const uint32_t n = n0 + 2 * (j - p.jb) + 1, st = n % NST;
                        if (!__all_sync(FULL, wait(&full[st], (n / NST) & 1))) give_up();
                        const int key = key0 + (r & 63), vr = 64 * hf + (r & 63);
                        if (key < c.t.lo || key >= c.t.hi) {
#pragma unroll 1
                            for (int d = r >> 6; d < HD / 8; d += 2)
                                *reinterpret_cast<uint4*>(ring + st * S::STAGE + (d / 8) * S::PANEL + sw128(vr, d & 7)) =
                                    make_uint4(0, 0, 0, 0);
                        }
                        fence_proxy_async();
                    }
                    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int q = 0; q < 2; q++) {
                        if (q) tmem_wait_ld();
                        uint32_t w[16];
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            const float x = ex2(fmaf(__uint_as_float(u[2 * e]), sl, base));
                            const float y = ex2(fmaf(__uint_as_float(u[2 * e + 1]), sl, base));
                            sum[(2 * e) & 3] += x;
                            sum[(2 * e + 1) & 3] += y;
                            w[e] = pack2(x, y, static_cast<T*>(nullptr));
                        }
                        if (q == 0) tmem_ld32_async(ts + 32, u);
                        tmem_st16_async(ts + 16 * q, w);  // over scores that have been read
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive(&p_full[2 * i + hf]);
                    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                }
            }
            if (act) {
                if (ok && !__all_sync(FULL, doze(&o_full[i], no & 1))) give_up();
                no++;
                tc_fence_after();
            }
            n0 += 2 * (p.je - p.jb);
            // ---- epilogue: this thread's columns of the row's sum over the halves and, if both have keys of the
            // same rows, over the streams ----
            const bool fold = !p.two && p.active(1);
            stream_sync(i, true);  // the maxima have been read
            xl[(2 * i + hf) * 128 + r] = l;
            const bool good = stream_sync(i, ok);
            float w0 = 1.f, w1 = 0.f, mt = m, lt = xl[2 * i * 128 + r] + xl[(2 * i + 1) * 128 + r];
            // The largest weight is 2^kLift at least, but for what m was rounded by, which the exact products in the
            // exponents bring back: scores beyond 2^24 may lose all their weights by that, and infinite ones do.
            if ((lt > 0.f && lt < Range<T>::kLeast) || m == INFINITY) lt = NAN;
            if (fold) {
                stream_sync(i, true);
                xl[(2 * i + hf) * 128 + r] = !good ? NAN : hf ? lt : m;
                __syncwarp();
                if (lane == 0) bar_arrive(xbar);
                if (good && !__all_sync(FULL, wait(xbar, nx & 1))) give_up();
                nx++;
                const float m0 = xl[r], m1 = xl[256 + r];
                mt = fmaxf(m0, m1);
                w0 = mt == -INFINITY ? 1.f : ex2(m0 - mt);
                w1 = mt == -INFINITY ? 1.f : ex2(m1 - mt);
                lt = xl[128 + r] * w0 + xl[384 + r] * w1;
                // Warps that gave up do not wait here, and may arrive twice in one phase: what was read need not be this
                // tile's.  They set the flag before they arrive.
                __syncwarp();
                if (*abort_flag) lt = NAN;
                tc_fence_after();
            }
            const bool whole = c.s == 0 && c.end == c.steps;
            const bool writer = p.two || fold || i == 0;
            // A wait that ran out: the accumulators hold nothing, and the rows are done over like those that are not finite.
            const bool fine = good && ok;
            if (!fine) lt = NAN;
            const int c0 = fold ? (2 * i + hf) * (HD / 4) : hf * (HD / 2), c1 = c0 + (fold ? HD / 4 : HD / 2);  // columns
            float* part = parts + (static_cast<size_t>(blockIdx.x) * 2 + (first_tile ? 0 : 1)) * kRows * (HD + 4);
            if (writer) {
                const float inv = lt != 0.f ? 1.f / lt : 0.f;
                float z = whole && lt == 0.f ? NAN : lt * 0.f;  // NaN once a value is not finite (or nothing has weight)
                const bool t0 = fine && (fold || act);
                const uint32_t ta = fold ? tO + lane_off : to;
#pragma unroll 1
                for (int col = c0; col < c1; col += 16) {
                    uint32_t o[16];
                    if (t0) {
                        tmem_ld16_async(ta + col, o);
                        tmem_wait_ld();
                    } else {  // (a part of a warp that gave up is not finite in its own columns either)
                        const uint32_t none = fine ? 0u : 0x7fc00000u;
#pragma unroll
                        for (int e = 0; e < 16; e++) o[e] = none;
                    }
                    if (fold && fine) {
                        uint32_t o1[16];
                        tmem_ld16_async(tO + 128 + lane_off + col, o1);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; e++)
                            o[e] = __float_as_uint(__uint_as_float(o[e]) * w0 + __uint_as_float(o1[e]) * w1);
                    }
#pragma unroll
                    for (int e = 0; e < 16; e++) z = fmaf(__uint_as_float(o[e]), 0.f, z);
                    if (!in) continue;
                    if (whole) {  // 32 bytes of this row
                        uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (static_cast<size_t>(tok) * a.H + h) * HD + col);
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            uint4 v;
                            uint32_t* vw = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
                            for (int k = 0; k < 4; k++)
                                vw[k] = pack2(__uint_as_float(o[8 * e + 2 * k]) * inv, __uint_as_float(o[8 * e + 2 * k + 1]) * inv,
                                              static_cast<T*>(nullptr));
                            dst[e] = v;
                        }
                    } else {  // [4-column group][row], so that a warp's stores are whole lines
                        uint4* dst = reinterpret_cast<uint4*>(part) + kRows;
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            dst[static_cast<size_t>(col / 4 + e) * kRows + row] =
                                make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                    }
                }
                // do over: a value that this row must not see may have met it as 0 x infinity (see tl_paged_attn.cu).
                // These columns only: the row's others are other warps', which may not see it and write theirs.
                const bool redo = in && z != z;
                if (whole) {
                    __syncwarp();
                    for (unsigned bad = __ballot_sync(FULL, redo); bad; bad &= bad - 1) {
                        const int src = __ffs(bad) - 1;
                        __syncwarp();
                        attend_row<T, HD>(a, c.b, __shfl_sync(FULL, tok, src), __shfl_sync(FULL, h, src), lane, c0 | (c1 << 16));
                    }
                } else if (in && hf == 0 && (!fold || i == 0)) {
                    *reinterpret_cast<float2*>(part + 4 * row) = make_float2(mt, lt);
                }
            }
            if (!whole && c.s == 0 && threadIdx.x == 0) {  // this block begins the tile: it says who has the rest
                Head hd;
                hd.parts = parts_of(c.steps, c.end, per);
                hd.slot = first_tile ? 0 : 1;
                hd.b = c.b;
                hd.rt = c.rt;
                hd.g = c.g;
                heads[blockIdx.x] = hd;
            }
            // Before the next tile's weights, which let products overwrite them: both halves, and (fold) both streams,
            // have read the accumulators.
            if (fold) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(xbar);
                if (good && !__all_sync(FULL, wait(xbar, nx & 1))) give_up();
                nx++;
            }
            tc_fence_before();
            stream_sync(i, true);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 17) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// Joins the parts of the tile that block blockIdx.x began (part i > 0: the first tile of block blockIdx.x + i).
// Block y takes 32 rows.  Reading, lane = row and warp = one 8th of the columns, as the parts lie; writing, a warp a
// row, through shared memory.
template <typename T, int HD>
__global__ void __launch_bounds__(256) k_attend_chunk_join(const __grid_constant__ AttendArgs a, const Head* heads, const float* parts) {
    constexpr int G = HD / 4 / 8;  // 4-column groups of a warp
    __shared__ float4 rows[32][HD / 4 + 1];
    __shared__ unsigned bad_rows;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) bad_rows = 0;
    pdl_wait();
    const Head h = heads[blockIdx.x];
    if (h.parts == 0) return;
    Cursor c;
    c.g = h.g;
    c.t = tile_of(a, h.b, h.rt, kRows);
    const int row0 = blockIdx.y * 32, row = row0 + lane;
    if (row0 >= c.t.nrows) return;
    const bool in = row < c.t.nrows;
    constexpr size_t rec = static_cast<size_t>(kRows) * (HD / 4 + 1);  // float4s of a part
    const float4* p0 = reinterpret_cast<const float4*>(parts) + (static_cast<size_t>(blockIdx.x) * 2 + h.slot) * rec;
    const float4* p1 = reinterpret_cast<const float4*>(parts) + (static_cast<size_t>(blockIdx.x) + 1) * 2 * rec;
    float M = -INFINITY, L = 0.f;
    float4 acc[G];
#pragma unroll
    for (int g = 0; g < G; g++) acc[g] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (in) {
#pragma unroll 1
        for (int i0 = 0; i0 < h.parts; i0 += 2) {  // two parts' loads at a time
            float2 s[2];
            float4 v[2][G];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int i = i0 + k;
                if (i < h.parts) {
                    const float4* p = i == 0 ? p0 : p1 + static_cast<size_t>(i - 1) * 2 * rec;
                    s[k] = *reinterpret_cast<const float2*>(p + row);
#pragma unroll
                    for (int g = 0; g < G; g++) v[k][g] = p[static_cast<size_t>(1 + warp * G + g) * kRows + row];
                } else {
                    s[k] = make_float2(-INFINITY, 0.f);
#pragma unroll
                    for (int g = 0; g < G; g++) v[k][g] = make_float4(0.f, 0.f, 0.f, 0.f);
                }
            }
            const float mx = fmaxf(M, fmaxf(s[0].x, s[1].x));
            const float f = mx == -INFINITY ? 1.f : ex2(M - mx), f0 = mx == -INFINITY ? 1.f : ex2(s[0].x - mx),
                        f1 = mx == -INFINITY ? 1.f : ex2(s[1].x - mx);
            M = mx;
            L = L * f + s[0].y * f0 + s[1].y * f1;
#pragma unroll
            for (int g = 0; g < G; g++) {
                acc[g].x = acc[g].x * f + v[0][g].x * f0 + v[1][g].x * f1;
                acc[g].y = acc[g].y * f + v[0][g].y * f0 + v[1][g].y * f1;
                acc[g].z = acc[g].z * f + v[0][g].z * f0 + v[1][g].z * f1;
                acc[g].w = acc[g].w * f + v[0][g].w * f0 + v[1][g].w * f1;
            }
        }
    }
    float z = L != 0.f ? L * 0.f : NAN;  // NaN once a value is not finite, or nothing has weight: the row is done over
    const float inv = L != 0.f ? 1.f / L : 0.f;
#pragma unroll
    for (int g = 0; g < G; g++) {
        z = fmaf(acc[g].x, 0.f, fmaf(acc[g].y, 0.f, fmaf(acc[g].z, 0.f, fmaf(acc[g].w, 0.f, z))));
        rows[lane][warp * G + g] = make_float4(acc[g].x * inv, acc[g].y * inv, acc[g].z * inv, acc[g].w * inv);
    }
    const unsigned mine = __ballot_sync(FULL, in && z != z);
    __syncthreads();
    if (lane == 0 && mine) atomicOr(&bad_rows, mine);
    __syncthreads();
#pragma unroll 1
    for (int rr = warp; rr < 32 && row0 + rr < c.t.nrows; rr += 8) {
        int tok, hh;
        row_of(a, c, row0 + rr, tok, hh);
        if ((bad_rows >> rr) & 1) {
            attend_row<T, HD>(a, h.b, tok, hh, lane);
        } else if (lane < HD / 4) {
            const float4 v = rows[rr][lane];
            reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (static_cast<size_t>(tok) * a.H + hh) * HD)[lane] =
                make_uint2(pack2(v.x, v.y, static_cast<T*>(nullptr)), pack2(v.z, v.w, static_cast<T*>(nullptr)));
        }
    }
}

// Map of Q: {64 columns, panels, heads, tokens}; a box is one panel of 128 rows, which are the heads of a group for
// 128 / group tokens.  (Where the group does not divide 128 the map is not used.)
template <int HD>
tl_status encode_q(CUtensorMap* map, const AttendArgs& a, tl_dtype dtype) {
    auto fn = encode_fn();
    if (!fn) return set_error(TL_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint32_t group = kHalf % a.group == 0 ? a.group : 1;
    const cuuint64_t dims[4] = {64, HD / 64, static_cast<cuuint64_t>(a.H), static_cast<cuuint64_t>(a.n_tokens)};
    const cuuint64_t strides[3] = {128, HD * 2, a.q_stride * 2};
    const cuuint32_t box[4] = {64, 1, group, kHalf / group};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    const CUresult r = fn(map, dtype == TL_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                          const_cast<void*>(a.q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(TL_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
    return TL_OK;
}

template <typename T, int HD>
tl_status run_chunk(const AttendArgs& a, const tl_paged_cache* c, void* workspace, cudaStream_t s) {
    using S = Shape<HD>;
    static_assert(S::SMEM <= 232448, "shared memory of a block");
    CUtensorMap mk, mv, mq;
    const int rows = std::min(kKB, 1 << a.shift);
    TL_TRY(encode_pages(&mk, c->k, c, rows, 1));
    TL_TRY(encode_pages(&mv, c->v, c, rows, 1));
    TL_TRY(encode_q<HD>(&mq, a, c->dtype));
    TL_CUDA_TRY(cudaFuncSetAttribute(k_attend_chunk<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     static_cast<int>(S::SMEM)));
    const int grid = std::min(sm_count(), kMaxBlocks);
    Head* heads = static_cast<Head*>(workspace);
    float* parts = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kHeadBytes);
    k_attend_chunk<T, HD><<<grid, kThreads, S::SMEM, s>>>(mk, mv, mq, a, heads, parts);
    TL_TRY(check_launch("paged_attention"));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid, kRows / 32);
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    TL_CUDA_TRY(cudaLaunchKernelEx(&cfg, k_attend_chunk_join<T, HD>, a, static_cast<const Head*>(heads),
                                   static_cast<const float*>(parts)));
    return TL_OK;
}

}  // namespace

size_t chunk_workspace(int hd) {
    return kHeadBytes + static_cast<size_t>(std::min(sm_count(), kMaxBlocks)) * 2 * kRows * (hd + 4) * 4;
}

tl_status attend_chunk(const AttendArgs& a, const tl_paged_cache* c, void* workspace, cudaStream_t s) {
    const bool half = c->dtype == TL_F16;
    if (c->head_dim == 128)
        return half ? run_chunk<__half, 128>(a, c, workspace, s) : run_chunk<__nv_bfloat16, 128>(a, c, workspace, s);
    return half ? run_chunk<__half, 64>(a, c, workspace, s) : run_chunk<__nv_bfloat16, 64>(a, c, workspace, s);
}

}  // namespace paged
}  // namespace tl
