// tl_paged_attn.cu -- tl_paged_attention: causal GQA attention of new tokens
// over a paged KV cache.
#include <math.h>

#include <algorithm>

#include "tl_paged_attn.cuh"

namespace tl {
namespace paged {
namespace {

// Warp = one (token, head): lanes hold HD / 32 dims, one online softmax over
// the attended keys.
template <typename T, int HD>
__global__ void __launch_bounds__(128) k_attend_rows(AttendArgs a) {
    const int lane = threadIdx.x & 31;
    const long long u = blockIdx.x * 4ll + (threadIdx.x >> 5);
    if (u >= static_cast<long long>(a.n_tokens) * a.H) return;
    const int t = static_cast<int>(u / a.H), h = static_cast<int>(u % a.H);
    const int b = sequence_of(a, t);
    if (b < 0) return;
    attend_row<T, HD>(a, b, t, h, lane);
}

template <typename T>
void launch_rows(const AttendArgs& a, int hd, cudaStream_t s) {
    const unsigned grid = static_cast<unsigned>((static_cast<long long>(a.n_tokens) * a.H + 3) / 4);
    if (hd == 128) k_attend_rows<T, 128><<<grid, 128, 0, s>>>(a);
    else k_attend_rows<T, 64><<<grid, 128, 0, s>>>(a);
}

}  // namespace
}  // namespace paged
}  // namespace tl

using namespace tl;
using namespace tl::paged;

extern "C" {

tl_status tl_paged_attention_workspace(const tl_paged_cache* cache, size_t n_tokens, size_t n_heads, size_t n_seq,
                                       size_t max_blocks, size_t* bytes) {
    clear_error();
    TL_TRY(check_cache("tl_paged_attention_workspace", cache));
    TL_REQUIRE(bytes, "tl_paged_attention_workspace: no result");
    TL_REQUIRE(n_heads > 0 && n_heads % cache->n_kv_heads == 0, "tl_paged_attention_workspace: %zu heads, %zu kv heads",
               n_heads, cache->n_kv_heads);
    (void)n_tokens; (void)n_seq; (void)max_blocks;
    *bytes = 16;
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
    TL_REQUIRE(n_tokens <= 0x7fffffffull / n_heads, "tl_paged_attention: %zu tokens x %zu heads", n_tokens, n_heads);
    TL_REQUIRE(q_stride >= n_heads * cache->head_dim && q_stride <= (1ull << 36), "tl_paged_attention: q_stride %zu",
               q_stride);
    TL_REQUIRE(aligned16(out) && aligned16(q) && q_stride * dtype_size(cache->dtype) % 16 == 0,
               "tl_paged_attention: out, q and q_stride must be 16-byte aligned");
    TL_REQUIRE(scale == scale && fabsf(scale) <= 3.0e38f, "tl_paged_attention: scale %g", static_cast<double>(scale));
    (void)workspace; (void)workspace_bytes;
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
    a.max_blocks = static_cast<int>(max_blocks);
    a.n_blocks = static_cast<int>(cache->n_blocks);
    a.shift = __builtin_ctzll(cache->block_size);
    a.window = window == 0 || window > 0x7fffffffull ? 0 : static_cast<int>(window);
    a.scale = scale;
    const cudaStream_t s = as_stream(stream);
    const int hd = static_cast<int>(cache->head_dim);
    if (cache->dtype == TL_F32) launch_rows<float>(a, hd, s);
    else if (cache->dtype == TL_F16) launch_rows<__half>(a, hd, s);
    else launch_rows<__nv_bfloat16>(a, hd, s);
    return check_launch("paged_attention");
}

}  // extern "C"
