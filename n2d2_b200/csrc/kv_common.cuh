// The paged cache as kernels see it, and the argument checks that appending to it and attending over it share.
#pragma once
#include "token_common.cuh"

namespace n2d2b {

struct KvArgs {
    int8_t *k, *v;
    float *k_scales, *v_scales;
    const int *table, *lengths, *starts;
    int nb_pages, heads, row;       // row: entries of a sequence's row of the page table
    int nb_tokens, max_new;
};

// A sequence's part of the call, with what the device arrays say brought inside the call's bounds
struct KvSequence {
    int length;     // tokens it holds
    int first_row;  // row of its first new token
    int count;      // new tokens
    int begin;      // position of the first of them; negative when there are more than the length holds
};
__device__ __forceinline__ KvSequence kv_sequence(const KvArgs& c, int b)
{
    KvSequence s;
    s.length = max(c.lengths[b], 0);
    int first = b, end = b + 1;
    if (c.starts) { first = c.starts[b]; end = c.starts[b + 1]; }
    first = min(max(first, 0), c.nb_tokens);
    end = min(max(end, first), c.nb_tokens);
    s.first_row = first;
    s.count = min(end - first, c.max_new);
    s.begin = s.length - s.count;
    return s;
}

static inline int kv_check(const n2d2b_kv_cache* cache, const n2d2b_kv_batch* batch, KvArgs& a)
{
    if (!cache || !batch) return set_error(N2D2B_ERR_INVALID, "cache and batch must not be NULL");
    if (cache->nb_pages < 1 || cache->nb_heads < 1)
        return set_error(N2D2B_ERR_INVALID, "a cache has at least one page and one head (got %d, %d)", cache->nb_pages, cache->nb_heads);
    if (cache->page_tokens != 16 && cache->page_tokens != 32 && cache->page_tokens != 64 && cache->page_tokens != 128)
        return set_error(N2D2B_ERR_INVALID, "page_tokens must be 16, 32, 64 or 128 (got %d)", cache->page_tokens);
    if (cache->head_size != 64 && cache->head_size != 128) return set_error(N2D2B_ERR_INVALID, "head_size must be 64 or 128 (got %d)", cache->head_size);
    if ((long long)cache->nb_pages * cache->nb_heads > 2147483647ll / cache->page_tokens)
        return set_error(N2D2B_ERR_TOO_LARGE, "pages x heads x page_tokens exceeds 2^31 - 1");
    if (!cache->k || !cache->v || !cache->k_scales || !cache->v_scales) return set_error(N2D2B_ERR_INVALID, "the cache's buffers must not be NULL");
    if (!token_aligned(cache->k, 16) || !token_aligned(cache->v, 16) || !token_aligned(cache->k_scales, 4) || !token_aligned(cache->v_scales, 4))
        return set_error(N2D2B_ERR_INVALID, "the cache's codes must start on 16 bytes and its scales on 4");
    if (batch->nb_sequences < 0 || batch->nb_tokens < 0 || batch->max_new < 0 || batch->pages_per_sequence < 1)
        return set_error(N2D2B_ERR_INVALID, "invalid batch: %d sequences, %d tokens, at most %d new, %d pages a sequence", batch->nb_sequences,
                         batch->nb_tokens, batch->max_new, batch->pages_per_sequence);
    if (batch->nb_sequences > 32767) return set_error(N2D2B_ERR_TOO_LARGE, "nb_sequences = %d exceeds 32767", batch->nb_sequences);
    // (kernels count in steps of 128 tokens and look two steps ahead)
    if (batch->pages_per_sequence > (2147483647 - 511) / cache->page_tokens)
        return set_error(N2D2B_ERR_TOO_LARGE, "pages_per_sequence x page_tokens exceeds 2^31 - 512");
    if (batch->nb_sequences > 0 && (!batch->page_table || !batch->lengths)) return set_error(N2D2B_ERR_INVALID, "page_table and lengths must not be NULL");
    if (!token_aligned(batch->page_table, 4) || !token_aligned(batch->lengths, 4) || !token_aligned(batch->starts, 4))
        return set_error(N2D2B_ERR_INVALID, "page_table, lengths and starts must start on 4 bytes");
    a.k = cache->k; a.v = cache->v; a.k_scales = cache->k_scales; a.v_scales = cache->v_scales;
    a.table = batch->page_table; a.lengths = batch->lengths; a.starts = batch->starts;
    a.nb_pages = cache->nb_pages; a.heads = cache->nb_heads; a.row = batch->pages_per_sequence;
    a.nb_tokens = batch->nb_tokens;
    // a bound may be as loose as the caller likes: no sequence has more new tokens than the call has rows, and blocks are launched for no more
    a.max_new = batch->starts ? batch->max_new : (batch->max_new < 1 ? batch->max_new : 1);
    if (a.max_new > batch->nb_tokens) a.max_new = batch->nb_tokens;
    return 0;
}

// ----------------------------------------------------------------------------- attention
struct AttendArgs {
    KvArgs c;
    const void* q;
    void* out;
    long long q_stride, out_stride;
    float scale_log2;      // scale * log2(e)
    int group;             // query heads of a key head
    int causal, window;
    int log_page;
    int* status;
};

// What stands for a scale of zero (up to TOKEN_TINY) of a page's values in the exponents: any number would do, as its codes are zeros.  This one is below the scales that a
// page of ordinary values has beside it, so its probabilities take no bits from theirs, and its reciprocal leaves the softmax's sum in 32 bits room for 2^40 tokens.
static constexpr float KV_NOTHING = 8.271806125530277e-25f;    // 2^-80

// (bytes 0, 1) and (bytes 2, 3) of four codes + 128 as halves 1024 + u
__device__ __forceinline__ unsigned splice(unsigned w, unsigned sel)
{
    unsigned r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(w), "r"(0x64646464u), "r"(sel));
    return r;
}
__device__ __forceinline__ unsigned less_1152(unsigned h)
{
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&h), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const unsigned*>(&d);
}
__device__ __forceinline__ float exp2_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ unsigned pack_half2(float a, float b)
{
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ float ld_cluster(unsigned addr)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_cluster4(unsigned addr)
{
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
// Steps of 128 tokens that a row may see
static inline long long attend_steps(const AttendArgs& a)
{
    const long long capacity = (long long)a.c.row << a.log_page, most = a.window && (long long)a.window + a.c.max_new < capacity ? (long long)a.window + a.c.max_new : capacity;
    return (most + 127) / 128 + (a.window ? 1 : 0);
}
// Streams (blocks of a cluster) that the tokens of a tile are cut into where a block has a multiprocessor to itself: as many as leave no two blocks on
// one, of at least `least` steps each.  Clusters of eight only find room beside one another on about three quarters of the multiprocessors (16
// tiles of 4000 tokens: 23.5 us as 16 clusters of 8, the last of which wait, 17.0 as clusters of 4).
static inline int attend_streams(long long tiles, long long steps, int least, int most)
{
    int streams = 1;
    while (streams < most && tiles * streams * 2 <= (streams == 4 ? token_sms() * 3 / 4 : token_sms()) && streams * 2 * least <= steps) streams *= 2;
    return streams;
}

// Many rows of a key head on the tensor cores (kv_attention_prompt.cu)
cudaError_t launch_attention_prompt(const AttendArgs& a, int head_size, bool half, int sequences, cudaStream_t s);

}  // namespace n2d2b
