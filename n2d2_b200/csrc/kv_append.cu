// New keys and values into the paged 8-bit cache.
//
// For a page and head that gains tokens: s' = max(s, max|new| / 127), old codes round(q * (s / s')), new codes round(x * (1 / s')).
// A block takes one page of one head, of the keys or of the values, and is the only one to touch its codes and scale; the new
// values stay in registers between the maximum and the rounding.
//
// Four prompts of up to 4000 tokens (8 heads of 128, keys and values): 15 us, 2.7 TB/s; bound by the short life of its 4000 blocks, each a chain of lengths, page
// number, values, reduction and store.  One token to each of 64 sequences: 5 us back to back, that chain once, and the codes of a page rescaled where its scale
// grows.  A block for several pages would have fewer of these chains, but no page of a decoding step has a neighbour to share one with.
#include <cstdio>
#include <cstring>
#include "kv_common.cuh"

namespace n2d2b {

template <typename T, int D>
__global__ void __launch_bounds__(256) kv_append_kernel(const KvArgs c, const T* new_k, const T* new_v, long long stride, int page)
{
    pdl_launch_dependents();
    pdl_wait();
    constexpr int PER = D / 8;          // 16-byte vectors of a token
    constexpr int KEEP = 128 * PER / 256;
    __shared__ unsigned tops[8];
    const int b = blockIdx.z >> 1, head = blockIdx.y, values = blockIdx.z & 1;
    const KvSequence s = kv_sequence(c, b);
    const int begin = max(s.begin, 0);
    const int p = begin / page + (int)blockIdx.x;
    // (page numbers are compared before they are multiplied: p * page stays below 2^31 for the pages of a row)
    if (s.count < 1 || p >= c.row) return;
    const int lo = max(begin, p * page), hi = min(s.length, (p + 1) * page);
    if (lo >= hi) return;
    const int number = c.table[(size_t)b * c.row + p];
    if (number < 0 || number >= c.nb_pages) return;
    const T* x = (values ? new_v : new_k) + (size_t)(s.first_row + (lo - s.begin)) * stride + (size_t)head * D;
    float* const scale = (values ? c.v_scales : c.k_scales) + (size_t)number * c.heads + head;
    int8_t* const codes = (values ? c.v : c.k) + ((size_t)number * c.heads + head) * page * D;

    const int n = (hi - lo) * PER;
    uint4 kept[KEEP];
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
        const int at = threadIdx.x + i * 256;
        if (at < n) kept[i] = *reinterpret_cast<const uint4*>(x + (size_t)(at / PER) * stride + (at % PER) * 8);
    }
    // (a scale that counts as zero is 0 here: the reciprocals of such leave 32 bits)
    const float held = lo > p * page ? *scale : 0.0f, before = held <= TOKEN_TINY ? 0.0f : held;
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
        const int at = threadIdx.x + i * 256;
        if (at < n) {
            float v[8];
            Elem<T>::unpack(kept[i], v);
#pragma unroll
            for (int e = 0; e < 8; e += 2) most = largest(most, v[e], v[e + 1]);
        }
    }
    unsigned top = __reduce_max_sync(0xffffffffu, magnitude(most));
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, tops[i]);

    float step = __uint_as_float(top) * TOKEN_STEP;
    if (step <= TOKEN_TINY) step = 0.0f;
    if (top >= 0x7f800000u) step = __int_as_float(0x7fffffff);
    const float after = (before >= step || before != before) ? before : step;
    const float inverse = after > 0.0f ? 1.0f / after : 0.0f;
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
        const int at = threadIdx.x + i * 256;
        if (at < n) {
            float v[8];
            Elem<T>::unpack(kept[i], v);
            *reinterpret_cast<uint2*>(codes + (size_t)(lo - p * page) * D + (size_t)at * 8) = make_uint2(pack_codes(v, inverse), pack_codes(v + 4, inverse));
        }
    }
    if (lo > p * page && after != held) {
        const float ratio = after > 0.0f ? before / after : 0.0f;
        const int old = (lo - p * page) * D / 4;
        for (int i = threadIdx.x; i < old; i += 256) {
            unsigned* const w = reinterpret_cast<unsigned*>(codes) + i;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (float)(int8_t)(*w >> (8 * e));
            *w = pack_codes(v, ratio);
        }
    }
    if (threadIdx.x == 0) *scale = after;
}

template <typename T>
static cudaError_t launch_append(const KvArgs& c, const void* k, const void* v, long long stride, int page, int head_size, int sequences, cudaStream_t s)
{
    // new tokens of a sequence lie in at most this many pages, none behind its row of the table
    const long long pages = ((long long)c.max_new + page - 2) / page + 1;
    const dim3 grid((unsigned)(pages < c.row ? pages : c.row), (unsigned)c.heads, (unsigned)(2 * sequences));
    if (head_size == 64) return launch_token(kv_append_kernel<T, 64>, grid, 256, 0, 1, s, c, (const T*)k, (const T*)v, stride, page);
    return launch_token(kv_append_kernel<T, 128>, grid, 256, 0, 1, s, c, (const T*)k, (const T*)v, stride, page);
}

}  // namespace n2d2b

extern "C" int n2d2b_kv_append(int device, const n2d2b_kv_cache* cache, const n2d2b_kv_batch* batch, const void* k, const void* v, int dtype, int64_t stride,
                               n2d2b_stream stream)
{
    using namespace n2d2b;
    KvArgs c;
    if (int rc = kv_check(cache, batch, c)) return rc;
    if (dtype != N2D2B_F16 && dtype != N2D2B_BF16) return set_error(N2D2B_ERR_INVALID, "dtype must be N2D2B_F16 or N2D2B_BF16 (got %d)", dtype);
    if (batch->nb_sequences == 0 || batch->nb_tokens == 0 || c.max_new == 0) return 0;
    if (!k || !v) return set_error(N2D2B_ERR_INVALID, "k and v must not be NULL");
    const int64_t width = (int64_t)cache->nb_heads * cache->head_size;
    if (stride == 0) stride = width;
    if (stride < width || stride % 8) return set_error(N2D2B_ERR_INVALID, "stride must be 0 or a multiple of 8 of at least %lld", (long long)width);
    if (!token_aligned(k, 16) || !token_aligned(v, 16)) return set_error(N2D2B_ERR_INVALID, "k and v must start on 16 bytes");
    if (cache->nb_heads > 65535) return set_error(N2D2B_ERR_TOO_LARGE, "nb_heads = %d exceeds 65535", cache->nb_heads);
    const TokenDevice on(device);
    if (on.err != cudaSuccess) return set_error(N2D2B_ERR_CUDA, "device %d is not usable: %s", device, cudaGetErrorString(on.err));
    cudaError_t e;
    if (dtype == N2D2B_F16) e = launch_append<__half>(c, k, v, stride, cache->page_tokens, cache->head_size, batch->nb_sequences, (cudaStream_t)stream);
    else e = launch_append<__nv_bfloat16>(c, k, v, stride, cache->page_tokens, cache->head_size, batch->nb_sequences, (cudaStream_t)stream);
    if (e != cudaSuccess) return set_error(N2D2B_ERR_CUDA, "append launch failed: %s", cudaGetErrorString(e));
    return 0;
}
