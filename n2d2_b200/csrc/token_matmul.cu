// Matrix product of 8-bit codes with scales for each token and each output channel.
//
//   out[i][j] = (sum_k a[i][k] w[j][k]) * sa[i] * sw[j] + bias[j]
//
// The sums are exact in 32 bits, so any split of k gives the same bits.
#include <cstdio>
#include <cstring>
#include "token_common.cuh"

namespace n2d2b {

struct MatmulArgs {
    const int8_t *a, *w;
    const float *a_scales, *w_scales, *bias;
    void* out;
    long long a_stride, w_stride, out_stride;
    int M, N, K;
};

template <typename T>
__device__ __forceinline__ void store_scaled(const MatmulArgs& p, int i, int j, int acc, float sa, float sw, float bias)
{
    float v = (float)acc * sa * sw;
    if (p.bias) v += bias;
    ((T*)p.out)[(size_t)i * p.out_stride + j] = Elem<T>::from_float(v);
}

// Rows of any address and stride: 64 x 64 outputs a block, 4 x 4 a thread, 64 bytes of k a step through shared memory.
template <typename T>
__global__ void __launch_bounds__(256) matmul_i8_any_kernel(const MatmulArgs p)
{
    pdl_launch_dependents();
    pdl_wait();
    constexpr int PITCH = 17;   // words of a row: 16 and one against bank conflicts
    __shared__ int as[64 * PITCH], ws[64 * PITCH];
    const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < p.K; k0 += 64) {
        for (int i = threadIdx.x; i < 2 * 64 * 64; i += 256) {
            const int which = i >> 12, row = (i >> 6) & 63, k = k0 + (i & 63);
            const int g = which ? n0 + row : m0 + row;
            int8_t v = 0;
            if (k < p.K && g < (which ? p.N : p.M)) v = which ? p.w[(size_t)g * p.w_stride + k] : p.a[(size_t)g * p.a_stride + k];
            ((int8_t*)((which ? ws : as) + row * PITCH))[i & 63] = v;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            int av[4], wv[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) { av[e] = as[(ty + 16 * e) * PITCH + k]; wv[e] = ws[(tx + 16 * e) * PITCH + k]; }
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int f = 0; f < 4; ++f) acc[e][f] = __dp4a(av[e], wv[f], acc[e][f]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int f = 0; f < 4; ++f) {
        const int j = n0 + tx + 16 * f;
        if (j >= p.N) continue;
        const float sw = p.w_scales[j], bias = p.bias ? p.bias[j] : 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = m0 + ty + 16 * e;
            if (i < p.M) store_scaled<T>(p, i, j, acc[e][f], p.a_scales[i], sw, bias);
        }
    }
}

template <typename T>
static cudaError_t launch_matmul(const MatmulArgs& p, cudaStream_t s)
{
    const dim3 grid((unsigned)((p.N + 63) / 64), (unsigned)((p.M + 63) / 64));
    return launch_token(matmul_i8_any_kernel<T>, grid, 256, 0, 1, s, p);
}

}  // namespace n2d2b

extern "C" int n2d2b_matmul_i8(int device, const n2d2b_matmul* matmul, n2d2b_stream stream)
{
    using namespace n2d2b;
    if (!matmul) return set_error(N2D2B_ERR_INVALID, "matmul must not be NULL");
    const n2d2b_matmul& d = *matmul;
    if (d.dtype != N2D2B_F32 && d.dtype != N2D2B_F16 && d.dtype != N2D2B_BF16)
        return set_error(N2D2B_ERR_INVALID, "dtype must be N2D2B_F32, N2D2B_F16 or N2D2B_BF16 (got %d)", d.dtype);
    if (d.m < 0 || d.n < 1 || d.k < 1) return set_error(N2D2B_ERR_INVALID, "invalid size: %d x %d x %d", d.m, d.n, d.k);
    if (d.k > 131071) return set_error(N2D2B_ERR_TOO_LARGE, "k = %d exceeds 131071, beyond which sums could leave 32 bits", d.k);
    if (d.m > 65535 * 64) return set_error(N2D2B_ERR_TOO_LARGE, "m = %d exceeds %d", d.m, 65535 * 64);
    if (d.m == 0) return 0;
    if (!d.a || !d.a_scales || !d.w || !d.w_scales || !d.out) return set_error(N2D2B_ERR_INVALID, "a, w, their scales and out must not be NULL");
    if (!token_aligned(d.out, token_item(d.dtype)) || !token_aligned(d.a_scales, 4) || !token_aligned(d.w_scales, 4) || !token_aligned(d.bias, 4))
        return set_error(N2D2B_ERR_INVALID, "buffers must start on a whole element");
    MatmulArgs p;
    p.a = d.a; p.w = d.w; p.a_scales = d.a_scales; p.w_scales = d.w_scales; p.bias = d.bias; p.out = d.out;
    p.M = d.m; p.N = d.n; p.K = d.k;
    p.a_stride = d.a_stride ? d.a_stride : d.k;
    p.w_stride = d.w_stride ? d.w_stride : d.k;
    p.out_stride = d.out_stride ? d.out_stride : d.n;
    if (p.a_stride < d.k || p.w_stride < d.k || p.out_stride < d.n)
        return set_error(N2D2B_ERR_INVALID, "strides must be 0 or at least a row (k = %d for a and w, n = %d for out)", d.k, d.n);
    const TokenDevice on(device);
    if (on.err != cudaSuccess) return set_error(N2D2B_ERR_CUDA, "device %d is not usable: %s", device, cudaGetErrorString(on.err));
    cudaError_t e;
    if (d.dtype == N2D2B_F32) e = launch_matmul<float>(p, (cudaStream_t)stream);
    else if (d.dtype == N2D2B_F16) e = launch_matmul<__half>(p, (cudaStream_t)stream);
    else e = launch_matmul<__nv_bfloat16>(p, (cudaStream_t)stream);
    if (e != cudaSuccess) return set_error(N2D2B_ERR_CUDA, "matrix product launch failed: %s", cudaGetErrorString(e));
    return 0;
}
