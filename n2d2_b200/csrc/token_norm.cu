// Root-mean-square norm with the residual's addition and an output in 8 bits with a scale for each token.
//
//   h = round(x + r)          stored in the inputs' type
//   u = h * w                 32 bits
//   s = max |u| / 127         code = round(u / s), scale = s / sqrt(mean(h^2) + eps), or s alone where no norm is wanted
//
// The factor 1 / sqrt(...) is the same for a whole row, so it cancels out of the codes: they are taken of u, do not depend on the
// order in which the squares are summed, and the row's sum and maximum come out of one pass and one reduction.
//
// Bound by memory: 7 bytes a value with a residual of 16 bits.  8192 rows of 4096 in bf16: 39 us, 5.99 TB/s (91 % of what a copy reaches); 8 rows:
// 2.5 us back to back, the launch, two loads one behind the other and the reduction.  Rows that are not whole vectors of 16 bytes go by an element an access: 8192 of 4095
// 122 us, 2048 of 8191 67.
#include <cstdio>
#include <cstring>
#include "token_common.cuh"

namespace n2d2b {

__device__ int g_token_status;

int* token_status_word()
{
    static std::atomic<int*> known[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return nullptr;
    if (dev >= 0 && dev < 64)
        if (int* p = known[dev].load(std::memory_order_acquire)) return p;
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, g_token_status) != cudaSuccess) return nullptr;
    if (dev >= 0 && dev < 64) known[dev].store((int*)p, std::memory_order_release);
    return (int*)p;
}

int token_sms()
{
    static std::atomic<int> known[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return current_sms();
    int n = known[dev].load(std::memory_order_relaxed);
    if (!n) {
        n = current_sms();
        known[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

bool token_byte_map(CUtensorMap* map, const void* base, unsigned long long columns, unsigned long long rows, unsigned long long pitch,
                    unsigned box_columns, unsigned box_rows, CUtensorMapSwizzle swizzle)
{
    typedef CUresult (*Encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                               const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static std::atomic<void*> entry;
    void* fn = entry.load(std::memory_order_acquire);
    if (!fn) {
        cudaDriverEntryPointQueryResult qr;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qr) != cudaSuccess || !fn) return false;
        entry.store(fn, std::memory_order_release);
    }
    const cuuint64_t dims[2] = {columns, rows}, strides[1] = {pitch};
    const cuuint32_t box[2] = {box_columns, box_rows}, steps[2] = {1, 1};
    return ((Encode)fn)(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct NormArgs {
    const void *x, *residual, *weight;
    void* total;
    int8_t* codes;
    float* scales;
    long long x_stride, residual_stride, total_stride, codes_stride;
    int columns, skip_norm;
    float eps, least;       // least: sums of squares below it have lost some that count beside eps
};

// Sum and maximum over the block; every thread gets both
__device__ __forceinline__ void block_sum_max(float& sum, unsigned& top)
{
    __shared__ float sums[32];
    __shared__ unsigned tops[32];
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    const int warps = (int)blockDim.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) { sums[threadIdx.x >> 5] = sum; tops[threadIdx.x >> 5] = top; }
    __syncthreads();
    sum = lane < warps ? sums[lane] : 0.0f;
    top = lane < warps ? tops[lane] : 0u;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
}

// The scale of a row h whose squares left 32 bits: their sum again, of the row times a power of two; *scale holds the step.  (2^75 keeps the sum below 2^121, as it was
// below 2^-60 times the columns, and the squares of the smallest normal values at 2^-102; 2^-80 keeps 2^31 of the largest squares below 2^127.)  A function of its own and an element at a
// time, for kernels that it takes no registers from: within them 8192 rows of 4096 took 43 to 48 us instead of 39.
template <typename T>
__device__ __noinline__ void scale_again(const T* h, int columns, float by, float eps, float* scale)
{
    float sum = 0.0f;
    unsigned unused = 0;
#pragma unroll 1
    for (int i = threadIdx.x; i < columns; i += blockDim.x) {
        const float v = Elem<T>::to_float(h[i]) * by;
        sum = fmaf(v, v, sum);
    }
    __syncthreads();        // all threads have read what the first reduction left
    block_sum_max(sum, unused);
    if (threadIdx.x == 0) *scale = (float)((double)*scale * by * rsqrtf(sum / (float)columns + eps * by * by));      // (1 / h itself may leave 32 bits)
}

// A block takes a row.  ITER > 0: a thread keeps its ITER vectors of the row in registers; ITER = 0: rows of any length, read a
// second time for their codes.  VEC elements per access: 16 bytes, or one where addresses, strides or the width do not allow that.
// As many threads a multiprocessor as their vectors leave registers for: left to itself the compiler takes a few more, and 2048 rows of 8192 in 32 bits 44 us instead of
// 37, 8192 of 4096 in bf16 41 instead of 39.
template <typename T, int VEC, int ITER>
__global__ void __launch_bounds__(512, ITER < 4 || VEC == 1 ? 4 : VEC == 4 ? 3 : 2) rmsnorm_quantize_kernel(const NormArgs a)
{
    pdl_launch_dependents();
    pdl_wait();
    const long long row = blockIdx.x;
    const T* x = (const T*)a.x + row * a.x_stride;
    const T* r = a.residual ? (const T*)a.residual + row * a.residual_stride : nullptr;
    T* total = a.residual ? (T*)a.total + row * a.total_stride : nullptr;
    const T* w = (const T*)a.weight;
    int8_t* codes = a.codes + row * a.codes_stride;
    const int n = a.columns / VEC;

    auto load = [](const T* p, float* v) {
        if (VEC == 1) v[0] = Elem<T>::to_float(p[0]);
        else Elem<T>::unpack(*reinterpret_cast<const uint4*>(p), v);
    };
    auto sum_of = [&](int i, float* v) {   // h of vector i, stored where a sum is wanted
        load(x + (size_t)i * VEC, v);
        if (r) {
            float add[VEC];
            load(r + (size_t)i * VEC, add);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] += add[e];
            if (VEC == 1) {
                total[i] = Elem<T>::from_float(v[0]);
                v[0] = Elem<T>::to_float(Elem<T>::from_float(v[0]));
            } else {
                const uint4 packed = Elem<T>::pack(v);
                *reinterpret_cast<uint4*>(total + (size_t)i * VEC) = packed;
                Elem<T>::unpack(packed, v);
            }
        }
    };
    auto weigh = [&](int i, float* v, float& sum, float& top) {
        float f[VEC];
        if (w) load(w + (size_t)i * VEC, f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            sum = fmaf(v[e], v[e], sum);
            if (w) v[e] *= f[e];
        }
#pragma unroll
        for (int e = 0; e < VEC; e += 2) top = largest(top, v[e], v[VEC == 1 ? 0 : e + 1]);
    };
    auto store = [&](int i, const float* v, float inverse) {
        if (VEC == 1) codes[i] = (int8_t)code_of(v[0], inverse);
        else if (VEC == 4) *reinterpret_cast<unsigned*>(codes + (size_t)i * 4) = pack_codes(v, inverse);
        else *reinterpret_cast<uint2*>(codes + (size_t)i * 8) = make_uint2(pack_codes(v, inverse), pack_codes(v + 4, inverse));
    };

    float kept[(ITER ? ITER : 1) * VEC], sum = 0.0f;
    float most = 0.0f;
    if (ITER) {
#pragma unroll
        for (int k = 0; k < ITER; ++k) {
            const int i = threadIdx.x + k * blockDim.x;
            if (i < n) sum_of(i, kept + k * VEC);
        }
#pragma unroll
        for (int k = 0; k < ITER; ++k) {
            const int i = threadIdx.x + k * blockDim.x;
            if (i < n) weigh(i, kept + k * VEC, sum, most);
        }
    } else {
        for (int i = threadIdx.x; i < n; i += blockDim.x) {
            sum_of(i, kept);
            weigh(i, kept, sum, most);
        }
    }
    unsigned top = magnitude(most);
    block_sum_max(sum, top);
    float step = __uint_as_float(top) * TOKEN_STEP, inverse = 1.0f / step;
    if (step <= TOKEN_TINY) step = inverse = 0.0f;
    if (top >= 0x7f800000u) step = __int_as_float(0x7fffffff);
    // squares that left 32 bits: values above 2^63 or so, or below 2^-63 with no eps to speak of
    const bool large = step > 0.0f && sum == INFINITY && !a.skip_norm, small = step > 0.0f && sum < a.least;
    if (threadIdx.x == 0) a.scales[row] = step == 0.0f ? 0.0f : large || small || a.skip_norm ? step : step * rsqrtf(sum / (float)a.columns + a.eps);
    if (ITER) {
#pragma unroll
        for (int k = 0; k < ITER; ++k) {
            const int i = threadIdx.x + k * blockDim.x;
            if (i < n) store(i, kept + k * VEC, inverse);
        }
    } else {
        const T* h = total ? total : x;   // its own elements: what this thread stored above
        for (int i = threadIdx.x; i < n; i += blockDim.x) {
            float unused = 0.0f;
            load(h + (size_t)i * VEC, kept);
            weigh(i, kept, unused, most);
            store(i, kept, inverse);
        }
    }
    if (large || small) {
        if (a.residual) __syncthreads();        // (an element's sum may be another thread's)
        scale_again<T>(a.residual ? (const T*)a.total + row * a.total_stride : (const T*)a.x + row * a.x_stride, a.columns, large ? 0x1p-80f : 0x1p75f, a.eps, a.scales + row);
    }
}

template <typename T, int VEC>
static cudaError_t launch_norm(const NormArgs& a, int rows, cudaStream_t s)
{
    const int n = a.columns / VEC;
    // as many warps as the row fills with two vectors a thread
    const int threads = n >= 1024 ? 512 : (n + 63) / 64 * 32;
    const int iter = (n + threads - 1) / threads;
    const dim3 grid((unsigned)rows);
    if (iter <= 1) return launch_token(rmsnorm_quantize_kernel<T, VEC, 1>, grid, threads, 0, 1, s, a);
    if (iter <= 2) return launch_token(rmsnorm_quantize_kernel<T, VEC, 2>, grid, threads, 0, 1, s, a);
    if (iter <= 4) return launch_token(rmsnorm_quantize_kernel<T, VEC, 4>, grid, threads, 0, 1, s, a);
    return launch_token(rmsnorm_quantize_kernel<T, VEC, 0>, grid, threads, 0, 1, s, a);
}

template <typename T>
static cudaError_t launch_norm_of(const NormArgs& a, int rows, cudaStream_t s)
{
    constexpr int VEC = Elem<T>::VEC;
    const bool wide = a.columns % VEC == 0 && a.x_stride % VEC == 0 && token_aligned(a.x, 16) && a.codes_stride % VEC == 0 && token_aligned(a.codes, VEC)
                      && (!a.weight || token_aligned(a.weight, 16))
                      && (!a.residual || (token_aligned(a.residual, 16) && token_aligned(a.total, 16) && a.residual_stride % VEC == 0 && a.total_stride % VEC == 0));
    return wide ? launch_norm<T, VEC>(a, rows, s) : launch_norm<T, 1>(a, rows, s);
}

}  // namespace n2d2b

extern "C" int n2d2b_rmsnorm_quantize(int device, const n2d2b_norm* norm, n2d2b_stream stream)
{
    using namespace n2d2b;
    if (!norm) return set_error(N2D2B_ERR_INVALID, "norm must not be NULL");
    const n2d2b_norm& d = *norm;
    if (d.dtype != N2D2B_F32 && d.dtype != N2D2B_F16 && d.dtype != N2D2B_BF16)
        return set_error(N2D2B_ERR_INVALID, "dtype must be N2D2B_F32, N2D2B_F16 or N2D2B_BF16 (got %d)", d.dtype);
    if (d.rows < 0 || d.columns < 1) return set_error(N2D2B_ERR_INVALID, "invalid size: %d rows of %d columns", d.rows, d.columns);
    if (!(d.eps >= 0.0f)) return set_error(N2D2B_ERR_INVALID, "eps must not be negative");
    if (d.rows == 0) return 0;
    if (!d.x || !d.codes || !d.scales) return set_error(N2D2B_ERR_INVALID, "x, codes and scales must not be NULL");
    if (!d.residual != !d.total) return set_error(N2D2B_ERR_INVALID, "residual and total go together: both or neither");
    const int item = token_item(d.dtype);
    if (!token_aligned(d.x, item) || !token_aligned(d.residual, item) || !token_aligned(d.total, item) || !token_aligned(d.weight, item) || !token_aligned(d.scales, 4))
        return set_error(N2D2B_ERR_INVALID, "buffers must start on a whole element");
    NormArgs a;
    a.x = d.x; a.residual = d.residual; a.weight = d.weight; a.total = d.total; a.codes = d.codes; a.scales = d.scales;
    a.columns = d.columns;
    a.eps = d.eps;
    a.skip_norm = d.skip_norm;
    a.least = d.eps < 0x1p-60f && !d.skip_norm ? (0x1p-60f - d.eps) * (float)d.columns : 0.0f;
    a.x_stride = d.x_stride ? d.x_stride : d.columns;
    a.residual_stride = d.residual_stride ? d.residual_stride : d.columns;
    a.total_stride = d.total_stride ? d.total_stride : d.columns;
    a.codes_stride = d.codes_stride ? d.codes_stride : d.columns;
    if (a.x_stride < d.columns || a.residual_stride < d.columns || a.total_stride < d.columns || a.codes_stride < d.columns)
        return set_error(N2D2B_ERR_INVALID, "strides must be 0 or at least the %d columns of a row", d.columns);
    // (rows that another row's sum overwrites before they are read)
    if (d.total && ((d.total == d.x && a.total_stride != a.x_stride) || (d.total == d.residual && a.total_stride != a.residual_stride)))
        return set_error(N2D2B_ERR_INVALID, "total in the place of x or residual takes the same stride");
    const TokenDevice on(device);
    if (on.err != cudaSuccess) return set_error(N2D2B_ERR_CUDA, "device %d is not usable: %s", device, cudaGetErrorString(on.err));
    cudaError_t e;
    if (d.dtype == N2D2B_F32) e = launch_norm_of<float>(a, d.rows, (cudaStream_t)stream);
    else if (d.dtype == N2D2B_F16) e = launch_norm_of<__half>(a, d.rows, (cudaStream_t)stream);
    else e = launch_norm_of<__nv_bfloat16>(a, d.rows, (cudaStream_t)stream);
    if (e != cudaSuccess) return set_error(N2D2B_ERR_CUDA, "norm kernel launch failed: %s", cudaGetErrorString(e));
    return 0;
}

extern "C" int n2d2b_token_check(int device, n2d2b_stream stream)
{
    using namespace n2d2b;
    const TokenDevice on(device);
    if (on.err != cudaSuccess) return set_error(N2D2B_ERR_CUDA, "device %d is not usable: %s", device, cudaGetErrorString(on.err));
    int* const word = token_status_word();
    if (!word) return set_error(N2D2B_ERR_CUDA, "the status word of the token operators has no address on device %d", device);
    cudaStream_t s = (cudaStream_t)stream;
    int status = 0;
    cudaError_t e = cudaMemcpyAsync(&status, word, sizeof(int), cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e == cudaSuccess && status) e = cudaMemsetAsync(word, 0, sizeof(int), s);
    if (e == cudaSuccess && status) e = cudaStreamSynchronize(s);
    if (e != cudaSuccess) return set_error(N2D2B_ERR_CUDA, "the stream failed: %s", cudaGetErrorString(e));
    if (status) return set_error(N2D2B_ERR_TIMEOUT, "a kernel gave up waiting on a pipeline barrier (role %d); its output is incomplete", status);
    return 0;
}

extern "C" int n2d2b_token_selftest_wait_timeout(int device, unsigned limit_us, n2d2b_stream stream)
{
    using namespace n2d2b;
    const TokenDevice on(device);
    if (on.err != cudaSuccess) return set_error(N2D2B_ERR_CUDA, "device %d is not usable: %s", device, cudaGetErrorString(on.err));
    int* const word = token_status_word();
    if (!word) return set_error(N2D2B_ERR_CUDA, "the status word of the token operators has no address on device %d", device);
    return wait_timeout_selftest(word, limit_us, (cudaStream_t)stream);
}
