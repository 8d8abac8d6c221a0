// What the token operators (norm, matrix product, cache, attention of layers served in 8-bit integers) share: element
// types, the argument checks of their entry points, the status word of their bounded waits, launches.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include "../../include/n2d2b.h"
#include "host_internal.h"
#include "tc_common.cuh"

namespace n2d2b {

// A scale up to this counts as zero, as do the codes under it: the reciprocals of smaller ones leave 32 bits
static constexpr float TOKEN_TINY = 7.888609052210118e-31f;   // 2^-100
static constexpr float TOKEN_STEP = (float)(1.0 / 127.0);

// Makes `device` the current one and puts the caller's back; a call on the current device changes nothing
struct TokenDevice {
    int prev = -1;
    cudaError_t err;
    explicit TokenDevice(int device)
    {
        int now = -1;
        err = cudaGetDevice(&now);
        if (err == cudaSuccess && now != device) {
            err = cudaSetDevice(device);
            if (err == cudaSuccess) prev = now;
        }
    }
    ~TokenDevice() { if (prev >= 0) cudaSetDevice(prev); }
    TokenDevice(const TokenDevice&) = delete;
    TokenDevice& operator=(const TokenDevice&) = delete;
};

// The status word of these operators' bounded waits on the current device (token_norm.cu), or nullptr
int* token_status_word();
// Multiprocessors of the current device, asked for once
int token_sms();
// cuTensorMapEncodeTiled for a matrix of bytes: `rows` rows of `columns` bytes, `pitch` bytes apart
bool token_byte_map(CUtensorMap* map, const void* base, unsigned long long columns, unsigned long long rows, unsigned long long pitch,
                    unsigned box_columns, unsigned box_rows, CUtensorMapSwizzle swizzle);

static inline int token_item(int dtype) { return dtype == N2D2B_F32 ? 4 : 2; }
static inline bool token_aligned(const void* p, unsigned n) { return ((uintptr_t)p & (n - 1u)) == 0; }

// Kernel launch as a programmatic dependent of the kernel before it (see launch_pdl), with a cluster along x when cluster > 1
template <typename... P, typename... A>
static inline cudaError_t launch_token(void (*kernel)(P...), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t s, A&&... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

// ----------------------------------------------------------------------------- clusters
// TMEM is handed out at run time, and a block that waits for its share while blocks that hold theirs wait for it would wait for ever.  Four rules keep that from happening,
// the first two also those of a network's kernels, which may run beside these on another stream: a block lets the next kernel start only when it has its columns, so
// none that starts early takes what the kernel before it still needs; it gives them back before it waits for another block of its cluster, so that whoever holds columns needs nobody
// else's to finish (blocks of a pair, which share theirs, have a multiprocessor each); it asks for at least this much shared memory for each column (the multiprocessor's
// 228 KB over 512 columns, rounded up), so blocks of these kernels that share a multiprocessor never wait for one another; and it allocates behind griddepcontrol.wait.
static constexpr int TMEM_BYTES = 460;
__device__ __forceinline__ unsigned cluster_rank()
{
    unsigned r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ unsigned cluster_size()
{
    unsigned r;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ unsigned map_to_rank(unsigned addr, unsigned rank)
{
    unsigned r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}

// ----------------------------------------------------------------------------- element types
template <typename T> struct Elem;
template <> struct Elem<float> {
    static constexpr int VEC = 4;    // elements of a 16-byte access
    static __device__ __forceinline__ float to_float(float v) { return v; }
    static __device__ __forceinline__ float from_float(float v) { return v; }
    static __device__ __forceinline__ void unpack(const uint4& w, float* v)
    {
        v[0] = __uint_as_float(w.x); v[1] = __uint_as_float(w.y); v[2] = __uint_as_float(w.z); v[3] = __uint_as_float(w.w);
    }
    static __device__ __forceinline__ uint4 pack(const float* v)
    {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
};
template <> struct Elem<__half> {
    static constexpr int VEC = 8;
    static __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
    static __device__ __forceinline__ unsigned pack2(float a, float b)
    {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const unsigned*>(&h);
    }
    static __device__ __forceinline__ float2 unpack2(unsigned w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
    static __device__ __forceinline__ void unpack(const uint4& w, float* v)
    {
        const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { const float2 f = unpack2(u[i]); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
    }
    static __device__ __forceinline__ uint4 pack(const float* v)
    {
        return make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7]));
    }
};
template <> struct Elem<__nv_bfloat16> {
    static constexpr int VEC = 8;
    static __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
    static __device__ __forceinline__ unsigned pack2(float a, float b)
    {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const unsigned*>(&h);
    }
    static __device__ __forceinline__ float2 unpack2(unsigned w)
    {
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
    static __device__ __forceinline__ void unpack(const uint4& w, float* v)
    {
        const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { const float2 f = unpack2(u[i]); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
    }
    static __device__ __forceinline__ uint4 pack(const float* v)
    {
        return make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7]));
    }
};

// Nearest whole number (ties to even) of a value within the codes' range, in the lowest byte: the sum with 1.5 * 2^23 rounds it there.  The product with the
// reciprocal is rounded by itself first, as the codes' definition has it.  What is no number gets some code; its scale says what it is.
__device__ __forceinline__ unsigned code_of(float v, float inverse) { return __float_as_uint(__fadd_rn(__fmul_rn(v, inverse), 12582912.0f)); }
__device__ __forceinline__ unsigned pack_codes(const float* v, float inverse)
{
    const unsigned ab = __byte_perm(code_of(v[0], inverse), code_of(v[1], inverse), 0x0040), cd = __byte_perm(code_of(v[2], inverse), code_of(v[3], inverse), 0x0040);
    return __byte_perm(ab, cd, 0x5410);
}

// Magnitudes as whole numbers: their order is that of the values, with what is no number above everything, so a maximum keeps it
__device__ __forceinline__ unsigned magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// Largest magnitude, which stays no number once it is
__device__ __forceinline__ float largest(float top, float a, float b)
{
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(top), "f"(fabsf(a)), "f"(fabsf(b)));
    return d;
}

}  // namespace n2d2b
