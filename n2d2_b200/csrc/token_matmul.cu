// Matrix product of 8-bit codes with scales for each token and each output channel.
//
//   out[i][j] = (sum_k a[i][k] w[j][k]) * sa[i] * sw[j] + bias[j]
//
// The sums are exact in 32 bits, so any split of k gives the same bits.
//
// Few tokens are bound by bringing the weights (us a call of many, weights in L2 / in memory: 1 x 4096 x 4096 4.8 / 6.6, 48 x 6144 x 4096 9.1 / 10.4), many by
// the tensor pipe: 4096 x 4096 x 4096 57 us (2.4 POP/s with the clock that the power limit leaves; 48 to 54 in bursts of a few ms; 79 % of the pipe's cycles).
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

// ----------------------------------------------------------------------------- tensor cores
// Weights are the M operand of the MMAs (128 output channels to 128 TMEM lanes), tokens the N operand: a thread of the epilogue owns one output
// channel (its scale and bias sit in registers), a warp stores 32 neighbouring channels of a token at a time, and a call of
// few tokens has narrow tiles instead of empty rows.  A step of the ring is 128 bytes of k of every row, swizzled by TMA; rows and
// bytes beyond the matrices read as zero.
static constexpr int MM_K = 128, TILE_RING = 200 * 1024;

// Scales, bias and store of `left` columns (tokens, at most 32) of a warp's 32 lanes (channels)
template <typename T>
__device__ __forceinline__ void store_columns(const MatmulArgs& p, const unsigned* acc, const float* sa, int token, int left, int channel, float sw, float bias)
{
    T* out = (T*)p.out + (size_t)token * p.out_stride + channel;
    const bool there = channel < p.N;
    // eight at a time: their arithmetic first, then their stores (a value and its store in turn took 60 cycles a column, this takes 25; all 32 at
    // once no less, and their registers keep other blocks off the multiprocessor)
#pragma unroll
    for (int c = 0; c < 32; c += 8) {
        T v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = Elem<T>::from_float(fmaf((float)(int)acc[c + e] * sa[c + e], sw, bias));
        if (there && c + 8 <= left) {
#pragma unroll
            for (int e = 0; e < 8; ++e) out[(long long)e * p.out_stride] = v[e];
        } else if (there) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c + e < left) out[(long long)e * p.out_stride] = v[e];
        }
        out += 8 * p.out_stride;
    }
}

// 16 bytes of k of a row that starts anywhere, zero from byte `valid` on: aligned words that hold a wanted byte (none of `valid` 0, wherever p
// points), shifted into place
__device__ __forceinline__ uint4 load_bytes(const int8_t* p, int valid)
{
    const unsigned shift = (unsigned)((uintptr_t)p & 3u);
    const unsigned* const w = reinterpret_cast<const unsigned*>((uintptr_t)p - shift);
    unsigned x[5], r[4];
#pragma unroll
    for (int i = 0; i < 5; ++i) x[i] = valid > 0 && 4 * i < (int)shift + valid ? w[i] : 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r[i] = __funnelshift_r(x[i], x[i + 1], 8u * shift);
        const int left = valid - 4 * i;
        r[i] = left >= 4 ? r[i] : (left <= 0 ? 0u : r[i] & (0xffffffffu >> (32 - 8 * left)));
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}

// One tile of 128 channels x BN tokens a block.  Few tiles: the blocks of a cluster take parts of k and add their 32-bit sums up through
// distributed shared memory, each finishing a share of the tile.  Warp 0 loads, warp 1 issues the MMAs, four warps store.  BYTES: rows that TMA cannot read (not on 16
// bytes); twelve warps, the storing ones among them, bring them through registers first: 64 bytes a thread are under way at a time (with four warps
// 1156 x 1024 x 3277 took 112 us, with twelve 47, both with the operands in L2; 68 from memory).
template <bool BYTES> struct TileWarps { static constexpr int BRINGING = BYTES ? 12 : 4, THREADS = 64 + 32 * BRINGING; };
template <typename T, int BN, bool BYTES>
__global__ void __launch_bounds__(TileWarps<BYTES>::THREADS, 1) matmul_i8_tile_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap a_map, const MatmulArgs p,
                                                                int stages, int* status)
{
    constexpr int STAGE = (128 + BN) * MM_K, COLUMNS = BN < 32 ? 32 : BN;
    unsigned char* const smem = (unsigned char*)(((uintptr_t)dyn_smem() + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) unsigned long long full[12], empty[12], done;
    __shared__ unsigned tmem_slot;
    __shared__ int abort_flag;
    __shared__ float sa[COLUMNS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        if (!BYTES) { prefetch_tensor_map(&w_map); prefetch_tensor_map(&a_map); }
        for (int i = 0; i < stages; ++i) { mbar_init(smem_u32(&full[i]), BYTES ? TileWarps<BYTES>::BRINGING : 1); mbar_init(smem_u32(&empty[i]), 1); }
        mbar_init(smem_u32(&done), 1);
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        pdl_wait();         // (see TMEM_BYTES)
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"((unsigned)COLUMNS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = tmem_slot;
    pdl_launch_dependents();
    pdl_wait();

    const unsigned rank = cluster_rank(), ranks = cluster_size();
    const int n0 = blockIdx.y * 128, t0 = blockIdx.z * BN;
    const int blocks = (p.K + MM_K - 1) / MM_K, per = (blocks + (int)ranks - 1) / (int)ranks;
    const int from = (int)rank * per, count = max(0, min(per, blocks - from));
    if (warp == 0) {
        for (int i = 0; !BYTES && i < count; ++i) {
            const int slot = i % stages;
            if (i >= stages && !mbar_wait_issuer(smem_u32(&empty[slot]), (unsigned)(i / stages - 1) & 1u, &abort_flag, status, 31)) break;
            if (elect_one()) {
                const unsigned bar = smem_u32(&full[slot]), dst = smem_u32(smem) + (unsigned)(slot * STAGE);
                mbar_expect_tx(bar, STAGE);
                tma_load_2d(dst, &w_map, bar, (from + i) * MM_K, n0);
                tma_load_2d(dst + 128 * MM_K, &a_map, bar, (from + i) * MM_K, t0);
            }
            __syncwarp();
        }
    } else if (warp == 1) {
        const unsigned idesc = (2u << 4) | (1u << 7) | (1u << 10) | (((unsigned)BN >> 3) << 17) | ((128u >> 4) << 24);
        const unsigned hi = (unsigned)(make_smem_desc(0u, 128) >> 32);
        bool ok = true;
        for (int i = 0; i < count && ok; ++i) {
            const int slot = i % stages;
            ok = mbar_wait_issuer(smem_u32(&full[slot]), (unsigned)(i / stages) & 1u, &abort_flag, status, 32);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
                const unsigned w = ((smem_u32(smem) + (unsigned)(slot * STAGE)) & 0x3ffffu) >> 4, a = w + 128 * MM_K / 16;
#pragma unroll
                for (int k = 0; k < MM_K / 32; ++k) tc_mma_i8_lohi(tmem, w + 2 * k, a + 2 * k, hi, idesc, i > 0 || k > 0);
                tc_commit(smem_u32(&empty[slot]));
                if (i == count - 1) tc_commit(smem_u32(&done));
            }
            __syncwarp();
        }
    } else {
        constexpr int BRINGING = 32 * TileWarps<BYTES>::BRINGING;
        for (int i = (int)threadIdx.x - 64; i < BN; i += BRINGING) sa[i] = t0 + i < p.M ? p.a_scales[t0 + i] : 0.0f;
        const int tid = (int)threadIdx.x - 64, chunk = tid & 7;
        for (int i = 0; BYTES && i < count; ++i) {
            const int slot = i % stages, k = (from + i) * MM_K + chunk * 16, valid = min(max(p.K - k, 0), 16);
            if (i >= stages && !mbar_wait_warp(smem_u32(&empty[slot]), (unsigned)(i / stages - 1) & 1u, &abort_flag, status, 31)) break;
            const unsigned dst = smem_u32(smem) + (unsigned)(slot * STAGE);
            // rows tid / 8, + BRINGING / 8, ...: four at a time, so that their loads are under way together
#pragma unroll 1
            for (int r0 = tid >> 3; r0 < 128 + BN; r0 += BRINGING / 2) {
                uint4 v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = r0 + BRINGING / 8 * e, row = r < 128 ? n0 + r : t0 + r - 128;
                    const bool there = r < 128 + BN && row < (r < 128 ? p.N : p.M);
                    const int8_t* const at = r < 128 ? p.w + (size_t)row * p.w_stride + k : p.a + (size_t)row * p.a_stride + k;
                    v[e] = load_bytes(at, there ? valid : 0);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = r0 + BRINGING / 8 * e;
                    if (r < 128 + BN)
                        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst + (unsigned)(r * MM_K + ((chunk ^ (r & 7)) << 4))), "r"(v[e].x), "r"(v[e].y),
                                     "r"(v[e].z), "r"(v[e].w) : "memory");
                }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&full[slot]));
        }
    }
    __syncthreads();
    const bool ok = count == 0 || mbar_wait_warp(smem_u32(&done), 0, &abort_flag, status, 33);
    tc_fence_after();
    if (!ok) __nanosleep(1000000);      // copies under way land before the block leaves
    // the ring is free: every MMA has read its operands
    int* const part = (int*)smem;       // [token][128 channels]
    if (warp >= 2 && warp < 6) {
        const int quad = warp & 3, channel = quad * 32 + lane;
        const float sw = ranks == 1 && n0 + channel < p.N ? p.w_scales[n0 + channel] : 0.0f;
        const float bias = ranks == 1 && p.bias && n0 + channel < p.N ? p.bias[n0 + channel] : 0.0f;
#pragma unroll 1
        for (int c = 0; c < BN; c += 32) {
            unsigned acc[32];
            tc_ld32(tmem + ((unsigned)(quad * 32) << 16) + (unsigned)c, acc);
            tc_wait_ld_into(acc);
            if (ranks == 1) {
                if (ok) store_columns<T>(p, acc, sa + c, t0 + c, min(BN - c, p.M - t0 - c), n0 + channel, sw, bias);
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (c + i < BN) part[(c + i) * 128 + channel] = count ? (int)acc[i] : 0;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {        // before the other blocks are waited for (see TMEM_BYTES)
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((unsigned)COLUMNS) : "memory");
    }
    if (ranks > 1) {
        cluster_sync();
        const int columns = min(BN, p.M - t0);
        for (int i = (int)(rank * blockDim.x + threadIdx.x); i < columns * 32; i += (int)(ranks * blockDim.x)) {
            const int c = i >> 5, channel = n0 + (i & 31) * 4;
            int4 sum = make_int4(0, 0, 0, 0);
            const unsigned at = smem_u32(part + i * 4);
            for (unsigned r = 0; r < ranks; ++r) {
                int4 v;
                asm volatile("ld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(map_to_rank(at, r)) : "memory");
                sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
            }
            const int s[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (channel + e < p.N)
                    ((T*)p.out)[(size_t)(t0 + c) * p.out_stride + channel + e] =
                        Elem<T>::from_float(fmaf((float)s[e] * sa[c], p.w_scales[channel + e], p.bias ? p.bias[channel + e] : 0.0f));
        }
        cluster_sync();     // no block leaves while another reads its sums
    }
}

// ---- pairs of blocks on tiles of 256 x 256
__device__ __forceinline__ void tma_load_2d_pair(unsigned dst, const CUtensorMap* tm, unsigned bar, int x, int y)
{
    // the barrier is the even block's of the pair, whichever block loads (bit 24 of a cluster address tells the two apart)
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(dst), "l"(tm), "r"(bar & 0xfeffffffu), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void tc_mma_i8_pair(unsigned d_tmem, unsigned a_lo, unsigned b_lo, unsigned desc_hi, unsigned idesc, unsigned accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %3};\n\t"
        "mov.b64 db, {%2, %3};\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], da, db, %4, p;\n\t}"
        ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(desc_hi), "r"(idesc), "r"(accumulate) : "memory");
}
// arrives at the barrier of that address in both blocks of the pair
__device__ __forceinline__ void tc_commit_pair(unsigned bar)
{
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((unsigned short)3) : "memory");
}
__device__ __forceinline__ void mbar_arrive_even(unsigned bar)
{
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(map_to_rank(bar, 0)) : "memory");
}

static constexpr int PAIR_STAGES = 6, PAIR_STAGE = 256 * MM_K, PAIR_THREADS = 320;
// all of TMEM, so all of the shared memory (see TMEM_BYTES)
static constexpr int PAIR_SMEM = 227 * 1024 - 1024;
static_assert(PAIR_STAGES * PAIR_STAGE + 1024 <= PAIR_SMEM, "the ring fits");

// Persistent: a pair of blocks (one cta_group::2) walks over tiles of 256 channels x 256 tokens.  Each block holds its 128 channels and
// half of the tokens of a step, so a byte is brought to a multiprocessor for twice the products of a single block's tile of 128 x 256; two
// accumulators: the eight storing warps drain one while the next tile's MMAs fill the other.
template <typename T>
__global__ void __launch_bounds__(PAIR_THREADS, 1) matmul_i8_pair_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap a_map,
                                                                         const MatmulArgs p, int tiles_n, int tiles, int* status)
{
    unsigned char* const smem = (unsigned char*)(((uintptr_t)dyn_smem() + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) unsigned long long full[PAIR_STAGES], empty[PAIR_STAGES], tfull[2], tempty[2];
    __shared__ unsigned tmem_slot;
    __shared__ int abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned rank = cluster_rank();
    if (threadIdx.x == 0) {
        prefetch_tensor_map(&w_map);
        prefetch_tensor_map(&a_map);
        for (int i = 0; i < PAIR_STAGES; ++i) { mbar_init(smem_u32(&full[i]), 1); mbar_init(smem_u32(&empty[i]), 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(smem_u32(&tfull[i]), 1); mbar_init(smem_u32(&tempty[i]), 16); }
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        pdl_wait();
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const unsigned tmem = tmem_slot;
    pdl_launch_dependents();
    pdl_wait();

    const int blocks = (p.K + MM_K - 1) / MM_K;
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const int mine = pair < tiles ? (tiles - pair + pairs - 1) / pairs : 0;
    if (warp == 0) {
        bool ok = true;
        int i = 0;
        for (int t = 0; t < mine && ok; ++t) {
            const int tile = pair + t * pairs, y_w = tile % tiles_n * 256 + (int)rank * 128, y_a = tile / tiles_n * 256 + (int)rank * 128;
            for (int k = 0; k < blocks; ++k, ++i) {
                const int slot = i % PAIR_STAGES;
                if (i >= PAIR_STAGES && !mbar_wait_issuer(smem_u32(&empty[slot]), (unsigned)(i / PAIR_STAGES - 1) & 1u, &abort_flag, status, 34)) { ok = false; break; }
                if (elect_one()) {
                    const unsigned bar = smem_u32(&full[slot]), dst = smem_u32(smem) + (unsigned)(slot * PAIR_STAGE);
                    if (rank == 0) mbar_expect_tx(bar, 2 * PAIR_STAGE);
                    tma_load_2d_pair(dst, &w_map, bar, k * MM_K, y_w);
                    tma_load_2d_pair(dst + 128 * MM_K, &a_map, bar, k * MM_K, y_a);
                }
                __syncwarp();
            }
        }
        if (!ok) __nanosleep(1000000);      // copies under way land before the block leaves
    } else if (warp == 1 && rank == 0) {
        const unsigned idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((256u >> 3) << 17) | ((256u >> 4) << 24);
        const unsigned hi = (unsigned)(make_smem_desc(0u, 128) >> 32);
        bool ok = true;
        int i = 0;
        for (int t = 0; t < mine && ok; ++t) {
            const unsigned d = tmem + (unsigned)((t & 1) * 256);
            if (t >= 2 && !mbar_wait_issuer(smem_u32(&tempty[t & 1]), (unsigned)(t / 2 - 1) & 1u, &abort_flag, status, 35)) break;
            tc_fence_after();
            for (int k = 0; k < blocks; ++k, ++i) {
                const int slot = i % PAIR_STAGES;
                if (!mbar_wait_issuer(smem_u32(&full[slot]), (unsigned)(i / PAIR_STAGES) & 1u, &abort_flag, status, 36)) { ok = false; break; }
                tc_fence_after();
                if (elect_one()) {
                    const unsigned w = ((smem_u32(smem) + (unsigned)(slot * PAIR_STAGE)) & 0x3ffffu) >> 4, a = w + 128 * MM_K / 16;
#pragma unroll
                    for (int q = 0; q < MM_K / 32; ++q) tc_mma_i8_pair(d, w + 2 * q, a + 2 * q, hi, idesc, k > 0 || q > 0);
                    tc_commit_pair(smem_u32(&empty[slot]));
                    if (k == blocks - 1) tc_commit_pair(smem_u32(&tfull[t & 1]));
                }
                __syncwarp();
            }
        }
    } else if (warp >= 2) {
        const int quad = warp & 3, half = (warp - 2) >> 2;
        for (int t = 0; t < mine; ++t) {
            const int tile = pair + t * pairs, channel = tile % tiles_n * 256 + (int)rank * 128 + quad * 32 + lane, t0 = tile / tiles_n * 256 + half * 128;
            const float sw = channel < p.N ? p.w_scales[channel] : 0.0f, bias = p.bias && channel < p.N ? p.bias[channel] : 0.0f;
            if (!mbar_wait_warp(smem_u32(&tfull[t & 1]), (unsigned)(t / 2) & 1u, &abort_flag, status, 37)) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < 128; c += 32) {
                if (t0 + c >= p.M) break;
                const float mine_sa = t0 + c + lane < p.M ? p.a_scales[t0 + c + lane] : 0.0f;
                unsigned acc[32];
                tc_ld32(tmem + ((unsigned)(quad * 32) << 16) + (unsigned)((t & 1) * 256 + half * 128 + c), acc);
                tc_wait_ld_into(acc);
                float sa[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) sa[i] = __shfl_sync(0xffffffffu, mine_sa, i);
                store_columns<T>(p, acc, sa, t0 + c, p.M - t0 - c, channel, sw, bias);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_even(smem_u32(&tempty[t & 1]));
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync();         // neither block leaves while the other's MMAs or arrivals reach into it
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// ---- a few tokens: no tiles
// A warp takes two output channels, 512 bytes of k of both at a time, and M tokens: loads straight to registers, four products an instruction, one
// sum over the warp at the end.  None of what a tile needs before its first and after its last byte (barriers, TMEM, a cluster's join).  1 x 4096 x
// 4096: 3.9 us back to back with the weights in L2, 6.6 (2.5 TB/s) with them in memory; from three or four tokens on the products take longer than the bytes.
template <typename T, int M, bool BYTES>
__global__ void __launch_bounds__(256) matmul_i8_rows_kernel(const MatmulArgs p)
{
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, n = ((int)blockIdx.x * 8 + (int)(threadIdx.x >> 5)) * 2;
    if (n >= p.N) return;
    const int8_t* const w0 = p.w + (size_t)n * p.w_stride;
    const int8_t* const w1 = n + 1 < p.N ? w0 + p.w_stride : w0;
    const int8_t* a[M];
#pragma unroll
    for (int m = 0; m < M; ++m) a[m] = p.a + (size_t)(m < p.M ? m : 0) * p.a_stride;
    int acc[2][M] = {};
    const auto load = [](const int8_t* from, int valid) { return BYTES ? load_bytes(from, valid) : *reinterpret_cast<const uint4*>(from); };
#pragma unroll 4
    for (int k = lane * 16; k < p.K; k += 512) {
        const int valid = min(p.K - k, 16);
        const uint4 x0 = load(w0 + k, valid), x1 = load(w1 + k, valid);
#pragma unroll
        for (int m = 0; m < M; ++m) {
            const uint4 y = load(a[m] + k, valid);
            acc[0][m] = __dp4a((int)x0.w, (int)y.w, __dp4a((int)x0.z, (int)y.z, __dp4a((int)x0.y, (int)y.y, __dp4a((int)x0.x, (int)y.x, acc[0][m]))));
            acc[1][m] = __dp4a((int)x1.w, (int)y.w, __dp4a((int)x1.z, (int)y.z, __dp4a((int)x1.y, (int)y.y, __dp4a((int)x1.x, (int)y.x, acc[1][m]))));
        }
    }
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int sum = __reduce_add_sync(0xffffffffu, acc[r][m]);
            if (lane == 2 * m + r && m < p.M && n + r < p.N)
                ((T*)p.out)[(size_t)m * p.out_stride + n + r] = Elem<T>::from_float(fmaf((float)sum * p.a_scales[m], p.w_scales[n + r], p.bias ? p.bias[n + r] : 0.0f));
        }
}

template <typename T, int M>
static cudaError_t launch_few(const MatmulArgs& p, bool bytes, cudaStream_t s)
{
    const dim3 grid((unsigned)((p.N + 15) / 16));
    return bytes ? launch_token(matmul_i8_rows_kernel<T, M, true>, grid, 256, 0, 1, s, p) : launch_token(matmul_i8_rows_kernel<T, M, false>, grid, 256, 0, 1, s, p);
}

// Blocks that share a multiprocessor so that all of a call run at once, four at most (their rings get the smaller for it)
static int tile_residents(const MatmulArgs& p, int sms, int bn, int split)
{
    const long long ctas = (long long)((p.N + 127) / 128) * ((p.M + bn - 1) / bn) * split, each = (ctas + sms - 1) / sms;
    const int most = bn >= 256 ? 1 : bn == 128 ? 2 : 4;
    return each < most ? (int)each : most;
}

template <typename T, int BN, bool BYTES>
static cudaError_t launch_tile(const MatmulArgs& p, int split, int* status, cudaStream_t s)
{
    static SmemLimitSet set;
    CUtensorMap w_map = {}, a_map = {};
    if (BYTES) {
    } else if (!token_byte_map(&w_map, p.w, p.K, p.N, p.w_stride, MM_K, 128, CU_TENSOR_MAP_SWIZZLE_128B)
        || !token_byte_map(&a_map, p.a, p.K, p.M, p.a_stride, MM_K, BN, CU_TENSOR_MAP_SWIZZLE_128B))
        return cudaErrorInvalidValue;
    constexpr int STAGE = (128 + BN) * MM_K;
    const int blocks = (p.K + MM_K - 1) / MM_K, room = TILE_RING / tile_residents(p, token_sms(), BN, split) / STAGE;
    int stages = (blocks + split - 1) / split;
    stages = stages < room ? stages : room;
    stages = stages < 12 ? stages : 12;
    const int part = split > 1 ? BN * 128 * 4 : 0;
    const int need = (stages * STAGE > part ? stages * STAGE : part) + 1024, least = (BN < 32 ? 32 : BN) * TMEM_BYTES, bytes = need > least ? need : least;
    const cudaError_t e = raise_smem_limit(matmul_i8_tile_kernel<T, BN, BYTES>, set, TILE_RING + 1024);
    if (e != cudaSuccess) return e;
    const dim3 grid((unsigned)split, (unsigned)((p.N + 127) / 128), (unsigned)((p.M + BN - 1) / BN));
    return launch_token(matmul_i8_tile_kernel<T, BN, BYTES>, grid, TileWarps<BYTES>::THREADS, bytes, split, s, w_map, a_map, p, stages, status);
}

template <typename T>
static cudaError_t launch_pair(const MatmulArgs& p, int sms, int* status, cudaStream_t s)
{
    static SmemLimitSet set;
    CUtensorMap w_map, a_map;
    if (!token_byte_map(&w_map, p.w, p.K, p.N, p.w_stride, MM_K, 128, CU_TENSOR_MAP_SWIZZLE_128B)
        || !token_byte_map(&a_map, p.a, p.K, p.M, p.a_stride, MM_K, 128, CU_TENSOR_MAP_SWIZZLE_128B))
        return cudaErrorInvalidValue;
    const cudaError_t e = raise_smem_limit(matmul_i8_pair_kernel<T>, set, PAIR_SMEM);
    if (e != cudaSuccess) return e;
    const int tiles_n = (p.N + 255) / 256, tiles = tiles_n * ((p.M + 255) / 256);
    const int pairs = tiles < sms / 2 ? tiles : sms / 2;
    return launch_token(matmul_i8_pair_kernel<T>, dim3((unsigned)(2 * pairs)), PAIR_THREADS, PAIR_SMEM, 2, s, w_map, a_map, p, tiles_n, tiles, status);
}

// Cycles that a call is expected to take, by the number of tokens of a tile and of blocks that share one (0 tokens: pairs).  The constants are fitted to
// a sweep of both over 25 shapes from 1 x 4096 x 4096 to 4096 x 4096 x 4096: what it chooses takes 0.1 % longer than the best on average, 6 % at
// most (150 x 1000 x 8000); the other choices take up to four times as long.
static double expected_cycles(const MatmulArgs& p, int sms, int bn, int split, bool bytes)
{
    const double blocks = (p.K + MM_K - 1) / MM_K;
    if (bn == 0) {
        const long long tiles = (long long)((p.N + 255) / 256) * ((p.M + 255) / 256), waves = (tiles + sms / 2 - 1) / (sms / 2);
        return 5000 + waves * (blocks * 705 > 7400 ? blocks * 705 : 7400);     // (a tile's stores run beside the next one's products)
    }
    const long long ctas = (long long)((p.N + 127) / 128) * ((p.M + bn - 1) / bn) * split, each = (ctas + sms - 1) / sms;
    if (split == 8 && each > 1) return 1e30;       // (clusters of eight find no place beside one another: 14.4 us instead of 9.7 for 48 x 6144 x 4096)
    const long long residents = tile_residents(p, sms, bn, split), rounds = (each + residents - 1) / residents;
    // a step's MMAs (128 cycles for 256 tokens, no fewer than 50 an MMA), or its bytes at 45 a cycle (through registers: 5.7, and a block's rate does not rise where others leave early)
    const double mma = bn >= 128 ? bn * 2 : 200, load = (128 + bn) * MM_K / (bytes ? 5.7 : 45.0), share = bytes ? (double)each : ctas > sms ? (double)ctas / sms : 1.0;
    return 3000 + share * (((p.K + MM_K - 1) / MM_K + split - 1) / split) * (mma > load ? mma : load) + rounds * (1050 + bn * 9.0) + (split > 1 ? 2700 + bn * (26 + 0.4 * split) : 0.0);
}

template <typename T, bool BYTES>
static cudaError_t launch_tiles(const MatmulArgs& p, int bn, int split, int* status, cudaStream_t s)
{
    switch (bn) {
    case 16: return launch_tile<T, 16, BYTES>(p, split, status, s);
    case 32: return launch_tile<T, 32, BYTES>(p, split, status, s);
    case 64: return launch_tile<T, 64, BYTES>(p, split, status, s);
    case 128: return launch_tile<T, 128, BYTES>(p, split, status, s);
    default: return launch_tile<T, 256, BYTES>(p, split, status, s);
    }
}

template <typename T>
static cudaError_t launch_matmul(const MatmulArgs& p, cudaStream_t s)
{
    const bool bytes = !token_aligned(p.a, 16) || !token_aligned(p.w, 16) || p.a_stride % 16 || p.w_stride % 16;
    // one or two tokens, up to eight where the products are few (us with the weights in L2, tiles / without: 1 x 4096 x 4096 6.6 / 3.9, 2 x 4096 x 4096 6.6 / 4.5, 4 x 1024 x 4096
    // 5.4 / 4.7, 8 x 4096 x 4096 6.7 / 7.0, 4 x 8192 x 4096 8.8 / 13.8).  Unaligned rows: one token, up to four short ones (1 x 4096 x 5999 23.8 / 17.2, 4 x
    // 10000 x 511 10.5 / 6.9, 4 x 1000 x 999 6.1 / 5.3, 2 x 4096 x 2001 9.3 / 10.8, 4 x 4096 x 4001 14.5 / 24.5, 6 x 1000 x 999 6.1 / 8.1)
    if (bytes ? p.M == 1 || (p.M <= 4 && p.M * p.K <= 4000) : p.M <= 2 || (p.M <= 8 && (long long)p.M * p.N * p.K <= 1 << 25)) {
        const bool words = bytes || p.K % 16;
        if (p.M == 1) return launch_few<T, 1>(p, words, s);
        if (p.M == 2) return launch_few<T, 2>(p, words, s);
        return p.M <= 4 ? launch_few<T, 4>(p, words, s) : launch_few<T, 8>(p, words, s);
    }
    int* const status = token_status_word();
    if (!status) return cudaErrorInvalidSymbol;
    const int sms = token_sms(), blocks = (p.K + MM_K - 1) / MM_K;
    int best_bn = 0, best_split = 1;
    double best = bytes ? 1e30 : expected_cycles(p, sms, 0, 1, false);
    for (int bn = 16; bn <= 256; bn *= 2) {
        if ((p.M + bn - 1) / bn > 65535) continue;
        for (int split = 1; split <= 8 && split <= blocks; split *= 2) {
            const double c = expected_cycles(p, sms, bn, split, bytes);
            if (c < best) { best = c; best_bn = bn; best_split = split; }
        }
        if (bn >= p.M) break;
    }
    if (best_bn == 0) return launch_pair<T>(p, sms, status, s);
    return bytes ? launch_tiles<T, true>(p, best_bn, best_split, status, s) : launch_tiles<T, false>(p, best_bn, best_split, status, s);
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
    if (d.n > 65535 * 128) return set_error(N2D2B_ERR_TOO_LARGE, "n = %d exceeds %d", d.n, 65535 * 128);
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
