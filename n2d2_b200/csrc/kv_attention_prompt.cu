// Attention of many new tokens over the paged 8-bit cache, on the tensor cores (the mathematics: kv_attention.cu).
//
// A block takes 256 rows (new token x query head of one key head, two tiles of 128) and walks over the tokens they see, 128 at a time.
//   warp 0       issues the MMAs: S = Q K^T (128 x 128, 32-bit sums in TMEM), O += P V with P read from TMEM in S's place
//   warp 1       the scales of the pages
//   warps 4-7    bring keys through registers and write their codes as halves (exact) where the MMAs read them, swizzled; 8-11 the same for values
//   warps 12-19  a thread holds one row of one tile: scores to probabilities, running maximum and sum, at the end O / sum
// While the tensor pipe works on one tile, the other tile's rows are in the hands of their threads, 32 scores at a time with the next 32 on
// their way.  A row's maximum only moves, and the output so far is only rescaled, when a score is more than 2^8 above it: below that the
// probabilities stay inside 16 bits and their sum in 32 whatever the maximum they are taken against.  A probability of 1 is 2^5 to 2^6 there, so one
// keeps its 11 bits down to 2^-19 and is off by at most 2^-30 below that, 2^-29 with the times its row's maximum moved since.  The softmax's sum is held on 2^-4 of that scale: it adds reciprocals of the values' scales
// from 2^-121 to 2^100.
//
// 4096 new tokens over 8192 (32 query heads, 8 key heads of 128, bf16): 509 us, 810 TFLOP/s, 48 % of what a large matrix product reaches.  Bound by
// the latency of a row's chain (scores out of TMEM, maximum, exponentials, back into TMEM) with two warps of rows to a scheduler: no pipe is more than
// 43 % busy (tensor 43, exponentials 31, ALU 31, issue 45).  Measured and dropped: steps of 64 tokens with a second buffer of scores (540 us: products of 64
// columns take as long as of 100), probabilities before the maximum (553), the maximum in a pass of its own (603: TMEM is read twice).
#include <cstdio>
#include <cstring>
#include "kv_common.cuh"

namespace n2d2b {

static constexpr int PR_THREADS = 640, PR_BLOCK = 128, PR_CONSTS = 4, PR_POLYNOMIAL = 6;
static constexpr float PR_SUM = 4.0f;                        // powers of two that the sum's probabilities are below those of the products (0x1p-4f at the end)
static constexpr float PR_BITS = 6.0f, PR_ROOM = 8.0f;       // a probability of 1 is 2^5 to 2^6, the largest before the maximum moves 2^14
template <int D> struct PromptSmem {
    static constexpr int TILE = 128 * D * 2;                 // 128 rows (or tokens) of halves, in blocks of 64 columns
    static constexpr int Q = 0, K = Q + 2 * TILE, V = K + 2 * TILE, NEED = V + 2 * TILE + 1024;
    static constexpr int BYTES = NEED > 227 * 1024 - 4096 ? NEED : 227 * 1024 - 4096;   // all of TMEM: a multiprocessor to itself
    static constexpr int PITCH = D + 4;                      // floats of a row of a part, in the tiles' place at the end
    static_assert(256 * PITCH * 4 <= 6 * TILE, "a part fits");
};

__device__ __forceinline__ void tc_mma_f16_ss(unsigned d_tmem, unsigned a_lo, unsigned b_lo, unsigned desc_hi, unsigned idesc, unsigned accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %3};\n\t"
        "mov.b64 db, {%2, %3};\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n\t}"
        ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(desc_hi), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tc_mma_f16_ts(unsigned d_tmem, unsigned a_tmem, unsigned b_lo, unsigned desc_hi, unsigned idesc, unsigned accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
        "mov.b64 db, {%2, %3};\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "r"(b_lo), "r"(desc_hi), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tc_ld16(unsigned taddr, unsigned* v)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
                   "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tc_st16(unsigned taddr, const unsigned* v)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
                 "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]));     // (no memory clobber: loads may pass it)
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void sts128(unsigned addr, unsigned x, unsigned y, unsigned z, unsigned w)
{
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// Two 32-bit values to an instruction
typedef unsigned long long Pair;
__device__ __forceinline__ Pair pair_of(float a, float b)
{
    Pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 both_of(Pair p)
{
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
    return r;
}
__device__ __forceinline__ Pair fma_pair(Pair a, Pair b, Pair c)
{
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ Pair add_pair(Pair a, Pair b)
{
    Pair d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max_of(float a, float b, float c)
{
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ Pair mul_pair(Pair a, Pair b)
{
    Pair d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// The larger one; no number if either is none
__device__ __forceinline__ float max_or_nan(float a, float b)
{
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
// 2^x for x up to 14 without the exponential unit, which a quarter of the probabilities is kept from (it takes 8 cycles for a warp's 32 and would bound
// the kernel): x = n + f with n whole, 2^f on [-1/2, 1/2] by the polynomial of degree 4 with the smallest relative error (2.6e-6, from an exchange
// iteration), times the number with the exponent n.  That is 0 from n = -127 down, and what is no number stays that, whatever the bits of its n make of the factor.
__device__ __forceinline__ Pair exp2_pair(Pair x)
{
    const float2 v = both_of(x);
    x = pair_of(max_or_nan(v.x, -127.0f), max_or_nan(v.y, -127.0f));
    const Pair r = add_pair(x, pair_of(12582912.0f, 12582912.0f));      // 1.5 * 2^23: n in the lowest bits
    const Pair f = fma_pair(add_pair(r, pair_of(-12582912.0f, -12582912.0f)), pair_of(-1.0f, -1.0f), x);
    Pair p = pair_of(0.009570102207362652f, 0.009570102207362652f);
    p = fma_pair(p, f, pair_of(0.05591785907745361f, 0.05591785907745361f));
    p = fma_pair(p, f, pair_of(0.240247443318367f, 0.240247443318367f));
    p = fma_pair(p, f, pair_of(0.6931217908859253f, 0.6931217908859253f));
    p = fma_pair(p, f, pair_of(0.9999992847442627f, 0.9999992847442627f));
    const float2 n = both_of(r);
    return mul_pair(p, pair_of(__uint_as_float((__float_as_uint(n.x) << 23) + 0x3f800000u), __uint_as_float((__float_as_uint(n.y) << 23) + 0x3f800000u)));
}
template <bool M> struct Masked { static constexpr bool value = M; };

struct PromptBars {
    unsigned long long k_full[2], k_empty[2], v_full[2], v_empty[2], q_full[2], s_full[2], p_full[2], o_full[2], c_full[PR_CONSTS], c_empty[PR_CONSTS];
};

template <typename T, int D>
__global__ void __launch_bounds__(PR_THREADS, 1) kv_attention_prompt_kernel(const AttendArgs a, int tiles, int sequences)
{
    typedef PromptSmem<D> S;
    unsigned char* const smem = (unsigned char*)(((uintptr_t)dyn_smem() + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) PromptBars bars;
    __shared__ float4 consts[PR_CONSTS][PR_BLOCK / 16];     // scale of the keys, log2 and reciprocal (times 2^-PR_SUM) of the values', for 16 tokens
    __shared__ float part_top[256], part_sum[256];
    __shared__ unsigned tmem_slot;
    __shared__ int abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&bars.k_full[i]), 4);
            mbar_init(smem_u32(&bars.v_full[i]), 4);
            mbar_init(smem_u32(&bars.q_full[i]), 4);
            mbar_init(smem_u32(&bars.p_full[i]), 4);
            mbar_init(smem_u32(&bars.k_empty[i]), 1);
            mbar_init(smem_u32(&bars.v_empty[i]), 1);
            mbar_init(smem_u32(&bars.s_full[i]), 1);
            mbar_init(smem_u32(&bars.o_full[i]), 1);
        }
        for (int i = 0; i < PR_CONSTS; ++i) { mbar_init(smem_u32(&bars.c_full[i]), 1); mbar_init(smem_u32(&bars.c_empty[i]), 8); }
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        pdl_wait();         // (see TMEM_BYTES)
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = tmem_slot;
    pdl_launch_dependents();
    pdl_wait();

    // the rows with the most to see come first
    const unsigned rank = cluster_rank(), ranks = cluster_size(), id = blockIdx.x / ranks;
    const int head = (int)(id % (unsigned)a.c.heads), b = (int)(id / (unsigned)a.c.heads % (unsigned)sequences);
    const int tile = tiles - 1 - (int)(id / (unsigned)a.c.heads / (unsigned)sequences);
    const KvSequence s = kv_sequence(a.c, b);
    const int row0 = tile * 256, rows = s.count * a.group - row0;
    const bool any = rows > 0, two = rows > 128;
    const int t_first = row0 / a.group, t_last = (min(row0 + 256, s.count * a.group) - 1) / a.group;
    int lo = 0, hi = any ? s.length : 0;
    if (a.causal) {
        hi = min(hi, s.begin + t_last + 1);
        if (a.window) lo = max(0, s.begin + t_first + 1 - a.window);
    }
    const int capacity = a.c.row << a.log_page;
    hi = min(hi, capacity);
    // the blocks of a cluster take a part of the tokens each
    const int all = hi > lo ? (hi + PR_BLOCK - 1) / PR_BLOCK - lo / PR_BLOCK : 0, per = (all + (int)ranks - 1) / (int)ranks;
    const int j_lo = lo / PR_BLOCK + (int)rank * per, blocks = max(0, min(per, all - (int)rank * per));
    const unsigned base = smem_u32(smem);

    if (warp < 4) {
        fewer_registers<40>();
        if (warp == 1) {
            // lane i: scales of tokens 16 i .. 16 i + 15 of a block, ahead of the keys
            auto number_of = [&](int j) -> int {
                const int token = (j_lo + j) * PR_BLOCK + lane * 16;
                return lane < 8 && j < blocks && token < hi ? a.c.table[(size_t)b * a.c.row + (token >> a.log_page)] : 0;
            };
            float k_scale = 0.0f, v_scale = 0.0f;
            bool bad = false;
            auto turn_to = [&](int page_number) {
                bad = (unsigned)page_number >= (unsigned)a.c.nb_pages;
                const int at = (bad ? 0 : page_number) * a.c.heads + head;
                k_scale = a.c.k_scales[at];
                v_scale = a.c.v_scales[at];
            };
            if (blocks > 0) turn_to(number_of(0));
            int number = number_of(1);
            for (int j = 0; j < blocks; ++j) {
                if (j >= PR_CONSTS && !mbar_wait_issuer(smem_u32(&bars.c_empty[j & (PR_CONSTS - 1)]), (unsigned)(j / PR_CONSTS - 1) & 1u, &abort_flag, a.status, 46)) break;
                if (lane < 8) {
                    const float scale = v_scale <= TOKEN_TINY ? KV_NOTHING : v_scale, log = __log2f(scale);       // (all codes are 0 there)
                    consts[j & (PR_CONSTS - 1)][lane] = make_float4(bad ? __int_as_float(0x7fffffff) : k_scale, log, exp2_approx(-log - PR_SUM), 0.0f);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&bars.c_full[j & (PR_CONSTS - 1)]));
                if (j + 1 < blocks) turn_to(number);
                number = number_of(j + 2);
            }
        } else if (warp == 0 && blocks > 0) {
            const unsigned hi_k = (unsigned)(make_smem_desc(0u, 128) >> 32);
            const unsigned idesc_s = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
            const unsigned idesc_o = (1u << 4) | (1u << 16) | (((unsigned)D >> 3) << 17) | ((128u >> 4) << 24);   // values: tokens are rows
            const unsigned q_lo = ((base + S::Q) & 0x3ffffu) >> 4, k_lo = ((base + S::K) & 0x3ffffu) >> 4, v_lo = ((base + S::V) & 0x3ffffu) >> 4;
            const int n = two ? 2 : 1;
            auto scores = [&](int i, int j) {       // S of tile i, block j
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        const unsigned at = (unsigned)((k >> 2) * 1024 + (k & 3) * 2);
                        tc_mma_f16_ss(tmem + (unsigned)(i * 128), q_lo + (unsigned)(i * (S::TILE / 16)) + at, k_lo + (unsigned)((j & 1) * (S::TILE / 16)) + at, hi_k,
                                      idesc_s, k > 0);
                    }
                    tc_commit(smem_u32(&bars.s_full[i]));
                    if (i == n - 1) tc_commit(smem_u32(&bars.k_empty[j & 1]));
                }
                __syncwarp();
            };
            bool ok = true;
            for (int i = 0; i < n && ok; ++i) ok = mbar_wait_issuer(smem_u32(&bars.q_full[i]), 0, &abort_flag, a.status, 41);
            if (ok) ok = mbar_wait_issuer(smem_u32(&bars.k_full[0]), 0, &abort_flag, a.status, 42);
            if (ok) {
                tc_fence_after();
                for (int i = 0; i < n; ++i) scores(i, 0);
            }
            for (int j = 0; j < blocks && ok; ++j) {
                ok = mbar_wait_issuer(smem_u32(&bars.v_full[j & 1]), (unsigned)(j >> 1) & 1u, &abort_flag, a.status, 43);
                if (ok && j + 1 < blocks) ok = mbar_wait_issuer(smem_u32(&bars.k_full[(j + 1) & 1]), (unsigned)((j + 1) >> 1) & 1u, &abort_flag, a.status, 42);
                for (int i = 0; i < n && ok; ++i) {
                    ok = mbar_wait_issuer(smem_u32(&bars.p_full[i]), (unsigned)j & 1u, &abort_flag, a.status, 44);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < PR_BLOCK / 16; ++k)
                            tc_mma_f16_ts(tmem + 256u + (unsigned)(i * 128), tmem + (unsigned)(i * 128 + k * 8),
                                          (v_lo + (unsigned)((j & 1) * (S::TILE / 16)) + (unsigned)(k * 128)) | (1024u << 16), hi_k, idesc_o, j > 0 || k > 0);
                        if (i == n - 1) tc_commit(smem_u32(&bars.v_empty[j & 1]));
                        if (j == blocks - 1) tc_commit(smem_u32(&bars.o_full[i]));
                    }
                    __syncwarp();
                    // (in order behind the product that reads P where this writes S)
                    if (j + 1 < blocks) scores(i, j + 1);
                }
            }
        }
    } else if (warp < 12) {
        fewer_registers<88>();
        const bool keys = warp < 8;
        const int tid = (threadIdx.x - 128) & 127;
        constexpr int CHUNKS = D / 16, ROWS = 128 / CHUNKS, PASSES = 128 / ROWS;   // 16 codes a chunk, tokens of a pass, passes of a block
        // eight lanes write two rows' halves of a 64-column block: no two on one bank
        const int row = CHUNKS == 8 ? (tid >> 5) * 4 + ((tid >> 4) & 1) * 2 + ((tid >> 2) & 1) : tid / CHUNKS;
        const int chunk = CHUNKS == 8 ? ((tid >> 3) & 1) * 4 + (tid & 3) : tid % CHUNKS;
        const int8_t* const from = (keys ? a.c.k : a.c.v) + chunk * 16;
        // lane i: page number of tokens 16 i .. 16 i + 15 of a block, asked for two blocks ahead
        auto number_of = [&](int j) -> int {
            const int token = (j_lo + j) * PR_BLOCK + lane * 16;
            return lane < 8 && j < blocks && token < hi ? a.c.table[(size_t)b * a.c.row + (token >> a.log_page)] : 0;
        };
        uint4 x[PASSES];
        auto load = [&](int number) {
            const int first = (((unsigned)number < (unsigned)a.c.nb_pages ? number : 0) * a.c.heads + head) << a.log_page;
#pragma unroll
            for (int i = 0; i < PASSES; ++i) {
                const int t = i * ROWS + row;          // token of the block
                const int line = __shfl_sync(0xffffffffu, first, t >> 4) + (t & ((1 << a.log_page) - 1));
                x[i] = *reinterpret_cast<const uint4*>(from + (size_t)(unsigned)line * D);
            }
        };
        const unsigned full = smem_u32(keys ? bars.k_full : bars.v_full), empty = smem_u32(keys ? bars.k_empty : bars.v_empty);
        const unsigned to = base + (keys ? S::K : S::V) + (unsigned)((chunk >> 2) * 16384 + row * 128);
        if (blocks > 0) load(number_of(0));
        int number = number_of(1);
        for (int j = 0; j < blocks; ++j) {
            if (j >= 2 && !mbar_wait_warp(empty + 8u * (j & 1), (unsigned)((j >> 1) - 1) & 1u, &abort_flag, a.status, 45)) break;
#pragma unroll
            for (int i = 0; i < PASSES; ++i) {
                const unsigned w[4] = {x[i].x ^ 0x80808080u, x[i].y ^ 0x80808080u, x[i].z ^ 0x80808080u, x[i].w ^ 0x80808080u};
                unsigned h[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) { h[2 * e] = less_1152(splice(w[e], 0x4140)); h[2 * e + 1] = less_1152(splice(w[e], 0x4342)); }
                const unsigned line = to + (unsigned)((j & 1) * S::TILE + i * ROWS * 128), c = (((unsigned)(chunk & 3) * 2) ^ (unsigned)((i * ROWS + row) & 7)) << 4;
                sts128(line + c, h[0], h[1], h[2], h[3]);
                sts128(line + (c ^ 16u), h[4], h[5], h[6], h[7]);
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(full + 8u * (j & 1));
            if (j + 1 < blocks) {
                load(number);
                number = number_of(j + 2);
            }
        }
    } else {
        more_registers<128>();
        const int i = (warp - 12) >> 2, r = threadIdx.x - 384 - i * 128;     // tile and row
        const int row = row0 + i * 128 + r, t = row / a.group, h = row - t * a.group;
        const bool there = row < s.count * a.group;
        const int pos = s.begin + t;
        int see_lo = 0, see_hi = 0;
        if (there) {
            see_hi = a.causal ? min(s.length, pos + 1) : s.length;
            if (a.causal && a.window) see_lo = max(0, pos + 1 - a.window);
        }
        float sum = there && see_hi > capacity ? __int_as_float(0x7fffffff) : 0.0f, top = -INFINITY, row_scale = 0.0f;
        if (blocks > 0 && (i == 0 || two)) {
            const T* const q = (const T*)a.q + (size_t)(s.first_row + t) * a.q_stride + (size_t)(head * a.group + h) * D;
            unsigned largest = 0;
#pragma unroll 4
            for (int e = 0; e < D / 8; ++e) {
                uint4 w = make_uint4(0, 0, 0, 0);
                if (there) w = *reinterpret_cast<const uint4*>(q + 8 * e);
                float f[8];
                Elem<T>::unpack(w, f);
#pragma unroll
                for (int x = 0; x < 8; ++x) largest = max(largest, magnitude(f[x]));
            }
            // a power of two brings the row's largest value into [1, 4); the sign of the scale goes with it.  A row that is not finite becomes no numbers
            // altogether: a score of -inf would count as one that is not seen.
            const int exponent = min((int)(largest >> 23), 253);
            const bool finite = largest < 0x7f800000u, scaled = exponent > 0 && finite;
            const float up = finite ? copysignf(scaled ? __int_as_float((254 - exponent) << 23) : 1.0f, a.scale_log2) : __int_as_float(0x7fffffff);
            row_scale = fabsf(a.scale_log2) * (scaled ? __int_as_float(exponent << 23) : 1.0f);
#pragma unroll 4
            for (int e = 0; e < D / 8; ++e) {
                uint4 w = make_uint4(0, 0, 0, 0);
                if (there) w = *reinterpret_cast<const uint4*>(q + 8 * e);
                float f[8];
                Elem<T>::unpack(w, f);
                sts128(base + S::Q + (unsigned)(i * S::TILE + (e >> 3) * 16384 + r * 128 + (((e & 7) ^ (r & 7)) << 4)), pack_half2(f[0] * up, f[1] * up),
                       pack_half2(f[2] * up, f[3] * up), pack_half2(f[4] * up, f[5] * up), pack_half2(f[6] * up, f[7] * up));
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bars.q_full[i]));
        }
        const unsigned lanes = (unsigned)((warp & 3) * 32) << 16;
        const unsigned s_at = tmem + lanes + (unsigned)(i * 128), o_at = tmem + lanes + 256u + (unsigned)(i * 128);
        bool ok = true;
        if (i == 1 && !two) {
            for (int j = 0; j < blocks; ++j) {      // a tile without rows: only hands the constants on
                if (!mbar_wait_issuer(smem_u32(&bars.c_full[j & (PR_CONSTS - 1)]), (unsigned)(j / PR_CONSTS) & 1u, &abort_flag, a.status, 47)) break;
                if (lane == 0) mbar_arrive(smem_u32(&bars.c_empty[j & (PR_CONSTS - 1)]));
            }
        } else {
            for (int j = 0; j < blocks; ++j) {
                const int j0 = (j_lo + j) * PR_BLOCK;
                ok = mbar_wait_warp(smem_u32(&bars.c_full[j & (PR_CONSTS - 1)]), (unsigned)(j / PR_CONSTS) & 1u, &abort_flag, a.status, 47)
                     && mbar_wait_warp(smem_u32(&bars.s_full[i]), (unsigned)j & 1u, &abort_flag, a.status, 48);
                if (!ok) break;
                tc_fence_after();
                const float4* const group = consts[j & (PR_CONSTS - 1)];
                const bool whole = __all_sync(0xffffffffu, see_lo <= j0 && see_hi >= j0 + PR_BLOCK);
                const unsigned first = (unsigned)(see_lo - j0), span = (unsigned)max(see_hi - see_lo, 0);

                // scores 32 q .. 32 q + 31 to probabilities
                auto quarter = [&](const int q, unsigned* x, const float4* f, auto masked) {
                    constexpr bool MASKED = decltype(masked)::value;
                    if (MASKED) {       // what a row does not see becomes -inf
#pragma unroll
                        for (int c = 0; c < 32; ++c)
                            if ((unsigned)(32 * q + c) - first >= span) x[c] = 0xff800000u;
                    }
                    float best = -INFINITY;
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        float m[5];
#pragma unroll
                        for (int e = 0; e < 5; ++e) m[e] = max_of(__uint_as_float(x[16 * g + 3 * e]), __uint_as_float(x[16 * g + 3 * e + 1]), __uint_as_float(x[16 * g + 3 * e + 2]));
                        const float most = max_of(max_of(m[0], m[1], m[2]), max_of(m[3], m[4], __uint_as_float(x[16 * g + 15])), -INFINITY);
                        best = fmaxf(best, MASKED && most == -INFINITY ? -INFINITY : fmaf(most, f[g].x * row_scale, f[g].y));
                    }
                    const bool moves = best > top + (PR_BITS + PR_ROOM) || (top == -INFINITY && best > top);       // (each row for itself: another row's numbers change nothing in it)
                    if (__any_sync(0xffffffffu, moves)) {
                        // a whole number, so that the factor is a power of two and halves only lose what falls off their lower end
                        const float raised = ceilf(best) - PR_BITS, fade = !moves ? 1.0f : (top == -INFINITY ? 0.0f : __int_as_float((127 + (int)fmaxf(top - raised, -127.0f)) << 23));
                        if (moves) top = raised;
                        sum *= fade;
                        tc_wait_st();       // what the quarters before stored: only this orders the loads behind it
#pragma unroll 1
                        for (int c = 0; c < 16 * q; c += 16) {        // this block's probabilities so far
                            unsigned p[16];
                            tc_ld16(s_at + (unsigned)c, p);
                            tc_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                asm volatile("" : "+r"(p[e])::"memory");
                                // (in 32 bits: factors below 2^-24 are no halves, but up to 2^14 times them are)
                                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p[e]));
                                p[e] = pack_half2(f.x * fade, f.y * fade);
                            }
                            tc_st16(s_at + (unsigned)c, p);
                        }
                        if (j > 0) {
#pragma unroll 1
                            for (int c = 0; c < D; c += 16) {
                                unsigned o[16];
                                tc_ld16(o_at + (unsigned)c, o);
                                tc_wait_ld();
#pragma unroll
                                for (int e = 0; e < 16; ++e) {
                                    asm volatile("" : "+r"(o[e])::"memory");
                                    o[e] = __float_as_uint(__uint_as_float(o[e]) * fade);
                                }
                                tc_st16(o_at + (unsigned)c, o);
                            }
                        }
                    }
                    const float from = top == -INFINITY ? 0.0f : top;
                    unsigned packed[16];
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        const float one_by = f[g].x * row_scale, one_add = f[g].y - from;
                        const Pair by = pair_of(one_by, one_by), add = pair_of(one_add, one_add);
                        Pair part[2] = {pair_of(0.0f, 0.0f), pair_of(0.0f, 0.0f)};
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            const float v0 = __uint_as_float(x[16 * g + e]), v1 = __uint_as_float(x[16 * g + e + 1]);
                            Pair p = fma_pair(pair_of(v0, v1), by, add);
                            if ((e & 6) == PR_POLYNOMIAL) p = exp2_pair(p);
                            else {
                                const float2 t = both_of(p);
                                p = pair_of(exp2_approx(t.x), exp2_approx(t.y));
                            }
                            float2 y = both_of(p);
                            if (MASKED) {       // (whatever the scales of a page it does not see)
                                y = make_float2(v0 == -INFINITY ? 0.0f : y.x, v1 == -INFINITY ? 0.0f : y.y);
                                p = pair_of(y.x, y.y);
                            }
                            part[(e >> 1) & 1] = add_pair(part[(e >> 1) & 1], p);
                            packed[8 * g + (e >> 1)] = pack_half2(y.x, y.y);
                        }
                        const float2 sums = both_of(add_pair(part[0], part[1]));
                        const float both = sums.x + sums.y;
                        if (!MASKED || both != 0.0f) sum = fmaf(both, f[g].z, sum);
                    }
                    tc_st16(s_at + (unsigned)(16 * q), packed);
                };
                auto block = [&](auto masked) {
                    // (the probabilities of 32 scores take 16 columns: they never reach what is still on its way)
                    unsigned xa[32], xb[32];
                    float4 fa[2] = {group[0], group[1]}, fb[2];
                    tc_ld32(s_at, xa);
                    tc_wait_ld_into(xa);
                    tc_ld32(s_at + 32u, xb);
                    fb[0] = group[2]; fb[1] = group[3];
                    quarter(0, xa, fa, masked);
                    tc_wait_ld_into(xb);
                    tc_ld32(s_at + 64u, xa);
                    fa[0] = group[4]; fa[1] = group[5];
                    quarter(1, xb, fb, masked);
                    tc_wait_ld_into(xa);
                    tc_ld32(s_at + 96u, xb);
                    fb[0] = group[6]; fb[1] = group[7];
                    quarter(2, xa, fa, masked);
                    tc_wait_ld_into(xb);
                    quarter(3, xb, fb, masked);
                };
                if (whole) block(Masked<false>());
                else block(Masked<true>());
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(smem_u32(&bars.p_full[i]));
                    mbar_arrive(smem_u32(&bars.c_empty[j & (PR_CONSTS - 1)]));
                }
            }
            if (ok && blocks > 0) ok = mbar_wait_warp(smem_u32(&bars.o_full[i]), 0, &abort_flag, a.status, 49);
            if (ranks > 1) {
                // the part goes where the tiles were: both tiles' products are through
                if (ok && blocks > 0 && two) ok = mbar_wait_warp(smem_u32(&bars.o_full[i ^ 1]), 0, &abort_flag, a.status, 49);
                tc_fence_after();
                float* const to = (float*)smem + (size_t)(i * 128 + r) * S::PITCH;
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    unsigned o[32];
                    tc_ld32(o_at + (unsigned)c, o);
                    tc_wait_ld_into(o);
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        *reinterpret_cast<uint4*>(to + c + e) = blocks > 0 ? make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]) : make_uint4(0, 0, 0, 0);
                }
                part_top[i * 128 + r] = top;
                part_sum[i * 128 + r] = sum;
            } else {
            tc_fence_after();
            const float inv = sum == 0.0f ? 0.0f : 0x1p-4f / sum;
            T* const out = (T*)a.out + (size_t)(s.first_row + t) * a.out_stride + (size_t)(head * a.group + h) * D;
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                unsigned o[32];
                tc_ld32(o_at + (unsigned)c, o);
                tc_wait_ld_into(o);
                if (there) {
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        float f[8];
#pragma unroll
                        for (int y = 0; y < 8; ++y) f[y] = sum == 0.0f ? 0.0f : __uint_as_float(o[e + y]) * inv;
                        *reinterpret_cast<uint4*>(out + c + e) = Elem<T>::pack(f);
                    }
                }
            }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {        // before the other blocks are waited for (see TMEM_BYTES)
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
    if (ranks > 1) {
        cluster_sync();
        // every block finishes a share of the outputs
        const int there = max(0, min(rows, 256)) * (D / 4);
        for (int e = (int)(rank * PR_THREADS + threadIdx.x); e < there; e += (int)ranks * PR_THREADS) {
            const int r = e / (D / 4), d = e % (D / 4) * 4;
            const unsigned at = base + (unsigned)(r * S::PITCH + d) * 4u, at_top = smem_u32(part_top + r), at_sum = smem_u32(part_sum + r);
            float m = -INFINITY;
            for (unsigned k = 0; k < ranks; ++k) m = fmaxf(m, ld_cluster(map_to_rank(at_top, k)));
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            float l = 0.0f;
            for (unsigned k = 0; k < ranks; ++k) {
                const float t = ld_cluster(map_to_rank(at_top, k));
                const float f = t == m ? 1.0f : exp2_approx(t - m);
                const float4 x = ld_cluster4(map_to_rank(at, k));
                o.x = fmaf(x.x, f, o.x); o.y = fmaf(x.y, f, o.y); o.z = fmaf(x.z, f, o.z); o.w = fmaf(x.w, f, o.w);
                l = fmaf(ld_cluster(map_to_rank(at_sum, k)), f, l);
            }
            const float inv = l == 0.0f ? 0.0f : 0x1p-4f / l;
            const int row = row0 + r, t = row / a.group, h = row - t * a.group;
            T* const out = (T*)a.out + (size_t)(s.first_row + t) * a.out_stride + (size_t)(head * a.group + h) * D + d;
            *reinterpret_cast<uint2*>(out) = make_uint2(Elem<T>::pack2(o.x * inv, o.y * inv), Elem<T>::pack2(o.z * inv, o.w * inv));
        }
        cluster_sync();     // no block leaves while another reads its part
    }
}

template <typename T, int D>
static cudaError_t launch_prompt_of(const AttendArgs& a, int sequences, cudaStream_t s)
{
    static SmemLimitSet set;
    const cudaError_t e = raise_smem_limit(kv_attention_prompt_kernel<T, D>, set, PromptSmem<D>::BYTES);
    if (e != cudaSuccess) return e;
    const long long tiles = ((long long)a.c.max_new * a.group + 255) / 256, blocks = tiles * a.c.heads * sequences;
    // where half of the multiprocessors would have nothing to do, clusters share the tokens, at least two steps to a block
    const int split = attend_streams(blocks, attend_steps(a), 2, 8);
    return launch_token(kv_attention_prompt_kernel<T, D>, dim3((unsigned)(blocks * split)), PR_THREADS, PromptSmem<D>::BYTES, split, s, a, (int)tiles, sequences);
}

cudaError_t launch_attention_prompt(const AttendArgs& a, int head_size, bool half, int sequences, cudaStream_t s)
{
    if (half) return head_size == 64 ? launch_prompt_of<__half, 64>(a, sequences, s) : launch_prompt_of<__half, 128>(a, sequences, s);
    return head_size == 64 ? launch_prompt_of<__nv_bfloat16, 64>(a, sequences, s) : launch_prompt_of<__nv_bfloat16, 128>(a, sequences, s);
}

}  // namespace n2d2b
