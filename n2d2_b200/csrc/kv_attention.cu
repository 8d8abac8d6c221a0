// Attention over the paged 8-bit cache.
//
//   s_j = scale * sK(page of j) * (q . k_j),   out = (sum_j e^(s_j) sV(page of j) v_j) / (sum_j e^(s_j))      over visible j
//
// in one pass over the tokens, with the running maximum of t_j = s_j log2(e) + log2 sV(page of j): the values' scales ride in the
// exponent, so that p_j = 2^(t_j - max) is at most 1 whatever the scales are and enters the second product in few bits; the softmax's sum
// adds p_j / sV(page of j): the p_j of that sum are about 1, as the scales go from 2^-100 to 2^121 and their reciprocals fill 32 bits.
//
// kv_attention_rows_kernel: 4, 8 or 16 rows (new token x query head of one key head) a tile, for few rows: bound by reading the cache.  The
// codes go into the int8 tensor cores as they lie in memory: widening them in registers took 224 integer instructions a warp for 32
// tokens of 128, which held a kernel of that kind to 4.5 TB/s at best.  The other operand is cut into bytes instead, which costs nothing as
// it has few columns: a query into three signed digits of a 22-bit number (on a scale of its own row), a probability into four unsigned
// ones of a 32-bit number (2^28 for 1).  Both products are exact in 32 bits.
//   S^T [128 tokens][3 digits x rows] = K Q^T,   O^T [head_size][4 digits x rows] = V^T P^T
// A thread holds a token's scores for all rows, later one element of every row's output.  The tokens of a sequence are split over a cluster of
// up to 16 blocks, whose parts are joined through distributed shared memory at the end: nothing is kept in memory between kernels.
//
// 48 sequences of up to 8000 tokens (8 key heads of 128, 32 query heads, bf16): 81 (back to back) to 85 us, 5.7 to 6.0 TB/s; one of 65000: 33 us, 4.0 TB/s (128 of the
// multiprocessors, a cluster of 16 for each head; the blocks' beginning and end take 8 us of it); 100 tokens, heads of 64: 5.7 us a call.
#include <cstdio>
#include <cstring>
#include "kv_common.cuh"

namespace n2d2b {

__device__ __forceinline__ void tc_ld8(unsigned taddr, unsigned* v)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "r"(taddr) : "memory");
}
template <int N> __device__ __forceinline__ void tc_ld_into(unsigned taddr, unsigned* v)
{
#pragma unroll
    for (int i = 0; i < N; i += 8) tc_ld8(taddr + (unsigned)i, v + i);
    tc_wait_ld();
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(v[i])::"memory");
}
// Whether any of a group's four warps that hold tokens says so
__device__ __forceinline__ bool any_of_128(int group, bool say)
{
    unsigned r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, %2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(r) : "r"((unsigned)say), "r"(1 + group) : "memory");
    return r != 0;
}

// Operands of different swizzles or orders: each has its own upper word
__device__ __forceinline__ void tc_mma_i8_mixed(unsigned d_tmem, unsigned a_lo, unsigned b_lo, unsigned a_hi, unsigned b_hi, unsigned idesc, unsigned accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %3};\n\t"
        "mov.b64 db, {%2, %4};\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], da, db, %5, p;\n\t}"
        ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(a_hi), "r"(b_hi), "r"(idesc), "r"(accumulate) : "memory");
}

// x * by for a whole number below 2^22 and a power of two: x as the lower bits of 1.5 * 2^23, which is subtracted again (exact; the
// conversion instruction has an eighth of the rate of these)
__device__ __forceinline__ float float_of(unsigned x, float by) { return fmaf(__uint_as_float(x + 0x4b400000u), by, -12582912.0f * by); }

static constexpr int ROWS_BLOCK = 128, ROWS_GROUP = 192;
static constexpr int ROWS_FLUSH = 512;          // blocks whose sums stay within 32 bits: 512 x 128 x 255 x 128 < 2^31
// The whole number of a probability of 1, and the powers of two that a score may be above the maximum before that moves: 2^32, the most there can be, is taken as
// 2^32 - 1.  The bits go to the small ones and not to the room: a probability is off by at most 2^-29 of the largest, so that the tokens beside one that takes 0.999 of
// a row and holds zeros keep their bits (with 2^23 for 1 they were off by up to a quarter).
static constexpr float ROWS_ONE = 0x1p28f, ROWS_ROOM = 4.0f;
static constexpr float ROWS_NONE = -3.0e38f;    // the maximum of nothing
// R: rows of a tile (4, 8 or 16); GROUPS: streams of tokens in a block
template <int D, int R, int GROUPS> struct RowsSmem {
    static constexpr int STAGE = 2 * ROWS_BLOCK * D;                                 // keys, then values
    static constexpr int NQ = R == 16 ? 48 : 32, NP = R == 16 ? 64 : 32;             // columns of the two products
    static constexpr int Q = 0, GROUP = (NQ * D + 1023) / 1024 * 1024;               // a group: probabilities of two blocks, then its ring
    static constexpr int RING = 2 * NP * ROWS_BLOCK, MOST = D == 128 ? 3 : 6;        // stages of a ring
    static constexpr int S_COLUMNS = NP, COLUMNS = NP * 4;                           // of TMEM, a group's: scores of two blocks, then the output
    static constexpr int PITCH = D + 4;                                              // floats of a row of a part, in the ring's place
    static_assert(R * PITCH * 4 <= STAGE && RING % 1024 == 0, "a part fits");
    static __host__ __device__ constexpr int group_bytes(int stages) { return RING + stages * STAGE; }
    static constexpr int bytes(int stages)
    {
        const int need = GROUP + GROUPS * group_bytes(stages) + 1024, least = GROUPS * COLUMNS * TMEM_BYTES;
        return need > least ? need : least;
    }
};

template <typename T, int D, int R, int GROUPS>
__global__ void __launch_bounds__(ROWS_GROUP * GROUPS, GROUPS == 2 ? 1 : R == 16 ? 2 : 3) kv_attention_rows_kernel(const __grid_constant__ CUtensorMap k_map,
                                                                                            const __grid_constant__ CUtensorMap v_map, const AttendArgs a, int stages)
{
    typedef RowsSmem<D, R, GROUPS> S;
    unsigned char* const smem = (unsigned char*)(((uintptr_t)dyn_smem() + 1023) & ~(uintptr_t)1023);
    struct Bars { unsigned long long full[S::MOST], o_done[S::MOST], s_full[2], p_full[2]; };
    __shared__ __align__(8) Bars all_bars[GROUPS];
    __shared__ __align__(8) unsigned long long q_full;
    __shared__ float row_scales[R], tops[GROUPS][4][R], sums[GROUPS][4][R], own_top[GROUPS][R], own_sum[GROUPS][R];
    __shared__ unsigned tmem_slot, all_fresh[GROUPS][2];
    __shared__ int abort_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, group = GROUPS == 1 ? 0 : warp / 6, role = warp - 6 * group;
    if (warp == 4) {
        if (elect_one()) {
            prefetch_tensor_map(&k_map);
            prefetch_tensor_map(&v_map);
            for (int g = 0; g < GROUPS; ++g) {
                Bars& m = all_bars[g];
                for (int i = 0; i < stages; ++i) { mbar_init(smem_u32(&m.full[i]), 1); mbar_init(smem_u32(&m.o_done[i]), 1); }
                for (int i = 0; i < 2; ++i) { mbar_init(smem_u32(&m.s_full[i]), 1); mbar_init(smem_u32(&m.p_full[i]), 4); }
            }
            mbar_init(smem_u32(&q_full), 4);
            abort_flag = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
        pdl_wait();         // (see TMEM_BYTES)
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"((unsigned)(S::COLUMNS * GROUPS)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = tmem_slot + (unsigned)(group * S::COLUMNS), o_tmem = tmem + 2 * S::S_COLUMNS;
    Bars& bars = all_bars[group];
    unsigned* const fresh = all_fresh[group];
    pdl_launch_dependents();
    pdl_wait();

    const int b = blockIdx.z, head = blockIdx.y % a.c.heads, row0 = (int)(blockIdx.y / a.c.heads) * R;
    const unsigned rank = cluster_rank(), ranks = cluster_size();
    const KvSequence s = kv_sequence(a.c, b);
    const int rows = s.count * a.group - row0;          // rows of the tile that exist (none: every block of the cluster only passes by)
    const int t_first = row0 / a.group, t_last = (min(row0 + R, s.count * a.group) - 1) / a.group;
    int lo = 0, hi = rows > 0 ? s.length : 0;
    if (a.causal) {
        hi = min(hi, s.begin + t_last + 1);
        if (a.window) lo = max(0, s.begin + t_first + 1 - a.window);
    }
    const int capacity = a.c.row << a.log_page;         // tokens behind the row of the table are nowhere
    hi = min(hi, capacity);
    const int all = hi > lo ? (hi + ROWS_BLOCK - 1) / ROWS_BLOCK - lo / ROWS_BLOCK : 0, parts = (int)ranks * GROUPS, per = (all + parts - 1) / parts;
    const int first = ((int)rank * GROUPS + group) * per, j_lo = lo / ROWS_BLOCK + first, blocks = max(0, min(per, all - first));
    const unsigned base = smem_u32(smem), at_group = (unsigned)(S::GROUP + group * S::group_bytes(stages));

    if (role == 5) {
        // ---- copies: a block into the slot of the block `stages` before it, once the products that read it are through
        const int page = 1 << a.log_page, pages = page < ROWS_BLOCK ? ROWS_BLOCK >> a.log_page : 1;
        auto look_up = [&](int j) -> int {  // lane i: page i of block j; page 0 where there is none that anybody sees
            const int token = (j_lo + j) * ROWS_BLOCK + lane * page;
            return lane < pages && j < blocks && token < hi ? a.c.table[(size_t)b * a.c.row + (token >> a.log_page)] : 0;
        };
        int number = look_up(0), slot = 0;
        unsigned phase = 1;
        for (int j = 0; j < blocks; ++j) {
            const int line = (((unsigned)number < (unsigned)a.c.nb_pages ? number : 0) * a.c.heads + head) * page;
            number = look_up(j + 1);
            if (j >= stages && !mbar_wait_issuer(smem_u32(&bars.o_done[slot]), phase, &abort_flag, a.status, 24)) {
                __nanosleep(1000000);       // copies under way land before the ring is given to the parts
                break;
            }
            const unsigned bar = smem_u32(&bars.full[slot]), dst = base + at_group + (unsigned)(S::RING + slot * S::STAGE);
            if (elect_one()) mbar_expect_tx(bar, S::STAGE);
            __syncwarp();
#pragma unroll 2
            for (int i = 0; i < pages; ++i) {
                const int y = __shfl_sync(0xffffffffu, line, i);
                if (elect_one()) {
                    tma_load_2d(dst + (unsigned)(i * page * D), &k_map, bar, 0, y);
                    tma_load_2d(dst + (unsigned)((ROWS_BLOCK + i * page) * D), &v_map, bar, 0, y);
                }
                __syncwarp();
            }
            if (++slot == stages) { slot = 0; phase ^= 1u; }
        }
    } else if (role == 4) {
        // ---- products: the scores of a block while the probabilities of the block before are made
        const unsigned idesc_s = (2u << 4) | (1u << 7) | (1u << 10) | (((unsigned)S::NQ >> 3) << 17) | ((128u >> 4) << 24);
        const unsigned idesc_o = (2u << 4) | (1u << 7) | (1u << 15) | (1u << 16) | (((unsigned)S::NP >> 3) << 17) | (((unsigned)D >> 4) << 24);   // tokens are rows of both operands
        const unsigned hi_d = (unsigned)(make_smem_desc(0u, D) >> 32), hi_p = (unsigned)(make_smem_desc(0u, S::NP) >> 32);
        const unsigned q_lo = ((base + S::Q) & 0x3ffffu) >> 4, p_lo = ((base + at_group) & 0x3ffffu) >> 4, ring = ((base + at_group + S::RING) & 0x3ffffu) >> 4;
        int slot_s = 0, slot_o = 0;
        unsigned phase_s = 0;
        auto scores = [&](int j) -> bool {
            if (!mbar_wait_warp(smem_u32(&bars.full[slot_s]), phase_s, &abort_flag, a.status, 21)) return false;
            tc_fence_after();
            if (elect_one()) {
                const unsigned k = ring + (unsigned)(slot_s * (S::STAGE / 16));
#pragma unroll
                for (int i = 0; i < D / 32; ++i) tc_mma_i8_lohi(tmem + (unsigned)((j & 1) * S::S_COLUMNS), k + 2 * i, q_lo + 2 * i, hi_d, idesc_s, i > 0);
                tc_commit(smem_u32(&bars.s_full[j & 1]));
            }
            __syncwarp();
            if (++slot_s == stages) { slot_s = 0; phase_s ^= 1u; }
            return true;
        };
        bool ok = blocks == 0 || (mbar_wait_issuer(smem_u32(&q_full), 0, &abort_flag, a.status, 22) && scores(0));
        for (int j = 0; j < blocks && ok; ++j) {
            if (j + 1 < blocks) ok = scores(j + 1);
            ok = ok && mbar_wait_warp(smem_u32(&bars.p_full[j & 1]), (unsigned)(j >> 1) & 1u, &abort_flag, a.status, 23);
            if (!ok) break;
            tc_fence_after();
            const unsigned keep = *(volatile unsigned*)&fresh[j & 1] ? 0u : 1u;
            if (elect_one()) {
                const unsigned v = ring + (unsigned)(slot_o * (S::STAGE / 16) + ROWS_BLOCK * D / 16), p = p_lo + (unsigned)((j & 1) * (ROWS_BLOCK * S::NP / 16));
#pragma unroll
                for (int i = 0; i < ROWS_BLOCK / 32; ++i)
                    tc_mma_i8_mixed(o_tmem, v + (unsigned)(i * 32 * D / 16), p + (unsigned)(i * 32 * S::NP / 16), hi_d, hi_p, idesc_o, i > 0 ? 1u : keep);
                tc_commit(smem_u32(&bars.o_done[slot_o]));
            }
            __syncwarp();
            if (++slot_o == stages) slot_o = 0;
        }
    } else {
        // ---- a token of each block, later an element of the head, to a thread; its warp's quarter of TMEM
        const int quad = warp & 3, place = quad * 32 + lane;
        if (group == 0) {
            // queries: TPR threads bring a row, D / TPR values each
            constexpr int TPR = R < 8 ? 16 : 128 / R, V = D / TPR;
            const int r = tid / TPR, part = tid % TPR, row = row0 + r, t = row / a.group, h = row - t * a.group;
            const T* const q = (const T*)a.q + (size_t)(s.first_row + t) * a.q_stride + (size_t)(head * a.group + h) * D + part * V;
            float v[V];
#pragma unroll
            for (int i = 0; i < V / 4; ++i) {
                uint2 w = make_uint2(0, 0);
                if (r < R && r < rows) w = *reinterpret_cast<const uint2*>(q + 4 * i);
                const float2 x = Elem<T>::unpack2(w.x), y = Elem<T>::unpack2(w.y);
                v[4 * i] = x.x; v[4 * i + 1] = x.y; v[4 * i + 2] = y.x; v[4 * i + 3] = y.y;
            }
            unsigned largest = 0;
#pragma unroll
            for (int i = 0; i < V; ++i) largest = max(largest, magnitude(v[i]));
#pragma unroll
            for (int o = 1; o < TPR; o *= 2) largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, o));
            // the row's largest value becomes 2^20 .. 2^22: what is no smaller than a 2^-12 of it keeps all of its bits
            const int exponent = min(max((int)(largest >> 23), 1), 253);
            const float up = __int_as_float((254 - exponent) << 23);
            if (r < R) {
                if (part == 0) row_scales[r] = largest >= 0x7f800000u ? __int_as_float(0x7fffffff) : a.scale_log2 * (__int_as_float(exponent << 23) * 0x1p-20f);
                unsigned digits[3][V / 4];
#pragma unroll
                for (int i = 0; i < V / 4; ++i) {
                    digits[0][i] = digits[1][i] = digits[2][i] = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int whole = __float2int_rn(v[4 * i + e] * up * 1048576.0f), low = (int)(int8_t)whole, rest = (whole - low) >> 8, middle = (int)(int8_t)rest;
                        digits[2][i] |= ((unsigned)low & 0xffu) << (8 * e);
                        digits[1][i] |= ((unsigned)middle & 0xffu) << (8 * e);
                        digits[0][i] |= ((unsigned)((rest - middle) >> 8) & 0xffu) << (8 * e);
                    }
                }
#pragma unroll
                for (int d = 0; d < 3; ++d)
#pragma unroll
                    for (int i = 0; i < V / 4; ++i)
                        *reinterpret_cast<unsigned*>(smem + S::Q + swz_off(3 * r + d, part * V + 4 * i, D)) = digits[d][i];
            }
            for (int i = tid; i < (S::NQ - 3 * R) * D / 4; i += 128) *reinterpret_cast<unsigned*>(smem + S::Q + 3 * R * D + 4 * i) = 0;
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&q_full));
        }
        unsigned char* const p_smem = smem + at_group;
        if (4 * R < S::NP)                  // columns that no row has
            for (int i = place; i < 2 * S::NP * ROWS_BLOCK / 16; i += 128) *reinterpret_cast<uint4*>(p_smem + 16 * i) = make_uint4(0, 0, 0, 0);
        bool ok = mbar_wait_warp(smem_u32(&q_full), 0, &abort_flag, a.status, 29);

        // from: the maximum that a row's probabilities are taken against
        float row_scale[R], from[R], sum[R], acc[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            row_scale[r] = row_scales[r];
            from[r] = ROWS_NONE;
            acc[r] = 0.0f;
            const int pos = s.begin + (row0 + r) / a.group;
            sum[r] = place == 0 && (a.causal ? pos : s.length - 1) >= capacity ? __int_as_float(0x7fffffff) : 0.0f;
        }
        const unsigned lanes = (unsigned)(quad * 32) << 16;
        int pending = 0;
        // slots and phases of the block before and of the one before that
        int slot1 = 0, slot2 = 0;
        unsigned phase1 = 0, phase2 = 0;
        auto flush = [&]() {                // the sums of the blocks so far, out of TMEM
            unsigned x[4 * R];
            tc_fence_after();
            tc_ld_into<4 * R>(o_tmem + lanes, x);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float high = fmaf((float)(int)x[4 * r + 3], 256.0f, (float)(int)x[4 * r + 2]), low = fmaf((float)(int)x[4 * r + 1], 256.0f, (float)(int)x[4 * r]);
                acc[r] = fmaf(fmaf(high, 65536.0f, low), 1.0f / ROWS_ONE, acc[r]);
            }
            pending = 0;
        };
        // a token's page number is asked for two blocks ahead and its scales one, each used an iteration after it was asked for
        const int token0 = j_lo * ROWS_BLOCK + place;
        auto number_of = [&](int j) -> int {
            const int token = token0 + j * ROWS_BLOCK;
            return j < blocks && token < hi ? a.c.table[(size_t)b * a.c.row + (token >> a.log_page)] : 0;
        };
        float k_next = 0.0f, v_next = 0.0f;
        bool bad_next = false;
        auto scales_of = [&](int number) {
            bad_next = (unsigned)number >= (unsigned)a.c.nb_pages;
            const size_t at = (size_t)(bad_next ? 0 : number) * a.c.heads + head;
            k_next = a.c.k_scales[at];
            v_next = a.c.v_scales[at];
        };
        if (blocks > 0) scales_of(number_of(0));
        int number_next = number_of(1);
        // (a wait that gave up ends no loop: the four warps meet at barriers without a limit, and the rest of the loop waits for nothing)
#pragma unroll 1
        for (int j = 0; j < blocks; ++j) {
            const int token = token0 + j * ROWS_BLOCK, j0 = token - place;
            const float k_scale = bad_next ? __int_as_float(0x7fffffff) : k_next, v_scale = v_next <= TOKEN_TINY ? KV_NOTHING : v_next;   // (all codes are 0 there)
            if (j + 1 < blocks) scales_of(number_next);
            number_next = number_of(j + 2);
            const float v_log = __log2f(v_scale), v_inverse = exp2_approx(-v_log);
            const bool whole = j0 + ROWS_BLOCK <= s.length && (!a.causal || (j0 + ROWS_BLOCK - 1 <= s.begin + t_first && (!a.window || j0 > s.begin + t_last - a.window)));
            ok = ok && mbar_wait_warp(smem_u32(&bars.s_full[j & 1]), (unsigned)(j >> 1) & 1u, &abort_flag, a.status, 25);
            tc_fence_after();
            unsigned x[(3 * R + 7) / 8 * 8];
            tc_ld_into<(3 * R + 7) / 8 * 8>(tmem + lanes + (unsigned)((j & 1) * S::S_COLUMNS), x);
            float t[R], over = 0.0f;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float whole_number = float_of(x[3 * r], 65536.0f) + (float_of(x[3 * r + 1], 256.0f) + float_of(x[3 * r + 2], 1.0f));
                t[r] = fmaf(whole_number, k_scale * row_scale[r], v_log);
            }
            if (!whole) {
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const int pos = s.begin + (row0 + r) / a.group;
                    if (!(token < s.length && (!a.causal || (token <= pos && (!a.window || token > pos - a.window))))) t[r] = -INFINITY;
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r) over = fmaxf(over, t[r] - from[r]);
            // below that room nothing leaves the digits
            const bool move = any_of_128(group, over > ROWS_ROOM);
            if (move) {
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    float m = t[r];
#pragma unroll
                    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                    if (lane == 0) tops[group][quad][r] = m;
                }
                any_of_128(group, false);
            }
            if (pending && (move || pending == ROWS_FLUSH)) {
                ok = ok && mbar_wait_warp(smem_u32(&bars.o_done[slot1]), phase1, &abort_flag, a.status, 26);
                flush();
            }
            if (move) {
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const float m = fmaxf(fmaxf(fmaxf(tops[group][0][r], tops[group][1][r]), fmaxf(tops[group][2][r], tops[group][3][r])), from[r]);
                    const float fade = exp2_approx(from[r] - m);
                    from[r] = m;
                    sum[r] *= fade;
                    acc[r] *= fade;
                }
            }
            unsigned digits[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float p = exp2_approx(t[r] - from[r]);
                if (whole || p != 0.0f) sum[r] = fmaf(p, v_inverse, sum[r]);     // (the scale of a page that a row does not see may be anything)
                digits[r] = __float2uint_rn(p * ROWS_ONE);                       // its bytes are the digits, the lowest first
            }
            // the place is free when the products of the block before the last are through
            if (j >= 2) ok = ok && mbar_wait_warp(smem_u32(&bars.o_done[slot2]), phase2, &abort_flag, a.status, 28);
#pragma unroll
            for (int r = 0; r < R; r += 4)
                *reinterpret_cast<uint4*>(p_smem + (j & 1) * S::NP * ROWS_BLOCK + swz_off(place, 4 * r, S::NP)) = make_uint4(digits[r], digits[r + 1], digits[r + 2], digits[r + 3]);
            if (place == 0) fresh[j & 1] = pending == 0;
            ++pending;
            fence_async_smem();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bars.p_full[j & 1]));
            if (j >= 1) {
                slot2 = slot1;
                phase2 = phase1;
                if (++slot1 == stages) { slot1 = 0; phase1 ^= 1u; }
            }
        }
        if (pending) {
            ok = ok && mbar_wait_warp(smem_u32(&bars.o_done[slot1]), phase1, &abort_flag, a.status, 27);
            flush();
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int o = 16; o; o >>= 1) sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], o);
            if (lane == 0) sums[group][quad][r] = sum[r];
            if (place == 0) own_top[group][r] = from[r];
        }
        // every product of the group is through: the part goes where its ring was.  Heads of 64 take the first 16 lanes of each 32 of TMEM.
        float* const own = (float*)(smem + at_group + S::RING);
        any_of_128(group, false);
        if (D == 128 || lane < 16) {
#pragma unroll
            for (int r = 0; r < R; ++r) own[r * S::PITCH + (D == 128 ? place : quad * 16 + lane)] = acc[r];
        }
        if (place < R) own_sum[group][place] = sums[group][0][place] + sums[group][1][place] + sums[group][2][place] + sums[group][3][place];
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 4) {        // before the other blocks are waited for (see TMEM_BYTES)
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_slot), "r"((unsigned)(S::COLUMNS * GROUPS)) : "memory");
    }
    if (ranks > 1) cluster_sync();
    // every block of the cluster finishes a share of the outputs
    const int there = min(max(rows, 0), R);
    for (int i = (int)rank * ROWS_GROUP * GROUPS + tid; i < there * (D / 4); i += (int)ranks * ROWS_GROUP * GROUPS) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        float m = ROWS_NONE;
        for (unsigned k = 0; k < ranks; ++k)
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) m = fmaxf(m, ld_cluster(map_to_rank(smem_u32(&own_top[g][r]), k)));
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float l = 0.0f;
        for (unsigned k = 0; k < ranks; ++k)
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                const float f = exp2_approx(ld_cluster(map_to_rank(smem_u32(&own_top[g][r]), k)) - m);
                const float4 x = ld_cluster4(map_to_rank(base + (unsigned)(S::GROUP + g * S::group_bytes(stages) + S::RING + (r * S::PITCH + d) * 4), k));
                o.x = fmaf(x.x, f, o.x); o.y = fmaf(x.y, f, o.y); o.z = fmaf(x.z, f, o.z); o.w = fmaf(x.w, f, o.w);
                l = fmaf(ld_cluster(map_to_rank(smem_u32(&own_sum[g][r]), k)), f, l);
            }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const int row = row0 + r, t = row / a.group, h = row - t * a.group;
        T* const out = (T*)a.out + (size_t)(s.first_row + t) * a.out_stride + (size_t)(head * a.group + h) * D + d;
        *reinterpret_cast<uint2*>(out) = make_uint2(Elem<T>::pack2(o.x * inv, o.y * inv), Elem<T>::pack2(o.z * inv, o.w * inv));
    }
    if (ranks > 1) cluster_sync();   // no block leaves while another reads its part
}

template <typename T, int D, int R, int GROUPS>
static cudaError_t launch_rows_of(const CUtensorMap& k_map, const CUtensorMap& v_map, const AttendArgs& a, int split, int stages, int sequences, cudaStream_t s)
{
    static SmemLimitSet set, wide;
    typedef RowsSmem<D, R, GROUPS> S;
    cudaError_t e = raise_smem_limit(kv_attention_rows_kernel<T, D, R, GROUPS>, set, S::bytes(S::MOST));
    if (e != cudaSuccess) return e;
    if (split > 8) {
        int dev = 0;
        cudaGetDevice(&dev);
        const unsigned long long bit = dev >= 0 && dev < 64 ? 1ull << dev : 0ull;
        if (!(wide.load(std::memory_order_relaxed) & bit)) {
            e = cudaFuncSetAttribute(kv_attention_rows_kernel<T, D, R, GROUPS>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (e != cudaSuccess) return e;
            wide.fetch_or(bit, std::memory_order_relaxed);
        }
    }
    const long long tiles = ((long long)a.c.max_new * a.group + R - 1) / R;
    return launch_token(kv_attention_rows_kernel<T, D, R, GROUPS>, dim3((unsigned)split, (unsigned)(tiles * a.c.heads), (unsigned)sequences), ROWS_GROUP * GROUPS,
                        S::bytes(stages < S::MOST ? stages : S::MOST), split, s, k_map, v_map, a, stages < S::MOST ? stages : S::MOST);
}

template <typename T, int D, int R>
static cudaError_t launch_rows(const CUtensorMap& k_map, const CUtensorMap& v_map, const AttendArgs& a, int sequences, cudaStream_t s)
{
    const long long rows = (long long)a.c.max_new * a.group, blocks = (rows + R - 1) / R * a.c.heads * sequences;
    const long long steps = attend_steps(a);
    // Streams of tokens to a tile: as many as give each multiprocessor two, at least two blocks to a stream.  One stream of 128 x 128 codes takes about 1300
    // cycles a block, half of what a multiprocessor's share of the memory takes for two.  Measured (streams to a tile: us): 8 tiles of 65000 tokens 4: 93,
    // 8: 51, 16: 33; 32 tiles of 15800 (heads of 64) 4: 31, 8: 21, 16: 36; 128 tiles of 2000 1: 19.6, 2: 14.0, 4: 19.0; 384 tiles of 8000 and
    // fewer 1: 91, 2: 81, 4: 90.  Two streams share a block (14.0 and 81 us; as clusters of two blocks 14.8 and 84), more are clusters.
    // Tiles of 16 rows have a multiprocessor to themselves (their share of TMEM takes 115 KB of shared memory); sixteen such neighbours are hard to come
    // by: 8 tiles of 4000 tokens 22.6 us as clusters of 16, 13.1 as clusters of 8.
    int streams = 1;
    if (R == 16) streams = attend_streams(blocks, steps, 1, 8);
    else while (streams < 16 && (blocks * streams * 2 <= 2 * token_sms() || (streams == 1 && steps >= 16)) && streams * 2 * 2 <= steps) streams *= 2;
    const int groups = R < 16 && streams == 2 ? 2 : 1, split = streams / groups;
    // (a slot is filled again two blocks later: three at least, unless there are no more blocks than slots)
    const long long per = (steps + split * groups - 1) / (split * groups);
    const int stages = per < 8 ? (int)per : 8;
    if (R < 16 && groups == 2) return launch_rows_of<T, D, R < 16 ? R : 8, 2>(k_map, v_map, a, split, stages, sequences, s);
    return launch_rows_of<T, D, R, 1>(k_map, v_map, a, split, stages, sequences, s);
}

template <typename T, int D>
static cudaError_t launch_rows_by_count(const CUtensorMap& k_map, const CUtensorMap& v_map, const AttendArgs& a, int sequences, cudaStream_t s)
{
    const long long rows = (long long)a.c.max_new * a.group;
    if (rows <= 4) return launch_rows<T, D, 4>(k_map, v_map, a, sequences, s);
    if (rows <= 8) return launch_rows<T, D, 8>(k_map, v_map, a, sequences, s);
    return launch_rows<T, D, 16>(k_map, v_map, a, sequences, s);
}

template <typename T> struct Half { static constexpr bool value = false; };
template <> struct Half<__half> { static constexpr bool value = true; };

template <typename T>
static cudaError_t launch_attention(const n2d2b_kv_cache& cache, const AttendArgs& a, int sequences, cudaStream_t s)
{
    // Tiles of 16 rows or of 256: a step of 128 tokens takes the former about 2000 cycles and the latter 5000 (7000 with one of its halves empty, which
    // then waits for its own products); 12000 and 15000 go with the blocks themselves.  Measured (us, 16 rows a tile / 256): 8 sequences of 8 new tokens of 4
    // heads over 4000 38 / 70, 1 of 12 over 20000 50 / 92, 8 of 12 over 4000 44 / 66, 32 of 16 over 600 57 / 40, 32 of 32 over 1000 133 / 60, 8 of 64 of one
    // head over 64 15 / 9.
    const long long rows = (long long)a.c.max_new * a.group, key_heads = (long long)sequences * a.c.heads, steps = attend_steps(a);
    if (rows > 16 || a.c.heads > 65535) {
        const long long few = (rows + 15) / 16 * key_heads, many = (rows + 255) / 256 * key_heads;
        const int few_streams = attend_streams(few, steps, 1, 8), many_streams = attend_streams(many, steps, 2, 8);
        const double sms = token_sms(), few_waves = few * few_streams / sms, many_waves = many * many_streams / sms;
        const double few_cycles = (few_waves > 1 ? few_waves : 1) * ((steps + few_streams - 1) / few_streams * 2000.0 + 12000);
        const double many_cycles = (many_waves > 1 ? many_waves : 1) * ((steps + many_streams - 1) / many_streams * (rows > 128 ? 5000.0 : 7000.0) + 15000);
        if (many_cycles < few_cycles || (rows + 15) / 16 * a.c.heads > 65535) return launch_attention_prompt(a, cache.head_size, Half<T>::value, sequences, s);
    }
    CUtensorMap k_map, v_map;
    const unsigned long long lines = (unsigned long long)cache.nb_pages * cache.nb_heads * cache.page_tokens;
    const unsigned box = cache.page_tokens;
    const CUtensorMapSwizzle swizzle = cache.head_size == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    if (!token_byte_map(&k_map, cache.k, cache.head_size, lines, cache.head_size, cache.head_size, box, swizzle)
        || !token_byte_map(&v_map, cache.v, cache.head_size, lines, cache.head_size, cache.head_size, box, swizzle))
        return cudaErrorInvalidValue;
    return cache.head_size == 64 ? launch_rows_by_count<T, 64>(k_map, v_map, a, sequences, s) : launch_rows_by_count<T, 128>(k_map, v_map, a, sequences, s);
}

}  // namespace n2d2b

extern "C" int n2d2b_kv_attention(int device, const n2d2b_kv_cache* cache, const n2d2b_kv_batch* batch, const n2d2b_attention* attention, n2d2b_stream stream)
{
    using namespace n2d2b;
    AttendArgs a;
    if (int rc = kv_check(cache, batch, a.c)) return rc;
    if (!attention) return set_error(N2D2B_ERR_INVALID, "attention must not be NULL");
    const n2d2b_attention& d = *attention;
    if (d.dtype != N2D2B_F16 && d.dtype != N2D2B_BF16) return set_error(N2D2B_ERR_INVALID, "dtype must be N2D2B_F16 or N2D2B_BF16 (got %d)", d.dtype);
    if (d.nb_query_heads < 1 || d.nb_query_heads % cache->nb_heads)
        return set_error(N2D2B_ERR_INVALID, "nb_query_heads must be a multiple of the cache's %d heads (got %d)", cache->nb_heads, d.nb_query_heads);
    if (d.window < 0 || (d.window > 0 && !d.causal)) return set_error(N2D2B_ERR_INVALID, "a window must not be negative and needs causal attention");
    if (!(d.scale > -INFINITY && d.scale < INFINITY)) return set_error(N2D2B_ERR_INVALID, "scale must be finite");
    if (batch->nb_sequences == 0 || batch->nb_tokens == 0 || a.c.max_new == 0) return 0;
    if (!d.q || !d.out) return set_error(N2D2B_ERR_INVALID, "q and out must not be NULL");
    const int64_t width = (int64_t)d.nb_query_heads * cache->head_size;
    a.q_stride = d.q_stride ? d.q_stride : width;
    a.out_stride = d.out_stride ? d.out_stride : width;
    if (a.q_stride < width || a.q_stride % 8 || a.out_stride < width || a.out_stride % 8)
        return set_error(N2D2B_ERR_INVALID, "strides must be 0 or multiples of 8 of at least %lld", (long long)width);
    if (!token_aligned(d.q, 16) || !token_aligned(d.out, 16)) return set_error(N2D2B_ERR_INVALID, "q and out must start on 16 bytes");
    a.group = d.nb_query_heads / cache->nb_heads;
    const long long rows = (long long)a.c.max_new * a.group;
    if (rows > (1 << 30) || (rows + 255) / 256 * cache->nb_heads * batch->nb_sequences >= (1ll << 27))
        return set_error(N2D2B_ERR_TOO_LARGE, "max_new x query heads (x nb_sequences) exceeds what one call takes: 2^30 rows of a key head, 2^27 tiles of 256 of them");
    a.q = d.q; a.out = d.out;
    a.scale_log2 = d.scale * 1.4426950408889634f;
    a.causal = d.causal ? 1 : 0;
    a.window = (int64_t)d.window < (int64_t)batch->pages_per_sequence * cache->page_tokens ? d.window : 0;
    a.log_page = cache->page_tokens == 16 ? 4 : cache->page_tokens == 32 ? 5 : cache->page_tokens == 64 ? 6 : 7;
    const TokenDevice on(device);
    if (on.err != cudaSuccess) return set_error(N2D2B_ERR_CUDA, "device %d is not usable: %s", device, cudaGetErrorString(on.err));
    a.status = token_status_word();
    if (!a.status) return set_error(N2D2B_ERR_CUDA, "the status word of the token operators has no address on device %d", device);
    cudaError_t e;
    if (d.dtype == N2D2B_F16) e = launch_attention<__half>(*cache, a, batch->nb_sequences, (cudaStream_t)stream);
    else e = launch_attention<__nv_bfloat16>(*cache, a, batch->nb_sequences, (cudaStream_t)stream);
    if (e != cudaSuccess) return set_error(N2D2B_ERR_CUDA, "attention launch failed: %s", cudaGetErrorString(e));
    return 0;
}
