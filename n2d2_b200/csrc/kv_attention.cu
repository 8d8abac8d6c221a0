// Attention over the paged 8-bit cache.
//
//   s_j = scale * sK(page of j) * (q . k_j),   out = (sum_j e^(s_j) sV(page of j) v_j) / (sum_j e^(s_j))      over visible j
//
// in one pass over the tokens, with the running maximum of t_j = s_j log2(e) + log2 sV(page of j): the values' scales ride in the
// exponent, so that p_j = 2^(t_j - max) is at most 1 whatever the scales are and enters the second product in 16 bits; the softmax's sum
// adds p_j / sV(page of j).
//
// kv_attention_rows_kernel: 8 or 16 rows (new token x query head of one key head) a tile, for few rows: bound by reading the cache.
// Codes become 16-bit floats in registers (bytes spliced into 1024 + u, minus 1152: exact) on their way into mma.m16n8k16; the products'
// inner indices are permuted so that a thread's operands are consecutive bytes of a token.  Every warp streams 32 tokens at a
// time through a ring of its own by TMA and keeps its own maximum, sums and output; the tokens of a sequence are split over the
// warps of a cluster of up to 16 blocks, whose parts are joined through distributed shared memory at the end, so nothing has to be kept in
// memory between kernels.
#include <cstdio>
#include <cstring>
#include "kv_common.cuh"

namespace n2d2b {

__device__ __forceinline__ void mma_f16(float* d, const unsigned* a, unsigned b0, unsigned b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 lds128(unsigned addr)
{
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint2 lds64(unsigned addr)
{
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
    return v;
}
static constexpr int ROWS_UNIT = 32;
template <int D, int NT, int WARPS> struct RowsSmem {
    static constexpr int STAGES = 256 / D;
    static constexpr int STAGE = 2 * ROWS_UNIT * D;                    // keys, then values
    static constexpr int RING = WARPS * STAGES * STAGE;
    static constexpr int ROWS = 8 * NT;
    static constexpr int PITCH = D + 4;                                // floats of a row of a part
    static constexpr int PART = ROWS * PITCH;
    static constexpr int BYTES = RING + 1024;                          // the parts take the ring's place
    static_assert(((WARPS + 1) * PART + 4 * WARPS * ROWS) * 4 <= RING, "parts fit in the ring");
};

// 8 x 8 halves, transposed across the warp
__device__ __forceinline__ unsigned transpose8(unsigned v)
{
    unsigned r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// Tokens are the M side of both products (16 to an MMA), rows the N side: 8 rows cost no more than they need, and a tile of NT * 8 rows shares
// the widening of the codes.  S^T = K Q^T comes out with a thread holding two rows of a token; as halves and transposed across the warp it
// is the operand of O^T = V^T P^T.
template <typename T, int D, int NT, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 12 / WARPS) kv_attention_rows_kernel(const __grid_constant__ CUtensorMap k_map,
                                                                                   const __grid_constant__ CUtensorMap v_map, const AttendArgs a)
{
    typedef RowsSmem<D, NT, WARPS> S;
    unsigned char* const smem = (unsigned char*)(((uintptr_t)dyn_smem() + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) unsigned long long full[WARPS][S::STAGES];
    __shared__ int abort_flag;
    pdl_launch_dependents();
    if (threadIdx.x == 0) {
        prefetch_tensor_map(&k_map);
        prefetch_tensor_map(&v_map);
        for (int i = 0; i < WARPS * S::STAGES; ++i) mbar_init(smem_u32(&full[0][0]) + 8 * i, 1);
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    pdl_wait();

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c4 = lane & 3;
    const int b = blockIdx.z, head = blockIdx.y % a.c.heads, row0 = (int)(blockIdx.y / a.c.heads) * S::ROWS;
    const unsigned rank = cluster_rank(), ranks = cluster_size();
    const KvSequence s = kv_sequence(a.c, b);
    const int rows = s.count * a.group - row0;          // rows of the tile that exist
    if (rows <= 0) return;                              // (the whole cluster)

    // what the tile's rows see
    const int t_first = row0 / a.group, t_last = min(row0 + S::ROWS - 1, s.count * a.group - 1) / a.group;
    int lo = 0, hi = s.length;
    if (a.causal) {
        hi = min(hi, s.begin + t_last + 1);
        if (a.window) lo = max(0, s.begin + t_first + 1 - a.window);
    }
    const int capacity = a.c.row << a.log_page;         // tokens behind the row of the table are nowhere
    hi = min(hi, capacity);
    const int u_lo = lo / ROWS_UNIT, u_hi = hi > lo ? (hi + ROWS_UNIT - 1) / ROWS_UNIT : u_lo;
    const int per_rank = (u_hi - u_lo + (int)ranks - 1) / (int)ranks;
    const int u0 = u_lo + (int)rank * per_rank, u1 = min(u0 + per_rank, u_hi);

    // this warp's units: u0 + warp, + WARPS, ...
    const int mine = u1 - u0 > warp ? (u1 - u0 - warp + WARPS - 1) / WARPS : 0;
    const unsigned ring = smem_u32(smem) + (unsigned)(warp * S::STAGES * S::STAGE);
    const unsigned bars = smem_u32(&full[warp][0]);
    const bool small = a.log_page == 4;                 // a unit is two pages
    struct Pages { PageOf first, second; } held, ahead; // lane i: of unit i of this and of the next 32 of this warp
    auto fetch_pages = [&](Pages& to, int from) {
        const int i = from + lane, token = (u0 + warp + i * WARPS) * ROWS_UNIT;
        to.first = page_of(a.c, b, head, token >> a.log_page, i < mine);
        to.second = to.first;
        if (small) to.second = page_of(a.c, b, head, (token >> 4) + 1, i < mine && token + 16 < hi);
    };
    auto issue = [&](const Pages& from, int i) {        // unit i into its slot; every lane calls
        const int n0 = __shfl_sync(0xffffffffu, from.first.number, i & 31), n1 = __shfl_sync(0xffffffffu, from.second.number, i & 31);
        if (elect_one()) {
            const unsigned bar = bars + 8u * (unsigned)(i % S::STAGES), dst = ring + (unsigned)((i % S::STAGES) * S::STAGE);
            const int token = (u0 + warp + i * WARPS) * ROWS_UNIT, page = 1 << a.log_page;
            const int y0 = (n0 * a.c.heads + head) * page + (token & (page - 1));
            mbar_expect_tx(bar, S::STAGE);
            tma_load_2d(dst, &k_map, bar, 0, y0);
            tma_load_2d(dst + ROWS_UNIT * D, &v_map, bar, 0, y0);
            if (small) {
                const int y1 = (n1 * a.c.heads + head) * page;
                tma_load_2d(dst + 16 * D, &k_map, bar, 0, y1);
                tma_load_2d(dst + ROWS_UNIT * D + 16 * D, &v_map, bar, 0, y1);
            }
        }
        __syncwarp();
    };
    if (mine > 0) fetch_pages(held, 0);
    for (int i = 0; i < S::STAGES - 1 && i < mine; ++i) issue(held, i);

    // queries: lanes of a quad hold row g of each 8, a quarter of its values each
    float scale_of_g[NT];
    unsigned qb[NT][D / 16][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int row = row0 + 8 * n + g, t = row / a.group, h = row - t * a.group;
        float v[D / 4];
        unsigned top = 0;
        const T* q = (const T*)a.q + (size_t)(s.first_row + t) * a.q_stride + (size_t)(head * a.group + h) * D + c4 * (D / 4);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (8 * n + g < rows) w = *reinterpret_cast<const uint4*>(q + 8 * i);
            Elem<T>::unpack(w, v + 8 * i);
        }
#pragma unroll
        for (int i = 0; i < D / 4; ++i) top = max(top, magnitude(v[i]));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // a power of two brings the row's largest value into [1, 4): exact, and a row of any size fits in halves
        const int exponent = min((int)(top >> 23), 253);
        const bool scaled = exponent > 0 && top < 0x7f800000u;
        const float up = scaled ? __int_as_float((254 - exponent) << 23) : 1.0f;
        scale_of_g[n] = a.scale_log2 * (scaled ? __int_as_float(exponent << 23) : 1.0f);
        // the order of the products' inner index is that of a word's bytes 0, 2 and 1, 3 (see widen)
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
            qb[n][k][0] = pack_half2(v[4 * k] * up, v[4 * k + 2] * up);
            qb[n][k][1] = pack_half2(v[4 * k + 1] * up, v[4 * k + 3] * up);
        }
    }
    // a thread's rows are 2 c4 and 2 c4 + 1 of each 8
    int pos[NT][2];
    float row_scale[NT][2], top[NT][2], sum[NT][2];
    float acc[D / 16][NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            row_scale[n][r] = __shfl_sync(0xffffffffu, scale_of_g[n], (2 * c4 + r) * 4);
            pos[n][r] = s.begin + (row0 + 8 * n + 2 * c4 + r) / a.group;
            top[n][r] = -INFINITY;
            sum[n][r] = (a.causal ? pos[n][r] : s.length - 1) >= capacity && g == 0 ? __int_as_float(0x7fffffff) : 0.0f;
        }
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[d][n][e] = 0.0f;

    // offsets of a thread's operands inside a slot, as the copies swizzle them (rows of 128 bytes: chunk ^ row mod 8; of 64: chunk ^ (row / 2) mod 4)
    unsigned k_off[2], v_off[2];
    if (D == 128) {
        k_off[0] = (unsigned)(g * 128 + (((2 * c4) ^ g) << 4));
        k_off[1] = (unsigned)(g * 128 + (((2 * c4 + 1) ^ g) << 4));
        v_off[0] = (unsigned)(2 * c4 * 128 + ((g ^ (2 * c4)) << 4));
        v_off[1] = (unsigned)((2 * c4 + 1) * 128 + ((g ^ (2 * c4 + 1)) << 4));
    } else {
        k_off[0] = k_off[1] = (unsigned)(g * 64 + ((c4 ^ ((g >> 1) & 3)) << 4));
        v_off[0] = (unsigned)(2 * c4 * 64 + (((g >> 1) ^ c4) << 4) + ((g & 1) << 3));
        v_off[1] = v_off[0] + 64;
    }

    bool ok = true;
    int issued = min(S::STAGES - 1, mine);
#pragma unroll 1
    for (int i = 0; i < mine; ++i) {
        // pages of the 32 units after these, read long before they are needed
        if ((i & 31) == 0) {
            if (i) held = ahead;
            if (i + 32 < mine) fetch_pages(ahead, i + 32);
        }
        if (issued < mine) {        // into the slot that the unit before this one has left
            issue((issued >> 5) == (i >> 5) ? held : ahead, issued);
            ++issued;
        }
        const float ks[2] = {__shfl_sync(0xffffffffu, held.first.k_scale, i & 31), __shfl_sync(0xffffffffu, held.second.k_scale, i & 31)};
        const float vl[2] = {__shfl_sync(0xffffffffu, held.first.v_log, i & 31), __shfl_sync(0xffffffffu, held.second.v_log, i & 31)};
        const float vi[2] = {__shfl_sync(0xffffffffu, held.first.v_inverse, i & 31), __shfl_sync(0xffffffffu, held.second.v_inverse, i & 31)};
        const unsigned slot = ring + (unsigned)((i % S::STAGES) * S::STAGE);
        ok = mbar_wait_warp(bars + 8u * (unsigned)(i % S::STAGES), (unsigned)(i / S::STAGES) & 1u, &abort_flag, a.status, 21);
        if (!ok) break;

        float sc[2][NT][4];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[m][n][e] = 0.0f;
            unsigned w[2][D / 16];      // a token of the first and of the second 8
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int h = 0; h < D / 64; ++h) {
                    const uint4 x = lds128(slot + (unsigned)((2 * m + r) * 8 * D) + k_off[h]);
                    w[r][4 * h] = x.x; w[r][4 * h + 1] = x.y; w[r][4 * h + 2] = x.z; w[r][4 * h + 3] = x.w;
                }
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                const unsigned ka[4] = {widen_even(w[0][k]), widen_even(w[1][k]), widen_odd(w[0][k]), widen_odd(w[1][k])};
#pragma unroll
                for (int n = 0; n < NT; ++n) mma_f16(sc[m][n], ka, qb[n][k][0], qb[n][k][1]);
            }
        }
        const int j0 = (u0 + warp + i * WARPS) * ROWS_UNIT;
        const bool whole = j0 + ROWS_UNIT <= s.length && (!a.causal || (j0 + ROWS_UNIT - 1 <= s.begin + t_first && (!a.window || j0 > s.begin + t_last - a.window)));
        float best[NT][2];
        bool grown = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                best[n][r] = top[n][r];
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int j = j0 + 16 * m + 8 * e + g;
                        float v = fmaf(sc[m][n][2 * e + r], ks[m] * row_scale[n][r], vl[m]);
                        if (!whole) {
                            const bool seen = j < s.length && (!a.causal || (j <= pos[n][r] && (!a.window || j > pos[n][r] - a.window)));
                            v = seen ? v : -INFINITY;
                        }
                        sc[m][n][2 * e + r] = v;
                        best[n][r] = fmaxf(best[n][r], v);
                    }
                grown |= best[n][r] > top[n][r] + 8.0f || (top[n][r] == -INFINITY && best[n][r] > top[n][r]);
            }
        // the maximum only moves when a score is more than 2^8 above it: below that, nothing leaves 16 bits
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float m = best[n][r];
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                    const float fade = m == top[n][r] ? 1.0f : exp2_approx(top[n][r] - m);
                    top[n][r] = m;
                    sum[n][r] *= fade;
#pragma unroll
                    for (int d = 0; d < D / 16; ++d) { acc[d][n][r] *= fade; acc[d][n][2 + r] *= fade; }
                }
        }
        unsigned pb[2][NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float from[2] = {top[n][0] == -INFINITY ? 0.0f : top[n][0], top[n][1] == -INFINITY ? 0.0f : top[n][1]};
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float p[2];
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        p[r] = exp2_approx(sc[m][n][2 * e + r] - from[r]);
                        // (the scale of a page that a row does not see may be anything)
                        if (whole) sum[n][r] = fmaf(p[r], vi[m], sum[n][r]);
                        else sum[n][r] = p[r] == 0.0f ? sum[n][r] : fmaf(p[r], vi[m], sum[n][r]);
                    }
                    pb[m][n][e] = transpose8(pack_half2(p[0], p[1]));
                }
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const unsigned at = slot + (unsigned)(ROWS_UNIT * D + m * 16 * D);
            unsigned x[4][D / 32];     // four tokens, D / 8 consecutive codes of each
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const unsigned from = at + v_off[t & 1] + (unsigned)((t >> 1) * 8 * D);
                if (D == 128) {
                    const uint4 y = lds128(from);
                    x[t][0] = y.x; x[t][1] = y.y; x[t][D / 32 - 2] = y.z; x[t][D / 32 - 1] = y.w;
                } else {
                    const uint2 y = lds64(from);
                    x[t][0] = y.x; x[t][1] = y.y;
                }
            }
#pragma unroll
            for (int w = 0; w < D / 32; ++w) {
                // a word holds four codes of a token: bytes 0, 1 and 2, 3 beside those of the next token
                const unsigned a01 = __byte_perm(x[0][w], x[1][w], 0x5410), a23 = __byte_perm(x[0][w], x[1][w], 0x7632);
                const unsigned b01 = __byte_perm(x[2][w], x[3][w], 0x5410), b23 = __byte_perm(x[2][w], x[3][w], 0x7632);
                const unsigned va[4] = {widen_even(a01), widen_odd(a01), widen_even(b01), widen_odd(b01)};
                const unsigned vb[4] = {widen_even(a23), widen_odd(a23), widen_even(b23), widen_odd(b23)};
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    mma_f16(acc[2 * w][n], va, pb[m][n][0], pb[m][n][1]);
                    mma_f16(acc[2 * w + 1][n], vb, pb[m][n][0], pb[m][n][1]);
                }
            }
        }
        __syncwarp();
    }
    // copies under way (after a wait that gave up) land before the ring is given to the parts
    if (!ok)
        for (int i = 0; i < issued; ++i) mbar_wait_for(bars + 8u * (unsigned)(i % S::STAGES), (unsigned)(i / S::STAGES) & 1u, &abort_flag, a.status, 21, 1000000ull);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int o = 4; o < 32; o *= 2) sum[n][r] += __shfl_xor_sync(0xffffffffu, sum[n][r], o);
    __syncthreads();

    // parts: [warp][row][D] and, behind them, maxima and sums; then the block's own part behind those
    float* const parts = (float*)smem;
    float* const part_top = parts + WARPS * S::PART;              // [warp][row], then sums
    float* const part_sum = part_top + WARPS * S::ROWS;
    float* const own = part_sum + WARPS * S::ROWS;                // [row][PITCH]
    __shared__ float own_top[S::ROWS], own_sum[S::ROWS];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = 8 * n + 2 * c4 + r;
            float* const to = parts + warp * S::PART + row * S::PITCH + g * (D / 8);
#pragma unroll
            for (int d = 0; d < D / 16; d += 2)
                *reinterpret_cast<float4*>(to + 2 * d) = make_float4(acc[d][n][r], acc[d][n][2 + r], acc[d + 1][n][r], acc[d + 1][n][2 + r]);
            if (g == 0) {
                part_top[warp * S::ROWS + row] = top[n][r];
                part_sum[warp * S::ROWS + row] = sum[n][r];
            }
        }
    __syncthreads();
    const int there = min(rows, S::ROWS);
    for (int i = threadIdx.x; i < there * (D / 4); i += WARPS * 32) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) m = fmaxf(m, part_top[w * S::ROWS + r]);
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float l = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float t = part_top[w * S::ROWS + r];
            // a part that saw nothing but what is no number keeps it
            const float f = t == m ? 1.0f : exp2_approx(t - m);
            const float4 x = *reinterpret_cast<const float4*>(parts + w * S::PART + r * S::PITCH + d);
            o.x = fmaf(x.x, f, o.x); o.y = fmaf(x.y, f, o.y); o.z = fmaf(x.z, f, o.z); o.w = fmaf(x.w, f, o.w);
            l = fmaf(part_sum[w * S::ROWS + r], f, l);
        }
        *reinterpret_cast<float4*>(own + r * S::PITCH + d) = o;
        if (d == 0) { own_top[r] = m; own_sum[r] = l; }
    }
    if (ranks > 1) cluster_sync();
    else __syncthreads();
    // every block of the cluster finishes a share of the outputs
    for (int i = (int)rank * WARPS * 32 + (int)threadIdx.x; i < there * (D / 4); i += (int)ranks * WARPS * 32) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        const unsigned at = smem_u32(own + r * S::PITCH + d), at_top = smem_u32(own_top + r), at_sum = smem_u32(own_sum + r);
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
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const int row = row0 + r, t = row / a.group, h = row - t * a.group;
        T* const out = (T*)a.out + (size_t)(s.first_row + t) * a.out_stride + (size_t)(head * a.group + h) * D + d;
        *reinterpret_cast<uint2*>(out) = make_uint2(Elem<T>::pack2(o.x * inv, o.y * inv), Elem<T>::pack2(o.z * inv, o.w * inv));
    }
    if (ranks > 1) cluster_sync();   // no block leaves while another reads its part
}

template <typename T, int D, int NT, int WARPS>
static cudaError_t launch_rows_of(const CUtensorMap& k_map, const CUtensorMap& v_map, const AttendArgs& a, int split, int sequences, cudaStream_t s)
{
    static SmemLimitSet set, wide;
    typedef RowsSmem<D, NT, WARPS> S;
    cudaError_t e = raise_smem_limit(kv_attention_rows_kernel<T, D, NT, WARPS>, set, S::BYTES);
    if (e != cudaSuccess) return e;
    if (split > 8) {
        int dev = 0;
        cudaGetDevice(&dev);
        const unsigned long long bit = dev >= 0 && dev < 64 ? 1ull << dev : 0ull;
        if (!(wide.load(std::memory_order_relaxed) & bit)) {
            e = cudaFuncSetAttribute(kv_attention_rows_kernel<T, D, NT, WARPS>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (e != cudaSuccess) return e;
            wide.fetch_or(bit, std::memory_order_relaxed);
        }
    }
    const long long tiles = ((long long)a.c.max_new * a.group + S::ROWS - 1) / S::ROWS;
    return launch_token(kv_attention_rows_kernel<T, D, NT, WARPS>, dim3((unsigned)split, (unsigned)(tiles * a.c.heads), (unsigned)sequences), WARPS * 32, S::BYTES,
                        split, s, k_map, v_map, a);
}

template <typename T, int D>
static cudaError_t launch_rows(const CUtensorMap& k_map, const CUtensorMap& v_map, const AttendArgs& a, int sequences, cudaStream_t s)
{
    const long long rows = (long long)a.c.max_new * a.group, blocks = (rows + (rows > 8 ? 15 : 7)) / (rows > 8 ? 16 : 8) * a.c.heads * sequences;
    const long long most = a.window ? min((long long)a.c.row << a.log_page, (long long)a.window + a.c.max_new) : (long long)a.c.row << a.log_page;
    int split = 1;
    // a block of twelve warps for each multiprocessor, parts of a sequence long enough for all of them; short ones go to blocks of four
    while (split < 8 && blocks * split * 2 <= token_sms() + blocks / 2 && split * 2 * 12 * ROWS_UNIT <= most) split *= 2;
    const int warps = most >= 12 * ROWS_UNIT ? 12 : 4;
    if (rows <= 8) return warps > 4 ? launch_rows_of<T, D, 1, 12>(k_map, v_map, a, split, sequences, s) : launch_rows_of<T, D, 1, 4>(k_map, v_map, a, split, sequences, s);
    return warps > 4 ? launch_rows_of<T, D, 2, 12>(k_map, v_map, a, split, sequences, s) : launch_rows_of<T, D, 2, 4>(k_map, v_map, a, split, sequences, s);
}

template <typename T> struct Half { static constexpr bool value = false; };
template <> struct Half<__half> { static constexpr bool value = true; };

template <typename T>
static cudaError_t launch_attention(const n2d2b_kv_cache& cache, const AttendArgs& a, int sequences, cudaStream_t s)
{
    // from here on the tensor cores' tiles of 128 rows are filled well enough
    if ((long long)a.c.max_new * a.group > 64 && sequences * (long long)a.c.heads * (((long long)a.c.max_new * a.group + 255) / 256) < (1ll << 27))
        return launch_attention_prompt(a, cache.head_size, Half<T>::value, sequences, s);
    CUtensorMap k_map, v_map;
    const unsigned long long rows = (unsigned long long)cache.nb_pages * cache.nb_heads * cache.page_tokens;
    const unsigned box = cache.page_tokens < ROWS_UNIT ? 16 : ROWS_UNIT;
    const CUtensorMapSwizzle swizzle = cache.head_size == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    if (!token_byte_map(&k_map, cache.k, cache.head_size, rows, cache.head_size, cache.head_size, box, swizzle)
        || !token_byte_map(&v_map, cache.v, cache.head_size, rows, cache.head_size, cache.head_size, box, swizzle))
        return cudaErrorInvalidValue;
    return cache.head_size == 64 ? launch_rows<T, 64>(k_map, v_map, a, sequences, s) : launch_rows<T, 128>(k_map, v_map, a, sequences, s);
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
    if (((long long)a.c.max_new * a.group + 15) / 16 * cache->nb_heads > 65535)
        return set_error(N2D2B_ERR_TOO_LARGE, "max_new x query heads exceeds %d rows", 65535 * 16);
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
