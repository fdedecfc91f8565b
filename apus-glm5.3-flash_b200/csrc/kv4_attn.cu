// kv4_attn.cu — attention of a few rows a sequence over the 4-bit cache
// (apus_gcuda_kv4_attn_dev).
//
//   z_tj = scale log2(e) q_t . k_j,  m_t = max_j z_tj,
//   out_t = sum_j 2^(z_tj - m_t) v_j / sum_j 2^(z_tj - m_t)
//
// over the visible positions j, in one pass with a running maximum and sum.
// With k_j = s_jg c_jd and v_j = r_jg e_jd (scale of the group g of 32 dims
// times an integer code), both contractions run on integer codes:
//   z_tj  = sum_g s_jg (sum_{d in g} q_td c_jd)
//   out_td = sum_j (p_tj r_jg) e_jd      for d in g
// so the scales cost one multiply per position, group and query column, not
// one per element.
//
// Bound: HBM at long contexts (a position of a head is 9/8 dim bytes), with
// the unpacking of the codes close behind it, so the unpacking is what the
// layout serves.  mma.sync m16n8k16 with the cached positions (scores) or the
// dims (output) as its 16 rows and the query columns (rows of the step times
// heads of the group) as its 8: tcgen05 needs 64 rows of a tile at least and
// operands in shared memory, so the codes would have to be unpacked into it
// first, and at 1 to 16 columns its rate buys nothing.
//   * Key codes 0-15 enter as f16 subnormals: a 4-bit field at bits 0-3 or
//     4-7 of a half is c 2^-24 or c 2^-20 as it stands, so one AND unpacks two
//     codes.  The factor 16 goes into the query's fragments, the offset 8 into
//     the accumulator's start, -8 sum q, and 2^24 into the column's scale.
//   * Value codes of two positions are paired by one byte permute, OR-ed into
//     the mantissa of 128.0 (BF16) and 136 is subtracted: exact integers.
//   * Weights stay fp32 up to the product with the value's scale; p and p r are
//     rounded to BF16 (2^-9 each, any range; f16 would lose small scales).
//
// Work: a CTA of four warps takes a chunk of one sequence's positions for one
// cache head and 8 NT columns.  Every warp streams its own units of U
// positions through its own two stages (bulk copies of whole cache blocks, an
// mbarrier each) with its own maximum, sum and output tile, so the loop has no
// CTA barrier; the warps are joined once at the end.  Chunks are joined by a
// second kernel when a sequence has several.
#include <type_traits>

#include "attn_dev.h"
#include "common.cuh"
#include "pipe.cuh"

namespace apus {

__device__ int g_kv4a_err;   // attn_dev.h's codes

namespace kv4 {
constexpr int WARPS = 4, THREADS = 32 * WARPS, STAGES = 2;
// Positions of a unit: one page where a page is at most 9 KB, half a page of
// dim 256, so that two stages of four warps leave room for three CTAs an SM.
template <int D> struct Cfg {
    static constexpr int U = D == 256 ? 32 : 64;
    static constexpr int NG = D / 32;                       // scale groups
    static constexpr int KC = 0, VC = U * D / 2, KS = U * D, VS = KS + U * NG * 2;
    static constexpr int STAGE = VS + U * NG * 2;           // 72 D U / 64
    static constexpr int SMEM = WARPS * STAGES * STAGE;
};
constexpr float NEG_INF = -__builtin_huge_valf();
}  // namespace kv4

struct Kv4AttnArgs {
    Kv4View v;
    RowsView q, out;
    int group;                // query heads of a cache head
    float zscale;             // scale * log2(e)
    const uint8_t *sel;
    long sel_stride;
    int pool;
    uint64_t pool_magic;      // ceil(2^36 / pool): j / pool = j * magic >> 36 for j < 2^28, pool <= 128
    int chunk_pos, nchunk, ncb;
    float *part;
};

APUS_DEV void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
APUS_DEV void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
APUS_DEV uint32_t movmatrix(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
APUS_DEV uint32_t pack_bf16(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
APUS_DEV uint32_t pack_f16(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
APUS_DEV uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
// All ones in each half whose sign bit is set.
APUS_DEV uint32_t sign_bf16x2(uint32_t x) {
    uint32_t d;
    asm("prmt.b32 %0, %1, 0, 0xbb99;" : "=r"(d) : "r"(x));
    return d;
}
APUS_DEV float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The low four bits of each half as the BF16 integers code - 8.
APUS_DEV uint32_t code_bf16x2(uint32_t x) {
    const uint32_t u = (x & 0x000f000fu) | 0x43004300u;      // 128 + code
    uint32_t d;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(u), "r"(0x43084308u));
    return d;
}
template <int N> APUS_DEV void lds_words(uint32_t (&w)[N], const uint8_t *p) {
    if constexpr (N == 1) w[0] = *(const uint32_t *)p;
    else if constexpr (N == 2) { const uint2 t = *(const uint2 *)p; w[0] = t.x; w[1] = t.y; }
    else { const uint4 t = lds128(p); w[0] = t.x; w[1] = t.y; w[2] = t.z; w[3] = t.w; }
}

template <int D, int NT>
__global__ void __launch_bounds__(kv4::THREADS, NT == 1 ? 3 : 2) k_kv4_attn(const Kv4AttnArgs a) {
    using C = kv4::Cfg<D>;
    constexpr int NG = C::NG, U = C::U, SUB = U / 16, COLS = 8 * NT, UPP = KV4_PAGE / U;
    constexpr float NEG_INF = kv4::NEG_INF;
    extern __shared__ __align__(128) uint8_t kv4_dyn[];
    __shared__ __align__(8) uint64_t full[kv4::WARPS][kv4::STAGES];
    __shared__ int abort_flag;
    __shared__ float join_m[kv4::WARPS][COLS], join_l[kv4::WARPS][COLS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
    const int chunk = blockIdx.x, head = (int)(blockIdx.y / (unsigned)a.ncb), cb = (int)(blockIdx.y % (unsigned)a.ncb);
    const int seq = blockIdx.z;

    const Kv4Seq sq = kv4_seq(a.v.cu[seq], a.v.cu[seq + 1], a.v.len[seq], a.v.rows, a.v.max_rows, a.v.max_len);
    if (sq.bad && threadIdx.x == 0) atomicExch(&g_kv4a_err, (int)ATTN_ERR_SEQ);
    const int cols = sq.n * a.group, c0 = cb * COLS;
    if (c0 >= cols) return;
    const int cend = min(c0 + COLS, cols);
    // the positions that the first and the last row of the block see
    const int lim_row0 = sq.len - sq.n + 1;
    const int lim0 = lim_row0 + c0 / a.group, lim1 = lim_row0 + (cend - 1) / a.group;
    const int p0 = chunk * a.chunk_pos, p1 = min(p0 + a.chunk_pos, lim1);
    if (p0 >= p1 && a.nchunk > 1) return;      // the joining kernel knows it too

    if (threadIdx.x == 0) {
        for (int w = 0; w < kv4::WARPS; w++)
            for (int s = 0; s < kv4::STAGES; s++) mbar_init(&full[w][s], 1);
        abort_flag = 0;
        fence_barrier_init();
    }
    // ---- this block's units: all of them, or those an indexer kept something in
    const int units_all = p1 > p0 ? (p1 - p0 + U - 1) / U : 0;
    uint16_t *list = (uint16_t *)(kv4_dyn + C::SMEM);
    __shared__ int list_n;
    if (a.sel) {
        if (threadIdx.x == 0) list_n = 0;
        __syncthreads();
        // a unit counts when a row of the block sees one of its positions
        for (int u0 = 0; u0 < units_all; u0 += kv4::THREADS) {
            const int u = u0 + threadIdx.x;
            bool any = false;
            if (u < units_all) {
                const int b = p0 + u * U, e = min(b + U, p1);
                const long q0 = b / a.pool, q1 = min((long)((e - 1) / a.pool) + 1, a.sel_stride);
                for (int t = c0 / a.group; t <= (cend - 1) / a.group && !any; t++) {
                    const int lim = lim_row0 + t;
                    if (lim <= b) continue;
                    any = e > lim - lim % a.pool;
                    const uint8_t *sr = a.sel + (long)(sq.row0 + t) * a.sel_stride;
                    for (long i = q0; i < q1; i++) any |= sr[i] != 0;
                }
            }
            // kept in order: the sums do not depend on timing
            const unsigned bal = __ballot_sync(0xffffffffu, any);
            __shared__ int wcount[kv4::WARPS];
            if (lane == 0) wcount[warp] = __popc(bal);
            __syncthreads();
            int at = list_n;
            for (int w = 0; w < warp; w++) at += wcount[w];
            if (any) list[at + __popc(bal & ((1u << lane) - 1))] = (uint16_t)u;
            __syncthreads();
            if (threadIdx.x == 0)
                for (int w = 0; w < kv4::WARPS; w++) list_n += wcount[w];
            __syncthreads();
        }
    } else {
        __syncthreads();
    }
    const int units = a.sel ? list_n : units_all;
    volatile int *ab = &abort_flag;

    // ---- the query's fragments: column g of each n tile, dims in the order in
    // which a lane meets the key codes (dim 8 q4 + i of a group is code i)
    uint32_t Q[NT][NG][4];
    float cinit[NT][NG][2], fac[NT][2];
    int lim[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const int c = c0 + nt * 8 + g;
        const bool on = c < cols;
        const uint16_t *qp = a.q.p + (long)(sq.row0 + (on ? c / a.group : 0)) * a.q.rs +
                             (long)(head * a.group + (on ? c % a.group : 0)) * a.q.hs;
        uint4 raw[NG];
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < NG; j++) {
            raw[j] = on ? *(const uint4 *)(qp + 32 * j + 8 * q4) : make_uint4(0, 0, 0, 0);
            const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
            for (int i = 0; i < 4; i++) top = max(top, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // a power of two that brings the largest magnitude to [2^14, 2^15): f16
        // holds every BF16 within 2^-28 of it exactly, smaller ones to 2^-39 of it
        const int e = top ? max((int)(top >> 7) - 127, -100) : 0;
        const float up = __int_as_float((127 + 14 - e) << 23);
        const float f = a.zscale * __int_as_float((127 + e - 14) << 23) * 16777216.0f;
#pragma unroll
        for (int j = 0; j < NG; j++) {
            const float x[8] = {bf16lo(raw[j].x), bf16hi(raw[j].x), bf16lo(raw[j].y), bf16hi(raw[j].y),
                                bf16lo(raw[j].z), bf16hi(raw[j].z), bf16lo(raw[j].w), bf16hi(raw[j].w)};
            float qs = 0.f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float down = (i & 1) ? up * 0.0625f : up;    // codes in the high nibbles stand 16 times higher
                const uint32_t h = pack_f16(x[i] * down, x[i + 4] * down);
                Q[nt][j][i] = h;
                const float2 back = __half22float2(*(const __half2 *)&h);
                qs += (back.x + back.y) * ((i & 1) ? 16.0f : 1.0f);
            }
            qs += __shfl_xor_sync(0xffffffffu, qs, 1);
            qs += __shfl_xor_sync(0xffffffffu, qs, 2);
            qs *= -8.0f / 16777216.0f;                             // the codes' offset
            cinit[nt][j][0] = __shfl_sync(0xffffffffu, qs, 8 * q4);
            cinit[nt][j][1] = __shfl_sync(0xffffffffu, qs, 8 * q4 + 4);
        }
        fac[nt][0] = __shfl_sync(0xffffffffu, f, 8 * q4);
        fac[nt][1] = __shfl_sync(0xffffffffu, f, 8 * q4 + 4);
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int cc = min(c0 + nt * 8 + 2 * q4 + u, cols - 1);
            lim[nt][u] = lim_row0 + cc / a.group;
        }
    }

    float O[NT][D / 16][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int i = 0; i < D / 16; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) O[nt][i][e] = 0.f;
        m[nt][0] = m[nt][1] = NEG_INF;
        l[nt][0] = l[nt][1] = 0.f;
    }

    // ---- this warp's units warp, warp + WARPS, ...: lane i holds the page of
    // the i-th of the next 32
    const int mine = units > warp ? (units - warp + kv4::WARPS - 1) / kv4::WARPS : 0;
    uint8_t *stages = kv4_dyn + warp * kv4::STAGES * C::STAGE;
    const int32_t *table = a.v.table + (long)seq * a.v.table_stride;
    int my_unit = 0, my_page = -1;
    auto fetch_ids = [&](int i0) {     // units i0 .. i0 + 31 of this warp
        const int i = i0 + lane;
        my_page = -1;
        if (i < mine) {
            const int u = warp + i * kv4::WARPS;
            my_unit = a.sel ? list[u] : u;
            const int page = table[(p0 + my_unit * U) / KV4_PAGE];
            if (kv4_page_ok(page, a.v.num_pages)) my_page = page;
            else atomicExch(&g_kv4a_err, (int)ATTN_ERR_PAGE);
        }
    };
    struct Unit { int page, u; };
    auto load = [&](int i) -> Unit {   // unit i of this warp into stage i % STAGES (whole warp)
        if (i >= mine) return Unit{-1, 0};
        if ((i & 31) == 0) fetch_ids(i);
        const int page = __shfl_sync(0xffffffffu, my_page, i & 31), u = __shfl_sync(0xffffffffu, my_unit, i & 31);
        if (lane == 0) {
            uint64_t *bar = &full[warp][i % kv4::STAGES];
            uint8_t *dst = stages + (i % kv4::STAGES) * C::STAGE;
            if (page >= 0) {
                const uint8_t *src = a.v.pages + kv4_block_at(page, head, a.v.heads, D);
                mbar_arrive_expect_tx(bar, C::STAGE);
                if (UPP == 1) {
                    bulk_g2s(dst, src, C::STAGE, bar);
                } else {
                    const int h = (p0 / U + u) % UPP;
                    bulk_g2s(dst + C::KC, src + h * (U * D / 2), U * D / 2, bar);
                    bulk_g2s(dst + C::VC, src + kv4_v_codes(D) + h * (U * D / 2), U * D / 2, bar);
                    bulk_g2s(dst + C::KS, src + kv4_k_scales(D) + h * (U * NG * 2), U * NG * 2, bar);
                    bulk_g2s(dst + C::VS, src + kv4_v_scales(D) + h * (U * NG * 2), U * NG * 2, bar);
                }
            } else {
                mbar_arrive(bar);      // no page: nothing to read, the unit is left out
            }
        }
        return Unit{page, u};
    };

    // the cached position of row r of a 16-row fragment: rows 2 q, 2 q + 1 are
    // positions q, 4 + (q ^ 1), so that the quads of one shared-memory access
    // fall in different banks for keys and for values
    const int pg = (g & 1) ? 4 + ((g >> 1) ^ 1) : (g >> 1), vp1 = 4 + (q4 ^ 1);

    auto process = [&](const uint8_t *st, int pos0, auto masked_t) {
        constexpr bool MASKED = decltype(masked_t)::value;
        float z[NT][SUB][4];
        // ---- scores
#pragma unroll
        for (int sub = 0; sub < SUB; sub++) {
            const int ra = sub * 16 + pg;
            uint32_t wa[NG], wb[NG];
            constexpr int JB = NG < 4 ? NG : 4;
#pragma unroll
            for (int h = 0; h < NG / JB; h++) {
                uint32_t ta[JB], tb[JB];
                const int off = kv4_k_word(D, pg, h * JB, q4) * 4;
                lds_words<JB>(ta, st + C::KC + ra * (D / 2) + off);
                lds_words<JB>(tb, st + C::KC + (ra + 8) * (D / 2) + off);
#pragma unroll
                for (int i = 0; i < JB; i++) { wa[h * JB + i] = ta[i]; wb[h * JB + i] = tb[i]; }
            }
            uint32_t sa[NG / 2], sb[NG / 2];
            lds_words<NG / 2>(sa, st + C::KS + ra * NG * 2);
            lds_words<NG / 2>(sb, st + C::KS + (ra + 8) * NG * 2);
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < 4; e++) z[nt][sub][e] = 0.f;
#pragma unroll
            for (int j = 0; j < NG; j++) {
                const uint32_t a0 = wa[j] & 0x000f000fu, a1 = wb[j] & 0x000f000fu;
                const uint32_t a2 = wa[j] & 0x00f000f0u, a3 = wb[j] & 0x00f000f0u;
                const uint32_t xa = wa[j] >> 8, xb = wb[j] >> 8;
                const uint32_t e0 = xa & 0x000f000fu, e1 = xb & 0x000f000fu;
                const uint32_t e2 = xa & 0x00f000f0u, e3 = xb & 0x00f000f0u;
                const float fa = (j & 1) ? bf16hi(sa[j / 2]) : bf16lo(sa[j / 2]);
                const float fb = (j & 1) ? bf16hi(sb[j / 2]) : bf16lo(sb[j / 2]);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float c[4] = {cinit[nt][j][0], cinit[nt][j][1], cinit[nt][j][0], cinit[nt][j][1]};
                    mma_f16(c, a0, a1, a2, a3, Q[nt][j][0], Q[nt][j][1]);
                    mma_f16(c, e0, e1, e2, e3, Q[nt][j][2], Q[nt][j][3]);
                    z[nt][sub][0] = fmaf(fa, c[0], z[nt][sub][0]);
                    z[nt][sub][1] = fmaf(fa, c[1], z[nt][sub][1]);
                    z[nt][sub][2] = fmaf(fb, c[2], z[nt][sub][2]);
                    z[nt][sub][3] = fmaf(fb, c[3], z[nt][sub][3]);
                }
            }
        }
        // ---- running maximum: raised only when a score passes it by more than
        // 2^8, which keeps every weight and sum well inside fp32 and BF16
        bool over = false;
        uint32_t hide = 0;             // bit nt * SUB * 4 + sub * 4 + e (MASKED)
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            int tail[2] = {0, 0};      // where each column's incomplete pool begins
            const uint8_t *srow[2] = {nullptr, nullptr};
            if (MASKED && a.sel) {
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    tail[u] = lim[nt][u] > 0 ? lim[nt][u] - lim[nt][u] % a.pool : 0;
                    srow[u] = a.sel + (long)(sq.row0 + lim[nt][u] - lim_row0) * a.sel_stride;
                }
            }
#pragma unroll
            for (int sub = 0; sub < SUB; sub++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float v = z[nt][sub][e] * fac[nt][e & 1];
                    if (MASKED) {
                        const int j = pos0 + sub * 16 + (e >> 1) * 8 + pg;
                        bool see = j < lim[nt][e & 1];
                        if (a.sel && see && j < tail[e & 1]) {
                            const long pl = (long)(((uint64_t)(uint32_t)j * a.pool_magic) >> 36);
                            see = pl < a.sel_stride && srow[e & 1][pl] != 0;
                        }
                        if (!see) { v = NEG_INF; hide |= 1u << ((nt * SUB + sub) * 4 + e); }
                    }
                    z[nt][sub][e] = v;
                    over |= v > m[nt][e & 1] + 8.0f;
                }
        }
        if (__any_sync(0xffffffffu, over)) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    float x = m[nt][u];
#pragma unroll
                    for (int sub = 0; sub < SUB; sub++) x = fmaxf(x, fmaxf(z[nt][sub][u], z[nt][sub][u + 2]));
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
                    if (!(x > m[nt][u] + 8.0f)) continue;          // each column by its own scores alone
                    const float down = m[nt][u] == NEG_INF ? 0.f : ex2(m[nt][u] - x);
                    m[nt][u] = x;
                    l[nt][u] *= down;
#pragma unroll
                    for (int i = 0; i < D / 16; i++) { O[nt][i][u] *= down; O[nt][i][u + 2] *= down; }
                }
        }
        // ---- weights and output
#pragma unroll
        for (int sub = 0; sub < SUB; sub++) {
            uint32_t b0[NT], b1[NT], k0[NT], k1[NT];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float p[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float mm = m[nt][e & 1];
                    p[e] = ex2(z[nt][sub][e] - (MASKED && mm == NEG_INF ? 0.f : mm));
                    // a hidden position's weight is -0: it adds nothing to the sum, and its
                    // sign marks it below, where a NaN scale must not reach the product
                    if (MASKED && (hide >> ((nt * SUB + sub) * 4 + e) & 1)) p[e] = -0.0f;
                    l[nt][e & 1] += p[e];
                }
                b0[nt] = movmatrix(pack_bf16(p[0], p[1]));
                b1[nt] = movmatrix(pack_bf16(p[2], p[3]));
                if (MASKED) {
                    k0[nt] = ~sign_bf16x2(b0[nt]);
                    k1[nt] = ~sign_bf16x2(b1[nt]);
                }
            }
            // the four positions of this lane: 0, 1 and 2, 3 are the two pairs of a fragment
            const int r[4] = {sub * 16 + q4, sub * 16 + vp1, sub * 16 + 8 + q4, sub * 16 + 8 + vp1};
            uint32_t w[4][D / 64], s[4][NG / 2];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                lds_words<D / 64>(w[i], st + C::VC + r[i] * (D / 2) + kv4_v_word(D, (i & 1) ? vp1 : q4, g, 0) * 4);
                lds_words<NG / 2>(s[i], st + C::VS + r[i] * NG * 2);
            }
#pragma unroll
            for (int j = 0; j < NG; j++) {
                const uint32_t pick = (j & 1) ? 0x7632 : 0x5410;
                const uint32_t s01 = __byte_perm(s[0][j / 2], s[1][j / 2], pick);
                const uint32_t s23 = __byte_perm(s[2][j / 2], s[3][j / 2], pick);
                const uint32_t x = __byte_perm(w[0][j / 2], w[1][j / 2], pick);
                const uint32_t y = __byte_perm(w[2][j / 2], w[3][j / 2], pick);
                const uint32_t x0 = code_bf16x2(x), x1 = code_bf16x2(x >> 4), x2 = code_bf16x2(x >> 8),
                               x3 = code_bf16x2(x >> 12);
                const uint32_t y0 = code_bf16x2(y), y1 = code_bf16x2(y >> 4), y2 = code_bf16x2(y >> 8),
                               y3 = code_bf16x2(y >> 12);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    uint32_t w0 = mul_bf16x2(b0[nt], s01), w1 = mul_bf16x2(b1[nt], s23);
                    if (MASKED) { w0 &= k0[nt]; w1 &= k1[nt]; }
                    mma_bf16(O[nt][2 * j], x0, x1, y0, y1, w0, w1);
                    mma_bf16(O[nt][2 * j + 1], x2, x3, y2, y3, w0, w1);
                }
            }
        }
    };

    // ---- the stream
    static_assert(kv4::STAGES == 2, "the units in flight are held in two variables");
    Unit now = load(0), next = load(1);
    for (int i = 0; i < mine; i++) {
        const bool got = mbar_wait(&full[warp][i % 2], (i / 2) & 1, ab, &g_kv4a_err, (int)ATTN_ERR_WAIT);
        if (!__all_sync(0xffffffffu, got)) break;
        const uint8_t *st = stages + (i % 2) * C::STAGE;
        const int pos0 = p0 + now.u * U;
        if (now.page >= 0) {
            if (!a.sel && pos0 + U <= lim0) process(st, pos0, std::false_type{});
            else process(st, pos0, std::true_type{});
        }
        __syncwarp();
        now = next;
        next = load(i + 2);
    }

    // ---- join the warps (the stages are free once every warp is here)
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int u = 0; u < 2; u++) {
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) l[nt][u] += __shfl_xor_sync(0xffffffffu, l[nt][u], off);
            if (g == 0) {
                join_m[warp][nt * 8 + 2 * q4 + u] = m[nt][u];
                join_l[warp][nt * 8 + 2 * q4 + u] = l[nt][u];
            }
        }
    __syncthreads();
    float *jo = (float *)kv4_dyn;     // [WARPS][COLS][D]
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int u = 0; u < 2; u++) {
            float *row = jo + ((size_t)warp * COLS + nt * 8 + 2 * q4 + u) * D;
#pragma unroll
            for (int j = 0; j < NG; j++)
                *(float4 *)(row + 32 * j + 4 * g) = make_float4(O[nt][2 * j][u], O[nt][2 * j][u + 2],
                                                               O[nt][2 * j + 1][u], O[nt][2 * j + 1][u + 2]);
        }
    __syncthreads();
    const bool last = a.nchunk == 1;
    float *part = a.part + (((size_t)seq * gridDim.y + blockIdx.y) * a.nchunk + chunk) * (size_t)(COLS * (D + 2));
    for (int i = threadIdx.x; i < COLS * (D / 4); i += kv4::THREADS) {
        const int c = i / (D / 4), d = (i % (D / 4)) * 4;
        float mx = NEG_INF;
#pragma unroll
        for (int w = 0; w < kv4::WARPS; w++) mx = fmaxf(mx, join_m[w][c]);
        float sum = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kv4::WARPS; w++) {
            if (join_m[w][c] == NEG_INF && join_l[w][c] == 0.f) continue;
            const float k = ex2(join_m[w][c] - mx);
            const float4 x = *(const float4 *)(jo + ((size_t)w * COLS + c) * D + d);
            sum += join_l[w][c] * k;
            o.x += x.x * k; o.y += x.y * k; o.z += x.z * k; o.w += x.w * k;
        }
        if (!last) {
            *(float4 *)(part + 2 * COLS + c * D + d) = o;
            if (d == 0) { part[c] = mx; part[COLS + c] = sum; }
        } else if (c0 + c < cend) {
            const float inv = sum == 0.f ? 0.f : 1.0f / sum;
            uint16_t *op = a.out.p + (long)(sq.row0 + (c0 + c) / a.group) * a.out.rs +
                           (long)(head * a.group + (c0 + c) % a.group) * a.out.hs + d;
            *(uint2 *)op = make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
        }
    }
}

// Joins the chunks of one column: weights 2^(m_c - max m), in chunk order.
template <int D>
__global__ void __launch_bounds__(128) k_kv4_join(const Kv4AttnArgs a, int cols_block) {
    constexpr int L = D / 4, P = 128 / L;      // lanes over the dims, parts over the chunks
    extern __shared__ float kj_dyn[];          // [nchunk] weights, then [P][D] sums
    __shared__ float total;
    const int seq = blockIdx.z, head = blockIdx.y, c = blockIdx.x;
    const Kv4Seq sq = kv4_seq(a.v.cu[seq], a.v.cu[seq + 1], a.v.len[seq], a.v.rows, a.v.max_rows, a.v.max_len);
    const int cols = sq.n * a.group;
    if (c >= cols) return;
    const int cb = c / cols_block, cc = c % cols_block;
    const int lim1 = sq.len - sq.n + 1 + (min((cb + 1) * cols_block, cols) - 1) / a.group;
    const int n = lim1 > 0 ? min((lim1 + a.chunk_pos - 1) / a.chunk_pos, a.nchunk) : 0;
    const size_t stride = (size_t)cols_block * (D + 2);
    const float *base = a.part + (((size_t)seq * a.v.heads + head) * a.ncb + cb) * a.nchunk * stride;
    float *sums = kj_dyn + (a.nchunk + 3) / 4 * 4;
    if (threadIdx.x < 32) {
        float mx = kv4::NEG_INF;
        for (int i = threadIdx.x; i < n; i += 32) mx = fmaxf(mx, base[i * stride + cc]);
#pragma unroll
        for (int off = 16; off; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
        float sum = 0.f;
        for (int i = threadIdx.x; i < n; i += 32) {
            const float mi = base[i * stride + cc], li = base[i * stride + cols_block + cc];
            const float k = mi == kv4::NEG_INF && li == 0.f ? 0.f : ex2(mi - mx);
            kj_dyn[i] = k;
            sum += li * k;
        }
#pragma unroll
        for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        if (threadIdx.x == 0) total = sum;
    }
    __syncthreads();
    const int d = (threadIdx.x % L) * 4, part = threadIdx.x / L;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = part; i < n; i += P) {
        const float k = kj_dyn[i];
        if (k == 0.f) continue;                // a chunk that saw nothing
        const float4 x = *(const float4 *)(base + i * stride + 2 * cols_block + cc * D + d);
        o.x += x.x * k; o.y += x.y * k; o.z += x.z * k; o.w += x.w * k;
    }
    *(float4 *)(sums + part * D + d) = o;
    __syncthreads();
    if (part) return;
#pragma unroll
    for (int i = 1; i < P; i++) {
        const float4 x = *(const float4 *)(sums + i * D + d);
        o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w;
    }
    const float inv = total == 0.f ? 0.f : 1.0f / total;
    uint16_t *op = a.out.p + (long)(sq.row0 + c / a.group) * a.out.rs + (long)(head * a.group + c % a.group) * a.out.hs + d;
    *(uint2 *)op = make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
}

}  // namespace apus
using namespace apus;

namespace {

// How a batch is cut: columns of a block and positions of a chunk.
constexpr long MAX_CHUNK = 1024;              // pages: bounds the list of units in shared memory
constexpr long MAX_POS = 1l << 28;            // bounds the joining kernel's weights
struct Kv4Plan { int nt, ncb, chunk_pages, nchunk; size_t bytes; };

Kv4Plan kv4_plan(const Kv4View &v, size_t q_heads) {
    Kv4Plan p;
    const long group = (long)q_heads / v.heads, cols = group * v.max_rows;
    p.nt = cols > 8 && v.dim <= 128 ? 2 : 1;
    p.ncb = (int)((cols + 8 * p.nt - 1) / (8 * p.nt));
    const long pages = (v.max_len + KV4_PAGE - 1) / KV4_PAGE, base = (long)v.nseq * v.heads * p.ncb;
    const long slots = 148 * 3 * 4;
    long want = (base * pages + slots - 1) / slots;          // pages of a chunk for that many CTAs
    if (want < 8) want = 8;                                  // two pages a warp at least
    if (want < (pages + 255) / 256) want = (pages + 255) / 256;
    if (want > MAX_CHUNK) want = MAX_CHUNK;
    if (want > pages) want = pages > 0 ? pages : 1;
    p.chunk_pages = (int)want;
    p.nchunk = pages > 0 ? (int)((pages + want - 1) / want) : 1;
    p.bytes = p.nchunk > 1 ? (size_t)base * p.nchunk * (8 * p.nt) * (v.dim + 2) * sizeof(float) : 0;
    return p;
}

int kv4_attn_args(const char *what, const ApusKv4Cache *c, const ApusKv4Batch *b, size_t q_heads, size_t rows,
                  Kv4View *view) {
    if (kv4_check(what, c, b, rows, view)) return -1;
    if (!q_heads || q_heads > 65535 || q_heads % c->heads) {
        gcuda_set_error("%s: %zu query heads over %zu heads", what, q_heads, c->heads);
        return -1;
    }
    if (b->max_len > (size_t)MAX_POS) {
        gcuda_set_error("%s: %zu positions (at most %ld)", what, b->max_len, MAX_POS);
        return -1;
    }
    const size_t cols = q_heads / c->heads * b->max_rows;
    if (cols > (size_t)1 << 30 || ((cols + 7) / 8) * c->heads > 65535) {
        gcuda_set_error("%s: %zu rows of a sequence for %zu query heads are too many for one call", what, b->max_rows,
                        q_heads);
        return -1;
    }
    return 0;
}

template <int D, int NT>
int kv4_attn_launch(const Kv4AttnArgs &a, cudaStream_t st) {
    using C = kv4::Cfg<D>;
    const int smem = C::SMEM + (a.sel ? (a.chunk_pos / C::U) * 2 : 0);
    if (gcuda_smem_limit_once((const void *)k_kv4_attn<D, NT>, smem)) return -1;
    k_kv4_attn<D, NT><<<dim3(a.nchunk, a.v.heads * a.ncb, a.v.nseq), kv4::THREADS, smem, st>>>(a);
    if (gcuda_check(cudaGetLastError(), "kv4_attn launch")) return -1;
    if (a.nchunk == 1) return 0;
    const int jsmem = ((a.nchunk + 3) / 4 * 4 + (128 / (D / 4)) * D) * 4;
    k_kv4_join<D><<<dim3(a.group * a.v.max_rows, a.v.heads, a.v.nseq), 128, jsmem, st>>>(a, 8 * NT);
    return gcuda_check(cudaGetLastError(), "kv4_attn join launch");
}

}  // namespace

extern "C" size_t apus_gcuda_kv4_attn_workspace(const ApusKv4Cache *cache, const ApusKv4Batch *batch, size_t q_heads) {
    Kv4View v;
    if (kv4_attn_args("kv4_attn_workspace", cache, batch, q_heads, 0, &v)) return 0;
    if (!v.nseq || !v.max_rows) return 0;
    return kv4_plan(v, q_heads).bytes;
}

extern "C" int apus_gcuda_kv4_attn_dev(const ApusKv4Cache *cache, const ApusKv4Batch *batch, const ApusHeadRows *q,
                                       const ApusHeadRows *out, float scale, const uint8_t *sel, size_t sel_stride,
                                       size_t pool, void *workspace, size_t workspace_bytes, void *stream) {
    const char *what = "kv4_attn";
    if (!q || !out) { gcuda_set_error("%s: no rows given", what); return -1; }
    Kv4AttnArgs a{};
    if (kv4_attn_args(what, cache, batch, q->heads, q->rows, &a.v)) return -1;
    if (attn_check_rows(what, q, cache->dim, false) || attn_check_rows(what, out, cache->dim, true)) return -1;
    if (q->rows != out->rows || q->heads != out->heads) {
        gcuda_set_error("%s: %zu rows of %zu heads in, %zu of %zu out", what, q->rows, q->heads, out->rows, out->heads);
        return -1;
    }
    if (sel && (pool < 1 || pool > 128 || sel_stride >= ((size_t)1 << 31))) {
        gcuda_set_error("%s: selection of %zu pools of %zu positions (1..128)", what, sel_stride, pool);
        return -1;
    }
    if (!q->rows || !a.v.nseq || !a.v.max_rows) return 0;
    const Kv4Plan p = kv4_plan(a.v, q->heads);
    if (p.bytes && (!workspace || workspace_bytes < p.bytes || ((uintptr_t)workspace & 15))) {
        gcuda_set_error("%s: workspace of %zu bytes at %p (%zu needed, 16-byte aligned)", what, workspace_bytes,
                        workspace, p.bytes);
        return -1;
    }
    a.q = rows_view(q);
    a.out = rows_view(out);
    a.group = (int)(q->heads / cache->heads);
    a.zscale = scale * 1.4426950408889634f;
    a.sel = sel;
    a.sel_stride = (long)sel_stride;
    a.pool = sel ? (int)pool : 1;
    a.pool_magic = (((uint64_t)1 << 36) + (uint64_t)a.pool - 1) / (uint64_t)a.pool;
    a.chunk_pos = p.chunk_pages * KV4_PAGE;
    a.nchunk = p.nchunk;
    a.ncb = p.ncb;
    a.part = (float *)workspace;
    cudaStream_t st = (cudaStream_t)stream;
    if (cache->dim == 64) return p.nt == 2 ? kv4_attn_launch<64, 2>(a, st) : kv4_attn_launch<64, 1>(a, st);
    if (cache->dim == 128) return p.nt == 2 ? kv4_attn_launch<128, 2>(a, st) : kv4_attn_launch<128, 1>(a, st);
    return kv4_attn_launch<256, 1>(a, st);
}

int kv4_attn_error_read_and_clear(void) {
    int v = 0, z = 0;
    cudaMemcpyFromSymbol(&v, g_kv4a_err, sizeof v);
    if (v) cudaMemcpyToSymbol(g_kv4a_err, &z, sizeof z);
    return v;
}
