// kv4_attn.cu — attention of a few rows a sequence over the 4-bit cache
// (apus_gcuda_kv4_attn_dev).
//
//   z_tj = scale log2(e) q_t . k_j,  m_t = max_j z_tj,
//   out_t = sum_j 2^(z_tj - m_t) v_j / sum_j 2^(z_tj - m_t)
//
// over the visible positions j, in one pass with running maxima and sums.
// With k_j = s_jg c_jd and v_j = r_jg e_jd (scale of the group g of 32 dims
// times an integer code), both contractions run on integer codes:
//   z_tj  = sum_g s_jg (sum_{d in g} q_td c_jd)
//   out_td = sum_j (p_tj r_jg) e_jd      for d in g
// so the scales cost one multiply per position, group and query column, not
// one per element.
//
// Bound: HBM at long contexts (a position of a head is 9/8 dim bytes), with
// the unpacking of the codes close behind it, so the unpacking is what the
// layout serves.  mma.sync with the query columns (rows of the step times
// heads of the group) in tiles of 8: tcgen05 needs 64 rows of a tile at least
// and operands in shared memory, so the codes would have to be unpacked into
// it first, and at 1 to 16 columns its rate buys nothing.
//   * m16n8k16 on f16 with the positions (scores) or the dims (output) as its
//     16 rows and the query columns as its 8.  The other way round the weights
//     would need no transpose, but half the rows would idle and their zeros cost
//     a register each (measured: 372 instructions for 16 positions of dim 128).
//   * Key codes 0-15 enter as f16 subnormals: a field at bits 0-3 or 4-7 of a
//     half is c 2^-24 or c 2^-20 as it stands, so one AND unpacks two codes.  The
//     factor 16 goes into the query's fragments, the offset 8 is taken off the
//     sum, and 2^24 goes into the column's scale.
//   * Value codes of two positions are paired by one byte permute, OR-ed into
//     the mantissa of 1024 and the offset is subtracted: exact integers.
//   * Scales are unpacked once a unit, not once a lane that needs them: fp32 for
//     the keys; for the values f16 below 2, with a power of two a position that
//     goes into the weight's exponent.  Two f16 roundings (2^-11 each) a weight.
//   * So there are two running maxima: ml of z for the sum of the weights, 2^(z - ml),
//     and m of (z - ml) + E (2^E a position's power of two) for the output's, whose
//     exponentials are computed a second time.  One weight for both, times 2^-E in the
//     sum, lost a position whose values are zero or 2^127 below the others', or
//     overflowed; and z + E without z - ml first rounds E away where scores are huge.
// (E4M3 mma.sync looks four times as fast but is carried out as conversions and
// f16 products: 50 conversions for 16 positions of dim 128, and no faster.)
//
// Work: a segment is one sequence's positions for one cache head and 8 NT
// columns.  All segments' pages in a row are cut into equal runs, one a CTA,
// one wave of CTAs (lengths are read on the device, so ragged batches balance
// too), or, of few segments, each into runs of its own; a segment that a cut
// divides is put together by a second kernel.
// Inside a CTA four warps each stream units of U positions of their own
// through two stages of their own with their own maximum, sum and output
// tile, so the loop has no CTA barrier; the warps are joined once a segment.
// Units come by cp.async, nine 16-byte pieces a lane: bulk copies of one or four
// pieces a unit cost their issuing warp about 250 cycles each, as much as two
// fragments' work.  Under a selection the positions that any of the columns keeps
// are listed, with a bit for each row that keeps them, and gathered row by row, so
// what no column keeps is neither read nor computed.
//
// Measured (us a call in a captured graph; bytes that it has to read, of 6.55 TB/s): one
// sequence of 131072 positions, 64 heads over 8 of 128: 42.4 (54%); 48 sequences of up
// to 8192, 32 over 8: 70.7 (53%); 4 rows over 4363 positions of 64 heads of 256: 32
// (38%); 4 rows of 512 pools of 4 out of 32771: 46; 513 positions, 32 over 8: 8.7.
// No pipe is full: 334 instructions for 16 positions of dim 128 (812 at dim 256) take
// 57% of the issue slots in the stream and 48% of the half-rate pipe (LOP3, shifts), and
// would take 19.5 of the 42.4 us by themselves.  A warp takes 16 positions at a time
// through one chain (scores, maxima, exponentials, transpose, output), with three warps
// a scheduler: fixed latencies are the first stall.  About 8 thousand cycles a launch go
// by before and after the stream.  A fourth CTA an SM (128 registers, the query in shared
// memory) took 8% longer; two scores an instruction (packed fp32) took 3% off; two
// fragments in flight a warp have not been tried.  The sum's own maximum and exponentials
// cost 2 to 4%.
#include <algorithm>
#include <type_traits>

#include "attn_dev.h"
#include "common.cuh"
#include "pipe.cuh"

namespace apus {

__device__ int g_kv4a_err;   // attn_dev.h's codes

namespace kv4 {
constexpr int WARPS = 4, THREADS = 32 * WARPS, STAGES = 2;
// CTAs an SM holds: as many as the registers allow (168 and 255 a thread).
constexpr int resident(int nt) { return nt == 1 ? 3 : 2; }
// Positions of a unit: 4608 bytes of cache.
template <int D> struct Cfg {
    static constexpr int U = 4096 / D;
    static constexpr int NG = D / 32;                       // scale groups
    static constexpr int KC = 0, VC = U * D / 2, KS = U * D, VS = KS + U * NG * 2;
    static constexpr int STAGE = VS + U * NG * 2;           // 72 D U / 64
    // a unit's scales as the loop wants them: keys' fp32 [U][NG], values' f16
    // pairs of positions, and each position's exponent E
    static constexpr int KF = STAGES * STAGE, VH = KF + U * NG * 4, PW = VH + U * NG * 2;
    static constexpr int WARP_SMEM = PW + U * 4;
    // the query's fragments, 512 bytes a group: 32 registers at dim 256, which the loop
    // has not (28 bytes are spilt as it is, and read eight times a warp in a launch);
    // below they stay in registers
    static constexpr bool QS = D == 256;
    static constexpr int QF = WARPS * WARP_SMEM, SMEM = QF + (QS ? NG * 512 : 0);
};
// Selected positions at a time: an offset in bits 0-15, above them a bit for
// each row of the block that keeps the position.
constexpr int LIST = 4096, LIST_SPAN = 65536, LOOK = 4;     // LOOK: pools that a thread looks at together
constexpr float NEG_INF = -__builtin_huge_valf();
// A maximum is raised when a term passes it by more than 2^OVER (the output's weights
// are f16) or 2^L_OVER (the sum is fp32 and has room for 2^67 such terms).
constexpr float OVER = 13.0f, L_OVER = 60.0f;
// A partial result: m, sum and ml of each column, then its dims.
constexpr int part_floats(int cols, int dim) { return cols * (dim + 3); }
}  // namespace kv4

struct Kv4AttnArgs {
    Kv4View v;
    RowsView q, out;
    int group;                // query heads of a cache head
    uint64_t group_magic;     // ceil(2^40 / group): c / group = c * magic >> 40 (a column and a head are below 2^20, 2^16)
    float zscale;             // scale * log2(e)
    const uint8_t *sel;
    long sel_stride;
    int pool;
    uint64_t pool_magic;      // ceil(2^36 / pool): j / pool = j * magic >> 36 for j < 2^28, pool <= 128
    int whole;                // no segment is cut: a page of work stands for a segment
    int min_pages;            // pages of a run at least
    int slots, segs;          // CTAs that run at once; segments at most
    long *plan;               // workspace: runs, units of work in all, pages of a unit, first unit of each sequence
    float *part;              // workspace: two partial results a CTA
};

// Quotients without the long way round of 64-bit division where they fit 32.
APUS_DEV long div_long(long a, long b) {
    return ((unsigned long)(a | b) >> 32) == 0 ? (long)((uint32_t)a / (uint32_t)b) : a / b;
}
APUS_DEV int row_of(const Kv4AttnArgs &a, int c) { return (int)(((uint64_t)(uint32_t)c * a.group_magic) >> 40); }

APUS_DEV int pool_of(const Kv4AttnArgs &a, int j) { return (int)(((uint64_t)(uint32_t)j * a.pool_magic) >> 36); }

constexpr int KJ_RUNS = ATTN_SMS * 4;     // runs at most (a multiple of 4)

// The work: sequence s has heads * ncb segments of `units` units of `unit`
// pages (one at least, so that a row that sees nothing is written too).
struct Kv4Work { Kv4Seq sq; int ncb; long units; };
APUS_DEV Kv4Work kv4_work(const Kv4AttnArgs &a, int s, int cols_block, int unit) {
    Kv4Work w;
    w.sq = kv4_seq(a.v.cu[s], a.v.cu[s + 1], a.v.len[s], a.v.rows, a.v.max_rows, a.v.max_len);
    w.ncb = (w.sq.n * a.group + cols_block - 1) / cols_block;
    const int pages = max(1, (w.sq.len + KV4_PAGE - 1) / KV4_PAGE);
    w.units = a.whole ? 1 : unit == 1 ? pages : (int)((uint32_t)(pages + unit - 1) / (uint32_t)unit);
    return w;
}

// c += a . b
APUS_DEV void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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
// cp.async of 4, 8 or 16 bytes.
template <int N> APUS_DEV void cp_async_n(void *dst, const void *src) {
    if constexpr (N == 16) cp_async16(dst, src);
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(dst)), "l"(src), "n"(N) : "memory");
}
APUS_DEV float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^e; 0 below the normal range.  The maxima are whole numbers, so that what they
// rescale is not rounded.  (The difference of two infinities, NaN, counts as 0: it
// arises where no position is seen, or in rows that are NaN already.)
APUS_DEV float pow2(int e) { return __int_as_float(max(min(e, 127) + 127, 0) << 23); }
// o 2^m / sum, by two factors: m goes from -140 to 187, and the result alone has to fit.
struct Kv4Norm {
    float inv, a, b;
    APUS_DEV Kv4Norm(float sum, float m) {
        const int d = max(min((int)m, 250), -250);
        inv = sum == 0.f ? 0.f : 1.0f / sum;
        a = pow2(d >> 1);
        b = pow2(d - (d >> 1));
    }
    APUS_DEV float operator()(float o) const { return o * inv * a * b; }
};
// 8x8 transpose of f16 pairs across the warp.
APUS_DEV uint32_t movmatrix(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
APUS_DEV uint32_t mul_f16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
// All ones in each half whose sign bit is set.
APUS_DEV uint32_t sign_x2(uint32_t x) {
    uint32_t d;
    asm("prmt.b32 %0, %1, 0, 0xbb99;" : "=r"(d) : "r"(x));
    return d;
}
// Constants of the code unpacking, kept in registers: an instruction takes one
// immediate, and the compiler would split (x & mask) | magic in two.
struct CodeConst { uint32_t lo, hi, magic, scale, off; };
APUS_DEV CodeConst code_const() {
    CodeConst k;
    asm volatile("mov.b32 %0, 0x000f000f;" : "=r"(k.lo));
    asm volatile("mov.b32 %0, 0x00f000f0;" : "=r"(k.hi));
    asm volatile("mov.b32 %0, 0x64006400;" : "=r"(k.magic));
    asm volatile("mov.b32 %0, 0x2c002c00;" : "=r"(k.scale));
    asm volatile("mov.b32 %0, 0xd480d480;" : "=r"(k.off));
    return k;
}
// Bits 0-3 (4-7) of each half as the f16 integers code - 8: OR-ed into the
// mantissa of 1024 the code counts 1 (16), and the rest is exact.
APUS_DEV uint32_t code_lo(uint32_t x, const CodeConst &k) {
    uint32_t u, d;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(u) : "r"(x), "r"(k.lo), "r"(k.magic));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(u), "r"(0x64086408u));
    return d;
}
APUS_DEV uint32_t code_hi(uint32_t x, const CodeConst &k) {
    uint32_t u, d;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(u) : "r"(x), "r"(k.hi), "r"(k.magic));
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(u), "r"(k.scale), "r"(k.off));
    return d;
}
template <int N> APUS_DEV void lds_floats(float (&f)[N], const float *p) {
    if constexpr (N == 2) { const float2 t = *(const float2 *)p; f[0] = t.x; f[1] = t.y; }
    else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 t = *(const float4 *)(p + i);
            f[i] = t.x; f[i + 1] = t.y; f[i + 2] = t.z; f[i + 3] = t.w;
        }
    }
}
template <int N> APUS_DEV void lds_pairs(uint32_t (&w)[N], const uint32_t *p) {
    if constexpr (N == 2) { const uint2 t = *(const uint2 *)p; w[0] = t.x; w[1] = t.y; }
    else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 t = lds128(p + i);
            w[i] = t.x; w[i + 1] = t.y; w[i + 2] = t.z; w[i + 3] = t.w;
        }
    }
}
template <int N> APUS_DEV void lds_words(uint32_t (&w)[N], const uint8_t *p) {
    if constexpr (N == 1) w[0] = *(const uint32_t *)p;
    else if constexpr (N == 2) { const uint2 t = *(const uint2 *)p; w[0] = t.x; w[1] = t.y; }
    else { const uint4 t = lds128(p); w[0] = t.x; w[1] = t.y; w[2] = t.z; w[3] = t.w; }
}

template <int D, int NT, bool SEL>
__global__ void __launch_bounds__(kv4::THREADS, kv4::resident(NT)) k_kv4_attn(const Kv4AttnArgs a) {
    using C = kv4::Cfg<D>;
    constexpr int NG = C::NG, U = C::U, COLS = 8 * NT, UPP = KV4_PAGE / U;
    constexpr float NEG_INF = kv4::NEG_INF;
    extern __shared__ __align__(128) uint8_t kv4_dyn[];
    __shared__ float join_m[kv4::WARPS][COLS], join_l[kv4::WARPS][COLS], join_ml[kv4::WARPS][COLS];
    __shared__ long scan_s[kv4::WARPS];
    __shared__ long found_s[2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;

    // ---- this CTA's run of units [x, xe)
    pdl_launch_dependents();
    // weights of the sequences, THREADS at a time: this thread's, the pages
    // before it and (through `before`) those of all
    int unit = 1, per_unit = 0, pages = 0;      // (this thread's sequence: segments, pages of one)
    auto scan = [&](int s0, long &w, long &before, bool again) -> long {
        const int s = s0 + threadIdx.x;
        w = 0;
        if (s < a.v.nseq) {
            if (!again) {
                const Kv4Work k = kv4_work(a, s, COLS, 1);
                if (k.sq.bad && blockIdx.x == 0) atomicExch(&g_kv4a_err, (int)ATTN_ERR_SEQ);
                per_unit = a.v.heads * k.ncb;
                pages = (int)k.units;
            }
            w = (long)per_unit * (unit == 1 ? pages : (int)((uint32_t)(pages + unit - 1) / (uint32_t)unit));
        }
        long incl = w;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const long o = __shfl_up_sync(0xffffffffu, incl, off);
            if (lane >= off) incl += o;
        }
        if (lane == 31) scan_s[warp] = incl;
        __syncthreads();
        long at = before + incl - w;
        for (int k = 0; k < kv4::WARPS; k++) {
            if (k < warp) at += scan_s[k];
            before += scan_s[k];
        }
        __syncthreads();
        return at;
    };
    // Runs that end with their segments, where these are few: with `unit` pages a
    // run, there are at most total / unit + segs of them.  A run across a border has
    // two pieces to set up and join, which takes as long as 1.5 pages (513 positions,
    // 8 segments: 10.1 us, and 8.4 with runs of their own).
    long total, w0 = 0, at0 = 0;
#pragma unroll 1
    for (bool again = false;; again = true) {
        total = 0;
#pragma unroll 1
        for (int s0 = 0; s0 < a.v.nseq; s0 += kv4::THREADS) at0 = scan(s0, w0, total, again && a.v.nseq <= kv4::THREADS);
        if (again || a.whole || a.segs >= a.slots) break;
        const long u = max((long)a.min_pages, div_long(total + a.slots - a.segs - 1, a.slots - a.segs));
        if (u != a.min_pages && 2 * u * a.slots > 2 * total + 3 * a.slots) break;
        unit = (int)u;
    }
    const long runs = min((long)gridDim.x, max(1l, unit > 1 ? total : div_long(total, a.min_pages)));
    if (blockIdx.x >= runs && blockIdx.x != 0) return;
    long x = div_long(total * blockIdx.x, runs);
    const long xe = div_long(total * (blockIdx.x + 1), runs);
    // the sequence in which it begins, and that sequence's first unit
    long before = 0;
    for (int s0 = 0; s0 < a.v.nseq; s0 += kv4::THREADS) {
        if (a.v.nseq > kv4::THREADS) at0 = scan(s0, w0, before, false);
        const int s = s0 + threadIdx.x;
        if (s < a.v.nseq && w0 && at0 <= x && x < at0 + w0) { found_s[0] = s; found_s[1] = at0; }
        if (blockIdx.x == 0 && a.plan && s < a.v.nseq) a.plan[3 + s] = at0;
    }
    if (blockIdx.x == 0 && a.plan && threadIdx.x == 0) { a.plan[0] = runs; a.plan[1] = total; a.plan[2] = unit; }
    if (x >= xe) return;
    __syncthreads();
    int seq = (int)found_s[0];
    long seq_x = found_s[1];
    uint8_t *const own = kv4_dyn + warp * C::WARP_SMEM, *const stages = own;
    uint32_t *list = (uint32_t *)(kv4_dyn + C::SMEM);     // LIST entries and 16 that no row keeps
    __shared__ int wcount[kv4::WARPS];

    while (x < xe) {
    // ---- the next piece: units of one segment
    Kv4Work wk = kv4_work(a, seq, COLS, unit);
    while (x >= seq_x + (long)a.v.heads * wk.ncb * wk.units) {
        seq_x += (long)a.v.heads * wk.ncb * wk.units;
        wk = kv4_work(a, ++seq, COLS, unit);
    }
    const Kv4Seq sq = wk.sq;
    const int seg = (int)div_long(x - seq_x, wk.units);
    const long seg_x = seq_x + seg * wk.units;
    const int head = wk.ncb == 1 ? seg : seg / wk.ncb, cb = seg - head * wk.ncb;
    const long piece_e = min(xe, seg_x + wk.units);
    const bool starts = x == seg_x, ends = piece_e == seg_x + wk.units;
    const int cols = sq.n * a.group, c0 = cb * COLS;
    const int cend = min(c0 + COLS, cols);
    // the positions that the first and the last row of the block see
    const int lim_row0 = sq.len - sq.n + 1;
    const int lim0 = lim_row0 + row_of(a, c0), lim1 = lim_row0 + row_of(a, cend - 1);
    const int p0 = a.whole ? 0 : (int)(x - seg_x) * unit * KV4_PAGE;
    const int p1 = a.whole ? lim1 : (int)min((piece_e - seg_x) * unit * KV4_PAGE, (long)lim1);
    const int32_t *table = a.v.table + (long)seq * a.v.table_stride;

    // the query rows of this lane's columns, on their way while the first units are fetched
    uint4 raw[NT][NG];
    auto fetch_query = [&]() {
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int c = c0 + nt * 8 + g, t = row_of(a, min(c, cols - 1));
            const uint16_t *qp = a.q.p + (long)(sq.row0 + t) * a.q.rs + (long)(head * a.group + min(c, cols - 1) - t * a.group) * a.q.hs;
#pragma unroll
            for (int j = 0; j < NG; j++)
                raw[nt][j] = c < cols ? *(const uint4 *)(qp + 32 * j + 8 * q4) : make_uint4(0, 0, 0, 0);
        }
    };
    if (!SEL) fetch_query();
    // the query's fragments, the columns' offsets, factors and limits (SEL: the
    // bit of the column's row in a list entry; below)
    uint32_t Q[C::QS ? 1 : NT][C::QS ? 1 : NG][4];
    float cinit[NT][NG][2], fac[NT][2];
    int lim[NT][2];
    // columns 2 q4, 2 q4 + 1: output and its maximum, the sum of this lane's weights and
    // its maximum
    float O[NT][D / 16][4], m[NT][2], l[NT][2], ml[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int i = 0; i < D / 16; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) O[nt][i][e] = 0.f;
        m[nt][0] = m[nt][1] = ml[nt][0] = ml[nt][1] = NEG_INF;
        l[nt][0] = l[nt][1] = 0.f;
    }

    // the cached position of place r of a 16-position fragment: places 2 q,
    // 2 q + 1 are positions q, 4 + (q ^ 1), so that the quads of one
    // shared-memory access fall in different banks for keys and for values
    const int pg = (g & 1) ? 4 + ((g >> 1) ^ 1) : (g >> 1), vp1 = 4 + (q4 ^ 1);

    const CodeConst cc = code_const();
    // A unit's scales as the loop below wants them.  A position's value scales
    // are 2^E times numbers below 2, exact in f16 (those below 2^-24 of the
    // largest become 0); E is kept to -126 .. 126, so that 2^-E is a normal number
    // (a scale of 2^127 is then below 4, and a weight of 2^13 times that fits f16).
    // Whole warp; a lane takes four scales of each kind.
    auto prepare = [&](const uint8_t *st) {
        static_assert(U * NG == 128, "four scales of keys and of values a lane");
        const uint2 k = *(const uint2 *)(st + C::KS + lane * 8), v = *(const uint2 *)(st + C::VS + lane * 8);
        *(float4 *)(own + C::KF + lane * 16) = make_float4(bf16lo(k.x), bf16hi(k.x), bf16lo(k.y), bf16hi(k.y));
        const float vf[4] = {bf16lo(v.x), bf16hi(v.x), bf16lo(v.y), bf16hi(v.y)};
        float top[2];                              // largest scale of this lane's position (NG 2: two)
        top[0] = fmaxf(vf[0], vf[1]);
        top[1] = fmaxf(vf[2], vf[3]);
        if constexpr (NG > 2) {
            top[0] = fmaxf(top[0], top[1]);
            if constexpr (NG == 8) top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], 1));
            top[1] = top[0];
        }
        float inv[2];
#pragma unroll
        for (int u = 0; u < (NG == 2 ? 2 : 1); u++) {
            int e = (int)(__float_as_uint(top[u]) >> 23) - 127;    // a NaN's or an infinity's scales stay what they are
            e = max(min(e, 126), -126);
            inv[u] = __int_as_float((127 - e) << 23);
            const int r = NG == 2 ? 2 * lane + u : lane / (NG / 4);
            *(float *)(own + C::PW + r * 4) = (float)e;
        }
        if constexpr (NG > 2) inv[1] = inv[0];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = (lane * 4 + i) / NG, j = (lane * 4 + i) % NG, e = (r >> 2) & 1;
            const int at = (((r >> 3) * 4 + ((r & 3) ^ e)) * NG + j) * 2 + e;
            ((__half *)(own + C::VH))[at] = __float2half_rn(vf[i] * inv[i >> 1]);
        }
        __syncwarp();
    };

    // 16 positions at place `at` of a stage: the positions from pos0 on, or (SEL)
    // those that the list names
    auto process = [&](const uint8_t *st, int at, int pos0, const uint32_t *names, auto masked_t) {
        constexpr bool MASKED = decltype(masked_t)::value;
        float z[NT][4];                // positions pg (0, 1), pg + 8 (2, 3); columns 2 q4 (0, 2), 2 q4 + 1
        float pw[2];                   // their exponents E
        {
            uint32_t wa[NG], wb[NG];
            constexpr int JB = NG < 4 ? NG : 4;
#pragma unroll
            for (int h = 0; h < NG / JB; h++) {
                uint32_t ta[JB], tb[JB];
                const uint8_t *kp = st + C::KC + (at + pg) * (D / 2) + kv4_k_word(D, pg, h * JB, q4) * 4;
                lds_words<JB>(ta, kp);
                lds_words<JB>(tb, kp + 8 * (D / 2));
#pragma unroll
                for (int i = 0; i < JB; i++) { wa[h * JB + i] = ta[i]; wb[h * JB + i] = tb[i]; }
            }
            float sa[NG], sb[NG];
            uint64_t z2[NT][2];
            lds_floats<NG>(sa, (const float *)(own + C::KF) + (at + pg) * NG);
            lds_floats<NG>(sb, (const float *)(own + C::KF) + (at + pg + 8) * NG);
            pw[0] = *(const float *)(own + C::PW + (at + pg) * 4);
            pw[1] = *(const float *)(own + C::PW + (at + pg + 8) * 4);
#pragma unroll
            for (int j = 0; j < NG; j++) {
                const uint32_t xa = wa[j] >> 8, xb = wb[j] >> 8;
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float c[4] = {0.f, 0.f, 0.f, 0.f};
                    uint4 qf;
                    if constexpr (C::QS) qf = lds128(kv4_dyn + C::QF + j * 512 + lane * 16);
                    else qf = make_uint4(Q[nt][j][0], Q[nt][j][1], Q[nt][j][2], Q[nt][j][3]);
                    mma_f16(c, wa[j] & 0x000f000fu, wb[j] & 0x000f000fu, wa[j] & 0x00f000f0u, wb[j] & 0x00f000f0u, qf.x, qf.y);
                    mma_f16(c, xa & 0x000f000fu, xb & 0x000f000fu, xa & 0x00f000f0u, xb & 0x00f000f0u, qf.z, qf.w);
                    const uint64_t off = f32_pair(cinit[nt][j][0], cinit[nt][j][1]);
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const uint64_t s = h ? f32_pair(sb[j], sb[j]) : f32_pair(sa[j], sa[j]);
                        const uint64_t x = add_f32x2(f32_pair(c[2 * h], c[2 * h + 1]), off);
                        z2[nt][h] = j ? fma_f32x2(s, x, z2[nt][h]) : mul_f32x2(s, x);
                    }
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const uint64_t f = f32_pair(fac[nt][0], fac[nt][1]);
                f32_unpair(mul_f32x2(z2[nt][0], f), z[nt][0], z[nt][1]);
                f32_unpair(mul_f32x2(z2[nt][1], f), z[nt][2], z[nt][3]);
            }
        }
        // ---- running maxima: ml of z, m of y + E, y = z - ml, so of what a position adds
        // to the output: its weight times 2^E, and times a scale below 2, then fits f16
        // with the largest at 2^5 to 2^13 whatever the scales' range (what is below 2^-30
        // of the largest may add nothing).
        uint32_t hide = 0;             // bit nt * 4 + i (MASKED)
        bool over = false;
        float y[NT][4], ye[NT][4];     // y and y + E - m
        auto relate = [&](int nt) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint64_t d = add_f32x2(f32_pair(z[nt][2 * h], z[nt][2 * h + 1]), f32_pair(-ml[nt][0], -ml[nt][1]));
                f32_unpair(d, y[nt][2 * h], y[nt][2 * h + 1]);
                f32_unpair(add_f32x2(add_f32x2(d, f32_pair(pw[h], pw[h])), f32_pair(-m[nt][0], -m[nt][1])), ye[nt][2 * h],
                           ye[nt][2 * h + 1]);
            }
        };
        uint32_t name[2] = {0, 0};
        if (SEL) { name[0] = names[pg]; name[1] = names[pg + 8]; }
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            if (MASKED) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const bool see = SEL ? (name[i >> 1] >> lim[nt][i & 1] & 1) != 0
                                         : pos0 + (i >> 1) * 8 + pg < lim[nt][i & 1];
                    if (!see) { z[nt][i] = NEG_INF; hide |= 1u << (nt * 4 + i); }
                }
            }
            relate(nt);
            over |= fmaxf(fmaxf(fmaxf(y[nt][0], y[nt][1]), y[nt][2]), y[nt][3]) > kv4::L_OVER;
            over |= fmaxf(fmaxf(fmaxf(ye[nt][0], ye[nt][1]), ye[nt][2]), ye[nt][3]) > kv4::OVER;
        }
        if (__any_sync(0xffffffffu, over)) {
            auto highest = [&](float x, float x2) {
                x = fmaxf(x, x2);
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
                return x;
            };
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                for (int u = 0; u < 2; u++) {                      // each column by its own scores alone
                    const float x = highest(z[nt][u], z[nt][u + 2]), up = floorf(x) - ml[nt][u];
                    if (!(x - ml[nt][u] > kv4::L_OVER)) continue;
                    l[nt][u] *= pow2((int)-up);
                    ml[nt][u] = floorf(x);
                    m[nt][u] -= up;                                // (of -inf: stays that)
                }
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const float x = highest(z[nt][u] - ml[nt][u] + pw[0], z[nt][u + 2] - ml[nt][u] + pw[1]), to = floorf(x) - 5.0f;
                    if (!(x - m[nt][u] > kv4::OVER)) continue;
                    const float down = pow2((int)(m[nt][u] - to));
                    m[nt][u] = to;
#pragma unroll
                    for (int i = 0; i < D / 16; i++) { O[nt][i][u] *= down; O[nt][i][u + 2] *= down; }
                }
                relate(nt);
            }
        }
        // ---- weights (times 2^E), brought to the order of the output's operand:
        // column g, positions 0, 1 and 2, 3 of the lane
        uint32_t b0[NT], b1[NT], k0[NT], k1[NT];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float p[4];
            uint64_t sum = f32_pair(l[nt][0], l[nt][1]);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float w[2];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    p[2 * h + u] = ex2(ye[nt][2 * h + u]);
                    w[u] = ex2(y[nt][2 * h + u]);
                    // a hidden position adds nothing to the sum, and its weight is -0: the sign
                    // marks it below, where a NaN scale must not reach the product
                    if (MASKED && (hide >> (nt * 4 + 2 * h + u) & 1)) { p[2 * h + u] = -0.0f; w[u] = 0.f; }
                }
                sum = add_f32x2(sum, f32_pair(w[0], w[1]));
            }
            f32_unpair(sum, l[nt][0], l[nt][1]);
            b0[nt] = movmatrix(pack_f16(p[0], p[1]));
            b1[nt] = movmatrix(pack_f16(p[2], p[3]));
            if (MASKED) {
                k0[nt] = ~sign_x2(b0[nt]);
                k1[nt] = ~sign_x2(b1[nt]);
            }
        }
        // ---- output
        uint32_t w[4][D / 64], va[NG], vb[NG];
#pragma unroll
        for (int i = 0; i < 4; i++)
            lds_words<D / 64>(w[i], st + C::VC + (at + (i >> 1) * 8 + ((i & 1) ? vp1 : q4)) * (D / 2) +
                                        kv4_v_word(D, (i & 1) ? vp1 : q4, g, 0) * 4);
        lds_pairs<NG>(va, (const uint32_t *)(own + C::VH) + ((at >> 3) * 4 + q4) * NG);
        lds_pairs<NG>(vb, (const uint32_t *)(own + C::VH) + ((at >> 3) * 4 + 4 + q4) * NG);
#pragma unroll
        for (int j = 0; j < NG; j++) {
            const uint32_t pick = (j & 1) ? 0x7632 : 0x5410;
            const uint32_t x = __byte_perm(w[0][j / 2], w[1][j / 2], pick);
            const uint32_t y = __byte_perm(w[2][j / 2], w[3][j / 2], pick);
            const uint32_t x0 = code_lo(x, cc), x1 = code_hi(x, cc), x2 = code_lo(x >> 8, cc), x3 = code_hi(x >> 8, cc);
            const uint32_t y0 = code_lo(y, cc), y1 = code_hi(y, cc), y2 = code_lo(y >> 8, cc), y3 = code_hi(y >> 8, cc);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                uint32_t w0 = mul_f16x2(b0[nt], va[j]), w1 = mul_f16x2(b1[nt], vb[j]);
                if (MASKED) { w0 &= k0[nt]; w1 &= k1[nt]; }
                mma_f16(O[nt][2 * j], x0, x1, y0, y1, w0, w1);
                mma_f16(O[nt][2 * j + 1], x2, x3, y2, y3, w0, w1);
            }
        }
    };

    // ---- the stream: this warp's units warp, warp + WARPS, ... of the piece, or
    // of one list of selected positions after the other
    int done = p0;
    do {
        int base = p0, filled = p1 > p0 ? p1 - p0 : 0;     // positions, the first of them (SEL: of the list)
        if constexpr (SEL) {
            // list the positions from `done` on that a row keeps, as many as the list
            // holds.  Pools are whole but for the first, which the piece's begin may
            // cut, and the last; a row sees all of its own incomplete pool.
            __syncthreads();
            const int t0 = lim0 - lim_row0, nt = lim1 - lim0 + 1;          // rows of the block
            const uint8_t *const sel0 = a.sel + (long)(sq.row0 + t0) * a.sel_stride;
            const int span = min(p1, done + kv4::LIST_SPAN);
            base = done;
            filled = 0;
            // pools looked at together: at least one, with room in the list for twice as
            // many positions, so `done` advances each time
            const int round = min(kv4::THREADS * kv4::LOOK, kv4::LIST / 2 / a.pool);
            const int tail0 = lim0 > 0 ? pool_of(a, lim0) * a.pool : 0;      // where the first row's incomplete pool begins
            while (done < span && filled + round * a.pool <= kv4::LIST) {
                const int pl0 = pool_of(a, done);
                uint32_t rows[kv4::LOOK] = {};
                for (int t = 0; t < nt; t++) {
#pragma unroll
                    for (int k = 0; k < kv4::LOOK; k++) {
                        const int pl = pl0 + k * kv4::THREADS + (int)threadIdx.x;
                        if (pl - pl0 < round && pl < a.sel_stride && pl * a.pool < span && sel0[(long)t * a.sel_stride + pl])
                            rows[k] |= 1u << t;
                    }
                }
                int cnt = 0, b[kv4::LOOK], n[kv4::LOOK];
#pragma unroll
                for (int k = 0; k < kv4::LOOK; k++) {
                    const int at = k * kv4::THREADS + (int)threadIdx.x, first = (pl0 + at) * a.pool;
                    b[k] = max(first, done);
                    n[k] = 0;
                    if (at >= round || first >= span) continue;
                    if (first + a.pool > tail0)            // some row's incomplete pool, or behind a row's last
                        for (int t = 0; t < nt; t++) {
                            const int lim = lim0 + t;
                            if (first >= lim) rows[k] &= ~(1u << t);
                            else if (first + a.pool > lim) rows[k] |= 1u << t;
                        }
                    if (rows[k]) n[k] = min(first + a.pool, span) - b[k];
                    cnt += n[k];
                }
                int incl = cnt;
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) {
                    const int o = __shfl_up_sync(0xffffffffu, incl, off);
                    if (lane >= off) incl += o;
                }
                if (lane == 31) wcount[warp] = incl;
                __syncthreads();
                int at = filled + incl - cnt;
                for (int w = 0; w < warp; w++) at += wcount[w];
#pragma unroll
                for (int k = 0; k < kv4::LOOK; k++)
                    for (int i = 0; i < n[k]; i++) {
                        // row t sees positions below lim0 + t
                        const int j = b[k] + i, from = j < lim0 ? 0 : j - lim0 + 1;
                        list[at++] = (uint32_t)(j - base) | (rows[k] >> from << from) << 16;
                    }
                for (int w = 0; w < kv4::WARPS; w++) filled += wcount[w];
                done = min(span, (pl0 + round) * a.pool);
                __syncthreads();
            }
            if (threadIdx.x < 16) list[filled + threadIdx.x] = 0;
            __syncthreads();
        }
        const int units = (filled + U - 1) / U;
        const int mine = units > warp ? (units - warp + kv4::WARPS - 1) / kv4::WARPS : 0;
        int my_page = -1;                  // lane i: page of the i-th of 32 units
        unsigned there = 0;                // bit s: stage s holds a unit (not one of a page out of range)
        auto load = [&](int i, int s) {    // unit i of this warp into stage s (whole warp)
            if (i < mine) {
                const int u = warp + i * kv4::WARPS;
                uint8_t *dst = stages + s * C::STAGE;
                constexpr int CH = D / 32;                 // 16-byte pieces of a row of codes
                if constexpr (!SEL) {
                    if ((i & 31) == 0) {
                        my_page = -1;
                        if (i + lane < mine) {
                            const int page = table[(p0 + (u + lane * kv4::WARPS) * U) / KV4_PAGE];
                            if (kv4_page_ok(page, a.v.num_pages)) my_page = page;
                            else atomicCAS(&g_kv4a_err, 0, (int)ATTN_ERR_PAGE);
                        }
                    }
                    const int page = __shfl_sync(0xffffffffu, my_page, i & 31);
                    there = (there & ~(1u << s)) | ((page >= 0 ? 1u : 0u) << s);
                    if (page >= 0) {
                        const int h = u % UPP;             // pieces begin at a page
                        const uint8_t *src = a.v.pages + kv4_block_at(page, head, a.v.heads, D);
                        const uint8_t *kc = src + h * (U * D / 2) + lane * 16;
#pragma unroll
                        for (int k = 0; k < U * CH / 32; k++) {
                            cp_async16(dst + C::KC + lane * 16 + k * 512, kc + k * 512);
                            cp_async16(dst + C::VC + lane * 16 + k * 512, kc + kv4_v_codes(D) + k * 512);
                        }
                        // scales: 16 pieces of the keys', 16 of the values'
                        cp_async16(dst + C::KS + lane * 16, src + (lane < 16 ? kv4_k_scales(D) : kv4_v_scales(D)) +
                                                                h * 256 + (lane & 15) * 16);
                        static_assert(U * NG * 2 == 256 && C::VS == C::KS + 256, "scales of a unit");
                    }
                } else {
                    constexpr int RPL = (U + 31) / 32;     // rows a lane finds
                    const int u0 = u * U;
                    const uint8_t *src[RPL];
                    int off[RPL];
#pragma unroll
                    for (int e = 0; e < RPL; e++) {
                        const int r = e * 32 + lane;
                        src[e] = nullptr;
                        off[e] = 0;
                        if (r < U && u0 + r < filled) {
                            const int j = base + (int)(list[u0 + r] & 0xffffu), page = table[j / KV4_PAGE];
                            off[e] = j & (KV4_PAGE - 1);
                            if (kv4_page_ok(page, a.v.num_pages)) src[e] = a.v.pages + kv4_block_at(page, head, a.v.heads, D);
                            else {
                                atomicCAS(&g_kv4a_err, 0, (int)ATTN_ERR_PAGE);
                                list[u0 + r] &= 0xffffu;   // no row sees it
                            }
                        }
                    }
#pragma unroll
                    for (int k = 0; k < U * CH; k += 32) {
                        const int row = (k + lane) / CH, c = (k + lane) % CH, e = (k / CH) / 32;
                        const uint8_t *sp = (const uint8_t *)__shfl_sync(0xffffffffu, (unsigned long long)src[e], row & 31);
                        const int o = __shfl_sync(0xffffffffu, off[e], row & 31);
                        // the row moves from place o of its page to place `row`
                        // of the stage, and its pieces as the layout has them there
                        const int kx = D == 256 ? (((o ^ row) >> 2) & 1) << 2 : 0;
                        const int vx = D == 256 ? ((o ^ row) & 3) << 1 : D == 128 ? (((o ^ row) >> 1) & 1) << 1 : 0;
                        if (sp) {
                            cp_async16(dst + C::KC + row * (D / 2) + (c ^ kx) * 16, sp + o * (D / 2) + c * 16);
                            cp_async16(dst + C::VC + row * (D / 2) + (c ^ vx) * 16,
                                       sp + kv4_v_codes(D) + o * (D / 2) + c * 16);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < RPL; e++) {
                        const int r = e * 32 + lane;
                        if (src[e]) {
                            cp_async_n<NG * 2>(dst + C::KS + r * NG * 2, src[e] + kv4_k_scales(D) + off[e] * NG * 2);
                            cp_async_n<NG * 2>(dst + C::VS + r * NG * 2, src[e] + kv4_v_scales(D) + off[e] * NG * 2);
                        }
                    }
                    there |= 1u << s;
                }
            }
            cp_async_commit();
        };
        for (int s = 0; s < kv4::STAGES; s++) load(s, s);
        if (!SEL || base == p0) {      // once a piece, while its first units are on their way
            if (SEL) fetch_query();
            // ---- the query's fragments: column g of each n tile, dims in the order
            // in which a lane meets the key codes (dim 8 q4 + i of a group is code i
            // of its word)
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                uint32_t top = 0;
#pragma unroll
                for (int j = 0; j < NG; j++) {
                    const uint32_t w[4] = {raw[nt][j].x, raw[nt][j].y, raw[nt][j].z, raw[nt][j].w};
#pragma unroll
                    for (int i = 0; i < 4; i++) top = max(top, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
                }
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // a power of two that brings the largest magnitude to [2^14, 2^15): f16
                // holds every BF16 within 2^-24 of it exactly, smaller ones to 2^-35 of it
                const int e = top ? max((int)(top >> 7) - 127, -100) : 0;
                const float up = __int_as_float((127 + 14 - e) << 23);
                float f = a.zscale * __int_as_float((127 + e - 14) << 23) * 16777216.0f;
                if (top >= 0x7f80u) f = __int_as_float(0x7fc00000);    // a NaN or an infinity: the row is NaN
#pragma unroll
                for (int j = 0; j < NG; j++) {
                    const float x[8] = {bf16lo(raw[nt][j].x), bf16hi(raw[nt][j].x), bf16lo(raw[nt][j].y), bf16hi(raw[nt][j].y),
                                        bf16lo(raw[nt][j].z), bf16hi(raw[nt][j].z), bf16lo(raw[nt][j].w), bf16hi(raw[nt][j].w)};
                    float qs = 0.f;
                    uint32_t frag[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        // codes in the high nibbles stand 16 times higher
                        const float down = (i & 1) ? up * 0.0625f : up;
                        const uint32_t h = pack_f16(x[i] * down, x[i + 4] * down);
                        frag[i] = h;
                        const float2 back = __half22float2(*(const __half2 *)&h);
                        qs += (back.x + back.y) * ((i & 1) ? 16.0f : 1.0f);
                    }
                    if constexpr (C::QS) {
                        if ((j & 3) == warp) *(uint4 *)(kv4_dyn + C::QF + j * 512 + lane * 16) = make_uint4(frag[0], frag[1], frag[2], frag[3]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; i++) Q[nt][j][i] = frag[i];
                    }
                    qs += __shfl_xor_sync(0xffffffffu, qs, 1);
                    qs += __shfl_xor_sync(0xffffffffu, qs, 2);
                    qs *= -8.0f / 16777216.0f;                               // the codes' offset
                    cinit[nt][j][0] = __shfl_sync(0xffffffffu, qs, 8 * q4);
                    cinit[nt][j][1] = __shfl_sync(0xffffffffu, qs, 8 * q4 + 4);
                }
                // what follows goes by the columns whose scores this lane holds
                fac[nt][0] = __shfl_sync(0xffffffffu, f, 8 * q4);
                fac[nt][1] = __shfl_sync(0xffffffffu, f, 8 * q4 + 4);
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int t = row_of(a, min(c0 + nt * 8 + 2 * q4 + u, cols - 1));
                    lim[nt][u] = SEL ? 16 + lim_row0 + t - lim0 : lim_row0 + t;
                }
            }
            if (C::QS) __syncthreads();
        }
        int s = 0;
        for (int i = 0; i < mine; i++) {
            cp_async_wait<kv4::STAGES - 1>();
            __syncwarp();
            if (there >> s & 1) {
                const uint8_t *st = stages + s * C::STAGE;
                const int u0 = (warp + i * kv4::WARPS) * U;
                prepare(st);
                if (!SEL && p0 + u0 + U <= lim0) {
#pragma unroll 1
                    for (int at = 0; at < U; at += 16) process(st, at, p0 + u0 + at, nullptr, std::false_type{});
                } else {
#pragma unroll 1
                    for (int at = 0; at < U && u0 + at < filled; at += 16)
                        process(st, at, p0 + u0 + at, list + u0 + at, std::true_type{});
                }
            }
            __syncwarp();
            load(i + kv4::STAGES, s);
            s = s == kv4::STAGES - 1 ? 0 : s + 1;
        }
        cp_async_wait<0>();
    } while (SEL && done < p1);

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
                join_ml[warp][nt * 8 + 2 * q4 + u] = ml[nt][u];
            }
        }
    __syncthreads();
    constexpr int JD = D + 4;         // rows a bank group apart
    float *jo = (float *)kv4_dyn;     // [WARPS][COLS][JD]
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int u = 0; u < 2; u++) {
            float *row = jo + (warp * COLS + nt * 8 + 2 * q4 + u) * JD;
#pragma unroll
            for (int j = 0; j < NG; j++)
                *(float4 *)(row + 32 * j + 4 * g) = make_float4(O[nt][2 * j][u], O[nt][2 * j][u + 2],
                                                               O[nt][2 * j + 1][u], O[nt][2 * j + 1][u + 2]);
        }
    __syncthreads();
    const bool last = starts && ends;
    float *part = a.part + ((size_t)blockIdx.x * 2 + (starts ? 1 : 0)) * (size_t)kv4::part_floats(COLS, D);
    for (int i = threadIdx.x; i < (cend - c0) * (D / 4); i += kv4::THREADS) {
        const int c = i / (D / 4), d = (i % (D / 4)) * 4;
        float mx = NEG_INF, mxl = NEG_INF;         // ml of all, m relative to that
#pragma unroll
        for (int w = 0; w < kv4::WARPS; w++) mxl = fmaxf(mxl, join_ml[w][c]);
#pragma unroll
        for (int w = 0; w < kv4::WARPS; w++) mx = fmaxf(mx, join_m[w][c] + (join_ml[w][c] - mxl));
        float sum = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kv4::WARPS; w++) {
            if (join_ml[w][c] == NEG_INF && join_l[w][c] == 0.f) continue;
            const float up = join_ml[w][c] - mxl, k = pow2((int)(join_m[w][c] + up - mx));
            const float4 x = *(const float4 *)(jo + (w * COLS + c) * JD + d);
            sum += join_l[w][c] * pow2((int)up);
            o.x += x.x * k; o.y += x.y * k; o.z += x.z * k; o.w += x.w * k;
        }
        if (!last) {
            *(float4 *)(part + 3 * COLS + c * D + d) = o;
            if (d == 0) { part[c] = mx; part[COLS + c] = sum; part[2 * COLS + c] = mxl; }
        } else {
            const Kv4Norm norm(sum, mx);
            const int t = row_of(a, c0 + c);
            uint16_t *op = a.out.p + (long)(sq.row0 + t) * a.out.rs +
                           (long)(head * a.group + c0 + c - t * a.group) * a.out.hs + d;
            *(uint2 *)op = make_uint2(pack_bf16(norm(o.x), norm(o.y)), pack_bf16(norm(o.z), norm(o.w)));
        }
    }
    __syncthreads();        // the stages are the next piece's
    x = piece_e;
    }
}

// Joins the pieces of one column of a segment that was cut: the maxima ml, then the m
// relative to the largest of them, then the sums with factors from these, in the order
// of the runs.  What it reads is on its way
// together: each thread's first AHEAD pieces before the weights are known.
// Two forms (kv4_attn_launch): WIDE for few columns, which may be cut into many
// pieces; the other for many, of few pieces each.
template <int D, bool WIDE>
__global__ void __launch_bounds__(WIDE ? 256 : 128, WIDE ? 2 : 12) k_kv4_join(const Kv4AttnArgs a, int cols_block) {
    constexpr int L = D / 4, P = (WIDE ? 256 : 128) / L, AHEAD = WIDE ? 8 : 1;
        // lanes over the dims, parts over the pieces
    extern __shared__ float kj_dyn[];                 // m (then weights), sums and ml of the pieces, then [P][D] sums
    __shared__ float total_s, max_s;
    const int seq = blockIdx.z, head = blockIdx.y;
    Kv4Work wk = kv4_work(a, seq, cols_block, 1);
    const Kv4Seq sq = wk.sq;
    pdl_wait();                                       // the partial results and the plan
    const long runs = a.plan[0], total = a.plan[1], first = a.plan[3 + seq];
    const int unit = (int)a.plan[2];
    if (unit > 1) wk.units = (uint32_t)((int)wk.units + unit - 1) / (uint32_t)unit;
    for (int c = blockIdx.x; c < sq.n * a.group; c += gridDim.x) {
        const int cb = c / cols_block, cc = c % cols_block;
        const long b = first + ((long)head * wk.ncb + cb) * wk.units, e = b + wk.units;
        // runs of the first and the last unit
        const long i0 = runs == total ? b : div_long((b + 1) * runs - 1, total);
        const long i1 = runs == total ? e - 1 : div_long(e * runs - 1, total);
        if (i0 == i1) continue;                       // written by its only run
        const int n = (int)(i1 - i0) + 1, stride = kv4::part_floats(cols_block, D);
        const float *const parts = a.part + (size_t)i0 * 2 * (size_t)stride;
        auto piece = [&](int i) { return parts + (size_t)(2 * i + (i == 0 ? 1 : 0)) * (size_t)stride; };
        const int d = (threadIdx.x % L) * 4, part = threadIdx.x / L, at = 3 * cols_block + cc * D + d;
        float4 y[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; u++)
            y[u] = part + u * P < n ? *(const float4 *)(piece(part + u * P) + at) : make_float4(0.f, 0.f, 0.f, 0.f);
        if (threadIdx.x < 32) {
            float mx = kv4::NEG_INF, mxl = kv4::NEG_INF;
            // (a lane finds its own pieces' in shared memory again)
            float *const km = kj_dyn, *const kl = kj_dyn + KJ_RUNS, *const kml = kj_dyn + 2 * KJ_RUNS;
#pragma unroll(WIDE ? 4 : 1)
            for (int i = threadIdx.x; i < n; i += 32) {
                km[i] = piece(i)[cc];
                kl[i] = piece(i)[cols_block + cc];
                const float mli = kml[i] = piece(i)[2 * cols_block + cc];
                mxl = fmaxf(mxl, mli);
            }
#pragma unroll
            for (int off = 16; off; off >>= 1) mxl = fmaxf(mxl, __shfl_xor_sync(0xffffffffu, mxl, off));
#pragma unroll(WIDE ? 4 : 1)
            for (int i = threadIdx.x; i < n; i += 32) mx = fmaxf(mx, km[i] + (kml[i] - mxl));
#pragma unroll
            for (int off = 16; off; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
            float sum = 0.f;
#pragma unroll(WIDE ? 4 : 1)
            for (int i = threadIdx.x; i < n; i += 32) {
                const float mi = km[i], li = kl[i], mli = kml[i];
                const bool none = mli == kv4::NEG_INF && li == 0.f;
                kj_dyn[i] = none ? 0.f : pow2((int)(mi + (mli - mxl) - mx));
                sum += none ? 0.f : li * pow2((int)(mli - mxl));
            }
#pragma unroll
            for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
            if (threadIdx.x == 0) { total_s = sum; max_s = mx; }
        }
        __syncthreads();
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        auto add = [&](const float4 &x, float k) { o.x += x.x * k; o.y += x.y * k; o.z += x.z * k; o.w += x.w * k; };
#pragma unroll
        for (int u = 0; u < AHEAD; u++)
            if (part + u * P < n) add(y[u], kj_dyn[part + u * P]);
#pragma unroll 4
        for (int i = part + AHEAD * P; i < n; i += P) add(*(const float4 *)(piece(i) + at), kj_dyn[i]);
        float *const sums = kj_dyn + 3 * KJ_RUNS;
        *(float4 *)(sums + part * D + d) = o;
        __syncthreads();
        if (part == 0) {
#pragma unroll
            for (int i = 1; i < P; i++) add(*(const float4 *)(sums + i * D + d), 1.0f);
            const Kv4Norm norm(total_s, max_s);
            const int t = row_of(a, c);
            uint16_t *op = a.out.p + (long)(sq.row0 + t) * a.out.rs + (long)(head * a.group + c - t * a.group) * a.out.hs + d;
            *(uint2 *)op = make_uint2(pack_bf16(norm(o.x), norm(o.y)), pack_bf16(norm(o.z), norm(o.w)));
        }
        __syncthreads();                              // the next column's weights and sums
    }
}

}  // namespace apus
using namespace apus;

namespace {

// How a batch is cut: columns of a block, CTAs, whether segments stay whole.
constexpr long MAX_POS = 1l << 28;
constexpr long WHOLE_PAGES = 8, MIN_PAGES = 2;
struct Kv4Plan { int nt, grid, whole, slots, segs; size_t plan_bytes, bytes; };

Kv4Plan kv4_plan(const Kv4View &v, size_t q_heads) {
    Kv4Plan p;
    const long cols = (long)q_heads / v.heads * v.max_rows;
    p.nt = cols > 8 && v.dim <= 128 ? 2 : 1;
    const long pages = v.max_len > KV4_PAGE ? (v.max_len + KV4_PAGE - 1) / KV4_PAGE : 1;
    const long segs = (long)v.nseq * v.heads * ((cols + 8 * p.nt - 1) / (8 * p.nt));
    p.whole = pages <= WHOLE_PAGES;
    const long most = p.whole ? segs : segs * ((pages + MIN_PAGES - 1) / MIN_PAGES);
    p.slots = ATTN_SMS * kv4::resident(p.nt);
    p.segs = (int)(segs < p.slots ? segs : p.slots);
    p.grid = (int)(most < p.slots ? most : p.slots);
    p.plan_bytes = ((size_t)v.nseq + 3) * sizeof(long);
    p.plan_bytes = (p.plan_bytes + 15) / 16 * 16;
    p.bytes = p.whole ? 0 : p.plan_bytes + (size_t)p.grid * 2 * kv4::part_floats(8 * p.nt, v.dim) * sizeof(float);
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

template <int D, int NT, bool SEL>
int kv4_attn_launch(const Kv4AttnArgs &a, int grid, cudaStream_t st) {
    using C = kv4::Cfg<D>;
    const int smem = C::SMEM + (SEL ? (kv4::LIST + 16) * 4 : 0);
    if (gcuda_smem_limit_once((const void *)k_kv4_attn<D, NT, SEL>, smem)) return -1;
    if (attn_launch("kv4_attn launch", k_kv4_attn<D, NT, SEL>, dim3((unsigned)grid), kv4::THREADS, smem, st, false, a)) return -1;
    if (a.whole) return 0;
    // the joining kernel starts while the first drains, and waits for it: a block a
    // column, up to 64 (max_rows may be far above the rows that there are).  The wide
    // form where all blocks are resident at once (131072 positions, 8 segments: 43 us,
    // 47 with the other; 48 sequences, 384 segments: 69 us, 79 with the wide form, each
    // before the sums had maxima of their own).
    const long bx = std::min((long)a.group * a.v.max_rows, 64l);
    const bool wide = bx * a.v.heads * a.v.nseq <= 2 * ATTN_SMS;
    return attn_launch("kv4_attn join launch", wide ? k_kv4_join<D, true> : k_kv4_join<D, false>,
                       dim3((unsigned)bx, a.v.heads, a.v.nseq), wide ? 256 : 128, (3 * KJ_RUNS + (wide ? 256 : 128) * 4) * 4, st,
                       true, a, 8 * NT);
}
template <int D, int NT> int kv4_attn_launch(const Kv4AttnArgs &a, int grid, cudaStream_t st) {
    return a.sel ? kv4_attn_launch<D, NT, true>(a, grid, st) : kv4_attn_launch<D, NT, false>(a, grid, st);
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
    if (kv4_attn_args(what, cache, batch, q->heads, q->rows, &a.v) || attn_check_scale(what, scale)) return -1;
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
    a.group_magic = (((uint64_t)1 << 40) + (uint64_t)a.group - 1) / (uint64_t)a.group;
    a.zscale = scale * 1.4426950408889634f;
    a.sel = sel;
    a.sel_stride = (long)sel_stride;
    a.pool = sel ? (int)pool : 1;
    a.pool_magic = (((uint64_t)1 << 36) + (uint64_t)a.pool - 1) / (uint64_t)a.pool;
    a.whole = p.whole;
    a.min_pages = p.whole ? 1 : (int)MIN_PAGES;
    a.slots = p.slots;
    a.segs = p.segs;
    a.plan = p.whole ? nullptr : (long *)workspace;
    a.part = p.whole ? nullptr : (float *)((char *)workspace + p.plan_bytes);
    cudaStream_t st = (cudaStream_t)stream;
    if (cache->dim == 64) return p.nt == 2 ? kv4_attn_launch<64, 2>(a, p.grid, st) : kv4_attn_launch<64, 1>(a, p.grid, st);
    if (cache->dim == 128) return p.nt == 2 ? kv4_attn_launch<128, 2>(a, p.grid, st) : kv4_attn_launch<128, 1>(a, p.grid, st);
    return kv4_attn_launch<256, 1>(a, p.grid, st);
}

int kv4_attn_error_read_and_clear(void) {
    int v = 0, z = 0;
    cudaMemcpyFromSymbol(&v, g_kv4a_err, sizeof v);
    if (v) cudaMemcpyToSymbol(g_kv4a_err, &z, sizeof z);
    return v;
}
