// kv4_cache.cu — the 4-bit cache's rows: quantised as they are written
// (apus_gcuda_kv4_append_dev) and read back (apus_gcuda_kv4_read_dev).
//
// Per group of 32 dims: s = bf16(max |x| / 7), code = clamp(rint(x / s), -7,
// 7) + 8, value (code - 8) * s.  A quotient of two 8-bit significands is never
// closer than 2^-13 (relative) to a rounding border without lying on it, so
// correctly rounded fp32 quotients take the same decisions as exact arithmetic.
// They come from one approximate reciprocal a group, y = x r, and one correction
// by the remainder, y + r (x - y s): the remainder is exact in a fused
// multiply-add, so the correction leaves y off by 2^-44, and where the quotient is
// a number and a half it comes out as that.  Rounding, offset and conversion are
// one addition of 1.5 2^23 + 8, which leaves the code in the low bits.  Scales
// below 1e-20 take divisions.
//
// Both are streams bound by HBM once there are some thousand rows (append
// reads 2 * dim * 2 bytes a row and head and writes 2 * (dim / 2 + dim / 16);
// read the other way) and by latency below.  A thread takes eight dims (one
// 16-byte access on the BF16 side) of a row, for IT of its keys and values of
// heads: where a row stands is looked up once for them, which costs as much as
// two of them, and their loads are in flight together (one at a time, 256 rows of
// 64 heads of 256 took 22 us to write and read back).  The four threads of a scale
// group are neighbours.  Eight dims are one word of key codes; of value codes,
// which interleave two scale groups, a thread and the one four lanes away hold
// the halves of two words, which one shuffle turns into a whole word each.
#include "attn_dev.h"
#include "common.cuh"

namespace apus {

// Packed BF16 of two floats.
APUS_DEV uint32_t kv4_pack(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}

__device__ int g_kv4_err;   // an id, length or row range out of bounds (attn_dev.h)

// Sequence of a row: the last s with cu[s] <= row (cu ascends; with entries
// out of order the search still ends, and kv4_seq's bounds hold).
APUS_DEV int seq_of_row(const int32_t *cu, int nseq, int row) {
    int lo = 0, hi = nseq - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (cu[mid] <= row) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Place of a row in its page: in = it belongs to a sequence, page < 0 = it
// stands before position 0 or in no page.
struct Kv4Place { int page, off; bool in; };
APUS_DEV Kv4Place kv4_place(const Kv4View &v, int row, bool report) {
    const int s = seq_of_row(v.cu, v.nseq, row);
    const Kv4Seq q = kv4_seq(v.cu[s], v.cu[s + 1], v.len[s], v.rows, v.max_rows, v.max_len);
    Kv4Place pl{-1, 0, row >= q.row0 && row < q.row0 + q.n};
    const int pos = q.len - q.n + (row - q.row0);
    if (!pl.in || pos < 0) return pl;
    const int page = v.table[(long)s * v.table_stride + pos / KV4_PAGE];
    if (kv4_page_ok(page, v.num_pages)) {
        pl.page = page;
        pl.off = pos & (KV4_PAGE - 1);
    } else if (report) {
        atomicCAS(&g_kv4_err, 0, (int)ATTN_ERR_PAGE);
    }
    return pl;
}

// Reports every sequence out of bounds, those that no row leads to among them (the
// grid's first row of blocks, a thread a sequence while there are enough).
APUS_DEV void kv4_report(const Kv4View &v) {
    if (blockIdx.y || blockIdx.x >= 256) return;      // (at most 65535 sequences)
#pragma unroll 1
    for (int s = blockIdx.x * 256 + threadIdx.x; s < v.nseq; s += min(gridDim.x, 256) * 256)
        if (kv4_seq(v.cu[s], v.cu[s + 1], v.len[s], v.rows, v.max_rows, v.max_len).bad)
            atomicExch(&g_kv4_err, (int)ATTN_ERR_SEQ);
}

// Thread -> eight dims (c) of a row; items blockIdx.y * IT .. + IT - 1 of the
// row: keys and values of head 0, of head 1, ...
template <int D> struct Kv4Part {
    static constexpr int C = D / 8, ROWS = 256 / C;         // threads of a row, rows of a block
    int c;
    long row;
    APUS_DEV Kv4Part() {
        c = threadIdx.x % C;
        row = (long)blockIdx.x * ROWS + threadIdx.x / C;
    }
};

template <int D, int IT>
__global__ void __launch_bounds__(256) k_kv4_append(Kv4View v, RowsView k, RowsView x) {
    const Kv4Part<D> me;
    const int c = me.c, items = 2 * v.heads, it0 = blockIdx.y * IT;
    const bool on = me.row < v.rows;             // the same for all threads of a row
    uint4 raw[IT];
#pragma unroll
    for (int i = 0; i < IT; i++) {
        const RowsView &src = (i + it0) & 1 ? x : k;
        raw[i] = on && it0 + i < items ? *(const uint4 *)(src.p + me.row * src.rs + ((it0 + i) >> 1) * src.hs + c * 8)
                                       : make_uint4(0, 0, 0, 0);
    }
    Kv4Place pl{-1, 0, false};
    if (on) pl = kv4_place(v, (int)me.row, c == 0);
    kv4_report(v);
    const int j = c >> 2, q4 = c & 3;            // group of 32 dims, quarter of it
#pragma unroll
    for (int i = 0; i < IT; i++) {
        // the largest magnitude as BF16 bits, so a NaN or an infinity wins
        uint32_t top2 = __vmaxu2(__vmaxu2(raw[i].x & 0x7fff7fffu, raw[i].y & 0x7fff7fffu),
                                 __vmaxu2(raw[i].z & 0x7fff7fffu, raw[i].w & 0x7fff7fffu));
        top2 = __vmaxu2(top2, __shfl_xor_sync(0xffffffffu, top2, 1));
        top2 = __vmaxu2(top2, __shfl_xor_sync(0xffffffffu, top2, 2));
        const uint32_t top = max(top2 & 0xffffu, top2 >> 16);
        const float f[8] = {bf16lo(raw[i].x), bf16hi(raw[i].x), bf16lo(raw[i].y), bf16hi(raw[i].y),
                            bf16lo(raw[i].z), bf16hi(raw[i].z), bf16lo(raw[i].w), bf16hi(raw[i].w)};
        const bool fine = top < 0x7f80u;
        const float amax = bf16_f32((uint16_t)top);
        float s7;                                // amax / 7, rounded
        if (amax >= 1e-20f) {
            const float y0 = amax * 0.14285714285714285f;
            s7 = fmaf(fmaf(-y0, 7.0f, amax), 0.14285714285714285f, y0);
        } else {
            s7 = __fdiv_rn(amax, 7.0f);
        }
        const uint16_t sb = fine ? (uint16_t)kv4_pack(s7, 0.0f) : (uint16_t)0x7fc0;
        const float s = bf16_f32(sb);
        uint32_t word = 0x88888888u;             // all zeros
        if (fine && s >= 1e-20f) {               // amax / s is 7.03 at most: nothing to clamp
            float r;
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
            word = 0;
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const float y0 = f[u] * r, y = fmaf(fmaf(-y0, s, f[u]), r, y0);
                word += __float_as_uint(y + 12582920.0f) << (4 * u);     // 0x4b400000 + code
            }
            word -= 0x4b400000u * 0x11111111u;
        } else if (fine && s > 0.0f) {
            word = 0;
#pragma unroll 1
            for (int u = 0; u < 8; u++) {
                const uint32_t pair = u < 2 ? raw[i].x : u < 4 ? raw[i].y : u < 6 ? raw[i].z : raw[i].w;
                const float y = __fdiv_rn((u & 1) ? bf16hi(pair) : bf16lo(pair), s);
                word |= (uint32_t)((int)rintf(fminf(fmaxf(y, -7.0f), 7.0f)) + 8) << (4 * u);
            }
        }
        const int val = (it0 + i) & 1;
        // values: this thread has dims 32 j + 8 q4 .., the halves of words g = 2 q4
        // (low 16 bits) and 2 q4 + 1; an even group keeps the first, an odd one the second
        const uint32_t give = (j & 1) ? (word & 0xffffu) : (word >> 16);
        const uint32_t got = __shfl_xor_sync(0xffffffffu, give, 4);
        if (pl.page < 0 || it0 + i >= items) continue;
        uint8_t *block = v.pages + kv4_block_at(pl.page, (it0 + i) >> 1, v.heads, D);
        uint32_t *codes = (uint32_t *)(block + (val ? kv4_v_codes(D) : 0) + pl.off * (D / 2));
        if (!val) codes[kv4_k_word(D, pl.off, j, q4)] = word;
        else if (!(j & 1)) codes[kv4_v_word(D, pl.off, 2 * q4, j >> 1)] = (word & 0xffffu) | (got << 16);
        else codes[kv4_v_word(D, pl.off, 2 * q4 + 1, j >> 1)] = got | (word & 0xffff0000u);
        if (q4 == 0)
            ((uint16_t *)(block + (val ? kv4_v_scales(D) : kv4_k_scales(D))))[pl.off * (D / 32) + j] = sb;
    }
}

template <int D, int IT>
__global__ void __launch_bounds__(256) k_kv4_read(Kv4View v, RowsView k, RowsView x) {
    const Kv4Part<D> me;
    kv4_report(v);
    if (me.row >= v.rows) return;
    const int c = me.c, items = 2 * v.heads, it0 = blockIdx.y * IT;
    const Kv4Place pl = kv4_place(v, (int)me.row, c == 0);
    if (!pl.in) return;
    const int j = c >> 2, q4 = c & 3;
    uint32_t w[IT][2];
    uint16_t sb[IT];
#pragma unroll
    for (int i = 0; i < IT; i++) {
        w[i][0] = w[i][1] = 0;
        sb[i] = 0;
        if (pl.page < 0 || it0 + i >= items) continue;
        const int val = (it0 + i) & 1;
        const uint8_t *block = v.pages + kv4_block_at(pl.page, (it0 + i) >> 1, v.heads, D);
        const uint32_t *codes = (const uint32_t *)(block + (val ? kv4_v_codes(D) : 0) + pl.off * (D / 2));
        if (!val) {
            w[i][0] = codes[kv4_k_word(D, pl.off, j, q4)];
        } else {
            w[i][0] = codes[kv4_v_word(D, pl.off, 2 * q4, j >> 1)];
            w[i][1] = codes[kv4_v_word(D, pl.off, 2 * q4 + 1, j >> 1)];
        }
        sb[i] = ((const uint16_t *)(block + (val ? kv4_v_scales(D) : kv4_k_scales(D))))[pl.off * (D / 32) + j];
    }
#pragma unroll
    for (int i = 0; i < IT; i++) {
        if (it0 + i >= items) return;
        const int val = (it0 + i) & 1, sh = (j & 1) * 16;
        const uint32_t word = val ? ((w[i][0] >> sh) & 0xffffu) | ((w[i][1] >> sh) << 16) : w[i][0];
        const float s = bf16_f32(sb[i]);
        float f[8];
#pragma unroll
        for (int u = 0; u < 8; u++) f[u] = (__uint_as_float(((word >> (4 * u)) & 15u) | 0x4b400000u) - 12582920.0f) * s;
        const RowsView &dst = val ? x : k;
        // a row in no page reads as zeros: its scale is 0 (and -8 times 0 is -0)
        *(uint4 *)(dst.p + me.row * dst.rs + ((it0 + i) >> 1) * dst.hs + c * 8) =
            pl.page < 0 ? make_uint4(0, 0, 0, 0)
                        : make_uint4(kv4_pack(f[0], f[1]), kv4_pack(f[2], f[3]), kv4_pack(f[4], f[5]), kv4_pack(f[6], f[7]));
    }
}

}  // namespace apus
using namespace apus;

static int kv4_rows_check(const char *what, const ApusKv4Cache *c, const ApusKv4Batch *b, const ApusHeadRows *k,
                          const ApusHeadRows *v, bool output, Kv4View *view) {
    if (kv4_check(what, c, b, k ? k->rows : 0, view)) return -1;
    if (attn_check_rows(what, k, c->dim, output) || attn_check_rows(what, v, c->dim, output)) return -1;
    if (k->rows != v->rows || k->heads != c->heads || v->heads != c->heads) {
        gcuda_set_error("%s: %zu rows of %zu heads and %zu of %zu, cache of %zu heads", what, k->rows, k->heads,
                        v->rows, v->heads, c->heads);
        return -1;
    }
    return 0;
}

template <int D, bool READ, int IT>
static int kv4_rows_launch(const char *what, const Kv4View &view, const ApusHeadRows *k, const ApusHeadRows *v,
                           void *stream) {
    const long bx = ((long)k->rows + Kv4Part<D>::ROWS - 1) / Kv4Part<D>::ROWS, by = (2l * view.heads + IT - 1) / IT;
    const dim3 grid((unsigned)bx, (unsigned)by);
    return attn_launch(what, READ ? k_kv4_read<D, IT> : k_kv4_append<D, IT>, grid, 256, 0, (cudaStream_t)stream, false, view,
                       rows_view(k), rows_view(v));
}

// Four items a thread where that still gives every SM two blocks (256 rows of 64
// heads of 256 written and read back: 13.9 us; two items 14.1, eight 15.2), two
// below (the grid's second axis takes 65535, so two up to 65535 heads).
template <int D, bool READ>
static int kv4_rows_launch(const char *what, const Kv4View &view, const ApusHeadRows *k, const ApusHeadRows *v,
                           void *stream) {
    const long blocks = ((long)k->rows + Kv4Part<D>::ROWS - 1) / Kv4Part<D>::ROWS * ((2l * view.heads + 3) / 4);
    return blocks >= 2 * ATTN_SMS ? kv4_rows_launch<D, READ, 4>(what, view, k, v, stream)
                                  : kv4_rows_launch<D, READ, 2>(what, view, k, v, stream);
}

template <bool READ>
static int kv4_rows(const char *what, const ApusKv4Cache *c, const ApusKv4Batch *b, const ApusHeadRows *k,
                    const ApusHeadRows *v, void *stream) {
    Kv4View view;
    if (kv4_rows_check(what, c, b, k, v, READ, &view)) return -1;
    if (!k->rows || !b->nseq || !b->max_rows) return 0;
    if (c->dim == 64) return kv4_rows_launch<64, READ>(what, view, k, v, stream);
    if (c->dim == 128) return kv4_rows_launch<128, READ>(what, view, k, v, stream);
    return kv4_rows_launch<256, READ>(what, view, k, v, stream);
}

extern "C" int apus_gcuda_kv4_append_dev(const ApusKv4Cache *cache, const ApusKv4Batch *batch, const ApusHeadRows *k,
                                         const ApusHeadRows *v, void *stream) {
    return kv4_rows<false>("kv4_append", cache, batch, k, v, stream);
}

extern "C" int apus_gcuda_kv4_read_dev(const ApusKv4Cache *cache, const ApusKv4Batch *batch, const ApusHeadRows *k,
                                       const ApusHeadRows *v, void *stream) {
    return kv4_rows<true>("kv4_read", cache, batch, k, v, stream);
}

int kv4_cache_error_read_and_clear(void) {
    int v = 0, z = 0;
    cudaMemcpyFromSymbol(&v, g_kv4_err, sizeof v);
    if (v) cudaMemcpyToSymbol(g_kv4_err, &z, sizeof z);
    return v;
}
