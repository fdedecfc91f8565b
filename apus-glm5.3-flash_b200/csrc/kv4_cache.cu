// kv4_cache.cu — the 4-bit cache's rows: quantised as they are written
// (apus_gcuda_kv4_append_dev) and read back (apus_gcuda_kv4_read_dev).
//
// Per group of 32 dims: s = bf16(max |x| / 7), code = clamp(rint(x / s), -7,
// 7) + 8, value (code - 8) * s.  Divisions are IEEE divisions of BF16 values
// in fp32; a quotient of two 8-bit significands is never closer than 2^-13
// (relative) to a rounding border without lying on it, so fp32 takes the same
// decisions as exact arithmetic.
//
// Both are streams bound by HBM once there are some thousand rows (append
// reads 2 * dim * 2 bytes a row and head and writes 2 * (dim / 2 + dim / 16);
// read the other way) and by latency below.  A thread takes eight dims of one
// head's key or value row: one 16-byte access on the BF16 side; the four
// threads of a scale group are neighbours.  Its eight dims are one word of key
// codes; of value codes, which interleave two scale groups, a thread and the
// one four lanes away hold the halves of two words, which one shuffle turns
// into a whole word each.
#include "attn_dev.h"
#include "common.cuh"

namespace apus {

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

// Place of a row: false when the row belongs to no sequence (in = false), or
// stands before position 0 or in no page (in = true).
struct Kv4Place { uint8_t *block; int off; bool in; };
APUS_DEV bool kv4_place(const Kv4View &v, int row, int head, bool report, Kv4Place *pl) {
    pl->in = false;
    const int s = seq_of_row(v.cu, v.nseq, row);
    const Kv4Seq q = kv4_seq(v.cu[s], v.cu[s + 1], v.len[s], v.rows, v.max_rows, v.max_len);
    if (q.bad && report) atomicExch(&g_kv4_err, (int)ATTN_ERR_SEQ);
    if (row < q.row0 || row >= q.row0 + q.n) return false;
    pl->in = true;
    const int pos = q.len - q.n + (row - q.row0);
    if (pos < 0) return false;
    const int page = v.table[(long)s * v.table_stride + pos / KV4_PAGE];
    if (!kv4_page_ok(page, v.num_pages)) {
        if (report) atomicExch(&g_kv4_err, (int)ATTN_ERR_PAGE);
        return false;
    }
    pl->block = v.pages + kv4_block_at(page, head, v.heads, v.dim);
    pl->off = pos & (KV4_PAGE - 1);
    return true;
}

// What a thread of a block takes: eight dims (c) of the key or value row of
// one head; a block takes 1024 / D rows of one head, and the heads of a
// row block are neighbouring blocks.
template <int D> struct Kv4Part {
    static constexpr int C = D / 8, ROWS = 256 / (2 * C);
    int c, val, head;
    long row;
    APUS_DEV Kv4Part(int heads) {
        c = threadIdx.x % C;
        val = (threadIdx.x / C) & 1;
        head = (int)(blockIdx.x % (unsigned)heads);
        row = (long)(blockIdx.x / (unsigned)heads) * ROWS + threadIdx.x / (2 * C);
    }
};

template <int D>
__global__ void __launch_bounds__(256) k_kv4_append(Kv4View v, RowsView k, RowsView x) {
    const Kv4Part<D> me(v.heads);
    const int c = me.c, val = me.val, head = me.head, row = (int)me.row;
    const bool on = me.row < v.rows;             // the same for all threads of a scale group
    uint4 raw = make_uint4(0, 0, 0, 0);
    const RowsView &src = val ? x : k;
    if (on) raw = *(const uint4 *)(src.p + me.row * src.rs + head * src.hs + c * 8);
    Kv4Place pl;
    const bool put = on && kv4_place(v, row, head, c == 0, &pl);
    float f[8] = {bf16lo(raw.x), bf16hi(raw.x), bf16lo(raw.y), bf16hi(raw.y),
                  bf16lo(raw.z), bf16hi(raw.z), bf16lo(raw.w), bf16hi(raw.w)};
    // the largest magnitude as bits, so a NaN or an infinity wins
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const bool fine = top < 0x7f800000u;
    const uint16_t sb = fine ? bf16_bits(__fdiv_rn(__uint_as_float(top), 7.0f)) : (uint16_t)0x7fc0;
    const float s = bf16_f32(sb);
    uint32_t word = 0x88888888u;                 // all zeros
    if (fine && s > 0.0f) {
        word = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float q = fminf(fmaxf(rintf(__fdiv_rn(f[i], s)), -7.0f), 7.0f);
            word |= (uint32_t)((int)q + 8) << (4 * i);
        }
    }
    const int j = c >> 2, q4 = c & 3;            // group of 32 dims, quarter of it
    // values: this thread has dims 32 j + 8 q4 .., the halves of words g = 2 q4
    // (low 16 bits) and 2 q4 + 1; an even group keeps the first, an odd one the second
    const uint32_t give = (j & 1) ? (word & 0xffffu) : (word >> 16);
    const uint32_t got = __shfl_xor_sync(0xffffffffu, give, 4);
    if (!put) return;
    uint32_t *codes = (uint32_t *)(pl.block + (val ? kv4_v_codes(D) : 0) + pl.off * (D / 2));
    uint16_t *scale = (uint16_t *)(pl.block + (val ? kv4_v_scales(D) : kv4_k_scales(D))) + pl.off * (D / 32);
    if (!val) codes[kv4_k_word(D, pl.off, j, q4)] = word;
    else if (!(j & 1)) codes[kv4_v_word(D, pl.off, 2 * q4, j >> 1)] = (word & 0xffffu) | (got << 16);
    else codes[kv4_v_word(D, pl.off, 2 * q4 + 1, j >> 1)] = got | (word & 0xffff0000u);
    if (q4 == 0) scale[j] = sb;
}

template <int D>
__global__ void __launch_bounds__(256) k_kv4_read(Kv4View v, RowsView k, RowsView x) {
    const Kv4Part<D> me(v.heads);
    if (me.row >= v.rows) return;
    const int c = me.c, val = me.val, head = me.head, row = (int)me.row;
    Kv4Place pl;
    const bool have = kv4_place(v, row, head, c == 0, &pl);
    if (!pl.in) return;
    uint4 o = make_uint4(0, 0, 0, 0);
    if (have) {
        const int j = c >> 2, q4 = c & 3;
        const uint32_t *codes = (const uint32_t *)(pl.block + (val ? kv4_v_codes(D) : 0) + pl.off * (D / 2));
        const float s = bf16_f32(((const uint16_t *)(pl.block + (val ? kv4_v_scales(D) : kv4_k_scales(D))))
                                     [pl.off * (D / 32) + j]);
        uint32_t word;
        if (!val) word = codes[kv4_k_word(D, pl.off, j, q4)];
        else {
            const int sh = (j & 1) * 16;
            word = ((codes[kv4_v_word(D, pl.off, 2 * q4, j >> 1)] >> sh) & 0xffffu) |
                   ((codes[kv4_v_word(D, pl.off, 2 * q4 + 1, j >> 1)] >> sh) << 16);
        }
        uint32_t b[8];
#pragma unroll
        for (int i = 0; i < 8; i++) b[i] = bf16_bits((float)((int)((word >> (4 * i)) & 15u) - 8) * s);
        o = make_uint4(b[0] | b[1] << 16, b[2] | b[3] << 16, b[4] | b[5] << 16, b[6] | b[7] << 16);
    }
    const RowsView &dst = val ? x : k;
    *(uint4 *)(dst.p + me.row * dst.rs + head * dst.hs + c * 8) = o;
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

template <int D, bool READ>
static int kv4_rows_launch(const char *what, const Kv4View &view, const ApusHeadRows *k, const ApusHeadRows *v,
                           void *stream) {
    const long blocks = ((long)k->rows + Kv4Part<D>::ROWS - 1) / Kv4Part<D>::ROWS * view.heads;
    if (blocks >= (1l << 31)) { gcuda_set_error("%s: %zu rows of %d heads", what, k->rows, view.heads); return -1; }
    if (READ) k_kv4_read<D><<<(unsigned)blocks, 256, 0, (cudaStream_t)stream>>>(view, rows_view(k), rows_view(v));
    else k_kv4_append<D><<<(unsigned)blocks, 256, 0, (cudaStream_t)stream>>>(view, rows_view(k), rows_view(v));
    return gcuda_check(cudaGetLastError(), what);
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
