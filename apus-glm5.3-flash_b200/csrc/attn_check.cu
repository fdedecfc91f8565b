// attn_check.cu — the host's checks of the structs of
// include/apus_attn_gcuda.h.  No GPU is touched here: a call with bad
// arguments is refused before anything is launched.
#include "attn_dev.h"

int attn_check_dim(const char *what, size_t dim) {
    if (dim == 64 || dim == 128 || dim == 256) return 0;
    gcuda_set_error("%s: head dim %zu (64, 128 or 256)", what, dim);
    return -1;
}

int attn_check_scale(const char *what, float scale) {
    if (scale > 0.0f && scale < 1e30f) return 0;
    gcuda_set_error("%s: scale %g (positive)", what, (double)scale);
    return -1;
}

int attn_check_rows(const char *what, const ApusHeadRows *r, size_t dim, bool output) {
    if (!r) { gcuda_set_error("%s: no rows given", what); return -1; }
    const size_t lim = (size_t)1 << 31;
    if (r->rows >= lim || r->heads < 1 || r->heads > 65535) {
        gcuda_set_error("%s: %zu rows of %zu heads", what, r->rows, r->heads);
        return -1;
    }
    if (r->rows == 0) return 0;
    if (!r->p || ((uintptr_t)r->p & 15)) {
        gcuda_set_error("%s: rows at %p (16-byte aligned device memory)", what, (void *)r->p);
        return -1;
    }
    const bool many_rows = r->rows > 1, many_heads = r->heads > 1;
    if ((many_rows && (r->row_stride % 8 || r->row_stride < dim || r->row_stride >= lim)) ||
        (many_heads && (r->head_stride % 8 || r->head_stride < dim || r->head_stride >= ((size_t)1 << 38)))) {
        gcuda_set_error("%s: strides %zu, %zu (multiples of 8, at least the head dim %zu)", what, r->row_stride,
                        r->head_stride, dim);
        return -1;
    }
    if (output && many_rows && many_heads && r->row_stride < (r->heads - 1) * r->head_stride + dim &&
        r->head_stride < (r->rows - 1) * r->row_stride + dim) {
        gcuda_set_error("%s: output rows and heads overlap (strides %zu, %zu)", what, r->row_stride, r->head_stride);
        return -1;
    }
    return 0;
}

int kv4_check(const char *what, const ApusKv4Cache *c, const ApusKv4Batch *b, size_t rows, Kv4View *out) {
    if (!c || !b) { gcuda_set_error("%s: no cache or batch given", what); return -1; }
    if (attn_check_dim(what, c->dim)) return -1;
    if (c->heads < 1 || c->heads > 65535 || c->num_pages >= ((size_t)1 << 31)) {
        gcuda_set_error("%s: %zu pages of %zu heads", what, c->num_pages, c->heads);
        return -1;
    }
    if (c->num_pages && (!c->pages || ((uintptr_t)c->pages & 15))) {
        gcuda_set_error("%s: pages at %p (16-byte aligned device memory)", what, c->pages);
        return -1;
    }
    const size_t lim = (size_t)1 << 31;
    if (b->nseq > 65535 || b->max_rows >= lim || b->max_len >= lim - KV4_PAGE || b->table_stride >= lim) {
        gcuda_set_error("%s: %zu sequences of up to %zu rows, %zu positions", what, b->nseq, b->max_rows, b->max_len);
        return -1;
    }
    if (b->max_len > b->table_stride * KV4_PAGE) {
        gcuda_set_error("%s: %zu positions in a table of %zu pages", what, b->max_len, b->table_stride);
        return -1;
    }
    if (b->nseq && (!b->cu_rows || !b->kv_len || (b->table_stride && !b->page_table))) {
        gcuda_set_error("%s: a device array of the batch is missing", what);
        return -1;
    }
    if (out)
        *out = Kv4View{(uint8_t *)c->pages, (long)c->num_pages, (int)c->heads, (int)c->dim, b->cu_rows, b->kv_len,
                       b->page_table, (long)b->table_stride, (int)b->nseq, (int)rows, (int)b->max_rows,
                       (int)b->max_len};
    return 0;
}

extern "C" size_t apus_gcuda_kv4_page_bytes(size_t heads, size_t dim) {
    if (attn_check_dim("kv4_page_bytes", dim)) return 0;
    return heads * 72 * dim;
}
