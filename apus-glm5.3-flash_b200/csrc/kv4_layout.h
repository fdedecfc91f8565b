// kv4_layout.h — where a row of the 4-bit cache stands (the layout that
// include/apus_attn_gcuda.h states), and the bounds every kernel applies to
// what the host cannot see.  Plain C++ as well as device code, so the index
// arithmetic is tested without a GPU.
#pragma once
#include <stddef.h>
#include <stdint.h>

#ifdef __CUDACC__
#define KV4_FN __host__ __device__ __forceinline__
#else
#define KV4_FN static inline
#endif

enum { KV4_PAGE = 64, KV4_GROUP = 32 };

// Byte offsets inside one head's block of a page.
KV4_FN int kv4_block_bytes(int dim) { return 72 * dim; }
KV4_FN int kv4_v_codes(int dim) { return 32 * dim; }
KV4_FN int kv4_k_scales(int dim) { return 64 * dim; }
KV4_FN int kv4_v_scales(int dim) { return 68 * dim; }

// Word (of a position's row of codes) of the eight key codes of dims
// 32 j + 8 q .. + 7, at position p of the page: a lane q of a quad finds the
// words of up to four groups side by side.
KV4_FN int kv4_k_word(int dim, int p, int j, int q) {
    if (dim == 64) return 2 * q + j;
    if (dim == 128) return 4 * q + j;
    return 16 * ((j >> 2) ^ ((p >> 2) & 1)) + 4 * q + (j & 3);
}

// Word of the value codes of dims 64 jj + 4 g .. + 3 (codes 0-3) and
// 64 jj + 32 + 4 g .. + 3 (codes 4-7): a lane group g finds all its dims side
// by side; the XOR by the position spreads the four positions that a quad
// reads at once over the shared-memory banks.
KV4_FN int kv4_v_word(int dim, int p, int g, int jj) {
    if (dim == 64) return g;
    if (dim == 128) return 2 * (g ^ (((p >> 1) & 1) << 2)) + jj;
    return 4 * (g ^ ((p & 3) << 1)) + jj;
}

// Offset of one head's block; page ids reach past 32 bits of bytes.
KV4_FN size_t kv4_block_at(int page, int head, int heads, int dim) {
    return ((size_t)page * (size_t)heads + (size_t)head) * (size_t)kv4_block_bytes(dim);
}

// The rows and the length of a sequence.  A row range outside 0 .. rows or of
// more than max_rows counts as no rows, a length outside 0 .. max_len as 0;
// bad = 1 for either.
struct Kv4Seq { int row0, n, len, bad; };
KV4_FN struct Kv4Seq kv4_seq(int lo, int hi, int len, long rows, long max_rows, long max_len) {
    struct Kv4Seq s;
    const int range_ok = lo >= 0 && hi >= lo && hi <= rows && (long)hi - lo <= max_rows;
    const int len_ok = len >= 0 && len <= max_len;
    s.row0 = range_ok ? lo : 0;
    s.n = range_ok ? hi - lo : 0;
    s.len = len_ok ? len : 0;
    s.bad = !(range_ok && len_ok);
    return s;
}
KV4_FN int kv4_page_ok(int page, long num_pages) { return page >= 0 && page < num_pages; }
