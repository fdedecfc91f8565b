// attn_dev.h — what the translation units of include/apus_attn_gcuda.h share:
// the host's checks of arguments, and the device error word.
#pragma once
#include "gcuda.h"
#include "kv4_layout.h"
#include "../../include/apus_attn_gcuda.h"

static_assert(KV4_PAGE == APUS_KV4_PAGE && KV4_GROUP == APUS_KV4_GROUP, "public and internal layout");

// The worse, the larger (43: a bounded wait gave up).  A word takes two of them: the
// larger is exchanged in, the smaller goes only where none stands (atomicMax for both
// took 0.25 us of a short call).
enum { ATTN_ERR_PAGE = 41, ATTN_ERR_SEQ = 42, ATTN_ERR_WAIT = 43 };

// SMs of a B200, by which work is cut.  A constant: the workspace that a batch needs may
// be asked for on a host without a GPU, and has to be what the call then uses.
enum { ATTN_SMS = 148 };

// Device views of the public structs (sizes checked to fit ints).
struct Kv4View {
    uint8_t *pages;
    long num_pages;
    int heads, dim;
    const int32_t *cu, *len, *table;
    long table_stride;
    int nseq;
    int rows;                 // row capacity of the row arrays
    int max_rows, max_len;
};
struct RowsView {
    uint16_t *p;
    long rs, hs;              // row and head strides
};

// Argument checks (attn_check.cu); each records the reason and returns -1.
int attn_check_rows(const char *what, const ApusHeadRows *r, size_t dim, bool output);
int attn_check_dim(const char *what, size_t dim);
int attn_check_scale(const char *what, float scale);
int kv4_check(const char *what, const ApusKv4Cache *c, const ApusKv4Batch *b, size_t rows, Kv4View *out);
static inline RowsView rows_view(const ApusHeadRows *r) {
    return RowsView{r->p, (long)r->row_stride, (long)r->head_stride};
}
// Launches a kernel and goes by what this launch returns: cudaGetLastError would also
// give an error that an earlier call of the library left (a refused allocation, say).
template <class... P, class... A>
int attn_launch(const char *what, void (*kernel)(P...), dim3 grid, int threads, int smem, cudaStream_t stream, bool dependent,
                const A &...args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = stream;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = dependent ? 1 : 0;       // starts while the kernel before drains, and waits for it
    return gcuda_check(cudaLaunchKernelEx(&cfg, kernel, args...), what);
}
// the device error words
int kv4_cache_error_read_and_clear(void);
int kv4_attn_error_read_and_clear(void);
int prompt_attn_error_read_and_clear(void);
