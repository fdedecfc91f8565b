// prompt_attn.cu — causal attention over packed sequences with grouped heads
// (apus_gcuda_prompt_attn_dev):
//   out_i = sum_{j <= m - n + i} p_ij v_j,  p_i = softmax_j(scale q_i . k_j)
// for row i of n queries over m keys of one sequence.
#include "attn_dev.h"
#include "common.cuh"

namespace apus {

__device__ int g_pa_err;   // attn_dev.h's codes

struct PromptArgs {
    const int32_t *cu_q, *cu_k;
    int nseq, rows_q, rows_k, max_rows;
    RowsView q, k, v, out;
    int heads, group;          // query heads, query heads of a key head
    float zscale;              // scale * log2(e)
};

// A sequence's ranges; one that is out of bounds is empty.
struct PromptSeq { int q0, n, k0, m; };
APUS_DEV PromptSeq prompt_seq(const PromptArgs &a, int s, bool report) {
    const Kv4Seq q = kv4_seq(a.cu_q[s], a.cu_q[s + 1], 0, a.rows_q, a.max_rows, 0);
    const Kv4Seq k = kv4_seq(a.cu_k[s], a.cu_k[s + 1], 0, a.rows_k, a.rows_k, 0);
    if ((q.bad || k.bad) && report) atomicExch(&g_pa_err, (int)ATTN_ERR_SEQ);
    return PromptSeq{q.row0, q.n, k.row0, k.n};
}

// One warp a query row and head, the keys one after another; a lane holds
// D / 32 neighbouring dims.
template <int D>
__global__ void __launch_bounds__(128) k_prompt_rows(const PromptArgs a) {
    constexpr int E = D / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head = blockIdx.y;
    const long row = (long)blockIdx.x * 4 + warp;
    if (row >= a.rows_q) return;
    int lo = 0, hi = a.nseq - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.cu_q[mid] <= row) lo = mid;
        else hi = mid - 1;
    }
    const PromptSeq s = prompt_seq(a, lo, lane == 0);
    if (row < s.q0 || row >= s.q0 + s.n) return;
    const int seen = min(s.m, s.m - s.n + (int)(row - s.q0) + 1);
    const uint16_t *qp = a.q.p + row * a.q.rs + (long)head * a.q.hs + lane * E;
    const uint16_t *kp = a.k.p + (long)s.k0 * a.k.rs + (long)(head / a.group) * a.k.hs + lane * E;
    const uint16_t *vp = a.v.p + (long)s.k0 * a.v.rs + (long)(head / a.group) * a.v.hs + lane * E;
    float q[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < E; i++) { q[i] = bf16_f32(qp[i]) * a.zscale; o[i] = 0.f; }
    for (int j = 0; j < seen; j++) {
        float z = 0.f;
#pragma unroll
        for (int i = 0; i < E; i++) z = fmaf(q[i], bf16_f32(kp[(long)j * a.k.rs + i]), z);
#pragma unroll
        for (int off = 16; off; off >>= 1) z += __shfl_xor_sync(0xffffffffu, z, off);
        if (z > m) {
            const float down = exp2f(m - z);
            l *= down;
#pragma unroll
            for (int i = 0; i < E; i++) o[i] *= down;
            m = z;
        }
        const float p = exp2f(z - m);
        l += p;
#pragma unroll
        for (int i = 0; i < E; i++) o[i] = fmaf(p, bf16_f32(vp[(long)j * a.v.rs + i]), o[i]);
    }
    uint16_t *op = a.out.p + row * a.out.rs + (long)head * a.out.hs + lane * E;
#pragma unroll
    for (int i = 0; i < E; i++) op[i] = bf16_bits(l == 0.f ? 0.f : o[i] / l);
}

}  // namespace apus
using namespace apus;

extern "C" int apus_gcuda_prompt_attn_dev(const ApusPromptBatch *batch, const ApusHeadRows *q, const ApusHeadRows *k,
                                          const ApusHeadRows *v, const ApusHeadRows *out, size_t dim, float scale,
                                          void *stream) {
    const char *what = "prompt_attn";
    if (!batch) { gcuda_set_error("%s: no batch given", what); return -1; }
    if (attn_check_dim(what, dim)) return -1;
    if (attn_check_rows(what, q, dim, false) || attn_check_rows(what, k, dim, false) ||
        attn_check_rows(what, v, dim, false) || attn_check_rows(what, out, dim, true))
        return -1;
    if (q->rows != out->rows || q->heads != out->heads || k->rows != v->rows || k->heads != v->heads ||
        q->heads % k->heads) {
        gcuda_set_error("%s: q %zu rows of %zu heads, out %zu of %zu, k %zu of %zu, v %zu of %zu", what, q->rows,
                        q->heads, out->rows, out->heads, k->rows, k->heads, v->rows, v->heads);
        return -1;
    }
    if (batch->nseq > 65535 || batch->max_rows >= ((size_t)1 << 31) || (batch->nseq && (!batch->cu_q || !batch->cu_k))) {
        gcuda_set_error("%s: %zu sequences of up to %zu rows, or their device arrays missing", what, batch->nseq,
                        batch->max_rows);
        return -1;
    }
    if (!q->rows || !batch->nseq || !batch->max_rows) return 0;
    PromptArgs a{batch->cu_q, batch->cu_k, (int)batch->nseq, (int)q->rows, (int)k->rows, (int)batch->max_rows,
                 rows_view(q), rows_view(k), rows_view(v), rows_view(out), (int)q->heads, (int)(q->heads / k->heads),
                 scale * 1.4426950408889634f};
    const dim3 grid((unsigned)((q->rows + 3) / 4), (unsigned)q->heads);
    cudaStream_t st = (cudaStream_t)stream;
    if (dim == 64) k_prompt_rows<64><<<grid, 128, 0, st>>>(a);
    else if (dim == 128) k_prompt_rows<128><<<grid, 128, 0, st>>>(a);
    else k_prompt_rows<256><<<grid, 128, 0, st>>>(a);
    return gcuda_check(cudaGetLastError(), "prompt_attn launch");
}

int prompt_attn_error_read_and_clear(void) {
    int v = 0, z = 0;
    cudaMemcpyFromSymbol(&v, g_pa_err, sizeof v);
    if (v) cudaMemcpyToSymbol(g_pa_err, &z, sizeof z);
    return v;
}
