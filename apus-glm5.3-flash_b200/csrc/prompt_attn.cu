// prompt_attn.cu — causal attention over packed sequences with grouped heads
// (apus_gcuda_prompt_attn_dev):
//   out_i = sum_{j <= m - n + i} p_ij v_j,  p_i = softmax_j(scale q_i . k_j)
// for row i of n queries over m keys of one sequence, in one pass over the keys
// with a running maximum and sum.
//
// Both products run on tcgen05: a CTA takes NQ tiles of 128 query rows of one
// head and walks the keys in tiles of 128,
//   S (TMEM, fp32) = Q (shared) . K^T (shared),   O (TMEM, fp32) += P (TMEM) . V (shared),
// with P = 2^(scale log2(e) (S - maximum)) in BF16 written over S.  K and V come as
// tensor copies (128-byte swizzle) into a ring; V is read as it lies, rows of
// keys with the dims contiguous.
//
// Bound: at dim 256 the products (2048 tensor cycles a tile of 128 x 128), at
// dim 128 products and exponentials alike (1024 tensor cycles; 16384
// exponentials at 16 a cycle), at dim 64 the exponentials.
// Up to dim 128 two query tiles share an SM, so that each K and V tile serves 256
// rows and one tile's softmax runs under the other's products.  S has one place
// in TMEM, which the softmax frees as soon as it holds the scores in registers; P
// has a place of its own.  So the next S is there when a softmax ends, and the two
// softmaxes take turns at the exponentials (at dim 64, with an S place each, they
// ran in step and took 10% longer).  (With P
// written over S, a query tile waited 1400 of 3700 cycles for its own products;
// two S tiles of 64 keys made the products of S, which read 128 rows of Q for 64
// keys, the bound.)
//
// Roles: warp 0 copies, warp 1 issues the products of S, warp 3 those of O (one
// warp for both spent 3400 cycles on issuing 2048 cycles of products), warp 2
// looks after V tiles with keys that some row must not see, warps 4.. are one
// softmax group of 128 threads (a row each) a query tile.  The maximum is raised, and O rescaled, only
// when a score passes it by more than 2^8, so almost never.
//
// A hidden key's weight is 0, but 0 times a NaN or an infinity in its value would
// reach the row through the product.  So in tiles with hidden keys such values
// (and all rows behind the sequence) are set to 0 in shared memory before the
// product reads them; the first key with a NaN, a +inf and a -inf is kept for each
// dim, and the rows that see it get it added at the end.
#include "attn_dev.h"
#include "common.cuh"
#include "pipe.cuh"
#include "tc.cuh"

namespace apus {

__device__ int g_pa_err;   // attn_dev.h's codes

struct PromptArgs {
    const int32_t *cu_q, *cu_k;
    int nseq, rows_q, rows_k, max_rows;
    RowsView q, k, v, out;
    int heads, group;          // query heads, query heads of a key head
    float zscale;              // scale * log2(e), positive
};

// A sequence's ranges; one that is out of bounds is empty.
struct PromptSeq { int q0, n, k0, m; };
APUS_DEV PromptSeq prompt_seq(const PromptArgs &a, int s, bool report) {
    const Kv4Seq q = kv4_seq(a.cu_q[s], a.cu_q[s + 1], 0, a.rows_q, a.max_rows, 0);
    const Kv4Seq k = kv4_seq(a.cu_k[s], a.cu_k[s + 1], 0, a.rows_k, a.rows_k, 0);
    if ((q.bad || k.bad) && report) atomicExch(&g_pa_err, (int)ATTN_ERR_SEQ);
    return PromptSeq{q.row0, q.n, k.row0, k.n};
}

namespace pa {
constexpr int BM = 128, BN = 128;               // query rows of a tile, keys of a K or V tile
constexpr int PANEL = 128 * 128;                // bytes of 128 rows of 64 dims
template <int D> struct Cfg {
    static constexpr int NQ = D == 256 ? 1 : 2;             // query tiles of a CTA
    static constexpr int THREADS = 128 + 128 * NQ;
    static constexpr int SPAN = D == 256 ? 128 : D;         // dims of a ring stage
    static constexpr int PARTS = D / SPAN;                  // stages of a K or V tile
    static constexpr int STAGE = SPAN / 64 * PANEL;
    static constexpr int QTILE = D / 64 * PANEL;
    static constexpr int NST = D == 256 ? 5 : D == 128 ? 4 : 8;
    static constexpr int SMEM = NQ * QTILE + NST * STAGE + 1024;
    static constexpr int ROWS = NQ * BM;
    static constexpr int P_COL = 128, O_COL = 256;          // TMEM columns: S from 0, P (two places), O
    // D f32, A and B BF16, N >> 3 at bit 17, M >> 4 at bit 24; V has its dims
    // (N) contiguous: bit 16
    static constexpr uint32_t IDESC_S = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) |
                                        ((uint32_t)(BM >> 4) << 24);
    static constexpr uint32_t IDESC_O = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) |
                                        ((uint32_t)(SPAN >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
};
constexpr float RAISE = 8.0f;
}  // namespace pa

APUS_DEV float pa_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
APUS_DEV uint32_t pa_pack(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}

template <int D>
__global__ void __launch_bounds__(pa::Cfg<D>::THREADS, 1)
k_prompt_tc(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
            const __grid_constant__ CUtensorMap vmap, const PromptArgs a) {
    using C = pa::Cfg<D>;
    constexpr int NQ = C::NQ, NST = C::NST, PARTS = C::PARTS;
    extern __shared__ __align__(1024) uint8_t pa_dyn[];
    __shared__ __align__(8) uint64_t q_full[PARTS], full[NST], empty[NST], checked[NST], s_free, s_full[2], p_full[2], o_done[2];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag, poison, found_s[2], wsum[C::THREADS / 32];
    // first key (from the first looked after, 1023: none) with a NaN, +inf, -inf in
    // a dim, ten bits each; at most four tiles are looked after
    __shared__ uint32_t first_bad[D];
    // (a shuffle tells the compiler that it is the same for the warp, so that the
    // products' operands stay in uniform registers)
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;

    // ---- this CTA's rows: blocks of ROWS rows, a sequence's last block (the one
    // with the most keys) first
    const int head = (int)(blockIdx.x % (unsigned)a.heads), block = (int)(blockIdx.x / (unsigned)a.heads);
    if (tid == 0) found_s[0] = -1;
    for (int i = tid; i < D; i += C::THREADS) first_bad[i] = 0x3fffffffu;
    if (tid == 0) {
        for (int p = 0; p < PARTS; p++) mbar_init(&q_full[p], 1);
        for (int s = 0; s < NST; s++) { mbar_init(&full[s], 1); mbar_init(&empty[s], 2); mbar_init(&checked[s], 1); }   // empty: products, scan
        mbar_init(&s_free, 128);
        for (int i = 0; i < 2; i++) { mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 128); mbar_init(&o_done[i], 1); }
        abort_flag = 0;
        poison = 0;
        fence_barrier_init();
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    {
        int before = 0;
        for (int s0 = 0; s0 < a.nseq && before <= block; s0 += C::THREADS) {
            const int s = s0 + tid;
            const int w = s < a.nseq ? (prompt_seq(a, s, blockIdx.x == 0).n + C::ROWS - 1) / C::ROWS : 0;
            int incl = w;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int o = __shfl_up_sync(0xffffffffu, incl, off);
                if (lane >= off) incl += o;
            }
            if (lane == 31) wsum[warp] = incl;
            __syncthreads();
            int at = before + incl - w;
            for (int k = 0; k < C::THREADS / 32; k++) {
                if (k < warp) at += wsum[k];
                before += wsum[k];
            }
            if (at <= block && block < at + w) { found_s[0] = s; found_s[1] = w - 1 - (block - at); }
            __syncthreads();
        }
    }
    if (found_s[0] < 0) {
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
        if (warp == 2)
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_slot), "r"(512) : "memory");
        return;
    }
    const PromptSeq sq = prompt_seq(a, found_s[0], false);
    const int r0 = found_s[1] * C::ROWS;                    // first row of the block, in the sequence
    const int khead = head / a.group;
    // key tiles of each query tile, the first of them with keys that a row must
    // not see, and the first that is looked after
    int nt[2] = {0, 0}, first_mask[2] = {0, 0}, mask_from = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < NQ; i++) {
        const int ra = r0 + i * pa::BM, rb = min(ra + pa::BM, sq.n);
        if (ra < sq.n) {
            nt[i] = (max(0, min(sq.m, sq.m - sq.n + rb)) + pa::BN - 1) / pa::BN;
            first_mask[i] = max(0, min(sq.m, sq.m - sq.n + ra + 1)) / pa::BN;
            if (nt[i] > 0) mask_from = min(mask_from, first_mask[i]);
        }
    }
    const int ntmax = max(nt[0], nt[1]);

    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
    volatile int *ab = &abort_flag;
    uint8_t *qs = pa_dyn + ((1024 - (smem_u32(pa_dyn) & 1023)) & 1023), *ring = qs + NQ * C::QTILE;

    // The ring holds K 0, K 1, V 0, K 2, V 1, ..., the order in which they are
    // used.  is_v, tile of ring entry e (each PARTS stages).
    const int entries = 2 * ntmax;
    // The P of query tile i and key tile j: one place a query tile, or (NQ 1) two
    // that take turns; its barriers p_full and o_done and how often they were used.
    auto p_at = [](int i, int j) { return NQ == 2 ? i : (j & 1); };
    auto p_use = [](int j) { return NQ == 2 ? j : (j >> 1); };
    auto entry = [&](int e, bool &is_v, int &tile) {
        if (e == 0) { is_v = false; tile = 0; }
        else if (e == entries - 1) { is_v = true; tile = ntmax - 1; }
        else { is_v = !(e & 1); tile = is_v ? (e >> 1) - 1 : (e + 1) >> 1; }
    };
    if (warp == 0) {
        if (lane == 0 && ntmax > 0) {   // ---- copies
            int g = 0;
            bool ok = true;
            for (int e = 0; e < entries && ok; e++) {
                bool is_v;
                int tile;
                entry(e, is_v, tile);
                for (int part = 0; part < PARTS && ok; part++, g++) {
                    const int s = g % NST;
                    if (e == 0) {       // this part of Q, then of the first K: the first product can begin
                        mbar_arrive_expect_tx(&q_full[part], NQ * C::STAGE);
                        for (int i = 0; i < NQ; i++)
                            for (int p = part * (C::SPAN / 64); p < (part + 1) * (C::SPAN / 64); p++)
                                tma_load_3d(qs + i * C::QTILE + p * pa::PANEL, &qmap, p * 64, head,
                                            sq.q0 + r0 + i * pa::BM, &q_full[part]);
                    }
                    if (g >= NST && !(ok = mbar_wait(&empty[s], ((g / NST) - 1) & 1, ab, &g_pa_err, (int)ATTN_ERR_WAIT))) break;
                    mbar_arrive_expect_tx(&full[s], C::STAGE);
                    for (int p = 0; p < C::SPAN / 64; p++)
                        tma_load_3d(ring + s * C::STAGE + p * pa::PANEL, is_v ? &vmap : &kmap, part * C::SPAN + p * 64, khead,
                                    sq.k0 + tile * pa::BN, &full[s]);
                }
            }
        }
    } else if (warp == 1) {             // ---- S = Q . K^T (the whole warp, one elected lane issuing)
        const int n0 = __shfl_sync(0xffffffffu, nt[0], 0), n1 = __shfl_sync(0xffffffffu, nt[1], 0);
        bool ok = true;
        auto wait = [&](uint64_t *bar, int parity) {
            if (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity)))
                ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, ab, &g_pa_err, (int)ATTN_ERR_WAIT));
        };
        // The uses of S: key tile j of query tile 0, then of query tile 1, while they
        // have tiles left.  S is free again as soon as a softmax has it in registers,
        // so the softmax that ends finds its next S there.
        int use = 0;
        for (int j = 0; j < max(n0, n1) && ok; j++)
#pragma unroll
            for (int i = 0; i < NQ; i++) {
                if (!ok || j >= (i == 0 ? n0 : n1)) continue;
                const bool first = i == 0 || j >= n0, last = i == NQ - 1 || j >= n1;   // to use this K tile
                if (use > 0) wait(&s_free, (use - 1) & 1);
                tc_fence_after();
                use++;
#pragma unroll
                for (int part = 0; part < PARTS; part++) {
                    const int gg = (j == 0 ? 0 : 2 * j - 1) * PARTS + part;
                    if (use == 1) wait(&q_full[part], 0);
                    if (first) wait(&full[gg % NST], (gg / NST) & 1);
                    if (!ok) break;
                    const uint32_t kb = smem_u32(ring) + (gg % NST) * C::STAGE;
                    const uint32_t qb = smem_u32(qs) + i * C::QTILE + part * (C::SPAN / 64) * pa::PANEL;
#pragma unroll
                    for (int k = 0; k < C::SPAN / 16; k++) {
                        const uint32_t off = (k >> 2) * pa::PANEL + (k & 3) * 32;
                        tc_mma_warp(tmem, umma_desc_sw128(qb + off), umma_desc_sw128(kb + off), C::IDESC_S, (part | k) != 0);
                    }
                    if (last) tc_commit_warp(&empty[gg % NST]);
                }
                if (ok) tc_commit_warp(&s_full[i]);
            }
    } else if (warp == 3) {             // ---- O += P . V
        const int n0 = __shfl_sync(0xffffffffu, nt[0], 0), n1 = __shfl_sync(0xffffffffu, nt[1], 0);
        const int mf = __shfl_sync(0xffffffffu, mask_from, 0), n = max(n0, n1);
        bool ok = true;
        auto wait = [&](uint64_t *bar, int parity) {
            if (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity)))
                ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, ab, &g_pa_err, (int)ATTN_ERR_WAIT));
        };
        for (int j = 0; j < n && ok; j++)
#pragma unroll
            for (int i = 0; i < NQ; i++) {
                if (!ok || j >= (i == 0 ? n0 : n1)) continue;
                const bool first = i == 0 || j >= n0, last = i == NQ - 1 || j >= n1;   // to use this V tile
                wait(&p_full[p_at(i, j)], p_use(j) & 1);
                tc_fence_after();
#pragma unroll
                for (int part = 0; part < PARTS; part++) {
                    const int gg = (j == n - 1 ? 2 * n - 1 : 2 * j + 2) * PARTS + part;
                    if (first) wait(&full[gg % NST], (gg / NST) & 1);
                    if (first && j >= mf) wait(&checked[gg % NST], (gg / NST) & 1);
                    if (!ok) break;
                    const uint32_t vb = smem_u32(ring) + (gg % NST) * C::STAGE;
#pragma unroll
                    for (int k = 0; k < pa::BN / 16; k++)
                        tc_mma_ts_warp(tmem + C::O_COL + i * D + part * C::SPAN, tmem + C::P_COL + p_at(i, j) * 64 + k * 8,
                                       umma_desc_mn_sw128(vb + k * 2048, pa::PANEL), C::IDESC_O, k ? 1u : (uint32_t)(j > 0));
                    if (last) tc_commit_warp(&empty[gg % NST]);
                }
                if (ok) tc_commit_warp(&o_done[p_at(i, j)]);
            }
    } else if (warp == 2) {             // ---- V tiles with hidden keys
        int g = 0;
        bool ok = true;
        for (int e = 0; e < entries && ok; e++) {
            bool is_v;
            int tile;
            entry(e, is_v, tile);
            for (int part = 0; part < PARTS; part++, g++) {
                const int s = g % NST;
                const bool got = mbar_wait(&full[s], (g / NST) & 1, ab, &g_pa_err, (int)ATTN_ERR_WAIT);
                ok = __all_sync(0xffffffffu, got);
                if (!ok) break;
                if (is_v && tile >= mask_from) {
                    uint8_t *st = ring + s * C::STAGE;
                    const int behind = sq.m - tile * pa::BN;        // rows from here on belong to no key
                    // eight 16-byte pieces at a time: an exponent of all ones carries
                    // into the sign bit
                    for (int i = lane * 16; i < C::STAGE; i += 8 * 32 * 16) {
                        uint4 w[8];
#pragma unroll
                        for (int k = 0; k < 8; k++) w[k] = lds128(st + i + k * 512);
                        if (behind < pa::BN) {
#pragma unroll
                            for (int k = 0; k < 8; k++)
                                if ((((i + k * 512) / 128) & 127) >= behind) {
                                    w[k] = make_uint4(0, 0, 0, 0);
                                    *(uint4 *)(st + i + k * 512) = w[k];
                                }
                        }
                        uint32_t bad = 0;
#pragma unroll
                        for (int k = 0; k < 8; k++)
                            bad |= ((w[k].x & 0x7f807f80u) + 0x00800080u) | ((w[k].y & 0x7f807f80u) + 0x00800080u) |
                                   ((w[k].z & 0x7f807f80u) + 0x00800080u) | ((w[k].w & 0x7f807f80u) + 0x00800080u);
                        if (!(bad & 0x80008000u)) continue;
#pragma unroll 1
                        for (int k = 0; k < 8; k++) {
                            const int at = i + k * 512, r = (at / 128) & 127;
                            // the piece's place in its row is swizzled by the row
                            const int d0 = part * C::SPAN + (at / pa::PANEL) * 64 + (((at >> 4) & 7) ^ (r & 7)) * 8;
                            uint16_t *h = (uint16_t *)(st + at);
                            for (int u = 0; u < 8; u++) {
                                const uint16_t x = h[u];
                                if ((x & 0x7f80) != 0x7f80) continue;
                                h[u] = 0;
                                const int sh = ((x & 0x7f) ? 0 : (x >> 15) ? 2 : 1) * 10;
                                const uint32_t key = (uint32_t)((tile - mask_from) * pa::BN + r);
                                uint32_t old = first_bad[d0 + u], was;
                                while (key < ((old >> sh) & 1023u)) {
                                    was = old;
                                    old = atomicCAS(&first_bad[d0 + u], was, (was & ~(1023u << sh)) | (key << sh));
                                    if (old == was) break;
                                }
                                poison = 1;
                            }
                        }
                    }
                    static_assert(C::STAGE % (8 * 32 * 16) == 0, "whole batches of pieces");
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&checked[s]);
                    mbar_arrive(&empty[s]);
                }
            }
        }
    } else {                            // ---- softmax, one row a thread
        const int i = (warp - 4) >> 2;                      // query tile
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const int rt = (warp & 3) * 32 + lane, row = r0 + i * pa::BM + rt;      // row in the sequence
        const int nti = nt[i];
        const int seen = max(0, min(sq.m, sq.m - sq.n + min(row, sq.n - 1) + 1));   // keys that it sees
        const uint32_t o_col = tmem + lanes + C::O_COL + i * D;
        float m = -INFINITY, l = 0.f;
        const float raise = pa::RAISE / a.zscale;
        bool ok = true;
        auto wait = [&](uint64_t *bar, int parity) {
            if (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity)))
                ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, ab, &g_pa_err, (int)ATTN_ERR_WAIT));
            tc_fence_after();
        };
        for (int j = 0; j < nti; j++) {
            wait(&s_full[i], j & 1);
            if (!ok) break;
            float v[128];
            tc_ld128(tmem + lanes, v);
            tc_fence_before();
            mbar_arrive(&s_free);
            if (j >= first_mask[i]) {
                const int lim = seen - j * pa::BN;
#pragma unroll
                for (int c = 0; c < 128; c++) v[c] = c < lim ? v[c] : -INFINITY;
            }
            float mx[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
            for (int c = 4; c < 128; c += 4)
#pragma unroll
                for (int u = 0; u < 4; u++) mx[u] = fmaxf(mx[u], v[c + u]);
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            const bool up = top > m + raise;
            if (__any_sync(0xffffffffu, up)) {
                const float down = !up ? 1.0f : m == -INFINITY ? 0.f : pa_ex2((m - top) * a.zscale);
                if (up) m = top;
                l *= down;
                if (j > 0) {                 // O is the product's of j - 1 until that is done
                    wait(&o_done[p_at(i, j - 1)], p_use(j - 1) & 1);
                    if (!ok) break;
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        uint32_t o[32];
                        tc_ld32(o_col + c, o);
#pragma unroll
                        for (int u = 0; u < 32; u++) o[u] = __float_as_uint(__uint_as_float(o[u]) * down);
                        tc_st32(o_col + c, o);
                    }
                }
            }
            const float mz = m == -INFINITY ? 0.f : m * a.zscale;
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
            uint32_t pk[2][32];
#pragma unroll
            for (int c = 0; c < 128; c += 2) {
                const float p0 = pa_ex2(fmaf(v[c], a.zscale, -mz)), p1 = pa_ex2(fmaf(v[c + 1], a.zscale, -mz));
                sum[c & 2] += p0;
                sum[(c & 2) + 1] += p1;
                pk[c / 64][(c % 64) / 2] = pa_pack(p0, p1);
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            // P's place is read by the product of j - 1 (NQ 1: j - 2) until that is done
            if (j >= (NQ == 2 ? 1 : 2)) {
                wait(&o_done[p_at(i, j)], (p_use(j) - 1) & 1);
                if (!ok) break;
            }
            const uint32_t p_col = tmem + lanes + C::P_COL + p_at(i, j) * 64;
            tc_st32(p_col, pk[0]);
            tc_st32(p_col + 32, pk[1]);
            tc_wait_st();
            tc_fence_before();
            mbar_arrive(&p_full[p_at(i, j)]);
        }
        if (NQ == 1 && ok && nti > 1) wait(&o_done[p_at(i, nti - 2)], p_use(nti - 2) & 1);
        if (ok && nti > 0) wait(&o_done[p_at(i, nti - 1)], p_use(nti - 1) & 1);
        // a query tile that sees no key: its rows of Q may still be on their way
        if (nti == 0 && ntmax > 0)
            for (int p = 0; p < PARTS; p++) wait(&q_full[p], 0);
        if (ok) {
            const float inv = l == 0.f ? 0.f : 1.0f / l;
            // through this warp's rows of the Q tile, which nothing reads any more, so
            // that rows are stored whole: 16-byte pieces, swizzled by the row
            uint8_t *own = qs + i * C::QTILE + (warp & 3) * 32 * (D * 2);
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                uint32_t o[32];
                if (nti > 0) tc_ld32(o_col + c, o);
                if (*(volatile int *)&poison) {
#pragma unroll
                    for (int u = 0; u < 32; u++) {
                        float x = __uint_as_float(o[u]);
                        const uint32_t f = first_bad[c + u];
                        const int rel = seen - mask_from * pa::BN;       // looked-after keys that the row sees
                        if (rel > (int)(f & 1023u)) x = __int_as_float(0x7fc00000);
                        if (rel > (int)((f >> 10) & 1023u)) x += INFINITY;
                        if (rel > (int)(f >> 20)) x -= INFINITY;
                        o[u] = __float_as_uint(x);
                    }
                }
#pragma unroll
                for (int h = 0; h < 4; h++) {
                    uint32_t w[4];
#pragma unroll
                    for (int u = 0; u < 4; u++)
                        w[u] = nti > 0 ? pa_pack(__uint_as_float(o[8 * h + 2 * u]) * inv,
                                                 __uint_as_float(o[8 * h + 2 * u + 1]) * inv) : 0u;
                    *(uint4 *)(own + lane * (D * 2) + (((c / 8 + h) ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            __syncwarp();
            constexpr int PIECES = D / 8, RPS = 32 / PIECES > 0 ? 32 / PIECES : 1;     // pieces of a row, rows of a store
            const int left = sq.n - (row - lane);                                      // rows of this warp that exist
#pragma unroll 4
            for (int r = 0; r < 32; r += RPS) {
                const int rr = r + (RPS > 1 ? lane / PIECES : 0), p = RPS > 1 ? lane % PIECES : lane;
                if (rr < left)
                    *(uint4 *)(a.out.p + (long)(sq.q0 + row - lane + rr) * a.out.rs + (long)head * a.out.hs + p * 8) =
                        lds128(own + rr * (D * 2) + ((p ^ (rr & 7)) << 4));
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 2)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

}  // namespace apus
using namespace apus;

// 3-D BF16 tensor map of rows of heads (dims, heads, rows): boxes of 64 dims of
// one head of 128 rows in the 128-byte swizzle; zeros past the last row.
static int pa_map(CUtensorMap *m, const ApusHeadRows *r, size_t dim) {
    static PFN_cuTensorMapEncodeTiled_v12000 enc = nullptr;
    if (!enc) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess) {
            gcuda_set_error("prompt_attn: no tensor map encoder");
            return -1;
        }
        enc = (PFN_cuTensorMapEncodeTiled_v12000)p;
    }
    // the stride of an axis of one is not looked at, but has to be a valid one
    const cuuint64_t dims[3] = {dim, r->heads, r->rows};
    const cuuint64_t strides[2] = {r->heads > 1 ? r->head_stride * 2 : dim * 2, r->rows > 1 ? r->row_stride * 2 : dim * 2};
    const cuuint32_t box[3] = {64, 1, 128}, es[3] = {1, 1, 1};
    if (enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, r->p, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
        gcuda_set_error("prompt_attn: tensor map of %zu rows of %zu heads, strides %zu, %zu", r->rows, r->heads,
                        r->row_stride, r->head_stride);
        return -1;
    }
    return 0;
}

template <int D>
static int pa_launch(const PromptArgs &a, const ApusHeadRows *q, const ApusHeadRows *k, const ApusHeadRows *v,
                     cudaStream_t st) {
    using C = pa::Cfg<D>;
    const long blocks = ((long)a.rows_q / C::ROWS + a.nseq) * a.heads;
    if (blocks >= (1l << 31)) { gcuda_set_error("prompt_attn: %d rows of %d heads", a.rows_q, a.heads); return -1; }
    CUtensorMap qm, km, vm;
    if (pa_map(&qm, q, D) || pa_map(&km, k, D) || pa_map(&vm, v, D)) return -1;
    if (gcuda_smem_limit_once((const void *)k_prompt_tc<D>, C::SMEM)) return -1;
    k_prompt_tc<D><<<(unsigned)blocks, C::THREADS, C::SMEM, st>>>(qm, km, vm, a);
    return gcuda_check(cudaGetLastError(), "prompt_attn launch");
}

extern "C" int apus_gcuda_prompt_attn_dev(const ApusPromptBatch *batch, const ApusHeadRows *q, const ApusHeadRows *k,
                                          const ApusHeadRows *v, const ApusHeadRows *out, size_t dim, float scale,
                                          void *stream) {
    const char *what = "prompt_attn";
    if (!batch) { gcuda_set_error("%s: no batch given", what); return -1; }
    if (attn_check_dim(what, dim) || attn_check_scale(what, scale)) return -1;
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
    // without keys every row gives zeros; the tensor maps need a row to stand on
    ApusHeadRows kk = *k, vv = *v;
    if (!k->rows) { kk = vv = *q; kk.heads = vv.heads = 1; }
    if (dim == 64) return pa_launch<64>(a, q, &kk, &vv, (cudaStream_t)stream);
    if (dim == 128) return pa_launch<128>(a, q, &kk, &vv, (cudaStream_t)stream);
    return pa_launch<256>(a, q, &kk, &vv, (cudaStream_t)stream);
}

int prompt_attn_error_read_and_clear(void) {
    int v = 0, z = 0;
    cudaMemcpyFromSymbol(&v, g_pa_err, sizeof v);
    if (v) cudaMemcpyToSymbol(g_pa_err, &z, sizeof z);
    return v;
}
