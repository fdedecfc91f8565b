// prompt_attn.cu — causal attention over packed sequences with grouped heads
// (apus_gcuda_prompt_attn_dev):
//   out_i = sum_{j <= m - n + i} p_ij v_j,  p_i = softmax_j(scale q_i . k_j)
// for row i of n queries over m keys of one sequence, in one pass over the keys
// with a running maximum and sum.
//
// Both products run on tcgen05: an item is NQ tiles of 128 query rows of one
// head, and a CTA walks the keys in tiles of 128,
//   S (TMEM, fp32) = Q (shared) . K^T (shared),   O (TMEM, fp32) += P (TMEM) . V (shared),
// with P = 2^(scale log2(e) (S - maximum)) in BF16.  K and V come as tensor copies
// (128-byte swizzle) into a ring; V is read as it lies, rows of keys with the dims
// contiguous.
//
// Bound: at dim 256 the products (2048 tensor cycles a tile of 128 x 128), at
// dim 128 products and exponentials alike (1024 tensor cycles; 16384
// exponentials at 16 a cycle), at dim 64 the exponentials.
// Up to dim 128 an item has two query tiles, so that each K and V tile serves 256
// rows and one tile's softmax runs under the other's products.  S has one place
// in TMEM, which the softmax frees as soon as it holds the scores in registers; P
// has a place of its own.  So the next S is there when a softmax ends, and the two
// softmaxes take turns at the exponentials (at dim 64, with an S place each, they
// ran in step and took 10% longer).  (With P written over S, a query tile waited
// 1400 of 3700 cycles for its own products; two S tiles of 64 keys made the
// products of S, which read 128 rows of Q for 64 keys, the bound.)
//
// Roles: warp 0 copies, warp 1 issues the products of S, warp 3 those of O (one
// warp for both spent 3400 cycles on issuing 2048 cycles of products), warp 2
// looks after V tiles with keys that some row must not see, warps 4.. are one
// softmax group of 128 threads (a row each) a query tile.  The maximum is raised,
// and O rescaled, only when a score passes it by more than 2^8, so almost never.
// Warps 0, 1 and 3 issue as whole warps with one elected lane: in a branch that
// one lane takes, moving the operands to uniform registers cost more than the
// issue (1210 against 995 TFLOP/s at dim 256 for the copies alone).
//
// Items: a CTA that is done asks for the item of one that has not begun
// (clusterlaunchcontrol), so the next item's copies and first products run under
// the last one's end.  One CTA an item spent 12.7 thousand cycles on set-up, first
// copies and the end, where 2048 rows of 64 heads of 256 take 37 thousand: 172 -> 162
// us; seven ragged prompts, 4099 rows of 32 heads over 8 of 128: 81 -> 75 us.  Heads
// that do not fit L2 together follow one another (L2_SHARE): 162 -> 144 us.
//
// Measured (captured graphs of a few milliseconds, at 1965 MHz): dim 128, 8192 rows
// after 4096 keys, 32 heads over 8: 0.79 ms, 1390 TFLOP/s; dim 256, 8192 rows of 16
// heads: 1290 TFLOP/s, 2400 cycles a tile of 2048 (a ring of five half tiles in place of
// four, the same; quarters, V by keys, 730; two softmax groups that take turns, 1160);
// 2048 rows of 64 heads: 139 us, tensor pipe 54% active; dim 64, 8192 rows of 32 heads
// over 8: 346 us, 794 TFLOP/s.  Over a tenth of a second and more the power limit holds
// the clock near 1530 MHz: 0.92 ms, and 162 us for the 2048 rows.
//
// A hidden key's weight is 0, but 0 times a NaN or an infinity in its value would
// reach the row through the product.  So in tiles with hidden keys such values
// (and all rows behind the sequence) are set to 0 in shared memory before the
// product reads them; the first key with a NaN, a +inf and a -inf is kept for each
// dim, and the rows that see it get it added at the end.
#include <atomic>

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
    if ((q.bad || k.bad) && report) atomicCAS(&g_pa_err, 0, (int)ATTN_ERR_SEQ);
    return PromptSeq{q.row0, q.n, k.row0, k.n};
}

namespace pa {
constexpr int BM = 128, BN = 128;               // query rows of a tile, keys of a K or V tile
constexpr int PANEL = 128 * 128;                // bytes of 128 rows of 64 dims
template <int D> struct Cfg {
    static constexpr int NQ = D == 256 ? 1 : 2;             // query tiles of an item
    static constexpr int THREADS = 128 + 128 * NQ;
    static constexpr int SPAN = D == 256 ? 128 : D;         // dims of a ring stage
    static constexpr int PARTS = D / SPAN;                  // stages of a K or V tile
    static constexpr int QTILE = D / 64 * PANEL, STAGE = SPAN / 64 * PANEL;
    static constexpr int NST = D == 64 ? 8 : 4;
    static constexpr int OUT = 32 * 128;                    // a softmax warp's rows on their way out, 64 dims of each
    static constexpr int SMEM = NQ * QTILE + NST * STAGE + 4 * NQ * OUT + 1024;
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
// Bytes of keys and values that items next to one another read: all items that
// run at once read them at their own places, so what does not stay in L2 (126 MB)
// comes from HBM for each block of rows.  64 heads of 256, 2048 rows: 144 us (all
// heads together, 134 MB: 165; 64 MB 149, 32 MB 144), 4096 rows of the same heads: 490
// (573), each when this was chosen; 139 and 475 since.
constexpr int L2_SHARE = 48 << 20;
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

// acc + 0 x for two BF16.
APUS_DEV uint32_t pa_times_0(uint32_t x, uint32_t acc) {
    uint32_t d;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(x), "r"(0u), "r"(acc));
    return d;
}

// A bounded wait.
APUS_DEV bool pa_wait(uint64_t *bar, uint32_t parity, volatile int *ab) {
    return mbar_wait(bar, parity, ab, &g_pa_err, (int)ATTN_ERR_WAIT);
}

// An item: ROWS query rows from r0 on of a sequence, for one head.  n < 0: no more.
struct PaItem { int q0, n, k0, m, r0, head, first; };     // first: of the whole call

// Key tiles of each query tile, the first of them with keys that some row must
// not see, and the first that is looked after.
template <int NQ> struct PaTiles { int nt[NQ], first_mask[NQ], mask_from, ntmax; };
template <int NQ> APUS_DEV PaTiles<NQ> pa_tiles(const PaItem &it) {
    PaTiles<NQ> t;
    t.mask_from = 0x7fffffff;
    t.ntmax = 0;
#pragma unroll
    for (int i = 0; i < NQ; i++) {
        const int ra = it.r0 + i * pa::BM, rb = min(ra + pa::BM, it.n);
        t.nt[i] = t.first_mask[i] = 0;
        if (ra < it.n) {
            t.nt[i] = (max(0, min(it.m, it.m - it.n + rb)) + pa::BN - 1) / pa::BN;
            t.first_mask[i] = max(0, min(it.m, it.m - it.n + ra + 1)) / pa::BN;
            if (t.nt[i] > 0) t.mask_from = min(t.mask_from, t.first_mask[i]);
        }
        t.ntmax = max(t.ntmax, t.nt[i]);
    }
    return t;
}

template <int D>
__global__ void __launch_bounds__(pa::Cfg<D>::THREADS, 1)
k_prompt_tc(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
            const __grid_constant__ CUtensorMap vmap, const PromptArgs a) {
    using C = pa::Cfg<D>;
    constexpr int NQ = C::NQ, NST = C::NST, PARTS = C::PARTS;
    extern __shared__ __align__(1024) uint8_t pa_dyn[];
    __shared__ __align__(16) uint4 clc_answer;
    __shared__ __align__(8) uint64_t q_full[PARTS], q_empty, full[NST], empty[NST], checked[NST], s_free, s_full[2],
        p_full[2], o_done[2], item_full[2], item_empty[2], clc_full;
    __shared__ PaItem items[2];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag, poison[2];
    // first key (from the first looked after, 1023: none) with a NaN, +inf, -inf in
    // a dim, ten bits each; at most four tiles are looked after.  Items take turns.
    __shared__ uint32_t first_bad[2][D];
    // (a shuffle tells the compiler that it is the same for the warp, so that the
    // products' operands stay in uniform registers)
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;

    if (tid == 0) {
        for (int p = 0; p < PARTS; p++) mbar_init(&q_full[p], 1);
        mbar_init(&q_empty, 1);
        for (int s = 0; s < NST; s++) { mbar_init(&full[s], 1); mbar_init(&empty[s], 2); mbar_init(&checked[s], 1); }   // empty: products, scan
        mbar_init(&s_free, 128);
        for (int i = 0; i < 2; i++) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 128);
            mbar_init(&o_done[i], 1);
            mbar_init(&item_full[i], 1);
            mbar_init(&item_empty[i], C::THREADS / 32 - 1);
        }
        mbar_init(&clc_full, 1);
        abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // warp 0: the blocks of rows of 128 sequences from c0 on, four a lane; `before`:
    // blocks before them
    int c0 = 0, before = 0, cw = 0, cincl = 0;
    auto blocks_of = [&](int s) { return s < a.nseq ? (prompt_seq(a, s, true).n + C::ROWS - 1) / C::ROWS : 0; };
    auto chunk = [&]() {
        cw = 0;
#pragma unroll
        for (int u = 0; u < 4; u++) cw += blocks_of(c0 + 4 * lane + u);
        cincl = cw;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, cincl, off);
            if (lane >= off) cincl += o;
        }
    };
    if (warp == 0) chunk();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
    volatile int *ab = &abort_flag;
    uint8_t *qs = pa_dyn + ((1024 - (smem_u32(pa_dyn) & 1023)) & 1023), *ring = qs + NQ * C::QTILE;

    // The next item (whole warp; not warp 0): false behind the last.  A softmax warp
    // gives its place back (done_with) when it is through with it, so whoever has
    // item k + 2 knows that the rows of item k are written.
    auto done_with = [&](int k) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_empty[k & 1]);
    };
    auto next_item = [&](int k, PaItem &it) -> bool {
        const bool got = mbar_try_wait(&item_full[k & 1], (k >> 1) & 1) ||
                         pa_wait(&item_full[k & 1], (k >> 1) & 1, ab);
        if (!__all_sync(0xffffffffu, got)) return false;
        it = items[k & 1];
        if (warp < 4) done_with(k);
        return __all_sync(0xffffffffu, it.n >= 0);      // (a vote: the same for the warp, as above)
    };
    // The ring holds an item's K 0, K 1, V 0, K 2, V 1, ..., the order in which
    // they are used, each PARTS stages; is_v, tile of its entry e.
    auto entry = [](int e, int ntmax, bool &is_v, int &tile) {
        if (e == 0) { is_v = false; tile = 0; }
        else if (e == 2 * ntmax - 1) { is_v = true; tile = ntmax - 1; }
        else { is_v = !(e & 1); tile = is_v ? (e >> 1) - 1 : (e + 1) >> 1; }
    };
    // The P of query tile i and the CTA's use u of it: one place a query tile, or
    // (NQ 1) two that take turns; how often that place was used before.
    auto p_at = [](int i, unsigned u) { return NQ == 2 ? i : (int)(u & 1); };
    auto p_use = [](unsigned u) { return NQ == 2 ? u : u >> 1; };

    if (warp < 4) {
    // Three warpgroups share 384 x 168 registers: the softmax keeps 128 scores a
    // thread, so the first gives 80 of its up (88 x 128 + 208 x 256 = 168 x 384).
    if constexpr (NQ == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 0) {                    // ---- items and copies
        // Items in the order of the sequences; in a sequence equal parts of the heads
        // whose keys and values take up to L2_SHARE bytes, of a part the last block of
        // ROWS rows (the one with the most keys) first, and the heads of a block one
        // after the other.
        unsigned idx = blockIdx.x, g = 0, asked = 0;
        int k = 0, loaded = 0;
        bool ok = true;
        auto ask = [&]() {              // for the next item: that of a CTA not yet begun, which then never begins
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_arrive_expect_tx(&clc_full, 16);
            asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
                         ::"r"(smem_u32(&clc_answer)), "r"(smem_u32(&clc_full)) : "memory");
        };
        auto wait = [&](uint64_t *bar, unsigned parity) {
            if (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) ok = __all_sync(0xffffffffu, pa_wait(bar, parity, ab));
        };
        auto publish = [&](const PaItem &it) {
            if (k >= 2) ok = __all_sync(0xffffffffu, pa_wait(&item_empty[k & 1], ((k >> 1) - 1) & 1, ab));
            if (ok && lane == 0) {
                items[k & 1] = it;
                mbar_arrive(&item_full[k & 1]);
            }
            k++;
        };
        while (true) {
            const int block = (int)(idx / (unsigned)a.heads);
            if (block < before) { c0 = before = 0; chunk(); }
            int sum = __shfl_sync(0xffffffffu, cincl, 31);
            while (block >= before + sum && c0 + 128 < a.nseq) {
                before += sum;
                c0 += 128;
                chunk();
                sum = __shfl_sync(0xffffffffu, cincl, 31);
            }
            bool pending = false;
            if (block < before + sum) {
                const int rel = block - before;
                const int src = __ffs(__ballot_sync(0xffffffffu, cincl - cw <= rel && rel < cincl)) - 1;
                // the sequence among the lane's four, its first block and their number
                int s = c0 + 4 * lane, left = rel - (cincl - cw), w = 0;
                PromptSeq sq{0, 0, 0, 0};
                if (lane == src)
#pragma unroll 1
                    for (int u = 0; u < 4; u++, s++) {
                        sq = prompt_seq(a, s, false);
                        w = (sq.n + C::ROWS - 1) / C::ROWS;
                        if (left < w) break;
                        left -= w;
                    }
                PaItem it;
                it.q0 = __shfl_sync(0xffffffffu, sq.q0, src);
                it.n = __shfl_sync(0xffffffffu, sq.n, src);
                it.k0 = __shfl_sync(0xffffffffu, sq.k0, src);
                it.m = __shfl_sync(0xffffffffu, sq.m, src);
                w = __shfl_sync(0xffffffffu, w, src);
                left = __shfl_sync(0xffffffffu, left, src);
                // place in the sequence's items -> heads together, block, head
                const unsigned local = idx - (unsigned)(block - left) * (unsigned)a.heads;
                const unsigned kheads = (unsigned)(a.heads / a.group);
                const unsigned fit = max(1u, (unsigned)(pa::L2_SHARE / (4 * D)) / (unsigned)max(it.m, 1));
                const unsigned parts = (kheads + fit - 1) / fit, share = (kheads + parts - 1) / parts * (unsigned)a.group;
                const unsigned h0 = local / (share * (unsigned)w) * share, in = local - h0 * (unsigned)w;
                const unsigned hn = min(share, (unsigned)a.heads - h0), nth = in / hn;
                const int head = (int)(h0 + (in - nth * hn));
                it.r0 = (w - 1 - (int)nth) * C::ROWS;
                it.head = head;
                it.first = idx == 0;
                publish(it);
                const int ntmax = __shfl_sync(0xffffffffu, pa_tiles<NQ>(it).ntmax, 0), khead = head / a.group, entries = 2 * ntmax;
                const int k_row = it.k0, q_row = it.q0 + it.r0;
                auto load_q = [&](int part) {
                    mbar_arrive_expect_tx_warp(&q_full[part], NQ * C::STAGE);
                    for (int i = 0; i < NQ; i++)
                        for (int p = part * (C::SPAN / 64); p < (part + 1) * (C::SPAN / 64); p++)
                            tma_load_3d_warp(qs + i * C::QTILE + p * pa::PANEL, &qmap, p * 64, head, q_row + i * pa::BM, &q_full[part]);
                };
                for (int e = 0; e < entries && ok; e++) {
                    bool is_v;
                    int tile;
                    entry(e, ntmax, is_v, tile);
#pragma unroll
                    for (int part = 0; part < PARTS; part++, g++) {
                        const unsigned s = g % NST;
                        if (g >= NST) wait(&empty[s], (g / NST - 1) & 1);
                        if (!ok) break;
                        mbar_arrive_expect_tx_warp(&full[s], C::STAGE);
                        uint8_t *st = ring + s * C::STAGE;
#pragma unroll
                        for (int p = 0; p < C::SPAN / 64; p++)
                            tma_load_3d_warp(st + p * pa::PANEL, is_v ? &vmap : &kmap, part * C::SPAN + p * 64, khead,
                                             k_row + tile * pa::BN, &full[s]);
                        // part by part, so that the first product can begin; later, Q is
                        // the last item's until that has no more products of S
                        if (e == 0 && loaded == 0) load_q(part);
                    }
                    if (e == 0 && loaded > 0 && ok) {
                        wait(&q_empty, (loaded - 1) & 1);
                        if (!ok) break;
                        for (int part = 0; part < PARTS; part++) load_q(part);
                    }
                    // early enough that the answer is there when the copies end
                    if (ok && e == max(0, entries - 4)) { if (lane == 0) ask(); pending = true; }
                }
                if (ntmax > 0) loaded++;
            }
            if (!ok && !pending) break;
            int more = 0;
            unsigned nx = 0;
            if (lane == 0) {
                if (!pending) ask();
                // an answer in flight is waited for whatever happens, but not for ever
                const long long t0 = clock64();
                while (!mbar_try_wait(&clc_full, asked & 1))
                    if (clock64() - t0 > (1ll << 31)) {
                        abort_flag = 1;
                        atomicExch(&g_pa_err, (int)ATTN_ERR_WAIT);
                        ok = false;
                        break;
                    }
                if (ok)
                    asm volatile(
                        "{\n .reg .b128 r;\n .reg .pred p;\n ld.shared.b128 r, [%2];\n"
                        " clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n selp.b32 %0, 1, 0, p;\n"
                        " @p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n}"
                        : "=r"(more), "+r"(nx) : "r"(smem_u32(&clc_answer)) : "memory");
            }
            asked++;
            ok = __shfl_sync(0xffffffffu, (int)ok, 0);
            more = __shfl_sync(0xffffffffu, more, 0);
            idx = __shfl_sync(0xffffffffu, nx, 0);
            if (!ok || !more) break;
        }
        if (ok) publish(PaItem{0, -1, 0, 0, 0, 0, 0});
    } else if (warp == 1) {             // ---- S = Q . K^T (the whole warp, one elected lane issuing)
        bool ok = true;
        auto wait = [&](uint64_t *bar, unsigned parity) {
            if (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity)))
                ok = __all_sync(0xffffffffu, pa_wait(bar, parity, ab));
        };
        PaItem it;
        unsigned use = 0, g0 = 0, loaded = 0;
        for (int k = 0; ok && next_item(k, it); k++) {
            const PaTiles<NQ> t = pa_tiles<NQ>(it);
            const int n0 = __shfl_sync(0xffffffffu, t.nt[0], 0), n1 = __shfl_sync(0xffffffffu, NQ == 2 ? t.nt[NQ - 1] : 0, 0);
            const int n = max(n0, n1);
            g0 = __shfl_sync(0xffffffffu, g0, 0);
            use = __shfl_sync(0xffffffffu, use, 0);
            loaded = __shfl_sync(0xffffffffu, loaded, 0);
            // The uses of S: key tile j of query tile 0, then of query tile 1, while they
            // have tiles left.  S is free again as soon as a softmax has it in registers,
            // so the softmax that ends finds its next S there.
            for (int j = 0; j < n && ok; j++)
#pragma unroll
                for (int i = 0; i < NQ; i++) {
                    if (!ok || j >= (i == 0 ? n0 : n1)) continue;
                    const bool first = i == 0 || j >= n0, last = i == NQ - 1 || j >= n1;   // to use this K tile
                    if (use > 0) wait(&s_free, (use - 1) & 1);
                    tc_fence_after();
                    use++;
#pragma unroll
                    for (int part = 0; part < PARTS; part++) {
                        const unsigned gg = g0 + (unsigned)((j == 0 ? 0 : 2 * j - 1) * PARTS + part);
                        if (j == 0 && first) wait(&q_full[part], loaded & 1);
                        if (first) wait(&full[gg % NST], (gg / NST) & 1);
                        if (!ok) break;
                        const uint32_t kb = smem_u32(ring) + (gg % NST) * C::STAGE;
                        const uint32_t qb = smem_u32(qs) + i * C::QTILE + part * (C::SPAN / 64) * pa::PANEL;
#pragma unroll
                        for (int kk = 0; kk < C::SPAN / 16; kk++) {
                            const uint32_t off = (kk >> 2) * pa::PANEL + (kk & 3) * 32;
                            tc_mma_warp(tmem, umma_desc_sw128(qb + off), umma_desc_sw128(kb + off), C::IDESC_S, (part | kk) != 0);
                        }
                        if (last) tc_commit_warp(&empty[gg % NST]);
                    }
                    if (ok) tc_commit_warp(&s_full[i]);
                }
            if (ok && n > 0) {
                tc_commit_warp(&q_empty);
                loaded++;
            }
            g0 += (unsigned)(2 * n * PARTS);
        }
    } else if (warp == 3) {             // ---- O += P . V
        bool ok = true;
        auto wait = [&](uint64_t *bar, unsigned parity) {
            if (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity)))
                ok = __all_sync(0xffffffffu, pa_wait(bar, parity, ab));
        };
        PaItem it;
        unsigned g0 = 0, used[2] = {0, 0};
        for (int k = 0; ok && next_item(k, it); k++) {
            const PaTiles<NQ> t = pa_tiles<NQ>(it);
            const int n0 = __shfl_sync(0xffffffffu, t.nt[0], 0), n1 = __shfl_sync(0xffffffffu, NQ == 2 ? t.nt[NQ - 1] : 0, 0);
            const int mf = __shfl_sync(0xffffffffu, t.mask_from, 0), n = max(n0, n1);
            g0 = __shfl_sync(0xffffffffu, g0, 0);
            used[0] = __shfl_sync(0xffffffffu, used[0], 0); used[1] = __shfl_sync(0xffffffffu, used[1], 0);
            for (int j = 0; j < n && ok; j++)
#pragma unroll
                for (int i = 0; i < NQ; i++) {
                    if (!ok || j >= (i == 0 ? n0 : n1)) continue;
                    const bool first = i == 0 || j >= n0, last = i == NQ - 1 || j >= n1;   // to use this V tile
                    const unsigned u = used[i]++;
                    wait(&p_full[p_at(i, u)], p_use(u) & 1);
                    tc_fence_after();
#pragma unroll
                    for (int part = 0; part < PARTS; part++) {
                        const unsigned gg = g0 + (unsigned)((j == n - 1 ? 2 * n - 1 : 2 * j + 2) * PARTS + part);
                        if (first) wait(&full[gg % NST], (gg / NST) & 1);
                        if (first && j >= mf) wait(&checked[gg % NST], (gg / NST) & 1);
                        if (!ok) break;
                        const uint32_t vb = smem_u32(ring) + (gg % NST) * C::STAGE;
#pragma unroll
                        for (int kk = 0; kk < pa::BN / 16; kk++)
                            tc_mma_ts_warp(tmem + C::O_COL + i * D + part * C::SPAN, tmem + C::P_COL + p_at(i, u) * 64 + kk * 8,
                                           umma_desc_mn_sw128(vb + kk * 2048, pa::PANEL), C::IDESC_O,
                                           kk ? 1u : (uint32_t)(j > 0));
                        if (last) tc_commit_warp(&empty[gg % NST]);
                    }
                    if (ok) tc_commit_warp(&o_done[p_at(i, u)]);
                }
            g0 += (unsigned)(2 * n * PARTS);
        }
    } else {                            // ---- V tiles with hidden keys
        unsigned g = 0;
        bool ok = true;
        auto wait = [&](uint64_t *bar, unsigned parity) {
            if (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) ok = __all_sync(0xffffffffu, pa_wait(bar, parity, ab));
        };
        PaItem it;
        for (int k = 0; ok && next_item(k, it); k++) {
            const PaTiles<NQ> t = pa_tiles<NQ>(it);
            // sequences out of bounds behind the last one with rows are reported too
            if (it.first)
#pragma unroll 4
                for (int s = 128 + lane; s < a.nseq; s += 32) prompt_seq(a, s, true);
            uint32_t *const bad_key = first_bad[k & 1];
            for (int i = lane; i < D; i += 32) bad_key[i] = 0x3fffffffu;
            if (lane == 0) poison[k & 1] = 0;
            __syncwarp();
            const int ntmax = __shfl_sync(0xffffffffu, t.ntmax, 0), entries = 2 * ntmax;
            const int mask_from = __shfl_sync(0xffffffffu, t.mask_from, 0);
            g = __shfl_sync(0xffffffffu, g, 0);
            for (int e = 0; e < entries && ok; e++) {
                bool is_v;
                int tile;
                entry(e, ntmax, is_v, tile);
                for (int part = 0; part < PARTS; part++, g++) {
                    const unsigned s = g % NST;
                    wait(&full[s], (g / NST) & 1);
                    if (!ok) break;
                    if (is_v && tile >= mask_from) {
                        uint8_t *st = ring + s * C::STAGE;
                        const int key0 = tile * pa::BN;
                        const int behind = it.m - key0;                 // rows from here on belong to no key
                        // eight 16-byte pieces at a time: 0 times a NaN or an infinity is NaN
                        // and stays in the sum, 0 times anything else adds nothing
                        for (int i = lane * 16; i < C::STAGE; i += 8 * 32 * 16) {
                            uint4 w[8];
#pragma unroll
                            for (int u = 0; u < 8; u++) w[u] = lds128(st + i + u * 512);
                            if (behind < pa::BN) {
#pragma unroll
                                for (int u = 0; u < 8; u++)
                                    if ((((i + u * 512) / 128) & 127) >= behind) {
                                        w[u] = make_uint4(0, 0, 0, 0);
                                        *(uint4 *)(st + i + u * 512) = w[u];
                                    }
                            }
                            uint32_t sum[4] = {0, 0, 0, 0};
#pragma unroll
                            for (int u = 0; u < 8; u++) {
                                sum[0] = pa_times_0(w[u].x, sum[0]);
                                sum[1] = pa_times_0(w[u].y, sum[1]);
                                sum[2] = pa_times_0(w[u].z, sum[2]);
                                sum[3] = pa_times_0(w[u].w, sum[3]);
                            }
                            if (!((sum[0] | sum[1] | sum[2] | sum[3]) & 0x7fff7fffu)) continue;
#pragma unroll 1
                            for (int u = 0; u < 8; u++) {
                                const int at = i + u * 512, r = (at / 128) & 127;
                                // the piece's place in its row is swizzled by the row
                                const int d0 = part * C::SPAN + (at / pa::PANEL) * 64 + (((at >> 4) & 7) ^ (r & 7)) * 8;
                                uint16_t *h = (uint16_t *)(st + at);
                                for (int x8 = 0; x8 < 8; x8++) {
                                    const uint16_t x = h[x8];
                                    if ((x & 0x7f80) != 0x7f80) continue;
                                    h[x8] = 0;
                                    const int sh = ((x & 0x7f) ? 0 : (x >> 15) ? 2 : 1) * 10;
                                    const uint32_t key = (uint32_t)(key0 - mask_from * pa::BN + r);
                                    uint32_t old = bad_key[d0 + x8], was;
                                    while (key < ((old >> sh) & 1023u)) {
                                        was = old;
                                        old = atomicCAS(&bad_key[d0 + x8], was, (was & ~(1023u << sh)) | (key << sh));
                                        if (old == was) break;
                                    }
                                    poison[k & 1] = 1;
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
        }
    }
    } else {                            // ---- softmax, one row a thread
        if constexpr (NQ == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int i = (warp - 4) >> 2;                      // query tile
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t o_col = tmem + lanes + C::O_COL + i * D;
        const float raise = pa::RAISE / a.zscale;
        bool ok = true;
        auto wait = [&](uint64_t *bar, unsigned parity) {
            if (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity)))
                ok = __all_sync(0xffffffffu, pa_wait(bar, parity, ab));
            tc_fence_after();
        };
        unsigned used = 0;              // key tiles of the items before
        for (int k = 0; ok; k++) {
            int nti, first_mask, seen;
            {
                PaItem it;
                if (!next_item(k, it)) break;
                const PaTiles<NQ> t = pa_tiles<NQ>(it);
                nti = __shfl_sync(0xffffffffu, i == 0 ? t.nt[0] : t.nt[NQ - 1], 0);
                first_mask = __shfl_sync(0xffffffffu, i == 0 ? t.first_mask[0] : t.first_mask[NQ - 1], 0);
                used = __shfl_sync(0xffffffffu, used, 0);
                const int row = it.r0 + i * pa::BM + (warp & 3) * 32 + lane;    // row in the sequence
                seen = max(0, min(it.m, it.m - it.n + min(row, it.n - 1) + 1));       // keys that it sees
            }
            float m = -INFINITY, l = 0.f;
            for (int j = 0; j < nti; j++) {
                const unsigned u = used + (unsigned)j;
                wait(&s_full[i], u & 1);
                if (!ok) break;
                float v[128];
                tc_ld128(tmem + lanes, v);
                tc_fence_before();
                mbar_arrive(&s_free);
                if (j >= first_mask) {
                    const int lim = seen - j * pa::BN;
#pragma unroll
                    for (int c = 0; c < 128; c++) v[c] = c < lim ? v[c] : -INFINITY;
                }
                float mx[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
                for (int c = 4; c < 128; c += 4)
#pragma unroll
                    for (int h = 0; h < 4; h++) mx[h] = fmaxf(mx[h], v[c + h]);
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                const bool up = top > m + raise;
                if (__any_sync(0xffffffffu, up)) {
                    const float down = !up ? 1.0f : m == -INFINITY ? 0.f : pa_ex2((m - top) * a.zscale);
                    if (up) m = top;
                    l *= down;
                    if (j > 0) {                 // O is the product's of j - 1 until that is done
                        wait(&o_done[p_at(i, u - 1)], p_use(u - 1) & 1);
                        if (!ok) break;
#pragma unroll 1
                        for (int c = 0; c < D; c += 32) {
                            uint32_t o[32];
                            tc_ld32(o_col + c, o);
#pragma unroll
                            for (int h = 0; h < 32; h++) o[h] = __float_as_uint(__uint_as_float(o[h]) * down);
                            tc_st32(o_col + c, o);
                        }
                    }
                }
                float mz = m == -INFINITY ? 0.f : m * a.zscale;
                // a product that is rounded to 2^-7 and more: the difference first, which is
                // exact for neighbours (from 2^31 on, the rounding alone reached 2^127)
                const bool huge = fabsf(mz) > 65536.0f;      // each row by its own scores alone
                if (__any_sync(0xffffffffu, huge)) {
                    const uint64_t down = huge ? f32_pair(-m, -m) : 0;
#pragma unroll
                    for (int c = 0; c < 128; c += 2) f32_unpair(add_f32x2(f32_pair(v[c], v[c + 1]), down), v[c], v[c + 1]);
                    if (huge) mz = 0.f;
                }
                // two scores an instruction (packed fp32): the loop is a quarter shorter (seven
                // ragged prompts of 32 heads over 8 of 128, 4099 rows: 66 -> 63 us)
                const uint64_t scale2 = f32_pair(a.zscale, a.zscale), mz2 = f32_pair(-mz, -mz);
                uint64_t sum[2] = {0, 0};
                uint32_t pk[2][32];
#pragma unroll
                for (int c = 0; c < 128; c += 2) {
                    float p0, p1;
                    f32_unpair(fma_f32x2(f32_pair(v[c], v[c + 1]), scale2, mz2), p0, p1);
                    p0 = pa_ex2(p0);
                    p1 = pa_ex2(p1);
                    sum[(c >> 1) & 1] = add_f32x2(sum[(c >> 1) & 1], f32_pair(p0, p1));
                    pk[c / 64][(c % 64) / 2] = pa_pack(p0, p1);
                }
                {
                    float s0, s1;
                    f32_unpair(add_f32x2(sum[0], sum[1]), s0, s1);
                    l += s0 + s1;
                }
                // P's place is read by the product of its last use until that is done
                if (p_use(u) > 0) {
                    wait(&o_done[p_at(i, u)], (p_use(u) - 1) & 1);
                    if (!ok) break;
                }
                const uint32_t p_col = tmem + lanes + C::P_COL + p_at(i, u) * 64;
                tc_st32(p_col, pk[0]);
                tc_st32(p_col + 32, pk[1]);
                tc_wait_st();
                tc_fence_before();
                mbar_arrive(&p_full[p_at(i, u)]);
            }
            used += (unsigned)nti;
            if (NQ == 1 && ok && nti > 1) wait(&o_done[p_at(i, used - 2)], p_use(used - 2) & 1);
            if (ok && nti > 0) wait(&o_done[p_at(i, used - 1)], p_use(used - 1) & 1);
            if (!ok) break;
            const float inv = l == 0.f ? 0.f : 1.0f / l;
            // (the addresses below are the same for every item: kept out of the registers
            // of the loop above, which has none left)
            int ln = lane;
            asm volatile("" : "+r"(ln));
            uint8_t *const own = ring + NST * C::STAGE + (warp - 4) * C::OUT;
            const PaItem it = items[k & 1];
            int mask_from;
            bool bad;
            {
                const PaTiles<NQ> t = pa_tiles<NQ>(it);
                mask_from = t.mask_from;
                bad = mask_from < t.ntmax && *(volatile int *)&poison[k & 1];
            }
            const int row0 = it.r0 + i * pa::BM + (warp & 3) * 32, left = it.n - row0;      // this warp's first row, rows that exist
            uint16_t *const op = a.out.p + (long)(it.q0 + row0) * a.out.rs + (long)it.head * a.out.hs;
            // through shared memory, so that a store covers 128 bytes of four rows:
            // 16-byte pieces, swizzled by the row
#pragma unroll 1
            for (int c = 0; c < D; c += 64) {
                float o[64];
                if (nti > 0) tc_ld64(o_col + c, o);
                else
#pragma unroll
                    for (int h = 0; h < 64; h++) o[h] = 0.f;
#pragma unroll
                for (int h = 0; h < 8; h++) {
                    uint32_t w[4];
#pragma unroll
                    for (int x = 0; x < 4; x++) w[x] = pa_pack(o[8 * h + 2 * x] * inv, o[8 * h + 2 * x + 1] * inv);
                    *(uint4 *)(own + ln * 128 + ((h ^ (ln & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                }
                if (bad)
#pragma unroll 1
                    for (int d = 0; d < 64; d++) {
                        const uint32_t f = first_bad[k & 1][c + d];
                        const int rel = seen - mask_from * pa::BN;       // looked-after keys that the row sees
                        uint16_t *o = (uint16_t *)(own + ln * 128 + (((d >> 3) ^ (ln & 7)) << 4)) + (d & 7);
                        const bool pos = rel > (int)((f >> 10) & 1023u), neg = rel > (int)(f >> 20);
                        if (rel > (int)(f & 1023u) || (pos && (neg || *o == 0xff80)) || (neg && *o == 0x7f80)) *o = 0x7fff;
                        else if ((pos || neg) && (*o & 0x7fff) <= 0x7f80) *o = pos ? 0x7f80 : 0xff80;
                    }
                __syncwarp();
                // (a warp's row 4 r + ln / 8, piece ln % 8)
                uint16_t *to = op + (long)(ln >> 3) * a.out.rs + c + (ln & 7) * 8;
#pragma unroll
                for (int r = 0; r < 32; r += 4) {
                    const int rr = r + (ln >> 3);
                    const uint4 x = lds128(own + rr * 128 + (((ln & 7) ^ (rr & 7)) << 4));
                    if (rr < left) *(uint4 *)to = x;
                    to += 4 * a.out.rs;
                }
                __syncwarp();
            }
            tc_fence_before();          // before the next item's first product writes O (after this thread's next p_full)
            done_with(k);
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
    // looked up again after a failure; first calls of several threads may each look it up
    static std::atomic<PFN_cuTensorMapEncodeTiled_v12000> encoder{nullptr};
    PFN_cuTensorMapEncodeTiled_v12000 enc = encoder.load(std::memory_order_acquire);
    if (!enc) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess) {
            gcuda_set_error("prompt_attn: no tensor map encoder");
            return -1;
        }
        enc = (PFN_cuTensorMapEncodeTiled_v12000)p;
        encoder.store(enc, std::memory_order_release);
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
    return attn_launch("prompt_attn launch", k_prompt_tc<D>, dim3((unsigned)blocks), C::THREADS, C::SMEM, st, false, qm, km, vm, a);
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
