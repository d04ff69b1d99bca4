// GQA attention, head_dim 256, of a tree of drafted tokens over a paged bf16 KV cache, on the Blackwell tensor cores.
//
// Node i of sequence b hangs below node parents[b][i] < i (or, -1, below the last cached token) and attends the cached keys
// 0 .. ctx_len[b] - 1, its ancestors and itself:  softmax(q_i K^T / 16) V.  The chained verify (gqa_decode_tc.cu) has at most 16 query rows
// per KV head; a tree has up to 64 nodes x (H / KV) query heads, so here the rows fill the 128 of a tensor-core tile and a K / V tile is
// read once for all of them.  Bound: HBM (2 KiB per key and pair of KV heads) up to about 128 rows per KV head, the tensor pipe beyond.
//
// Work: a (sequence, KV head) is a "pair"; its keys come in 128-key tiles, the last tile holding the nodes themselves (from the call's
// k_new / v_new).  The tiles of all pairs laid end to end are cut into equal ranges, one per SM, so that one long sequence occupies the
// whole GPU as well as many short ones; a pair that is cut leaves fp32 partials, which a second small kernel joins (overlapping its
// launch with this kernel's end).  Every block derives the plan from ctx_len itself.  More than 128 rows take several row tiles: the blocks
// then form groups, one block per row tile, that walk the same range side by side, so that one of them brings a tile out of HBM and
// the others find it in L2 (with the row tiles one after the other in the plan, 2 x 64 nodes over 64 k tokens read everything twice:
// 112 us against 98).
//
// Roles: warps 0-3 softmax (one thread per query row; warps without rows sleep), warp 4 issues the MMAs, warps 5 and 6 are the TMA
// producers of K and V, warp 7 appends the nodes' rows to the cache and makes their value rows fit for the product.  Per tile
//     S [128 x 128]  = Q K^T      16 MMAs; K travels in slabs of 64 dims x 128 keys
//     P              = 2^(S sc - m), written over S in tensor memory as bf16 hi + lo pairs (weights exact to 2^-17, as in the chained
//                      and prefill kernels; hi alone would put an error of the size of the output's own rounding on every weight)
//     O [128 x 256] += P V        16 MMAs; V travels in chunks of 32 keys x 256 dims, read N-major
// with S / P double buffered, so the scores of the next tile (also of the next pair's first one) are formed while the softmax of this
// one runs.  The running maximum is only raised when a tile exceeds it by more than 2^8, which keeps rescales of O rare.
//
// Pages: the boxes of the page maps hold gcd(page_size, 128) keys (K) and gcd(page_size, 32) keys (V), so a box never crosses a page and any
// page size works; pages of a multiple of 32 / 128 keys take the fewest copies.  (The 128-byte swizzle goes by shared-memory address bits,
// so small boxes side by side form the same image as one large box.)
//
// Masked places never reach the sums: scores are replaced, not multiplied; value rows behind the context and of unused nodes are zeroed in
// shared memory; non-finite values of a node are zeroed there too (their weight is 0 for nodes that do not see it, and 0 x NaN is NaN)
// and added back in the epilogue of the rows that do see it.
// Every wait is bounded; one that gives up sets the device status word and the block runs out its loops.  No block leaves before the copies and
// products that it issued are over, whichever role gave up.
#include <cstring>
#include "gqa_common.cuh"
#include "sm100_prims.cuh"

namespace gdn {

using namespace sm100;

constexpr int TA_THREADS = 256, TA_TK = 128;
constexpr int TA_MAX_B = 256;                                         // sequences per launch (the plan lives in shared memory)
constexpr int TA_SLOT = 16384, TA_NK = 5, TA_NV = 5;                  // K slab: 128 keys x 64 dims; V chunk: 32 keys x 256 dims
constexpr int TA_Q_BYTES = 65536;                                     // 128 rows, or two buffers of up to 64 rows
constexpr int TA_SMEM = TA_Q_BYTES + (TA_NK + TA_NV) * TA_SLOT;
constexpr uint32_t TAM_O = 0, TAM_SP0 = 256;
constexpr int TA_TAIL = 3;                                            // plan weight of a pair's end (its nodes and epilogue, 8 us) in tiles (2.6 us)
constexpr float TA_RAISE = 8.f;                                       // log2 units
enum {
    AB_QFULL = 0, AB_QEMPTY = 2, AB_KFULL = 4, AB_KEMPTY = AB_KFULL + TA_NK, AB_VFULL = AB_KEMPTY + TA_NK, AB_VEMPTY = AB_VFULL + TA_NV,
    AB_SDONE = AB_VEMPTY + TA_NV, AB_PREADY = AB_SDONE + 2, AB_PFREE = AB_PREADY + 2, AB_ODONE = AB_PFREE + 2, AB_OFREE, AB_LAST, AB_NODES, AB_DRAIN, AB_COUNT
};

struct TreeAttnPlan {
    TreeAttnArgs a;
    float* part;                 // [2 * G][64 column groups][rows][4]: partial O; then [2 * G][rows][2]: (m, l)
    float* part_ml;
    int* info;                   // a cut pair's first block, the pair and its number of partials (0: not cut), in the order the merge kernel's
                                 // grid has: by pair where there are at most G pairs (`by_pair`), by first block otherwise
    bool by_pair;
    int G;                       // blocks
    int group, nodes, rows;      // query heads per KV head, nodes per row tile, rows per tile
    int row_tiles, q_bufs, q_slab;       // row tiles per (sequence, KV head); Q buffers; bytes of a Q slab (64 dims of all rows)
    int k_box, v_box;            // keys per copy
};

struct TreeSeg { int b, kvh, t0, n, span, tiles, ctx; };          // tiles [t0, t0 + n) of a pair with `tiles` of them; span: of the plan

// {i, ancestors} of nodes lane and lane + 32 of one tree, as bit masks (0 = unused); par0 / par1: their parents (-2 beyond N)
__device__ __noinline__ void warp_lines(int par0, int par1, unsigned long long& l0, unsigned long long& l1, bool& bad) {
    const int lane = threadIdx.x & 31;
    const bool late0 = par0 >= lane, late1 = par1 >= lane + 32;      // a parent that does not precede its child
    if (late0) par0 = -2;
    if (late1) par1 = -2;
    bad = late0 || late1;
    int at0 = par0 < -1 ? -2 : par0, at1 = par1 < -1 ? -2 : par1;    // >= 0: still walking, -1: reached the root, -2: unused
    l0 = 1ull << lane; l1 = 1ull << (lane + 32);
    const bool in0 = par0 >= -1, in1 = par1 >= -1;
#pragma unroll 1
    while (__any_sync(0xffffffffu, at0 >= 0 || at1 >= 0)) {
        if (at0 >= 0) l0 |= 1ull << at0;
        if (at1 >= 0) l1 |= 1ull << at1;
        const int a0 = __shfl_sync(0xffffffffu, par0, at0 & 31), b0 = __shfl_sync(0xffffffffu, par1, at0 & 31);
        const int a1 = __shfl_sync(0xffffffffu, par0, at1 & 31), b1 = __shfl_sync(0xffffffffu, par1, at1 & 31);
        if (at0 >= 0) at0 = at0 < 32 ? a0 : b0;
        if (at1 >= 0) at1 = at1 < 32 ? a1 : b1;
    }
    if (at0 != -1) l0 = 0;
    if (at1 != -1) l1 = 0;
    bad = bad || (in0 && !l0) || (in1 && !l1);
}

__device__ __forceinline__ unsigned long long shfl64(unsigned long long v, int src) {
    return (unsigned long long)__shfl_sync(0xffffffffu, (uint32_t)v, src) | (unsigned long long)__shfl_sync(0xffffffffu, (uint32_t)(v >> 32), src) << 32;
}

// tcgen05.mma with the accumulate flag in a register
__device__ __forceinline__ void mma_ss_r(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .b64 da, db;\n\t.reg .pred p;\n\tmov.b64 da, {%1, %2};\n\tmov.b64 db, {%3, %4};\n\tsetp.ne.b32 p, %6, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n\t}"
                 ::"r"(d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void mma_ts_r(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .b64 db;\n\t.reg .pred p;\n\tmov.b64 db, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}"
                 ::"r"(d), "r"(a_tmem), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(acc) : "memory");
}

__device__ __forceinline__ bool bf16_not_finite(uint32_t bits) { return (bits & 0x7f80u) == 0x7f80u; }

// first tile of block g when G blocks share N tiles: the first N % G blocks take one more (32-bit: a division costs a tenth of a 64-bit one)
__device__ __forceinline__ int range_lo(int g, int G, int N) { const int q = N / G; return g * q + min(g, N - q * G); }

// The rest of a bounded wait whose first poll failed; out of line, because a wait is needed in two dozen places and the code of the
// roles' loops has to stay small (they run side by side out of one instruction cache).
__device__ __noinline__ bool tree_wait_slow(uint32_t addr, uint32_t parity, volatile int* abort, int* status) {
    for (uint32_t i = 0; i < WAIT_POLLS; i++) {
        if (mbar_test_wait(addr, parity)) return true;
        if ((i & 63u) == 63u && *abort) return false;
        __nanosleep(20);
    }
    *abort = 1;
    atomicExch(status, 2);
    return false;
}

__global__ void __launch_bounds__(TA_THREADS, 1)
tree_attn_kernel(const __grid_constant__ TreeAttnPlan p, const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                 const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmKn, const __grid_constant__ CUtensorMap tmVn) {
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ uint64_t bars[AB_COUNT];
    __shared__ int s_cum[TA_MAX_B + 1];                              // tiles of all pairs of the sequences before
    __shared__ int s_ctx[TA_MAX_B];                                  // contexts, -1 = skipped
    __shared__ int2 s_box[2][32];                                    // (page, row) of the boxes of a producer's tile
    __shared__ unsigned long long s_badv[2];
    __shared__ uint32_t tmem_slot;
    __shared__ int s_abort;
    const TreeAttnArgs& a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t sbase = smem_addr(smem);
    if (sbase & 1023u) { if (tid == 0) atomicExch(a.status, 4); return; }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");               // nothing an earlier kernel wrote is read before this

    GDN_BSTAMP(0);
    // ---- plan ----
    const long long cap = (long long)a.max_pages * a.page_size;
    const int rt = blockIdx.x % p.row_tiles, grp = blockIdx.x / p.row_tiles;      // row tile and group of this block
    // context of sequence b as the kernel uses it, -1 = skipped (negative, or the nodes do not fit the table)
    auto context = [&](int b) -> int {
        const int ctx = a.ctx_len[b];
        if (ctx < 0 || ctx > cap) return -1;
        if ((long long)ctx + a.N > cap) {                            // (rare: only then do the tree's unused nodes matter)
            int last = a.N - 1;
#pragma unroll 1
            while (last >= 0 && a.parents[(size_t)b * a.N + last] < -1) last--;
            if ((long long)ctx + last >= cap) return -1;
        }
        return ctx;
    };
    if (warp == 0) {
        int run = 0;
#pragma unroll 1
        for (int b0 = 0; b0 < a.B; b0 += 32) {
            const int b = b0 + lane;
            int x = 0;
            if (b < a.B) {
                const int ctx = context(b);
                if (ctx < 0 && blockIdx.x == 0) atomicExch(a.status, 1);
                s_ctx[b] = ctx;
                x = ((max(ctx, 0) + TA_TK - 1) / TA_TK + 1 + TA_TAIL) * a.KV;
            }
            const int own = x;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, x, o); if (lane >= o) x += y; }
            if (b < a.B) s_cum[b] = run + x - own;
            run += __shfl_sync(0xffffffffu, x, 31);
        }
        if (lane == 0) s_cum[a.B] = run;
    }
    auto bar = [&](int i) -> uint32_t { return smem_addr(&bars[i]); };
    const int n_warps = (p.rows + 31) / 32;                          // softmax warps with rows
    if (tid == 32) {
        for (int i = 0; i < AB_COUNT; i++) mbar_init(bar(i), (i >= AB_PREADY && i < AB_PREADY + 2) || i == AB_OFREE ? n_warps : 1);
        s_abort = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tmQ); tma_prefetch_desc(&tmK); tma_prefetch_desc(&tmV); tma_prefetch_desc(&tmKn); tma_prefetch_desc(&tmVn);
    }
    if (warp == 4) { tmem_alloc(smem_addr(&tmem_slot), 512); tmem_relinquish(); }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tb = tmem_slot;
    GDN_BSTAMP(1);
    const int N_all = s_cum[a.B];
    const int G = min((int)gridDim.x / p.row_tiles, N_all);
    const int lo = grp < G ? range_lo(grp, G, N_all) : 0, hi = grp < G ? range_lo(grp + 1, G, N_all) : 0;

    auto aborted = [&]() -> bool { return *(volatile int*)&s_abort != 0; };
    // bounded; a failure tells the whole block to stop computing
    auto wait = [&](int b, uint32_t parity) -> bool {
        return mbar_test_wait(bar(b), parity & 1u) || tree_wait_slow(bar(b), parity & 1u, &s_abort, a.status);
    };
    // the same for a whole warp: every lane gets the same answer, whatever a lane saw of an abort
    auto warp_wait = [&](int b, uint32_t parity) -> bool {
        if (__all_sync(0xffffffffu, mbar_test_wait(bar(b), parity & 1u))) return true;
        int got = 0;
        if (lane == 0) got = tree_wait_slow(bar(b), parity & 1u, &s_abort, a.status);
        return __shfl_sync(0xffffffffu, got, 0) != 0;
    };
    // the part of the block's range that starts at tile x: it ends with the pair or with the range
    auto segment = [&](int x) -> TreeSeg {
        int l = 0, r = a.B - 1;
#pragma unroll 1
        while (l < r) { const int m = (l + r + 1) >> 1; if (s_cum[m] <= x) l = m; else r = m - 1; }
        TreeSeg s;
        s.b = l;
        s.ctx = s_ctx[l];
        s.tiles = (max(s.ctx, 0) + TA_TK - 1) / TA_TK + 1;
        const int off = x - s_cum[l], len = s.tiles + TA_TAIL;
        s.kvh = off / len;
        s.t0 = off - s.kvh * len;
        s.span = min(len - s.t0, hi - x);
        s.n = min(s.tiles - s.t0, s.span);                           // (0 or less where the range starts in a pair's tail)
        return s;
    };
    const uint32_t sQ = sbase, sK = sbase + TA_Q_BYTES, sV = sK + TA_NK * TA_SLOT;
    // keys of tile t of a segment's pair (the last tile holds the nodes)
    auto limit_of = [&](const TreeSeg& s, int t) -> int { return t == s.tiles - 1 ? a.N : min(TA_TK, s.ctx - t * TA_TK); };

    // nothing to join, as far as is known (every pair starts in exactly one block, and only that one writes its entry)
    auto clear_info = [&]() {
        if (!p.by_pair) { *reinterpret_cast<int2*>(p.info + 2 * blockIdx.x) = make_int2(0, 0); return; }
#pragma unroll 1
        for (int x = lo; x < hi;) {
            const TreeSeg s = segment(x);
            x += s.span;
            if (s.t0 == 0) p.info[2 * ((s.b * a.KV + s.kvh) * p.row_tiles + rt) + 1] = 0;
        }
    };
    if (tid == 0) clear_info();
    if (warp == 5 || warp == 6) {
        // ================= producers: warp 5 Q and K, warp 6 V =================
        // Lane i works out page and row of box i of a tile (a tile has at most 32 boxes where the page size is a multiple of 4); page
        // numbers come in windows of 32 table entries, one per lane, the next window requested a window ahead, because a plain load
        // takes microseconds under the copies.  Then lane j is the producer of the tile's j-th ring slot: it polls that slot and
        // issues that slot's copies.  (One lane doing all of it, slot after slot, took 7 .. 13 k cycles a tile; the memory needs 5.7 k.)
        const bool isk = warp == 5;
        const int box = isk ? p.k_box : p.v_box, per_tile = TA_TK / box, per_chunk = 32 / min(box, 32);
        const int first_empty = isk ? AB_KEMPTY : AB_VEMPTY, first_full = isk ? AB_KFULL : AB_VFULL, ring = isk ? TA_NK : TA_NV;
        const uint32_t base = isk ? sK : sV;
        uint64_t stream_policy;                                      // the cache is read once per row tile: first to leave L2 unless a second row tile follows
        if (p.row_tiles == 1) asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(stream_policy));
        else asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(stream_policy));
        uint32_t nr = 0, nq = 0, nseg = 0, part = 0;                 // slots and Q buffers filled so far; lanes that filled one of a tile given up
        bool okp = true;
#pragma unroll 1
        for (int x = lo; x < hi && okp;) {
            const TreeSeg s = segment(x);
            x += s.span;
            if (s.n <= 0) continue;
            if (isk) {
                const int qb = nseg % p.q_bufs;
                if (nseg >= (uint32_t)p.q_bufs && !warp_wait(AB_QEMPTY + qb, nseg / p.q_bufs - 1)) { okp = false; break; }
                if (lane == 0) {
                    mbar_expect_tx(bar(AB_QFULL + qb), p.rows * 512);
                    for (int j = 0; j < 4; j++)
                        tma_load_3d(sQ + qb * (TA_Q_BYTES / 2) + j * p.q_slab, &tmQ, bar(AB_QFULL + qb), 64 * j, s.kvh * p.group, s.b * a.N + rt * p.nodes);
                }
                nq++;
            }
            const int* table = a.block_table + (size_t)s.b * a.max_pages;
            const int entries = s.ctx > 0 ? (s.ctx - 1) / a.page_size + 1 : 0;      // those that hold context
            auto entry = [&](int e) -> int { return e < entries ? table[e] : 0; };
            auto checked = [&](int pg) -> int {                      // a bad page number is reported, and page 0 read in its place
                if (pg >= 0 && pg < a.n_pages) return pg;
                atomicExch(a.status, 1);
                return 0;
            };
            int w = s.t0 * TA_TK / a.page_size;                      // first entry of the current window
            int cur = entry(w + lane), nxt = entry(w + 32 + lane);
#pragma unroll 1
            for (int t = s.t0; t < s.t0 + s.n && okp; t++) {
                const int limit = limit_of(s, t);
                const bool nodes = t == s.tiles - 1;
                if (!nodes && per_tile <= 32) {
                    const int first = t * TA_TK / a.page_size;
#pragma unroll 1
                    while (first >= w + 32) { w += 32; cur = nxt; nxt = entry(w + 32 + lane); }
                    const int key = min(t * TA_TK + lane * box, s.ctx - 1), e = key / a.page_size - w;      // (boxes behind the context are not copied)
                    const int p0 = __shfl_sync(0xffffffffu, cur, e & 31), p1 = __shfl_sync(0xffffffffu, nxt, e & 31);
                    s_box[warp - 5][lane] = make_int2(checked(e < 32 ? p0 : p1), key - (w + e) * a.page_size);
                    __syncwarp();
                }
                // K: four slabs of 64 dims, all boxes each; V: chunks of 32 keys, its boxes whole rows
                const int steps = isk ? 4 : (limit + 31) / 32, j = lane;
                const uint32_t mine = nr + lane, slot = mine % ring, round = mine / ring;
                const uint32_t full = bar(first_full + slot), empty = bar(first_empty + slot), dst = base + slot * TA_SLOT;
                const int i0 = isk ? 0 : j * per_chunk;              // this lane's boxes [i0, i0 + cnt)
                const int cnt = isk ? (limit + box - 1) / box : (min(32, limit - 32 * j) + box - 1) / box;
                bool todo = lane < steps;
#pragma unroll 1
                for (uint32_t polls = 0; __any_sync(0xffffffffu, todo); polls++) {
                    if (todo && (round == 0 || mbar_test_wait(empty, (round - 1) & 1u))) {
                        todo = false;
                        if (nodes) {
                            mbar_expect_tx(full, isk ? 64 * 128 : TA_SLOT);
                            if (isk) tma_load_3d(dst, &tmKn, full, 64 * j, s.kvh, s.b * a.N);
                            else for (int k = 0; k < 4; k++) tma_load_3d(dst + k * 4096, &tmVn, full, 64 * k, s.kvh, s.b * a.N + 32 * j);
                        } else {
                            mbar_expect_tx(full, cnt * box * (isk ? 128 : 512));
#pragma unroll 1
                            for (int i = 0; i < cnt; i++) {
                                int2 at;
                                if (per_tile <= 32) at = s_box[warp - 5][i0 + i];
                                else {                               // (page sizes that are not a multiple of 4: looked up in place)
                                    const int key = t * TA_TK + (i0 + i) * box, e = key / a.page_size;
                                    at = make_int2(checked(table[e]), key - e * a.page_size);
                                }
                                // V: the four 64-dim blocks of 32 rows are the chunk's image; of smaller boxes each block is a copy of its own
                                const int copies = isk || box == 32 ? 1 : 4;
#pragma unroll 1
                                for (int k = 0; k < copies; k++)
                                    asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4, %5, %6, %7}], [%2], %8;"
                                                 ::"r"(dst + i * box * 128 + k * 4096), "l"(isk ? &tmK : &tmV), "r"(full), "r"(0), "r"(at.y), "r"(isk ? j : k), "r"(s.kvh), "r"(at.x), "l"(stream_policy) : "memory");
                            }
                        }
                    } else if (todo) {
                        __nanosleep(20);
                    }
                    if ((polls & 63u) == 63u && __any_sync(0xffffffffu, aborted() || polls > WAIT_POLLS)) { okp = false; break; }
                }
                if (!okp) {
                    if (lane == 0 && !aborted()) { s_abort = 1; atomicExch(a.status, 2); }
                    part = __ballot_sync(0xffffffffu, lane < steps && !todo);
                    break;
                }
                nr += steps;
                __syncwarp();                                        // (s_box is rewritten by the next tile)
            }
            nseg++;
        }
        // Every copy has to land before the block leaves, also where another role gives up: lane i sees to the last one into slot i (a
        // tile fills at most `ring` slots, so a tile given up added at most one), lanes behind it to the Q buffers.
        const uint32_t first_use = lane < ring ? lane : lane - ring, every = lane < ring ? ring : p.q_bufs;
        uint32_t uses = lane < ring ? nr : isk && lane < ring + p.q_bufs ? nq : 0;
        uses = uses > first_use ? (uses - 1 - first_use) / every + 1 : 0;
        if (lane < ring && (part >> (lane + ring - nr % ring) % ring & 1)) uses++;
        if (uses) mbar_wait(bar(lane < ring ? first_full + lane : AB_QFULL + first_use), (uses - 1) & 1u, DRAIN_POLLS);
    } else if (warp == 4) {
        // ================= MMA issuer =================
        if (lane == 0) {
            constexpr uint32_t I_QK = idesc_bf16(128, 128, 0, 0), I_QN = idesc_bf16(128, 64, 0, 0);
            constexpr uint32_t I_PV = idesc_bf16(128, 256, 0, 1);    // B = V read N-major (dims contiguous)
            constexpr uint32_t HI = smem_desc_hi_sw128(1024);
            uint32_t k_slot = 0, k_round = 0, v_slot = 0, v_round = 0, n = 0, nseg = 0;      // ring positions; tiles and segments so far
            bool ok = true;
            // the P V product of tile m with `limit` keys; first / last: of its segment (the ps-th)
            auto issue_pv = [&](uint32_t m, int limit, bool first, bool last, uint32_t ps) -> bool {
                const uint32_t sp = tb + TAM_SP0 + (m & 1) * 128;
                if (!wait(AB_PREADY + (m & 1), m >> 1)) return false;
                if (first && ps > 0 && !wait(AB_OFREE, ps - 1)) return false;      // the epilogue before has read O
                GDN_TSTAMP(m * 16 + 2);
                uint32_t acc = first ? 0 : 1;                        // the first product of a segment overwrites O
#pragma unroll 2
                for (int c = 0; 32 * c < limit; c++) {
                    if (!wait(AB_VFULL + v_slot, v_round)) return false;
                    tc_fence_after_sync();
                    const uint32_t vlo = smem_desc_lo(sV + v_slot * TA_SLOT, 4096), acol = sp + 32 * c;
                    mma_ts_r(tb + TAM_O, acol, vlo, HI, I_PV, acc);  // hi and lo of keys 32 c .. 32 c + 15, then of the other 16
                    mma_ts_w<true>(tb + TAM_O, acol + 16, vlo, HI, I_PV);
                    if (limit - 32 * c > 16) {
                        mma_ts_w<true>(tb + TAM_O, acol + 8, vlo + 128, HI, I_PV);
                        mma_ts_w<true>(tb + TAM_O, acol + 24, vlo + 128, HI, I_PV);
                    }
                    acc = 1;
                    mma_commit(bar(AB_VEMPTY + v_slot));
                    if (++v_slot == TA_NV) { v_slot = 0; v_round++; }
                }
                mma_commit(bar(AB_PFREE + (m & 1)));
                if (last) mma_commit(bar(AB_ODONE));
                GDN_TSTAMP(m * 16 + 3);
                return true;
            };
            int p_limit = 0;
            bool p_have = false, p_first = false, p_last = false;
            uint32_t p_seg = 0;
#pragma unroll 1
            for (int x = lo; x < hi && ok;) {
                const TreeSeg s = segment(x);
                x += s.span;
                if (s.n <= 0) continue;
                const int qb = nseg % p.q_bufs;
                if (!wait(AB_QFULL + qb, nseg / p.q_bufs)) { ok = false; break; }
                const uint32_t qlo = smem_desc_lo(sQ + qb * (TA_Q_BYTES / 2), 16);
#pragma unroll 1
            for (int t = s.t0; t < s.t0 + s.n && ok; t++, n++) {
                    // the buffer of tile n held P of tile n - 2, whose product was issued before: MMAs of one thread run in order
                    const uint32_t sp = tb + TAM_SP0 + (n & 1) * 128;
                    const uint32_t idesc = t == s.tiles - 1 ? I_QN : I_QK;
                    GDN_TSTAMP(n * 16 + 0);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        if (!wait(AB_KFULL + k_slot, k_round)) { ok = false; break; }
                        tc_fence_after_sync();
                        const uint32_t klo = smem_desc_lo(sK + k_slot * TA_SLOT, 16), ql = qlo + j * (p.q_slab >> 4);
                        mma_ss_r(sp, ql, HI, klo, HI, idesc, j);     // (the first product of a tile overwrites S)
#pragma unroll
                        for (int kk = 1; kk < 4; kk++) mma_ss_w<true>(sp, ql + kk * 2, HI, klo + kk * 2, HI, idesc);
                        mma_commit(bar(AB_KEMPTY + k_slot));
                        if (++k_slot == TA_NK) { k_slot = 0; k_round++; }
                    }
                    if (!ok) break;
                    mma_commit(bar(AB_SDONE + (n & 1)));
                    GDN_TSTAMP(n * 16 + 1);
                    if (t == s.t0 + s.n - 1) mma_commit(bar(AB_QEMPTY + qb));
                    if (p_have) ok = issue_pv(n - 1, p_limit, p_first, p_last, p_seg);
                    if (t == s.tiles - 1) mma_commit(bar(AB_LAST));  // the chunks before the nodes' have been consumed
                    p_have = true; p_limit = limit_of(s, t); p_first = t == s.t0; p_last = t == s.t0 + s.n - 1; p_seg = nseg;
                }
                nseg++;
            }
            if (ok && p_have) ok = issue_pv(n - 1, p_limit, p_first, p_last, p_seg);
            mma_commit(bar(AB_DRAIN));                               // no product may run on after the block, whichever role gave up
            mbar_wait(bar(AB_DRAIN), 0, DRAIN_POLLS);
        }
    } else if (warp == 7) {
        // ================= nodes: their rows into the cache, by the block that has a pair's first tile; their value rows fit for the product =================
        uint32_t nv = 0, node_tiles = 0;                             // V chunks and node tiles so far
        bool ok = true;
#pragma unroll 1
        for (int x = lo; x < hi && ok;) {
            const TreeSeg s = segment(x);
            x += s.span;
            if (s.n <= 0) continue;
            const bool has_nodes = s.t0 + s.n == s.tiles, append = s.t0 == 0 && rt == 0 && s.ctx >= 0;
            unsigned long long used = 0;
            if (append || has_nodes) {
                const int* par = a.parents + (size_t)s.b * a.N;
                unsigned long long l0, l1;
                bool bad;
                warp_lines(s.ctx >= 0 && lane < a.N ? par[lane] : -2, s.ctx >= 0 && lane + 32 < a.N ? par[lane + 32] : -2, l0, l1, bad);
                if (bad && append) atomicExch(a.status, 1);
                used = __ballot_sync(0xffffffffu, l0 != 0) | (unsigned long long)__ballot_sync(0xffffffffu, l1 != 0) << 32;
            }
            auto append_rows = [&]() {                               // four rows of K and V in flight
                const int* table = a.block_table + (size_t)s.b * a.max_pages;
                int page[2];
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const int i = lane + 32 * k;
                    page[k] = used >> i & 1 ? table[(s.ctx + i) / a.page_size] : -1;
                    if ((used >> i & 1) && (page[k] < 0 || page[k] >= a.n_pages)) { atomicExch(a.status, 1); page[k] = -1; }
                }
#pragma unroll 1
                for (int i0 = 0; i0 < a.N; i0 += 4) {
                    uint4 kr[4], vr[4];
                    size_t dst[4];
                    bool on[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int i = i0 + k, pg = __shfl_sync(0xffffffffu, i0 < 32 ? page[0] : page[1], i & 31);
                        on[k] = i < a.N && pg >= 0;
                        dst[k] = (((size_t)pg * a.KV + s.kvh) * a.page_size + (s.ctx + i) % a.page_size) * ATT_D;
                        if (on[k]) {
                            const size_t src = (((size_t)s.b * a.N + i) * a.KV + s.kvh) * ATT_D;
                            kr[k] = reinterpret_cast<const uint4*>(a.k_new + src)[lane];
                            vr[k] = reinterpret_cast<const uint4*>(a.v_new + src)[lane];
                        }
                    }
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        if (on[k]) {
                            reinterpret_cast<uint4*>(a.k_pages + dst[k])[lane] = kr[k];
                            reinterpret_cast<uint4*>(a.v_pages + dst[k])[lane] = vr[k];
                        }
                }
            };
            // a long range has time for the copies before its nodes' tile comes up, a short one after it
            if (append && s.n >= 4) append_rows();
            nv += (max(min(s.ctx, (s.t0 + s.n) * TA_TK) - s.t0 * TA_TK, 0) + 31) / 32;
            if (has_nodes) {
                // value rows of unused nodes (and behind the last) and the non-finite values of the others are zeroed, once the chunks
                // before these have been consumed (a parity of the ring cannot tell a phase from the one two before).  The wait lasts as
                // long as the segment, and so does its bound.
                int got = 0;
                if (lane == 0) {
                    for (long long i = 0; i < (long long)(WAIT_POLLS / 2) * (s.n + 1) && !got && !aborted(); i++) {
                        got = mbar_test_wait(bar(AB_LAST), node_tiles & 1u);
                        if (!got) __nanosleep(100);
                    }
                    if (!got && !aborted()) { s_abort = 1; atomicExch(a.status, 2); }
                }
                ok = __shfl_sync(0xffffffffu, got, 0) != 0;
                unsigned long long seen_bad = 0;
#pragma unroll 1
                for (int c = 0; c < (a.N + 31) / 32 && ok; c++) {
                    const uint32_t slot = (nv + c) % TA_NV;
                    ok = warp_wait(AB_VFULL + slot, (nv + c) / TA_NV);
                    if (!ok) break;
                    unsigned char* chunk = smem + TA_Q_BYTES + TA_NK * TA_SLOT + slot * TA_SLOT + (lane >> 3) * 4096;      // lane = 16-byte column of a row
#pragma unroll 4
                    for (int r = 0; r < 32; r++) {
                        uint4* at = reinterpret_cast<uint4*>(chunk + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
                        if (!(used >> (32 * c + r) & 1)) { *at = make_uint4(0, 0, 0, 0); continue; }
                        const uint4 v = *at;
                        uint32_t w[4] = {v.x, v.y, v.z, v.w};
                        // an exponent of ones in either half carries into the half's top bit
                        const uint32_t E = 0x7f807f80u, one = 0x00800080u;
                        if (!((((w[0] & E) + one) | ((w[1] & E) + one) | ((w[2] & E) + one) | ((w[3] & E) + one)) & 0x80008000u)) continue;
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            if (bf16_not_finite(w[q])) w[q] &= 0xffff0000u;
                            if (bf16_not_finite(w[q] >> 16)) w[q] &= 0xffffu;
                        }
                        seen_bad |= 1ull << (32 * c + r);
                        *at = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
                if (!ok) break;
                fence_proxy_async_smem();
                __syncwarp();
                const uint32_t b0 = __reduce_or_sync(0xffffffffu, (uint32_t)seen_bad), b1 = __reduce_or_sync(0xffffffffu, (uint32_t)(seen_bad >> 32));
                if (lane == 0) {
                    s_badv[node_tiles & 1] = b0 | (unsigned long long)b1 << 32;      // (last read before the product two node tiles ago)
                    mbar_arrive(bar(AB_NODES));
                }
                node_tiles++;
                nv += (a.N + 31) / 32;
            }
            if (append && s.n < 4) append_rows();
        }
    } else if (warp < n_warps) {
        // ================= softmax and epilogue: thread = row = node * group + head =================
        const float sc = 0.0625f * 1.4426950408889634f;              // 256^-1/2, scores kept in log2 units
        const int row = tid, local = row / p.group;
        const uint32_t tl = tb + ((uint32_t)(warp * 32) << 16);      // this warp's TMEM lanes
        uint32_t n = 0, nv = 0, nseg = 0, node_tiles = 0;
        bool ok = true;
#pragma unroll 1
        for (int x = lo; x < hi;) {
            const TreeSeg s = segment(x);
            x += s.span;
            if (s.n <= 0) continue;
            const int node = rt * p.nodes + local;
            const bool real = row < p.rows && node < a.N;
            const bool has_nodes = s.t0 + s.n == s.tiles;
            int par0 = -2, par1 = -2;                                // requested early, used at the last tile
            if (has_nodes && s.ctx >= 0) {
                const int* par = a.parents + (size_t)s.b * a.N;
                if (lane < a.N) par0 = par[lane];
                if (lane + 32 < a.N) par1 = par[lane + 32];
            }
            unsigned long long line = 0, badv = 0;
            float m_run = -INFINITY, l_run = 0.f;
#pragma unroll 1
            for (int t = s.t0; t < s.t0 + s.n && ok; t++, n++) {
                const int limit = limit_of(s, t), chunks = (limit + 31) / 32;
                const bool nodes = t == s.tiles - 1;
                const uint32_t sp = tl + TAM_SP0 + (n & 1) * 128;
                if (nodes) {                                         // the ancestors of this row's node
                    unsigned long long l0, l1;
                    bool bad;
                    warp_lines(par0, par1, l0, l1, bad);
                    const unsigned long long x0 = shfl64(l0, node & 31), x1 = shfl64(l1, node & 31);
                    line = real ? (node < 32 ? x0 : x1) : 0;
                }
                if (!warp_wait(AB_SDONE + (n & 1), n >> 1)) { ok = false; break; }
                tc_fence_after_sync();
                if (warp == 0) GDN_TSTAMP(n * 16 + 4);
                // Two passes over the scores, 32 columns at a time in rolled loops: the code of a tile has to stay small (unrolled over the 128
                // columns it drove the producers' and the issuer's code out of the instruction cache, and every step of theirs took
                // hundreds of cycles).  Masked scores are replaced by -inf.
                auto scores = [&](int g, float (&v)[32]) {
                    uint32_t r[32];
                    tmem_ld32(sp + 32 * g, r);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
                    if (nodes || limit < 32 * g + 32) {
                        const uint32_t see = nodes ? (uint32_t)(line >> (32 * g)) : (1u << (limit - 32 * g)) - 1u;
#pragma unroll
                        for (int i = 0; i < 32; i++) v[i] = (see >> i & 1) ? v[i] : -INFINITY;
                    }
                };
                float mt = -INFINITY;
#pragma unroll 1
                for (int g = 0; g < chunks; g++) {
                    float v[32];
                    scores(g, v);
#pragma unroll
                    for (int i = 0; i < 32; i += 4) mt = fmaxf(mt, fmaxf(fmaxf(v[i], v[i + 1]), fmaxf(v[i + 2], v[i + 3])));
                }
                if (warp == 0) GDN_TSTAMP(n * 16 + 5);
                mt *= sc;                                            // (sc > 0: the maximum of the scaled scores)
                // raise the reference only when it is far behind (or not set yet); O is rescaled then -- all lanes take part in the
                // tensor-memory round trip, each with its own factor
                const bool raise = mt > m_run + TA_RAISE || (m_run == -INFINITY && mt != -INFINITY);
                if (__any_sync(0xffffffffu, raise)) {
                    const float m_new = raise ? mt : m_run;
                    const float alpha = (m_run == -INFINITY) ? 0.f : exp2f(m_run - m_new);
                    l_run *= alpha;
                    m_run = m_new;
                    if (t > s.t0) {                                  // O holds the tiles before this one: P V of tile n - 1 must have landed
                        if (!warp_wait(AB_PFREE + ((n - 1) & 1), (n - 1) >> 1)) { ok = false; break; }
                        tc_fence_after_sync();
#pragma unroll 1
                        for (int c0 = 0; c0 < 256; c0 += 32) {
                            uint32_t o[32];
                            tmem_ld32(tl + TAM_O + c0, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                            tmem_st32(tl + TAM_O + c0, o);
                        }
                        tmem_wait_st();
                    }
                }
                __syncwarp();                                        // (each lane chose its own factor; tensor-memory accesses take a converged warp)
                // p = 2^(s sc - m) (a masked score gives 0) as bf16 hi + lo, written over the scores group by group: the 32 score
                // columns of keys 32 g .. 32 g + 31 become 16 columns of hi pairs and 16 columns of lo pairs
                const float nm = (m_run == -INFINITY) ? 0.f : -m_run;
#pragma unroll 1
                for (int g = 0; g < chunks; g++) {
                    float v[32];
                    scores(g, v);
                    uint32_t ph[16], pl[16];
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        float p0, p1;
                        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p0) : "f"(fmaf(v[i], sc, nm)));
                        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p1) : "f"(fmaf(v[i + 1], sc, nm)));
                        l_run += p0 + p1;
                        ph[i >> 1] = pack_bf16x2(p0, p1);
                        pl[i >> 1] = pack_bf16x2(p0 - __uint_as_float(ph[i >> 1] << 16), p1 - __uint_as_float(ph[i >> 1] & 0xffff0000u));
                    }
                    tmem_st16(sp + 32 * g, ph);
                    tmem_st16(sp + 32 * g + 16, pl);
                }
                tmem_wait_st();
                if (warp == 0) GDN_TSTAMP(n * 16 + 6);
                if (nodes) {                                         // warp 7 has made the nodes' value rows ready
                    if (!warp_wait(AB_NODES, node_tiles)) { ok = false; break; }
                    badv = *(volatile unsigned long long*)&s_badv[node_tiles & 1];
                    node_tiles++;
                } else if (limit & 15) {
                    // value rows behind the context are zeroed, up to the next multiple of 16 keys, before the product reads them.  These warps
                    // do not wait for every phase of the V ring, and a parity cannot tell a phase from the one two before: once the
                    // product of the tile before is done, the chunks before this tile's have all been consumed.
                    if (n > 0 && !warp_wait(AB_PFREE + ((n - 1) & 1), (n - 1) >> 1)) { ok = false; break; }
                    const int slot = (nv + chunks - 1) % TA_NV, r0 = limit & 31, r1 = (r0 + 15) & ~15;
                    if (!warp_wait(AB_VFULL + slot, (nv + chunks - 1) / TA_NV)) { ok = false; break; }
#pragma unroll 1
                    for (int i = row; i < (r1 - r0) * 32; i += n_warps * 32) {
                        const int r = r0 + (i >> 5), ch = i & 31;
                        *reinterpret_cast<uint4*>(smem + TA_Q_BYTES + TA_NK * TA_SLOT + slot * TA_SLOT + (ch >> 3) * 4096 + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async_smem();
                }
                nv += chunks;
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(AB_PREADY + (n & 1)));
                if (warp == 0) GDN_TSTAMP(n * 16 + 7);
            }
            if (!ok) break;
            GDN_BSTAMP(nseg == 0 ? 3 : 6);
            // ---- epilogue: O / l, or a partial (m, l, O) where the pair goes on in another block ----
            if (!warp_wait(AB_ODONE, nseg)) break;
            tc_fence_after_sync();
            GDN_BSTAMP(nseg == 0 ? 4 : 7);
            const bool whole = s.n == s.tiles;
            const int slot = 2 * (int)blockIdx.x + (s.t0 == 0 ? 1 : 0);
            float* part = p.part + (size_t)slot * (64 * 4) * p.rows;
            const float inv = l_run == 0.f ? 1.f : 1.f / l_run;
            __nv_bfloat16* orow = a.out + (((size_t)s.b * a.N + node) * a.H + s.kvh * p.group + (row - local * p.group)) * ATT_D;
            const unsigned long long add = line & badv;
#pragma unroll 1
            for (int c0 = 0; c0 < 256; c0 += 32) {
                uint32_t u[32];
                __syncwarp();                                        // (rows add and store different things below; the load takes a converged warp)
                tmem_ld32(tl + TAM_O + c0, u);
                tmem_wait_ld();
                if (add) {
#pragma unroll 1
                    for (unsigned long long r = add; r; r &= r - 1) {
                        const __nv_bfloat16* v = a.v_new + (((size_t)s.b * a.N + (__ffsll((long long)r) - 1)) * a.KV + s.kvh) * ATT_D + c0;
#pragma unroll
                        for (int i = 0; i < 32; i++) {
                            const float f = __bfloat162float(v[i]);
                            if (!isfinite(f)) u[i] = __float_as_uint(__uint_as_float(u[i]) + f);
                        }
                    }
                }
                if (real && whole) {
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        uint4 v;
                        v.x = pack_bf16x2(__uint_as_float(u[i]) * inv, __uint_as_float(u[i + 1]) * inv);
                        v.y = pack_bf16x2(__uint_as_float(u[i + 2]) * inv, __uint_as_float(u[i + 3]) * inv);
                        v.z = pack_bf16x2(__uint_as_float(u[i + 4]) * inv, __uint_as_float(u[i + 5]) * inv);
                        v.w = pack_bf16x2(__uint_as_float(u[i + 6]) * inv, __uint_as_float(u[i + 7]) * inv);
                        if (!line) v = make_uint4(0, 0, 0, 0);       // an unused node
                        *reinterpret_cast<uint4*>(orow + c0 + i) = v;
                    }
                } else if (row < p.rows && !whole) {
                    // partials are stored column group by column group, rows side by side: a warp writes 512 contiguous bytes
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *reinterpret_cast<float4*>(part + ((size_t)((c0 + i) >> 2) * p.rows + row) * 4) =
                            make_float4(__uint_as_float(u[i]), __uint_as_float(u[i + 1]), __uint_as_float(u[i + 2]), __uint_as_float(u[i + 3]));
                }
            }
            if (row < p.rows && !whole) *reinterpret_cast<float2*>(p.part_ml + ((size_t)slot * p.rows + row) * 2) = make_float2(m_run, l_run);
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(AB_OFREE));
            GDN_BSTAMP(nseg == 0 ? 5 : 8);
            if (tid == 0 && s.t0 == 0 && !whole) {
                // the pair that starts in this block and goes on in the next ones is joined by the merge kernel
                int parts = 1;
#pragma unroll 1
                while (range_lo(grp + parts, G, N_all) < hi - s.n + s.tiles) parts++;
                const int pair = (s.b * a.KV + s.kvh) * p.row_tiles + rt;
                *reinterpret_cast<int2*>(p.info + 2 * (p.by_pair ? pair : (int)blockIdx.x)) = make_int2(p.by_pair ? (int)blockIdx.x : pair, parts);
            }
            nseg++;
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (tid == 0 && aborted()) clear_info();                         // (every role is through: what gave up shows)
    if (warp == 4) { __syncwarp(); tmem_dealloc(tb, 512); }          // (one lane of it was the issuer)
    GDN_BSTAMP(9);
}

// Joins the partials of a cut pair (blockIdx.x: the pair, or the main block that it starts in): a thread holds four columns of a row, or of every
// 2nd or 4th partial of it.  Bound: latency (a few hundred KiB out of L2), so what a block needs is requested at once, and where rows are few
// several threads share one: one sequence with 16 k cached tokens and 16 nodes 36 -> 28 us (74 partials a pair, four threads a row), with 64
// nodes 37.5 -> 33.3, four sequences with 8 k 31.3 -> 28.3 (two threads a row).  Sixteen partials in flight a thread leave room for one block
// per SM, six for two: 16 sequences (about 5 partials a pair) 43 us with six, 46 with sixteen; 2 sequences x 64 nodes (18 a pair) 98.5 and 95.6,
// 9 sequences (8 a pair) 27.5 and 25.7.
constexpr int TM_THREADS = 512;
constexpr int TM_FEW = 6, TM_MANY = 16;                              // partials requested at once where pairs have few of them, and many

template <int ROWS, int AHEAD>
__global__ void __launch_bounds__(TM_THREADS) tree_attn_merge_kernel(const __grid_constant__ TreeAttnPlan p) {
    constexpr int GROUPS = TM_THREADS / (64 * ROWS);                 // threads that share a row's columns: each takes every GROUPS-th partial
    __shared__ float s_w[148][ROWS], s_l[148][ROWS];
    __shared__ unsigned char s_live[ROWS];
    __shared__ float4 s_acc[GROUPS][64 * ROWS];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int2 info = *reinterpret_cast<const int2*>(p.info + 2 * blockIdx.x);
    const int first = p.by_pair ? info.x : blockIdx.x, pair = p.by_pair ? blockIdx.x : info.x, parts = info.y;
    GDN_BSTAMP(10);
    if (parts == 0) return;
    const TreeAttnArgs& a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = tid & (ROWS - 1), row = blockIdx.y * ROWS + r, cg = tid / ROWS % 64, grp = tid / (64 * ROWS);
    const bool in = row < p.rows;
    auto slot = [&](int k) -> size_t { return 2 * (first + k * p.row_tiles) + (k == 0 ? 1 : 0); };
    // (requested at once: the rows' (m, l), the first partials and the tree; a dependent round trip to L2 costs most of a microsecond)
    const float4* part = reinterpret_cast<const float4*>(p.part) + (size_t)cg * p.rows + row;
    const size_t step = (size_t)64 * p.rows;                         // float4s of a slot
    float4 o[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; k++)
        if (in && grp + k * GROUPS < parts) o[k] = __ldcg(part + slot(grp + k * GROUPS) * step);
    for (int k = tid / ROWS; k < parts; k += TM_THREADS / ROWS) {
        const float2 ml = in ? __ldcg(reinterpret_cast<const float2*>(p.part_ml + (slot(k) * p.rows + row) * 2)) : make_float2(-INFINITY, 0.f);
        s_w[k][r] = ml.x;
        s_l[k][r] = ml.y;
    }
    const int rt = pair % p.row_tiles, kvh = pair / p.row_tiles % a.KV, b = pair / p.row_tiles / a.KV;
    if (warp == 8) {                                                 // which of the rows belong to nodes in use
        unsigned long long l0, l1;
        bool bad;
        const int* par = a.parents + (size_t)b * a.N;
        warp_lines(lane < a.N ? par[lane] : -2, lane + 32 < a.N ? par[lane + 32] : -2, l0, l1, bad);
        const int node = rt * p.nodes + (blockIdx.y * ROWS + (lane & (ROWS - 1))) / p.group;
        const unsigned long long x0 = shfl64(l0, node & 31), x1 = shfl64(l1, node & 31);
        if (lane < ROWS) s_live[lane] = node < a.N && (node < 32 ? x0 : x1) != 0;
    }
    __syncthreads();
    if (warp < ROWS) {                                               // the row's common maximum; weights over the row's sum
        float mx = -INFINITY, sum = 0.f;
        for (int k = lane; k < parts; k += 32) mx = fmaxf(mx, s_w[k][warp]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        for (int k = lane; k < parts; k += 32) {
            const float m = s_w[k][warp], w = m == -INFINITY ? 0.f : exp2f(m - mx);
            sum = fmaf(w, s_l[k][warp], sum);
            s_w[k][warp] = w;
        }
        sum = warp_sum(sum);
        const float inv = sum == 0.f ? 1.f : 1.f / sum;
        for (int k = lane; k < parts; k += 32) s_w[k][warp] *= inv;
    }
    __syncthreads();
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float w, float4 x) {
        acc.x = fmaf(w, x.x, acc.x); acc.y = fmaf(w, x.y, acc.y); acc.z = fmaf(w, x.z, acc.z); acc.w = fmaf(w, x.w, acc.w);
    };
#pragma unroll
    for (int k = 0; k < AHEAD; k++)
        if (in && grp + k * GROUPS < parts) add(s_w[grp + k * GROUPS][r], o[k]);
    if (in)
#pragma unroll (AHEAD / 2)
        for (int k = grp + AHEAD * GROUPS; k < parts; k += GROUPS) add(s_w[k][r], __ldcg(part + slot(k) * step));
    if (GROUPS > 1) {
        s_acc[grp][cg * ROWS + r] = acc;
        __syncthreads();
        if (grp > 0) return;
#pragma unroll
        for (int g = 1; g < GROUPS; g++) add(1.f, s_acc[g][cg * ROWS + r]);
    }
    const int node = rt * p.nodes + row / p.group;
    if (!in || node >= a.N) return;
    const uint2 v = s_live[r] ? make_uint2(pack_bf16x2(acc.x, acc.y), pack_bf16x2(acc.z, acc.w)) : make_uint2(0, 0);
    *reinterpret_cast<uint2*>(a.out + (((size_t)b * a.N + node) * a.H + kvh * p.group + row % p.group) * ATT_D + 4 * cg) = v;
    GDN_BSTAMP(11);
}

// ---- host side ----
static int tree_sms() {                                               // (at least 8, the largest number of row tiles)
    static int sms[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { cudaGetLastError(); return 148; }
    if (!sms[dev]) {
        int n = 0;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) { cudaGetLastError(); n = 148; }
        sms[dev] = n < 148 ? n : 148;                                // (the merge kernel keeps the weights of at most 148 partials)
    }
    return sms[dev];
}

static void tree_shape(TreeAttnPlan& p, int N, int H, int KV) {
    p.group = H / KV;
    p.nodes = 128 / p.group < N ? 128 / p.group : N;
    p.rows = p.nodes * p.group;
    p.row_tiles = (N + p.nodes - 1) / p.nodes;
    p.q_bufs = p.rows <= 64 ? 2 : 1;                                 // a second Q buffer hides the load between pairs where it fits
    p.q_slab = (p.rows + 7) / 8 * 1024;
}

size_t tree_attn_workspace_bytes(int B, int N, int H, int KV) {
    (void)B;
    TreeAttnPlan p{};
    tree_shape(p, N, H, KV);
    const size_t G = 148;
    return G * 16 + 2 * G * p.rows * (ATT_D + 2) * sizeof(float);
}

// tiles of the longest plan a launch can meet, for contexts up to `cap` rows
long long tree_attn_plan_tiles(int B, int N, int H, int KV, long long cap) {
    TreeAttnPlan p{};
    tree_shape(p, N, H, KV);
    return (long long)(B < TA_MAX_B ? B : TA_MAX_B) * KV * p.row_tiles * ((cap + TA_TK - 1) / TA_TK + 1 + TA_TAIL);
}

typedef CUresult (*TreeEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                 CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static bool tree_map(CUtensorMap* m, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
    static TreeEncodeFn fn = nullptr;
    if (!fn) {
        cudaDriverEntryPointQueryResult qr;
        void* f = nullptr;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &qr) != cudaSuccess || qr != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            return false;
        }
        fn = reinterpret_cast<TreeEncodeFn>(f);
    }
    const cuuint32_t es[5] = {1, 1, 1, 1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static int gcd_of(int x, int y) { while (y) { const int r = x % y; x = y; y = r; } return x; }

static int launch_pdl(const void* fn, dim3 grid, int threads, size_t smem, cudaStream_t st, void** args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 1;
    cudaLaunchKernelExC(&cfg, fn, args);
    return check_launch("tree_attn");
}

int launch_tree_attn(const TreeAttnArgs& all, void* workspace, size_t workspace_bytes, cudaStream_t st) {
    (void)workspace_bytes;
    static bool attr_set[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && !attr_set[dev]) {
        if (cudaFuncSetAttribute(tree_attn_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, TA_SMEM) != cudaSuccess)
            return check_launch("tree_attn smem attribute");
        attr_set[dev] = true;
    }
    for (int b0 = 0; b0 < all.B; b0 += TA_MAX_B) {
        TreeAttnPlan p{};
        p.a = all;
        TreeAttnArgs& a = p.a;
        a.B = all.B - b0 < TA_MAX_B ? all.B - b0 : TA_MAX_B;
        a.q += (size_t)b0 * a.N * a.H * ATT_D; a.out += (size_t)b0 * a.N * a.H * ATT_D;
        a.k_new += (size_t)b0 * a.N * a.KV * ATT_D; a.v_new += (size_t)b0 * a.N * a.KV * ATT_D;
        a.block_table += (size_t)b0 * a.max_pages; a.ctx_len += b0; a.parents += (size_t)b0 * a.N;
        tree_shape(p, a.N, a.H, a.KV);
        p.G = tree_sms() / p.row_tiles * p.row_tiles;
        const int pairs = a.B * a.KV * p.row_tiles;
        p.by_pair = pairs <= p.G;                                    // (fewer merge blocks that find nothing to do: each wave of them costs a microsecond)
        p.info = static_cast<int*>(workspace);
        p.part_ml = reinterpret_cast<float*>(static_cast<char*>(workspace) + 148 * 16);
        p.part = p.part_ml + 2 * 148 * (size_t)p.rows * 2;
        p.k_box = gcd_of(a.page_size, TA_TK);
        p.v_box = gcd_of(a.page_size, 32);
        CUtensorMap tq, tk, tv, tkn, tvn;
        // q, k_new, v_new: (dim, head, row); pages: (64 dims, row, 64-dim block, KV head, page), so that one copy can bring whole rows
        const cuuint64_t row = ATT_D * 2, P = a.page_size;
        const cuuint64_t dq[3] = {ATT_D, (cuuint64_t)a.H, (cuuint64_t)a.B * a.N}, dn[3] = {ATT_D, (cuuint64_t)a.KV, (cuuint64_t)a.B * a.N};
        const cuuint64_t sq[2] = {row, row * a.H}, sn[2] = {row, row * a.KV};
        const cuuint64_t dp[5] = {64, P, 4, (cuuint64_t)a.KV, (cuuint64_t)a.n_pages}, sp[4] = {row, 128, row * P, row * P * a.KV};
        const cuuint32_t bq[3] = {64, (cuuint32_t)p.group, (cuuint32_t)p.nodes}, bkn[3] = {64, 1, 64}, bvn[3] = {64, 1, 32};
        const cuuint32_t bk[5] = {64, (cuuint32_t)p.k_box, 1, 1, 1}, bv[5] = {64, (cuuint32_t)p.v_box, p.v_box == 32 ? 4u : 1u, 1, 1};
        if (!tree_map(&tq, a.q, 3, dq, sq, bq) || !tree_map(&tk, a.k_pages, 5, dp, sp, bk) || !tree_map(&tv, a.v_pages, 5, dp, sp, bv) ||
            !tree_map(&tkn, a.k_new, 3, dn, sn, bkn) || !tree_map(&tvn, a.v_new, 3, dn, sn, bvn)) {
            set_error("gqa_tree_attn: tensor maps could not be made");
            return GDN_E_UNSUPPORTED;
        }
        void* args[] = {&p, &tq, &tk, &tv, &tkn, &tvn};
        int rc = launch_pdl((const void*)tree_attn_kernel, dim3(p.G), TA_THREADS, TA_SMEM, st, args);
        if (rc) return rc;
        void* margs[] = {&p};
        // as few rows a block as leave it an SM of its own; with eight, by the mean number of partials of a pair
        const int eights = pairs * ((p.rows + 7) / 8), rows = eights * 4 <= p.G ? 2 : eights * 2 <= p.G ? 4 : 8;
        const void* merge = rows == 2 ? (const void*)tree_attn_merge_kernel<2, TM_MANY>
                            : rows == 4 ? (const void*)tree_attn_merge_kernel<4, TM_MANY>
                            : p.G > TM_FEW * pairs ? (const void*)tree_attn_merge_kernel<8, TM_MANY> : (const void*)tree_attn_merge_kernel<8, TM_FEW>;
        rc = launch_pdl(merge, dim3(p.by_pair ? pairs : p.G, (p.rows + rows - 1) / rows), TM_THREADS, 0, st, margs);
        if (rc) return rc;
    }
    return GDN_OK;
}

}  // namespace gdn

#ifdef GDN_TIMING
extern "C" __attribute__((visibility("default"))) int gdn_timing_log_tree(long long* out_host, int n) {
    return cudaMemcpyFromSymbol(out_host, gdn::g_tlog, sizeof(long long) * n) == cudaSuccess ? 0 : -5;
}
#endif
