// Speculative decoding with a tree of drafted tokens on the GatedDeltaNet layers: verify, accept, commit.
//
// Node i of a sequence's tree hangs below node parents[i] < i, or (-1) below the last token of the slot; a smaller value marks an
// unused node.  The chained verify (gdn_decode.cu) writes a state snapshot after every token, 1 MiB per layer, node and sequence;
// here nothing is written but y.  The rule S <- g S; d = beta (v - S k); S <- S + d k^T; y = S q unrolled along the path root .. i gives
// a form in which only the state S0 before the tree occurs.  With G_i = the log-decays summed over the path, M_ia = e^(G_i - G_a):
//     u_i = beta_i (v_i - e^G_i S0 k_i) - sum over ancestors a of i:  beta_i M_ia (k_i . k_a) u_a
//     y_i = e^G_i S0 q_i + sum over a in {i, ancestors}:  M_ia (q_i . k_a) u_a
// so the state is read once whatever the tree's size.  After the target has chosen, `commit` advances state and conv window along the
// accepted path, for all layers in one launch.
//
// Conv, silu, norm, gates and the solve stay in fp32 here until y (bf16) or the state (fp32) is stored.  The operands of verify's tensor-core products -- S0, K
// and Q, with 17 nodes and more also u and A -- are each the sum of two bf16 numbers hi + lo (exact to 2^-17), and lo x lo is left out (2^-16 of the
// factors at most).  The single-token and chained kernels round to bf16 after each of these operations as the reference's graph does, so
// results agree with them to bf16 rounding, not bit for bit.
#include <cuda.h>
#include <type_traits>
#include "gdn_common.cuh"
#include "launchers.cuh"
#include "sm100_prims.cuh"

namespace gdn {


__device__ __forceinline__ float log_decay_f(float A_log, float x) { return -expf(A_log) * (fmaxf(x, 0.f) + log1pf(expf(-fabsf(x)))); }
__device__ __forceinline__ float sigmoid_f(float x) { return 1.f / (1.f + expf(-x)); }

// The set {i, ancestors of i} of a tree node as a bit mask, 0 for an unused node.  par: the tree's parents (N of them), already loaded.
// A parent that does not precede its child, or that is unused, makes the node unused and sets `bad`.
__device__ __forceinline__ unsigned long long tree_line(const int* par, int i, bool& bad) {
    unsigned long long line = 0;
    int at = i;
    while (at >= 0) {
        line |= 1ull << at;
        const int p = par[at];
        if (p >= at) { bad = true; return 0; }
        if (p < -1) { bad = at != i; return 0; }                    // (an unused node itself is no mistake, a used one below it is)
        at = p;
    }
    return line;
}

// ----------------------------------------------------------------------------------------------------------------------
// verify: one block per (sequence, head), two blocks per SM.  NP = nodes padded to 16, 32 or 64.  Bound: issue slots and latency
// (some 40 k warp instructions a head at 64 nodes, half of the slots used; the state alone would take a quarter of the time).  Measured: 64
// sequences x 64 nodes 87 us, 16 x 27 16.5 us, one sequence x 8 nodes 9.0 us (states that L2 does not hold).
//     [P1 | P2] = S0 [K; Q]^T     on the tensor cores, rows = value rows d: S0 in tensor memory, [K; Q] in shared memory
//     G         = [K; Q] K^T      on the tensor cores
// each operand as bf16 hi + lo and the three products that matter (what is dropped is 2^-16 of the factors; K and Q rounded to bf16
// alone would put an error of the size of y's own rounding on every product).  The solve is fp32: thread d of four warps solves
//     u_i = beta_i (v_i - e^G_i P1_i) - sum_j L_ij u_j
// for its value row in blocks of 16 nodes.  Up to 16 nodes thread d of the other four follows with
//     y_i = e^G_i P2_i + sum_j A_ij u_j;
// with more, where it would follow block by block, this sum is another product, u and A as hi + lo (when it was made one, 64 sequences x 64
// nodes 86 us against 90, x 32 nodes 52.8 against 54.1, one sequence x 32 nodes 11.1 either way).  L and A are dense with zeros outside the
// ancestors; zeros do not stop NaN, so a head with a non-finite q, k, v or gate takes the sums over the ancestors one by one instead, and y's rows of
// unused nodes are selected, whatever the state holds.
// M_ij is 2 to the difference of two sums G, which can be far larger than their difference (a path through tokens that wipe the state out).
// G is summed in 64 bits and split into hi = fp32(G) and lo; with u'_i = 2^-lo_i u_i in place of u the solve needs 2^(hi_i - hi_j) only, and
// lo enters factors of single nodes: beta_i 2^-lo_i on v, 2^lo_i on A's row.
// Shared memory: [K; Q] hi and lo (1 KiB a node), later L and A; a region that receives the state (two halves of 32 KiB where
// NP = 64, so that two blocks fit an SM) and then holds v and u.
// ----------------------------------------------------------------------------------------------------------------------
using namespace sm100;

constexpr int TV_THREADS = 256;
constexpr float LOG2E = 1.4426950408889634f, TV_WIPED = -160.f;      // 2^-160 is below the smallest fp32 number
// Waits of verify that gave up.  A copy or product is only issued when the waits before it were not among them (as seen behind a barrier, so that
// all threads see the same); y is unspecified then, and the block leaves when what was issued is over.
enum { FAIL_STATE0 = 1, FAIL_STATE1 = 2, FAIL_PRODUCT = 4, FAIL_Y = 8 };
template <int NP> struct TreeVerify {
    static constexpr int HALVES = NP == 64 ? 2 : 1;                  // pieces the state arrives in
    static constexpr int SLAB = 2 * NP * 128;                        // bytes of 64 dims of [K; Q]
    static constexpr int KQ_BYTES = 4 * SLAB;                        // hi (two slabs), lo
    static constexpr int ST_BYTES = 65536 / HALVES;
    static constexpr int SMEM = KQ_BYTES + ST_BYTES + DV * 4;        // + a row of zeros behind the last u
    static constexpr uint32_t TM_HI = 0, TM_LO = 64, TM_P = 128, TM_G = 0;       // G replaces S0 (products of one thread run in order)
    static constexpr bool Y_MMA = NP >= 32;                          // y's sums on the tensor cores
    static constexpr int A_LO = NP * 128;                            // (A as operand: hi, then lo)
    static constexpr uint32_t TM_UHI = 0, TM_ULO = 32, TM_Y = 64;    // u and y replace G and the rest of S0
};

__device__ __forceinline__ void split_bf16(float x, float y, uint32_t& hi, uint32_t& lo) {
    hi = pack_bf16x2(x, y);
    lo = pack_bf16x2(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xffff0000u));
}

// two fp32 fused multiply-adds in one instruction (sm_100): x += a * b on both halves
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float x, float y) { f32x2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y)); return r; }
__device__ __forceinline__ float2 unpack2(f32x2 v) { float2 r; asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v)); return r; }
__device__ __forceinline__ void fma2(f32x2& x, f32x2 a, f32x2 b) { asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(x) : "l"(a), "l"(b)); }
// The documented errors of the fast exp, 2 + 1.173 |x| ulp, and of the fast division, 2 ulp, make 2^-18 of the value up to |x| = 40 (below -40 the value is
// smaller than 2^-52), a thousandth of y's rounding to bf16.
__device__ __forceinline__ float silu_fast(float x) { return __fdividef(x, 1.f + __expf(-x)); }

__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}

template <int NP>
__global__ void __launch_bounds__(TV_THREADS, 2) tree_verify_kernel(const TreeDeltaArgs a, const __grid_constant__ CUtensorMap tmS) {
    using C = TreeVerify<NP>;
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ uint64_t bars[2];                                     // state landed; products done
    __shared__ unsigned long long s_line[NP];
    __shared__ int s_par[NP];
    __shared__ __align__(16) const __nv_bfloat16* s_row[NP][4];      // conv rows of a node: t-3 .. t along its path
    __shared__ float s_lg[NP], s_beta[NP];
    __shared__ __align__(16) float s_G[NP], s_grow[NP], s_bgrow[NP];  // G (log2), rounded to fp32; e^G; beta 2^(G rounded)
    __shared__ float s_up[NP], s_bdown[NP];                          // with lo = what the rounding of G dropped: 2^lo; beta 2^-lo
    __shared__ __align__(4) unsigned char s_list[NP / 16][NP];       // per block of 16 nodes: their ancestors in earlier blocks,
    __shared__ int s_cnt[NP / 16];                                   // in fours (filled up with NP, the row of zeros)
    __shared__ uint32_t s_tmem;
    __shared__ int s_odd, s_fail;                                    // a non-finite value in this head; waits that gave up (FAIL_*)
    const int N = a.N, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int b = blockIdx.x / HV, h = blockIdx.x % HV;
    const uint32_t sKQ = smem_addr(smem), sST = sKQ + C::KQ_BYTES;
    const uint32_t b_state = smem_addr(&bars[0]), b_mma = smem_addr(&bars[1]);
    if (sKQ & 1023u) { if (tid == 0) atomicExch(a.status, 4); return; }
    GDN_BSTAMP(0);
    // every row of the tree is first touched in the conv, a few rows at a time: asked for now, they come out of L2 then
    for (int k = tid; k < N * 6; k += TV_THREADS) {
        const __nv_bfloat16* line = a.proj + ((size_t)b * N + k / 6) * a.row_stride + (k % 6 >> 1) * KD + h * DK + (k & 1) * 64;
        asm volatile("prefetch.global.L2 [%0];" ::"l"(line));
    }
    // everything that only needs the block's own numbers, in one round of loads
    const int slot = a.slots[b], pos = a.pos[b];
    const int par = tid < N ? a.parents[(size_t)b * N + tid] : -2;
    float lg = 0.f, beta = 0.f;
    if (tid < N) {
        const __nv_bfloat16* row = a.proj + ((size_t)b * N + tid) * a.row_stride;
        const __nv_bfloat16 rb = row[CD + KD + h], ra = row[CD + KD + HV + h];
        const float A_log = a.A_log[h], dt_bias = a.dt_bias[h];
        beta = sigmoid_f(__bfloat162float(rb));
        lg = log_decay_f(A_log, __bfloat162float(ra) + dt_bias) * LOG2E;
        if (lg < TV_WIPED) lg = TV_WIPED;                            // (the decay is zero in fp32 either way; sums stay in range; NaN passes)
    }
    if (slot < 0 || slot >= a.n_slots || pos < 0) {                  // rows of a bad sequence: zeros
        if (tid == 0) atomicExch(a.status, 1);
        for (int i = tid; i < N * DV; i += TV_THREADS) a.y[((size_t)b * N + i / DV) * KD + h * DV + i % DV] = __float2bfloat16_rn(0.f);
        return;
    }
    auto load_state = [&](int half) {                                // two (or all four) boxes of 32 key columns
        constexpr int BOXES = 4 / C::HALVES;
        mbar_expect_tx(b_state, BOXES * 16384);
        for (int k = 0; k < BOXES; k++) tma_load_2d(sST + k * 16384, &tmS, b_state, 32 * (half * BOXES + k), (slot * HV + h) * DV);
    };
    if (tid == 0) {
        mbar_init(b_state, 1); mbar_init(b_mma, 1);
        s_odd = s_fail = 0;
        fence_barrier_init();
        load_state(0);
    }
    // (tensor memory is allocated, read and written by converged warps: wherever lanes may have parted before, they meet first)
    if (warp == 7) { __syncwarp(); tmem_alloc(smem_addr(&s_tmem), 256); tmem_relinquish(); }
    if (tid < NP) { s_par[tid] = par; s_lg[tid] = lg; }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tb = s_tmem;
    if (tid < NP) {
        bool bad = false;
        const unsigned long long line = tid < N ? tree_line(s_par, tid, bad) : 0;
        if (bad) atomicExch(a.status, 1);
        double sum = 0.;
        for (unsigned long long m = line; m; m &= m - 1) sum += s_lg[__ffsll((long long)m) - 1];
        const float g = (float)sum;
        s_line[tid] = line;
        s_beta[tid] = beta;
        const float lo = (float)(sum - g), up = exp2f(lo), e = exp2f(g);
        s_G[tid] = g;
        s_up[tid] = up;
        s_bdown[tid] = line ? __fdividef(beta, up) : 0.f;
        s_grow[tid] = line ? e * up : 0.f;
        s_bgrow[tid] = line ? beta * e : 0.f;
        if (line && !(isfinite(g) && isfinite(beta))) s_odd = 1;
    } else if (tid < 2 * NP) {                                       // (two threads a node: the one above and this one)
        const int i = tid - NP;
        const __nv_bfloat16* window = a.conv_pool + ((size_t)slot * 2 + (pos & 1)) * 3 * CD;
        for (int t = 3, e = 3 + i; t >= 0; t--) {                    // e: 0..2 the window, 3 + j node j
            s_row[i][t] = i >= N ? window : e >= 3 ? a.proj + ((size_t)b * N + e - 3) * a.row_stride : window + (size_t)e * CD;
            e = e >= 3 ? (s_par[e - 3] >= 0 && s_par[e - 3] < e - 3 ? 3 + s_par[e - 3] : 2) : e - 1;
        }
    }
    __syncthreads();
    GDN_BSTAMP(1);
    if (warp >= 8 - NP / 16) {                                       // the lists, one block of nodes per warp
        const int I = warp - (8 - NP / 16);
        unsigned long long rel = 0;
        for (int i = 0; i < 16; i++) rel |= s_line[16 * I + i];
        rel &= (1ull << (16 * I)) - 1;
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int j = lane + 32 * k;
            if (j < NP && (rel >> j & 1)) s_list[I][__popcll(rel & ((1ull << j) - 1))] = (unsigned char)j;
        }
        const int cnt = __popcll(rel);
        if (lane < 3 && cnt + lane < NP) s_list[I][cnt + lane] = NP;
        if (lane == 0) s_cnt[I] = cnt;
    }
    // ---- conv over the path, silu, norm: a node per warp, four channels per lane, two nodes' loads in flight; GROUPS = 2: q and k,
    //      1: v ----
    auto front = [&](auto first_group, auto groups, auto&& put) {
        constexpr int G0 = decltype(first_group)::value, GROUPS = decltype(groups)::value;
        const int ch = h * DK + 4 * lane;
        f32x2 w[GROUPS][4][2];                                       // taps of channels 0, 1 and of 2, 3
#pragma unroll
        for (int g = 0; g < GROUPS; g++) {
            float f[4][4];
#pragma unroll
            for (int c = 0; c < 4; c++) unpack_bf16x4(*reinterpret_cast<const uint2*>(a.conv_w + (size_t)((G0 + g) * KD + ch + c) * 4), f[c]);
#pragma unroll
            for (int k = 0; k < 4; k++) { w[g][k][0] = pack2(f[0][k], f[1][k]); w[g][k][1] = pack2(f[2][k], f[3][k]); }
        }
        uint2 raw[2][GROUPS][4];
        auto fetch = [&](int i0) {
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const __nv_bfloat16* row = s_row[i0 + 8 * n][k] + ch;
#pragma unroll
                    for (int g = 0; g < GROUPS; g++) raw[n][g][k] = *reinterpret_cast<const uint2*>(row + (G0 + g) * KD);
                }
        };
        fetch(warp);
#pragma unroll 1
        for (int i0 = warp; i0 < NP; i0 += 16) {
            f32x2 sum[2][GROUPS][2];
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int g = 0; g < GROUPS; g++) {
                    sum[n][g][0] = sum[n][g][1] = 0;
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint2 r = raw[n][g][k];
                        fma2(sum[n][g][0], pack2(__uint_as_float(r.x << 16), __uint_as_float(r.x & 0xffff0000u)), w[g][k][0]);
                        fma2(sum[n][g][1], pack2(__uint_as_float(r.y << 16), __uint_as_float(r.y & 0xffff0000u)), w[g][k][1]);
                    }
                }
            if (i0 + 16 < NP) fetch(i0 + 16);                        // (arrive during what follows)
            float x[2][GROUPS][4], ss[2 * GROUPS];
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const bool on = s_line[i0 + 8 * n] != 0;
#pragma unroll
                for (int g = 0; g < GROUPS; g++) {
                    const float2 a0 = unpack2(sum[n][g][0]), a1 = unpack2(sum[n][g][1]);
                    float (&y)[4] = x[n][g];
                    y[0] = on ? silu_fast(a0.x) : 0.f; y[1] = on ? silu_fast(a0.y) : 0.f;
                    y[2] = on ? silu_fast(a1.x) : 0.f; y[3] = on ? silu_fast(a1.y) : 0.f;
                    ss[n * GROUPS + g] = (y[0] * y[0] + y[1] * y[1]) + (y[2] * y[2] + y[3] * y[3]);
                    if (!(ss[n * GROUPS + g] < INFINITY)) s_odd = 1;
                }
            }
            if (G0 == 0) {
                // the four sums over the warp in seven shuffles: each quarter of the lanes ends up with one of them
                const bool up = lane & 16, odd = lane & 8;
                const float t0 = (up ? ss[1] : ss[0]) + __shfl_xor_sync(0xffffffffu, up ? ss[0] : ss[1], 16);
                const float t1 = (up ? ss[2 * GROUPS - 1] : ss[2 * GROUPS - 2]) + __shfl_xor_sync(0xffffffffu, up ? ss[2 * GROUPS - 2] : ss[2 * GROUPS - 1], 16);
                float q = (odd ? t1 : t0) + __shfl_xor_sync(0xffffffffu, odd ? t0 : t1, 8);
                q += __shfl_xor_sync(0xffffffffu, q, 4);
                q += __shfl_xor_sync(0xffffffffu, q, 2);
                q += __shfl_xor_sync(0xffffffffu, q, 1);
                const float r = rsqrtf(q + 1e-6f);                   // lanes 0-7: node 0 q, 16-23: node 0 k, 8-15: node 1 q, 24-31: node 1 k
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int g = 0; g < GROUPS; g++) {
                        const float scale = __shfl_sync(0xffffffffu, r, 16 * g + 8 * n) * (g == 0 ? 0.08838834764831845f : 1.f);
#pragma unroll
                        for (int c = 0; c < 4; c++) x[n][g][c] *= scale;
                    }
            }
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int g = 0; g < GROUPS; g++) put(g, i0 + 8 * n, x[n][g]);
        }
    };
    // (a warp's nodes are 8 apart, so the swizzle of its rows is one)
    const uint32_t put_at = (lane >> 4) * C::SLAB + ((((lane >> 1) & 7) ^ warp) << 4) + (lane & 1) * 8;
    auto put_kq = [&](int row, const float (&x)[4]) {                // rows 0 .. NP - 1: K, then Q
        uint2 hi, lo;
        split_bf16(x[0], x[1], hi.x, lo.x);
        split_bf16(x[2], x[3], hi.y, lo.y);
        const uint32_t at = put_at + row * 128;
        *reinterpret_cast<uint2*>(smem + at) = hi;
        *reinterpret_cast<uint2*>(smem + 2 * C::SLAB + at) = lo;
    };
    front(std::integral_constant<int, 0>(), std::integral_constant<int, 2>(), [&](int g, int i, const float (&x)[4]) { put_kq((g == 0 ? NP : 0) + i, x); });
    GDN_BSTAMP(2);
    fence_proxy_async_smem();
    // ---- the state into tensor memory as hi + lo: lane = value row, warps 0-3 and 4-7 take every other box of 32 key columns ----
    const uint32_t tl = tb + ((uint32_t)((warp & 3) * 32) << 16);
    const int d = (warp & 3) * 32 + lane;
    auto gave_up = [&](int which) { atomicOr(&s_fail, which); atomicExch(a.status, 2); };
    bool whole = C::HALVES == 1;                                     // the last piece of the state is on its way
#pragma unroll 1
    for (int k = 0; k < 2; k++) {
        const int box = 2 * k + (warp >> 2);
        if (k == 0) { if (!mbar_wait(b_state, 0)) gave_up(FAIL_STATE0); }
        else if (C::HALVES == 2 && whole) { if (!mbar_wait(b_state, 1)) gave_up(FAIL_STATE1); }
        __syncwarp();                                                // (lanes poll on their own)
        const unsigned char* src = smem + C::KQ_BYTES + (C::HALVES == 2 ? box & 1 : box) * 16384 + d * 128;
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int c = 0; c < 8; c++) {
            const float4 s = *reinterpret_cast<const float4*>(src + ((c ^ (d & 7)) << 4));
            split_bf16(s.x, s.y, hi[2 * c], lo[2 * c]);
            split_bf16(s.z, s.w, hi[2 * c + 1], lo[2 * c + 1]);
        }
        tmem_st16(tl + C::TM_HI + 16 * box, hi);
        tmem_st16(tl + C::TM_LO + 16 * box, lo);
        if (k == 0 && C::HALVES == 2) {
            __syncthreads();                                         // the first half has been read
            whole = !(s_fail & FAIL_STATE0);
            if (tid == 0 && whole) load_state(1);
        }
    }
    tmem_wait_st();
    tc_fence_before_sync();
    __syncthreads();
    GDN_BSTAMP(3);
    const bool product = !(s_fail & (FAIL_STATE0 | FAIL_STATE1));
    if (tid == TV_THREADS - 32 && product) {
        tc_fence_after_sync();
        constexpr uint32_t HI = smem_desc_hi_sw128(1024);
        constexpr uint32_t I_P = idesc_bf16(128, 2 * NP, 0, 0), I_G = idesc_bf16(128, NP, 0, 0);
        const uint32_t kq = smem_desc_lo(sKQ, 16);
#pragma unroll
        for (int ks = 0; ks < 8; ks++) {
            const uint32_t bh = kq + (ks >> 2) * (C::SLAB >> 4) + (ks & 3) * 2, bl = bh + 2 * (C::SLAB >> 4);
            if (ks == 0) mma_ts_w<false>(tb + C::TM_P, tb + C::TM_HI, bh, HI, I_P);
            else mma_ts_w<true>(tb + C::TM_P, tb + C::TM_HI + 8 * ks, bh, HI, I_P);
            mma_ts_w<true>(tb + C::TM_P, tb + C::TM_HI + 8 * ks, bl, HI, I_P);
            mma_ts_w<true>(tb + C::TM_P, tb + C::TM_LO + 8 * ks, bh, HI, I_P);
        }
#pragma unroll
        for (int ks = 0; ks < 8; ks++) {
            const uint32_t xh = kq + (ks >> 2) * (C::SLAB >> 4) + (ks & 3) * 2, xl = xh + 2 * (C::SLAB >> 4);
            if (ks == 0) mma_ss_w<false>(tb + C::TM_G, xh, HI, xh, HI, I_G);
            else mma_ss_w<true>(tb + C::TM_G, xh, HI, xh, HI, I_G);
            mma_ss_w<true>(tb + C::TM_G, xh, HI, xl, HI, I_G);
            mma_ss_w<true>(tb + C::TM_G, xl, HI, xh, HI, I_G);
        }
        mma_commit(b_mma);
    }
    GDN_BSTAMP(4);
    float* su = reinterpret_cast<float*>(smem + C::KQ_BYTES);        // [NP][128]: v, then u
    front(std::integral_constant<int, 2>(), std::integral_constant<int, 1>(), [&](int, int i, const float (&x)[4]) {
        const float m = s_bdown[i];
        *reinterpret_cast<float4*>(su + i * DV + 4 * lane) = s_line[i] ? make_float4(m * x[0], m * x[1], m * x[2], m * x[3]) : make_float4(0.f, 0.f, 0.f, 0.f);
    });
    if (tid < DV) su[NP * DV + tid] = 0.f;
    GDN_BSTAMP(5);
    if (product && !mbar_wait(b_mma, 0)) gave_up(FAIL_PRODUCT);
    __syncwarp();
    tc_fence_after_sync();
    GDN_BSTAMP(6);
    // ---- L[j][i] = beta_i M_ij (k_i . k_j) and A[j][i] = M_ij (q_i . k_j), j along rows, so that a thread reads them for four i at a time ----
    float* sL = reinterpret_cast<float*>(smem);
    float* sA = sL + NP * NP;
    if (d < 2 * NP) {
        const bool isq = d >= NP;
        const int i = isq ? d - NP : d;
        const unsigned long long line = isq ? s_line[i] : s_line[i] & ~(1ull << i);
        const float g = s_G[i], mul = isq ? s_up[i] : s_beta[i];
        float* dst = (isq ? sA : sL) + i;
        unsigned char* arow = reinterpret_cast<unsigned char*>(sA) + i * 128;        // Y_MMA: A's rows as operand images, hi and lo
        for (int j0 = (warp >> 2) * 16; j0 < NP; j0 += 32) {
            uint32_t r[16];
            __syncwarp();
            tmem_ld16(tl + C::TM_G + j0, r);
            tmem_wait_ld();
            const uint32_t on = (uint32_t)(line >> j0);
            float m[16];
#pragma unroll
            for (int c = 0; c < 16; c++) {
                float e;
                asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g - s_G[j0 + c]));
                m[c] = on >> c & 1 ? mul * e * __uint_as_float(r[c]) : 0.f;
            }
            if (C::Y_MMA && isq) {
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    uint4 hi, lo;
                    split_bf16(m[8 * q], m[8 * q + 1], hi.x, lo.x);
                    split_bf16(m[8 * q + 2], m[8 * q + 3], hi.y, lo.y);
                    split_bf16(m[8 * q + 4], m[8 * q + 5], hi.z, lo.z);
                    split_bf16(m[8 * q + 6], m[8 * q + 7], hi.w, lo.w);
                    const int at = ((j0 / 8 + q) ^ (i & 7)) << 4;
                    *reinterpret_cast<uint4*>(arow + at) = hi;
                    *reinterpret_cast<uint4*>(arow + C::A_LO + at) = lo;
                }
            } else {
#pragma unroll
                for (int c = 0; c < 16; c++) dst[(j0 + c) * NP] = m[c];
            }
        }
    }
    if (C::Y_MMA) fence_proxy_async_smem();
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    GDN_BSTAMP(7);
    const bool solver = warp < 4;
    __nv_bfloat16* out = a.y + (size_t)b * N * KD + h * DV + d;
    const bool plain = !s_odd, y_product = C::Y_MMA && plain && product && !(s_fail & FAIL_PRODUCT);
    // which of the 32 nodes from i0 on are in use: the sums of the others are zeros times whatever the state holds, and 0 x NaN is NaN
    auto used_from = [&](int i0) -> uint32_t { return __ballot_sync(0xffffffffu, i0 + lane < NP && s_line[i0 + lane < NP ? i0 + lane : 0]); };
    if (plain) {
#pragma unroll 1
        for (int I = 0; I < NP / 16; I++) {
            if (C::Y_MMA && !solver) break;
            f32x2 x[8];                                              // nodes 16 I + 2 k, + 1
            {
                uint32_t r[16];
                tmem_ld16(tl + C::TM_P + (solver ? 0 : NP) + 16 * I, r);
                tmem_wait_ld();
                const float4* grow = reinterpret_cast<const float4*>((solver ? s_bgrow : s_grow) + 16 * I);
                float f[16];
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const float4 m = grow[q];
                    f[4 * q] = m.x * __uint_as_float(r[4 * q]); f[4 * q + 1] = m.y * __uint_as_float(r[4 * q + 1]);
                    f[4 * q + 2] = m.z * __uint_as_float(r[4 * q + 2]); f[4 * q + 3] = m.w * __uint_as_float(r[4 * q + 3]);
                }
                if (solver)
#pragma unroll
                    for (int c = 0; c < 16; c++) f[c] = su[(16 * I + c) * DV + d] - f[c];
#pragma unroll
                for (int k = 0; k < 8; k++) x[k] = pack2(f[2 * k], f[2 * k + 1]);
            }
            const float* coef = (solver ? sL : sA) + 16 * I;
            const float sign = solver ? -1.f : 1.f;
            auto add = [&](int j, float u) {                         // x += coef[j] u
                const ulonglong2* row = reinterpret_cast<const ulonglong2*>(coef + (j & (NP - 1)) * NP);      // (NP, with u = 0: any row)
                const f32x2 uu = pack2(u, u);
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const ulonglong2 m = row[q];
                    fma2(x[2 * q], m.x, uu);
                    fma2(x[2 * q + 1], m.y, uu);
                }
            };
            // nodes of earlier blocks, only those that are an ancestor of one of these, four at a time
            for (int k = 0; k < s_cnt[I]; k += 4) {
                const uint32_t js = *reinterpret_cast<const uint32_t*>(&s_list[I][k]);
                float u[4];
#pragma unroll
                for (int q = 0; q < 4; q++) u[q] = sign * su[(js >> 8 * q & 255) * DV + d];
#pragma unroll
                for (int q = 0; q < 4; q++) add(js >> 8 * q & 255, u[q]);
            }
            if (solver) {
                float us[16];
#pragma unroll
                for (int c = 0; c < 16; c++) {                       // (entries up to c are zero)
                    const float2 p = unpack2(x[c / 2]);
                    const float u = c & 1 ? p.y : p.x;
                    us[c] = u;
                    su[(16 * I + c) * DV + d] = u;
                    const f32x2 uu = pack2(-u, -u);
                    const ulonglong2* row = reinterpret_cast<const ulonglong2*>(coef + (16 * I + c) * NP);
#pragma unroll
                    for (int q = c / 4; q < 4; q++) {
                        const ulonglong2 m = row[q];
                        if (4 * q + 1 > c) fma2(x[2 * q], m.x, uu);
                        if (4 * q + 3 > c) fma2(x[2 * q + 1], m.y, uu);
                    }
                }
                if (C::Y_MMA) {
                    uint32_t hi[8], lo[8];
#pragma unroll
                    for (int q = 0; q < 8; q++) split_bf16(us[2 * q], us[2 * q + 1], hi[q], lo[q]);
                    tmem_st8(tl + C::TM_UHI + 8 * I, hi);
                    tmem_st8(tl + C::TM_ULO + 8 * I, lo);
                } else {
                    __threadfence_block();
                    asm volatile("bar.arrive %0, 256;" ::"r"(1 + I) : "memory");
                }
            } else {
                asm volatile("bar.sync %0, 256;" ::"r"(1 + I) : "memory");
                const uint32_t used = used_from(16 * I);
#pragma unroll
                for (int c = 0; c < 16; c++) {                       // (entries before c are zero)
                    const float u = su[(16 * I + c) * DV + d];
                    const f32x2 uu = pack2(u, u);
                    const ulonglong2* row = reinterpret_cast<const ulonglong2*>(coef + (16 * I + c) * NP);
#pragma unroll
                    for (int q = c / 4; q < 4; q++) {
                        const ulonglong2 m = row[q];
                        fma2(x[2 * q], m.x, uu);
                        fma2(x[2 * q + 1], m.y, uu);
                    }
                }
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const float2 v = unpack2(x[k]);
                    if (16 * I + 2 * k < N) out[(size_t)(16 * I + 2 * k) * KD] = __float2bfloat16_rn(used >> 2 * k & 1 ? v.x : 0.f);
                    if (16 * I + 2 * k + 1 < N) out[(size_t)(16 * I + 2 * k + 1) * KD] = __float2bfloat16_rn(used >> (2 * k + 1) & 1 ? v.y : 0.f);
                }
            }
        }
        if constexpr (C::Y_MMA) {
            // y = e^G P2 + U A^T, rows = value rows: u as hi + lo out of tensor memory, A as hi + lo out of shared memory
            constexpr int MINE = NP / 2;                             // nodes whose y this warp's group writes
            auto load = [&](uint32_t col, uint32_t (&r)[MINE]) {
                if constexpr (MINE == 32) tmem_ld32(tl + col, r);
                else tmem_ld16(tl + col, r);
                tmem_wait_ld();
            };
            float f[MINE];
            uint32_t r[MINE];
            const int i0 = MINE * (warp >> 2);
            const uint32_t used = used_from(i0);
            load(C::TM_P + NP + i0, r);
#pragma unroll
            for (int c = 0; c < MINE; c++) f[c] = s_grow[i0 + c] * __uint_as_float(r[c]);
            tmem_wait_st();
            tc_fence_before_sync();
            __syncthreads();
            if (tid == TV_THREADS - 32 && y_product) {
                tc_fence_after_sync();
                constexpr uint32_t HI = smem_desc_hi_sw128(1024), I_Y = idesc_bf16(128, NP, 0, 0);
                const uint32_t ah = smem_desc_lo(sKQ + NP * NP * 4, 16), al = ah + (C::A_LO >> 4);
#pragma unroll
                for (int ks = 0; ks < NP / 16; ks++) {
                    if (ks == 0) mma_ts_w<false>(tb + C::TM_Y, tb + C::TM_UHI, ah, HI, I_Y);
                    else mma_ts_w<true>(tb + C::TM_Y, tb + C::TM_UHI + 8 * ks, ah + 2 * ks, HI, I_Y);
                    mma_ts_w<true>(tb + C::TM_Y, tb + C::TM_UHI + 8 * ks, al + 2 * ks, HI, I_Y);
                    mma_ts_w<true>(tb + C::TM_Y, tb + C::TM_ULO + 8 * ks, ah + 2 * ks, HI, I_Y);
                }
                mma_commit(b_mma);
            }
            if (y_product && !mbar_wait(b_mma, 1)) gave_up(FAIL_Y);
            __syncwarp();
            tc_fence_after_sync();
            load(C::TM_Y + i0, r);
#pragma unroll
            for (int c = 0; c < MINE; c++)
                if (i0 + c < N) out[(size_t)(i0 + c) * KD] = __float2bfloat16_rn(used >> c & 1 ? f[c] + __uint_as_float(r[c]) : 0.f);
        }
    } else if (solver) {
        // A's entries: as they are, or from their operand images (of a non-finite one hi alone)
        auto coef_a = [&](int j, int i) -> float {
            if (!C::Y_MMA) return sA[j * NP + i];
            const unsigned char* at = reinterpret_cast<const unsigned char*>(sA) + i * 128 + (((j >> 3) ^ (i & 7)) << 4) + (j & 7) * 2;
            const float hi = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(at)), lo = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(at + C::A_LO));
            return isfinite(hi) ? hi + lo : hi;
        };
        // a non-finite value somewhere: only what lies on a node's own path enters its sums
        for (int i0 = 0; i0 < NP; i0 += 16) {
            uint32_t r1[16], r2[16];
            __syncwarp();
            tmem_ld16(tl + C::TM_P + i0, r1);
            tmem_ld16(tl + C::TM_P + NP + i0, r2);
            tmem_wait_ld();
            for (int c = 0; c < 16 && i0 + c < N; c++) {
                const int i = i0 + c;
                float p1 = 0.f, p2 = 0.f;
#pragma unroll
                for (int k = 0; k < 16; k++) if (k == c) { p1 = __uint_as_float(r1[k]); p2 = __uint_as_float(r2[k]); }
                const unsigned long long line = s_line[i];
                const float grow = s_grow[i];
                float u = su[i * DV + d] - s_bgrow[i] * p1, y = grow * p2;
                for (unsigned long long m = line & ~(1ull << i); m; m &= m - 1) {
                    const int j = __ffsll((long long)m) - 1;
                    u = fmaf(-sL[j * NP + i], su[j * DV + d], u);
                    y = fmaf(coef_a(j, i), su[j * DV + d], y);
                }
                y = fmaf(coef_a(i, i), u, y);
                su[i * DV + d] = u;                                  // (column d is this thread's)
                out[(size_t)i * KD] = __float2bfloat16_rn(line ? y : 0.f);
            }
        }
    }
    GDN_BSTAMP(8);
    tc_fence_before_sync();
    __syncthreads();
    GDN_BSTAMP(9);
    if (s_fail && tid == 0) {                                        // copies and products in flight end first
        mbar_wait(b_state, C::HALVES == 2 && whole, DRAIN_POLLS);
        if (product) mbar_wait(b_mma, y_product, DRAIN_POLLS);
    }
    __syncthreads();
    if (warp == 7) { __syncwarp(); tmem_dealloc(tb, 256); }
}

typedef CUresult (*StateEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                  CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// the pool as rows of 128 fp32 key columns; box = 32 columns x the 128 value rows of a head
static bool state_map(CUtensorMap* m, const float* pool, int n_slots) {
    static StateEncodeFn fn = nullptr;
    if (!fn) {
        cudaDriverEntryPointQueryResult qr;
        void* f = nullptr;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &qr) != cudaSuccess || qr != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            return false;
        }
        fn = reinterpret_cast<StateEncodeFn>(f);
    }
    const cuuint64_t dims[2] = {DK, (cuuint64_t)n_slots * HV * DV}, strides[1] = {DK * 4};
    const cuuint32_t box[2] = {32, DV}, es[2] = {1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, const_cast<float*>(pool), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int NP>
static int run_tree_verify(const TreeDeltaArgs& a, const CUtensorMap& tm, cudaStream_t st) {
    static bool attr_set[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && !attr_set[dev]) {
        if (cudaFuncSetAttribute(tree_verify_kernel<NP>, cudaFuncAttributeMaxDynamicSharedMemorySize, TreeVerify<NP>::SMEM) != cudaSuccess)
            return check_launch("tree_verify smem attribute");
        attr_set[dev] = true;
    }
    tree_verify_kernel<NP><<<a.B * HV, TV_THREADS, TreeVerify<NP>::SMEM, st>>>(a, tm);
    return check_launch("tree_verify");
}

int launch_tree_verify(const TreeDeltaArgs& a, cudaStream_t st) {
    if (a.B <= 0 || a.N <= 0) return GDN_OK;
    CUtensorMap tm;
    if (!state_map(&tm, a.ssm_pool, a.n_slots)) {
        set_error("gdn_tree_verify: the state's tensor map could not be made");
        return GDN_E_UNSUPPORTED;
    }
    if (a.N <= 16) return run_tree_verify<16>(a, tm, st);
    if (a.N <= 32) return run_tree_verify<32>(a, tm, st);
    return run_tree_verify<64>(a, tm, st);
}

// ----------------------------------------------------------------------------------------------------------------------
// accept: one warp per sequence walks from the first root to the first child that carries the token the target chose.  Bound: latency (a ballot
// and two shuffles a step); 24 sequences x 32 nodes 2.2 us.
// ----------------------------------------------------------------------------------------------------------------------
__global__ void tree_accept_kernel(const int* __restrict__ parents, const int* __restrict__ toks, const int* __restrict__ ids, int* __restrict__ path,
                                   int* __restrict__ n_path, int* status, int B, int N) {
    const int b = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (b >= B) return;
    const size_t o = (size_t)b * N;
    int par[2], tok[2], id[2];                                       // nodes lane and lane + 32
    bool bad = false;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int i = lane + 32 * k;
        par[k] = i < N ? parents[o + i] : -2;
        tok[k] = i < N ? toks[o + i] : 0;
        id[k] = i < N ? ids[o + i] : 0;
        if (par[k] >= i) { bad = true; par[k] = -2; }                // a parent has to precede its child
    }
    const uint32_t used0 = __ballot_sync(0xffffffffu, par[0] >= -1), used1 = __ballot_sync(0xffffffffu, par[1] >= -1);
    const unsigned long long used = used0 | (unsigned long long)used1 << 32;
#pragma unroll
    for (int k = 0; k < 2; k++) bad = bad || (par[k] >= 0 && !(used >> par[k] & 1));
    if (__any_sync(0xffffffffu, bad) && lane == 0) atomicExch(status, 1);
    int n = 0, at = -1, want = 0;
    while (n < N) {
        const uint32_t h0 = __ballot_sync(0xffffffffu, par[0] == at && (at < 0 || tok[0] == want)), h1 = __ballot_sync(0xffffffffu, par[1] == at && (at < 0 || tok[1] == want));
        const int next = h0 ? __ffs(h0) - 1 : h1 ? 31 + __ffs(h1) : -1;
        if (next < 0) break;
        if (lane == 0) path[o + n] = next;
        n++;
        at = next;
        const int w0 = __shfl_sync(0xffffffffu, id[0], next & 31), w1 = __shfl_sync(0xffffffffu, id[1], next & 31);
        want = next < 32 ? w0 : w1;
    }
    for (int i = n + lane; i < N; i += 32) path[o + i] = -1;
    if (lane == 0) n_path[b] = n;
}

int launch_tree_accept(const int* parents, const int* toks, const int* ids, int* path, int* n_path, int* status, int B, int N, cudaStream_t st) {
    if (B <= 0) return GDN_OK;
    tree_accept_kernel<<<(B + 3) / 4, 128, 0, st>>>(parents, toks, ids, path, n_path, status, B, N);
    return check_launch("tree_accept");
}

// ----------------------------------------------------------------------------------------------------------------------
// commit: one block per (layer, sequence, head), two per SM.  Bound: HBM, the state once in and once out (2 MiB per layer and sequence).
// One bulk copy brings a head's state into shared memory while the path's tokens go through conv, norm and gates; then half of it at a time
// lies in registers, a row on 8 lanes of 4 float4 each, so that a quarter warp reads and writes 128 contiguous bytes.  While the states
// stream, a load that misses L2 takes 5 us, so a block asks L2 for the rows that a block of a later layer will need (32 KiB against its 128
// of state, and the states are marked to leave L2 first).  24 sequences x 18 layers, accept and compaction included: 203 us (commit
// alone 199, 4.8 TB/s), without the prefetch 249, two layers ahead instead of one 202 (against 200 then).  Measured and not kept: state by plain loads (256), three blocks per SM with 80
// registers (204 .. 215), half heads on four blocks (305), 512 threads a head (309), persistent blocks with a ring of bulk copies (225 .. 380,
// 25 against 14 us for one sequence).
// ----------------------------------------------------------------------------------------------------------------------
constexpr int CM_THREADS = 256, CM_STEPS = 8;                        // tokens of the path prepared at a time
constexpr int STATE_BYTES = DV * DK * 4;
constexpr int CM_GENERATION = 300;                                   // blocks between a prefetch and its use: as many as are resident
constexpr int CM_PATH = 64, CM_AHEAD = 8;                            // path entries kept in shared memory; raw rows in flight

// silu to a few fp32 ulp: expf's own error and an approximate division
__device__ __forceinline__ float silu_ulp(float x) { return __fdividef(x, 1.f + expf(-x)); }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) { f32x2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }

__global__ void __launch_bounds__(CM_THREADS, 2) tree_commit_kernel(const __grid_constant__ TreeCommitArgs a) {
    extern __shared__ __align__(1024) unsigned char smem[];          // the state as it comes in
    __shared__ uint64_t s_bar;
    __shared__ __align__(16) float s_k[CM_STEPS][DK];
    __shared__ float s_v[CM_STEPS][DV], s_g[CM_STEPS], s_beta[CM_STEPS], s_red[CM_STEPS][4];
    __shared__ int s_path[CM_PATH];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int h = blockIdx.x % HV, b = blockIdx.x / HV, layer = blockIdx.y;
    const bool isv = tid >= 128;                                     // threads 0-127: channel of k (and the window of q's), the others: of v
    const int c = tid & 127, ch = (isv ? 2 : 1) * KD + h * DK + c, chq = h * DK + c;
    const int* path = a.path + (size_t)b * a.E;
    const int first = tid < CM_PATH && tid < a.E ? path[tid] : 0;
    const int slot = a.slots[b], dst = a.dst_slots[b], pos = a.pos[b], n = a.n_path[b];
    const int o0 = min(tid, a.B - 1), so0 = a.slots[o0], to0 = a.dst_slots[o0], no0 = a.n_path[o0];
    const uint2 taps = *reinterpret_cast<const uint2*>(a.conv_w[layer] + (size_t)ch * 4);
    const float A_log = a.A_log[layer][h], dt_bias = a.dt_bias[layer][h];
    bool bad = slot < 0 || slot >= a.n_slots || dst < 0 || dst >= a.n_slots || pos < 0 || n < 0 || n > a.E;
    if (!bad && n == 0 && slot == dst) return;
    const uint32_t landed = smem_addr(&s_bar);
    const bool loads = !bad;                                         // (uniform)
    if (tid == 0 && loads) {
        mbar_init(landed, 1);
        fence_barrier_init();
        mbar_expect_tx(landed, STATE_BYTES);
        const char* src = reinterpret_cast<const char*>(a.ssm_pool[layer] + (size_t)slot * STATE_ELEMS + (size_t)h * DV * DK);
        uint64_t once;                                               // (read once: first to leave L2)
        asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(once));
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;"
                     ::"r"(smem_addr(smem)), "l"(src), "r"(STATE_BYTES), "r"(landed), "l"(once) : "memory");
    }
    if (tid < CM_PATH) s_path[tid] = first;
    bad = bad || (tid < n && tid < CM_PATH && (first < 0 || first >= a.N));
    // another sequence that writes what this one reads or writes, or reads what it writes, would make the result a matter of order: both
    // are refused (the pools' last slot takes the padding of a batch and is nobody's)
    auto clash = [&](int o, int so, int to, int no) -> bool {
        const int last = a.n_slots - 1;
        return o != b && (so != to || no != 0) && ((to == slot && slot != last) || ((to == dst || so == dst) && dst != last));
    };
    bad = bad || clash(o0, so0, to0, no0);
    for (int o = tid + CM_THREADS; o < a.B; o += CM_THREADS) bad = bad || clash(o, a.slots[o], a.dst_slots[o], a.n_path[o]);
    if (!bad)
        for (int j = CM_PATH + tid; j < n; j += CM_THREADS) bad = bad || path[j] < 0 || path[j] >= a.N;
    if (__syncthreads_or(bad)) {
        if (tid == 0) { atomicExch(a.status, 1); if (loads) mbar_wait(landed, 0, DRAIN_POLLS); }      // (nothing may land after the block)
        return;
    }
    auto node = [&](int j) -> int { return j < CM_PATH ? s_path[j] : path[j]; };
    const __nv_bfloat16* rows = a.proj[layer] + (size_t)b * a.N * a.row_stride;
    const __nv_bfloat16* win = a.conv_pool[layer] + ((size_t)slot * 2 + (pos & 1)) * 3 * CD;
    // A load that misses L2 while the states stream takes 5 us, one that hits 0.8: the rows that this sequence's block of a later layer
    // will read (about one generation of blocks ahead) are asked for now.
    const int later = layer + a.ahead;
    if (later < gridDim.y) {
        const __nv_bfloat16* rows2 = a.proj[later] + (size_t)b * a.N * a.row_stride;
        const __nv_bfloat16* win2 = a.conv_pool[later] + ((size_t)slot * 2 + (pos & 1)) * 3 * CD;
        for (int i = tid; i < (n + 3) * 8; i += CM_THREADS) {
            const int r = i >> 3, part = (i & 7) >> 1;               // parts: q, k, v (two lines each), gates
            const __nv_bfloat16* base = r < 3 ? win2 + (size_t)r * CD : rows2 + (size_t)node(r - 3) * a.row_stride;
            const __nv_bfloat16* line = part < 3 ? base + part * KD + h * DK + (i & 1) * 64 : base + CD + KD;
            if (part == 0 ? r >= n : part < 3 || (r >= 3 && !(i & 1))) asm volatile("prefetch.global.L2 [%0];" ::"l"(line));
        }
    }
    // raw row r of the sequence: 0..2 the window, 3 + j the path's tokens
    auto raw = [&](int r, int chan) -> __nv_bfloat16 { return r < 3 ? win[(size_t)r * CD + chan] : rows[(size_t)node(r - 3) * a.row_stride + chan]; };
    __nv_bfloat16 x0 = win[ch], x1 = win[CD + ch], x2 = win[2 * CD + ch], q0, q1, q2;
    if (!isv) { q0 = raw(n, chq); q1 = raw(n + 1, chq); q2 = raw(n + 2, chq); }
    __nv_bfloat16 x[CM_AHEAD];                                       // the next raw rows
    auto fetch = [&](int j0) {
#pragma unroll
        for (int q = 0; q < CM_AHEAD; q++)
            if (j0 + q < n) x[q] = rows[(size_t)node(j0 + q) * a.row_stride + ch];
    };
    fetch(0);
    __nv_bfloat16 raw_a, raw_b;
    auto fetch_gates = [&](int j) {
        const __nv_bfloat16* r = rows + (size_t)node(j) * a.row_stride + CD + KD + h;
        raw_b = r[0]; raw_a = r[HV];
    };
    if (tid < min(n, CM_STEPS)) fetch_gates(tid);
    // this thread's part of the state, in two halves: rows row + 8 half + 4 i, columns col + 32 m
    const int row = warp * 16 + (lane >> 3), col = (lane & 7) * 4;
    float* out = a.ssm_pool[layer] + (size_t)dst * STATE_ELEMS + (size_t)h * DV * DK;
    // The state has landed?  Decided for the whole block: one that gives up writes nothing, and waits for the copy before it leaves.
    auto state_is_here = [&]() -> bool {
        if (!__syncthreads_or(!mbar_wait(landed, 0))) return true;
        if (tid == 0) { atomicExch(a.status, 2); mbar_wait(landed, 0, DRAIN_POLLS); }
        return false;
    };
    ulonglong2 S[2][4];
    auto take = [&](int half) {
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int m = 0; m < 4; m++) S[i][m] = *reinterpret_cast<const ulonglong2*>(smem + ((row + 8 * half + 4 * i) * DK + col + 32 * m) * 4);
    };
    auto put = [&](int half, bool last) {
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int m = 0; m < 4; m++) {
                const int e = (row + 8 * half + 4 * i) * DK + col + 32 * m;
                if (last) {
                    const float2 lo = unpack2(S[i][m].x), hi = unpack2(S[i][m].y);
                    __stcs(reinterpret_cast<float4*>(out + e), make_float4(lo.x, lo.y, hi.x, hi.y));
                } else {
                    *reinterpret_cast<ulonglong2*>(smem + e * 4) = S[i][m];
                }
            }
    };
    float w[4];
    unpack_bf16x4(taps, w);
    for (int j0 = 0; j0 < n; j0 += CM_STEPS) {
        const int cnt = min(CM_STEPS, n - j0);
        if (j0) {
            __syncthreads();                                         // the steps before have read the shared rows
            if (tid < cnt) fetch_gates(j0 + tid);
        }
        if (tid < cnt) {
            s_beta[tid] = sigmoid_f(__bfloat162float(raw_b));
            s_g[tid] = expf(log_decay_f(A_log, __bfloat162float(raw_a) + dt_bias));
        }
        for (int j1 = 0; j1 < cnt; j1 += CM_AHEAD) {
            if (j0 + j1) fetch(j0 + j1);
#pragma unroll
            for (int q = 0; q < CM_AHEAD; q++) {
                if (j1 + q >= cnt) break;
                const float f = fmaf(__bfloat162float(x[q]), w[3], fmaf(__bfloat162float(x2), w[2], fmaf(__bfloat162float(x1), w[1], __bfloat162float(x0) * w[0])));
                const float v = silu_ulp(f);
                x0 = x1; x1 = x2; x2 = x[q];
                if (isv) s_v[j1 + q][c] = v;
                else {
                    s_k[j1 + q][c] = v;
                    const float ss = warp_sum(v * v);
                    if (lane == 0) s_red[j1 + q][warp] = ss;
                }
            }
        }
        if (j0 == 0) {                                               // (a barrier, which the rows above need too)
            if (!state_is_here()) return;
        } else {
            __syncthreads();
        }
#pragma unroll 1
        for (int half = 0; half < 2; half++) {
            take(half);
            for (int j = 0; j < cnt; j++) {
                // k is used as it left the conv; its length enters the two places where k does
                const float r = rsqrtf((s_red[j][0] + s_red[j][1]) + (s_red[j][2] + s_red[j][3]) + 1e-6f);
                const float g = s_g[j], beta = s_beta[j];
                const f32x2 gg = pack2(g, g);
                ulonglong2 k[4];
#pragma unroll
                for (int m = 0; m < 4; m++) k[m] = *reinterpret_cast<const ulonglong2*>(&s_k[j][col + 32 * m]);
                float p[2];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    f32x2 p0 = 0, p1 = 0;
#pragma unroll
                    for (int m = 0; m < 4; m++) {
                        S[i][m].x = mul2(S[i][m].x, gg); S[i][m].y = mul2(S[i][m].y, gg);
                        fma2(p0, S[i][m].x, k[m].x); fma2(p1, S[i][m].y, k[m].y);
                    }
                    const float2 a0 = unpack2(p0), a1 = unpack2(p1);
                    p[i] = (a0.x + a0.y) + (a1.x + a1.y);
                }
                // the two rows' sums over their eight lanes: one exchange leaves lane l with row l & 1's, two more complete it
                const bool odd = lane & 1;
                float x = (odd ? p[1] : p[0]) + __shfl_xor_sync(0xffffffffu, odd ? p[0] : p[1], 1);
                x += __shfl_xor_sync(0xffffffffu, x, 2);
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                const float u = (s_v[j][row + 8 * half + 4 * (lane & 1)] - x * r) * beta * r;      // of row `row + 8 half + 4 (lane & 1)`
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const float ui = __shfl_sync(0xffffffffu, u, (lane & 24) + i);
                    const f32x2 uu = pack2(ui, ui);
#pragma unroll
                    for (int m = 0; m < 4; m++) { fma2(S[i][m].x, uu, k[m].x); fma2(S[i][m].y, uu, k[m].y); }
                }
            }
            put(half, j0 + cnt >= n);
        }
    }
    if (n == 0) {
        if (!state_is_here()) return;
        for (int half = 0; half < 2; half++) { take(half); put(half, true); }
    }
    // a window buffer that is read and written in one call (n even): every channel has been read by the thread that writes it
    __nv_bfloat16* wout = a.conv_pool[layer] + ((size_t)dst * 2 + (((unsigned)pos + (unsigned)n) & 1)) * 3 * CD;
    wout[ch] = x0; wout[CD + ch] = x1; wout[2 * CD + ch] = x2;
    if (!isv) { wout[chq] = q0; wout[CD + chq] = q1; wout[2 * CD + chq] = q2; }
}

int launch_tree_commit(const TreeCommitArgs& a, int n_layers, cudaStream_t st) {
    if (a.B <= 0 || n_layers <= 0) return GDN_OK;
    static bool attr_set[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && !attr_set[dev]) {
        if (cudaFuncSetAttribute(tree_commit_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, STATE_BYTES) != cudaSuccess) return check_launch("tree_commit smem attribute");
        attr_set[dev] = true;
    }
    TreeCommitArgs with = a;
    with.ahead = (CM_GENERATION + a.B * HV - 1) / (a.B * HV);
    tree_commit_kernel<<<dim3((unsigned)(a.B * HV), n_layers), CM_THREADS, STATE_BYTES, st>>>(with);
    return check_launch("tree_commit");
}

}  // namespace gdn

#ifdef GDN_TIMING
extern "C" __attribute__((visibility("default"))) int gdn_timing_log_delta(long long* out_host, int n) {
    return cudaMemcpyFromSymbol(out_host, gdn::g_tlog, sizeof(long long) * n) == cudaSuccess ? 0 : -5;
}
#endif
