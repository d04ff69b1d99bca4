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
// Conv, silu, norm and gates stay in fp32 here, and nothing is rounded before y (bf16) or the state (fp32): the single-token and
// chained kernels round to bf16 after each of these operations as the reference's graph does, so results agree with them to
// bf16 rounding, not bit for bit.
#include "gdn_common.cuh"
#include "launchers.cuh"

namespace gdn {

constexpr int TREE_MAX = 64;

__device__ __forceinline__ float silu_f(float x) { return x / (1.f + expf(-x)); }
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
// verify: one block per (sequence, head)
// ----------------------------------------------------------------------------------------------------------------------
constexpr int TV_THREADS = 256;

__global__ void __launch_bounds__(TV_THREADS) tree_verify_kernel(const TreeDeltaArgs a) {
    extern __shared__ __align__(16) float sm[];
    const int N = a.N, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int b = blockIdx.x / HV, h = blockIdx.x % HV;
    float *sq = sm, *sk = sq + N * DK, *su = sk + N * DK;            // q, k, v (then u) of the nodes
    float *skk = su + N * DK, *sqk = skk + N * N;                    // M (k.k) beta, M (q.k)
    __shared__ int s_par[TREE_MAX];
    __shared__ unsigned long long s_line[TREE_MAX];
    __shared__ float s_lg[TREE_MAX], s_beta[TREE_MAX], s_G[TREE_MAX];
    const int slot = a.slots[b], pos = a.pos[b];
    if (slot < 0 || slot >= a.n_slots || pos < 0) {                  // rows of a bad sequence: zeros
        if (tid == 0) atomicExch(a.status, 1);
        for (int i = tid; i < N * DV; i += TV_THREADS) a.y[((size_t)b * N + i / DV) * KD + h * DV + i % DV] = __float2bfloat16_rn(0.f);
        return;
    }
    if (tid < N) s_par[tid] = a.parents[(size_t)b * N + tid];
    __syncthreads();
    if (tid < N) {
        bool bad = false;
        s_line[tid] = tree_line(s_par, tid, bad);
        if (bad) atomicExch(a.status, 1);
        const __nv_bfloat16* row = a.proj + ((size_t)b * N + tid) * a.row_stride;
        s_beta[tid] = sigmoid_f(ldbf(row + CD + KD + h));
        s_lg[tid] = log_decay_f(a.A_log[h], ldbf(row + CD + KD + HV + h) + a.dt_bias[h]);
    }
    __syncthreads();
    if (tid < N) {
        float g = 0.f;
        for (unsigned long long m = s_line[tid]; m; m &= m - 1) g += s_lg[__ffsll((long long)m) - 1];
        s_G[tid] = g;
    }
    // conv over the path + silu + norms: one node per warp, four channels of q, k and v per lane
    const __nv_bfloat16* window = a.conv_pool + ((size_t)slot * 2 + (pos & 1)) * 3 * CD;
    for (int i = warp; i < N; i += TV_THREADS / 32) {
        if (!s_line[i]) continue;
        const __nv_bfloat16* row[4];
        for (int t = 3, e = 3 + i; t >= 0; t--) {                    // rows: window 0..2, then nodes
            row[t] = e >= 3 ? a.proj + ((size_t)b * N + e - 3) * a.row_stride : window + (size_t)e * CD;
            e = e >= 3 ? (s_par[e - 3] >= 0 ? 3 + s_par[e - 3] : 2) : e - 1;
        }
#pragma unroll
        for (int g = 0; g < 3; g++) {
            const int ch = g * KD + h * DK + 4 * lane;
            float acc[4] = {0.f, 0.f, 0.f, 0.f}, w[4][4];
#pragma unroll
            for (int c = 0; c < 4; c++) unpack_bf16x4(*reinterpret_cast<const uint2*>(a.conv_w + (size_t)(ch + c) * 4), w[c]);
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int c = 0; c < 4; c++) acc[c] = fmaf(ldbf(row[t] + ch + c), w[c][t], acc[c]);
            float ss = 0.f;
#pragma unroll
            for (int c = 0; c < 4; c++) { acc[c] = silu_f(acc[c]); ss += acc[c] * acc[c]; }
            float scale = 1.f;
            if (g < 2) scale = rsqrtf(warp_sum(ss) + 1e-6f) * (g == 0 ? 0.08838834764831845f : 1.f);
            float* dst = (g == 0 ? sq : g == 1 ? sk : su) + i * DK + 4 * lane;
#pragma unroll
            for (int c = 0; c < 4; c++) dst[c] = acc[c] * scale;
        }
    }
    __syncthreads();
    for (int p = tid; p < N * N; p += TV_THREADS) {
        const int i = p / N, j = p % N;
        float kk = 0.f, qk = 0.f;
        if (s_line[i] >> j & 1) {
            for (int c = 0; c < DK; c++) { kk = fmaf(sk[i * DK + c], sk[j * DK + c], kk); qk = fmaf(sq[i * DK + c], sk[j * DK + c], qk); }
            const float M = expf(s_G[i] - s_G[j]);
            kk *= M * s_beta[i]; qk *= M;
        }
        skk[p] = kk; sqk[p] = qk;
    }
    __syncthreads();
    // two threads per value row, 64 key columns of S0 each
    const int d = tid >> 1, half = tid & 1;
    float S[DK / 2];
    const float4* src = reinterpret_cast<const float4*>(a.ssm_pool + ((size_t)slot * HV + h) * DV * DK + d * DK + half * 64);
#pragma unroll
    for (int c = 0; c < 16; c++) *reinterpret_cast<float4*>(&S[4 * c]) = src[c];
    for (int i = 0; i < N; i++) {
        __nv_bfloat16* out = a.y + ((size_t)b * N + i) * KD + h * DV + d;
        const unsigned long long line = s_line[i];
        if (!line) { if (half == 0) *out = __float2bfloat16_rn(0.f); continue; }
        float p1 = 0.f, p2 = 0.f;
#pragma unroll
        for (int c = 0; c < 64; c++) { p1 = fmaf(S[c], sk[i * DK + half * 64 + c], p1); p2 = fmaf(S[c], sq[i * DK + half * 64 + c], p2); }
        p1 += __shfl_xor_sync(0xffffffffu, p1, 1);
        p2 += __shfl_xor_sync(0xffffffffu, p2, 1);
        const float grow = expf(s_G[i]);
        float u = s_beta[i] * (su[i * DK + d] - grow * p1), y = grow * p2;
        for (unsigned long long m = line & ~(1ull << i); m; m &= m - 1) {
            const int j = __ffsll((long long)m) - 1;
            u = fmaf(-skk[i * N + j], su[j * DK + d], u);
            y = fmaf(sqk[i * N + j], su[j * DK + d], y);
        }
        y = fmaf(sqk[i * N + i], u, y);
        __syncwarp();
        if (half == 0) { su[i * DK + d] = u; *out = __float2bfloat16_rn(y); }      // column d belongs to these two threads
        __syncwarp();
    }
}

int launch_tree_verify(const TreeDeltaArgs& a, cudaStream_t st) {
    if (a.B <= 0 || a.N <= 0) return GDN_OK;
    const int smem = (3 * a.N * DK + 2 * a.N * a.N) * 4;
    if (cudaFuncSetAttribute(tree_verify_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (3 * TREE_MAX * DK + 2 * TREE_MAX * TREE_MAX) * 4) != cudaSuccess)
        return check_launch("tree_verify smem attribute");
    tree_verify_kernel<<<a.B * HV, TV_THREADS, smem, st>>>(a);
    return check_launch("tree_verify");
}

// ----------------------------------------------------------------------------------------------------------------------
// accept: one warp per sequence walks from the first root to the first child that carries the token the target chose
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
// commit: one block per (layer, sequence, head).  Bound: HBM, the state once in and once out (2 MiB per layer and sequence).  The
// state lies in registers -- a row on 8 lanes of 4 float4 each, so that a quarter warp reads 128 contiguous bytes -- and is requested
// before the conv / norm / gate work of the path's tokens, which hides behind its latency.
// ----------------------------------------------------------------------------------------------------------------------
constexpr int CM_THREADS = 256, CM_STEPS = 16;                      // tokens of the path prepared at a time

__global__ void __launch_bounds__(CM_THREADS, 2) tree_commit_kernel(const __grid_constant__ TreeCommitArgs a) {
    __shared__ float s_k[CM_STEPS][DK], s_v[CM_STEPS][DV], s_g[CM_STEPS], s_beta[CM_STEPS], s_red[CM_STEPS][4];
    __shared__ int s_bad;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int layer = blockIdx.y, b = blockIdx.x / HV, h = blockIdx.x % HV;
    const int slot = a.slots[b], dst = a.dst_slots[b], pos = a.pos[b], n = a.n_path[b];
    const int* path = a.path + (size_t)b * a.E;
    if (tid == 0) s_bad = 0;
    __syncthreads();
    if (slot < 0 || slot >= a.n_slots || dst < 0 || dst >= a.n_slots || pos < 0 || n < 0 || n > a.E) { if (tid == 0) atomicExch(a.status, 1); return; }
    for (int j = tid; j < n; j += CM_THREADS)
        if (path[j] < 0 || path[j] >= a.N) s_bad = 1;
    __syncthreads();
    if (s_bad) { if (tid == 0) atomicExch(a.status, 1); return; }
    if (n == 0 && slot == dst) return;
    // ---- the state ----
    const size_t head = (size_t)h * DV * DK;
    const int row = warp * 16 + (lane >> 3), col = (lane & 7) * 4;   // rows row + 4 i, columns col + 32 m
    float4 S[4][4];
    {
        const float* src = a.ssm_pool[layer] + (size_t)slot * STATE_ELEMS + head;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int m = 0; m < 4; m++) S[i][m] = __ldcs(reinterpret_cast<const float4*>(src + (row + 4 * i) * DK + col + 32 * m));
    }
    // ---- the conv window: thread t < 128 owns channel t of q and of k, the others channel t - 128 of v ----
    const int c = tid & 127;
    const bool isv = tid >= 128;
    const __nv_bfloat16* proj = a.proj[layer] + (size_t)b * a.N * a.row_stride;
    const __nv_bfloat16* win = a.conv_pool[layer] + ((size_t)slot * 2 + (pos & 1)) * 3 * CD;
    __nv_bfloat16* wout = a.conv_pool[layer] + ((size_t)dst * 2 + (((unsigned)pos + (unsigned)n) & 1)) * 3 * CD;
    const int ch = (isv ? 2 : 1) * KD + h * DK + c, chq = h * DK + c;
    float w[4];
    unpack_bf16x4(*reinterpret_cast<const uint2*>(a.conv_w[layer] + (size_t)ch * 4), w);
    // raw row r of the sequence: r = 0..2 the window, 3 + j the path's tokens
    auto raw = [&](int r, int chan) -> __nv_bfloat16 { return r < 3 ? win[(size_t)r * CD + chan] : proj[(size_t)path[r - 3] * a.row_stride + chan]; };
    __nv_bfloat16 x0 = raw(0, ch), x1 = raw(1, ch), x2 = raw(2, ch);
    __nv_bfloat16 q0, q1, q2;
    if (!isv) { q0 = raw(n, chq); q1 = raw(n + 1, chq); q2 = raw(n + 2, chq); }
    for (int j0 = 0; j0 < n; j0 += CM_STEPS) {
        const int cnt = min(CM_STEPS, n - j0);
        __syncthreads();                                             // the steps before have read the shared rows
        if (tid < cnt) {
            const __nv_bfloat16* r = proj + (size_t)path[j0 + tid] * a.row_stride;
            s_beta[tid] = sigmoid_f(ldbf(r + CD + KD + h));
            s_g[tid] = expf(log_decay_f(a.A_log[layer][h], ldbf(r + CD + KD + HV + h) + a.dt_bias[layer][h]));
        }
        for (int j = 0; j < cnt; j++) {
            const __nv_bfloat16 x3 = raw(3 + j0 + j, ch);
            float v = fmaf(__bfloat162float(x3), w[3], fmaf(__bfloat162float(x2), w[2], fmaf(__bfloat162float(x1), w[1], __bfloat162float(x0) * w[0])));
            v = silu_f(v);
            x0 = x1; x1 = x2; x2 = x3;
            if (isv) s_v[j][c] = v;
            else {
                s_k[j][c] = v;
                const float ss = warp_sum(v * v);
                if (lane == 0) s_red[j][warp] = ss;
            }
        }
        __syncthreads();
        if (!isv)
            for (int j = 0; j < cnt; j++) s_k[j][c] *= rsqrtf(s_red[j][0] + s_red[j][1] + s_red[j][2] + s_red[j][3] + 1e-6f);
        __syncthreads();
        for (int j = 0; j < cnt; j++) {
            const float g = s_g[j], beta = s_beta[j];
            float4 k[4];
#pragma unroll
            for (int m = 0; m < 4; m++) k[m] = *reinterpret_cast<const float4*>(&s_k[j][col + 32 * m]);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float p = 0.f;
#pragma unroll
                for (int m = 0; m < 4; m++) {
                    float4& s = S[i][m];
                    s.x *= g; s.y *= g; s.z *= g; s.w *= g;
                    p = fmaf(s.x, k[m].x, fmaf(s.y, k[m].y, fmaf(s.z, k[m].z, fmaf(s.w, k[m].w, p))));
                }
                p += __shfl_xor_sync(0xffffffffu, p, 1);
                p += __shfl_xor_sync(0xffffffffu, p, 2);
                p += __shfl_xor_sync(0xffffffffu, p, 4);
                const float d = (s_v[j][row + 4 * i] - p) * beta;
#pragma unroll
                for (int m = 0; m < 4; m++) {
                    float4& s = S[i][m];
                    s.x = fmaf(d, k[m].x, s.x); s.y = fmaf(d, k[m].y, s.y); s.z = fmaf(d, k[m].z, s.z); s.w = fmaf(d, k[m].w, s.w);
                }
            }
        }
    }
    float* out = a.ssm_pool[layer] + (size_t)dst * STATE_ELEMS + head;
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int m = 0; m < 4; m++) __stcs(reinterpret_cast<float4*>(out + (row + 4 * i) * DK + col + 32 * m), S[i][m]);
    // a window buffer that is read and written in one call (n even): every channel has been read by the thread that writes it
    wout[ch] = x0; wout[CD + ch] = x1; wout[2 * CD + ch] = x2;
    if (!isv) { wout[chq] = q0; wout[CD + chq] = q1; wout[2 * CD + chq] = q2; }
}

int launch_tree_commit(const TreeCommitArgs& a, int n_layers, cudaStream_t st) {
    if (a.B <= 0 || n_layers <= 0) return GDN_OK;
    tree_commit_kernel<<<dim3((unsigned)(a.B * HV), n_layers), CM_THREADS, 0, st>>>(a);
    return check_launch("tree_commit");
}

}  // namespace gdn
