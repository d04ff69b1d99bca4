// Attention of a tree of drafted tokens over a paged cache (see gqa_tree_attn in the header).
#include "gqa_common.cuh"

namespace gdn {

// one warp per (sequence, node, query head)
__global__ void __launch_bounds__(128) tree_attn_kernel(const TreeAttnArgs a) {
    const int lane = threadIdx.x & 31, item = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (item >= a.B * a.N * a.H) return;
    const int h = item % a.H, i = item / a.H % a.N, b = item / a.H / a.N, kvh = h / (a.H / a.KV);
    const int ctx = a.ctx_len[b];
    const int* par = a.parents + (size_t)b * a.N;
    uint4* out = reinterpret_cast<uint4*>(a.out + (size_t)item * ATT_D);
    unsigned long long line = 0;
    for (int at = i; at >= 0;) {
        line |= 1ull << at;
        const int p = par[at];
        if (p >= at || (p < -1 && at != i)) { if (lane == 0) atomicExch(a.status, 1); }
        if (p >= at || p < -1) { line = 0; break; }
        at = p;
    }
    const long long rows = (long long)a.max_pages * a.page_size;
    int last = a.N - 1;                                              // the last node in use
    while (last >= 0 && par[last] < -1) last--;
    if (ctx < 0 || (long long)ctx + last >= rows) { line = 0; if (lane == 0) atomicExch(a.status, 1); }
    if (!line) { out[lane] = make_uint4(0, 0, 0, 0); return; }
    float q[8], o[8] = {}, m = -INFINITY, l = 0.f;
    auto unpack = [](uint4 u, float* f) {
        unpack_bf16x4(make_uint2(u.x, u.y), f);
        unpack_bf16x4(make_uint2(u.z, u.w), f + 4);
    };
    unpack(reinterpret_cast<const uint4*>(a.q + (size_t)item * ATT_D)[lane], q);
    auto step = [&](const uint4 ku, const uint4 vu) {
        float k[8], v[8], s = 0.f;
        unpack(ku, k); unpack(vu, v);
#pragma unroll
        for (int c = 0; c < 8; c++) s = fmaf(q[c], k[c], s);
        s = warp_sum(s) * 0.0625f;
        const float mn = fmaxf(m, s), al = mn == -INFINITY ? 1.f : expf(m - mn), p = mn == -INFINITY ? 0.f : expf(s - mn);
        m = mn; l = l * al + p;
#pragma unroll
        for (int c = 0; c < 8; c++) o[c] = fmaf(p, v[c], o[c] * al);
    };
    const int* table = a.block_table + (size_t)b * a.max_pages;
    for (int t = 0; t < ctx; t++) {
        int page = table[t / a.page_size];
        if (page < 0 || page >= a.n_pages) { if (lane == 0) atomicExch(a.status, 1); page = 0; }
        const size_t off = (((size_t)page * a.KV + kvh) * a.page_size + t % a.page_size) * ATT_D;
        step(reinterpret_cast<const uint4*>(a.k_pages + off)[lane], reinterpret_cast<const uint4*>(a.v_pages + off)[lane]);
    }
    for (unsigned long long r = line; r; r &= r - 1) {
        const size_t off = (((size_t)b * a.N + (__ffsll((long long)r) - 1)) * a.KV + kvh) * ATT_D;
        step(reinterpret_cast<const uint4*>(a.k_new + off)[lane], reinterpret_cast<const uint4*>(a.v_new + off)[lane]);
    }
    const float inv = l == 0.f ? 1.f : 1.f / l;
    out[lane] = make_uint4(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv), pack_bf16x2(o[4] * inv, o[5] * inv), pack_bf16x2(o[6] * inv, o[7] * inv));
    if (h % (a.H / a.KV) == 0) {                                     // the node's rows into the cache
        const int page = table[(ctx + i) / a.page_size];
        if (page < 0 || page >= a.n_pages) { if (lane == 0) atomicExch(a.status, 1); return; }
        const size_t src = (((size_t)b * a.N + i) * a.KV + kvh) * ATT_D, dst = (((size_t)page * a.KV + kvh) * a.page_size + (ctx + i) % a.page_size) * ATT_D;
        reinterpret_cast<uint4*>(a.k_pages + dst)[lane] = reinterpret_cast<const uint4*>(a.k_new + src)[lane];
        reinterpret_cast<uint4*>(a.v_pages + dst)[lane] = reinterpret_cast<const uint4*>(a.v_new + src)[lane];
    }
}

size_t tree_attn_workspace_bytes(int, int, int, int) { return 16; }

int launch_tree_attn(const TreeAttnArgs& a, void*, size_t, cudaStream_t st) {
    if (a.B <= 0 || a.N <= 0) return GDN_OK;
    tree_attn_kernel<<<(a.B * a.N * a.H + 3) / 4, 128, 0, st>>>(a);
    return check_launch("tree_attn");
}

}  // namespace gdn
