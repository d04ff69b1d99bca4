// Strided in-place copies for state admission, snapshot moves and prefix-cache checkpoints.
//
// Replaces the reference's `blit` kernel (qwen35/batch.py:349-372):
//     dst.flat[d0 + y*dstride + i] = src.flat[s0 + y*sstride + i]   for i < n, y < ny
// Offsets and strides are in elements of `elem_size` bytes (2 = bf16, 4 = fp32).  Rows are copied with 16-byte accesses when
// every address involved is 16-byte aligned, element by element otherwise.
#include "gdn_common.cuh"
#include "launchers.cuh"

namespace gdn {

template <typename T>
__global__ void state_copy_kernel(T* __restrict__ dst, const T* __restrict__ src, long long n, long long dstride, long long sstride) {
    const long long y = blockIdx.y;
    T* d = dst + y * dstride;
    const T* s = src + y * sstride;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) d[i] = s[i];
}

template <typename T>
static int run(void* dst, const void* src, long long n, long long d0, long long s0, int ny, long long dstride, long long sstride, cudaStream_t st) {
    long long blocks = (n + 255) / 256;
    if (blocks > 148 * 8) blocks = 148 * 8;
    state_copy_kernel<T><<<dim3((unsigned)blocks, ny), 256, 0, st>>>(static_cast<T*>(dst) + d0, static_cast<const T*>(src) + s0, n, dstride, sstride);
    return check_launch("state_copy");
}

int launch_state_copy(void* dst, const void* src, int elem_size, long long n, long long d0, long long s0, int ny, long long dstride,
                      long long sstride, cudaStream_t st) {
    if (n <= 0 || ny <= 0) return GDN_OK;
    if (elem_size != 2 && elem_size != 4) { set_error("state_copy: elem_size must be 2 or 4, got %d", elem_size); return GDN_E_DTYPE; }
    if (ny > 65535) { set_error("state_copy: ny = %d exceeds 65535", ny); return GDN_E_SHAPE; }
    const long long per16 = 16 / elem_size;
    const bool vec = (n % per16 == 0) && (d0 % per16 == 0) && (s0 % per16 == 0) && (dstride % per16 == 0) && (sstride % per16 == 0) &&
                     (reinterpret_cast<uintptr_t>(dst) % 16 == 0) && (reinterpret_cast<uintptr_t>(src) % 16 == 0);
    if (vec) return run<uint4>(dst, src, n / per16, d0 / per16, s0 / per16, ny, dstride / per16, sstride / per16, st);
    if (elem_size == 4) return run<uint32_t>(dst, src, n, d0, s0, ny, dstride, sstride, st);
    return run<uint16_t>(dst, src, n, d0, s0, ny, dstride, sstride, st);
}

// Row scatter of the speculative mode's hidden-state history (the reference's `hrec` kernel, qwen35/batch.py:375-399):
//     hist[slots[b], pos[b], :] = rows[b, :]        hist [n_slots, Lh, H] bf16, rows [B, H] bf16
// The indices live on the device; a row whose slot or position is out of range is skipped and reported through the status word.
__global__ void hrec_kernel(__nv_bfloat16* __restrict__ hist, const __nv_bfloat16* __restrict__ rows, const int* __restrict__ slots,
                            const int* __restrict__ pos, int n_slots, int Lh, int H, int* status) {
    const int b = blockIdx.y;
    const int s = slots[b], p = pos[b];
    if (s < 0 || s >= n_slots || p < 0 || p >= Lh) { if (threadIdx.x == 0 && blockIdx.x == 0) atomicExch(status, 1); return; }
    __nv_bfloat16* d = hist + ((size_t)s * Lh + p) * H;
    const __nv_bfloat16* r = rows + (size_t)b * H;
    const bool vec = (H % 8 == 0) && (reinterpret_cast<uintptr_t>(d) % 16 == 0) && (reinterpret_cast<uintptr_t>(r) % 16 == 0);
    if (vec) {
        for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < H / 8; i += gridDim.x * blockDim.x)
            reinterpret_cast<uint4*>(d)[i] = reinterpret_cast<const uint4*>(r)[i];
    } else {
        for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < H; i += gridDim.x * blockDim.x) d[i] = r[i];
    }
}

int launch_hrec(void* hist, const void* rows, const int* slots, const int* pos, int B, int n_slots, int Lh, int H, int* status, cudaStream_t st) {
    if (B <= 0 || H <= 0) return GDN_OK;
    if (B > 65535) { set_error("hrec: B = %d exceeds 65535", B); return GDN_E_SHAPE; }
    hrec_kernel<<<dim3(1, B), 128, 0, st>>>(static_cast<__nv_bfloat16*>(hist), static_cast<const __nv_bfloat16*>(rows), slots, pos, n_slots, Lh, H, status);
    return check_launch("hrec");
}

// ----------------------------------------------------------------------------------------------------------------------
// Entries of many equally shaped pools at once: for every pool and pair, entry dst <- entry src (K/V pages of all layers, recurrent
// states, conv windows).  An entry is n_sub sub-blocks of sub_bytes; the first `len` bytes of each are copied (len is per pair: the
// filled rows of a page).  Pool pointers and pairs travel as kernel arguments, so nothing is uploaded and a call can be captured.
// Bound: HBM (every byte once in, once out).  A block moves one 16 KiB chunk with four independent 16-byte accesses per thread; the
// pairs are the fastest index of the grid, so that the copies of one source (a fork) find its chunk in L2.  300 pages in 12 pools 74 us
// (6.4 TB/s read and write); a slot's states, windows and last pages into seven others, three launches, 31 us.
// ----------------------------------------------------------------------------------------------------------------------
constexpr int EC_THREADS = 256, EC_PER = 4;

template <typename T>
__global__ void __launch_bounds__(EC_THREADS) entries_copy_kernel(const __grid_constant__ EntriesArgs a, long long chunks) {
    const int pair = blockIdx.x % a.n_pairs;
    const long long rest = blockIdx.x / a.n_pairs;
    const long long chunk = rest % chunks;
    const int sub = (int)(rest / chunks);
    const long long len = (a.per_pair ? 2ll * a.len[pair] : a.len_all) / (long long)sizeof(T);
    const long long i0 = chunk * (EC_THREADS * EC_PER) + threadIdx.x;
    if (i0 >= len) return;
    char* pool = static_cast<char*>(a.pool[blockIdx.y]);
    const T* src = reinterpret_cast<const T*>(pool + a.src[pair] * a.entry_bytes + sub * a.sub_bytes);
    T* dst = reinterpret_cast<T*>(pool + a.dst[pair] * a.entry_bytes + sub * a.sub_bytes);
    T v[EC_PER];
#pragma unroll
    for (int k = 0; k < EC_PER; k++)
        if (i0 + k * EC_THREADS < len) v[k] = src[i0 + k * EC_THREADS];
#pragma unroll
    for (int k = 0; k < EC_PER; k++)
        if (i0 + k * EC_THREADS < len) dst[i0 + k * EC_THREADS] = v[k];
}

int launch_entries_copy(const EntriesArgs& a, int n_pools, cudaStream_t st) {
    long long longest = a.per_pair ? 0 : a.len_all;
    bool vec = a.entry_bytes % 16 == 0 && a.sub_bytes % 16 == 0 && longest % 16 == 0;
    for (int i = 0; i < a.n_pairs && a.per_pair; i++) {
        longest = 2ll * a.len[i] > longest ? 2ll * a.len[i] : longest;
        vec = vec && a.len[i] % 8 == 0;
    }
    for (int i = 0; i < n_pools; i++) vec = vec && reinterpret_cast<uintptr_t>(a.pool[i]) % 16 == 0;
    if (n_pools <= 0 || a.n_pairs <= 0 || longest <= 0) return GDN_OK;
    const long long unit = vec ? 16 : 2;                             // (element sizes are 2 or 4 bytes)
    const long long chunks = (longest / unit + EC_THREADS * EC_PER - 1) / (EC_THREADS * EC_PER);
    const long long blocks = chunks * a.n_sub * a.n_pairs;
    if (blocks > 0x7fffffffll) { set_error("entries_copy: %lld blocks in one launch", blocks); return GDN_E_SHAPE; }
    const dim3 grid((unsigned)blocks, n_pools);
    if (vec) entries_copy_kernel<uint4><<<grid, EC_THREADS, 0, st>>>(a, chunks);
    else entries_copy_kernel<uint16_t><<<grid, EC_THREADS, 0, st>>>(a, chunks);
    return check_launch("entries_copy");
}

// ----------------------------------------------------------------------------------------------------------------------
// Compaction of cached rows: row base[b] + keep[b][j] of sequence b moves to row base[b] + j, for every pool (K and V of all layers)
// and head.  keep is strictly ascending, so keep[j] >= j and a row is only ever overwritten after it was read: a thread owns a
// 16-byte column of a (pool, sequence, head) and walks the rows in order, eight loads in flight before their eight stores.  Bound:
// latency (a round keeps a handful of rows); the index words of 32 rows are fetched by the 32 lanes at once, so that the dependent
// chain is keep -> page -> row whatever the number of rows.  24 sequences, 12 pools, one to seven rows: 3.0 us.
// ----------------------------------------------------------------------------------------------------------------------
constexpr int RC_WARPS = 4, RC_ROWS = 8;

template <typename T>
__global__ void __launch_bounds__(32 * RC_WARPS) rows_compact_kernel(const __grid_constant__ RowsArgs a) {
    const int lane = threadIdx.x & 31;
    const int item = blockIdx.x * RC_WARPS + (threadIdx.x >> 5);     // (sequence, head); blockIdx.y = pool
    if (item >= a.B * a.heads) return;
    const int b = item / a.heads, h = item % a.heads;
    const int n = a.n_keep[b], base = a.base[b];
    const long long rows = (long long)a.max_pages * a.page_size;
    if (n < 0 || n > a.L || base < 0) { if (lane == 0) atomicExch(a.status, 1); return; }
    T* pool = static_cast<T*>(a.pool[blockIdx.y]);
    const long long row_units = a.row_bytes / (long long)sizeof(T);
    const int* keep = a.keep + (size_t)b * a.L;
    int before = -1;                                                 // last kept row of the rows already moved
    for (int j0 = 0; j0 < n; j0 += 32) {
        // lane l: where row j0 + l comes from and goes to (in rows of the pool), or "bad"
        const int j = j0 + lane, k = j < n ? keep[j] : 0x7fffffff;
        int prev = __shfl_up_sync(0xffffffffu, k, 1);
        if (lane == 0) prev = before;
        before = __shfl_sync(0xffffffffu, k, 31);
        long long from = 0, to = 0;
        bool ok = true;
        if (j < n) {
            const long long s = (long long)base + k, d = (long long)base + j;
            ok = k > prev && s < rows;
            if (ok) {
                const int sp = a.table[(size_t)b * a.max_pages + s / a.page_size], dp = a.dst_table[(size_t)b * a.max_pages + d / a.page_size];
                ok = sp >= 0 && sp < a.n_pages && dp >= 0 && dp < a.n_pages;
                from = ((long long)sp * a.heads + h) * a.page_size + s % a.page_size;
                to = ((long long)dp * a.heads + h) * a.page_size + d % a.page_size;
            }
        }
        const uint32_t bad = __ballot_sync(0xffffffffu, !ok);
        const int cnt = min(min(32, n - j0), bad ? __ffs(bad) - 1 : 32);      // rows from the first bad entry on stay where they are
        for (int r0 = 0; r0 < cnt; r0 += RC_ROWS) {
            long long f[RC_ROWS], t[RC_ROWS];
#pragma unroll
            for (int i = 0; i < RC_ROWS; i++) { f[i] = __shfl_sync(0xffffffffu, from, (r0 + i) & 31); t[i] = __shfl_sync(0xffffffffu, to, (r0 + i) & 31); }
            for (long long c = lane; c < row_units; c += 32) {
                T v[RC_ROWS];
#pragma unroll
                for (int i = 0; i < RC_ROWS; i++)
                    if (r0 + i < cnt && f[i] != t[i]) v[i] = pool[f[i] * row_units + c];
#pragma unroll
                for (int i = 0; i < RC_ROWS; i++)
                    if (r0 + i < cnt && f[i] != t[i]) pool[t[i] * row_units + c] = v[i];
            }
        }
        if (bad) { if (lane == 0) atomicExch(a.status, 1); return; }
    }
}

int launch_rows_compact(const RowsArgs& a, int n_pools, cudaStream_t st) {
    if (n_pools <= 0 || a.B <= 0 || a.L <= 0) return GDN_OK;
    bool vec = a.row_bytes % 16 == 0;
    for (int i = 0; i < n_pools; i++) vec = vec && reinterpret_cast<uintptr_t>(a.pool[i]) % 16 == 0;
    const dim3 grid((unsigned)(((long long)a.B * a.heads + RC_WARPS - 1) / RC_WARPS), n_pools);
    if (vec) rows_compact_kernel<uint4><<<grid, 32 * RC_WARPS, 0, st>>>(a);
    else rows_compact_kernel<uint16_t><<<grid, 32 * RC_WARPS, 0, st>>>(a);
    return check_launch("rows_compact");
}

}  // namespace gdn
