// The paged K/V cache of the Global blocks: block tables and slot maps of an
// engine step from request lengths, and the rows of the step's tokens written
// by them. Pages hold `page` positions of every head, [H][page][d], so one
// page of one head is a contiguous run for the attention that reads it.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "common.cuh"
#include "kernels.h"

namespace rhz {
namespace {

// ------------------------------------------------------------------ block tables and slot maps

constexpr int TABLE_THREADS = 512;   // requests per scan step, one per thread
constexpr int TABLE_ROWS = 1024;     // slot-map rows per CTA

// Exclusive scan of one int64 per thread over the CTA, the total to `total`.
__device__ __forceinline__ int64_t scan_exclusive(int64_t x, int64_t *sums, int64_t &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int NW = TABLE_THREADS / 32;
    int64_t incl = x;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += y;
    }
    __syncthreads();  // the sums of the scan before have been read
    if (lane == 31) sums[warp] = incl;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        const int64_t s = sums[w];
        if (w < warp) before += s;
        total += s;
    }
    return before + incl - x;
}

// With need_i = pages request i lacks for its cached + fresh positions and
// off_i = cursor + sum of need over the requests before it, request i gets
// the free-list entries [off_i, off_i + granted_i), granted_i =
// clamp(num_free - off_i, 0, need_i).
//
// Bound by latency: 20 bytes a request in, 8 a token out. So it is one launch
// without any exchange between CTAs: every CTA scans all requests itself (from
// L2, 512 per step) and then writes only its share of the slot map, of the new
// table entries and, CTA 0, the per-request results. A slot takes its page
// from the table where the request held it before the call and from the free
// list where it is new, so no CTA reads what another writes.
__global__ void __launch_bounds__(TABLE_THREADS) kv_tables_kernel(const KvTablesArgs a, int shift) {
    __shared__ int64_t s_sums[TABLE_THREADS / 32];
    __shared__ int64_t s_row[TABLE_THREADS];       // first slot-map row of each request of the step
    __shared__ int64_t s_off[TABLE_THREADS];       // its free-list offset
    __shared__ int32_t s_cached[TABLE_THREADS], s_held[TABLE_THREADS], s_now[TABLE_THREADS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t start = a.cursor ? max(*a.cursor, 0) : 0;
    // Rows of the slot map that this CTA writes.
    const int64_t per = (a.max_tokens + gridDim.x - 1) / gridDim.x;
    const int64_t lo = min(blockIdx.x * per, a.max_tokens), hi = min(lo + per, a.max_tokens);
    int64_t rows = 0, off = start, taken = 0, missing = 0;  // carried over the steps
    for (int64_t base = 0; base < a.n; base += TABLE_THREADS) {
        const int64_t i = base + tid;
        const bool in = i < a.n;
        const int64_t cached = in ? max(a.cached[i], 0) : 0, fresh = in ? max(a.fresh[i], 0) : 0;
        const int64_t held = in ? min(static_cast<int64_t>(max(a.held[i], 0)), a.width) : 0;
        const int64_t wanted = fresh > 0 ? (cached + fresh + (int64_t{1} << shift) - 1) >> shift : 0;
        const int64_t need = max(min(wanted, a.width) - held, int64_t{0});
        int64_t total_rows, total_need;
        const int64_t row = rows + scan_exclusive(fresh, s_sums, total_rows);
        const int64_t at = off + scan_exclusive(need, s_sums, total_need);
        const int64_t granted = min(max(a.num_free - at, int64_t{0}), need);
        s_row[tid] = row;
        s_off[tid] = at;
        s_cached[tid] = static_cast<int32_t>(cached);
        s_held[tid] = static_cast<int32_t>(held);
        s_now[tid] = static_cast<int32_t>(held + granted);
        if (blockIdx.x == 0) {
            if (in) {
                a.cu_seqlens[i] = static_cast<int32_t>(row);
                a.held_out[i] = static_cast<int32_t>(held + granted);
            }
            taken += granted;
            missing += max(wanted - held, int64_t{0}) - granted;
        }
        __syncthreads();
        const int count = static_cast<int>(min(a.n - base, static_cast<int64_t>(TABLE_THREADS)));
        // New table entries: a warp per request of this CTA's share.
        const int64_t nw = static_cast<int64_t>(gridDim.x) * (TABLE_THREADS / 32);
        for (int64_t r = warp * static_cast<int64_t>(gridDim.x) + blockIdx.x; r < count; r += nw)
            for (int p = s_held[r] + lane; p < s_now[r]; p += 32)
                a.block_table[(base + r) * a.width + p] = a.free_blocks[s_off[r] + p - s_held[r]];
        // Slots of this CTA's rows that belong to the step's requests.
        const int64_t b = max(lo, rows), e = min(hi, rows + total_rows);
        for (int64_t t = b + tid; t < e; t += TABLE_THREADS) {
            int x = 0, y = count;  // the last request whose first row is <= t
            while (y - x > 1) {
                const int mid = (x + y) >> 1;
                if (s_row[mid] <= t) x = mid; else y = mid;
            }
            const int64_t pos = s_cached[x] + (t - s_row[x]);
            const int64_t p = pos >> shift;
            int32_t block = -1;
            if (p < s_held[x]) block = a.block_table[(base + x) * a.width + p];
            else if (p < s_now[x]) block = a.free_blocks[s_off[x] + p - s_held[x]];
            a.slot_map[t] = block < 0 ? -1 : (static_cast<int64_t>(block) << shift) + (pos & ((1 << shift) - 1));
        }
        rows += total_rows;
        off += total_need;
    }
    for (int64_t t = max(lo, rows) + tid; t < hi; t += TABLE_THREADS) a.slot_map[t] = -1;
    if (blockIdx.x == 0) {
        int64_t all_taken, all_missing;
        scan_exclusive(taken, s_sums, all_taken);
        scan_exclusive(missing, s_sums, all_missing);
        if (tid == 0) {
            a.cu_seqlens[a.n] = static_cast<int32_t>(rows);
            *a.cursor_out = static_cast<int32_t>(start + all_taken);
            *a.missing = static_cast<int32_t>(min(all_missing, static_cast<int64_t>(INT32_MAX)));
        }
    }
}

// ------------------------------------------------------------------ append

// One warp per token: the slot is one load, and the token's K and V rows (kv
// heads of d channels, contiguous) move as V-byte vectors, four of each tensor
// in flight per lane. Bound by HBM: every byte is read once and written once.
template <typename V>
__global__ void __launch_bounds__(256) kv_append_kernel(const KvAppendArgs a, int elem, int shift) {
    const int lane = threadIdx.x & 31;
    const int64_t t = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    if (t >= a.tokens) return;
    const int64_t slot = a.slot_map[t];
    const int64_t block = slot >> shift;
    if (slot < 0 || block >= a.num_blocks) return;
    const int per_head = a.d * elem / static_cast<int>(sizeof(V)), per_row = per_head * a.H;
    const V *ks = reinterpret_cast<const V *>(static_cast<const char *>(a.k) + t * a.k_stride * elem);
    const V *vs = reinterpret_cast<const V *>(static_cast<const char *>(a.v) + t * a.v_stride * elem);
    // [block][head][row][d]: heads are page * d apart.
    const int64_t at = ((block * a.H << shift) + (slot & ((1 << shift) - 1))) * per_head;
    V *kd = static_cast<V *>(a.k_cache) + at, *vd = static_cast<V *>(a.v_cache) + at;
    constexpr int U = 4;
    for (int j0 = lane; j0 < per_row; j0 += 32 * U) {
        V kx[U], vx[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + 32 * u;
            if (j < per_row) {
                kx[u] = __ldcs(ks + j);
                vx[u] = __ldcs(vs + j);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + 32 * u;
            if (j < per_row) {
                const int head = j / per_head;
                const int64_t to = (static_cast<int64_t>(head) << shift) * per_head + (j - head * per_head);
                kd[to] = kx[u];
                vd[to] = vx[u];
            }
        }
    }
}

int log2_of(int x) {
    int s = 0;
    while ((1 << s) < x) ++s;
    return s;
}

}  // namespace

int launch_kv_tables(const KvTablesArgs &a) {
    int64_t grid = (a.max_tokens + TABLE_ROWS - 1) / TABLE_ROWS;
    if (grid < 1) grid = 1;
    if (grid > 148 * 4) grid = 148 * 4;  // four CTAs of 512 threads fill an SM
    kv_tables_kernel<<<static_cast<unsigned>(grid), TABLE_THREADS, 0, a.stream>>>(a, log2_of(a.page));
    return check_launch("kv_tables_kernel");
}

int launch_kv_append(const KvAppendArgs &a) {
    if (a.tokens == 0) return RHZ_OK;
    const int elem = a.dtype == RHZ_DTYPE_BF16 ? 2 : 4;
    // 16-byte vectors need every row of either side on a 16-byte boundary;
    // d % 4 == 0 leaves at least 8 otherwise.
    const bool wide = (a.d * elem) % 16 == 0 && (a.k_stride * elem) % 16 == 0 &&
                      (a.v_stride * elem) % 16 == 0 && aligned(a.k, 16) && aligned(a.v, 16);
    // A warp per token; two tokens to a CTA while there are few, so that a
    // decode step's rows spread over the SMs.
    const int warps = a.tokens < 148 * 16 ? 2 : 8;
    const unsigned grid = static_cast<unsigned>((a.tokens + warps - 1) / warps);
    if (wide)
        kv_append_kernel<uint4><<<grid, 32 * warps, 0, a.stream>>>(a, elem, log2_of(a.page));
    else
        kv_append_kernel<uint2><<<grid, 32 * warps, 0, a.stream>>>(a, elem, log2_of(a.page));
    return check_launch("kv_append_kernel");
}

}  // namespace rhz
