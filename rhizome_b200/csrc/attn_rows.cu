// Softmax attention of few query rows per sequence over the paged cache: one
// token or a small drafted tree, bf16, head widths 64 and 128.
//
// What bounds it is reading K and V once: a (sequence, K/V head) pair has at
// most 16 rows here, 16 multiply-adds to a byte, a sixteenth of what the tensor
// cores could take at HBM's rate. So the unit of work is one warp's: a chunk of
// one pair's keys (Split in attn_common.cuh), read in tiles of 32 keys that
// the warp's own ring of TMA copies brings in; no warp waits for another. The
// products run as mma.sync m16n8k16 from that ring (rows as m, so that every
// row of the group shares each K and V byte), the softmax stays in registers.
// Four warps with 48 KB in flight each keep an SM's share of HBM busy (44 KB
// would cover one microsecond of it). 512 sequences of U{1..8192} keys, one
// token, 32 heads over 8, pages of 16: 1,350 us, 6.2 TB/s, 0.95 of a plain copy's
// rate, and 26 us to join the chunks; 74 sequences of 8,192 keys and four tokens: 448 us,
// 5.5 TB/s (rows of masked nodes and one round of units more for some SMs).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "attn_common.cuh"
#include "attn_device.cuh"
#include "sm100.cuh"
#include "tmap.h"

namespace rhz {
namespace {

using namespace attn;

constexpr int WARPS = 4;
constexpr int KEYS = 32;         // keys of a tile
constexpr int STAGES = 3;        // tiles in a warp's ring
constexpr int MAX_SEQ = 4096;    // sequences of a launch: their chunk counts fit in shared memory

// Sticky: a bounded wait of this kernel ran out.
__device__ int g_rows_timeout;

// A unit as the warp's copying side hands it to its computing side.
struct Unit {
    int32_t seq, kvh, first, m, live, cached, kbeg, kend, chunk, chunks;
};
constexpr int UNITS = STAGES + 2;  // units that the copies may be ahead by, and the current one

struct RowsArgs {
    AttnArgs a;
    Parts parts;
    Split split;
    int group;
    int rows;   // rows per TMA box: min(page, 32)
    float c2;   // scale * log2 e
};

template <int D>
struct Cfg {
    static constexpr int TILE = KEYS * D * 2;        // K or V of a tile
    static constexpr int RING = STAGES * 2 * TILE;   // per warp
    static constexpr int OFF_CUM = WARPS * RING;     // prefix sums of the sequences' chunks
    static constexpr int OFF_UNITS = OFF_CUM + (MAX_SEQ + 4) * 4;
    static constexpr int OFF_BARS = OFF_UNITS + WARPS * UNITS * 64;
    static constexpr int OFF_VALID = OFF_BARS + WARPS * 32;
    static constexpr int OFF_SUMS = OFF_VALID + WARPS * 32;
    static constexpr int BYTES = OFF_SUMS + 64 + 1024;
};
static_assert(sizeof(Unit) <= 64 && STAGES <= 4, "shared-memory layout");

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
        "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Byte of (key, 16-byte piece c of its channels) in a tile: halves of 64
// channels, 128-byte rows, 128-byte swizzle.
__device__ __forceinline__ uint32_t piece_at(int key, int c) {
    return (c >> 3) * (KEYS * 128) + key * 128 + (((c & 7) ^ (key & 7)) << 4);
}

// Fragments (PTX, g = lane / 4, t = lane % 4): a score or
// output tile n holds rows g and g + 8, columns 8 n + 2 t and the next.
template <int D>
__global__ void __launch_bounds__(32 * WARPS, 1)
    attn_rows_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                     const __grid_constant__ RowsArgs g) {
    using C = Cfg<D>;
    extern __shared__ char smem_raw[];
    char *smem = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t{1023});
    const uint32_t base = sm100::smem_u32(smem);
    const AttnArgs &a = g.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int *cum = reinterpret_cast<int *>(smem + C::OFF_CUM);
    const int n_seq = static_cast<int>(a.n_seq);

    if (threadIdx.x < WARPS * STAGES) bar_init(base + C::OFF_BARS + 32 * (threadIdx.x / STAGES) + 8 * (threadIdx.x % STAGES), 1);
    sm100::mbar_fence_init();
    {
        // cum[i] = chunks of the sequences before i that have rows.
        int *sums = reinterpret_cast<int *>(smem + C::OFF_SUMS);
        int before = 0;
        for (int b = 0; b < n_seq; b += 32 * WARPS) {
            const int i = b + threadIdx.x;
            int c = 0;
            if (i < n_seq) {
                const Seq s = seq_of(a, i);
                c = s.m > 0 ? static_cast<int>(g.split.chunks(s.keys)) : 0;
            }
            int incl = c;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, incl, off);
                if (lane >= off) incl += y;
            }
            __syncthreads();
            if (lane == 31) sums[warp] = incl;
            __syncthreads();
            int at = before + incl - c;
            for (int w = 0; w < WARPS; ++w) {
                if (w < warp) at += sums[w];
                before += sums[w];
            }
            if (i < n_seq) cum[i] = at;
        }
        if (threadIdx.x == 0) cum[n_seq] = before;
        __syncthreads();
    }
    const int total = cum[n_seq] * a.Hkv;
    const int step = gridDim.x * WARPS;
    const uint32_t ring = base + warp * C::RING;
    const uint32_t bars = base + C::OFF_BARS + 32 * warp, valid_at = base + C::OFF_VALID + 32 * warp;
    Unit *units = reinterpret_cast<Unit *>(smem + C::OFF_UNITS + warp * UNITS * 64);
    auto unit_at = [&](int k) -> Unit & { return *reinterpret_cast<Unit *>(reinterpret_cast<char *>(units) + (k % UNITS) * 64); };

    // ---- the copying side: tile by tile through the warp's units
    int c_unit = blockIdx.x * WARPS + warp;  // index of the unit being copied
    int c_count = 0;                         // units begun
    int c_key = 0, c_end = 0, c_seq = 0, c_kvh = 0;
    uint32_t c_tile = 0;                     // tiles issued
    int c_ids = 0, c_page = -1000;           // this lane's block of the 32 pages from c_page on
    // The next unit with keys; units without any are begun too (their rows are
    // written), so the computing side sees every one. False past the last.
    auto begin_unit = [&]() -> bool {
        if (c_unit >= total) return false;
        const int x = c_unit / a.Hkv;
        int lo = 0, hi = n_seq;  // the last sequence with cum <= x that has chunks
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (cum[mid] <= x) lo = mid; else hi = mid;
        }
        const Seq s = seq_of(a, lo);
        Unit u;
        u.seq = lo;
        u.kvh = c_unit - x * a.Hkv;
        u.first = static_cast<int>(s.first);
        u.m = static_cast<int>(s.m);
        u.live = static_cast<int>(s.live);
        u.cached = static_cast<int>(s.cached);
        u.chunk = x - cum[lo];
        u.chunks = cum[lo + 1] - cum[lo];
        const int span = static_cast<int>(g.split.span(s.keys));
        u.kbeg = u.chunk * span;
        u.kend = min(static_cast<int>(s.keys), u.kbeg + span);
        __syncwarp();
        if (lane == 0) unit_at(c_count) = u;
        __syncwarp();
        ++c_count;
        c_unit += step;
        c_key = u.kbeg;
        c_end = s.live > 0 ? u.kend : u.kbeg;
        c_seq = u.seq;
        c_kvh = u.kvh;
        c_page = -1000;
        return true;
    };
    // Issues the next tile, if there is one and the computing side (at unit
    // k) is near enough that its descriptor has a place.
    auto copy = [&](int k) {
        while (c_key >= c_end) {
            if (c_count - k >= UNITS - 1 || !begin_unit()) return;
        }
        const int st = c_tile % STAGES;
        const int first = c_key >> a.shift;
        const int pieces = KEYS / g.rows;  // pages of a tile that come by boxes of their own
        const int last = (min(c_key + KEYS, c_end) - 1) >> a.shift;
        if (c_page < 0 || last >= c_page + 32) {
            c_page = first;
            c_ids = first + lane < a.width ? a.block_table[c_seq * a.width + first + lane] : -1;
        }
        const int key = c_key + lane * g.rows;  // of this lane's piece
        const int id = __shfl_sync(0xffffffffu, c_ids, min(max((key >> a.shift) - c_page, 0), 31));
        const bool there = lane < pieces && key < c_end && id >= 0 && id < a.num_blocks;
        const uint32_t mask = __ballot_sync(0xffffffffu, there);
        uint32_t valid = ~0u;
        if (__popc(mask) != pieces) valid = __ballot_sync(0xffffffffu, mask >> (lane / g.rows) & 1u);
        const uint32_t bar = bars + 8 * st;
        if (lane == 0) {
            sts(valid_at + 4 * st, valid);
            bar_expect(bar, __popc(mask) * g.rows * D * 4);
        }
        __syncwarp();
        if (there) {
            const int row = static_cast<int>(((static_cast<int64_t>(id) * a.Hkv + c_kvh) << a.shift) + (key & ((1 << a.shift) - 1)));
            const uint32_t dst = ring + st * 2 * C::TILE + lane * g.rows * 128;
#pragma unroll
            for (int h = 0; h < D / 64; ++h) {
                load_2d(dst + h * KEYS * 128, &tm_k, h * 64, row, bar);
                load_2d(dst + C::TILE + h * KEYS * 128, &tm_v, h * 64, row, bar);
            }
        }
        c_key += KEYS;
        ++c_tile;
    };

    // ---- the computing side
    const int gq = lane >> 2, tq = lane & 3;
    uint32_t tile = 0;
    // Fills the ring's free places.
    auto top_up = [&](int k) {
        while (c_tile - tile < STAGES) {
            const uint32_t was = c_tile;
            copy(k);
            if (c_tile == was) break;
        }
    };
    bool ok = true;
    for (int k = 0; ok; ++k) {
        if (k >= c_count && !begin_unit()) break;
        const Unit u = unit_at(k);
        __syncwarp();
        top_up(k);  // (the copies stop where too many units lie ahead: some may have no keys)
        // Q as A fragments, the rows' sight.
        uint32_t q[D / 16][4];
        int all[2];
        uint64_t bits[2];
        const int used = min(u.live, 16 / g.group) * g.group;  // rows with a token that takes part
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = gq + 8 * i, t = r / g.group, of = r - t * g.group;
            all[i] = 0;
            bits[i] = 0;
            const bool has = r < used;
            if (has) {
                if (a.parent) {
                    bits[i] = ancestors(a.parent + u.first, t);
                    all[i] = bits[i] ? u.cached : 0;
                } else {
                    all[i] = u.cached + t + 1;
                }
            }
            const __nv_bfloat16 *src = static_cast<const __nv_bfloat16 *>(a.q) + static_cast<int64_t>(u.first + t) * a.q_stride +
                                       static_cast<int64_t>(u.kvh * g.group + of) * D + 2 * tq;
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
                q[c][i & 1] = has ? *reinterpret_cast<const uint32_t *>(src + 16 * c) : 0u;
                q[c][2 + (i & 1)] = has ? *reinterpret_cast<const uint32_t *>(src + 16 * c + 8) : 0u;
            }
        }
        float acc[D / 8][4], top[2], sum[2];
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            top[i] = -INFINITY;
            sum[i] = 0.f;
        }
        bool bad = false;
        const int end = u.live > 0 ? u.kend : u.kbeg;
        // Keys below `full` are seen by every row that sees anything.
        const int full = a.parent ? u.cached : u.cached + 1;
        for (int key = u.kbeg; key < end; key += KEYS, ++tile) {
            const int st = tile % STAGES;
            const uint32_t bar = bars + 8 * st;
            bool came = bar_try(bar, (tile / STAGES) & 1);
            if (!came) {
                const uint32_t since = clock_ns();
                for (uint32_t i = 1; !came && ((i & 63u) != 0 || clock_ns() - since <= WAIT_NS); ++i) came = bar_try(bar, (tile / STAGES) & 1);
            }
            ok = __all_sync(0xffffffffu, came);
            if (!ok) {
                atomicExch(&g_rows_timeout, 1);
                break;
            }
            const uint32_t kt = ring + st * 2 * C::TILE, vt = kt + C::TILE;
            const uint32_t valid = lds(valid_at + 4 * st);
            const bool edge = valid != ~0u || key + KEYS > full;
            if (edge) {
                // V of keys behind the sequence or without a page becomes zero, and so do
                // values that are not finite where not every row looks; those are noted.
                const bool exists = key + lane < end && (valid >> lane & 1u);
                if (!exists || key + lane >= full) {
                    for (int c = 0; c < D / 8; ++c) {
                        const uint32_t at = vt + piece_at(lane, c);
                        if (!exists) {
                            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
                        } else {
                            uint32_t w[4];
                            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                                         : "r"(at)
                                         : "memory");
                            if (odd_word(w[0]) || odd_word(w[1]) || odd_word(w[2]) || odd_word(w[3])) {
                                bad = true;
                                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(finite_word(w[0])),
                                             "r"(finite_word(w[1])), "r"(finite_word(w[2])), "r"(finite_word(w[3]))
                                             : "memory");
                            }
                        }
                    }
                }
                sm100::fence_proxy_async_smem();  // before a copy writes here again
                __syncwarp();
            }
            // Scores: 4 tiles of 8 keys.
            float x[4][4];
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[n][e] = 0.f;
#pragma unroll
            for (int c = 0; c < D / 16; ++c)
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    uint32_t b[4];
                    ldsm4(b, kt + piece_at(16 * n + (lane & 7) + ((lane >> 4) << 3), 2 * c + ((lane >> 3) & 1)));
                    mma(x[2 * n], q[c], b[0], b[1]);
                    mma(x[2 * n + 1], q[c], b[2], b[3]);
                }
            // Softmax.
            uint32_t p[2][4];
            bool moved = false;
            float keep[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float best = top[i];
                uint32_t m = ~0u;
                if (edge) m = seen_word(all[i], bits[i], key) & valid;
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float &s = x[n][2 * i + e];
                        s *= g.c2;
                        if (edge && !(m >> (8 * n + 2 * tq + e) & 1u)) s = -INFINITY;
                        best = fmaxf(best, s);
                    }
                best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 1));
                best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 2));
                const float from = best == -INFINITY ? 0.f : best;
                keep[i] = best == top[i] ? 1.f : ex2(top[i] - from);
                moved |= best != top[i];
                top[i] = best;
                float part = 0.f;
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float &s = x[n][2 * i + e];
                        s = ex2(s - from);
                        part += s;
                    }
                sum[i] = sum[i] * keep[i] + part;
            }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int n = 0; n < D / 8; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[n][e] *= keep[e >> 1];
            }
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                p[n][0] = pack_bf16(x[2 * n][0], x[2 * n][1]);
                p[n][1] = pack_bf16(x[2 * n][2], x[2 * n][3]);
                p[n][2] = pack_bf16(x[2 * n + 1][0], x[2 * n + 1][1]);
                p[n][3] = pack_bf16(x[2 * n + 1][2], x[2 * n + 1][3]);
            }
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int c = 0; c < D / 16; ++c) {
                    uint32_t b[4];
                    ldsm4t(b, vt + piece_at(16 * n + (lane & 7) + (((lane >> 3) & 1) << 3), 2 * c + (lane >> 4)));
                    mma(acc[2 * c], p[n], b[0], b[1]);
                    mma(acc[2 * c + 1], p[n], b[2], b[3]);
                }
            __syncwarp();  // every lane has read the tile
            copy(k);
        }
        if (!ok) break;
        bool some[2];  // rows that see a key
        const bool split = u.chunks > 1;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float l = sum[i];
            l += __shfl_xor_sync(0xffffffffu, l, 1);
            l += __shfl_xor_sync(0xffffffffu, l, 2);
            const int r = gq + 8 * i, t = r / g.group, of = r - t * g.group;
            const bool none = all[i] == 0 && bits[i] == 0;
            if (none) l = 0.f;  // sees nothing: whole tiles did not ask
            // (Where every score is -inf the row is zeros, whatever 0 * inf left in the sums; a chunk keeps that for the join.)
            some[i] = r < used && !none && (split || l != 0.f);
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const float l2 = l == 0.f ? -INFINITY : top[i] + log2f(l);
            if (r >= used) continue;
            const int64_t token = u.first + t;
            const int head = u.kvh * g.group + of;
            if (split) {
                const int64_t row = g.parts.row(u.chunk, token, head);
                if (tq == 0) g.parts.lse[row] = l2;
                float2 *dst = reinterpret_cast<float2 *>(g.parts.o + row * D + 2 * tq);
#pragma unroll
                for (int n = 0; n < D / 8; ++n)
                    dst[4 * n] = none ? make_float2(0.f, 0.f) : make_float2(acc[n][2 * i] * inv, acc[n][2 * i + 1] * inv);
            } else {
                if (tq == 0 && a.lse) a.lse[token * a.H + head] = l2 * LN2;
                uint32_t *dst = reinterpret_cast<uint32_t *>(static_cast<__nv_bfloat16 *>(a.o) + (token * a.H + head) * D + 2 * tq);
#pragma unroll
                for (int n = 0; n < D / 8; ++n)
                    dst[4 * n] = l == 0.f ? 0u : pack_bf16(acc[n][2 * i] * inv, acc[n][2 * i + 1] * inv);
            }
        }
        if (__any_sync(0xffffffffu, bad)) {
            const int r = lane & 15, t = r / g.group;  // lane r takes row r
            const bool some0 = __shfl_sync(0xffffffffu, static_cast<int>(some[0]), 4 * (lane & 7));
            const bool some1 = __shfl_sync(0xffffffffu, static_cast<int>(some[1]), 4 * (lane & 7));
            add_odd_values<D>(a, g.parts, {u.first, u.m, u.live, u.cached, u.cached + u.live}, {u.seq, u.kvh, u.chunk, u.chunks},
                              max(full, u.kbeg), end, lane < 16 && (lane & 8 ? some1 : some0), t, u.kvh * g.group + (r - t * g.group), lane);
        }
        if (u.chunk == 0) {
            if (g.parts.count && u.kvh == 0)
                for (int t = lane; t < u.m; t += 32) g.parts.count[u.first + t] = t * g.group < used ? u.chunks : 1;
            // Rows that take no part.
            for (int64_t r = used; r < static_cast<int64_t>(u.m) * g.group; ++r) {
                const int64_t token = u.first + r / g.group;
                const int head = u.kvh * g.group + static_cast<int>(r % g.group);
                if (lane == 0 && a.lse) a.lse[token * a.H + head] = -INFINITY;
                uint32_t *dst = reinterpret_cast<uint32_t *>(static_cast<__nv_bfloat16 *>(a.o) + (token * a.H + head) * D);
                for (int c = lane; c < D / 2; c += 32) dst[c] = 0u;
            }
        }
    }
    if (!ok)  // copies in flight land before the CTA leaves
        for (uint32_t t = tile; t < c_tile; ++t)
            for (uint32_t i = 0; i < (1u << 20) && !bar_try(bars + 8 * (t % STAGES), (t / STAGES) & 1); ++i) {
            }
}

template <int D>
int launch_t(const AttnArgs &a, const Parts &parts, Split split) {
    RowsArgs g{};
    g.a = a;
    g.parts = parts;
    g.split = split;
    g.group = a.H / a.Hkv;
    const int page = 1 << a.shift;
    g.rows = page < KEYS ? page : KEYS;
    g.c2 = a.scale * LOG2E;
    CUtensorMap tk, tv;
    const uint64_t d[2] = {D, static_cast<uint64_t>(a.num_blocks * a.Hkv) << a.shift};
    const uint64_t s[1] = {D * 2};
    const uint32_t b[2] = {64, static_cast<uint32_t>(g.rows)};
    int st = encode_tmap(&tk, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.k, d, s, b, CU_TENSOR_MAP_SWIZZLE_128B);
    if (st == RHZ_OK) st = encode_tmap(&tv, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.v, d, s, b, CU_TENSOR_MAP_SWIZZLE_128B);
    if (st != RHZ_OK) return st;
    int sms = 148;
    bool sm100 = true;
    st = device_info(&sms, &sm100);
    if (st != RHZ_OK) return st;
    const int64_t units = a.n_seq * a.Hkv * parts.most;  // at most
    if (units > INT32_MAX) return set_error(RHZ_ERR_SHAPE, "attention over %lld units exceeds int32 indexing", (long long)units);
    const int64_t ctas = (units + WARPS - 1) / WARPS;
    const unsigned grid = static_cast<unsigned>(ctas < sms ? ctas : sms);
    cudaError_t e = cudaFuncSetAttribute(attn_rows_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::BYTES);
    if (e != cudaSuccess) return set_error(RHZ_ERR_DEVICE, "attn_rows_kernel: %s", cudaGetErrorString(e));
    attn_rows_kernel<D><<<grid, 32 * WARPS, Cfg<D>::BYTES, a.stream>>>(tk, tv, g);
    return check_launch("attn_rows_kernel");
}

}  // namespace

// One 16-row tile: with two, 74 sequences of 8,192 keys and 32 rows took 1,088 us
// here and 552 us as a row tile of the tcgen05 form.
bool attn_rows_supports(const AttnArgs &a) {
    return a.paged && a.dtype == RHZ_DTYPE_BF16 && (a.d == 64 || a.d == 128) && a.most * (a.H / a.Hkv) <= 16;
}

int launch_attn_rows(const AttnArgs &a, const Parts &parts, Split split) {
    int st = RHZ_OK;
    for (int64_t from = 0; st == RHZ_OK && from < a.n_seq; from += MAX_SEQ) {  // rows, parents and partial results go by token
        AttnArgs g = a;
        g.n_seq = a.n_seq - from < MAX_SEQ ? a.n_seq - from : MAX_SEQ;
        g.cu_seqlens += from;
        g.cached += from;
        g.block_table += from * a.width;
        st = a.d == 128 ? launch_t<128>(g, parts, split) : launch_t<64>(g, parts, split);
    }
    return st;
}

int attn_rows_status(int *flag, bool clear) {
    cudaError_t e = cudaMemcpyFromSymbol(flag, g_rows_timeout, sizeof(int));
    if (e == cudaSuccess && clear && *flag) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_rows_timeout, &zero, sizeof(int));
    }
    if (e != cudaSuccess) return set_error(RHZ_ERR_DEVICE, "attention status: %s", cudaGetErrorString(e));
    return RHZ_OK;
}

}  // namespace rhz
