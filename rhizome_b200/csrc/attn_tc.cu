// Softmax attention with grouped heads on the 5th-generation tensor cores:
// bf16, head widths 64 and 128, packed causal prompts and drafted trees (or
// pieces of a prompt) over the paged cache.
//
// One persistent CTA per SM works through units: 2 x 128 query rows (two
// tiles) of one (sequence, K/V head), over that pair's keys or a chunk of
// them, 64 keys at a time:
//   S_x = Q_x K^T            (tcgen05, both operands in shared memory, f32 in TMEM)
//   P_x = exp2(c S_x - c m)  (one warpgroup per tile, a thread per row)
//   O_x += P_x V             (tcgen05, P as a bf16 A operand in TMEM, over S's columns)
// P is rounded to bf16 because the product takes one type, the type of V; its
// sum is taken in f32 before the rounding. The maximum m is kept lazily: it is
// looked for only when a step's sum exceeds 2^16 (so the one in use may lag by as
// much), and then O is rescaled only if it has grown by more than 2^8.
//
// Roles: warps 0-3 and 4-7 the softmax of tiles 0 and 1, warps 8 and 9 the
// products of a tile each, warp 10 copies Q and K, warp 11 resolves units ahead
// of the others and copies V. Scores are held twice per tile, so the order
// PV_x(e), QK_x(e + 2) lets the tensor cores work on one step while the softmax
// is on another, and S_x(e + 2) complete implies PV_x(e) complete.
//
// What bounds it: no one pipe, but the chain of scores, softmax, probabilities
// and product of each row tile. Of a step of 2 x 128 x 64 products at d = 128 the
// tensor pipe needs 1,024 cycles at its rate (8 PV products of 64 cycles, 16 QK of
// 32; a QK product, both operands from shared memory, takes 51 alone and 36
// between PV products, so 1,090 to 1,330), the exponentials 1,024 of the SM's 16
// special-function lanes. A step takes 1,660 cycles in one prompt of 32,768 tokens
// (both pipes 62% active) and 1,790 in 16 packed ones (57%); an instruction waits
// 2.5 cycles for the one before it and 1.8 for memory, tensor memory mostly. One prompt
// of 32,768 tokens (32 heads over 8): 7.2 ms in a launch of its own, 8.2 ms among
// others under the power cap, 1.1 PFLOP/s, 0.66 of a large library product. Steps
// of 64 keys with P and S held twice took 8.16 ms where steps of 128 took 8.73, an
// issuing thread per tile and operands in uniform registers 7.86. Measured and
// not kept, on the 128-key form: part of the exponentials as polynomials on the
// FMA pipe (9.06 -> 9.30 ms and more with the share), the two tiles taking turns
// at the exponentials (8.73 -> 8.80 ms).
// Over the cache with one row tile only one of the softmax warpgroups works, 64
// keys in 0.88 us per SM: 74 sequences of 8,192 keys and 32 rows 552 us, of which
// reading them once is 379.
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
using namespace sm100;

constexpr int ROWS = 128;   // query rows of a tile
constexpr int KEYS = 64;    // keys of a step
constexpr int THREADS = 384;
constexpr int WARP_MMA = 8, WARP_TMA = 10, WARP_SCHED = 11;  // (two of the first)
constexpr int GROUP = 192;  // sequences whose unit counts the scheduler holds at a time
constexpr float FREE = 65536.f;  // 2^16: probabilities may reach this against a maximum that was not looked for
constexpr float LAZY = 8.f; // a row's maximum may grow by 2^LAZY before O is rescaled

// Sticky: a bounded wait of this kernel ran out.
__device__ int g_attn_timeout;

// A unit, resolved by the scheduler warp.
struct Unit {
    int32_t valid;
    int32_t seq, kvh;
    int32_t first, t0, m, live;  // query rows: first row, this unit's first token, tokens, those taking part
    int32_t cached, keys;        // keys before the sequence's own, and in all
    int32_t kbeg, n0, n1;        // first key, steps of either row tile
    int32_t chunk, chunks;
};

template <int D>
struct Cfg {
    static constexpr int HALVES = D / 64;                  // 64 channels: one 128-byte row
    static constexpr int Q_TILE = ROWS * D * 2;
    static constexpr int TILE = KEYS * D * 2;              // K or V of a step
    static constexpr int STAGES = D == 128 ? 4 : 8;        // of either in flight
    static constexpr int OFF_Q = 0;
    static constexpr int OFF_K = 2 * Q_TILE;
    static constexpr int OFF_V = OFF_K + STAGES * TILE;
    static constexpr int OFF_OUT = OFF_V + STAGES * TILE;  // 4 KB per softmax warp: output rows on their way out
    static constexpr int OFF_BAR = OFF_OUT + 8 * 4096;     // barriers, units, scheduler's counts
    static constexpr int OFF_UNIT = OFF_BAR + 448;
    static constexpr int OFF_MASK = OFF_UNIT + 256;
    static constexpr int OFF_MISC = OFF_MASK + 128;
    static constexpr int OFF_COUNT = OFF_MISC + 64;
    static constexpr int BYTES = OFF_COUNT + GROUP * 5 + 1024;
    static constexpr uint32_t ID_QK = idesc_bf16(ROWS, KEYS, false, false);
    static constexpr uint32_t ID_PV = idesc_bf16(ROWS, D, false, true);
};

// Barriers, 8 bytes each, from OFF_BAR. Everything in shared memory that the
// main loop touches is addressed by 32-bit addresses: as generic pointers the
// loop's invariants alone would push its score registers out to memory.
enum Bar : uint32_t {
    K_FULL = 0, K_EMPTY = 8, V_FULL = 16, V_EMPTY = 24, Q_FULL = 32, Q_EMPTY = 33,
    S_FULL = 34, P_FULL = 38,  // [row tile][parity of the step]
    PV_DONE = 42, O_FULL = 44, // [row tile]: a step's output product, a unit's last
    U_FULL = 46, U_EMPTY = 50, DRAIN = 54, NUM_BARS = 55
};
static_assert(NUM_BARS * 8 <= 448 && 4 * sizeof(Unit) <= 256, "shared-memory layout");

struct TcArgs {
    AttnArgs a;
    Parts parts;
    Split split;
    int tok;     // tokens of a row tile: 128 / group
    int group;   // query heads per K/V head
    int rows_shift;  // log2 of the rows per TMA box of a paged step
    float c2;    // scale * log2 e
};

__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(one));
    return one != 0;
}

// D[tmem] (+)= A * B, bf16 with f32 sums: descriptors as their low words and
// the high word that they share; A in shared memory, or in tensor memory.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, bool more) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d),
        "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(static_cast<uint32_t>(more))
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t hi, uint32_t idesc, bool more) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "mov.b64 b, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
        "r"(a_tmem), "r"(b_lo), "r"(hi), "r"(idesc), "r"(static_cast<uint32_t>(more))
        : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// Bounded wait of one thread (WAIT_NS) that also ends when another role gave up;
// *stop in shared memory tells the others.
__device__ __forceinline__ bool wait1(uint32_t bar, uint32_t parity, uint32_t stop) {
    uint32_t since = 0;
    for (uint32_t i = 0; !bar_try(bar, parity); ++i) {
        if ((i & 63u) != 63u) continue;
        if (lds(stop) != 0) return false;
        const uint32_t now = clock_ns();
        if (i == 63u) since = now;
        if (now - since > WAIT_NS) {
            sts(stop, 1);
            atomicExch(&g_attn_timeout, 1);
            return false;
        }
    }
    return true;
}

// For copies and products in flight when a role gave up: bounded the same way.
__device__ __forceinline__ void drain_wait(uint32_t bar, uint32_t parity) {
    for (uint32_t i = 0; i < (1u << 20) && !bar_try(bar, parity); ++i) {
    }
}

// The same for a whole warp: all its lanes go on or none does.
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, uint32_t stop) {
    return __all_sync(0xffffffffu, wait1(bar, parity, stop));
}

// (a * b + c) on two f32 at once.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t &>(d))
        : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)),
          "l"(reinterpret_cast<uint64_t &>(c)));
    return d;
}

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t &>(d))
        : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)));
    return d;
}

// 8 consecutive 32-bit columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&v)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(taddr));
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(v[0]),
                 "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// V of a step that not every row sees whole, a step's 64 keys by a warpgroup,
// two threads to a key: rows behind the sequence or without a page become
// zero, and so do values that are not finite at keys from `full` on, which are
// noted at `spoiled`. (A probability of zero does not keep them out of a
// product.) Both row tiles read these keys, so `full` is the unit's, and each
// tile's warpgroup cleans every such step before its own product. What one has
// replaced the other no longer finds, so the note comes first.
template <int D, bool PAGED>
__device__ __forceinline__ void clean_values(uint32_t tile, uint32_t mask, int key, int keys, int full, int r,
                                             uint32_t spoiled, int mark) {
    const int kr = r >> 1;
    const uint32_t vrow = tile + kr * 128 + (D == 128 ? (r & 1) * (KEYS * 128) : 0);
    const bool exists = key + kr < keys && (!PAGED || (lds(mask + 4 * (kr >> 5)) >> (kr & 31) & 1u));
    if (!exists || key + kr >= full) {
#pragma unroll 1
        for (int c = 0; c < D / 16; ++c) {  // 16-byte pieces; lanes start at different ones: different banks
            const int piece = D == 128 ? ((c + kr) & 7) : ((c + kr) & 3) + 4 * (r & 1);
            const uint32_t at = vrow + piece * 16;
            if (!exists) {
                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
            } else {
                uint32_t ws[4];
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(ws[0]), "=r"(ws[1]), "=r"(ws[2]), "=r"(ws[3])
                             : "r"(at)
                             : "memory");
                if (odd_word(ws[0]) || odd_word(ws[1]) || odd_word(ws[2]) || odd_word(ws[3])) {
                    sts(spoiled, mark);
                    __threadfence_block();
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(finite_word(ws[0])), "r"(finite_word(ws[1])),
                                 "r"(finite_word(ws[2])), "r"(finite_word(ws[3]))
                                 : "memory");
                }
            }
        }
    }
    fence_proxy_async_smem();
}

template <int D, bool PAGED>
__global__ void __launch_bounds__(THREADS, 1)
    attn_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                   const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ TcArgs g) {
    using C = Cfg<D>;
    extern __shared__ char smem_raw[];
    char *smem = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t{1023});
    const uint32_t base = smem_u32(smem);
    const uint32_t bars = base + C::OFF_BAR, abort = base + C::OFF_MISC + 4;
    Unit *units = reinterpret_cast<Unit *>(smem + C::OFF_UNIT);
    // Keys of a step with memory behind them, 8 bytes a step, 16 steps (K's copies,
    // which write it, are at most two steps more than its ring ahead of any softmax that reads).
    const uint32_t masks = base + C::OFF_MASK;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + C::OFF_MISC);
    // Unit i met values that are not finite where not every row sees them: word
    // i & 3 is i + 1. (Unit i + 4 comes when every warp is done with i.)
    const uint32_t spoiled = base + C::OFF_MISC + 16;
    int *counts = reinterpret_cast<int *>(smem + C::OFF_COUNT);
    uint8_t *costs = reinterpret_cast<uint8_t *>(counts + GROUP);
    const AttnArgs &a = g.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::STAGES; ++i) {
            bar_init(bars + 8 * (K_FULL + i), 1);
            bar_init(bars + 8 * (K_EMPTY + i), 2);
            bar_init(bars + 8 * (V_FULL + i), 1);
            bar_init(bars + 8 * (V_EMPTY + i), 2);
        }
        bar_init(bars + 8 * Q_FULL, 1);
        bar_init(bars + 8 * Q_EMPTY, 2);
        for (int x = 0; x < 2; ++x) {
            bar_init(bars + 8 * (PV_DONE + x), 1);
            bar_init(bars + 8 * (O_FULL + x), 1);
            for (int h = 0; h < 2; ++h) {
                bar_init(bars + 8 * (S_FULL + 2 * x + h), 1);
                bar_init(bars + 8 * (P_FULL + 2 * x + h), 4);
            }
        }
        for (int i = 0; i < 4; ++i) {
            bar_init(bars + 8 * (U_FULL + i), 1);
            bar_init(bars + 8 * (U_EMPTY + i), WARP_SCHED);
        }
        bar_init(bars + 8 * DRAIN, 2);
        sts(abort, 0);
        for (int i = 0; i < 4; ++i) sts(spoiled + 4 * i, 0);
        mbar_fence_init();
    }
    if (warp == WARP_MMA) tmem_alloc(tmem_slot, 512);
    if (warp == WARP_TMA && lane == 0) {
        prefetch_tmap(&tm_q);
        prefetch_tmap(&tm_k);
        prefetch_tmap(&tm_v);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    // Units come through a ring of four. The copying and the issuing warps take
    // theirs out at once, the softmax warps leave it there until they are done.
    auto next_unit = [&](int i, Unit &u) -> bool {
        if (!wait(bars + 8 * (U_FULL + (i & 3)), (i >> 2) & 1, abort)) return false;
        u = units[i & 3];
        __syncwarp();
        if (lane == 0) bar_arrive(bars + 8 * (U_EMPTY + (i & 3)));
        return u.valid != 0;
    };

    // 384 x 168 registers at launch: 256 x 208 for the softmax, 128 x 88 for the rest.
    if (warp < WARP_MMA) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        // Softmax of tile x: thread r of the warpgroup is row r.
        const int x = warp >> 2, r = threadIdx.x & 127;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + x * 128, to = tmem + lanes + 256 + x * 128;
        uint32_t sn = 0, on = 0, it = 0;  // steps and units done (mod 2^32) of this row tile, steps before the unit
        uint32_t sp = 0;          // phases of S_FULL waited for, one bit per half
        const int row_token = r / g.group, row_head = r - row_token * g.group;
        for (int i = 0; wait(bars + 8 * (U_FULL + (i & 3)), (i >> 2) & 1, abort); ++i) {
            const Unit &u = units[i & 3];
            if (!u.valid) break;
            const int token = u.t0 + x * g.tok + row_token;
            const bool used = row_token < g.tok && token < u.m;
            int all = 0;         // what the row sees: keys below `all`, and of the 64 from there on those in `bits`
            uint64_t bits = 0;
            if (used && token < u.live) {
                if (PAGED && a.parent) {
                    bits = ancestors(a.parent + u.first, token);
                    all = bits ? u.cached : 0;
                } else {
                    all = u.cached + token + 1;
                }
            }
            // Tiles below `full` are seen whole by every live row of the warpgroup's tile.
            const int full = PAGED && a.parent ? u.cached : u.cached + u.t0 + x * g.tok + 1;
            auto full_both = [&]() { return u.cached + (PAGED && a.parent ? 0 : u.t0 + 1); };  // and by those of both tiles
            const int kbeg = u.kbeg;
            const bool sees = all > 0 || bits != 0;  // (rows that do not are computed and thrown away)
            float top = -INFINITY, sum = 0.f;
            bool ok = true;
            const int n = x ? u.n1 : u.n0;
            // Halves that every live row sees whole.
            const int whole = min(max(full - kbeg, 0) / KEYS, n);
            const int clean = max(full_both() - kbeg, 0) / KEYS;  // steps before this one need no clean_values
            bool loaded = false;  // v holds step e's scores
            float v[2][32];
            auto load = [&](int h) {
                tc_fence_after();
#pragma unroll
                for (int w = 0; w < 2; ++w) tmem_ld32(ts + KEYS * h + 32 * w, v[w]);
            };
            for (int e = 0; e < n; ++e, ++sn) {
                const int h = e & 1, key = kbeg + e * KEYS;
                bool edge = e >= whole;
                if (!loaded) {
                    ok = wait(bars + 8 * (S_FULL + 2 * x + h), sp >> h & 1, abort);
                    if (!ok) break;
                    load(h);
                }
                uint32_t there[2] = {~0u, ~0u};
                const uint32_t nth = it + e;
                if (PAGED) {
                    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];"
                                 : "=r"(there[0]), "=r"(there[1])
                                 : "r"(masks + 8 * (nth & 15))
                                 : "memory");
                    edge |= (there[0] & there[1]) != ~0u;
                }
                if (edge || e >= clean) {
                    // Not before the scores are there: only then is V's place in the ring
                    // at most one lap from its turn, and the parity tells. (A warpgroup
                    // without steps in a unit runs ahead of the ring.)
                    const int vs = nth % C::STAGES;
                    ok = wait(bars + 8 * (V_FULL + vs), (nth / C::STAGES) & 1, abort);
                    if (!ok) break;
                    clean_values<D, PAGED>(base + C::OFF_V + vs * C::TILE, masks + 8 * (nth & 15), key, u.keys, full_both(), r, spoiled + 4 * (i & 3), i + 1);
                }
                tmem_wait_ld();
                sp ^= 1u << h;
                loaded = false;
                const float2 c2 = make_float2(g.c2, g.c2);
                float2 part[2];
                uint32_t p[32];
                // p = exp2(c s - c top) and its sum.
                auto exponentials = [&]() {
                    const float from = top == -INFINITY ? 0.f : -top * g.c2;
                    const float2 f2 = make_float2(from, from);
                    part[0] = part[1] = make_float2(0.f, 0.f);
#pragma unroll
                    for (int b = 0; b < 32; b += 8) {
                        float2 y[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const int c = 2 * (b + k);
                            y[k] = fma2(make_float2(v[c / 32][c % 32], v[c / 32][c % 32 + 1]), c2, f2);
                        }
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            y[k].x = ex2(y[k].x);
                            y[k].y = ex2(y[k].y);
                        }
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            part[k & 1] = add2(part[k & 1], y[k]);
                            p[b + k] = pack_bf16(y[k].x, y[k].y);
                        }
                    }
                    part[0] = add2(part[0], part[1]);
                };
                // Without looking for the maximum first: against the one in use
                // no probability of these 64 is above FREE if their sum is not
                // (the search took 280 of a step's 1,900 cycles).
                bool settled = false;
                if (e > 0 && !edge) {
                    exponentials();
                    settled = __all_sync(0xffffffffu, !sees || (part[0].x + part[0].y <= FREE && top > -INFINITY));
                    if (!settled) {
                        load(h);
                        tmem_wait_ld();
                    }
                }
                if (!settled) {
                    if (edge) {
#pragma unroll
                        for (int w = 0; w < 2; ++w) {
                            const uint32_t m = seen_word(all, bits, key + 32 * w) & there[w];
                            if (m != ~0u) {
#pragma unroll
                                for (int k = 0; k < 32; ++k) v[w][k] = m >> k & 1u ? v[w][k] : -INFINITY;
                            }
                        }
                    }
                    float best[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int k = 0; k < 32; k += 4)
#pragma unroll
                        for (int w = 0; w < 4; ++w) best[w] = max3(best[w], v[w >> 1][k + 2 * (w & 1)], v[w >> 1][k + 2 * (w & 1) + 1]);
                    const float peak = fmaxf(max3(best[0], best[1], best[2]), best[3]);
                    if (e == 0) {
                        top = peak;
                    } else if (__any_sync(0xffffffffu, sees && (peak - top) * g.c2 > LAZY)) {
                        const float now = fmaxf(top, peak);
                        const float keep = now == top ? 1.f : ex2((top - now) * g.c2);
                        top = now;
                        sum *= keep;
                        // O holds every step before this one (that step sn - 2 is done follows
                        // from S, so the parity tells step sn - 1 from it)
                        ok = wait(bars + 8 * (PV_DONE + x), (sn - 1) & 1, abort);
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < D; c += 8) {  // few registers: the scores are held meanwhile
                            uint32_t o[8];
                            tmem_ld8(to + c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int k = 0; k < 8; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * keep);
                            tmem_st8(to + c, o);
                        }
                    }
                    exponentials();
                }
                tmem_st32u(ts + KEYS * h, p);
                // The next step's scores come while the probabilities go, if they are there already.
                if (e + 1 < n && __all_sync(0xffffffffu, bar_test(bars + 8 * (S_FULL + 2 * x + (h ^ 1)), sp >> (h ^ 1) & 1))) {
                    load(h ^ 1);
                    loaded = true;
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(bars + 8 * (P_FULL + 2 * x + h));
                sum += part[0].x + part[0].y;
                if (loaded) tmem_wait_ld();
            }
            if (!ok) break;
            it += max(u.n0, u.n1);
            bool bad = false;
            if (n > 0) {
                if (!wait(bars + 8 * (O_FULL + x), on & 1, abort)) break;
                ++on;
                tc_fence_after();
                bad = lds(spoiled + 4 * (i & 3)) == i + 1;  // written before this tile's P of that step was handed over
            }
            if (!sees) sum = 0.f;
            const int64_t row = u.first + token;
            const int head = u.kvh * g.group + row_head;
            const bool split = PAGED && u.chunks > 1;
            // Rows leave through the warp's 4 KB of shared memory, 128 bytes of
            // each at a time, so that eight lanes write a row's whole line. The
            // loops stay rolled: this code runs once in a unit, and fetching
            // its instructions is most of its time.
            // (Where every score is -inf the row is zeros, whatever 0 * inf left in O; a chunk keeps that for the join.)
            const bool some = n > 0 && sees && (split || sum != 0.f);
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            const uint32_t mine = used && some ? static_cast<uint32_t>(split ? g.parts.row(0, row, head) : row * a.H + head) : ~0u;
            const uint32_t out = base + C::OFF_OUT + warp * 4096;
            char *dst = split ? reinterpret_cast<char *>(g.parts.o + g.parts.row(u.chunk, 0, 0) * D) : static_cast<char *>(a.o);
            const int row_bytes = split ? D * 4 : D * 2;
            if (n > 0) {
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    float o[32];
                    tmem_ld32(to + c, o);
                    tmem_wait_ld();
                    const float2 scale = make_float2(inv, inv), none = make_float2(0.f, 0.f);
                    uint32_t w[32];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float2 y = fma2(make_float2(o[2 * e], o[2 * e + 1]), scale, none);
                        w[2 * e] = __float_as_uint(y.x);
                        w[2 * e + 1] = __float_as_uint(y.y);
                    }
                    int pieces = 8, at = c * 4, first = 0;
                    if (!split) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) w[e] = pack_bf16(__uint_as_float(w[2 * e]), __uint_as_float(w[2 * e + 1]));
                        pieces = 4;
                        first = c >> 3 & 4;
                        at = (c - 32) * 2;
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (e < pieces)
                            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(out + lane * 128 + (((first + e) ^ (lane & 7)) << 4)),
                                         "r"(w[4 * e]), "r"(w[4 * e + 1]), "r"(w[4 * e + 2]), "r"(w[4 * e + 3])
                                         : "memory");
                    if (!split && !(c & 32)) continue;
                    __syncwarp();
#pragma unroll 2
                    for (int k = 0; k < 8; ++k) {
                        const int rr = 4 * k + (lane >> 3);
                        const uint32_t to_row = __shfl_sync(0xffffffffu, mine, rr);
                        uint4 q;
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                     : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w)
                                     : "r"(out + rr * 128 + (((lane & 7) ^ (rr & 7)) << 4))
                                     : "memory");
                        if (to_row != ~0u)
                            *reinterpret_cast<uint4 *>(dst + static_cast<int64_t>(to_row) * row_bytes + at + (lane & 7) * 16) = q;
                    }
                    __syncwarp();
                }
            }
            if (used && !some) {  // a row that sees nothing, or nothing but scores of -inf
                uint32_t *z = reinterpret_cast<uint32_t *>(dst + (split ? g.parts.row(0, row, head) : row * a.H + head) * row_bytes);
#pragma unroll 1
                for (int c = 0; c < row_bytes / 4; ++c) z[c] = 0u;
            }
            if (used) {
                const float l2 = sum == 0.f ? -INFINITY : top * g.c2 + log2f(sum);
                if (split) g.parts.lse[g.parts.row(u.chunk, row, head)] = l2;
                else if (a.lse) a.lse[row * a.H + head] = l2 * LN2;
            }
            if (PAGED && used && g.parts.count && u.chunk == 0 && head == 0) g.parts.count[row] = u.chunks;
            if (bad)
                add_odd_values<D>(a, g.parts, {u.first, u.m, u.live, u.cached, u.keys}, {u.seq, u.kvh, u.chunk, u.chunks},
                                  max(full_both(), kbeg), min(u.keys, kbeg + n * KEYS), used && some, token, head, lane);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(bars + 8 * (U_EMPTY + (i & 3)));
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        // Copies of K or V: the steps' pages are found and issued here by two
        // warps, one each (a box takes its issuing warp some 60 cycles, and a
        // step has 16 of them where a page is 16 positions; one warp for both
        // needed 1,700 cycles a step). Lane l copies half l % HALVES of page l / HALVES.
        const int rows = 1 << g.rows_shift, pages = KEYS >> g.rows_shift;
        int ids = -1, page0 = 0;  // the table's entries of 32 pages at a time, a lane each
        int place = 0;            // the first row of this lane's page in the cache
        uint32_t there = 0;       // lanes whose page has memory behind it
        auto find_pages = [&](const Unit &u, int j) {
            const int key = u.kbeg + j * KEYS;
            const int last = (min(key + KEYS, u.keys) - 1) >> a.shift;
            if (j == 0 || last >= page0 + 32) {
                page0 = key >> a.shift;
                ids = page0 + lane < a.width ? a.block_table[u.seq * a.width + page0 + lane] : -1;
            }
            const int mine = key + (lane / C::HALVES << g.rows_shift);
            const int block = __shfl_sync(0xffffffffu, ids, min(max((mine >> a.shift) - page0, 0), 31));
            const bool has = lane < pages * C::HALVES && mine < u.keys && block >= 0 && block < a.num_blocks;
            there = __ballot_sync(0xffffffffu, has);
            place = static_cast<int>(((static_cast<int64_t>(block) * a.Hkv + u.kvh) << a.shift) + (mine & ((1 << a.shift) - 1)));
        };
        auto copy_step = [&](const Unit &u, int j, uint32_t full, uint32_t dst, const CUtensorMap *tm) {
            if (PAGED) {
                if (lane == 0) bar_expect(full, __popc(there) * (rows * 128));
                __syncwarp();
                if (there >> lane & 1u)
                    load_2d(dst + lane % C::HALVES * (KEYS * 128) + (lane / C::HALVES << g.rows_shift) * 128, tm, lane % C::HALVES * 64, place, full);
            } else {
                if (lane == 0) bar_expect(full, C::TILE);
                __syncwarp();
                if (lane < C::HALVES) load_3d(dst + lane * (KEYS * 128), tm, lane * 64, u.kvh, u.first + u.kbeg + j * KEYS, full);
            }
            __syncwarp();
        };
        if (warp == WARP_SCHED) {
            // Resolves units, and copies V.
            // Units in order of falling cost, level by level, dealt to the CTAs in
            // snake order. Packed: unit l of a sequence is its row block l, which sees
            // more keys than those before, and a level is all sequences' units of one
            // l. Paged: a sequence's chunks are equal, and a level is every unit of the
            // sequences with chunks of this many steps (48 trees over caches of
            // U{1..8192} keys: 199 us; by the chunks' places alone, which leaves some
            // CTAs a third more than others, 232 us).
            // (The launch refuses more units than 31 bits count.)
            const int pair = 2 * g.tok, n_seq = static_cast<int>(a.n_seq), G = gridDim.x;
            int before = 0;                          // units of the groups before this one
            int group = -1, total = 0, level = 0;    // of this group: units, current l
            int passed = 0, here = 0;                // units of higher l, sequences with a unit l
            auto units_at = [&](int j, int l) { return PAGED ? (costs[j] == l ? counts[j] : 0) : static_cast<int>(counts[j] > l); };
            auto at_level = [&](int l) {
                int n = 0;
#pragma unroll 1
                for (int j = lane; j < GROUP; j += 32) n += units_at(j, l);
                return static_cast<int>(__reduce_add_sync(0xffffffffu, n));
            };
            // Unit i of this CTA, passed on to the other roles.
            bool ok = true;
            auto resolve = [&](int i) -> Unit {
                bool going = true;
                const int64_t x64 = static_cast<int64_t>(i) * G + ((i & 1) ? G - 1 - blockIdx.x : blockIdx.x);
                const int x = static_cast<int>(min(x64, static_cast<int64_t>(INT32_MAX)));
                const int want = x / a.Hkv;
                Unit u{};
#pragma unroll 1
                while (group < 0 || want - before >= total) {
                    before += total;
                    ++group;
                    if (group * GROUP >= n_seq) {
                        going = false;
                        break;
                    }
                    total = 0;
                    int most = 0;
                    __syncwarp();
#pragma unroll 1
                    for (int j = lane; j < GROUP; j += 32) {
                        const int q = group * GROUP + j;
                        int n = 0;
                        if (q < n_seq) {
                            const Seq s = seq_of(a, q);
                            n = (s.m + pair - 1) / pair * (PAGED ? g.split.chunks(s.keys) : 1);
                            if (PAGED) {  // a step of one row tile takes three quarters of a step of two
                                const int steps = min(g.split.span(s.keys) / KEYS, 63);
                                costs[j] = static_cast<uint8_t>(s.live > g.tok ? steps : steps * 3 / 4);
                            }
                        }
                        counts[j] = n;
                        total += n;
                        most = max(most, PAGED ? (n > 0 ? costs[j] + 1 : 0) : n);
                    }
                    total = __reduce_add_sync(0xffffffffu, total);
                    most = __reduce_max_sync(0xffffffffu, most);
                    __syncwarp();
                    level = most - 1;
                    passed = 0;
                    here = most > 0 ? at_level(level) : 0;
                }
                if (going) {
#pragma unroll 1
                    while (want - before >= passed + here) {
                        passed += here;
                        --level;
                        here = at_level(level);
                    }
                    int k = want - before - passed;  // unit k of this level, then of its sequence
                    int q = 0;
#pragma unroll 1
                    for (int j = 0; j < GROUP; j += 32) {
                        const int mine = units_at(j + lane, level);
                        int upto = mine;
#pragma unroll
                        for (int off = 1; off < 32; off <<= 1) {
                            const int y = __shfl_up_sync(0xffffffffu, upto, off);
                            if (lane >= off) upto += y;
                        }
                        const uint32_t past = __ballot_sync(0xffffffffu, upto > k);
                        if (past) {
                            const int at = __ffs(past) - 1;
                            q = group * GROUP + j + at;
                            k -= __shfl_sync(0xffffffffu, upto - mine, at);
                            break;
                        }
                        k -= __shfl_sync(0xffffffffu, upto, 31);
                    }
                    const int l = PAGED ? k : level;  // of the sequence's units
                    const Seq s = seq_of(a, q);
                    const int chunks = PAGED ? g.split.chunks(s.keys) : 1;
                    u.valid = 1;
                    u.seq = q;
                    u.kvh = x - want * a.Hkv;
                    u.first = s.first;
                    u.m = s.m;
                    u.live = s.live;
                    u.cached = s.cached;
                    u.keys = s.keys;
                    const int block = l / chunks;
                    u.chunk = l - block * chunks;
                    u.chunks = chunks;
                    u.t0 = block * pair;
                    int stop = s.keys;
                    if (PAGED) {
                        const int span = g.split.span(s.keys);
                        u.kbeg = u.chunk * span;
                        stop = min(stop, u.kbeg + span);
                    }
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const int t = u.t0 + y * g.tok;
                        int end = t >= u.live ? 0 : stop;
                        if (!(PAGED && a.parent)) end = min(end, s.cached + t + g.tok);
                        const int steps = max(end - u.kbeg + KEYS - 1, 0) / KEYS;
                        (y ? u.n1 : u.n0) = steps;
                    }
                }
                ok = ok && (i < 4 || wait(bars + 8 * (U_EMPTY + (i & 3)), ((i >> 2) - 1) & 1, abort));
                if (ok && lane == 0) {
                    units[i & 3] = u;
                    bar_arrive(bars + 8 * (U_FULL + (i & 3)));
                }
                __syncwarp();
                return u;
            };
            Unit u = resolve(0);
            uint32_t vn = 0;  // tiles issued
#pragma unroll 1
            for (int i = 0; ok && u.valid; ++i) {
                const int steps = max(u.n0, u.n1), early = max(min(steps, C::STAGES), 1);
                Unit after;
#pragma unroll 1
                for (int j = 0; ok && j < max(steps, 1); ++j) {
                    if (steps > 0) {
                        if (PAGED) find_pages(u, j);
                        const int st = vn % C::STAGES;
                        ok = vn < C::STAGES || wait(bars + 8 * (V_EMPTY + st), (vn / C::STAGES - 1) & 1, abort);
                        if (!ok) break;
                        copy_step(u, j, bars + 8 * (V_FULL + st), base + C::OFF_V + st * C::TILE, &tm_v);
                        ++vn;
                    }
                    if (j + 1 == early) after = resolve(i + 1);  // well before K's copies come to it
                }
                u = after;
            }
            if (lds(abort))  // copies in flight land before the CTA leaves
                for (uint32_t k = vn > C::STAGES ? vn - C::STAGES : 0; k < vn; ++k)
                    drain_wait(bars + 8 * (V_FULL + k % C::STAGES), (k / C::STAGES) & 1);
        } else if (warp == WARP_TMA) {
            // Copies Q, and K as far ahead as its ring allows. (K and V have a ring
            // each: in one, a K whose place was free waited behind a V whose place was not.)
            Unit u;
            uint32_t qn = 0, kn = 0;  // Q loads and tiles issued
            bool ok = true;
#pragma unroll 1
            for (int i = 0; ok && next_unit(i, u); ++i) {
                const int steps = max(u.n0, u.n1);
                if (steps == 0) continue;
                if (qn > 0) ok = wait(bars + 8 * Q_EMPTY, (qn - 1) & 1, abort);
                if (!ok) break;
                if (lane == 0) {
                    const uint32_t bytes = static_cast<uint32_t>(g.tok * g.group) * D * 2;
                    bar_expect(bars + 8 * Q_FULL, bytes * ((u.n0 > 0) + (u.n1 > 0)));
                    for (int x = 0; x < 2; ++x)
                        for (int h = 0; (x ? u.n1 : u.n0) > 0 && h < C::HALVES; ++h)
                            load_3d(base + C::OFF_Q + x * C::Q_TILE + h * (ROWS * 128), &tm_q, h * 64, u.kvh * g.group,
                                    u.first + u.t0 + x * g.tok, bars + 8 * Q_FULL);
                }
                ++qn;
#pragma unroll 1
                for (int j = 0; j < steps; ++j) {
                    if (PAGED) find_pages(u, j);
                    const int st = kn % C::STAGES;
                    ok = kn < C::STAGES || wait(bars + 8 * (K_EMPTY + st), (kn / C::STAGES - 1) & 1, abort);
                    if (!ok) break;
                    if (PAGED && lane < 2) {  // which of the step's keys have memory behind them
                        uint32_t w = ~0u;
                        if (__popc(there) != pages * C::HALVES) {
                            w = 0;
#pragma unroll 1
                            for (int b = 0; b < 32; b += 8)  // (pages are eight positions at least)
                                w |= (there >> ((lane * 32 + b) >> g.rows_shift) * C::HALVES & 1u) * 0xffu << b;
                        }
                        sts(masks + 8 * (kn & 15) + 4 * lane, w);
                    }
                    __syncwarp();
                    copy_step(u, j, bars + 8 * (K_FULL + st), base + C::OFF_K + st * C::TILE, &tm_k);
                    ++kn;
                }
            }
            if (lds(abort)) {  // copies in flight land before the CTA leaves
                for (uint32_t k = kn > C::STAGES ? kn - C::STAGES : 0; k < kn; ++k)
                    drain_wait(bars + 8 * (K_FULL + k % C::STAGES), (k / C::STAGES) & 1);
                if (qn > 0) drain_wait(bars + 8 * Q_FULL, (qn - 1) & 1);
            }
        } else if (warp < WARP_TMA) {
            // Products of row tile x. One thread per tile: a step's twelve products
            // take one thread some 1,100 cycles to issue, as long as the tensor cores take for them.
            // The warp stays together and its values are broadcast, so that they
            // live in uniform registers, which the products take their operands from.
            const int x = __shfl_sync(0xffffffffu, warp, 0) - WARP_MMA;
            const bool chosen = elect_one();
            // A descriptor's address field counts 16 bytes: steps are added to
            // its low word (addresses stay below 2^18, so nothing carries).
            const uint64_t like = sdesc_sw128(0, 16, 1024), like_v = sdesc_sw128(0, KEYS * 128, 1024);
            const uint32_t hi = static_cast<uint32_t>(like >> 32), hi_v = static_cast<uint32_t>(like_v >> 32);
            const uint32_t t0 = __shfl_sync(0xffffffffu, tmem, 0);
            const uint32_t q_lo = static_cast<uint32_t>(like) + ((base + C::OFF_Q + x * C::Q_TILE) >> 4);
            const uint32_t k_lo = static_cast<uint32_t>(like) + ((base + C::OFF_K) >> 4);
            const uint32_t v_lo = static_cast<uint32_t>(like_v) + ((base + C::OFF_V) >> 4);
            auto qk = [&](int h, int st) {
                const uint32_t ka = k_lo + st * (C::TILE >> 4), d = t0 + x * 128 + h * KEYS;
                if (chosen) {
#pragma unroll
                    for (int k = 0; k < D / 16; ++k)
                        mma_ss(d, q_lo + (((k >> 2) * (ROWS * 128) + (k & 3) * 32) >> 4), ka + (((k >> 2) * (KEYS * 128) + (k & 3) * 32) >> 4),
                               hi, C::ID_QK, k > 0);
                    commit(bars + 8 * (S_FULL + 2 * x + h));
                }
                __syncwarp();
            };
            auto pv = [&](int h, int st, bool more) {
                const uint32_t va = v_lo + st * (C::TILE >> 4);
                const uint32_t p = t0 + x * 128 + h * KEYS, d = t0 + 256 + x * 128;
                if (chosen) {
#pragma unroll
                    for (int k = 0; k < KEYS / 16; ++k) mma_ts(d, p + 8 * k, va + k * (2048 >> 4), hi_v, C::ID_PV, more || k > 0);
                    commit(bars + 8 * (PV_DONE + x));
                }
                __syncwarp();
            };
            auto done = [&](uint32_t bar) {  // arrives when every product so far is done
                if (chosen) commit(bar);
                __syncwarp();
            };
            Unit u;
            uint32_t qn = 0, pp = 0;     // pp: phases of P_FULL waited for, one bit per parity
            int ks = 0, vs = 0;          // places of the rings
            uint32_t kp = 0, vp = 0;     // and the parities of their laps
            bool ok = true;
            auto next = [](int &st, uint32_t &lap) {
                if (++st == C::STAGES) {
                    st = 0;
                    lap ^= 1;
                }
            };
#pragma unroll 1
            for (int i = 0; ok && next_unit(i, u); ++i) {
                const int steps = __shfl_sync(0xffffffffu, max(u.n0, u.n1), 0);
                const int n = __shfl_sync(0xffffffffu, x ? u.n1 : u.n0, 0);
                if (steps == 0) continue;
                ok = wait(bars + 8 * Q_FULL, qn & 1, abort);
                if (!ok) break;
                // Step e: P is there; its product, then the scores of step e + 2 in its
                // place. (Steps -2 and -1 are the first two scores. Every place of the
                // rings is waited for and released also where this row tile has no use
                // for it: an arrival on EMPTY belongs to the lap whose FULL it follows.)
#pragma unroll 1
                for (int e = -2; e < steps; ++e) {
                    const int h = e & 1;
                    if (e >= 0) {
                        ok = wait(bars + 8 * (V_FULL + vs), vp, abort);
                        if (!ok) break;
                        if (e < n) {
                            ok = wait(bars + 8 * (P_FULL + 2 * x + h), pp >> h & 1, abort);
                            if (!ok) break;
                            pp ^= 1u << h;
                            tc_fence_after();
                            pv(h, vs, e > 0);
                            if (e + 1 == n) done(bars + 8 * (O_FULL + x));
                        }
                        done(bars + 8 * (V_EMPTY + vs));
                        next(vs, vp);
                    }
                    if (e + 2 < steps) {
                        ok = wait(bars + 8 * (K_FULL + ks), kp, abort);
                        if (!ok) break;
                        if (e + 2 < n) qk(h, ks);
                        done(bars + 8 * (K_EMPTY + ks));
                        next(ks, kp);
                        if (e + 3 == steps) done(bars + 8 * Q_EMPTY);
                    }
                }
                ++qn;
            }
            if (lds(abort) && chosen) {  // products in flight finish before TMEM is freed
                commit(bars + 8 * DRAIN);
                drain_wait(bars + 8 * DRAIN, 0);
            }
            __syncwarp();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == WARP_MMA) {
        tc_fence_after();
        tmem_relinquish();
        tmem_dealloc(tmem, 512);
    }
}

template <int D, bool PAGED>
int launch_t(const AttnArgs &a, const Parts &parts, Split split) {
    TcArgs g{};
    g.a = a;
    g.parts = parts;
    g.split = split;
    g.group = a.H / a.Hkv;
    g.tok = ROWS / g.group;
    g.c2 = a.scale * LOG2E;
    const int page = 1 << a.shift;
    g.rows_shift = PAGED && page < KEYS ? a.shift : 6;
    CUtensorMap tq, tk, tv;
    const uint64_t qd[3] = {D, static_cast<uint64_t>(a.H), static_cast<uint64_t>(a.total_tokens)};
    const uint64_t qs[2] = {D * 2, static_cast<uint64_t>(a.q_stride) * 2};
    const uint32_t qb[3] = {64, static_cast<uint32_t>(g.group), static_cast<uint32_t>(g.tok)};
    int st = encode_tmap(&tq, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, a.q, qd, qs, qb, CU_TENSOR_MAP_SWIZZLE_128B);
    if (st != RHZ_OK) return st;
    for (int kv = 0; kv < 2; ++kv) {
        CUtensorMap *m = kv ? &tv : &tk;
        const void *p = kv ? a.v : a.k;
        if (PAGED) {
            const uint64_t d[2] = {D, static_cast<uint64_t>(a.num_blocks * a.Hkv) << a.shift};
            const uint64_t s[1] = {D * 2};
            const uint32_t b[2] = {64, 1u << g.rows_shift};
            st = encode_tmap(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, p, d, s, b, CU_TENSOR_MAP_SWIZZLE_128B);
        } else {
            const uint64_t d[3] = {D, static_cast<uint64_t>(a.Hkv), static_cast<uint64_t>(a.total_tokens)};
            const uint64_t s[2] = {D * 2, static_cast<uint64_t>(kv ? a.v_stride : a.k_stride) * 2};
            const uint32_t b[3] = {64, 1, KEYS};
            st = encode_tmap(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, p, d, s, b, CU_TENSOR_MAP_SWIZZLE_128B);
        }
        if (st != RHZ_OK) return st;
    }
    int sms = 148;
    bool sm100 = true;
    st = device_info(&sms, &sm100);
    if (st != RHZ_OK) return st;
    const int64_t pair = 2 * g.tok;
    const int64_t units = (a.total_tokens / pair + a.n_seq) * (PAGED ? parts.most : 1) * a.Hkv;  // at most
    if (units > INT32_MAX) return set_error(RHZ_ERR_SHAPE, "attention over %lld units exceeds int32 indexing", (long long)units);
    const unsigned grid = static_cast<unsigned>(units < sms ? units : sms);
    cudaError_t e = cudaFuncSetAttribute(attn_tc_kernel<D, PAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::BYTES);
    if (e != cudaSuccess) return set_error(RHZ_ERR_DEVICE, "attn_tc_kernel: %s", cudaGetErrorString(e));
    attn_tc_kernel<D, PAGED><<<grid, THREADS, Cfg<D>::BYTES, a.stream>>>(tq, tk, tv, g);
    return check_launch("attn_tc_kernel");
}

}  // namespace

bool attn_tc_supports(const AttnArgs &a) {
    return a.dtype == RHZ_DTYPE_BF16 && (a.d == 64 || a.d == 128);
}

int launch_attn_tc(const AttnArgs &a, const Parts &parts, Split split) {
    if (a.paged)
        return a.d == 128 ? launch_t<128, true>(a, parts, split) : launch_t<64, true>(a, parts, split);
    return a.d == 128 ? launch_t<128, false>(a, parts, split) : launch_t<64, false>(a, parts, split);
}

int attn_tc_status(int *flag, bool clear) {
    cudaError_t e = cudaMemcpyFromSymbol(flag, g_attn_timeout, sizeof(int));
    if (e == cudaSuccess && clear && *flag) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_attn_timeout, &zero, sizeof(int));
    }
    if (e != cudaSuccess) return set_error(RHZ_ERR_DEVICE, "attention status: %s", cudaGetErrorString(e));
    return RHZ_OK;
}

}  // namespace rhz
