// Softmax attention with grouped heads on the 5th-generation tensor cores:
// bf16, head widths 64 and 128, packed causal prompts and drafted trees (or
// pieces of a prompt) over the paged cache.
//
// One persistent CTA per SM works through units: 2 x 128 query rows (two
// tiles) of one (sequence, K/V head), over that pair's keys or a chunk of
// them, 128 keys at a time:
//   S_x = Q_x K^T          (tcgen05, both operands in shared memory, f32 in TMEM)
//   P_x = exp2(c S_x - c m)  (one warpgroup per tile, a thread per row)
//   O_x += P_x V           (tcgen05, P as a bf16 A operand in TMEM, over S's columns)
// with the running maximum m kept lazily: O is rescaled only when a row's
// maximum has grown by more than 2^8 since m was set, so probabilities stay
// below 2^8 and the product is rarely interrupted.
//
// Roles: warps 0-3 and 4-7 the softmax of tiles 0 and 1, warp 8 issues every
// product, warp 9 every copy, warp 10 resolves units ahead of the others.
// While one tile's softmax runs, the tensor cores work on the other tile. The
// order PV_x(j), QK_x(j + 1) on the one issuing thread also means that S_x(j)
// complete implies PV_x(j - 1) complete, so a rescale of O needs no further wait.
//
// What bounds it: 128 x 128 exponentials cost the SM's 16 special-function
// lanes 1,024 cycles, the two products of a d = 128 tile 1,024 tensor cycles.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "attn_common.cuh"
#include "sm100.cuh"
#include "tmap.h"

namespace rhz {
namespace {

using namespace attn;
using namespace sm100;

constexpr int ROWS = 128;   // query rows of a tile
constexpr int KEYS = 128;   // keys of a tile
constexpr int THREADS = 384;  // the last warp only fills its warpgroup (registers move by warpgroup)
constexpr int WARP_MMA = 8, WARP_TMA = 9, WARP_SCHED = 10;
constexpr int GROUP = 256;  // sequences whose unit counts the scheduler holds at a time
#ifndef POLY_
#define POLY_ 0
#endif
constexpr int POLY = POLY_;      // of 8 pairs of exponentials, so many by polynomial
constexpr float LAZY = 8.f; // a row's maximum may grow by 2^LAZY before O is rescaled

// Sticky: a bounded wait of this kernel ran out.
__device__ int g_attn_timeout;

// A unit, resolved by the scheduler warp.
struct Unit {
    int32_t valid;
    int32_t seq, kvh;
    int32_t first, t0, m, live;  // query rows: first row, this unit's first token, tokens, those taking part
    int32_t cached, keys;        // keys before the sequence's own, and in all
    int32_t kbeg, n0, n1;        // first key, key tiles of either row tile
    int32_t chunk, chunks;
};

template <int D>
struct Cfg {
    static constexpr int HALVES = D / 64;
    static constexpr int TILE = KEYS * D * 2;              // a K, V or Q tile in bytes
    static constexpr int STAGES = D == 128 ? 4 : 8;        // K and V tiles in flight
    static constexpr int OFF_Q = 0;
    static constexpr int OFF_KV = 2 * TILE;
    static constexpr int OFF_OUT = OFF_KV + STAGES * TILE; // 4 KB per softmax warp: output rows on their way out
    static constexpr int OFF_BAR = OFF_OUT + 8 * 4096;     // barriers, units, scheduler's counts
    static constexpr int OFF_UNIT = OFF_BAR + 256;
    static constexpr int OFF_MASK = OFF_UNIT + 128;
    static constexpr int OFF_MISC = OFF_MASK + 128;
    static constexpr int OFF_COUNT = OFF_MISC + 64;
    static constexpr int BYTES = OFF_COUNT + GROUP * 4 + 1024;
    static constexpr uint32_t ID_QK = idesc_bf16(ROWS, KEYS, false, false);
    static constexpr uint32_t ID_PV = idesc_bf16(ROWS, D, false, true);
};

struct Bars {
    uint64_t kv_full[8], kv_empty[8];
    uint64_t q_full, q_empty;
    uint64_t s_full[2], p_full[2][2], o_full[2];  // P in two halves of 64 keys
    uint64_t u_full[2], u_empty[2];
    uint64_t drain;
};
static_assert(sizeof(Bars) <= 256 && 2 * sizeof(Unit) <= 128, "shared-memory layout");

struct TcArgs {
    AttnArgs a;
    Parts parts;
    Split split;
    int tok;     // tokens of a row tile: 128 / group
    int group;   // query heads per K/V head
    int rows;    // rows per TMA box of a paged tile
    float c2;    // scale * log2 e
};

// Bounded wait of one thread that also ends when another role gave up.
__device__ bool wait1(uint64_t *bar, uint32_t parity, volatile int *abort) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = globaltimer_ns();
    for (uint32_t i = 1;; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 63u) == 0) {
            if (*abort) return false;
            if (globaltimer_ns() - t0 > 2000000000ull) {
                *abort = 1;
                atomicExch(&g_attn_timeout, 1);
                return false;
            }
        }
    }
}

// The same for a whole warp: all its lanes go on or none does.
__device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity, volatile int *abort) {
    return __all_sync(0xffffffffu, wait1(bar, parity, abort));
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
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

// 2^x without the special-function unit, two at once: x = n + f with n the
// nearest integer (the low bits of x + 1.5 * 2^23), |f| <= 1/2, then a
// degree-5 polynomial in f (least maximal relative error among those with
// constant term 1: 2^-22.4 in f32 arithmetic, as close as ex2.approx) and n
// added to the exponent. x is held at -127, where f = 0 and the sum of
// exponents is exactly 0.
__device__ __forceinline__ float2 ex2_poly(float2 x) {
    constexpr float MAGIC = 12582912.f;
    x.x = fmaxf(x.x, -127.f);
    x.y = fmaxf(x.y, -127.f);
    const float2 t = add2(x, make_float2(MAGIC, MAGIC));
    const float2 n = add2(t, make_float2(-MAGIC, -MAGIC));
    const float2 f = fma2(n, make_float2(-1.f, -1.f), x);
    float2 p = make_float2(0.001326472731307149f, 0.001326472731307149f);
    p = fma2(p, f, make_float2(0.009671512991189957f, 0.009671512991189957f));
    p = fma2(p, f, make_float2(0.05550733581185341f, 0.05550733581185341f));
    p = fma2(p, f, make_float2(0.24022242426872253f, 0.24022242426872253f));
    p = fma2(p, f, make_float2(0.6931470036506653f, 0.6931470036506653f));
    p = fma2(p, f, make_float2(1.f, 1.f));
    return make_float2(__uint_as_float((__float_as_uint(t.x) << 23) + __float_as_uint(p.x)),
                       __uint_as_float((__float_as_uint(t.y) << 23) + __float_as_uint(p.y)));
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}

// Bits of the 32 keys from `start` that a row sees (`all`: keys below it are
// seen; `bits`: the 64 keys from `all` on).
__device__ __forceinline__ uint32_t seen_word(int all, uint64_t bits, int start) {
    const int n = all - start;  // keys of this word below `all`
    if (n >= 32) return ~0u;
    if (n > 0) return ((1u << n) - 1u) | static_cast<uint32_t>(bits << n);
    return n > -64 ? static_cast<uint32_t>(bits >> -n) : 0u;
}

// One row by plain arithmetic from global memory, a warp per row: for tiles
// that hold values which are not finite where some rows must not see them
// (the tensor cores' 0 * NaN would reach every row of the tile).
template <int D, bool PAGED>
__device__ __noinline__ void plain_row(const TcArgs &g, const Unit &u, int row, const Sight &sight, int kend, int lane) {
    constexpr int C = D / 32;  // channels of a lane
    const AttnArgs &a = g.a;
    const int64_t token = u.first + u.t0 + row / g.group;
    const int head = u.kvh * g.group + row % g.group;
    const __nv_bfloat16 *q = static_cast<const __nv_bfloat16 *>(a.q) + token * a.q_stride + static_cast<int64_t>(head) * D + lane * C;
    float qx[C], acc[C], top = -INFINITY, sum = 0.f;
    for (int e = 0; e < C; ++e) {
        qx[e] = __bfloat162float(q[e]);
        acc[e] = 0.f;
    }
    for (int key = u.kbeg; key < kend; ++key) {
        if (!sight.sees(key)) continue;
        int64_t kat, vat;
        if (PAGED) {
            const int64_t block = a.block_table[u.seq * a.width + (key >> a.shift)];
            if (block < 0 || block >= a.num_blocks) continue;
            kat = vat = (((block * a.Hkv + u.kvh) << a.shift) + (key & ((1 << a.shift) - 1))) * D;
        } else {
            kat = (static_cast<int64_t>(u.first) + key) * a.k_stride + static_cast<int64_t>(u.kvh) * D;
            vat = (static_cast<int64_t>(u.first) + key) * a.v_stride + static_cast<int64_t>(u.kvh) * D;
        }
        float s = 0.f;
        for (int e = 0; e < C; ++e) s = fmaf(qx[e], __bfloat162float(static_cast<const __nv_bfloat16 *>(a.k)[kat + lane * C + e]), s);
        for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
        s *= g.c2;
        const float best = fmaxf(top, s), from = best == -INFINITY ? 0.f : best;
        const float keep = ex2(top - from), p = ex2(s - from);
        top = best;
        sum = sum * keep + p;
        for (int e = 0; e < C; ++e)
            acc[e] = fmaf(p, __bfloat162float(static_cast<const __nv_bfloat16 *>(a.v)[vat + lane * C + e]), acc[e] * keep);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const float l2 = sum == 0.f ? -INFINITY : top + log2f(sum);
    if (u.chunks > 1) {
        const int64_t r = g.parts.row(u.chunk, token, head);
        if (lane == 0) g.parts.lse[r] = l2;
        for (int e = 0; e < C; ++e) g.parts.o[r * D + lane * C + e] = acc[e] * inv;
    } else {
        if (lane == 0 && a.lse) a.lse[token * a.H + head] = l2 * LN2;
        for (int e = 0; e < C; ++e)
            static_cast<__nv_bfloat16 *>(a.o)[(token * a.H + head) * D + lane * C + e] = __float2bfloat16_rn(acc[e] * inv);
    }
}

template <int D, bool PAGED>
__global__ void __launch_bounds__(THREADS, 1)
    attn_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                   const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ TcArgs g) {
    using C = Cfg<D>;
    extern __shared__ char smem_raw[];
    char *smem = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t{1023});
    const uint32_t base = smem_u32(smem);
    Bars &bar = *reinterpret_cast<Bars *>(smem + C::OFF_BAR);
    Unit *units = reinterpret_cast<Unit *>(smem + C::OFF_UNIT);
    uint32_t(*masks)[4] = reinterpret_cast<uint32_t(*)[4]>(smem + C::OFF_MASK);  // per ring stage: keys with memory behind them
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + C::OFF_MISC);
    volatile int *abort = reinterpret_cast<volatile int *>(smem + C::OFF_MISC + 4);
    // Unit i of tile x met values that are not finite where not every row sees
    // them: [x][i & 3] == i + 1. (A warp that sets the flag of unit i + 4 has
    // seen the descriptor of i + 4, so every warp has read that of i + 2 and is done with i.)
    volatile int(*spoiled)[4] = reinterpret_cast<volatile int(*)[4]>(smem + C::OFF_MISC + 16);
    int *counts = reinterpret_cast<int *>(smem + C::OFF_COUNT);
    const AttnArgs &a = g.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::STAGES; ++i) {
            mbar_init(&bar.kv_full[i], 1);
            mbar_init(&bar.kv_empty[i], 1);
        }
        mbar_init(&bar.q_full, 1);
        mbar_init(&bar.q_empty, 1);
        for (int x = 0; x < 2; ++x) {
            mbar_init(&bar.s_full[x], 1);
            mbar_init(&bar.p_full[x][0], 4);
            mbar_init(&bar.p_full[x][1], 4);
            mbar_init(&bar.o_full[x], 1);
            mbar_init(&bar.u_full[x], 1);
            mbar_init(&bar.u_empty[x], 10);
        }
        mbar_init(&bar.drain, 1);
        *abort = 0;
        for (int i = 0; i < 8; ++i) spoiled[i >> 2][i & 3] = 0;
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

    // Units come through a ring of two.
    auto next_unit = [&](int i, Unit &u) -> bool {
        if (!wait(&bar.u_full[i & 1], (i >> 1) & 1, abort)) return false;
        u = units[i & 1];
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.u_empty[i & 1]);
        return u.valid != 0;
    };

    // 384 x 168 registers at launch: 256 x 208 for the softmax, 128 x 88 for the rest.
    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        // Softmax of tile x: thread r of the warpgroup is row r.
        const int x = warp >> 2, r = threadIdx.x & 127;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + x * 128, to = tmem + lanes + 256 + x * 128;
        Unit u;
        uint32_t sn = 0, on = 0, it = 0;  // S tiles and outputs waited for, ring position of the unit's first tile
        for (int i = 0; next_unit(i, u); ++i) {
            const int token = u.t0 + x * g.tok + r / g.group;
            const bool used = r < g.tok * g.group && token < u.m;
            Seq s;
            s.first = u.first; s.m = u.m; s.live = u.live; s.cached = u.cached; s.keys = u.keys;
            Sight sight{0, 0};
            if (used) sight = sight_of(a, s, token);
            const int all = static_cast<int>(sight.all);
            // Tiles below `full` are seen whole by every live row of the warpgroup's tile.
            const int t_first = u.t0 + x * g.tok;
            const int full = PAGED && a.parent ? u.cached : u.cached + t_first + 1;
            float top = -INFINITY, sum = 0.f;
            bool ok = true;
            const int n = x ? u.n1 : u.n0;
            for (int j = 0; j < n; ++j, ++sn) {
                const int key = u.kbeg + j * KEYS;
                bool edge = key + KEYS > full;
                const uint32_t vt = it + 2 * j + 1;  // this tile's V in the ring
                const int vs = vt % C::STAGES;
                uint32_t there[4] = {~0u, ~0u, ~0u, ~0u};
                if (PAGED || edge) {
                    ok = wait(&bar.kv_full[vs], (vt / C::STAGES) & 1, abort);
                    if (!ok) break;
                    if (PAGED) {
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            there[w] = masks[vs][w];
                            edge |= there[w] != ~0u;
                        }
                    }
                }
                ok = wait(&bar.s_full[x], sn & 1, abort);
                if (!ok) break;
                tc_fence_after();
                float v[4][32];
#pragma unroll
                for (int w = 0; w < 4; ++w) tmem_ld32(ts + 32 * w, v[w]);
                tmem_wait_ld();
                if (edge) {
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t m = seen_word(all, sight.bits, key + 32 * w) & there[w];
                        if (m != ~0u) {
#pragma unroll
                            for (int e = 0; e < 32; ++e) v[w][e] = m >> e & 1u ? v[w][e] : -INFINITY;
                        }
                    }
                    // V: rows behind the sequence or without a page become zero,
                    // values that are not finite in rows not everyone sees are noted.
                    char *vrow = smem + C::OFF_KV + vs * C::TILE + r * 128;
                    const bool exists = key + r < u.keys && (!PAGED || (masks[vs][warp & 3] >> lane & 1u));
                    bool bad = false;
                    if (!exists || key + r >= full) {
#pragma unroll 1
                        for (int h = 0; h < C::HALVES; ++h)
#pragma unroll 2
                            for (int c = 0; c < 8; ++c) {
                                // (lanes start at different 16-byte pieces: different banks)
                                uint4 *p = reinterpret_cast<uint4 *>(vrow + h * 16384 + ((c + lane) & 7) * 16);
                                if (!exists) {
                                    *p = make_uint4(0u, 0u, 0u, 0u);
                                } else {
                                    const uint4 q = *p;
                                    const uint32_t ws[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                                    for (int e = 0; e < 4; ++e)
                                        bad |= (ws[e] & 0x7f80u) == 0x7f80u || (ws[e] & 0x7f800000u) == 0x7f800000u;
                                }
                            }
                    }
                    if (bad) spoiled[x][i & 3] = i + 1;
                    fence_proxy_async_smem();
                }
                float best[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < 32; ++e)
#pragma unroll
                    for (int w = 0; w < 4; ++w) best[w] = fmaxf(best[w], v[w][e]);
                const float peak = fmaxf(fmaxf(best[0], best[1]), fmaxf(best[2], best[3]));
                if (j == 0) {
                    top = peak;
                } else if (__any_sync(0xffffffffu, (peak - top) * g.c2 > LAZY)) {
                    const float now = fmaxf(top, peak);
                    const float keep = now == top ? 1.f : ex2((top - now) * g.c2);
                    top = now;
                    sum *= keep;
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        float o[32];
                        tmem_ld32(to + c, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] *= keep;
                        tmem_st32(to + c, o);
                    }
                }
                const float from = top == -INFINITY ? 0.f : -top * g.c2;
                const float2 c2 = make_float2(g.c2, g.c2), f2 = make_float2(from, from);
                float2 part[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
auto exponentials = [&](auto poly) {  // pairs of each eight that go by polynomial
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t p[32];
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            float2 y = fma2(make_float2(v[2 * half + e / 16][2 * (e % 16)], v[2 * half + e / 16][2 * (e % 16) + 1]), c2, f2);
                            if (e % 8 < decltype(poly)::value) {
                                y = ex2_poly(y);
                            } else {
                                y.x = ex2(y.x);
                                y.y = ex2(y.y);
                            }
                            part[e & 1] = add2(part[e & 1], y);
                            p[e] = pack_bf16(y.x, y.y);
                        }
                        tmem_st32u(ts + 32 * half, p);
                        tmem_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&bar.p_full[x][half]);
                    }
                };
                if (edge) exponentials(std::integral_constant<int, 0>{});  // masked scores give exact zeros
                else exponentials(std::integral_constant<int, POLY>{});
                part[0] = add2(part[0], part[1]);
                sum += part[0].x + part[0].y;
            }
            if (!ok) break;
            it += 2 * max(u.n0, u.n1);
            bool bad = false;
            if (n > 0) {
                if (!wait(&bar.o_full[x], on & 1, abort)) break;
                ++on;
                tc_fence_after();
                bad = spoiled[x][i & 3] == i + 1;  // written before its warp's last p_full arrival
            }
            const bool blind = sight.all == 0 && sight.bits == 0;  // sees nothing: whole tiles above did not ask
            if (blind) sum = 0.f;
            const int64_t row = u.first + token;
            const int head = u.kvh * g.group + r % g.group;
            if (bad) {
                const int kend = min(u.keys, u.kbeg + n * KEYS);
                for (int w = 0; w < 32; ++w) {  // the warp takes its own 32 rows
                    const int rr = (warp & 3) * 32 + w;
                    const Sight theirs{__shfl_sync(0xffffffffu, sight.all, w), __shfl_sync(0xffffffffu, sight.bits, w)};
                    if (__shfl_sync(0xffffffffu, static_cast<int>(used), w))
                        plain_row<D, PAGED>(g, u, x * g.tok * g.group + rr, theirs, kend, lane);
                }
            } else {
                // Rows leave through the warp's 4 KB of shared memory, 128 bytes of
                // each at a time, so that eight lanes write a row's whole line (a
                // thread writing its own row took 6,600 cycles per unit).
                const bool split = PAGED && u.chunks > 1;
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                const float l2 = sum == 0.f ? -INFINITY : top * g.c2 + log2f(sum);
                const uint32_t mine = used ? static_cast<uint32_t>(split ? g.parts.row(0, row, head) : row * a.H + head) : ~0u;
                char *out = smem + C::OFF_OUT + warp * 4096;
                char *dst = split ? reinterpret_cast<char *>(g.parts.o + g.parts.row(u.chunk, 0, 0) * D) : static_cast<char *>(a.o);
                const int row_bytes = split ? D * 4 : D * 2;
                auto leave = [&](int at) {  // 128 bytes of every row, from byte `at` of the row
                    __syncwarp();
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int rr = 4 * k + (lane >> 3);
                        const uint32_t to = __shfl_sync(0xffffffffu, mine, rr);
                        const uint4 q = *reinterpret_cast<const uint4 *>(out + rr * 128 + (((lane & 7) ^ (rr & 7)) << 4));
                        if (to != ~0u) *reinterpret_cast<uint4 *>(dst + static_cast<int64_t>(to) * row_bytes + at + (lane & 7) * 16) = q;
                    }
                    __syncwarp();
                };
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    float o[32];
                    if (n > 0) {
                        tmem_ld32(to + c, o);
                        tmem_wait_ld();
                    }
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = n > 0 && !blind ? o[e] * inv : 0.f;
                    if (split) {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            *reinterpret_cast<float4 *>(out + lane * 128 + ((e ^ (lane & 7)) << 4)) =
                                make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                        leave(c * 4);
                    } else {
                        const int h = (c & 32) >> 3;  // the row's lower or upper 64 bytes
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            *reinterpret_cast<uint4 *>(out + lane * 128 + (((h + e) ^ (lane & 7)) << 4)) =
                                make_uint4(pack_bf16(o[8 * e], o[8 * e + 1]), pack_bf16(o[8 * e + 2], o[8 * e + 3]),
                                           pack_bf16(o[8 * e + 4], o[8 * e + 5]), pack_bf16(o[8 * e + 6], o[8 * e + 7]));
                        if (c & 32) leave((c - 32) * 2);
                    }
                }
                if (used) {
                    if (split) g.parts.lse[g.parts.row(u.chunk, row, head)] = l2;
                    else if (a.lse) a.lse[row * a.H + head] = l2 * LN2;
                }
            }
            if (used && g.parts.count && u.chunk == 0 && head == 0) g.parts.count[row] = u.chunks;
            tc_fence_before();
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == WARP_SCHED) {
            // Units in order of falling cost: unit l of a sequence is its row block
            // l / chunks (later blocks see more keys), and all sequences' units
            // of one l come together, the highest l first; dealt to the CTAs in
            // snake order.
            // (The launch refuses more units than 31 bits count.)
            const int pair = 2 * g.tok, n_seq = static_cast<int>(a.n_seq), G = gridDim.x;
            int before = 0;                          // units of the groups before this one
            int group = -1, total = 0, level = 0;    // of this group: units, current l
            int passed = 0, here = 0;                // units of higher l, sequences with a unit l
            auto at_level = [&](int l) {
                int n = 0;
#pragma unroll 1
                for (int i = lane; i < GROUP; i += 32) n += __popc(__ballot_sync(0xffffffffu, counts[i] > l));
                return n;
            };
            bool going = true;
#pragma unroll 1
            for (int i = 0; going; ++i) {
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
                            n = (static_cast<int>(s.m) + pair - 1) / pair * (PAGED ? static_cast<int>(g.split.chunks(s.keys)) : 1);
                        }
                        counts[j] = n;
                        total += n;
                        most = max(most, n);
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
                    int k = want - before - passed;  // the k-th sequence with a unit at this level
                    int q = 0;
#pragma unroll 1
                    for (int j = 0; j < GROUP; j += 32) {
                        const bool has = counts[j + lane] > level;
                        const uint32_t b = __ballot_sync(0xffffffffu, has);
                        if (k < __popc(b)) {
                            const uint32_t kth = __ballot_sync(0xffffffffu, has && __popc(b & ((1u << lane) - 1u)) == k);
                            q = group * GROUP + j + __ffs(kth) - 1;
                            break;
                        }
                        k -= __popc(b);
                    }
                    const Seq s = seq_of(a, q);
                    const int keys = static_cast<int>(s.keys), cached = static_cast<int>(s.cached);
                    const int chunks = PAGED ? static_cast<int>(g.split.chunks(s.keys)) : 1;
                    u.valid = 1;
                    u.seq = q;
                    u.kvh = x - want * a.Hkv;
                    u.first = static_cast<int>(s.first);
                    u.m = static_cast<int>(s.m);
                    u.live = static_cast<int>(s.live);
                    u.cached = cached;
                    u.keys = keys;
                    const int block = level / chunks;
                    u.chunk = level - block * chunks;
                    u.chunks = chunks;
                    u.t0 = block * pair;
                    int stop = keys;
                    if (PAGED) {
                        const int span = static_cast<int>(g.split.span(s.keys));
                        u.kbeg = u.chunk * span;
                        stop = min(stop, u.kbeg + span);
                    }
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const int t = u.t0 + y * g.tok;
                        int end = t >= u.live ? 0 : stop;
                        if (!(PAGED && a.parent)) end = min(end, cached + t + g.tok);
                        const int tiles = max(end - u.kbeg + KEYS - 1, 0) / KEYS;
                        (y ? u.n1 : u.n0) = tiles;
                    }
                }
                if (i >= 2 && !wait(&bar.u_empty[i & 1], ((i >> 1) - 1) & 1, abort)) break;
                if (lane == 0) {
                    units[i & 1] = u;
                    mbar_arrive(&bar.u_full[i & 1]);
                }
                __syncwarp();
            }
        } else if (warp == WARP_TMA) {
            // K and V tiles in the order K0 V0 K1 V1 ..: one ring for both.
            Unit u;
            uint32_t it = 0, qn = 0;  // tiles and Q loads issued
            bool ok = true;
            for (int i = 0; ok && next_unit(i, u); ++i) {
                const int tiles = max(u.n0, u.n1);
                if (tiles == 0) continue;
                if (qn > 0) ok = wait(&bar.q_empty, (qn - 1) & 1, abort);
                if (!ok) break;
                if (lane == 0) {
                    const uint32_t bytes = static_cast<uint32_t>(g.tok * g.group) * D * 2;
                    mbar_arrive_expect_tx(&bar.q_full, bytes * ((u.n0 > 0) + (u.n1 > 0)));
                    for (int x = 0; x < 2; ++x)
                        for (int h = 0; (x ? u.n1 : u.n0) > 0 && h < C::HALVES; ++h)
                            tma_load_3d(smem + C::OFF_Q + x * C::TILE + h * 16384, &tm_q, h * 64, u.kvh * g.group,
                                        u.first + u.t0 + x * g.tok, &bar.q_full);
                }
                ++qn;
                const int rows = g.rows, pages = KEYS / rows;
                for (int j = 0; j < tiles && ok; ++j) {
                    const int key = u.kbeg + j * KEYS;
                    int at = 0;          // this lane's page: its first row in the cache
                    bool there = false;
                    uint32_t valid = 1;
                    if (PAGED) {
                        const int mine = key + lane * rows;
                        if (lane < pages && mine < u.keys) {
                            const int64_t block = a.block_table[u.seq * a.width + (mine >> a.shift)];
                            there = block >= 0 && block < a.num_blocks;
                            at = static_cast<int>(((block * a.Hkv + u.kvh) << a.shift) + (mine & ((1 << a.shift) - 1)));
                        }
                        valid = __ballot_sync(0xffffffffu, there);
                    }
                    for (int kv = 0; kv < 2; ++kv, ++it) {
                        const int st = it % C::STAGES;
                        const uint32_t lap = it / C::STAGES;
                        if (lap > 0 && !wait(&bar.kv_empty[st], (lap - 1) & 1, abort)) {
                            ok = false;
                            break;
                        }
                        char *dst = smem + C::OFF_KV + st * C::TILE;
                        const CUtensorMap *tm = kv ? &tm_v : &tm_k;
                        if (PAGED) {
                            if (kv == 1 && lane < 4) {  // which of the tile's keys have memory behind them
                                uint32_t w = ~0u;
                                if (__popc(valid) != pages) {
                                    w = 0;
                                    for (int b = 0; b < 32; ++b) w |= (valid >> ((lane * 32 + b) / rows) & 1u) << b;
                                }
                                masks[st][lane] = w;
                            }
                            __syncwarp();
                            if (lane == 0) mbar_arrive_expect_tx(&bar.kv_full[st], __popc(valid) * rows * D * 2);
                            __syncwarp();
                            if (there)
                                for (int h = 0; h < C::HALVES; ++h)
                                    asm volatile(
                                        "cp.async.bulk.tensor.2d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
                                            smem_u32(dst + h * 16384 + lane * rows * 128)),
                                        "l"(reinterpret_cast<uint64_t>(tm)), "r"(h * 64), "r"(at), "r"(smem_u32(&bar.kv_full[st]))
                                        : "memory");
                        } else if (lane == 0) {
                            mbar_arrive_expect_tx(&bar.kv_full[st], C::TILE);
                            for (int h = 0; h < C::HALVES; ++h)
                                tma_load_3d(dst + h * 16384, tm, h * 64, u.kvh, u.first + key, &bar.kv_full[st]);
                        }
                        __syncwarp();
                    }
                }
            }
            if (*abort) {  // copies in flight land before the CTA leaves
                for (uint32_t k = it > C::STAGES ? it - C::STAGES : 0; k < it; ++k)
                    mbar_wait(&bar.kv_full[k % C::STAGES], (k / C::STAGES) & 1, 1000000000ull);
                if (qn > 0) mbar_wait(&bar.q_full, (qn - 1) & 1, 1000000000ull);
            }
        } else if (warp == WARP_MMA) {
            Unit u;
            uint32_t it = 0, qn = 0, pn0 = 0, pn1 = 0;
            bool ok = true;
            for (int i = 0; ok && next_unit(i, u); ++i) {
                const int tiles = max(u.n0, u.n1);
                if (tiles == 0) continue;
                if (lane == 0) {
                    // A descriptor's address field counts 16 bytes: steps are added to it.
                    const uint64_t dq = sdesc_sw128(base + C::OFF_Q, 16, 1024);
                    const uint64_t dk = sdesc_sw128(base + C::OFF_KV, 16, 1024);
                    const uint64_t dv = sdesc_sw128(base + C::OFF_KV, 16384, 1024);
                    auto qk = [&](int x, int st) {
                        const uint64_t qa = dq + x * (C::TILE >> 4), ka = dk + st * (C::TILE >> 4);
#pragma unroll
                        for (int k = 0; k < D / 16; ++k) {
                            const uint32_t off = ((k >> 2) * 16384 + (k & 3) * 32) >> 4;
                            umma_f16(tmem + x * 128, qa + off, ka + off, C::ID_QK, k > 0);
                        }
                        umma_commit(&bar.s_full[x]);
                    };
                    auto pv = [&](int x, int st, int half, bool more) {
                        const uint64_t va = dv + st * (C::TILE >> 4) + half * (8192 >> 4);
                        const uint32_t p = tmem + x * 128 + half * 32;
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            umma_f16_ta(tmem + 256 + x * 128, p + 8 * k, va + k * (2048 >> 4), C::ID_PV, more || k + half > 0);
                    };
                ok = wait1(&bar.q_full, qn & 1, abort) && wait1(&bar.kv_full[it % C::STAGES], (it / C::STAGES) & 1, abort);
                    if (ok) {
#pragma unroll 1
                        for (int x = 0; x < 2; ++x)
                            if ((x ? u.n1 : u.n0) > 0) qk(x, it % C::STAGES);
                        umma_commit(&bar.kv_empty[it % C::STAGES]);
                        if (tiles == 1) umma_commit(&bar.q_empty);
                        ++it;
                    }
                    for (int j = 0; ok && j < tiles; ++j) {
                        const int vs = it % C::STAGES;
                        const uint32_t kt = it + 1;
                        const int ks = kt % C::STAGES;
                        ok = wait1(&bar.kv_full[vs], (it / C::STAGES) & 1, abort);
                        bool have_k = false;
#pragma unroll 1
                        for (int x = 0; ok && x < 2; ++x) {
                            const int n = x ? u.n1 : u.n0;
                            if (j < n) {
                                uint32_t &pn = x ? pn1 : pn0;
#pragma unroll 1
                                for (int half = 0; ok && half < 2; ++half) {
                                    ok = wait1(&bar.p_full[x][half], pn & 1, abort);
                                    if (!ok) break;
                                    tc_fence_after();
                                    pv(x, vs, half, j > 0);
                                }
                                if (!ok) break;
                                ++pn;
                                if (j + 1 == n) umma_commit(&bar.o_full[x]);
                            }
                            if (j + 1 < n) {
                                if (!have_k) {
                                    ok = wait1(&bar.kv_full[ks], (kt / C::STAGES) & 1, abort);
                                    if (!ok) break;
                                    have_k = true;
                                }
                                qk(x, ks);
                            }
                        }
                        if (!ok) break;
                        umma_commit(&bar.kv_empty[vs]);
                        if (j + 1 < tiles) {
                            umma_commit(&bar.kv_empty[ks]);
                            if (j + 2 == tiles) umma_commit(&bar.q_empty);
                            it += 2;
                        } else {
                            it += 1;
                        }
                    }
                }
                ++qn;
                ok = __shfl_sync(0xffffffffu, static_cast<int>(ok), 0) != 0;
            }
            if (*abort && lane == 0) {  // products in flight finish before TMEM is freed
                umma_commit(&bar.drain);
                mbar_wait(&bar.drain, 0, 1000000000ull);
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
    g.rows = PAGED && page < KEYS ? page : KEYS;
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
            const uint32_t b[2] = {64, static_cast<uint32_t>(g.rows)};
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
