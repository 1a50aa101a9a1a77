// What the two tensor-core forms of the attention share on the device:
// barriers and copies by 32-bit shared-memory addresses, the bits of the keys
// that a row sees, and values that are not finite.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "attn_common.cuh"

namespace rhz {
namespace attn {

__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 1000;\n\t"  // suspended for about 1 us at most
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
// The limit of a wait, 2 s by the card's clock (its low word: differences are
// good to 4 s), looked at every 64 tries.
constexpr uint32_t WAIT_NS = 2000000000u;
__device__ __forceinline__ uint32_t clock_ns() {
    uint32_t t;
    asm volatile("mov.u32 %0, %%globaltimer_lo;" : "=r"(t));
    return t;
}
__device__ __forceinline__ uint32_t lds(uint32_t at) {
    uint32_t x;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(x) : "r"(at) : "memory");
    return x;
}
__device__ __forceinline__ void sts(uint32_t at, uint32_t x) {
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(x) : "memory");
}
__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap *tm, int c0, int c1, int c2, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(tm)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void load_2d(uint32_t dst, const CUtensorMap *tm, int c0, int c1, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(tm)), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}

__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
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

// Where a unit's keys are and its results go.
struct Place {
    int seq, kvh, chunk, chunks;
};

// Whether one of the two bf16 in a word is not finite, and the word without
// those that are not.
__device__ __forceinline__ bool odd_word(uint32_t w) {
    return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}
__device__ __forceinline__ uint32_t finite_word(uint32_t w) {
    if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
    if ((w & 0x7f800000u) == 0x7f800000u) w &= 0x0000ffffu;
    return w;
}

// Values that are not finite at keys that not every row of a tile sees. The
// tensor cores' 0 * NaN would take them to every row, so the kernels replace
// them by zero in shared memory and, once a unit's rows are written, come here
// for the keys [from, to) that this can be (two row tiles' tokens, or a tree's
// nodes, and a step at most).
// What a row that sees such a key has to get follows without its probability:
// that is positive, so an infinity stays one, and what was written is finite
// there or not finite already. Only where the key's score is itself not finite
// (its K row is not) it is 0 * inf or worse, a NaN. A lane of the warp has one
// row: token t of the sequence and a head, with `takes` false where it is none
// or sees no key at all.
template <int D>
__device__ __noinline__ void add_odd_values(const AttnArgs &a, const Parts &parts, const Seq s, const Place at, int from, int to, bool takes,
                                            int t, int head, int lane) {
    constexpr int W = D / 64;  // words of a lane
    const Sight sight = takes ? sight_of(a, s, t) : Sight{0, 0};
    const uint32_t row = static_cast<uint32_t>(s.first + t) * a.H + head;
    __syncwarp();  // the rows were written by other lanes of this warp
    for (int key = from; key < to; ++key) {
        int64_t kat, vat;
        if (a.paged) {
            const int64_t block = a.block_table[at.seq * a.width + (key >> a.shift)];
            if (block < 0 || block >= a.num_blocks) continue;
            kat = vat = (((block * a.Hkv + at.kvh) << a.shift) + (key & ((1 << a.shift) - 1))) * D;
        } else {
            kat = (static_cast<int64_t>(s.first) + key) * a.k_stride + static_cast<int64_t>(at.kvh) * D;
            vat = (static_cast<int64_t>(s.first) + key) * a.v_stride + static_cast<int64_t>(at.kvh) * D;
        }
        const uint32_t *kw = reinterpret_cast<const uint32_t *>(static_cast<const __nv_bfloat16 *>(a.k) + kat) + lane * W;
        const uint32_t *vw = reinterpret_cast<const uint32_t *>(static_cast<const __nv_bfloat16 *>(a.v) + vat) + lane * W;
        uint32_t v[W];
        bool odd = false, odd_k = false;
        for (int e = 0; e < W; ++e) {
            v[e] = vw[e];
            odd |= odd_word(v[e]);
            odd_k |= odd_word(kw[e]);
        }
        if (!__any_sync(0xffffffffu, odd)) continue;
        odd_k = __any_sync(0xffffffffu, odd_k);
        for (uint32_t who = __ballot_sync(0xffffffffu, takes && sight.sees(key)); who != 0; who &= who - 1) {
            const uint32_t to_row = __shfl_sync(0xffffffffu, row, __ffs(who) - 1);
            if (!odd) continue;
            for (int c = 0; c < 2 * W; ++c) {
                const float x = __uint_as_float(c & 1 ? v[c >> 1] & 0xffff0000u : v[c >> 1] << 16);
                if (isfinite(x)) continue;
                const float add = odd_k ? NAN : x;
                const int64_t place = static_cast<int64_t>(to_row) * D + lane * 2 * W + c;
                if (at.chunks > 1) {
                    float *o = parts.o + parts.row(at.chunk, 0, 0) * D + place;
                    *o += add;
                } else {
                    __nv_bfloat16 *o = static_cast<__nv_bfloat16 *>(a.o) + place;
                    *o = __float2bfloat16_rn(__bfloat162float(*o) + add);
                }
            }
        }
    }
}

}  // namespace attn
}  // namespace rhz
