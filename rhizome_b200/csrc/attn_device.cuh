// What the two tensor-core forms of the attention share on the device:
// barriers and copies by 32-bit shared-memory addresses, the bits of the keys
// that a row sees, and the plain-arithmetic form of one row.
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

// Where a row's keys are and its result goes.
struct RowPlace {
    int seq, kvh, first, kbeg, kend, chunk, chunks;
};

// One row by plain arithmetic from global memory, a warp per row: for tiles
// that hold values which are not finite where some rows must not see them
// (the tensor cores' 0 * NaN would reach every row of the tile).
template <int D>
__device__ __noinline__ void plain_row(const AttnArgs &a, const Parts &parts, float c2, const RowPlace at, int t, int of_group,
                                       const Sight sight, int lane) {
    constexpr int C = D / 32;  // channels of a lane
    const int64_t token = at.first + t;
    const int head = at.kvh * (a.H / a.Hkv) + of_group;
    const __nv_bfloat16 *q = static_cast<const __nv_bfloat16 *>(a.q) + token * a.q_stride + static_cast<int64_t>(head) * D + lane * C;
    float qx[C], acc[C], top = -INFINITY, sum = 0.f;
    for (int e = 0; e < C; ++e) {
        qx[e] = __bfloat162float(q[e]);
        acc[e] = 0.f;
    }
    for (int key = at.kbeg; key < at.kend; ++key) {
        if (!sight.sees(key)) continue;
        int64_t kat, vat;
        if (a.paged) {
            const int64_t block = a.block_table[at.seq * a.width + (key >> a.shift)];
            if (block < 0 || block >= a.num_blocks) continue;
            kat = vat = (((block * a.Hkv + at.kvh) << a.shift) + (key & ((1 << a.shift) - 1))) * D;
        } else {
            kat = (static_cast<int64_t>(at.first) + key) * a.k_stride + static_cast<int64_t>(at.kvh) * D;
            vat = (static_cast<int64_t>(at.first) + key) * a.v_stride + static_cast<int64_t>(at.kvh) * D;
        }
        float s = 0.f;
        for (int e = 0; e < C; ++e) s = fmaf(qx[e], __bfloat162float(static_cast<const __nv_bfloat16 *>(a.k)[kat + lane * C + e]), s);
        for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
        s *= c2;
        const float best = fmaxf(top, s), from = best == -INFINITY ? 0.f : best;
        const float keep = ex2(top - from), p = ex2(s - from);
        top = best;
        sum = sum * keep + p;
        for (int e = 0; e < C; ++e)
            acc[e] = fmaf(p, __bfloat162float(static_cast<const __nv_bfloat16 *>(a.v)[vat + lane * C + e]), acc[e] * keep);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const float l2 = sum == 0.f ? -INFINITY : top + log2f(sum);
    if (at.chunks > 1) {
        const int64_t r = parts.row(at.chunk, token, head);
        if (lane == 0) parts.lse[r] = l2;
        for (int e = 0; e < C; ++e) parts.o[r * D + lane * C + e] = acc[e] * inv;
    } else {
        if (lane == 0 && a.lse) a.lse[token * a.H + head] = l2 * LN2;
        for (int e = 0; e < C; ++e)
            static_cast<__nv_bfloat16 *>(a.o)[(token * a.H + head) * D + lane * C + e] = __float2bfloat16_rn(acc[e] * inv);
    }
}

}  // namespace attn
}  // namespace rhz
