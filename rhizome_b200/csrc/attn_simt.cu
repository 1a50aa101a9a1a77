// Softmax attention with grouped heads in fp32 arithmetic, for every width and
// type (the f32 path, and bf16 at widths the tensor-core forms do not tile),
// the joining of split key axes, and the choice of form.
//
// For a row with query q over the keys j it sees:
//   s_j = scale q . k_j,  m = max s_j,  p_j = exp(s_j - m),
//   o = sum_j p_j v_j / sum_j p_j,  lse = m + log sum_j p_j,
// in one pass over the keys with the running m and sum; a row that sees no key
// gives o = 0 and lse = -inf.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <type_traits>

#include "attn_common.cuh"

namespace rhz {
namespace {

using namespace attn;

constexpr int THREADS = 256;
constexpr int KEYS = 64;                       // keys per tile
constexpr Split ROWS_SPLIT{512, 64};

// A bound of more rows than a tree has (pieces of a prompt) lowers the most
// chunks by the row blocks that a sequence can have, to four: the blocks fill
// the SMs themselves, and the scratch, which the most chunks of the table's
// width size, was 5 GB for 8,192 rows of 32 heads over 131,072 positions (0.5 GB
// in four chunks, 21.2 -> 17.8 ms; 2,048 rows over 65,536 keys 2.9 -> 2.4 ms). What
// it costs is a lone row in such a call: over 131,000 keys 437 us, not 134.
int chunks_beside(int64_t blocks, int wanted, int most) {
    const int64_t few = wanted / blocks;
    const int least = most < 4 ? most : 4;
    return few < least ? least : few < most ? static_cast<int>(few) : most;
}

// Keys per chunk and chunks at most on the tcgen05 form (64 at most: the join
// has two per lane). A unit costs some 3 us beside its keys, and its rows' partial
// results are written and read again, so chunks are as long as an even deal
// allows: 74 trees of 64 nodes over 8,192 keys took 768 us in chunks of 2,048,
// 706 of 4,096 and 612 of 8,192, but 48 trees over U{1..8192} keys 232, 238
// and 316. The bound gives one long sequence two units per SM (131,072 keys and
// 24 nodes: 112 us in 37 chunks, 141 in 32).
Split tc_split(const AttnArgs &a) {
    int most = 2 * 148 / a.Hkv;
    most = most < 1 ? 1 : most < 64 ? most : 64;
    const int pair = 2 * (128 / (a.H / a.Hkv));  // tokens of a unit
    if (a.most > MAX_NODES) most = chunks_beside((a.most + pair - 1) / pair, most, most);
    return {2560, most};
}

// The rule counts blocks of 64 rows, four to an SM, also where 16 go to a CTA, so
// that the bits are the same.
Split simt_split(const AttnArgs &a) {
    const int tok = 64 / (a.H / a.Hkv);
    const int most = a.most > MAX_NODES ? chunks_beside((a.most + tok - 1) / tok * a.Hkv, 4 * 148, 64) : 64;
    return {256, most};
}

// Four consecutive elements as f32 (d % 4 == 0, 16-byte aligned bases).
__device__ __forceinline__ float4 get4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
__device__ __forceinline__ float4 get4(const __nv_bfloat16 *p) {
    float x[4];
    load4(p, true, 4, x);
    return make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void set4(float *p, const float4 x) { *reinterpret_cast<float4 *>(p) = x; }
__device__ __forceinline__ void set4(__nv_bfloat16 *p, const float4 x) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x.x, x.y), b = __floats2bfloat162_rn(x.z, x.w);
    *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const uint32_t *>(&a),
                                               *reinterpret_cast<const uint32_t *>(&b));
}

__device__ __forceinline__ bool finite4(const float4 x) {
    return isfinite(x.x) && isfinite(x.y) && isfinite(x.z) && isfinite(x.w);
}

// The unit of a CTA: block b of a sequence's rows, chunk c of its keys.
struct Found {
    int32_t seq, block, chunk;
};

// Unit x of the batch, `most` to a block; seq -1 where there is none. Block j of
// a sequence whose first row is f has number f / tok + i + j, i the sequence's
// index: rounding f down loses less than the one block that i adds, so no two
// blocks meet and the numbers stay below total / tok + n_seq. The CTA finds i by
// a search that divides the sequences by its threads in each step. (Walking over
// them all instead, every CTA took as long as there are sequences: 65,536 f32
// prompts of one token, 2 heads of 32 channels, 22.1 ms against 2.5.)
__device__ Found find_unit(const AttnArgs &a, int x, int tok, Split split, int most) {
    __shared__ Found found;
    const int unit = x / most;
    auto number = [&](int i) { return seq_of(a, i).first / tok + i; };  // (the launch refuses more than 31 bits count)
    int lo = 0, hi = static_cast<int>(a.n_seq);  // number(lo) <= unit once a step is done
    do {
        const int step = (hi - lo + THREADS - 1) / THREADS;
        const int i = lo + static_cast<int>(threadIdx.x) * step;
        const int below = __syncthreads_count(i < hi && number(i) <= unit);
        if (below == 0) return {-1, 0, 0};
        lo += (below - 1) * step;
        hi = min(hi, lo + step);
    } while (hi - lo > 1);
    if (threadIdx.x == 0) {
        const Seq s = seq_of(a, lo);
        const int block = unit - number(lo), chunk = x - unit * most;
        const bool there = static_cast<int64_t>(block) * tok < s.m && chunk < (a.paged ? split.chunks(s.keys) : 1);
        found = there ? Found{lo, block, chunk} : Found{-1, 0, 0};
    }
    __syncthreads();
    return found;
}

// One CTA per (unit, K/V head): ROWS rows over the keys of one chunk, K and V
// tiles of 64 keys as f32 in shared memory. Thread (ty, tx) of 16 x 16 owns
// rows ty * RM .. and, of a tile's scores, keys tx + 16 j; of the outputs,
// channels 4 (tx + 16 g). Row strides of d + 4 floats keep the 16-byte reads
// of eight neighbouring keys on different banks. Bound by the shared-memory
// reads of the score product (five 16-byte reads to 16 RM / 4 multiply-adds),
// so 64 rows where a sequence has them, 16 where it does not.
template <typename T, int ROWS, int NG>
__global__ void __launch_bounds__(THREADS) attn_simt_kernel(const AttnArgs a, const Parts parts,
                                                            Split split) {
    constexpr int RM = ROWS / 16;
    extern __shared__ float4 smem4[];
    const int d = a.d, ld = d + 4, tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    float *sq = reinterpret_cast<float *>(smem4), *sk = sq + ROWS * ld, *sv = sk + KEYS * ld,
          *sp = sv + KEYS * d;
    const int G = a.H / a.Hkv, tok = ROWS / G, kvh = blockIdx.y;
    const Found f = find_unit(a, blockIdx.x, tok, split, parts.most);
    if (f.seq < 0) return;
    const Seq s = seq_of(a, f.seq);
    const int64_t t0 = static_cast<int64_t>(f.block) * tok;
    const int used = static_cast<int>(min(static_cast<int64_t>(tok), s.m - t0)) * G;
    const int64_t chunks = a.paged ? split.chunks(s.keys) : 1;
    int64_t kbeg = 0, kend = min(static_cast<int64_t>(s.keys), s.cached + t0 + tok);
    if (a.paged) {
        if (a.parent) kend = s.keys;
        kbeg = static_cast<int64_t>(f.chunk) * split.span(s.keys);
        kend = min(kend, kbeg + split.span(s.keys));
    }

    const int cols = d / 4;  // 4-channel groups of a row
    for (int e = tid; e < ROWS * cols; e += THREADS) {
        const int r = e / cols, c = 4 * (e - r * cols);
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < used)
            x = get4(static_cast<const T *>(a.q) + (s.first + t0 + r / G) * a.q_stride +
                     static_cast<int64_t>(kvh * G + r % G) * d + c);
        set4(sq + r * ld + c, x);
    }
    Sight sight[RM];
    float top[RM], sum[RM], acc[RM][NG][4];
#pragma unroll
    for (int i = 0; i < RM; ++i) {
        const int r = ty * RM + i;
        sight[i] = r < used ? sight_of(a, s, t0 + r / G) : Sight{0, 0};
        top[i] = -INFINITY;
        sum[i] = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][g][e] = 0.f;
    }
    const float c2 = a.scale * LOG2E;
    for (int64_t k0 = kbeg; k0 < kend; k0 += KEYS) {
        __syncthreads();
        bool odd = false;  // some value here is not finite
        for (int e = tid; e < KEYS * cols; e += THREADS) {
            const int r = e / cols, c = 4 * (e - r * cols);
            const int64_t key = k0 + r;
            float4 kx = make_float4(0.f, 0.f, 0.f, 0.f), vx = kx;
            if (key < kend) {
                int64_t kat = (s.first + key) * a.k_stride + static_cast<int64_t>(kvh) * d + c;
                int64_t vat = (s.first + key) * a.v_stride + static_cast<int64_t>(kvh) * d + c;
                bool there = true;
                if (a.paged) {
                    const int64_t block = a.block_table[f.seq * a.width + (key >> a.shift)];
                    there = block >= 0 && block < a.num_blocks;
                    kat = vat = (((block * a.Hkv + kvh) << a.shift) + (key & ((1 << a.shift) - 1))) * d + c;
                }
                if (there) {
                    kx = get4(static_cast<const T *>(a.k) + kat);
                    vx = get4(static_cast<const T *>(a.v) + vat);
                }
            }
            odd |= !finite4(vx);
            set4(sk + r * ld + c, kx);
            set4(sv + r * d + c, vx);
        }
        odd = __syncthreads_or(odd);
        // Scores.
        float x[RM][4];
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) x[i][j] = 0.f;
        for (int c = 0; c < d; c += 4) {
            float4 kx[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) kx[j] = get4(sk + (tx + 16 * j) * ld + c);
#pragma unroll
            for (int i = 0; i < RM; ++i) {
                const float4 qx = get4(sq + (ty * RM + i) * ld + c);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    x[i][j] = fmaf(qx.x, kx[j].x, fmaf(qx.y, kx[j].y, fmaf(qx.z, kx[j].z, fmaf(qx.w, kx[j].w, x[i][j]))));
            }
        }
        bool there[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t key = k0 + tx + 16 * j;
            there[j] = key < kend;
            if (a.paged && there[j]) {
                const int64_t block = a.block_table[f.seq * a.width + (key >> a.shift)];
                there[j] = block >= 0 && block < a.num_blocks;
            }
        }
#pragma unroll
        for (int i = 0; i < RM; ++i) {
            bool in[4];
            float best = top[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                in[j] = there[j] && sight[i].sees(k0 + tx + 16 * j);
                x[i][j] *= c2;
                if (in[j]) best = fmaxf(best, x[i][j]);
            }
#pragma unroll
            for (int off = 1; off < 16; off <<= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, off));
            const float from = best == -INFINITY ? 0.f : best;
            const float keep = exp2f(top[i] - from);
            top[i] = best;
            float part = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p = in[j] ? exp2f(x[i][j] - from) : 0.f;
                part += p;
                // A masked key must not touch the row, 0 * NaN would: where the
                // tile holds such values, -1 marks what the product skips.
                sp[(ty * RM + i) * (KEYS + 4) + tx + 16 * j] = odd && !in[j] ? -1.f : p;
            }
            sum[i] = sum[i] * keep + part;  // this thread's keys; joined at the end
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][g][e] *= keep;
        }
        __syncwarp();  // a row's probabilities come from and go to one half-warp
        auto products = [&](auto guarded) {
            for (int j = 0; j < KEYS; j += 4) {
                float4 p4[RM];
#pragma unroll
                for (int i = 0; i < RM; ++i) p4[i] = get4(sp + (ty * RM + i) * (KEYS + 4) + j);
#pragma unroll
                for (int jj = 0; jj < 4; ++jj)
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        const int c = 4 * (tx + 16 * g);
                        if (c >= d) continue;
                        const float4 vx = get4(sv + (j + jj) * d + c);
#pragma unroll
                        for (int i = 0; i < RM; ++i) {
                            const float p = jj == 0 ? p4[i].x : jj == 1 ? p4[i].y : jj == 2 ? p4[i].z : p4[i].w;
                            if (decltype(guarded)::value && p < 0.f) continue;
                            acc[i][g][0] = fmaf(p, vx.x, acc[i][g][0]);
                            acc[i][g][1] = fmaf(p, vx.y, acc[i][g][1]);
                            acc[i][g][2] = fmaf(p, vx.z, acc[i][g][2]);
                            acc[i][g][3] = fmaf(p, vx.w, acc[i][g][3]);
                        }
                    }
            }
        };
        if (odd) products(std::true_type{});
        else products(std::false_type{});
    }
#pragma unroll
    for (int i = 0; i < RM; ++i) {
        float l = sum[i];
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
        const int r = ty * RM + i;
        if (r >= used) continue;
        const int64_t token = s.first + t0 + r / G;
        const int head = kvh * G + r % G;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const float l2 = l == 0.f ? -INFINITY : top[i] + log2f(l);
        auto result = [&](int g) {  // (zeros where every score is -inf, whatever 0 * inf left in the sums; a chunk keeps that for the join)
            return l == 0.f && chunks == 1 ? make_float4(0.f, 0.f, 0.f, 0.f)
                                           : make_float4(acc[i][g][0] * inv, acc[i][g][1] * inv, acc[i][g][2] * inv, acc[i][g][3] * inv);
        };
        if (chunks > 1) {
            const int64_t row = parts.row(f.chunk, token, head);
            if (tx == 0) parts.lse[row] = l2;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const int c = 4 * (tx + 16 * g);
                if (c < d) set4(parts.o + row * d + c, result(g));
            }
        } else {
            if (tx == 0 && a.lse) a.lse[token * a.H + head] = l2 * LN2;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const int c = 4 * (tx + 16 * g);
                if (c < d) set4(static_cast<T *>(a.o) + (token * a.H + head) * d + c, result(g));
            }
        }
        if (parts.count && tx == 0 && f.chunk == 0 && head == 0) parts.count[token] = static_cast<int32_t>(chunks);
    }
}

// Joins the chunks of a row: o = sum_c 2^(lse_c - lse) o_c in order of
// position, one warp per (token, head). Rows of one chunk are final already.
template <typename T, int FLIGHT>
__global__ void __launch_bounds__(256) attn_join_kernel(const AttnArgs a, const Parts parts) {
    const int lane = threadIdx.x & 31;
    const int64_t row = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    const int64_t token = row / a.H;
    cudaGridDependencySynchronize();  // launched early: the chunks' results are there from here on
    if (token >= a.total_tokens || token >= a.cu_seqlens[a.n_seq] || token < a.cu_seqlens[0]) return;
    const int head = static_cast<int>(row - token * a.H);
    const int chunks = min(parts.count[token], parts.most);
    if (chunks <= 1) return;
    float top = -INFINITY, mine[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int c = lane + 32 * u;
        mine[u] = c < chunks ? parts.lse[parts.row(c, token, head)] : -INFINITY;
        top = fmaxf(top, mine[u]);  // a NaN stays in mine[] and reaches the sum
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    const float from = top == -INFINITY ? 0.f : top;
    float total = 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        mine[u] = exp2f(mine[u] - from);
        total += mine[u];
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
    const float inv = total == 0.f ? 0.f : 1.f / total;
    // FLIGHT chunks' loads at a time: with four, 64 chunks of a row took a
    // warp 39 us, sixteen round trips to memory (sixteen: 12 us); for many rows
    // of few chunks, four leave room for more warps (27 us against 48 us for
    // the rows of 48 trees).
    float acc[2][4] = {};
    const float *src = parts.o + parts.row(0, token, head) * a.d + 4 * lane;
    const int64_t next = parts.tokens * a.H * a.d;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        const bool has = 4 * lane + 128 * g < a.d;
        for (int c0 = 0; c0 < chunks && 128 * g < a.d; c0 += FLIGHT) {
            float4 x[FLIGHT];
#pragma unroll
            for (int k = 0; k < FLIGHT; ++k)
                if (has && c0 + k < chunks) x[k] = get4(src + (c0 + k) * next + 128 * g);
#pragma unroll
            for (int k = 0; k < FLIGHT; ++k) {
                const int c = c0 + k;
                const float w = __shfl_sync(0xffffffffu, c < 32 ? mine[0] : mine[1], c & 31);
                if (!has || c >= chunks) continue;
                acc[g][0] = fmaf(w, x[k].x, acc[g][0]);
                acc[g][1] = fmaf(w, x[k].y, acc[g][1]);
                acc[g][2] = fmaf(w, x[k].z, acc[g][2]);
                acc[g][3] = fmaf(w, x[k].w, acc[g][3]);
            }
        }
    }
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        const int col = 4 * lane + 128 * g;
        if (col < a.d)
            set4(static_cast<T *>(a.o) + (token * a.H + head) * a.d + col,
                 total == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f)
                              : make_float4(acc[g][0] * inv, acc[g][1] * inv, acc[g][2] * inv, acc[g][3] * inv));
    }
    if (lane == 0 && a.lse)
        a.lse[token * a.H + head] = total == 0.f ? -INFINITY : (top + log2f(total)) * LN2;
}

int launch_join(const AttnArgs &a, const Parts &parts) {
    // Its launch overlaps the end of the kernel before it.
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>((a.total_tokens * a.H + 7) / 8));
    cfg.blockDim = dim3(256);
    cfg.stream = a.stream;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    const bool few = parts.most <= 8, bf16 = a.dtype == RHZ_DTYPE_BF16;
    auto *kernel = bf16 ? (few ? attn_join_kernel<__nv_bfloat16, 4> : attn_join_kernel<__nv_bfloat16, 16>)
                        : (few ? attn_join_kernel<float, 4> : attn_join_kernel<float, 16>);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a, parts);
    if (e != cudaSuccess) return set_error(RHZ_ERR_DEVICE, "attn_join_kernel: %s", cudaGetErrorString(e));
    return check_launch("attn_join_kernel");
}

template <typename T, int ROWS, int NG>
int launch_simt_t(const AttnArgs &a, const Parts &parts, Split split) {
    auto bytes = [](int d) { return 4 * ((ROWS + KEYS) * (d + 4) + KEYS * d + ROWS * (KEYS + 4)); };
    const int tok = ROWS / (a.H / a.Hkv);
    const int64_t units = (a.total_tokens / tok + a.n_seq) * parts.most;
    if (units > INT32_MAX) return set_error(RHZ_ERR_SHAPE, "attention over %lld units exceeds the grid", (long long)units);
    cudaError_t e = cudaFuncSetAttribute(attn_simt_kernel<T, ROWS, NG>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         bytes(64 * NG));  // for every d, whatever another thread launches
    if (e != cudaSuccess) return set_error(RHZ_ERR_DEVICE, "attn_simt_kernel: %s", cudaGetErrorString(e));
    dim3 grid(static_cast<unsigned>(units), static_cast<unsigned>(a.Hkv));
    attn_simt_kernel<T, ROWS, NG><<<grid, THREADS, bytes(a.d), a.stream>>>(a, parts, split);
    return check_launch("attn_simt_kernel");
}

template <typename T, int ROWS>
int launch_simt_r(const AttnArgs &a, const Parts &parts, Split split) {
    if (a.d <= 64) return launch_simt_t<T, ROWS, 1>(a, parts, split);
    if (a.d <= 128) return launch_simt_t<T, ROWS, 2>(a, parts, split);
    return launch_simt_t<T, ROWS, 4>(a, parts, split);
}

// The tokens a sequence may have at most: a paged call says so, a packed one
// is judged by its whole stream.
int64_t rows_bound(const AttnArgs &a) {
    const int64_t t = a.paged && a.most < a.total_tokens ? a.most : a.total_tokens;
    return t * (a.H / a.Hkv);
}

// 16 rows to a CTA where a sequence has no more, or where 64 would leave SMs
// without work; a row's arithmetic is the same in both, so the batch may choose.
// f32, d = 32, 2 heads over 1: one prompt of 1,000 tokens 103 us in 64 rows, 55
// in 16; 8 prompts, 8 over 4: 349 and 508; one of 1,000 with d = 128, 8 over 4, at
// 128 CTAs of 64 rows: 266 and 253.
int launch_simt(const AttnArgs &a, const Parts &parts, Split split) {
    const int group = a.H / a.Hkv;
    const int64_t wide = (a.total_tokens / (64 / group) + a.n_seq) * parts.most * a.Hkv;  // CTAs of 64 rows, at most
    const bool few = group <= 16 && (rows_bound(a) <= 16 || wide <= 148);
    if (a.dtype == RHZ_DTYPE_BF16)
        return few ? launch_simt_r<__nv_bfloat16, 16>(a, parts, split) : launch_simt_r<__nv_bfloat16, 64>(a, parts, split);
    return few ? launch_simt_r<float, 16>(a, parts, split) : launch_simt_r<float, 64>(a, parts, split);
}

Split split_of(const AttnArgs &a) {
    return attn_rows_supports(a) ? ROWS_SPLIT : attn_tc_supports(a) ? tc_split(a) : simt_split(a);
}

int64_t chunk_bound(const AttnArgs &a) {
    return a.paged ? split_of(a).bound(a.width << a.shift) : 1;
}

}  // namespace

size_t attn_ws_bytes(const AttnArgs &a) {
    return parts_bytes(a.total_tokens, a.H, a.d, chunk_bound(a));
}

int launch_attn(const AttnArgs &a) {
    if (a.n_seq == 0 || a.total_tokens == 0) return RHZ_OK;
    const int64_t chunks = chunk_bound(a);
    const Parts parts = parts_at(a.ws, a.total_tokens, a.H, a.d, chunks);
    const Split split = split_of(a);
    // A cache of no pages has no tensor map; nothing is seen there.
    const bool none = a.paged && a.num_blocks == 0;
    const int st = none                    ? launch_simt(a, parts, split)
                   : attn_rows_supports(a) ? launch_attn_rows(a, parts, split)
                   : attn_tc_supports(a)   ? launch_attn_tc(a, parts, split)
                                           : launch_simt(a, parts, split);
    if (st != RHZ_OK || chunks <= 1) return st;
    return launch_join(a, parts);
}

int attn_status(int *flag, bool clear) {
    int x = 0, y = 0;
    int st = attn_tc_status(&x, clear);
    if (st == RHZ_OK) st = attn_rows_status(&y, clear);
    *flag = x | y;
    return st;
}

}  // namespace rhz
