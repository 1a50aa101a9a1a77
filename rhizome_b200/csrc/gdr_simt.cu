// SIMT kernels of the GDR library (sm_100a):
//   - gdr_step_kernel: one position of the recurrence for a ragged batch of
//     sequences whose states live in a slot pool (decode, memory bound);
//   - gdr_multistep_kernel, gdr_tree_kernel: a few drafted positions per
//     sequence, a chain or a tree of them, with the state after every one;
//   - gdr_seq_kernel: the recurrence applied position by position over whole
//     sequences in fp32 (the rtol-1e-5 path, and the path for head widths the
//     tensor-core kernel does not tile).
//
// All follow gated_delta_step (crates/ops/src/delta.rs:93-127) per row:
//   sk_i = sum_j S_ij k_j
//   S_ij <- alpha (S_ij - (beta sk_i) k_j) + (beta v_i) k_j
//   o_i  = sum_j S_ij q_j
// Rows (the v index i) are independent, so a (sequence, head) can be split
// into row blocks across warps and CTAs with no cross-CTA reduction.
//
// Register layout: a warp owns RPW consecutive rows; lane l owns the column
// vectors j = 128 c + 4 l + e (c < NV, e < 4). A row's partial dot products
// are combined with a transposing butterfly: RPW values per lane are halved
// at each of the first log2(RPW) xor-shuffle levels, so the sums of 16 rows
// cost 16 shuffles (plus 16 to broadcast them back) instead of 5 per row.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "common.cuh"
#include "kernels.h"

namespace rhz {
namespace {

constexpr unsigned FULL = 0xffffffffu;

template <int N> struct Log2 { static constexpr int value = 1 + Log2<N / 2>::value; };
template <> struct Log2<1> { static constexpr int value = 0; };

// After the call, v[0] on lane l holds the full 32-lane sum of row
// (l >> (5 - log2 N)); every lane of that row's group holds it.
template <int N>
__device__ __forceinline__ void transpose_reduce(float (&v)[N], int lane) {
#pragma unroll
    for (int half = N / 2, off = 16; half >= 1; half /= 2, off /= 2) {
        const bool upper = (lane & off) != 0;
#pragma unroll
        for (int i = 0; i < half; ++i) {
            float send = upper ? v[i] : v[i + half];
            float keep = upper ? v[i + half] : v[i];
            v[i] = keep + __shfl_xor_sync(FULL, send, off);
        }
    }
#pragma unroll
    for (int off = 16 >> Log2<N>::value; off >= 1; off /= 2) v[0] += __shfl_xor_sync(FULL, v[0], off);
}

// Row sums of s[r][.] . x[.] for this warp's RPW rows. Returns (via out[r])
// the full sum of every row on every lane; `mine` gets the sum of the row
// this lane represents (row index lane >> SHIFT).
template <int RPW, int NV>
__device__ __forceinline__ void row_dots(const float (&s)[RPW][NV][4], const float (&x)[NV][4],
                                         int lane, float (&out)[RPW], float &mine) {
    float p[RPW];
#pragma unroll
    for (int r = 0; r < RPW; ++r) {
        float acc = 0.f;
#pragma unroll
        for (int c = 0; c < NV; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc = fmaf(s[r][c][e], x[c][e], acc);
        p[r] = acc;
    }
    transpose_reduce<RPW>(p, lane);
    mine = p[0];
    constexpr int SHIFT = 5 - Log2<RPW>::value;
#pragma unroll
    for (int r = 0; r < RPW; ++r) out[r] = __shfl_sync(FULL, p[0], r << SHIFT);
}

template <int RPW, int NV>
__device__ __forceinline__ void rank1_update(float (&s)[RPW][NV][4], const float (&kk)[NV][4],
                                             const float (&sk)[RPW], const float (&vr)[RPW],
                                             float a, float b) {
#pragma unroll
    for (int r = 0; r < RPW; ++r) {
        const float bsk = b * sk[r];
        const float bv = b * vr[r];
#pragma unroll
        for (int c = 0; c < NV; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float decayed = a * (s[r][c][e] - bsk * kk[c][e]);
                s[r][c][e] = decayed + bv * kk[c][e];
            }
    }
}

__device__ __forceinline__ int nvalid(int d, int j) {
    int n = d - j;
    return n < 0 ? 0 : (n > 4 ? 4 : n);
}

// ------------------------------------------------------------------ decode

template <typename T, int RPW, int NV, int WARPS>
__global__ void __launch_bounds__(WARPS * 32)
    gdr_step_kernel(T *__restrict__ o, float *__restrict__ pool, const int32_t *__restrict__ slots,
                    const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
                    const float *__restrict__ alpha, const float *__restrict__ beta,
                    int64_t num_slots, int H, int d, bool vec) {
    const int64_t item = blockIdx.x;  // sequence * H + head
    const int64_t seq = item / H;
    const int h = static_cast<int>(item - seq * H);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row0 = blockIdx.y * (WARPS * RPW) + warp * RPW;
    if (row0 >= d) return;
    constexpr int SHIFT = 5 - Log2<RPW>::value;
    const int myrow = row0 + (lane >> SHIFT);
    const bool writer = (lane & ((1 << SHIFT) - 1)) == 0 && myrow < d;

    const int64_t slot = slots ? static_cast<int64_t>(slots[seq]) : seq;
    T *op = o + item * d;
    if (slot < 0 || slot >= num_slots) {
        if (writer) op[myrow] = from_f32<T>(nanf(""));
        return;
    }
    const T *qp = q + item * d, *kp = k + item * d, *vp = v + item * d;
    float *S = pool + (static_cast<int64_t>(slot) * H + h) * static_cast<int64_t>(d) * d;

    float s[RPW][NV][4];
#pragma unroll
    for (int r = 0; r < RPW; ++r) {
        const int row = row0 + r;
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            const int j = 128 * c + 4 * lane;
            if (row < d) {
                load4(S + static_cast<int64_t>(row) * d + j, vec, nvalid(d, j), s[r][c]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) s[r][c][e] = 0.f;
            }
        }
    }
    float kk[NV][4], qq[NV][4], vr[RPW];
#pragma unroll
    for (int c = 0; c < NV; ++c) {
        const int j = 128 * c + 4 * lane;
        load4(kp + j, vec, nvalid(d, j), kk[c]);
        load4(qp + j, vec, nvalid(d, j), qq[c]);
    }
#pragma unroll
    for (int r = 0; r < RPW; ++r) vr[r] = row0 + r < d ? to_f32(vp[row0 + r]) : 0.f;
    const float a = alpha[item], b = beta[item];

    float sk[RPW], mine;
    row_dots<RPW, NV>(s, kk, lane, sk, mine);
    rank1_update<RPW, NV>(s, kk, sk, vr, a, b);
#pragma unroll
    for (int r = 0; r < RPW; ++r) {
        const int row = row0 + r;
        if (row < d) {
#pragma unroll
            for (int c = 0; c < NV; ++c) {
                const int j = 128 * c + 4 * lane;
                store4(S + static_cast<int64_t>(row) * d + j, vec, nvalid(d, j), s[r][c]);
            }
        }
    }
    float ov[RPW];
    row_dots<RPW, NV>(s, qq, lane, ov, mine);
    if (writer) op[myrow] = from_f32<T>(mine);
}

// ------------------------------------------------------------------ multistep

// gated_delta_multistep (delta.rs:201-230) for n sequences x H heads of up
// to Tn positions: the state rows stay in registers across the positions and
// the state after every position is written out (speculative decoding keeps
// them to roll back to the last accepted draft token). With pool == nullptr
// the state starts at zero and resets wherever the segment id changes (the
// reference's semantics; its reset at t = 0 discards `init`); otherwise it
// starts from pool[slot] and the pool is left untouched.
template <typename T, int RPW, int NV, int WARPS>
__global__ void __launch_bounds__(WARPS * 32)
    gdr_multistep_kernel(T *__restrict__ outs, float *__restrict__ states,
                         const float *__restrict__ pool, const int32_t *__restrict__ slots,
                         const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
                         const float *__restrict__ alpha, const float *__restrict__ beta,
                         const int64_t *__restrict__ segment, int64_t Tin, int Tn,
                         int64_t num_slots, int H, int d, bool vec) {
    const int64_t item = blockIdx.x;  // sequence * H + head
    const int64_t seq = item / H;
    const int h = static_cast<int>(item - seq * H);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row0 = blockIdx.y * (WARPS * RPW) + warp * RPW;
    if (row0 >= d) return;
    constexpr int SHIFT = 5 - Log2<RPW>::value;
    const int myrow = row0 + (lane >> SHIFT);
    const bool writer = (lane & ((1 << SHIFT) - 1)) == 0 && myrow < d;
    const int64_t dd = static_cast<int64_t>(d) * d;

    float s[RPW][NV][4];
    bool valid = true;
    if (pool) {
        const int64_t slot = slots ? static_cast<int64_t>(slots[seq]) : seq;
        valid = slot >= 0 && slot < num_slots;
        const float *S = valid ? pool + (slot * H + h) * dd : nullptr;
#pragma unroll
        for (int r = 0; r < RPW; ++r)
#pragma unroll
            for (int c = 0; c < NV; ++c) {
                const int j = 128 * c + 4 * lane;
                if (valid && row0 + r < d) {
                    load4(S + static_cast<int64_t>(row0 + r) * d + j, vec, nvalid(d, j), s[r][c]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[r][c][e] = 0.f;
                }
            }
    } else {
#pragma unroll
        for (int r = 0; r < RPW; ++r)
#pragma unroll
            for (int c = 0; c < NV; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[r][c][e] = 0.f;
    }
    const int64_t row_stride = static_cast<int64_t>(H) * d;
    for (int t = 0; t < Tn; ++t) {
        const int64_t tok = seq * Tin + t;
        if (!pool && segment && t > 0 && segment[tok] != segment[tok - 1]) {
#pragma unroll
            for (int r = 0; r < RPW; ++r)
#pragma unroll
                for (int c = 0; c < NV; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[r][c][e] = 0.f;
        }
        const T *qp = q + tok * row_stride + static_cast<int64_t>(h) * d;
        const T *kp = k + tok * row_stride + static_cast<int64_t>(h) * d;
        const T *vp = v + tok * row_stride + static_cast<int64_t>(h) * d;
        float kk[NV][4], qq[NV][4], vr[RPW];
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            const int j = 128 * c + 4 * lane;
            load4(kp + j, vec, nvalid(d, j), kk[c]);
            load4(qp + j, vec, nvalid(d, j), qq[c]);
        }
#pragma unroll
        for (int r = 0; r < RPW; ++r) vr[r] = row0 + r < d ? to_f32(vp[row0 + r]) : 0.f;
        const float a = alpha[tok * H + h], b = beta[tok * H + h];
        float sk[RPW], ov[RPW], mine;
        row_dots<RPW, NV>(s, kk, lane, sk, mine);
        rank1_update<RPW, NV>(s, kk, sk, vr, a, b);
        row_dots<RPW, NV>(s, qq, lane, ov, mine);
        T *op = outs + (seq * Tn + t) * row_stride + static_cast<int64_t>(h) * d;
        if (writer) op[myrow] = valid ? from_f32<T>(mine) : from_f32<T>(nanf(""));
        float *St = states + ((seq * Tn + t) * H + h) * dd;
#pragma unroll
        for (int r = 0; r < RPW; ++r) {
            if (row0 + r < d) {
#pragma unroll
                for (int c = 0; c < NV; ++c) {
                    const int j = 128 * c + 4 * lane;
                    store4(St + static_cast<int64_t>(row0 + r) * d + j, vec, nvalid(d, j), s[r][c]);
                }
            }
        }
    }
}

// ------------------------------------------------------------------ tree

// The recurrence over a tree of drafted tokens: node t of sequence i starts
// from the state of its parent node, S_t = step(S_parent(t)), or from the
// pool's slot where the parent is -1, and every node's state is written out.
// The rows of S never mix, so a warp that owns 4 NR rows walks the whole tree
// by itself: a node whose parent is the node before it finds the parent's
// rows in registers, any other reads back what this warp wrote for the parent
// (the same lanes at the same addresses, so program order is enough).
//
// The traffic that cannot be avoided is the d x d f32 state written per node
// and head. Eight lanes share a row here (lane 8 g + c: rows g + 4 i, columns
// 4 c + 32 j): a row's product is 4 NJ multiply-adds and three shuffles, and
// its sum is where it is needed, on the eight lanes that update the row. (A
// whole warp to a row, as in the kernels above, took twice as many
// instructions and was bound by them: 840 us for 32 trees of up to 64 nodes,
// 32 heads, against 404 us of traffic.) The tree's q, k, v, gates and parents
// come into shared memory first, all at once: fetched one node ahead they still
// kept every node waiting for memory (650 us). Only a parent's rows are
// fetched node by node, one ahead, unless the parent is the node before.
// EXACT: d == 32 NJ, no bounds checks on columns and rows.
template <typename T, int NR, int NJ, int WARPS, bool EXACT>
__global__ void __launch_bounds__(WARPS * 32)
    gdr_tree_kernel(T *__restrict__ o, float *states, const float *__restrict__ pool,
                    const int32_t *__restrict__ slots, const int32_t *__restrict__ cu,
                    const int32_t *__restrict__ parent, const T *__restrict__ q,
                    const T *__restrict__ k, const T *__restrict__ v,
                    const float *__restrict__ alpha, const float *__restrict__ beta,
                    int64_t total, int most, int64_t num_slots, int H, int d, bool vec) {
    const int64_t item = blockIdx.x;  // sequence * H + head
    const int64_t seq = item / H;
    const int h = static_cast<int>(item - seq * H);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row0 = (blockIdx.y * WARPS + warp) * (4 * NR) + (lane >> 3);  // and every fourth from there
    const int col0 = 4 * (lane & 7);
    const bool writer = (lane & 7) == 0;
    const int dd = d * d;
    const int64_t first = min(max(static_cast<int64_t>(cu[seq]), int64_t{0}), total);
    const int64_t last = min(max(static_cast<int64_t>(cu[seq + 1]), first), total);
    const int m = static_cast<int>(min(last - first, static_cast<int64_t>(INT32_MAX)));
    const int64_t slot = !pool ? 0 : slots ? static_cast<int64_t>(slots[seq]) : seq;
    const bool valid = !pool || (slot >= 0 && slot < num_slots);
    const float *root = pool && valid ? pool + (slot * H + h) * dd : nullptr;
    const int nodes = min(m, most);
    T *o0 = o + (first * H + h) * d;
    float *s0 = states + (first * H + h) * dd;
    const int64_t node_state = static_cast<int64_t>(H) * dd;
    const int node_row = H * d;

    // q, k, v [nodes][d], alpha, beta, parent [nodes].
    extern __shared__ float4 tree_smem[];
    T *sq = reinterpret_cast<T *>(tree_smem), *sk = sq + most * d, *sv = sk + most * d;
    float *sa = reinterpret_cast<float *>(sv + most * d + (most * d & 1)), *sb = sa + most;
    int *sp = reinterpret_cast<int *>(sb + most);
    {
        const int64_t at0 = (first * H + h) * d;
        if (EXACT) {
            constexpr int PER = 16 / sizeof(T), PIECES = 32 * NJ / PER;
            for (int e = threadIdx.x; e < nodes * PIECES; e += WARPS * 32) {
                const int t = e / PIECES, c = (e - t * PIECES) * PER;
                const int64_t from = at0 + static_cast<int64_t>(t) * node_row + c;
                *reinterpret_cast<uint4 *>(sq + t * d + c) = *reinterpret_cast<const uint4 *>(q + from);
                *reinterpret_cast<uint4 *>(sk + t * d + c) = *reinterpret_cast<const uint4 *>(k + from);
                *reinterpret_cast<uint4 *>(sv + t * d + c) = *reinterpret_cast<const uint4 *>(v + from);
            }
        } else {
            for (int e = threadIdx.x; e < nodes * d; e += WARPS * 32) {
                const int t = e / d;
                const int64_t from = at0 + static_cast<int64_t>(t) * node_row + (e - t * d);
                sq[e] = q[from];
                sk[e] = k[from];
                sv[e] = v[from];
            }
        }
        for (int t = threadIdx.x; t < nodes; t += WARPS * 32) {
            sa[t] = alpha[(first + t) * H + h];
            sb[t] = beta[(first + t) * H + h];
            sp[t] = parent ? parent[first + t] : t - 1;
        }
    }
    __syncthreads();

    // Nodes whose state is read again: some child is not the node after it.
    // The other states are stored so as to leave L2 first (those 32 trees: 532 ->
    // 515 us; 6.0 TB/s of HBM traffic, a sixth of it parents that had left L2).
    uint64_t again = 0;
#pragma unroll
    for (int u = 0; u < 64; u += 32) {
        const int t = lane + u, p = t < nodes ? sp[t] : -1;
        const uint64_t bit = p >= 0 && p < t - 1 ? uint64_t{1} << p : 0;
        again |= __reduce_or_sync(FULL, static_cast<uint32_t>(bit));
        again |= static_cast<uint64_t>(__reduce_or_sync(FULL, static_cast<uint32_t>(bit >> 32))) << 32;
    }
    float s[NR][NJ][4], ahead[NR][NJ][4];
    auto fetch = [&](const float *S, float (&to)[NR][NJ][4]) {  // this lane's part of a state, zeros without one
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int row = row0 + 4 * i, col = col0 + 32 * j;
                if (EXACT && S != nullptr) {
                    const float4 x = *reinterpret_cast<const float4 *>(S + row * d + col);
                    to[i][j][0] = x.x; to[i][j][1] = x.y; to[i][j][2] = x.z; to[i][j][3] = x.w;
                } else if (S != nullptr && row < d) {
                    load4(S + row * d + col, vec, nvalid(d, col), to[i][j]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) to[i][j][e] = 0.f;
                }
            }
    };
    // Sums over a row's columns of s[i][.] x[.], on all eight lanes of the row.
    auto dots = [&](const float (&x)[NJ][4], float (&sum)[NR]) {
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) part[e] = fmaf(s[i][j][e], x[j][e], part[e]);
            sum[i] = (part[0] + part[1]) + (part[2] + part[3]);
        }
#pragma unroll
        for (int off = 1; off < 8; off <<= 1)
#pragma unroll
            for (int i = 0; i < NR; ++i) sum[i] += __shfl_xor_sync(FULL, sum[i], off);
    };
    struct alignas(4 * sizeof(T)) Four { T x[4]; };
    auto columns = [&](const T *row, float (&x)[NJ][4]) {  // this lane's columns of a row in shared memory
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            if (EXACT) {
                const Four f = *reinterpret_cast<const Four *>(row + col0 + 32 * j);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[j][e] = to_f32(f.x[e]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[j][e] = col0 + 32 * j + e < d ? to_f32(row[col0 + 32 * j + e]) : 0.f;
            }
        }
    };
    uint64_t live = 0;  // nodes that take part: their parent is -1 or a live node before them
    auto begin = [&](int t) -> int {  // notes whether node t takes part; its parent
        const int p = sp[t];
        if (p == -1 || (p >= 0 && p < t && (live >> p & 1))) live |= uint64_t{1} << t;
        return p;
    };
    int held = -2;   // the node whose state s holds
    int ready = -2;  // the node whose state `ahead` holds (-1: the root's)
    int pn = nodes > 0 ? begin(0) : -2;
    if (live & 1) {
        fetch(root, ahead);
        ready = -1;
    }
    for (int t = 0; t < nodes; ++t) {
        const int p = pn;
        const bool takes_part = live >> t & 1;
        if (takes_part && p != held) {
            if (p != ready) fetch(p < 0 ? root : s0 + p * node_state, ahead);
            ready = -2;
#pragma unroll
            for (int i = 0; i < NR; ++i)
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[i][j][e] = ahead[i][j][e];
        }
        if (t + 1 < nodes) {
            pn = begin(t + 1);
            // A parent before t: its rows are written (by this warp) already.
            if ((live >> (t + 1) & 1) && pn != t) {
                fetch(pn < 0 ? root : s0 + pn * node_state, ahead);
                ready = pn;
            }
        }
        T *op = o0 + static_cast<int64_t>(t) * node_row;
        if (!takes_part) {
#pragma unroll
            for (int i = 0; i < NR; ++i)
                if (writer && (EXACT || row0 + 4 * i < d)) op[row0 + 4 * i] = from_f32<T>(0.f);
            continue;
        }
        held = t;
        const float a = sa[t], b = sb[t];
        float sum[NR], kk[NJ][4];
        columns(sk + t * d, kk);
        dots(kk, sum);
        float *St = s0 + t * node_state;
        const bool keep = again >> t & 1;
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const float vi = EXACT || row0 + 4 * i < d ? to_f32(sv[t * d + row0 + 4 * i]) : 0.f;
            const float bsk = b * sum[i], bv = b * vi;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float decayed = a * (s[i][j][e] - bsk * kk[j][e]);
                    s[i][j][e] = decayed + bv * kk[j][e];
                }
                const int row = row0 + 4 * i, col = col0 + 32 * j;
                float4 *to = reinterpret_cast<float4 *>(St + row * d + col);
                const float4 x = make_float4(s[i][j][0], s[i][j][1], s[i][j][2], s[i][j][3]);
                if (EXACT && keep)
                    *to = x;
                else if (EXACT)
                    __stcs(to, x);
                else if (row < d)
                    store4(St + row * d + col, vec, nvalid(d, col), s[i][j]);
            }
        }
        columns(sq + t * d, kk);
        dots(kk, sum);
#pragma unroll
        for (int i = 0; i < NR; ++i)
            if (writer && (EXACT || row0 + 4 * i < d)) op[row0 + 4 * i] = valid ? from_f32<T>(sum[i]) : from_f32<T>(nanf(""));
    }
    for (int t = nodes; t < m; ++t) {  // past the bound: not part of the tree
#pragma unroll
        for (int i = 0; i < NR; ++i)
            if (writer && (EXACT || row0 + 4 * i < d)) o0[static_cast<int64_t>(t) * node_row + row0 + 4 * i] = from_f32<T>(0.f);
    }
}

// ------------------------------------------------------------------ sequential

// Tile of TS positions staged in shared memory: k and q rows (all d
// columns), the CTA's v rows, alpha and beta.
template <typename T, int ROWS, int TS>
struct SeqTile {
    static size_t bytes(int d) {
        return (size_t(2) * TS * d + size_t(TS) * ROWS) * sizeof(float) + 2 * TS * sizeof(float);
    }
};

template <typename T, int RPW, int NV, int WARPS, int TS>
__global__ void __launch_bounds__(WARPS * 32)
    gdr_seq_kernel(T *__restrict__ o, const T *__restrict__ q, const T *__restrict__ k,
                   const T *__restrict__ v, const float *__restrict__ alpha,
                   const float *__restrict__ beta, const int32_t *__restrict__ cu_seqlens,
                   const int32_t *__restrict__ n_seq_dev, int64_t n_seq_host, int64_t seq_len,
                   int64_t total_tokens,
                   const float *__restrict__ state_in, const int32_t *__restrict__ in_slots,
                   float *__restrict__ state_out, const int32_t *__restrict__ out_slots,
                   int64_t num_slots, int H, int d, bool vec) {
    constexpr int ROWS = WARPS * RPW;
    constexpr int SHIFT = 5 - Log2<RPW>::value;
    extern __shared__ float4 smem_raw[];
    float *smem = reinterpret_cast<float *>(smem_raw);
    float *sk_ = smem;                       // [TS][d]
    float *sq_ = sk_ + TS * d;               // [TS][d]
    float *sv_ = sq_ + TS * d;               // [TS][ROWS]
    float *sa_ = sv_ + TS * ROWS;            // [TS]
    float *sb_ = sa_ + TS;                   // [TS]
    const int nthr = WARPS * 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rb0 = blockIdx.y * ROWS;
    const int row0 = rb0 + warp * RPW;
    const int myrow = row0 + (lane >> SHIFT);
    const bool writer = (lane & ((1 << SHIFT) - 1)) == 0 && myrow < d;
    const int64_t row_stride = static_cast<int64_t>(H) * d;  // token stride in q/k/v/o

    int64_t n_seq = n_seq_host;
    if (n_seq_dev) {
        const int64_t nd = *n_seq_dev;
        n_seq = nd < n_seq ? nd : n_seq;
    }
    const int64_t n_items = n_seq * H;

    // Persistent loop over (sequence, head) items; all threads of the CTA
    // take the same item, so the barriers below stay uniform.
    for (int64_t item = blockIdx.x; item < n_items; item += gridDim.x) {
        const int64_t seq = item / H;
        const int h = static_cast<int>(item - seq * H);
        int64_t t0, t1;
        if (cu_seqlens) {
            // Offsets are caller data: clamp them to the packed stream.
            t0 = cu_seqlens[seq];
            t1 = cu_seqlens[seq + 1];
            t0 = t0 < 0 ? 0 : (t0 > total_tokens ? total_tokens : t0);
            t1 = t1 < t0 ? t0 : (t1 > total_tokens ? total_tokens : t1);
        } else {
            t0 = seq * seq_len;
            t1 = t0 + seq_len;
        }

        // Initial state rows: zeros unless state_in is given (the reset at a
        // segment start, delta.rs:139-141, is the zero case).
        float s[RPW][NV][4];
        int64_t in_slot = -1;
        if (state_in) in_slot = in_slots ? static_cast<int64_t>(in_slots[seq]) : seq;
        const bool have_in = state_in && in_slot >= 0 && in_slot < num_slots;
        const float *Sin =
            have_in ? state_in + (in_slot * H + h) * static_cast<int64_t>(d) * d : nullptr;
#pragma unroll
        for (int r = 0; r < RPW; ++r) {
            const int row = row0 + r;
#pragma unroll
            for (int c = 0; c < NV; ++c) {
                const int j = 128 * c + 4 * lane;
                if (have_in && row < d) {
                    load4(Sin + static_cast<int64_t>(row) * d + j, vec, nvalid(d, j), s[r][c]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[r][c][e] = 0.f;
                }
            }
        }

        for (int64_t tt = t0; tt < t1; tt += TS) {
            const int n = static_cast<int>((t1 - tt) < TS ? (t1 - tt) : TS);
            __syncthreads();
            for (int idx = threadIdx.x; idx < n * d; idx += nthr) {
                const int t = idx / d, j = idx - t * d;
                const int64_t g = (tt + t) * row_stride + static_cast<int64_t>(h) * d + j;
                sk_[t * d + j] = to_f32(k[g]);
                sq_[t * d + j] = to_f32(q[g]);
            }
            for (int idx = threadIdx.x; idx < n * ROWS; idx += nthr) {
                const int t = idx / ROWS, r = idx - t * ROWS;
                const int row = rb0 + r;
                sv_[t * ROWS + r] =
                    row < d ? to_f32(v[(tt + t) * row_stride + static_cast<int64_t>(h) * d + row])
                            : 0.f;
            }
            for (int t = threadIdx.x; t < n; t += nthr) {
                sa_[t] = alpha[(tt + t) * H + h];
                sb_[t] = beta[(tt + t) * H + h];
            }
            __syncthreads();
            if (row0 < d) {
                for (int t = 0; t < n; ++t) {
                    float kk[NV][4], qq[NV][4], vr[RPW];
#pragma unroll
                    for (int c = 0; c < NV; ++c) {
                        const int j = 128 * c + 4 * lane;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const bool ok = j + e < d;
                            kk[c][e] = ok ? sk_[t * d + j + e] : 0.f;
                            qq[c][e] = ok ? sq_[t * d + j + e] : 0.f;
                        }
                    }
#pragma unroll
                    for (int r = 0; r < RPW; ++r) vr[r] = sv_[t * ROWS + warp * RPW + r];
                    float sk[RPW], ov[RPW], mine;
                    row_dots<RPW, NV>(s, kk, lane, sk, mine);
                    rank1_update<RPW, NV>(s, kk, sk, vr, sa_[t], sb_[t]);
                    row_dots<RPW, NV>(s, qq, lane, ov, mine);
                    if (writer) {
                        o[(tt + t) * row_stride + static_cast<int64_t>(h) * d + myrow] =
                            from_f32<T>(mine);
                    }
                }
            }
        }

        if (state_out && row0 < d) {
            const int64_t out_slot = out_slots ? static_cast<int64_t>(out_slots[seq]) : seq;
            if (out_slot >= 0 && out_slot < num_slots) {
                float *Sout = state_out + (out_slot * H + h) * static_cast<int64_t>(d) * d;
#pragma unroll
                for (int r = 0; r < RPW; ++r) {
                    const int row = row0 + r;
                    if (row < d) {
#pragma unroll
                        for (int c = 0; c < NV; ++c) {
                            const int j = 128 * c + 4 * lane;
                            store4(Sout + static_cast<int64_t>(row) * d + j, vec, nvalid(d, j),
                                   s[r][c]);
                        }
                    }
                }
            }
        }
    }
}

template <typename T, int RPW, int NV, int WARPS>
int launch_step_t(const StepArgs &a) {
    dim3 grid(static_cast<unsigned>(a.n * a.H), (a.d + WARPS * RPW - 1) / (WARPS * RPW));
    const bool vec = (a.d % 4) == 0;
    gdr_step_kernel<T, RPW, NV, WARPS><<<grid, WARPS * 32, 0, a.stream>>>(
        static_cast<T *>(a.o), a.pool, a.slots, static_cast<const T *>(a.q),
        static_cast<const T *>(a.k), static_cast<const T *>(a.v), a.alpha, a.beta, a.num_slots,
        a.H, a.d, vec);
    return check_launch("gdr_step_kernel");
}

template <typename T, int RPW, int NV, int WARPS, int TS>
int launch_seq_t(const SeqArgs &a) {
    constexpr int ROWS = WARPS * RPW;
    int sms = 148;
    bool sm100 = true;
    device_info(&sms, &sm100);
    const int64_t items = a.n_seq * a.H;
    const int row_blocks = (a.d + ROWS - 1) / ROWS;
    // Enough CTAs to fill every SM a few times over; the kernel loops over the
    // remaining (sequence, head) items.
    int64_t gx = static_cast<int64_t>(sms) * 16 / row_blocks;
    if (gx < 1) gx = 1;
    if (gx > items) gx = items;
    dim3 grid(static_cast<unsigned>(gx), row_blocks);
    const size_t smem = SeqTile<T, ROWS, TS>::bytes(a.d);
    auto kern = gdr_seq_kernel<T, RPW, NV, WARPS, TS>;
    if (smem > 48 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             static_cast<int>(smem));
        if (e != cudaSuccess) return set_error(RHZ_ERR_DEVICE, "gdr_seq_kernel smem: %s", cudaGetErrorString(e));
    }
    const bool vec = (a.d % 4) == 0;
    kern<<<grid, WARPS * 32, smem, a.stream>>>(
        static_cast<T *>(a.o), static_cast<const T *>(a.q), static_cast<const T *>(a.k),
        static_cast<const T *>(a.v), a.alpha, a.beta, a.cu_seqlens, a.n_seq_dev, a.n_seq, a.seq_len,
        a.cu_seqlens ? a.total_tokens : a.n_seq * a.seq_len,
        a.state_in, a.in_slots, a.state_out, a.out_slots, a.num_slots, a.H, a.d, vec);
    return check_launch("gdr_seq_kernel");
}

template <typename T, int RPW, int NV, int WARPS>
int launch_multistep_t(const MultistepArgs &a) {
    dim3 grid(static_cast<unsigned>(a.n * a.H), (a.d + WARPS * RPW - 1) / (WARPS * RPW));
    const bool vec = (a.d % 4) == 0;
    gdr_multistep_kernel<T, RPW, NV, WARPS><<<grid, WARPS * 32, 0, a.stream>>>(
        static_cast<T *>(a.outs), a.states, a.pool, a.slots, static_cast<const T *>(a.q),
        static_cast<const T *>(a.k), static_cast<const T *>(a.v), a.alpha, a.beta, a.segment,
        a.T, a.Tn, a.num_slots, a.H, a.d, vec);
    return check_launch("gdr_multistep_kernel");
}

template <typename T, int NR, int NJ, int WARPS>
int launch_tree_t(const TreeArgs &a) {
    dim3 grid(static_cast<unsigned>(a.n * a.H), (a.d + WARPS * 4 * NR - 1) / (WARPS * 4 * NR));
    const bool vec = (a.d % 4) == 0;
    auto *kernel = a.d == 32 * NJ ? gdr_tree_kernel<T, NR, NJ, WARPS, true> : gdr_tree_kernel<T, NR, NJ, WARPS, false>;
    const size_t smem = static_cast<size_t>(a.most) * (3 * a.d * sizeof(T) + 3 * 4) + 16;
    // The bound of every call of this kernel, so that no thread lowers it under another's launch.
    constexpr int BOUND = 64 * (3 * 32 * NJ * static_cast<int>(sizeof(T)) + 3 * 4) + 16;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, BOUND);
    if (e != cudaSuccess) return set_error(RHZ_ERR_DEVICE, "gdr_tree_kernel: %s", cudaGetErrorString(e));
    kernel<<<grid, WARPS * 32, smem, a.stream>>>(
        static_cast<T *>(a.o), a.states, a.pool, a.slots, a.cu_seqlens, a.parent,
        static_cast<const T *>(a.q), static_cast<const T *>(a.k), static_cast<const T *>(a.v),
        a.alpha, a.beta, a.total_tokens, a.most, a.num_slots, a.H, a.d, vec);
    return check_launch("gdr_tree_kernel");
}

template <typename T>
int launch_tree_d(const TreeArgs &a) {
    if (a.d <= 32) return launch_tree_t<T, 2, 1, 4>(a);
    if (a.d <= 64) return launch_tree_t<T, 2, 2, 8>(a);
    if (a.d <= 128) return launch_tree_t<T, 2, 4, 8>(a);
    return launch_tree_t<T, 1, 8, 8>(a);
}

}  // namespace

int launch_tree(const TreeArgs &a) {
    if (a.n == 0 || a.total_tokens == 0) return RHZ_OK;
    return a.dtype == RHZ_DTYPE_BF16 ? launch_tree_d<__nv_bfloat16>(a) : launch_tree_d<float>(a);
}

int launch_multistep(const MultistepArgs &a) {
    if (a.n == 0 || a.Tn == 0) return RHZ_OK;
    if (a.dtype == RHZ_DTYPE_BF16) {
        if (a.d <= 128) return launch_multistep_t<__nv_bfloat16, 8, 1, 8>(a);
        return launch_multistep_t<__nv_bfloat16, 4, 2, 8>(a);
    }
    if (a.d <= 128) return launch_multistep_t<float, 8, 1, 8>(a);
    return launch_multistep_t<float, 4, 2, 8>(a);
}

int launch_step(const StepArgs &a) {
    if (a.n == 0) return RHZ_OK;
    // d <= 128: one vector column per lane; 129..256: two. 64 rows per CTA
    // keep registers near 64/thread so three CTAs (96 KB of state loads in
    // flight) share an SM.
    if (a.dtype == RHZ_DTYPE_BF16) {
        if (a.d <= 128) return launch_step_t<__nv_bfloat16, 8, 1, 8>(a);
        return launch_step_t<__nv_bfloat16, 4, 2, 8>(a);
    }
    if (a.d <= 128) return launch_step_t<float, 8, 1, 8>(a);
    return launch_step_t<float, 4, 2, 8>(a);
}

int launch_seq(const SeqArgs &a) {
    if (a.n_seq == 0) return RHZ_OK;
    if (a.dtype == RHZ_DTYPE_BF16) {
        if (a.d <= 128) return launch_seq_t<__nv_bfloat16, 4, 1, 4, 32>(a);
        return launch_seq_t<__nv_bfloat16, 4, 2, 4, 16>(a);
    }
    if (a.d <= 128) return launch_seq_t<float, 4, 1, 4, 32>(a);
    return launch_seq_t<float, 4, 2, 4, 16>(a);
}

}  // namespace rhz
