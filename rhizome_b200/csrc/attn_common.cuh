// What the attention kernels share: which keys a row sees, how the key axis
// of a paged sequence is split, and where partial results go.
//
// Rows. A (sequence, K/V head) pair's query rows are ordered (token, head of
// the group): row r is token r / G, query head g * G + r % G, G = H / Hkv, so
// the rows of a tile share every K and V tile they read and a short sequence
// still fills tiles when the group is large.
#pragma once

#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "common.cuh"
#include "kernels.h"

namespace rhz {
namespace attn {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr int MAX_NODES = 64;  // drafted tokens of one sequence (one bit each)

// Splitting the key axis. A paged sequence of L keys is cut into equal chunks
// of span(L) keys, anchored at its first key, each computed by itself and joined
// afterwards in order of position. The rule looks at this sequence's length
// alone, so a sequence's result does not depend on what else is in the batch.
struct Split {
    int keys;  // per chunk, where that makes no more than
    int most;  // chunks of a sequence
    // (Lengths fit 31 bits: the entry refuses wider tables.)
    __host__ __device__ int span(int64_t L) const {
        const uint32_t l = static_cast<uint32_t>(L), w = (l + keys - 1) / keys;
        const uint32_t n = w < 1 ? 1 : w < static_cast<uint32_t>(most) ? w : most;
        return static_cast<int>((l + n * 128 - 1) / (n * 128) * 128);
    }
    __host__ __device__ int chunks(int64_t L) const {
        if (L <= keys) return 1;
        const uint32_t c = span(L);
        return static_cast<int>((static_cast<uint32_t>(L) + c - 1) / c);
    }
    // The most chunks that any length up to L can have.
    int64_t bound(int64_t L) const {
        const int64_t c = (L + keys - 1) / keys;
        return c < 1 ? 1 : (c < most ? c : most);
    }
};

// Partial results in the workspace: chunk counts [tokens], then log-sum-exp
// (base 2) [chunk][tokens][H], then normalised outputs [chunk][tokens][H][d].
struct Parts {
    int32_t *count;
    float *lse, *o;
    int64_t tokens;
    int H, d, most;  // most: chunks that the workspace has room for
    __device__ int64_t row(int64_t c, int64_t token, int head) const {
        return (c * tokens + token) * H + head;
    }
};

inline size_t up256(size_t x) { return (x + 255) / 256 * 256; }

inline size_t parts_bytes(int64_t tokens, int H, int d, int64_t chunks) {
    if (chunks <= 1 || tokens <= 0) return 0;
    const size_t rows = static_cast<size_t>(chunks) * tokens * H;
    return up256(tokens * sizeof(int32_t)) + up256(rows * sizeof(float)) + rows * d * sizeof(float);
}

inline Parts parts_at(void *ws, int64_t tokens, int H, int d, int64_t chunks) {
    Parts p{};
    p.tokens = tokens;
    p.H = H;
    p.d = d;
    p.most = static_cast<int>(chunks);
    if (chunks <= 1 || ws == nullptr) return p;
    char *b = static_cast<char *>(ws);
    const size_t rows = static_cast<size_t>(chunks) * tokens * H;
    p.count = reinterpret_cast<int32_t *>(b);
    p.lse = reinterpret_cast<float *>(b + up256(tokens * sizeof(int32_t)));
    p.o = reinterpret_cast<float *>(b + up256(tokens * sizeof(int32_t)) + up256(rows * sizeof(float)));
    return p;
}

// One sequence as the kernels see it: offsets clamped to the buffers, so that
// no cu_seqlens, length or table can lead outside them.
struct Seq {
    int first;   // first query row
    int m;       // query rows
    int live;    // of which take part (m, at most `most`)
    int cached;  // keys before the sequence's own rows (0 packed)
    int keys;    // cached + live
};

// (The entries refuse token counts and tables beyond 31 bits.)
__device__ __forceinline__ Seq seq_of(const AttnArgs &a, int64_t i) {
    const int total = static_cast<int>(a.total_tokens);
    Seq s;
    s.first = min(max(a.cu_seqlens[i], 0), total);
    s.m = min(max(a.cu_seqlens[i + 1], s.first), total) - s.first;
    s.cached = 0;
    s.live = s.m;
    if (a.paged) {
        const int room = static_cast<int>(a.width << a.shift);
        s.cached = min(max(a.cached[i], 0), room);
        // Rows whose own key has no table entry take no part either.
        s.live = min(min(s.m, static_cast<int>(a.most)), room - s.cached);
    }
    s.keys = s.cached + s.live;
    return s;
}

// Ancestors of drafted token t, itself included, as bits; 0 where t takes no
// part: its parent is not -1 or an earlier token, or some ancestor's is not.
__device__ __forceinline__ uint64_t ancestors(const int32_t *parent, int64_t t) {
    uint64_t bits = 0;
    int64_t p = t;
    while (p >= 0) {
        bits |= uint64_t{1} << p;
        const int64_t up = parent[p];
        if (up < -1 || up >= p) return 0;
        p = up;
    }
    return bits;
}

// The keys that one row sees: all below `all`, and of the 64 from `all` on
// those whose bit is set.
struct Sight {
    int64_t all;
    uint64_t bits;
    __device__ __forceinline__ bool sees(int64_t key) const {
        if (key < all) return true;
        const int64_t b = key - all;
        return b < 64 && (bits >> b & 1);
    }
};

__device__ __forceinline__ Sight sight_of(const AttnArgs &a, const Seq &s, int64_t t) {
    if (t >= s.live) return {0, 0};
    if (a.paged && a.parent) {
        const uint64_t bits = ancestors(a.parent + s.first, t);
        return {bits ? s.cached : 0, bits};
    }
    return {s.cached + t + 1, 0};
}

}  // namespace attn

// The tensor-core form (attn_tc.cu): bf16, d = 64 or 128.
bool attn_tc_supports(const AttnArgs &a);
int launch_attn_tc(const AttnArgs &a, const attn::Parts &parts, attn::Split split);
int attn_tc_status(int *flag, bool clear);
// The form for few rows per sequence over the paged cache (attn_rows.cu).
bool attn_rows_supports(const AttnArgs &a);
int launch_attn_rows(const AttnArgs &a, const attn::Parts &parts, attn::Split split);
int attn_rows_status(int *flag, bool clear);

}  // namespace rhz
