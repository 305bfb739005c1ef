// kv_layout.h -- where the quantised KV cache keeps its values.
//
// A kv head of a slot is a run of records of 32 positions, K and V apart:
//   [head_dim / 32 blocks][64 lanes]  integers, 16 bytes a lane (Q8_0) or 8 (Q4_0)
//   [head_dim / 32 blocks][32]        fp16 scales, one per position
//   V only: [32] fp16 e and [32] fp16 2^-e, where 2^e is past the position's
//   largest |scale| and half of it is not (e at least -14)
// so that one 16-byte load per lane is an operand of v_mfma_f32_16x16x32_f16
// once its bytes are halves, without LDS or lane exchanges: lane (g, c) = (lane
// >> 4, lane & 15) of a block holds
//   K  dims 8 g .. 8 g + 7 of positions c and 16 + c (A operands of K q^T, one
//      MFMA per 16 positions and block of 32 dims: a scale never changes inside
//      one product),
//   V  dims c and 16 + c of positions 4 g .. 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3,
//      which are the rows that lane (g, .) holds of two such score tiles: the
//      probabilities are the B operand of V^T p^T where they stand.
// Scales and exponents are ordered by those rows too: position p at 8 g + j.
// Q8_0 integers are stored as q + 128, Q4_0 as q + 8: a byte b becomes the half
// 1024 + b by setting its high byte to 0x64, and one packed add takes 1024 and
// the offset off again.
#pragma once

#include "common.h"

namespace llmdot {

constexpr int KV_GROUP = 32;   // positions per record

__host__ __device__ constexpr int kv_block_bytes(bool q4) { return q4 ? 512 : 1024; }
__host__ __device__ constexpr int kv_record_bytes(bool q4, int blocks, bool v) {
    return blocks * (kv_block_bytes(q4) + 64) + (v ? 128 : 0);
}

// Order of a position within its record's scales.
__host__ __device__ constexpr int kv_row(int p) { return (p & 12) * 2 + (p & 3) + (p >> 4) * 4; }

// Byte of element (position p of the record, dim r of its block); Q4_0: the
// nibble is kv_k_high / kv_v_high.
__host__ __device__ constexpr int kv_k_byte(bool q4, int p, int r) {
    const int lane = (r >> 3) * 16 + (p & 15), t = p >> 4;
    return q4 ? lane * 8 + t * 4 + (r & 3) : lane * 16 + t * 8 + (r & 7);
}
__host__ __device__ constexpr int kv_k_high(int r) { return (r >> 2) & 1; }
__host__ __device__ constexpr int kv_v_byte(bool q4, int p, int r) {
    const int lane = ((p >> 2) & 3) * 16 + (r & 15), j = (p & 3) + (p >> 4) * 4;
    return q4 ? lane * 8 + j : lane * 16 + (r >> 4) * 8 + j;
}
__host__ __device__ constexpr int kv_v_high(int r) { return r >> 4; }

// Division by a number that the host knows: n / d for 0 <= n < 2^31, with
// 2^(l-1) < d <= 2^l and m = floor(2^32 (2^l - d) / d) + 1 (Granlund and
// Montgomery's invariant division).
struct Divisor {
    uint32_t d, m, l;
    Divisor() = default;
    explicit Divisor(int v) : d((uint32_t)v), m(0), l(0) {
        while (l < 31 && ((uint32_t)1 << l) < d) l++;
        m = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << l) - d)) / d + 1);
    }
    __device__ __forceinline__ int div(int n) const {
        return (int)((__umulhi(m, (uint32_t)n) + (uint32_t)n) >> l);
    }
    __device__ __forceinline__ int mod(int n, int quotient) const { return n - quotient * (int)d; }
};

struct KvView {
    uint8_t *k, *v;             // [slots][kv_heads][groups] records
    int slots, kv_heads, head_dim, capacity, groups;
    int k_q4, v_q4;
    int k_rec, v_rec;           // bytes of a record
};
__host__ __device__ inline int64_t kv_group_index(const KvView& c, int slot, int head, int group) {
    return ((int64_t)slot * c.kv_heads + head) * c.groups + group;
}

struct KvRows {                 // llmdot_hip_token_batch
    int batch, tokens;
    const int32_t *slots, *starts, *counts;
};
// Sequence b's tokens as the kernels see them: rows lo .. hi - 1 of the call are
// positions start + lo .. start + hi - 1, all inside the slot (lo = hi: none).
struct KvSpan {
    int slot, start, lo, hi;
};
struct KvAsked { int slot, start, count; };   // a sequence as the arrays have it
__device__ __forceinline__ KvAsked kv_asked(const KvRows& r, int b) {
    const int32_t* counts = r.counts ? r.counts : r.starts;   // no branch around a load
    const int count = counts[b];
    return {r.slots[b], r.starts[b], r.counts ? count : r.tokens};
}
// Selects, not branches: with an early way out the compiler asks for the three
// numbers one after the other, each a trip to HBM.  Unsigned sums wrap where a
// start is far outside, and are not used then.
__device__ __forceinline__ KvSpan kv_span(const KvRows& r, const KvView& c, KvAsked a) {
    const int n = a.count < r.tokens ? a.count : r.tokens;
    const bool there = (a.slot >= 0) & (a.slot < c.slots) & (n > 0) & (a.start < c.capacity) & (a.start > -r.tokens);
    const int back = (int)(0u - (uint32_t)a.start), room = (int)((uint32_t)c.capacity - (uint32_t)a.start);
    const int lo = back > 0 ? back : 0, most = n < room ? n : room, hi = most > lo ? most : lo;
    return {there ? a.slot : 0, there ? a.start : 0, there ? lo : 0, there ? hi : 0};
}
__device__ __forceinline__ KvSpan kv_span(const KvRows& r, const KvView& c, int b) {
    return kv_span(r, c, kv_asked(r, b));
}

}  // namespace llmdot
