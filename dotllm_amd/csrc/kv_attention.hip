// kv_attention.hip -- attention over the quantised KV cache (layout: kv_layout.h).
//
// out = sum_t softmax_t(scale q . k_t) v_t with k_t = dk qk, v_t = dv qv: integers
// times a scale per position and block of 32 dims.  One pass over the keys with
// the running maximum and sum, on v_mfma_f32_16x16x32_f16:
//   scores  S^T = K q^T: one MFMA covers exactly one block, so K's integers are
//     exact operands and its scale multiplies the MFMA's result (one FMA per
//     block and score).  q enters as two halves (22 bits), scaled by a power of
//     two per row.
//   values  O^T += V^T P'^T with P' = p dv, the probability with V's scale on it,
//     again two halves, per block; the score tile's lanes hold P' where the MFMA
//     wants it.  The running reference is the maximum of s + e, 2^e past the
//     position's largest |dv|: then p 2^e <= 2^14 and P' <= 2^14 whatever V's
//     range, so halves neither overflow nor lose small values.  p 2^e = ph + pl
//     and dv 2^-e are halves, and ph dvn = hi + r exactly (r an fma), so
//     P' = hi + (pl dvn + r) costs three packed instructions for two values.
// Scores, statistics and sums are fp32.
//
// Bound by the issue of vector instructions for prompts (the MFMAs, 2 x 2 of 16
// rows x 32 keys x 32 dims a block, run under them for the most part); by the
// chain lengths -> queries and records -> joined wavefronts -> joined chunks for
// single tokens.  Measured on an MI355X, whole calls:
//   8 kv heads x 4 x 128, Q8_0: one token at 4096 positions 9.0 us; a prompt of
//   2048 tokens 106 to 109 us (320 TFLOP/s of 4 hd per visible pair); 32 sequences of up
//   to 250 positions behind 6000 shared ones 22 us.
//   8 x 4 x 64, Q8_0 and Q4_0: 16 sequences of up to 8000 positions 16.7 us (2.9 TB/s).
//   32 x 1 x 96, Q8_0: 4 x 5 drafted tokens at up to 2400 positions, window 2047, 11.1 us.
#include "kernels.h"
#include "kv_layout.h"

#include <math.h>

#include <algorithm>
#include <type_traits>

namespace llmdot {

namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int THREADS = 256, WAVES = 4;
constexpr float P_EXP = 6.f, SLACK = 8.f;   // probabilities are held times 2^6, and at most 2^8 times that

// ---- operands ----
// Bytes b of w (unsigned, off more than the integer) as halves: 0x6400 + b is 1024 + b.
__device__ __forceinline__ h2 byte_halves(uint32_t w, uint32_t sel, _Float16 off) {
    const uint32_t x = __builtin_amdgcn_perm(0x64646464u, w, sel);
    return __builtin_bit_cast(h2, x) - h2{off, off};
}
__device__ __forceinline__ h8 join(h2 a, h2 b, h2 c, h2 d) {
    return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
constexpr uint32_t LOW_PAIR = 0x04010400u, HIGH_PAIR = 0x04030402u;

// A lane's 16 integers of a block: operands for (K) positions c and 16 + c, (V) dims c and 16 + c.
template <bool Q4>
struct Ints {
    typename std::conditional<Q4, u2, u4>::type w;
    __device__ __forceinline__ void load(const uint8_t* block, int lane) {
        w = *reinterpret_cast<const decltype(w)*>(block + lane * sizeof(w));
    }
    // K: each half of the lane's bytes is one operand (Q4_0: low nibbles are dims 0 .. 3, high 4 .. 7)
    __device__ __forceinline__ h8 k(int t) const {
        if constexpr (Q4) {
            const uint32_t lo = w[t] & 0x0F0F0F0Fu, hi = (w[t] >> 4) & 0x0F0F0F0Fu;
            const _Float16 off = (_Float16)1032.f;
            return join(byte_halves(lo, LOW_PAIR, off), byte_halves(lo, HIGH_PAIR, off), byte_halves(hi, LOW_PAIR, off),
                        byte_halves(hi, HIGH_PAIR, off));
        } else {
            const _Float16 off = (_Float16)1152.f;
            return join(byte_halves(w[2 * t], LOW_PAIR, off), byte_halves(w[2 * t], HIGH_PAIR, off),
                        byte_halves(w[2 * t + 1], LOW_PAIR, off), byte_halves(w[2 * t + 1], HIGH_PAIR, off));
        }
    }
    // V: Q4_0 keeps dims c in the low nibbles and 16 + c in the high ones
    __device__ __forceinline__ h8 v(int t) const {
        if constexpr (Q4) {
            const uint32_t a = (w[0] >> (4 * t)) & 0x0F0F0F0Fu, b = (w[1] >> (4 * t)) & 0x0F0F0F0Fu;
            const _Float16 off = (_Float16)1032.f;
            return join(byte_halves(a, LOW_PAIR, off), byte_halves(a, HIGH_PAIR, off), byte_halves(b, LOW_PAIR, off),
                        byte_halves(b, HIGH_PAIR, off));
        } else {
            return k(t);
        }
    }
};

// Eight fp32 values as two planes of halves.
__device__ __forceinline__ void split8(const float* x, h8& hi, h8& lo) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const h2 h = __builtin_convertvector(f2{x[i], x[i + 1]}, h2);
        const h2 l = __builtin_convertvector(f2{fmaf((float)h[0], -1.f, x[i]), fmaf((float)h[1], -1.f, x[i + 1])}, h2);
        hi[i] = h[0]; hi[i + 1] = h[1];
        lo[i] = l[0]; lo[i + 1] = l[1];
    }
}

// One record's K or V of a block set, in registers.
template <bool Q4, int NB>
struct Record {
    Ints<Q4> q[NB];
    h8 d[NB];          // scales of the lane's positions
    __device__ __forceinline__ void load(const uint8_t* rec, int lane) {
#pragma unroll
        for (int i = 0; i < NB; i++) {
            q[i].load(rec + i * kv_block_bytes(Q4), lane);
            d[i] = *reinterpret_cast<const h8*>(rec + NB * kv_block_bytes(Q4) + i * 64 + (lane >> 4) * 16);
        }
    }
};
template <bool Q4, int NB>
struct VRecord : Record<Q4, NB> {
    h8 e, w;           // exponents, and 2^-e
    __device__ __forceinline__ void load(const uint8_t* rec, int lane) {
        Record<Q4, NB>::load(rec, lane);
        const uint8_t* tail = rec + NB * (kv_block_bytes(Q4) + 64) + (lane >> 4) * 16;
        e = *reinterpret_cast<const h8*>(tail);
        w = *reinterpret_cast<const h8*>(tail + 64);
    }
};

// ---- the running softmax of 16 query rows (one per column of the score tiles) ----
template <int NB>
struct Tile {
    h8 qh[NB], ql[NB];
    float qinv;            // turns an MFMA sum into a score times log2(e)
    int last, before;      // visible positions: before < p <= last
    float m, l;            // reference and (the lane's part of the) sum
    f4 o[2 * NB];          // dims 16 t + 4 g .. + 3 of row `lane & 15`

    __device__ __forceinline__ void init(const f4 (&q)[2 * NB], float scale) {
        float x[NB][8], top = 0.f;
#pragma unroll
        for (int i = 0; i < NB; i++) {
#pragma unroll
            for (int j = 0; j < 4; j++) { x[i][j] = q[2 * i][j]; x[i][4 + j] = q[2 * i + 1][j]; }
#pragma unroll
            for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(x[i][j]));
        }
        top = fmaxf(top, fx(lane_xor16, top));
        top = fmaxf(top, fx(lane_xor32, top));
        int e = 0;
        if (top > 0.f && top < INFINITY) (void)frexpf(top, &e);
        e = 13 - e;   // the row's largest lies in [2^12, 2^13)
#pragma unroll
        for (int i = 0; i < NB; i++) {
#pragma unroll
            for (int j = 0; j < 8; j++) x[i][j] = ldexpf(x[i][j], e);
            split8(x[i], qh[i], ql[i]);
        }
        qinv = ldexpf(scale * 1.44269504088896341f, -e);
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int t = 0; t < 2 * NB; t++) o[t] = f4{0.f, 0.f, 0.f, 0.f};
    }

    __device__ __forceinline__ void mask(float (&s)[8], int first, int g) const {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int p = first + (j >> 2) * 16 + g * 4 + (j & 3);
            if (p > last || p <= before) s[j] = -INFINITY;
        }
    }
    // The probabilities' planes for each block, and the new reference and sum.
    __device__ __forceinline__ void probabilities(float (&s)[8], const h8& w, h8& ph, h8& pl) {
        float mx = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
        mx = fmaxf(mx, fx(lane_xor16, mx));
        mx = fmaxf(mx, fx(lane_xor32, mx));
        // the reference follows the maximum only where it falls too far behind:
        // sums are rescaled a few times in a walk, not at most records
        if (__any(mx > m + SLACK)) {
            const float mn = mx > m + SLACK ? mx : m;
            const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= f;
#pragma unroll
            for (int t = 0; t < 2 * NB; t++) o[t] *= f;
        }
        const float ref = m == -INFINITY ? 0.f : m - P_EXP;
        float p[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            p[j] = __builtin_amdgcn_exp2f(s[j] - ref);
            l = fmaf(p[j], (float)w[j], l);
        }
        split8(p, ph, pl);
    }
};

// Scores (times log2 e) plus exponents of a record's 32 positions for R tiles:
// s[x][4 t + r] is position 16 t + 4 g + r.  All of a half's products go out
// before the first result is needed: one MFMA's result takes several others' time.
template <int NB, int R>
__device__ __forceinline__ void scores(const Tile<NB> (&t)[R], const h8 (&kf)[2][NB], const h8 (&dk)[NB], const h8& e,
                                       float (&s)[R][8]) {
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int x = 0; x < R; x++) {
            f4 sum{0.f, 0.f, 0.f, 0.f};
            constexpr int TOGETHER = 2;
#pragma unroll
            for (int i0 = 0; i0 < NB; i0 += TOGETHER) {
                f4 c[TOGETHER];
#pragma unroll
                for (int i = 0; i < TOGETHER && i0 + i < NB; i++)
                    c[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[h][i0 + i], t[x].ql[i0 + i], f4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < TOGETHER && i0 + i < NB; i++)
                    c[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[h][i0 + i], t[x].qh[i0 + i], c[i], 0, 0, 0);
#pragma unroll
                for (int i = 0; i < TOGETHER && i0 + i < NB; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) sum[r] = fmaf(c[i][r], (float)dk[i0 + i][4 * h + r], sum[r]);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) s[x][4 * h + r] = fmaf(sum[r], t[x].qinv, (float)e[4 * h + r]);
        }
}

// Work of one launch.  An entry is a tile of query rows with the records it
// sees; its records are cut into chunks, one workgroup each.
struct Plan {
    int rows;              // query rows of a tile
    int tiles;             // per sequence (own) or of the call (prefix)
    int entries;           // own: batch * tiles; prefix: tiles
    int items;             // workgroups per kv head
    int least;             // records per chunk, at least, as a rule
    Divisor by_tiles, by_batch;
    float per_record;      // chunks per record, at most
    int whole;             // every entry is one chunk, in the workspace (2) or straight in `out` (1)
    float *o, *ml;         // workspace: [items][kv_heads][rows] of head_dim and of 2
    uint32_t* arrived;     // finished chunks of each (entry, kv head), zero between calls
};

// Records [x, y) that tile `tile` of sequence b sees of its own slot.
__device__ __forceinline__ int2 own_records(const KvAttnArgs& a, const Plan& pl, const KvSpan& sp, int tile) {
    int i0 = a.by_group.div(tile * pl.rows), i1 = a.by_group.div(tile * pl.rows + pl.rows - 1) + 1;
    i0 = i0 < sp.lo ? sp.lo : i0;
    i1 = i1 > sp.hi ? sp.hi : i1;
    if (i0 >= i1) return int2{0, 0};
    const int first = a.window > 0 && sp.start + i0 >= a.window ? sp.start + i0 - a.window + 1 : 0;
    return int2{first / KV_GROUP, (sp.start + i1 - 1) / KV_GROUP + 1};
}

// An entry's place among the items: its records [r0, r1) in `count` chunks from
// item `first` on.
struct Cut {
    int entry, first, count, r0, r1;
    KvSpan span;           // of its sequence
    // where chunk k begins (k = count: the end), the same in every workgroup
    __device__ __forceinline__ int begin(int k) const {
        return k >= count ? r1 : r0 + (int)((float)k * ((float)(r1 - r0) * __builtin_amdgcn_rcpf((float)count)));
    }
};
__device__ __forceinline__ uint32_t wave_sum_u32(uint32_t v) {
    v += lane_xor1(v);
    v += lane_xor2(v);
    v += lane_mirror8(v);
    v += lane_mirror16(v);
    v += lane_xor16(v);
    return v + lane_xor32(v);
}
// Inclusive sums over the lanes: within rows of 16, then rows 0 and 2 into 1 and
// 3, then the lower half into the upper.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_or_zero(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, true);
}
__device__ __forceinline__ int wave_scan_int(int v) {
    v += dpp_or_zero<0x111, 0xF>(v);   // row_shr 1, 2, 4, 8
    v += dpp_or_zero<0x112, 0xF>(v);
    v += dpp_or_zero<0x114, 0xF>(v);
    v += dpp_or_zero<0x118, 0xF>(v);
    v += dpp_or_zero<0x142, 0xA>(v);   // row_bcast 15
    return v + dpp_or_zero<0x143, 0xC>(v);   // row_bcast 31
}
// The cut that holds `item`, or (by_entry) the one of entry `item`; entry -1: an
// item that no entry needs.  Every wavefront works it out from the lengths in
// memory: one ratio of chunks to records for the whole batch, as high as the
// items allow, so that long sequences get many workgroups and short ones few.
// An entry of n records gets floor(n ratio) + 1 chunks: with ratio a little
// under (items - entries) / records, all of them fit into the items; where the
// lengths are such that they fit, it is (items - entries / 2) / records or
// (items - 3 entries / 4) / records, and the longest chunk is that much shorter.
__device__ __forceinline__ Cut find_cut(const KvAttnArgs& a, const Plan& pl, int item, bool by_entry) {
    auto ratio_at = [&](float give, float records) {
        return fminf(pl.per_record, ((float)pl.items - give * (float)pl.entries) * __builtin_amdgcn_rcpf(records));
    };
    auto chunks = [&](float ratio, int n) { return n > 0 ? (int)((float)n * ratio) + 1 : 0; };
    if (pl.entries == 1) {
        const KvSpan sp = kv_span(a.rows, a.cache, 0);
        const int2 r = own_records(a, pl, sp, 0);
        const int n = r.y - r.x;
        const int count = chunks(ratio_at(0.5f, (float)n), n);
        return Cut{by_entry || item < count ? 0 : -1, 0, count, r.x, r.y, sp};
    }
    const int lane = threadIdx.x & 63;
    KvSpan sp{0, 0, 0, 0};
    int2 r{0, 0};
    auto look = [&](int e) {
        if (e < pl.entries) {
            const int b = pl.by_tiles.div(e);
            sp = kv_span(a.rows, a.cache, b);
            r = own_records(a, pl, sp, pl.by_tiles.mod(e, b));
        } else {
            r = int2{0, 0};
        }
    };
    float total = 0.f;
    for (int e0 = 0; e0 < pl.entries; e0 += 64) {
        look(e0 + lane);
        total += (float)wave_sum_u32((uint32_t)(r.y - r.x));   // at most 64 * 2^25
    }
    float ratio = ratio_at(1.f, total) * (1.f - 0x1p-18f);
    if (pl.entries <= 64) {
#pragma unroll
        for (float give : {0.75f, 0.5f}) {
            const float more = ratio_at(give, total);
            if (wave_sum_u32((uint32_t)chunks(more, r.y - r.x)) <= (uint32_t)pl.items) ratio = more;
        }
    }
    int before = 0;
    for (int e0 = 0; e0 < pl.entries; e0 += 64) {
        const int e = e0 + lane;
        if (pl.entries > 64) look(e);
        const int n = chunks(ratio, r.y - r.x);
        const int upto = wave_scan_int(n);
        const bool mine = by_entry ? e == item : item >= before + upto - n && item < before + upto;
        const uint64_t who = __ballot(mine);
        if (who) {
            const int at = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)who) - 1);
            auto of = [&](int v) { return __builtin_amdgcn_readlane(v, at); };
            const int count = of(n);
            return Cut{e0 + at, before + of(upto) - count, count, of(r.x), of(r.y),
                       KvSpan{of(sp.slot), of(sp.start), of(sp.lo), of(sp.hi)}};
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return Cut{-1, 0, 0, 0, 0, KvSpan{0, 0, 0, 0}};
}

// Partial results cross XCDs inside a launch (the last workgroup of an entry
// joins it): written through, and read past, the XCD's own L2.
__device__ __forceinline__ void store_through(float* p, f2 v) {
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), __builtin_bit_cast(uint64_t, v), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f2 load_past(const float* p) {
    return __builtin_bit_cast(f2, __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED,
                                                    __HIP_MEMORY_SCOPE_AGENT));
}

// (reference, sum) pairs and what they weigh joined: running values times f, the new ones times w.
__device__ __forceinline__ void join_weights(float& m, float mk, float& f, float& w) {
    const float mn = fmaxf(m, mk);
    f = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
    w = mk == mn ? 1.f : __builtin_amdgcn_exp2f(mk - mn);   // -inf twice: nothing, or what is no number
    m = mn;
}

// Takes the 16 query rows from `first_row` on of a kv head (own rows: of sequence
// b; a prefix's: of all sequences, the lane's as `asked`) for a tile: asks for the
// lane's part of them, narrows the range of positions that all of them see, and returns where the
// lane's row goes in `out` (-1: none).
template <int NB, bool PRE>
__device__ __forceinline__ int64_t load_rows(const KvAttnArgs& a, Tile<NB>& t, f4 (&q)[2 * NB], int first_row, int b,
                                             int head, const KvSpan& sp, const KvAsked& asked, int& edge_last,
                                             int& edge_before) {
    const int lane = threadIdx.x & 63, tokens = a.rows.tokens, group = (int)a.by_group.d;
    const int row = first_row + (lane & 15);
    int i, bb = b, token;
    KvSpan s = sp;
    bool there;
    if constexpr (PRE) {
        token = a.by_group.div(row);
        bb = a.by_tokens.div(token);
        i = a.by_tokens.mod(token, bb);
        there = bb < a.rows.batch;
        s = kv_span(a.rows, a.cache, asked);
    } else {
        token = i = a.by_group.div(row);
        there = i < tokens;
    }
    there = there && i >= s.lo && i < s.hi;
    const int64_t at = (int64_t)bb * tokens + i;
    const int h = head * group + a.by_group.mod(row, token);
    // rows that are not there read the call's first (kv head `head` of it) and count as zeros
    const float* src = a.q + (there ? at * a.q_stride + h * (NB * 32) : (int64_t)head * group * (NB * 32)) + 8 * (lane >> 4);
#pragma unroll
    for (int i = 0; i < NB; i++) {
        q[2 * i] = *reinterpret_cast<const f4*>(src + 32 * i);
        q[2 * i + 1] = *reinterpret_cast<const f4*>(src + 32 * i + 4);
    }
    // positions in the cache at hand; an empty row sees all of the chunk
    const int pos = s.start + i;
    t.last = !there ? 0x7fffffff : PRE ? a.prefix_len - 1 : pos;
    t.before = !there || a.window <= 0 ? -1 : (PRE ? a.prefix_len : 0) + pos - a.window;
    int el = t.last, eb = t.before;
#pragma unroll
    for (int k = 1; k < 16; k *= 2) {
        const int ol = __shfl_xor(el, k), ob = __shfl_xor(eb, k);
        el = el < ol ? el : ol;
        eb = eb > ob ? eb : ob;
    }
    el = __builtin_amdgcn_readfirstlane(el);
    eb = __builtin_amdgcn_readfirstlane(eb);
    edge_last = el < edge_last ? el : edge_last;
    edge_before = eb > edge_before ? eb : edge_before;
    return there ? at * a.out_stride + h * (NB * 32) : -1;
}

// One workgroup: 16 R query rows of a kv head over a chunk of records, every
// fourth of them to a wavefront.  Bound by instruction issue (about 200 vector
// instructions a record and tile at head_dim 64, 300 at 128), by the loads'
// latency where a wavefront has a record or two.  FUSE: the workgroup that
// finishes an entry's last chunk joins them; its wavefronts' products go before
// their neighbours' other work (16 long sequences of the 1B shape: 16.7 us, 17.5 without: two wavefronts of a SIMD drift
// apart, and one's MFMAs run under the other's vector instructions).
template <int NB, bool KQ4, bool VQ4, int R, bool PRE, bool FUSE>
__device__ __forceinline__ void attend_chunk(const KvAttnArgs& a, const Plan& pl, int wg, float* lds) {
    constexpr int HD = NB * 32, ROWS = 16 * R;
    const int kvh = a.cache.kv_heads, item = a.by_kv_heads.div(wg), head = wg - item * kvh, group = (int)a.by_group.d;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x & 63, g = lane >> 4;

    // which rows and records
    int b = 0, tile, r0, r1, entry = 0, chunks = 1, first_item = 0, at_item = item;   // at_item: place in the workspace
    KvSpan sp{0, 0, 0, 0};
    if constexpr (PRE) {
        const int per = pl.items / pl.entries, total = (a.prefix_len + KV_GROUP - 1) / KV_GROUP;
        const int low = a.window > 0 && a.prefix_len >= a.window ? (a.prefix_len - a.window + 1) / KV_GROUP : 0;
        tile = item / per;
        const int n = total - low, k = item % per;
        r0 = low + (int)((int64_t)n * k / per);
        r1 = low + (int)((int64_t)n * (k + 1) / per);
    } else {
        if (pl.whole) {
            const int k = pl.by_batch.div(item);
            b = pl.by_batch.mod(item, k);
            tile = pl.tiles - 1 - k;   // the longest first
            at_item = b * pl.tiles + tile;
            sp = kv_span(a.rows, a.cache, b);
            const int2 r = own_records(a, pl, sp, tile);
            r0 = r.x;
            r1 = r.y;
        } else {
            const Cut c = find_cut(a, pl, item, false);
            if (c.entry < 0) return;
            entry = c.entry;
            chunks = c.count;
            first_item = c.first;
            b = pl.by_tiles.div(entry);
            tile = pl.by_tiles.mod(entry, b);
            r0 = c.begin(item - c.first);
            r1 = c.begin(item - c.first + 1);
            sp = c.span;
        }
        if (pl.whole && r0 >= r1) return;
    }
    const KvView& cache = PRE ? a.prefix : a.cache;
    const int slot = PRE ? a.prefix_slot : sp.slot;
    const int64_t base = kv_group_index(cache, slot, head, 0);
    const uint8_t* kb = cache.k + base * cache.k_rec;
    const uint8_t* vb = cache.v + base * cache.v_rec;
    constexpr int64_t KREC = kv_record_bytes(KQ4, NB, false), VREC = kv_record_bytes(VQ4, NB, true);
    Record<KQ4, NB> k;
    VRecord<VQ4, NB> v;
    int rec = r0 + wave;
    auto load_record = [&] {
        if (rec < r1) {
            k.load(kb + rec * KREC, lane);
            v.load(vb + rec * VREC, lane);
        }
    };
    // A prefix's rows are known only once their sequences' lengths are there: their
    // lengths, its record, then the queries.  Loads come back in order, so an own
    // chunk asks for its queries, which are needed first, before its record.
    KvAsked asked[R];
    if constexpr (PRE) {
#pragma unroll
        for (int x = 0; x < R; x++) {
            const int seq = a.by_tokens.div(a.by_group.div(tile * ROWS + x * 16 + (lane & 15)));
            asked[x] = kv_asked(a.rows, seq < a.rows.batch ? seq : 0);
        }
        load_record();
    }
    Tile<NB> t[R];
    int64_t out_at[R];     // element of `out` (-1: not a row)
    int edge_last = 0x7fffffff, edge_before = -1;   // records inside need no mask
    const int tokens = a.rows.tokens;
    {
        f4 q[R][2 * NB];
#pragma unroll
        for (int x = 0; x < R; x++)
            out_at[x] = load_rows<NB, PRE>(a, t[x], q[x], tile * ROWS + x * 16, b, head, sp, asked[x], edge_last, edge_before);
        if constexpr (!PRE) load_record();
#pragma unroll
        for (int x = 0; x < R; x++) {
            if (out_at[x] < 0) {
#pragma unroll
                for (int i = 0; i < 2 * NB; i++) q[x][i] = f4{0.f, 0.f, 0.f, 0.f};
            }
            t[x].init(q[x], a.scale);
        }
    }
    if (PRE && edge_last > a.prefix_len - 1) edge_last = a.prefix_len - 1;
    if (PRE && a.window > 0) {
        // rows whose windows begin behind the chunk (a prompt's, all but the first few): nothing to join
        int before = 0x7fffffff;
#pragma unroll
        for (int x = 0; x < R; x++)
            if (out_at[x] >= 0 && t[x].before < before) before = t[x].before;
#pragma unroll
        for (int k = 1; k < 16; k *= 2) {
            const int o = __shfl_xor(before, k);
            before = o < before ? o : before;
        }
        const int end = r1 * KV_GROUP < a.prefix_len ? r1 * KV_GROUP : a.prefix_len;
        if (__builtin_amdgcn_readfirstlane(before) >= end - 1) {
            if (wave == 0 && g == 0) {
#pragma unroll
                for (int x = 0; x < R; x++) {
                    const int64_t part = ((int64_t)at_item * kvh + head) * ROWS + x * 16 + (lane & 15);
                    *reinterpret_cast<f2*>(pl.ml + part * 2) = f2{-INFINITY, 0.f};
                }
            }
            return;
        }
    }

    for (; rec < r1; rec += WAVES) {
        const int next = rec + WAVES < r1 ? rec + WAVES : rec;
        float s[R][8];
        {
            h8 kf[2][NB];
#pragma unroll
            for (int i = 0; i < NB; i++) { kf[0][i] = k.q[i].k(0); kf[1][i] = k.q[i].k(1); }
            if constexpr (FUSE) __builtin_amdgcn_s_setprio(1);
            scores<NB, R>(t, kf, k.d, v.e, s);
            if constexpr (FUSE) __builtin_amdgcn_s_setprio(0);
        }
        k.load(kb + next * KREC, lane);
        if (rec * KV_GROUP + KV_GROUP - 1 > edge_last || rec * KV_GROUP <= edge_before) {
#pragma unroll
            for (int x = 0; x < R; x++) t[x].mask(s[x], rec * KV_GROUP, g);
        }
        h8 ph[R], pl8[R];
#pragma unroll
        for (int x = 0; x < R; x++) t[x].probabilities(s[x], v.w, ph[x], pl8[x]);
        if constexpr (FUSE) __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < NB; i++) {
            const h8 d = v.d[i] * v.w;
            const h8 v0 = v.q[i].v(0), v1 = v.q[i].v(1);
#pragma unroll
            for (int x = 0; x < R; x++) {
                const h8 hi = ph[x] * d;
                const h8 lo = __builtin_elementwise_fma(pl8[x], d, __builtin_elementwise_fma(ph[x], d, -hi));
                t[x].o[2 * i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, hi, t[x].o[2 * i], 0, 0, 0);
                t[x].o[2 * i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, hi, t[x].o[2 * i + 1], 0, 0, 0);
                t[x].o[2 * i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, lo, t[x].o[2 * i], 0, 0, 0);
                t[x].o[2 * i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, lo, t[x].o[2 * i + 1], 0, 0, 0);
            }
        }
        if constexpr (FUSE) __builtin_amdgcn_s_setprio(0);
        v.load(vb + next * VREC, lane);
    }
#pragma unroll
    for (int x = 0; x < R; x++) {
        t[x].l += fx(lane_xor16, t[x].l);
        t[x].l += fx(lane_xor32, t[x].l);
    }

    const bool direct = pl.whole == 1 || (FUSE && chunks == 1);
    {
        // the wavefronts' records meet in LDS, each wavefront summing a share of the dims in order
        auto so = reinterpret_cast<float (*)[16 * R][HD + 4]>(lds);
        auto sm = reinterpret_cast<float (*)[16 * R][2]>(lds + WAVES * 16 * R * (HD + 4));
#pragma unroll
        for (int x = 0; x < R; x++) {
            const int row = x * 16 + (lane & 15);
            if (g == 0) { sm[wave][row][0] = t[x].m; sm[wave][row][1] = t[x].l; }
#pragma unroll
            for (int d = 0; d < 2 * NB; d++) *reinterpret_cast<f4*>(&so[wave][row][16 * d + 4 * g]) = t[x].o[d];
        }
        __syncthreads();
#pragma unroll
        for (int x = 0; x < R; x++) {
            const int row = x * 16 + (lane & 15);
            float mx = -INFINITY, sum = 0.f, f[WAVES];
#pragma unroll
            for (int w = 0; w < WAVES; w++) mx = fmaxf(mx, sm[w][row][0]);
#pragma unroll
            for (int w = 0; w < WAVES; w++) {
                const float mw = sm[w][row][0];
                f[w] = mw == mx ? 1.f : __builtin_amdgcn_exp2f(mw - mx);
                sum = fmaf(f[w], sm[w][row][1], sum);
            }
            const int64_t part = ((int64_t)at_item * kvh + head) * ROWS + row;
            const float inv = 1.f / sum;
            if (out_at[x] < 0) continue;
            for (int d = wave; d < 2 * NB; d += WAVES) {
                f4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < WAVES; w++) acc += f[w] * *reinterpret_cast<const f4*>(&so[w][row][16 * d + 4 * g]);
                float* o = pl.o + part * HD + 16 * d + 4 * g;
                if (direct) {
                    *reinterpret_cast<f4*>(a.out + out_at[x] + 16 * d + 4 * g) = acc * inv;
                } else if constexpr (FUSE) {
                    store_through(o, f2{acc[0], acc[1]});
                    store_through(o + 2, f2{acc[2], acc[3]});
                } else {
                    *reinterpret_cast<f4*>(o) = acc;
                }
            }
            if (!direct && wave == 0 && g == 0) {
                if constexpr (FUSE) store_through(pl.ml + part * 2, f2{mx, sum});
                else *reinterpret_cast<f2*>(pl.ml + part * 2) = f2{mx, sum};
            }
        }
    }

    if constexpr (FUSE) {
        if (direct) return;
        // every store of this workgroup is past the L2 before it counts itself in
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        int& is_last = *reinterpret_cast<int*>(lds + WAVES * 16 * R * (HD + 6));
        __syncthreads();
        if (threadIdx.x == 0) {
            uint32_t* count = pl.arrived + (entry * kvh + head) * COUNTER_STRIDE;
            const uint32_t was = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            is_last = was + 1 == (uint32_t)chunks;
            if (is_last) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!is_last) return;
        // rows x (HD / 4) lanes, the chunks of a row in as many sets as the threads allow
        constexpr int LANES = HD / 4, SETS = THREADS / LANES;
        const int set = threadIdx.x / LANES, d = threadIdx.x % LANES * 4;
        const int i0 = a.by_group.div(tile * ROWS), i1 = a.by_group.div(tile * ROWS + ROWS - 1) + 1;
        const int lo = (sp.lo > i0 ? sp.lo : i0) * group, hi = (sp.hi < i1 ? sp.hi : i1) * group;   // its rows
        const int begin = lo > tile * ROWS ? lo - tile * ROWS : 0, end = hi - tile * ROWS < ROWS ? hi - tile * ROWS : ROWS;
        const int rows = end - begin;
        int share = 1;                                     // sets that split a row's chunks
        while (share * 2 * rows <= SETS) share *= 2;
        auto jo = reinterpret_cast<float (*)[HD]>(lds);
        auto jm = reinterpret_cast<float (*)[2]>(lds + SETS * HD);
        const int at_once = SETS / share, my = set / share, part_of = set % share;
        for (int q0 = 0; q0 < rows; q0 += at_once) {
            const int q = q0 + my;
            const bool on = my < at_once && q < rows;
            float m = -INFINITY, l = 0.f;
            f4 acc{0.f, 0.f, 0.f, 0.f};
            if (on) {
                constexpr int FLIGHT = 8;                  // chunks whose loads are out together
                for (int c0 = part_of; c0 < chunks; c0 += FLIGHT * share) {
                    f2 ml[FLIGHT], oa[FLIGHT], ob[FLIGHT];
#pragma unroll
                    for (int z = 0; z < FLIGHT; z++) {
                        const int c = c0 + z * share < chunks ? c0 + z * share : c0;
                        const int64_t part = ((int64_t)(first_item + c) * kvh + head) * ROWS + begin + q;
                        ml[z] = load_past(pl.ml + part * 2);
                        oa[z] = load_past(pl.o + part * HD + d);
                        ob[z] = load_past(pl.o + part * HD + d + 2);
                    }
#pragma unroll
                    for (int z = 0; z < FLIGHT; z++) {
                        if (c0 + z * share >= chunks) break;
                        float f, w;
                        join_weights(m, ml[z][0], f, w);
                        l = fmaf(l, f, w * ml[z][1]);
                        acc = acc * f + f4{oa[z][0], oa[z][1], ob[z][0], ob[z][1]} * w;
                    }
                }
                *reinterpret_cast<f4*>(&jo[set][d]) = acc;
                if (d == 0) { jm[set][0] = m; jm[set][1] = l; }
            }
            __syncthreads();
            if (on && part_of == 0) {
                for (int c = 1; c < share && c < chunks; c++) {
                    float f, w;
                    join_weights(m, jm[set + c][0], f, w);
                    l = fmaf(l, f, w * jm[set + c][1]);
                    acc = acc * f + *reinterpret_cast<const f4*>(&jo[set + c][d]) * w;
                }
                const int row = tile * ROWS + begin + q, i = a.by_group.div(row);
                const int64_t at = ((int64_t)b * tokens + i) * a.out_stride + (head * group + a.by_group.mod(row, i)) * HD;
                *reinterpret_cast<f4*>(a.out + at + d) = acc * (1.f / l);
            }
            __syncthreads();
        }
    }
}

// The call's own chunks, and (RP) the prefix's before them, 16 RP rows to a wavefront.
template <int NB, bool KQ4, bool VQ4, int R, int RP>
__global__ __launch_bounds__(THREADS, NB == 8 ? 1 : 2) void kv_attention_kernel(KvAttnArgs a, Plan own, Plan pre) {
    constexpr int MOST = RP > R ? RP : R;
    __shared__ __align__(16) float lds[WAVES * 16 * MOST * (NB * 32 + 6) + 4];
    if constexpr (RP > 0) {
        const int before = pre.items * a.cache.kv_heads;
        if ((int)blockIdx.x < before) attend_chunk<NB, KQ4, VQ4, RP, true, false>(a, pre, blockIdx.x, lds);
        else attend_chunk<NB, KQ4, VQ4, R, false, false>(a, own, blockIdx.x - before, lds);
    } else {
        attend_chunk<NB, KQ4, VQ4, R, false, R == 1>(a, own, blockIdx.x, lds);
    }
}

// The chunks of a row (the prefix's, then its own) joined: one workgroup per row,
// hd / 4 lanes to a chunk and as many chunks at a time as fit; the order of the
// sums depends on their number alone.  Bound by its chain of loads (lengths, plan,
// parts): 4.4 us for 1024 rows of 8 + 2 chunks.
__global__ __launch_bounds__(THREADS) void kv_attention_join(KvAttnArgs a, Plan own, Plan pre) {
    const int kvh = a.cache.kv_heads, group = (int)a.by_group.d, hd = a.cache.head_dim;
    // rows of a token: kv head by kv head
    const int x = a.by_group.div(blockIdx.x), hr = a.by_group.mod(blockIdx.x, x), token = a.by_kv_heads.div(x),
              head = a.by_kv_heads.mod(x, token), h = head * group + hr;
    const int b = a.by_tokens.div(token), i = a.by_tokens.mod(token, b);
    const KvAsked asked = kv_asked(a.rows, b);

    const int lanes = hd / 4, sets = THREADS / lanes;
    const int set = threadIdx.x / lanes, d = threadIdx.x % lanes * 4;
    float m = -INFINITY, l = 0.f;
    f4 acc{0.f, 0.f, 0.f, 0.f};
    auto take = [&](f2 ml, f4 o) {
        if (ml[0] == -INFINITY) return;   // saw nothing: its sums may not have been written
        float f, w;
        join_weights(m, ml[0], f, w);
        l = fmaf(l, f, w * ml[1]);
        acc = acc * f + o * w;
    };
    // a set's chunks: of the prefix (whose place needs no lengths: the first is on
    // its way while they come), then the row's own
    const int prow = token * group + hr;
    const int pchunks = pre.items ? pre.items / pre.entries : 0, ptile = pre.items ? prow / pre.rows : 0;
    auto pre_part = [&](int k) { return ((int64_t)(ptile * pchunks + k) * kvh + head) * pre.rows + prow % pre.rows; };
    f2 ml0{-INFINITY, 0.f};
    f4 o0{0.f, 0.f, 0.f, 0.f};
    if (set < sets && set < pchunks) {
        ml0 = *reinterpret_cast<const f2*>(pre.ml + pre_part(set) * 2);
        o0 = *reinterpret_cast<const f4*>(pre.o + pre_part(set) * hd + d);
    }
    const KvSpan sp = kv_span(a.rows, a.cache, asked);
    if (i < sp.lo || i >= sp.hi) return;
    const int row = i * group + hr, tile = row / own.rows, trow = row % own.rows;
    Cut c{0, 0, 1, 0, 0, sp};
    if (!own.whole) {
        c = find_cut(a, own, b * own.tiles + tile, true);
    } else {
        c.first = b * own.tiles + tile;
    }
    const int n = pchunks + c.count;
    if (set < sets) {
        if (set < pchunks) take(ml0, o0);
#pragma unroll 4
        for (int k = set < pchunks ? set + sets : set; k < n; k += sets) {
            const bool of_pre = k < pchunks;
            const int64_t part = of_pre ? pre_part(k) : ((int64_t)(c.first + k - pchunks) * kvh + head) * own.rows + trow;
            take(*reinterpret_cast<const f2*>((of_pre ? pre.ml : own.ml) + part * 2),
                 *reinterpret_cast<const f4*>((of_pre ? pre.o : own.o) + part * hd + d));
        }
    }
    __shared__ float so[THREADS * 4], sml[THREADS / 16][2];
    if (set < sets) {
        *reinterpret_cast<f4*>(so + set * hd + d) = acc;
        if (d == 0) { sml[set][0] = m; sml[set][1] = l; }
    }
    __syncthreads();
    if (set != 0) return;
    const int used = n < sets ? n : sets;
    for (int k = 1; k < used; k++) {
        float f, w;
        join_weights(m, sml[k][0], f, w);
        l = fmaf(l, f, w * sml[k][1]);
        acc = acc * f + *reinterpret_cast<const f4*>(so + k * hd + d) * w;
    }
    const int64_t at = (int64_t)token * a.out_stride + h * hd + d;
    *reinterpret_cast<f4*>(a.out + at) = acc * (1.f / l);
}

// ---- host ----
constexpr int PRE_R = 2;
constexpr int TARGET = 512;        // workgroups: two per CU (16 long sequences of the 1B shape: 16.7 us, 23.5 with 256)
constexpr int PRE_TARGET = 256;    // of a prefix: its chunks' results cost more than an idle wavefront (22.1 us against 25.2 at 512)
static_assert(TARGET <= MAX_SEQUENCES);   // entries * kv_heads <= TARGET where chunks are counted

struct Plans {
    Plan own{}, pre{};
    int r;                 // tiles of a wavefront
    bool fused;            // chunks joined by the workgroup that finishes last
    size_t bytes = 0;
};

int rows_per_wave(int blocks) { return blocks == 8 ? 1 : 2; }   // tiles of 16: registers for two wavefronts per SIMD

// Shapes of the launch, from sizes that the host knows (lengths are on the
// device).  16 rows or fewer of a kv head and sequence (decode): tiles of 16
// rows, more: of 32 (16 at head_dim 256, whose tiles leave no registers for
// two wavefronts per SIMD): a record's integers become halves once for two tiles
// (a 7B prompt of 2048 tokens: 107 us, 132 in tiles of 16).  A tile's keys go over the wavefronts of its
// workgroup and, where tiles are too few for the card, in chunks over several.
Plans make_plans(const KvView& c, int heads, int batch, int tokens, bool prefix, int prefix_len, uint8_t* work) {
    Plans p;
    const int group = heads / c.kv_heads, r = rows_per_wave(c.head_dim / 32);
    // beside a prefix the call's own chunks get the other half of the workgroups (431 tokens of 2 heads at
    // position 3234 behind 11433: 30 us, 36 with all of them, whose last then wait for a place)
    const int64_t rows = (int64_t)tokens * group, want = (prefix ? TARGET - PRE_TARGET : TARGET) / c.kv_heads;
    auto tiles_of = [](int64_t n, int per) { return (int)((n + per - 1) / per); };
    p.r = rows <= 16 ? 1 : r;
    Plan& o = p.own;
    o.rows = 16 * p.r;
    o.tiles = tiles_of(rows, o.rows);
    o.entries = batch * o.tiles;
    // two records a wavefront pay for a chunk's own time (4096 keys of the 7B shape: 9.0 us, at one 9.2, at four 10.9)
    o.least = 2 * WAVES;
    o.per_record = 1.f / (float)o.least * (1.f - 0x1p-18f);
    o.by_tiles = Divisor(o.tiles);
    o.by_batch = Divisor(batch);
    const int64_t most = tiles_of(c.groups, o.least);   // chunks of an entry
    o.items = o.entries;
    if (o.entries < want && most > 1)
        o.items = (int)std::max<int64_t>(std::min(want, o.entries * (most + 1)), o.entries * 3 / 2 + 1);
    o.whole = o.items == o.entries ? prefix ? 2 : 1 : 0;
    p.fused = !prefix && p.r == 1 && !o.whole;
    size_t at = 0;
    auto take = [&](size_t n) {
        uint8_t* q = work + at;
        at += (n + 15) & ~(size_t)15;
        return q;
    };
    auto take_parts = [&](Plan& x) {
        const size_t n = (size_t)x.items * c.kv_heads * x.rows;
        x.o = reinterpret_cast<float*>(take(n * c.head_dim * 4));
        x.ml = reinterpret_cast<float*>(take(n * 8));
    };
    o.arrived = reinterpret_cast<uint32_t*>(take(COUNTER_BYTES));
    if (prefix) {
        Plan& x = p.pre;
        x.rows = 16 * std::min(PRE_R, r);
        x.tiles = x.entries = tiles_of(batch * rows, x.rows);
        x.least = 4;
        const int64_t most_pre = PRE_TARGET / c.kv_heads;
        int64_t chunks = x.entries < most_pre ? most_pre / x.entries : 1;
        if (prefix_len >= 0) chunks = std::max<int64_t>(1, std::min<int64_t>(chunks, tiles_of(prefix_len, KV_GROUP) / x.least));
        x.items = (int)(x.entries * chunks);
        take_parts(x);
    }
    if (o.whole != 1) take_parts(o);
    p.bytes = at;
    return p;
}

template <int NB, bool KQ4, bool VQ4, int RP>
void launch_own(const Plans& p, const KvAttnArgs& a, hipStream_t s) {
    const dim3 grid((uint32_t)((p.own.items + p.pre.items) * a.cache.kv_heads));
    if (p.r == 1) kv_attention_kernel<NB, KQ4, VQ4, 1, RP><<<grid, THREADS, 0, s>>>(a, p.own, p.pre);
    else kv_attention_kernel<NB, KQ4, VQ4, NB == 8 ? 1 : 2, RP><<<grid, THREADS, 0, s>>>(a, p.own, p.pre);
}

template <int NB, bool KQ4, bool VQ4>
hipError_t launch_types(KvAttnArgs a, hipStream_t s) {
    a.by_group = Divisor(a.heads / a.cache.kv_heads);
    a.by_tokens = Divisor(a.rows.tokens);
    a.by_kv_heads = Divisor(a.cache.kv_heads);
    const Plans p = make_plans(a.cache, a.heads, a.rows.batch, a.rows.tokens, a.prefix_len > 0, a.prefix_len, a.work);
    if (p.pre.items) launch_own<NB, KQ4, VQ4, NB == 8 ? 1 : PRE_R>(p, a, s);
    else launch_own<NB, KQ4, VQ4, 0>(p, a, s);
    if (p.own.whole != 1 && !p.fused) {
        const int64_t rows = (int64_t)a.rows.batch * a.rows.tokens * a.heads;
        kv_attention_join<<<dim3((uint32_t)rows), THREADS, 0, s>>>(a, p.own, p.pre);
    }
    return hipGetLastError();
}

template <int NB>
hipError_t launch_blocks(const KvAttnArgs& a, hipStream_t s) {
    if (a.cache.k_q4) return a.cache.v_q4 ? launch_types<NB, true, true>(a, s) : launch_types<NB, true, false>(a, s);
    return a.cache.v_q4 ? launch_types<NB, false, true>(a, s) : launch_types<NB, false, false>(a, s);
}

}  // namespace

bool kv_attention_supported(int head_dim) {
    return head_dim == 64 || head_dim == 96 || head_dim == 128 || head_dim == 256;
}

size_t kv_attention_workspace(const KvView& c, int heads, int batch, int tokens, bool prefix) {
    const size_t without = make_plans(c, heads, batch, tokens, false, 0, nullptr).bytes;
    return prefix ? std::max(without, make_plans(c, heads, batch, tokens, true, -1, nullptr).bytes) : without;
}

size_t kv_attention_workspace_upto(const KvView& c, int heads, int tokens) {
    size_t most = 0;
    for (int t = 1; t <= tokens; t++) most = std::max(most, kv_attention_workspace(c, heads, 1, t, false));
    return most;
}

hipError_t launch_kv_attention(const KvAttnArgs& a, hipStream_t s) {
    switch (a.cache.head_dim) {
        case 64: return launch_blocks<2>(a, s);
        case 96: return launch_blocks<3>(a, s);
        case 128: return launch_blocks<4>(a, s);
        case 256: return launch_blocks<8>(a, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace llmdot
