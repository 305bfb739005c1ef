// kv_cache.hip -- the quantised KV cache: rows quantised as they are written,
// and read back (layout: kv_layout.h).
//
// Bound by the bytes, by the launch where there are few: 2048 rows of 8 x 128 as
// Q8_0 are written in 10 us and read in 6 (38 MB together), 32768 read in 66 us
// (340 MB, 5.2 TB/s); 7 ragged sequences of up to 1500 positions of 8 x 64 as
// Q4_0 are read in 5.6 us (3.3 TB/s).
#include "kernels.h"
#include "kv_layout.h"

#include <type_traits>

namespace llmdot {

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4a __attribute__((ext_vector_type(4)));

constexpr float HALF_MAX = 65504.f;

__device__ __forceinline__ float max8(float v) {   // over each 8 consecutive lanes
    v = fmaxf(v, fx(lane_xor1, v));
    v = fmaxf(v, fx(lane_xor2, v));
    return fmaxf(v, fx(lane_mirror8, v));
}

// lroundf: to the nearest integer, halves away from zero (x - trunc(x) is exact).
__device__ __forceinline__ int round_away(float x) {
    const float t = truncf(x);
    return (int)t + (fabsf(x - t) >= 0.5f ? (x < 0.f ? -1 : 1) : 0);
}

// Four elements x of a block (8 lanes to a block, elements 4 l .. 4 l + 3 in
// lane l) as stored integers (q + 128, Q4_0: q + 8), a byte each, and the
// block's scale: the formulas of llmdot_hip_quantize, operation for operation.
// NaN elements have no magnitude there and are held as 0.
template <bool Q4>
__device__ __forceinline__ uint32_t quantize4(f4 x, int lane8, _Float16& scale) {
#pragma clang fp contract(off)
    float m = 0.f;
    int at = 0;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (fabsf(x[i]) > m) { m = fabsf(x[i]); at = i; }
    const float top = max8(m);
    float s;
    if constexpr (Q4) {
        // the signed value of the block's first largest magnitude becomes -8
        const bool mine = m == top && top > 0.f;
        float first = mine ? (float)(4 * lane8 + at) : 32.f;
        first = -max8(-first);
        const float v = x[at & 3];
        float signed_top = (mine && first == (float)(4 * lane8 + at)) ? v : 0.f;
        signed_top = sum8(signed_top);
        s = signed_top / -8.0f;
    } else {
        s = top / 127.0f;
    }
    s = fminf(fmaxf(s, -HALF_MAX), HALF_MAX);
    scale = (_Float16)s;
    const float d = (float)scale;
    // x / d is rounded to 32 bits before it becomes an integer.  The product with
    // 1 / d is within 2^-15 of that quotient (which is under 129), so only one that
    // near a half needs the division itself (10.4 -> 10.0 us for 2048 rows of 8 x 128).
    const float inv = d != 0.f ? 1.f / d : 0.f;
    f4 t = x * inv;
    bool near = false;
#pragma unroll
    for (int i = 0; i < 4; i++) near |= fabsf(fabsf(t[i]) - floorf(fabsf(t[i])) - 0.5f) < 0x1p-14f;
    if (__any(near)) {
#pragma unroll
        for (int i = 0; i < 4; i++) t[i] = d != 0.f ? x[i] / d : 0.f;
    }
    uint32_t out = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float r = t[i] == t[i] ? t[i] : 0.f;      // NaN
        r = fminf(fmaxf(r, -128.f), 128.f);       // infinities, before the conversion
        int q = round_away(r);
        if constexpr (Q4) q = (q < -8 ? -8 : q > 7 ? 7 : q) + 8;
        else q = (q < -127 ? -127 : q > 127 ? 127 : q) + 128;
        out |= (uint32_t)q << (8 * i);
    }
    return out;
}

constexpr int THREADS = 256, SETS = THREADS / 8;   // eight lanes to a block of 32 elements

// The part of a call that one workgroup moves: positions p0 .. p1 - 1 of one
// record of one kv head of one sequence.
struct Piece {
    KvSpan sp;
    int b, head, first, p0, p1;   // first: position of the record's first
    int64_t at;                   // index of the record
    __device__ __forceinline__ int64_t row(const KvRows& rows, int p) const {
        return (int64_t)b * rows.tokens + (first + p - sp.start);
    }
};
__device__ __forceinline__ Piece piece_of(const KvView& c, const KvRows& rows, const Divisor& by_groups,
                                          const Divisor& by_heads) {
    Piece x;
    // the kv heads of the same rows side by side: together they read or write whole rows
    const int rest = by_heads.div(blockIdx.x);
    x.head = by_heads.mod(blockIdx.x, rest);
    x.b = by_groups.div(rest);
    const int gi = by_groups.mod(rest, x.b);
    x.sp = kv_span(rows, c, x.b);
    const int group = (x.sp.start + x.sp.lo) / KV_GROUP + gi;
    x.first = group * KV_GROUP;
    x.p0 = x.sp.start + x.sp.lo - x.first;
    x.p1 = x.sp.start + x.sp.hi - x.first;
    x.p0 = x.p0 < 0 ? 0 : x.p0;
    x.p1 = x.p1 > KV_GROUP ? KV_GROUP : x.p1;
    x.at = kv_group_index(c, x.sp.slot, x.head, group);
    return x;
}

// Quantises a piece of k and v.  Records written whole are put together in LDS
// and leave in 16-byte stores (a V byte of a position lies 16 bytes from the
// next dim's); others store what is theirs, a byte belonging to one position.
// Bound by reading the fp32 rows.
template <int NB, bool KQ4, bool VQ4>
__global__ __launch_bounds__(THREADS) void kv_write_kernel(KvView c, KvRows rows, const float* k, int64_t ks,
                                                           const float* v, int64_t vs, Divisor by_groups,
                                                           Divisor by_heads) {
    constexpr int HD = NB * 32, KREC = kv_record_bytes(KQ4, NB, false), VREC = kv_record_bytes(VQ4, NB, true);
    const Piece x = piece_of(c, rows, by_groups, by_heads);
    if (x.sp.lo >= x.sp.hi || x.p0 >= x.p1) return;
    const int tid = threadIdx.x, lane8 = tid & 7, n = (x.p1 - x.p0) * NB;

    // positions that a later sequence of the call writes too are left to it
    __shared__ uint32_t taken;
    __shared__ __align__(16) uint8_t image[KREC + VREC];
    __shared__ float vscale[KV_GROUP][NB];
    uint32_t skip = 0;
    if (rows.batch > 1) {
        if (tid == 0) taken = 0;
        __syncthreads();
        for (int o = x.b + 1 + tid; o < rows.batch; o += THREADS) {
            const KvSpan so = kv_span(rows, c, o);
            if (so.slot != x.sp.slot) continue;
            int q0 = so.start + so.lo - x.first, q1 = so.start + so.hi - x.first;
            q0 = q0 < 0 ? 0 : q0;
            q1 = q1 > KV_GROUP ? KV_GROUP : q1;
            if (q0 < q1) atomicOr(&taken, (uint32_t)((((uint64_t)1 << (q1 - q0)) - 1) << q0));
        }
        __syncthreads();
        skip = taken;
    }
    const bool whole = x.p1 - x.p0 == KV_GROUP && skip == 0;
    uint8_t* kr = whole ? image : c.k + x.at * KREC;
    uint8_t* vr = whole ? image + KREC : c.v + x.at * VREC;

    constexpr int FLIGHT = NB < 4 ? NB : 4;   // blocks of a lane whose loads are out together
    // every lane of a group of eight takes part in its exchanges
    for (int i0 = tid / 8; i0 < n; i0 += SETS * FLIGHT) {
        f4 xk[FLIGHT], xv[FLIGHT];
#pragma unroll
        for (int z = 0; z < FLIGHT; z++) {
            const int i = i0 + z * SETS < n ? i0 + z * SETS : i0, p = x.p0 + i / NB;
            const int64_t row = x.row(rows, p);
            const int col = x.head * HD + i % NB * 32 + lane8 * 4;
            xk[z] = *reinterpret_cast<const f4*>(k + row * ks + col);
            xv[z] = *reinterpret_cast<const f4*>(v + row * vs + col);
        }
#pragma unroll
        for (int z = 0; z < FLIGHT; z++) {
            const int i = i0 + z * SETS;
            if (i >= n) break;
            const int p = x.p0 + i / NB, blk = i % NB, r = lane8 * 4;
            const bool keep = !(skip >> p & 1);
            _Float16 d;
            uint32_t w = quantize4<KQ4>(xk[z], lane8, d);
            if constexpr (KQ4) {
                // dims r .. r + 3 are the low nibbles, the next lane's the high ones
                const uint32_t other = lane_xor1(w);
                if (keep && !(lane8 & 1))
                    *reinterpret_cast<uint32_t*>(kr + blk * 512 + kv_k_byte(true, p, r)) = w | other << 4;
            } else if (keep) {
                *reinterpret_cast<uint32_t*>(kr + blk * 1024 + kv_k_byte(false, p, r)) = w;
            }
            if (keep && lane8 == 0)
                *reinterpret_cast<_Float16*>(kr + NB * kv_block_bytes(KQ4) + blk * 64 + kv_row(p) * 2) = d;
            w = quantize4<VQ4>(xv[z], lane8, d);
            if constexpr (VQ4) w |= (uint32_t)__shfl_down((int)w, 4, 8) << 4;   // dims r + 16 ..: the high nibbles
            if (keep && (!VQ4 || lane8 < 4)) {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    vr[blk * kv_block_bytes(VQ4) + kv_v_byte(VQ4, p, r + j)] = (uint8_t)(w >> (8 * j));
            }
            if (lane8 == 0) {
                if (keep) *reinterpret_cast<_Float16*>(vr + NB * kv_block_bytes(VQ4) + blk * 64 + kv_row(p) * 2) = d;
                vscale[p][blk] = fabsf((float)d);
            }
        }
    }
    __syncthreads();
    if (tid >= x.p0 && tid < x.p1 && !(skip >> tid & 1)) {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < NB; i++) m = fmaxf(m, vscale[tid][i]);
        int e = -14;
        if (m > 0x1p-15f) (void)frexpf(m, &e);
        _Float16* tail = reinterpret_cast<_Float16*>(vr + NB * (kv_block_bytes(VQ4) + 64)) + kv_row(tid);
        tail[0] = (_Float16)e;
        tail[32] = (_Float16)ldexpf(1.f, -e);
    }
    if (!whole) return;
    __syncthreads();
    for (int i = tid * 16; i < KREC; i += THREADS * 16)
        *reinterpret_cast<u32x4a*>(c.k + x.at * KREC + i) = *reinterpret_cast<const u32x4a*>(image + i);
    for (int i = tid * 16; i < VREC; i += THREADS * 16)
        *reinterpret_cast<u32x4a*>(c.v + x.at * VREC + i) = *reinterpret_cast<const u32x4a*>(image + KREC + i);
}

// The values of a piece.  The records pass through LDS, whole whatever part of
// them is asked for.  Bound by writing the fp32 rows.
template <int NB, bool KQ4, bool VQ4>
__global__ __launch_bounds__(THREADS) void kv_read_kernel(KvView c, KvRows rows, float* k, int64_t ks, float* v, int64_t vs,
                                                          Divisor by_groups, Divisor by_heads) {
    constexpr int HD = NB * 32, KREC = kv_record_bytes(KQ4, NB, false), VREC = kv_record_bytes(VQ4, NB, true);
    const Piece x = piece_of(c, rows, by_groups, by_heads);
    if (x.sp.lo >= x.sp.hi || x.p0 >= x.p1) return;
    __shared__ __align__(16) uint8_t image[KREC + VREC];
    const int tid = threadIdx.x, r = (tid & 7) * 4;
    constexpr int KN = (KREC + THREADS * 16 - 1) / (THREADS * 16), VN = (VREC + THREADS * 16 - 1) / (THREADS * 16);
    u32x4a in[KN + VN];
#pragma unroll
    for (int i = 0; i < KN; i++) {
        const int o = (i * THREADS + tid) * 16;
        in[i] = *reinterpret_cast<const u32x4a*>(c.k + x.at * KREC + (o < KREC ? o : 0));
    }
#pragma unroll
    for (int i = 0; i < VN; i++) {
        const int o = (i * THREADS + tid) * 16;
        in[KN + i] = *reinterpret_cast<const u32x4a*>(c.v + x.at * VREC + (o < VREC ? o : 0));
    }
#pragma unroll
    for (int i = 0; i < KN; i++) {
        const int o = (i * THREADS + tid) * 16;
        if (o < KREC) *reinterpret_cast<u32x4a*>(image + o) = in[i];
    }
#pragma unroll
    for (int i = 0; i < VN; i++) {
        const int o = (i * THREADS + tid) * 16;
        if (o < VREC) *reinterpret_cast<u32x4a*>(image + KREC + o) = in[KN + i];
    }
    __syncthreads();
    const uint8_t *kr = image, *vr = image + KREC;
    const int n = (x.p1 - x.p0) * NB;
    for (int i = tid / 8; i < n; i += SETS) {
        const int p = x.p0 + i / NB, blk = i % NB;
        const int64_t row = x.row(rows, p);
        const int col = x.head * HD + blk * 32 + r;
        const float dk = (float)*reinterpret_cast<const _Float16*>(kr + NB * kv_block_bytes(KQ4) + blk * 64 + kv_row(p) * 2);
        const float dv = (float)*reinterpret_cast<const _Float16*>(vr + NB * kv_block_bytes(VQ4) + blk * 64 + kv_row(p) * 2);
        uint32_t w = *reinterpret_cast<const uint32_t*>(kr + blk * kv_block_bytes(KQ4) + kv_k_byte(KQ4, p, r));
        if constexpr (KQ4) w = (kv_k_high(r) ? w >> 4 : w) & 0x0F0F0F0Fu;
        f4 xk, xv;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            xk[j] = dk * (float)((int)(w >> (8 * j) & 255) - (KQ4 ? 8 : 128));
            uint32_t u = vr[blk * kv_block_bytes(VQ4) + kv_v_byte(VQ4, p, r + j)];
            if constexpr (VQ4) u = (kv_v_high(r) ? u >> 4 : u) & 15;
            xv[j] = dv * (float)((int)u - (VQ4 ? 8 : 128));
        }
        *reinterpret_cast<f4*>(k + row * ks + col) = xk;
        *reinterpret_cast<f4*>(v + row * vs + col) = xv;
    }
}

// One wavefront per head row of a token (q heads, then k, then v).  Bound by the
// launch for a token, by reading and writing the rows for a prompt.
__global__ __launch_bounds__(64) void rope_rows_kernel(PfAttnArgs a, const int32_t* start, float* q_out, float* k_out,
                                                       float* v_out) {
    const int hd = a.head_dim, t = blockIdx.x, lane = threadIdx.x, half = a.rope_half;
    int h = blockIdx.y;
    const float *in = a.q, *norm = a.q_norm;
    float* out = q_out;
    int split = a.q_split, heads = a.heads;
    int64_t part = a.q_part;
    bool turns = true;
    if (h >= a.heads + a.kv_heads) {
        h -= a.heads + a.kv_heads;
        in = a.v; norm = nullptr; out = v_out; split = a.v_split; part = a.v_part; heads = a.kv_heads; turns = false;
    } else if (h >= a.heads) {
        h -= a.heads;
        in = a.k; norm = a.k_norm; out = k_out; split = a.k_split; part = a.k_part; heads = a.kv_heads;
    }
    const int64_t row = ((int64_t)t * heads + h) * hd;
    __shared__ float x[256];
    float ss = 0.f;
    for (int d = lane; d < hd; d += 64) {
        float v = in[row + d];
        for (int p = 1; p < split; p++) v += in[row + p * part + d];
        x[d] = v;
        ss += v * v;
    }
    if (norm) {
        const float inv = 1.f / sqrtf(wave_sum(ss) / (float)hd + a.eps);
        for (int d = lane; d < hd; d += 64) x[d] = norm[d] * x[d] * inv;
    }
    __syncthreads();
    const int64_t pos = *start + t;
    for (int d = lane; d < hd; d += 64) {
        const int64_t c = pos * half;
        out[row + d] = turns ? rope_elem(x, d, half, a.cos_tab + c, a.sin_tab + c) : x[d];
    }
}

// Records that a run of `tokens` positions can touch.
int run_groups(int tokens, const KvView& c) {
    const int64_t n = ((int64_t)tokens + KV_GROUP - 2) / KV_GROUP + 1;
    return n < c.groups ? (int)n : c.groups;
}

template <int NB, typename F>
void for_types(const KvView& c, F&& f) {
    using std::bool_constant;
    using std::integral_constant;
    const integral_constant<int, NB> nb;
    if (c.k_q4) c.v_q4 ? f(nb, bool_constant<true>(), bool_constant<true>()) : f(nb, bool_constant<true>(), bool_constant<false>());
    else c.v_q4 ? f(nb, bool_constant<false>(), bool_constant<true>()) : f(nb, bool_constant<false>(), bool_constant<false>());
}
template <typename F>
hipError_t for_shape(const KvView& c, F&& f) {
    switch (c.head_dim) {
        case 64: for_types<2>(c, f); break;
        case 96: for_types<3>(c, f); break;
        case 128: for_types<4>(c, f); break;
        case 256: for_types<8>(c, f); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_rope_rows(const PfAttnArgs& a, const int32_t* start, float* q_out, float* k_out, float* v_out,
                            hipStream_t s) {
    if (a.T <= 0 || a.head_dim > 256) return hipErrorInvalidValue;
    rope_rows_kernel<<<dim3(a.T, a.heads + 2 * a.kv_heads), 64, 0, s>>>(a, start, q_out, k_out, v_out);
    return hipGetLastError();
}

KvView kv_view(int slots, int kv_heads, int head_dim, int capacity, bool k_q4, bool v_q4) {
    KvView v{};
    v.slots = slots; v.kv_heads = kv_heads; v.head_dim = head_dim; v.capacity = capacity;
    v.groups = (capacity + KV_GROUP - 1) / KV_GROUP;
    v.k_q4 = k_q4; v.v_q4 = v_q4;
    v.k_rec = kv_record_bytes(k_q4, head_dim / 32, false);
    v.v_rec = kv_record_bytes(v_q4, head_dim / 32, true);
    return v;
}

hipError_t launch_kv_write(const KvView& c, const KvRows& rows, const float* k, int64_t ks, const float* v, int64_t vs,
                           hipStream_t s) {
    const int groups = run_groups(rows.tokens, c);
    const dim3 grid((uint32_t)groups * c.kv_heads * rows.batch);
    return for_shape(c, [&](auto nb, auto kq4, auto vq4) {
        kv_write_kernel<nb(), kq4(), vq4()><<<grid, THREADS, 0, s>>>(c, rows, k, ks, v, vs, Divisor(groups), Divisor(c.kv_heads));
    });
}

hipError_t launch_kv_read(const KvView& c, const KvRows& rows, float* k, int64_t ks, float* v, int64_t vs,
                          hipStream_t s) {
    const int groups = run_groups(rows.tokens, c);
    const dim3 grid((uint32_t)groups * c.kv_heads * rows.batch);
    return for_shape(c, [&](auto nb, auto kq4, auto vq4) {
        kv_read_kernel<nb(), kq4(), vq4()><<<grid, THREADS, 0, s>>>(c, rows, k, ks, v, vs, Divisor(groups), Divisor(c.kv_heads));
    });
}

}  // namespace llmdot
