// kv_cache.hip -- the quantised KV cache: rows quantised as they are written,
// and read back (layout: kv_layout.h).
#include "kernels.h"
#include "kv_layout.h"

namespace llmdot {

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));

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
    uint32_t out = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float r = d != 0.f ? x[i] / d : 0.f;
        r = r == r ? r : 0.f;                     // NaN
        r = fminf(fmaxf(r, -128.f), 128.f);       // infinities, before the conversion
        int q = round_away(r);
        if constexpr (Q4) q = (q < -8 ? -8 : q > 7 ? 7 : q) + 8;
        else q = (q < -127 ? -127 : q > 127 ? 127 : q) + 128;
        out |= (uint32_t)q << (8 * i);
    }
    return out;
}

constexpr int WRITE_THREADS = 256;

// One workgroup: the new positions of one record (32 positions of one kv head of
// one sequence), K and V.  Eight lanes take a block of 32 elements.
template <bool KQ4, bool VQ4>
__global__ __launch_bounds__(WRITE_THREADS) void kv_write_kernel(KvView c, KvRows rows, const float* k, int64_t ks,
                                                                 const float* v, int64_t vs, int groups) {
    const int gi = blockIdx.x % groups, rest = blockIdx.x / groups;
    const int head = rest % c.kv_heads, b = rest / c.kv_heads;
    const KvSpan sp = kv_span(rows, c, b);
    if (sp.lo >= sp.hi) return;
    const int group = (sp.start + sp.lo) / KV_GROUP + gi;
    const int first = group * KV_GROUP;
    int p0 = sp.start + sp.lo - first, p1 = sp.start + sp.hi - first;   // the record's positions p0 .. p1 - 1
    p0 = p0 < 0 ? 0 : p0;
    p1 = p1 > KV_GROUP ? KV_GROUP : p1;
    if (p0 >= p1) return;

    // positions that a later sequence of the call writes too are left to it
    __shared__ uint32_t taken;
    __shared__ float vscale[KV_GROUP][8];
    const int tid = threadIdx.x;
    if (tid == 0) taken = 0;
    __syncthreads();
    for (int o = b + 1 + tid; o < rows.batch; o += WRITE_THREADS) {
        const KvSpan so = kv_span(rows, c, o);
        if (so.slot != sp.slot) continue;
        int q0 = so.start + so.lo - first, q1 = so.start + so.hi - first;
        q0 = q0 < 0 ? 0 : q0;
        q1 = q1 > KV_GROUP ? KV_GROUP : q1;
        if (q0 < q1) atomicOr(&taken, (uint32_t)((((uint64_t)1 << (q1 - q0)) - 1) << q0));
    }
    __syncthreads();

    const int blocks = c.head_dim / 32, lane8 = tid & 7;
    const int64_t at = kv_group_index(c, sp.slot, head, group);
    uint8_t* kr = c.k + at * c.k_rec;
    uint8_t* vr = c.v + at * c.v_rec;
    const int n = (p1 - p0) * blocks;
    // every lane of a group of eight takes part in its exchanges
    for (int i = tid / 8; i < n; i += WRITE_THREADS / 8) {
        const int p = p0 + i / blocks, blk = i % blocks;
        const int64_t row = (int64_t)b * rows.tokens + (first + p - sp.start);
        const int col = head * c.head_dim + blk * 32 + lane8 * 4;
        const f4 xk = *reinterpret_cast<const f4*>(k + row * ks + col);
        const f4 xv = *reinterpret_cast<const f4*>(v + row * vs + col);
        const bool keep = !(taken >> p & 1);
        const int r = lane8 * 4;
        _Float16 d;
        uint32_t w = quantize4<KQ4>(xk, lane8, d);
        if constexpr (KQ4) {
            // dims r .. r + 3 are the low nibbles, the next lane's the high ones
            const uint32_t other = lane_xor1(w);
            if (keep && !(lane8 & 1))
                *reinterpret_cast<uint32_t*>(kr + blk * 512 + kv_k_byte(true, p, r)) = w | other << 4;
        } else if (keep) {
            *reinterpret_cast<uint32_t*>(kr + blk * 1024 + kv_k_byte(false, p, r)) = w;
        }
        const int krow = blocks * kv_block_bytes(KQ4) + blk * 64 + kv_row(p) * 2;
        if (keep && lane8 == 0) *reinterpret_cast<_Float16*>(kr + krow) = d;
        w = quantize4<VQ4>(xv, lane8, d);
        if constexpr (VQ4) w |= (uint32_t)__shfl_down((int)w, 4, 8) << 4;   // dims r + 16 ..: the high nibbles
        if (keep && (!VQ4 || lane8 < 4)) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                vr[blk * kv_block_bytes(VQ4) + kv_v_byte(VQ4, p, r + j)] = (uint8_t)(w >> (8 * j));
        }
        const int vrow = blocks * kv_block_bytes(VQ4) + blk * 64 + kv_row(p) * 2;
        if (lane8 == 0) {
            if (keep) *reinterpret_cast<_Float16*>(vr + vrow) = d;
            vscale[p][blk] = fabsf((float)d);
        }
    }
    __syncthreads();
    if (tid >= p0 && tid < p1 && !(taken >> tid & 1)) {
        float m = 0.f;
        for (int i = 0; i < blocks; i++) m = fmaxf(m, vscale[tid][i]);
        int e = -14;
        if (m > 0x1p-15f) (void)frexpf(m, &e);
        _Float16* tail = reinterpret_cast<_Float16*>(vr + blocks * (kv_block_bytes(VQ4) + 64)) + kv_row(tid);
        tail[0] = (_Float16)e;
        tail[32] = (_Float16)ldexpf(1.f, -e);
    }
}

// The inverse: eight lanes to a block of 32 elements.
template <bool KQ4, bool VQ4>
__global__ __launch_bounds__(WRITE_THREADS) void kv_read_kernel(KvView c, KvRows rows, float* k, int64_t ks, float* v,
                                                                int64_t vs, int groups) {
    const int gi = blockIdx.x % groups, rest = blockIdx.x / groups;
    const int head = rest % c.kv_heads, b = rest / c.kv_heads;
    const KvSpan sp = kv_span(rows, c, b);
    if (sp.lo >= sp.hi) return;
    const int group = (sp.start + sp.lo) / KV_GROUP + gi;
    const int first = group * KV_GROUP;
    int p0 = sp.start + sp.lo - first, p1 = sp.start + sp.hi - first;
    p0 = p0 < 0 ? 0 : p0;
    p1 = p1 > KV_GROUP ? KV_GROUP : p1;
    if (p0 >= p1) return;
    const int tid = threadIdx.x, blocks = c.head_dim / 32, r = (tid & 7) * 4;
    const int64_t at = kv_group_index(c, sp.slot, head, group);
    const uint8_t* kr = c.k + at * c.k_rec;
    const uint8_t* vr = c.v + at * c.v_rec;
    const int n = (p1 - p0) * blocks;
    for (int i = tid / 8; i < n; i += WRITE_THREADS / 8) {
        const int p = p0 + i / blocks, blk = i % blocks;
        const int64_t row = (int64_t)b * rows.tokens + (first + p - sp.start);
        const int col = head * c.head_dim + blk * 32 + r;
        const float dk = (float)*reinterpret_cast<const _Float16*>(kr + blocks * kv_block_bytes(KQ4) + blk * 64 + kv_row(p) * 2);
        const float dv = (float)*reinterpret_cast<const _Float16*>(vr + blocks * kv_block_bytes(VQ4) + blk * 64 + kv_row(p) * 2);
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

// Records that a run of `tokens` positions can touch.
int run_groups(int tokens, const KvView& c) {
    const int64_t n = ((int64_t)tokens + KV_GROUP - 2) / KV_GROUP + 1;
    return n < c.groups ? (int)n : c.groups;
}

}  // namespace

hipError_t launch_kv_write(const KvView& c, const KvRows& rows, const float* k, int64_t ks, const float* v, int64_t vs,
                           hipStream_t s) {
    const int groups = run_groups(rows.tokens, c);
    const dim3 grid((uint32_t)groups * c.kv_heads * rows.batch);
    auto go = [&](auto kernel) { kernel<<<grid, WRITE_THREADS, 0, s>>>(c, rows, k, ks, v, vs, groups); };
    if (c.k_q4) c.v_q4 ? go(kv_write_kernel<true, true>) : go(kv_write_kernel<true, false>);
    else c.v_q4 ? go(kv_write_kernel<false, true>) : go(kv_write_kernel<false, false>);
    return hipGetLastError();
}

hipError_t launch_kv_read(const KvView& c, const KvRows& rows, float* k, int64_t ks, float* v, int64_t vs,
                          hipStream_t s) {
    const int groups = run_groups(rows.tokens, c);
    const dim3 grid((uint32_t)groups * c.kv_heads * rows.batch);
    auto go = [&](auto kernel) { kernel<<<grid, WRITE_THREADS, 0, s>>>(c, rows, k, ks, v, vs, groups); };
    if (c.k_q4) c.v_q4 ? go(kv_read_kernel<true, true>) : go(kv_read_kernel<true, false>);
    else c.v_q4 ? go(kv_read_kernel<false, true>) : go(kv_read_kernel<false, false>);
    return hipGetLastError();
}

}  // namespace llmdot
