// kv_attention.hip -- attention over the quantised KV cache (layout: kv_layout.h).
#include "kernels.h"
#include "kv_layout.h"

#include <math.h>

namespace llmdot {

namespace {

__device__ __forceinline__ float kv_k_value(const KvView& c, const uint8_t* rec, int p, int d) {
    const int blocks = c.head_dim / 32, blk = d >> 5, r = d & 31;
    uint32_t u = rec[blk * kv_block_bytes(c.k_q4) + kv_k_byte(c.k_q4, p, r)];
    if (c.k_q4) u = (kv_k_high(r) ? u >> 4 : u) & 15;
    const float s = (float)*reinterpret_cast<const _Float16*>(rec + blocks * kv_block_bytes(c.k_q4) + blk * 64 + kv_row(p) * 2);
    return s * (float)((int)u - (c.k_q4 ? 8 : 128));
}
__device__ __forceinline__ float kv_v_value(const KvView& c, const uint8_t* rec, int p, int d) {
    const int blocks = c.head_dim / 32, blk = d >> 5, r = d & 31;
    uint32_t u = rec[blk * kv_block_bytes(c.v_q4) + kv_v_byte(c.v_q4, p, r)];
    if (c.v_q4) u = (kv_v_high(r) ? u >> 4 : u) & 15;
    const float s = (float)*reinterpret_cast<const _Float16*>(rec + blocks * kv_block_bytes(c.v_q4) + blk * 64 + kv_row(p) * 2);
    return s * (float)((int)u - (c.v_q4 ? 8 : 128));
}

// One wavefront per query head of a token: 64 keys at a time, one per lane,
// with the running maximum and sum; then the lanes take the dims.
__global__ __launch_bounds__(64) void kv_attention_simple(KvAttnArgs a) {
    const KvView& c = a.cache;
    const int h = blockIdx.x % a.heads, rest = blockIdx.x / a.heads;
    const int i = rest % a.rows.tokens, b = rest / a.rows.tokens;
    const KvSpan sp = kv_span(a.rows, c, b);
    if (i < sp.lo || i >= sp.hi) return;
    const int hd = c.head_dim, lane = threadIdx.x, head = h / (a.heads / c.kv_heads);
    const int64_t row = (int64_t)b * a.rows.tokens + i;
    const float* q = a.q + row * a.q_stride + h * hd;
    __shared__ float qs[256], ps[64];
    for (int d = lane; d < hd; d += 64) qs[d] = q[d] * a.scale;
    __syncthreads();
    const int P = a.prefix_len;
    const int64_t end = (int64_t)P + sp.start + i + 1;
    const int64_t begin = a.window > 0 && end > a.window ? end - a.window : 0;
    float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int64_t t0 = begin; t0 < end; t0 += 64) {
        const int64_t t = t0 + lane;
        float s = -INFINITY;
        if (t < end) {
            const bool pre = t < P;
            const KvView& w = pre ? a.prefix : c;
            const int p = (int)(pre ? t : t - P);
            const uint8_t* rec = w.k + kv_group_index(w, pre ? a.prefix_slot : sp.slot, head, p / KV_GROUP) * w.k_rec;
            s = 0.f;
            for (int d = 0; d < hd; d++) s = fmaf(qs[d], kv_k_value(w, rec, p % KV_GROUP, d), s);
        }
        const float mn = fmaxf(m, wave_max(s));
        const float p = t < end ? expf(s - mn) : 0.f;
        const float f = m == -INFINITY ? 0.f : expf(m - mn);
        l = l * f + wave_sum(p);
        m = mn;
        ps[lane] = p;
        __syncthreads();
        for (int x = 0; x < 4; x++) acc[x] *= f;
        for (int j = 0; j < 64 && t0 + j < end; j++) {
            const int64_t u = t0 + j;
            const bool pre = u < P;
            const KvView& w = pre ? a.prefix : c;
            const int pp = (int)(pre ? u : u - P);
            const uint8_t* rec = w.v + kv_group_index(w, pre ? a.prefix_slot : sp.slot, head, pp / KV_GROUP) * w.v_rec;
            for (int x = 0; x < 4 && x * 64 + lane < hd; x++)
                acc[x] = fmaf(ps[j], kv_v_value(w, rec, pp % KV_GROUP, x * 64 + lane), acc[x]);
        }
        __syncthreads();
    }
    float* o = a.out + row * a.out_stride + h * hd;
    for (int x = 0; x < 4 && x * 64 + lane < hd; x++) o[x * 64 + lane] = acc[x] / l;
}

}  // namespace

bool kv_attention_supported(int head_dim) {
    return head_dim == 64 || head_dim == 96 || head_dim == 128 || head_dim == 256;
}

size_t kv_attention_workspace(const KvView&, int, int, int, bool) { return 0; }

hipError_t launch_kv_attention(const KvAttnArgs& a, hipStream_t s) {
    const dim3 grid((uint32_t)a.rows.batch * a.rows.tokens * a.heads);
    kv_attention_simple<<<grid, 64, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace llmdot
