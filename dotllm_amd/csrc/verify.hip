// verify.hip -- speculative sampling: which drafted tokens stand against the
// target's probabilities, and the token that follows them.
//
// With p = softmax(target / T) and q = softmax(draft / T), draft i stands if
// u_i q(d_i) < p(d_i); the next token is the first t with sum_{t' <= t} r > u sum r,
// r = max(p - q, 0) at the first draft that does not stand (p after the last).
// Whole numbers come out, so exponentials and sums are in 64 bits: the order of
// the sums would otherwise decide draws next to one of the 2 V borders (a 32-bit
// cumulative sum over 128k tokens puts some 2% of the draws next to one).
//
// Three launches, each over slices of 2048 logits so that a single sequence
// fills the card: maximum and mass of every row's slices (the only pass over all
// rows); the drafts decided, by every workgroup for itself, and the residual's
// mass in the slices of the one row that matters; the slice that holds the
// draw, scanned.
#include "kernels.h"
#include "common.h"

#include <math.h>

namespace llmdot {

namespace {

constexpr int VT = 256;              // threads
constexpr int PER = 8;               // logits per thread
constexpr int SLICE = VT * PER;

// Maximum and mass of a slice (greedy: the maximum's first index).
struct SliceStats {
    double z;      // sum of exp((x - mx) / T)
    float mx;
    int32_t arg;
};
// A sequence's decision: the row that the next token comes from.
struct Verdict {
    double zp, zq;         // masses of its target and draft rows
    float mp, mq;          // and maxima
    int32_t accepted;
    int32_t one;           // drafts without probabilities: the token that did not stand, else -1
    int32_t has_q;
    int32_t pad;
};
struct SliceMass {
    double r, p;           // residual, and the target's own mass
};
struct Work {              // in the workspace
    SliceStats* stats;     // [batch][rows][slices], target rows first
    Verdict* verdict;      // [batch]
    SliceMass* mass;       // [batch][slices]
    int rows, slices;
};

// 2^y for y <= 0 by its Taylor series about the nearest integer (12 terms:
// 2e-16 of the value for |f| <= 1/2); y under -1200 and NaN give 0.
__device__ __forceinline__ double exp2_64(double y) {
    y = fmax(y, -1200.0);
    const double k = rint(y), f = y - k;
    double r = 2.5678435993488206e-11;                       // ln2^12 / 12!
    r = fma(r, f, 4.4455382718708116e-10);
    r = fma(r, f, 7.0549116208011234e-09);
    r = fma(r, f, 1.0178086009239699e-07);
    r = fma(r, f, 1.3215486790144309e-06);
    r = fma(r, f, 1.5252733804059841e-05);
    r = fma(r, f, 1.5403530393381608e-04);
    r = fma(r, f, 1.3333558146428443e-03);
    r = fma(r, f, 9.6181291076284772e-03);
    r = fma(r, f, 5.5504108664821580e-02);
    r = fma(r, f, 2.4022650695910071e-01);
    r = fma(r, f, 6.9314718055994531e-01);
    r = fma(r, f, 1.0);
    return ldexp(r, (int)k);
}

// exp((x - mx) / T), c = log2(e) / T; NaN has no mass, and where the maximum is
// +infinity only the infinities have some.
__device__ __forceinline__ double mass(float x, float mx, double c) {
    if (mx == INFINITY) return x == INFINITY ? 1.0 : 0.0;
    return exp2_64(((double)x - (double)mx) * c);
}
__device__ __forceinline__ double rate(double temperature) { return 1.4426950408889634074 / temperature; }

__device__ __forceinline__ int draft_count(const VerifyArgs& a, int b) {
    const int n = a.counts ? a.counts[b] : a.drafts;
    return n < 0 ? 0 : n > a.drafts ? a.drafts : n;
}
__device__ __forceinline__ const float* target_row(const VerifyArgs& a, int b, int i) {
    return a.target + ((int64_t)b * (a.drafts + 1) + i) * a.vocab;
}
__device__ __forceinline__ const float* draft_row(const VerifyArgs& a, int b, int i) {
    return a.draft + ((int64_t)b * a.drafts + i) * a.vocab;
}

// A thread's logits of a slice (consecutive ones), `pad` past the row's end.
__device__ __forceinline__ void load_slice(const float* row, int first, int vocab, float pad, float (&x)[PER]) {
    const int t0 = first + threadIdx.x * PER;
    if (t0 + PER <= vocab) {
#pragma unroll
        for (int j = 0; j < PER; j += 4) {   // rows begin at any multiple of 4 bytes
            const u32x4 w = ld16_a4(reinterpret_cast<const uint8_t*>(row + t0 + j));
            x[j] = __uint_as_float(w.x); x[j + 1] = __uint_as_float(w.y);
            x[j + 2] = __uint_as_float(w.z); x[j + 3] = __uint_as_float(w.w);
        }
    } else {
#pragma unroll
        for (int j = 0; j < PER; j++) x[j] = t0 + j < vocab ? row[t0 + j] : pad;
    }
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int k = 1; k < 64; k *= 2) v += __shfl_xor(v, k);
    return v;
}

template <bool GREEDY>
__global__ __launch_bounds__(VT) void verify_stats(VerifyArgs a, Work w) {
    const int slice = blockIdx.x % w.slices, b = blockIdx.x / w.slices, row = blockIdx.y;
    const int n = draft_count(a, b);
    const bool of_target = row <= a.drafts;
    const int i = of_target ? row : row - a.drafts - 1;
    if (of_target ? i > n : i >= n) return;
    float x[PER];
    load_slice(of_target ? target_row(a, b, i) : draft_row(a, b, i), slice * SLICE, a.vocab, -INFINITY, x);
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < PER; j++) m = fmaxf(m, x[j]);   // NaN passes by
    __shared__ float sm[VT / 64];
    __shared__ double sz[VT / 64];
    __shared__ int sa[VT / 64];
    const int wave = threadIdx.x / 64, lane = threadIdx.x & 63;
    const float wm = wave_max(m);
    if (lane == 0) sm[wave] = wm;
    __syncthreads();
    float mx = sm[0];
#pragma unroll
    for (int k = 1; k < VT / 64; k++) mx = fmaxf(mx, sm[k]);
    double z = 0.0;
    int arg = -1;
    if constexpr (GREEDY) {
        int at = 0x7fffffff;
#pragma unroll
        for (int j = PER - 1; j >= 0; j--)
            if (x[j] == mx) at = slice * SLICE + threadIdx.x * PER + j;
#pragma unroll
        for (int k = 1; k < 64; k *= 2) {
            const int o = __shfl_xor(at, k);
            at = o < at ? o : at;
        }
        if (lane == 0) sa[wave] = at;
        __syncthreads();
        arg = sa[0];
#pragma unroll
        for (int k = 1; k < VT / 64; k++) arg = sa[k] < arg ? sa[k] : arg;
    } else {
        const double c = rate((double)a.temperature);
        if (mx > -INFINITY)
#pragma unroll
            for (int j = 0; j < PER; j++) z += mass(x[j], mx, c);
        z = wave_sum64(z);
        if (lane == 0) sz[wave] = z;
        __syncthreads();
        z = sz[0];
#pragma unroll
        for (int k = 1; k < VT / 64; k++) z += sz[k];
    }
    if (threadIdx.x == 0) w.stats[((int64_t)b * w.rows + row) * w.slices + slice] = SliceStats{z, mx, arg};
}

// A row's maximum and mass from its slices, by 16 lanes (every lane gets them).
__device__ __forceinline__ void join_slices(const SliceStats* s, int slices, int lane16, double c, float& mx, double& z) {
    float m = -INFINITY;
    for (int k = lane16; k < slices; k += 16) m = fmaxf(m, s[k].mx);
    mx = max16(m);
    z = 0.0;
    for (int k = lane16; k < slices; k += 16) {
        const SliceStats t = s[k];
        // the slice's mass against the row's maximum
        if (t.mx > -INFINITY) z += t.z * mass(t.mx, mx, c);
    }
#pragma unroll
    for (int k = 1; k < 16; k *= 2) z += __shfl_xor(z, k);
}
// The same for the first maximum.
__device__ __forceinline__ int join_first(const SliceStats* s, int slices, int lane16) {
    float m = -INFINITY;
    for (int k = lane16; k < slices; k += 16) m = fmaxf(m, s[k].mx);
    m = max16(m);
    if (m == -INFINITY) return -1;
    int at = 0x7fffffff;
    for (int k = lane16; k < slices; k += 16)
        if (s[k].mx == m && s[k].arg < at) at = s[k].arg;
#pragma unroll
    for (int k = 1; k < 16; k *= 2) {
        const int o = __shfl_xor(at, k);
        at = o < at ? o : at;
    }
    return at;
}

// How many leading drafts of sequence b stand (the whole workgroup; 16 lanes a draft).
template <bool GREEDY>
__device__ int decide(const VerifyArgs& a, const Work& w, int b, int n, int* fail) {
    const int set = threadIdx.x / 16, lane16 = threadIdx.x & 15;
    if (threadIdx.x == 0) *fail = n;
    __syncthreads();
    const SliceStats* stats = w.stats + (int64_t)b * w.rows * w.slices;
    const double c = GREEDY ? 0.0 : rate((double)a.temperature);
    for (int i0 = 0; i0 < n; i0 += VT / 16) {
        const int i = i0 + set;
        if (i < n) {
            const int t = a.draft_tokens[(int64_t)b * a.drafts + i];
            bool stands = t >= 0 && t < a.vocab;
            if constexpr (GREEDY) {
                stands = join_first(stats + (int64_t)i * w.slices, w.slices, lane16) == t && stands;
            } else {
                float mp, mq;
                double zp, zq, q = 1.0;
                join_slices(stats + (int64_t)i * w.slices, w.slices, lane16, c, mp, zp);
                if (a.draft) {
                    join_slices(stats + (int64_t)(a.drafts + 1 + i) * w.slices, w.slices, lane16, c, mq, zq);
                    q = stands && zq > 0.0 ? mass(draft_row(a, b, i)[t], mq, c) / zq : 0.0;
                }
                const double p = stands && zp > 0.0 ? mass(target_row(a, b, i)[t], mp, c) / zp : 0.0;
                stands = (double)a.uniforms[(int64_t)b * (a.drafts + 1) + i] * q < p && stands;
            }
            if (!stands && lane16 == 0) atomicMin(fail, i);
        }
        __syncthreads();
        if (*fail < n) break;   // the same for all: nothing writes it between here and the next barrier
        __syncthreads();
    }
    return *fail;
}

__device__ __forceinline__ double residual(float x, float y, const Verdict& v, int t, double c, double& p) {
    p = v.zp > 0.0 ? mass(x, v.mp, c) / v.zp : 0.0;
    const double q = v.has_q ? mass(y, v.mq, c) / v.zq : t == v.one ? 1.0 : 0.0;
    return fmax(p - q, 0.0);
}

__global__ __launch_bounds__(VT) void verify_residual(VerifyArgs a, Work w) {
    __shared__ int fail;
    __shared__ Verdict sv;
    __shared__ double sr[VT / 64], sp[VT / 64];
    const int slice = blockIdx.x % w.slices, b = blockIdx.x / w.slices;
    const int n = draft_count(a, b);
    const int acc = decide<false>(a, w, b, n, &fail);
    const double c = rate((double)a.temperature);
    const SliceStats* stats = w.stats + (int64_t)b * w.rows * w.slices;
    if (threadIdx.x < 16) {
        Verdict v{0.0, 0.0, 0.f, 0.f, acc, -1, 0, 0};
        join_slices(stats + (int64_t)acc * w.slices, w.slices, threadIdx.x, c, v.mp, v.zp);
        if (acc < n) {
            if (a.draft) {
                join_slices(stats + (int64_t)(a.drafts + 1 + acc) * w.slices, w.slices, threadIdx.x, c, v.mq, v.zq);
                v.has_q = v.zq > 0.0;
            } else {
                v.one = a.draft_tokens[(int64_t)b * a.drafts + acc];
            }
        }
        if (threadIdx.x == 0) {
            sv = v;
            if (slice == 0) w.verdict[b] = v;
        }
    }
    __syncthreads();
    const Verdict v = sv;
    float x[PER], y[PER];
    load_slice(target_row(a, b, acc), slice * SLICE, a.vocab, -INFINITY, x);
    if (v.has_q) load_slice(draft_row(a, b, acc), slice * SLICE, a.vocab, -INFINITY, y);
    double r = 0.0, s = 0.0;
#pragma unroll
    for (int j = 0; j < PER; j++) {
        double p;
        r += residual(x[j], v.has_q ? y[j] : 0.f, v, slice * SLICE + threadIdx.x * PER + j, c, p);
        s += p;
    }
    r = wave_sum64(r);
    s = wave_sum64(s);
    if ((threadIdx.x & 63) == 0) { sr[threadIdx.x / 64] = r; sp[threadIdx.x / 64] = s; }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < VT / 64; k++) { r += sr[k]; s += sp[k]; }
        w.mass[(int64_t)b * w.slices + slice] = SliceMass{r, s};
    }
}

__device__ __forceinline__ void write_tokens(const VerifyArgs& a, int b, int acc, int next) {
    for (int i = threadIdx.x; i <= a.drafts; i += VT)
        a.tokens_out[(int64_t)b * (a.drafts + 1) + i] =
            i < acc ? a.draft_tokens[(int64_t)b * a.drafts + i] : i == acc ? next : -1;
    if (threadIdx.x == 0) a.accepted_out[b] = acc;
}

__global__ __launch_bounds__(VT) void verify_greedy(VerifyArgs a, Work w) {
    __shared__ int fail;
    const int b = blockIdx.x;
    const int acc = decide<true>(a, w, b, draft_count(a, b), &fail);
    const int next = join_first(w.stats + ((int64_t)b * w.rows + acc) * w.slices, w.slices, threadIdx.x & 15);
    write_tokens(a, b, acc, next);
}

// Inclusive sums over the workgroup's threads, in thread order.
__device__ __forceinline__ double block_scan(double v, double* sh) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
#pragma unroll
    for (int k = 1; k < 64; k *= 2) {
        const double o = __shfl_up(v, k);
        if (lane >= k) v += o;
    }
    __syncthreads();
    if (lane == 63) sh[wave] = v;
    __syncthreads();
    for (int k = 0; k < wave; k++) v += sh[k];
    return v;
}

__global__ __launch_bounds__(VT) void verify_select(VerifyArgs a, Work w) {
    __shared__ double sh[VT / 64], before_at;
    __shared__ int first, last;
    const int b = blockIdx.x, tid = threadIdx.x;
    Verdict v = w.verdict[b];
    const SliceMass* m = w.mass + (int64_t)b * w.slices;
    const double u = (double)a.uniforms[(int64_t)b * (a.drafts + 1) + a.drafts];
    const double c = rate((double)a.temperature);
    // runs of slices per thread
    const int per = (w.slices + VT - 1) / VT, k0 = tid * per < w.slices ? tid * per : w.slices,
              k1 = k0 + per < w.slices ? k0 + per : w.slices;
    bool of_p = false;
    double mine = 0.0, upto = 0.0, total = 0.0;
    for (int pass = 0; pass < 2; pass++) {
        of_p = pass == 1;
        mine = 0.0;
        for (int k = k0; k < k1; k++) mine += of_p ? m[k].p : m[k].r;
        upto = block_scan(mine, sh);
        if (tid == VT - 1) before_at = upto;
        __syncthreads();
        total = before_at;
        if (total > 0.0) break;   // the same for all
        __syncthreads();
    }
    int next = -1;
    if (total > 0.0) {
        if (of_p) { v.has_q = 0; v.one = -1; }
        const double want = u * total;
        if (tid == 0) { first = w.slices; last = -1; }
        __syncthreads();
        double cum = upto - mine;
        int found = w.slices, some = -1;
        for (int k = k0; k < k1; k++) {
            const double s = of_p ? m[k].p : m[k].r;
            cum += s;
            if (s > 0.0) {
                some = k;
                if (cum > want && found == w.slices) found = k;
            }
        }
        if (found < w.slices) atomicMin(&first, found);
        if (some >= 0) atomicMax(&last, some);
        __syncthreads();
        const int slice = first < w.slices ? first : last;   // a draw past the last border by rounding
        __syncthreads();
        if (slice >= k0 && slice < k1) {
            double s = upto - mine;
            for (int k = k0; k < slice; k++) s += of_p ? m[k].p : m[k].r;
            before_at = s;
        }
        if (tid == 0) { first = 0x7fffffff; last = -1; }
        __syncthreads();
        float x[PER], y[PER];
        load_slice(target_row(a, b, v.accepted), slice * SLICE, a.vocab, -INFINITY, x);
        if (v.has_q) load_slice(draft_row(a, b, v.accepted), slice * SLICE, a.vocab, -INFINITY, y);
        double r[PER], sum = 0.0;
        const int t0 = slice * SLICE + tid * PER;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            double p;
            r[j] = residual(x[j], v.has_q ? y[j] : 0.f, v, t0 + j, c, p);
            sum += r[j];
        }
        cum = before_at + (block_scan(sum, sh) - sum);
        int at = 0x7fffffff, most = -1;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            cum += r[j];
            if (r[j] > 0.0) {
                most = t0 + j;
                if (cum > want && at == 0x7fffffff) at = t0 + j;
            }
        }
        if (at != 0x7fffffff) atomicMin(&first, at);
        if (most >= 0) atomicMax(&last, most);
        __syncthreads();
        next = first != 0x7fffffff ? first : last;
    }
    write_tokens(a, b, v.accepted, next);
}

size_t layout(int batch, int drafts, int vocab, bool draft, uint8_t* base, Work* w) {
    w->slices = (vocab + SLICE - 1) / SLICE;
    w->rows = drafts + 1 + (draft ? drafts : 0);
    size_t at = 0;
    auto take = [&](size_t n) {
        uint8_t* p = base + at;
        at += (n + 15) & ~(size_t)15;
        return p;
    };
    w->stats = reinterpret_cast<SliceStats*>(take(sizeof(SliceStats) * (size_t)batch * w->rows * w->slices));
    w->verdict = reinterpret_cast<Verdict*>(take(sizeof(Verdict) * (size_t)batch));
    w->mass = reinterpret_cast<SliceMass*>(take(sizeof(SliceMass) * (size_t)batch * w->slices));
    return at;
}

}  // namespace

size_t verify_workspace(int batch, int drafts, int vocab) {
    Work w;
    return layout(batch, drafts, vocab, true, nullptr, &w);
}

hipError_t launch_verify(const VerifyArgs& a, hipStream_t s) {
    Work w;
    const bool greedy = a.temperature <= 0.f;
    layout(a.batch, a.drafts, a.vocab, a.draft && !greedy, a.work, &w);
    const dim3 grid((uint32_t)w.slices * a.batch, w.rows);
    if (greedy) {
        verify_stats<true><<<grid, VT, 0, s>>>(a, w);
        verify_greedy<<<dim3(a.batch), VT, 0, s>>>(a, w);
    } else {
        verify_stats<false><<<grid, VT, 0, s>>>(a, w);
        verify_residual<<<dim3((uint32_t)w.slices * a.batch), VT, 0, s>>>(a, w);
        verify_select<<<dim3(a.batch), VT, 0, s>>>(a, w);
    }
    return hipGetLastError();
}

}  // namespace llmdot
