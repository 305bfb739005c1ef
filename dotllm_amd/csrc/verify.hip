// verify.hip -- speculative sampling: which drafted tokens stand against the
// target's probabilities, and the token that follows them.
//
// With p = softmax(target / T) and q = softmax(draft / T), draft i stands if
// u_i q(d_i) < p(d_i), i.e. u_i eq Zp < ep Zq with e = exp((x - max) / T); the
// next token is the first t with sum_{t' <= t} r > u sum r, r = max(p - q, 0).
// Whole numbers come out, so every exponential and sum is in 64 bits: a token
// whose border lies within rounding of the draw would otherwise change with the
// order of the sums (a 32-bit cumulative sum over 128k tokens puts some 2% of
// the draws next to one).
#include "kernels.h"
#include "common.h"

#include <math.h>

namespace llmdot {

namespace {

constexpr int VT = 256;

// e = exp((x - max) / T) of a logit; NaN has no mass, and where the maximum is
// +infinity only the infinities have some.
__device__ __forceinline__ double mass(float x, float mx, double inv_t) {
    if (mx == INFINITY) return x == INFINITY ? 1.0 : 0.0;
    if (!(x > -INFINITY)) return 0.0;
    return exp(((double)x - (double)mx) * inv_t);
}

__device__ double block_sum(double v, double* sh) {
    const int tid = threadIdx.x;
    __syncthreads();
    sh[tid] = v;
    __syncthreads();
    for (int n = VT / 2; n > 0; n /= 2) {
        if (tid < n) sh[tid] += sh[tid + n];
        __syncthreads();
    }
    return sh[0];
}
__device__ float block_max(float v, double* sh) {
    const int tid = threadIdx.x;
    __syncthreads();
    sh[tid] = v;
    __syncthreads();
    for (int n = VT / 2; n > 0; n /= 2) {
        if (tid < n) sh[tid] = fmax(sh[tid], sh[tid + n]);
        __syncthreads();
    }
    return (float)sh[0];
}

struct Row {
    float mx;
    double z;   // 0: no mass
};
__device__ Row row_stats(const float* x, int vocab, double inv_t, double* sh) {
    float m = -INFINITY;
    for (int t = threadIdx.x; t < vocab; t += VT) m = fmaxf(m, x[t]);   // fmaxf passes NaN by
    Row r;
    r.mx = block_max(m, sh);
    double z = 0.0;
    if (r.mx > -INFINITY)
        for (int t = threadIdx.x; t < vocab; t += VT) z += mass(x[t], r.mx, inv_t);
    r.z = block_sum(z, sh);
    return r;
}

__device__ int row_argmax(const float* x, int vocab, double* sh) {
    float m = -INFINITY;
    for (int t = threadIdx.x; t < vocab; t += VT) m = fmaxf(m, x[t]);
    m = block_max(m, sh);
    if (m == -INFINITY) return -1;
    double first = vocab;
    for (int t = threadIdx.x; t < vocab && first == vocab; t += VT)
        if (x[t] == m) first = t;
    return -(int)block_max(-(float)first, sh);
}

// One workgroup per sequence, row by row.
__global__ __launch_bounds__(VT) void verify_simple(VerifyArgs a) {
    __shared__ double sh[VT];
    const int b = blockIdx.x, tid = threadIdx.x;
    int n = a.counts ? a.counts[b] : a.drafts;
    n = n < 0 ? 0 : n > a.drafts ? a.drafts : n;
    const double inv_t = a.temperature > 0.f ? 1.0 / (double)a.temperature : 0.0;
    const float* target = a.target + (int64_t)b * (a.drafts + 1) * a.vocab;
    const float* draft = a.draft ? a.draft + (int64_t)b * a.drafts * a.vocab : nullptr;
    const int32_t* d = a.draft_tokens + (int64_t)b * a.drafts;
    const float* u = a.uniforms + (int64_t)b * (a.drafts + 1);
    int acc = 0;
    int next = -1;
    for (; acc < n; acc++) {
        const float* x = target + (int64_t)acc * a.vocab;
        const int t = d[acc];
        const bool inside = t >= 0 && t < a.vocab;
        if (a.temperature <= 0.f) {
            if (row_argmax(x, a.vocab, sh) != t) break;
            continue;
        }
        const Row p = row_stats(x, a.vocab, inv_t, sh);
        double q = 1.0;
        if (draft && inside) {
            const float* y = draft + (int64_t)acc * a.vocab;
            const Row r = row_stats(y, a.vocab, inv_t, sh);
            q = r.z > 0.0 ? mass(y[t], r.mx, inv_t) / r.z : 0.0;
        }
        if (!inside || !(p.z > 0.0) || !((double)u[acc] * q < mass(x[t], p.mx, inv_t) / p.z)) break;
    }
    const float* x = target + (int64_t)acc * a.vocab;
    if (a.temperature <= 0.f) {
        next = row_argmax(x, a.vocab, sh);
    } else {
        const Row p = row_stats(x, a.vocab, inv_t, sh);
        Row r{0.f, 0.0};
        const float* y = nullptr;
        int one = -1;
        if (acc < n) {
            if (draft) {
                y = draft + (int64_t)acc * a.vocab;
                r = row_stats(y, a.vocab, inv_t, sh);
                if (!(r.z > 0.0)) y = nullptr;
            } else {
                one = d[acc];
            }
        }
        auto residual = [&](int t) {
            const double pt = p.z > 0.0 ? mass(x[t], p.mx, inv_t) / p.z : 0.0;
            const double qt = y ? mass(y[t], r.mx, inv_t) / r.z : t == one ? 1.0 : 0.0;
            return fmax(pt - qt, 0.0);
        };
        for (int pass = 0; pass < 2 && next < 0; pass++) {
            if (pass) { y = nullptr; one = -1; }
            double total = 0.0;
            for (int t = tid; t < a.vocab; t += VT) total += residual(t);
            total = block_sum(total, sh);
            if (!(total > 0.0)) continue;
            const double want = (double)u[a.drafts] * total;
            // runs of consecutive tokens per thread, then the run that holds the draw
            const int per = (a.vocab + VT - 1) / VT, t0 = tid * per, t1 = t0 + per < a.vocab ? t0 + per : a.vocab;
            double mine = 0.0;
            for (int t = t0; t < t1; t++) mine += residual(t);
            __syncthreads();
            sh[tid] = mine;
            __syncthreads();
            double before = 0.0;
            for (int j = 0; j < tid; j++) before += sh[j];
            int found = a.vocab, last = -1;
            double cum = before;
            for (int t = t0; t < t1; t++) {
                const double v = residual(t);
                cum += v;
                if (v > 0.0) last = t;
                if (v > 0.0 && cum > want && found == a.vocab) found = t;
            }
            const int f = -(int)block_max(-(float)found, sh), e = (int)block_max((float)last, sh);
            next = f < a.vocab ? f : e;   // a draw past the last border by rounding
        }
    }
    if (tid <= a.drafts)
        for (int i = tid; i <= a.drafts; i += VT)
            a.tokens_out[(int64_t)b * (a.drafts + 1) + i] = i < acc ? d[i] : i == acc ? next : -1;
    if (tid == 0) a.accepted_out[b] = acc;
}

}  // namespace

size_t verify_workspace(int, int, int) { return 0; }

hipError_t launch_verify(const VerifyArgs& a, hipStream_t s) {
    verify_simple<<<dim3(a.batch), VT, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace llmdot
