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
// Two launches, each over slices of 1024 or 4096 logits so that a single sequence
// fills the card: maximum and mass of every row's slices (the only pass over all
// rows); then every workgroup decides its sequence's drafts for itself and sums
// the residual in its slice of the one row that matters, and the last of them
// finds the slice that holds the draw and scans it.  Bound by reading the logits
// and, about as long, by the 64-bit exponentials: 16 sequences of 5 drafts, 128256
// logits and a draft model take 32.5 us (statistics 17, draw 17; 53 MB), one of 4
// drafts and 32000 logits 10.4 (3 + 8: latencies).
#include "kernels.h"
#include "common.h"

#include <math.h>

namespace llmdot {

namespace {

constexpr int VT = 256;              // threads
constexpr int WAVES = VT / 64;
constexpr int QUAD = 4;              // consecutive logits of a thread; quads of a slice lie VT * QUAD apart

// Maximum and mass of a slice (greedy: the maximum's first index).
struct SliceStats {
    double z;      // sum of exp((x - mx) / T)
    float mx;
    int32_t arg;
};
// A sequence's decision: the row that the next token comes from.
struct Decision {
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
    float* picked;         // [batch][rows] logit of each row's drafted token
    uint32_t* drawn;       // [MAX_SEQUENCES] workgroups done with a sequence, zero between launches
    SliceStats* stats;     // [batch][rows][slices], target rows first
    SliceMass* mass;       // [batch][slices]
    int rows, slices;
};

// exp((x - mx) / T) for the logits x of a row with maximum mx.  2^y with y =
// (x - mx) log2(e) / T: the nearest integer goes into the exponent, the rest
// (|f| <= 1/2) through a polynomial of degree 10 whose largest relative error
// there is the least (2.2e-16, by Remez's exchange; 2.8e-16 with these doubles).
// Adding and taking off 1.5 * 2^52 rounds to the integer and leaves it in the
// low word: no conversions, which take four times an FMA's time.  Logits under
// 2^-1000 of the maximum, -infinity and NaN have no mass.
struct Series {            // kept in scalar registers: as operands an FMA takes them in place
    double c[11];
    __device__ __forceinline__ Series() {
        constexpr double k[11] = {1.0, 6.9314718055994973e-01, 2.4022650695908768e-01, 5.5504108664458839e-02,
                                  9.6181291080346207e-03, 1.3333558228560802e-03, 1.5403529961092289e-04,
                                  1.5252658116891647e-05, 1.3215662854692098e-06, 1.0208537850876446e-07,
                                  7.0372755249486504e-09};
#pragma unroll
        for (int i = 0; i < 11; i++) {
            c[i] = k[i];
            asm("" : "+s"(c[i]));   // a number like any other to the compiler
        }
    }
    __device__ __forceinline__ double exp2(double f) const {
        double r = fma(c[10], f, c[9]);
#pragma unroll
        for (int i = 8; i >= 0; i--) r = fma(r, f, c[i]);
        return r;
    }
};
constexpr double BIG = 6755399441055744.0;
// One such number, for any x up to mx: 0 for NaN, 1 for the maximum itself.
__device__ __forceinline__ double mass_of(float x, float mx, const VerifyArgs& a, const Series& series) {
    const double d = (double)x - (double)mx, t = fma(d, a.rate, BIG);
    const uint64_t u = __builtin_bit_cast(uint64_t, series.exp2(fma(d, a.rate, BIG - t)));
    const double v = __builtin_bit_cast(double, u + (__builtin_bit_cast(uint64_t, t) << 52));
    return x == mx ? 1.0 : d * a.rate > -1000.0 ? v : 0.0;
}
// The masses of a slice's logits.
struct Masses {
    double c, m;           // y = c (x - m)
    float least;           // logits above it have a mass
    // a maximum of +infinity: only the infinities pass `least`, and y is 0 for them
    __device__ __forceinline__ Masses(float mx, const VerifyArgs& a) {
        const bool infinite = mx == INFINITY, none = !(mx > -INFINITY);
        m = infinite || none ? 0.0 : (double)mx;
        c = infinite ? 0.0 : a.rate;
        // where floats (or doubles) lie further apart than the masses reach, the maximum stays above
        const float low = __double2float_rd(m - a.reach);
        least = none ? INFINITY : infinite ? 3.4028234663852886e38f : low < mx ? low : below(mx);
    }
    __device__ __forceinline__ double of(float x, const Series& series) const {
        uint32_t k;
        const uint64_t u = significand(x, series, k);
        const bool some = x > least;
        const uint32_t high = some ? (uint32_t)(u >> 32) + (k << 20) : 0, low = some ? (uint32_t)u : 0;
        return __builtin_bit_cast(double, (uint64_t)high << 32 | low);
    }
    // `of` for sums that hold the maximum's own mass of 1: logits without mass count
    // 2^-1000 or less each.  For a finite maximum with `least` no further below it
    // than an exponent reaches.
    __device__ __forceinline__ bool steady(float mx) const {
        return mx > -INFINITY && mx < INFINITY && ((double)least - m) * c > -1020.0;
    }
    __device__ __forceinline__ double beside(float x, const Series& series) const {
        uint32_t k;
        const uint64_t u = significand(x, series, k);
        return __builtin_bit_cast(double, u + ((uint64_t)k << 52));
    }

private:
    __device__ __forceinline__ static float below(float v) {   // the next float, v finite
        const uint32_t u = __builtin_bit_cast(uint32_t, v);
        return __builtin_bit_cast(float, v > 0.f ? u - 1 : v < 0.f ? u + 1 : 0x80000001u);
    }
    // 2^f as a double's bits, and the integer modulo 2^32; x = m gives f = 0 whatever c
    __device__ __forceinline__ uint64_t significand(float x, const Series& series, uint32_t& k) const {
        const double d = (double)__builtin_amdgcn_fmed3f(x, least, 3.4028234663852886e38f) - m;
        const double t = fma(d, c, BIG);
        k = (uint32_t)__builtin_bit_cast(uint64_t, t);
        return __builtin_bit_cast(uint64_t, series.exp2(fma(d, c, BIG - t)));
    }
};

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

// A thread's logits of a slice of Q quads per thread; -infinity past the row's end.
template <int Q>
__device__ __forceinline__ void load_slice(const float* row, int slice, int vocab, float (&x)[Q][QUAD]) {
    const int first = slice * Q * (VT * QUAD) + (int)threadIdx.x * QUAD;
    // no branch around a load: the ones behind it would wait for it
    if ((slice + 1) * Q * (VT * QUAD) <= vocab) {
#pragma unroll
        for (int j = 0; j < Q; j++) {   // rows begin at any multiple of 4 bytes
            const u32x4 w = ld16_a4(reinterpret_cast<const uint8_t*>(row + first + j * (VT * QUAD)));
            x[j][0] = __uint_as_float(w.x); x[j][1] = __uint_as_float(w.y);
            x[j][2] = __uint_as_float(w.z); x[j][3] = __uint_as_float(w.w);
        }
    } else {
#pragma unroll
        for (int j = 0; j < Q; j++)
#pragma unroll
            for (int i = 0; i < QUAD; i++) {
                const int t = first + j * (VT * QUAD) + i;
                const float v = row[t < vocab ? t : vocab - 1];
                x[j][i] = t < vocab ? v : -INFINITY;
            }
    }
}

// Results that another workgroup of the same launch reads: past the XCD's own L2.
template <typename T>
__device__ __forceinline__ void store_through(T* p, const T& v) {
    static_assert(sizeof(T) % 8 == 0, "whole words");
    uint64_t w[sizeof(T) / 8];
    __builtin_memcpy(w, &v, sizeof(T));
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 8); i++)
        __hip_atomic_store(reinterpret_cast<uint64_t*>(p) + i, w[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T>
__device__ __forceinline__ T load_past(const T* p) {
    uint64_t w[sizeof(T) / 8];
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 8); i++)
        w[i] = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p) + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    T v;
    __builtin_memcpy(&v, w, sizeof(T));
    return v;
}
// Whether this workgroup is the last of `of` to get here (thread 0 has stored
// its result through); the counter is left at zero.
__device__ __forceinline__ bool last_of(uint32_t* count, uint32_t of) {
    __shared__ int last;
    if (threadIdx.x == 0) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const uint32_t was = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = was + 1 == of;
        if (last) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return last;
}

// 64-bit values over lanes, without the LDS.
template <typename F>
__device__ __forceinline__ double lanes64(F f, double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)f((uint32_t)u) | (uint64_t)f((uint32_t)(u >> 32)) << 32);
}
__device__ __forceinline__ double sum16_64(double v) {
    v += lanes64(lane_xor1, v);
    v += lanes64(lane_xor2, v);
    v += lanes64(lane_mirror8, v);
    return v + lanes64(lane_mirror16, v);
}
__device__ __forceinline__ double wave_sum64(double v) {
    v = sum16_64(v);
    v += lanes64(lane_xor16, v);
    return v + lanes64(lane_xor32, v);
}
__device__ __forceinline__ int wave_min_int(int v) {
    auto step = [&](uint32_t (*f)(uint32_t)) { const int o = (int)f((uint32_t)v); v = o < v ? o : v; };
    step(lane_xor1); step(lane_xor2); step(lane_mirror8); step(lane_mirror16); step(lane_xor16); step(lane_xor32);
    return v;
}

__device__ __forceinline__ void write_tokens(const VerifyArgs& a, int b, int acc, int next) {
    for (int i = threadIdx.x; i <= a.drafts; i += VT)
        a.tokens_out[(int64_t)b * (a.drafts + 1) + i] =
            i < acc ? a.draft_tokens[(int64_t)b * a.drafts + i] : i == acc ? next : -1;
    if (threadIdx.x == 0) a.accepted_out[b] = acc;
}

// A row's maximum and mass from its slices, by 16 lanes (every lane gets them).
__device__ __forceinline__ void join_slices(const VerifyArgs& a, const SliceStats* s, int slices, int lane16,
                                            const Series& series, float& mx, double& z) {
    mx = -INFINITY;
    z = 0.0;
    for (int k = lane16; k < slices; k += 16) {
        const SliceStats t = s[k];
        const bool more = t.mx > mx;   // against the larger maximum
        const float m = more ? t.mx : mx;
        const double f = mass_of(more ? mx : t.mx, m, a, series);
        z = more ? z * f + t.z : z + t.z * f;
        mx = m;
    }
    const float m = max16(mx);
    z = sum16_64(z * mass_of(mx, m, a, series));
    mx = m;
}
// The first of a row's maxima, from its slices.
__device__ __forceinline__ int join_first(const SliceStats* s, int slices, int lane16) {
    float mx = -INFINITY;
    int at = 0x7fffffff;
    for (int k = lane16; k < slices; k += 16) {   // ascending: an equal maximum further on is not the first
        const SliceStats t = s[k];
        if (t.mx > mx) { mx = t.mx; at = t.arg; }
    }
    const float m = max16(mx);
    if (m == -INFINITY) return -1;
    at = mx == m ? at : 0x7fffffff;
#pragma unroll
    for (int k = 1; k < 16; k *= 2) {
        const int o = __shfl_xor(at, k);
        at = o < at ? o : at;
    }
    return at;
}

// The leading drafts of sequence b that stand, and the statistics of the rows
// behind the first that does not, by the whole workgroup: 16 lanes a draft.  All
// loads are of known addresses, so they are out at once.
template <bool GREEDY>
__device__ __forceinline__ Decision decide(const VerifyArgs& a, const Work& w, int b) {
    __shared__ int fail;
    __shared__ Decision of_set[VT / 16];
    const int set = threadIdx.x / 16, lane16 = threadIdx.x & 15, n = draft_count(a, b);
    if (threadIdx.x == 0) fail = n;
    __syncthreads();
    const SliceStats* stats = w.stats + (int64_t)b * w.rows * w.slices;
    const float* picked = w.picked + (int64_t)b * w.rows;
    const Series series;
    for (int i0 = 0;; i0 += VT / 16) {
        const int i = i0 + set;
        if (i <= n) {
            const bool drafted = i < a.drafts, with_q = drafted && w.rows > a.drafts + 1;
            const int t = drafted ? a.draft_tokens[(int64_t)b * a.drafts + i] : -1;
            const double u = (double)a.uniforms[(int64_t)b * (a.drafts + 1) + i];
            bool stands = t >= 0 && t < a.vocab;
            Decision v{0.0, 0.0, 0.f, 0.f, i, -1, 0, 0};
            if constexpr (GREEDY) {
                v.one = join_first(stats + (int64_t)i * w.slices, w.slices, lane16);
                stands = stands && v.one == t;
            } else {
                const float xt = picked[i], yt = with_q ? picked[a.drafts + 1 + i] : 0.f;
                join_slices(a, stats + (int64_t)i * w.slices, w.slices, lane16, series, v.mp, v.zp);
                double q = 1.0;
                if (with_q) {
                    join_slices(a, stats + (int64_t)(a.drafts + 1 + i) * w.slices, w.slices, lane16, series, v.mq, v.zq);
                    q = v.zq > 0.0 ? mass_of(yt, v.mq, a, series) / v.zq : 0.0;
                }
                const double p = v.zp > 0.0 ? mass_of(xt, v.mp, a, series) / v.zp : 0.0;
                stands = stands && u * q < p;
                // after the last draft the next token is the target's alone
                v.has_q = with_q && i < n && v.zq > 0.0;
                if (!a.draft && i < n) v.one = t;
            }
            if (lane16 == 0) {
                of_set[set] = v;
                if (!stands) atomicMin(&fail, i);
            }
        }
        __syncthreads();
        const int acc = fail;   // the same for all threads: the next write waits for the barrier
        const Decision v = of_set[acc < i0 + VT / 16 ? acc - i0 : 0];
        __syncthreads();
        if (acc < i0 + VT / 16) return v;
    }
}

template <bool GREEDY, int Q>
__global__ __launch_bounds__(VT) void verify_stats(VerifyArgs a, Work w) {
    const int slice = blockIdx.x % w.slices, b = blockIdx.x / w.slices, row = blockIdx.y;
    const int n = draft_count(a, b);
    const bool of_target = row <= a.drafts;
    const int i = of_target ? row : row - a.drafts - 1;
    if (of_target ? i > n : i >= n) return;
    const float* logits = of_target ? target_row(a, b, i) : draft_row(a, b, i);
    float x[Q][QUAD];
    load_slice<Q>(logits, slice, a.vocab, x);
    if (threadIdx.x == 0 && i < a.drafts) {
        const int t = a.draft_tokens[(int64_t)b * a.drafts + i];
        if (t >= 0 && t < a.vocab && t / (Q * VT * QUAD) == slice) w.picked[(int64_t)b * w.rows + row] = logits[t];
    }
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < Q; j++)
#pragma unroll
        for (int k = 0; k < QUAD; k++) m = fmaxf(m, x[j][k]);   // NaN passes by
    __shared__ float sm[WAVES];
    __shared__ double sz[WAVES];
    __shared__ int sa[WAVES];
    const int wave = threadIdx.x / 64, lane = threadIdx.x & 63;
    m = wave_max(m);
    if (lane == 0) sm[wave] = m;
    __syncthreads();
    float mx = sm[0];
#pragma unroll
    for (int k = 1; k < WAVES; k++) mx = fmaxf(mx, sm[k]);
    double z = 0.0;
    int arg = -1;
    if constexpr (GREEDY) {
        int at = 0x7fffffff;
#pragma unroll
        for (int j = Q - 1; j >= 0; j--)
#pragma unroll
            for (int k = QUAD - 1; k >= 0; k--)
                if (x[j][k] == mx) at = (slice * Q + j) * (VT * QUAD) + (int)threadIdx.x * QUAD + k;
        at = wave_min_int(at);
        if (lane == 0) sa[wave] = at;
        __syncthreads();
        arg = sa[0];
#pragma unroll
        for (int k = 1; k < WAVES; k++) arg = sa[k] < arg ? sa[k] : arg;
    } else {
        const Masses e(mx, a);
        const Series series;
        if (e.steady(mx)) {
#pragma unroll
            for (int j = 0; j < Q; j++)
#pragma unroll
                for (int k = 0; k < QUAD; k++) z += e.beside(x[j][k], series);
        } else {
#pragma unroll
            for (int j = 0; j < Q; j++)
#pragma unroll
                for (int k = 0; k < QUAD; k++) z += e.of(x[j][k], series);
        }
        z = wave_sum64(z);
        if (lane == 0) sz[wave] = z;
        __syncthreads();
        z = sz[0];
#pragma unroll
        for (int k = 1; k < WAVES; k++) z += sz[k];
    }
    if (threadIdx.x == 0) w.stats[((int64_t)b * w.rows + row) * w.slices + slice] = SliceStats{z, mx, arg};
}

__global__ __launch_bounds__(VT) void verify_greedy(VerifyArgs a, Work w) {
    const int b = blockIdx.x;
    const Decision v = decide<true>(a, w, b);
    write_tokens(a, b, v.accepted, v.one);
}

// max(p - q, 0) of a token, and p.
struct Residual {
    Series series;
    Masses p, q;
    double ip, iq;         // 1 / masses, 0 without any
    int one;
    __device__ __forceinline__ Residual(const Decision& v, const VerifyArgs& a)
        : p(v.mp, a), q(v.mq, a), ip(v.zp > 0.0 ? 1.0 / v.zp : 0.0), iq(v.has_q ? 1.0 / v.zq : 0.0), one(v.one) {}
    __device__ __forceinline__ double of(float x, float y, int t, double& pt) const {
        pt = p.of(x, series) * ip;
        return fmax(pt - (iq > 0.0 ? q.of(y, series) * iq : t == one ? 1.0 : 0.0), 0.0);
    }
};

// Inclusive sums over the wavefront's lanes: within rows of 16, then rows 0 and 2
// into 1 and 3, then the lower half into the upper.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp64(double v) {   // 0 where the lane or its row takes no part
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xF, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xF, true);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_scan64(double v) {
    v += dpp64<0x111, 0xF>(v);   // row_shr 1, 2, 4, 8
    v += dpp64<0x112, 0xF>(v);
    v += dpp64<0x114, 0xF>(v);
    v += dpp64<0x118, 0xF>(v);
    v += dpp64<0x142, 0xA>(v);   // row_bcast 15
    return v + dpp64<0x143, 0xC>(v);   // row_bcast 31
}
__device__ __forceinline__ double lane64(double v, int lane) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

template <int Q>
__global__ __launch_bounds__(VT) void verify_draw(VerifyArgs a, Work w) {
    __shared__ double sr[WAVES], sp[WAVES], part[Q][WAVES];
    __shared__ int next;
    const int slice = blockIdx.x % w.slices, b = blockIdx.x / w.slices;
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    Decision v = decide<false>(a, w, b);
    const double u = (double)a.uniforms[(int64_t)b * (a.drafts + 1) + a.drafts];
    const float* target = target_row(a, b, v.accepted);
    const float* draft = v.has_q ? draft_row(a, b, v.accepted) : target;
    const Residual e(v, a);
    float x[Q][QUAD], y[Q][QUAD];
    auto token = [&](int s, int j, int k) { return (s * Q + j) * (VT * QUAD) + (int)threadIdx.x * QUAD + k; };
    load_slice<Q>(target, slice, a.vocab, x);
    load_slice<Q>(draft, slice, a.vocab, y);
    double r = 0.0, s = 0.0;
#pragma unroll
    for (int j = 0; j < Q; j++)
#pragma unroll
        for (int k = 0; k < QUAD; k++) {
            double p;
            r += e.of(x[j][k], y[j][k], token(slice, j, k), p);
            s += p;
        }
    r = wave_sum64(r);
    s = wave_sum64(s);
    if (lane == 0) { sr[wave] = r; sp[wave] = s; }
    __syncthreads();
    SliceMass* m = w.mass + (int64_t)b * w.slices;
    if (threadIdx.x == 0) {
        for (int k = 1; k < WAVES; k++) { r += sr[k]; s += sp[k]; }
        store_through(m + slice, SliceMass{r, s});
    }
    if (!last_of(w.drawn + b * COUNTER_STRIDE, (uint32_t)w.slices)) return;

    // every wavefront adds the slices up for itself, a lane a slice
    auto slice_of = [&](int k0) {
        return k0 + lane < w.slices ? load_past(m + k0 + lane) : SliceMass{0.0, 0.0};
    };
    double total = 0.0, total_p = 0.0;
    SliceMass mine{0.0, 0.0};
    for (int k0 = 0; k0 < w.slices; k0 += 64) {
        mine = slice_of(k0);
        total += wave_sum64(mine.r);
        total_p += wave_sum64(mine.p);
    }
    const bool of_p = !(total > 0.0);   // nothing left over: the target's own distribution
    if (of_p) {
        total = total_p;
        v.has_q = 0;
        v.one = -1;
    }
    if (!(total > 0.0)) {
        write_tokens(a, b, v.accepted, -1);
        return;
    }
    const double want = u * total;
    // the piece (of those that the lanes hold, `cum` before them) that holds the
    // draw, else the last with any mass: a draw past the last border by rounding
    double cum = 0.0, before = 0.0;
    int at = -1;
    auto search = [&](double x1, int k0) {
        const double upto = cum + wave_scan64(x1);
        const uint64_t over = __ballot(x1 > 0.0 && upto > want), any = __ballot(x1 > 0.0);
        if (any) {
            const int k = over ? __ffsll((unsigned long long)over) - 1 : 63 - __clzll((long long)any);
            at = k0 + k;
            before = lane64(upto - x1, __builtin_amdgcn_readfirstlane(k));
        }
        cum = lane64(upto, 63);
        return over != 0;
    };
    for (int k0 = 0; k0 < w.slices; k0 += 64) {
        if (w.slices > 64) mine = slice_of(k0);
        if (search(of_p ? mine.p : mine.r, k0)) break;
    }
    const int chosen = at;
    const Residual e2(v, a);
    load_slice<Q>(target, chosen, a.vocab, x);
    load_slice<Q>(draft, chosen, a.vocab, y);
    // sums of the slice's pieces: a quad of each of a wavefront's lanes
#pragma unroll
    for (int j = 0; j < Q; j++) {
        double sum = 0.0, p;
#pragma unroll
        for (int k = 0; k < QUAD; k++) sum += e2.of(x[j][k], y[j][k], token(chosen, j, k), p);
        sum = wave_sum64(sum);
        if (lane == 0) part[j][wave] = sum;
    }
    if (threadIdx.x == 0) next = -1;
    __syncthreads();
    cum = before;
    search(lane < Q * WAVES ? part[lane / WAVES][lane % WAVES] : 0.0, 0);
    if (at % WAVES == wave) {   // one wavefront looks through the piece
        const int piece = at / WAVES, t0 = token(chosen, piece, 0);
        double r1[QUAD], sum = 0.0, p;
#pragma unroll
        for (int k = 0; k < QUAD; k++) {
            float xk = x[0][k], yk = y[0][k];
#pragma unroll
            for (int j = 1; j < Q; j++) { xk = piece == j ? x[j][k] : xk; yk = piece == j ? y[j][k] : yk; }
            r1[k] = e2.of(xk, yk, t0 + k, p);
            sum += r1[k];
        }
        cum = before;
        search(sum, 0);
        if (lane == at) {
            int found = -1;
            bool over = false;
#pragma unroll
            for (int k = 0; k < QUAD; k++) {
                before += r1[k];
                if (r1[k] > 0.0 && !over) {
                    found = t0 + k;
                    over = before > want;
                }
            }
            next = found;
        }
    }
    __syncthreads();
    write_tokens(a, b, v.accepted, next);
}

// Logits of a slice: small ones where there are few slices to a row anyway (one
// sequence, vocabulary 32000: 10.4 us, 15.6 in slices of 4096), else large ones,
// whose statistics every workgroup reads again (16 of 128256: 32.5, 49 of 1024).
int quads_of(int vocab) { return vocab <= 32768 ? 1 : 4; }

size_t layout(int batch, int drafts, int vocab, bool draft, uint8_t* base, Work* w) {
    const int slice = VT * QUAD * quads_of(vocab);
    w->slices = (vocab + slice - 1) / slice;
    w->rows = drafts + 1 + (draft ? drafts : 0);
    size_t at = 0;
    auto take = [&](size_t n) {
        uint8_t* p = base + at;
        at += (n + 15) & ~(size_t)15;
        return p;
    };
    w->drawn = reinterpret_cast<uint32_t*>(take(COUNTER_BYTES));
    w->picked = reinterpret_cast<float*>(take(sizeof(float) * (size_t)batch * w->rows));
    w->mass = reinterpret_cast<SliceMass*>(take(sizeof(SliceMass) * (size_t)batch * w->slices));
    w->stats = reinterpret_cast<SliceStats*>(take(sizeof(SliceStats) * (size_t)batch * w->rows * w->slices));
    return at;
}

template <int Q>
void launch_sized(const VerifyArgs& a, const Work& w, hipStream_t s) {
    const dim3 slices((uint32_t)w.slices * a.batch), rows(slices.x, w.rows);
    if (a.temperature <= 0.f) {
        verify_stats<true, Q><<<rows, VT, 0, s>>>(a, w);
        verify_greedy<<<dim3(a.batch), VT, 0, s>>>(a, w);
    } else {
        verify_stats<false, Q><<<rows, VT, 0, s>>>(a, w);
        verify_draw<Q><<<slices, VT, 0, s>>>(a, w);
    }
}

}  // namespace

size_t verify_workspace(int batch, int drafts, int vocab) {
    Work w;
    return layout(batch, drafts, vocab, true, nullptr, &w);
}

hipError_t launch_verify(VerifyArgs a, hipStream_t s) {
    Work w;
    a.rate = a.temperature > 0.f ? 1.4426950408889634074 / (double)a.temperature : 0.0;
    a.reach = a.temperature > 0.f ? 1000.0 / a.rate : 0.0;
    layout(a.batch, a.drafts, a.vocab, a.draft && a.temperature > 0.f, a.work, &w);
    if (quads_of(a.vocab) == 1) launch_sized<1>(a, w, s);
    else launch_sized<4>(a, w, s);
    return hipGetLastError();
}

}  // namespace llmdot
