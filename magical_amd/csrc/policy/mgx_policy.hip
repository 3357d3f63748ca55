// mgx_policy.hip -- the operators of include/mgx_policy.h: what lies between a policy's action scores and the engine's actions.
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <type_traits>

#include "../../../include/mgx_policy.h"

namespace {

constexpr float NEG_INF = -__builtin_inff();

// The rows of scores a call works on; an action that is not open reads as -inf.
template <typename T> struct Scores {
    const T *x;
    const uint8_t *mask;
    int64_t rows, n, stride, mask_stride;
    float inv_t;        // 1 / temperature
    double inv_t64;
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__hip_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half(v); }
template <> __device__ __forceinline__ __hip_bfloat16 from_f32<__hip_bfloat16>(float v) { return __float2bfloat16(v); }

template <typename T> struct Row {
    const T *x;
    const uint8_t *mask;
    __device__ Row(const Scores<T> &s, int64_t r) : x(s.x + r * s.stride), mask(s.mask ? s.mask + r * s.mask_stride : nullptr) {}
    __device__ __forceinline__ float at(int64_t j) const {
        const float v = to_f32(x[j]);
        return mask && !mask[j] ? NEG_INF : v;
    }
};

struct Actions {
    const void *p;
    int bytes;
    __device__ __forceinline__ int64_t at(int64_t r) const { return bytes == 8 ? ((const int64_t *)p)[r] : ((const int32_t *)p)[r]; }
};

constexpr int BLOCK = 256, WAVES = BLOCK / 64;

template <typename V, typename F> __device__ __forceinline__ V wave_all(V v, F f) {
    for (int o = 1; o < 64; o <<= 1) v = f(v, __shfl_xor(v, o));
    return v;
}
template <typename V, typename F> __device__ __forceinline__ V block_all(V v, V *lds, F f) {
    v = wave_all(v, f);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
    for (int w = 1; w < WAVES; w++) v = f(v, lds[w]);
    return v;
}

// is (v, i) a better alternative than (w, k)?  Higher score first, then the lower index.
__device__ __forceinline__ bool better(float v, int i, float w, int k) { return v > w || (v == w && i < k); }

// e^d for d <= 0 in 64 bits: d = k log 2 + r with |r| <= log 2 / 2 (log 2 in two parts, so that r is exact to 2^-53), Taylor's series to
// the 13th power (the next term is below 2^-57), times 2^k.  NaN stays NaN, -inf gives 0.
__device__ __forceinline__ double exp64(double d) {
    const double k = rint(d * 1.4426950408889634);
    double r = fma(k, -0x1.62e42fefa3800p-1, d);
    r = fma(k, -0x1.ef35793c76730p-45, r);
    double p = 1.0 / 6227020800.0;
    p = fma(p, r, 1.0 / 479001600.0);
    p = fma(p, r, 1.0 / 39916800.0);
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return d < -800.0 ? 0.0 : ldexp(p, (int)k);
}

// ---------------------------------------------------------------------------------------------------------------- short rows
// A row of up to 2048 scores stays in the registers of G lanes (4 ... 64, so that several rows share a wavefront), E a lane: one read of the
// scores, all sums by lane exchanges, no LDS, no barrier.

template <typename V, typename F> __device__ __forceinline__ V group_all(V v, int G, F f) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1)
        if (o < G) v = f(v, __shfl_xor(v, o));
    return v;
}
__device__ __forceinline__ float f_max(float a, float b) { return fmaxf(a, b); }

// W consecutive scores from j on, in one load where they are all there (gfx950 loads any alignment)
template <int W, typename T> __device__ __forceinline__ void load(const Row<T> &row, int j, int n, float (&x)[W]) {
    if (j + W <= n) {
        T v[W];
        __builtin_memcpy(v, row.x + j, sizeof v);
#pragma unroll
        for (int k = 0; k < W; k++) x[k] = to_f32(v[k]);
        if (row.mask) {
            uint8_t b[W];
            __builtin_memcpy(b, row.mask + j, W);
#pragma unroll
            for (int k = 0; k < W; k++) x[k] = b[k] ? x[k] : NEG_INF;
        }
    } else {
#pragma unroll
        for (int k = 0; k < W; k++) x[k] = j + k < n ? row.at(j + k) : NEG_INF;
    }
}

// lane g of a row's G lanes holds W-wide pieces: x[e] is score place(g, e)
template <int G, int E> struct Spread {
    static constexpr int W = E % 4 == 0 && G == 64 ? 4 : 1;
    static __device__ __forceinline__ int place(int g, int e) { return e / W * (G * W) + g * W + e % W; }
    template <typename T> static __device__ __forceinline__ void load_row(const Row<T> &row, int g, int n, float (&x)[E]) {
#pragma unroll
        for (int e = 0; e < E; e += W) {
            float v[W];
            load<W>(row, place(g, e), n, v);
#pragma unroll
            for (int k = 0; k < W; k++) x[e + k] = v[k];
        }
    }
};

template <typename T, int G, int E>
__global__ __launch_bounds__(BLOCK) void k_log_probs_short(Scores<T> sc, Actions actions, int top, float *log_prob, float *entropy,
                                                           float *top_log_probs, int32_t *top_actions) {
    using S = Spread<G, E>;
    const int g = threadIdx.x % G, n = (int)sc.n;
    for (int64_t r = (int64_t)blockIdx.x * (BLOCK / G) + threadIdx.x / G; r < sc.rows; r += (int64_t)gridDim.x * (BLOCK / G)) {
        const Row<T> row(sc, r);
        float x[E];
        S::load_row(row, g, n, x);
        float m = x[0];
#pragma unroll
        for (int e = 1; e < E; e++) m = fmaxf(m, x[e]);
        m = group_all(m, G, f_max);
        const bool some = m > NEG_INF;
        const float ref = some ? m : 0.0f;
        float s = 0, t = 0;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const float d = (x[e] - ref) * sc.inv_t, p = expf(d);
            s += p;
            t += p * fmaxf(d, -1e30f);          // (not open: 0 x a finite number)
        }
        s = group_all(s, G, [](float a, float b) { return a + b; });
        t = group_all(t, G, [](float a, float b) { return a + b; });
        const bool undefined = !(s == s);
        const float log_s = logf(s), nan = __builtin_nanf("");
        if (g == 0) {
            const int64_t a = actions.at(r);
            float lp = 0.0f;
            if (a >= n || (a >= 0 && undefined)) lp = nan;
            else if (a >= 0) lp = some ? (row.at(a) - ref) * sc.inv_t - log_s : NEG_INF;
            log_prob[r] = lp;
            entropy[r] = undefined ? nan : some ? log_s - t / s : 0.0f;
        }
        // the best alternatives, one after the other: every lane's best of what is left, then the group's
        for (int k = 0; k < top; k++) {
            float v = NEG_INF;
            int i = 0x7fffffff;
#pragma unroll
            for (int e = 0; e < E; e++) {
                const bool b = x[e] > v;          // (a lane's places ascend: of equal scores the first)
                v = b ? x[e] : v;
                i = b ? S::place(g, e) : i;
            }
#pragma unroll
            for (int o = 1; o < G; o <<= 1) {
                const float ov = __shfl_xor(v, o);
                const int oi = __shfl_xor(i, o);
                const bool b = better(ov, oi, v, i);
                v = b ? ov : v;
                i = b ? oi : i;
            }
#pragma unroll
            for (int e = 0; e < E; e++) x[e] = S::place(g, e) == i ? NEG_INF : x[e];
            if (g == 0) {
                const bool there = v > NEG_INF && !undefined;
                top_actions[r * top + k] = there ? i : -1;
                top_log_probs[r * top + k] = there ? (v - ref) * sc.inv_t - log_s : NEG_INF;
            }
        }
    }
}

template <typename T, int G, int E>
__global__ __launch_bounds__(BLOCK) void k_backward_short(Scores<T> sc, Actions actions, const float *entropy, const float *g_lp,
                                                          int64_t g_lp_stride, const float *g_h, int64_t g_h_stride, T *grad) {
    using S = Spread<G, E>;
    const int g = threadIdx.x % G, n = (int)sc.n;
    for (int64_t r = (int64_t)blockIdx.x * (BLOCK / G) + threadIdx.x / G; r < sc.rows; r += (int64_t)gridDim.x * (BLOCK / G)) {
        const Row<T> row(sc, r);
        float x[E];
        S::load_row(row, g, n, x);
        const int64_t a = actions.at(r);
        const float h = entropy[r];
        const float gl = g_lp && a >= 0 ? g_lp[r * g_lp_stride] : 0.0f, gh = g_h ? g_h[r * g_h_stride] : 0.0f;
        // maximum and sum again (cheaper than 8 bytes a row written and read)
        float m = x[0];
#pragma unroll
        for (int e = 1; e < E; e++) m = fmaxf(m, x[e]);
        m = group_all(m, G, f_max);
        const float ref = m > NEG_INF ? m : 0.0f;
        float s = 0;
        float p[E];
#pragma unroll
        for (int e = 0; e < E; e++) {
            p[e] = expf((x[e] - ref) * sc.inv_t);
            s += p[e];
        }
        s = group_all(s, G, [](float a, float b) { return a + b; });
        const float inv_s = 1.0f / s, log_s = logf(s);
        T out[E];
#pragma unroll
        for (int e = 0; e < E; e++) {
            const float lp = (x[e] - ref) * sc.inv_t - log_s;
            float v = -(p[e] * inv_s) * (gl + gh * (fmaxf(lp, -1e30f) + h));
            if (S::place(g, e) == a) v += gl;
            out[e] = from_f32<T>(x[e] == NEG_INF ? 0.0f : v * sc.inv_t);
        }
        T *to = grad + r * sc.n;
#pragma unroll
        for (int e = 0; e < E; e += S::W) {
            const int j = S::place(g, e);
            if (j + S::W <= n) __builtin_memcpy(to + j, out + e, S::W * sizeof(T));
            else
#pragma unroll
                for (int k = 0; k < S::W; k++)
                    if (j + k < n) to[j + k] = out[e + k];
        }
    }
}

__device__ __forceinline__ double uniform_at(const void *uniforms, int bytes, int64_t r) {
    const double u = bytes == 8 ? ((const double *)uniforms)[r] : (double)((const float *)uniforms)[r];
    return u > 0.0 ? (u < 1.0 ? u : 1.0) : 0.0;          // (NaN: 0)
}

// Lane g holds the E consecutive scores from g * E on: a running sum in index order is a lane's sum, a scan over the lanes, and a second
// look at the one lane in which the target lies.
template <typename T, int G, int E>
__global__ __launch_bounds__(BLOCK) void k_sample_short(Scores<T> sc, const void *uniforms, int uniform_bytes, int32_t *action,
                                                        float *log_prob, float *entropy) {
    constexpr int W = E % 8 == 0 ? 8 : E % 4 == 0 ? 4 : 1;
    const int g = threadIdx.x % G, n = (int)sc.n;
    for (int64_t r = (int64_t)blockIdx.x * (BLOCK / G) + threadIdx.x / G; r < sc.rows; r += (int64_t)gridDim.x * (BLOCK / G)) {
        const Row<T> row(sc, r);
        float x[E];
#pragma unroll
        for (int e = 0; e < E; e += W) {
            float v[W];
            load<W>(row, g * E + e, n, v);
#pragma unroll
            for (int k = 0; k < W; k++) x[e + k] = v[k];
        }
        float m = x[0];
#pragma unroll
        for (int e = 1; e < E; e++) m = fmaxf(m, x[e]);
        m = group_all(m, G, f_max);
        const bool some = m > NEG_INF;
        const double ref = some ? m : 0.0;
        double p[E], s = 0, t = 0;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const double d = ((double)x[e] - ref) * sc.inv_t64;
            p[e] = exp64(d);
            s += p[e];
            t = fma(p[e], fmax(d, -1e300), t);
        }
        double upto = s;          // the lanes' running sum, this one's included
#pragma unroll
        for (int o = 1; o < G; o <<= 1) {
            const double v = __shfl_up(upto, o, G);
            if (g >= o) upto += v;
        }
        const double total = __shfl(upto, G - 1, G);
        t = group_all(t, G, [](double a, double b) { return a + b; });
        const bool undefined = !(total == total), none = undefined || !some;
        const double target = uniform_at(uniforms, uniform_bytes, r) * total;
        // the first lane that passes the target, or else (rounding; a number of 1) the last one with anything in it
        const int first_lane = (threadIdx.x & 63) - g;
        const uint64_t in_group = G == 64 ? ~0ull : ((1ull << (G & 63)) - 1) << first_lane;
        const uint64_t past = __ballot(s > 0.0 && upto > target) & in_group, any = __ballot(s > 0.0) & in_group;
        const int owner = none ? first_lane : past ? __ffsll((unsigned long long)past) - 1 : 63 - __clzll((long long)any);
        if ((threadIdx.x & 63) == owner) {
            double c = upto - s;
            c = g == 0 ? 0.0 : c;
            int a = -1;
            bool found = false;
#pragma unroll
            for (int e = 0; e < E; e++) {
                c += p[e];
                if (p[e] > 0.0 && !found) { a = g * E + e; found = c > target; }
            }
            action[r] = none ? -1 : a;
            if (log_prob) log_prob[r] = undefined ? __builtin_nanf("") : some ? (float)(((double)row.at(a) - ref) * sc.inv_t64 - log(total)) : NEG_INF;
            if (entropy) entropy[r] = undefined ? __builtin_nanf("") : some ? (float)(log(total) - t / total) : 0.0f;
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------- rows of any length
template <typename T>
__global__ __launch_bounds__(BLOCK) void k_log_probs(Scores<T> sc, Actions actions, int top, float *log_prob, float *entropy, float *stats,
                                                     float *top_log_probs, int32_t *top_actions) {
    __shared__ float lds[WAVES], lds_v[WAVES];
    __shared__ int lds_i[WAVES];
    for (int64_t r = blockIdx.x; r < sc.rows; r += gridDim.x) {
    const Row<T> row(sc, r);
    const int n = (int)sc.n;
    float m = NEG_INF;
    for (int j = threadIdx.x; j < n; j += BLOCK) m = fmaxf(m, row.at(j));
    m = block_all(m, lds, [](float a, float b) { return fmaxf(a, b); });
    const bool some = m > NEG_INF;
    const float ref = some ? m : 0.0f;
    float s = 0, t = 0;
    for (int j = threadIdx.x; j < n; j += BLOCK) {
        const float x = row.at(j), d = (x - ref) * sc.inv_t, e = expf(d);
        s += e;
        t += e * fmaxf(d, -1e30f);          // (not open: 0 x a finite number)
    }
    s = block_all(s, lds, [](float a, float b) { return a + b; });
    t = block_all(t, lds, [](float a, float b) { return a + b; });
    const bool undefined = !(s == s);
    const float log_s = logf(s), nan = __builtin_nanf("");
    if (threadIdx.x == 0) {
        const int64_t a = actions.at(r);
        float lp = 0.0f;
        if (a >= n || (a >= 0 && undefined)) lp = nan;
        else if (a >= 0) lp = some ? (row.at(a) - ref) * sc.inv_t - log_s : NEG_INF;
        log_prob[r] = lp;
        entropy[r] = undefined ? nan : some ? log_s - t / s : 0.0f;
        if (stats) { stats[2 * r] = ref; stats[2 * r + 1] = log_s; }
    }
    // the best alternatives, one after the other: the best one behind the last one found
    float pv = -NEG_INF;
    int pi = -1;
    for (int k = 0; k < top; k++) {
        float v = NEG_INF;
        int i = 0x7fffffff;
        if (!undefined)
            for (int j = threadIdx.x; j < n; j += BLOCK) {
                const float x = row.at(j);
                if (better(pv, pi, x, j) && better(x, j, v, i)) { v = x; i = j; }
            }
        for (int o = 1; o < 64; o <<= 1) {
            const float ov = __shfl_xor(v, o);
            const int oi = __shfl_xor(i, o);
            if (better(ov, oi, v, i)) { v = ov; i = oi; }
        }
        __syncthreads();
        if ((threadIdx.x & 63) == 0) { lds_v[threadIdx.x >> 6] = v; lds_i[threadIdx.x >> 6] = i; }
        __syncthreads();
        for (int w = 0; w < WAVES; w++)
            if (better(lds_v[w], lds_i[w], v, i)) { v = lds_v[w]; i = lds_i[w]; }
        if (threadIdx.x == 0) {
            top_actions[r * top + k] = v > NEG_INF ? i : -1;
            top_log_probs[r * top + k] = v > NEG_INF ? (v - ref) * sc.inv_t - log_s : NEG_INF;
        }
        pv = v; pi = i;
    }
    __syncthreads();
    }
}

template <typename T>
__global__ __launch_bounds__(BLOCK) void k_log_probs_backward(Scores<T> sc, Actions actions, const float *stats, const float *entropy,
                                                              const float *g_lp, int64_t g_lp_stride, const float *g_h, int64_t g_h_stride,
                                                              T *grad) {
    for (int64_t r = blockIdx.x; r < sc.rows; r += gridDim.x) {
    const Row<T> row(sc, r);
    const int n = (int)sc.n;
    const int64_t a = actions.at(r);
    const float ref = stats[2 * r], log_s = stats[2 * r + 1], h = entropy[r];
    const float gl = g_lp && a >= 0 ? g_lp[r * g_lp_stride] : 0.0f, gh = g_h ? g_h[r * g_h_stride] : 0.0f;
    for (int j = threadIdx.x; j < n; j += BLOCK) {
        const float x = row.at(j), lp = (x - ref) * sc.inv_t - log_s, p = expf(lp);
        float g = -p * (gl + gh * (fmaxf(lp, -1e30f) + h));
        if (j == a) g += gl;
        grad[r * sc.n + j] = from_f32<T>(x > NEG_INF || x != x ? g * sc.inv_t : 0.0f);
    }
    }
}

template <typename T>
__global__ __launch_bounds__(BLOCK) void k_sample(Scores<T> sc, const void *uniforms, int uniform_bytes, int32_t *action, float *log_prob,
                                                  float *entropy) {
    __shared__ float lds[WAVES];
    __shared__ double lds64[WAVES];
    __shared__ int found, lds_last[WAVES];
    for (int64_t r = blockIdx.x; r < sc.rows; r += gridDim.x) {
    const Row<T> row(sc, r);
    const int n = (int)sc.n, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float m = NEG_INF;
    for (int j = threadIdx.x; j < n; j += BLOCK) m = fmaxf(m, row.at(j));
    m = block_all(m, lds, [](float a, float b) { return fmaxf(a, b); });
    const bool some = m > NEG_INF;
    const double ref = some ? m : 0.0;
    double s = 0, t = 0;
    for (int j = threadIdx.x; j < n; j += BLOCK) {
        const double d = ((double)row.at(j) - ref) * sc.inv_t64, e = exp(d);
        s += e;
        t += e * fmax(d, -1e300);
    }
    s = block_all(s, lds64, [](double a, double b) { return a + b; });
    t = block_all(t, lds64, [](double a, double b) { return a + b; });
    const bool undefined = !(s == s);
    double u = uniform_bytes == 8 ? ((const double *)uniforms)[r] : (double)((const float *)uniforms)[r];
    u = u > 0.0 ? (u < 1.0 ? u : 1.0) : 0.0;
    const double target = u * s;
    // running sums in index order, BLOCK actions at a time; the last action with e > 0 stands in where rounding leaves none above the target
    if (threadIdx.x == 0) found = 0x7fffffff;
    __syncthreads();
    double before = 0;
    int last = -1;
    for (int j0 = 0; j0 < n; j0 += BLOCK) {
        const int j = j0 + threadIdx.x;
        const double e = j < n ? exp(((double)row.at(j) - ref) * sc.inv_t64) : 0.0;
        double c = e;
        for (int o = 1; o < 64; o <<= 1) {
            const double v = __shfl_up(c, o);
            if (lane >= o) c += v;
        }
        __syncthreads();
        if (lane == 63) lds64[wave] = c;
        __syncthreads();
        double base = before;
        for (int w = 0; w < wave; w++) base += lds64[w];
        for (int w = 0; w < WAVES; w++) before += lds64[w];
        if (e > 0.0) last = j;
        if (e > 0.0 && base + c > target) atomicMin(&found, j);
        __syncthreads();
        if (found != 0x7fffffff) break;
    }
    for (int o = 1; o < 64; o <<= 1) last = max(last, __shfl_xor(last, o));
    if (lane == 0) lds_last[wave] = last;
    __syncthreads();
    for (int w = 0; w < WAVES; w++) last = max(last, lds_last[w]);
    if (threadIdx.x == 0) {
        const int a = found != 0x7fffffff ? found : last;
        const bool none = undefined || !some;
        const double log_s = log(s);
        action[r] = none ? -1 : a;
        if (log_prob) log_prob[r] = undefined ? __builtin_nanf("") : some ? (float)(((double)row.at(a) - ref) * sc.inv_t64 - log_s) : NEG_INF;
        if (entropy) entropy[r] = undefined ? __builtin_nanf("") : some ? (float)(log_s - t / s) : 0.0f;
    }
    __syncthreads();
    }
}

thread_local char g_err[256] = "";          // (no allocation: nothing may throw across the C boundary)
int fail(int code, const char *msg) { snprintf(g_err, sizeof g_err, "%s", msg); return code; }

// the caller's current device is left as it was
struct DeviceGuard {
    int prev = -1;
    bool ok = true;
    explicit DeviceGuard(int device) {
        if (hipGetDevice(&prev) != hipSuccess) prev = -1;
        if (prev != device) ok = hipSetDevice(device) == hipSuccess;
    }
    ~DeviceGuard() { if (prev >= 0) (void)hipSetDevice(prev); }
};

int check_scores(int dtype, const void *logits, int64_t rows, int64_t n, int64_t row_stride, const uint8_t *mask, int64_t mask_row_stride,
                 double temperature) {
    if (dtype < MGX_REAL_F32 || dtype > MGX_REAL_BF16) return fail(MGX_ERR_ARG, "bad dtype");
    if (rows < 0 || rows > 0x7fffffff || n < 1 || n > (1 << 30)) return fail(MGX_ERR_ARG, "rows: 0 ... 2^31 - 1, n: 1 ... 2^30");
    if (row_stride < 0 || (mask && mask_row_stride < 0)) return fail(MGX_ERR_ARG, "negative row stride");
    if (rows && !logits) return fail(MGX_ERR_ARG, "logits is NULL");
    if (!(temperature > 0) || !std::isfinite(temperature) || !std::isfinite((float)(1.0 / temperature)) || !((float)(1.0 / temperature) > 0))
        return fail(MGX_ERR_ARG, "temperature must be positive and finite");
    return MGX_OK;
}

template <typename T>
Scores<T> scores(const void *logits, int64_t rows, int64_t n, int64_t row_stride, const uint8_t *mask, int64_t mask_row_stride, double temperature) {
    return {(const T *)logits, mask, rows, n, row_stride, mask_row_stride, (float)(1.0 / temperature), 1.0 / temperature};
}

// one workgroup per row, as many as a grid of 2^32 work items takes
template <typename... P, typename... A> int launch(void (*kernel)(P...), int64_t blocks, int threads, void *stream, A... args) {
    const int64_t most = 0xffffffffLL / threads;
    void *ptrs[] = {(void *)&args...};
    static_assert(sizeof...(P) == sizeof...(A) && (std::is_same_v<P, A> && ...), "argument types are the kernel's");
    const hipError_t err = hipLaunchKernel((const void *)kernel, dim3((unsigned)(blocks < most ? blocks : most)), dim3(threads), ptrs, 0,
                                           (hipStream_t)stream);
    return err == hipSuccess ? (int)MGX_OK : fail(MGX_ERR_HIP, hipGetErrorString(err));
}

constexpr int SHORT_MAX = 2048;
template <int G_, int E_> struct Shape { static constexpr int G = G_, E = E_; };
// f(lanes a row and scores a lane) for rows of n <= SHORT_MAX: the fewest lanes that keep 4 ... 8 scores each, then a whole wavefront
template <typename F> int by_length(int64_t n, F f) {
    if (n <= 32)
        switch ((n + 3) / 4) {
            case 1: return f(Shape<4, 1>());
            case 2: return f(Shape<4, 2>());
            case 3: return f(Shape<4, 3>());
            case 4: return f(Shape<4, 4>());
            case 5: return f(Shape<4, 5>());
            case 6: return f(Shape<4, 6>());
            case 7: return f(Shape<4, 7>());
            default: return f(Shape<4, 8>());
        }
    if (n <= 48) return f(Shape<8, 6>());
    if (n <= 64) return f(Shape<8, 8>());
    if (n <= 96) return f(Shape<16, 6>());
    if (n <= 128) return f(Shape<16, 8>());
    if (n <= 192) return f(Shape<32, 6>());
    if (n <= 256) return f(Shape<32, 8>());
    if (n <= 384) return f(Shape<64, 6>());
    if (n <= 512) return f(Shape<64, 8>());
    if (n <= 768) return f(Shape<64, 12>());
    if (n <= 1024) return f(Shape<64, 16>());
    if (n <= 1536) return f(Shape<64, 24>());
    return f(Shape<64, 32>());
}
int64_t short_blocks(int64_t rows, int G) { return (rows * G + BLOCK - 1) / BLOCK; }

// f(a value of the scores' element type)
template <typename F> int by_dtype(int dtype, F f) {
    switch (dtype) {
        case MGX_REAL_F32: return f(float());
        case MGX_REAL_F16: return f(__half());
        default: return f(__hip_bfloat16());
    }
}

}  // namespace

extern "C" {

const char *mgx_policy_last_error(void) { return g_err; }

int64_t mgx_policy_workspace_bytes(int, int, int64_t, int64_t, int) { return 0; }

int64_t mgx_policy_stats_bytes(int64_t rows, int64_t n) { return n > SHORT_MAX ? rows * 8 : 0; }

int mgx_policy_log_probs(int device, int dtype, const void *logits, int64_t rows, int64_t n, int64_t row_stride, const uint8_t *mask,
                         int64_t mask_row_stride, double temperature, const void *actions, int action_bytes, int top, float *log_prob,
                         float *entropy, float *stats, float *top_log_probs, int32_t *top_actions, void *workspace,
                         int64_t workspace_bytes, void *stream) {
    if (int rc = check_scores(dtype, logits, rows, n, row_stride, mask, mask_row_stride, temperature)) return rc;
    if (action_bytes != 4 && action_bytes != 8) return fail(MGX_ERR_ARG, "action_bytes: 4 or 8");
    if (top < 0 || top > MGX_POLICY_MAX_TOP || top > n) return fail(MGX_ERR_ARG, "top: 0 ... min(n, 64)");
    if (rows == 0) return MGX_OK;
    if (!actions || !log_prob || !entropy || (top && (!top_log_probs || !top_actions))) return fail(MGX_ERR_ARG, "NULL argument");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(MGX_ERR_HIP, "hipSetDevice failed");
    return by_dtype(dtype, [&](auto v) {
        using T = decltype(v);
        const Scores<T> sc = scores<T>(logits, rows, n, row_stride, mask, mask_row_stride, temperature);
        if (n <= SHORT_MAX)
            return by_length(n, [&](auto shape) {
                constexpr int G = decltype(shape)::G, E = decltype(shape)::E;
                return launch(k_log_probs_short<T, G, E>, short_blocks(rows, G), BLOCK, stream, sc, Actions{actions, action_bytes}, top,
                              log_prob, entropy, top_log_probs, top_actions);
            });
        return launch(k_log_probs<T>, rows, BLOCK, stream, sc, Actions{actions, action_bytes}, top, log_prob, entropy, stats, top_log_probs,
                      top_actions);
    });
}

int mgx_policy_log_probs_backward(int device, int dtype, const void *logits, int64_t rows, int64_t n, int64_t row_stride,
                                  const uint8_t *mask, int64_t mask_row_stride, double temperature, const void *actions,
                                  int action_bytes, const float *stats, const float *entropy, const float *grad_log_prob,
                                  int64_t grad_log_prob_stride, const float *grad_entropy, int64_t grad_entropy_stride, void *grad,
                                  void *stream) {
    if (int rc = check_scores(dtype, logits, rows, n, row_stride, mask, mask_row_stride, temperature)) return rc;
    if (action_bytes != 4 && action_bytes != 8) return fail(MGX_ERR_ARG, "action_bytes: 4 or 8");
    if (grad_log_prob_stride < 0 || grad_entropy_stride < 0) return fail(MGX_ERR_ARG, "negative stride");
    if (rows == 0) return MGX_OK;
    if (!actions || (!stats && mgx_policy_stats_bytes(rows, n)) || !entropy || !grad) return fail(MGX_ERR_ARG, "NULL argument");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(MGX_ERR_HIP, "hipSetDevice failed");
    return by_dtype(dtype, [&](auto v) {
        using T = decltype(v);
        const Scores<T> sc = scores<T>(logits, rows, n, row_stride, mask, mask_row_stride, temperature);
        if (n <= SHORT_MAX)
            return by_length(n, [&](auto shape) {
                constexpr int G = decltype(shape)::G, E = decltype(shape)::E;
                return launch(k_backward_short<T, G, E>, short_blocks(rows, G), BLOCK, stream, sc, Actions{actions, action_bytes}, entropy,
                              grad_log_prob, grad_log_prob_stride, grad_entropy, grad_entropy_stride, (T *)grad);
            });
        return launch(k_log_probs_backward<T>, rows, BLOCK, stream, sc, Actions{actions, action_bytes}, stats, entropy, grad_log_prob,
                      grad_log_prob_stride, grad_entropy, grad_entropy_stride, (T *)grad);
    });
}

int mgx_policy_sample(int device, int dtype, const void *logits, int64_t rows, int64_t n, int64_t row_stride, const uint8_t *mask,
                      int64_t mask_row_stride, double temperature, const void *uniforms, int uniform_bytes, int32_t *action,
                      float *log_prob, float *entropy, void *workspace, int64_t workspace_bytes, void *stream) {
    if (int rc = check_scores(dtype, logits, rows, n, row_stride, mask, mask_row_stride, temperature)) return rc;
    if (uniform_bytes != 4 && uniform_bytes != 8) return fail(MGX_ERR_ARG, "uniform_bytes: 4 or 8");
    if (rows == 0) return MGX_OK;
    if (!uniforms || !action) return fail(MGX_ERR_ARG, "NULL argument");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(MGX_ERR_HIP, "hipSetDevice failed");
    return by_dtype(dtype, [&](auto v) {
        using T = decltype(v);
        const Scores<T> sc = scores<T>(logits, rows, n, row_stride, mask, mask_row_stride, temperature);
        if (n <= SHORT_MAX)
            return by_length(n, [&](auto shape) {
                constexpr int G = decltype(shape)::G, E = decltype(shape)::E;
                return launch(k_sample_short<T, G, E>, short_blocks(rows, G), BLOCK, stream, sc, uniforms, uniform_bytes, action, log_prob,
                              entropy);
            });
        return launch(k_sample<T>, rows, BLOCK, stream, sc, uniforms, uniform_bytes, action, log_prob, entropy);
    });
}

}  // extern "C"
