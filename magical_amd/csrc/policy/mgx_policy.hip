// mgx_policy.hip -- the operators of include/mgx_policy.h: what lies between a policy's action scores and the engine's actions.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
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
    float inv_t, inv_t2;        // 1 / temperature, log2(e) / temperature: exponentials are taken to the base 2, as the hardware does
    double inv_t2_64;
};

using half = _Float16;
using bf16 = __bf16;
template <typename T> __device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f32(float v) { return (T)v; }          // to nearest, ties to even

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
// is (v, i) a better alternative than (w, k)?  Higher score first, then the lower index.
__device__ __forceinline__ bool better(float v, int i, float w, int k) { return v > w || (v == w && i < k); }

// 2^y for y <= 0 in 64 bits: y = k + f with |f| <= 1 / 2, a polynomial for 2^f (interpolated at the Chebyshev points of [-1/2, 1/2] in 60
// digits: off by 3.1e-16 at most), times 2^k.  Below -1100 (and for NaN, which the callers look for themselves) it is 0.
__device__ __forceinline__ double exp2_64(double y) {
    y = fmax(y, -1100.0);
    const double k = rint(y), f = y - k;
    double p = 0x1.e6063f7217bc6p-28;
    p = fma(p, f, 0x1.b675bca4eeebbp-24);
    p = fma(p, f, 0x1.62bfd47773353p-20);
    p = fma(p, f, 0x1.ffcb54062e698p-17);
    p = fma(p, f, 0x1.430913096fd9fp-13);
    p = fma(p, f, 0x1.5d87fe9d7a584p-10);
    p = fma(p, f, 0x1.3b2ab6fba1ddap-7);
    p = fma(p, f, 0x1.c6b08d703ce49p-5);
    p = fma(p, f, 0x1.ebfbdff82c598p-3);
    p = fma(p, f, 0x1.62e42fefa3a19p-1);
    p = fma(p, f, 1.0);
    return ldexp(p, (int)k);
}
constexpr double LOG2_E = 1.4426950408889634, LN_2 = 0.6931471805599453;

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
            const float d = (x[e] - ref) * sc.inv_t2, p = __builtin_amdgcn_exp2f(d);
            s += p;
            t = fmaf(p, fmaxf(d, -1e30f), t);          // (not open: 0 x a finite number)
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
            entropy[r] = undefined ? nan : some ? log_s - t / s * (float)LN_2 : 0.0f;
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
            p[e] = __builtin_amdgcn_exp2f((x[e] - ref) * sc.inv_t2);
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
        bool nan = false;
#pragma unroll
        for (int e = 0; e < E; e++) {
            nan |= x[e] != x[e];
            const double d = fmax(((double)x[e] - ref) * sc.inv_t2_64, -1100.0);
            p[e] = exp2_64(d);
            s += p[e];
            t = fma(p[e], d, t);
        }
        double upto = s;          // the lanes' running sum, this one's included
#pragma unroll
        for (int o = 1; o < G; o <<= 1) {
            const double v = __shfl_up(upto, o, G);
            if (g >= o) upto += v;
        }
        const double total = __shfl(upto, G - 1, G);
        t = group_all(t, G, [](double a, double b) { return a + b; });
        const int first_lane = (threadIdx.x & 63) - g;
        const uint64_t in_group = G == 64 ? ~0ull : ((1ull << (G & 63)) - 1) << first_lane;
        const bool undefined = (__ballot(nan) & in_group) || m == -NEG_INF, none = undefined || !some;
        const double target = uniform_at(uniforms, uniform_bytes, r) * total;
        // the first lane that passes the target, or else (rounding; a number of 1) the last one with anything in it
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
            if (log_prob)
                log_prob[r] = undefined ? __builtin_nanf("") : some ? (float)(((double)row.at(a) - ref) * sc.inv_t2_64 * LN_2 - log(total)) : NEG_INF;
            if (entropy) entropy[r] = undefined ? __builtin_nanf("") : some ? (float)(log(total) - t / total * LN_2) : 0.0f;
        }
    }
}

// ----------------------------------------------------------------------------------------------------------------- long rows
// A workgroup goes over a row, or over one part of it where there are few rows, in tiles of U 16-byte vectors a lane: running maximum, sum and
// weighted sum per lane, joined at the end.

template <typename T> struct Tile {
    static constexpr int V = 16 / sizeof(T), U = 4, SIZE = BLOCK * U * V;
    // vector u of a tile in this thread: a wavefront's 64 vectors are neighbours, and its places ascend with the tile and u
    static __device__ __forceinline__ int64_t place(int64_t tile, int u) { return tile * SIZE + (u * BLOCK + (int)threadIdx.x) * V; }
    static __device__ __forceinline__ void load_tile(const Row<T> &row, int64_t tile, int n, float (&x)[U][V]) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t j = place(tile, u);
            if (j < n) load<V>(row, (int)j, n, x[u]);
            else
#pragma unroll
                for (int k = 0; k < V; k++) x[u][k] = NEG_INF;
        }
    }
};

// Maximum m, s = sum 2^d, t = sum d 2^d with d = (x - m) inv_t2, of scores seen so far (none: m = -inf, s = t = 0).  A NaN or +inf among
// them makes s NaN.
struct Softmax {
    float m = NEG_INF, s = 0, t = 0;
    __device__ __forceinline__ void to(float new_m, float inv_t2) {          // the same scores against a larger maximum
        const float d = (m - new_m) * inv_t2, c = __builtin_amdgcn_exp2f(d);
        t = s == 0 ? 0 : c * fmaf(fmaxf(d, -1e30f), s, t);
        s = s == 0 ? 0 : c * s;
        m = new_m;
    }
    __device__ __forceinline__ void join(Softmax o, float inv_t2) {
        const float top = fmaxf(m, o.m);
        if (top > NEG_INF) { to(top, inv_t2); o.to(top, inv_t2); }
        s += o.s;
        t += o.t;
    }
};

// The best k <= 64 scores a wavefront has seen, lane i the i-th best (score, index); -inf and -1 where there are fewer.
struct Best {
    float v = NEG_INF, last_v = NEG_INF;
    int i = -1, last_i = -1, k;          // last: the k-th
    __device__ explicit Best(int k_) : k(k_) {}
    __device__ __forceinline__ bool wants(float x, int j) const { return better(x, j, last_v, last_i); }
    // every lane offers one score (-inf: none)
    __device__ __forceinline__ void offer(float x, int j) {
        uint64_t who = __ballot(wants(x, j));
        while (who) {
            const int lane = __ffsll((unsigned long long)who) - 1;
            const float cv = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
            const int ci = __builtin_amdgcn_readlane(j, lane);
            const int at = __popcll(__ballot(better(v, i, cv, ci)));
            const float sv = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x138, 0xf, 0xf, false));
            const int si = __builtin_amdgcn_update_dpp(0, i, 0x138, 0xf, 0xf, false);          // (one lane up)
            const int me = threadIdx.x & 63;
            v = me < at ? v : me == at ? cv : sv;
            i = me < at ? i : me == at ? ci : si;
            last_v = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), k - 1));
            last_i = __builtin_amdgcn_readlane(i, k - 1);
            who &= ~(1ull << lane);
            who &= __ballot(wants(x, j));
        }
    }
};

struct LogProbOut {
    float *log_prob, *entropy, *stats, *top_log_probs;
    int32_t *top_actions;
    int top;
};

// a row's results from its sums (one lane) and its best (one wavefront)
template <typename T> __device__ void finish_row(const Scores<T> &sc, int64_t r, const Actions &actions, const Softmax &all, const Best &best,
                                                 const LogProbOut &out) {
    const int lane = threadIdx.x & 63, n = (int)sc.n;
    const bool some = all.m > NEG_INF, undefined = !(all.s == all.s);
    const float ref = some ? all.m : 0.0f, log_s = logf(all.s), nan = __builtin_nanf("");
    if (lane == 0) {
        const int64_t a = actions.at(r);
        const Row<T> row(sc, r);
        float lp = 0.0f;
        if (a >= n || (a >= 0 && undefined)) lp = nan;
        else if (a >= 0) lp = some ? (row.at(a) - ref) * sc.inv_t - log_s : NEG_INF;
        out.log_prob[r] = lp;
        out.entropy[r] = undefined ? nan : some ? log_s - all.t / all.s * (float)LN_2 : 0.0f;
        if (out.stats) { out.stats[2 * r] = ref; out.stats[2 * r + 1] = log2f(all.s); }
    }
    if (lane < out.top) {
        const bool there = best.i >= 0 && !undefined;
        out.top_actions[r * out.top + lane] = there ? best.i : -1;
        out.top_log_probs[r * out.top + lane] = there ? (best.v - ref) * sc.inv_t - log_s : NEG_INF;
    }
}

// what one part of a row leaves for the join: its sums, and `top` best behind them
__device__ __forceinline__ int part_words(int top) { return 4 + 2 * top; }

template <typename T>
__global__ __launch_bounds__(BLOCK) void k_log_probs_long(Scores<T> sc, Actions actions, LogProbOut out, int parts, int64_t part_tiles,
                                                          float *workspace) {
    using L = Tile<T>;
    __shared__ float lds[WAVES][3];
    __shared__ float lds_v[WAVES][64];
    __shared__ int lds_i[WAVES][64];
    const int n = (int)sc.n, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, top = out.top;
    for (int64_t b = blockIdx.x; b < sc.rows * parts; b += gridDim.x) {
        const int64_t r = b / parts, part = b % parts;
        const Row<T> row(sc, r);
        const int64_t tiles = (n + L::SIZE - 1) / L::SIZE, first = part * part_tiles, behind = first + part_tiles < tiles ? first + part_tiles : tiles;
        Softmax a;
        Best best(top ? top : 1);
        for (int64_t tile = first; tile < behind; tile++) {
            float x[L::U][L::V], um[L::U];
            L::load_tile(row, tile, n, x);
            float m = NEG_INF;
#pragma unroll
            for (int u = 0; u < L::U; u++) {
                um[u] = x[u][0];
#pragma unroll
                for (int k = 1; k < L::V; k++) um[u] = fmaxf(um[u], x[u][k]);
                m = fmaxf(m, um[u]);
            }
            if (m > a.m) a.to(m, sc.inv_t2);
            const float ref = a.m > NEG_INF ? a.m : 0.0f;
#pragma unroll
            for (int u = 0; u < L::U; u++)
#pragma unroll
                for (int k = 0; k < L::V; k++) {
                    const float d = (x[u][k] - ref) * sc.inv_t2, p = __builtin_amdgcn_exp2f(d);
                    a.s += p;
                    a.t = fmaf(p, fmaxf(d, -1e30f), a.t);
                }
            // (a later score that only equals the k-th best is behind it)
            if (top && __ballot(m > best.last_v)) {
#pragma unroll
                for (int u = 0; u < L::U; u++)
                    if (__ballot(um[u] > best.last_v))
#pragma unroll
                        for (int k = 0; k < L::V; k++) best.offer(x[u][k], (int)(L::place(tile, u) + k));
            }
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            Softmax other;
            other.m = __shfl_xor(a.m, o);
            other.s = __shfl_xor(a.s, o);
            other.t = __shfl_xor(a.t, o);
            a.join(other, sc.inv_t2);
        }
        __syncthreads();
        if (lane == 0) { lds[wave][0] = a.m; lds[wave][1] = a.s; lds[wave][2] = a.t; }
        if (top) { lds_v[wave][lane] = best.v; lds_i[wave][lane] = best.i; }
        __syncthreads();
        if (wave == 0) {
            for (int w = 1; w < WAVES; w++) {
                Softmax o;
                o.m = lds[w][0];
                o.s = lds[w][1];
                o.t = lds[w][2];
                a.join(o, sc.inv_t2);
                if (top) best.offer(lane < top ? lds_v[w][lane] : NEG_INF, lds_i[w][lane]);
            }
            if (parts == 1) finish_row(sc, r, actions, a, best, out);
            else {
                float *to = workspace + b * part_words(top);
                if (lane == 0) { to[0] = a.m; to[1] = a.s; to[2] = a.t; }
                if (lane < top) { to[4 + lane] = best.v; to[4 + top + lane] = __builtin_bit_cast(float, best.i); }
            }
        }
    }
}

// one wavefront a row: the parts' sums and best
template <typename T>
__global__ __launch_bounds__(64) void k_log_probs_join(Scores<T> sc, Actions actions, LogProbOut out, int parts, const float *workspace) {
    const int lane = threadIdx.x, top = out.top;
    for (int64_t r = blockIdx.x; r < sc.rows; r += gridDim.x) {
        const float *from = workspace + r * parts * part_words(top);
        Softmax a;
        for (int p = lane; p < parts; p += 64) {
            const float *f = from + (int64_t)p * part_words(top);
            Softmax o;
            o.m = f[0];
            o.s = f[1];
            o.t = f[2];
            a.join(o, sc.inv_t2);
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            Softmax other;
            other.m = __shfl_xor(a.m, o);
            other.s = __shfl_xor(a.s, o);
            other.t = __shfl_xor(a.t, o);
            a.join(other, sc.inv_t2);
        }
        Best best(top ? top : 1);
        for (int64_t c0 = 0; c0 < (int64_t)parts * top; c0 += 64) {
            const int64_t c = c0 + lane;
            float v = NEG_INF;
            int i = -1;
            if (c < (int64_t)parts * top) {
                const float *f = from + c / top * part_words(top) + 4;
                v = f[c % top];
                i = __builtin_bit_cast(int, f[top + c % top]);
            }
            best.offer(v, i);
        }
        finish_row(sc, r, actions, a, best, out);
    }
}

template <typename T>
__global__ __launch_bounds__(BLOCK) void k_backward_long(Scores<T> sc, Actions actions, const float *stats, const float *entropy, const float *g_lp,
                                                         int64_t g_lp_stride, const float *g_h, int64_t g_h_stride, T *grad) {
    using L = Tile<T>;
    const int n = (int)sc.n;
    for (int64_t r = blockIdx.y; r < sc.rows; r += gridDim.y) {
        const Row<T> row(sc, r);
        const int64_t a = actions.at(r);
        const float ref = stats[2 * r], log2_s = stats[2 * r + 1], h = entropy[r];
        const float gl = g_lp && a >= 0 ? g_lp[r * g_lp_stride] : 0.0f, gh = g_h ? g_h[r * g_h_stride] : 0.0f;
        // dx = p (c0 + c1 log2 p) + 1[j = a] g_lp / T
        const float c0 = -(gl + gh * h) * sc.inv_t, c1 = -gh * (float)LN_2 * sc.inv_t;
        float x[L::U][L::V];
        L::load_tile(row, blockIdx.x, n, x);
        T *to = grad + r * sc.n;
#pragma unroll
        for (int u = 0; u < L::U; u++) {
            const int64_t j = L::place(blockIdx.x, u);
            const int given = a >= j && a < j + L::V ? (int)(a - j) : -1;
            T v[L::V];
#pragma unroll
            for (int k = 0; k < L::V; k++) {
                const float lp = (x[u][k] - ref) * sc.inv_t2 - log2_s, p = __builtin_amdgcn_exp2f(lp);
                float g = p * fmaf(c1, fmaxf(lp, -1e30f), c0);
                if (k == given) g += gl * sc.inv_t;
                v[k] = from_f32<T>(x[u][k] == NEG_INF ? 0.0f : g);
            }
            if (j + L::V <= n) __builtin_memcpy(to + j, v, sizeof v);
            else
#pragma unroll
                for (int k = 0; k < L::V; k++)
                    if (j + k < n) to[j + k] = v[k];
        }
    }
}

// ---- drawing: the row's segments of 64 vectors (one a lane), each with its own maximum and 64-bit sums, then the one segment the target lies in
struct Segment {
    double s, t;        // sum 2^d, sum d 2^d
    float m;            // its maximum (-inf: nothing open)
    int nan;
};
__device__ __forceinline__ double wave_sum(double v) { return wave_all(v, [](double a, double b) { return a + b; }); }

// the four segments of a wavefront's part of a tile: (tile, u, wave) is segment (tile * U + u) * WAVES + wave
template <typename T> __device__ __forceinline__ void sum_segments(const Scores<T> &sc, const Row<T> &row, int64_t tile, int64_t segments, Segment *to) {
    using L = Tile<T>;
    const int n = (int)sc.n, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float x[L::U][L::V];
    L::load_tile(row, tile, n, x);
    float m = NEG_INF;
    bool nan = false;
#pragma unroll
    for (int u = 0; u < L::U; u++)
#pragma unroll
        for (int k = 0; k < L::V; k++) {
            m = fmaxf(m, x[u][k]);
            nan |= x[u][k] != x[u][k];
        }
    m = wave_all(m, f_max);
    const double ref = m > NEG_INF ? m : 0.0;
    double t = 0;
    const int any_nan = __ballot(nan) != 0;
#pragma unroll
    for (int u = 0; u < L::U; u++) {
        double s = 0;
#pragma unroll
        for (int k = 0; k < L::V; k++) {
            const double d = fmax(((double)x[u][k] - ref) * sc.inv_t2_64, -1100.0), p = exp2_64(d);
            s += p;
            t = fma(p, d, t);
        }
        s = wave_sum(s);
        if (u == L::U - 1) t = wave_sum(t);
        const int64_t seg = (tile * L::U + u) * WAVES + wave;
        // (the tile's t, all against one maximum, goes with its last segment that there is)
        if (lane == 0 && seg < segments) to[seg] = {s, 0.0, m, any_nan};
    }
    if (lane == 0) {
        int64_t seg = (tile * L::U + L::U - 1) * WAVES + wave;
        while (seg >= segments) seg -= WAVES;
        if (seg >= tile * L::U * WAVES) to[seg].t = t;
    }
}

// One wavefront: the row's action from its segments.
template <typename T>
__device__ void draw(const Scores<T> &sc, int64_t r, const Segment *seg, int64_t segments, const void *uniforms, int uniform_bytes, int32_t *action,
                     float *log_prob, float *entropy) {
    constexpr int V = Tile<T>::V;
    const int lane = threadIdx.x & 63, n = (int)sc.n;
    const Row<T> row(sc, r);
    // every lane has a run of neighbouring segments
    const int64_t each = (segments + 63) / 64, lo = lane * each < segments ? lane * each : segments, hi = lo + each < segments ? lo + each : segments;
    float m = NEG_INF;
    int nan = 0;
    for (int64_t g = lo; g < hi; g++) { m = fmaxf(m, seg[g].m); nan |= seg[g].nan; }
    m = wave_all(m, f_max);
    const bool some = m > NEG_INF, undefined = __ballot(nan) || m == -NEG_INF;
    if (undefined || !some) {
        if (lane == 0) {
            action[r] = -1;
            if (log_prob) log_prob[r] = undefined ? __builtin_nanf("") : NEG_INF;
            if (entropy) entropy[r] = undefined ? __builtin_nanf("") : 0.0f;
        }
        return;
    }
    const double ref = m;
    const auto weight = [&](const Segment &g, double &d) {
        d = fmax(((double)g.m - ref) * sc.inv_t2_64, -1100.0);
        return exp2_64(d);
    };
    double s = 0, t = 0;
    for (int64_t g = lo; g < hi; g++) {
        double d;
        const double w = weight(seg[g], d);
        s += w * seg[g].s;
        t += w * fma(d, seg[g].s, seg[g].t);
    }
    double upto = s;
    for (int o = 1; o < 64; o <<= 1) {
        const double v = __shfl_up(upto, o);
        if (lane >= o) upto += v;
    }
    const double total = __shfl(upto, 63);
    t = wave_sum(t);
    const double target = uniform_at(uniforms, uniform_bytes, r) * total;
    // the first run that passes the target, or else (rounding; a number of 1) the last one with anything in it; then the segment in it
    uint64_t past = __ballot(s > 0.0 && upto > target), any = __ballot(s > 0.0);
    const int run = past ? __ffsll((unsigned long long)past) - 1 : 63 - __clzll((long long)any);
    double before = __shfl(lane == 0 ? 0.0 : upto - s, run);
    int64_t found = -1;
    double found_before = 0;
    for (int64_t g = run * each; g < (run + 1) * each && g < segments; g++) {
        double d;
        const double w = weight(seg[g], d) * seg[g].s;
        if (w > 0.0) { found = g; found_before = before; }
        before += w;
        if (w > 0.0 && before > target) break;
    }
    // ... and the action in the segment
    float x[V];
    const int64_t j = (found * 64 + lane) * V;
    if (j < n) load<V>(row, (int)j, n, x);
    else
#pragma unroll
        for (int k = 0; k < V; k++) x[k] = NEG_INF;
    double p[V];
    s = 0;
#pragma unroll
    for (int k = 0; k < V; k++) {
        p[k] = exp2_64(((double)x[k] - ref) * sc.inv_t2_64);
        s += p[k];
    }
    upto = s;
    for (int o = 1; o < 64; o <<= 1) {
        const double v = __shfl_up(upto, o);
        if (lane >= o) upto += v;
    }
    past = __ballot(s > 0.0 && found_before + upto > target);
    any = __ballot(s > 0.0);
    const bool tiny = !any;          // (the segment's sum is above 0 and all its terms round to it: the first one that is open)
    if (tiny) {
        bool open = false;
#pragma unroll
        for (int k = 0; k < V; k++) open |= x[k] > NEG_INF;
        past = __ballot(open);
    }
    const int owner = past ? __ffsll((unsigned long long)past) - 1 : 63 - __clzll((long long)any);
    if (lane == owner) {
        double c = found_before + (lane == 0 ? 0.0 : upto - s);
        int a = -1;
        float xa = 0;
        bool done = false;
#pragma unroll
        for (int k = 0; k < V; k++) {
            c += p[k];
            if ((tiny ? x[k] > NEG_INF : p[k] > 0.0) && !done) { a = (int)j + k; xa = x[k]; done = tiny || c > target; }
        }
        action[r] = a;
        if (log_prob) log_prob[r] = (float)(((double)xa - ref) * sc.inv_t2_64 * LN_2 - log(total));
        if (entropy) entropy[r] = (float)(log(total) - t / total * LN_2);
    }
}

// parts == 1: a workgroup sums a row's segments and its first wavefront draws; else only the sums, for k_draw
template <typename T>
__global__ __launch_bounds__(BLOCK) void k_sample_long(Scores<T> sc, const void *uniforms, int uniform_bytes, int32_t *action, float *log_prob,
                                                       float *entropy, int parts, int64_t part_tiles, int64_t segments, Segment *workspace) {
    using L = Tile<T>;
    const int64_t tiles = (sc.n + L::SIZE - 1) / L::SIZE;
    for (int64_t b = blockIdx.x; b < sc.rows * parts; b += gridDim.x) {
        const int64_t r = b / parts, first = b % parts * part_tiles, behind = first + part_tiles < tiles ? first + part_tiles : tiles;
        const Row<T> row(sc, r);
        Segment *seg = workspace + r * segments;
        for (int64_t tile = first; tile < behind; tile++) sum_segments(sc, row, tile, segments, seg);
        if (parts == 1) {
            __syncthreads();
            if (threadIdx.x < 64) draw(sc, r, seg, segments, uniforms, uniform_bytes, action, log_prob, entropy);
        }
    }
}
template <typename T>
__global__ __launch_bounds__(64) void k_draw(Scores<T> sc, const void *uniforms, int uniform_bytes, int32_t *action, float *log_prob, float *entropy,
                                             int64_t segments, const Segment *workspace) {
    for (int64_t r = blockIdx.x; r < sc.rows; r += gridDim.x)
        draw(sc, r, workspace + r * segments, segments, uniforms, uniform_bytes, action, log_prob, entropy);
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
    if (!(temperature > 0) || !std::isfinite((float)(LOG2_E / temperature)) || !((float)(1.0 / temperature) >= FLT_MIN))
        return fail(MGX_ERR_ARG, "temperature: positive, and its reciprocal a normal fp32 number");
    return MGX_OK;
}

template <typename T>
Scores<T> scores(const void *logits, int64_t rows, int64_t n, int64_t row_stride, const uint8_t *mask, int64_t mask_row_stride, double temperature) {
    return {(const T *)logits, mask, rows, n, row_stride, mask_row_stride, (float)(1.0 / temperature),
            (float)(LOG2_E / temperature), LOG2_E / temperature};
}

// a grid of at most 2^32 work items; the kernels go on from there in strides of the grid (its last dimension)
template <typename... P, typename... A> int launch(void (*kernel)(P...), dim3 blocks, int threads, void *stream, A... args) {
    void *ptrs[] = {(void *)&args...};
    static_assert(sizeof...(P) == sizeof...(A) && (std::is_same_v<P, A> && ...), "argument types are the kernel's");
    const int64_t most = 0xffffffffLL / threads;
    if (blocks.y > most / blocks.x) blocks.y = (unsigned)(most / blocks.x);
    const hipError_t err = hipLaunchKernel((const void *)kernel, blocks, dim3(threads), ptrs, 0, (hipStream_t)stream);
    return err == hipSuccess ? (int)MGX_OK : fail(MGX_ERR_HIP, hipGetErrorString(err));
}
template <typename... P, typename... A> int launch(void (*kernel)(P...), int64_t blocks, int threads, void *stream, A... args) {
    return launch(kernel, dim3((unsigned)std::min<int64_t>(blocks, 0xffffffffLL / threads)), threads, stream, args...);
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
// How many workgroups share a long row: enough to give every one of the 256 CUs some, no more than the row has tiles.
struct Split {
    int parts;
    int64_t part_tiles;
};
Split split(int dtype, int64_t rows, int64_t n) {
    const int64_t size = dtype == MGX_REAL_F32 ? Tile<float>::SIZE : Tile<half>::SIZE, tiles = (n + size - 1) / size;
    const int64_t wanted = std::max<int64_t>(1, std::min<int64_t>(tiles, 1024 / std::max<int64_t>(rows, 1))), each = (tiles + wanted - 1) / wanted;
    return {(int)((tiles + each - 1) / each), each};
}
int64_t n_segments(int dtype, int64_t n) {
    const int64_t size = 64 * (dtype == MGX_REAL_F32 ? Tile<float>::V : Tile<half>::V);
    return (n + size - 1) / size;
}

int64_t short_blocks(int64_t rows, int G) { return (rows * G + BLOCK - 1) / BLOCK; }

// f(a value of the scores' element type)
template <typename F> int by_dtype(int dtype, F f) {
    switch (dtype) {
        case MGX_REAL_F32: return f(float());
        case MGX_REAL_F16: return f(half());
        default: return f(bf16());
    }
}

}  // namespace

extern "C" {

const char *mgx_policy_last_error(void) { return g_err; }

int64_t mgx_policy_workspace_bytes(int op, int dtype, int64_t rows, int64_t n, int top) {
    if (n <= SHORT_MAX || rows <= 0) return 0;
    if (op == MGX_POLICY_SAMPLE) return rows * n_segments(dtype, n) * (int64_t)sizeof(Segment);
    const Split sp = split(dtype, rows, n);
    return sp.parts == 1 ? 0 : rows * sp.parts * (4 + 2 * (int64_t)top) * 4;
}

int64_t mgx_policy_stats_bytes(int64_t rows, int64_t n) { return n > SHORT_MAX ? rows * 8 : 0; }

int mgx_policy_log_probs(int device, int dtype, const void *logits, int64_t rows, int64_t n, int64_t row_stride, const uint8_t *mask,
                         int64_t mask_row_stride, double temperature, const void *actions, int action_bytes, int top, float *log_prob,
                         float *entropy, float *stats, float *top_log_probs, int32_t *top_actions, void *workspace,
                         int64_t workspace_bytes, void *stream) {
    if (int rc = check_scores(dtype, logits, rows, n, row_stride, mask, mask_row_stride, temperature)) return rc;
    if (action_bytes != 4 && action_bytes != 8) return fail(MGX_ERR_ARG, "action_bytes: 4 or 8");
    if (top < 0 || top > MGX_POLICY_MAX_TOP || top > n) return fail(MGX_ERR_ARG, "top: 0 ... min(n, 64)");
    if (rows == 0) return MGX_OK;
    if (const int64_t need = mgx_policy_workspace_bytes(MGX_POLICY_LOG_PROBS, dtype, rows, n, top))
        if (!workspace || workspace_bytes < need) return fail(MGX_ERR_ARG, "workspace: smaller than mgx_policy_workspace_bytes()");
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
        const Split sp = split(dtype, rows, n);
        const LogProbOut out{log_prob, entropy, stats, top_log_probs, top_actions, top};
        const Actions given{actions, action_bytes};
        const int rc = launch(k_log_probs_long<T>, rows * sp.parts, BLOCK, stream, sc, given, out, sp.parts, sp.part_tiles, (float *)workspace);
        if (rc || sp.parts == 1) return rc;
        return launch(k_log_probs_join<T>, rows, 64, stream, sc, given, out, sp.parts, (const float *)workspace);
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
        return launch(k_backward_long<T>, dim3((unsigned)((n + Tile<T>::SIZE - 1) / Tile<T>::SIZE), (unsigned)std::min<int64_t>(rows, 65535)), BLOCK,
                      stream, sc, Actions{actions, action_bytes}, stats, entropy, grad_log_prob, grad_log_prob_stride, grad_entropy,
                      grad_entropy_stride, (T *)grad);
    });
}

int mgx_policy_sample(int device, int dtype, const void *logits, int64_t rows, int64_t n, int64_t row_stride, const uint8_t *mask,
                      int64_t mask_row_stride, double temperature, const void *uniforms, int uniform_bytes, int32_t *action,
                      float *log_prob, float *entropy, void *workspace, int64_t workspace_bytes, void *stream) {
    if (int rc = check_scores(dtype, logits, rows, n, row_stride, mask, mask_row_stride, temperature)) return rc;
    if (uniform_bytes != 4 && uniform_bytes != 8) return fail(MGX_ERR_ARG, "uniform_bytes: 4 or 8");
    if (rows == 0) return MGX_OK;
    if (const int64_t need = mgx_policy_workspace_bytes(MGX_POLICY_SAMPLE, dtype, rows, n, 0))
        if (!workspace || workspace_bytes < need) return fail(MGX_ERR_ARG, "workspace: smaller than mgx_policy_workspace_bytes()");
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
        const Split sp = split(dtype, rows, n);
        const int64_t segments = n_segments(dtype, n);
        const int rc = launch(k_sample_long<T>, rows * sp.parts, BLOCK, stream, sc, uniforms, uniform_bytes, action, log_prob, entropy, sp.parts,
                              sp.part_tiles, segments, (Segment *)workspace);
        if (rc || sp.parts == 1) return rc;
        return launch(k_draw<T>, rows, 64, stream, sc, uniforms, uniform_bytes, action, log_prob, entropy, segments, (const Segment *)workspace);
    });
}

}  // extern "C"
