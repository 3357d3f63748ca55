// mgx_policy.hip -- the operators of include/mgx_policy.h: what lies between a policy's action scores and the engine's actions.
//
// Times in these comments, unless one says otherwise: of a call among ten of its kind in a captured graph, on the same scores, the median, on an MI355X;
// scores that fit the 256 MB cache in front of the memory come from there in part.  A copy of 1 GiB moves 5.1 TB/s on it.
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
constexpr double LOG2_E = 1.4426950408889634, LN_2 = 0.6931471805599453;

// The rows of scores a call works on; an action that is not open reads as -inf.
template <typename T> struct Scores {
    const T *x;
    const uint8_t *mask;
    int64_t rows, n, stride, mask_stride;
    float inv_t, inv_t2;        // 1 / temperature, log2(e) / temperature: exponentials are taken to the base 2, as the hardware does
    double inv_t2_64;
    // Two scores may be further apart than the largest fp32 number (3e38 and -3e38).  Over a T of up to 1e36 their quotient is one whose exponential is 0
    // all the same; over a larger one the difference is taken of their halves (unit 1 / 2, else 1), in one operation.  (Told by what is there already:
    // two more arguments made 983040 x 18 fp32 17.9 us of 17.2.)
    __host__ __device__ __forceinline__ bool by_halves() const { return __builtin_bit_cast(uint32_t, inv_t2) < __builtin_bit_cast(uint32_t, 1.44e-36f); }
    // one score's (v - ref) / T as a result, which is to be finite over smaller T too: always by halves
    __device__ __forceinline__ float over_t(float v, float ref) const { return 2.0f * (fmaf(v, 0.5f, -0.5f * ref) * inv_t); }
};

using half = _Float16;
using bf16 = __bf16;
template <typename T> __device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f32(float v) { return (T)v; }          // to nearest, ties to even

// Differences of scores, in a loop's scalar registers (worked out on their bits: there is no scalar unit for floats; the long rows' kernel is given it,
// 65536 x 1500 bf16 44.7 us, itself 45.7, without halves 42.9).
struct Difference {
    float unit, per_t2;         // per_t2: log2(e) / (T unit)
    template <typename T> __host__ __device__ __forceinline__ explicit Difference(const Scores<T> &sc) {
        const uint32_t one_exponent = sc.by_halves() ? 1u << 23 : 0;
        unit = __builtin_bit_cast(float, 0x3f800000u - one_exponent);
        per_t2 = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, sc.inv_t2) + one_exponent);
    }
    __device__ __forceinline__ float operator()(float v, float unit_ref) const { return fmaf(v, unit, -unit_ref); }
    __device__ __forceinline__ float over_t2(float v, float unit_ref) const { return (*this)(v, unit_ref) * per_t2; }
};

template <typename T> struct Row {
    const T *x;
    const uint8_t *mask;
    __device__ Row(const Scores<T> &s, int64_t r) : x(s.x + r * s.stride), mask(s.mask ? s.mask + r * s.mask_stride : nullptr) {}
    __device__ __forceinline__ float at(int64_t j) const {
        const float v = to_f32(x[j]);
        return mask && !mask[j] ? NEG_INF : v;
    }
};

// The larger of two; a NaN wins.  (fmaxf would quiet each operand first, an instruction a score; two of these are one on gfx950.)
__device__ __forceinline__ float max_of(float a, float b) { return __builtin_elementwise_maximum(a, b); }

struct Actions {
    const void *p;
    int bytes;
    __device__ __forceinline__ int64_t at(int64_t r) const { return bytes == 8 ? ((const int64_t *)p)[r] : ((const int32_t *)p)[r]; }
};

constexpr int BLOCK = 256, WAVES = BLOCK / 64;

// A whole vector of results.  stream: it is not kept in the caches (STREAM_BYTES below).
template <typename T, int W> __device__ __forceinline__ void store_bytes(T *to, const T (&v)[W], bool stream) {
    if constexpr (sizeof v == 16) {
        using Words = uint32_t __attribute__((ext_vector_type(4), aligned(2)));
        if (stream) {
            Words w;
            __builtin_memcpy(&w, v, 16);
            __builtin_nontemporal_store(w, (Words *)to);
            return;
        }
    }
    __builtin_memcpy(to, v, sizeof v);
}

template <typename T> constexpr uint32_t neg_inf_bits = sizeof(T) == 4 ? 0xff800000u : std::is_same_v<T, half> ? 0xfc00u : 0xff80u;

// N pieces of W neighbouring scores of a row, as they lie in memory (16-bit scores two a word), with their mask bytes.  One load a piece and
// one for its mask (gfx950 loads any alignment); what is behind the row's end is -inf.  SMALL: n may be less than W.
template <typename T, int W, int N, bool SMALL = false> struct Pieces {
    static constexpr int BITS = 8 * sizeof(T), WORDS = W * BITS / 32, MASK_WORDS = W / 4;
    uint32_t w[N][WORDS], open[N][MASK_WORDS];
    static_assert(W % 4 == 0);
    using Bits = std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>;
    static constexpr uint32_t CLOSED = sizeof(T) == 4 ? neg_inf_bits<T> : neg_inf_bits<T> << 16 | neg_inf_bits<T>;
    // v shifted down by `bits` (0 ... 64 * words), zeros from above
    static __device__ __forceinline__ uint64_t down(uint64_t v, int bits) { return bits < 64 ? v >> bits : 0; }
    template <int M> static __device__ __forceinline__ void shift_down(uint32_t (&v)[M], int bits) {
        if constexpr (M == 1) v[0] = bits < 32 ? v[0] >> bits : 0;
        else if constexpr (M == 2) {
            const uint64_t r = down((uint64_t)v[1] << 32 | v[0], bits);
            v[0] = (uint32_t)r;
            v[1] = (uint32_t)(r >> 32);
        } else {
            static_assert(M == 4);
            const uint64_t lo = (uint64_t)v[1] << 32 | v[0], hi = (uint64_t)v[3] << 32 | v[2];
            const uint64_t low = bits < 64 ? lo >> bits | hi << 1 << (63 - bits) : down(hi, bits - 64), high = down(hi, bits);
            v[0] = (uint32_t)low;
            v[1] = (uint32_t)(low >> 32);
            v[2] = (uint32_t)high;
            v[3] = (uint32_t)(high >> 32);
        }
    }
    // Piece p from place j on.  Where the row ends inside it (or before it), the row's last W scores are loaded instead and shifted down.
    __device__ __forceinline__ void fetch(const Row<T> &row, int p, int j, int n, bool whole) {
        if (whole) __builtin_memcpy(w[p], row.x + j, W * sizeof(T));
        else if (!SMALL || n >= W) {
            const int from = j < n - W ? j : n - W, bits = (j - from < W ? j - from : W) * BITS;
            __builtin_memcpy(w[p], row.x + from, W * sizeof(T));
#pragma unroll
            for (int k = 0; k < WORDS; k++) w[p][k] ^= CLOSED;
            shift_down(w[p], bits);
#pragma unroll
            for (int k = 0; k < WORDS; k++) w[p][k] ^= CLOSED;
        } else {
#pragma unroll
            for (int k = 0; k < WORDS; k++) w[p][k] = CLOSED;
#pragma unroll
            for (int k = 0; k < W; k++)
                if (j + k < n) {
                    Bits b;
                    __builtin_memcpy(&b, row.x + j + k, sizeof b);
                    w[p][k * BITS / 32] = BITS == 32 ? b : (k % 2 ? (w[p][k / 2] & 0xffff) | (uint32_t)b << 16 : (w[p][k / 2] & 0xffff0000u) | b);
                }
        }
    }
    __device__ __forceinline__ void fetch_mask(const Row<T> &row, int p, int j, int n, bool whole) {
        if (whole) __builtin_memcpy(open[p], row.mask + j, W);
        else if (!SMALL || n >= W) {
            const int from = j < n - W ? j : n - W;
            __builtin_memcpy(open[p], row.mask + from, W);
            shift_down(open[p], (j - from < W ? j - from : W) * 8);
        } else {
#pragma unroll
            for (int k = 0; k < MASK_WORDS; k++) open[p][k] = 0;
#pragma unroll
            for (int k = 0; k < W; k++)
                if (j + k < n) open[p][k / 4] |= (uint32_t)row.mask[j + k] << (k % 4 * 8);
        }
    }
    // piece p from place(p) on.  The wavefront's pieces below `whole` are all there in every lane, those from `live` on in none.
    template <typename F> __device__ __forceinline__ void load(const Row<T> &row, int n, int whole, int live, F place) {
#pragma unroll
        for (int p = 0; p < N; p++)
            if (p < live) fetch(row, p, place(p), n, p < whole);
            else
#pragma unroll
                for (int k = 0; k < WORDS; k++) w[p][k] = CLOSED;
        if (row.mask) {
#pragma unroll
            for (int p = 0; p < N; p++)
                if (p < live) fetch_mask(row, p, place(p), n, p < whole);
                else
#pragma unroll
                    for (int k = 0; k < MASK_WORDS; k++) open[p][k] = 0;
        }
    }
    // W values of type T to `to` from place j on, as far as the row goes
    static __device__ __forceinline__ void store(T *to, int j, int n, bool whole, const T (&v)[W], bool stream) {
        if (whole || j + W <= n) return store_bytes(to + j, v, stream);
        uint32_t q[WORDS];
        __builtin_memcpy(q, v, sizeof v);
        int left = n - j;
        if (left <= 0) return;
#pragma unroll
        for (int half = W / 2; half >= 1; half /= 2) {          // 4, 2 and 1 of them, as many as are left
            const int words = half * BITS / 32;
            if (left & half) {
                __builtin_memcpy(to + j, q, half * sizeof(T));
                j += half;
#pragma unroll
                for (int k = 0; k < words; k++) q[k] = q[words + k];
            }
        }
    }
    __device__ __forceinline__ float score(int p, int k) const {
        if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, w[p][k]);
        else if constexpr (std::is_same_v<T, half>) return (float)__builtin_bit_cast(half, (uint16_t)(w[p][k / 2] >> (k % 2 * 16)));
        else return __builtin_bit_cast(float, k % 2 ? w[p][k / 2] & 0xffff0000u : w[p][k / 2] << 16);
    }
    // the N * W scores in fp32, -inf where the mask rules them out (a byte less 1 is negative if it was 0, and only then: spread to all bits,
    // its sign selects)
    __device__ __forceinline__ void scores(const Row<T> &row, float *x) {
        if (row.mask)
#pragma unroll
            for (int p = 0; p < N; p++)
#pragma unroll
                for (int k = 0; k < WORDS; k++) {
                    uint32_t shut;
                    if constexpr (sizeof(T) == 4) shut = (uint32_t)(((int32_t)(open[p][k / 4] >> (k % 4 * 8) & 0xff) - 1) >> 31);
                    else {
                        using Two16 = short __attribute__((ext_vector_type(2)));
                        const Two16 bytes = __builtin_bit_cast(Two16, __builtin_amdgcn_perm(0, open[p][k / 2], k % 2 ? 0x0c030c02 : 0x0c010c00));
                        shut = __builtin_bit_cast(uint32_t, (Two16)((bytes - (Two16){1, 1}) >> (Two16){15, 15}));
                    }
                    w[p][k] = (shut & CLOSED) | (~shut & w[p][k]);
                }
#pragma unroll
        for (int p = 0; p < N; p++)
#pragma unroll
            for (int k = 0; k < W; k++) x[p * W + k] = score(p, k);
    }
};

// ---- lane exchanges in the vector unit.  Partner values of a butterfly over G lanes: quads, then half rows, rows of 16, and the two swaps of
// gfx950 (the mirrors reach the other half, whose lanes all hold the same by then).
// (lanes without a source get 0; where only some rows take part, so do the others)
template <int CTRL, int ROWS = 0xf> __device__ __forceinline__ int dpp(int v) {
    if constexpr (ROWS == 0xf) return __builtin_amdgcn_mov_dpp(v, CTRL, 0xf, 0xf, true);
    else return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS = 0xf> __device__ __forceinline__ float dpp(float v) { return __builtin_bit_cast(float, dpp<CTRL, ROWS>(__builtin_bit_cast(int, v))); }
template <int CTRL, int ROWS = 0xf> __device__ __forceinline__ double dpp(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)dpp<CTRL, ROWS>((int)(uint32_t)b), hi = (uint32_t)dpp<CTRL, ROWS>((int)(uint32_t)(b >> 32));
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
constexpr int DPP_XOR1 = 0xB1, DPP_XOR2 = 0x4E, DPP_HALF_MIRROR = 0x141, DPP_MIRROR = 0x140, DPP_WAVE_SHR1 = 0x138, DPP_ROW_SHR = 0x110,
              DPP_BCAST15 = 0x142, DPP_BCAST31 = 0x143;
template <typename V> struct Two { V a, b; };
// the values of this lane's and its partner's 16 (32) lanes, the lower ones' first
__device__ __forceinline__ Two<int> swap16(int v) { const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false); return {(int)r[0], (int)r[1]}; }
__device__ __forceinline__ Two<int> swap32(int v) { const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false); return {(int)r[0], (int)r[1]}; }
template <int N> __device__ __forceinline__ Two<int> swap(int v) { if constexpr (N == 16) return swap16(v); else return swap32(v); }
template <int N> __device__ __forceinline__ Two<float> swap(float v) {
    const Two<int> r = swap<N>(__builtin_bit_cast(int, v));
    return {__builtin_bit_cast(float, r.a), __builtin_bit_cast(float, r.b)};
}
template <int N> __device__ __forceinline__ Two<double> swap(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const Two<int> lo = swap<N>((int)(uint32_t)b), hi = swap<N>((int)(uint32_t)(b >> 32));
    return {__builtin_bit_cast(double, (uint64_t)(uint32_t)hi.a << 32 | (uint32_t)lo.a), __builtin_bit_cast(double, (uint64_t)(uint32_t)hi.b << 32 | (uint32_t)lo.b)};
}
// f over the G lanes of a group (f commutes: all lanes get the same bits)
template <int G, typename V, typename F> __device__ __forceinline__ V group_all(V v, F f) {
    if constexpr (G > 1) v = f(v, dpp<DPP_XOR1>(v));
    if constexpr (G > 2) v = f(v, dpp<DPP_XOR2>(v));
    if constexpr (G > 4) v = f(v, dpp<DPP_HALF_MIRROR>(v));
    if constexpr (G > 8) v = f(v, dpp<DPP_MIRROR>(v));
    if constexpr (G > 16) { const Two<V> t = swap<16>(v); v = f(t.a, t.b); }
    if constexpr (G > 32) { const Two<V> t = swap<32>(v); v = f(t.a, t.b); }
    return v;
}
template <int G> __device__ __forceinline__ float group_max(float v) { return group_all<G>(v, [](float a, float b) { return max_of(a, b); }); }
template <int G, typename V> __device__ __forceinline__ V group_sum(V v) { return group_all<G>(v, [](V a, V b) { return a + b; }); }
// running sum over the G lanes of a group, this lane (number g) included
template <int G> __device__ __forceinline__ double group_scan(double v, int g) {
    const auto step = [&](double from, int o) { v += G >= 16 || g >= o ? from : 0.0; };          // (a row's first lanes get 0 from outside)
    if constexpr (G > 1) step(dpp<DPP_ROW_SHR + 1>(v), 1);
    if constexpr (G > 2) step(dpp<DPP_ROW_SHR + 2>(v), 2);
    if constexpr (G > 4) step(dpp<DPP_ROW_SHR + 4>(v), 4);
    if constexpr (G > 8) step(dpp<DPP_ROW_SHR + 8>(v), 8);
    if constexpr (G > 16) v += dpp<DPP_BCAST15, 0xa>(v);
    if constexpr (G > 32) v += dpp<DPP_BCAST31, 0xc>(v);
    return v;
}
__device__ __forceinline__ float lane_of(float v, int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane)); }
__device__ __forceinline__ double lane_of(double v, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ int first_lane(uint64_t b) { return __ffsll((unsigned long long)b) - 1; }
__device__ __forceinline__ int last_lane(uint64_t b) { return 63 - __clzll((long long)b); }

// what lanes of a wavefront have written to LDS is there for its others
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// is (v, i) a better alternative than (w, k)?  Higher score first, then the lower index.
__device__ __forceinline__ bool better(float v, int i, float w, int k) { return v > w || (v == w && i < k); }

// a * b + c with c in scalar registers.  (The compiler would copy the constant into vector registers first, two moves a step.)
__device__ __forceinline__ double fma_64(double a, double b, double c) {
    double r;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
    return r;
}
// For drawing: scores as differences to a maximum, in 64 bits, and 2^(d * inv_t2) of them.  A difference below 2^-1000's counts as that, -inf
// and NaN too (the callers look for NaN themselves), and what is below NOTHING as no probability at all.
constexpr double NOTHING = 0x1p-990;
__device__ __forceinline__ double or_nothing(double p) { return p > NOTHING ? p : 0.0; }
struct Exp64 {
    double inv_t2, least;
    __device__ __forceinline__ explicit Exp64(double inv_t2_) : inv_t2(inv_t2_), least(-1000.0 / inv_t2_) {}
    __device__ __forceinline__ double below(float x, double ref) const { return fmax((double)x - ref, least); }
    // y = d * inv_t2 = k + f with |f| <= 1 / 2 (k by adding 1.5 * 2^52, whose last bits then are k); a polynomial for 2^f (interpolated at the
    // Chebyshev points of [-1/2, 1/2] in 60 digits: off by 3.1e-16 at most); k added to its exponent
    __device__ __forceinline__ double operator()(double d) const {
        const double shifted = fma_64(d, inv_t2, 0x1.8p52), f = fma(d, inv_t2, 0x1.8p52 - shifted);
        using Words = uint32_t __attribute__((ext_vector_type(2)));
        double p = 0x1.e6063f7217bc6p-28;
        p = fma_64(p, f, 0x1.b675bca4eeebbp-24);
        p = fma_64(p, f, 0x1.62bfd47773353p-20);
        p = fma_64(p, f, 0x1.ffcb54062e698p-17);
        p = fma_64(p, f, 0x1.430913096fd9fp-13);
        p = fma_64(p, f, 0x1.5d87fe9d7a584p-10);
        p = fma_64(p, f, 0x1.3b2ab6fba1ddap-7);
        p = fma_64(p, f, 0x1.c6b08d703ce49p-5);
        p = fma_64(p, f, 0x1.ebfbdff82c598p-3);
        p = fma_64(p, f, 0x1.62e42fefa3a19p-1);
        p = fma_64(p, f, 1.0);
        Words w = __builtin_bit_cast(Words, p);
        w.y += __builtin_bit_cast(Words, shifted).x << 20;
        return __builtin_bit_cast(double, w);
    }
};

// ---------------------------------------------------------------------------------------------------------------- short rows
// A row stays in the registers of G lanes (1 ... 64), E scores a lane: one read of the scores, all sums by lane exchanges, no barrier.  What
// bounds it: memory (983040 x 18 fp32: 17.1 us where its 86 MB take 17 at a copy's rate; backward 27 where its 161 MB take 31: part of them lies
// in the cache), from some dozen scores a row on the vector unit, which issues some 15 instructions a score, 20 with a mask (61440 x 324 bf16
// with a mask: 15.4 us, 12 of them issued, where memory would take 8; backward 22.8, 16 issued, 16 of memory).  Lane g holds pieces of W
// neighbouring scores (16 bytes, or 4 scores): x[e] is score place(g, e).
template <int G, int E, int W> struct Spread {
    static __device__ __forceinline__ int place(int g, int e) { return e / W * (G * W) + g * W + e % W; }
    template <typename T> static __device__ __forceinline__ void load_row(const Row<T> &row, int g, int n, float (&x)[E]) {
        Pieces<T, W, E / W, G == 1> p;
        p.load(row, n, n / (G * W), E / W, [&](int k) { return place(g, k * W); });
        p.scores(row, x);
    }
};
template <int E> __device__ __forceinline__ float lane_max(const float (&x)[E]) {
    float m = x[0];
#pragma unroll
    for (int e = 1; e < E; e++) m = max_of(m, x[e]);
    return m;
}

struct Given {          // a row's action and its score
    int64_t a;
    float x;
    template <typename T> __device__ __forceinline__ Given(const Actions &actions, const Row<T> &row, int64_t r, int n)
        : a(actions.at(r)), x(a >= 0 && a < n ? row.at(a) : NEG_INF) {}
};

// A wavefront's run of `bytes` bytes from LDS (at a multiple of 16) to memory, in 16-byte vectors and a rest of `unit` bytes each, by its first `lanes` lanes.
template <int UNIT> __device__ __forceinline__ void store_run(void *out, const unsigned char *run, int bytes, int lane, int lanes, bool stream) {
    unsigned char *const to = (unsigned char *)out;
    for (int at = lane * 16; at + 16 <= bytes; at += lanes * 16) {
        uint32_t v[4];
        __builtin_memcpy(v, __builtin_assume_aligned(run + at, 16), 16);
        store_bytes((uint32_t *)(to + at), v, stream);
    }
    for (int at = (bytes & ~15) + lane * UNIT; at < bytes; at += lanes * UNIT) __builtin_memcpy(to + at, run + at, UNIT);
}

// Rows in one lane put their alternatives together in LDS, as k_backward_lane does with the gradients (288296 x 18 fp16, a lane storing its own: 5
// alternatives 11.9 us, 8 17.9, 18 56; by way of LDS 12.4, 15.9, 28).
template <typename T, int G, int E, int W>
__global__ __launch_bounds__(BLOCK) void k_log_probs_short(Scores<T> sc, Actions actions, int top, float *log_prob, float *entropy,
                                                           float *top_log_probs, int32_t *top_actions) {
    static_assert(G <= 32, "the best of a group: exchanges over 32 lanes");
    using S = Spread<G, E, W>;
    extern __shared__ __align__(16) unsigned char lds_bytes[];          // (staged: [wavefronts][2][64][top])
    const int g = threadIdx.x % G, n = (int)sc.n;
    constexpr bool staged = G == 1;
    const int lane = threadIdx.x & 63;
    float *const run_log_probs = (float *)lds_bytes + (threadIdx.x >> 6) * 128 * top;
    int32_t *const run_actions = (int32_t *)(run_log_probs + 64 * top);
    for (int64_t r = (int64_t)blockIdx.x * (BLOCK / G) + threadIdx.x / G; r < sc.rows; r += (int64_t)gridDim.x * (BLOCK / G)) {
        const Row<T> row(sc, r);
        const Given given(actions, row, r, n);
        float x[E];
        S::load_row(row, g, n, x);
        const float m = group_max<G>(lane_max(x));
        const bool some = m > NEG_INF;
        const float ref = some ? m : 0.0f;
        float s = 0, t = 0;
        const auto add = [&](float d) {
            const float p = __builtin_amdgcn_exp2f(d);
            s += p;
            t = fmaf(p, fmaxf(d, -1e30f), t);          // (not open: 0 x a finite number)
        };
        if (!sc.by_halves())
#pragma unroll
            for (int e = 0; e < E; e++) add((x[e] - ref) * sc.inv_t2);
        else
#pragma unroll
            for (int e = 0; e < E; e++) add(fmaf(x[e], 0.5f, -0.5f * ref) * (2.0f * sc.inv_t2));
        s = group_sum<G>(s);
        t = group_sum<G>(t);
        const bool undefined = !(s == s);
        const float log_s = logf(s), nan = __builtin_nanf("");
        if (g == 0) {
            float lp = 0.0f;
            if (given.a >= n || (given.a >= 0 && undefined)) lp = nan;
            else if (given.a >= 0) lp = some ? sc.over_t(given.x, ref) - log_s : NEG_INF;
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
            const auto take = [&](float ov, int oi) {
                const bool b = better(ov, oi, v, i);
                v = b ? ov : v;
                i = b ? oi : i;
            };
            if constexpr (G > 1) take(dpp<DPP_XOR1>(v), dpp<DPP_XOR1>(i));
            if constexpr (G > 2) take(dpp<DPP_XOR2>(v), dpp<DPP_XOR2>(i));
            if constexpr (G > 4) take(dpp<DPP_HALF_MIRROR>(v), dpp<DPP_HALF_MIRROR>(i));
            if constexpr (G > 8) take(dpp<DPP_MIRROR>(v), dpp<DPP_MIRROR>(i));
            if constexpr (G > 16) { const auto ov = swap<16>(v); const auto oi = swap<16>(i); take(ov.a, oi.a); take(ov.b, oi.b); }
            if (k + 1 < top)
#pragma unroll
                for (int e = 0; e < E; e++) x[e] = S::place(g, e) == i ? NEG_INF : x[e];
            if (g == 0) {
                const bool there = v > NEG_INF && !undefined;
                const int action = there ? i : -1;
                const float lp = there ? sc.over_t(v, ref) - log_s : NEG_INF;
                if constexpr (staged) {
                    run_actions[lane * top + k] = action;
                    run_log_probs[lane * top + k] = lp;
                } else {
                    top_actions[r * top + k] = action;
                    top_log_probs[r * top + k] = lp;
                }
            }
        }
        if constexpr (staged)
            if (top) {          // (the lanes with a row are the wavefront's first)
                wave_sync();
                const int64_t r0 = r - lane;
                const int lanes = (int)(sc.rows - r0 < 64 ? sc.rows - r0 : 64), bytes = lanes * top * 4;
                store_run<4>(top_actions + r0 * top, (const unsigned char *)run_actions, bytes, lane, lanes, false);
                store_run<4>(top_log_probs + r0 * top, (const unsigned char *)run_log_probs, bytes, lane, lanes, false);
                wave_sync();
            }
    }
}

struct Upstream {          // gradients to the log probabilities and entropies, one value a row (stride 0: one for all), or NULL
    const float *lp, *h;
    int64_t lp_stride, h_stride;
    // (behind the last action the log probability is NaN: whatever flows back through it is, too)
    __device__ __forceinline__ float to_log_prob(int64_t r, int64_t a, int64_t n) const {
        const float g = lp && a >= 0 ? lp[r * lp_stride] : 0.0f;
        return a < n || g == 0 ? g : __builtin_nanf("");
    }
    __device__ __forceinline__ float to_entropy(int64_t r) const { return h ? h[r * h_stride] : 0.0f; }
};

// The gradient is p (c0 + c1 log2 p), with log2 p no lower than LEAST_LOG2: p is 0 there in fp32, so is the product, and -inf stays out of it.  That takes
// moderate c0 and c1: of larger ones (a gradient to the entropy over a tiny temperature) the product with log2 p overflows, and 0 x inf is NaN, or what
// fp32 has no exponential for is no longer nothing; and NaN has to stay out of the places that are not open.  Rows with such factors are worked out
// place by place in 64 bits (983040 x 18 fp32 57 us for 28, 1024 x 104976 bf16 277 for 67).
constexpr float LEAST_LOG2 = -256.0f, MODERATE = 0x1p40f;
__device__ __forceinline__ bool moderate(float c0, float c1) { return fabsf(c0) <= MODERATE && fabsf(c1) <= MODERATE; }
// (All that the row's factors were made of is read again, so that nothing stays in registers for it.)
template <typename T> struct RowGradient64 {
    const Scores<T> &sc;
    const Row<T> row;
    const int64_t a;
    const float ref, log2_s, gl, gh, h;
    __device__ __forceinline__ RowGradient64(const Scores<T> &sc_, int64_t r, const Actions &actions, const float *entropy, const Upstream &up, float ref_, float log2_s_)
        : sc(sc_), row(sc_, r), a(actions.at(r)), ref(ref_), log2_s(log2_s_), gl(up.to_log_prob(r, a, sc_.n)), gh(up.to_entropy(r)), h(entropy[r]) {}
    __device__ __forceinline__ T at(int64_t j) const {
        const float x = row.at(j);
        if (x == NEG_INF || (gl == 0 && gh == 0)) return from_f32<T>(0.0f);          // (nothing flows back into the row, be its scores what they may)
        // (nothing overflows: the factors are fp32 numbers.  Below 2^-1000 a p makes 0 of them; where it is NaN, so is h)
        const double l2 = ((double)x - ref) * sc.inv_t2_64 - log2_s, factor = (double)gl + (double)gh * (h + l2 * LN_2);
        return from_f32<T>((float)(((j == a ? (double)gl : 0.0) - Exp64(1.0)(fmax(l2, -1000.0)) * factor) * (sc.inv_t2_64 * LN_2)));
    }
};

template <typename T, int G, int E, int W>
__global__ __launch_bounds__(BLOCK) void k_backward_short(Scores<T> sc, Actions actions, const float *entropy, Upstream up, T *grad, bool stream) {
    using S = Spread<G, E, W>;
    const int g = threadIdx.x % G, n = (int)sc.n;
    const Difference diff(sc);
    for (int64_t r = (int64_t)blockIdx.x * (BLOCK / G) + threadIdx.x / G; r < sc.rows; r += (int64_t)gridDim.x * (BLOCK / G)) {
        const Row<T> row(sc, r);
        const int64_t a = actions.at(r);
        const float h = entropy[r], gl = up.to_log_prob(r, a, n), gh = up.to_entropy(r);
        float x[E];
        S::load_row(row, g, n, x);
        // maximum and sum again (cheaper than 8 bytes a row written and read)
        const float m = group_max<G>(lane_max(x)), ref = m > NEG_INF ? m : 0.0f, unit_ref = diff.unit * ref;
        float s = 0, p[E];
#pragma unroll
        for (int e = 0; e < E; e++) {
            p[e] = __builtin_amdgcn_exp2f(diff.over_t2(x[e], unit_ref));
            s += p[e];
        }
        s = group_sum<G>(s);
        // dx = p (c0 + c1 log2 p), and g_lp / T more at j = a (nothing open: s = 0, and with it both factors)
        const float inv_s = s == 0 ? 0.0f : 1.0f / s, log2_s = log2f(s), c0 = -(gl + gh * h) * sc.inv_t * inv_s, c1 = -gh * (float)LN_2 * sc.inv_t * inv_s;
        T *to = grad + r * sc.n;
        if (moderate(c0, c1)) {
#pragma unroll
            for (int e = 0; e < E; e += W) {
                T out[W];
#pragma unroll
                for (int k = 0; k < W; k++) out[k] = from_f32<T>(p[e + k] * fmaf(c1, fmaxf(diff.over_t2(x[e + k], unit_ref) - log2_s, LEAST_LOG2), c0));
                Pieces<T, W, 1>::store(to, S::place(g, e), n, e / W < n / (G * W), out, stream);
            }
            if (a >= 0 && a < n && (int)(a / W) % G == g) {          // (the lane that has just written this place)
                const float xa = row.at(a), d = diff.over_t2(xa, unit_ref), pa = __builtin_amdgcn_exp2f(d);
                to[a] = from_f32<T>(xa == NEG_INF ? 0.0f : fmaf(pa, fmaf(c1, fmaxf(d - log2_s, LEAST_LOG2), c0), gl * sc.inv_t));
            }
        } else {
            const RowGradient64<T> exact(sc, r, actions, entropy, up, ref, log2_s);
#pragma unroll 1
            for (int j = g; j < n; j += G) to[j] = exact.at(j);
        }
    }
}

// Up to 32 scores a row, a lane each.  The gradients of a wavefront's 64 rows are one run of memory: they are put together in LDS and stored in 16-byte
// vectors, neighbours by neighbours (983040 rows of 18 fp32: 28 us; a lane storing its own row writes 16 bytes every 72: 130; four lanes a row, a
// score a store: 37).
template <typename T, int G, int E, int W>
__global__ __launch_bounds__(BLOCK) void k_backward_lane(Scores<T> sc, Actions actions, const float *entropy, Upstream up, T *grad, bool stream) {
    static_assert(G == 1);
    extern __shared__ __align__(16) unsigned char lds_bytes[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = (int)sc.n;
    const Difference diff(sc);
    T *const mine = (T *)lds_bytes + (wave * 64 + lane) * n;
    const unsigned char *const run = lds_bytes + wave * 64 * n * sizeof(T);
    for (int64_t r0 = ((int64_t)blockIdx.x * WAVES + wave) * 64; r0 < sc.rows; r0 += (int64_t)gridDim.x * BLOCK) {
        const int64_t r = r0 + lane;
        if (r < sc.rows) {
            const Row<T> row(sc, r);
            const Given given(actions, row, r, n);
            const float h = entropy[r], gl = up.to_log_prob(r, given.a, n), gh = up.to_entropy(r);
            float x[E];
            Spread<1, E, W>::load_row(row, 0, n, x);
            const float m = lane_max(x), ref = m > NEG_INF ? m : 0.0f, unit_ref = diff.unit * ref;
            float s = 0, p[E];
#pragma unroll
            for (int e = 0; e < E; e++) {
                p[e] = __builtin_amdgcn_exp2f(diff.over_t2(x[e], unit_ref));
                s += p[e];
            }
            const float inv_s = s == 0 ? 0.0f : 1.0f / s, log2_s = log2f(s), c0 = -(gl + gh * h) * sc.inv_t * inv_s, c1 = -gh * (float)LN_2 * sc.inv_t * inv_s;
#pragma unroll
            for (int e = 0; e < E; e++)
                if (e < n) mine[e] = from_f32<T>(p[e] * fmaf(c1, fmaxf(diff.over_t2(x[e], unit_ref) - log2_s, LEAST_LOG2), c0));
            if (given.a >= 0 && given.a < n) {
                const float d = diff.over_t2(given.x, unit_ref), pa = __builtin_amdgcn_exp2f(d);
                mine[given.a] = from_f32<T>(given.x == NEG_INF ? 0.0f : fmaf(pa, fmaf(c1, fmaxf(d - log2_s, LEAST_LOG2), c0), gl * sc.inv_t));
            }
            if (!moderate(c0, c1)) {
                const RowGradient64<T> exact(sc, r, actions, entropy, up, ref, log2_s);
#pragma unroll 1
                for (int j = 0; j < n; j++) mine[j] = exact.at(j);
            }
        }
        wave_sync();
        const int bytes = (int)(sc.rows - r0 < 64 ? sc.rows - r0 : 64) * n * (int)sizeof(T);
        store_run<(int)sizeof(T)>(grad + r0 * n, run, bytes, lane, 64, stream);
        wave_sync();
    }
}

__device__ __forceinline__ double uniform_at(const void *uniforms, int bytes, int64_t r) {
    const double u = bytes == 8 ? ((const double *)uniforms)[r] : (double)((const float *)uniforms)[r];
    return u > 0.0 ? (u < 1.0 ? u : 1.0) : 0.0;          // (NaN: 0)
}
struct Drawn {
    int32_t *action;
    float *log_prob, *entropy;          // either may be NULL
    __device__ __forceinline__ void put(int64_t r, int a, float lp, float h) const {
        action[r] = a;
        if (log_prob) log_prob[r] = lp;
        if (entropy) entropy[r] = h;
    }
};

// The place, among the E of the lane that a draw falls into, that passes the target (else the last one with anything in it), and its score.
template <int E> __device__ __forceinline__ int in_lane(const float (&x)[E], const double (&p)[E], double c, double target, float &xa) {
    int a = -1;
    bool found = false;
#pragma unroll
    for (int e = 0; e < E; e++) {
        c += p[e];
        if (p[e] > NOTHING && !found) { a = e; xa = x[e]; found = c > target; }
    }
    if (a < 0)          // (each below NOTHING, their sum above it: the first one that is open)
#pragma unroll
        for (int e = E - 1; e >= 0; e--)
            if (x[e] > NEG_INF) { a = e; xa = x[e]; }
    return a;
}

// Lane g holds the E consecutive scores from g * E on: a running sum in index order is a lane's sum, a scan over the lanes, and a second
// look at the one lane in which the target lies.
template <typename T, int G, int E, int W>
__global__ __launch_bounds__(BLOCK) void k_sample_short(Scores<T> sc, const void *uniforms, int uniform_bytes, Drawn out) {
    const int g = threadIdx.x % G, n = (int)sc.n;
    for (int64_t r = (int64_t)blockIdx.x * (BLOCK / G) + threadIdx.x / G; r < sc.rows; r += (int64_t)gridDim.x * (BLOCK / G)) {
        const Row<T> row(sc, r);
        const double u = uniform_at(uniforms, uniform_bytes, r);
        float x[E];
        {
            Pieces<T, W, E / W, G == 1> p;
            p.load(row, n, G == 1 ? n / W : n / (G * E) * (E / W), E / W, [&](int k) { return g * E + k * W; });
            p.scores(row, x);
        }
        const float m = group_max<G>(lane_max(x));
        const bool some = m > NEG_INF;
        const double ref = some ? m : 0.0;
        const Exp64 exp64(sc.inv_t2_64);
        double p[E], s = 0, t = 0;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const double d = exp64.below(x[e], ref);
            p[e] = exp64(d);
            s += p[e];
            t = fma(p[e], d, t);
        }
        const double upto = group_scan<G>(s, g), total = __shfl(upto, G - 1, G);
        t = group_sum<G>(t);
        const int group = (threadIdx.x & 63) - g;
        const uint64_t in_group = G == 64 ? ~0ull : ((1ull << (G & 63)) - 1) << group;
        const bool undefined = m != m || m == -NEG_INF, none = undefined || !some;
        const double target = u * total;
        // the first lane that passes the target, or else (rounding; a number of 1) the last one with anything in it
        const uint64_t past = __ballot(s > NOTHING && upto > target) & in_group, any = __ballot(s > NOTHING) & in_group;
        const int owner = none ? group : past ? first_lane(past) : last_lane(any);
        if ((threadIdx.x & 63) == owner) {
            const double c = g == 0 ? 0.0 : upto - s;
            float xa = 0;
            const int a = g * E + in_lane(x, p, c, target, xa);
            const double log_s = log(total);
            const float nil = undefined ? __builtin_nanf("") : NEG_INF;
            out.put(r, none ? -1 : a, none ? nil : (float)(((double)xa - ref) * sc.inv_t2_64 * LN_2 - log_s),
                    undefined ? nil : some ? (float)(log_s - t / total * sc.inv_t2_64 * LN_2) : 0.0f);
        }
    }
}

// ----------------------------------------------------------------------------------------------------------------- long rows
// A wavefront or workgroup goes over a row, or over one part of it where there are few rows, in tiles of U 16-byte vectors a lane: running
// maximum, sum and weighted sum per lane, joined at the end; every score is read once.  What bounds it: memory (1024 x 104976 bf16, 215 MB: 37.6 us, part
// of them from the cache, 43 ... 46 after other work; backward 66, 67 ... 74 after other work, for 430 MB), with masks and alternatives the vector unit
// too (4096 x 5832 bf16, a mask, five alternatives: 22 us, 13 of them issued, where memory would take 14), and with few rows two launches, each a
// chain of load, exchange and rank (7 x 50021 fp32, 20 alternatives: 8 and 5 us under the profiler).  Loading the next tile ahead of the present one's
// arithmetic made it slower when it was tried (58 -> 64 and 22 -> 28 us): registers, and other wavefronts hide the loads already.

// ROW_WAVES: wavefronts that go over the tile together (1, or the workgroup's 4)
template <typename T, int ROW_WAVES, int VECTORS = 4> struct Tile {
    static constexpr int V = 16 / sizeof(T), U = VECTORS, LANES = 64 * ROW_WAVES, SIZE = LANES * U * V;
    static __device__ __forceinline__ int lane() { return (int)threadIdx.x % LANES; }
    static __device__ __forceinline__ int wave() { return ROW_WAVES == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6); }
    // vector u of a tile in this lane: a wavefront's 64 vectors are neighbours, and its places ascend with the tile and u
    static __device__ __forceinline__ int64_t place(int64_t tile, int u) { return tile * SIZE + (u * LANES + lane()) * V; }
    Pieces<T, V, U> p;
    __device__ __forceinline__ void load(const Row<T> &row, int64_t tile, int n) {
        p.load(row, n, (int)((n - tile * SIZE) / (LANES * V)), live(tile, n), [&](int u) { return (int)place(tile, u); });
    }
    // how many of its U vectors begin inside the row in some lane of this wavefront
    static __device__ __forceinline__ int live(int64_t tile, int n) { return (int)((n - tile * SIZE - wave() * 64 * V + LANES * V - 1) / (LANES * V)); }
    static __host__ __device__ __forceinline__ int count(int64_t n) { return (int)((n + SIZE - 1) / SIZE); }
};

// Maximum m, s = sum 2^d, t = sum d 2^d with d = (x - m) log2(e) / T, of scores seen so far (none: m = -inf, s = t = 0).  A NaN or +inf among
// them makes s NaN.
struct Softmax {
    float m = NEG_INF, s = 0, t = 0;
    __device__ __forceinline__ void to(float new_m, const Difference &diff) {          // the same scores against a larger maximum
        const float d = diff.over_t2(m, diff.unit * new_m), c = __builtin_amdgcn_exp2f(d);
        t = s == 0 ? 0 : c * fmaf(fmaxf(d, -1e30f), s, t);
        s = s == 0 ? 0 : c * s;
        m = new_m;
    }
    __device__ __forceinline__ void join(Softmax o, const Difference &diff) {
        const float top = fmaxf(m, o.m);
        if (top > NEG_INF) { to(top, diff); o.to(top, diff); }
        s += o.s;
        t += o.t;
    }
    __device__ __forceinline__ void join_wave(const Difference &diff) {
        const float top = group_max<64>(m);
        if (top > NEG_INF) to(top, diff);
        s = group_sum<64>(s);
        t = group_sum<64>(t);
    }
};

// The best alternatives a wavefront has seen, as 64-bit keys: the score's order in the upper half (larger is better), the index's complement in
// the lower (equal scores: the lower index).  0 is none.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);          // (+ 0: the two zeros are one score)
    return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float score_of(uint32_t order) { return __builtin_bit_cast(float, order ^ (order >> 31 ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ uint64_t key_of(float x, int j) { return x > NEG_INF ? (uint64_t)order_of(x) << 32 | (uint32_t)~j : 0; }
__device__ __forceinline__ int index_of(uint64_t key) { return (int)~(uint32_t)key; }

// It collects, in LDS and unsorted, whatever beats the k-th best it knows (k <= 64); when that gets full, and at the end, every key's rank is
// counted and the k best stay, in order.  (Keeping a sorted list and pushing scores in one by one took five times as long: a chain of
// dependent exchanges for each, and unrolled over a tile's 32 scores a lane more code than the instruction cache likes.)
struct Top {
    static constexpr int CAPACITY = 128;
    uint64_t *keys;          // LDS [CAPACITY], the wavefront's own
    uint64_t bound = 0;      // what a key has to exceed
    int count = 0, k;
    __device__ Top(uint64_t *lds, int k_) : keys(lds), k(k_) {}
    // Before the first offers: x are N scores that each lane is going to offer, the best of some each.  The k-th best of these 64 N bounds the
    // k-th best of all from below; found bit by bit (16 of them: the bound may be lower), it keeps most of the scores out that would not last.
    // For one alternative it is the best of them.  (32768 x 2500 bf16: 47 us, bit by bit 54.)
    template <int N> __device__ __forceinline__ void expect(const float (&x)[N]) {
        if (k == 1) {
            const float most = group_max<64>(lane_max(x));
            if (most > NEG_INF) bound = ((uint64_t)order_of(most) << 32) - 1;
            return;
        }
        uint32_t order[N], at_least = 0;
#pragma unroll
        for (int i = 0; i < N; i++) order[i] = x[i] > NEG_INF ? order_of(x[i]) >> 16 : 0;
        for (uint32_t bit = 0x8000; bit; bit >>= 1) {
            int reach = 0;
#pragma unroll
            for (int i = 0; i < N; i++) reach += __popcll(__ballot(order[i] >= (at_least | bit)));
            if (reach >= k) at_least |= bit;
        }
        if (at_least) bound = ((uint64_t)at_least << 48) - 1;
    }
    // the least score that can still get in, offered from further on in the row (an equal one with a lower index could too: there are none);
    // one up from the bound's, and never -inf, which is not open
    __device__ __forceinline__ float least_score() const { return fmaxf(score_of((uint32_t)(bound >> 32) + 1), -FLT_MAX); }          // (no bound: a NaN's bits)
    // every lane offers one key (0: none)
    __device__ __forceinline__ void offer(uint64_t key) {
        uint64_t who = __ballot(key > bound);
        if (!who) return;
        if (count + __popcll(who) > CAPACITY) {
            sort();
            who = __ballot(key > bound);
        }
        const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
        if (key > bound) keys[count + before] = key;
        count += __popcll(who);
        wave_sync();
    }
    // the k best in order
    __device__ __forceinline__ void sort() {
        const int lane = threadIdx.x & 63;
        const uint64_t a = lane < count ? keys[lane] : 0, b = lane + 64 < count ? keys[lane + 64] : 0;
        int rank_a = 0, rank_b = 0;
#pragma unroll 4
        for (int c = 0; c < count; c++) {
            const uint64_t other = keys[c];
            rank_a += other > a;
            rank_b += other > b;
        }
        wave_sync();
        if (a && rank_a < k) keys[rank_a] = a;
        if (b && rank_b < k) keys[rank_b] = b;
        wave_sync();
        if (count >= k) {
            count = k;
            bound = keys[k - 1];
        }
    }
};

struct LogProbOut {
    float *log_prob, *entropy, *stats, *top_log_probs;
    int32_t *top_actions;
    int top;
};

// a row's results from its sums (one lane) and its best (one wavefront; sorted)
template <typename T> __device__ __forceinline__ void finish_row(const Scores<T> &sc, int64_t r, const Given &given, const Softmax &all,
                                                                 const Top &best, const LogProbOut &out) {
    const int lane = threadIdx.x & 63, n = (int)sc.n;
    const bool some = all.m > NEG_INF, undefined = !(all.s == all.s);
    const float ref = some ? all.m : 0.0f, log_s = logf(all.s), nan = __builtin_nanf("");
    if (lane == 0) {
        float lp = 0.0f;
        if (given.a >= n || (given.a >= 0 && undefined)) lp = nan;
        else if (given.a >= 0) lp = some ? sc.over_t(given.x, ref) - log_s : NEG_INF;
        out.log_prob[r] = lp;
        out.entropy[r] = undefined ? nan : some ? log_s - all.t / all.s * (float)LN_2 : 0.0f;
        if (out.stats) { out.stats[2 * r] = ref; out.stats[2 * r + 1] = all.s == 0 ? 0.0f : log2f(all.s); }
    }
    if (lane < out.top) {
        const bool there = lane < best.count && !undefined;
        const uint64_t key = there ? best.keys[lane] : 0;
        out.top_actions[r * out.top + lane] = there ? index_of(key) : -1;
        out.top_log_probs[r * out.top + lane] = there ? sc.over_t(score_of((uint32_t)(key >> 32)), ref) - log_s : NEG_INF;
    }
}

// What the parts of a row leave for the join: [rows][parts][top] keys and [rows][parts][4] sums.
struct Partials {
    uint64_t *keys;
    float *sums;
};

// One wavefront (ROW_WAVES 1) or workgroup (4) goes over a row; SPLIT: a workgroup over blockIdx.x-th part of part_tiles tiles of it.
template <typename T, bool TOP, int ROW_WAVES, bool SPLIT>
__global__ __launch_bounds__(BLOCK) void k_log_probs_long(Scores<T> sc, Actions actions, LogProbOut out, int part_tiles, Partials to, Difference diff) {
    using L = Tile<T, ROW_WAVES>;
    __shared__ float lds[WAVES][3];
    __shared__ uint64_t lds_keys[TOP ? WAVES : 1][TOP ? Top::CAPACITY : 1];
    __shared__ int lds_count[WAVES];
    __shared__ uint4 lds_scores[TOP ? BLOCK : 1][TOP ? L::U : 1];
    const int n = (int)sc.n, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), top = TOP ? out.top : 0;
    const int first = SPLIT ? (int)blockIdx.x * part_tiles : 0, behind = SPLIT ? min(first + part_tiles, L::count(n)) : L::count(n);
    constexpr int ROWS = WAVES / ROW_WAVES;          // of a workgroup
    const int64_t r0 = (SPLIT ? blockIdx.y : (int64_t)blockIdx.x * ROWS) + (ROW_WAVES == 1 ? wave : 0);
    for (int64_t r = r0; r < sc.rows; r += SPLIT ? gridDim.y : (int64_t)gridDim.x * ROWS) {
        const Row<T> row(sc, r);
        const Given given(actions, row, r, n);
        Softmax a;
        Top best(lds_keys[TOP ? wave : 0], TOP ? top : 1);
        for (int tile = first; tile < behind; tile++) {
            L now;
            now.load(row, tile, n);
            float x[L::U * L::V], um[L::U];
            now.p.scores(row, x);
#pragma unroll
            for (int u = 0; u < L::U; u++) {
                um[u] = x[u * L::V];
#pragma unroll
                for (int k = 1; k < L::V; k++) um[u] = max_of(um[u], x[u * L::V + k]);
            }
            const float m = lane_max(um);
            if (m > a.m) a.to(m, diff);
            const float ref = a.m > NEG_INF ? diff.unit * a.m : 0.0f;
            const int live = L::live(tile, n);
            float s = 0, t = 0;          // (the tile's own: scores next to nothing each are added up before they meet a large sum)
#pragma unroll
            for (int u = 0; u < L::U; u++)
                if (u < live)
#pragma unroll
                    for (int k = u * L::V; k < (u + 1) * L::V; k++) {
                        const float d = diff.over_t2(x[k], ref), p = __builtin_amdgcn_exp2f(d);
                        s += p;
                        t = fmaf(p, fmaxf(d, -1e30f), t);
                    }
            a.s += s;
            a.t += t;
            if constexpr (TOP) {
                if (tile == first) best.expect(um);
                const float least = best.least_score();          // (the wavefront's places ascend with the tiles; expect()'s bound lies between two scores)
                if (__ballot(m >= least)) {
                    uint32_t mine = 0;          // which of the lane's scores are in question; taken one by one, by way of LDS (its own place: no waits)
#pragma unroll
                    for (int k = L::U * L::V - 1; k >= 0; k--) mine = mine + mine + (x[k] >= least);
                    if (mine)
#pragma unroll
                        for (int u = 0; u < L::U; u++) __builtin_memcpy(&lds_scores[threadIdx.x][u], now.p.w[u], 16);
                    while (__ballot(mine != 0)) {
                        const int k = __ffs((int)mine) - 1, j = (int)L::place(tile, k / L::V) + k % L::V;
                        T score;
                        __builtin_memcpy(&score, (const unsigned char *)lds_scores[threadIdx.x] + (mine ? k : 0) * sizeof(T), sizeof(T));
                        best.offer(mine ? key_of(to_f32(score), j) : 0);
                        mine &= mine - 1;
                    }
                }
            }
        }
        a.join_wave(diff);
        if constexpr (ROW_WAVES == 1) {
            if constexpr (TOP) best.sort();
            finish_row(sc, r, given, a, best, out);
            wave_sync();
        } else {
            __syncthreads();
            if (lane == 0) { lds[wave][0] = a.m; lds[wave][1] = a.s; lds[wave][2] = a.t; lds_count[wave] = best.count; }
            __syncthreads();
            if (wave == 0) {
                for (int w = 1; w < WAVES; w++) {
                    Softmax o;
                    o.m = lds[w][0];
                    o.s = lds[w][1];
                    o.t = lds[w][2];
                    a.join(o, diff);
                    if constexpr (TOP)
                        for (int c = 0; c < lds_count[w]; c += 64) best.offer(c + lane < lds_count[w] ? lds_keys[w][c + lane] : 0);
                }
                if constexpr (TOP) best.sort();
                if constexpr (SPLIT) {
                    const int64_t b = r * gridDim.x + blockIdx.x;
                    if (lane == 0) { to.sums[b * 4] = a.m; to.sums[b * 4 + 1] = a.s; to.sums[b * 4 + 2] = a.t; }
                    if (lane < top) to.keys[b * top + lane] = lane < best.count ? best.keys[lane] : 0;
                } else finish_row(sc, r, given, a, best, out);
            }
            __syncthreads();
        }
    }
}

// one wavefront a row: the parts' sums and best
template <typename T>
__global__ __launch_bounds__(64) void k_log_probs_join(Scores<T> sc, Actions actions, LogProbOut out, int parts, Partials from) {
    __shared__ uint64_t lds_keys[Top::CAPACITY];
    const int lane = threadIdx.x, top = out.top;
    const Difference diff(sc);
    for (int64_t r = blockIdx.x; r < sc.rows; r += gridDim.x) {
        const uint64_t *keys = from.keys + r * parts * top;
        const float *sums = from.sums + r * parts * 4;
        const Given given(actions, Row<T>(sc, r), r, (int)sc.n);
        Softmax a;
        for (int p = lane; p < parts; p += 64) {
            Softmax o;
            o.m = sums[p * 4];
            o.s = sums[p * 4 + 1];
            o.t = sums[p * 4 + 2];
            a.join(o, diff);
        }
        a.join_wave(diff);
        Top best(lds_keys, top ? top : 1);
        if (top) {
            for (int c0 = 0; c0 < parts * top; c0 += 512) {          // eight keys a lane at a time
                uint64_t key[8];
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const int c = c0 + k * 64 + lane;
                    key[k] = c < parts * top ? keys[c] : 0;
                }
                if (c0 == 0) {          // (64 samples bound up to half as many well; eight times as many take eight times as long)
                    float x[8];
#pragma unroll
                    for (int k = 0; k < 8; k++) x[k] = key[k] ? score_of((uint32_t)(key[k] >> 32)) : NEG_INF;
                    const float most[1] = {lane_max(x)};
                    if (top <= 32) best.expect(most);
                    else best.expect(x);
                }
                for (int k = 0; k < 8; k++) {
                    uint64_t v = key[0];
#pragma unroll
                    for (int i = 0; i < 7; i++) key[i] = key[i + 1];
                    best.offer(v);
                }
            }
            best.sort();
        }
        finish_row(sc, r, given, a, best, out);
        wave_sync();
    }
}

// blockIdx.x: the tile, of a wavefront (ROW_WAVES 1, four rows a workgroup) or a workgroup (4)
template <typename T, int ROW_WAVES, int U>
__global__ __launch_bounds__(BLOCK) void k_backward_long(Scores<T> sc, Actions actions, const float *stats, const float *entropy, Upstream up,
                                                         T *grad, bool stream) {
    using L = Tile<T, ROW_WAVES, U>;
    constexpr int ROWS = WAVES / ROW_WAVES;
    const int n = (int)sc.n;
    const Difference diff(sc);
    for (int64_t r = (int64_t)blockIdx.y * ROWS + (ROW_WAVES == 1 ? __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) : 0); r < sc.rows;
         r += (int64_t)gridDim.y * ROWS) {
        const Row<T> row(sc, r);
        // (the row's own values are asked for before its scores: they come in that order, and 1024 x 104976 bf16 takes 66 us, the other way round 76)
        const int64_t a = actions.at(r);
        const float unit_ref = diff.unit * stats[2 * r], log2_s = stats[2 * r + 1], h = entropy[r];
        const float gl = up.to_log_prob(r, a, n), gh = up.to_entropy(r);
        // dx = p (c0 + c1 log2 p), and g_lp / T more at j = a
        const float c0 = -(gl + gh * h) * sc.inv_t, c1 = -gh * (float)LN_2 * sc.inv_t;
        L tile;
        tile.load(row, blockIdx.x, n);
        float x[L::U * L::V];
        tile.p.scores(row, x);
        T *to = grad + r * sc.n;
        const int live = L::live(blockIdx.x, n);
#pragma unroll
        for (int u = 0; u < L::U; u++) {
            if (u >= live) break;
            const int64_t j = L::place(blockIdx.x, u);
            T v[L::V];
#pragma unroll
            for (int k = 0; k < L::V; k++) {
                const float l2 = fmaf(diff(x[u * L::V + k], unit_ref), diff.per_t2, -log2_s);
                v[k] = from_f32<T>(__builtin_amdgcn_exp2f(l2) * fmaf(c1, fmaxf(l2, LEAST_LOG2), c0));
            }
            if (j < n) Pieces<T, L::V, 1>::store(to, (int)j, n, false, v, stream);
            if (a >= j && a < j + L::V && a < n) {          // (the lane that has just written this place)
                const float xa = row.at(a), l2 = fmaf(diff(xa, unit_ref), diff.per_t2, -log2_s);
                to[a] = from_f32<T>(xa == NEG_INF ? 0.0f : fmaf(__builtin_amdgcn_exp2f(l2), fmaf(c1, fmaxf(l2, LEAST_LOG2), c0), gl * sc.inv_t));
            }
        }
        if (__ballot(!moderate(c0, c1))) {          // (one row a wavefront: a scalar branch.  Over what has just been written, each lane its own)
            const RowGradient64<T> exact(sc, r, actions, entropy, up, stats[2 * r], stats[2 * r + 1]);
#pragma unroll 1
            for (int i = 0; i < L::U * L::V; i++) {
                const int64_t j = L::place(blockIdx.x, i / L::V) + i % L::V;
                if (j < n) to[j] = exact.at(j);
            }
        }
    }
}

// ---- drawing: the row's segments of 64 vectors (one a lane), each with its own maximum and 64-bit sums, then the one segment the target lies in,
// read once more.  What bounds it: the 64-bit exponentials, 20 instructions each (4096 x 5832 bf16: 28 us, of which the vector unit issues
// for 21; memory would take 9); with few rows two launches (16 x 104976 fp32: 11.0 us).  32 bits would not do: a border between two actions is off by
// some 2^-24 there, and with ten thousand actions a random number lies that close to one every thousandth time.
struct Segment {
    double s, t;        // sums of the exponentials, and of these times their differences to the maximum
    float m;            // its maximum (-inf: nothing open; NaN: there is one)
};

// The segments of a wavefront's vectors of a tile: (tile, u, wave) is segment (tile * U + u) * ROW_WAVES + wave.  put(segment, its sums) for
// each that there is; t of all of them, against one maximum, comes with the last.
template <typename T, int ROW_WAVES, typename F>
__device__ __forceinline__ void sum_segments(const Row<T> &row, int n, const Exp64 &exp64, int tile, Tile<T, ROW_WAVES> &now, F put) {
    using L = Tile<T, ROW_WAVES>;
    const int live = min(L::live(tile, n), (int)L::U);
    float x[L::U * L::V];
    now.p.scores(row, x);
    const float m = group_max<64>(lane_max(x));
    const double ref = m > NEG_INF ? m : 0.0;
    double t = 0;
#pragma unroll
    for (int u = 0; u < L::U; u++) {
        if (u >= live) break;
        double s = 0;
#pragma unroll
        for (int k = 0; k < L::V; k++) {
            const double d = exp64.below(x[u * L::V + k], ref), p = exp64(d);
            s += p;
            t = fma(p, d, t);
        }
        s = group_sum<64>(s);
        if (u + 1 == live) t = group_sum<64>(t);
        put((tile * L::U + u) * ROW_WAVES + L::wave(), Segment{s, u + 1 == live ? t : 0.0, m});
    }
}

// One wavefront: the row's action.  Every lane has a run of `each` neighbouring segments from lane * each on; of(k) is its k-th (empty from
// `each` on), and again(run, k) the k-th of another lane's.  STEP segments are looked at together.
template <int STEP, typename T, typename F, typename A>
__device__ __forceinline__ void draw(const Scores<T> &sc, const Row<T> &row, const Exp64 &exp64, int64_t r, int each, F of, A again, double u, const Drawn &out) {
    constexpr int V = 16 / sizeof(T);
    const int lane = threadIdx.x & 63, n = (int)sc.n;
    float m = NEG_INF;
    for (int k = 0; k < each; k += STEP) {
        Segment g[STEP];
#pragma unroll
        for (int i = 0; i < STEP; i++) g[i] = of(k + i);
#pragma unroll
        for (int i = 0; i < STEP; i++) m = max_of(m, g[i].m);
    }
    m = group_max<64>(m);
    const bool some = m > NEG_INF, undefined = m != m || m == -NEG_INF;
    if (undefined || !some) {
        if (lane == 0) out.put(r, -1, undefined ? __builtin_nanf("") : NEG_INF, undefined ? __builtin_nanf("") : 0.0f);
        return;
    }
    const double ref = m;
    double s = 0, t = 0;
    for (int k = 0; k < each; k += STEP) {
        Segment g[STEP];
#pragma unroll
        for (int i = 0; i < STEP; i++) g[i] = of(k + i);
#pragma unroll
        for (int i = 0; i < STEP; i++) {
            const double d = exp64.below(g[i].m, ref), w = exp64(d);
            s += or_nothing(w * g[i].s);          // (a run of segments in which nothing is open is to have a sum of 0)
            t = fma(w, fma(d, g[i].s, g[i].t), t);
        }
    }
    double upto = group_scan<64>(s, lane);
    const double total = lane_of(upto, 63);
    t = group_sum<64>(t);
    const double target = u * total;
    // the first run that passes the target, or else (rounding; a number of 1) the last one with anything in it; then the segment in it
    uint64_t past = __ballot(s > 0 && upto > target), any = __ballot(s > 0);
    const int run = past ? first_lane(past) : last_lane(any);
    double before = lane_of(lane == 0 ? 0.0 : upto - s, run), found_before = before;
    int found = run * each;
    if (each > 1)
        for (int k0 = 0; k0 < each; k0 += 64) {
            const Segment g = k0 + lane < each ? again(run, k0 + lane) : Segment{0, 0, NEG_INF};
            const double w = or_nothing(exp64(exp64.below(g.m, ref)) * g.s), sum = group_scan<64>(w, lane);
            past = __ballot(w > 0 && before + sum > target);
            any = __ballot(w > 0);
            if (any) {
                const int k = past ? first_lane(past) : last_lane(any);
                found = run * each + k0 + k;
                found_before = before + lane_of(lane == 0 ? 0.0 : sum - w, k);
            }
            if (past) break;
            before += lane_of(sum, 63);
        }
    // ... and the action in the segment
    const int64_t j = ((int64_t)found * 64 + lane) * V;
    Pieces<T, V, 1> piece;
    piece.load(row, n, 0, 1, [&](int) { return (int)j; });
    float x[V];
    piece.scores(row, x);
    double p[V];
    s = 0;
#pragma unroll
    for (int k = 0; k < V; k++) {
        p[k] = exp64(exp64.below(x[k], ref));
        s += p[k];
    }
    upto = group_scan<64>(s, lane);
    past = __ballot(s > NOTHING && found_before + upto > target);
    any = __ballot(s > NOTHING);
    if (!any) {          // (the segment's sum is above NOTHING and none of its lanes': the first one with something open)
        bool open = false;
#pragma unroll
        for (int k = 0; k < V; k++) open |= x[k] > NEG_INF;
        past = __ballot(open);
    }
    const int owner = past ? first_lane(past) : last_lane(any);
    if (lane == owner) {
        float xa = 0;
        const int k = in_lane(x, p, found_before + (lane == 0 ? 0.0 : upto - s), target, xa);
        const double log_s = log(total);
        out.put(r, (int)j + k, (float)(((double)xa - ref) * sc.inv_t2_64 * LN_2 - log_s), (float)(log_s - t / total * sc.inv_t2_64 * LN_2));
    }
}

// rows of up to 64 segments: one wavefront each, lane i keeps the i-th segment's sums
template <typename T>
__global__ __launch_bounds__(BLOCK) void k_sample_wave(Scores<T> sc, const void *uniforms, int uniform_bytes, Drawn out) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const Exp64 exp64(sc.inv_t2_64);
    for (int64_t r = (int64_t)blockIdx.x * WAVES + wave; r < sc.rows; r += (int64_t)gridDim.x * WAVES) {
        const Row<T> row(sc, r);
        const double u = uniform_at(uniforms, uniform_bytes, r);
        Segment mine{0, 0, NEG_INF};
        const int n = (int)sc.n;
        for (int tile = 0; tile < Tile<T, 1>::count(n); tile++) {
            Tile<T, 1> now;
            now.load(row, tile, n);
            sum_segments(row, n, exp64, tile, now, [&](int g, const Segment &v) {
                mine.s = lane == g ? v.s : mine.s;
                mine.t = lane == g ? v.t : mine.t;
                mine.m = lane == g ? v.m : mine.m;
            });
        }
        draw<1>(sc, row, exp64, r, 1, [&](int) { return mine; }, [&](int, int) { return mine; }, u, out);
    }
}

// longer rows: workgroups sum a tile each, a wavefront draws
template <typename T>
__global__ __launch_bounds__(BLOCK) void k_sample_parts(Scores<T> sc, int segments, Segment *workspace) {
    using L = Tile<T, WAVES>;
    const Exp64 exp64(sc.inv_t2_64);
    for (int64_t r = blockIdx.y; r < sc.rows; r += gridDim.y) {
        const Row<T> row(sc, r);
        Segment *to = workspace + r * segments;
        L now;
        now.load(row, blockIdx.x, (int)sc.n);
        sum_segments(row, (int)sc.n, exp64, (int)blockIdx.x, now, [&](int g, const Segment &v) { if ((threadIdx.x & 63) == 0) to[g] = v; });
    }
}
constexpr int LDS_SEGMENTS = 512;          // as many are looked at in LDS
template <typename T>
__global__ __launch_bounds__(BLOCK) void k_draw(Scores<T> sc, const void *uniforms, int uniform_bytes, Drawn out, int segments, const Segment *workspace) {
    __shared__ Segment lds[LDS_SEGMENTS];
    const Exp64 exp64(sc.inv_t2_64);
    for (int64_t r = blockIdx.x; r < sc.rows; r += gridDim.x) {
        const double u = uniform_at(uniforms, uniform_bytes, r);
        const Segment *seg = workspace + r * segments;
        if (segments <= LDS_SEGMENTS) {
            for (int g = threadIdx.x; g < segments; g += BLOCK) lds[g] = seg[g];
            seg = lds;
        }
        __syncthreads();
        const int lane = threadIdx.x, each = (segments + 63) / 64;
        const auto at = [&](int run, int k) {
            const int g = run * each + k;
            return k < each && g < segments ? seg[g] : Segment{0, 0, NEG_INF};
        };
        if (threadIdx.x < 64) draw<8>(sc, Row<T>(sc, r), exp64, r, each, [&](int k) { return at(lane, k); }, at, u, out);
        __syncthreads();
    }
}

thread_local char g_err[256] = "";          // (no allocation: nothing may throw across the C boundary)
int fail(int code, const char *msg) { snprintf(g_err, sizeof g_err, "%s", msg); return code; }
// an error of HIP's: reported here, and not again by the next call, another library's, that asks for the last one
int fail_hip(const char *msg) { (void)hipGetLastError(); return fail(MGX_ERR_HIP, msg); }

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
    return {(const T *)logits, mask, rows, n, row_stride, mask_row_stride, (float)(1.0 / temperature), (float)(LOG2_E / temperature), LOG2_E / temperature};
}

// a grid of at most 2^32 work items; the kernels go on from there in strides of the grid (its last dimension)
template <typename... P, typename... A> int launch_lds(void (*kernel)(P...), dim3 blocks, int threads, int lds, void *stream, A... args) {
    void *ptrs[] = {(void *)&args...};
    static_assert(sizeof...(P) == sizeof...(A) && (std::is_same_v<P, A> && ...), "argument types are the kernel's");
    const int64_t most = 0xffffffffLL / threads;
    if (blocks.y > most / blocks.x) blocks.y = (unsigned)(most / blocks.x);
    const hipError_t err = hipLaunchKernel((const void *)kernel, blocks, dim3(threads), ptrs, (size_t)lds, (hipStream_t)stream);
    return err == hipSuccess ? (int)MGX_OK : fail_hip(hipGetErrorString(err));
}
template <typename... P, typename... A> int launch(void (*kernel)(P...), dim3 blocks, int threads, void *stream, A... args) {
    return launch_lds(kernel, blocks, threads, 0, stream, args...);
}
template <typename... P, typename... A> int launch(void (*kernel)(P...), int64_t blocks, int threads, void *stream, A... args) {
    return launch(kernel, dim3((unsigned)std::min<int64_t>(blocks, 0xffffffffLL / threads)), threads, stream, args...);
}

// Gradients of this size go past the caches: a quarter of the 256 MB that memory has in front of it would be filled with what is read
// once, much later, and written back while the next kernels read.  1024 x 104976 bf16 (215 MB): backward 78 -> 67 us, forward and
// backward in turn 113 -> 103; 983040 x 18 fp32 (71 MB): 28.2 -> 27.0 and 44.7 -> 44.2; 61440 x 324 bf16 (40 MB): no difference.
constexpr int64_t STREAM_BYTES = 64 << 20;
// Rows of up to 2 KB of scores stay in a few lanes' registers.  Measured against a wavefront a row that goes over it in tiles, 65536 rows (log
// probabilities / with five alternatives / draws, us): 600 bf16 24 / 58 / 75 against 37 / 75 / 117, 1000 bf16 30 / 73 / 90 against 37 / 76 / 118;
// longer ones, as they are now, against registers (log probabilities / draws): 1500 bf16 45 / 139 against 44 / 126, 1000 fp32 45 / 108 against 44 / 120.
template <typename T> constexpr bool is_short(int64_t n) { return n * (int64_t)sizeof(T) <= 2048; }
// The backward pass, which needs no second look, keeps rows of up to 2048 scores there, and needs nothing of the forward pass for them (65536
// x 1500: bf16 69 us, fp32 134; in tiles, from the forward pass's statistics, 77 and 168).
constexpr int BACKWARD_SHORT_MAX = 2048;
template <int G_, int E_, int W_> struct Shape { static constexpr int G = G_, E = E_, W = W_; };
// f(lanes a row, scores a lane, scores a load): up to 32 scores in one lane (no exchanges at all: 983040 x 18 fp32 17.1 us, over four lanes 23.4;
// 61 rows 3.1, over four lanes 2.8; drawing 983040 x 18 bf16 32 us, over four lanes 54); beyond, the fewest lanes that hold the row in four
// pieces of W scores each, or 64 lanes with up to MOST pieces.
template <int W, int G, int MOST, typename F> int by_pieces(int64_t n, F f) {
    const int64_t c = (n + G * W - 1) / (G * W);
    if constexpr (G == 4) if (c <= 2) return f(Shape<G, 2 * W, W>());
    if (c <= 3) return f(Shape<G, 3 * W, W>());
    if constexpr (G < 64 || MOST == 4) return f(Shape<G, 4 * W, W>());
    else {
        if (c <= 4) return f(Shape<G, 4 * W, W>());
        if (c <= 6) return f(Shape<G, 6 * W, W>());
        return f(Shape<G, 8 * W, W>());
    }
}
template <int W, int LONGEST, typename F> int by_lanes(int64_t n, F f) {
    const int64_t lanes = (n + 4 * W - 1) / (4 * W);
    if (lanes <= 4) return by_pieces<W, 4, 4>(n, f);
    if (lanes <= 8) return by_pieces<W, 8, 4>(n, f);
    if (lanes <= 16) return by_pieces<W, 16, 4>(n, f);
    if constexpr (LONGEST <= 32 * 4 * W) return by_pieces<W, 32, 4>(n, f);
    else {
        if (lanes <= 32) return by_pieces<W, 32, 4>(n, f);
        return by_pieces<W, 64, LONGEST / (64 * W)>(n, f);
    }
}
template <typename F> int by_length_32(int64_t n, F f) {
    switch ((n + 3) / 4) {
        case 1: return f(Shape<1, 4, 4>());
        case 2: return f(Shape<1, 8, 4>());
        case 3: return f(Shape<1, 12, 4>());
        case 4: return f(Shape<1, 16, 4>());
        case 5: return f(Shape<1, 20, 4>());
        case 6: return f(Shape<1, 24, 4>());
        case 7: return f(Shape<1, 28, 4>());
        default: return f(Shape<1, 32, 4>());
    }
}
template <typename T, int LONGEST, typename F> int by_length(int64_t n, F f) {
    return n <= 32 ? by_length_32(n, f) : by_lanes<16 / sizeof(T), LONGEST>(n, f);
}
// Drawing for up to 16384 rows, which do not fill the GPU: short rows over four lanes.  (64-bit exponentials one after the other: 4096 x 18 fp32 4.2 us, in
// one lane 5.0; 65536 x 18 6.4, in one lane 5.2.)
// Beyond 32 scores, 16 a lane at most, whatever their type; with 32 of 16 bits in fewer lanes there is less overlap of wavefronts' exponentials and fewer
// exchanges (46394 x 242 fp16 20.0 us against 22.2; 51738 x 616 60.8 against 56.6).
template <typename T, typename F> int by_length_to_draw(int64_t rows, int64_t n, F f) {
    if (n > 32) return by_lanes<4, 2048 / sizeof(T)>(n, f);
    if (rows > 16384 || n < 8) return by_length_32(n, f);
    return n <= 16 ? f(Shape<4, 4, 4>()) : f(Shape<4, 8, 4>());
}
// How a long row is shared out: a wavefront a row (no exchange between wavefronts) where these are many or the rows not that long, else a
// workgroup, or several where that leaves CUs without one (no more than the row has tiles).  Measured (log probabilities / with five
// alternatives, us; wavefront against workgroup): 512 x 2500 bf16 4.5 against 4.4, 2048 x 2500 5.2 / 8.1 against 7.1 / 13.7; 512 x 5832 5.8 / 9.7
// against 4.8 / 7.9, 2048 x 5832 7.5 / 11.8 against 8.3 / 15.3, 4096 x 5832 13.0 / 17.3 against 15.6 / 27.9; 1024 x 20000 15.3 / 26.2 against 12.4 /
// 17.7, 2048 x 20000 19.3 / 30.3 against 20.3 / 30.4, 4096 x 20000 29.9 / 41.9 against 31.9 / 49.6.
struct Split {
    int row_waves, parts, part_tiles;
};
template <typename T> Split split(int64_t rows, int64_t n) {
    const int64_t wave_tiles = Tile<T, 1>::count(n);
    if (wave_tiles <= 2 || rows >= 4096 || (rows >= 2048 && wave_tiles <= 8)) return {1, 1, 0};
    const int64_t tiles = Tile<T, WAVES>::count(n), wanted = std::max<int64_t>(1, std::min<int64_t>(tiles, 1024 / std::max<int64_t>(rows, 1)));
    const int64_t each = (tiles + wanted - 1) / wanted;
    return {WAVES, (int)((tiles + each - 1) / each), (int)each};
}
// The backward pass of a longer row has a tile of a wavefront's or of a workgroup's size for each wavefront or workgroup; smaller tiles leave less of the last one empty.
// Measured (us): 32768 x 2500 bf16 75 against 100, 16384 x 5832 61 against 69, 8192 x 20000 113 against 120, 3000 x 40001 76 against 74, 1024 x
// 104976 67 either way.
// Up to two wavefront's tiles, halves of them (16-bit scores alone are that short here): 32768 x 2100 bf16 76 -> 57, x 2500 75 -> 58, x 4000 90 -> 91; longer
// rows 61 -> 65 (16384 x 5832); quarters, when they were tried, 1.2 ... 1.4 times halves.
template <typename T> bool backward_by_waves(int64_t n) { return Tile<T, 1>::count(n) <= 12; }
// Short rows' alternatives come one after the other, a pass over the registers each; from nine on, of rows of some length, a wavefront a row that
// collects and ranks them is faster (7 x 500 fp32, 20 of them: 5.6 us against 13.2 in passes).
template <typename T> bool in_lanes(int64_t n, int top) { return is_short<T>(n) && !(n > 256 && top > 8); }
template <typename T> int n_segments(int64_t n) { return (int)((n + 64 * (16 / sizeof(T)) - 1) / (64 * (16 / sizeof(T)))); }
// Drawing: a wavefront a row up to 12 tiles where there are rows enough, else a workgroup a tile and a second kernel.  Measured (us; the first against the
// second): 16 x 2500 bf16 8.2 against 8.6; 16 x 5832 12.1 against 9.3, 1024 x 5832 12.7 against 14.0, 4096 x 5832 28 against 43; 1024 x 20000
// 32 against 28, 2048 x 20000 43 against 48, 4096 x 20000 73 against 89; longer rows, fp32, 2048 x 20000 52 by the second (76 against 57 when the rule was made).
template <typename T> bool sample_by_waves(int64_t rows, int64_t n) {
    const int64_t tiles = Tile<T, 1>::count(n);
    return tiles <= 2 || (tiles <= 4 && rows >= 512) || (tiles <= 12 && rows >= 2048);          // (at most 48 segments: a lane each)
}

dim3 short_blocks(int64_t rows, int G) { return dim3((unsigned)std::min<int64_t>((rows * G + BLOCK - 1) / BLOCK, 0xffffffffLL / BLOCK)); }

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
    if (n <= 0 || rows <= 0) return 0;
    const auto bytes = [&](auto v) -> int64_t {
        using T = decltype(v);
        if (op == MGX_POLICY_SAMPLE ? is_short<T>(n) : in_lanes<T>(n, top)) return 0;
        if (op == MGX_POLICY_SAMPLE) return sample_by_waves<T>(rows, n) ? 0 : rows * n_segments<T>(n) * (int64_t)sizeof(Segment);
        const Split sp = split<T>(rows, n);
        return sp.parts == 1 ? 0 : rows * sp.parts * (16 + 8 * (int64_t)top);
    };
    return dtype == MGX_REAL_F32 ? bytes(float()) : bytes(half());
}

int64_t mgx_policy_stats_bytes(int64_t rows, int64_t n) { return n > BACKWARD_SHORT_MAX ? rows * 8 : 0; }

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
    if (!guard.ok) return fail_hip("hipSetDevice failed");
    const Actions given{actions, action_bytes};
    return by_dtype(dtype, [&](auto v) {
        using T = decltype(v);
        const Scores<T> sc = scores<T>(logits, rows, n, row_stride, mask, mask_row_stride, temperature);
        if (in_lanes<T>(n, top))
            return by_length<T, 2048 / sizeof(T)>(n, [&](auto shape) {
                constexpr int G = decltype(shape)::G, E = decltype(shape)::E, W = decltype(shape)::W;
                return launch_lds(k_log_probs_short<T, G, E, W>, short_blocks(rows, G), BLOCK, G == 1 ? BLOCK * top * 8 : 0, stream, sc,
                                  given, top, log_prob, entropy, top_log_probs, top_actions);
            });
        const Split sp = split<T>(rows, n);
        // (shorter rows whose alternatives take this way: the backward call has no use for statistics, and their memory need not be there)
        const LogProbOut out{log_prob, entropy, mgx_policy_stats_bytes(rows, n) ? stats : nullptr, top_log_probs, top_actions, top};
        const Partials partials{(uint64_t *)workspace, workspace ? (float *)((uint64_t *)workspace + rows * sp.parts * top) : nullptr};
        if (sp.row_waves == 1)
            return launch(top ? k_log_probs_long<T, true, 1, false> : k_log_probs_long<T, false, 1, false>, (rows + WAVES - 1) / WAVES, BLOCK, stream,
                          sc, given, out, 0, partials, Difference(sc));
        if (sp.parts == 1)
            return launch(top ? k_log_probs_long<T, true, WAVES, false> : k_log_probs_long<T, false, WAVES, false>, rows, BLOCK, stream, sc, given,
                          out, 0, partials, Difference(sc));
        if (const int rc = launch(top ? k_log_probs_long<T, true, WAVES, true> : k_log_probs_long<T, false, WAVES, true>,
                                  dim3((unsigned)sp.parts, (unsigned)rows), BLOCK, stream, sc, given, out, sp.part_tiles, partials, Difference(sc)))
            return rc;
        return launch(k_log_probs_join<T>, rows, 64, stream, sc, given, out, sp.parts, partials);
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
    if (!guard.ok) return fail_hip("hipSetDevice failed");
    const Actions given{actions, action_bytes};
    const bool stream_out = rows * n * (dtype == MGX_REAL_F32 ? 4 : 2) >= STREAM_BYTES;
    const Upstream up{grad_log_prob, grad_entropy, grad_log_prob_stride, grad_entropy_stride};
    return by_dtype(dtype, [&](auto v) {
        using T = decltype(v);
        const Scores<T> sc = scores<T>(logits, rows, n, row_stride, mask, mask_row_stride, temperature);
        if (n <= BACKWARD_SHORT_MAX)
            return by_length<T, BACKWARD_SHORT_MAX>(n, [&](auto shape) {
                constexpr int G = decltype(shape)::G, E = decltype(shape)::E, W = decltype(shape)::W;
                if constexpr (G == 1)
                    return launch_lds(k_backward_lane<T, G, E, W>, short_blocks(rows, 1), BLOCK, (int)(BLOCK * n * sizeof(T)), stream, sc, given, entropy,
                                      up, (T *)grad, stream_out);
                else return launch(k_backward_short<T, G, E, W>, short_blocks(rows, G), BLOCK, stream, sc, given, entropy, up, (T *)grad, stream_out);
            });
        if (backward_by_waves<T>(n)) {
            const unsigned by_fours = (unsigned)std::min<int64_t>((rows + WAVES - 1) / WAVES, 65535);
            if constexpr (sizeof(T) == 2)
                if (Tile<T, 1>::count(n) <= 2)
                    return launch(k_backward_long<T, 1, 2>, dim3((unsigned)Tile<T, 1, 2>::count(n), by_fours), BLOCK, stream, sc, given, stats, entropy, up,
                                  (T *)grad, stream_out);
            return launch(k_backward_long<T, 1, 4>, dim3((unsigned)Tile<T, 1>::count(n), by_fours), BLOCK, stream, sc, given, stats, entropy, up,
                          (T *)grad, stream_out);
        }
        return launch(k_backward_long<T, WAVES, 4>, dim3((unsigned)Tile<T, WAVES>::count(n), (unsigned)std::min<int64_t>(rows, 65535)), BLOCK,
                      stream, sc, given, stats, entropy, up, (T *)grad, stream_out);
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
    if (!guard.ok) return fail_hip("hipSetDevice failed");
    const Drawn out{action, log_prob, entropy};
    return by_dtype(dtype, [&](auto v) {
        using T = decltype(v);
        const Scores<T> sc = scores<T>(logits, rows, n, row_stride, mask, mask_row_stride, temperature);
        if (is_short<T>(n))
            return by_length_to_draw<T>(rows, n, [&](auto shape) {
                constexpr int G = decltype(shape)::G, E = decltype(shape)::E, W = decltype(shape)::W;
                return launch(k_sample_short<T, G, E, W>, short_blocks(rows, G), BLOCK, stream, sc, uniforms, uniform_bytes, out);
            });
        if (sample_by_waves<T>(rows, n))
            return launch(k_sample_wave<T>, (rows + WAVES - 1) / WAVES, BLOCK, stream, sc, uniforms, uniform_bytes, out);
        const int segments = n_segments<T>(n);
        if (const int rc = launch(k_sample_parts<T>, dim3((unsigned)Tile<T, WAVES>::count(n), (unsigned)std::min<int64_t>(rows, 65535)), BLOCK, stream, sc,
                                  segments, (Segment *)workspace))
            return rc;
        return launch(k_draw<T>, rows, BLOCK, stream, sc, uniforms, uniform_bytes, out, segments, (const Segment *)workspace);
    });
}

}  // extern "C"
