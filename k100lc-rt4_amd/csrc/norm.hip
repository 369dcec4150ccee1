// norm.hip -- what stands between one block and the next, and the quantizer with one scale a token.
//
//   y1 = post_w ? y * post_w / rms(y) : y
//   h' = round(h + scale * gate * y1)                       (to h's type: what is stored is what is normed)
//   n  = h' * (w + w_offset) / rms(h'),   rms(x) = sqrt(mean(x^2) + eps)
//
// n goes out as floats or as int8 codes, one scale a token or one a 128-group.  A code is the nearest integer
// to most * n / max|n|, and 1 / rms cancels in that quotient, so codes go by p = h' (w + w_offset) alone.
//
// Results are those of 64-bit arithmetic.  p is exact in it and a quotient off by 2^-51, so a code has one right value.  A sum of
// squares passes through n roundings, 34 for 5120 elements and 86 for 65536, and is off by n 2^-53 of itself, 1 / rms by half of
// that: 2^-47.6 at most, which can move a residual behind a norm, or a float result, over a border that it lies next to.
// A 64-bit conversion costs four fp32 operations, so what fp32 decides is left to it: a quotient, or a residual
// of 16 bits, is formed in fp32 with a bound of its error, and in 64 bits by the lanes whose rounding that leaves open
// (one of 8000 codes, of 4000 residuals).
//
// 4096 tokens of 5120 (bf16, post norm, gate, token codes): 62 us from memory (58 where the last-level cache holds a part); their
// 147 MB take 31 at the rate of a large copy, and the vector ALU works for 40 of them (74 instructions an element, active 71% of
// the cycles), at the 4 waves a SIMD that 123 registers leave.  Without the check of products' range, `least`, 93 registers and
// 57 us; held to 96 registers, which spills, 82; two chunks a thread, 81.  A tenth of y zero, which that check leaves to 64 bits:
// 67; every other row zero: 63.  Without post norm and gate: token codes 55, group codes 53, bf16 47; without y 31, 30, 26.
// 4 rows of 5120: 5.4 us.  1000 rows of 17408 to codes alone: 19 us for 52 MB (16 to 17 from the cache).
#include <type_traits>

#include "ffn_dev.h"
#include "rt4_internal.h"

namespace rt4 {

namespace {

constexpr int kMaxWaves = 16;

// Eight elements as they are in memory.  VEC: rows are whole chunks of 8, aligned for vector access.  Others: whole chunks by
// the same loads and stores, which global memory takes at any alignment (1000 rows of 17401 bf16 to codes: 20 us, element by
// element 34), the row's last by elements.
template <class T>
struct Raw {
    uint4 d[sizeof(T) / 2];
};
template <bool VEC, class T>
__device__ __forceinline__ Raw<T> load_raw(const T* row, int i, int K) {
    Raw<T> r = {};
    if (VEC) {
        if (i < K)
#pragma unroll
            for (int k = 0; k < (int)sizeof(T) / 2; k++) r.d[k] = reinterpret_cast<const uint4*>(row + i)[k];
    } else if (i + 8 <= K) {
        __builtin_memcpy(&r, row + i, sizeof(r));
    } else if (i < K) {
        T t[8];
#pragma unroll
        for (int e = 0; e < 8; e++) t[e] = i + e < K ? row[i + e] : (T)0.f;
        __builtin_memcpy(&r, t, sizeof(r));
    }
    return r;
}
// Element e of eight as fp32: one operation (bf16 is the upper half of an fp32 value).
template <class T>
__device__ __forceinline__ float elem(const uint4* d, int e) {
    const uint32_t q[8] = {d[0].x, d[0].y, d[0].z, d[0].w, sizeof(T) == 4 ? d[1].x : 0, sizeof(T) == 4 ? d[1].y : 0, sizeof(T) == 4 ? d[1].z : 0, sizeof(T) == 4 ? d[1].w : 0};
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, q[e]);
    else if constexpr (__is_same(T, bf16)) return __builtin_bit_cast(float, e & 1 ? q[e >> 1] & 0xFFFF0000u : q[e >> 1] << 16);
    else return (float)__builtin_bit_cast(f16, (uint16_t)(e & 1 ? q[e >> 1] >> 16 : q[e >> 1]));
}
template <class T>
__device__ __forceinline__ float elem(const Raw<T>& r, int e) {
    return elem<T>(r.d, e);
}
// The same of a type known at the launch: loaded as it is (no wait), widened where it is used.
struct RawAny {
    uint4 d[2];
};
template <bool VEC>
__device__ __forceinline__ RawAny load_any(const void* p, long long at, int type, int i, int K) {
    RawAny r = {};
    if (type == kF32) {
        const Raw<float> t = load_raw<VEC>(static_cast<const float*>(p) + at, i, K);
        r.d[0] = t.d[0], r.d[1] = t.d[1];
    } else {
        r.d[0] = load_raw<VEC>(static_cast<const f16*>(p) + at, i, K).d[0];
    }
    return r;
}
template <class T>
__device__ __forceinline__ void widen16(const RawAny& r, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = elem<T>(r.d, e);
}
__device__ __forceinline__ void widen(const RawAny& r, int type, float (&v)[8]) {
    if (type == kF32) __builtin_memcpy(v, r.d, sizeof(v));
    else if (type == kBF16) widen16<bf16>(r, v);
    else widen16<f16>(r, v);
}
template <bool VEC, class T>
__device__ __forceinline__ void store8(T* row, int i, int K, const T (&t)[8]) {
    if (VEC) {
        uint4 d[sizeof(T) / 2];
        __builtin_memcpy(d, t, sizeof(t));
        if (i < K)
#pragma unroll
            for (int k = 0; k < (int)sizeof(T) / 2; k++) reinterpret_cast<uint4*>(row + i)[k] = d[k];
    } else if (i + 8 <= K) {
        __builtin_memcpy(row + i, t, sizeof(t));
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (i + e < K) row[i + e] = t[e];
    }
}

// The fp32 value of v, which 16-bit results are rounded from (as they are wherever such sums are formed in fp32).  The
// empty asm keeps the compiler from joining the two roundings into one.
__device__ __forceinline__ float f32_of(double v) {
    float f = (float)v;
    asm("" : "+v"(f));
    return f;
}

__device__ __forceinline__ double max2(double a, double b) { return a > b ? a : b; }

// Sums (and maxima) over the workgroup, the same in every thread: waves in order through LDS.
__device__ __forceinline__ double block_sum(double v, double* lds) {
    v = wave_sum(v);
    if (blockDim.x == 64) return v;
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0;
    for (int i = 0; i < (int)(blockDim.x >> 6); i++) s += lds[i];
    return s;
}
__device__ __forceinline__ void block_sum_max(double& s, double& m, double* lds) {
    s = wave_sum(s);
    m = wave_reduce(m, max2);
    if (blockDim.x == 64) return;
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s, lds[kMaxWaves + (threadIdx.x >> 6)] = m;
    __syncthreads();
    s = 0;
    m = 0;
    for (int i = 0; i < (int)(blockDim.x >> 6); i++) s += lds[i], m = max2(m, lds[kMaxWaves + i]);
}

// The magnitude that a maximum takes: NaN counts as infinite, so that a row that holds either is known by its maximum.
__device__ __forceinline__ double magnitude(double p) { return p == p ? fabs(p) : __builtin_inf(); }
// The same in fp32 as bits, which order as magnitudes do, NaN above all.
__device__ __forceinline__ uint32_t magnitude_bits(float p) { return __builtin_bit_cast(uint32_t, p) & 0x7FFFFFFFu; }

// 1 / sqrt(mean + eps) from a sum of squares, to 2^-50: the hardware's estimate and two Newton steps.
__device__ __forceinline__ double inv_rms(double sum, double inv_k, double eps) {
    const double x = fma(sum, inv_k, eps);
    double r = __builtin_amdgcn_rsq(x);
    if (x > 0 && x < __builtin_inf()) {
        r = fma(r * 0.5, fma(-x * r, r, 1.0), r);
        r = fma(r * 0.5, fma(-x * r, r, 1.0), r);
    }
    return r;
}

// The code of p in a group of maximum a, f = most / a (0 codes where a is 0 or not finite).
__device__ __forceinline__ int code_of(double p, double f, double a, double most) {
    const double q = p * f;
    double r = rint(q);
    if (fabs(q - r) > 0.5 - 0x1p-40) r = rint(p * most / a);
    return (int)r;
}
// Codes of 8 values p = v * w (w the weight with its offset, an fp32 value) from fp32 products: six roundings (w's sum, the
// product, the maximum's, the factor's 2, the quotient's) of at most 2^-24 each leave the quotient, below 128, off by 2^-14.4
// at most.  Where it lies within 2^-14 of a half, 64 bits decide.
// The sum of the quotient and 3 * 2^22 is rounded to an integer (ties to even), which its low byte holds.
template <class P>
__device__ __forceinline__ uint2 codes_of(const float (&hi)[8], P exact, float f32, double a, double most, bool interleaved) {
    constexpr float M = 0x1.8p23f;
    bool open = false;
    uint32_t c[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float t = fmaf(hi[e], f32, M);
        open |= !(fabsf(fmaf(hi[e], f32, M - t)) < 0.5f - 0x1p-14f);
        c[e] = __builtin_bit_cast(uint32_t, t);
    }
    if (open) {
        const double f = most / a;
#pragma unroll
        for (int e = 0; e < 8; e++) c[e] = (uint32_t)code_of(exact(e), f, a, most);
    }
    const auto four = [&](int p, int q, int r, int s) {
        return __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[s], c[r], 0x0c0c0400u), __builtin_amdgcn_perm(c[q], c[p], 0x0c0c0400u), 0x05040100u);
    };
    return interleaved ? make_uint2(four(0, 2, 4, 6), four(1, 3, 5, 7)) : make_uint2(four(0, 1, 2, 3), four(4, 5, 6, 7));
}
// h + t for a 16-bit residual, t formed in fp32 with at most 6 roundings, each of at most 2^-24 (see `least`): where both ends
// of the error's range round to the same bits, those; otherwise `open` is set, and 64 bits decide.
template <class T>
__device__ __forceinline__ T sum_of(float h, float t, bool& open) {
    typedef T two __attribute__((ext_vector_type(2)));
    typedef float two32 __attribute__((ext_vector_type(2)));
    const float v = h + t, e = fabsf(h) + fabsf(t);
    const two32 ends = {fmaf(e, -0x1p-21f, v), fmaf(e, 0x1p-21f, v)};
    const two r = __builtin_convertvector(ends, two);
    const uint32_t b = __builtin_bit_cast(uint32_t, r);
    open |= (b & 0xFFFFu) != b >> 16;
    return r[1];
}
// The lesser of m and the magnitudes of eight products, NaN where one of them is.  At 2^-100 and above all of them were rounded to
// 24 bits; a NaN may come of an overflow on the way.
__device__ __forceinline__ float least(float m, const float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) m = __builtin_elementwise_minimum(__builtin_elementwise_minimum(m, fabsf(v[e])), fabsf(v[e + 1]));
    return m;
}
// The scale that belongs to maximum a: 1 for zeros (as the other quantizers), so where r = 1 / rms is 0 for an infinite value in
// another group; NaN where a value was not finite.
__device__ __forceinline__ float scale_of(double a, double r, double most) {
    if (!(a < __builtin_inf()) || r != r) return __builtin_nanf("");
    return a > 0 && r > 0 ? (float)(a * r / most) : 1.f;
}

// One workgroup a row; a thread holds C chunks of 8 elements, chunk c at (c * threads + thread) * 8.  What lies behind the
// row's end is zeros, of values and of weights.
template <int C, int MOST, bool VEC, class TH, bool HASY, bool NORM>
__global__ __launch_bounds__(MOST) void norm_k(BlockNorm a) {
    __shared__ double lds[3 * kMaxWaves];
    __shared__ unsigned long long top;           // the row's exact maximum, as bits (they order as the values do)
    const int K = a.K, NT = blockDim.x;
    const size_t m = blockIdx.x;
    const TH* hrow = static_cast<const TH*>(a.h) + m * a.ldh;
    Raw<TH> hr[C];
    RawAny yr[HASY ? C : 1];
    const auto place = [&](int c) { return (c * NT + (int)threadIdx.x) * 8; };
    // Between passes over the chunks: what a pass has widened or loaded is not kept for the next (the compiler would keep 40
    // registers a chunk).
    uint32_t zero = 0;                           // (of the weights' place, for the same reason)
    const auto next_pass = [&]() {
        asm volatile("" : "+s"(zero));
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int k = 0; k < (int)sizeof(TH) / 2; k++) asm volatile("" : "+v"(hr[c].d[k].x), "+v"(hr[c].d[k].y), "+v"(hr[c].d[k].z), "+v"(hr[c].d[k].w));
    };
#pragma unroll
    for (int c = 0; c < C; c++) hr[c] = load_raw<VEC>(hrow, place(c), K);
    if constexpr (HASY) {
#pragma unroll
        for (int c = 0; c < C; c++) yr[c] = load_any<VEC>(a.y, (long long)m * a.ldy, a.y_type, place(c), K);
    }
    if (threadIdx.x == 0) top = 0;
    if constexpr (HASY) {
        const auto factors = [&](int c, Raw<float>& pw, RawAny& g) {
            if (a.post_w) pw = load_raw<VEC>(a.post_w, place(c), K);
            if (a.gate) g = load_any<VEC>(a.gate, (long long)m * a.ldg, a.y_type, place(c), K);
        };
        Raw<float> pw, pw1;                      // this chunk's, and the next one's on its way
        RawAny gr, gr1;
        factors(0, pw, gr);
        double k = a.scale;
        if (a.post_w) {
            double s = 0;
#pragma unroll
            for (int c = 0; c < C; c++) {
                float v[8];
                widen(yr[c], a.y_type, v);
#pragma unroll
                for (int e = 0; e < 8; e++) s = fma((double)v[e], (double)v[e], s);
            }
            k *= inv_rms(block_sum(s, lds + 2 * kMaxWaves), a.inv_k, a.eps);
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int i = 0; i < 2; i++) asm volatile("" : "+v"(yr[c].d[i].x), "+v"(yr[c].d[i].y), "+v"(yr[c].d[i].z), "+v"(yr[c].d[i].w));
        }
        const float k32 = (float)k;
        const bool k_fine = fabsf(k32) >= 0x1p-126f && fabsf(k32) < __builtin_inff();
        TH* orow = static_cast<TH*>(a.h_out) + m * a.ldho;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int i = place(c);
            if (c + 1 < C) factors(c + 1, pw1, gr1);
            const auto exact = [&](TH (&t)[8]) {
                float y[8], g[8];
                widen(yr[c], a.y_type, y);
                if (a.gate) widen(gr, a.y_type, g);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    double v = (double)y[e] * k;
                    if (a.gate) v *= (double)g[e];
                    if (a.post_w) v *= (double)elem(pw, e);
                    t[e] = (TH)f32_of((double)elem(hr[c], e) + v);
                }
            };
            TH t[8];
            if constexpr (sizeof(TH) == 4) {
                exact(t);
            } else {
                float y[8];
                widen(yr[c], a.y_type, y);
#pragma unroll
                for (int e = 0; e < 8; e++) y[e] *= k32;
                float small = least(0x1p0f, y);
                if (a.gate) {
                    float g[8];
                    widen(gr, a.y_type, g);
#pragma unroll
                    for (int e = 0; e < 8; e++) y[e] *= g[e];
                    small = least(small, y);
                }
                if (a.post_w) {
#pragma unroll
                    for (int e = 0; e < 8; e++) y[e] *= elem(pw, e);
                    small = least(small, y);
                }
                bool open = !(k_fine && small >= 0x1p-100f);
#pragma unroll
                for (int e = 0; e < 8; e++) t[e] = sum_of<TH>(elem(hr[c], e), y[e], open);
                if (open && i < K) exact(t);
            }
            store8<VEC>(orow, i, K, t);
            if (!VEC)                            // (what lies behind the row: 0 times an infinite k is NaN)
#pragma unroll
                for (int e = 0; e < 8; e++) t[e] = i + e < K ? t[e] : (TH)0.f;
            __builtin_memcpy(&hr[c], t, sizeof(t));
            if (VEC && i >= K) hr[c] = Raw<TH>{};
            pw = pw1, gr = gr1;
            __builtin_amdgcn_sched_barrier(0);   // (chunks mixed need more registers than there are)
        }
    }
    if (!a.n) return;
    next_pass();
    const float off32 = (float)a.w_offset;
    const bool off_fine = off32 == a.w_offset;   // else a weight may cancel all of it but its rounding: 64 bits throughout
    const auto weights = [&](int c) {
        Raw<float> w = {};
        if (NORM) w = load_raw<VEC>(a.w + zero, place(c), K);
        return w;
    };
    double s = 0;
    uint32_t bits = 0;                           // the largest fp32 product
    Raw<float> w, w1;                            // this chunk's weights, and the next one's on their way
    if (a.form == kToken) w = weights(0);
#pragma unroll
    for (int c = 0; c < C; c++) {
        if (a.form == kToken && c + 1 < C) w1 = weights(c + 1);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float v = elem(hr[c], e);
            if (NORM) s = fma((double)v, (double)v, s);
        }
        if (a.form == kToken)
#pragma unroll
            for (int e = 0; e < 8; e++) bits = max(bits, magnitude_bits(NORM ? elem(hr[c], e) * (elem(w, e) + off32) : elem(hr[c], e)));
        w = w1;
        __builtin_amdgcn_sched_barrier(0);
    }
    next_pass();
    w = weights(0);                              // (from the cache, under way during the reductions)
    const float most32 = bits < 0x7F800000u ? __builtin_bit_cast(float, bits) : __builtin_inff();
    double r = 1, most = most32;
    if (NORM || a.form == kToken) {
        block_sum_max(s, most, lds);
        if (NORM) r = inv_rms(s, a.inv_k, a.eps);
    }
    if (a.form <= kF16) {
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int i = place(c);
            if (c + 1 < C) w1 = weights(c + 1);
            float n[8];
#pragma unroll
            for (int e = 0; e < 8; e++) n[e] = f32_of((double)elem(hr[c], e) * ((double)elem(w, e) + a.w_offset) * r);
            if (a.form == kF32) {
                store8<VEC>(static_cast<float*>(a.n) + m * K, i, K, n);
            } else if (a.form == kBF16) {
                bf16 t[8];
#pragma unroll
                for (int e = 0; e < 8; e++) t[e] = (bf16)n[e];
                store8<VEC>(static_cast<bf16*>(a.n) + m * K, i, K, t);
            } else {
                f16 t[8];
#pragma unroll
                for (int e = 0; e < 8; e++) t[e] = (f16)n[e];
                store8<VEC>(static_cast<f16*>(a.n) + m * K, i, K, t);
            }
            w = w1;
            __builtin_amdgcn_sched_barrier(0);
        }
    } else if (a.form == kToken) {
        // The exact maximum: of the values whose fp32 product is within its error of the largest.  Where fp32 does not hold the
        // products, of all values, and all codes in 64 bits.
        const bool range = off_fine && most > 0x1p-100 && most < __builtin_inf();
        if constexpr (NORM) {                    // (without a norm the products are the values themselves)
            if (!range || most32 >= (float)most * (1 - 0x1p-21f)) {
                double mine = 0;
#pragma unroll
                for (int c = 0; c < C; c++) {
                    const Raw<float> v = weights(c);
#pragma unroll
                    for (int e = 0; e < 8; e++) mine = max2(mine, magnitude((double)elem(hr[c], e) * ((double)elem(v, e) + a.w_offset)));
                }
                atomicMax(&top, (unsigned long long)__double_as_longlong(mine));
            }
            next_pass();
            __syncthreads();
            most = __longlong_as_double((long long)top);
        }
        const bool fine = most > 0 && most < __builtin_inf();
        const float f32 = fine && range ? 127.f / (float)most : __builtin_nanf("");   // (NaN: every quotient is left open)
        int8_t* qrow = static_cast<int8_t*>(a.n) + m * K;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int i = place(c);
            if (c + 1 < C) w1 = weights(c + 1);
            uint2 q = make_uint2(0, 0);
            float hi[8];
#pragma unroll
            for (int e = 0; e < 8; e++) hi[e] = NORM ? elem(hr[c], e) * (elem(w, e) + off32) : elem(hr[c], e);
            if (fine)
                q = codes_of(hi, [&](int e) { return NORM ? (double)elem(hr[c], e) * ((double)elem(w, e) + a.w_offset) : (double)hi[e]; }, f32, most, 127., false);
            if (VEC) {
                if (i < K) *reinterpret_cast<uint2*>(qrow + i) = q;
            } else if (i + 8 <= K) {
                __builtin_memcpy(qrow + i, &q, sizeof(q));
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (i + e < K) qrow[i + e] = (int8_t)((e < 4 ? q.x : q.y) >> 8 * (e & 3));
            }
            w = w1;
            __builtin_amdgcn_sched_barrier(0);
        }
        if (threadIdx.x == 0) a.n_scale[m] = scale_of(most, r, 127);
    } else if constexpr (NORM) {                 // K % 128 == 0: a 128-group is a run of 16 lanes
        const double levels = a.form == kAct ? 127 : 119;
        int8_t* qrow = static_cast<int8_t*>(a.n) + m * K;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int i = place(c);
            if (c + 1 < C) w1 = weights(c + 1);
            const auto exact = [&](int e) { return (double)elem(hr[c], e) * ((double)elem(w, e) + a.w_offset); };
            double g = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) g = max2(g, magnitude(exact(e)));
            g = max2(g, pair_of<0>(g));
            g = max2(g, pair_of<1>(g));
            g = max2(g, pair_of<2>(g));
            g = max2(g, pair_of<3>(g));
            const bool fine = g > 0 && g < __builtin_inf() && r > 0;
            const float f32 = off_fine && g > 0x1p-100 && g < 0x1p100 ? (float)levels / (float)g : __builtin_nanf("");
            uint2 q = make_uint2(0, 0);
            float hi[8];
#pragma unroll
            for (int e = 0; e < 8; e++) hi[e] = elem(hr[c], e) * (elem(w, e) + off32);
            if (fine) q = codes_of(hi, exact, f32, g, levels, true);
            if (i < K) {
                *reinterpret_cast<uint2*>(qrow + i) = q;
                const int gi = i >> 7;
                if ((threadIdx.x & 15) == 0) a.n_scale[a.form == kAct ? m * (K >> 7) + gi : (size_t)gi * a.M + m] = scale_of(g, r, levels);
            }
            w = w1;
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}

template <class TH, bool HASY, bool NORM>
void launch_chunks(const BlockNorm& a, hipStream_t st) {
    // Few rows: many waves a row.  Many: few waves a row, whose reductions cost little; 3 chunks a thread (5 without y) leave
    // registers for as many rows a CU as hide each other's latencies (4096 tokens of 5120, bf16, post norm and gate: 3 chunks 62
    // us, 2 81).  Waves enough to fill the CUs either way.
    // Forms of 2 to 5 chunks hold 512 threads.  So rows above 12288 elements take 5 chunks, with y at 149 to 188 registers and 2
    // or 3 waves a SIMD, and rows above 20480 take 8 at 1024 threads, whose 128 registers do not hold them with a norm: 40 to 344
    // bytes of a lane go to scratch without y, 556 to 788 with it (1000 rows with a post norm: of 12288 elements 34 us, of 17408
    // 68, of 20480 70, of 24576 184; without y 27, 26, 29, 79).
    const int lanes = (a.K + 7) / 8, most = HASY ? 3 : 5;
    const auto go = [&](auto k, int C) {
        hipLaunchKernelGGL(k, dim3((unsigned)a.M), dim3((unsigned)(((lanes + C - 1) / C + 63) / 64 * 64)), 0, st, a);
    };
    const int all = (lanes + 63) / 64, least = (all + most - 1) / most, want = a.M < 2048 ? 2048 / a.M : 1;
    int waves = want < least ? least : want;
    if (waves > 16) waves = 16;
    const int C = (all + waves - 1) / waves;
    const auto pick = [&](auto vec) {
        constexpr bool V = decltype(vec)::value;
        if (C <= 1) go(norm_k<1, 1024, V, TH, HASY, NORM>, 1);
        else if (C <= 2 && lanes <= 2 * 512) go(norm_k<2, 512, V, TH, HASY, NORM>, 2);
        else if (C <= 3 && lanes <= 3 * 512) go(norm_k<3, 512, V, TH, HASY, NORM>, 3);
        else if (C <= 5 && lanes <= 5 * 512) go(norm_k<5, 512, V, TH, HASY, NORM>, 5);
        else go(norm_k<8, 1024, V, TH, HASY, NORM>, 8);
    };
    if (a.vec) pick(std::true_type{});
    else pick(std::false_type{});
}
template <class TH>
void launch_y(const BlockNorm& a, hipStream_t st) {
    if (a.y) launch_chunks<TH, true, true>(a, st);
    else if (a.w || !a.n) launch_chunks<TH, false, true>(a, st);
    else launch_chunks<TH, false, false>(a, st);
}

}  // namespace

hipError_t launch_block_norm(const BlockNorm& a, hipStream_t st) {
    if (a.h_type == kF32) launch_y<float>(a, st);
    else if (a.h_type == kBF16) launch_y<bf16>(a, st);
    else launch_y<f16>(a, st);
    return hipGetLastError();
}

}  // namespace rt4
