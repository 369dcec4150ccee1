// norm.hip -- what stands between one block and the next, and the quantizer with one scale a token.
//
//   y1 = post_w ? y * post_w / rms(y) : y
//   h' = round(h + scale * gate * y1)                       (to h's type: what is stored is what is normed)
//   n  = h' * (w + w_offset) / rms(h'),   rms(x) = sqrt(mean(x^2) + eps)
//
// n goes out as floats or as int8 codes, one scale a token or one a 128-group.  A code is the nearest integer
// to most * n / max|n|, and 1 / rms cancels in that quotient, so codes go by p = h' (w + w_offset) alone.
// Everything between loads and stores is 64-bit: p is exact, the quotient is off by 2^-51, so a code differs
// from its definition only where the quotient is within that of a half (and exact halves are divided out).
// The kernel is bound by memory all the same: ~25 64-bit operations an element, 13 us of the chip's vector rate
// for 4096 rows of 5120, whose bytes take 31.
#include <type_traits>

#include "ffn_dev.h"
#include "rt4_internal.h"

namespace rt4 {

namespace {

constexpr int kMaxWaves = 16;

// Eight elements as they are in memory.
template <class T>
struct Raw {
    uint4 d[sizeof(T) / 2];
};
template <class T>
__device__ __forceinline__ Raw<T> load_raw(const T* row, int i, int K, bool vec) {
    Raw<T> r = {};
    if (vec && i + 8 <= K) {
#pragma unroll
        for (int k = 0; k < (int)sizeof(T) / 2; k++) r.d[k] = reinterpret_cast<const uint4*>(row + i)[k];
    } else {
        T t[8];
#pragma unroll
        for (int e = 0; e < 8; e++) t[e] = i + e < K ? row[i + e] : (T)0.f;
        __builtin_memcpy(&r, t, sizeof(r));
    }
    return r;
}
template <class T>
__device__ __forceinline__ float elem(const Raw<T>& r, int e) {
    T t[8];
    __builtin_memcpy(t, &r, sizeof(r));
    return (float)t[e];
}
template <class T>
__device__ __forceinline__ void store8(T* row, int i, int K, bool vec, const T (&t)[8]) {
    if (vec && i + 8 <= K) {
        uint4 d[sizeof(T) / 2];
        __builtin_memcpy(d, t, sizeof(t));
#pragma unroll
        for (int k = 0; k < (int)sizeof(T) / 2; k++) reinterpret_cast<uint4*>(row + i)[k] = d[k];
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
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0;
    for (int i = 0; i < (int)(blockDim.x >> 6); i++) s += lds[i];
    return s;
}
__device__ __forceinline__ void block_sum_max(double& s, double& m, double* lds) {
    s = wave_sum(s);
    m = wave_reduce(m, max2);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s, lds[kMaxWaves + (threadIdx.x >> 6)] = m;
    __syncthreads();
    s = 0;
    m = 0;
    for (int i = 0; i < (int)(blockDim.x >> 6); i++) s += lds[i], m = max2(m, lds[kMaxWaves + i]);
}

// The magnitude that a maximum takes: NaN counts as infinite, so that a row that holds either is known by its maximum.
__device__ __forceinline__ double magnitude(double p) { return p == p ? fabs(p) : __builtin_inf(); }

// The code of p in a group of maximum a, f = most / a (0 codes where a is 0 or not finite).
__device__ __forceinline__ int code_of(double p, double f, double a, double most) {
    const double q = p * f;
    double r = rint(q);
    if (fabs(q - r) > 0.5 - 0x1p-40) r = rint(p * most / a);
    return (int)r;
}
__device__ __forceinline__ uint2 pack8(const int (&c)[8]) {
    return make_uint2((uint32_t)(c[0] & 0xFF) | (uint32_t)(c[1] & 0xFF) << 8 | (uint32_t)(c[2] & 0xFF) << 16 | (uint32_t)(c[3] & 0xFF) << 24,
                      (uint32_t)(c[4] & 0xFF) | (uint32_t)(c[5] & 0xFF) << 8 | (uint32_t)(c[6] & 0xFF) << 16 | (uint32_t)(c[7] & 0xFF) << 24);
}
// The scale that belongs to maximum a: 1 for zeros (as the other quantizers), NaN where a value was not finite.
__device__ __forceinline__ float scale_of(double a, double r, double most) {
    const double s = a * r / most;
    return a > 0 ? (a < __builtin_inf() ? (float)s : __builtin_nanf("")) : r == r ? 1.f : __builtin_nanf("");
}

struct None {};

// One workgroup a row; a thread holds C chunks of 8 elements, chunk c at (c * threads + thread) * 8.
template <int C, class TH, class TY, bool NORM>
__global__ __launch_bounds__(1024) void norm_k(BlockNorm a) {
    constexpr bool HASY = !__is_same(TY, None);
    using Y = std::conditional_t<HASY, TY, TH>;
    __shared__ double lds[3 * kMaxWaves];
    const int K = a.K, NT = blockDim.x;
    const size_t m = blockIdx.x;
    const bool vec = a.vec;
    const TH* hrow = static_cast<const TH*>(a.h) + m * a.ldh;
    Raw<TH> hr[C];
    Raw<Y> yr[HASY ? C : 1], gr[HASY ? C : 1];
#pragma unroll
    for (int c = 0; c < C; c++) hr[c] = load_raw(hrow, (c * NT + (int)threadIdx.x) * 8, K, vec);
    if constexpr (HASY) {
        const TY* yrow = static_cast<const TY*>(a.y) + m * a.ldy;
#pragma unroll
        for (int c = 0; c < C; c++) yr[c] = load_raw(yrow, (c * NT + (int)threadIdx.x) * 8, K, vec);
        if (a.gate) {
            const TY* grow = static_cast<const TY*>(a.gate) + m * a.ldg;
#pragma unroll
            for (int c = 0; c < C; c++) gr[c] = load_raw(grow, (c * NT + (int)threadIdx.x) * 8, K, vec);
        }
    }
    float hv[C][8];
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int e = 0; e < 8; e++) hv[c][e] = elem(hr[c], e);
    if constexpr (HASY) {
        double k = a.scale;
        if (a.post_w) {
            double s = 0;
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const double v = elem(yr[c], e);
                    s = fma(v, v, s);
                }
            s = block_sum(s, lds + 2 * kMaxWaves);
            k *= 1 / sqrt(s / K + a.eps);
        }
        TH* orow = static_cast<TH*>(a.h_out) + m * a.ldho;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int i = (c * NT + (int)threadIdx.x) * 8;
            Raw<float> pw;
            if (a.post_w) pw = load_raw(a.post_w, i, K, a.wvec);
            TH t[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                double v = (double)elem(yr[c], e) * k;
                if (a.gate) v *= (double)elem(gr[c], e);
                if (a.post_w) v *= (double)elem(pw, e);
                t[e] = (TH)f32_of((double)hv[c][e] + v);
                hv[c][e] = (float)t[e];
            }
            if (i < K) store8(orow, i, K, vec, t);
            if (i + 8 > K)                       // what lies behind the row stays out of the sums (0 times an infinite k is NaN)
#pragma unroll
                for (int e = 0; e < 8; e++) hv[c][e] = i + e < K ? hv[c][e] : 0.f;
        }
    }
    if (!a.n) return;
    double s = 0, most = 0;
    double p[C][8];
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int i = (c * NT + (int)threadIdx.x) * 8;
        Raw<float> w = {};
        if (NORM) w = load_raw(a.w, i, K, a.wvec);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const double v = hv[c][e];
            s = fma(v, v, s);
            p[c][e] = NORM ? v * ((double)elem(w, e) + a.w_offset) : v;
            most = max2(most, magnitude(i + e < K ? p[c][e] : 0.));
        }
    }
    double r = 1;
    if (NORM || a.form == kToken) {
        block_sum_max(s, most, lds);
        if (NORM) r = 1 / sqrt(s / K + a.eps);
    }
    if (a.form <= kF16) {
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int i = (c * NT + (int)threadIdx.x) * 8;
            if (i >= K) continue;
            if (a.form == kF32) {
                float t[8];
#pragma unroll
                for (int e = 0; e < 8; e++) t[e] = (float)(p[c][e] * r);
                store8(static_cast<float*>(a.n) + m * K, i, K, a.nvec, t);
            } else if (a.form == kBF16) {
                bf16 t[8];
#pragma unroll
                for (int e = 0; e < 8; e++) t[e] = (bf16)f32_of(p[c][e] * r);
                store8(static_cast<bf16*>(a.n) + m * K, i, K, a.nvec, t);
            } else {
                f16 t[8];
#pragma unroll
                for (int e = 0; e < 8; e++) t[e] = (f16)f32_of(p[c][e] * r);
                store8(static_cast<f16*>(a.n) + m * K, i, K, a.nvec, t);
            }
        }
    } else if (a.form == kToken) {
        const bool fine = most > 0 && most < __builtin_inf();
        const double f = fine ? 127 / most : 0.;
        int8_t* qrow = static_cast<int8_t*>(a.n) + m * K;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int i = (c * NT + (int)threadIdx.x) * 8;
            if (i >= K) continue;
            int q[8];
#pragma unroll
            for (int e = 0; e < 8; e++) q[e] = fine ? code_of(p[c][e], f, most, 127) : 0;
            if (a.nvec && i + 8 <= K) {
                *reinterpret_cast<uint2*>(qrow + i) = pack8(q);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (i + e < K) qrow[i + e] = (int8_t)q[e];
            }
        }
        if (threadIdx.x == 0) a.n_scale[m] = scale_of(most, r, 127);
    } else {                                     // K % 128 == 0: a 128-group is a run of 16 lanes
        const double top = a.form == kAct ? 127 : 119;
        int8_t* qrow = static_cast<int8_t*>(a.n) + m * K;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int i = (c * NT + (int)threadIdx.x) * 8;
            double g = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) g = max2(g, magnitude(p[c][e]));
            g = max2(g, pair_of<0>(g));
            g = max2(g, pair_of<1>(g));
            g = max2(g, pair_of<2>(g));
            g = max2(g, pair_of<3>(g));
            if (i >= K) continue;
            const bool fine = g > 0 && g < __builtin_inf();
            const double f = fine ? top / g : 0.;
            int q[8];
#pragma unroll
            for (int e = 0; e < 8; e++) q[e] = fine ? code_of(p[c][e], f, g, top) : 0;
            *reinterpret_cast<uint2*>(qrow + i) = interleave8(q);
            const int gi = i >> 7;
            if ((threadIdx.x & 15) == 0) a.n_scale[a.form == kAct ? m * (K >> 7) + gi : (size_t)gi * a.M + m] = scale_of(g, r, top);
        }
    }
}

template <int C, class TH, class TY, bool NORM>
void launch(const BlockNorm& a, int threads, hipStream_t st) {
    hipLaunchKernelGGL((norm_k<C, TH, TY, NORM>), dim3((unsigned)a.M), dim3((unsigned)threads), 0, st, a);
}
template <class TH, class TY, bool NORM>
void launch_chunks(const BlockNorm& a, hipStream_t st) {
    const int lanes = (a.K + 7) / 8;
    // One chunk a thread while that is at most a workgroup; with many rows two, so that a CU holds several rows.
    int C = 1;
    while (lanes > C * 1024 || (C < 2 && a.M >= 1024 && lanes > 64)) C *= 2;
    const int threads = ((lanes + C - 1) / C + 63) / 64 * 64;
    if (C == 1) launch<1, TH, TY, NORM>(a, threads, st);
    else if (C == 2) launch<2, TH, TY, NORM>(a, threads, st);
    else if (C == 4) launch<4, TH, TY, NORM>(a, threads, st);
    else launch<8, TH, TY, NORM>(a, threads, st);
}
template <class TH>
void launch_y(const BlockNorm& a, hipStream_t st) {
    if (!a.y) a.w ? launch_chunks<TH, None, true>(a, st) : launch_chunks<TH, None, false>(a, st);
    else if (a.y_type == kF32) launch_chunks<TH, float, true>(a, st);
    else if (a.y_type == kBF16) launch_chunks<TH, bf16, true>(a, st);
    else launch_chunks<TH, f16, true>(a, st);
}

}  // namespace

hipError_t launch_block_norm(const BlockNorm& a, hipStream_t st) {
    if (a.h_type == kF32) launch_y<float>(a, st);
    else if (a.h_type == kBF16) launch_y<bf16>(a, st);
    else launch_y<f16>(a, st);
    return hipGetLastError();
}

}  // namespace rt4
