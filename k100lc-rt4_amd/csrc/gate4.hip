// gate4.hip -- the first half of a gated feed-forward block on RT4 weights, 1 to 4 rows (a decode step).
//
//   h[m][n] = act(g[m][n]) * u[m][n],   g, u = Σ_g f16(ws[n][g]) sa[m][g] Σ_{k in g} code[n][k] xq[m][k]
//
// A stream of weights, read once: a wave owns 4 weight rows (gate and up rows of 2 channels) and goes through them 1 KB of
// each at a time, a lane 32 codes of a row (a quarter of a 128-group).  The activation codes and scales of all tokens lie in
// LDS, where a lane takes the 32 codes of each token that meet its weights, for all 4 rows; so a wave's registers hold
// little but weights, of this KB and of the next, and a CU many waves.  The vector ALU needs 12 operations to unpack 16
// bytes of codes to int8 (times 16), and 8 v_dot4 and 3 for the fold a token.
// A wave goes on to further pairs without a pause, so that loads and arithmetic overlap throughout.
// The quarter sums are exact and folded as rt4_gemv_w4a8_q folds group sums, fp32(16 I) * (f16(ws) / 16 * sa).
#include <atomic>
#include <type_traits>

#include "ffn_dev.h"
#include "rt4_internal.h"

namespace rt4 {

namespace {

constexpr int kMaxWaves = 8;

// LDS: the codes in two planes for each token (first and second 16 bytes of every 32, so that a wave reads 1 KB in a row) of
// K/2 bytes, then the scales over 16 (the codes are unpacked times 16), [K/128][M].
template <int M>
__global__ __launch_bounds__(64 * kMaxWaves) void gate4_k(Gate4 a) {
    typedef unsigned v4 __attribute__((ext_vector_type(4)));
    extern __shared__ __align__(16) unsigned char smem[];
    const int lane = threadIdx.x & 63, W = blockDim.x >> 6;
    const int RS = a.K >> 1, NG = a.K >> 7;
    // A wave's channel pairs, and the pieces of a pair: whole KB of all four rows, and what is left behind them, where it is at
    // most half a KB, by half a wave for each channel.
    const int first = uniform((int)(blockIdx.x * W + (threadIdx.x >> 6))) * 2, stride = gridDim.x * W * 2;
    const int left = RS & 1023, whole = RS - left + (left > 512 ? 1024 : 0), end = whole + (left > 0 && left <= 512 ? 1024 : 0);
    v4 pw[2][4];                                 // two pieces: codes and scales
    uint32_t ps[2][4];
    struct Place {
        int n0, o;
    };
    const auto next = [&](Place c) {
        c.o += 1024;
        if (c.o >= end) c.o = 0, c.n0 += stride;
        return c;
    };
    const int tb = whole + (lane & 31) * 16;
    const auto load = [&](auto buf, Place c) __attribute__((always_inline)) {   // past the rows' end the last piece (it is not folded)
        constexpr int Q = decltype(buf)::value;
        if (c.n0 >= a.N) return;
        const int other = c.n0 + 1 < a.N;        // rows to the second channel's (the first's again past the last)
        if (c.o < whole) {
            const uint32_t b = min(c.o + lane * 16, RS - 16);
#pragma unroll
            for (int r = 0; r < 4; r++)
                pw[Q][r] = __builtin_nontemporal_load(reinterpret_cast<const v4*>(reinterpret_cast<const unsigned char*>(a.w[r >> 1]) + (size_t)(c.n0 + (r & other)) * RS + b));
#pragma unroll
            for (int r = 0; r < 4; r++) ps[Q][r] = (a.ws[r >> 1])[(size_t)(c.n0 + (r & other)) * NG + (b >> 6)];
        } else {
            const uint32_t b = min(tb, RS - 16), half = lane >> 5 & other;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                pw[Q][j] = __builtin_nontemporal_load(reinterpret_cast<const v4*>(reinterpret_cast<const unsigned char*>(a.w[j]) + (size_t)c.n0 * RS + (half * (uint32_t)RS + b)));
                ps[Q][j] = a.ws[j][(size_t)c.n0 * NG + (half * NG + (b >> 6))];
            }
        }
    };
    typedef std::integral_constant<int, 0> zero;
    typedef std::integral_constant<int, 1> one;
    Place at{first, 0};
    load(zero{}, at);
#pragma unroll
    for (int m = 0; m < M; m++)
        for (int c = threadIdx.x; c < a.K >> 4; c += blockDim.x)
            reinterpret_cast<v4*>(smem)[(2 * m + (c & 1)) * (RS >> 4) + (c >> 1)] = reinterpret_cast<const v4*>(a.xq + (size_t)m * a.K)[c];
    float* sl = reinterpret_cast<float*>(smem + (size_t)M * a.K);
#pragma unroll
    for (int m = 0; m < M; m++)
        for (int g = threadIdx.x; g < NG; g += blockDim.x) sl[g * M + m] = a.sa[(size_t)m * NG + g] * 0.0625f;
    __syncthreads();
    float y[4][M] = {}, yt[2][M] = {};
    const auto fold = [&](auto buf, int b, auto rows, auto& y) __attribute__((always_inline)) {
        constexpr int Q = decltype(buf)::value, R = decltype(rows)::value;
        if (b >= RS) return;
        float sa[M], s[R];
#pragma unroll
        for (int m = 0; m < M; m++) sa[m] = sl[(b >> 6) * M + m];
#pragma unroll
        for (int r = 0; r < R; r++) s[r] = f16_bits_to_f32((uint16_t)ps[Q][r]);
        uint32_t c[R][8];
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int e = 0; e < 4; e++) c[r][2 * e] = even_x16(pw[Q][r][e]), c[r][2 * e + 1] = odd_x16(pw[Q][r][e]);
#pragma unroll
        for (int m = 0; m < M; m++) {
            const v4 x[2] = {*reinterpret_cast<const v4*>(smem + (2 * m) * RS + b), *reinterpret_cast<const v4*>(smem + (2 * m + 1) * RS + b)};
#pragma unroll
            for (int r = 0; r < R; r++) {
                int I = 0;
#pragma unroll
                for (int e = 0; e < 8; e++) I = __builtin_amdgcn_sdot4((int)c[r][e], (int)x[e >> 2][e & 3], I, false);
                y[r][m] = fmaf((float)I, s[r] * sa[m], y[r][m]);
            }
        }
    };
    // Sums over the lanes, several in one register: halves of the wave for the channels, then rows of 16 for gate and up.
    const auto finish = [&](int n0) __attribute__((always_inline)) {
        float g = 0.f, u = 0.f;                  // lane 32 c + m (and its copy 16 lanes on): channel c, token m
#pragma unroll
        for (int m = 0; m < M; m++) {
            float z[2];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, y[2 * j][m]), __builtin_bit_cast(uint32_t, y[2 * j + 1][m]), false, false);
                z[j] = __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]) + yt[j][m];
                y[2 * j][m] = y[2 * j + 1][m] = yt[j][m] = 0.f;
            }
            const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, z[0]), __builtin_bit_cast(uint32_t, z[1]), false, false);
            float v = __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
            v += pair_of<0>(v);
            v += pair_of<1>(v);
            v += pair_of<2>(v);
            v += pair_of<3>(v);
            const auto h = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
            g = (lane & 15) == m ? __builtin_bit_cast(float, (uint32_t)h[0]) : g;
            u = (lane & 15) == m ? __builtin_bit_cast(float, (uint32_t)h[1]) : u;
        }
        const int m = lane & 15, n = n0 + (lane >> 5);
        if (m < M && !(lane & 16) && n < a.N) a.out[(size_t)m * a.N + n] = activate(g, a.act) * u;
    };
    const auto use = [&](auto buf, Place c) __attribute__((always_inline)) {
        if (c.o < whole) fold(buf, c.o + lane * 16, std::integral_constant<int, 4>{}, y);
        else fold(buf, tb, std::integral_constant<int, 2>{}, yt);
        if (c.o + 1024 >= end) finish(c.n0);
    };
    while (at.n0 < a.N) {                        // the next piece is under way while one is used
        const Place b = next(at);
        load(one{}, b);
        __builtin_amdgcn_sched_barrier(0);
        use(zero{}, at);
        if (b.n0 >= a.N) return;
        at = next(b);
        load(zero{}, at);
        __builtin_amdgcn_sched_barrier(0);
        use(one{}, b);
    }
}

constexpr size_t lds_bytes(int rows, int K) { return (size_t)rows * K + (size_t)rows * (K >> 7) * 4; }

// The limit of a launch's LDS is the kernel's on a device, shared by all threads that call it: it is raised once, to what the
// largest K needs, and never lowered under another thread's launch.
template <int M>
hipError_t raise_lds_limit() {
    constexpr int kMaxDev = 64;
    static std::atomic<bool> raised[kMaxDev];
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const bool known = dev >= 0 && dev < kMaxDev;
    if (known && raised[dev].load(std::memory_order_acquire)) return hipSuccess;
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(gate4_k<M>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds_bytes(M, kGate4MaxK));
    if (e == hipSuccess && known) raised[dev].store(true, std::memory_order_release);
    return e;
}

template <int M>
hipError_t launch_rows(const Gate4& a, int cus, hipStream_t st) {
    const size_t lds = lds_bytes(M, a.K);
    if (lds > 65536) {                           // (what a launch is granted without asking)
        const hipError_t e = raise_lds_limit<M>();
        if (e != hipSuccess) return e;
    }
    // Two workgroups a CU (one where LDS holds no more), of as many waves as leave every CU one at least (4 rows of 5120 x 17408:
    // 8 waves 22.4 us, 6 25.8, 4 24.4; one row of 2048 x 2051: 4 waves 3.1 us, 8 3.4, 3 3.5).
    const int slots = cus * (lds <= 80 * 1024 ? 2 : 1), pairs = (a.N + 1) / 2;
    const int waves = pairs / cus < 1 ? 1 : pairs / cus < kMaxWaves ? pairs / cus : kMaxWaves;
    const int groups = (pairs + waves - 1) / waves;
    hipLaunchKernelGGL((gate4_k<M>), dim3((unsigned)(groups < slots ? groups : slots)), dim3(64 * waves), lds, st, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_gate4(const Gate4& a, int cus, hipStream_t st) {
    switch (a.rows) {
        case 1: return launch_rows<1>(a, cus, st);
        case 2: return launch_rows<2>(a, cus, st);
        case 3: return launch_rows<3>(a, cus, st);
        default: return launch_rows<4>(a, cus, st);
    }
}

}  // namespace rt4
