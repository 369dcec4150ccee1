// gate4.hip -- the first half of a gated feed-forward block on RT4 weights, 1 to 4 rows (a decode step).
//
//   h[m][n] = act(g[m][n]) * u[m][n],   g, u = Σ_g f16(ws[n][g]) sa[m][g] Σ_{k in g} code[n][k] xq[m][k]
//
// A stream of weights, read once: a wave owns 4 weight rows (gate and up rows of 2 channels) and goes through them 1 KB of
// each at a time, a lane 32 codes of a row (a quarter of a 128-group).  The activation codes and scales of all tokens lie in
// LDS, where a lane takes the 32 codes of each token that meet its weights, for all 4 rows; so a wave's registers hold
// little but weights, of this KB and of the next, and a CU many waves.  The vector ALU needs 12 operations to unpack 16
// bytes of codes to int8 (times 16), and 8 v_dot4 and 3 for the fold a token.
// The quarter sums are exact and folded as rt4_gemv_w4a8_q folds group sums, fp32(16 I) * (f16(ws) / 16 * sa).
#include "ffn_dev.h"
#include "rt4_internal.h"

namespace rt4 {

namespace {

constexpr int kMaxWaves = 8;

// LDS: the codes in two planes (first and second 16 bytes of every 32, so that a wave reads 1 KB in a row), M planes pairs of
// K/2 bytes each, then the scales [K/128][M].
template <int M>
__global__ __launch_bounds__(64 * kMaxWaves) void gate4_k(Gate4 a) {
    typedef unsigned v4 __attribute__((ext_vector_type(4)));
    extern __shared__ __align__(16) unsigned char smem[];
    const int lane = threadIdx.x & 63, W = blockDim.x >> 6;
    const int n0 = uniform((int)(blockIdx.x * W + (threadIdx.x >> 6))) * 2;
    const int RS = a.K >> 1, NG = a.K >> 7;
    const unsigned char* wp[4];
    const uint16_t* sp[4];
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const size_t n = min(n0 + (r & 1), a.N - 1);
        wp[r] = reinterpret_cast<const unsigned char*>(a.w[r >> 1]) + n * RS;
        sp[r] = a.ws[r >> 1] + n * NG;
    }
    struct Piece {
        v4 w[4];
        uint16_t s[4];
    } p[2];
    const auto load = [&](Piece& q, int o) {     // the lanes' pieces of the KB at o; past the rows' end the last piece (not folded)
        const uint32_t b = min(o + lane * 16, RS - 16);
#pragma unroll
        for (int r = 0; r < 4; r++) q.w[r] = __builtin_nontemporal_load(reinterpret_cast<const v4*>(wp[r] + b));
#pragma unroll
        for (int r = 0; r < 4; r++) q.s[r] = sp[r][b >> 6];
    };
    load(p[0], 0);
    for (int i = threadIdx.x; i < M * (a.K >> 4); i += blockDim.x) {
        const int m = i / (a.K >> 4), c = i - m * (a.K >> 4);
        reinterpret_cast<v4*>(smem)[(2 * m + (c & 1)) * (RS >> 4) + (c >> 1)] = reinterpret_cast<const v4*>(a.xq)[i];
    }
    float* sl = reinterpret_cast<float*>(smem + (size_t)M * a.K);
    for (int i = threadIdx.x; i < M * NG; i += blockDim.x) sl[i % NG * M + i / NG] = a.sa[i];
    __syncthreads();
    float y[4][M] = {};
    const auto fold = [&](const Piece& q, int o) {
        const int b = o + lane * 16;
        if (b >= RS) return;
        float sa[M];
#pragma unroll
        for (int m = 0; m < M; m++) sa[m] = sl[(b >> 6) * M + m];
        float s[4];
#pragma unroll
        for (int r = 0; r < 4; r++) s[r] = f16_bits_to_f32(q.s[r]) * 0.0625f;
        uint32_t c[4][8];
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int e = 0; e < 4; e++) c[r][2 * e] = even_x16(q.w[r][e]), c[r][2 * e + 1] = odd_x16(q.w[r][e]);
#pragma unroll
        for (int m = 0; m < M; m++) {
            const v4 x[2] = {*reinterpret_cast<const v4*>(smem + (2 * m) * RS + b), *reinterpret_cast<const v4*>(smem + (2 * m + 1) * RS + b)};
#pragma unroll
            for (int r = 0; r < 4; r++) {
                int I = 0;
#pragma unroll
                for (int e = 0; e < 8; e++) I = __builtin_amdgcn_sdot4((int)c[r][e], (int)x[e >> 2][e & 3], I, false);
                y[r][m] = fmaf((float)I, s[r] * sa[m], y[r][m]);
            }
        }
    };
    int o = 0;
    for (; o + 2048 < RS; o += 2048) {
        load(p[1], o + 1024);
        __builtin_amdgcn_sched_barrier(0);
        fold(p[0], o);
        load(p[0], o + 2048);
        __builtin_amdgcn_sched_barrier(0);
        fold(p[1], o + 1024);
    }
    if (o + 1024 < RS) {
        load(p[1], o + 1024);
        __builtin_amdgcn_sched_barrier(0);
        fold(p[0], o);
        fold(p[1], o + 1024);
    } else {
        fold(p[0], o);
    }
    float g = 0.f, u = 0.f;                      // lane 2 m + c: token m, channel c
#pragma unroll
    for (int m = 0; m < M; m++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const float v = wave_sum(y[r][m]);
            if (r < 2) g = lane == 2 * m + r ? v : g;
            else u = lane == 2 * m + r - 2 ? v : u;
        }
    const int m = lane >> 1, n = n0 + (lane & 1);
    if (m < M && n < a.N) a.out[(size_t)m * a.N + n] = activate(g, a.act) * u;
}

template <int M>
hipError_t launch_rows(const Gate4& a, int waves, hipStream_t st) {
    const size_t lds = (size_t)M * a.K + (size_t)M * (a.K >> 7) * 4;
    if (lds > 65536) {                           // (what a launch is granted without asking)
        hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(gate4_k<M>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((gate4_k<M>), dim3((unsigned)((a.N + 2 * waves - 1) / (2 * waves))), dim3(64 * waves), lds, st, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_gate4(const Gate4& a, int cus, hipStream_t st) {
    // Waves share the activations in LDS, as far as that leaves every CU two workgroups.
    int waves = kMaxWaves;
    while (waves > 1 && (a.N + 2 * waves - 1) / (2 * waves) < 2 * cus) waves >>= 1;
    switch (a.rows) {
        case 1: return launch_rows<1>(a, waves, st);
        case 2: return launch_rows<2>(a, waves, st);
        case 3: return launch_rows<3>(a, waves, st);
        default: return launch_rows<4>(a, waves, st);
    }
}

}  // namespace rt4
