// gate4.hip -- the first half of a gated feed-forward block on RT4 weights, 1 to 4 rows (a decode step).
//
//   h[m][n] = act(g[m][n]) * u[m][n],   g, u = Σ_g f16(ws[n][g]) sa[m][g] Σ_{k in g} code[n][k] xq[m][k]
#include "ffn_dev.h"
#include "rt4_internal.h"

namespace rt4 {

namespace {

// A wave owns one output column: lane l takes 16 bytes (a quarter of a 128-group) of both its weight rows.
template <int M>
__global__ __launch_bounds__(256) void gate4_k(Gate4 a) {
    const int lane = threadIdx.x & 63;
    const int n = uniform((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
    if (n >= a.N) return;
    const int RS = a.K >> 1, NG = a.K >> 7;
    float y[2][M] = {};
    for (int o = lane * 16; o < RS; o += 1024) {
        const int g = o >> 6;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const uint4 w = *reinterpret_cast<const uint4*>(reinterpret_cast<const unsigned char*>(a.w[j]) + (size_t)n * RS + o);
            const float s = f16_bits_to_f32(a.ws[j][(size_t)n * NG + g]) * 0.0625f;
#pragma unroll
            for (int m = 0; m < M; m++) {
                const uint4* xp = reinterpret_cast<const uint4*>(a.xq + (size_t)m * a.K + 2 * o);
                const uint4 x0 = xp[0], x1 = xp[1];
                int I = 0;
                I = __builtin_amdgcn_sdot4((int)even_x16(w.x), (int)x0.x, I, false);
                I = __builtin_amdgcn_sdot4((int)odd_x16(w.x), (int)x0.y, I, false);
                I = __builtin_amdgcn_sdot4((int)even_x16(w.y), (int)x0.z, I, false);
                I = __builtin_amdgcn_sdot4((int)odd_x16(w.y), (int)x0.w, I, false);
                I = __builtin_amdgcn_sdot4((int)even_x16(w.z), (int)x1.x, I, false);
                I = __builtin_amdgcn_sdot4((int)odd_x16(w.z), (int)x1.y, I, false);
                I = __builtin_amdgcn_sdot4((int)even_x16(w.w), (int)x1.z, I, false);
                I = __builtin_amdgcn_sdot4((int)odd_x16(w.w), (int)x1.w, I, false);
                y[j][m] = fmaf((float)I, s * a.sa[(size_t)m * NG + g], y[j][m]);
            }
        }
    }
#pragma unroll
    for (int m = 0; m < M; m++) {
        const float g = wave_sum(y[0][m]), u = wave_sum(y[1][m]);
        if (lane == 0) a.out[(size_t)m * a.N + n] = activate(g, a.act) * u;
    }
}

template <int M>
void launch_rows(const Gate4& a, hipStream_t st) {
    const dim3 grid((unsigned)((a.N + 3) / 4));
    hipLaunchKernelGGL((gate4_k<M>), grid, dim3(256), 0, st, a);
}

}  // namespace

hipError_t launch_gate4(const Gate4& a, hipStream_t st) {
    switch (a.rows) {
        case 1: launch_rows<1>(a, st); break;
        case 2: launch_rows<2>(a, st); break;
        case 3: launch_rows<3>(a, st); break;
        default: launch_rows<4>(a, st); break;
    }
    return hipGetLastError();
}

}  // namespace rt4
