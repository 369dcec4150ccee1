// linear8.hip -- products of int8 codes with a scale for each token and each channel, and the first half of
// a gated feed-forward block on them.
//
//   c[m][n] = sx[m] sw[n] Σ_k xq[m][k] wq[n][k]                     (exact int32 sums, K < 2^17)
//   h[m][n] = act(sx[m] sg[n] Σ_k xq[m][k] wg[n][k]) * (sx[m] su[n] Σ_k xq[m][k] wu[n][k])
#include "ffn_dev.h"
#include "rt4_internal.h"

namespace rt4 {

namespace {

template <class T>
__device__ __forceinline__ void store_out(const Linear8& a, int m, int n, float v) {
    static_cast<T*>(a.out)[(size_t)m * a.ldo + n] = (T)v;
}

// One output from its sums: the sums are converted once (2^-24), the scales applied one after the other.
template <int ACT>
__device__ __forceinline__ float finish(int i0, int i1, float sx, float s0, float s1) {
    const float g = (float)i0 * sx * s0;
    return ACT < 0 ? g : activate<ACT>(g) * ((float)i1 * sx * s1);
}

// A wave owns 32 x 32 outputs and loads the operands of v_mfma_i32_32x32x32_i8 from memory.
template <int ACT, class T>
__global__ __launch_bounds__(256) void linear8_k(Linear8 a) {
    constexpr int NW = ACT < 0 ? 1 : 2;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int m0 = blockIdx.y * 32, n0 = (blockIdx.x * 4 + w) * 32;
    if (n0 >= a.N) return;
    const int r = lane & 31, kh = (lane >> 5) * 16;
    const int8_t* xp = a.x + (size_t)min(m0 + r, a.M - 1) * a.ldx;
    const int8_t* wp[NW];
    v16i acc[NW];
#pragma unroll
    for (int j = 0; j < NW; j++) {
        wp[j] = a.w[j] + (size_t)min(n0 + r, a.N - 1) * a.ldw[j];
#pragma unroll
        for (int i = 0; i < 16; i++) acc[j][i] = 0;
    }
    for (int k = kh; k < a.K + kh; k += 32) {
        v4i x = {0, 0, 0, 0}, v[NW] = {};
        if (k < a.K) {
            x = *reinterpret_cast<const v4i*>(xp + k);
#pragma unroll
            for (int j = 0; j < NW; j++) v[j] = *reinterpret_cast<const v4i*>(wp[j] + k);
        }
#pragma unroll
        for (int j = 0; j < NW; j++) acc[j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(x, v[j], acc[j], 0, 0, 0);
    }
    const int n = n0 + r;
    if (n >= a.N) return;
    const float s0 = a.sw[0][n], s1 = NW == 2 ? a.sw[NW - 1][n] : 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int m = m0 + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3);
        if (m < a.M) store_out<T>(a, m, n, finish<ACT>(acc[0][i], acc[NW - 1][i], a.sx[m], s0, s1));
    }
}

template <int ACT>
void launch_type(const Linear8& a, dim3 grid, hipStream_t st) {
    if (a.type == kF32) hipLaunchKernelGGL((linear8_k<ACT, float>), grid, dim3(256), 0, st, a);
    else if (a.type == kBF16) hipLaunchKernelGGL((linear8_k<ACT, bf16>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((linear8_k<ACT, f16>), grid, dim3(256), 0, st, a);
}

}  // namespace

hipError_t launch_linear8(const Linear8& a, hipStream_t st) {
    const dim3 grid((unsigned)((a.N + 127) / 128), (unsigned)((a.M + 31) / 32));
    if (a.act < 0) launch_type<-1>(a, grid, st);
    else if (a.act == 0) launch_type<0>(a, grid, st);
    else launch_type<1>(a, grid, st);
    return hipGetLastError();
}

}  // namespace rt4
