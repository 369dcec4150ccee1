// attn_tree.hip -- attention of a tree of new tokens over an int4-KV cache, gfx950
// (rt4_attention_tree; one token and a chain are trees too).  No counterpart in the
// reference, whose decode attention (src/k_fa.hip:154-240) stays the caller's.
//
// Formats of qq, qsc, kc, ksc, vc, vsc are those in the header of attn.hip, with B
// caches one after the other; the new tokens' own keys are one more 64-key tile per
// sequence and KV head in the same format.  Row b * T + i is node i of sequence b.
//   S[i][k] = sum over the two 128-dim groups of I_g qs_g ks_g (I_g the codes' exact dot
//   product), k over the cache's keys before kv_len[b] and the nodes that are i or above
//   it; out = softmax(S) V.  A node that hangs under no root sees nothing: zeros.
// P stays in fp32 (the reference's decode attention does the same; the prefill's int4 P
// would cost a relative 1e-2 per row when there are few keys).
#include "rt4_dev.h"
#include "rt4_internal.h"

namespace rt4 {
namespace {

constexpr int HD = 256, KDW = HD / 8, BNK = 64;
constexpr float L2E = 1.4426950408889634f;
typedef unsigned long long u64;

// Nodes that node i of sequence b sees: itself and those above it, none where it hangs
// under no root.  Lane i of the wave has node i.
__device__ __forceinline__ u64 tree_sees(const int* parent, int T) {
    const int i = threadIdx.x & 63;
    const int par = i < T ? parent[i] : -2;
    const bool root = i == 0 && par == -1, node = i > 0 && par >= 0 && par < i;
    int up = node ? par : i;
    u64 anc = 1ull << i;
#pragma unroll
    for (int s = 0; s < 6; s++) {        // pointer doubling: 2^6 covers the deepest chain
        anc |= __shfl(anc, up);
        up = __shfl(up, up);
    }
    return (root || node) && __shfl((int)root, 0) && (anc & 1) ? anc : 0;
}

// One workgroup per (row, head).
__global__ __launch_bounds__(256) void attn_tree_k(const AttnTree A) {
    __shared__ float sp[BNK], red[4];
    const int tid = threadIdx.x, head = blockIdx.x, i = blockIdx.y, b = blockIdx.z, vh = head / A.ratio, KVH = A.n_heads / A.ratio;
    const u64 sees = __shfl(tree_sees(A.parent + (size_t)b * A.T, A.T), i);
    const size_t row = (size_t)b * A.T + i;
    float* out = A.out + ((size_t)head * A.TP + row) * HD;
    if (!sees) {
        out[tid] = 0.f;
        return;
    }
    int len = A.kv_len ? A.kv_len[b] : 0;
    len = len < 0 ? 0 : len > A.kv_cap ? A.kv_cap : len;
    const int nt = (len + BNK - 1) / BNK;
    const size_t seq = (size_t)b * KVH + vh;
    const int key = tid >> 2, part = tid & 3;
    uint32_t q[8];
    for (int e = 0; e < 8; e++) q[e] = A.qq[((size_t)head * A.TP + row) * KDW + 8 * part + e];
    const float qs = A.qsc[((size_t)head * 2 + (part >> 1)) * A.TP + row] * L2E;
    float m = -1e30f, l = 0.f, o = 0.f;
    for (int t = 0; t <= nt; t++) {
        const bool draft = t == nt;
        const int cap = draft ? BNK : A.kv_cap, k0 = draft ? 0 : t * BNK;
        const uint32_t* kc = (draft ? A.kd : A.kc) + (seq * cap + k0 + key) * KDW + 8 * part;
        const float* ksc = (draft ? A.ksd : A.ksc) + (seq * 2 + (part >> 1)) * cap + k0 + key;
        int dot = 0;
        for (int e = 0; e < 8; e++) dot = __builtin_amdgcn_sdot8((int)q[e], (int)kc[e], dot, false);
        float s = (float)dot * (qs * ksc[0]);
        s += __shfl_xor(s, 1);
        s += __shfl_xor(s, 2);
        if (!(draft ? sees >> key & 1 : k0 + key < len)) s = -INFINITY;
        float mt = s;
        for (int x = 4; x < 64; x <<= 1) mt = fmaxf(mt, __shfl_xor(mt, x));
        __syncthreads();
        if ((tid & 63) == 0) red[tid >> 6] = mt;
        __syncthreads();
        mt = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), m);
        const float alpha = exp2f(m - mt), p = exp2f(s - mt);
        m = mt;
        if (part == 0) sp[key] = p;
        __syncthreads();
        const uint32_t* vc = (draft ? A.vd : A.vc) + (seq * (cap / 8) + k0 / 8) * HD + tid;
        const float vs = (draft ? A.vsd : A.vsc)[(seq * (cap / BNK) + k0 / BNK) * HD + tid];
        float acc = 0.f, sum = 0.f;
        for (int g = 0; g < 8; g++) {
            const uint32_t w = vc[(size_t)g * HD];
            for (int e = 0; e < 8; e++) {
                const float pe = sp[8 * g + e];
                acc += pe * (float)((int)(w << (28 - 4 * e)) >> 28);
                sum += pe;
            }
        }
        o = o * alpha + acc * vs;
        l = l * alpha + sum;
    }
    out[tid] = o / l;
}

}  // namespace

hipError_t launch_attn_tree(const AttnTree& a, hipStream_t st) {
    hipLaunchKernelGGL(attn_tree_k, dim3(a.n_heads, a.T, a.B), dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace rt4
