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

typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

__device__ __forceinline__ int lane_id() { return threadIdx.x & 63; }

// Max over the four lanes that hold one query row's keys (lanes 16 and 32 apart).
__device__ __forceinline__ float max_groups(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}

// 16 int8 operand bytes (16 x code) of two code dwords.
__device__ __forceinline__ v4i bytes16(uint32_t a, uint32_t b) {
    return v4i{(int)even_x16(a), (int)odd_x16(a), (int)even_x16(b), (int)odd_x16(b)};
}

// The eight codes of a V dword as fp16, key pairs (0,4) (1,5) (2,6) (3,7): the nibble + 8 under
// the exponent of 1024 is 1024 + u (or 1024 + 16 u one nibble up), from which a packed add (or
// fma) takes the code exactly.
__device__ __forceinline__ v8h codes_f16(uint32_t w) {
    const uint32_t x = w ^ 0x88888888u, y = x >> 8;
    const uint32_t t[4] = {(x & 0x000F000Fu) | 0x64006400u, (x & 0x00F000F0u) | 0x64006400u, (y & 0x000F000Fu) | 0x64006400u,
                           (y & 0x00F000F0u) | 0x64006400u};
    union {
        v2h p[4];
        v8h v;
    } r;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const v2h a = __builtin_bit_cast(v2h, t[k]);
        r.p[k] = (k & 1) ? a * v2h{(_Float16)0.0625f, (_Float16)0.0625f} + v2h{(_Float16)-72.f, (_Float16)-72.f}
                         : a + v2h{(_Float16)-1032.f, (_Float16)-1032.f};
    }
    return r.v;
}

constexpr float kPBits = 7.f;            // P is held times 2^7: at most 2^15 with the lazy maximum
constexpr float kLazy = 8.f;             // the running maximum moves when a tile exceeds it by 2^8

// A workgroup owns 16 NB query rows of one (sequence, KV head) -- rows r * T + i, r the head in
// the group, i the node -- and a range of the keys' 64-key tiles, the draft tile last; its four
// waves take every fourth tile and keep their own softmax state, joined through LDS at the end.
template <int NB>
__global__ __launch_bounds__(256, 1) void attn_tree_k(const AttnTree A, const TreePlan P, float* __restrict__ opart,
                                                      float2* __restrict__ mlpart) {
    constexpr int RW = 16 * NB;
    __shared__ __align__(16) float ol[4][16][HD];
    __shared__ float ml[2][4][RW];
    const int tid = threadIdx.x, lane = lane_id(), w = uniform(tid >> 6), c = lane & 15, g = lane >> 4;
    // the row groups of one unit (sequence, KV head, split) on one XCD: workgroups go round the 8
    const int rg = (int)(blockIdx.x / 8) % P.groups;
    const int unit = (int)(blockIdx.x / (8 * P.groups)) * 8 + (int)(blockIdx.x % 8);
    const int KVH = A.n_heads / A.ratio, R = A.T * A.ratio;
    if (unit >= A.B * KVH * P.splits) return;
    const int split = unit % P.splits, seq = unit / P.splits, b = seq / KVH, vh = seq % KVH;
    int len = A.kv_len ? A.kv_len[b] : 0;
    len = uniform(len < 0 ? 0 : len > A.kv_cap ? A.kv_cap : len);
    const int nt = (len + BNK - 1) / BNK;                      // tile nt is the draft tile
    const int t0 = (int)((long long)(nt + 1) * split / P.splits), t1 = (int)((long long)(nt + 1) * (split + 1) / P.splits);

    // Q operands: column c of block nb is row n
    v4i qop[NB][4];
    float qs0[NB], qs1[NB];
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
        int n = rg * RW + nb * 16 + c;
        n = n < R ? n : R - 1;
        const size_t head = (size_t)vh * A.ratio + n / A.T, row = (size_t)b * A.T + n % A.T;
        const uint32_t* qr = A.qq + (head * A.TP + row) * KDW + 4 * g;
        const v4u d0 = *reinterpret_cast<const v4u*>(qr), d1 = *reinterpret_cast<const v4u*>(qr + 16);
        qop[nb][0] = bytes16(d0.x, d0.y);
        qop[nb][1] = bytes16(d0.z, d0.w);
        qop[nb][2] = bytes16(d1.x, d1.y);
        qop[nb][3] = bytes16(d1.z, d1.w);
        qs0[nb] = A.qsc[(head * 2) * A.TP + row] * (L2E / 256.f);   // (both operands are 16 x code)
        qs1[nb] = A.qsc[(head * 2 + 1) * A.TP + row] * (L2E / 256.f);
    }

    v4f O[NB][16];
    float m[NB], l[NB];
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
        m[nb] = -1e30f;
        l[nb] = 0.f;
#pragma unroll
        for (int t = 0; t < 16; t++) O[nb][t] = v4f{0.f, 0.f, 0.f, 0.f};
    }

    v4u K[4][2], V[2][4];
    v4f ks[4][2], vs[4];
    auto load_k = [&](int t) __attribute__((always_inline)) {
        const bool d = t == nt;
        const size_t cap = d ? BNK : A.kv_cap, k0 = d ? 0 : (size_t)t * BNK;
        const uint32_t* kb = (d ? A.kd : A.kc) + (seq * cap + k0) * KDW;
        const float* sb = (d ? A.ksd : A.ksc) + (size_t)seq * 2 * cap + k0;
        // operand row 4g + i of subtile 2h + p is key 32h + 8g + 4p + i: a lane's scores of subtiles
        // 2h and 2h + 1 are then one V dword's eight keys
        const uint32_t ko = (uint32_t)((8 * (c >> 2) + (c & 3)) * KDW + 4 * g);
#pragma unroll
        for (int sub = 0; sub < 4; sub++) {
            const int at = 32 * (sub >> 1) + 4 * (sub & 1);
            K[sub][0] = *reinterpret_cast<const v4u*>(kb + ko + at * KDW);
            K[sub][1] = *reinterpret_cast<const v4u*>(kb + ko + at * KDW + 16);
            ks[sub][0] = *reinterpret_cast<const v4f*>(sb + 8 * g + at);
            ks[sub][1] = *reinterpret_cast<const v4f*>(sb + cap + 8 * g + at);
        }
    };
    auto load_v = [&](int t) __attribute__((always_inline)) {
        const bool d = t == nt;
        const size_t cap = d ? BNK : A.kv_cap, k0 = d ? 0 : (size_t)t * BNK;
        const uint32_t* vb = (d ? A.vd : A.vc) + (seq * (cap / 8) + k0 / 8) * HD;
        const float* sb = (d ? A.vsd : A.vsc) + (seq * (cap / BNK) + k0 / BNK) * HD;
        // dim tile 4q + j, column c is dim 64q + 4c + j
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int q = 0; q < 4; q++) V[h][q] = *reinterpret_cast<const v4u*>(vb + (4 * h + g) * HD + 64 * q + 4 * c);
#pragma unroll
        for (int q = 0; q < 4; q++) vs[q] = *reinterpret_cast<const v4f*>(sb + 64 * q + 4 * c);
    };

    int t = t0 + w;
    if (t < t1) {
        load_k(t);
        load_v(t);
    }
    for (; t < t1; t += 4) {
        // S^T = K Q^T: lane (c, g) gets row c, keys 32h + 8g + 4p + i
        float s[NB][16];
#pragma unroll
        for (int sub = 0; sub < 4; sub++) {
            const v4i a0 = bytes16(K[sub][0].x, K[sub][0].y), a1 = bytes16(K[sub][0].z, K[sub][0].w);
            const v4i a2 = bytes16(K[sub][1].x, K[sub][1].y), a3 = bytes16(K[sub][1].z, K[sub][1].w);
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
                v4i x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
                x = __builtin_amdgcn_mfma_i32_16x16x64_i8(a0, qop[nb][0], x, 0, 0, 0);
                y = __builtin_amdgcn_mfma_i32_16x16x64_i8(a2, qop[nb][2], y, 0, 0, 0);
                x = __builtin_amdgcn_mfma_i32_16x16x64_i8(a1, qop[nb][1], x, 0, 0, 0);
                y = __builtin_amdgcn_mfma_i32_16x16x64_i8(a3, qop[nb][3], y, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; i++)
                    s[nb][4 * sub + i] = fmaf((float)x[i] * ks[sub][0][i], qs0[nb], ((float)y[i] * ks[sub][1][i]) * qs1[nb]);
            }
        }
        const int tn = t + 4;
        const bool draft = t == nt;
        if (tn < t1) load_k(tn);
        if (draft || (t + 1) * BNK > len) {                    // a tile with keys that some row may not see
            const u64 sees = draft ? tree_sees(A.parent + (size_t)b * A.T, A.T) : 0;
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
                int n = rg * RW + nb * 16 + c;
                n = n < R ? n : R - 1;
                u64 ok = __shfl(sees, n % A.T);
                if (!draft) ok = (1ull << (len - t * BNK)) - 1;
                ok >>= 8 * g;
#pragma unroll
                for (int e = 0; e < 16; e++)
                    if (!(ok >> (32 * (e >> 3) + (e & 7)) & 1)) s[nb][e] = -INFINITY;
            }
        }
        v8h ph[NB][2], pl[NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            float mt = s[nb][0];
#pragma unroll
            for (int e = 1; e < 16; e++) mt = fmaxf(mt, s[nb][e]);
            mt = max_groups(mt);
            if (__any(mt > m[nb] + kLazy)) {
                const float mn = fmaxf(m[nb], mt), alpha = __builtin_amdgcn_exp2f(m[nb] - mn);
                m[nb] = mn;
                l[nb] *= alpha;
                float ar[4];
#pragma unroll
                for (int i = 0; i < 4; i++) ar[i] = __shfl(alpha, 4 * g + i);
#pragma unroll
                for (int d = 0; d < 16; d++)
#pragma unroll
                    for (int i = 0; i < 4; i++) O[nb][d][i] *= ar[i];
            }
            const float ref = kPBits - m[nb];
            float sum = 0.f;
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const v2f p = {__builtin_amdgcn_exp2f(s[nb][8 * h + i] + ref), __builtin_amdgcn_exp2f(s[nb][8 * h + 4 + i] + ref)};
                    sum += p[0] + p[1];
                    const v2h hi = __builtin_convertvector(p, v2h);
                    const v2f r = {p[0] - (float)hi[0], p[1] - (float)hi[1]};
                    const v2h lo = __builtin_convertvector(r, v2h);
                    ph[nb][h][2 * i] = hi[0];
                    ph[nb][h][2 * i + 1] = hi[1];
                    pl[nb][h][2 * i] = lo[0];
                    pl[nb][h][2 * i + 1] = lo[1];
                }
            l[nb] += sum;
        }
        // O += P V: rows 4g + i, dim 64q + 4c + j
#pragma unroll
        for (int d = 0; d < 16; d++) {
            const v8h v0 = codes_f16(V[0][d >> 2][d & 3]), v1 = codes_f16(V[1][d >> 2][d & 3]);
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
                v4f a = {0.f, 0.f, 0.f, 0.f};
                a = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[nb][0], v0, a, 0, 0, 0);
                a = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl[nb][0], v0, a, 0, 0, 0);
                a = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[nb][1], v1, a, 0, 0, 0);
                a = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl[nb][1], v1, a, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; i++) O[nb][d][i] = fmaf(a[i], vs[d >> 2][d & 3], O[nb][d][i]);
            }
        }
        if (tn < t1) load_v(tn);
    }

    // join the waves
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
        float s = l[nb] + __shfl_xor(l[nb], 16);
        s += __shfl_xor(s, 32);
        if (g == 0) {
            ml[0][w][nb * 16 + c] = m[nb];
            ml[1][w][nb * 16 + c] = s;
        }
    }
    const u64 sees = P.splits == 1 ? tree_sees(A.parent + (size_t)b * A.T, A.T) : 0;
    const size_t prow = (size_t)unit * P.groups * RW + rg * RW;
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
        if (nb) __syncthreads();
#pragma unroll
        for (int q = 0; q < 4; q++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                *reinterpret_cast<v4f*>(&ol[w][4 * g + i][64 * q + 4 * c]) =
                    v4f{O[nb][4 * q][i], O[nb][4 * q + 1][i], O[nb][4 * q + 2][i], O[nb][4 * q + 3][i]};
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int r = 4 * k + w, n = rg * RW + nb * 16 + r;      // wave w joins row r, lane 4 dims
            float M = ml[0][0][nb * 16 + r];
            for (int x = 1; x < 4; x++) M = fmaxf(M, ml[0][x][nb * 16 + r]);
            v4f o = {0.f, 0.f, 0.f, 0.f};
            float ls = 0.f;
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const float f = __builtin_amdgcn_exp2f(ml[0][x][nb * 16 + r] - M);
                ls = fmaf(ml[1][x][nb * 16 + r], f, ls);
                const v4f v = *reinterpret_cast<const v4f*>(&ol[x][r][4 * lane]);
#pragma unroll
                for (int i = 0; i < 4; i++) o[i] = fmaf(v[i], f, o[i]);
            }
            if (P.splits > 1) {
                *reinterpret_cast<v4f*>(opart + (prow + nb * 16 + r) * HD + 4 * lane) = o;
                if (lane == 0) mlpart[prow + nb * 16 + r] = make_float2(M, ls);
            } else if (n < R) {
                const int i = n % A.T;
                const bool live = __shfl(sees, i) != 0;
                const size_t head = (size_t)vh * A.ratio + n / A.T;
                float* dst = A.out + (head * A.TP + (size_t)b * A.T + i) * HD + 4 * lane;
                *reinterpret_cast<v4f*>(dst) = live ? v4f{o[0] / ls, o[1] / ls, o[2] / ls, o[3] / ls} : v4f{0.f, 0.f, 0.f, 0.f};
            }
        }
    }
}

// Sums the splits' states: one wave per row, four dims a lane.
__global__ __launch_bounds__(256) void attn_tree_join_k(const AttnTree A, const TreePlan P, const float* __restrict__ opart,
                                                        const float2* __restrict__ mlpart) {
    const int KVH = A.n_heads / A.ratio, R = A.T * A.ratio, lane = lane_id();
    const int n = (int)blockIdx.x * 4 + uniform(threadIdx.x >> 6), seq = blockIdx.y, b = seq / KVH, vh = seq % KVH;
    if (n >= R) return;
    const int i = n % A.T;
    const bool live = __shfl(tree_sees(A.parent + (size_t)b * A.T, A.T), i) != 0;
    const size_t step = (size_t)P.groups * 16 * P.blocks, row = (size_t)seq * P.splits * step + n;
    // lane s has split s's state
    const float2 x = lane < P.splits ? mlpart[row + lane * step] : make_float2(-1e30f, 0.f);
    float M = x.x;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o));
    const float f = __builtin_amdgcn_exp2f(x.x - M);
    float ls = x.y * f;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) ls += __shfl_xor(ls, o);
    v4f o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int s = 0; s < P.splits; s++) {
        const v4f v = *reinterpret_cast<const v4f*>(opart + (row + s * step) * HD + 4 * lane);
        const float fs = __shfl(f, s);
#pragma unroll
        for (int k = 0; k < 4; k++) o[k] = fmaf(v[k], fs, o[k]);
    }
    const size_t head = (size_t)vh * A.ratio + n / A.T;
    *reinterpret_cast<v4f*>(A.out + (head * A.TP + (size_t)b * A.T + i) * HD + 4 * lane) =
        live ? v4f{o[0] / ls, o[1] / ls, o[2] / ls, o[3] / ls} : v4f{0.f, 0.f, 0.f, 0.f};
}

}  // namespace

TreePlan tree_plan(int B, int T, int n_heads, int ratio, int kv_max, int kv_splits, int cus) {
    const int R = T * ratio;
    TreePlan p = {1, 1, 1};
    // rows per workgroup: 1400 cycles of unpacking a tile against about 2000 per block of 16 rows
    long best = 0;
    for (int nb = 1; nb <= kTreeMaxBlocks; nb++) {
        const int rg = (R + 16 * nb - 1) / (16 * nb);
        const long cost = (long)rg * (1400 + 2000 * nb);
        if (nb == 1 || cost < best) best = cost, p.blocks = nb, p.groups = rg;
    }
    const long units = (long)B * (n_heads / ratio) * p.groups;
    const long tiles = kv_max / BNK + 2;
    long s = kv_splits ? kv_splits : cus / units;
    if (!kv_splits && s > (tiles + 3) / 4) s = (tiles + 3) / 4;      // a tile for every wave
    p.splits = s < 1 ? 1 : s > kTreeMaxSplits ? kTreeMaxSplits : (int)s;
    return p;
}

size_t tree_part_bytes(const AttnTree& a, const TreePlan& p) {
    if (p.splits == 1) return 0;
    const size_t rows = (size_t)a.B * (a.n_heads / a.ratio) * p.splits * p.groups * 16 * p.blocks;
    return rows * (HD * sizeof(float) + sizeof(float2));
}

hipError_t launch_attn_tree(const AttnTree& a, const TreePlan& p, void* ws, hipStream_t st) {
    const int KVH = a.n_heads / a.ratio;
    const size_t units = (size_t)a.B * KVH * p.splits, rows = units * p.groups * 16 * p.blocks;
    float* opart = static_cast<float*>(ws);
    float2* mlpart = reinterpret_cast<float2*>(opart + rows * HD);
    const dim3 grid((unsigned)((units + 7) / 8 * 8 * p.groups));
    switch (p.blocks) {
        case 1: hipLaunchKernelGGL(attn_tree_k<1>, grid, dim3(256), 0, st, a, p, opart, mlpart); break;
        case 2: hipLaunchKernelGGL(attn_tree_k<2>, grid, dim3(256), 0, st, a, p, opart, mlpart); break;
        default: hipLaunchKernelGGL(attn_tree_k<3>, grid, dim3(256), 0, st, a, p, opart, mlpart); break;
    }
    if (p.splits > 1)
        hipLaunchKernelGGL(attn_tree_join_k, dim3((a.T * a.ratio + 3) / 4, a.B * KVH), dim3(256), 0, st, a, p, opart, mlpart);
    return hipGetLastError();
}

}  // namespace rt4
