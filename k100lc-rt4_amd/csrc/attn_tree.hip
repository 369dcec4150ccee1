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
// Scores are exact integers times two fp32 scales (the reference's decode attention has fp32
// scores, P and sums too; the prefill's int4 P would cost a relative 1e-2 per row when there are
// few keys).  P is two fp16 parts, high and low, so that P V runs on the fp16 matrix instructions with
// V's codes exact: off by at most 2^-22 of itself or 2^-38 of the row's largest so far; states and sums
// are fp32.
//
// What bounds it (24 query heads over 4 KV heads):
//   1 node over 1000 keys: 6.1 us and the join 3.8, the start of two launches; the loop is one step
//   4 nodes over 32701 keys: 16.6 and 3.9 us, 36.7 MB at 1.8 TB/s, four steps after 2.7 us of start
//   16 sequences of 8 nodes over up to 16384 keys: 55 to 62 us in all, 118 to 156 MB at 2.4 TB/s with 18 GFLOP beside it
//   61 nodes over 131001 keys: 279 to 285 us in all, 196 GFLOP at 0.7 PFLOP/s; P's two parts make them 294,
//   which take 222 us at the rates of large int8 and fp16 products, the softmax beside them
#include <algorithm>

#include "rt4_dev.h"
#include "rt4_internal.h"

namespace rt4 {
namespace {

constexpr int HD = 256, KDW = HD / 8, BNK = 64;
constexpr float L2E = 1.4426950408889634f;

typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

__device__ __forceinline__ int lane_id() { return threadIdx.x & 63; }

// Maxima by the instruction itself: fmaxf first quiets operands that it cannot see made (a third of
// the scores' maximum was that).
__device__ __forceinline__ float max2(float a, float b) {
    float r;
    asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
// Max over the four lanes that hold one query row's keys (lanes 16 and 32 apart).
__device__ __forceinline__ float max_groups(float v) {
    v = with_half<16>(v, max2);
    return with_half<32>(v, max2);
}

// 16 int8 operand bytes (16 x code) of two code dwords.
__device__ __forceinline__ v4i bytes16(uint32_t a, uint32_t b) {
    return v4i{(int)even_x16(a), (int)odd_x16(a), (int)even_x16(b), (int)odd_x16(b)};
}

// P is held times 2^kPBits, and the running maximum moves when a score exceeds it by 2^kLazy, so that P is
// at most 2^15 and fp16 holds it.  What is below 2^-(25 + kPBits) of the largest adds to the sum of P and
// not to P V: over the n keys of a run at most n 2^-38 of the largest |V|, where the fp32 sums over the
// n / 64 tiles may be off by n 2^-30.  (7 and 8: n 2^-32, 1e-4 of the output where one key is 22 nats above
// 32768 others and its value small.  The lower floor moves the maximum more often: 1.9% on average over 45
// sizes, 61 nodes over 131001 keys 282 -> 288 us.  The low part times 2^11, which needs no floor: 4.2%.)
constexpr float kPBits = 13.f, kLazy = 2.f, kPScale = 1.f / 8192;        // 2^-kPBits

// The eight codes of a V dword times 2^-kPBits as fp16, key pairs (0,4) (1,5) (2,6) (3,7): a nibble with its
// sign bit flipped is u = code + 8, and under the exponent of 1024 it reads 1024 + u (1024 + 16 u one nibble
// up), from which a packed fma makes the scaled code exactly (its 2^-17 is subnormal, and exact).  So the sums
// of P V are as large as the values that go into them, and overflow no sooner.
__device__ __forceinline__ v8h codes_f16(uint32_t w) {
    const uint32_t y = w >> 8;
    const uint32_t t[4] = {(w & 0x000F000Fu) ^ 0x64086408u, (w & 0x00F000F0u) ^ 0x64806480u, (y & 0x000F000Fu) ^ 0x64086408u,
                           (y & 0x00F000F0u) ^ 0x64806480u};
    union {
        v2h p[4];
        v8h v;
    } r;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const v2h a = __builtin_bit_cast(v2h, t[k]);
        const _Float16 m = (_Float16)(k & 1 ? kPScale / 16 : kPScale), c = (_Float16)(k & 1 ? -72 * kPScale : -1032 * kPScale);
        r.p[k] = a * v2h{m, m} + v2h{c, c};
    }
    return r.v;
}

// p + n elements in bytes, held in scalar registers (or the compiler loads the pointers from the
// kernel's arguments again at every use).
template <class T>
__device__ __forceinline__ const char* at(const T* p, size_t n) {
    const char* r = reinterpret_cast<const char*>(sptr(p + n));
    asm volatile("" : "+s"(r));
    return r;
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const char* p, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p), 0, bytes, 0x00020000);     // 32-bit data format
}

// How the key tiles of the sequences (the cache's, then the draft tile) are shared out, lengths being
// known here only.  A unit is a run of tiles of one sequence, for each KV head and row group a
// workgroup: `fixed` units a sequence, or runs of one length, the shortest by which there are at most
// `units` of them (at least B), no sequence has more than kTreeMaxSplits and none is shorter than a
// step.  So a batch's longest sequence takes no longer than its share.  An idle sequence has the draft
// tile alone, whatever its length.
struct Run {
    int b, split, splits, first, len, tiles;    // sequence, which of its units, their number, the first's, its cached keys and tiles
};
__device__ __forceinline__ int tiles_of_len(int len) { return (len + BNK - 1) / BNK + 1; }
// ceil(t / q) for t and q up to 2^19: the quotient of t + q - 1 + 1/2 is off by less than 2^-22 of
// itself, which is below the 1 / 2q that lies between it and the next integers.
__device__ __forceinline__ int ceil_div(int t, int q) {
    return (int)(((float)(t + q - 1) + 0.5f) * __builtin_amdgcn_rcpf((float)q));
}
// Unit x, b -1 past the last one.  By a whole wave; every lane gets it.
__device__ __forceinline__ Run run_of(const AttnTree& A, const TreePlan& P, int x) {
    const int lane = lane_id();
    auto len_of = [&](int b) __attribute__((always_inline)) {
        if (b >= A.B || !A.kv_len) return 0;
        const int len = A.kv_len[b];
        return A.parent[(size_t)b * A.T] != -1 || len < 0 ? 0 : len > A.kv_cap ? A.kv_cap : len;
    };
    auto tiles_of = [&](int b, int len) __attribute__((always_inline)) { return b < A.B ? tiles_of_len(len) : 0; };
    if (A.B == 1) {                                            // (the same without the reductions)
        const int len = uniform(len_of(0)), t = tiles_of_len(len), q = max(max(2, (t + P.units - 1) / P.units), (t + kTreeMaxSplits - 1) / kTreeMaxSplits);
        const int n = P.fixed ? min(P.fixed, t) : (t + q - 1) / q;
        return Run{x < n ? 0 : -1, x, n, 0, len, t};
    }
    const int held_len = len_of(lane), held = tiles_of(lane, held_len);
    int q = 0;
    if (!P.fixed) {
        int total = wave_sum(held), most = wave_max(held);
        for (int b0 = 64; b0 < A.B; b0 += 64) {
            const int t = tiles_of(b0 + lane, len_of(b0 + lane));
            total += wave_sum(t);
            most = max(most, wave_max(t));
        }
        // between an even share of all tiles and one that allows for a shorter run at every sequence's end
        // (that one where there are more sequences than lanes)
        q = max(max(2, (total + P.units - 1) / P.units), (most + kTreeMaxSplits - 1) / kTreeMaxSplits);
        int hi = P.units > A.B ? max(q, min(most, (total + P.units - A.B - 1) / (P.units - A.B))) : max(q, most);
        if (A.B > 64) q = hi;
        while (q < hi) {
            const int mid = (q + hi) / 2;
            if (wave_sum(ceil_div(held, mid)) <= P.units) hi = mid;
            else q = mid + 1;
        }
    }
    Run r = {-1, 0, 0, 0, 0, 0};
    int before = 0;
    for (int b0 = 0; b0 < A.B; b0 += 64) {
        const int len = b0 ? len_of(b0 + lane) : held_len, t = b0 ? tiles_of(b0 + lane, len) : held;
        const int n = P.fixed ? min(P.fixed, t) : ceil_div(t, q);
        const int end = before + wave_scan(n);
        const u64 hit = __ballot(x >= end - n && x < end);
        if (hit) {
            const int k = __ffsll((unsigned long long)hit) - 1;
            r.b = b0 + k;
            r.splits = __builtin_amdgcn_readlane(n, k);
            r.first = __builtin_amdgcn_readlane(end, k) - r.splits;
            r.split = x - r.first;
            r.len = __builtin_amdgcn_readlane(len, k);
            r.tiles = __builtin_amdgcn_readlane(t, k);
            return r;
        }
        before = __builtin_amdgcn_readlane(end, 63);
    }
    return r;
}

// n / T for a row n of a KV head's (T at most 64, n below 2^26).
__device__ __forceinline__ int by_nodes(int n, const AttnTree& A, const TreePlan& P) { return A.T == 1 ? n : (int)__umulhi((unsigned)n, P.inv_nodes); }

// Products x[4g + r] * y[c] of four 16x16 tiles in their accumulator layout on the matrix core
// (registers 4b + r: tile b, x from lane 16b + 4g + r, y from lane 16b + c), each rounded once.
__device__ __forceinline__ v16f outer16(float x_of_lane, float y) {
    const v16f z = {};
    return __builtin_amdgcn_mfma_f32_16x16x1f32(x_of_lane, y, z, 0, 0, 0);
}

// A workgroup owns 16 NB query rows of one (sequence, KV head) -- rows r * T + i, r the head in
// the group, i the node -- and a range of the keys' 64-key tiles, the draft tile last, two tiles a
// step.  Wave w makes S and P of its 32 keys of a step (each K dword is unpacked once), the P
// fragments go through LDS in operand order, and wave w multiplies them with its 64 dims of V (each
// V dword is unpacked once), so that no state has to be joined across waves but the row sums.  A
// step's P x V runs beside the next step's scores; two workgroups share a CU.
template <int NB>
__global__ __launch_bounds__(256, 2) void attn_tree_k(const AttnTree A, const TreePlan P, float* __restrict__ opart,
                                                      float2* __restrict__ mlpart, int2* __restrict__ runs) {
    constexpr int RW = 16 * NB;
    constexpr bool QL = NB > 2;                                // Q operands in LDS instead of registers
    __shared__ __align__(16) v8h pf[NB][4][2][64];             // P: [32 keys][high, low part][lane]
    __shared__ __align__(16) v4i qf[QL ? NB : 1][4][64];
    __shared__ float mx[4][RW];
    __shared__ u64 sees_l[RW];                                 // the draft keys a row sees (0: it is no node's)
    __shared__ size_t row_l[RW];                               // its row of qq and out
    const int tid = threadIdx.x, lane = lane_id(), w = uniform(tid >> 6), c = lane & 15, g = lane >> 4;
    // the row groups of one unit (sequence, KV head, split) on one XCD: workgroups go round the 8
    const int rg = (int)(blockIdx.x / 8) % P.groups;
    const int unit = (int)(blockIdx.x / (8 * P.groups)) * 8 + (int)(blockIdx.x % 8);
    const int KVH = A.n_heads / A.ratio, R = A.T * A.ratio;
    const Run run = run_of(A, P, unit / KVH);
    if (run.b < 0) return;
    const int b = uniform(run.b), vh = unit % KVH, len = uniform(run.len);
    const size_t seq = (size_t)b * KVH + vh;
    const int tiles = run.tiles, nt = tiles - 1;       // tile nt is the draft tile
    const int t0 = uniform(tiles * run.split / run.splits), t1 = uniform(tiles * (run.split + 1) / run.splits);     // (below 2^26)
    if (P.fixed != 1 && run.split == 0 && vh == 0 && rg == 0 && tid == 0) runs[b] = make_int2(run.first, run.splits);

    const int hS = w & 1;                                      // half of the tile whose scores this wave makes
    v4u K[2][2], V[4];
    v4f vs[2];
    float ks[2];
    // Buffer loads: a per-lane offset that stays for the whole loop and a scalar offset per tile (a KV
    // head's cache is below 2^31 bytes), from the cache or the draft tile.
    // K: operand row 4g + i of subtile p is key 8g + 4p + i, so a lane's scores are the eight keys of one
    // V dword; lane 16 b + j supplies the scales of group b / 2, row j.  V: dim tile j, column c is dim
    // 64w + 4c + j.
    const char *kc = at(A.kc, seq * A.kv_cap * KDW), *kd = at(A.kd, seq * BNK * KDW);
    const char *ksc = at(A.ksc, seq * 2 * A.kv_cap), *ksd = at(A.ksd, seq * 2 * BNK);
    const char *vc = at(A.vc, seq * (A.kv_cap / 8) * HD), *vd = at(A.vd, seq * (BNK / 8) * HD);
    const char *vsc = at(A.vsc, seq * (A.kv_cap / BNK) * HD), *vsd = at(A.vsd, seq * HD);
    const int ko = ((8 * (c >> 2) + (c & 3)) * KDW + 4 * g) * 4 + 32 * hS * KDW * 4;
    const int so = (8 * (c >> 2) + (c & 3) + 32 * hS) * 4;
    const int vo = (g * HD + 4 * c + 64 * w) * 4, wo = (4 * c + 64 * w) * 4;
    auto load_k = [&](int tp) __attribute__((always_inline)) {
        int t = tp + (w >> 1);
        t = t < t1 ? t : t1 - 1;
        const bool d = t == nt;
        const int cap = d ? BNK : A.kv_cap;
        const auto rk = rsrc(d ? kd : kc, cap * KDW * 4), rs = rsrc(d ? ksd : ksc, 2 * cap * 4);
        const int k0 = d ? 0 : t * BNK;
#pragma unroll
        for (int p = 0; p < 2; p++) {
#pragma unroll
            for (int G = 0; G < 2; G++)
                K[p][G] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rk, ko + (4 * p * KDW + 16 * G) * 4, k0 * (KDW * 4), 0));
            ks[p] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rs, so + 16 * p + (g >> 1) * cap * 4, k0 * 4, 0));
        }
    };
    auto load_v = [&](int tp, int x) __attribute__((always_inline)) {
        int t = tp + x;
        t = t < t1 ? t : t1 - 1;                               // (past the range: P is zero)
        const bool d = t == nt;
        const auto rv = rsrc(d ? vd : vc, (d ? BNK : A.kv_cap) / 8 * HD * 4);
        const int t8 = d ? 0 : t * (BNK / 8 * HD * 4);
        V[2 * x] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rv, vo, t8, 0));
        V[2 * x + 1] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rv, vo, t8 + 4 * HD * 4, 0));
    };
    auto load_vs = [&](int tp, int x) __attribute__((always_inline)) {
        int t = tp + x;
        t = t < t1 ? t : t1 - 1;
        const bool d = t == nt;
        const auto rs = rsrc(d ? vsd : vsc, (d ? 1 : A.kv_cap / BNK) * HD * 4);
        vs[x] = __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(rs, wo, d ? 0 : t * (HD * 4), 0));
    };
    // Loads in the order in which they are needed, since they come back in that order: the tree, K, Q, V
    const int par = lane < A.T ? A.parent[(size_t)b * A.T + lane] : -2;
    if (t0 < t1) load_k(t0);
    // Q operands (column c of block nb is row n) and this lane's column scales: lane 16 b + c has those
    // of group b / 2, block 2 pr + b % 2
    auto row_of = [&](int n) __attribute__((always_inline)) {      // of qq and out
        n = n < R ? n : 0;
        const int head = by_nodes(n, A, P);
        return ((size_t)vh * A.ratio + head) * A.TP + (size_t)b * A.T + (n - head * A.T);
    };
    v4u qd[QL ? 1 : NB][2];
    float qs[(NB + 1) / 2], m[NB], l[NB];
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
        m[nb] = 0.f;
        l[nb] = 0.f;
        if (QL && nb != w) continue;
        const uint32_t* qr = A.qq + row_of(rg * RW + nb * 16 + c) * KDW + 4 * g;
#pragma unroll
        for (int k = 0; k < 2; k++) qd[QL ? 0 : nb][k] = *reinterpret_cast<const v4u*>(qr + 16 * k);
    }
#pragma unroll
    for (int pr = 0; pr < (NB + 1) / 2; pr++) {
        const int nb = 2 * pr + (g & 1), n = rg * RW + (nb < NB ? nb : 0) * 16 + c;
        const size_t head = (size_t)vh * A.ratio + by_nodes(n < R ? n : 0, A, P);
        qs[pr] = A.qsc[row_of(n) + (head + (g >> 1)) * A.TP];
    }
    if (t0 < t1) {
#pragma unroll
        for (int x = 0; x < 2; x++) {
            load_v(t0, x);
            load_vs(t0, x);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    {
        const u64 sees = tree_sees(par, A.T);
        const int n = rg * RW + tid, in = n < R ? n : 0;
        const u64 x = __shfl(sees, in - by_nodes(in, A, P) * A.T);
        if (tid < RW) {
            sees_l[tid] = n < R ? x : 0;
            row_l[tid] = row_of(n);
        }
    }
    v4i qop[QL ? 1 : NB][4];
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
        if (QL && nb != w) continue;
        const v4u (&d)[2] = qd[QL ? 0 : nb];
        v4i (&q)[4] = qop[QL ? 0 : nb];
        q[0] = bytes16(d[0].x, d[0].y);
        q[1] = bytes16(d[0].z, d[0].w);
        q[2] = bytes16(d[1].x, d[1].y);
        q[3] = bytes16(d[1].z, d[1].w);
        if (QL)
#pragma unroll
            for (int k = 0; k < 4; k++) qf[nb][k][lane] = q[k];
    }
#pragma unroll
    for (int pr = 0; pr < (NB + 1) / 2; pr++) qs[pr] *= L2E / 256.f;     // (both operands are 16 x code)
    __syncthreads();

    v4f O[NB][4];
#pragma unroll
    for (int nb = 0; nb < NB; nb++)
#pragma unroll
        for (int j = 0; j < 4; j++) O[nb][j] = v4f{0.f, 0.f, 0.f, 0.f};

    float s[NB][8];
    // S^T = K Q^T less the reference: lane (c, g) gets row c, keys 8g + 4p + i; publishes the rows' maxima
    auto scores = [&](int tp) __attribute__((always_inline)) {
        const int t = tp + (w >> 1);
#pragma unroll
        for (int p = 0; p < 2; p++) {
            const v4i a0 = bytes16(K[p][0].x, K[p][0].y), a1 = bytes16(K[p][0].z, K[p][0].w);
            const v4i a2 = bytes16(K[p][1].x, K[p][1].y), a3 = bytes16(K[p][1].z, K[p][1].w);
            v16f sc;
            v4i qn[4];                                         // the next block's operands, read while this one's are in use
            auto read_q = [&](int nb) __attribute__((always_inline)) {
#pragma unroll
                for (int k = 0; k < 4; k++) qn[k] = QL ? qf[nb][k][lane] : qop[QL ? 0 : nb][k];
            };
            read_q(0);
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
                const v4i q0 = qn[0], q1 = qn[1], q2 = qn[2], q3 = qn[3];
                if (nb + 1 < NB) read_q(nb + 1);
                if (NB > 2) __builtin_amdgcn_sched_barrier(0); // (or the compiler holds all blocks' operands at once and spills)
                if (nb % 2 == 0) sc = outer16(ks[p], qs[nb / 2]);
                const v4i z = {0, 0, 0, 0};
                v4i x = __builtin_amdgcn_mfma_i32_16x16x64_i8(a0, q0, z, 0, 0, 0);
                v4i y = __builtin_amdgcn_mfma_i32_16x16x64_i8(a2, q2, z, 0, 0, 0);
                x = __builtin_amdgcn_mfma_i32_16x16x64_i8(a1, q1, x, 0, 0, 0);
                y = __builtin_amdgcn_mfma_i32_16x16x64_i8(a3, q3, y, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float v = fmaf((float)x[i], sc[4 * (nb % 2) + i], fmaf((float)y[i], sc[8 + 4 * (nb % 2) + i], kPBits - m[nb]));
                    asm volatile("" : "+v"(v));                // (computed here: sunk below the mask's branch, its operands of all
                    s[nb][4 * p + i] = v;                      // blocks stay live and spill)
                }
            }
        }
        load_k(tp + 2);
        if (t >= nt || (t + 1) * BNK > len || t >= t1) {       // keys that some row may not see
            const u64 tail = t < nt && t < t1 ? (1ull << (len - t * BNK)) - 1 : 0;
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
                u64 ok = t == nt && t < t1 ? sees_l[nb * 16 + c] : tail;
                ok >>= 32 * hS + 8 * g;
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (!(ok >> e & 1)) s[nb][e] = -INFINITY;
            }
        }
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            float mt = max3(max3(s[nb][0], s[nb][1], s[nb][2]), s[nb][3], s[nb][4]);
            mt = max_groups(max3(max2(mt, s[nb][5]), s[nb][6], s[nb][7]));
            if (g == 0) mx[w][nb * 16 + c] = mt;
        }
    };
    // Moves the references (all waves alike) where a score exceeds them by much, at first in any case
    auto move = [&](bool first) __attribute__((always_inline)) {
        float mt[NB];
        bool any = first;
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            const int r = nb * 16 + c;
            mt[nb] = max3(max2(mx[0][r], mx[1][r]), mx[2][r], mx[3][r]) - kPBits;
            any |= mt[nb] > kLazy;
        }
        if (__builtin_expect(!__any(any), 1)) return;
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            // (a row that sees nothing yet keeps its reference: -inf would not come back)
            if (NB > 2) __builtin_amdgcn_sched_barrier(0);
            const float up = first ? (mt[nb] > -INFINITY ? mt[nb] : 0.f) : fmaxf(mt[nb], 0.f);
            m[nb] += up;
#pragma unroll
            for (int e = 0; e < 8; e++) s[nb][e] -= up;
            if (first) continue;
            const float alpha = __builtin_amdgcn_exp2f(-up);
            l[nb] *= alpha;
            float ar[4];
#pragma unroll
            for (int i = 0; i < 4; i++) ar[i] = __shfl(alpha, 4 * g + i);
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) O[nb][j][i] *= ar[i];
        }
    };
    // P, and its fragments into LDS
    auto weights = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            if (NB > 2) __builtin_amdgcn_sched_barrier(0);
            v8h ph, pl;
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const v2f p = {__builtin_amdgcn_exp2f(s[nb][i]), __builtin_amdgcn_exp2f(s[nb][4 + i])};
                sum += p[0] + p[1];
                const v2h hi = __builtin_convertvector(p, v2h);
                const uint32_t hb = __builtin_bit_cast(uint32_t, hi);
                v2f r;                                         // p - hi, the conversion back within the instruction
                asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r[0]) : "v"(hb), "v"(p[0]));
                asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r[1]) : "v"(hb), "v"(p[1]));
                const v2h lo = __builtin_convertvector(r, v2h);
                ph[2 * i] = hi[0];
                ph[2 * i + 1] = hi[1];
                pl[2 * i] = lo[0];
                pl[2 * i + 1] = lo[1];
            }
            l[nb] += sum;
            pf[nb][w][0][lane] = ph;
            pf[nb][w][1][lane] = pl;
        }
    };
    // O += P V: rows 4g + i, dims 64w + 4c + j
    auto product = [&](int tn) __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < 2; x++) {
            v8h v[2][4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                v[0][j] = codes_f16(V[2 * x][j]);
                v[1][j] = codes_f16(V[2 * x + 1][j]);
            }
            __builtin_amdgcn_sched_barrier(0);
            load_v(tn, x);
            v8h pn[4];                                         // likewise
            auto read_p = [&](int nb) __attribute__((always_inline)) {
#pragma unroll
                for (int k = 0; k < 4; k++) pn[k] = pf[nb][2 * x + k / 2][k % 2][lane];
            };
            read_p(0);
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
                const v8h p0 = pn[0], p1 = pn[1], p2 = pn[2], p3 = pn[3];
                if (nb + 1 < NB) read_p(nb + 1);
                if (NB > 2) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    v4f a = {0.f, 0.f, 0.f, 0.f};
                    a = __builtin_amdgcn_mfma_f32_16x16x32_f16(p0, v[0][j], a, 0, 0, 0);
                    a = __builtin_amdgcn_mfma_f32_16x16x32_f16(p1, v[0][j], a, 0, 0, 0);
                    a = __builtin_amdgcn_mfma_f32_16x16x32_f16(p2, v[1][j], a, 0, 0, 0);
                    a = __builtin_amdgcn_mfma_f32_16x16x32_f16(p3, v[1][j], a, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        float o = fmaf(a[i], vs[x][j], O[nb][j][i]);
                        if (x) asm volatile("" : "+v"(o));     // (nor are these, below the branch of the references)
                        O[nb][j][i] = o;
                    }
                }
            }
            load_vs(tn, x);
        }
    };

    if (t0 < t1) {
        scores(t0);
        __syncthreads();
        move(true);
        weights();
        __syncthreads();
        for (int tp = t0 + 2; tp < t1; tp += 2) {
            product(tp);
            __builtin_amdgcn_sched_barrier(0);
            scores(tp);
            __syncthreads();                                   // the fragments are read, the maxima are there
            move(false);
            weights();
            __syncthreads();
        }
        product(t1);
    }

    // row sums of the four waves; every wave holds the same references
    __syncthreads();
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
        float t = l[nb] + __shfl_xor(l[nb], 16);
        t += __shfl_xor(t, 32);
        if (g == 0) mx[w][nb * 16 + c] = t * kPScale;
    }
    __syncthreads();
    const size_t prow = ((size_t)unit * P.groups + rg) * RW;
    if (P.fixed != 1) {                                        // attn_tree_join_k sums the splits
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (rg * RW + nb * 16 + 4 * g + i >= R) continue;
                v4f* to = reinterpret_cast<v4f*>(opart + (prow + nb * 16 + 4 * g + i) * HD + 64 * w + 4 * c);
                const v4f o = {O[nb][0][i], O[nb][1][i], O[nb][2][i], O[nb][3][i]};
                if (P.stream) {
                    asm volatile("" ::: "memory");             // (or both stores become one, a plain one)
                    __builtin_nontemporal_store(o, to);
                    asm volatile("" ::: "memory");
                } else {
                    *to = o;
                }
            }
            if (w == 0 && g == 0) {
                const int r = nb * 16 + c;
                mlpart[prow + r] = make_float2(m[nb], mx[0][r] + mx[1][r] + mx[2][r] + mx[3][r]);
            }
        }
        return;
    }
#pragma unroll
    for (int nb = 0; nb < NB; nb++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = nb * 16 + 4 * g + i;
            if (rg * RW + r >= R) continue;
            const float ls = mx[0][r] + mx[1][r] + mx[2][r] + mx[3][r];
            *reinterpret_cast<v4f*>(A.out + row_l[r] * HD + 64 * w + 4 * c) =
                sees_l[r] ? v4f{O[nb][0][i] / ls, O[nb][1][i] / ls, O[nb][2][i] / ls, O[nb][3][i] / ls} : v4f{0.f, 0.f, 0.f, 0.f};
        }
}

// Sums the splits' states, W waves per row (all of a wave's loads in flight at once), four dims a lane:
// four waves where a row has many splits, else one, which needs no exchange through LDS.
template <int W>
__global__ __launch_bounds__(256) void attn_tree_join_k(const AttnTree A, const TreePlan P, const float* __restrict__ opart,
                                                        const float2* __restrict__ mlpart, const int2* __restrict__ runs) {
    __shared__ __align__(16) v4f ol[W == 1 ? 1 : 4][64];
    const int KVH = A.n_heads / A.ratio, lane = lane_id(), w = uniform(threadIdx.x >> 6);
    const int n = W == 1 ? 4 * blockIdx.x + w : blockIdx.x, s0 = W == 1 ? 0 : w;
    const int seq = blockIdx.y, b = seq / KVH, vh = seq % KVH, in_head = by_nodes(n, A, P), i = n - in_head * A.T;
    if (n >= A.T * A.ratio) return;
    const int2 run = runs[b];                                  // the sequence's first unit and their number
    const size_t step = (size_t)KVH * P.groups * 16 * P.blocks, row = (size_t)run.x * step + (size_t)vh * P.groups * 16 * P.blocks + n;
    const int splits = uniform(run.y), par = lane < A.T ? A.parent[(size_t)b * A.T + lane] : -2;
    // lane s has the states of splits s and s + 64
    float2 x[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
        x[k] = mlpart[row + min(lane + 64 * k, splits - 1) * step];
        if (lane + 64 * k >= splits) x[k] = make_float2(-INFINITY, 0.f);
    }
    const float* src = opart + row * HD + 4 * lane;
    v4f v[16];
    auto read = [&](int h) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < 16; k++) {
            const int s = s0 + W * (16 * h + k);               // (past the last split: that one, times 0;
            v[k] = *reinterpret_cast<const v4f*>(src + min(s, splits - 1) * step * HD);   // under a condition each load waits)
        }
    };
    read(0);
    __builtin_amdgcn_sched_barrier(0);
    const bool live = __shfl(tree_sees(par, A.T), i) != 0;
    const float M = wave_max(fmaxf(x[0].x, x[1].x));
    const float f[2] = {__builtin_amdgcn_exp2f(x[0].x - M), __builtin_amdgcn_exp2f(x[1].x - M)};
    const float ls = wave_sum(x[0].y * f[0] + x[1].y * f[1]);
    v4f o = {0.f, 0.f, 0.f, 0.f};
    for (int h = 0; s0 + W * 16 * h < splits; h++) {
        if (h) read(h);
#pragma unroll
        for (int k = 0; k < 16; k++) {
            const int s = s0 + W * (16 * h + k);
            const float fs = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, s < 64 ? f[0] : f[1]), s & 63));
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = fmaf(v[k][e], fs, o[e]);
        }
    }
    if constexpr (W > 1) {
        ol[w][lane] = o;
        __syncthreads();
        if (w) return;
#pragma unroll
        for (int k = 1; k < 4; k++) o += ol[k][lane];
    }
    const size_t head = (size_t)vh * A.ratio + in_head;
    *reinterpret_cast<v4f*>(A.out + (head * A.TP + (size_t)b * A.T + i) * HD + 4 * lane) =
        live ? v4f{o[0] / ls, o[1] / ls, o[2] / ls, o[3] / ls} : v4f{0.f, 0.f, 0.f, 0.f};
}

}  // namespace

// The rows per workgroup and the units by a model of the time in us: a step of two tiles takes 1.3, 2.2
// or 3.0 (1 to 3 blocks) with one workgroup on a CU and 1.6, 2.5 or 3.3 with two, the joining launch 4
// and its states (1 KB a row and unit, written and read) 0.35 a MB, all sequences as long as the longest.
// A unit's row groups stay on one XCD (an eighth of the CUs), so the XCD with the most units decides; where
// they are more workgroups than it takes at once, every XCD still has a unit, in whole rounds (64 nodes of
// 64 heads over 1 KV head and 65536 keys 388 us; all on one XCD 3308, rounds counted in parts 433).
// Over 241 sweeps of blocks and units, 1 to 16 sequences of 500 to 131000 keys and 1 to 64 nodes, the
// choice by these figures takes 0.8% longer than the best on average and 12% at most where lengths are
// alike (1.5% and 29% where they are drawn between 0 and the longest).
// (4 to 6 blocks fit too: 276 to 283 us where 3 take 283, 64 nodes over 131001 keys, and 43 against 37,
// 16 nodes over 32000.  A join in the same launch by the last workgroup of a row group took 14 us where
// both launches take 10, one node over 1000 keys; 1024 threads a workgroup, four teams on a quarter of
// the keys each that join in LDS, 16 at 500 keys where both launches take 11.)
TreePlan tree_plan(int B, int T, int n_heads, int ratio, int kv_max, int kv_splits, int cus) {
    constexpr double one[] = {1.3, 2.2, 3.0}, two[] = {1.6, 2.5, 3.3};
    const int R = T * ratio;
    const long KVH = n_heads / ratio, tiles = (kv_max + BNK - 1) / BNK + 1, xcd = cus > 8 ? cus / 8 : 1;
    TreePlan p = {1, 1, 0, 0};
    double best = 0;
    for (int nb = 1; nb <= kTreeMaxBlocks; nb++) {
        const int rg = (R + 16 * nb - 1) / (16 * nb);
        if (nb > 1 && rg == (R + 16 * nb - 17) / (16 * nb - 16)) continue;      // no fewer groups than with fewer blocks
        for (int k = 0; k < 5; k++) {                          // a unit a sequence, or k / 2 workgroups a CU
            if (kv_splits && k != (kv_splits > 1)) continue;
            // (one a XCD at least, where its row groups are more workgroups than the XCD takes at once)
            long units = kv_splits ? (long)B * kv_splits : k ? std::max(1l, k * xcd / 2 / rg) * 8 / KVH : B;
            const long most = std::min((tiles + 1) / 2, (long)kTreeMaxSplits) * B;     // (run_of has no more)
            units = units < B ? B : kv_splits || units < most ? units : most;
            const long each = units / B, wgs = (units * KVH + 7) / 8 * rg, steps = ((tiles + each - 1) / each + 1) / 2;
            const double rounds = fmax(1.0, wgs / (2.0 * xcd));
            const double run = steps * (wgs <= xcd ? one[nb - 1] : two[nb - 1] * (k && !kv_splits ? ceil(rounds) : rounds));
            const double cost = run + (k == 0 ? 0 : 4 + 0.35e-3 * KVH * R * units);
            if (best == 0 || cost < best) best = cost, p = TreePlan{nb, rg, (int)units, kv_splits ? kv_splits : k == 0};
        }
    }
    p.inv_nodes = (unsigned)(((1ull << 32) + T - 1) / T);
    // States of more than 6 MB are written past the L2, which would write them back at the end of the
    // launch (4 ragged sequences of 16 nodes, 25 MB: 28.6 -> 26.8 us; 4 of 8 nodes over 2000 keys, 8 MB:
    // 18.9 -> 18.1), fewer through it (1.5 MB: 11.4 us, past it 12.1; 6 MB: 18.4, 19.2), and so where
    // the caches are over 120 MB, which leaves them no place behind it (61 nodes over 131001 keys, 147
    // MB: 282 us, past it 284; 16 sequences of 16 nodes over 8000, 143 MB: 101, 107).
    p.stream = p.units * KVH * R > 6144 && KVH * B * (long)kv_max * (HD + 24) < 120000000;
    return p;
}

// Units that a launch may have.
static size_t max_units(const AttnTree& a, const TreePlan& p) { return p.fixed ? (size_t)a.B * p.fixed : (size_t)p.units; }

size_t tree_part_bytes(const AttnTree& a, const TreePlan& p) {
    if (p.fixed == 1) return 0;
    const size_t rows = max_units(a, p) * (a.n_heads / a.ratio) * p.groups * 16 * p.blocks;
    return rows * (HD * sizeof(float) + sizeof(float2)) + a.B * sizeof(int2);
}

hipError_t launch_attn_tree(const AttnTree& a, const TreePlan& p, void* ws, hipStream_t st) {
    const int KVH = a.n_heads / a.ratio;
    const size_t units = max_units(a, p) * KVH, rows = units * p.groups * 16 * p.blocks;
    float* opart = static_cast<float*>(ws);
    float2* mlpart = reinterpret_cast<float2*>(opart + rows * HD);
    int2* runs = reinterpret_cast<int2*>(mlpart + rows);
    const dim3 grid((unsigned)((units + 7) / 8 * 8 * p.groups));
    switch (p.blocks) {
        case 1: hipLaunchKernelGGL(attn_tree_k<1>, grid, dim3(256), 0, st, a, p, opart, mlpart, runs); break;
        case 2: hipLaunchKernelGGL(attn_tree_k<2>, grid, dim3(256), 0, st, a, p, opart, mlpart, runs); break;
        default: hipLaunchKernelGGL(attn_tree_k<3>, grid, dim3(256), 0, st, a, p, opart, mlpart, runs); break;
    }
    if (p.fixed != 1) {
        const int R = a.T * a.ratio;
        if ((p.fixed ? p.fixed : p.units / a.B) > 16)
            hipLaunchKernelGGL(attn_tree_join_k<4>, dim3(R, a.B * KVH), dim3(256), 0, st, a, p, opart, mlpart, runs);
        else
            hipLaunchKernelGGL(attn_tree_join_k<1>, dim3((R + 3) / 4, a.B * KVH), dim3(256), 0, st, a, p, opart, mlpart, runs);
    }
    return hipGetLastError();
}

}  // namespace rt4
