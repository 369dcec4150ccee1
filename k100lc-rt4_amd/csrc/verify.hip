// verify.hip -- which drafted tokens a target model's logits accept, and the token that
// follows them, gfx950 (rt4_verify_tree; no counterpart in the reference, which compares
// argmaxes on the host, src/model.cpp:1838-1926).
//
// p = softmax(l / temp) of a row.  At a node the children are tested in index order:
// after j rejections the token's distribution is r_j, and child c (token x, uniform u)
// is accepted iff u < r_j(x) / q(x), q the distribution it was proposed from.
//   - proposals chosen outright (no draft probabilities): q is 1 at x, so r_{j+1} is r_j
//     without x, renormalized: accept iff u W < p(x), W = 1 - sum of the rejected p.
//   - proposals drawn from q: r_{j+1} = max(r_j - q, 0) / its sum.  With r_j = max(p -
//     a_j q, 0) / W_j that is max(p - (a_j + W_j) q, 0) / W_{j+1}, so one number per
//     rejection describes the residual: a_0 = 0, W_0 = 1, a_{j+1} = a_j + W_j, W_j = sum
//     of max(p - a_j q, 0).
// The last token is the smallest x whose cumulated residual exceeds u_0 times its total.
//
// A drawn index has to be the definition's, so everything that decides it is held in 64
// bits: with V ~ 250k tokens of like weight a cumulated sum in 32 bits (2^-24) misplaces
// one draw in about twenty.
#include <climits>

#include "rt4_dev.h"
#include "rt4_internal.h"

namespace rt4 {
namespace {

constexpr int CH = kVerifyChunk;         // logits per workgroup: 256 threads x 16
constexpr int PT = CH / 256;

typedef unsigned long long u64;

struct RowStat {                         // of a chunk or of a row: largest logit, its lowest index, sum of exp((l - m) / temp)
    float m;
    int i;
    double s;
};

// exp((l - m) * it), 1 at the maximum (also where that is +inf), 0 for -inf and NaN.
__device__ __forceinline__ double weight(float l, float m, double it) {
    if (l == m) return m > -INFINITY ? 1.0 : 0.0;
    return l > -INFINITY && l < m ? exp(((double)l - (double)m) * it) : 0.0;
}

// (max, lowest index) of two.
__device__ __forceinline__ void max_of(float& m, int& i, float m2, int i2) {
    if (m2 > m || (m2 == m && i2 < i)) {
        m = m2;
        i = i2;
    }
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// The whole row's statistics from its chunks', by one wave, in a fixed order.
__device__ __forceinline__ RowStat row_of_chunks(const float* cm, const int* ci, const double* cs, int C, double it) {
    const int lane = threadIdx.x & 63;
    RowStat r = {-INFINITY, INT_MAX, 0.0};
    for (int c = lane; c < C; c += 64) max_of(r.m, r.i, cm[c], ci[c]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) max_of(r.m, r.i, __shfl_xor(r.m, o), __shfl_xor(r.i, o));
    for (int c = lane; c < C; c += 64) r.s += cs[c] * weight(cm[c], r.m, it);
    r.s = wave_sum(r.s);
    return r;
}

__device__ __forceinline__ double inv_temp(const float* temp, int b) {
    const float t = temp ? temp[b] : 1.f;
    return t > 0.f ? 1.0 / (double)t : 0.0;                  // 0: greedy
}

// A wave's view of sequence b's tree: lane i is node i.
struct Tree {
    int par;
    u64 anc;                             // the node and those above it; 0: not in the tree
};
__device__ __forceinline__ Tree tree_of(const int* parent, int b, int T) {
    const int i = threadIdx.x & 63;
    Tree t;
    t.par = i < T ? parent[(size_t)b * T + i] : -2;
    const bool root = i == 0 && t.par == -1, node = i > 0 && t.par >= 0 && t.par < i;
    int up = node ? t.par : i;
    u64 anc = 1ull << i;
#pragma unroll
    for (int s = 0; s < 6; s++) {        // pointer doubling: 2^6 covers the deepest chain
        anc |= __shfl(anc, up);
        up = __shfl(up, up);
    }
    const bool rooted = __shfl((int)root, 0);
    t.anc = (root || node) && rooted && (anc & 1) ? anc : 0;
    if (!t.anc) t.par = -2;
    return t;
}

// Statistics of a chunk of a row.  grid (C, B * T), 256 threads.
__global__ __launch_bounds__(256) void verify_stats_k(const float* __restrict__ logits, size_t ldl, const int* __restrict__ parent,
                                                      const float* __restrict__ temp, int T, int V, float* __restrict__ cm,
                                                      int* __restrict__ ci, double* __restrict__ cs) {
    __shared__ float sm[4];
    __shared__ int si[4];
    __shared__ double ss[4];
    const int row = blockIdx.y, b = row / T, c = blockIdx.x, C = gridDim.x, w = threadIdx.x >> 6;
    const double it = inv_temp(temp, b);
    const float* l = logits + (size_t)row * ldl;
    float v[PT], m = -INFINITY;
    int mi = INT_MAX;
#pragma unroll
    for (int e = 0; e < PT; e++) {
        const int i = c * CH + e * 256 + threadIdx.x;
        v[e] = i < V ? l[i] : -INFINITY;
        if (!(v[e] == v[e])) v[e] = -INFINITY;
        if (v[e] > m) m = v[e], mi = i;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) max_of(m, mi, __shfl_xor(m, o), __shfl_xor(mi, o));
    if ((threadIdx.x & 63) == 0) sm[w] = m, si[w] = mi;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; k++) max_of(m, mi, sm[k], si[k]);
    double s = 0;
    if (it > 0) {
#pragma unroll
        for (int e = 0; e < PT; e++) s += weight(v[e], m, it);
    }
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) ss[w] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        const size_t at = (size_t)row * C + c;
        cm[at] = m;
        ci[at] = mi;
        cs[at] = ss[0] + ss[1] + ss[2] + ss[3];
    }
}

// Statistics of the rows, from their chunks'.  grid B * T, 64 threads.
__global__ __launch_bounds__(64) void verify_rows_k(const float* __restrict__ cm, const int* __restrict__ ci,
                                                    const double* __restrict__ cs, const float* __restrict__ temp, int T, int C,
                                                    RowStat* __restrict__ rows) {
    const int row = blockIdx.x;
    const RowStat r = row_of_chunks(cm + (size_t)row * C, ci + (size_t)row * C, cs + (size_t)row * C, C, inv_temp(temp, row / T));
    if (threadIdx.x == 0) rows[row] = r;
}

// Residual mass of level j (1 ..): chunk sums of max(p - a_j q, 0) for the rows with more
// than j children.  aw [level][row]: a_j; part [level][row][C].  grid (C, B * T).
__global__ __launch_bounds__(256) void verify_mass_k(const float* __restrict__ logits, size_t ldl, const float* __restrict__ q,
                                                     size_t ldq, const int* __restrict__ parent, const float* __restrict__ temp,
                                                     int T, int V, int level, const RowStat* __restrict__ rows,
                                                     double* __restrict__ av, double* __restrict__ part) {
    __shared__ double ss[4];
    const int row = blockIdx.y, b = row / T, c = blockIdx.x, C = gridDim.x, R = gridDim.y;
    const Tree t = tree_of(parent, b, T);
    if (__popcll(__ballot(t.par == row % T)) <= level) return;
    const double it = inv_temp(temp, b);
    if (!(it > 0)) return;
    double a = 1.0;
    if (level > 1) {
        const double* prev = part + ((size_t)(level - 1) * R + row) * C;
        double w = 0;
        for (int k = threadIdx.x & 63; k < C; k += 64) w += prev[k];
        a = av[(size_t)(level - 1) * R + row] + wave_sum(w);
    }
    const RowStat r = rows[row];
    const double is = r.s > 0 ? 1.0 / r.s : 0.0;
    double s = 0;
#pragma unroll
    for (int e = 0; e < PT; e++) {
        const int i = c * CH + e * 256 + threadIdx.x;
        if (i < V)
            s += fmax(weight(logits[(size_t)row * ldl + i], r.m, it) * is - a * (double)q[(size_t)row * ldq + i], 0.0);
    }
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) ss[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        part[((size_t)level * R + row) * C + c] = ss[0] + ss[1] + ss[2] + ss[3];
        if (c == 0) av[(size_t)level * R + row] = a;
    }
}

// What the draw of a sequence's last token needs.
struct Draw {
    int row, nrej;                       // row -1: nothing to draw
    double a;
    int rej[64];
};

// The path of each sequence.  grid B, 64 threads: lane i is node i.  Whether a node is
// accepted, once reached, depends on its parent's row and its earlier siblings alone, so
// all nodes are tested at once and the path is the set whose ancestors all passed.
__global__ __launch_bounds__(64) void verify_walk_k(int* __restrict__ tokens, int* __restrict__ path, int* __restrict__ count,
                                                    int* __restrict__ kv_len, const float* __restrict__ logits, size_t ldl,
                                                    const int* __restrict__ draft, const int* __restrict__ parent,
                                                    const float* __restrict__ u, const float* __restrict__ temp,
                                                    const float* __restrict__ q, size_t ldq, int T, int V, int C, int levels,
                                                    const RowStat* __restrict__ rows, const double* __restrict__ av,
                                                    const double* __restrict__ part, Draw* __restrict__ draw) {
    const int b = blockIdx.x, i = threadIdx.x, R = gridDim.x * T;
    const double it = inv_temp(temp, b);
    const Tree t = tree_of(parent, b, T);
    const bool kid = t.anc && i > 0;
    const int tok = kid ? draft[(size_t)b * T + i] : -1;
    const bool real = tok >= 0 && tok < V;
    const size_t prow = (size_t)b * T + (kid ? t.par : 0);
    const RowStat r = rows[prow];
    double pc = 0, qc = 0;
    if (kid && real && it > 0 && r.s > 0) pc = weight(logits[prow * ldl + tok], r.m, it) / r.s;
    if (kid && real && q) qc = q[prow * ldq + tok];
    u64 sib = 0, same = 0;               // earlier siblings; those with this token
    for (int j = 1; j < T; j++) {
        const int pj = __shfl(t.par, j), tj = __shfl(tok, j);      // (by every lane)
        const bool s = pj == t.par && j < i && kid;
        sib |= (u64)s << j;
        same |= (u64)(s && tj == tok) << j;
    }
    const bool first = !same;
    double W = 1.0, a = 0.0;
    bool tested = kid;
    if (q) {
        const int rank = __popcll(sib);
        tested = kid && rank < levels;
        for (int k = 1; k < levels; k++) {                   // (wave-uniform loops: part is summed by the whole wave)
            for (int n = 0; n < T; n++) {
                const size_t pr = (size_t)b * T + n;
                if (__popcll(__ballot(kid && t.par == n)) <= k || !(it > 0)) continue;
                double w = 0;
                for (int c = i; c < C; c += 64) w += part[((size_t)k * R + pr) * C + c];
                w = wave_sum(w);
                if (kid && t.par == n && rank == k) W = w, a = av[(size_t)k * R + pr];
            }
        }
    } else {
        for (int j = 1; j < T; j++) {
            const double pj = __shfl(pc, j);
            const bool fj = __shfl((int)first, j);
            if (fj && (sib >> j & 1)) W -= pj;
        }
    }
    const double ui = kid ? (double)u[(size_t)b * T + i] : 0.0;
    bool yes = q ? ui * W * qc < pc - a * qc : first && ui * W < pc;
    if (!(it > 0)) yes = tok == r.i;
    yes = yes && tested && real;
    const u64 yesm = __ballot(yes);
    const u64 okm = __ballot(yes && !(sib & yesm));
    const bool on = t.anc && !(t.anc & ~okm & ~1ull);
    const u64 onm = __ballot(on);
    const int n = __popcll(onm), pos = __popcll(onm & ((1ull << i) - 1));
    const int last = n ? 63 - __clzll(onm) : 0;
    // outputs: -1 wherever no value belongs
    if (i < T) {
        if (i >= n) path[(size_t)b * T + i] = -1;
        if (i >= n - 1) tokens[(size_t)b * T + i] = -1;
    }
    if (on) path[(size_t)b * T + pos] = i;
    if (on && i > 0) tokens[(size_t)b * T + pos - 1] = tok;
    const bool rejected = kid && t.par == last && n;
    const u64 rejm = __ballot(rejected && (q ? tested : real && first));
    Draw* d = draw + b;
    if (rejm >> i & 1) d->rej[__popcll(rejm & ((1ull << i) - 1))] = tok;
    // the residual's a after its children: a of the last one tested plus that one's W
    if (q && rejm && i == 63 - __clzll(rejm)) d->a = a + W;
    if (i == 0) {
        count[b] = n;
        if (kv_len) kv_len[b] += n;
        d->row = n ? b * T + last : -1;
        d->nrej = q ? 0 : __popcll(rejm);
        if (q && !rejm) d->a = 0.0;
    }
}

// Residual weight of token i of the row a draw is from.
__device__ __forceinline__ double residual(const float* l, const float* q, const RowStat& r, double is, double it, double a, int i) {
    const double w = weight(l[i], r.m, it);
    return q ? fmax(w * is - a * (double)q[i], 0.0) : w;
}

// Weights of thread's 16 consecutive tokens of chunk c, and their sum.
__device__ __forceinline__ double chunk_weights(double (&w)[PT], const float* l, const float* q, const RowStat& r, double it,
                                                const Draw& d, int c, int V) {
    const double is = r.s > 0 ? 1.0 / r.s : 0.0;
    double s = 0;
#pragma unroll
    for (int e = 0; e < PT; e++) {
        const int i = c * CH + (int)threadIdx.x * PT + e;
        w[e] = i < V ? residual(l, q, r, is, it, d.a, i) : 0.0;
        for (int k = 0; k < d.nrej; k++)
            if (d.rej[k] == i) w[e] = 0.0;
        s += w[e];
    }
    return s;
}

// Chunk sums of the residual.  grid (C, B).
__global__ __launch_bounds__(256) void verify_residual_k(const float* __restrict__ logits, size_t ldl, const float* __restrict__ q,
                                                         size_t ldq, const float* __restrict__ temp, int V,
                                                         const RowStat* __restrict__ rows, const Draw* __restrict__ draw,
                                                         double* __restrict__ sums) {
    __shared__ double ss[4];
    const int b = blockIdx.y, c = blockIdx.x;
    const double it = inv_temp(temp, b);
    const Draw& d = draw[b];
    if (d.row < 0 || !(it > 0)) return;
    double w[PT];
    double s = chunk_weights(w, logits + d.row * ldl, q ? q + d.row * ldq : nullptr, rows[d.row], it, d, c, V);
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) ss[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) sums[(size_t)b * gridDim.x + c] = ss[0] + ss[1] + ss[2] + ss[3];
}

// The last token.  grid B, 256 threads.
__global__ __launch_bounds__(256) void verify_draw_k(int* __restrict__ tokens, const int* __restrict__ count,
                                                     const float* __restrict__ logits, size_t ldl, const float* __restrict__ u,
                                                     const float* __restrict__ temp, const float* __restrict__ q, size_t ldq, int T,
                                                     int V, int C, const RowStat* __restrict__ rows, const Draw* __restrict__ draw,
                                                     const double* __restrict__ sums) {
    __shared__ double part[256];
    __shared__ int s_chunk, s_tok;
    __shared__ double s_r;
    const int b = blockIdx.x, tid = threadIdx.x;
    const double it = inv_temp(temp, b);
    const Draw& d = draw[b];
    if (d.row < 0) return;
    const RowStat r = rows[d.row];
    if (tid == 0) {
        s_chunk = -1;
        s_tok = r.i < V ? r.i : -1;                          // greedy, or nothing left
        if (it > 0) {
            double total = 0, acc = 0;
            for (int c = 0; c < C; c++) total += sums[(size_t)b * C + c];
            const double want = (double)u[(size_t)b * T] * total;
            for (int c = 0; c < C; c++) {
                const double s = sums[(size_t)b * C + c];
                if (s > 0) {
                    s_chunk = c;                             // the last one with weight if rounding leaves none
                    s_r = want - acc;
                }
                acc += s;
                if (acc > want) break;
            }
        }
    }
    __syncthreads();
    const int c = s_chunk;
    if (c >= 0) {
        double w[PT];
        part[tid] = chunk_weights(w, logits + d.row * ldl, q ? q + d.row * ldq : nullptr, r, it, d, c, V);
        __syncthreads();
        if (tid == 0) {
            double acc = 0;
            int th = 0, with = 0;
            for (th = 0; th < 256; th++) {
                if (part[th] > 0) with = th;
                if (acc + part[th] > s_r) break;
                acc += part[th];
            }
            if (th == 256) {
                th = with;
                s_r = INFINITY;
            } else {
                s_r -= acc;
            }
            s_chunk = th;
        }
        __syncthreads();
        if (tid == s_chunk) {
            double acc = 0;
            int at = -1;
            for (int e = 0; e < PT; e++) {
                if (w[e] > 0) at = e;
                acc += w[e];
                if (acc > s_r) break;
            }
            s_tok = c * CH + tid * PT + at;
        }
        __syncthreads();
    }
    if (tid == 0) tokens[(size_t)b * T + count[b] - 1] = s_tok;
}

size_t up16(size_t n) { return (n + 15) & ~size_t(15); }

}  // namespace

size_t verify_ws_bytes(int B, int T, int V, int levels) {
    const size_t R = (size_t)B * T, C = (V + CH - 1) / CH;
    return up16(R * C * 4) * 2 + up16(R * C * 8) + up16(R * sizeof(RowStat)) + up16(R * levels * 8) + up16(R * C * levels * 8) +
           up16(B * sizeof(Draw)) + up16(B * C * 8);
}

hipError_t launch_verify_tree(int* tokens, int* path, int* count, int* kv_len, const float* logits, size_t ldl, const int* draft,
                              const int* parent, const float* u, const float* temp, const float* q, size_t ldq, int B, int T, int V,
                              int levels, void* ws, hipStream_t st) {
    const int R = B * T, C = (V + CH - 1) / CH;
    unsigned char* p = static_cast<unsigned char*>(ws);
    auto take = [&](size_t n) { unsigned char* r = p; p += up16(n); return r; };
    float* cm = reinterpret_cast<float*>(take((size_t)R * C * 4));
    int* ci = reinterpret_cast<int*>(take((size_t)R * C * 4));
    double* cs = reinterpret_cast<double*>(take((size_t)R * C * 8));
    RowStat* rows = reinterpret_cast<RowStat*>(take((size_t)R * sizeof(RowStat)));
    double* av = reinterpret_cast<double*>(take((size_t)R * levels * 8));
    double* part = reinterpret_cast<double*>(take((size_t)R * C * levels * 8));
    Draw* draw = reinterpret_cast<Draw*>(take((size_t)B * sizeof(Draw)));
    double* sums = reinterpret_cast<double*>(take((size_t)B * C * 8));
    hipLaunchKernelGGL(verify_stats_k, dim3(C, R), dim3(256), 0, st, logits, ldl, parent, temp, T, V, cm, ci, cs);
    hipLaunchKernelGGL(verify_rows_k, dim3(R), dim3(64), 0, st, cm, ci, cs, temp, T, C, rows);
    for (int k = 1; k < levels; k++)
        hipLaunchKernelGGL(verify_mass_k, dim3(C, R), dim3(256), 0, st, logits, ldl, q, ldq, parent, temp, T, V, k, rows, av, part);
    hipLaunchKernelGGL(verify_walk_k, dim3(B), dim3(64), 0, st, tokens, path, count, kv_len, logits, ldl, draft, parent, u, temp, q,
                       ldq, T, V, C, levels, rows, av, part, draw);
    hipLaunchKernelGGL(verify_residual_k, dim3(C, B), dim3(256), 0, st, logits, ldl, q, ldq, temp, V, rows, draw, sums);
    hipLaunchKernelGGL(verify_draw_k, dim3(B), dim3(256), 0, st, tokens, count, logits, ldl, u, temp, q, ldq, T, V, C, rows, draw,
                       sums);
    return hipGetLastError();
}

}  // namespace rt4
