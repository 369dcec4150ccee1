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

// e^x for -708 < x <= 0: 2^n e^r, n the integer nearest x log2(e) (its bits are the low ones of x log2(e)
// + 1.5 * 2^52), |r| <= ln(2) / 2, e^r by its Taylor sum to r^11 (the rest is below 7e-15).  Half the
// instructions of the library's exp, and no branch.
__device__ __forceinline__ double exp_small(double x) {
    constexpr double M = 6755399441055744.0;
    const double t = fma(x, 1.4426950408889634, M), n = t - M;
    double r = fma(n, -0.69314718055994529, x);
    r = fma(n, -2.3190468138462996e-17, r);
    double p = 1.0 / 39916800;
    p = fma(p, r, 1.0 / 3628800);
    p = fma(p, r, 1.0 / 362880);
    p = fma(p, r, 1.0 / 40320);
    p = fma(p, r, 1.0 / 5040);
    p = fma(p, r, 1.0 / 720);
    p = fma(p, r, 1.0 / 120);
    p = fma(p, r, 1.0 / 24);
    p = fma(p, r, 1.0 / 6);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return __hiloint2double(__double2hiint(p) + (int)((uint32_t)__double2loint(t) << 20), __double2loint(p));
}

// exp((l - m) * it), 1 at the maximum (also where that is +inf), 0 for -inf and NaN.
__device__ __forceinline__ double weight(float l, float m, double it) {
    const double x = ((double)l - (double)m) * it, e = exp_small(x);
    return l == m ? (m > -INFINITY ? 1.0 : 0.0) : x > -708.0 && l < m ? e : 0.0;
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
__device__ __forceinline__ RowStat row_of_chunks(const RowStat* ch, int C, double it) {
    const int lane = threadIdx.x & 63;
    RowStat r = {-INFINITY, INT_MAX, 0.0}, first = r;
    if (lane < C) first = ch[lane];                          // (held: most rows have at most 64 chunks)
    max_of(r.m, r.i, first.m, first.i);
    for (int c = lane + 64; c < C; c += 64) max_of(r.m, r.i, ch[c].m, ch[c].i);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) max_of(r.m, r.i, __shfl_xor(r.m, o), __shfl_xor(r.i, o));
    r.s = first.s * weight(first.m, r.m, it);
    for (int c = lane + 64; c < C; c += 64) r.s += ch[c].s * weight(ch[c].m, r.m, it);
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

struct Draw;
struct Verify {                          // the arguments of rt4_verify_tree and its workspace
    int *tokens, *path, *count, *kv_len;
    const float* logits;
    size_t ldl;
    const int *draft, *parent;
    const float *u, *temp, *q;
    size_t ldq;
    RowStat* ch;                         // [row][C] chunk statistics
    double *av, *part;                   // residual levels: a and chunk sums, [level][row], [level][row][C]
    Draw* draw;
    double* sums;                        // [B][C] residual mass of the last token's row
    int B, T, V, C, levels;
};

// Statistics of a chunk of a row: one read of the logits, held in registers between the maximum and
// the sum.  grid (C, B * T), 256 threads.  Rows of nodes that hang under nothing are not read.
template <bool ALIGNED>
__global__ __launch_bounds__(256) void verify_stats_k(const float* __restrict__ logits, size_t ldl, const int* __restrict__ parent,
                                                      const float* __restrict__ temp, int T, int V, RowStat* __restrict__ ch) {
    __shared__ float sm[4];
    __shared__ int si[4];
    __shared__ double ss[4];
    const int row = blockIdx.y, b = row / T, c = blockIdx.x, w = threadIdx.x >> 6;
    if (parent[(size_t)b * T] != -1 || (row % T && parent[row] < 0)) return;
    const float* l = logits + (size_t)row * ldl;
    // element e of thread i: 1024 (e / 4) + 4 i + e % 4
    float v[PT], m = -INFINITY;
    const int at = c * CH + 4 * (int)threadIdx.x;
    if (ALIGNED && (c + 1) * CH <= V) {
#pragma unroll
        for (int e = 0; e < PT; e += 4) {
            const float4 q = *reinterpret_cast<const float4*>(l + at + 256 * e);
            v[e] = q.x, v[e + 1] = q.y, v[e + 2] = q.z, v[e + 3] = q.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < PT; e++) {
            const int i = at + 256 * (e & ~3) + (e & 3);
            v[e] = i < V ? l[i] : -INFINITY;
        }
    }
    const double it = inv_temp(temp, b);
#pragma unroll
    for (int e = 0; e < PT; e++) m = fmaxf(m, v[e]);           // (drops NaN)
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if ((threadIdx.x & 63) == 0) sm[w] = m;
    __syncthreads();
    m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    int mi = INT_MAX;
    double s = 0;
#pragma unroll
    for (int e = PT - 1; e >= 0; e--) {
        if (v[e] == m && m > -INFINITY) mi = at + 256 * (e & ~3) + (e & 3);
        if (it > 0) s += weight(v[e], m, it);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const int x = __shfl_xor(mi, o);
        mi = x < mi ? x : mi;
    }
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) si[w] = mi, ss[w] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        const int i01 = si[0] < si[1] ? si[0] : si[1], i23 = si[2] < si[3] ? si[2] : si[3];
        ch[(size_t)row * gridDim.x + c] = RowStat{m, i01 < i23 ? i01 : i23, ss[0] + ss[1] + ss[2] + ss[3]};
    }
}

// Residual mass of level j (1 ..): chunk sums of max(p - a_j q, 0) for the rows with more
// than j children.  av [level][row]: a_j; part [level][row][C].  grid (C, B * T).
__global__ __launch_bounds__(256) void verify_mass_k(const float* __restrict__ logits, size_t ldl, const float* __restrict__ q,
                                                     size_t ldq, const int* __restrict__ parent, const float* __restrict__ temp,
                                                     int T, int V, int level, const RowStat* __restrict__ ch,
                                                     double* __restrict__ av, double* __restrict__ part) {
    __shared__ double ss[4];
    const int row = blockIdx.y, b = row / T, c = blockIdx.x, C = gridDim.x, R = gridDim.y;
    const Tree t = tree_of(parent, b, T);
    if (__popcll(__ballot(t.par == row % T)) <= level) return;
    const double it = inv_temp(temp, b);
    if (!(it > 0)) return;
    float l[PT], pq[PT];
#pragma unroll
    for (int e = 0; e < PT; e++) {
        const int i = c * CH + e * 256 + threadIdx.x;
        l[e] = i < V ? logits[(size_t)row * ldl + i] : -INFINITY;
        pq[e] = i < V ? q[(size_t)row * ldq + i] : 0.f;
    }
    double a = 1.0;
    if (level > 1) {
        const double* prev = part + ((size_t)(level - 1) * R + row) * C;
        double w = 0;
        for (int k = threadIdx.x & 63; k < C; k += 64) w += prev[k];
        a = av[(size_t)(level - 1) * R + row] + wave_sum(w);
    }
    const RowStat r = row_of_chunks(ch + (size_t)row * C, C, it);
    const double is = r.s > 0 ? 1.0 / r.s : 0.0;
    double s = 0;
#pragma unroll
    for (int e = 0; e < PT; e++) s += fmax(weight(l[e], r.m, it) * is - a * (double)pq[e], 0.0);
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
    int row, n, nrej, pad;               // row -1: nothing to draw; n accepted nodes; nrej tokens left out (no q)
    double a;                            // q: the residual is max(p - a q, 0)
    RowStat r;                           // of the row
    int rej[64];
};

// The path of sequence b, by one wave, lane i node i; rows: the statistics of its T rows.  Whether a
// node is accepted, once reached, depends on its parent's row and its earlier siblings alone, so all
// nodes are tested at once and the path is the set whose ancestors all passed.
__device__ void walk(const Verify& A, int b, double it, const RowStat* rows, bool write, Draw* d) {
    const int i = threadIdx.x & 63, T = A.T, V = A.V, R = A.B * T, C = A.C;
    const Tree t = tree_of(A.parent, b, T);
    const bool kid = t.anc && i > 0;
    const int tok = kid ? A.draft[(size_t)b * T + i] : -1;
    const bool real = tok >= 0 && tok < V;
    const int pn = kid ? t.par : 0;
    const size_t prow = (size_t)b * T + pn;
    const float lt = kid && real ? A.logits[prow * A.ldl + tok] : -INFINITY;
    const double qc = kid && real && A.q ? (double)A.q[prow * A.ldq + tok] : 0.0;
    const double ui = kid ? (double)A.u[(size_t)b * T + i] : 0.0;
    const RowStat r = rows[pn];
    const double pc = it > 0 && r.s > 0 ? weight(lt, r.m, it) / r.s : 0.0;
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
    if (A.q) {
        const int rank = __popcll(sib);
        tested = kid && rank < A.levels;
        for (int k = 1; k < A.levels; k++) {                 // (wave-uniform loops: part is summed by the whole wave)
            for (int n = 0; n < T; n++) {
                const size_t pr = (size_t)b * T + n;
                if (__popcll(__ballot(kid && t.par == n)) <= k || !(it > 0)) continue;
                double w = 0;
                for (int c = i; c < C; c += 64) w += A.part[((size_t)k * R + pr) * C + c];
                w = wave_sum(w);
                if (kid && t.par == n && rank == k) W = w, a = A.av[(size_t)k * R + pr];
            }
        }
    } else {
        for (int j = 1; j < T; j++) {
            const double pj = __shfl(pc, j);
            const bool fj = __shfl((int)first, j);
            if (fj && (sib >> j & 1)) W -= pj;
        }
    }
    bool yes = A.q ? ui * W * qc < pc - a * qc : first && ui * W < pc;
    if (!(it > 0)) yes = tok == r.i;
    yes = yes && tested && real;
    const u64 yesm = __ballot(yes);
    const u64 okm = __ballot(yes && !(sib & yesm));
    const bool on = t.anc && !(t.anc & ~okm & ~1ull);
    const u64 onm = __ballot(on);
    const int n = __popcll(onm), pos = __popcll(onm & ((1ull << i) - 1));
    const int last = n ? 63 - __clzll(onm) : 0;
    const bool rejected = kid && t.par == last && n;
    const u64 rejm = __ballot(rejected && (A.q ? tested : real && first));
    if (rejm >> i & 1) d->rej[__popcll(rejm & ((1ull << i) - 1))] = tok;
    // the residual's a after its children: a of the last one tested plus that one's W
    if (A.q && rejm && i == 63 - __clzll(rejm)) d->a = a + W;
    if (i == 0) {
        d->row = n ? b * T + last : -1;
        d->n = n;
        d->nrej = A.q ? 0 : __popcll(rejm);
        if (!A.q || !rejm) d->a = 0.0;
        d->r = rows[last];
    }
    if (!write) return;
    // -1 wherever no value belongs
    if (i < T) {
        if (i >= n) A.path[(size_t)b * T + i] = -1;
        if (i >= n) A.tokens[(size_t)b * T + i] = -1;          // (the last token comes after the draw)
    }
    if (on) A.path[(size_t)b * T + pos] = i;
    if (on && i > 0) A.tokens[(size_t)b * T + pos - 1] = tok;
    if (i == 0) {
        A.count[b] = n;
        if (A.kv_len) A.kv_len[b] += n;
    }
}

// Residual weights of thread's E consecutive tokens from `at` on; their sum.
template <int E>
__device__ __forceinline__ double residuals(double (&w)[E], const Verify& A, const Draw& d, double it, int at) {
    const float* l = A.logits + (size_t)d.row * A.ldl;
    const float* q = A.q ? A.q + (size_t)d.row * A.ldq : nullptr;
    const double is = d.r.s > 0 ? 1.0 / d.r.s : 0.0;
    double s = 0;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const int i = at + e;
        w[e] = 0.0;
        if (i < A.V) {
            w[e] = weight(l[i], d.r.m, it);
            if (q) w[e] = fmax(w[e] * is - d.a * (double)q[i], 0.0);
        }
    }
    for (int k = 0; k < d.nrej; k++) {
        const int i = d.rej[k] - at;
#pragma unroll
        for (int e = 0; e < E; e++)
            if (i == e) w[e] = 0.0;
    }
#pragma unroll
    for (int e = 0; e < E; e++) s += w[e];
    return s;
}

// Statistics of sequence b's rows into LDS, a wave per row.
__device__ __forceinline__ void rows_to_lds(const Verify& A, int b, double it, RowStat* rows) {
    for (int n = threadIdx.x >> 6; n < A.T; n += blockDim.x >> 6) {
        const RowStat r = row_of_chunks(A.ch + ((size_t)b * A.T + n) * A.C, A.C, it);
        if ((threadIdx.x & 63) == 0) rows[n] = r;
    }
    __syncthreads();
}

// With draft probabilities, the walk and the chunk sums of the residual: every workgroup of a
// sequence walks for itself (a launch less), the first one writes.  grid (C, B), 256 threads.
__global__ __launch_bounds__(256) void verify_residual_k(const Verify A) {
    __shared__ double ss[4];
    __shared__ RowStat rows[64];
    __shared__ Draw d;
    const int b = blockIdx.y, c = blockIdx.x;
    const double it = inv_temp(A.temp, b);
    rows_to_lds(A, b, it, rows);
    if (threadIdx.x < 64) walk(A, b, it, rows, c == 0, &d);
    __syncthreads();
    if (c == 0 && threadIdx.x < sizeof(Draw) / 4) reinterpret_cast<int*>(A.draw + b)[threadIdx.x] = reinterpret_cast<const int*>(&d)[threadIdx.x];
    if (d.row < 0 || !(it > 0)) return;
    double w[PT];
    double s = residuals(w, A, d, it, c * CH + (int)threadIdx.x * PT);
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) ss[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) A.sums[(size_t)b * A.C + c] = ss[0] + ss[1] + ss[2] + ss[3];
}

// The last token, after the walk where there are no draft probabilities.  grid B, 1024 threads.
//
// Without them a chunk's mass is the sum that verify_stats_k left, less the rejected tokens'.  Where
// hardly anything is left that difference says little, and the chunks are summed anew.
__global__ __launch_bounds__(1024) void verify_draw_k(const Verify A) {
    constexpr int E = CH / 1024;
    __shared__ RowStat rows[64];
    __shared__ Draw d;
    __shared__ double part[16], s_total, s_r;
    __shared__ int s_chunk, s_wave, s_tok;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const double it = inv_temp(A.temp, b);
    if (!A.q) {
        rows_to_lds(A, b, it, rows);
        if (tid < 64) walk(A, b, it, rows, true, &d);
    } else if (tid < (int)(sizeof(Draw) / 4)) {
        reinterpret_cast<int*>(&d)[tid] = reinterpret_cast<const int*>(A.draw + b)[tid];
    }
    __syncthreads();
    if (d.row < 0) return;
    int* out = A.tokens + (size_t)b * A.T + d.n - 1;
    const int best = d.r.i < A.V ? d.r.i : -1;
    if (!(it > 0) || best < 0) {                               // greedy, or a row with nothing in it
        if (tid == 0) *out = best;
        return;
    }
    const RowStat* ch = A.ch + (size_t)d.row * A.C;
    double* sums = A.sums + (size_t)b * A.C;
    if (w == 0) {
        if (tid == 0) s_chunk = -1, s_tok = best;              // (nothing left: the largest)
        double total = 0, all = 0;
        for (int c = lane; c < A.C; c += 64) {
            double s = sums[c];
            if (!A.q) {
                s = ch[c].s * weight(ch[c].m, d.r.m, it);
                all += s;
                for (int k = 0; k < d.nrej; k++)
                    if (d.rej[k] / CH == c) s -= weight(A.logits[(size_t)d.row * A.ldl + d.rej[k]], d.r.m, it);
                s = fmax(s, 0.0);
                sums[c] = s;
            }
            total += s;
        }
        total = wave_sum(total);
        all = wave_sum(all);
        if (tid == 0) s_total = !A.q && total < 1e-6 * all ? -1.0 : total;
    }
    __syncthreads();
    if (s_total < 0) {
        for (int c = 0; c < A.C; c++) {
            double x[E];
            const double s = wave_sum(residuals(x, A, d, it, c * CH + tid * E));
            if (lane == 0) part[w] = s;
            __syncthreads();
            if (tid == 0) {
                double t = 0;
                for (int k = 0; k < 16; k++) t += part[k];
                sums[c] = t;
            }
            __syncthreads();
        }
    }
    if (w == 0) {
        // the first chunk whose cumulated sum exceeds u times the total; lane order is chunk order
        double total = 0;
        for (int c = lane; c < A.C; c += 64) total += sums[c];
        total = wave_sum(total);
        const double want = (double)A.u[(size_t)b * A.T] * total;
        double acc = 0;
        int pick = -1, some = -1;
        double before = 0, sbefore = 0;
        for (int c0 = 0; c0 < A.C && pick < 0; c0 += 64) {
            const double s = c0 + lane < A.C ? sums[c0 + lane] : 0.0;
            double x = s;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const double y = __shfl_up(x, o);
                if (lane >= o) x += y;
            }
            const u64 hit = __ballot(acc + x > want && s > 0), any = __ballot(s > 0);
            if (any) {
                some = 63 - __clzll(any);
                sbefore = acc + __shfl(x - s, some);
                some += c0;
            }
            if (hit) {
                pick = __ffsll((unsigned long long)hit) - 1;
                before = acc + __shfl(x - s, pick);
                pick += c0;
            }
            acc += __shfl(x, 63);
        }
        if (pick < 0) pick = some, before = sbefore;           // (rounding left none: the last one with mass)
        if (lane == 0) {
            s_chunk = pick;
            s_r = want - before;
        }
    }
    __syncthreads();
    const int c = s_chunk;
    if (c >= 0) {
        double x[E];
        const double mine = residuals(x, A, d, it, c * CH + tid * E);
        double inc = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double y = __shfl_up(inc, o);
            if (lane >= o) inc += y;
        }
        if (lane == 63) part[w] = inc;
        if (tid == 0) s_wave = -1;
        __syncthreads();
        double base = 0;
        for (int k = 0; k < w; k++) base += part[k];
        const double r = s_r;
        // the wave, then the lane, then the token in which the sum first exceeds r; the last token with
        // weight where none does
        const u64 hit = __ballot(base + inc > r && mine > 0), any = __ballot(mine > 0);
        if (lane == 0 && hit) atomicMin(reinterpret_cast<unsigned*>(&s_wave), (unsigned)w);
        __syncthreads();
        int ws = s_wave;
        if (ws < 0) {                                          // none: the last wave with any
            __syncthreads();
            if (lane == 0 && any) atomicMax(&s_wave, w);
            __syncthreads();
            ws = s_wave;
        }
        if (w == ws) {
            const int ln = hit ? __ffsll((unsigned long long)hit) - 1 : 63 - __clzll(any);
            if (lane == ln) {
                double acc = base + inc - mine;
                int at = -1;
                for (int e = 0; e < E; e++) {
                    if (x[e] > 0) at = e;
                    acc += x[e];
                    if (acc > r && x[e] > 0) break;
                }
                s_tok = c * CH + tid * E + at;
            }
        }
        __syncthreads();
    }
    if (tid == 0) *out = s_tok;
}

size_t up16(size_t n) { return (n + 15) & ~size_t(15); }

}  // namespace

size_t verify_ws_bytes(int B, int T, int V, int levels) {
    const size_t R = (size_t)B * T, C = (V + CH - 1) / CH;
    return up16(R * C * sizeof(RowStat)) + up16(R * levels * 8) + up16(R * C * levels * 8) + up16(B * sizeof(Draw)) + up16(B * C * 8);
}

hipError_t launch_verify_tree(int* tokens, int* path, int* count, int* kv_len, const float* logits, size_t ldl, const int* draft,
                              const int* parent, const float* u, const float* temp, const float* q, size_t ldq, int B, int T, int V,
                              int levels, void* ws, hipStream_t st) {
    const int R = B * T, C = (V + CH - 1) / CH;
    unsigned char* p = static_cast<unsigned char*>(ws);
    auto take = [&](size_t n) { unsigned char* r = p; p += up16(n); return r; };
    RowStat* ch = reinterpret_cast<RowStat*>(take((size_t)R * C * sizeof(RowStat)));
    double* av = reinterpret_cast<double*>(take((size_t)R * levels * 8));
    double* part = reinterpret_cast<double*>(take((size_t)R * C * levels * 8));
    Draw* draw = reinterpret_cast<Draw*>(take((size_t)B * sizeof(Draw)));
    double* sums = reinterpret_cast<double*>(take((size_t)B * C * 8));
    const Verify a = {tokens, path, count, kv_len, logits, ldl, draft, parent, u, temp, q, ldq, ch, av, part, draw, sums, B, T, V, C, levels};
    if (((uintptr_t)logits & 15) == 0 && ldl % 4 == 0)
        hipLaunchKernelGGL(verify_stats_k<true>, dim3(C, R), dim3(256), 0, st, logits, ldl, parent, temp, T, V, ch);
    else
        hipLaunchKernelGGL(verify_stats_k<false>, dim3(C, R), dim3(256), 0, st, logits, ldl, parent, temp, T, V, ch);
    for (int k = 1; k < levels; k++)
        hipLaunchKernelGGL(verify_mass_k, dim3(C, R), dim3(256), 0, st, logits, ldl, q, ldq, parent, temp, T, V, k, ch, av, part);
    if (q) hipLaunchKernelGGL(verify_residual_k, dim3(C, B), dim3(256), 0, st, a);
    hipLaunchKernelGGL(verify_draw_k, dim3(B), dim3(1024), 0, st, a);
    return hipGetLastError();
}

}  // namespace rt4
