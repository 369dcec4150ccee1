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
//
// What bounds it: where the logits are many their read and the arithmetic on them, which take the same
// time and do not overlap wholly (8 chains of 16 nodes, V = 248320, every row read: verify_stats_k 33.8 us,
// 127 MB at 3.8 TB/s, which a copy reads in 25.7, and vector instructions in 69% of the SIMDs' cycles, 30 a
// logit; trees with an idle sequence and padding among them, 85 to 92 MB: 22.3 us; then 7.5 to 8 for walk and
// draw), else a chain of short launches, each the start of one and two or three trips to memory (4 rows of
// 248320 with draft probabilities 4.2 + 9.8 us; with siblings 5.3 more for each), or one launch
// (verify_small_k).
#include <climits>

#include "rt4_dev.h"
#include "rt4_internal.h"

namespace rt4 {
namespace {

constexpr int CH = kVerifyChunk;         // logits per workgroup: 256 threads x 16
constexpr int PT = CH / 256;

struct RowStat {                         // of a chunk or of a row: largest logit, its lowest index, sum of exp((l - m) / temp)
    float m;
    int i;
    double s;
};

// exp((l - m) / temp) for a finite m, it = log2(e) / temp: 1 at the maximum, 0 for -inf and NaN (and where m
// is -inf).  2^y = 2^n 2^f, n the integer nearest y (its bits are the low ones of y + 1.5 * 2^52), |f| <= 1/2,
// 2^f = 1 + f q(f), q of degree 9 interpolating (2^f - 1) / f at Chebyshev nodes: off by less than 6e-16.
// What the 64-bit unit has to do for a logit counts with many rows: 19 instructions, 88 MB of logits in 22
// us (30 instructions of an exp to the base e with its special cases by selects: 29 us).
__device__ __forceinline__ double weight_finite(float l, float m, double it) {
    constexpr double M = 6755399441055744.0;
    const double y = fmax(((double)l - (double)m) * it, -2000.0);
    const double t = y + M, f = y - (t - M);
    double q = 7.0709778665081383e-09;
    q = fma(q, f, 1.0205905413765595e-07);
    q = fma(q, f, 1.3215451633221434e-06);
    q = fma(q, f, 1.5252672924850737e-05);
    q = fma(q, f, 0.00015403530424776529);
    q = fma(q, f, 0.0013333558200794592);
    q = fma(q, f, 0.0096181291076186653);
    q = fma(q, f, 0.05550410866465167);
    q = fma(q, f, 0.24022650695910075);
    q = fma(q, f, 0.69314718055994617);
    return __builtin_ldexp(fma(q, f, 1.0), __double2loint(t));
}
// Where m is +inf, the logits above this weigh the same and the rest nothing: those that are +inf, at an
// infinite temperature all but -inf.
__device__ __forceinline__ float weightless(double it) { return it == 0.0 ? -INFINITY : 3.402823466e38f; }
// The same as weight_finite for any m.
__device__ __forceinline__ double weight(float l, float m, double it) {
    return m == INFINITY ? (l > weightless(it) ? 1.0 : 0.0) : weight_finite(l, m, it);
}
// Logits of a row whose largest is m, made such that weight_finite(l, m) is right.
template <int N>
__device__ __forceinline__ void make_finite(float (&l)[N], float& m, double it) {
    if (m < INFINITY) return;
    const float none = weightless(it);
#pragma unroll
    for (int e = 0; e < N; e++) l[e] = l[e] > none ? 0.f : -INFINITY;
    m = 0.f;
}

// The whole row's statistics from its chunks', by one wave, in a fixed order.  keep [64]: the first
// chunks' masses.
__device__ __forceinline__ RowStat row_of_chunks(const RowStat* ch, int C, double it, double* keep = nullptr) {
    const int lane = threadIdx.x & 63;
    RowStat first = {-INFINITY, INT_MAX, 0.0};
    if (lane < C) first = ch[lane];                          // (held: most rows have at most 64 chunks)
    RowStat r = first;
    for (int c = lane + 64; c < C; c += 64)
        if (ch[c].m > r.m) r.m = ch[c].m, r.i = ch[c].i;     // (chunks in ascending order: the first of equals stays)
    const float m = wave_max(r.m);
    r.i = wave_min(r.m == m ? r.i : INT_MAX);
    r.m = m;
    r.s = first.s * weight(first.m, r.m, it);
    if (keep) keep[lane] = r.s;
    for (int c = lane + 64; c < C; c += 64) r.s += ch[c].s * weight(ch[c].m, r.m, it);
    r.s = wave_sum(r.s);
    return r;
}

__device__ __forceinline__ double inv_temp(const float* temp, int b) {     // log2(e) / temp
    const float t = temp ? temp[b] : 1.f;
    return t > 0.f ? 1.4426950408889634 / (double)t : -1.0;                 // -1: greedy (0: an infinite temperature)
}

__device__ __forceinline__ double lane_of(double v, int j) {     // (j the same in every lane)
    return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), j), __builtin_amdgcn_readlane(__double2loint(v), j));
}

// A wave's view of sequence b's tree: lane i is node i.
struct Tree {
    int par;
    u64 anc;                             // the node and those above it; 0: not in the tree
};
__device__ __forceinline__ Tree tree_of(int par, int T) {      // (par: node i's parent, -2 past the last node)
    Tree t;
    t.anc = tree_sees(par, T);
    t.par = t.anc ? par : -2;
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
    double* sums;                        // [B][C] residual mass of the last token's row
    int* cnt;                            // [B] workgroups that have written theirs, 0 between launches
    int B, T, V, C, levels;
};

struct __attribute__((packed, aligned(4))) Quad {    // (loads of 16 bytes need an alignment of 4 here)
    float f[4];
};

// 16 logits of a row, element e at `at` + STRIDE (e / 4) + e % 4; `rest` past the row's end, which is within
// the span of the threads that load together unless `whole`.
template <int STRIDE>
__device__ __forceinline__ void load16(float (&v)[PT], const float* row, int at, bool whole, int V, float rest) {
    if (whole) {
#pragma unroll
        for (int e = 0; e < PT; e += 4) {
            const Quad q = *reinterpret_cast<const Quad*>(row + at + STRIDE / 4 * e);
#pragma unroll
            for (int k = 0; k < 4; k++) v[e + k] = q.f[k];
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < PT; e++) {                             // (unconditional loads: under a condition each waits)
        const int i = at + STRIDE * (e / 4) + e % 4;
        v[e] = row[i < V ? i : V - 1];
    }
#pragma unroll
    for (int e = 0; e < PT; e++)
        if (at + STRIDE * (e / 4) + e % 4 >= V) v[e] = rest;
}
// Lowest index of a wave's largest logit m and its sum of weights.
template <int STRIDE>
__device__ __forceinline__ RowStat stat16(float (&v)[PT], int at, float m, double it) {
    RowStat r = {m, INT_MAX, 0.0};
#pragma unroll
    for (int e = PT - 1; e >= 0; e--)
        if (v[e] == m && m > -INFINITY) r.i = at + STRIDE * (e / 4) + e % 4;
    if (it >= 0) {
        float mf = m;
        make_finite(v, mf, it);
#pragma unroll
        for (int e = 0; e < PT; e++) r.s += weight_finite(v[e], mf, it);
    }
    r.i = wave_min(r.i);
    r.s = wave_sum(r.s);
    return r;
}

// Statistics of a chunk of a row: one read of the logits, held in registers between the maximum and
// the sum.  grid (C, B * T), 256 threads.  Rows of nodes that hang under nothing are not read.
__global__ __launch_bounds__(256) void verify_stats_k(const float* __restrict__ logits, size_t ldl, const int* __restrict__ parent,
                                                      const float* __restrict__ temp, int T, int V, RowStat* __restrict__ ch) {
    __shared__ float sm[4];
    __shared__ int si[4];
    __shared__ double ss[4];
    const int row = blockIdx.y, b = row / T, c = blockIdx.x, w = threadIdx.x >> 6;
    if (parent[(size_t)b * T] != -1 || (row % T && parent[row] < 0)) return;
    const float* l = logits + (size_t)row * ldl;
    float v[PT], m = -INFINITY;
    const int at = c * CH + 4 * (int)threadIdx.x;
    load16<1024>(v, l, at, (c + 1) * CH <= V, V, -INFINITY);
    const double it = inv_temp(temp, b);
#pragma unroll
    for (int e = 0; e < PT; e++) m = fmaxf(m, v[e]);           // (drops NaN)
    m = wave_max(m);
    if ((threadIdx.x & 63) == 0) sm[w] = m;
    __syncthreads();
    m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    const RowStat part = stat16<1024>(v, at, m, it);
    if ((threadIdx.x & 63) == 0) si[w] = part.i, ss[w] = part.s;
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
    const int i = threadIdx.x & 63, n = row % T, par = i < T ? parent[(size_t)b * T + i] : -2;
    if (__builtin_amdgcn_readlane(par, 0) != -1) return;       // idle
    if (__popcll(__ballot(i > n && par == n)) <= level) return;     // (padding's children are counted too, to no harm)
    const double it = inv_temp(temp, b);
    if (!(it >= 0)) return;
    float l[PT], pq[PT];
    const int at = c * CH + 4 * (int)threadIdx.x;
    load16<1024>(l, logits + (size_t)row * ldl, at, (c + 1) * CH <= V, V, -INFINITY);
    load16<1024>(pq, q + (size_t)row * ldq, at, (c + 1) * CH <= V, V, 0.f);
    double a = 1.0;
    if (level > 1) {
        const double* prev = part + ((size_t)(level - 1) * R + row) * C;
        double w = 0;
        for (int k = threadIdx.x & 63; k < C; k += 64) w += prev[k];
        a = av[(size_t)(level - 1) * R + row] + wave_sum(w);
    }
    const RowStat r = row_of_chunks(ch + (size_t)row * C, C, it);
    const double is = r.s > 0 ? 1.0 / r.s : 0.0;
    float mf = r.m;
    make_finite(l, mf, it);
    double s = 0;
#pragma unroll
    for (int e = 0; e < PT; e++) s += fmax(weight_finite(l[e], mf, it) * is - a * (double)pq[e], 0.0);
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
    double rejw[64];                     // their weights
};

// What one wave reads of sequence b's tree, lane i node i.
struct Nodes {
    Tree t;
    int tok;
    float lt;                            // its token's logit in its parent's row
    double qc, u;                        // and probability there; its uniform
};
// Earlier siblings of lane i's node (nodes are in index order), by one wave; kids [64] in LDS, the wave's own.
__device__ __forceinline__ u64 siblings(const Tree& t, u64* kids) {
    const int i = threadIdx.x & 63;
    const bool kid = t.anc && i > 0;
    kids[i] = 0;
    __builtin_amdgcn_wave_barrier();
    if (kid) atomicOr(kids + t.par, 1ull << i);
    __builtin_amdgcn_wave_barrier();
    return kid ? kids[t.par] & ((1ull << i) - 1) : 0;
}
__device__ __forceinline__ Nodes read_nodes(const Verify& A, int b) {
    const int i = threadIdx.x & 63;
    Nodes n;
    int tok = i < A.T ? A.draft[(size_t)b * A.T + i] : -1;
    const float u = i < A.T ? A.u[(size_t)b * A.T + i] : 0.f;
    const int par = i < A.T ? A.parent[(size_t)b * A.T + i] : -2;
    // (what a node names is read while the tree is made out: padding reads too)
    const bool named = i > 0 && par >= 0 && par < i && tok >= 0 && tok < A.V;
    const size_t prow = (size_t)b * A.T + (named ? par : 0);
    const float lt = A.logits[prow * A.ldl + (named ? tok : 0)], qc = A.q ? A.q[prow * A.ldq + (named ? tok : 0)] : 0.f;
    n.t = tree_of(par, A.T);
    const bool kid = n.t.anc && i > 0, real = kid && named;
    n.tok = kid ? tok : -1;
    n.lt = real ? lt : -INFINITY;
    n.qc = real ? (double)qc : 0.0;
    n.u = kid ? (double)u : 0.0;
    return n;
}

// The path of sequence b, by one wave, lane i node i; rows: the statistics of its T rows.  Whether a
// node is accepted, once reached, depends on its parent's row and its earlier siblings alone, so all
// nodes are tested at once and the path is the set whose ancestors all passed.
__device__ void walk(const Verify& A, int b, double it, const Nodes& nd, const RowStat* rows, const double* mass, u64* kids, bool write, Draw* d) {
    const int i = threadIdx.x & 63, T = A.T, R = A.B * T;
    const Tree t = nd.t;
    const bool kid = t.anc && i > 0;
    const int tok = nd.tok, pn = kid ? t.par : 0;
    const size_t prow = (size_t)b * T + pn;
    const bool real = tok >= 0 && tok < A.V;
    const RowStat r = rows[pn];
    const double wt = it >= 0 ? weight(nd.lt, r.m, it) : 0.0, pc = r.s > 0 ? wt / r.s : 0.0;
    const u64 sib = siblings(t, kids);
    double W = 1.0, a = 0.0;
    bool tested = kid, first = true;                           // first: no earlier sibling has its token
    if (A.q) {
        const int rank = __popcll(sib);
        tested = kid && rank < A.levels;
        if (tested && rank > 0) W = mass[i], a = A.av[(size_t)rank * R + prow];
    } else {
        // the k-th earlier siblings of all nodes at once; that one has been compared with its own k by then
        for (u64 rest = sib; __any(rest != 0); rest &= rest - 1) {
            const int j = rest ? __ffsll((unsigned long long)rest) - 1 : i, tj = __shfl(tok, j);
            const double pj = __shfl(first ? pc : 0.0, j);
            if (rest) {
                W -= pj;
                first = first && tj != tok;
            }
        }
    }
    bool yes = A.q ? nd.u * W * nd.qc < pc - a * nd.qc : first && nd.u * W < pc;
    if (!(it >= 0)) yes = tok == r.i;
    yes = yes && tested && real;
    const u64 yesm = __ballot(yes);
    const u64 okm = __ballot(yes && !(sib & yesm));
    const bool on = t.anc && !(t.anc & ~okm & ~1ull);
    const u64 onm = __ballot(on);
    const int n = __popcll(onm), pos = __popcll(onm & ((1ull << i) - 1));
    const int last = n ? 63 - __clzll(onm) : 0;
    const bool rejected = kid && t.par == last && n;
    const u64 rejm = __ballot(rejected && (A.q ? tested : real && first));
    if (rejm >> i & 1) {
        const int k = __popcll(rejm & ((1ull << i) - 1));
        d->rej[k] = tok;
        d->rejw[k] = wt;
    }
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
    // -1 wherever no value belongs (the last token comes after the draw)
    if (i < T && i >= n) {
        A.path[(size_t)b * T + i] = -1;
        A.tokens[(size_t)b * T + i] = -1;
    }
    if (on) A.path[(size_t)b * T + pos] = i;
    if (on && i > 0) A.tokens[(size_t)b * T + pos - 1] = tok;
    if (i == 0) {
        A.count[b] = n;
        if (A.kv_len) A.kv_len[b] += n;
    }
}

// Residual weights of four tokens from `at` on; their sum.
__device__ __forceinline__ double residuals(double (&w)[4], const Verify& A, const Draw& d, double it, int at) {
    const float* l = A.logits + (size_t)d.row * A.ldl + at;
    const float* q = A.q ? A.q + (size_t)d.row * A.ldq + at : nullptr;
    const double is = d.r.s > 0 ? 1.0 / d.r.s : 0.0;
    Quad lv, qv = {};
    if (at + 4 <= A.V) {
        lv = *reinterpret_cast<const Quad*>(l);
        if (q) qv = *reinterpret_cast<const Quad*>(q);
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            lv.f[e] = at + e < A.V ? l[e] : -INFINITY;
            if (q) qv.f[e] = at + e < A.V ? q[e] : 0.f;
        }
    }
    float mf = d.r.m;
    make_finite(lv.f, mf, it);
#pragma unroll
    for (int e = 0; e < 4; e++) {
        w[e] = weight_finite(lv.f[e], mf, it);
        if (q) w[e] = fmax(w[e] * is - d.a * (double)qv.f[e], 0.0);
    }
    for (int k = 0; k < d.nrej; k++) {
        const int i = d.rej[k] - at;
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (i == e) w[e] = 0.0;
    }
    return w[0] + w[1] + w[2] + w[3];
}

// Statistics of sequence b's rows into LDS, a wave per row, beside what the first wave reads of its
// tree, and the walk.  mass [64]: the residual's sum that a later sibling is tested against; keep: the
// rows' first 64 chunks' masses.
__device__ __forceinline__ void walk_sequence(const Verify& A, int b, double it, RowStat* rows, double* mass, double (*keep)[64],
                                              bool write, Draw* d) {
    __shared__ u64 kids[64];
    const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6), waves = blockDim.x >> 6;
    Nodes nd;
    if (w == 0) nd = read_nodes(A, b);
    for (int n = w; n < A.T; n += waves) {
        const RowStat r = row_of_chunks(A.ch + ((size_t)b * A.T + n) * A.C, A.C, it, keep ? keep[n] : nullptr);
        if (lane == 0) rows[n] = r;
    }
    if (A.q && A.levels > 1 && it >= 0) {
        const int par = lane < A.T ? A.parent[(size_t)b * A.T + lane] : -2;
        for (int i = 1 + w; i < A.T; i += waves) {             // (of padding too: nothing reads that)
            const int pn = __builtin_amdgcn_readlane(par, i);
            const int k = __popcll(__ballot(lane > pn && lane < i && par == pn));
            if (pn < 0 || pn >= i || k < 1 || k >= A.levels) continue;
            const double* src = A.part + ((size_t)k * A.B * A.T + (size_t)b * A.T + pn) * A.C;
            double s = 0;
            for (int c = lane; c < A.C; c += 64) s += src[c];
            s = wave_sum(s);
            if (lane == 0) mass[i] = s;
        }
    }
    __syncthreads();
    if (w == 0) walk(A, b, it, nd, rows, mass, kids, write, d);
    __syncthreads();
}

// The first thread at which the masses' running sum (in thread order) exceeds r, or u times their total
// where r is negative; where rounding leaves none, the last one with any; -1 where there is no mass.
// Every thread gets it; r becomes what of it is left there.  kDrawThreads threads.
constexpr int kDrawThreads = 1024, kDrawWaves = kDrawThreads / 64;
struct PickLds {
    double part[kDrawWaves], left;
    int at;
};
__device__ __forceinline__ int block_pick(double mine, double u, double& r, PickLds& L) {
    const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6);
    const double inc = wave_scan(mine);
    if (lane == 63) L.part[w] = inc;
    if (threadIdx.x == 0) L.at = -1;
    __syncthreads();
    // lane k has wave k's (sums over them one after the other, in every wave, took 1 us more)
    const double part = lane < kDrawWaves ? L.part[lane] : 0.0, upto = wave_scan(part);
    if (r < 0) r = u * lane_of(upto, 63);
    const u64 over = __ballot(upto > r && part > 0), some = __ballot(part > 0);
    const int ws = over ? __ffsll((unsigned long long)over) - 1 : 63 - __clzll(some);    // -1: none
    if (w == ws) {
        const double base = ws ? lane_of(upto, ws - 1) : 0.0;
        const u64 hit = __ballot(base + inc > r && mine > 0), any = __ballot(mine > 0);
        if (lane == (hit ? __ffsll((unsigned long long)hit) - 1 : 63 - __clzll(any))) {
            L.at = threadIdx.x;
            L.left = r - (base + inc - mine);
        }
    }
    __syncthreads();
    r = L.left;
    return L.at;
}
// Of a thread's E masses from `left` on: the first at which their sum exceeds it, else the last with any;
// `left` becomes what of it is left there.
template <int E>
__device__ __forceinline__ int thread_pick(const double (&x)[E], double& left) {
    int at = -1;
    double acc = 0, before = 0;
    bool done = false;
#pragma unroll
    for (int e = 0; e < E; e++) {
        if (!done && x[e] > 0) at = e, before = acc;
        acc += x[e];
        done = done || (acc > left && x[e] > 0);
    }
    left -= before;
    return at;
}

// The last token, chunk tid having `mass`: by running sums over chunks, then over the tokens of one.  False
// where that one has none (its mass was rounding alone).
static_assert(kVerifyMaxV / CH == kDrawThreads && 4 * kDrawThreads == CH, "a thread has a chunk, and four tokens of one");
__device__ __forceinline__ bool pick_token(double mass, const Verify& A, const Draw& d, double it, double u, PickLds& L, int best,
                                           int* out) {
    const int tid = threadIdx.x;
    double r = -1.0;
    const int chunk = block_pick(mass, u, r, L);
    if (chunk < 0) {                                           // nothing left: the largest
        if (tid == 0) *out = best;
        return true;
    }
    __syncthreads();                                           // (every thread has its answer)
    const int at = chunk * CH + 4 * tid;
    double x[4], left = fmax(r, 0.0);
    const int th = block_pick(residuals(x, A, d, it, at), u, left, L);
    if (th == tid) *out = at + thread_pick(x, left);
    return th >= 0;
}

// With draft probabilities, the walk, the chunk sums of the residual and the last token.  Every workgroup of a
// sequence walks for itself (a launch less), the first one writes the path; the last to write its sum draws
// (another launch less, 3 us of the host's).  Sums go through the L2 to where all XCDs see them (agent
// scope), are there before the workgroup counts itself in, and are read from there; nobody waits.  grid (C, B),
// kDrawThreads threads.
__global__ __launch_bounds__(kDrawThreads) void verify_residual_k(const Verify A) {
    __shared__ double ss[kDrawWaves];
    __shared__ RowStat rows[64];
    __shared__ double mass[64];
    __shared__ Draw d;
    __shared__ PickLds L;
    __shared__ bool s_last;
    const int b = blockIdx.y, c = blockIdx.x, tid = threadIdx.x;
    const double it = inv_temp(A.temp, b), u = (double)A.u[(size_t)b * A.T];
    walk_sequence(A, b, it, rows, mass, nullptr, c == 0, &d);
    if (d.row < 0) return;
    int* out = A.tokens + (size_t)b * A.T + d.n - 1;
    const int best = d.r.i < A.V ? d.r.i : -1;
    if (!(it >= 0) || best < 0) {                              // greedy, or a row with nothing in it
        if (c == 0 && tid == 0) *out = best;
        return;
    }
    double w[4];
    const double s = wave_sum(residuals(w, A, d, it, c * CH + 4 * tid));
    if ((tid & 63) == 0) ss[tid >> 6] = s;
    __syncthreads();
    u64* sums = reinterpret_cast<u64*>(A.sums + (size_t)b * A.C);
    if (tid == 0) {
        double t = 0;
        for (int k = 0; k < kDrawWaves; k++) t += ss[k];
        __hip_atomic_store(sums + c, __builtin_bit_cast(u64, t), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        s_last = __hip_atomic_fetch_add(A.cnt + b, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == A.C - 1;
    }
    __syncthreads();
    if (!s_last) return;
    if (tid == 0) __hip_atomic_store(A.cnt + b, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const double m = tid < A.C ? __builtin_bit_cast(double, __hip_atomic_load(sums + tid, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) : 0.0;
    if (!pick_token(m, A, d, it, u, L, best, out) && tid == 0) *out = best;
}

// Without them, the walk and the last token, after verify_stats_k.  grid B, kDrawThreads threads.
//
// A chunk's mass is the sum that verify_stats_k left, less the rejected tokens'.  Where hardly anything is
// left that difference says little, and the chunks are summed anew; so they are where the chunk that is
// picked turns out to hold rejected tokens alone.
__global__ __launch_bounds__(kDrawThreads) void verify_draw_k(const Verify A) {
    __shared__ RowStat rows[64];
    __shared__ Draw d;
    __shared__ PickLds L;
    __shared__ double s_sum[kDrawWaves], keep[64][64];
    const int b = blockIdx.x, tid = threadIdx.x;
    const double it = inv_temp(A.temp, b), u = (double)A.u[(size_t)b * A.T];
    walk_sequence(A, b, it, rows, nullptr, keep, true, &d);
    if (d.row < 0) return;
    int* out = A.tokens + (size_t)b * A.T + d.n - 1;
    const int best = d.r.i < A.V ? d.r.i : -1;
    if (!(it >= 0) || best < 0) {                              // greedy, or a row with nothing in it
        if (tid == 0) *out = best;
        return;
    }
    double mass = 0, gone = 0;
    if (tid < 64) {
        mass = keep[d.row - b * A.T][tid];
    } else if (tid < A.C) {
        const RowStat s = A.ch[(size_t)d.row * A.C + tid];
        mass = s.s * weight(s.m, d.r.m, it);
    }
    for (int k = 0; k < d.nrej; k++) {
        if (d.rej[k] / CH == tid) mass -= d.rejw[k];
        gone += d.rejw[k];
    }
    mass = fmax(mass, 0.0);
    for (bool anew = d.r.s - gone < 1e-6 * d.r.s;; anew = true) {
        if (anew)
            for (int c = 0; c < A.C; c++) {
                double x[4];
                const double s = wave_sum(residuals(x, A, d, it, c * CH + 4 * tid));
                if ((tid & 63) == 0) s_sum[tid >> 6] = s;
                __syncthreads();
                if (tid == c) {
                    mass = 0;
                    for (int k = 0; k < kDrawWaves; k++) mass += s_sum[k];
                }
                __syncthreads();
            }
        if (pick_token(mass, A, d, it, u, L, best, out)) return;
        if (anew) {
            if (tid == 0) *out = best;
            return;
        }
    }
}

// The whole verification in one launch, a workgroup a sequence, where its rows are few pieces of 1024 logits
// (a wave each) and no residual levels are needed; verify_one_launch says where.
// grid B, 1024 threads; A.C: pieces in a row.
constexpr int SP = 1024, kSmallPieces = 32;
__global__ __launch_bounds__(1024) void verify_small_k(const Verify A) {
    __shared__ RowStat ch[kSmallPieces], rows[64];
    __shared__ double keep[kSmallPieces][64];
    __shared__ u64 kids[64];
    __shared__ Draw d;
    __shared__ PickLds L;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = uniform(tid >> 6), C = A.C;
    const double it = inv_temp(A.temp, b), u = (double)A.u[(size_t)b * A.T];
    Nodes nd;
    if (w == 0) nd = read_nodes(A, b);
    for (int p = w; p < A.T * C; p += 16) {
        const int n = p / C, c = p - n * C, at = c * SP + 4 * lane;
        float v[PT], m = -INFINITY;
        load16<256>(v, A.logits + ((size_t)b * A.T + n) * A.ldl, at, (c + 1) * SP <= A.V, A.V, -INFINITY);
#pragma unroll
        for (int e = 0; e < PT; e++) m = fmaxf(m, v[e]);       // (drops NaN)
        const RowStat r = stat16<256>(v, at, wave_max(m), it);
        if (lane == 0) ch[p] = r;
    }
    __syncthreads();
    for (int n = w; n < A.T; n += 16) {
        const RowStat r = row_of_chunks(ch + n * C, C, it, keep[n]);
        if (lane == 0) rows[n] = r;
    }
    __syncthreads();
    if (w == 0) walk(A, b, it, nd, rows, nullptr, kids, true, &d);
    __syncthreads();
    if (d.row < 0) return;
    int* out = A.tokens + (size_t)b * A.T + d.n - 1;
    const int best = d.r.i < A.V ? d.r.i : -1, row = d.row - b * A.T;
    if (!(it >= 0) || best < 0) {                              // greedy, or a row with nothing in it
        if (tid == 0) *out = best;
        return;
    }
    double gone = 0;
    for (int k = 0; k < d.nrej; k++) gone += d.rejw[k];
    for (bool anew = A.q || d.r.s - gone < 1e-6 * d.r.s;; anew = true) {       // (see verify_draw_k)
        if (anew) {
            for (int c = w; c < C; c += 16) {
                double s = 0, x[4];
#pragma unroll
                for (int k = 0; k < 4; k++) s += residuals(x, A, d, it, c * SP + 256 * k + 4 * lane);
                s = wave_sum(s);
                if (lane == 0) keep[row][c] = s;
            }
            __syncthreads();
        }
        double mine = tid < C ? keep[row][tid] : 0.0, r = -1.0;
        if (!anew) {
            for (int k = 0; k < d.nrej; k++)
                if (d.rej[k] / SP == tid) mine -= d.rejw[k];
            mine = fmax(mine, 0.0);
        }
        const int owner = block_pick(mine, u, r, L);
        if (owner < 0) {                                       // nothing left: the largest
            if (tid == 0) *out = best;
            return;
        }
        __syncthreads();                                       // (every thread has its answer)
        const int at = owner * SP + 4 * tid;
        double x[4] = {}, left = fmax(r, 0.0);
        const int th = block_pick(tid < SP / 4 ? residuals(x, A, d, it, at) : 0.0, u, left, L);
        if (th == tid) *out = at + thread_pick(x, left);
        if (th >= 0) return;
        if (anew) {
            if (tid == 0) *out = best;
            return;
        }
    }
}

size_t up16(size_t n) { return (n + 15) & ~size_t(15); }

}  // namespace

// Whether verify_small_k takes it, by the faster of the two in a call as it is made: eager calls are bound by
// the host, whose 3 us for a launch it saves, captured ones by the device, where one CU's 64-bit rate counts.
// Eagerly it gains as far as 32 pieces go: one row of 32768 logits 16.3 -> 13.0 us, 7 pieces for each of 4 rows
// 16.1 -> 13.0, a row of 20480 with draft probabilities 16.9 -> 15.0 (32 rows of 1000 16.5 -> 17.4).
// In a graph it gains up to about 20 pieces, or 24 with draft probabilities, whose residual counts as a row more:
// one row of 19 pieces 10.4 -> 10.1 us, of 20 9.7 -> 10.0, of 24 9.8 -> 10.8, of 32 9.8 -> 12.5; 16 x 2 rows of
// 10 11.1 -> 10.7, of 12 10.5 -> 11.3; 4 rows of 5 10.4 -> 10.5, of 6 10.8 -> 11.2; with draft probabilities one
// row of 12 12.5 -> 11.9, of 13 12.6 -> 13.4, 2 rows of 8 12.1 -> 11.9, of 9 12.6 -> 13.2, 6 of 3 13.0 -> 12.0.
OneLaunch verify_one_launch(int T, int V, int levels, bool q) {
    const int pieces = (V + SP - 1) / SP;
    if (levels != 1 || (q ? 3 : 2) * T * pieces + 2 * T > 2 * kSmallPieces + 2) return kNever;
    return (q ? (T + 1) * pieces <= 24 : T * pieces <= 20) ? kAlways : kEager;
}

size_t verify_ws_bytes(int B, int T, int V, int levels) {
    const size_t R = (size_t)B * T, C = (V + CH - 1) / CH;
    return up16(R * C * sizeof(RowStat)) + up16(R * levels * 8) + up16(R * C * levels * 8) + up16(B * C * 8);
}

hipError_t launch_verify_tree(int* tokens, int* path, int* count, int* kv_len, const float* logits, size_t ldl, const int* draft,
                              const int* parent, const float* u, const float* temp, const float* q, size_t ldq, int B, int T, int V,
                              int levels, void* ws, int* cnt, hipStream_t st) {
    const int R = B * T, C = (V + CH - 1) / CH;
    unsigned char* p = static_cast<unsigned char*>(ws);
    auto take = [&](size_t n) { unsigned char* r = p; p += up16(n); return r; };
    RowStat* ch = reinterpret_cast<RowStat*>(take((size_t)R * C * sizeof(RowStat)));
    double* av = reinterpret_cast<double*>(take((size_t)R * levels * 8));
    double* part = reinterpret_cast<double*>(take((size_t)R * C * levels * 8));
    double* sums = reinterpret_cast<double*>(take((size_t)B * C * 8));
    const Verify a = {tokens, path, count, kv_len, logits, ldl, draft, parent, u, temp, q, ldq, ch, av, part, sums, cnt, B, T, V, C, levels};
    if (!ws) {
        Verify one = a;
        one.C = (V + SP - 1) / SP;
        hipLaunchKernelGGL(verify_small_k, dim3(B), dim3(1024), 0, st, one);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(verify_stats_k, dim3(C, R), dim3(256), 0, st, logits, ldl, parent, temp, T, V, ch);
    for (int k = 1; k < levels; k++)
        hipLaunchKernelGGL(verify_mass_k, dim3(C, R), dim3(256), 0, st, logits, ldl, q, ldq, parent, temp, T, V, k, ch, av, part);
    if (q)
        hipLaunchKernelGGL(verify_residual_k, dim3(C, B), dim3(kDrawThreads), 0, st, a);
    else
        hipLaunchKernelGGL(verify_draw_k, dim3(B), dim3(kDrawThreads), 0, st, a);
    return hipGetLastError();
}

}  // namespace rt4
