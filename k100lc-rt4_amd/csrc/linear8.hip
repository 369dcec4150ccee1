// linear8.hip -- products of int8 codes with a scale for each token and each channel, and the first half of
// a gated feed-forward block on them.
//
//   c[m][n] = sx[m] sw[n] Σ_k xq[m][k] wq[n][k]                     (exact int32 sums, K < 2^17)
//   h[m][n] = act(sx[m] sg[n] Σ_k xq[m][k] wg[n][k]) * (sx[m] su[n] Σ_k xq[m][k] wu[n][k])
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "ffn_dev.h"
#include "rt4_internal.h"

namespace rt4 {

namespace {

// One output from its sums: each is converted once (2^-24), the scales applied one after the other.
template <int NW>
__device__ __forceinline__ float finish(int i0, int i1, float sx, float s0, float s1, int act) {
    const float g = (float)i0 * sx * s0;
    return NW == 1 ? g : activate(g, act) * ((float)i1 * sx * s1);
}

// ---- Tiles on the matrix cores.  A workgroup of WM x WN waves owns BM tokens and BN weight rows, a wave 32 TM x 32 TN of
// them as fragments of v_mfma_i32_32x32x32_i8 with the weights as A: a lane then holds one token (lane & 31) and runs of 4
// channels (8 (i >> 2) + 4 (lane >> 5) + (i & 3)).  With two weight matrices (NW) the first half of a wave's fragments are
// gate rows and the second half the up rows of the same channels, so both factors of an output meet in one lane.
//
// Steps are 128 codes deep: whole cache lines of a row.  Operands arrive by DMA (8 rows x 128 bytes an instruction) in a
// ring of ST stages; in a stage, chunk c (16 bytes) of row r lies at slot c ^ (r >> 1 & 7), which puts the 16 rows that one
// cycle of a read serves into 16 different bank groups.  One barrier a step, before its last quarter: by then every wave
// has read the stage for the last time, and the DMA of the step ST further on goes into it from there on.
template <int TM_, int TN_, int WM_, int WN_, int ST_>
struct Tile {
    static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, ST = ST_, W = WM * WN;
    static constexpr int BM = 32 * TM * WM, BN = 32 * TN * WN, STAGE = (BM + BN) * 128, LDS = ST * STAGE;
    static constexpr int PA = BM / 8 / W, PB = BN / 8 / W, P = PA + PB;   // DMA instructions of a wave a step
    static_assert(BM % (8 * W) == 0 && BN % (8 * W) == 0 && TN % 2 == 0 && WM <= 2, "");
    static_assert(LDS <= 160 * 1024 && 32 * (TN * 32 * 4 + 16) * W <= LDS, "a slab of fp32 outputs fits a wave's share");
};

struct Where {                           // a workgroup's tile and steps
    int tile, part, m0, n0, s0, s1;
};

template <class C, int NW>
__device__ __forceinline__ Where where(const Linear8& a, int splits, int b, int blocks) {
    const int nm = (a.M + C::BM - 1) / C::BM, nn = (a.N + C::BN / NW - 1) / (C::BN / NW);
    // Workgroups go round the XCDs: each takes a run of the list, in which tiles that share operands are neighbours.
    const int x = b & 7, per = blocks >> 3, rem = blocks & 7, t = x * per + min(x, rem) + (b >> 3);
    Where w;
    w.part = t % splits;
    w.tile = t / splits;
    constexpr int GM = 4;
    const int first = w.tile / (GM * nn) * GM, rows = min(GM, nm - first), in = w.tile - first * nn;
    w.m0 = (first + in % rows) * C::BM;
    w.n0 = in / rows * (C::BN / NW);
    const int steps = (a.K + 127) >> 7;
    w.s0 = (int)((long long)steps * w.part / splits);
    w.s1 = (int)((long long)steps * (w.part + 1) / splits);
    return w;
}

// The scales of a lane's channels: runs of 4 from n0 + 8 q + 4 (lane >> 5).
template <int NC>
__device__ __forceinline__ void load_scales(float (&s)[NC * 16], const float* sw, int n0, int N) {
    const int hi = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int q = 0; q < NC * 4; q++) {
        const int n = n0 + 8 * q + 4 * hi;
        if (n + 4 <= N) __builtin_memcpy(&s[4 * q], sw + n, 16);
        else
#pragma unroll
            for (int e = 0; e < 4; e++) s[4 * q + e] = sw[min(n + e, N - 1)];
    }
}

// 32 tokens x 32 NC channels of a wave from its sums: through the wave's own LDS, out in 16-byte pieces of rows.
template <int NW, class T, int NC>
__device__ __forceinline__ void write_slab(const Linear8& a, const v16i* i0, const v16i* i1, const float* s0, const float* s1, int m0, int n0,
                                           unsigned char* lds) {
    constexpr int PITCH = NC * 32 * (int)sizeof(T) + 16, PER = 16 / (int)sizeof(T), LPR = NC * 32 / PER;
    const int lane = threadIdx.x & 63, ml = lane & 31, hi = lane >> 5;
    const float sx = a.sx[min(m0 + ml, a.M - 1)];
#pragma unroll
    for (int c = 0; c < NC; c++)
#pragma unroll
        for (int q = 0; q < 4; q++) {
            T t[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int k = 16 * c + 4 * q + e;
                t[e] = (T)finish<NW>(i0[c][4 * q + e], NW == 1 ? 0 : i1[c][4 * q + e], sx, s0[k], NW == 1 ? 0.f : s1[k], a.act);
            }
            __builtin_memcpy(lds + ml * PITCH + (32 * c + 8 * q + 4 * hi) * sizeof(T), t, sizeof(t));
        }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const bool vec = ((uintptr_t)a.out & 15) == 0 && a.ldo * (int)sizeof(T) % 16 == 0;
    const int col = lane % LPR * PER, n = n0 + col;
#pragma unroll
    for (int k = 0; k < 32 * LPR / 64; k++) {
        const int r = lane / LPR + k * (64 / LPR), m = m0 + r;
        const uint4 d = *reinterpret_cast<const uint4*>(lds + r * PITCH + col * sizeof(T));
        if (m < a.M && n < a.N) {
            T* o = static_cast<T*>(a.out) + (size_t)m * a.ldo + n;
            if (vec && n + PER <= a.N) {
                *reinterpret_cast<uint4*>(o) = d;
            } else {
                T t[PER];
                __builtin_memcpy(t, &d, 16);
#pragma unroll
                for (int e = 0; e < PER; e++)
                    if (n + e < a.N) o[e] = t[e];
            }
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// All outputs of a wave.
template <class C, int NW, int ROWS>
__device__ __forceinline__ void write_wave(const Linear8& a, const v16i (&acc)[ROWS][C::TN], int m0, int n0, unsigned char* lds) {
    constexpr int NC = C::TN / NW;
    float s0[NC * 16], s1[NC * 16];
    load_scales<NC>(s0, a.sw[0], n0, a.N);
    if (NW == 2) load_scales<NC>(s1, a.sw[1], n0, a.N);
    const auto all = [&](auto t) {
#pragma unroll
        for (int i = 0; i < ROWS; i++)
            write_slab<NW, decltype(t), NC>(a, acc[i], acc[i] + (NW == 2 ? NC : 0), s0, s1, m0 + 32 * i, n0, lds);
    };
    if (a.type == kF32) all(float{});
    else if (a.type == kBF16) all(bf16{});
    else all(f16{});
}

template <int N>
__device__ __forceinline__ void wait_dma_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// part null: whole tiles; else this workgroup's sums (of one of `splits` runs of steps), a fragment's registers as they are.
template <class C, int NW>
__global__ __launch_bounds__(64 * C::W, 1) void linear8_tile_k(Linear8 a, int splits, int4* part) {
    constexpr int TM = C::TM, TN = C::TN, ST = C::ST, PA = C::PA, P = C::P, FR = TM + TN, MF = TM * TN;
    extern __shared__ __align__(16) unsigned char smem[];
    const int lane = threadIdx.x & 63, w = uniform((int)(threadIdx.x >> 6)), wm = w / C::WN, wn = w % C::WN;
    const Where at = where<C, NW>(a, splits, blockIdx.x, gridDim.x);

    // DMA: a wave brings PA pieces of 8 token rows and PB of weight rows.  Rows past the end read the last one (their
    // outputs are dropped).  Chunks of the last step that lie past K: the row's first chunk of that step instead, and the
    // tokens' codes there are cleared before they are used.
    const int steps = (a.K + 127) >> 7, whole = (a.K >> 4) & 7;
    uint32_t voff[P];
    const int even = (lane & 7) ^ (lane >> 4);    // chunk that a lane brings of even pieces; of odd ones it is even ^ 4
    const int pa0 = w * PA, pb0 = w * C::PB;     // first pieces
    const auto chunk = [&](int t) { return even ^ ((t < PA ? pa0 + t : pb0 + t - PA) & 1) * 4; };
    const auto mat = [&](int t) { return NW == 1 ? 0 : C::WM == 2 ? w & 1 : t - PA >= 2 * TN; };   // whose rows a weight piece is
#pragma unroll
    for (int t = 0; t < P; t++) {
        const int c = chunk(t);
        if (t < PA) {
            voff[t] = (uint32_t)min((pa0 + t) * 8 + (lane >> 3), a.M - 1 - at.m0) * (uint32_t)a.ldx + c * 16;
        } else {
            int r = (pb0 + t - PA) * 8 + (lane >> 3);                                  // channel in the tile
            if (NW == 2) r = (C::WM == 2 ? w >> 1 : w) * 16 * TN + (C::WM == 2 ? t - PA : (t - PA) % (2 * TN)) * 8 + (lane >> 3);
            voff[t] = (uint32_t)min(r, a.N - 1 - at.n0) * (uint32_t)(mat(t) ? a.ldw[1] : a.ldw[0]) + c * 16;
        }
    }
    const size_t k0 = (size_t)at.s0 * 128;
    const int8_t* ga = a.x + (size_t)at.m0 * a.ldx + k0;
    const int8_t* gb[NW];
#pragma unroll
    for (int j = 0; j < NW; j++) gb[j] = a.w[j] + (size_t)at.n0 * a.ldw[j] + k0;
    const uint32_t lds0 = lds_addr(smem);
    const uint32_t la = lds0 + (uint32_t)pa0 * 1024, lb = lds0 + C::BM * 128 + (uint32_t)pb0 * 1024;
    int issue = at.s0;                           // next step to bring
    uint32_t in = 0, out = 0;                    // byte offsets of the stages to fill and to read
    const auto next = [](uint32_t s) { return s == (uint32_t)(ST - 1) * C::STAGE ? 0u : s + C::STAGE; };
    const auto begin_issue = [&]() {
        if (whole && issue == steps - 1) {
#pragma unroll
            for (int t = 0; t < P; t++) {
                const int c = chunk(t);
                voff[t] -= c >= whole ? c * 16 : 0;
            }
        }
    };
    const auto dma_piece = [&](int t) {          // (t is a constant wherever loops are unrolled)
        if (t < PA) dma16<0>(voff[t], ga, la + in + t * 1024);
        else dma16<0>(voff[t], gb[NW == 1 ? 0 : mat(t)], lb + in + (t - PA) * 1024);
    };
    const auto issued = [&]() {
        issue++;
        ga += 128;
#pragma unroll
        for (int j = 0; j < NW; j++) gb[j] += 128;
        in = next(in);
    };
    // Pieces of a step that are brought behind the barrier, and in the first quarter of the step that follows.
    constexpr int P3 = P / 2;

    v16i acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][j][e] = 0;

    uint32_t ro[4];                              // a lane's place in a 32-row fragment, by quarter of the step
#pragma unroll
    for (int p = 0; p < 4; p++) ro[p] = (uint32_t)(lane & 31) * 128 + ((uint32_t)(2 * p + (lane >> 5)) ^ (lane >> 1 & 7)) * 16;
    const uint32_t oa = (uint32_t)(wm * TM) * 4096, ob = C::BM * 128 + (uint32_t)(wn * TN) * 4096;
    v4i fa[2][TM], fb[2][TN];
    const auto read = [&](int p, int f) {        // fragment f of quarter p of the stage at `out`
        if (f < TN) fb[p & 1][f] = *reinterpret_cast<const v4i*>(smem + (ro[p] + (out + ob)) + f * 4096);
        else fa[p & 1][f - TN] = *reinterpret_cast<const v4i*>(smem + (ro[p] + (out + oa)) + (f - TN) * 4096);
    };
    const auto clear_tail = [&]() {              // by all waves, after the last step has arrived
        for (int r = threadIdx.x; r < C::BM; r += 64 * C::W)
            for (int c = whole; c < 8; c++) *reinterpret_cast<v4i*>(smem + out + r * 128 + (c ^ (r >> 1 & 7)) * 16) = v4i{0, 0, 0, 0};
        __syncthreads();
    };
    // A quarter's products, among them the reads of the next quarter and pieces LO .. HI-1 of the DMA.
    const auto quarter = [&](auto pc, auto lo_, auto hi_, bool ahead) {
        constexpr int Q = decltype(pc)::value, LO = decltype(lo_)::value, HI = decltype(hi_)::value;
#pragma unroll
        for (int q = 0; q < MF; q++) {
            acc[q / TN][q % TN] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[Q & 1][q % TN], fa[Q & 1][q / TN], acc[q / TN][q % TN], 0, 0, 0);
            if (ahead)
#pragma unroll
                for (int o = q * 2 * FR / MF; o < (q + 1) * 2 * FR / MF; o++)
                    if (o < FR) read((Q + 1) & 3, o);
#pragma unroll
            for (int o = LO + q * (HI - LO) / MF; o < LO + (q + 1) * (HI - LO) / MF; o++) dma_piece(o);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // M1: step s + ST - 1 is still being brought; M2: there is a step s + ST.
    const auto step = [&](int s, auto m1, auto m2) {
        constexpr bool M1 = decltype(m1)::value, M2 = decltype(m2)::value;
#define RT4_C(x) std::integral_constant<int, (x)>{}
        quarter(RT4_C(0), RT4_C(P3), RT4_C(M1 ? P : P3), true);
        if (M1) issued();
        quarter(RT4_C(1), RT4_C(0), RT4_C(0), true);
        quarter(RT4_C(2), RT4_C(0), RT4_C(0), true);
        out = next(out);
        if (M1) wait_dma_barrier<(ST - 2) * P>();
        else wait_dma_barrier<0>();
        if (whole && s + 2 == steps && s + 1 < at.s1) clear_tail();
        if (M2) begin_issue();
        if (M1) quarter(RT4_C(3), RT4_C(0), RT4_C(M2 ? P3 : 0), true);
        else quarter(RT4_C(3), RT4_C(0), RT4_C(0), s + 1 < at.s1);
#undef RT4_C
    };
    typedef std::true_type yes;
    typedef std::false_type no;
#pragma unroll
    for (int p = 0; p < ST - 1; p++)
        if (issue < at.s1) {
            begin_issue();
#pragma unroll
            for (int t = 0; t < P; t++) dma_piece(t);
            issued();
        }
    if (at.s1 - at.s0 >= ST) wait_dma_barrier<(ST - 2) * P>();
    else wait_dma_barrier<0>();
    if (whole && at.s0 == steps - 1) clear_tail();
#pragma unroll
    for (int f = 0; f < FR; f++) read(0, f);
    if (issue < at.s1) {
        begin_issue();
#pragma unroll
        for (int t = 0; t < P3; t++) dma_piece(t);
    }
    int s = at.s0;
    for (; s < at.s1 - ST; s++) step(s, yes{}, yes{});
    if (s == at.s1 - ST) step(s++, yes{}, no{});
    for (; s < at.s1; s++) step(s, no{}, no{});

    if (part) {
        int4* o = part + ((size_t)(at.tile * splits + at.part) * C::W + w) * (MF * 256) + lane;
#pragma unroll
        for (int i = 0; i < TM; i++)
#pragma unroll
            for (int j = 0; j < TN; j++)
#pragma unroll
                for (int q = 0; q < 4; q++)
                    o[((i * TN + j) * 4 + q) * 64] = make_int4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
        return;
    }
    __syncthreads();                             // the stages are free for the outputs
    write_wave<C, NW, TM>(a, acc, at.m0 + wm * TM * 32, at.n0 + wn * (TN / NW) * 32, smem + (size_t)w * (C::LDS / C::W));
}

// Sums the runs of split tiles: a wave takes 32 tokens of a tile's wave.
template <class C, int NW>
__global__ __launch_bounds__(256) void linear8_join_k(Linear8 a, int splits, const int4* part, int waves) {
    constexpr int TM = C::TM, TN = C::TN, SLAB = 32 * (TN / NW * 32 * 4 + 16);
    __shared__ __align__(16) unsigned char smem[4 * SLAB];
    const int lane = threadIdx.x & 63, id = uniform((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
    if (id >= waves) return;                     // whole waves; no barrier follows
    const int i = id % TM, w = id / TM % C::W, tile = id / (TM * C::W);
    const int nm = (a.M + C::BM - 1) / C::BM, nn = (a.N + C::BN / NW - 1) / (C::BN / NW);
    constexpr int GM = 4;
    const int first = tile / (GM * nn) * GM, rows = min(GM, nm - first), in = tile - first * nn;
    const int m0 = (first + in % rows) * C::BM + (w / C::WN * TM + i) * 32, n0 = in / rows * (C::BN / NW) + w % C::WN * (TN / NW) * 32;
    if (m0 >= a.M || n0 >= a.N) return;
    v16i acc[1][TN];
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[0][j][e] = 0;
    const int4* p = part + ((size_t)tile * splits * C::W + w) * (TM * TN * 256) + i * TN * 256 + lane;
    for (int s = 0; s < splits; s++, p += (size_t)C::W * (TM * TN * 256))
#pragma unroll
        for (int j = 0; j < TN; j++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int4 v = p[(j * 4 + q) * 64];
                acc[0][j][4 * q] += v.x, acc[0][j][4 * q + 1] += v.y, acc[0][j][4 * q + 2] += v.z, acc[0][j][4 * q + 3] += v.w;
            }
    write_wave<C, NW, 1>(a, acc, m0, n0, smem + (threadIdx.x >> 6) * SLAB);
}

typedef Tile<4, 4, 2, 2, 2> T256x256;
typedef Tile<2, 4, 2, 2, 3> T128x256;
typedef Tile<2, 2, 2, 2, 2> T128x128;
typedef Tile<1, 2, 2, 2, 3> T64x128;
typedef Tile<1, 2, 1, 4, 2> T32x256;

template <class C, int NW>
hipError_t launch_tile(const Linear8& a, const Linear8Plan& p, void* part, hipStream_t st) {
    auto k = linear8_tile_k<C, NW>;
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(k, dim3((unsigned)(p.tiles * p.splits)), dim3(64 * C::W), C::LDS, st, a, p.splits, p.splits > 1 ? static_cast<int4*>(part) : nullptr);
    if (p.splits > 1) {
        const int waves = p.tiles * C::W * C::TM;
        hipLaunchKernelGGL((linear8_join_k<C, NW>), dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, st, a, p.splits, static_cast<const int4*>(part), waves);
    }
    return hipGetLastError();
}

// ---- Few tokens: dot products on the vector ALU, the weights streamed once.  A wave owns 4 weight rows (4 channels, or gate
// and up rows of 2) and goes through them 1 KB of each at a time, a lane 16 codes of each row, with the codes of every token
// beside them: each token's 16 bytes serve 4 rows.  The next loads are under way while 4 M v_dot4 an operand are done.  A
// workgroup is one wave, so that they spread evenly over the CUs.
template <int M, int NW>
__global__ __launch_bounds__(64) void linear8_dot_k(Linear8 a) {
    constexpr int RN = 4 / NW, U = M == 1 ? 4 : M <= 4 ? 2 : 1;      // channels of a wave; KB of each row at a time
    typedef int v4 __attribute__((ext_vector_type(4)));
    const int lane = threadIdx.x;
    const int n0 = blockIdx.x * RN;
    const int8_t* wp[4];
#pragma unroll
    for (int r = 0; r < 4; r++) wp[r] = a.w[r / RN] + (size_t)min(n0 + r % RN, a.N - 1) * a.ldw[r / RN];
    int sum[4][M] = {};
    v4 w[2][U][4], x[2][U][M];
    const auto load = [&](int b, int k0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int k = k0 + u * 1024 + lane * 16;
            const bool in = k < a.K;             // past the end: zeros for weights, anything for tokens
#pragma unroll
            for (int r = 0; r < 4; r++) w[b][u][r] = in ? __builtin_nontemporal_load(reinterpret_cast<const v4*>(wp[r] + (uint32_t)k)) : v4{0, 0, 0, 0};
#pragma unroll
            for (int m = 0; m < M; m++) x[b][u][m] = in ? *reinterpret_cast<const v4*>(a.x + (size_t)m * a.ldx + (uint32_t)k) : v4{0, 0, 0, 0};
        }
    };
    const auto dots = [&](int b) {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int m = 0; m < M; m++)
#pragma unroll
                    for (int r = 0; r < 4; r++) sum[r][m] = __builtin_amdgcn_sdot4(w[b][u][r][e], x[b][u][m][e], sum[r][m], false);
    };
    load(0, 0);
    int k = 0;
    for (; k + 2 * U * 1024 < a.K; k += 2 * U * 1024) {
        load(1, k + U * 1024);
        dots(0);
        load(0, k + 2 * U * 1024);
        dots(1);
    }
    if (k + U * 1024 < a.K) {
        load(1, k + U * 1024);
        dots(0);
        dots(1);
    } else {
        dots(0);
    }
    int g = 0, up = 0;                           // lane m RN + c: token m, channel c
#pragma unroll
    for (int m = 0; m < M; m++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int v = wave_sum(sum[r][m]);
            if (r < RN) g = lane == m * RN + r ? v : g;
            else up = lane == m * RN + r - RN ? v : up;
        }
    const int m = lane / RN, n = n0 + lane % RN;
    if (m >= M || n >= a.N) return;
    const float y = finish<NW>(g, up, a.sx[m], a.sw[0][n], NW == 2 ? a.sw[1][n] : 0.f, a.act);
    const size_t o = (size_t)m * a.ldo + n;
    if (a.type == kF32) static_cast<float*>(a.out)[o] = y;
    else if (a.type == kBF16) static_cast<bf16*>(a.out)[o] = (bf16)y;
    else static_cast<f16*>(a.out)[o] = (f16)y;
}

template <int M>
hipError_t launch_dot(const Linear8& a, hipStream_t st) {
    if (a.act < 0) hipLaunchKernelGGL((linear8_dot_k<M, 1>), dim3((unsigned)((a.N + 3) / 4)), dim3(64), 0, st, a);
    else hipLaunchKernelGGL((linear8_dot_k<M, 2>), dim3((unsigned)((a.N + 1) / 2)), dim3(64), 0, st, a);
    return hipGetLastError();
}

// Forms: the tiles' sizes, workgroups a CU holds, and what a step and a tile's beginning and end take (us).
struct Shape {
    int bm, bn, per_cu;
    double step, ends;
};
constexpr int kDotForm = 5, kDotMaxM = 8;
constexpr Shape kShapes[kDotForm] = {{256, 256, 1, 0.85, 8}, {128, 256, 1, 0.5, 5}, {128, 128, 2, 0.35, 4}, {64, 128, 2, 0.25, 3}, {32, 256, 2, 0.3, 3}};

}  // namespace

Linear8Plan linear8_plan(int M, int N, int K, int weights, int cus) {
    Linear8Plan p{kDotForm, 0, 1, 0};
    if (M <= kDotMaxM) return p;
    // An estimate of each form's time (us) with each number of splits.
    double best = 1e30;
    const int steps = (K + 127) / 128;
    for (int f = 0; f < kDotForm; f++) {
        const Shape& s = kShapes[f];
        const int tiles = ((M + s.bm - 1) / s.bm) * ((N + s.bn / weights - 1) / (s.bn / weights));
        for (int sp = 1; sp <= 16 && sp <= steps; sp++) {
            const int groups = tiles * sp, slots = cus * s.per_cu;
            const double rounds = (groups + slots - 1) / slots, share = groups < slots ? (double)groups / cus : s.per_cu;
            const double step = fmax(s.step * fmax(1., share), 0.) ;
            const double bytes = (double)tiles * sp * s.bm * s.bn * 4;
            const double t = rounds * ((double)((steps + sp - 1) / sp) * step + s.ends) + (sp > 1 ? 3 + 2 * bytes / 4e6 : 0);
            if (t < best) best = t, p = Linear8Plan{f, tiles, sp, sp > 1 ? (size_t)bytes : 0};
        }
    }
    return p;
}

hipError_t launch_linear8(const Linear8& a, const Linear8Plan& p, void* part, hipStream_t st) {
    const bool one = a.act < 0;
    switch (p.form) {
        case 0: return one ? launch_tile<T256x256, 1>(a, p, part, st) : launch_tile<T256x256, 2>(a, p, part, st);
        case 1: return one ? launch_tile<T128x256, 1>(a, p, part, st) : launch_tile<T128x256, 2>(a, p, part, st);
        case 2: return one ? launch_tile<T128x128, 1>(a, p, part, st) : launch_tile<T128x128, 2>(a, p, part, st);
        case 3: return one ? launch_tile<T64x128, 1>(a, p, part, st) : launch_tile<T64x128, 2>(a, p, part, st);
        case 4: return one ? launch_tile<T32x256, 1>(a, p, part, st) : launch_tile<T32x256, 2>(a, p, part, st);
    }
    switch (a.M) {
        case 1: return launch_dot<1>(a, st);
        case 2: return launch_dot<2>(a, st);
        case 3: return launch_dot<3>(a, st);
        case 4: return launch_dot<4>(a, st);
        case 5: return launch_dot<5>(a, st);
        case 6: return launch_dot<6>(a, st);
        case 7: return launch_dot<7>(a, st);
        default: return launch_dot<8>(a, st);
    }
}

}  // namespace rt4
