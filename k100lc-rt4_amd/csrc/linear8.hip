// linear8.hip -- products of int8 codes with a scale for each token and each channel, and the first half of
// a gated feed-forward block on them.
//
//   c[m][n] = sx[m] sw[n] Σ_k xq[m][k] wq[n][k]                     (exact int32 sums, K < 2^17)
//   h[m][n] = act(sx[m] sg[n] Σ_k xq[m][k] wg[n][k]) * (sx[m] su[n] Σ_k xq[m][k] wu[n][k])
//
// What bounds it, and where it stands:
//   up to 8 tokens   the weights' stream; 2 x 17408 x 5120 of one token 30.4 us, 5.9 TB/s; 5120 x 5120 7.6 us for a stream of 5.5:
//                    the launch, the first loads' latency, and a second round, since 266 registers leave one wave a SIMD and
//                    1280 waves do not fit the 1024 SIMDs
//   9 to 400 tokens  latency: a workgroup's steps, of 0.25 us, one after the other, where tiles are fewer than the CUs; 37 tokens
//                    of 4999 x 7056, 79 workgroups of 56 steps, 15.9 us with the weights in the last-level cache and 24 from
//                    memory, for a floor of 7.5; 100 tokens of 5120 x 17408 35 us for 19 (a launch that joins runs of split K: 7.8)
//   many tokens      the matrix cores, at the clock that power leaves them (1.7 to 1.8 GHz, busy 57 to 62% of the cycles): 4096
//                    tokens of 17408 x 5120 329 to 352 us by card, 2.1 to 2.2 Pop/s; 1000 of 2 x 17408 x 5120 178 to 193 us,
//                    1.85 to 2.0; 1024 of 5120 x 17408 95 us, 1.9 (a library's int8 product of 8192^3: 2.07)
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
// channels (8 (i >> 2) + 4 (lane >> 5) + (i & 3)).  With two weight matrices (NW) a fragment is 16 gate rows and the up rows
// of the same 16 channels, so both factors of an output meet in one lane, as registers i and i + 8.
//
// Steps are 128 codes deep: whole cache lines of a row.  Operands arrive by DMA (8 rows x 128 bytes an instruction) in a
// ring of ST stages; in a stage, chunk c (16 bytes) of row r lies at slot c ^ (r >> 1 & 7), which puts the 16 rows that one
// cycle of a read serves into 16 different bank groups.  One barrier a step, before its last quarter: by then every wave
// has read the stage for the last time, and the DMA of the step ST further on goes into it from there on.
template <int TM_, int TN_, int WM_, int WN_, int ST_, int PER_CU_>
struct Tile {
    static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, ST = ST_, W = WM * WN, PER_CU = PER_CU_;
    static constexpr int BM = 32 * TM * WM, BN = 32 * TN * WN, STAGE = (BM + BN) * 128;
    static constexpr int SLAB = 32 * (TN * 32 * 4 + 16) + TN * 128;       // a wave's share of LDS for fp32 outputs and scales
    static constexpr int LDS = ST * STAGE > W * SLAB ? ST * STAGE : W * SLAB;
    static constexpr int PA = BM / 8 / W, PB = BN / 8 / W, P = PA + PB;   // DMA instructions of a wave a step
    static_assert(BM % (8 * W) == 0 && BN % (8 * W) == 0 && (ST - 2) * P < 64, "");
    static_assert(LDS * PER_CU <= 160 * 1024 && W == 4, "");
};

struct Where {                           // a workgroup's tile and steps
    int tile, part, m0, n0, s0, s1;
};

template <class C, int NW>
__device__ __forceinline__ Where where(const Linear8& a, int splits, int b, int blocks) {
    const int nm = (a.M + C::BM - 1) / C::BM, nn = (a.N + C::BN / NW - 1) / (C::BN / NW);
    // Workgroups go round the XCDs: each takes a run of the list, in which tiles that share operands are neighbours: columns of GM
    // tiles, one beside the other (4096 tokens of 17408 x 5120: GM 4 340 to 345 us, 1 355 to 359, 2 349, 8 343; 2000 tokens 180,
    // 188 to 194, 184, 183).
    const int x = b & 7, per = blocks >> 3, rem = blocks & 7, t = x * per + min(x, rem) + (b >> 3);
    Where w;
    w.part = t % splits;
    w.tile = t / splits;
    constexpr int GM = 4;
    const int first = w.tile / (GM * nn) * GM, rows = min(GM, nm - first), in = w.tile - first * nn;
    w.m0 = (first + in % rows) * C::BM;
    w.n0 = in / rows * (C::BN / NW);
    const int steps = (a.K + 127) >> 7;
    w.s0 = steps * w.part / splits;
    w.s1 = steps * (w.part + 1) / splits;
    // The divisions above are done on the vector ALU.  Everything that goes by them is made scalar here, once: a base address
    // that v_readfirstlane writes needs five wait states before a load reads it, and before those in inline assembly the
    // compiler puts none.
    return Where{uniform(w.tile), uniform(w.part), uniform(w.m0), uniform(w.n0), uniform(w.s0), uniform(w.s1)};
}

// 32 tokens of a wave's TN fragments from their sums: through the wave's own LDS, out in 16-byte pieces of rows.
template <int NW, class T, int TN>
__device__ __forceinline__ void write_slab(const Linear8& a, const v16i* acc, const float* scales, int m0, int n0, unsigned char* lds) {
    constexpr int COLS = TN * 32 / NW, PITCH = COLS * (int)sizeof(T) + 16, PER = 16 / (int)sizeof(T), LPR = COLS / PER;
    const int lane = threadIdx.x & 63, ml = lane & 31, hi = lane >> 5;
    const float sx = a.sx[min(m0 + ml, a.M - 1)];
#pragma unroll
    for (int q = 0; q < COLS / 8; q++) {         // 8 channels: registers 4 (q % per) .. of fragment q / per
        constexpr int per = 4 / NW;
        const v16i& f = acc[q / per];
        float s[NW][4];
#pragma unroll
        for (int j = 0; j < NW; j++) __builtin_memcpy(s[j], scales + j * COLS + 8 * q + 4 * hi, 16);
        T t[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int r = 4 * (q % per) + e;
            t[e] = (T)finish<NW>(f[r], NW == 1 ? 0 : f[r + 8], sx, s[0][e], s[NW - 1][e], a.act);
        }
        __builtin_memcpy(lds + ml * PITCH + (8 * q + 4 * hi) * sizeof(T), t, sizeof(t));
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    static_assert(32 * LPR % 64 == 0, "");
#pragma unroll
    for (int k = 0; k < 32 * LPR / 64; k++) {
        const int id = lane + 64 * k, r = id / LPR, col = id % LPR * PER, m = m0 + r, n = n0 + col;
        const uint4 d = *reinterpret_cast<const uint4*>(lds + r * PITCH + col * sizeof(T));
        if (m < a.M && n < a.N) {
            T* o = static_cast<T*>(a.out) + (size_t)m * a.ldo + n;
            if (n + PER <= a.N) {                // (global memory takes 16 bytes at any alignment)
                __builtin_memcpy(o, &d, 16);
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

// All outputs of a wave, whose share of LDS holds its channels' scales behind the slab.
template <class C, int NW, int ROWS>
__device__ __forceinline__ void write_wave(const Linear8& a, const v16i (&acc)[ROWS][C::TN], int m0, int n0, unsigned char* lds) {
    constexpr int COLS = C::TN * 32 / NW;
    float* scales = reinterpret_cast<float*>(lds + C::SLAB - C::TN * 128);
    for (int i = threadIdx.x & 63; i < C::TN * 32; i += 64) scales[i] = a.sw[NW == 1 ? 0 : i / COLS][min(n0 + i % COLS, a.N - 1)];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const auto all = [&](auto t) {
#pragma unroll
        for (int i = 0; i < ROWS; i++) write_slab<NW, decltype(t), C::TN>(a, acc[i], scales, m0 + 32 * i, n0, lds);
    };
    if (a.type == kF32) all(float{});
    else if (a.type == kBF16) all(bf16{});
    else all(f16{});
}

template <int N>
__device__ __forceinline__ void wait_dma_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// A DMA in two parts: where its rows go (M0, which the compiler leaves alone; one wait state until its use), and the load,
// whose immediate offset is added to both addresses.
__device__ __forceinline__ void set_m0(uint32_t l) { asm volatile("s_mov_b32 m0, %0\n\ts_nop 0" ::"s"((uint32_t)__builtin_amdgcn_readfirstlane((int)l)) : "memory"); }
template <int IMM>
__device__ __forceinline__ void dma16_m0(uint32_t voff, const void* gbase) {
    asm volatile("global_load_lds_dwordx4 %0, %1 offset:%2" ::"v"(voff), "s"(sptr(gbase)), "n"(IMM) : "memory");
}

// part null: whole tiles; else this workgroup's sums (of one of `splits` runs of steps), a fragment's registers as they are.
template <class C, int NW>
__global__ __launch_bounds__(64 * C::W, 1) void linear8_tile_k(Linear8 a, int splits, int4* part) {
    constexpr int TM = C::TM, TN = C::TN, ST = C::ST, PA = C::PA, P = C::P, FR = TM + TN, MF = TM * TN, HALF = P / 2;
    __shared__ __align__(16) unsigned char smem[C::LDS];
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
    const auto mat = [&](int t) { return NW == 1 ? 0 : (pb0 + t - PA) >> 1 & 1; };    // whose rows a weight piece is: see above
#pragma unroll
    for (int t = 0; t < P; t++) {
        const int c = chunk(t);
        if (t < PA) {
            voff[t] = (uint32_t)min((pa0 + t) * 8 + (lane >> 3), a.M - 1 - at.m0) * (uint32_t)a.ldx + c * 16 + (3 - t % 4) * 1024;
        } else {
            const int b = pb0 + t - PA, r = (NW == 1 ? b : (b >> 2) * 2 + (b & 1)) * 8 + (lane >> 3);   // channel in the tile
            voff[t] = (uint32_t)min(r, a.N - 1 - at.n0) * (uint32_t)(mat(t) ? a.ldw[1] : a.ldw[0]) + c * 16 + (3 - (t - PA) % 4) * 1024;
        }
    }
    const size_t k0 = (size_t)at.s0 * 128;
    // An instruction's immediate offset counts for both addresses: pieces 1 KB apart in LDS need M0 set for every fourth
    // alone.  In memory it is taken out again: voff holds 3 KB less it, the bases 3 KB less.
    const int8_t* ga = a.x + (size_t)at.m0 * a.ldx + k0 - 3 * 1024;
    const int8_t* gb[NW];
#pragma unroll
    for (int j = 0; j < NW; j++) gb[j] = a.w[j] + (size_t)at.n0 * a.ldw[j] + k0 - 3 * 1024;
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
        const int u = t < PA ? t : t - PA;
        if (u % 4 == 0 || t == HALF) set_m0((t < PA ? la : lb) + in + u / 4 * 4096);
        const int8_t* g = t < PA ? ga : gb[NW == 1 ? 0 : mat(t)];
        switch (u % 4) {
            case 0: dma16_m0<0>(voff[t], g); break;
            case 1: dma16_m0<1 * 1024>(voff[t], g); break;
            case 2: dma16_m0<2 * 1024>(voff[t], g); break;
            default: dma16_m0<3 * 1024>(voff[t], g);
        }
    };
    const auto issued = [&]() {
        issue++;
        ga += 128;
#pragma unroll
        for (int j = 0; j < NW; j++) gb[j] += 128;
        in = next(in);
    };
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
    // Pieces of step s + ST are brought behind the barrier of step s and in the first quarter of the next.
    // M1: there is a step s + ST - 1; M2: there is a step s + ST.
    const auto step = [&](int s, auto m1, auto m2) {
        constexpr bool M1 = decltype(m1)::value, M2 = decltype(m2)::value;
#define RT4_C(x) std::integral_constant<int, (x)>{}
        quarter(RT4_C(0), RT4_C(HALF), RT4_C(M1 ? P : HALF), true);
        if (M1) issued();
        quarter(RT4_C(1), RT4_C(0), RT4_C(0), true);
        quarter(RT4_C(2), RT4_C(0), RT4_C(0), true);
        out = next(out);
        if (M1) wait_dma_barrier<(ST - 2) * P>();
        else wait_dma_barrier<0>();
        if (whole && s + 2 == steps && s + 1 < at.s1) clear_tail();
        if (M2) begin_issue();
        quarter(RT4_C(3), RT4_C(0), RT4_C(M2 ? HALF : 0), M1 || s + 1 < at.s1);
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
    if (at.s1 - at.s0 >= ST - 1) wait_dma_barrier<(ST - 2) * P>();
    else wait_dma_barrier<0>();
    if (whole && at.s0 == steps - 1) clear_tail();
#pragma unroll
    for (int f = 0; f < FR; f++) read(0, f);
    if (issue < at.s1) {
        begin_issue();
#pragma unroll
        for (int t = 0; t < HALF; t++) dma_piece(t);
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
    write_wave<C, NW, TM>(a, acc, at.m0 + wm * TM * 32, at.n0 + wn * (TN * 32 / NW), smem + (size_t)w * C::SLAB);
}

// Sums the runs of split tiles: a wave takes 32 tokens of a tile's wave.
template <class C, int NW>
__global__ __launch_bounds__(256) void linear8_join_k(Linear8 a, int splits, const int4* part, int waves) {
    constexpr int TM = C::TM, TN = C::TN;
    __shared__ __align__(16) unsigned char smem[4 * C::SLAB];
    const int lane = threadIdx.x & 63, id = uniform((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
    if (id >= waves) return;                     // whole waves; no barrier follows
    const int i = id % TM, w = id / TM % C::W, tile = id / (TM * C::W);
    const int nm = (a.M + C::BM - 1) / C::BM, nn = (a.N + C::BN / NW - 1) / (C::BN / NW);
    constexpr int GM = 4;
    const int first = tile / (GM * nn) * GM, rows = min(GM, nm - first), in = tile - first * nn;
    const int m0 = (first + in % rows) * C::BM + (w / C::WN * TM + i) * 32, n0 = in / rows * (C::BN / NW) + w % C::WN * (TN * 32 / NW);
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
    write_wave<C, NW, 1>(a, acc, m0, n0, smem + (threadIdx.x >> 6) * C::SLAB);
}

// Forms, by number: tiles whose counts fill rounds of workgroups for as many sizes as possible.
#define RT4_TILES(F)                                                                                                              \
    F(0, 4, 4, 2, 2, 2, 1) F(1, 2, 7, 4, 1, 2, 1) F(2, 2, 5, 4, 1, 3, 1) F(3, 2, 4, 2, 2, 3, 1) F(4, 1, 7, 4, 1, 3, 1)            \
    F(5, 1, 5, 4, 1, 4, 1) F(6, 2, 2, 2, 2, 2, 2) F(7, 1, 2, 2, 2, 3, 2) F(8, 1, 1, 2, 2, 4, 2)
template <class C, int NW>
hipError_t launch_tile(const Linear8& a, const Linear8Part& p, void* part, hipStream_t st) {
    auto k = linear8_tile_k<C, NW>;
    hipLaunchKernelGGL(k, dim3((unsigned)(p.tiles * p.splits)), dim3(64 * C::W), 0, st, a, p.splits, p.splits > 1 ? static_cast<int4*>(part) : nullptr);
    if (p.splits == 1) return hipGetLastError();
    auto j = linear8_join_k<C, NW>;
    const int waves = p.tiles * C::W * C::TM;
    hipLaunchKernelGGL(j, dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, st, a, p.splits, static_cast<const int4*>(part), waves);
    return hipGetLastError();
}

// ---- Few tokens: dot products on the vector ALU, the weights streamed once.  A wave owns 4 weight rows (4 channels, or gate
// and up rows of 2) and goes through them 1 KB of each at a time, a lane 16 codes of each row, with the codes of every token
// beside them: each token's 16 bytes serve 4 rows.  The next loads are under way while 4 M v_dot4 an operand are done.  A
// workgroup is one wave, so that they spread evenly over the CUs.
// U, the KB of each row at a time (1 token of 5120 x 5120, of 17408 x 5120, 4 tokens of the latter, 8 tokens, from memory): as it is
// 7.7, 17.6, 19.6, 25.2 us; 2 for one token 6.3, 15.5; 1 everywhere 6.4, 15.3, 18.4, 25.4; 2 for 5 to 8 tokens 33.6.
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

// 8 tokens by dot products and by tiles: 5120 x 5120 10.3 and 12.6 us, 17408 x 5120 25.2 and 25.3, 5120 x 17408 24.3 and 25.0, 2 x
// 2500 x 2560 8.1 and 9.2; but 2 x 17408 x 5120 42.6 and 38.5 (6 tokens 37.3 and 38.1).
constexpr int kDotMaxM = 8;
constexpr long long kMaxGroups = 1 << 24;        // workgroups of 256 threads in a grid
// A form's tile, workgroups a CU holds, and its measured cost (us): a step where few workgroups run, what is added to that
// where all do (power, the L2's rate), a tile's beginning and end; and the rate at which it streams weights (TB/s), which bounds
// few tokens.  Fitted to 1045 times of 54 sizes (M 16..4000, N 1000..17408, K 1024..17408, one and two weight matrices, every
// form, 1 to 4 splits); the form they choose takes 2% longer than the best one of each of these sizes.  On 24 sizes that the fit
// has not seen (M 14..2475, N 532..16714, K 1360..15776) it takes 8.5% longer on average, over 10% at 8 of them and 45% at worst
// (170 tokens of 2 x 4543 x 12912: 79 us, the best form 55).
struct Shape {
    int bm, bn, per_cu;
    double step, full, ends, rate;
};
constexpr double kCost[][4] = {{1.294, 0.406, 4.932, 4.5}, {0.875, 0.456, 19.139, 4.5}, {0.505, 0.46, 12.229, 4.5}, {0.688, 0.211, 3.819, 4}, {0.58, 0.134, 15.555, 4.3}, {0.577, 0.115, 8.16, 5.1}, {0.766, 0.454, 0, 3.6}, {0.359, 0.47, 0.199, 3.95}, {0.208, 0.227, 1.427, 4.3}};
#define RT4_SHAPE(f, tm, tn, wm, wn, st, pc) {32 * tm * wm, 32 * tn * wn, pc, kCost[f][0], kCost[f][1], kCost[f][2], kCost[f][3]},
constexpr Shape kShapes[] = {RT4_TILES(RT4_SHAPE)};
constexpr int kDotForm = sizeof(kShapes) / sizeof(kShapes[0]);
static_assert(kDotForm == sizeof(kCost) / sizeof(kCost[0]), "");

}  // namespace

namespace {

// Form f over M x N with K split into sp runs: the estimated time, and the number of tiles.
double estimate(int f, int M, int N, int K, int weights, int cus, int sp, long long* tiles_out) {
    const Shape& s = kShapes[f];
    const long long tiles = (long long)((M + s.bm - 1) / s.bm) * ((N + s.bn / weights - 1) / (s.bn / weights)), slots = (long long)cus * s.per_cu;
    const long long groups = tiles * sp;
    const int n = ((K + 127) / 128 + sp - 1) / sp;
    const double part = (double)(groups % slots) / slots;
    double t = groups / slots * (n * (s.step + s.full) + s.ends);
    if (part > 0) t += n * (s.step + s.full * part) + s.ends;
    if (sp > 1) t += 7.8 + 0.274e-6 * 4 * groups * s.bm * s.bn;      // the runs' sums, out and in again, and the launch that joins them
    *tiles_out = tiles;
    return 2 + std::max(t, (double)N * K * weights / s.rate * 1e-6);
}

// The form and number of splits of the lowest estimate.  (A grid counts its threads in 32 bits: large tiles alone for the
// largest products.)  Up to 8 splits: 100 tokens of 1024 x 131056 57 us, with up to 4 95, up to 16 66; 16 of 1000 x 17408 13.2,
// 15.1, 14.7; 9 of 512 x 65536 24.6, 36.4, 20.4.
double choose(int M, int N, int K, int weights, int cus, Linear8Part* p) {
    double best = 1e30;
    for (int f = 0; f < kDotForm; f++)
        for (int sp = 1; sp <= 8 && sp <= (K + 127) / 128; sp++) {
            long long tiles;
            const double t = estimate(f, M, N, K, weights, cus, sp, &tiles);
            if ((sp > 1 && tiles * sp > 2ll * cus * kShapes[f].per_cu) || tiles * sp >= kMaxGroups) break;
            if (t < best) best = t, *p = Linear8Part{f, N, (int)tiles, sp};
        }
    return best;
}

}  // namespace

Linear8Plan linear8_plan(int M, int N, int K, int weights, int cus) {
    Linear8Plan p{{{kDotForm, N, 0, 1}, {}}, 1, 0};
    if (M <= kDotMaxM) return p;
    double best = choose(M, N, K, weights, cus, &p.part[0]);
    // Or whole rounds of a form's tiles over the first channels, and what is left of a last round with few tiles by the form
    // that is best for it, in a launch of its own (4096 tokens of 17408 x 5120: 1088 tiles of 256 x 256, 4.25 rounds, in one launch
    // 354 us, four rounds and the rest apart 329; 1000 tokens of 2 x 17408 x 5120 190 and 178).
    for (int f = 0; f < kDotForm; f++) {
        const Shape& s = kShapes[f];
        const int nm = (M + s.bm - 1) / s.bm, bn = s.bn / weights;
        const long long slots = (long long)cus * s.per_cu, rounds = (long long)nm * ((N + bn - 1) / bn) / slots;
        const long long first = rounds * slots / nm * bn;
        if (rounds < 1 || first >= N) continue;
        long long tiles;
        Linear8Part rest;
        const double t = estimate(f, M, (int)first, K, weights, cus, 1, &tiles) + choose(M, N - (int)first, K, weights, cus, &rest);
        if (t < best && tiles < kMaxGroups) best = t, p = Linear8Plan{{{f, (int)first, (int)tiles, 1}, rest}, 2, 0};
    }
    for (int i = 0; i < p.parts; i++) {
        const Linear8Part& q = p.part[i];
        const size_t bytes = q.splits > 1 ? (size_t)4 * q.tiles * q.splits * kShapes[q.form].bm * kShapes[q.form].bn : 0;
        p.part_bytes = bytes > p.part_bytes ? bytes : p.part_bytes;
    }
    return p;
}

void linear8_tile(int form, int* bm, int* bn) {
    const bool tile = form < kDotForm;
    *bm = tile ? kShapes[form].bm : 0;
    *bn = tile ? kShapes[form].bn : 0;
}

namespace {

hipError_t launch_part(const Linear8& a, const Linear8Part& p, void* part, hipStream_t st) {
#define RT4_LAUNCH(f, ...) \
    if (p.form == f) return a.act < 0 ? launch_tile<Tile<__VA_ARGS__>, 1>(a, p, part, st) : launch_tile<Tile<__VA_ARGS__>, 2>(a, p, part, st);
    RT4_TILES(RT4_LAUNCH)
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

}  // namespace

hipError_t launch_linear8(const Linear8& a, const Linear8Plan& p, void* part, hipStream_t st) {
    int n = 0;
    for (int i = 0; i < p.parts; i++) {
        Linear8 b = a;
        b.N = p.part[i].N;
        b.out = static_cast<char*>(a.out) + (size_t)n * (a.type == kF32 ? 4 : 2);
        for (int j = 0; j < (a.act < 0 ? 1 : 2); j++) b.w[j] = a.w[j] + (size_t)n * a.ldw[j], b.sw[j] = a.sw[j] + n;
        const hipError_t e = launch_part(b, p.part[i], part, st);
        if (e != hipSuccess) return e;
        n += p.part[i].N;
    }
    return hipSuccess;
}

}  // namespace rt4
