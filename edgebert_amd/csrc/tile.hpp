// tile.hpp -- the product tiles of the gated feed-forward block (gated.hip):
// C(m, n) = sum over k of A(m, k) B(n, k), bf16 or fp32 operands, fp32 sums,
// each operand with its k contiguous (rows of activations, weights as stored)
// or strided (the transposed operands of gradients), and what becomes of a
// tile while it is still in registers.
#pragma once
#include "gemm16.hpp"
#include "layer.hpp"

namespace ebh {

// What is done with a tile.
enum Use : int {
    USE_STORE = 0,    // C = sum + bias, in T
    USE_PARTIAL = 1,  // one of several sums over ranges of k, fp32
    USE_GATE = 2,     // h = act(g) u, and g | u where they are kept
    USE_SLOPES = 3    // dg | du from dh, g and u, and their column sums
};

struct TileArgs {
    const void* A;
    const void* B;
    int lda, ldb;         // elements between rows in memory: of m and n, or of k where k is strided
    int M, N, K;          // USE_GATE: N = I, and B has 2 N rows
    int splits, kt_split; // ranges of k, of kt_split k-tiles (even) each
    void* C;
    int ldc;
    const float* bias;
    void* h;              // USE_GATE: [M, I]
    void* gu;             // USE_GATE: written if not null; USE_SLOPES: read, [M, 2 I]
    void* dgu;            // USE_SLOPES: [M, 2 I]
    float* colsum;        // USE_SLOPES: [blocks of rows][2 I], or null
    int I, act;
};

// ---------------------------------------------------------------------------
// Activations and their derivatives, on the hardware's exp2 and reciprocal (as
// fast_exp and gelu_tanh_fast in kernels.hpp): a few units of fp32's last place,
// far below a bf16 rounding and as good as the fp32 sums they are applied to.
// ---------------------------------------------------------------------------
__device__ __forceinline__ float logistic(float x) { return __builtin_amdgcn_rcpf(1.0f + fast_exp(-x)); }

// Within 30 of 0, where every activation and slope has long reached its limit; NaN stays NaN.
__device__ __forceinline__ float within_30(float g) { return g > 30.0f ? 30.0f : (g < -30.0f ? -30.0f : g); }

// The normal distribution function by formula 7.1.26 of Abramowitz and Stegun
// (erf to 1.5e-7, here 0.75e-7, little over fp32's own half step at 1):
// erfc(x) = e^(-x^2) (a1 t + .. + a5 t^5), t = 1 / (1 + p x), x = |g| / sqrt 2.
// No branches, no difference of near numbers for g < 0, and the exponential is
// the one the derivative needs: e = e^(-g^2 / 2).
__device__ __forceinline__ float normal_cdf(float g, float& e) {
    const float m = fabsf(within_30(g));          // e^(-450) is 0
    e = fast_exp(-0.5f * m * m);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f * 0.70710678118654752f, m, 1.0f));
    const float poly = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
    const float tail = 0.5f * poly * e;
    return g > 0.0f ? 1.0f - tail : tail;
}

template <int ACT>
__device__ __forceinline__ float act_of(float g) {
    if constexpr (ACT == 0) return g * logistic(g);
    else if constexpr (ACT == 1) return gelu_tanh_fast(g);
    else {
        float e;
        return g * normal_cdf(g, e);
    }
}

// a = act(g), d = act'(g).
template <int ACT>
__device__ __forceinline__ void act_and_slope(float g, float& a, float& d) {
    if constexpr (ACT == 0) {
        // 1 - s as the logistic function of -g: no difference of near numbers
        const float s = logistic(g);
        a = g * s;
        d = fmaf(a, logistic(-g), s);
    } else if constexpr (ACT == 1) {
        // g s(2 u): s + g s(2 u) s(-2 u) 2 u'.  Past |g| = 30 one of the two is 0,
        // and g^2 could pass the range
        const float c = within_30(g);
        const float u2 = 2.0f * 0.7978845608f * c * fmaf(0.044715f * c, c, 1.0f);
        const float du2 = 2.0f * 0.7978845608f * fmaf(3.0f * 0.044715f * c, c, 1.0f);
        const float s = logistic(u2);
        a = g * s;
        d = fmaf(c * s * logistic(-u2), du2, s);
    } else {
        float e;
        const float p = normal_cdf(g, e);
        a = g * p;
        d = fmaf(within_30(g), 0.3989422804014327f * e, p);
    }
}

// V values; act is uniform.
template <int V>
__device__ __forceinline__ void act_times(int act, const float* g, const float* u, float* h) {
    if (act == 0) {
#pragma unroll
        for (int e = 0; e < V; ++e) h[e] = act_of<0>(g[e]) * u[e];
    } else if (act == 1) {
#pragma unroll
        for (int e = 0; e < V; ++e) h[e] = act_of<1>(g[e]) * u[e];
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) h[e] = act_of<2>(g[e]) * u[e];
    }
}

// g, u -> dg, du of dh.
template <int V>
__device__ __forceinline__ void act_grads(int act, const float* dh, float* g, float* u) {
    auto each = [&](auto act_c) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            float a, d;
            act_and_slope<decltype(act_c)::value>(g[e], a, d);
            g[e] = dh[e] * u[e] * d;
            u[e] = dh[e] * a;
        }
    };
    if (act == 0) each(std::integral_constant<int, 0>{});
    else if (act == 1) each(std::integral_constant<int, 1>{});
    else each(std::integral_constant<int, 2>{});
}

// ---------------------------------------------------------------------------
// A tile's operands.  A k-tile is 128 bytes of k (64 bf16, 32 fp32) of BM rows of
// A and BN of B, in LDS as it comes from memory, in 16-byte chunks that direct
// loads put where the fragment reads find them without bank conflicts:
//  - k contiguous: rows of 8 chunks, chunk c of row r at c ^ chunk_swizzle16(r);
//    a lane's operand is one 16-byte read;
//  - k strided: rows of k, in units of 16 columns (32 bytes of bf16, 64 of
//    fp32), unit b of row k at b ^ f(k).  bf16 operands come from
//    ds_read_b64_tr_b16 (attention.hip has its lane layout): a 16-lane group q
//    reads rows 8 q + 0 .. 3, then + 4 .. 7, 32 bytes each, so the 8 rows that a
//    half-wave reads fall in 8 different units of the 256 bytes of all banks
//    with f(k) = (k & 3) + 4 ((k >> 3) & 1).  fp32 operands are four reads of a
//    word, at rows 4 q + e: f(k) = (k >> 2) & 3.
// Lane (r, q) = (lane % 16, lane / 16) of a fragment holds row r of 16 and, of a
// slice of half a k-tile, bf16 k = 8 q .. 8 q + 7, fp32 k = 4 q .. 4 q + 3 (one
// for each of four v_mfma_f32_16x16x4_f32).
// ---------------------------------------------------------------------------
constexpr uint32_t TILE_OUT = 0xFFFFFFE0u;    // an offset past every operand's k-tile
constexpr uint32_t TILE_NONE = 0x80000000u;   // past every output's rows in a tile, and block steps above it too

template <class T, bool STRIDED, int ROWS, int NT>
struct TileLoader {
    static constexpr int ES = sizeof(T), KT = 128 / ES, CE = 16 / ES;
    static constexpr int L = ROWS * 8 / NT;          // loads per thread and k-tile
    static constexpr int CPR = STRIDED ? ROWS * ES / 16 : 8;   // chunks per row in LDS
    static constexpr int CU = ES;                    // chunks per unit of 16 columns
    static constexpr int RPL = NT / CPR;             // rows a pass of loads covers
    static_assert(L * NT == ROWS * 8 && RPL >= 1 && (STRIDED || RPL % 32 == 0) && NT % CPR == 0, "passes of whole rows");

    static __device__ __forceinline__ int f(int k) {
        return ES == 2 ? (k & 3) + 4 * ((k >> 3) & 1) : (k >> 2) & 3;
    }

    uint32_t ldb;         // bytes between rows
    uint32_t voff[L];     // this thread's chunks, from the k-tile's start
    int chunk;            // k contiguous: the chunk's place in k
    uint64_t base;        // of the next k-tile to load
    int64_t size;         // k contiguous: bytes from there to the panel's end
    int left;             // k from there to the end
    int cols;             // k strided: columns from the panel's first to the operand's last

    // rows_of(r): the row of the operand's panel that goes to row r in LDS.
    template <class F>
    __device__ __forceinline__ void init(int64_t ld, int tid, F&& row_of) {
        ldb = (uint32_t)(ld * ES);
        chunk = 0;
#pragma unroll
        for (int i = 0; i < L; ++i) {
            const int r = tid / CPR + i * RPL, slot = tid % CPR;
            if constexpr (STRIDED) {
                voff[i] = (uint32_t)r * ldb + 16 * (slot ^ (CU * f(r)));
            } else {
                chunk = slot ^ chunk_swizzle16<8>(r);     // the same for all: passes are multiples of 16 rows
                voff[i] = (uint32_t)row_of(r) * ldb + 16 * chunk;
            }
        }
    }
    // A panel: rows (k contiguous) or columns (k strided) r0 .. of `rows`, from k0 of K on.
    __device__ __forceinline__ void at(const void* p, int64_t ld, int64_t r0, int64_t rows, int64_t k0, int64_t K) {
        left = (int)(K - k0);
        if constexpr (STRIDED) {
            base = uniform_u64(static_cast<const char*>(p) + (k0 * ld + r0) * ES);
            cols = (int)(rows - r0);
        } else {
            base = uniform_u64(static_cast<const char*>(p) + (r0 * ld + k0) * ES);
            size = ((rows - r0 - 1) * ld + K - k0) * ES;
            const int64_t most = 0xFFFF0000;              // offsets within a tile stay below it
            if (size > most) size = most;
        }
    }
    // The next k-tile into LDS at `lds` (this wave's part of the stage).
    __device__ __forceinline__ void issue(uint32_t lds) {
        uint32_t bytes;
        if constexpr (STRIDED) bytes = left > 0 ? (uint32_t)(min(left, KT) - 1) * ldb + (uint32_t)cols * ES : 0u;
        else bytes = left > 0 && size > 0 ? (uint32_t)size : 0u;
        const g16_v4i rsrc = {(int)(uint32_t)base, (int)((uint32_t)(base >> 32) & 0xffffu), __builtin_amdgcn_readfirstlane((int)bytes),
                              G16_RSRC_WORD3};
        // k ends inside this k-tile: what lies behind it in a row is not zeros
        const bool cut = !STRIDED && left < KT;
        const bool out = cut && chunk * CE >= left;
#pragma unroll
        for (int i = 0; i < L; ++i) load_lds16_buf(rsrc, out ? TILE_OUT : voff[i], 0, lds + i * NT * 16);
        left -= KT;
        if constexpr (STRIDED) {
            base += (uint64_t)KT * ldb;
        } else {
            base += 128;
            size -= 128;
        }
    }
};

template <class T, bool STRIDED, int ROWS>
struct TileReader {
    static constexpr int ES = sizeof(T), RB = ROWS * ES;
    uint32_t off;         // this lane's place
    __device__ __forceinline__ void init(int lane) {
        const int r = lane & 15, q = lane >> 4;
        if constexpr (!STRIDED) off = r * 128 + 16 * (q ^ chunk_swizzle16<8>(r));
        else if constexpr (ES == 2) off = (8 * q + (r >> 2)) * RB + 32 * ((r >> 2) + 4 * (q & 1)) + 8 * (r & 3);
        else off = 4 * q * RB + 64 * q + 4 * r;
    }
    // The operand of block b (16 rows or columns) and slice s, `st` the stage's LDS address.
    __device__ __forceinline__ g16_v4f read(const char* st, int b, int s) const {
        if constexpr (!STRIDED) {
            return *reinterpret_cast<const g16_v4f*>(st + (off ^ (64 * s)) + b * 2048);
        } else if constexpr (ES == 2) {
            typedef short v4s __attribute__((ext_vector_type(4)));
            typedef short v8s __attribute__((ext_vector_type(8)));
            const char* p = st + (off ^ (32 * b)) + s * 32 * RB;
            const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)p);
            const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)(p + 4 * RB));
            return __builtin_bit_cast(g16_v4f, v8s{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
        } else {
            const char* p = st + (off ^ (64 * b)) + s * 16 * RB;
            return g16_v4f{*reinterpret_cast<const float*>(p), *reinterpret_cast<const float*>(p + RB),
                           *reinterpret_cast<const float*>(p + 2 * RB), *reinterpret_cast<const float*>(p + 3 * RB)};
        }
    }
};

// Two neighbouring blocks' accumulators (lane (r, q): columns 4 q .. 4 q + 3 of
// row r) as eight consecutive columns: the second and fourth 16 lanes of the
// one change places with the first and third of the other.  Lane (r, q) then has
// columns 16 (q % 2) + 8 (q / 2) .. + 7 of the 32.
__device__ __forceinline__ void eight_columns(const g16_v4f& a, const g16_v4f& b, float* v) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(a[e]), __float_as_uint(b[e]), false, false);
        v[e] = __uint_as_float(s[0]);
        v[4 + e] = __uint_as_float(s[1]);
    }
}
__device__ __forceinline__ u4v_t pack8(const float* v) {
    return u4v_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
}
__device__ __forceinline__ void unpack8(const u4v_t& w, float* v) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[2 * e] = __uint_as_float(w[e] << 16);
        v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    }
}

// A persistent grid walks the work items (C tiles, N-fastest, times the ranges of
// k).  The k-tiles of a workgroup's items are one stream: the next one's loads
// are in flight while a tile is finished.  A k-tile's last MFMAs run after the
// next one's barrier (two sets of B fragments, so k-tiles come in pairs; one
// past the end of k is zeros).
template <class T, bool AKS, bool BKS, int BM, int BN, int WAVES_M, int WAVES_N, int NS, int USE>
__device__ __forceinline__ void tile_body(const TileArgs& p, char* const smem) {
    constexpr int NW = WAVES_M * WAVES_N, NT = 64 * NW, ES = sizeof(T), KT = 128 / ES;
    constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N, FM = WM / 16, FN = WN / 16;
    static_assert(FM * 16 == WM && WN == 64 && FN == 4, "waves of 64 columns");
    constexpr int SB = FM >= 8 ? 2 : 1, STEPS = FM / SB;
    static_assert(STEPS % 2 == 0, "steps alternate between two A sets");
    constexpr bool WIDE = ES == 2 && USE != USE_PARTIAL;   // eight bf16 columns a lane, else four fp32 ones
    constexpr int G = WIDE ? 2 : 4;                        // groups of columns a lane has in 64
    constexpr int BNC = USE == USE_GATE ? BN / 2 : BN;     // columns of C in a tile
    constexpr int ST_A = BM * 128, ST_B = BN * 128, B_OFF = NS * ST_A;
    constexpr int NLD = (BM + BN) * 8 / NT;                // loads per thread and k-tile
    constexpr int NSTO = FM * G / (USE == USE_GATE ? 2 : 1);   // stores per thread and tile, at least

    const int ntn = (p.N + BNC - 1) / BNC, ntiles = ((p.M + BM - 1) / BM) * ntn, nwork = ntiles * p.splits, nk = p.kt_split;
    // Workgroup b runs on XCD b % 8; each XCD's workgroups take consecutive items,
    // which share operand panels in that XCD's L2.
    const int grid = gridDim.x;
    int u0 = blockIdx.x, ustep = grid, uend = nwork;
    if ((grid & 7) == 0 && nwork % grid == 0) {
        u0 = (blockIdx.x & 7) * (grid >> 3) + (blockIdx.x >> 3);
    } else if ((grid & 7) == 0) {
        const int x = blockIdx.x & 7;
        ustep = grid >> 3;
        u0 = (int)((int64_t)x * nwork / 8) + (blockIdx.x >> 3);
        uend = (int)((int64_t)(x + 1) * nwork / 8);
    }
    const int my_tiles = u0 < uend ? (uend - u0 + ustep - 1) / ustep : 0;
    if (my_tiles == 0) return;   // uniform over the workgroup

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WAVES_N, wn = wave % WAVES_N;
    const uint32_t lds0 = (uint32_t)(uintptr_t)smem + (uint32_t)wave * 1024;

    TileLoader<T, AKS, BM, NT> la;
    TileLoader<T, BKS, BN, NT> lb;
    la.init(p.lda, tid, [](int r) { return r; });
    // USE_GATE: each wave's 64 columns are 32 of the gate's and the same 32 of the other's
    lb.init(p.ldb, tid, [&](int r) { return USE == USE_GATE ? (r >> 6) * 32 + (r & 31) + (r & 32 ? p.N : 0) : r; });
    int lt = 0, lkt = 0, li = 0;   // the stream's next k-tile: its item, its place in it, its number
    auto item = [&](int t, int& m0, int& n0, int& split) __attribute__((always_inline)) {
        const int u = u0 + t * ustep;
        split = u / ntiles;
        const int tile = u - split * ntiles, mt = tile / ntn;
        m0 = mt * BM;
        n0 = (tile - mt * ntn) * BNC;
    };
    auto cursors = [&](int t) __attribute__((always_inline)) {
        int m0, n0, split;
        item(t, m0, n0, split);
        const int64_t k0 = (int64_t)split * nk * KT;
        la.at(p.A, p.lda, m0, AKS ? p.M : min(p.M, m0 + BM), k0, p.K);
        lb.at(p.B, p.ldb, n0, USE == USE_GATE ? 2 * (int64_t)p.N : (BKS ? p.N : min(p.N, n0 + BN)), k0, p.K);
    };
    auto issue = [&]() __attribute__((always_inline)) {
        if (lt >= my_tiles) return;
        const uint32_t st = li % NS;
        la.issue(lds0 + st * ST_A);
        lb.issue(lds0 + B_OFF + st * ST_B);
        ++li;
        if (++lkt == nk) {
            lkt = 0;
            if (++lt < my_tiles) cursors(lt);
        }
    };

    TileReader<T, AKS, BM> ra;
    TileReader<T, BKS, BN> rb;
    ra.init(lane);
    rb.init(lane);
    g16_v4f acc[FM][FN], af[2][SB][2], bf[2][FN][2];
    int it = 0;
    // The stream's k-tile `it` is in LDS, and everyone is done with the one before.
    // Issued behind its loads: at most those of the k-tiles between, and a tile's stores.
    auto enter = [&](bool stores) __attribute__((always_inline)) {
        constexpr auto c = [](int v) { return v > 63 ? 63 : v; };
        const int ahead = li - it - 1;             // k-tiles in flight behind it
        if constexpr (NS > 2) {
            if (ahead >= NS - 2) {
                if (stores) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(c((NS - 2) * NLD + NSTO)) : "memory");
                else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(c((NS - 2) * NLD)) : "memory");
            } else if (stores) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(c(NSTO)) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        } else {
            if (stores) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(c(NSTO)) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        lds_barrier();
    };
    auto mfma_step = [&](int s, int as, int bs) __attribute__((always_inline)) {
#pragma unroll
        for (int sl = 0; sl < 2; ++sl)
#pragma unroll
            for (int e = 0; e < (ES == 2 ? 1 : 4); ++e)
#pragma unroll
                for (int i = 0; i < SB; ++i)
#pragma unroll
                    for (int j = 0; j < FN; ++j) {
                        g16_v4f& d = acc[s * SB + i][j];
                        if constexpr (ES == 2)
                            d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(g16_v8bf, bf[bs][j][sl]),
                                                                        __builtin_bit_cast(g16_v8bf, af[as][i][sl]), d, 0, 0, 0);
                        else
                            d = __builtin_amdgcn_mfma_f32_16x16x4f32(bf[bs][j][sl][e], af[as][i][sl][e], d, 0, 0, 0);
                    }
    };
    auto run_ktile = [&](auto set, bool first) __attribute__((always_inline)) {
        constexpr int P = decltype(set)::value;
        const char *sa = smem + (it % NS) * ST_A, *sb = smem + B_OFF + (it % NS) * ST_B;
        auto rd_a = [&](int s) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < SB; ++i)
#pragma unroll
                for (int sl = 0; sl < 2; ++sl) af[s & 1][i][sl] = ra.read(sa, wm * FM + s * SB + i, sl);
        };
        rd_a(0);
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int sl = 0; sl < 2; ++sl) bf[P][j][sl] = rb.read(sb, wn * FN + j, sl);
        if (!first) mfma_step(STEPS - 1, 1, P ^ 1);   // the previous k-tile's last step
#pragma unroll
        for (int s = 0; s + 1 < STEPS; ++s) {
            if (s == 0) issue();
            rd_a(s + 1);
            mfma_step(s, s & 1, P);
        }
        ++it;
    };

    auto finish = [&](int t) __attribute__((always_inline)) {
        int m0, n0, split;
        item(t, m0, n0, split);
        const int wrow = m0 + wm * WM;
        int el = lane;
        asm volatile("" : "+v"(el));   // formed here, not held across the k-loop
        const int r = el & 15, q = el >> 4;
        // Block pair or block g of the wave's columns: this lane's first column of C
        auto col = [&](int g) __attribute__((always_inline)) {
            return n0 + (USE == USE_GATE ? wn * 32 : wn * WN) + (WIDE ? 32 * g + 16 * (q & 1) + 8 * (q >> 1) : 16 * g + 4 * q);
        };
        constexpr int V = WIDE ? 8 : 4;
        auto values = [&](int i, int g, float* v) __attribute__((always_inline)) {
            if constexpr (WIDE) {
                eight_columns(acc[i][2 * g], acc[i][2 * g + 1], v);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = acc[i][g][e];
            }
        };
        // The wave's rows of a matrix, and a lane's place in block i's (less than 2^31
        // from the first: TILE_NONE is past every row's)
        auto rows = [&](const void* base, int64_t ld, int es) __attribute__((always_inline)) {
            const int left = __builtin_amdgcn_readfirstlane(min(p.M - wrow, WM));
            return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(static_cast<const char*>(base) + (int64_t)wrow * ld * es),
                                                     (short)0, (left > 0 ? left : 0) * (int)(ld * es), G16_RSRC_WORD3);
        };
        auto put = [&](const __amdgpu_buffer_rsrc_t& d, uint32_t off, const float* v) __attribute__((always_inline)) {
            if constexpr (WIDE) __builtin_amdgcn_raw_buffer_store_b128(pack8(v), d, off, 0, 0);
            else
                __builtin_amdgcn_raw_buffer_store_b128(
                    u4v_t{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])}, d, off, 0, 0);
        };
        auto unpack = [&](const u4v_t& w, float* v) __attribute__((always_inline)) {
            if constexpr (WIDE) {
                unpack8(w, v);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(w[e]);
            }
        };
        constexpr int OS = USE == USE_PARTIAL ? 4 : ES;      // bytes of a stored element
        if constexpr (USE == USE_STORE || USE == USE_PARTIAL) {
            char* const c = static_cast<char*>(p.C) + (USE == USE_PARTIAL ? (int64_t)split * p.M * p.ldc * 4 : 0);
            float b[G][V];
            uint32_t off[G];
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const int n = col(g);
                off[g] = n < p.N ? (uint32_t)(r * p.ldc * OS + n * OS) : TILE_NONE;
#pragma unroll
                for (int e = 0; e < V; ++e) b[g][e] = USE == USE_STORE && p.bias && n < p.N ? p.bias[n + e] : 0.0f;
            }
            const auto d = rows(c, p.ldc, OS);
            int step = 16 * p.ldc * OS;
            asm volatile("" : "+s"(step));   // its multiples are formed here, not held
#pragma unroll
            for (int i = 0; i < FM; ++i) {
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    float v[V];
                    values(i, g, v);
#pragma unroll
                    for (int e = 0; e < V; ++e) v[e] += b[g][e];
                    put(d, off[g] + i * step, v);
                }
            }
        } else {
            {
                const int64_t I = p.I;
                int row_h = p.I * ES;
                asm volatile("" : "+s"(row_h));   // its multiples are formed here, not held
                const int row_gu = 2 * row_h;
                if constexpr (USE == USE_GATE) {
                    const auto dh = rows(p.h, I, ES), dgu = rows(p.gu, 2 * I, ES);
#pragma unroll
                    for (int g = 0; g < G / 2; ++g) {
                        const int n = col(g);
                        const bool in = n < p.N;
                        float bg[V], bu[V];
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            bg[e] = p.bias && in ? p.bias[n + e] : 0.0f;
                            bu[e] = p.bias && in ? p.bias[I + n + e] : 0.0f;
                        }
                        uint32_t oh = in ? (uint32_t)(r * row_h + n * ES) : TILE_NONE;
                        uint32_t og = in ? (uint32_t)(r * row_gu + n * ES) : TILE_NONE;
#pragma unroll
                        for (int i = 0; i < FM; ++i) {
                            float gv[V], uv[V], hv[V];
                            values(i, g, gv);
                            values(i, G / 2 + g, uv);
#pragma unroll
                            for (int e = 0; e < V; ++e) {
                                gv[e] += bg[e];
                                uv[e] += bu[e];
                            }
                            act_times<V>(p.act, gv, uv, hv);
                            put(dh, oh, hv);
                            if (p.gu) {
                                put(dgu, og, gv);
                                put(dgu, og + row_h, uv);
                            }
                            oh += 16 * row_h;
                            og += 16 * row_gu;
                        }
                    }
                } else {
                    const auto src = rows(p.gu, 2 * I, ES), dst = rows(p.dgu, 2 * I, ES);
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const int n = col(g);
                        uint32_t og = n < p.N ? (uint32_t)(r * row_gu + n * ES) : TILE_NONE;
                        float cg[V] = {}, cu[V] = {};
                        u4v_t raw[2][2];           // g and u of this block of rows and the next
                        auto load = [&](int set, uint32_t at) __attribute__((always_inline)) {
                            raw[set][0] = __builtin_amdgcn_raw_buffer_load_b128(src, at, 0, 0);
                            raw[set][1] = __builtin_amdgcn_raw_buffer_load_b128(src, at + row_h, 0, 0);
                        };
                        load(0, og);
#pragma unroll
                        for (int i = 0; i < FM; ++i) {
                            float gv[V], uv[V], dh[V];
                            if (i + 1 < FM) load((i + 1) & 1, og + 16 * row_gu);
                            unpack(raw[i & 1][0], gv);
                            unpack(raw[i & 1][1], uv);
                            values(i, g, dh);
                            act_grads<V>(p.act, dh, gv, uv);
#pragma unroll
                            for (int e = 0; e < V; ++e) {
                                cg[e] += gv[e];
                                cu[e] += uv[e];
                            }
                            put(dst, og, gv);
                            put(dst, og + row_h, uv);
                            og += 16 * row_gu;
                            __builtin_amdgcn_sched_barrier(0);   // keeps the loads one block ahead, not all at once
                        }
                        if (p.colsum) {
                            // rows past the last are zeros: dh is, of operands that are
#pragma unroll
                            for (int e = 0; e < V; ++e)
#pragma unroll
                                for (int o = 1; o < 16; o <<= 1) {
                                    cg[e] += __shfl_xor(cg[e], o);
                                    cu[e] += __shfl_xor(cu[e], o);
                                }
                            if (r == 0 && n < p.N) {
                                float* at = p.colsum + (int64_t)(m0 / BM * WAVES_M + wm) * 2 * I + n;
#pragma unroll
                                for (int e = 0; e < V; ++e) {
                                    at[e] = cg[e];
                                    at[I + e] = cu[e];
                                }
                            }
                        }
                    }
                }
            }
        }
    };

    cursors(0);
#pragma unroll
    for (int d = 0; d < NS - 1; ++d) issue();
    typedef std::integral_constant<int, 0> set0;
    typedef std::integral_constant<int, 1> set1;
    for (int t = 0; t < my_tiles; ++t) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = g16_v4f{0.0f, 0.0f, 0.0f, 0.0f};
        enter(t > 0);
        run_ktile(set0{}, true);
        enter(NS > 2 && t > 0);
        run_ktile(set1{}, false);
        for (int kt = 2; kt < nk; kt += 2) {
            enter(false);
            run_ktile(set0{}, false);
            enter(false);
            run_ktile(set1{}, false);
        }
        mfma_step(STEPS - 1, 1, 1);
        finish(t);
    }
}

constexpr int tile_lds(int bm, int bn, int ns) { return (bm + bn) * 128 * ns; }

}  // namespace ebh
