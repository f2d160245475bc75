// tile.hpp -- the product tiles of the gated feed-forward block (gated.hip):
// C(m, n) = sum over k of A(m, k) B(n, k), bf16 or fp32 operands, fp32 sums,
// each operand with its k contiguous (rows of activations, weights as stored)
// or strided (the transposed operands of gradients), and what becomes of a
// tile while it is still in registers.
#pragma once
#include "gemm16.hpp"
#include "layer.hpp"

#pragma clang diagnostic ignored "-Winline-asm"   // m0 among the clobbers, a reserved register

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

// Within L of 0; NaN stays NaN.
template <int L>
__device__ __forceinline__ float within(float g) { return g > (float)L ? (float)L : (g < -(float)L ? -(float)L : g); }

// The normal distribution function by formula 7.1.26 of Abramowitz and Stegun
// (erf to 1.5e-7, here 0.75e-7, little over fp32's own half step at 1):
// erfc(x) = e^(-x^2) (a1 t + .. + a5 t^5), t = 1 / (1 + p x), x = |g| / sqrt 2.
// No branches, no difference of near numbers for g < 0, and the exponential is
// the one the derivative needs: e = e^(-g^2 / 2).
__device__ __forceinline__ float normal_cdf(float g, float& e) {
    const float m = fabsf(within<30>(g));          // e^(-450) is 0
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
    // x s(v) with s the logistic function: s = 1 / (1 + e), 1 - s = e s with e =
    // e^(-v), no difference of near numbers.  v is held where e is finite; s has
    // long reached its limit there, and g^2 stays in range.
    if constexpr (ACT == 0) {
        const float e = fast_exp(-within<80>(g));
        const float s = __builtin_amdgcn_rcpf(1.0f + e);
        a = g * s;
        d = fmaf(a, e * s, s);
    } else if constexpr (ACT == 1) {
        const float c = within<10>(g), c2 = c * c;     // v = 2 u = 87 at 10
        const float k = 2.0f * 0.7978845608f;
        const float e = fast_exp(-(c * fmaf(k * 0.044715f, c2, k)));
        const float s = __builtin_amdgcn_rcpf(1.0f + e);
        a = g * s;
        d = fmaf(c * s * (e * s), fmaf(3.0f * k * 0.044715f, c2, k), s);
    } else {
        float e;
        const float p = normal_cdf(g, e);
        a = g * p;
        d = fmaf(within<30>(g), 0.3989422804014327f * e, p);
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
// A tile's operands.  A k-tile is KB = 128 bytes of k (64 bf16, 32 fp32) of BM
// rows of A and BN of B, in LDS as it comes from memory, in 16-byte chunks that direct
// loads put where the fragment reads find them without bank conflicts:
//  - k contiguous: rows of 8 chunks, chunk c of row r at c ^ (r & 7); a lane's operand
//    is one 16-byte read.  LDS serves those of lanes 0-3, 12-15, 20-23 and 24-27 (and
//    the likes of them) at a time, here from 16 different places in the 256 bytes of
//    all banks: 4 clocks a read (counted), where c ^ (r & 7) ^ ((r >> 3) & 1) takes 8;
//  - k strided: rows of k, in units of 16 columns (32 bytes of bf16, 64 of
//    fp32), unit b of row k at b ^ f(k).  bf16 operands come from
//    ds_read_b64_tr_b16 (attention.hip has its lane layout): a 16-lane group q
//    reads rows 8 q + 0 .. 3, then + 4 .. 7, 32 bytes each, so the 8 rows that a
//    half-wave reads fall in 8 different units of the 256 bytes of all banks
//    with f(k) = (k & 3) + 4 ((k >> 3) & 1).  fp32 operands are four reads of a
//    word, at rows 4 q + e: f(k) = (k >> 2) & 3.
// Lane (r, q) = (lane % 16, lane / 16) of a fragment holds row r of 16 and, of a
// slice of 64 bytes of k, bf16 k = 8 q .. 8 q + 7, fp32 k = 4 q .. 4 q + 3 (one
// for each of four v_mfma_f32_16x16x4_f32).
// ---------------------------------------------------------------------------
constexpr uint32_t TILE_OUT = 0xFFFFFFE0u;    // an offset past every operand's k-tile
constexpr uint32_t TILE_NONE = 0x80000000u;   // past every output's rows in a tile, and block steps above it too

// Columns of a row of k in LDS: 192 bf16 are a row and a half of all banks, and take two.
template <bool STRIDED, int ROWS>
constexpr int tile_pitch() { return STRIDED && ROWS == 192 ? 256 : ROWS; }

template <class T, bool STRIDED, int ROWS, int KB, int NT>
struct TileLoader {
    static constexpr int ES = sizeof(T), KT = KB / ES, CE = 16 / ES, PITCH = tile_pitch<STRIDED, ROWS>();
    static constexpr int L = PITCH * (KB / 16) / NT;   // loads per thread and k-tile
    static constexpr int CPR = STRIDED ? PITCH * ES / 16 : KB / 16;   // chunks per row in LDS
    static constexpr int CU = ES;                    // chunks per unit of 16 columns
    static constexpr int RPL = NT / CPR;             // rows a pass of loads covers
    static_assert(L * NT == PITCH * (KB / 16) && RPL >= 1 && (STRIDED || RPL % 32 == 0) && NT % CPR == 0, "passes of whole rows");

    static __device__ __forceinline__ int f(int k) {
        return ES == 2 ? (k & 3) + 4 * ((k >> 3) & 1) : (k >> 2) & 3;
    }

    uint32_t ldb;         // bytes between rows
    // A pass's chunks lie RPL rows behind the one's before; strided, the swizzle has them
    // in another place where RPL is not its period (16 rows of k in bf16, fp32 too).
    static constexpr int BASES = !STRIDED || RPL % 16 == 0 ? 1 : 16 / RPL;
    static_assert(BASES <= L, "passes");
    uint32_t voff[BASES]; // this thread's chunks, from the k-tile's start
    uint32_t other;       // the gate's tile: bytes from the gate's rows to the other projection's
    int chunk;            // k contiguous: the chunk's place in k
    uint64_t base;        // of the next k-tile to load
    uint32_t size;        // k contiguous: bytes from there to the panel's end
    int left;             // k from there to the end
    uint32_t last;        // k strided: bytes of a row from the panel's first column to the operand's last

    // HALF > 0: every other HALF rows in LDS are the other projection's, `second` rows on.
    template <int HALF = 0>
    __device__ __forceinline__ void init(int64_t ld, int tid, int second = 0) {
        static_assert(HALF == 0 || (!STRIDED && (RPL == HALF || RPL % (2 * HALF) == 0)), "whole passes");
        ldb = (uint32_t)(ld * ES);
        other = (uint32_t)second * ldb;
        chunk = 0;
#pragma unroll
        for (int i = 0; i < BASES; ++i) {
            const int r = tid / CPR + i * RPL, slot = tid % CPR;
            if constexpr (STRIDED) {
                const int c = slot ^ (CU * f(r));
                voff[i] = c < ROWS / CE ? (uint32_t)r * ldb + 16 * c : TILE_NONE;
            } else {
                chunk = slot ^ (r & 7);                   // the same for all: passes are multiples of 16 rows
                const int row = HALF > 0 ? r / (2 * HALF) * HALF + r % HALF : r;
                voff[i] = (uint32_t)row * ldb + 16 * chunk + (HALF > 0 && r % (2 * HALF) >= HALF ? other : 0u);
            }
        }
    }
    // A panel: rows (k contiguous) or columns (k strided) r0 .. of `rows`, from k0 of K on.
    __device__ __forceinline__ void at(const void* p, int64_t ld, int64_t r0, int64_t rows, int64_t k0, int64_t K) {
        left = (int)(K - k0);
        if constexpr (STRIDED) {
            base = uniform_u64(static_cast<const char*>(p) + (k0 * ld + r0) * ES);
            last = (uint32_t)(rows - r0) * ES;
        } else {
            base = uniform_u64(static_cast<const char*>(p) + (r0 * ld + k0) * ES);
            size = left > 0 ? (uint32_t)((rows - r0 - 1) * ld + left) * ES : 0u;   // less than 2^32: layer_ops.cpp
        }
    }
    // The next k-tile's loads, into LDS at `lds` (this wave's part of the stage).
    template <int HALF = 0>
    __device__ __forceinline__ void load(uint32_t lds) const {
        uint32_t bytes;
        if constexpr (STRIDED) bytes = left > 0 ? (uint32_t)(min(left, KT) - 1) * ldb + last : 0u;
        else bytes = left > 0 ? size : 0u;
        const g16_v4i rsrc = {(int)(uint32_t)base, (int)((uint32_t)(base >> 32) & 0xffffu), (int)bytes, G16_RSRC_WORD3};
        // k ends inside this k-tile: what lies behind it in a row is not zeros
        const uint32_t out = !STRIDED && left < KT && chunk * CE >= left ? TILE_OUT : 0u;
        uint32_t v[BASES], row = ldb;
        asm volatile("" : "+s"(row));              // multiples are formed here, one after the other
#pragma unroll
        for (int i = 0; i < BASES; ++i) v[i] = voff[i];
#pragma unroll
        for (int i = 0; i < L; ++i) {
            uint32_t at = v[i % BASES];
            if constexpr (HALF > 0 && RPL < 2 * HALF) {
                // RPL rows on in LDS: the other projection's, or the gate's next ones
                static_assert(RPL == HALF, "a pass is one projection's");
                if (i & 1) {
                    at += other;
                    v[0] += HALF * row;
                }
            } else {
                v[i % BASES] += (HALF > 0 ? RPL / 2 : BASES * RPL) * row;
            }
            asm volatile(
                "s_add_u32 m0, %2, %3\n\t"
                "s_nop 0\n\t"
                "buffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(STRIDED ? at : at | out), "s"(rsrc), "s"(lds), "n"(i * NT * 16)
                : "memory", "m0", "scc");
        }
    }
    __device__ __forceinline__ void advance() {
        left -= KT;
        if constexpr (STRIDED) {
            base += (uint64_t)KT * ldb;
        } else {
            base += KB;
            size -= KB;
        }
    }
};

template <class T, bool STRIDED, int ROWS, int KB>
struct TileReader {
    static constexpr int ES = sizeof(T), RB = tile_pitch<STRIDED, ROWS>() * ES;
    uint32_t off;         // this lane's place
    __device__ __forceinline__ void init(int lane) {
        const int r = lane & 15, q = lane >> 4;
        if constexpr (!STRIDED) off = r * KB + 16 * (q ^ (r & 7));
        else if constexpr (ES == 2) off = (8 * q + (r >> 2)) * RB + 32 * ((r >> 2) + 4 * (q & 1)) + 8 * (r & 3);
        else off = 4 * q * RB + 64 * q + 4 * r;
    }
    // Strided: the blocks' places are formed anew in each k-tile, not held
    __device__ __forceinline__ void renew() {
        if constexpr (STRIDED) asm volatile("" : "+v"(off));
    }
    // The operand of block b (16 rows or columns) and slice s, `st` the stage's LDS address.
    __device__ __forceinline__ g16_v4f read(const char* st, int b, int s) const {
        if constexpr (!STRIDED) {
            return *reinterpret_cast<const g16_v4f*>(st + (off ^ (64 * s)) + b * 16 * KB);
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

// Two neighbouring blocks of a row, a lane's columns 4 q .. 4 q + 3 of each, as they
// lie in memory.  bf16: 16 bytes a lane, columns 16 (q % 2) + 8 (q / 2) .. + 7 of the
// 32: of the packed words, the second and fourth 16 lanes of the one block change
// places with the first and third of the other.
__device__ __forceinline__ u4v_t swap_blocks(const u4v_t& w) {
    const auto s = __builtin_amdgcn_permlane16_swap(w[0], w[2], false, false);
    const auto t = __builtin_amdgcn_permlane16_swap(w[1], w[3], false, false);
    return u4v_t{s[0], t[0], s[1], t[1]};
}
__device__ __forceinline__ u4v_t words(const float* v) {
    return u4v_t{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
}
// ES: bytes of an element in memory; o: the lane's places (of both blocks, where they
// are two).  AUX 2: non-temporal.
template <int ES, int AUX = 0>
__device__ __forceinline__ void put_blocks(const __amdgpu_buffer_rsrc_t& d, const uint32_t* o, uint32_t add, const float* a, const float* b) {
    if constexpr (ES == 2) {
        const u4v_t w = swap_blocks(u4v_t{pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]), pack_bf16x2(b[0], b[1]), pack_bf16x2(b[2], b[3])});
        __builtin_amdgcn_raw_buffer_store_b128(w, d, o[0] + add, 0, AUX);
    } else {
        __builtin_amdgcn_raw_buffer_store_b128(words(a), d, o[0] + add, 0, AUX);
        __builtin_amdgcn_raw_buffer_store_b128(words(b), d, o[1] + add, 0, AUX);
    }
}
template <int ES>
struct RawBlocks {
    u4v_t w[ES / 2];
    __device__ __forceinline__ void load(const __amdgpu_buffer_rsrc_t& d, const uint32_t* o, uint32_t add) {
#pragma unroll
        for (int k = 0; k < ES / 2; ++k) w[k] = __builtin_amdgcn_raw_buffer_load_b128(d, o[k] + add, 0, 0);
    }
    __device__ __forceinline__ void values(float* a, float* b) const {
        if constexpr (ES == 2) {
            const u4v_t v = swap_blocks(w[0]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                a[2 * e] = __uint_as_float(v[e] << 16);
                a[2 * e + 1] = __uint_as_float(v[e] & 0xffff0000u);
                b[2 * e] = __uint_as_float(v[2 + e] << 16);
                b[2 * e + 1] = __uint_as_float(v[2 + e] & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                a[e] = __uint_as_float(w[0][e]);
                b[e] = __uint_as_float(w[ES / 2 - 1][e]);
            }
        }
    }
};

// A persistent grid walks the work items (C tiles, N-fastest, times the ranges of
// k).  The k-tiles of a workgroup's items are one stream: the next one's loads
// are in flight while a tile is finished.  A k-tile's last MFMAs run after the
// next one's barrier (two sets of B fragments, so k-tiles come in pairs; one
// past the end of k is zeros).
template <class T, bool AKS, bool BKS, int BM, int BN, int WAVES_M, int WAVES_N, int KB, int NS, int USE>
__device__ __forceinline__ void tile_body(const TileArgs& p, char* const smem) {
    constexpr int NW = WAVES_M * WAVES_N, NT = 64 * NW, ES = sizeof(T), KT = KB / ES, SL = KB / 64;
    constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N, FM = WM / 16, FN = WN / 16;
    static_assert(FM * 16 == WM && FN * 16 == WN && FN % (USE == USE_GATE ? 4 : 2) == 0, "pairs of blocks");
    constexpr int SB = FM >= 8 ? 2 : 1, STEPS = FM / SB;
    static_assert(STEPS % 2 == 0, "steps alternate between two A sets");
    static_assert(NT == 256 || (NT == 512 && NS == 2), "turns of loading go with the two stages");
    constexpr int OS = USE == USE_PARTIAL ? 4 : ES;        // bytes of a stored element
    constexpr int FC = USE == USE_GATE ? FN / 2 : FN;      // blocks of a wave's columns of C
    constexpr int BNC = USE == USE_GATE ? BN / 2 : BN;     // columns of C in a tile
    constexpr int ST_A = BM * KB, ST_B = tile_pitch<BKS, BN>() * KB, B_OFF = NS * ST_A;
    constexpr int NLD = (ST_A + ST_B) / 16 / NT;                // loads per thread and k-tile
    constexpr int NSTO = FM * FC * OS / 4;                 // stores per thread and tile, at least

    const int ntn = (p.N + BNC - 1) / BNC, ntiles = ((p.M + BM - 1) / BM) * ntn, nwork = ntiles * (USE == USE_PARTIAL ? p.splits : 1), nk = p.kt_split;
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

    // Eight waves load by turns, one k-tile the first four and one the others (mfma_step).
    constexpr int LT = NT == 512 ? 256 : NT, HALF = USE == USE_GATE ? WN / 2 : 0;
    const uint32_t lds0 = (uint32_t)(uintptr_t)smem + (uint32_t)(wave % (LT / 64)) * 1024;
    TileLoader<T, AKS, BM, KB, LT> la;
    TileLoader<T, BKS, BN, KB, LT> lb;
    la.init(p.lda, tid % LT);
    // USE_GATE: half of each wave's columns are the gate's, the others the same ones of the other projection
    lb.template init<HALF>(p.ldb, tid % LT, p.N);
    int lt = 0, lkt = 0, li = 0;   // the stream's next k-tile: its item, its place in it, its number
    int ls = 0, its = 0;           // of three stages and more: its one, and that of the one being multiplied
    auto item = [&](int t, int& m0, int& n0, int& split) __attribute__((always_inline)) {
        int across = ntn, all = ntiles;
        asm volatile("" : "+s"(across), "+s"(all));   // their reciprocals are formed here, not held across the k-loop
        const int u = u0 + t * ustep;
        split = USE == USE_PARTIAL ? u / all : 0;
        const int tile = u - split * all, mt = tile / across;
        m0 = mt * BM;
        n0 = (tile - mt * across) * BNC;
    };
    typedef const __attribute__((address_space(4))) TileArgs* Args;
    auto cursors = [&](int t) __attribute__((always_inline)) {
        int m0, n0, split;
        item(t, m0, n0, split);
        const int64_t k0 = (int64_t)split * nk * KT;
        // The arguments (the kernel's only one, at its arguments' start) come from memory
        // anew, here and in finish(): held across the k-loop they would spill scalar
        // registers.
        Args ep = (Args)__builtin_amdgcn_kernarg_segment_ptr();
        asm volatile("" : "+s"(ep));
        const int M = ep->M, N = ep->N, K = ep->K, lda = ep->lda, ldb = ep->ldb;
        la.at(ep->A, lda, m0, AKS ? M : min(M, m0 + BM), k0, K);
        lb.at(ep->B, ldb, n0, USE == USE_GATE ? 2 * (int64_t)N : (BKS ? N : min(N, n0 + BN)), k0, K);
    };
    // The next k-tile's loads of A and of B, into the stage of its number, even or odd
    // (k-tiles come in pairs), or the next of three and more.
    auto load_a = [&](int par) __attribute__((always_inline)) {
        if (lt < my_tiles) la.load(lds0 + (uint32_t)(NS == 2 ? par : ls) * ST_A);
    };
    auto load_b = [&](int par) __attribute__((always_inline)) {
        if (lt < my_tiles) lb.template load<HALF>(lds0 + B_OFF + (uint32_t)(NS == 2 ? par : ls) * ST_B);
    };
    auto next = [&]() __attribute__((always_inline)) {
        if (lt >= my_tiles) return;
        la.advance();
        lb.advance();
        ++li;
        ls = ls + 1 == NS ? 0 : ls + 1;
        if (++lkt == nk) {
            lkt = 0;
            if (++lt < my_tiles) cursors(lt);
        }
    };

    TileReader<T, AKS, BM, KB> ra;
    TileReader<T, BKS, BN, KB> rb;
    ra.init(lane);
    rb.init(lane);
    g16_v4f acc[FM][FN], af[2][SB][SL], bf[2][FN][SL];
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
    // One step's MFMAs.  A load holds up its wave until the CU's address unit takes
    // it, 16 clocks for each: half of a k-tile's MFMA time for all of its loads.  So
    // of the two waves of a SIMD one loads, for both, while the other has the matrix
    // core (32,768 rows, 768 x 2,048: 326 -> 321 us forward, 696 -> 685 back, over
    // every wave's own loads one by one between its MFMAs); two workgroups of four
    // waves a CU do so of themselves, with A's and B's loads in one go each, after the
    // first FN MFMAs (`slot`) and the second.
    auto mfma_step = [&](int s, int as, int bs, int slot, int par) __attribute__((always_inline)) {
#pragma unroll
        for (int sl = 0; sl < SL; ++sl)
#pragma unroll
            for (int i = 0; i < SB; ++i) {
#pragma unroll
                for (int e = 0; e < (ES == 2 ? 1 : 4); ++e)
#pragma unroll
                    for (int j = 0; j < FN; ++j) {
                        g16_v4f& d = acc[s * SB + i][j];
                        if constexpr (ES == 2)
                            d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(g16_v8bf, bf[bs][j][sl]),
                                                                        __builtin_bit_cast(g16_v8bf, af[as][i][sl]), d, 0, 0, 0);
                        else
                            d = __builtin_amdgcn_mfma_f32_16x16x4f32(bf[bs][j][sl][e], af[as][i][sl][e], d, 0, 0, 0);
                    }
                if (NT == 256 && (slot == 0 || slot == 1)) {
                    __builtin_amdgcn_sched_barrier(0);
                    slot ? load_b(par) : load_a(par);
                    __builtin_amdgcn_sched_barrier(0);
                }
                ++slot;
            }
    };
    auto run_ktile = [&](auto set, bool first) __attribute__((always_inline)) {
        constexpr int P = decltype(set)::value;
        const int st = NS == 2 ? P : its;
        const char *sa = smem + st * ST_A, *sb = smem + B_OFF + st * ST_B;
        auto rd_a = [&](int s) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < SB; ++i)
#pragma unroll
                for (int sl = 0; sl < SL; ++sl) af[s & 1][i][sl] = ra.read(sa, wm * FM + s * SB + i, sl);
        };
        ra.renew();
        rb.renew();
        rd_a(0);
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int sl = 0; sl < SL; ++sl) bf[P][j][sl] = rb.read(sb, wn * FN + j, sl);
        __builtin_amdgcn_sched_barrier(0);            // reads stay ahead of the MFMAs that hide them
        constexpr int par = NS == 2 ? P ^ 1 : 0;
        if (NT == 512 && (wave >> 2) == P) {
            load_a(par);
            load_b(par);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (!first) mfma_step(STEPS - 1, 1, P ^ 1, 0, par);   // the previous k-tile's last step
        else if (NT == 256) {
            load_a(par);
            load_b(par);
        }
#pragma unroll
        for (int s = 0; s + 1 < STEPS; ++s) {
            rd_a(s + 1);
            __builtin_amdgcn_sched_barrier(0);
            mfma_step(s, s & 1, P, 2, par);
            __builtin_amdgcn_sched_barrier(0);
        }
        next();
        ++it;
        its = its + 1 == NS ? 0 : its + 1;
    };

    auto finish = [&](int t) __attribute__((always_inline)) {
        int m0, n0, split;
        item(t, m0, n0, split);
        Args ep = (Args)__builtin_amdgcn_kernarg_segment_ptr();
        asm volatile("" : "+s"(ep));
        const float* const biases = ep->bias;
        const int M = ep->M, N = ep->N, I = ep->I, act = ep->act;
        const int wrow = m0 + wm * WM;
        int el = lane;
        asm volatile("" : "+v"(el));   // formed here, not held across the k-loop
        const int r = el & 15, q = el >> 4;
        const int cbase = n0 + wn * FC * 16;          // the wave's first column of C
        auto col = [&](int j) __attribute__((always_inline)) { return cbase + 16 * j + 4 * q; };   // the lane's of block j
        // The lane's places of blocks 2 jp and 2 jp + 1 in its row r, rows `bytes` apart
        // (N is a multiple of 8: 8 or 4 columns are in or out together)
        auto places = [&](int jp, int bytes, uint32_t* o) __attribute__((always_inline)) {
            const int w = cbase + 32 * jp + 16 * (q & 1) + 8 * (q >> 1);
            if constexpr (OS == 2) {
                o[0] = w < N ? (uint32_t)(r * bytes + w * 2) : TILE_NONE;
            } else {
#pragma unroll
                for (int b = 0; b < 2; ++b) o[b] = col(2 * jp + b) < N ? (uint32_t)(r * bytes + col(2 * jp + b) * 4) : TILE_NONE;
            }
        };
        // The wave's rows of a matrix; a lane's places in them are less than 2^31 from
        // the first, and TILE_NONE is past them
        auto rows = [&](const void* base, int bytes) __attribute__((always_inline)) {
            const int left = __builtin_amdgcn_readfirstlane(min(M - wrow, WM));
            return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(static_cast<const char*>(base) + (int64_t)wrow * bytes),
                                                     (short)0, (left > 0 ? left : 0) * bytes, G16_RSRC_WORD3);
        };
        auto bias = [&](int j, const float* from, float* v) __attribute__((always_inline)) {
            const bool in = from && col(j) < N;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = in ? from[col(j) + e] : 0.0f;
        };
        // Rows outermost: a row's neighbouring pairs are stored one after the other, whole lines.
        if constexpr (USE == USE_STORE || USE == USE_PARTIAL) {
            int bytes = ep->ldc * OS;
            asm volatile("" : "+s"(bytes));   // its multiples are formed here, not held
            const auto d = rows(static_cast<char*>(ep->C) + (USE == USE_PARTIAL ? (int64_t)split * M * bytes : 0), bytes);
            float bv[FN][4];
            uint32_t o[FN / 2][2];
#pragma unroll
            for (int j = 0; j < FN; ++j)
                if (USE == USE_STORE) bias(j, biases, bv[j]);
#pragma unroll
            for (int jp = 0; jp < FN / 2; ++jp) places(jp, bytes, o[jp]);
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int jp = 0; jp < FN / 2; ++jp) {
                    float v[2][4];
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[b][e] = acc[i][2 * jp + b][e] + (USE == USE_STORE ? bv[2 * jp + b][e] : 0.0f);
                    put_blocks<OS>(d, o[jp], i * 16 * bytes, v[0], v[1]);
                }
        } else {
            void* const gu = ep->gu;
            int row_h = I * ES;
            asm volatile("" : "+s"(row_h));
            const int row_gu = 2 * row_h;
            uint32_t og[FC / 2][2];
#pragma unroll
            for (int jp = 0; jp < FC / 2; ++jp) places(jp, row_gu, og[jp]);
            if constexpr (USE == USE_GATE) {
                const auto dh = rows(ep->h, row_h), dgu = rows(gu, row_gu);
                uint32_t oh[FC / 2][2];
#pragma unroll
                for (int jp = 0; jp < FC / 2; ++jp) places(jp, row_h, oh[jp]);
                float bg[FC][4], bu[FC][4];
#pragma unroll
                for (int j = 0; j < FC; ++j) {
                    bias(j, biases, bg[j]);
                    bias(j, biases ? biases + I : nullptr, bu[j]);
                }
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int jp = 0; jp < FC / 2; ++jp) {
                        float g[2][4], u[2][4], hv[2][4];
#pragma unroll
                        for (int b = 0; b < 2; ++b)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                g[b][e] = acc[i][2 * jp + b][e] + bg[2 * jp + b][e];
                                u[b][e] = acc[i][FC + 2 * jp + b][e] + bu[2 * jp + b][e];
                            }
                        act_times<8>(act, g[0], u[0], hv[0]);
                        put_blocks<ES>(dh, oh[jp], i * 16 * row_h, hv[0], hv[1]);
                        if (gu) {   // not read before the backward pass: kept out of the caches
                            put_blocks<ES, 2>(dgu, og[jp], i * 16 * row_gu, g[0], g[1]);
                            put_blocks<ES, 2>(dgu, og[jp], i * 16 * row_gu + row_h, u[0], u[1]);
                        }
                        __builtin_amdgcn_sched_barrier(0);   // one pair's values at a time in registers
                    }
            } else {
                const auto src = rows(gu, row_gu), dst = rows(ep->dgu, row_gu);
                constexpr int PAIRS = FM * FN / 2, AHEAD = 2;   // pairs of blocks, and how many's g and u are on their way
                const bool sums = ep->colsum != nullptr;
                float cg[FN][4] = {}, cu[FN][4] = {};
                RawBlocks<ES> raw[AHEAD][2];
                // pair k, `rows16` rows of blocks on from where og has come to
                auto load = [&](int k, int rows16) __attribute__((always_inline)) {
                    raw[k % AHEAD][0].load(src, og[k % (FN / 2)], rows16 * 16 * row_gu);
                    raw[k % AHEAD][1].load(src, og[k % (FN / 2)], rows16 * 16 * row_gu + row_h);
                };
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) load(k, k / (FN / 2));
#pragma unroll
                for (int k = 0; k < PAIRS; ++k) {
                    const int i = k / (FN / 2), jp = k % (FN / 2);
                    float g[2][4], u[2][4], dh[2][4];
                    raw[k % AHEAD][0].values(g[0], g[1]);
                    raw[k % AHEAD][1].values(u[0], u[1]);
                    if (k + AHEAD < PAIRS) load(k + AHEAD, (k + AHEAD) / (FN / 2) - i);
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int e = 0; e < 4; ++e) dh[b][e] = acc[i][2 * jp + b][e];
                    act_grads<8>(act, dh[0], g[0], u[0]);
                    if (sums) {
#pragma unroll
                        for (int b = 0; b < 2; ++b)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                cg[2 * jp + b][e] += g[b][e];
                                cu[2 * jp + b][e] += u[b][e];
                            }
                    }
                    put_blocks<ES>(dst, og[jp], 0, g[0], g[1]);
                    put_blocks<ES>(dst, og[jp], row_h, u[0], u[1]);
                    og[jp][0] += 16 * row_gu;
                    og[jp][1] += 16 * row_gu;
                    __builtin_amdgcn_sched_barrier(0);   // keeps the loads so far ahead, not all of them
                }
                if (sums) {
                    asm volatile("" : "+s"(ep));
                    float* const colsum = ep->colsum;
                    // rows past the last are zeros: dh is, of operands that are
#pragma unroll
                    for (int j = 0; j < FN; ++j) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
#pragma unroll
                            for (int o = 1; o < 16; o <<= 1) {
                                cg[j][e] += __shfl_xor(cg[j][e], o);
                                cu[j][e] += __shfl_xor(cu[j][e], o);
                            }
                        if (r == 0 && col(j) < N) {
                            float* at = colsum + (int64_t)(m0 / BM * WAVES_M + wm) * 2 * I + col(j);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                at[e] = cg[j][e];
                                at[I + e] = cu[j][e];
                            }
                        }
                    }
                }
            }
        }
    };

    cursors(0);
#pragma unroll
    for (int d = 0; d < NS - 1; ++d) {
        if (NT == 256 || wave < 4) {
            load_a(d);
            load_b(d);
        }
        next();
    }
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
#pragma unroll 1
        for (int kt = 2; kt < nk; kt += 2) {
            enter(false);
            run_ktile(set0{}, false);
            enter(false);
            run_ktile(set1{}, false);
        }
        mfma_step(STEPS - 1, 1, 1, 2, 0);
        finish(t);
    }
}

template <bool BKS, int BM, int BN, int KB, int NS>
constexpr int tile_lds() { return (BM + tile_pitch<BKS, BN>()) * KB * NS; }

}  // namespace ebh
