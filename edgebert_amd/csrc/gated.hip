// gated.hip -- the gated feed-forward block and its gradients
// (ebh_op_gated_ffn / _bwd), as products on the tiles of tile.hpp.
#include <algorithm>

#include "tile.hpp"

namespace ebh {

// ---------------------------------------------------------------------------
// The tiles, largest first.  A kernel's operand orders: both k contiguous
// (forward), B strided (through the weights back), both strided (weight
// gradients, whose k are the tokens).
//
// Bound by the matrix cores.  32,768 tokens of 768 x 2,048 in bf16, as the kernels
// run in sequence: forward 325 us (with g | u kept: 400 MB stored), backward 690 us,
// 900-950 TFLOP/s with what is done in registers, where library products of these
// shapes alone reach 956-1,041.
// ---------------------------------------------------------------------------
struct TileShape {
    int bm, bn, waves_m, waves_n, ns;
};
constexpr int TILES = 5, TILE_KB = 128;
constexpr TileShape kTiles[TILES] = {
    {256, 256, 2, 4, 2},   // 8 waves, one workgroup a CU
    {256, 192, 4, 2, 2},
    {128, 128, 2, 2, 2},   // 4 waves, two a CU
    {64, 128, 2, 2, 3},
    {64, 64, 2, 2, 3},     // fp32, where few tokens leave CUs idle: 1,061 of 384 x 1,000 back, 108 -> 95 us
};
constexpr int tile_threads(int t) { return 64 * kTiles[t].waves_m * kTiles[t].waves_n; }

template <class T, bool AKS, bool BKS, int TILE, int USE>
__global__ __launch_bounds__(tile_threads(TILE), 2) void tile_kernel(TileArgs p) {
    constexpr TileShape S = kTiles[TILE];
    __shared__ __attribute__((aligned(16))) char smem[tile_lds<BKS, S.bm, S.bn, TILE_KB, S.ns>()];
    tile_body<T, AKS, BKS, S.bm, S.bn, S.waves_m, S.waves_n, TILE_KB, S.ns, USE>(p, smem);
}

// out[part][c] = sum over the part's rows of x[., c]: 64 columns and 16 slices of
// the rows a workgroup.
template <class T>
__global__ __launch_bounds__(1024) void sum_rows_kernel(const T* x, int64_t ld, int64_t rows, int cols, float* out) {
    __shared__ float part[16][64];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), slice = threadIdx.x >> 6;
    const int64_t n = (int64_t)gridDim.y * 16, k = (int64_t)blockIdx.y * 16 + slice;
    const int64_t r0 = rows * k / n, r1 = rows * (k + 1) / n;
    float s = 0.0f;
    if (c < cols) {
#pragma unroll 8
        for (int64_t r = r0; r < r1; ++r) s += to_f32(x[r * ld + c]);
    }
    part[slice][threadIdx.x & 63] = s;
    __syncthreads();
    if (slice == 0 && c < cols) {
        s = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) s += part[i][threadIdx.x & 63];
        out[(int64_t)blockIdx.y * cols + c] = s;
    }
}

// out = the sum of `parts` partial products of n4 x 4 elements, in order, + bias;
// rows of cols4 x 4 elements, ld apart.
template <class T>
__global__ __launch_bounds__(256) void sum_parts_kernel(const float4* x, int parts, uint32_t n4, uint32_t cols4, const float* bias, T* out, int ld) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= n4) return;
    float4 s = x[i];
#pragma unroll 4
    for (int k = 1; k < parts; ++k) {
        const float4 v = x[(int64_t)k * n4 + i];
        s.x += v.x;
        s.y += v.y;
        s.z += v.z;
        s.w += v.w;
    }
    const uint32_t row = i / cols4, c = 4 * (i - row * cols4);
    if (bias) {
        s.x += bias[c];
        s.y += bias[c + 1];
        s.z += bias[c + 2];
        s.w += bias[c + 3];
    }
    T* const o = out + (int64_t)row * ld + c;
    if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(s.x, s.y), pack_bf16x2(s.z, s.w));
    else *reinterpret_cast<float4*>(o) = s;
}

static int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// ---------------------------------------------------------------------------
// The choice of a tile and of splits over k, by estimated time: with n items on
// the busiest CU, rounds of one workgroup a CU (tiles 0 and 1) or of two, us:
//   launch + full rounds * (k/64 * full + epi) + a last one of one workgroup
//   (k/64 * one + epi / 2).
// Constants fitted to a sweep on MI355X of the five products at 70 .. 32,768
// tokens of H 384 .. 1,024, I 1,000 .. 4,096 and 1 .. 24 splits (rms error 4-14%,
// fp32 1-4%; the choice takes 1.01-1.02 times the best's time on average, at worst
// 1.23).
// What they say: the largest tile runs its k fastest but needs whole rounds of
// 256; few tiles are split over k, as long as writing and reading the partial
// sums (6 TB/s, and a launch) costs less than the idle CUs.
// ---------------------------------------------------------------------------
struct TileTime {
    float launch, full, epi, one;
};
static const TileTime kTimes[2][4][TILES] = {   // bf16, fp32; by Use
    {{{0.0f, 1.302f, 6.9f, 0}, {0.0f, 1.152f, 2.7f, 0}, {0.0f, 0.815f, 6.4f, 0.800f}, {3.9f, 0.634f, 0.0f, 0.429f}},
     {{1.2f, 1.363f, 11.3f, 0}, {2.8f, 1.165f, 7.8f, 0}, {2.5f, 0.883f, 5.0f, 0.644f}, {3.7f, 0.602f, 2.2f, 0.403f}},
     {{2.1f, 1.414f, 5.6f, 0}, {}, {3.5f, 1.082f, 0.4f, 0.617f}, {2.6f, 0.893f, 0.0f, 0.610f}},
     {{0.0f, 1.282f, 20.5f, 0}, {}, {0.0f, 0.732f, 14.4f, 0.505f}, {2.1f, 0.743f, 4.7f, 0.511f}}},
    {{{}, {}, {3.9f, 7.389f, 3.8f, 3.994f}, {0.0f, 4.211f, 2.7f, 2.493f}, {0.9f, 2.124f, 4.0f, 1.393f}},
     {{}, {}, {3.6f, 7.474f, 4.4f, 4.015f}, {3.3f, 4.096f, 2.2f, 2.393f}, {3.1f, 2.112f, 1.5f, 1.360f}},
     {{}, {}, {4.2f, 7.379f, 1.6f, 3.878f}, {3.8f, 4.063f, 1.0f, 2.269f}, {}},
     {{}, {}, {1.0f, 7.367f, 16.2f, 4.052f}, {2.7f, 3.850f, 7.5f, 2.404f}, {3.3f, 2.244f, 2.3f, 1.416f}}},
};

// Whether a product can have a tile: fp32 tiles are the small ones, and bf16's strided
// operands have at least 128 columns; the gate's waves have pairs of blocks of each
// projection.
constexpr bool has_tile(int t, bool bf16, bool a_strided, int use) {
    return (bf16 ? t < 4 : t >= 2) && !(bf16 && a_strided && t == 3) && !(t == 1 && (use == USE_GATE || use == USE_SLOPES)) && !(t == 4 && use == USE_GATE);
}

struct Plan {
    int tile, splits, kt_split;
    int64_t partial;   // bytes of partial sums
};

// An M x N product over K; most: bytes of partial sums there may be.
static Plan plan_product(int64_t M, int64_t N, int64_t K, bool bf16, bool a_strided, int use, int64_t most) {
    const int cus = device_cu_count(), KT = TILE_KB / (bf16 ? 2 : 4);
    const int64_t nk = std::max<int64_t>(2, up((K + KT - 1) / KT, 2));
    Plan best{0, 1, (int)nk, 0};
    double best_us = 1e30;
    for (int S : {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24}) {
        const int64_t per_split = up((nk + S - 1) / S, 2), bytes = S > 1 ? (int64_t)S * M * N * 4 : 0;
        if (S > 1 && (most <= 0 || bytes > most || (nk + per_split - 1) / per_split != S)) continue;
        for (int t = 0; t < TILES; ++t) {
            if (!has_tile(t, bf16, a_strided, use)) continue;
            const TileTime& c = kTimes[bf16 ? 0 : 1][S > 1 ? USE_PARTIAL : use][t];
            const int bn = kTiles[t].bn / (use == USE_GATE ? 2 : 1);
            const int64_t per = ((M + kTiles[t].bm - 1) / kTiles[t].bm * ((N + bn - 1) / bn) * S + cus - 1) / cus;
            const int64_t full = t < 2 ? per : per / 2, rem = t < 2 ? 0 : per & 1;
            const double k = (double)per_split * KT / 64.0;
            double us = c.launch + full * (k * c.full + c.epi) + rem * (k * c.one + 0.5 * c.epi);
            if (S > 1) us += 3.0 + bytes / 6.0e6;
            if (us < best_us) {
                best_us = us;
                best = Plan{t, S, (int)per_split, bytes};
            }
        }
    }
    return best;
}

// Launches tile t of those that a product can have.
template <class T, bool AKS, bool BKS, int USE, int TILE = 0>
static void launch_tile(const TileArgs& a, int t, dim3 grid, hipStream_t s) {
    if constexpr (TILE < TILES) {
        if constexpr (has_tile(TILE, sizeof(T) == 2, AKS, USE))
            if (t == TILE) {
                hipLaunchKernelGGL((tile_kernel<T, AKS, BKS, TILE, USE>), grid, dim3(tile_threads(TILE)), 0, s, a);
                return;
            }
        launch_tile<T, AKS, BKS, USE, TILE + 1>(a, t, grid, s);
    }
}

template <class T, bool AKS, bool BKS, int USE>
static void product(TileArgs a, const Plan& w, hipStream_t s) {
    a.splits = w.splits;
    a.kt_split = w.kt_split;
    const int bm = kTiles[w.tile].bm, bn = kTiles[w.tile].bn / (USE == USE_GATE ? 2 : 1);
    const int64_t items = ((int64_t)a.M + bm - 1) / bm * ((a.N + bn - 1) / bn) * a.splits;
    launch_tile<T, AKS, BKS, USE>(a, w.tile, dim3((unsigned)std::min<int64_t>(items, (int64_t)device_cu_count() * (w.tile < 2 ? 1 : 2))), s);
}

// C = A.B (+ bias), by way of partial sums where the plan splits k.
template <class T, bool AKS, bool BKS>
static void stored_product(TileArgs a, const Plan& w, float* partial, hipStream_t s) {
    if (w.splits == 1) {
        product<T, AKS, BKS, USE_STORE>(a, w, s);
        return;
    }
    T* const out = static_cast<T*>(a.C);
    const int ld = a.ldc;
    a.C = partial;
    a.ldc = a.N;
    product<T, AKS, BKS, USE_PARTIAL>(a, w, s);
    const uint32_t n4 = (uint32_t)((int64_t)a.M * a.N / 4);
    hipLaunchKernelGGL((sum_parts_kernel<T>), dim3((n4 + 255) / 256), dim3(256), 0, s, reinterpret_cast<const float4*>(partial), w.splits, n4,
                       (uint32_t)(a.N / 4), a.bias, out, ld);
}

static int col_parts(int64_t rows) { return (int)std::max<int64_t>(1, std::min<int64_t>(64, rows / 256)); }
template <class T>
static void sum_rows(const T* x, int64_t ld, int64_t rows, int cols, float* parts, float* out, hipStream_t s) {
    const int n = col_parts(rows);
    const unsigned cb = (unsigned)((cols + 63) / 64);
    hipLaunchKernelGGL((sum_rows_kernel<T>), dim3(cb, n), dim3(1024), 0, s, x, ld, rows, cols, n > 1 ? parts : out);
    if (n > 1) hipLaunchKernelGGL((sum_rows_kernel<float>), dim3(cb), dim3(1024), 0, s, parts, (int64_t)cols, (int64_t)n, cols, out);
}

// ---------------------------------------------------------------------------
// At most FEW_ROWS tokens, where the weights' bytes are the work: a workgroup has
// 16 columns and all of k, every 128 bytes of a weight row go to one wave as 32
// contiguous bytes a lane, straight into MFMA operands, and each wave sums its
// share of k; the waves' sums meet in LDS.  X comes from the caches.  One bf16 token
// of 768 x 2,048: 4.3 + 5.6 us for 9.4 MB of weights.
// ---------------------------------------------------------------------------
constexpr int FEW_ROWS = 64;
struct FewArgs {
    const void* X;      // [M, K], fp32 where it is split
    const void* W;      // [N, K] rows; the gate's and then the other projection's where GATE
    const float* bias;
    void* out;          // h or Y
    void* gu;           // GATE: [M, 2 N], or null
    float* hf;          // GATE, bf16: h before its rounding
    int M, N, K, ldx, ldo, act;
};

// SPLIT: X is fp32, and each value is two bf16 (16 of its bits: the products'
// operand errors are 2^-17 instead of 2^-9; the MFMAs are idle anyway).
template <class T, int MB, bool GATE, bool SPLIT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void few_kernel(FewArgs p) {
    constexpr int ES = sizeof(T), KT = 128 / ES, CE = 16 / ES, G = GATE ? 2 : 1, PASS = MB > 2 ? 2 : 4, XP = SPLIT ? 2 : 1;
    __shared__ __attribute__((aligned(16))) float red[WAVES * MB * G * 256];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, q = lane >> 4;
    const int n0 = blockIdx.x * 16;
    typedef std::conditional_t<SPLIT, float, T> TX;
    const T* const w0 = static_cast<const T*>(p.W) + (int64_t)min(n0 + r, p.N - 1) * p.K;
    const TX* x[MB];
#pragma unroll
    for (int b = 0; b < MB; ++b) x[b] = static_cast<const TX*>(p.X) + (int64_t)min(16 * b + r, p.M - 1) * p.ldx;
    g16_v4f acc[G][MB];
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int b = 0; b < MB; ++b) acc[g][b] = g16_v4f{0.0f, 0.0f, 0.0f, 0.0f};
    const int chunks = (p.K + KT - 1) / KT;
    for (int c0 = wave; c0 < chunks; c0 += WAVES * PASS) {
        g16_v4f wv[PASS][G][2], xv[PASS][MB][2][XP];
#pragma unroll
        for (int u = 0; u < PASS; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = (c0 + u * WAVES) * KT + q * (KT / 4) + h * CE;   // K is whole pieces of CE
                const bool in = k < p.K;
#pragma unroll
                for (int g = 0; g < G; ++g)
                    wv[u][g][h] = in ? *reinterpret_cast<const g16_v4f*>(w0 + (int64_t)g * p.N * p.K + k) : g16_v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int b = 0; b < MB; ++b)
#pragma unroll
                    for (int e = 0; e < XP; ++e)
                        xv[u][b][h][e] = in ? *reinterpret_cast<const g16_v4f*>(x[b] + k + 4 * e) : g16_v4f{0.0f, 0.0f, 0.0f, 0.0f};
            }
#pragma unroll
        for (int u = 0; u < PASS; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int b = 0; b < MB; ++b) {
                    if constexpr (SPLIT) {
                        const g16_v4f a = xv[u][b][h][0], c = xv[u][b][h][1];
                        u4v_t hi = {pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]), pack_bf16x2(c[0], c[1]), pack_bf16x2(c[2], c[3])}, lo;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float v0 = e < 2 ? a[2 * e] : c[2 * e - 4], v1 = e < 2 ? a[2 * e + 1] : c[2 * e - 3];
                            // of infinity and NaN, and what rounds to infinity, all is in hi
                            auto rest = [](float d) { return fabsf(d) < __builtin_inff() ? d : 0.0f; };
                            lo[e] = pack_bf16x2(rest(v0 - __uint_as_float(hi[e] << 16)), rest(v1 - __uint_as_float(hi[e] & 0xffff0000u)));
                        }
                        acc[0][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(g16_v8bf, wv[u][0][h]), __builtin_bit_cast(g16_v8bf, lo),
                                                                            acc[0][b], 0, 0, 0);
                        acc[0][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(g16_v8bf, wv[u][0][h]), __builtin_bit_cast(g16_v8bf, hi),
                                                                            acc[0][b], 0, 0, 0);
                    } else {
#pragma unroll
                        for (int g = 0; g < G; ++g) {
                            if constexpr (ES == 2)
                                acc[g][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(g16_v8bf, wv[u][g][h]),
                                                                                    __builtin_bit_cast(g16_v8bf, xv[u][b][h][0]), acc[g][b], 0, 0, 0);
                            else
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    acc[g][b] = __builtin_amdgcn_mfma_f32_16x16x4f32(wv[u][g][h][e], xv[u][b][h][0][e], acc[g][b], 0, 0, 0);
                        }
                    }
                }
    }
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int b = 0; b < MB; ++b) *reinterpret_cast<g16_v4f*>(red + ((wave * MB + b) * G + g) * 256 + r * 16 + 4 * q) = acc[g][b];
    __syncthreads();
    // four columns of a row a thread
    if (tid >= MB * 64) return;
    const int b = tid >> 6, row = 16 * b + r, n = n0 + 4 * q;
    if (row >= p.M || n >= p.N) return;
    g16_v4f v[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        v[g] = *reinterpret_cast<const g16_v4f*>(red + (b * G + g) * 256 + r * 16 + 4 * q);
        for (int w = 1; w < WAVES; ++w) v[g] += *reinterpret_cast<const g16_v4f*>(red + ((w * MB + b) * G + g) * 256 + r * 16 + 4 * q);
        if (p.bias) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[g][e] += p.bias[g * p.N + n + e];
        }
    }
    auto put = [&](void* base, int64_t at, const g16_v4f& o) __attribute__((always_inline)) {
        if constexpr (ES == 2) *reinterpret_cast<uint2*>(static_cast<T*>(base) + at) = make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
        else *reinterpret_cast<g16_v4f*>(static_cast<T*>(base) + at) = o;
    };
    if constexpr (GATE) {
        float gv[4] = {v[0][0], v[0][1], v[0][2], v[0][3]}, uv[4] = {v[1][0], v[1][1], v[1][2], v[1][3]}, hv[4];
        act_times<4>(p.act, gv, uv, hv);
        const g16_v4f h = {hv[0], hv[1], hv[2], hv[3]};
        put(p.out, (int64_t)row * p.N + n, h);
        if (p.hf) *reinterpret_cast<g16_v4f*>(p.hf + (int64_t)row * p.N + n) = h;
        if (p.gu) {
            put(p.gu, (int64_t)row * 2 * p.N + n, v[0]);
            put(p.gu, (int64_t)row * 2 * p.N + p.N + n, v[1]);
        }
    } else {
        put(p.out, (int64_t)row * p.ldo + n, v[0]);
    }
}

template <class T, bool GATE, bool SPLIT>
static void launch_few(const FewArgs& a, hipStream_t s) {
    // 4 waves and 32 columns' rows, or 8 and 16: as many bytes on their way
    constexpr int WAVES = GATE ? 4 : 8;
    const dim3 grid((unsigned)((a.N + 15) / 16)), block(64 * WAVES);
    switch ((a.M + 15) / 16) {
        case 1: hipLaunchKernelGGL((few_kernel<T, 1, GATE, SPLIT, WAVES>), grid, block, 0, s, a); break;
        case 2: hipLaunchKernelGGL((few_kernel<T, 2, GATE, SPLIT, WAVES>), grid, block, 0, s, a); break;
        case 3: hipLaunchKernelGGL((few_kernel<T, 3, GATE, SPLIT, WAVES>), grid, block, 0, s, a); break;
        default: hipLaunchKernelGGL((few_kernel<T, 4, GATE, SPLIT, WAVES>), grid, block, 0, s, a); break;
    }
}

template <class T>
static void few(const GatedArgs& g, hipStream_t s) {
    constexpr bool BF16 = sizeof(T) == 2;
    FewArgs a{};
    a.X = g.X;
    a.ldx = (int)g.ldx;
    a.W = g.Wgu;
    a.bias = g.bgu;
    a.out = g.h;
    a.gu = g.gu;
    a.hf = BF16 ? static_cast<float*>(g.ws) : nullptr;
    a.M = g.M;
    a.N = g.I;
    a.K = g.H;
    a.act = g.act;
    launch_few<T, true, false>(a, s);
    a.X = BF16 ? g.ws : g.h;
    a.ldx = g.I;
    a.W = g.Wd;
    a.bias = g.bd;
    a.out = g.Y;
    a.ldo = (int)g.ldy;
    a.N = g.H;
    a.K = g.I;
    launch_few<T, false, BF16>(a, s);
}

// Most bytes of partial sums: of outputs of a row a token, and of weights' gradients.
constexpr int64_t PARTIAL_ROWS = 64 << 20, PARTIAL_WEIGHTS = 512 << 20;

// At most FEW_ROWS tokens: few_kernel reads the weights once and needs no tiles.
// bf16: its h between the two products is kept in fp32 too, in the workspace.
static Plan down_plan(int M, int H, int I, bool bf16) { return plan_product(M, H, I, bf16, false, USE_STORE, PARTIAL_ROWS); }
int64_t gated_ws_bytes(int M, int H, int I, bool bf16) {
    if (M <= FEW_ROWS) return bf16 ? up((int64_t)M * I * 4, 256) : 0;
    return up(down_plan(M, H, I, bf16).partial, 256);
}

template <class T>
static void gated(const GatedArgs& g, hipStream_t s) {
    constexpr bool BF16 = sizeof(T) == 2;
    if (g.M <= FEW_ROWS) {
        few<T>(g, s);
        return;
    }
    TileArgs a{};
    a.A = g.X;
    a.lda = (int)g.ldx;
    a.B = g.Wgu;
    a.ldb = g.H;
    a.M = g.M;
    a.N = a.I = g.I;
    a.K = g.H;
    a.bias = g.bgu;
    a.h = g.h;
    a.gu = g.gu;
    a.act = g.act;
    product<T, false, false, USE_GATE>(a, plan_product(g.M, g.I, g.H, BF16, false, USE_GATE, 0), s);
    a.A = g.h;
    a.lda = g.I;
    a.B = g.Wd;
    a.ldb = g.I;
    a.C = g.Y;
    a.ldc = (int)g.ldy;
    a.N = g.H;
    a.K = g.I;
    a.bias = g.bd;
    stored_product<T, false, false>(a, down_plan(g.M, g.H, g.I, BF16), static_cast<float*>(g.ws), s);
}

// The backward's workspace: [dg du], its column sums by row blocks, partial
// sums of one product at a time, and partial column sums.
struct BwdSpace {
    int64_t colsum, partial, cols, bytes;
    Plan slopes, dx, wgu, wd;
};
static BwdSpace bwd_space(int M, int H, int I, bool bf16) {
    BwdSpace w;
    const int64_t I2 = 2 * (int64_t)I;
    w.slopes = plan_product(M, I, H, bf16, false, USE_SLOPES, 0);
    w.dx = plan_product(M, H, I2, bf16, false, USE_STORE, PARTIAL_ROWS);
    w.wgu = plan_product(I2, H, M, bf16, true, USE_STORE, PARTIAL_WEIGHTS);
    w.wd = plan_product(H, I, M, bf16, true, USE_STORE, PARTIAL_WEIGHTS);
    const TileShape& t = kTiles[w.slopes.tile];
    w.colsum = up(M * I2 * (bf16 ? 2 : 4), 256);
    w.partial = w.colsum + up(((int64_t)M + t.bm - 1) / t.bm * t.waves_m * I2 * 4, 256);
    w.cols = w.partial + up(std::max({w.dx.partial, w.wgu.partial, w.wd.partial}), 256);
    w.bytes = w.cols + up(64 * std::max<int64_t>(I2, H) * 4, 256);
    return w;
}
int64_t gated_bwd_ws_bytes(int M, int H, int I, bool bf16) { return bwd_space(M, H, I, bf16).bytes; }

template <class T>
static hipError_t gated_bwd(const GatedArgs& g, hipStream_t s) {
    const int64_t I2 = 2 * (int64_t)g.I;
    if (g.M == 0) {   // sums over no rows
        const int64_t words = sizeof(T) * g.H * (int64_t)g.I / 4;
        hipError_t e = hipSuccess;
        auto zero = [&](void* p, int64_t n) {
            if (p && e == hipSuccess) e = launch_zero_words(p, n, s);
        };
        zero(g.dWgu, 2 * words);
        zero(g.dWd, words);
        zero(g.dbgu, I2);
        zero(g.dbd, g.H);
        return e;
    }
    const BwdSpace w = bwd_space(g.M, g.H, g.I, sizeof(T) == 2);
    char* const ws = static_cast<char*>(g.ws);
    float* const colsum = reinterpret_cast<float*>(ws + w.colsum);
    float* const partial = reinterpret_cast<float*>(ws + w.partial);
    float* const cols = reinterpret_cast<float*>(ws + w.cols);
    TileArgs a{};
    a.act = g.act;
    a.I = g.I;
    if (g.dX || g.dWgu || g.dbgu) {
        a.A = g.dY;
        a.lda = (int)g.lddy;
        a.B = g.Wd;
        a.ldb = g.I;
        a.M = g.M;
        a.N = g.I;
        a.K = g.H;
        a.gu = g.gu;
        a.dgu = ws;
        a.colsum = g.dbgu ? colsum : nullptr;
        product<T, false, true, USE_SLOPES>(a, w.slopes, s);
        if (g.dbgu) {
            const TileShape& t = kTiles[w.slopes.tile];
            sum_rows<float>(colsum, I2, ((int64_t)g.M + t.bm - 1) / t.bm * t.waves_m, (int)I2, cols, g.dbgu, s);
        }
    }
    if (g.dbd) sum_rows<T>(static_cast<const T*>(g.dY), g.lddy, g.M, g.H, cols, g.dbd, s);
    if (g.dX) {
        a.A = ws;
        a.lda = (int)I2;
        a.B = g.Wgu;
        a.ldb = g.H;
        a.C = g.dX;
        a.ldc = (int)g.lddx;
        a.M = g.M;
        a.N = g.H;
        a.K = (int)I2;
        stored_product<T, false, true>(a, w.dx, partial, s);
    }
    a.K = g.M;
    if (g.dWgu) {
        a.A = ws;
        a.lda = (int)I2;
        a.B = g.X;
        a.ldb = (int)g.ldx;
        a.C = g.dWgu;
        a.ldc = g.H;
        a.M = (int)I2;
        a.N = g.H;
        stored_product<T, true, true>(a, w.wgu, partial, s);
    }
    if (g.dWd) {
        a.A = g.dY;
        a.lda = (int)g.lddy;
        a.B = g.h;
        a.ldb = g.I;
        a.C = g.dWd;
        a.ldc = g.I;
        a.M = g.H;
        a.N = g.I;
        stored_product<T, true, true>(a, w.wd, partial, s);
    }
    return hipGetLastError();
}

hipError_t launch_gated(const GatedArgs& a, bool bf16, hipStream_t s) {
    if (bf16) gated<uint16_t>(a, s);
    else gated<float>(a, s);
    return hipGetLastError();
}

hipError_t launch_gated_bwd(const GatedArgs& a, bool bf16, hipStream_t s) {
    return bf16 ? gated_bwd<uint16_t>(a, s) : gated_bwd<float>(a, s);
}

}  // namespace ebh
