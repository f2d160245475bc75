// gated.hip -- the gated feed-forward block and its gradients
// (ebh_op_gated_ffn / _bwd), as products on the tiles of tile.hpp.
#include <algorithm>

#include "tile.hpp"

namespace ebh {

// ---------------------------------------------------------------------------
// The tiles, largest first.  A kernel's operand orders: both k contiguous
// (forward), B strided (through the weights back), both strided (weight
// gradients, whose k are the tokens).
// ---------------------------------------------------------------------------
template <class T, bool AKS, bool BKS, int TILE, int USE>
__global__ __launch_bounds__(TILE == 0 ? 512 : 256, 2) void tile_kernel(TileArgs p) {
    constexpr int BM = TILE == 0 ? 256 : (TILE == 1 ? 128 : 64), BN = TILE == 0 ? 256 : 128, NS = TILE == 2 ? 3 : 2;
    __shared__ __attribute__((aligned(16))) char smem[tile_lds(BM, BN, NS)];
    tile_body<T, AKS, BKS, BM, BN, 2, TILE == 0 ? 4 : 2, NS, USE>(p, smem);
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

// out = the sum of `parts` partial products, in order; n a multiple of 4.
template <class T>
__global__ __launch_bounds__(256) void sum_parts_kernel(const float* x, int parts, int64_t n, T* out) {
    const int64_t i = 4 * (blockIdx.x * (int64_t)256 + threadIdx.x);
    if (i >= n) return;
    float4 s = *reinterpret_cast<const float4*>(x + i);
    for (int k = 1; k < parts; ++k) {
        const float4 v = *reinterpret_cast<const float4*>(x + k * n + i);
        s.x += v.x;
        s.y += v.y;
        s.z += v.z;
        s.w += v.w;
    }
    if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(out + i) = make_uint2(pack_bf16x2(s.x, s.y), pack_bf16x2(s.z, s.w));
    else *reinterpret_cast<float4*>(out + i) = s;
}

static int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// Which tile: the largest that fills the chip, else ...
static int pick_tile(int64_t M, int64_t N, bool f32, bool strided) {
    const int cus = device_cu_count();
    auto tiles = [&](int bm, int bn) { return (M + bm - 1) / bm * ((N + bn - 1) / bn); };
    if (!f32 && tiles(256, 256) >= cus) return 0;
    if (strided || tiles(128, 128) >= cus) return 1;
    return 2;
}

struct SplitPlan {
    int tile, splits, kt;
};
// Weight gradients: M x N products over `K` tokens.
static SplitPlan plan_split(int64_t M, int64_t N, int K, bool bf16) {
    const int cus = device_cu_count(), kt = (K + (bf16 ? 63 : 31)) / (bf16 ? 64 : 32);
    const int tile = bf16 && M * N >= 256 * 256 * 4 && kt >= 64 ? 0 : 1;
    const int bm = tile == 0 ? 256 : 128, slots = tile == 0 ? cus : 2 * cus;
    const int64_t tiles = up(M, bm) / bm * (up(N, bm) / bm);
    const int s = (int)std::max<int64_t>(1, std::min<int64_t>(slots / tiles, kt / 4));
    SplitPlan p{tile, s, std::max(2, (int)up((kt + s - 1) / s, 2))};
    p.splits = std::max(1, (kt + p.kt - 1) / p.kt);
    return p;
}

template <class T, bool AKS, bool BKS, int USE>
static void product(TileArgs a, int tile, hipStream_t s) {
    constexpr int KT = 128 / sizeof(T);
    if (a.splits == 0) {
        a.splits = 1;
        a.kt_split = std::max(2, (int)up((a.K + KT - 1) / KT, 2));
    }
    const int bm = tile == 0 ? 256 : (tile == 1 ? 128 : 64), bn = (tile == 0 ? 256 : 128) / (USE == USE_GATE ? 2 : 1);
    const int64_t items = (int64_t)((a.M + bm - 1) / bm) * ((a.N + bn - 1) / bn) * a.splits;
    const dim3 grid((unsigned)std::min<int64_t>(items, (int64_t)device_cu_count() * (tile == 0 ? 1 : 2)));
    if constexpr (sizeof(T) == 2)
        if (tile == 0) {
            hipLaunchKernelGGL((tile_kernel<T, AKS, BKS, 0, USE>), grid, dim3(512), 0, s, a);
            return;
        }
    if constexpr (!AKS)
        if (tile == 2) {
            hipLaunchKernelGGL((tile_kernel<T, AKS, BKS, 2, USE>), grid, dim3(256), 0, s, a);
            return;
        }
    hipLaunchKernelGGL((tile_kernel<T, AKS, BKS, 1, USE>), grid, dim3(256), 0, s, a);
}

static int col_parts(int64_t rows) { return (int)std::max<int64_t>(1, std::min<int64_t>(64, rows / 256)); }
template <class T>
static void sum_rows(const T* x, int64_t ld, int64_t rows, int cols, float* parts, float* out, hipStream_t s) {
    const int n = col_parts(rows);
    const unsigned cb = (unsigned)((cols + 63) / 64);
    hipLaunchKernelGGL((sum_rows_kernel<T>), dim3(cb, n), dim3(1024), 0, s, x, ld, rows, cols, n > 1 ? parts : out);
    if (n > 1) hipLaunchKernelGGL((sum_rows_kernel<float>), dim3(cb), dim3(1024), 0, s, parts, (int64_t)cols, (int64_t)n, cols, out);
}

// The backward's workspace: [dg du], its column sums by row blocks, partial
// weight gradients, and partial column sums.
struct BwdSpace {
    int64_t dgu, colsum, partial, cols, bytes;
    SplitPlan wgu, wd;
    int slopes_tile;
};
static BwdSpace bwd_space(int M, int H, int I, bool bf16) {
    BwdSpace w;
    const int64_t es = bf16 ? 2 : 4, I2 = 2 * (int64_t)I;
    w.slopes_tile = pick_tile(M, I, !bf16, false);
    const int bm = w.slopes_tile == 0 ? 256 : (w.slopes_tile == 1 ? 128 : 64);
    w.wgu = plan_split(I2, H, M, bf16);
    w.wd = plan_split(H, I, M, bf16);
    int64_t at = up(M * I2 * es, 256);
    w.dgu = 0;
    w.colsum = at;
    at += up((int64_t)((M + (int64_t)bm - 1) / bm) * 2 * I2 * 4, 256);
    w.partial = at;
    const int64_t pg = w.wgu.splits > 1 ? w.wgu.splits * I2 * H * 4 : 0, pd = w.wd.splits > 1 ? (int64_t)w.wd.splits * H * I * 4 : 0;
    at += up(std::max(pg, pd), 256);
    w.cols = at;
    at += up(64 * std::max<int64_t>(I2, H) * 4, 256);
    w.bytes = at;
    return w;
}

int64_t gated_ws_bytes(int, int, int, bool) { return 0; }
int64_t gated_bwd_ws_bytes(int M, int H, int I, bool bf16) { return bwd_space(M, H, I, bf16).bytes; }

template <class T>
static void gated(const GatedArgs& g, hipStream_t s) {
    constexpr bool F32 = sizeof(T) == 4;
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
    product<T, false, false, USE_GATE>(a, pick_tile(g.M, 2 * (int64_t)g.I, F32, false), s);
    a.A = g.h;
    a.lda = g.I;
    a.B = g.Wd;
    a.ldb = g.I;
    a.C = g.Y;
    a.ldc = (int)g.ldy;
    a.N = g.H;
    a.K = g.I;
    a.bias = g.bd;
    product<T, false, false, USE_STORE>(a, pick_tile(g.M, g.H, F32, false), s);
}

template <class T>
static void weight_gradient(TileArgs a, const SplitPlan& w, float* partial, void* out, hipStream_t s) {
    a.splits = w.splits;
    a.kt_split = w.kt;
    a.ldc = a.N;
    a.bias = nullptr;
    if (w.splits == 1) {
        a.C = out;
        product<T, true, true, USE_STORE>(a, w.tile, s);
        return;
    }
    a.C = partial;
    product<T, true, true, USE_PARTIAL>(a, w.tile, s);
    const int64_t n = (int64_t)a.M * a.N;
    hipLaunchKernelGGL((sum_parts_kernel<T>), dim3((unsigned)((n / 4 + 255) / 256)), dim3(256), 0, s, partial, w.splits, n, static_cast<T*>(out));
}

template <class T>
static void gated_bwd(const GatedArgs& g, hipStream_t s) {
    constexpr bool F32 = sizeof(T) == 4;
    const BwdSpace w = bwd_space(g.M, g.H, g.I, !F32);
    char* const ws = static_cast<char*>(g.ws);
    const int64_t I2 = 2 * (int64_t)g.I;
    if (g.M == 0) {   // sums over no rows
        const int64_t es = sizeof(T) / 2;   // in 16-bit halves of words
        if (g.dWgu) launch_zero_words(g.dWgu, I2 * g.H * es / 2, s);
        if (g.dWd) launch_zero_words(g.dWd, (int64_t)g.H * g.I * es / 2, s);
        if (g.dbgu) launch_zero_words(g.dbgu, I2, s);
        if (g.dbd) launch_zero_words(g.dbd, g.H, s);
        return;
    }
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
        product<T, false, true, USE_SLOPES>(a, w.slopes_tile, s);
        if (g.dbgu) {
            const int bm = w.slopes_tile == 0 ? 256 : (w.slopes_tile == 1 ? 128 : 64);
            sum_rows<float>(colsum, I2, (g.M + (int64_t)bm - 1) / bm * 2, (int)I2, cols, g.dbgu, s);
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
        product<T, false, true, USE_STORE>(a, pick_tile(g.M, g.H, F32, false), s);
    }
    a.K = g.M;
    if (g.dWgu) {
        a.A = ws;
        a.lda = (int)I2;
        a.B = g.X;
        a.ldb = (int)g.ldx;
        a.M = (int)I2;
        a.N = g.H;
        weight_gradient<T>(a, w.wgu, partial, g.dWgu, s);
    }
    if (g.dWd) {
        a.A = g.dY;
        a.lda = (int)g.lddy;
        a.B = g.h;
        a.ldb = g.I;
        a.M = g.H;
        a.N = g.I;
        weight_gradient<T>(a, w.wd, partial, g.dWd, s);
    }
}

hipError_t launch_gated(const GatedArgs& a, bool bf16, hipStream_t s) {
    if (bf16) gated<uint16_t>(a, s);
    else gated<float>(a, s);
    return hipGetLastError();
}

hipError_t launch_gated_bwd(const GatedArgs& a, bool bf16, hipStream_t s) {
    if (bf16) gated_bwd<uint16_t>(a, s);
    else gated_bwd<float>(a, s);
    return hipGetLastError();
}

}  // namespace ebh
