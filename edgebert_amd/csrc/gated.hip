// gated.hip -- the gated feed-forward block and its gradients
// (ebh_op_gated_ffn / _bwd).
#include <algorithm>

#include "layer.hpp"

namespace ebh {

// Activation and its derivative.
__device__ __forceinline__ float act_of(int act, float g) {
    if (act == 0) return g / (1.0f + expf(-g));
    if (act == 1) return gelu_tanh(g);
    return 0.5f * g * (1.0f + erff(g * 0.70710678118654752f));
}
__device__ __forceinline__ float act_slope(int act, float g) {
    if (act == 0) {
        const float s = 1.0f / (1.0f + expf(-g));
        return s * (1.0f + g * (1.0f - s));
    }
    if (act == 1) {
        const float t = tanhf(0.7978845608f * (g + 0.044715f * g * g * g));
        return 0.5f * (1.0f + t) + 0.5f * g * (1.0f - t * t) * 0.7978845608f * (1.0f + 3.0f * 0.044715f * g * g);
    }
    return 0.5f * (1.0f + erff(g * 0.70710678118654752f)) + g * expf(-0.5f * g * g) * 0.3989422804014327f;
}

// A product C(m, n) = sum over k of A(m, k) B(n, k) with operands in any
// orders (element strides), and what becomes of it.
enum Use : int { USE_STORE = 0, USE_GATE = 1, USE_SLOPES = 2 };
struct SimpleArgs {
    const void* A;
    const void* B;
    void* C;
    int64_t am, ak, bn, bk, ldc;
    int M, N, K;
    const float* bias;
    GatedArgs g;
    float* colsum;      // USE_SLOPES: [row blocks][2 I] sums before rounding
    void* dgu;
};

// 64 x 64 tiles, 16 x 16 threads of 4 x 4 outputs; USE_GATE: N = I, with a second
// sum for the rows of B that are I further on.
template <class T, int USE>
__global__ __launch_bounds__(256) void simple_kernel(SimpleArgs p) {
    __shared__ float sa[16][65], sb[16][65], sc[USE == USE_GATE ? 16 : 1][65];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int64_t m0 = (int64_t)blockIdx.y * 64, n0 = (int64_t)blockIdx.x * 64;
    const T* A = static_cast<const T*>(p.A);
    const T* B = static_cast<const T*>(p.B);
    float acc[4][4] = {}, acc2[4][4] = {};
    for (int k0 = 0; k0 < p.K; k0 += 16) {
        for (int e = threadIdx.x; e < 1024; e += 256) {
            const int r = e >> 4, k = e & 15;
            const bool in = k0 + k < p.K;
            sa[k][r] = in && m0 + r < p.M ? to_f32(A[(m0 + r) * p.am + (k0 + k) * p.ak]) : 0.0f;
            sb[k][r] = in && n0 + r < p.N ? to_f32(B[(n0 + r) * p.bn + (k0 + k) * p.bk]) : 0.0f;
            if (USE == USE_GATE) sc[k][r] = in && n0 + r < p.N ? to_f32(B[(n0 + r + p.N) * p.bn + (k0 + k) * p.bk]) : 0.0f;
        }
        __syncthreads();
        for (int k = 0; k < 16; ++k)
            for (int i = 0; i < 4; ++i)
                for (int j = 0; j < 4; ++j) {
                    acc[i][j] += sa[k][ty * 4 + i] * sb[k][tx * 4 + j];
                    if (USE == USE_GATE) acc2[i][j] += sa[k][ty * 4 + i] * sc[k][tx * 4 + j];
                }
        __syncthreads();
    }
    float cg[4] = {}, cu[4] = {};
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int64_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
            if (m >= p.M || n >= p.N) continue;
            const int64_t I = p.g.I;
            if (USE == USE_STORE) {
                store_as(static_cast<T*>(p.C) + m * p.ldc + n, acc[i][j] + (p.bias ? p.bias[n] : 0.0f));
            } else if (USE == USE_GATE) {
                const float g = acc[i][j] + (p.bias ? p.bias[n] : 0.0f), u = acc2[i][j] + (p.bias ? p.bias[I + n] : 0.0f);
                store_as(static_cast<T*>(p.g.h) + m * I + n, act_of(p.g.act, g) * u);
                if (p.g.gu) {
                    store_as(static_cast<T*>(p.g.gu) + m * 2 * I + n, g);
                    store_as(static_cast<T*>(p.g.gu) + m * 2 * I + I + n, u);
                }
            } else {
                const T* gu = static_cast<const T*>(p.g.gu) + m * 2 * I + n;
                const float g = to_f32(gu[0]), u = to_f32(gu[I]);
                const float dg = acc[i][j] * u * act_slope(p.g.act, g), du = acc[i][j] * act_of(p.g.act, g);
                T* out = static_cast<T*>(p.dgu) + m * 2 * I + n;
                store_as(out, dg);
                store_as(out + I, du);
                cg[j] += dg;
                cu[j] += du;
            }
        }
    if (USE == USE_SLOPES && p.colsum) {
        for (int j = 0; j < 4; ++j) {
            sa[ty][tx * 4 + j] = cg[j];
            sb[ty][tx * 4 + j] = cu[j];
        }
        __syncthreads();
        if (threadIdx.x < 64 && n0 + threadIdx.x < p.N) {
            float g = 0.0f, u = 0.0f;
            for (int k = 0; k < 16; ++k) {
                g += sa[k][threadIdx.x];
                u += sb[k][threadIdx.x];
            }
            float* at = p.colsum + (int64_t)blockIdx.y * 2 * p.g.I + n0 + threadIdx.x;
            at[0] = g;
            at[p.g.I] = u;
        }
    }
}

// out[c] = sum over rows of x[r, c], in order of r.
template <class T>
__global__ __launch_bounds__(256) void colsum_kernel(const T* x, int64_t ld, int rows, int cols, float* out) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= cols) return;
    float s = 0.0f;
    for (int64_t r = 0; r < rows; ++r) s += to_f32(x[r * ld + c]);
    out[c] = s;
}

static int64_t up16(int64_t v) { return (v + 15) / 16 * 16; }
int64_t gated_ws_bytes(int, int, int, bool) { return 0; }
int64_t gated_bwd_ws_bytes(int M, int, int I, bool bf16) {
    return up16((int64_t)M * 2 * I * (bf16 ? 2 : 4)) + ((int64_t)M + 63) / 64 * 2 * I * 4;
}

template <class T, int USE>
static void product(SimpleArgs a, hipStream_t s) {
    hipLaunchKernelGGL((simple_kernel<T, USE>), dim3((unsigned)((a.N + 63) / 64), (unsigned)((a.M + 63) / 64)), dim3(256), 0, s, a);
}

template <class T>
static void gated(const GatedArgs& g, hipStream_t s) {
    SimpleArgs a{};
    a.g = g;
    a.A = g.X; a.am = g.ldx; a.ak = 1;
    a.B = g.Wgu; a.bn = g.H; a.bk = 1;
    a.M = g.M; a.N = g.I; a.K = g.H;
    a.bias = g.bgu;
    product<T, USE_GATE>(a, s);
    a.A = g.h; a.am = g.I;
    a.B = g.Wd; a.bn = g.I;
    a.C = g.Y; a.ldc = g.ldy;
    a.N = g.H; a.K = g.I;
    a.bias = g.bd;
    product<T, USE_STORE>(a, s);
}

template <class T>
static void gated_bwd(const GatedArgs& g, hipStream_t s) {
    SimpleArgs a{};
    a.g = g;
    a.dgu = g.ws;
    const int64_t I2 = 2 * (int64_t)g.I;
    a.colsum = reinterpret_cast<float*>(static_cast<char*>(g.ws) + up16(g.M * I2 * sizeof(T)));
    a.A = g.dY; a.am = g.lddy; a.ak = 1;
    a.B = g.Wd; a.bn = 1; a.bk = g.I;
    a.M = g.M; a.N = g.I; a.K = g.H;
    if (g.M > 0) product<T, USE_SLOPES>(a, s);
    if (g.dbgu)
        hipLaunchKernelGGL((colsum_kernel<float>), dim3((unsigned)((I2 + 255) / 256)), dim3(256), 0, s, a.colsum, I2, (g.M + 63) / 64, (int)I2, g.dbgu);
    if (g.dbd)
        hipLaunchKernelGGL((colsum_kernel<T>), dim3((unsigned)((g.H + 255) / 256)), dim3(256), 0, s, static_cast<const T*>(g.dY), g.lddy, g.M, g.H, g.dbd);
    if (g.dX && g.M > 0) {
        a.A = g.ws; a.am = I2; a.ak = 1;
        a.B = g.Wgu; a.bn = 1; a.bk = g.H;
        a.C = g.dX; a.ldc = g.lddx;
        a.N = g.H; a.K = (int)I2;
        product<T, USE_STORE>(a, s);
    }
    if (g.dWgu) {
        a.A = g.ws; a.am = 1; a.ak = I2;
        a.B = g.X; a.bn = 1; a.bk = g.ldx;
        a.C = g.dWgu; a.ldc = g.H;
        a.M = (int)I2; a.N = g.H; a.K = g.M;
        product<T, USE_STORE>(a, s);
    }
    if (g.dWd) {
        a.A = g.dY; a.am = 1; a.ak = g.lddy;
        a.B = g.h; a.bn = 1; a.bk = g.I;
        a.C = g.dWd; a.ldc = g.I;
        a.M = g.H; a.N = g.I; a.K = g.M;
        product<T, USE_STORE>(a, s);
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
