// norm.hip -- layer norm and its gradients (ebh_op_layer_norm_fwd / _bwd).
#include <algorithm>

#include "layer.hpp"

namespace ebh {

__device__ __forceinline__ float block_sum(float v, float* red) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return red[0] + red[1] + red[2] + red[3];
}

// One workgroup per row; mean first, then the squared deviations from it.
template <class T>
__global__ __launch_bounds__(256) void norm_fwd_kernel(NormArgs p) {
    __shared__ float red[4];
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    T* y = static_cast<T*>(p.y) + row * p.ldy;
    float s = 0.0f, q = 0.0f;
    for (int c = threadIdx.x; c < p.H; c += 256) s += to_f32(x[c]);
    const float mean = block_sum(s, red) / (float)p.H;
    for (int c = threadIdx.x; c < p.H; c += 256) {
        const float d = to_f32(x[c]) - mean;
        q += d * d;
    }
    const float rstd = 1.0f / sqrtf(block_sum(q, red) / (float)p.H + p.eps);
    for (int c = threadIdx.x; c < p.H; c += 256) {
        float v = (to_f32(x[c]) - mean) * rstd;
        if (p.gamma) v *= p.gamma[c];
        if (p.beta) v += p.beta[c];
        store_as(y + c, v);
    }
    if (threadIdx.x == 0) {
        if (p.mean) p.mean[row] = mean;
        if (p.rstd) p.rstd[row] = rstd;
    }
}

// Partial sums of dy xh and dy over one of `chunks` ranges of the rows.
template <class T>
__global__ __launch_bounds__(256) void norm_cols_kernel(NormArgs p, int chunks) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= p.H) return;
    const int r0 = (int)((int64_t)p.rows * blockIdx.y / chunks), r1 = (int)((int64_t)p.rows * (blockIdx.y + 1) / chunks);
    float g = 0.0f, b = 0.0f;
    for (int64_t r = r0; r < r1; ++r) {
        const float dy = to_f32(static_cast<const T*>(p.dy)[r * p.lddy + c]);
        g += dy * ((to_f32(static_cast<const T*>(p.x)[r * p.ldx + c]) - p.mean[r]) * p.rstd[r]);
        b += dy;
    }
    p.partials[(int64_t)blockIdx.y * 2 * p.H + c] = g;
    p.partials[(int64_t)blockIdx.y * 2 * p.H + p.H + c] = b;
}

__global__ __launch_bounds__(256) void norm_sum_kernel(NormArgs p, int chunks) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= p.H) return;
    float g = 0.0f, b = 0.0f;
    for (int k = 0; k < chunks; ++k) {
        g += p.partials[(int64_t)k * 2 * p.H + c];
        b += p.partials[(int64_t)k * 2 * p.H + p.H + c];
    }
    if (p.dgamma) p.dgamma[c] = g;
    if (p.dbeta) p.dbeta[c] = b;
}

template <class T>
__global__ __launch_bounds__(256) void norm_bwd_kernel(NormArgs p) {
    __shared__ float red[4];
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    const T* dy = static_cast<const T*>(p.dy) + row * p.lddy;
    const T* dres = p.dres ? static_cast<const T*>(p.dres) + row * p.lddres : nullptr;
    T* dx = static_cast<T*>(p.dx) + row * p.lddx;
    const float mean = p.mean[row], rstd = p.rstd[row];
    float s = 0.0f, q = 0.0f;
    for (int c = threadIdx.x; c < p.H; c += 256) {
        const float g = to_f32(dy[c]) * (p.gamma ? p.gamma[c] : 1.0f);
        s += g;
        q += g * ((to_f32(x[c]) - mean) * rstd);
    }
    s = block_sum(s, red) / (float)p.H;
    q = block_sum(q, red) / (float)p.H;
    for (int c = threadIdx.x; c < p.H; c += 256) {
        const float g = to_f32(dy[c]) * (p.gamma ? p.gamma[c] : 1.0f);
        const float v = rstd * (g - s - (to_f32(x[c]) - mean) * rstd * q);
        store_as(dx + c, dres ? v + to_f32(dres[c]) : v);
    }
}

static int norm_chunks(int rows) { return std::max(1, std::min(256, rows / 16)); }
int64_t norm_bwd_partials(int rows, int H) { return (int64_t)norm_chunks(rows) * 2 * H; }

template <class T>
static void norm_bwd(const NormArgs& a, hipStream_t s) {
    const unsigned cols = (unsigned)((a.H + 255) / 256);
    const int chunks = norm_chunks(a.rows);
    if (a.dgamma || a.dbeta) {
        hipLaunchKernelGGL((norm_cols_kernel<T>), dim3(cols, chunks), dim3(256), 0, s, a, chunks);
        hipLaunchKernelGGL(norm_sum_kernel, dim3(cols), dim3(256), 0, s, a, chunks);
    }
    if (a.rows > 0) hipLaunchKernelGGL((norm_bwd_kernel<T>), dim3(a.rows), dim3(256), 0, s, a);
}

hipError_t launch_norm_fwd(const NormArgs& a, bool bf16, hipStream_t s) {
    if (bf16) hipLaunchKernelGGL((norm_fwd_kernel<uint16_t>), dim3(a.rows), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((norm_fwd_kernel<float>), dim3(a.rows), dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_norm_bwd(const NormArgs& a, bool bf16, hipStream_t s) {
    if (bf16) norm_bwd<uint16_t>(a, s);
    else norm_bwd<float>(a, s);
    return hipGetLastError();
}

}  // namespace ebh
