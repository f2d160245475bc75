// rope.hip -- rotary positions over packed rows (ebh_op_rope).
#include <algorithm>

#include "layer.hpp"

namespace ebh {

// cos and sin, times the magnitude, of pair i's angle at position pos.  The
// angle is formed in turns, in 64 bits: a 32-bit product pos * f is off by
// pos * f * 2^-24, 0.004 of a radian at position 65,536.
__device__ __forceinline__ float2 rope_angle(const RopeArgs& p, int i, int pos) {
    double f = exp2(-2.0 * i / p.rot * p.log2_base);
    if (p.scaling == 1) {
        f *= p.inv_factor;
    } else if (p.scaling == 3) {
        double g = (p.turns * f - p.slow) * p.inv_span;
        g = g < 0.0 ? 0.0 : (g > 1.0 ? 1.0 : g);
        f *= g + (1.0 - g) * p.inv_factor;
    }
    const double turns = (double)pos * f * 0.15915494309189535;   // 1 / (2 pi)
    const double q = rint(4.0 * turns);                            // quarter turns
    float s, c;
    sincospif((float)(2.0 * (turns - 0.25 * q)), &s, &c);          // |argument| <= 1/4
    const int quarter = (int)(q - 4.0 * floor(0.25 * q));
    float2 r = quarter == 0 ? make_float2(c, s) : (quarter == 1 ? make_float2(-s, c) : (quarter == 2 ? make_float2(-c, -s) : make_float2(s, -c)));
    if (p.transpose) r.y = -r.y;
    return make_float2((float)(r.x * p.magnitude), (float)(r.y * p.magnitude));
}

// One thread per pair of columns, or per two columns that pass.
template <class T>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs p) {
    const int tokens = p.n_dev ? min(p.T, *p.n_dev) : p.T;
    const int half = p.rot / 2, per = half + (p.d - p.rot + 1) / 2;
    const int64_t id = blockIdx.x * (int64_t)256 + threadIdx.x;
    const int64_t t = id / ((int64_t)per * p.n);
    if (t >= tokens) return;
    const int rem = (int)(id - t * per * p.n), head = rem / per, i = rem - head * per;
    const T* x = static_cast<const T*>(p.x) + t * p.ldx + (int64_t)head * p.d;
    T* y = static_cast<T*>(p.y) + t * p.ldy + (int64_t)head * p.d;
    if (i >= half) {
        for (int c = p.rot + 2 * (i - half); c < min(p.d, p.rot + 2 * (i - half) + 2); ++c) y[c] = x[c];
        return;
    }
    const float2 cs = rope_angle(p, i, p.pos[t]);
    const int ca = p.layout ? 2 * i : i, cb = p.layout ? 2 * i + 1 : i + half;
    const float a = to_f32(x[ca]), b = to_f32(x[cb]);
    store_as(y + ca, a * cs.x - b * cs.y);
    store_as(y + cb, a * cs.y + b * cs.x);
}

hipError_t launch_rope(const RopeArgs& a, bool bf16, hipStream_t s) {
    const int64_t n = (int64_t)a.T * a.n * (a.rot / 2 + (a.d - a.rot + 1) / 2), blocks = (n + 255) / 256;
    if (blocks > 0x7fffffff) return hipErrorInvalidValue;
    if (bf16) hipLaunchKernelGGL((rope_kernel<uint16_t>), dim3((unsigned)blocks), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((rope_kernel<float>), dim3((unsigned)blocks), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace ebh
