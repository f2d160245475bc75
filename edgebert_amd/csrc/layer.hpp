// layer.hpp -- launchers of what a rotary, gated encoder layer adds: rotary
// positions (rope.hip), layer norm with gradients (norm.hip) and the gated
// feed-forward block with gradients (gated.hip).  Arguments are checked by
// layer_ops.cpp.
#pragma once
#include "kernels.hpp"

namespace ebh {

struct RopeArgs {
    const void* x;
    void* y;
    int64_t ldx, ldy;
    const int* pos;
    const int* n_dev;   // actual tokens, read on device (nullptr: T)
    int T, n, d, rot, layout, scaling;
    int transpose;
    // log2 of the base (after NTK scaling), 1 / factor, turns of a unit
    // frequency over the original length, and the ends of the ramp
    double log2_base, inv_factor, turns, slow, inv_span, magnitude;
};
hipError_t launch_rope(const RopeArgs& a, bool bf16, hipStream_t s);

struct NormArgs {
    const void* x;
    void* y;            // forward
    const void* dy;     // backward
    const void* dres;
    void* dx;
    int64_t ldx, ldy, lddy, lddres, lddx;
    const float* gamma;
    const float* beta;
    float* mean;        // written by the forward, read by the backward
    float* rstd;
    int rows, H;
    float eps;
    float* dgamma;
    float* dbeta;
    float* partials;    // norm_bwd_partials floats
};
int64_t norm_bwd_partials(int rows, int H);
hipError_t launch_norm_fwd(const NormArgs& a, bool bf16, hipStream_t s);
hipError_t launch_norm_bwd(const NormArgs& a, bool bf16, hipStream_t s);

struct GatedArgs {
    const void* X;
    const void* Wgu;    // [2 I, H]
    const void* Wd;     // [H, I]
    const float* bgu;
    const float* bd;
    void* Y;
    void* h;            // [M, I]
    void* gu;           // [M, 2 I]
    const void* dY;
    void* dX;
    void* dWgu;
    void* dWd;
    float* dbgu;
    float* dbd;
    int64_t ldx, ldy, lddy, lddx;
    int M, H, I, act;
    void* ws;
};
int64_t gated_ws_bytes(int M, int H, int I, bool bf16);
int64_t gated_bwd_ws_bytes(int M, int H, int I, bool bf16);
hipError_t launch_gated(const GatedArgs& a, bool bf16, hipStream_t s);
hipError_t launch_gated_bwd(const GatedArgs& a, bool bf16, hipStream_t s);

// ---------------------------------------------------------------------------
// device helpers
// ---------------------------------------------------------------------------
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
__device__ __forceinline__ void store_as(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_as(uint16_t* p, float v) { *p = f32_to_bf16_rne(v); }

}  // namespace ebh
