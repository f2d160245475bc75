// layer_ops.cpp -- op-level entry points of edgebert_hip_ops.h for rotary
// positions, layer norm with gradients and the gated feed-forward block:
// argument checks and workspace sizes; the kernels are in rope.hip, norm.hip
// and gated.hip.
#include <cmath>

#include "../../include/edgebert_hip.h"
#include "../../include/edgebert_hip_ops.h"
#include "internal.hpp"
#include "layer.hpp"

namespace {

using ebh::set_error;
#define fail set_error

#define LAUNCH_TRY(expr)                                                                 \
    do {                                                                                 \
        hipError_t e_ = (expr);                                                          \
        if (e_ != hipSuccess) return fail(EBH_ERR_HIP, "%s failed: %s", #expr, hipGetErrorString(e_)); \
    } while (0)

bool known_dtype(int32_t dtype) { return dtype == EBH_DTYPE_F32 || dtype == EBH_DTYPE_BF16; }
bool aligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; }
uintptr_t element(int32_t dtype) { return dtype == EBH_DTYPE_BF16 ? 2 : 4; }

constexpr int32_t kNormMaxH = 8192, kFfnMaxDim = 65536, kFfnMaxRows = 1 << 30;
constexpr int32_t kRopeMaxT = 1 << 26;   // 2^23 workgroups of 256 lanes: a grid has less than 2^32

int check_ffn(int32_t M, int32_t H, int32_t I, int32_t dtype) {
    if (!known_dtype(dtype)) return fail(EBH_ERR_INVALID_ARG, "unknown dtype %d", dtype);
    if (M < 0 || M > kFfnMaxRows || H <= 0 || I <= 0 || H % 8 || I % 8 || H > kFfnMaxDim || I > kFfnMaxDim)
        return fail(EBH_ERR_INVALID_ARG, "bad FFN shape: M %d (at most %d), H %d, I %d (multiples of 8, at most %d)", M, kFfnMaxRows,
                    H, I, kFfnMaxDim);
    if (2 * (int64_t)H * I * (int64_t)element(dtype) >= 0xFFFF0000ll)   // 32-bit offsets within the weights
        return fail(EBH_ERR_INVALID_ARG, "FFN weights too large: 2 H I = %lld elements", 2 * (long long)H * I);
    return EBH_OK;
}

int check_ffn_stride(const char* name, int64_t ld, int32_t H) {
    if (ld < H || ld % 8 || ld > ebh::gemm_stride_max(4))
        return fail(EBH_ERR_INVALID_ARG, "%s %lld: a multiple of 8, at least %d and at most %lld", name, (long long)ld, H,
                    (long long)ebh::gemm_stride_max(4));
    return EBH_OK;
}

int check_workspace(const void* workspace, int64_t have, int64_t need) {
    if (need > 0 && (!workspace || have < need || !aligned(workspace, 16)))
        return fail(EBH_ERR_INVALID_ARG, "workspace of %lld bytes, 16-byte aligned, needed (got %lld at %p)", (long long)need,
                    (long long)have, workspace);
    return EBH_OK;
}

}  // namespace

extern "C" {

int ebh_op_rope(const void* x, int64_t ldx, void* y, int64_t ldy, int32_t dtype, const int32_t* pos,
                const int32_t* n_tokens, int32_t T, int32_t n_heads, int32_t head_dim, const ebh_rope* cfg,
                int32_t transpose, void* stream) {
    if (!cfg) return fail(EBH_ERR_INVALID_ARG, "null rope config");
    if (!known_dtype(dtype)) return fail(EBH_ERR_INVALID_ARG, "unknown dtype %d", dtype);
    if (T < 0 || T > kRopeMaxT || n_heads <= 0 || n_heads > 65536 || head_dim <= 0 || head_dim > 1024)
        return fail(EBH_ERR_INVALID_ARG, "bad rope shape: T %d (at most %d), %d heads of %d", T, kRopeMaxT, n_heads, head_dim);
    const ebh_rope& c = *cfg;
    if (c.rot_dim < 2 || c.rot_dim % 2 || c.rot_dim > head_dim)
        return fail(EBH_ERR_INVALID_ARG, "rot_dim %d: even, 2 .. head_dim %d", c.rot_dim, head_dim);
    if (c.layout != EBH_ROPE_HALF && c.layout != EBH_ROPE_INTERLEAVED)
        return fail(EBH_ERR_INVALID_ARG, "unknown rope layout %d", c.layout);
    if (c.scaling < EBH_ROPE_NONE || c.scaling > EBH_ROPE_WAVELENGTH)
        return fail(EBH_ERR_INVALID_ARG, "unknown rope scaling %d", c.scaling);
    if (!(c.base > 0.0) || !std::isfinite(c.base) || !std::isfinite(c.magnitude))
        return fail(EBH_ERR_INVALID_ARG, "rope base must be positive, base and magnitude finite");
    if (c.scaling != EBH_ROPE_NONE && (!(c.factor > 0.0) || !std::isfinite(c.factor)))
        return fail(EBH_ERR_INVALID_ARG, "rope factor must be positive and finite");
    if (c.scaling == EBH_ROPE_WAVELENGTH &&
        (c.original_len <= 0 || !std::isfinite(c.turns_fast) || !std::isfinite(c.turns_slow) || !(c.turns_fast > c.turns_slow)))
        return fail(EBH_ERR_INVALID_ARG, "rope by wavelength needs original_len > 0 and turns_fast > turns_slow");
    if (T == 0) return EBH_OK;
    const int64_t cols = (int64_t)n_heads * head_dim;
    if (!x || !y || !pos) return fail(EBH_ERR_INVALID_ARG, "null buffer");
    if (ldx < cols || ldy < cols) return fail(EBH_ERR_INVALID_ARG, "row strides must cover %lld columns", (long long)cols);
    if (!aligned(x, element(dtype)) || !aligned(y, element(dtype)) || !aligned(pos, 4) || !aligned(n_tokens, 4))
        return fail(EBH_ERR_INVALID_ARG, "operands must be aligned to their elements");
    if (x == y && ldx != ldy) return fail(EBH_ERR_INVALID_ARG, "in place, ldx and ldy must be the same");
    ebh::RopeArgs a{};
    a.x = x;
    a.y = y;
    a.ldx = ldx;
    a.ldy = ldy;
    a.pos = pos;
    a.n_dev = n_tokens;
    a.T = T;
    a.n = n_heads;
    a.d = head_dim;
    a.rot = c.rot_dim;
    a.layout = c.layout;
    a.scaling = c.scaling;
    a.transpose = transpose != 0;
    a.log2_base = std::log2(c.base);
    a.inv_factor = 1.0;
    a.magnitude = c.magnitude;
    if (c.scaling == EBH_ROPE_NTK) {
        // a single pair has frequency 1 whatever the base
        if (c.rot_dim > 2) a.log2_base += std::log2(c.factor) * c.rot_dim / (c.rot_dim - 2);
    } else if (c.scaling != EBH_ROPE_NONE) {
        a.inv_factor = 1.0 / c.factor;
    }
    if (c.scaling == EBH_ROPE_WAVELENGTH) {
        a.turns = c.original_len / 6.283185307179586;
        a.slow = c.turns_slow;
        a.inv_span = 1.0 / (c.turns_fast - c.turns_slow);
    }
    LAUNCH_TRY(ebh::launch_rope(a, dtype == EBH_DTYPE_BF16, static_cast<hipStream_t>(stream)));
    return EBH_OK;
}

int ebh_op_layer_norm_fwd(const void* x, int64_t ldx, int32_t dtype, const float* gamma, const float* beta,
                          int32_t rows, int32_t H, float eps, void* y, int64_t ldy, float* mean, float* rstd,
                          void* stream) {
    if (!known_dtype(dtype)) return fail(EBH_ERR_INVALID_ARG, "unknown dtype %d", dtype);
    if (rows < 0 || H <= 0 || H > kNormMaxH) return fail(EBH_ERR_INVALID_ARG, "bad LayerNorm shape: %d rows of %d", rows, H);
    if (!(eps >= 0.0f)) return fail(EBH_ERR_INVALID_ARG, "LayerNorm eps must not be negative");
    if (rows == 0) return EBH_OK;
    if (!x || !y) return fail(EBH_ERR_INVALID_ARG, "null buffer");
    if (ldx < H || ldy < H || (x == y && ldx != ldy))
        return fail(EBH_ERR_INVALID_ARG, "row strides must cover H, and be the same in place");
    const uintptr_t e = element(dtype);
    if (!aligned(x, e) || !aligned(y, e) || !aligned(gamma, 4) || !aligned(beta, 4) || !aligned(mean, 4) || !aligned(rstd, 4))
        return fail(EBH_ERR_INVALID_ARG, "operands must be aligned to their elements");
    ebh::NormArgs a{};
    a.x = x;
    a.ldx = ldx;
    a.y = y;
    a.ldy = ldy;
    a.gamma = gamma;
    a.beta = beta;
    a.mean = mean;
    a.rstd = rstd;
    a.rows = rows;
    a.H = H;
    a.eps = eps;
    LAUNCH_TRY(ebh::launch_norm_fwd(a, dtype == EBH_DTYPE_BF16, static_cast<hipStream_t>(stream)));
    return EBH_OK;
}

int64_t ebh_op_layer_norm_bwd_workspace(int32_t rows, int32_t H) {
    if (rows < 0 || H <= 0 || H > kNormMaxH) return fail(EBH_ERR_INVALID_ARG, "bad LayerNorm shape: %d rows of %d", rows, H);
    return ebh::norm_bwd_partials(rows, H) * 4;
}

int ebh_op_layer_norm_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, int32_t dtype,
                          const float* gamma, const float* mean, const float* rstd, const void* dres,
                          int64_t lddres, int32_t rows, int32_t H, void* dx, int64_t lddx, float* dgamma,
                          float* dbeta, void* workspace, int64_t workspace_bytes, void* stream) {
    if (!known_dtype(dtype)) return fail(EBH_ERR_INVALID_ARG, "unknown dtype %d", dtype);
    if (rows < 0 || H <= 0 || H > kNormMaxH) return fail(EBH_ERR_INVALID_ARG, "bad LayerNorm shape: %d rows of %d", rows, H);
    if (!aligned(dgamma, 4) || !aligned(dbeta, 4))
        return fail(EBH_ERR_INVALID_ARG, "operands must be aligned to their elements");
    if (rows > 0) {
        if (!dy || !x || !mean || !rstd || !dx) return fail(EBH_ERR_INVALID_ARG, "null buffer");
        if (lddy < H || ldx < H || lddx < H || (dres && lddres < H) || (dx == dy && lddx != lddy) || (dx == x && lddx != ldx) ||
            (dres && dx == dres && lddx != lddres))
            return fail(EBH_ERR_INVALID_ARG, "row strides must cover H, and be the same in place");
        const uintptr_t e = element(dtype);
        if (!aligned(dy, e) || !aligned(x, e) || !aligned(dres, e) || !aligned(dx, e) || !aligned(gamma, 4) ||
            !aligned(mean, 4) || !aligned(rstd, 4))
            return fail(EBH_ERR_INVALID_ARG, "operands must be aligned to their elements");
    }
    if (dgamma || dbeta) {
        const int rc = check_workspace(workspace, workspace_bytes, ebh::norm_bwd_partials(rows, H) * 4);
        if (rc) return rc;
    }
    if (rows == 0 && !dgamma && !dbeta) return EBH_OK;
    ebh::NormArgs a{};
    a.x = x;
    a.ldx = ldx;
    a.dy = dy;
    a.lddy = lddy;
    a.dres = dres;
    a.lddres = lddres;
    a.dx = dx;
    a.lddx = lddx;
    a.gamma = gamma;
    a.mean = const_cast<float*>(mean);
    a.rstd = const_cast<float*>(rstd);
    a.rows = rows;
    a.H = H;
    a.dgamma = dgamma;
    a.dbeta = dbeta;
    a.partials = static_cast<float*>(workspace);
    LAUNCH_TRY(ebh::launch_norm_bwd(a, dtype == EBH_DTYPE_BF16, static_cast<hipStream_t>(stream)));
    return EBH_OK;
}

int64_t ebh_op_gated_ffn_workspace(int32_t M, int32_t H, int32_t I, int32_t dtype) {
    const int rc = check_ffn(M, H, I, dtype);
    return rc ? rc : ebh::gated_ws_bytes(M, H, I, dtype == EBH_DTYPE_BF16);
}

int ebh_op_gated_ffn(const void* X, int64_t ldx, const void* Wgu, const float* bgu, const void* Wd,
                     const float* bd, void* Y, int64_t ldy, void* h, void* gu, int32_t M, int32_t H, int32_t I,
                     int32_t act, int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream) {
    int rc = check_ffn(M, H, I, dtype);
    if (rc) return rc;
    if (act < EBH_ACT_SILU || act > EBH_ACT_GELU_ERF) return fail(EBH_ERR_INVALID_ARG, "unknown activation %d", act);
    if (M == 0) return EBH_OK;
    if (!X || !Wgu || !Wd || !Y || !h) return fail(EBH_ERR_INVALID_ARG, "null buffer");
    if ((rc = check_ffn_stride("ldx", ldx, H)) || (rc = check_ffn_stride("ldy", ldy, H))) return rc;
    for (const void* p : {X, Wgu, (const void*)bgu, Wd, (const void*)bd, (const void*)Y, (const void*)h, (const void*)gu})
        if (!aligned(p, 16)) return fail(EBH_ERR_INVALID_ARG, "operands must be 16-byte aligned");
    const bool bf16 = dtype == EBH_DTYPE_BF16;
    if ((rc = check_workspace(workspace, workspace_bytes, ebh::gated_ws_bytes(M, H, I, bf16)))) return rc;
    ebh::GatedArgs a{};
    a.X = X;
    a.ldx = ldx;
    a.Wgu = Wgu;
    a.bgu = bgu;
    a.Wd = Wd;
    a.bd = bd;
    a.Y = Y;
    a.ldy = ldy;
    a.h = h;
    a.gu = gu;
    a.M = M;
    a.H = H;
    a.I = I;
    a.act = act;
    a.ws = workspace;
    LAUNCH_TRY(ebh::launch_gated(a, bf16, static_cast<hipStream_t>(stream)));
    return EBH_OK;
}

int64_t ebh_op_gated_ffn_bwd_workspace(int32_t M, int32_t H, int32_t I, int32_t dtype) {
    const int rc = check_ffn(M, H, I, dtype);
    return rc ? rc : ebh::gated_bwd_ws_bytes(M, H, I, dtype == EBH_DTYPE_BF16);
}

int ebh_op_gated_ffn_bwd(const void* dY, int64_t lddy, const void* X, int64_t ldx, const void* h, const void* gu,
                         const void* Wgu, const void* Wd, void* dX, int64_t lddx, void* dWgu, float* dbgu,
                         void* dWd, float* dbd, int32_t M, int32_t H, int32_t I, int32_t act, int32_t dtype,
                         void* workspace, int64_t workspace_bytes, void* stream) {
    int rc = check_ffn(M, H, I, dtype);
    if (rc) return rc;
    if (act < EBH_ACT_SILU || act > EBH_ACT_GELU_ERF) return fail(EBH_ERR_INVALID_ARG, "unknown activation %d", act);
    for (const void* p : {(const void*)dX, (const void*)dWgu, (const void*)dbgu, (const void*)dWd, (const void*)dbd})
        if (!aligned(p, 16)) return fail(EBH_ERR_INVALID_ARG, "operands must be 16-byte aligned");
    const bool bf16 = dtype == EBH_DTYPE_BF16;
    if (M > 0) {
        if (!dY || !X || !h || !gu || !Wgu || !Wd) return fail(EBH_ERR_INVALID_ARG, "null buffer");
        if ((rc = check_ffn_stride("lddy", lddy, H)) || (rc = check_ffn_stride("ldx", ldx, H)) ||
            (dX && (rc = check_ffn_stride("lddx", lddx, H))))
            return rc;
        for (const void* p : {dY, X, h, gu, Wgu, Wd})
            if (!aligned(p, 16)) return fail(EBH_ERR_INVALID_ARG, "operands must be 16-byte aligned");
        if ((rc = check_workspace(workspace, workspace_bytes, ebh::gated_bwd_ws_bytes(M, H, I, bf16)))) return rc;
    }
    if (M == 0 && !dWgu && !dbgu && !dWd && !dbd) return EBH_OK;
    ebh::GatedArgs a{};
    a.dY = dY;
    a.lddy = lddy;
    a.X = X;
    a.ldx = ldx;
    a.h = const_cast<void*>(h);
    a.gu = const_cast<void*>(gu);
    a.Wgu = Wgu;
    a.Wd = Wd;
    a.dX = dX;
    a.lddx = lddx;
    a.dWgu = dWgu;
    a.dbgu = dbgu;
    a.dWd = dWd;
    a.dbd = dbd;
    a.M = M;
    a.H = H;
    a.I = I;
    a.act = act;
    a.ws = workspace;
    LAUNCH_TRY(ebh::launch_gated_bwd(a, bf16, static_cast<hipStream_t>(stream)));
    return EBH_OK;
}

}  // extern "C"
