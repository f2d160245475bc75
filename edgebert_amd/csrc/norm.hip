// norm.hip -- layer norm and its gradients (ebh_op_layer_norm_fwd / _bwd).
//
// Bound by its bytes: the forward reads a row once and keeps it in registers for
// the mean, the squared deviations from it and the output; the backward reads x
// and dy (and dres) once for dx and for its share of dgamma and dbeta.  A row
// belongs to L lanes (a part of a wave, a wave or a whole workgroup), NV pieces
// of V columns each, 16 bytes where rows and pointers allow it; a persistent
// grid walks the rows with gamma, and the column sums, in registers, and with
// the next row on its way while this one is worked on.
//
// Columns: a workgroup's rows' sums of dy xh and dy meet in LDS, leave as one
// row of partial sums a workgroup, and a second kernel adds those in order: the
// result does not depend on timing.
//
// bf16 rows of 768: forward of 131,072 76 us, 5.3 TB/s; backward of 32,768 with
// dres 38 + 4 us (201 MB).  fp32: 2,161 rows of 384 forward 6.0 us, 1,061 of 769
// back 7.9 + 3.4 us.
#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "layer.hpp"

namespace ebh {

typedef float norm_v4 __attribute__((ext_vector_type(4)));
typedef unsigned int norm_u4 __attribute__((ext_vector_type(4)));

// V columns as they lie in memory: 16 bytes, or one element.
template <class T, int V>
struct Piece {
    typedef std::conditional_t<V == 1, T, norm_u4> Raw;
    Raw w;
    __device__ __forceinline__ void load(const T* p) { w = *reinterpret_cast<const Raw*>(p); }
    __device__ __forceinline__ void zero() { w = Raw{}; }
    __device__ __forceinline__ float get(int e) const {
        if constexpr (V == 1) return to_f32(w);
        else if constexpr (sizeof(T) == 4) return __uint_as_float(w[e]);
        else return __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    }
};
template <class T, int V>
__device__ __forceinline__ void put_piece(T* p, const float* v) {
    if constexpr (V == 1) store_as(p, v[0]);
    else if constexpr (sizeof(T) == 4) *reinterpret_cast<norm_v4*>(p) = norm_v4{v[0], v[1], v[2], v[3]};
    else
        *reinterpret_cast<norm_u4*>(p) = norm_u4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
}

// Sums over the L lanes of a row, the same in each of them; red holds two values a wave.
template <int L>
__device__ __forceinline__ void row_sum(float& a, float& b, float* red) {
#pragma unroll
    for (int o = (L < 64 ? L : 64) / 2; o > 0; o >>= 1) {
        a += __shfl_xor(a, o);
        b += __shfl_xor(b, o);
    }
    if constexpr (L > 64) {
        __syncthreads();                       // the last sums have been read
        if ((threadIdx.x & 63) == 0) {
            red[2 * (threadIdx.x >> 6)] = a;
            red[2 * (threadIdx.x >> 6) + 1] = b;
        }
        __syncthreads();
        a = b = 0.0f;
#pragma unroll
        for (int w = 0; w < L / 64; ++w) {
            a += red[2 * w];
            b += red[2 * w + 1];
        }
    }
}

constexpr int norm_threads(int L) { return L > 256 ? L : 256; }

// Whole workgroups of 1,024 lanes have 128 registers each: no next row, and gamma
// from the caches.
constexpr bool norm_holds(int L) { return L < 1024; }

template <class T, int V, int L, int NV>
__global__ __launch_bounds__(norm_threads(L)) void norm_fwd_kernel(NormArgs p) {
    constexpr int NT = norm_threads(L), R = NT / L, N = NV * V;   // rows of a workgroup, columns of a lane
    __shared__ float red[L > 64 ? L / 32 : 1];
    const int lane = threadIdx.x % L, pieces = p.H / V;
    const T* const x = static_cast<const T*>(p.x);
    T* const y = static_cast<T*>(p.y);
    const float inv = 1.0f / (float)p.H;
    constexpr bool HOLD = norm_holds(L);
    auto gamma = [&](int i, int e) { return lane + i * L < pieces && p.gamma ? p.gamma[(lane + i * L) * V + e] : 1.0f; };
    auto beta = [&](int i, int e) { return lane + i * L < pieces && p.beta ? p.beta[(lane + i * L) * V + e] : 0.0f; };
    float g[HOLD ? N : 1], b[HOLD ? N : 1];
    if constexpr (HOLD) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                g[i * V + e] = gamma(i, e);
                b[i * V + e] = beta(i, e);
            }
    }
    const int64_t stride = (int64_t)gridDim.x * R;
    Piece<T, V> next[NV];
    auto fetch = [&](int64_t row) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (row < p.rows && lane + i * L < pieces) next[i].load(x + row * p.ldx + (lane + i * L) * V);
            else next[i].zero();
        }
    };
    int64_t row = (int64_t)blockIdx.x * R + threadIdx.x / L;
    if (HOLD) fetch(row);
    // Rows of a workgroup go together (its sums have barriers where L > 64)
    for (int64_t row0 = (int64_t)blockIdx.x * R; row0 < p.rows; row0 += stride, row += stride) {
        float v[N];
        if (!HOLD) fetch(row);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) v[i * V + e] = next[i].get(e);
        if (HOLD) fetch(row + stride);
        float s = 0.0f, q = 0.0f, none = 0.0f;
#pragma unroll
        for (int k = 0; k < N; ++k) s += v[k];
        row_sum<L>(s, none, red);
        const float mean = s * inv;
        none = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (lane + i * L < pieces)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    v[i * V + e] -= mean;
                    q = fmaf(v[i * V + e], v[i * V + e], q);
                }
        row_sum<L>(q, none, red);
        const float rstd = 1.0f / sqrtf(q * inv + p.eps);
        if (row < p.rows) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (lane + i * L < pieces) {
                    float o[V];
#pragma unroll
                    for (int e = 0; e < V; ++e) o[e] = fmaf(v[i * V + e] * rstd, HOLD ? g[i * V + e] : gamma(i, e), HOLD ? b[i * V + e] : beta(i, e));
                    put_piece<T, V>(y + row * p.ldy + (lane + i * L) * V, o);
                }
            if (lane == 0) {
                if (p.mean) p.mean[row] = mean;
                if (p.rstd) p.rstd[row] = rstd;
            }
        }
    }
}

template <class T, int V, int L, int NV>
__global__ __launch_bounds__(norm_threads(L)) void norm_bwd_kernel(NormArgs p) {
    constexpr int NT = norm_threads(L), R = NT / L, N = NV * V, W = NT / 64;
    constexpr int LW = L < 64 ? L : 64;             // lanes of a row in a wave
    __shared__ float red[L > 64 ? L / 32 : 1];
    __shared__ float cols[L <= 64 ? W * LW * N : 1];
    const int lane = threadIdx.x % L, pieces = p.H / V;
    const T* const x = static_cast<const T*>(p.x);
    const T* const dy = static_cast<const T*>(p.dy);
    const T* const dres = static_cast<const T*>(p.dres);
    T* const dx = static_cast<T*>(p.dx);
    const float inv = 1.0f / (float)p.H;
    constexpr bool HOLD = norm_holds(L);
    auto gamma = [&](int i, int e) { return lane + i * L < pieces && p.gamma ? p.gamma[(lane + i * L) * V + e] : 1.0f; };
    float g[HOLD ? N : 1], sg[N], sb[N];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if (HOLD) g[i * V + e] = gamma(i, e);
            sg[i * V + e] = sb[i * V + e] = 0.0f;
        }
    const int64_t stride = (int64_t)gridDim.x * R;
    Piece<T, V> nx[NV], ny[NV], nr[NV];
    float nmean = 0.0f, nrstd = 0.0f;
    auto fetch = [&](int64_t row) {
        const bool live = row < p.rows;
        nmean = live ? p.mean[row] : 0.0f;
        nrstd = live ? p.rstd[row] : 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (lane + i * L) * V;
            if (live && lane + i * L < pieces) {
                nx[i].load(x + row * p.ldx + c);
                ny[i].load(dy + row * p.lddy + c);
                if (dres) nr[i].load(dres + row * p.lddres + c);
                else nr[i].zero();
            } else {
                nx[i].zero();
                ny[i].zero();
                nr[i].zero();
            }
        }
    };
    int64_t row = (int64_t)blockIdx.x * R + threadIdx.x / L;
    if (HOLD) fetch(row);
    for (int64_t row0 = (int64_t)blockIdx.x * R; row0 < p.rows; row0 += stride, row += stride) {
        if (!HOLD) fetch(row);
        const float mean = nmean, rstd = nrstd;
        float xh[N], d[N];
        Piece<T, V> r[NV];
        float s = 0.0f, q = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const bool in = lane + i * L < pieces;
            r[i] = nr[i];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int k = i * V + e;
                const float t = ny[i].get(e);
                // columns past the row, and rows past the last, add nothing
                xh[k] = in ? (nx[i].get(e) - mean) * rstd : 0.0f;
                d[k] = t * (HOLD ? g[k] : gamma(i, e));
                sg[k] = fmaf(t, xh[k], sg[k]);
                sb[k] += t;
                s += d[k];
                q = fmaf(d[k], xh[k], q);
            }
        }
        if (HOLD) fetch(row + stride);
        row_sum<L>(s, q, red);
        s *= inv;
        q *= inv;
        if (row < p.rows) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (lane + i * L < pieces) {
                    float o[V];
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const int k = i * V + e;
                        o[e] = rstd * (d[k] - s - xh[k] * q);
                        if (dres) o[e] += r[i].get(e);
                    }
                    put_piece<T, V>(dx + row * p.lddx + (lane + i * L) * V, o);
                }
        }
    }
    if (p.partials) {
        float* const out = p.partials + (int64_t)blockIdx.x * 2 * p.H;
        auto leave = [&](float* v, float* to) {
            if constexpr (L <= 64) {
                // the rows of a wave, then the waves
#pragma unroll
                for (int k = 0; k < N; ++k)
#pragma unroll
                    for (int o = L; o < 64; o <<= 1) v[k] += __shfl_xor(v[k], o);
                __syncthreads();
                if ((threadIdx.x & 63) < LW) {
#pragma unroll
                    for (int i = 0; i < NV; ++i)
#pragma unroll
                        for (int e = 0; e < V; ++e) cols[((threadIdx.x >> 6) * NV * LW + i * L + lane) * V + e] = v[i * V + e];
                }
                __syncthreads();
                for (int c = threadIdx.x; c < p.H; c += NT) {
                    float t = 0.0f;
#pragma unroll
                    for (int w = 0; w < W; ++w) t += cols[w * NV * LW * V + c];
                    to[c] = t;
                }
            } else {
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    if (lane + i * L < pieces)
#pragma unroll
                        for (int e = 0; e < V; ++e) to[(lane + i * L) * V + e] = v[i * V + e];
            }
        };
        leave(sg, out);
        leave(sb, out + p.H);
    }
}

// dgamma and dbeta from `parts` rows of [dgamma | dbeta] partial sums: 64 columns
// and 16 slices of the rows a workgroup.
__global__ __launch_bounds__(1024) void norm_cols_kernel(const float* partials, int parts, int H, float* dgamma, float* dbeta) {
    __shared__ float part[16][64];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), slice = threadIdx.x >> 6;
    float s = 0.0f;
    if (c < 2 * H) {
#pragma unroll 8
        for (int r = slice; r < parts; r += 16) s += partials[(int64_t)r * 2 * H + c];
    }
    part[slice][threadIdx.x & 63] = s;
    __syncthreads();
    if (slice == 0 && c < 2 * H) {
        s = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) s += part[i][threadIdx.x & 63];
        float* const out = c < H ? dgamma : dbeta;
        if (out) out[c < H ? c : c - H] = s;
    }
}

// Workgroups of the backward: two a CU, at least a few rows each.
static int bwd_blocks(int rows, int H) {
    const int rows_each = H > 1024 ? 1 : 4;          // at once, or more
    return (int)std::max<int64_t>(1, std::min<int64_t>(512, ((int64_t)rows + rows_each - 1) / rows_each));
}
int64_t norm_bwd_partials(int rows, int H) { return (int64_t)bwd_blocks(rows, H) * 2 * H; }

template <class T, int V, int L, int NV>
struct NormLaunch {
    static void fwd(const NormArgs& a, hipStream_t s) {
        constexpr int NT = norm_threads(L), R = NT / L;
        // a few workgroups a CU, so that gamma is read once for many rows
        const int64_t blocks = std::min<int64_t>(((int64_t)a.rows + R - 1) / R, NT == 256 ? 2048 : 512);
        hipLaunchKernelGGL((norm_fwd_kernel<T, V, L, NV>), dim3((unsigned)blocks), dim3(NT), 0, s, a);
    }
    static void bwd(const NormArgs& a, hipStream_t s) {
        hipLaunchKernelGGL((norm_bwd_kernel<T, V, L, NV>), dim3(bwd_blocks(a.rows, a.H)), dim3(norm_threads(L)), 0, s, a);
    }
};

// f(NormLaunch<T, V, L, NV>) of the first L lanes and NV pieces that hold a row: as
// few lanes as can, so that every lane of a wave has loads on its way, of at most
// 16 columns each (24 in bf16 rows of a wave or less, whose loads are few).
template <class T, int V, int L, int NV, int... REST, class F>
static void with_lanes(int H, F&& f) {
    if constexpr (sizeof...(REST) == 0) {
        f(NormLaunch<T, V, L, NV>{});
    } else {
        if (H <= L * NV * V) f(NormLaunch<T, V, L, NV>{});
        else with_lanes<T, V, REST...>(H, f);
    }
}
template <class T, class F>
static void with_row(int H, bool wide, F&& f) {
    if (!wide) with_lanes<T, 1, 16, 16, 64, 8, 64, 16, 256, 8, 256, 16, 1024, 8>(H, f);
    else if constexpr (sizeof(T) == 2) with_lanes<T, 8, 16, 1, 16, 2, 16, 3, 32, 2, 32, 3, 64, 2, 64, 3, 256, 1, 256, 2, 1024, 1>(H, f);
    else with_lanes<T, 4, 16, 1, 16, 2, 16, 4, 32, 3, 32, 4, 64, 3, 64, 4, 256, 2, 256, 4, 1024, 2>(H, f);
}

template <class T>
static bool whole_pieces(const NormArgs& a, std::initializer_list<const void*> rows, std::initializer_list<int64_t> strides) {
    constexpr int V = 16 / sizeof(T);
    if (a.H % V) return false;
    for (const void* q : rows)
        if ((uintptr_t)q & 15) return false;
    for (int64_t ld : strides)
        if (ld % V) return false;
    return true;
}

template <class T>
static void norm_fwd(const NormArgs& a, hipStream_t s) {
    auto f = [&](auto l) { l.fwd(a, s); };
    with_row<T>(a.H, whole_pieces<T>(a, {a.x, a.y}, {a.ldx, a.ldy}), f);
}

template <class T>
static void norm_bwd(NormArgs a, hipStream_t s) {
    if (!a.dgamma && !a.dbeta) a.partials = nullptr;
    auto f = [&](auto l) { l.bwd(a, s); };
    if (a.rows > 0) with_row<T>(a.H, whole_pieces<T>(a, {a.x, a.dy, a.dx, a.dres}, {a.ldx, a.lddy, a.lddx, a.dres ? a.lddres : 0}), f);
    if (a.partials)
        hipLaunchKernelGGL(norm_cols_kernel, dim3((unsigned)((2 * a.H + 63) / 64)), dim3(1024), 0, s, a.partials,
                           a.rows > 0 ? bwd_blocks(a.rows, a.H) : 0, a.H, a.dgamma, a.dbeta);
}

hipError_t launch_norm_fwd(const NormArgs& a, bool bf16, hipStream_t s) {
    if (bf16) norm_fwd<uint16_t>(a, s);
    else norm_fwd<float>(a, s);
    return hipGetLastError();
}

hipError_t launch_norm_bwd(const NormArgs& a, bool bf16, hipStream_t s) {
    if (bf16) norm_bwd<uint16_t>(a, s);
    else norm_bwd<float>(a, s);
    return hipGetLastError();
}

}  // namespace ebh
