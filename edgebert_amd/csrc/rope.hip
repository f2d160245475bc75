// rope.hip -- rotary positions over packed rows (ebh_op_rope).
//
// Bound by its bytes: each head's columns are read and written once.  What is
// left to get right is the angles' cost and where they come from.  They are the
// same for every head of a token, so a workgroup takes a few tokens, forms each
// angle's cos and sin once into LDS and then streams the tokens' rows past them,
// 16 bytes of each half (or 16 bytes of pairs) a lane, neighbouring lanes on
// neighbouring columns.  The first columns are on their way while the angles
// are formed.  32,768 tokens of 24 heads of 64 in bf16: 43 us, 4.7 TB/s (a copy
// of 1 GiB reaches 4.8); 16 tokens: 3.2 us.
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

typedef float rope_v4 __attribute__((ext_vector_type(4)));

// V columns as floats, by one access.
template <class T, int V>
struct RopeVec {
    float v[V];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (V == 1) {
            v[0] = to_f32(*p);
        } else if constexpr (sizeof(T) == 4) {
            const rope_v4 w = *reinterpret_cast<const rope_v4*>(p);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = w[e];
        } else {
            const uint4 w = *reinterpret_cast<const uint4*>(p);
            const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[2 * e] = __uint_as_float(u[e] << 16);
                v[2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u);
            }
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (V == 1) {
            store_as(p, v[0]);
        } else if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<rope_v4*>(p) = rope_v4{v[0], v[1], v[2], v[3]};
        } else {
            *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
        }
    }
};

// A quotient by a divisor known on the host: floor(n / d) = n m >> 32 for n d < 2^32,
// m = ceil(2^32 / d).  Here n < 8 tokens * 256 heads * d, d <= 1,024.
struct RopeDiv {
    uint32_t d, m;
};
static RopeDiv rope_div(uint32_t d) { return RopeDiv{d, (uint32_t)(((uint64_t)1 << 32) / d + (((uint64_t)1 << 32) % d != 0))}; }
__device__ __forceinline__ uint32_t quotient(uint32_t n, const RopeDiv& d) { return d.d == 1 ? n : __umulhi(n, d.m); }

struct RopeGrid {
    int tokens;        // of a workgroup
    int heads;         // of a workgroup (blockIdx.y takes the next ones)
    RopeDiv half, chunks, pass;   // pairs of a token, V-wide chunks of them in a head, V-wide chunks that pass
};

// LAYOUT as ebh_rope's.  V columns a chunk; half layout: V pairs from two accesses,
// interleaved: V / 2 pairs from one (V 1: one pair from two).
template <class T, int LAYOUT, int V>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs p, RopeGrid g) {
    extern __shared__ float2 cs[];     // [tokens][half]
    const int n_tokens = p.n_dev ? min(p.T, *p.n_dev) : p.T;
    const int t0 = blockIdx.x * g.tokens, nt = min(g.tokens, n_tokens - t0);
    if (nt <= 0) return;
    const int h0 = blockIdx.y * g.heads, nh = min(g.heads, p.n - h0), half = p.rot / 2;
    constexpr bool TWO = LAYOUT == 0 || V == 1;    // a chunk is two accesses
    const T* const x = static_cast<const T*>(p.x) + (int64_t)t0 * p.ldx + (int64_t)h0 * p.d;
    T* const y = static_cast<T*>(p.y) + (int64_t)t0 * p.ldy + (int64_t)h0 * p.d;
    const uint32_t per_token = g.chunks.d * nh, items = per_token * nt;

    struct Place {
        int64_t a, b;          // columns of the chunk's accesses, from x's rows
        int64_t ya;
        int at;                // its first pair's angle
    };
    auto place = [&](uint32_t id) {
        const uint32_t row = quotient(id, g.chunks);          // token and head
        const uint32_t c = id - row * g.chunks.d;
        const uint32_t t = row / (uint32_t)nh, head = row - t * nh;
        Place l;
        const int64_t first = (int64_t)head * p.d + (LAYOUT == 0 ? c * V : (V == 1 ? 2 * c : c * V));
        l.a = t * p.ldx + first;
        l.ya = t * p.ldy + first;
        l.b = LAYOUT == 0 ? half : 1;
        l.at = (int)t * half + (LAYOUT == 0 ? c * V : (V == 1 ? c : c * (V / 2)));
        return l;
    };
    constexpr int AHEAD = V == 1 ? 1 : 2;          // chunks on their way before the angles are there
    RopeVec<T, V> a[AHEAD], b[AHEAD];
    Place at[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
        const uint32_t id = threadIdx.x + k * 256;
        if (id < items) {
            at[k] = place(id);
            a[k].load(x + at[k].a);
            if (TWO) b[k].load(x + at[k].a + at[k].b);
        }
    }
    for (uint32_t id = threadIdx.x; id < (uint32_t)(nt * half); id += 256) {
        const uint32_t t = quotient(id, g.half);
        cs[id] = rope_angle(p, (int)(id - t * half), p.pos[t0 + t]);
    }
    __syncthreads();
    auto turn = [&](RopeVec<T, V>& u, RopeVec<T, V>& w, const Place& l) {
        if constexpr (TWO) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float2 r = cs[l.at + e];
                const float ux = u.v[e], wx = w.v[e];
                u.v[e] = ux * r.x - wx * r.y;
                w.v[e] = ux * r.y + wx * r.x;
            }
            u.store(y + l.ya);
            w.store(y + l.ya + l.b);
        } else {
#pragma unroll
            for (int e = 0; e < V / 2; ++e) {
                const float2 r = cs[l.at + e];
                const float ux = u.v[2 * e], wx = u.v[2 * e + 1];
                u.v[2 * e] = ux * r.x - wx * r.y;
                u.v[2 * e + 1] = ux * r.y + wx * r.x;
            }
            u.store(y + l.ya);
        }
    };
    for (uint32_t id0 = threadIdx.x; id0 < items; id0 += 256 * AHEAD) {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const uint32_t id = id0 + k * 256, nx = id + 256 * AHEAD;
            if (id >= items) break;
            RopeVec<T, V> u = a[k], w = b[k];
            const Place l = at[k];
            if (nx < items) {
                at[k] = place(nx);
                a[k].load(x + at[k].a);
                if (TWO) b[k].load(x + at[k].a + at[k].b);
            }
            turn(u, w, l);
        }
    }
    if (p.x != p.y && p.rot < p.d) {               // columns that pass
        const uint32_t n = g.pass.d * nh * nt;
        for (uint32_t id = threadIdx.x; id < n; id += 256) {
            const uint32_t row = quotient(id, g.pass), c = id - row * g.pass.d, t = row / (uint32_t)nh, head = row - t * nh;
            const int64_t col = (int64_t)head * p.d + p.rot + (int64_t)c * V;
            if constexpr (V > 1) *reinterpret_cast<uint4*>(y + t * p.ldy + col) = *reinterpret_cast<const uint4*>(x + t * p.ldx + col);
            else y[t * p.ldy + col] = x[t * p.ldx + col];
        }
    }
}

template <class T, int LAYOUT, int V>
static void launch(const RopeArgs& a, hipStream_t s) {
    const int half = a.rot / 2;
    RopeGrid g;
    // 8 tokens a workgroup where that leaves a few workgroups for every CU, fewer
    // down to one; then heads are shared out too, at least 256 chunks of them,
    // since every workgroup forms its tokens' angles anew
    const int64_t want = 4 * (int64_t)device_cu_count();
    const int chunks = LAYOUT == 0 || V == 1 ? half / (V == 1 ? 1 : V) : a.rot / V;
    g.tokens = (int)std::max<int64_t>(1, std::min<int64_t>(8, a.T / want));
    const int blocks_t = (a.T + g.tokens - 1) / g.tokens;
    const int least = std::max(1, 256 / chunks);
    const int64_t share = std::max<int64_t>(1, std::min<int64_t>((a.n + least - 1) / least, want / blocks_t));
    g.heads = (int)std::min<int64_t>(256, (a.n + share - 1) / share);
    g.half = rope_div((uint32_t)half);
    g.chunks = rope_div((uint32_t)chunks);
    g.pass = rope_div((uint32_t)std::max(1, (a.d - a.rot) / V));
    const dim3 grid((unsigned)blocks_t, (unsigned)((a.n + g.heads - 1) / g.heads));
    hipLaunchKernelGGL((rope_kernel<T, LAYOUT, V>), grid, dim3(256), g.tokens * half * sizeof(float2), s, a, g);
}

template <class T>
static void launch_typed(const RopeArgs& a, hipStream_t s) {
    constexpr int V = 16 / sizeof(T);
    auto whole = [](int64_t v) { return v % V == 0; };
    // 16-byte accesses: rows, heads, halves and what passes are whole ones
    const bool wide = whole(a.ldx) && whole(a.ldy) && whole(a.d) && whole(a.layout == 0 ? a.rot / 2 : a.rot) &&
                      (((uintptr_t)a.x | (uintptr_t)a.y) & 15) == 0;
    if (a.layout == 0) wide ? launch<T, 0, V>(a, s) : launch<T, 0, 1>(a, s);
    else wide ? launch<T, 1, V>(a, s) : launch<T, 1, 1>(a, s);
}

hipError_t launch_rope(const RopeArgs& a, bool bf16, hipStream_t s) {
    if (bf16) launch_typed<uint16_t>(a, s);
    else launch_typed<float>(a, s);
    return hipGetLastError();
}

}  // namespace ebh
