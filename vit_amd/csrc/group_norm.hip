// Group normalisation with an activation behind it, on channels-last maps (gfx950 / CDNA4): forward and backward.
//
// x [batch, pixels, channels], group g of a sample = channels g*Cg .. g*Cg + Cg - 1 of all its pixels:
//     h = (x - mean_g) rstd_g,   z = h w[c] + b[c],   y = act(z)
// Backward, with dz = dy act'(z) and n = pixels * Cg:
//     dx = rstd_g (dz w - m1_g - h m2_g),  m1 = sum_g(dz w) / n,  m2 = sum_g(dz w h) / n
//     dw[c] = sum dz h,  db[c] = sum dz   over samples and pixels
//
// Bound by HBM (forward: x read, y written; backward: x and dy read, dx written).  A lane owns V channels (16 bytes where
// the channel count and the pointers allow it, else one value) and walks down the pixels, so that a wave reads whole
// runs of a pixel's channels; statistics are kept per channel and put together into groups only at the end of a
// workgroup, which leaves the group width free (any divisor of the channels).
//
// Two forms.  Where the channels of some whole groups over all pixels of a sample fit one workgroup's registers (rows of 64
// bytes at least), it reads them once, does everything and writes the result.  Else two passes: one leaves the moments of
// every chunk of pixels, the next one puts them together again in every workgroup (a few hundred values) and applies them.
//
// All statistics in f32, without the cancellation that sums of squares have where the mean is large against the deviation:
// lanes add first and second moments about their first value, moments of parts are joined about a mean of their own.
#include <type_traits>

#include "vitk_common.h"
#include "vitk_kernels.h"

namespace vitk {

namespace {

constexpr int kT = 256;       // threads of the two-pass kernels

struct Mom {
    float n, mean, m2;
};

// sum over L neighbouring lanes (a power of two), in every lane of them
__device__ __forceinline__ float lanes_sum(float v, int L) {
    for (int o = L >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

__device__ __forceinline__ void lanes_sum2(float& a, float& b, int L) {
    for (int o = L >> 1; o > 0; o >>= 1) {
        const float x = __shfl_xor(a, o, 64), y = __shfl_xor(b, o, 64);
        a += x;
        b += y;
    }
}

// f(group, lane of it) for ng groups by the workgroup's threads, L neighbouring lanes to a group (power of two up to 64);
// every lane of a wave makes every call, with group < ng or not
template <int NT, class F>
__device__ __forceinline__ void by_groups(int ng, int L, F&& f) {
    const int per = NT / L;
    for (int g = 0; g < ng; g += per) f(g + (int)threadIdx.x / L, (int)threadIdx.x & (L - 1));
}

// V values of T: raw registers and their f32 values
template <class T, int V>
struct Raw;
template <>
struct Raw<bf16_t, 8> {
    u32x4 r;
    __device__ __forceinline__ void load(const bf16_t* p) { r = *reinterpret_cast<const u32x4*>(p); }
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[2 * j] = bf16_lo(r[j]);
            v[2 * j + 1] = bf16_hi(r[j]);
        }
    }
    __device__ __forceinline__ float plus(float t) const {             // t + the values, two to an instruction
        typedef bf16_t bf16x2 __attribute__((ext_vector_type(2)));
        const bf16x2 one = {(bf16_t)1.f, (bf16_t)1.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned u = r[j];
            t = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, u), one, t, false);
        }
        return t;
    }
    __device__ __forceinline__ static void store(bf16_t* p, const float (&v)[8]) {
        *reinterpret_cast<u32x4*>(p) = u32x4{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])};
    }
};
template <>
struct Raw<bf16_t, 1> {
    uint16_t r;
    __device__ __forceinline__ void load(const bf16_t* p) { r = *reinterpret_cast<const uint16_t*>(p); }
    __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = __builtin_bit_cast(float, (uint32_t)r << 16); }
    __device__ __forceinline__ static void store(bf16_t* p, const float (&v)[1]) {
        *reinterpret_cast<uint16_t*>(p) = (uint16_t)pack_bf16(v[0], 0.f);
    }
};
template <>
struct Raw<float, 4> {
    f32x4 r;
    __device__ __forceinline__ void load(const float* p) { r = *reinterpret_cast<const f32x4*>(p); }
    __device__ __forceinline__ void get(float (&v)[4]) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = r[j];
    }
    __device__ __forceinline__ float plus(float t) const { return t + ((r[0] + r[1]) + (r[2] + r[3])); }
    __device__ __forceinline__ static void store(float* p, const float (&v)[4]) {
        *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
    }
};
template <>
struct Raw<float, 1> {
    float r;
    __device__ __forceinline__ void load(const float* p) { r = *p; }
    __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = r; }
    __device__ __forceinline__ static void store(float* p, const float (&v)[1]) { *p = v[0]; }
};

__device__ __forceinline__ float sigmoid(float z) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504088896340736f));
}

// Phi(z) and exp(-z^2 / 2), for f32 results: gelu_erf's polynomial is off by up to 1.5e-7 of erf, 2e-7 of a result near 1 and
// 0.2 % of one at z = -5 (-1.4e-6), below half a step of bf16 but not of f32.  Here erfc(|z| / sqrt 2) exp(z^2 / 2) = t P(t),
// t = 1 / (1 + 0.3 |z|), with P of degree 9 fitted (least squares reweighted towards the largest relative error, |z| <= 14)
// to 4e-9; the two halves then share the exponential, whose argument's rounding, z^2 / 2 steps, is most of the error.
// 32 x 56 x 56 x 256 forward 47.5 us with gelu_erf, 51.7 with this, 68 with the library's erfcf.
__device__ __forceinline__ float normal_cdf(float z, float& e) {
    const float az = fabsf(z);
    const float t = __builtin_amdgcn_rcpf(fmaf(az, 0.3f, 1.0f));
    e = __builtin_amdgcn_exp2f(z * z * (-0.5f * 1.44269504088896340736f));
    float q = -0.0412258916f;
    q = fmaf(q, t, 0.224752828f);
    q = fmaf(q, t, -0.456138015f);
    q = fmaf(q, t, 0.383167386f);
    q = fmaf(q, t, -0.158498019f);
    q = fmaf(q, t, 0.192117453f);
    q = fmaf(q, t, 0.156850532f);
    q = fmaf(q, t, 0.220454782f);
    q = fmaf(q, t, 0.239145666f);
    q = fmaf(q, t, 0.239373267f);
    q = 0.5f * q * t * e;
    return z < 0.f ? q : 1.0f - q;
}

template <class T, int ACT>
__device__ __forceinline__ float act_of(float z) {
    if constexpr (ACT == GN_RELU) return z > 0.f ? z : (z == z ? 0.f : z);      // a NaN stays one
    if constexpr (ACT == GN_GELU) {
        if constexpr (sizeof(T) == 4) {
            float e;
            return z * normal_cdf(z, e);
        }
        return gelu_erf(z);
    }
    if constexpr (ACT == GN_SILU) return z * sigmoid(z);
    return z;
}

template <class T, int ACT>
__device__ __forceinline__ float dact_of(float z) {
    if constexpr (ACT == GN_RELU) return z > 0.f ? 1.f : 0.f;
    if constexpr (ACT == GN_GELU) {
        if constexpr (sizeof(T) == 4) {
            float e;
            const float cdf = normal_cdf(z, e);
            return fmaf(z * e, 0.39894228040143267794f, cdf);
        }
        return dgelu_erf(z);
    }
    if constexpr (ACT == GN_SILU) {
        const float s = sigmoid(z);
        return s * fmaf(z, 1.0f - s, 1.0f);
    }
    return 1.f;
}

// V neighbouring channels' weights and biases, all loads at once (1 and 0 where there are none)
template <int V>
__device__ __forceinline__ void load_params(const float* __restrict__ weight, const float* __restrict__ bias, int c, float (&w)[V], float (&sh)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
        w[j] = 1.f;
        sh[j] = 0.f;
    }
    if (weight) {
#pragma unroll
        for (int j = 0; j < V; ++j) w[j] = weight[c + j];
    }
    if (bias) {
#pragma unroll
        for (int j = 0; j < V; ++j) sh[j] = bias[c + j];
    }
}

// f(j, group) for V neighbouring channels from c on
template <int V, class F>
__device__ __forceinline__ void groups_of(int c, int Cg, F&& f) {
    int g = c / Cg, left = (g + 1) * Cg - c;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        f(j, g);
        if (--left == 0) {
            ++g;
            left = Cg;
        }
    }
}

struct Geometry {
    int S, C, G, Cg;          // pixels, channels, groups, channels of a group
    int cv;                   // lanes side by side in a slab = slab channels / V
    int slabs;                // slabs of cv * V channels (the last one may be short)
    int chunk;                // pixels of a workgroup
    int chunks;
    int L;                    // lanes that put a group together
};

// ---- forward, two passes over x ------------------------------------------------------------------------------

// Moments of every group over one chunk of pixels and one slab of channels:
// part[((b * chunks + chunk) * slabs + slab) * G + g] for the groups that the slab touches.
template <class T, int V>
__global__ __launch_bounds__(kT) void gn_moments(const T* __restrict__ x, Mom* __restrict__ part, Geometry q) {
    __shared__ float s_mean[kT * V], s_m2[kT * V];
    const int tid = threadIdx.x;
    const int rows = kT / q.cv;
    const int row = tid / q.cv, col = tid - row * q.cv;
    const int slab = blockIdx.y, b = blockIdx.z;
    const int c0 = slab * q.cv * V;
    const int wc = min(q.cv * V, q.C - c0);             // channels of this slab
    const int s0 = blockIdx.x * q.chunk, s1 = min(s0 + q.chunk, q.S);
    if (row < rows && col * V < wc) {
        float x0[V], a1[V], a2[V];
#pragma unroll
        for (int j = 0; j < V; ++j) x0[j] = a1[j] = a2[j] = 0.f;
        const T* p = x + ((int64_t)b * q.S) * q.C + c0 + col * V;
        int s = s0 + row;
        float n = 0.f;
        if (s < s1) {
            Raw<T, V> r;
            r.load(p + (int64_t)s * q.C);
            r.get(x0);
            n = 1.f;
            s += rows;
        }
        auto add = [&](const Raw<T, V>& r) {
            float v[V];
            r.get(v);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = v[j] - x0[j];
                a1[j] += d;
                a2[j] = fmaf(d, d, a2[j]);
            }
        };
        constexpr int U = 8;
        for (; s + (U - 1) * rows < s1; s += U * rows) {
            Raw<T, V> r[U];
#pragma unroll
            for (int u = 0; u < U; ++u) r[u].load(p + (int64_t)(s + u * rows) * q.C);
#pragma unroll
            for (int u = 0; u < U; ++u) add(r[u]);
            n += U;
        }
        for (; s < s1; s += rows) {
            Raw<T, V> r;
            r.load(p + (int64_t)s * q.C);
            add(r);
            n += 1.f;
        }
        const float inv = n > 0.f ? 1.0f / n : 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            s_mean[row * wc + col * V + j] = fmaf(a1[j], inv, x0[j]);
            s_m2[row * wc + col * V + j] = fmaxf(fmaf(-a1[j] * inv, a1[j], a2[j]), a2[j] == a2[j] ? 0.f : a2[j]);
        }
    }
    __syncthreads();
    const int g0 = c0 / q.Cg, g1 = (c0 + wc - 1) / q.Cg;
    Mom* out = part + (((int64_t)b * q.chunks + blockIdx.x) * q.slabs + slab) * q.G;
    const int len = s1 - s0;
    by_groups<kT>(g1 - g0 + 1, q.L, [&](int gi, int l) {
        const int g = g0 + gi;
        const bool on = g <= g1;
        const int lo = on ? max(g * q.Cg - c0, 0) : 0, hi = on ? min((g + 1) * q.Cg - c0, wc) : 0;
        const int live = min(rows, len);                             // rows that hold a pixel
        // lanes over the channels first, over the rows with what is left of them (groups of few channels have many rows)
        int sh = 0;
        while ((1 << sh) < q.L && (1 << sh) < hi - lo) ++sh;
        const int cl = l & ((1 << sh) - 1), cs = 1 << sh, r0 = l >> sh, rs = q.L >> sh;
        const float m0 = s_mean[lo], total = (float)len * (float)(hi - lo);
        float t = 0.f;
        for (int r = r0; r < live; r += rs) {
            const float n = (float)((len - r + rows - 1) / rows);
            for (int c = lo + cl; c < hi; c += cs) t = fmaf(n, s_mean[r * wc + c] - m0, t);
        }
        const float mean = m0 + lanes_sum(t, q.L) / total;
        t = 0.f;
        for (int r = r0; r < live; r += rs) {
            const float n = (float)((len - r + rows - 1) / rows);
            for (int c = lo + cl; c < hi; c += cs) {
                const float d = s_mean[r * wc + c] - mean;
                t += fmaf(n * d, d, s_m2[r * wc + c]);
            }
        }
        t = lanes_sum(t, q.L);
        if (on && l == 0) out[g] = Mom{total, mean, t};
    });
}

// mean and rstd of the groups g0..g1 of sample b from the partial moments, into shared memory (index g - g0).  The parts'
// moments are taken about the first part's mean; what that mean is off by counts at most (parts) times in the deviation,
// since the first part's own share of it does.
__device__ __forceinline__ void merge_groups(const Mom* __restrict__ part, const Geometry& q, int V, int b, int g0, int g1,
                                             float eps, float* s_mean, float* s_rstd) {
    by_groups<kT>(g1 - g0 + 1, q.L, [&](int gi, int l) {
        const bool on = g0 + gi <= g1;
        const int g = on ? g0 + gi : g1;
        const int first = (g * q.Cg) / (q.cv * V), last = ((g + 1) * q.Cg - 1) / (q.cv * V);   // slabs that touch the group
        const int ns = last - first + 1;
        const Mom* p = part + ((int64_t)b * q.chunks * q.slabs + first) * q.G + g;
        const float m0 = p->mean;
        float n = 0.f, t1 = 0.f, t2 = 0.f;
        auto at = [&](int i) {
            const int ch = ns == 1 ? i : i / ns, sl = i - ch * ns;
            return p[((int64_t)ch * q.slabs + sl) * q.G];
        };
        auto add = [&](const Mom& m) {
            const float d = m.mean - m0;
            n += m.n;
            t1 = fmaf(m.n, d, t1);
            t2 += fmaf(m.n * d, d, m.m2);
        };
        constexpr int U = 8;                                         // loads on their way at once
        int i = l;
        for (; i + (U - 1) * q.L < q.chunks * ns; i += U * q.L) {
            Mom m[U];
#pragma unroll
            for (int u = 0; u < U; ++u) m[u] = at(i + u * q.L);
#pragma unroll
            for (int u = 0; u < U; ++u) add(m[u]);
        }
        for (; i < q.chunks * ns; i += q.L) add(at(i));
        n = lanes_sum(n, q.L);
        t1 = lanes_sum(t1, q.L) / n;
        t2 = lanes_sum(t2, q.L) / n;
        if (on && l == 0) {
            s_mean[gi] = m0 + t1;
            const float var = t2 - t1 * t1;
            s_rstd[gi] = rsqrtf((var > 0.f || var != var ? var : 0.f) + eps);
        }
    });
}

template <class T, int V, int ACT>
__global__ __launch_bounds__(kT) void gn_apply(const T* __restrict__ x, const Mom* __restrict__ part,
                                               const float* __restrict__ weight, const float* __restrict__ bias,
                                               T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out,
                                               Geometry q, float eps) {
    __shared__ float s_mean[kT * V], s_rstd[kT * V];
    const int tid = threadIdx.x;
    const int rows = kT / q.cv;
    const int row = tid / q.cv, col = tid - row * q.cv;
    const int slab = blockIdx.y, b = blockIdx.z;
    const int c0 = slab * q.cv * V;
    const int wc = min(q.cv * V, q.C - c0);
    const int g0 = c0 / q.Cg, g1 = (c0 + wc - 1) / q.Cg;
    // the last chunks first: the moments' pass has read them last; the first values are on their way while the groups are
    // put together
    const int ch = q.chunks - 1 - blockIdx.x;
    const int s0 = ch * q.chunk, s1 = min(s0 + q.chunk, q.S);
    const int64_t base = ((int64_t)b * q.S) * q.C + c0 + col * V;
    const bool live = row < rows && col * V < wc;
    constexpr int U = 4;
    Raw<T, V> ahead[U];
    float a[V], sh[V];
    if (live) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s0 + row + u * rows < s1) ahead[u].load(x + base + (int64_t)(s0 + row + u * rows) * q.C);
        load_params<V>(weight, bias, c0 + col * V, a, sh);
    }
    merge_groups(part, q, V, b, g0, g1, eps, s_mean, s_rstd);
    __syncthreads();
    if (mean_out && blockIdx.x == 0)
        for (int g = g0 + tid; g <= g1; g += kT) {
            mean_out[b * q.G + g] = s_mean[g - g0];         // a group of several slabs is written by each, the same bits
            rstd_out[b * q.G + g] = s_rstd[g - g0];
        }
    if (!live) return;
    float mu[V];
    groups_of<V>(c0 + col * V, q.Cg, [&](int j, int g) {
        mu[j] = s_mean[g - g0];
        a[j] *= s_rstd[g - g0];
    });
    auto one = [&](const Raw<T, V>& r, int s) {
        float v[V];
        r.get(v);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = act_of<T, ACT>(fmaf(v[j] - mu[j], a[j], sh[j]));
        Raw<T, V>::store(y + base + (int64_t)s * q.C, v);
    };
    int s = s0 + row;
#pragma unroll
    for (int u = 0; u < U; ++u, s += rows)
        if (s < s1) one(ahead[u], s);
    for (; s + (U - 1) * rows < s1; s += U * rows) {
        Raw<T, V> r[U];
#pragma unroll
        for (int u = 0; u < U; ++u) r[u].load(x + base + (int64_t)(s + u * rows) * q.C);
#pragma unroll
        for (int u = 0; u < U; ++u) one(r[u], s + u * rows);
    }
    for (; s < s1; s += rows) {
        Raw<T, V> r;
        r.load(x + base + (int64_t)s * q.C);
        one(r, s);
    }
}

// ---- backward, two passes over x and dy ------------------------------------------------------------------------

// Per chunk and channel the sums of dz and dz h (chan[(b * chunks + chunk) * 2 + {0, 1}][C]), per chunk, slab and group
// those of dz w and dz w h (grp[((b * chunks + chunk) * slabs + slab) * G + g][2]).
template <class T, int V, int ACT>
__global__ __launch_bounds__(kT) void gn_bwd_sums(const T* __restrict__ x, const T* __restrict__ dy,
                                                  const float* __restrict__ weight, const float* __restrict__ bias,
                                                  const float* __restrict__ mean, const float* __restrict__ rstd,
                                                  float* __restrict__ chan, float* __restrict__ grp, Geometry q) {
    __shared__ float s_1[kT * V], s_2[kT * V];
    const int tid = threadIdx.x;
    const int rows = kT / q.cv;
    const int row = tid / q.cv, col = tid - row * q.cv;
    const int slab = blockIdx.y, b = blockIdx.z;
    const int c0 = slab * q.cv * V;
    const int wc = min(q.cv * V, q.C - c0);
    const int s0 = blockIdx.x * q.chunk, s1 = min(s0 + q.chunk, q.S);
    if (row < rows && col * V < wc) {
        float mu[V], rs[V], w[V], sh[V], a1[V], a2[V];
        load_params<V>(weight, bias, c0 + col * V, w, sh);
        groups_of<V>(c0 + col * V, q.Cg, [&](int j, int g) {
            mu[j] = mean[b * q.G + g];
            rs[j] = rstd[b * q.G + g];
            a1[j] = a2[j] = 0.f;
        });
        const int64_t base = ((int64_t)b * q.S) * q.C + c0 + col * V;
        auto add = [&](const Raw<T, V>& rx, const Raw<T, V>& rg) {
            float v[V], g[V];
            rx.get(v);
            rg.get(g);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float h = (v[j] - mu[j]) * rs[j];
                const float dz = ACT == GN_NONE ? g[j] : g[j] * dact_of<T, ACT>(fmaf(h, w[j], sh[j]));
                a1[j] += dz;
                a2[j] = fmaf(dz, h, a2[j]);
            }
        };
        int s = s0 + row;
        constexpr int U = 4;
        for (; s + (U - 1) * rows < s1; s += U * rows) {
            Raw<T, V> rx[U], rg[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                rx[u].load(x + base + (int64_t)(s + u * rows) * q.C);
                rg[u].load(dy + base + (int64_t)(s + u * rows) * q.C);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) add(rx[u], rg[u]);
        }
        for (; s < s1; s += rows) {
            Raw<T, V> rx, rg;
            rx.load(x + base + (int64_t)s * q.C);
            rg.load(dy + base + (int64_t)s * q.C);
            add(rx, rg);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            s_1[row * wc + col * V + j] = a1[j];
            s_2[row * wc + col * V + j] = a2[j];
        }
    }
    __syncthreads();
    float* o1 = chan + ((int64_t)b * q.chunks + blockIdx.x) * 2 * q.C + c0;
    // per channel: the rows in kT / wc parts, then the parts
    const int parts = min(max(kT / wc, 1), rows);
    if (parts > 1) {
        for (int i = tid; i < parts * wc; i += kT) {
            const int p = i / wc, c = i - p * wc;
            float t1 = 0.f, t2 = 0.f;
            for (int r = p; r < rows; r += parts) {
                t1 += s_1[r * wc + c];
                t2 += s_2[r * wc + c];
            }
            s_1[p * wc + c] = t1;                          // rows p, p + parts, ...: this thread's alone
            s_2[p * wc + c] = t2;
        }
        __syncthreads();
    }
    const int left = parts > 1 ? parts : rows;
    for (int c = tid; c < wc; c += kT) {
        float t1 = s_1[c], t2 = s_2[c];
        for (int r = 1; r < left; ++r) {
            t1 += s_1[r * wc + c];
            t2 += s_2[r * wc + c];
        }
        o1[c] = t1;
        o1[q.C + c] = t2;
        const float w = weight ? weight[c0 + c] : 1.f;
        s_1[c] = t1 * w;                                   // row 0, column c: read by this thread alone
        s_2[c] = t2 * w;
    }
    __syncthreads();
    const int g0 = c0 / q.Cg, g1 = (c0 + wc - 1) / q.Cg;
    float* og = grp + (((int64_t)b * q.chunks + blockIdx.x) * q.slabs + slab) * q.G * 2;
    by_groups<kT>(g1 - g0 + 1, q.L, [&](int gi, int l) {
        const int g = g0 + gi;
        const bool on = g <= g1;
        const int lo = on ? max(g * q.Cg - c0, 0) : 0, hi = on ? min((g + 1) * q.Cg - c0, wc) : 0;
        float t1 = 0.f, t2 = 0.f;
        for (int c = lo + l; c < hi; c += q.L) {
            t1 += s_1[c];
            t2 += s_2[c];
        }
        t1 = lanes_sum(t1, q.L);
        t2 = lanes_sum(t2, q.L);
        if (on && l == 0) {
            og[2 * g] = t1;
            og[2 * g + 1] = t2;
        }
    });
}

template <class T, int V, int ACT>
__global__ __launch_bounds__(kT) void gn_bwd_apply(const T* __restrict__ x, const T* __restrict__ dy,
                                                   const float* __restrict__ weight, const float* __restrict__ bias,
                                                   const float* __restrict__ mean, const float* __restrict__ rstd,
                                                   const float* __restrict__ grp, T* __restrict__ dx, Geometry q) {
    __shared__ float s_1[kT * V], s_2[kT * V];
    const int tid = threadIdx.x;
    const int rows = kT / q.cv;
    const int row = tid / q.cv, col = tid - row * q.cv;
    const int slab = blockIdx.y, b = blockIdx.z;
    const int c0 = slab * q.cv * V;
    const int wc = min(q.cv * V, q.C - c0);
    const int g0 = c0 / q.Cg, g1 = (c0 + wc - 1) / q.Cg;
    const float inv_n = 1.0f / ((float)q.S * (float)q.Cg);
    const int ch = q.chunks - 1 - blockIdx.x;
    const int s0 = ch * q.chunk, s1 = min(s0 + q.chunk, q.S);
    const int64_t base = ((int64_t)b * q.S) * q.C + c0 + col * V;
    const bool live = row < rows && col * V < wc;
    constexpr int U = 2;
    Raw<T, V> ax[U], ag[U];
    float mu[V], rs[V], w[V], sh[V];
    if (live) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s0 + row + u * rows < s1) {
                ax[u].load(x + base + (int64_t)(s0 + row + u * rows) * q.C);
                ag[u].load(dy + base + (int64_t)(s0 + row + u * rows) * q.C);
            }
        load_params<V>(weight, bias, c0 + col * V, w, sh);
        groups_of<V>(c0 + col * V, q.Cg, [&](int j, int g) {
            mu[j] = mean[b * q.G + g];
            rs[j] = rstd[b * q.G + g];
        });
    }
    by_groups<kT>(g1 - g0 + 1, q.L, [&](int gi, int l) {
        const bool on = g0 + gi <= g1;
        const int g = on ? g0 + gi : g1;
        const int first = (g * q.Cg) / (q.cv * V), last = ((g + 1) * q.Cg - 1) / (q.cv * V);
        const int ns = last - first + 1;
        const float* p = grp + (((int64_t)b * q.chunks * q.slabs + first) * q.G + g) * 2;
        float t1 = 0.f, t2 = 0.f;
        auto at = [&](int i) {
            const int c = ns == 1 ? i : i / ns, sl = i - c * ns;
            return *reinterpret_cast<const f32x2*>(p + ((int64_t)c * q.slabs + sl) * q.G * 2);
        };
        constexpr int UP = 8;                                        // loads on their way at once
        int i = l;
        for (; i + (UP - 1) * q.L < q.chunks * ns; i += UP * q.L) {
            f32x2 m[UP];
#pragma unroll
            for (int u = 0; u < UP; ++u) m[u] = at(i + u * q.L);
#pragma unroll
            for (int u = 0; u < UP; ++u) {
                t1 += m[u][0];
                t2 += m[u][1];
            }
        }
        for (; i < q.chunks * ns; i += q.L) {
            const f32x2 m = at(i);
            t1 += m[0];
            t2 += m[1];
        }
        t1 = lanes_sum(t1, q.L);
        t2 = lanes_sum(t2, q.L);
        if (on && l == 0) {
            s_1[gi] = t1 * inv_n;
            s_2[gi] = t2 * inv_n;
        }
    });
    __syncthreads();
    if (!live) return;
    float m1[V], m2[V];
    groups_of<V>(c0 + col * V, q.Cg, [&](int j, int g) {
        m1[j] = s_1[g - g0];
        m2[j] = s_2[g - g0];
    });
    auto one = [&](const Raw<T, V>& rx, const Raw<T, V>& rg, int s) {
        float v[V], g[V];
        rx.get(v);
        rg.get(g);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float h = (v[j] - mu[j]) * rs[j];
            const float dz = ACT == GN_NONE ? g[j] : g[j] * dact_of<T, ACT>(fmaf(h, w[j], sh[j]));
            v[j] = rs[j] * (fmaf(dz, w[j], -m1[j]) - h * m2[j]);
        }
        Raw<T, V>::store(dx + base + (int64_t)s * q.C, v);
    };
    int s = s0 + row;
#pragma unroll
    for (int u = 0; u < U; ++u, s += rows)
        if (s < s1) one(ax[u], ag[u], s);
    for (; s + (U - 1) * rows < s1; s += U * rows) {
        Raw<T, V> rx[U], rg[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            rx[u].load(x + base + (int64_t)(s + u * rows) * q.C);
            rg[u].load(dy + base + (int64_t)(s + u * rows) * q.C);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) one(rx[u], rg[u], s + u * rows);
    }
    for (; s < s1; s += rows) {
        Raw<T, V> rx, rg;
        rx.load(x + base + (int64_t)s * q.C);
        rg.load(dy + base + (int64_t)s * q.C);
        one(rx, rg, s);
    }
}

// ---- one pass: whole groups of a sample in one workgroup's registers -------------------------------------------

// Thread t holds chunk t % wv (V channels, all of one group) of pixels t / wv, + R, + 2 R, ... (R = NT / wv), at most NV.
struct Slab {
    int S, C, G, Cg;
    int W, wv;                // channels of a workgroup (whole groups), W / V
    int L;                    // lanes that put a group together
    int paired;
};

// Workgroup -> (slab, sample).  Paired: the two slabs of 64 bytes that share a 128-byte line go to workgroups 8 apart, which
// one XCD runs, so that its L2 fetches and writes whole lines.
__device__ __forceinline__ void slab_place(const Slab& q, int& slab, int& b) {
    const int n = q.C / q.W, id = blockIdx.x;
    if (q.paired) {
        const int pair = (id >> 4) * 8 + (id & 7), half = (id >> 3) & 1, m = n >> 1;
        b = pair / m;
        slab = (pair - b * m) * 2 + half;
    } else {
        b = id / n;
        slab = id - b * n;
    }
}

// sums of two values per thread over the threads of each group: s_out[0 / 1][group of the slab]; two barriers
template <int NT, int V>
__device__ __forceinline__ void slab_sums(const Slab& q, int R, float v1, float v2, float (*s_in)[NT], float (*s_out)[NT]) {
    const int tid = threadIdx.x, gv = q.Cg / V;                      // gv: threads side by side in a group
    s_in[0][tid] = v1;                                               // [pixel row][chunk] as the threads lie
    s_in[1][tid] = v2;
    __syncthreads();
    by_groups<NT>(q.W / q.Cg, q.L, [&](int g, int l) {
        const bool on = g < q.W / q.Cg;
        float t1 = 0.f, t2 = 0.f;
        if (on) {
            // lanes over a row's threads first, over the rows with what is left of them
            int sh = 0;
            while ((1 << sh) < q.L && (1 << sh) < gv) ++sh;
            for (int r = l >> sh; r < R; r += q.L >> sh)
                for (int c = l & ((1 << sh) - 1); c < gv; c += 1 << sh) {
                    const int at = r * q.wv + g * gv + c;
                    t1 += s_in[0][at];
                    t2 += s_in[1][at];
                }
        }
        lanes_sum2(t1, t2, q.L);
        if (on && l == 0) {
            s_out[0][g] = t1;
            s_out[1][g] = t2;
        }
    });
    __syncthreads();
}

template <class T, int V, int ACT, int NT, int NV>
__global__ __launch_bounds__(NT) void gn_slab(const T* __restrict__ x, const float* __restrict__ weight,
                                              const float* __restrict__ bias, T* __restrict__ y, float* __restrict__ mean_out,
                                              float* __restrict__ rstd_out, Slab q, float eps) {
    __shared__ float s_in[2][NT], s_out[2][NT];
    const int tid = threadIdx.x;
    const int R = NT / q.wv, row = tid / q.wv, col = tid - row * q.wv;
    int slab_id, b;
    slab_place(q, slab_id, b);
    const int c0 = slab_id * q.W;
    const int gl = col * V / q.Cg;                                   // group within the slab
    const int64_t base = ((int64_t)b * q.S) * q.C + c0 + col * V;
    const bool live = row < R;
    Raw<T, V> r[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (live && row + i * R < q.S) r[i].load(x + base + (int64_t)(row + i * R) * q.C);
    float w[V], sh[V];
    load_params<V>(weight, bias, c0 + col * V, w, sh);
    const float inv_n = 1.0f / ((float)q.S * (float)q.Cg);
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (live && row + i * R < q.S) {
            t = r[i].plus(t);
        }
    slab_sums<NT, V>(q, R, t, 0.f, s_in, s_out);
    const float mu0 = s_out[0][gl] * inv_n;
    // second moment about the mean as summed, and what that mean is off by
    float t1 = 0.f, t2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (live && row + i * R < q.S) {
            float v[V];
            r[i].get(v);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = v[j] - mu0;
                t1 += d;
                t2 = fmaf(d, d, t2);
            }
        }
    slab_sums<NT, V>(q, R, t1, t2, s_in, s_out);
    const float off = s_out[0][gl] * inv_n;
    const float var = fmaf(-off, off, s_out[1][gl] * inv_n);
    const float mu = mu0 + off, rstd = rsqrtf((var > 0.f || var != var ? var : 0.f) + eps);
    if (!live) return;
    if (mean_out && row == 0 && col * V % q.Cg == 0) {
        mean_out[b * q.G + c0 / q.Cg + gl] = mu;
        rstd_out[b * q.G + c0 / q.Cg + gl] = rstd;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) w[j] *= rstd;
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (row + i * R < q.S) {
            float v[V];
            r[i].get(v);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = act_of<T, ACT>(fmaf(v[j] - mu, w[j], sh[j]));
            Raw<T, V>::store(y + base + (int64_t)(row + i * R) * q.C, v);
        }
}

template <class T, int V, int ACT, int NT, int NV>
__global__ __launch_bounds__(NT) void gn_slab_bwd(const T* __restrict__ x, const T* __restrict__ dy,
                                                  const float* __restrict__ weight, const float* __restrict__ bias,
                                                  const float* __restrict__ mean, const float* __restrict__ rstd,
                                                  T* __restrict__ dx, float* __restrict__ chan, Slab q) {
    __shared__ float s_1[NT * V], s_2[NT * V];
    __shared__ float s_m[2][NT];
    const int tid = threadIdx.x;
    const int R = NT / q.wv, row = tid / q.wv, col = tid - row * q.wv;
    int slab_id, b;
    slab_place(q, slab_id, b);
    const int c0 = slab_id * q.W;
    const int gl = col * V / q.Cg;
    const int64_t base = ((int64_t)b * q.S) * q.C + c0 + col * V;
    const bool live = row < R;
    // gelu' and silu' cost more arithmetic than the memory leaves time for twice: their dz stays in registers
    constexpr bool HOLD = ACT == GN_GELU || ACT == GN_SILU;
    Raw<T, V> rx[NV], rg[NV];
    float held[HOLD ? NV : 1][V];
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (live && row + i * R < q.S) {
            rx[i].load(x + base + (int64_t)(row + i * R) * q.C);
            rg[i].load(dy + base + (int64_t)(row + i * R) * q.C);
        }
    float w[V], sh[V], a1[V], a2[V];
    const float mu = live ? mean[b * q.G + c0 / q.Cg + gl] : 0.f, rs = live ? rstd[b * q.G + c0 / q.Cg + gl] : 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) a1[j] = a2[j] = 0.f;
    load_params<V>(weight, bias, c0 + col * V, w, sh);
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (live && row + i * R < q.S) {
            float v[V], g[V];
            rx[i].get(v);
            rg[i].get(g);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float h = (v[j] - mu) * rs;
                const float dz = ACT == GN_NONE ? g[j] : g[j] * dact_of<T, ACT>(fmaf(h, w[j], sh[j]));
                if constexpr (HOLD) held[i][j] = dz;
                a1[j] += dz;
                a2[j] = fmaf(dz, h, a2[j]);
            }
        }
    if (live) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            s_1[row * q.W + col * V + j] = a1[j];
            s_2[row * q.W + col * V + j] = a2[j];
        }
    }
    __syncthreads();
    // per channel: the rows in NT / W parts, then the parts
    const int parts = NT / q.W < R ? (NT / q.W > 0 ? NT / q.W : 1) : R;
    for (int i = tid; i < parts * q.W; i += NT) {
        const int p = i / q.W, c = i - p * q.W;
        float t1 = 0.f, t2 = 0.f;
        for (int r = p; r < R; r += parts) {
            t1 += s_1[r * q.W + c];
            t2 += s_2[r * q.W + c];
        }
        s_1[p * q.W + c] = t1;                              // rows p, p + parts, ...: this thread's alone
        s_2[p * q.W + c] = t2;
    }
    __syncthreads();
    for (int c = tid; c < q.W; c += NT) {
        float t1 = s_1[c], t2 = s_2[c];
        for (int p = 1; p < parts; ++p) {
            t1 += s_1[p * q.W + c];
            t2 += s_2[p * q.W + c];
        }
        chan[(int64_t)b * 2 * q.C + c0 + c] = t1;
        chan[(int64_t)b * 2 * q.C + q.C + c0 + c] = t2;
        const float wc = weight ? weight[c0 + c] : 1.f;
        s_1[c] = t1 * wc;
        s_2[c] = t2 * wc;
    }
    __syncthreads();
    const float inv_n = 1.0f / ((float)q.S * (float)q.Cg);
    by_groups<NT>(q.W / q.Cg, q.L, [&](int g, int l) {
        const bool on = g < q.W / q.Cg;
        float t1 = 0.f, t2 = 0.f;
        if (on)
            for (int c = l; c < q.Cg; c += q.L) {
                t1 += s_1[g * q.Cg + c];
                t2 += s_2[g * q.Cg + c];
            }
        t1 = lanes_sum(t1, q.L);
        t2 = lanes_sum(t2, q.L);
        if (on && l == 0) {
            s_m[0][g] = t1 * inv_n;
            s_m[1][g] = t2 * inv_n;
        }
    });
    __syncthreads();
    if (!live) return;
    const float m1 = s_m[0][gl], m2 = s_m[1][gl];
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (row + i * R < q.S) {
            float v[V], g[V];
            rx[i].get(v);
            if constexpr (!HOLD) rg[i].get(g);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float h = (v[j] - mu) * rs;
                float dz;
                if constexpr (HOLD) dz = held[i][j];
                else dz = ACT == GN_NONE ? g[j] : g[j] * dact_of<T, ACT>(fmaf(h, w[j], sh[j]));
                v[j] = rs * (fmaf(dz, w[j], -m1) - h * m2);
            }
            Raw<T, V>::store(dx + base + (int64_t)(row + i * R) * q.C, v);
        }
}

// dweight[c] = sum of chan[r][1][c], dbias[c] = sum of chan[r][0][c] over the rows r, in a fixed order: a workgroup takes
// 64 of the 2 C columns, its 16 waves every 16th row each, then the 16 sums are added in wave order.
__global__ __launch_bounds__(1024) void gn_bwd_params(const float* __restrict__ chan, int rows, int C,
                                                      float* __restrict__ dweight, float* __restrict__ dbias) {
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int col = blockIdx.x * 64 + lane;
    const int64_t stride = 2 * (int64_t)C;
    float acc = 0.f;
    if (col < 2 * C) {
        int r = w;
        for (; r + 7 * 16 < rows; r += 8 * 16) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = chan[(int64_t)(r + 16 * j) * stride + col];
            acc += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
        }
        for (; r < rows; r += 16) acc += chan[(int64_t)r * stride + col];
    }
    red[w][lane] = acc;
    __syncthreads();
    if (w == 0 && col < 2 * C) {
        float t = red[0][lane];
#pragma unroll
        for (int j = 1; j < 16; ++j) t += red[j][lane];
        if (col < C) {
            if (dbias) dbias[col] = t;
        } else if (dweight) {
            dweight[col - C] = t;
        }
    }
}

// lanes to a group so that `threads` serve ng groups at once where they can
int lanes_of(int threads, int ng) {
    int L = 64;
    while (L > 1 && L * ng > threads) L >>= 1;
    return L;
}

int vec_of(int esize, int C, bool aligned) {
    const int v = 16 / esize;
    return aligned && C % v == 0 ? v : 1;
}

// How the work is cut: slabs of at most 256 lanes of V channels, and so many chunks of pixels that about 512 workgroups
// share the batch (two of 256 threads on every CU), with at least four pixels to a lane where there are that many and at
// most 128 chunks, since every workgroup of the second pass reads a sample's partial sums again: at 56 x 56 x 256, batch 16,
// in training 2,048 workgroups take 107 us, 512 of them 76.
Geometry geometry(int B, int S, int C, int G, int V) {
    Geometry q;
    q.S = S; q.C = C; q.G = G; q.Cg = C / G;
    const int lanes = C / V;
    q.slabs = (lanes + kT - 1) / kT;
    q.cv = (lanes + q.slabs - 1) / q.slabs;
    const int rows = kT / q.cv;
    int64_t chunks = 512 / ((int64_t)B * q.slabs);
    const int64_t most = S / (4 * (int64_t)rows);
    if (chunks > most) chunks = most;
    if (chunks > 128) chunks = 128;
    if (chunks < 1) chunks = 1;
    q.chunk = (int)((S + chunks - 1) / chunks);
    q.chunks = (S + q.chunk - 1) / q.chunk;
    q.L = lanes_of(kT, (q.cv * V + q.Cg - 1) / q.Cg + 1);
    return q;
}

constexpr int kSlabMost = 16;   // vectors of a thread at most (of x, and of dy again in the backward)

// The one-pass form's cut, or W = 0 where a sample's groups do not fit: as few whole groups as make rows of 128 bytes, of
// 64 where those do not fit, each vector within one group.  512 threads, or in the forward 1,024 for longer maps (128
// registers each; the backward holds twice as much).
Slab slab(int B, int S, int C, int G, int V, int esize, bool backward, int& threads) {
    Slab q = {S, C, G, C / G, 0, 0, 1, 0};
    if (V == 1 || q.Cg % V != 0) return q;
    for (threads = 512; threads <= (backward ? 512 : 1024); threads *= 2)
        for (const int bytes : {128, 64}) {
            int k = 1;
            while (k < G && (k * q.Cg * esize < bytes || G % k != 0)) ++k;
            const int64_t wv = (int64_t)k * q.Cg / V;
            if (wv > threads || (int64_t)B * (G / k) > 0x7FFFFFFF) continue;
            const int R = threads / (int)wv;
            if (((int64_t)S + R - 1) / R > kSlabMost) continue;
            q.W = k * q.Cg;
            q.wv = (int)wv;
            q.L = lanes_of(threads, k);
            q.paired = q.W * esize == 64 && (int64_t)B * (G / k) % 16 == 0 && (G / k) % 2 == 0;
            return q;
        }
    return q;
}

template <class F>
hipError_t by_act(int act, F&& f) {
    switch (act) {
        case GN_RELU: return f(std::integral_constant<int, GN_RELU>{});
        case GN_GELU: return f(std::integral_constant<int, GN_GELU>{});
        case GN_SILU: return f(std::integral_constant<int, GN_SILU>{});
        default: return f(std::integral_constant<int, GN_NONE>{});
    }
}

template <class T, int V>
hipError_t forward(const T* x, const float* weight, const float* bias, T* y, float* mean, float* rstd, Mom* part, int B,
                   int S, int C, int G, float eps, int act, hipStream_t s) {
    if constexpr (V > 1) {
        int threads;
        const Slab sl = slab(B, S, C, G, V, sizeof(T), false, threads);
        if (sl.W) {
            const int R = threads / sl.wv, nv = (S + R - 1) / R;
            return by_act(act, [&](auto a) {
                constexpr int A = decltype(a)::value;
                if ((int64_t)B * (C / sl.W) > 0x7FFFFFFF) return hipErrorInvalidValue;
                const dim3 grid(B * (C / sl.W)), block(threads);
                if (threads == 1024) hipLaunchKernelGGL((gn_slab<T, V, A, 1024, kSlabMost>), grid, block, 0, s, x, weight, bias, y, mean, rstd, sl, eps);
                else if (nv <= 4) hipLaunchKernelGGL((gn_slab<T, V, A, 512, 4>), grid, block, 0, s, x, weight, bias, y, mean, rstd, sl, eps);
                else hipLaunchKernelGGL((gn_slab<T, V, A, 512, kSlabMost>), grid, block, 0, s, x, weight, bias, y, mean, rstd, sl, eps);
                return hipGetLastError();
            });
        }
    }
    const Geometry q = geometry(B, S, C, G, V);
    const dim3 grid(q.chunks, q.slabs, B);
    hipLaunchKernelGGL((gn_moments<T, V>), grid, dim3(kT), 0, s, x, part, q);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    return by_act(act, [&](auto a) {
        hipLaunchKernelGGL((gn_apply<T, V, decltype(a)::value>), grid, dim3(kT), 0, s, x, part, weight, bias, y, mean, rstd, q, eps);
        return hipGetLastError();
    });
}

template <class T, int V>
hipError_t backward(const T* x, const float* weight, const float* bias, const T* dy, const float* mean, const float* rstd,
                    T* dx, float* dweight, float* dbias, float* ws, int B, int S, int C, int G, int act, hipStream_t s) {
    if constexpr (V > 1) {
        int threads;
        const Slab sl = slab(B, S, C, G, V, sizeof(T), true, threads);
        if (sl.W) {
            const int R = threads / sl.wv, nv = (S + R - 1) / R;
            hipError_t e = by_act(act, [&](auto a) {
                constexpr int A = decltype(a)::value;
                if ((int64_t)B * (C / sl.W) > 0x7FFFFFFF) return hipErrorInvalidValue;
                const dim3 grid(B * (C / sl.W)), block(512);
                if (nv <= 4) hipLaunchKernelGGL((gn_slab_bwd<T, V, A, 512, 4>), grid, block, 0, s, x, dy, weight, bias, mean, rstd, dx, ws, sl);
                else hipLaunchKernelGGL((gn_slab_bwd<T, V, A, 512, kSlabMost>), grid, block, 0, s, x, dy, weight, bias, mean, rstd, dx, ws, sl);
                return hipGetLastError();
            });
            if (e != hipSuccess || (!dweight && !dbias)) return e;
            hipLaunchKernelGGL(gn_bwd_params, dim3((2 * C + 63) / 64), dim3(1024), 0, s, ws, B, C, dweight, dbias);
            return hipGetLastError();
        }
    }
    const Geometry q = geometry(B, S, C, G, V);
    float* chan = ws;
    float* grp = ws + (int64_t)B * q.chunks * 2 * C;
    const dim3 grid(q.chunks, q.slabs, B);
    hipError_t e = by_act(act, [&](auto a) {
        hipLaunchKernelGGL((gn_bwd_sums<T, V, decltype(a)::value>), grid, dim3(kT), 0, s, x, dy, weight, bias, mean, rstd, chan, grp, q);
        hipError_t r = hipGetLastError();
        if (r != hipSuccess) return r;
        hipLaunchKernelGGL((gn_bwd_apply<T, V, decltype(a)::value>), grid, dim3(kT), 0, s, x, dy, weight, bias, mean, rstd, grp, dx, q);
        return hipGetLastError();
    });
    if (e != hipSuccess || (!dweight && !dbias)) return e;
    hipLaunchKernelGGL(gn_bwd_params, dim3((2 * C + 63) / 64), dim3(1024), 0, s, chan, B * q.chunks, C, dweight, dbias);
    return hipGetLastError();
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

// f32 values of scratch: what the forward (backward = false) or the backward needs at most, whatever the alignment
int64_t group_norm_workspace(int B, int S, int C, int G, bool bf16, bool backward) {
    int64_t most = 0;
    for (const bool al : {false, true}) {
        const Geometry q = geometry(B, S, C, G, vec_of(bf16 ? 2 : 4, C, al));
        const int64_t blocks = (int64_t)B * q.chunks;
        const int64_t n = backward ? blocks * 2 * C + blocks * q.slabs * G * 2 : blocks * q.slabs * G * 3;
        most = n > most ? n : most;
    }
    return most;
}

hipError_t launch_group_norm(const void* x, const float* weight, const float* bias, void* y, float* mean, float* rstd,
                             float* ws, int B, int S, int C, int G, float eps, int act, bool bf16, hipStream_t s) {
    Mom* part = reinterpret_cast<Mom*>(ws);
    const bool al = aligned(x) && aligned(y);
    if (bf16) {
        auto xb = reinterpret_cast<const bf16_t*>(x);
        auto yb = reinterpret_cast<bf16_t*>(y);
        return vec_of(2, C, al) == 8 ? forward<bf16_t, 8>(xb, weight, bias, yb, mean, rstd, part, B, S, C, G, eps, act, s)
                                     : forward<bf16_t, 1>(xb, weight, bias, yb, mean, rstd, part, B, S, C, G, eps, act, s);
    }
    auto xf = reinterpret_cast<const float*>(x);
    auto yf = reinterpret_cast<float*>(y);
    return vec_of(4, C, al) == 4 ? forward<float, 4>(xf, weight, bias, yf, mean, rstd, part, B, S, C, G, eps, act, s)
                                 : forward<float, 1>(xf, weight, bias, yf, mean, rstd, part, B, S, C, G, eps, act, s);
}

hipError_t launch_group_norm_backward(const void* x, const float* weight, const float* bias, const void* dy, const float* mean,
                                      const float* rstd, void* dx, float* dweight, float* dbias, float* ws, int B, int S,
                                      int C, int G, int act, bool bf16, hipStream_t s) {
    const bool al = aligned(x) && aligned(dy) && aligned(dx);
    if (bf16) {
        auto xb = reinterpret_cast<const bf16_t*>(x);
        auto gb = reinterpret_cast<const bf16_t*>(dy);
        auto db = reinterpret_cast<bf16_t*>(dx);
        return vec_of(2, C, al) == 8
                   ? backward<bf16_t, 8>(xb, weight, bias, gb, mean, rstd, db, dweight, dbias, ws, B, S, C, G, act, s)
                   : backward<bf16_t, 1>(xb, weight, bias, gb, mean, rstd, db, dweight, dbias, ws, B, S, C, G, act, s);
    }
    auto xf = reinterpret_cast<const float*>(x);
    auto gf = reinterpret_cast<const float*>(dy);
    auto df = reinterpret_cast<float*>(dx);
    return vec_of(4, C, al) == 4
               ? backward<float, 4>(xf, weight, bias, gf, mean, rstd, df, dweight, dbias, ws, B, S, C, G, act, s)
               : backward<float, 1>(xf, weight, bias, gf, mean, rstd, df, dweight, dbias, ws, B, S, C, G, act, s);
}

}  // namespace vitk
