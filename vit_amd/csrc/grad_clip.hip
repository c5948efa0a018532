// Global norm of a list of gradients and the clipping by it (gfx950 / CDNA4): what follows the backward pass of the
// training step (clip_grad_norm_ at main.py:221-223).
//
//     norm = sqrt(sum over all tensors of g^2)   or   max |g|
//     g   *= min(1, max_norm / (norm + 1e-6))
//
// Bound by HBM: the norm reads every gradient once, the scaling reads and writes it once more; nothing is computed to
// speak of.  One launch covers up to kTensors tensors (their addresses and sizes travel as kernel arguments: nothing has
// to be copied to the device first), whatever their sizes: the list is cut into pieces of 16 KiB, a fixed grid of
// workgroups walks the pieces.  Squares are added in f64: every f32 value has a square that f64 holds, so neither large
// nor tiny gradients lose their norm, and the matrix-free f64 rate (one multiply-add per element) is far above what
// memory delivers.  Every workgroup leaves one partial sum; the scaling kernel adds them itself, every workgroup the same
// sums in the same order (no atomics, no launch of its own, results reproducible), and ends at once where the norm is
// under the bound: a factor of 1 changes no value.
#include "vitk_common.h"
#include "vitk_kernels.h"

namespace vitk {

namespace {

constexpr int kTensors = kGradTensorsPerLaunch;
constexpr int kThreads = 256;
// Measured on all gradients of ViT-L/16 (304 M f32 values in 298 tensors), the norm's and the scaling's passes: pieces of
// 16 KiB and 4 loads in flight a lane 195 and 478 us, of 64 KiB and 8 loads 202 and 500, of 16 KiB and 2 loads 198 and 484.
constexpr int kUnroll = 4;
constexpr int kPieceBytes = 16384;        // 4 loads of 16 bytes per lane
// workgroups of a scaling launch: 1024 took 491 us, one to each piece 462, but 12 instead of 5.5 where the factor is 1
constexpr uint32_t kScaleGrid = 4096;
constexpr uint64_t kTypeBit = 1ull << 62;  // set in `size`: bf16

// Addresses come as integers: said to be global memory, or they would be loaded as generic ones.
#define VITK_GLOBAL __attribute__((address_space(1)))

struct GradTable {
    uint64_t addr[kTensors];
    uint64_t size[kTensors];          // elements, kTypeBit for bf16
    uint32_t first[kTensors + 1];     // first piece of each tensor within this launch
    int n;
};
static_assert(sizeof(GradTable) <= 3968, "kernel arguments are limited to 4 KiB");

// the tensor that holds piece p (wave-uniform)
__device__ __forceinline__ int tensor_of(const GradTable& t, uint32_t p) {
    int lo = 0, hi = t.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= p) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

template <bool INF>
struct Acc {
    double s = 0.0;      // sum of squares
    uint32_t m = 0;      // bits of the largest |g|: ordered as integers, a NaN above everything
    __device__ __forceinline__ void add(float g) {
        if constexpr (INF) {
            const uint32_t b = __builtin_bit_cast(uint32_t, g) & 0x7FFFFFFFu;
            m = b > m ? b : m;
        } else {
            const double d = (double)g;
            s = fma(d, d, s);
        }
    }
    __device__ __forceinline__ void add16(u32x4 v, bool bf16) {
        const f32x4 f = __builtin_bit_cast(f32x4, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (bf16) {
                add(bf16_lo(v[j]));
                add(bf16_hi(v[j]));
            } else {
                add(f[j]);
            }
        }
    }
};

__device__ __forceinline__ double shfl_xor_f64(double v, int o) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __shfl_xor((uint32_t)b, o, 64), hi = __shfl_xor((uint32_t)(b >> 32), o, 64);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

// max that a NaN on either side decides
__device__ __forceinline__ double max_nan(double a, double b) { return (b > a || b != b) ? b : a; }

template <bool INF>
__device__ __forceinline__ double block_reduce(double v, double* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const double w = shfl_xor_f64(v, o);
        v = INF ? max_nan(v, w) : v + w;
    }
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double r = red[0];
#pragma unroll
    for (int i = 1; i < kThreads / 64; ++i) r = INF ? max_nan(r, red[i]) : r + red[i];
    return r;
}

__device__ __forceinline__ float load1(const VITK_GLOBAL char* p, bool bf16) {
    return bf16 ? __builtin_bit_cast(float, (uint32_t)*(const VITK_GLOBAL uint16_t*)p << 16) : *(const VITK_GLOBAL float*)p;
}

// The byte range of piece p of a tensor, split into elements before the first 16-byte boundary, 16-byte vectors, and
// elements after the last one (views into communication buckets start at any element).
struct Piece {
    VITK_GLOBAL char* base;
    int head, vecs, tail;      // elements, 16-byte vectors, elements
    bool bf16;
    int esize;
};

__device__ __forceinline__ Piece piece_of(const GradTable& t, uint32_t p) {
    const int k = tensor_of(t, p);
    Piece r;
    const uint64_t sz = t.size[k];
    r.bf16 = (sz & kTypeBit) != 0;
    r.esize = r.bf16 ? 2 : 4;
    const uint64_t begin = t.addr[k], end = begin + (sz & ~kTypeBit) * r.esize;
    // pieces are cut at multiples of kPieceBytes from the 16-byte boundary at or below the tensor's start
    const uint64_t lo = (begin & ~15ull) + (uint64_t)(p - t.first[k]) * kPieceBytes;
    uint64_t a = lo < begin ? begin : lo, b = lo + kPieceBytes;
    b = b < end ? b : end;
    uint64_t va = (a + 15) & ~15ull, vb = b & ~15ull;
    if (va > b) va = b;                      // fewer bytes than up to the next boundary
    if (vb < va) vb = va;
    r.base = (VITK_GLOBAL char*)a;
    r.head = (int)(va - a) / r.esize;
    r.vecs = (int)((vb - va) >> 4);
    r.tail = (int)(b - vb) / r.esize;
    return r;
}

template <bool INF>
__global__ __launch_bounds__(kThreads) void grad_norm_partials(GradTable t, double* __restrict__ partials) {
    __shared__ double red[kThreads / 64];
    Acc<INF> acc;
    const uint32_t total = t.first[t.n];
    for (uint32_t p = blockIdx.x; p < total; p += gridDim.x) {
        const Piece q = piece_of(t, p);
        const VITK_GLOBAL u32x4* v = (const VITK_GLOBAL u32x4*)(q.base + q.head * q.esize);
        int i = threadIdx.x;
        for (; i + (kUnroll - 1) * kThreads < q.vecs; i += kUnroll * kThreads) {
            u32x4 w[kUnroll];
#pragma unroll
            for (int j = 0; j < kUnroll; ++j) w[j] = __builtin_nontemporal_load(v + i + j * kThreads);
            if (q.bf16) {
#pragma unroll
                for (int j = 0; j < kUnroll; ++j) acc.add16(w[j], true);
            } else {
#pragma unroll
                for (int j = 0; j < kUnroll; ++j) acc.add16(w[j], false);
            }
        }
        for (; i < q.vecs; i += kThreads) acc.add16(v[i], q.bf16);
        if ((int)threadIdx.x < q.head) acc.add(load1(q.base + threadIdx.x * q.esize, q.bf16));
        if ((int)threadIdx.x < q.tail)
            acc.add(load1((const VITK_GLOBAL char*)(v + q.vecs) + threadIdx.x * q.esize, q.bf16));
    }
    const double mine = INF ? (double)__builtin_bit_cast(float, acc.m) : acc.s;
    const double r = block_reduce<INF>(mine, red);
    if (threadIdx.x == 0) partials[blockIdx.x] = r;
}

template <bool INF>
__device__ __forceinline__ double norm_of(const double* __restrict__ partials, int n, double* red) {
    double v = 0.0;
    for (int i = threadIdx.x; i < n; i += 4 * kThreads) {
        double w[4];                                                 // loads on their way at once
#pragma unroll
        for (int u = 0; u < 4; ++u) w[u] = partials[i + u * kThreads < n ? i + u * kThreads : i];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const double x = i + u * kThreads < n ? w[u] : 0.0;
            v = INF ? max_nan(v, x) : v + x;
        }
    }
    const double r = block_reduce<INF>(v, red);
    return INF ? r : sqrt(r);
}

template <bool INF>
__global__ __launch_bounds__(kThreads) void grad_norm_finish(const double* __restrict__ partials, int n,
                                                             float* __restrict__ norm) {
    __shared__ double red[kThreads / 64];
    const double v = norm_of<INF>(partials, n, red);
    if (threadIdx.x == 0) *norm = (float)v;
}

template <bool INF>
__global__ __launch_bounds__(kThreads) void grad_scale(GradTable t, const double* __restrict__ partials, int n,
                                                       double max_norm, float* __restrict__ norm) {
    __shared__ double red[kThreads / 64];
    const double total_norm = norm_of<INF>(partials, n, red);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)total_norm;
    const double c = max_norm / (total_norm + 1e-6);
    if (c >= 1.0) return;                    // a NaN goes on, as a factor
    // the factor as mantissa and exponent: it may lie below f32's normal range while its products do not
    int e;
    const float f = (float)frexp(c, &e);
    auto mul = [&](float g) { return ldexpf(g * f, e); };
    const uint32_t total = t.first[t.n];
    for (uint32_t p = blockIdx.x; p < total; p += gridDim.x) {
        const Piece q = piece_of(t, p);
        VITK_GLOBAL u32x4* v = (VITK_GLOBAL u32x4*)(q.base + q.head * q.esize);
        auto scale = [&](u32x4 w) {
            f32x4 v4 = __builtin_bit_cast(f32x4, w);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (q.bf16) w[j] = pack_bf16(mul(bf16_lo(w[j])), mul(bf16_hi(w[j])));
                else v4[j] = mul(v4[j]);
            }
            return q.bf16 ? w : __builtin_bit_cast(u32x4, v4);
        };
        auto scale1 = [&](VITK_GLOBAL char* p) {
            const float g = mul(load1(p, q.bf16));
            if (q.bf16) *(VITK_GLOBAL uint16_t*)p = (uint16_t)pack_bf16(g, 0.f);
            else *(VITK_GLOBAL float*)p = g;
        };
        int i = threadIdx.x;
        for (; i + (kUnroll - 1) * kThreads < q.vecs; i += kUnroll * kThreads) {
            u32x4 w[kUnroll];
#pragma unroll
            for (int j = 0; j < kUnroll; ++j) w[j] = v[i + j * kThreads];
#pragma unroll
            for (int j = 0; j < kUnroll; ++j) v[i + j * kThreads] = scale(w[j]);
        }
        for (; i < q.vecs; i += kThreads) v[i] = scale(v[i]);
        if ((int)threadIdx.x < q.head) scale1(q.base + threadIdx.x * q.esize);
        if ((int)threadIdx.x < q.tail) scale1((VITK_GLOBAL char*)(v + q.vecs) + threadIdx.x * q.esize);
    }
}

// fills t with up to kTensors tensors from index i on; returns the next index.  The entry points take up to 16 TiB: at most
// 2^30 pieces and one more at either end of a tensor.
int fill(GradTable& t, const uint64_t* addr, const int64_t* size, const int* bf16, int n, int i) {
    t.n = 0;
    uint64_t pieces = 0;
    for (; i < n && t.n < kTensors; ++i) {
        if (size[i] == 0) continue;
        const uint64_t bytes = (uint64_t)size[i] * (bf16[i] ? 2 : 4) + (addr[i] & 15);
        const uint64_t more = (bytes + kPieceBytes - 1) / kPieceBytes;
        t.addr[t.n] = addr[i];
        t.size[t.n] = (uint64_t)size[i] | (bf16[i] ? kTypeBit : 0);
        t.first[t.n] = (uint32_t)pieces;
        pieces += more;
        ++t.n;
    }
    t.first[t.n] = (uint32_t)pieces;
    return i;
}

int grid_of(const GradTable& t) {
    const uint32_t p = t.first[t.n];
    return p < (uint32_t)kGradPartialsPerLaunch ? (int)p : kGradPartialsPerLaunch;
}

}  // namespace

// Partial sums the list leaves (what launch_grad_norm fills): at most kGradPartialsPerLaunch for each kTensors tensors.
int grad_partials(const uint64_t* addr, const int64_t* size, const int* bf16, int n) {
    GradTable t;
    int total = 0;
    for (int i = 0; i < n;) {
        i = fill(t, addr, size, bf16, n, i);
        if (t.n) total += grid_of(t);
    }
    return total;
}

hipError_t launch_grad_norm(const uint64_t* addr, const int64_t* size, const int* bf16, int n, bool inf, double* partials,
                            float* norm, hipStream_t s) {
    GradTable t;
    int at = 0;
    for (int i = 0; i < n;) {
        i = fill(t, addr, size, bf16, n, i);
        if (!t.n) continue;
        const int grid = grid_of(t);
        if (inf) hipLaunchKernelGGL((grad_norm_partials<true>), dim3(grid), dim3(kThreads), 0, s, t, partials + at);
        else hipLaunchKernelGGL((grad_norm_partials<false>), dim3(grid), dim3(kThreads), 0, s, t, partials + at);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        at += grid;
    }
    if (!norm) return hipSuccess;
    if (inf) hipLaunchKernelGGL((grad_norm_finish<true>), dim3(1), dim3(kThreads), 0, s, partials, at, norm);
    else hipLaunchKernelGGL((grad_norm_finish<false>), dim3(1), dim3(kThreads), 0, s, partials, at, norm);
    return hipGetLastError();
}

hipError_t launch_grad_scale(const uint64_t* addr, const int64_t* size, const int* bf16, int n, bool inf,
                             const double* partials, int npartials, double max_norm, float* norm, hipStream_t s) {
    GradTable t;
    for (int i = 0; i < n;) {
        i = fill(t, addr, size, bf16, n, i);
        if (!t.n) continue;
        const int grid = (int)(t.first[t.n] < kScaleGrid ? t.first[t.n] : kScaleGrid);
        if (inf) hipLaunchKernelGGL((grad_scale<true>), dim3(grid), dim3(kThreads), 0, s, t, partials, npartials, max_norm, norm);
        else hipLaunchKernelGGL((grad_scale<false>), dim3(grid), dim3(kThreads), 0, s, t, partials, npartials, max_norm, norm);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        norm = nullptr;                     // the first launch has written it
    }
    return hipSuccess;
}

}  // namespace vitk
