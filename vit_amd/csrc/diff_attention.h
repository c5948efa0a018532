// What the forward and backward kernels of differential attention share (gfx950 / CDNA4): the shape record, the LDS image
// of a tile of keys (or queries), and the 32 x 32 matrix tiles on it, for bf16 and f32 operands alike.
//
// All products are 32 x 32 tiles with f32 accumulators, whose layout is the same for both types: lane l holds column
// l & 31 and, as element i, row 8 (i >> 2) + 4 (l >> 5) + (i & 3).  Operands move in 16-byte chunks: 8 bf16 (one
// 32x32x16 instruction per pair of chunks, one in each half-wave) or 4 f32 (four 32x32x2 instructions); the order of the
// k index inside a product is whatever the two operands agree on, so a lane may feed four neighbouring f32 to four
// instructions.
#pragma once
#include "vitk_common.h"
#include "vitk_kernels.h"

namespace vitk {
namespace diff {

typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;

constexpr float kNoScore = -1.0e30f;       // the running maximum before the first key
constexpr float kLog2e = 1.44269504088896340736f;

template <class T>
struct Op;
template <>
struct Op<bf16_t> {
    typedef bf16x8 Chunk;
    static constexpr int kPer = 8;         // elements of a chunk
    __device__ __forceinline__ static f32x16 mma(Chunk a, Chunk b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Op<float> {
    typedef f32x4 Chunk;
    static constexpr int kPer = 4;
    __device__ __forceinline__ static f32x16 mma(Chunk a, Chunk b, f32x16 c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
        return c;
    }
};

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.f;
    return z;
}

// the other half-wave's value of the same column, combined with one's own
__device__ __forceinline__ float both_max(float v) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const auto sw = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const unsigned a = sw[0], b = sw[1];
    return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
__device__ __forceinline__ float both_sum(float v) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const auto sw = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const unsigned a = sw[0], b = sw[1];
    return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
}

// Rows of RB bytes in LDS, 16-byte chunk c of row r at slot c ^ swz(r).  Two kinds of reads have to be free of bank
// conflicts: one chunk of 16 rows in a row (ds_read_b128: 16 different slots), and four chunks of 4 rows (the transposed
// read: 4 rows in 4 different quarters of a 256-byte line).
template <int RB>
__device__ __forceinline__ int swz(int r) {
    if constexpr (RB == 128) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);     // two rows to a 256-byte line
    return ((r & 3) << 2) | ((r >> 2) & 3);
}

// bytes of an LDS row of `n` elements
template <class T, int N>
constexpr int row_bytes() {
    constexpr int b = N * (int)sizeof(T);
    static_assert(b <= 512, "row of an LDS tile");
    return b <= 128 ? 128 : b <= 256 ? 256 : 512;
}

// chunk c of row r
template <class T, int RB>
__device__ __forceinline__ typename Op<T>::Chunk chunk_at(const char* tile, int r, int c) {
    return *reinterpret_cast<const typename Op<T>::Chunk*>(tile + r * RB + ((c ^ swz<RB>(r)) << 4));
}

// Transposed operand: element j of a lane is tile[row0 + 8 (j >> 2) + 4 (lane >> 5) + (j & 3)][col0 + (lane & 31)], j < 8:
// the A operand of (tile slice)^T x B where B is an accumulator's elements 8 s .. 8 s + 7 (rows 16 s + ...).
// row0 is a multiple of 16, col0 of 32.
template <class T, int RB>
struct Trans;
template <int RB>
struct Trans<bf16_t, RB> {
    bf16x8 v;
    __device__ __forceinline__ void load(const char* tile, int row0, int col0, int lane) {
        const int hh = lane >> 5, sub = (lane >> 4) & 1, tq = (lane & 15) >> 2, tp = lane & 3;
        const int c = (col0 >> 3) + sub * 2 + (tp >> 1);
        const int r0 = row0 + 4 * hh + tq, r1 = r0 + 8;
        const char* a0 = tile + r0 * RB + ((c ^ swz<RB>(r0)) << 4) + (tp & 1) * 8;
        const char* a1 = tile + r1 * RB + ((c ^ swz<RB>(r1)) << 4) + (tp & 1) * 8;
        const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)a0);
        const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)a1);
        v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};
template <int RB>
struct Trans<float, RB> {
    float v[8];
    __device__ __forceinline__ void load(const char* tile, int row0, int col0, int lane) {
        const int hh = lane >> 5, n = col0 + (lane & 31);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int r = row0 + 8 * (j >> 2) + 4 * hh + (j & 3);
            v[j] = *reinterpret_cast<const float*>(tile + r * RB + (((n >> 2) ^ swz<RB>(r)) << 4) + (n & 3) * 4);
        }
    }
};

// B operand from elements 8 s .. 8 s + 7 of an accumulator tile
template <class T>
struct Slice;
template <>
struct Slice<bf16_t> {
    bf16x8 v;
    // the rounding to bf16 of a probability or of its gradient: 2^-9 relative, of terms that are then added in f32
    __device__ __forceinline__ void take(const f32x16& s, int st) {
        const u32x4 pk = {pack_bf16(s[8 * st], s[8 * st + 1]), pack_bf16(s[8 * st + 2], s[8 * st + 3]),
                          pack_bf16(s[8 * st + 4], s[8 * st + 5]), pack_bf16(s[8 * st + 6], s[8 * st + 7])};
        v = __builtin_bit_cast(bf16x8, pk);
    }
};
template <>
struct Slice<float> {
    float v[8];
    __device__ __forceinline__ void take(const f32x16& s, int st) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = s[8 * st + j];
    }
};
template <int RB>
__device__ __forceinline__ f32x16 mma_t(const Trans<bf16_t, RB>& a, const Slice<bf16_t>& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, c, 0, 0, 0);
}
template <int RB>
__device__ __forceinline__ f32x16 mma_t(const Trans<float, RB>& a, const Slice<float>& b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[j], b.v[j], c, 0, 0, 0);
    return c;
}

// column sums of the B operand in every element of the accumulator: a product with ones
__device__ __forceinline__ f32x16 ones_t(const Slice<bf16_t>& b, f32x16 c) {
    const u32x4 one = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, one), b.v, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 ones_t(const Slice<float>&, f32x16 c) { return c; }

// four neighbouring values to memory
__device__ __forceinline__ void store4(bf16_t* p, f32x4 v) {
    *reinterpret_cast<u32x2*>(p) = u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
}
__device__ __forceinline__ void store4(float* p, f32x4 v) { *reinterpret_cast<f32x4*>(p) = v; }

// 16 zero bytes to stage from where there is nothing: rows past the last visible key, columns past the head
static __device__ __align__(16) const unsigned kZeros[4] = {0, 0, 0, 0};

// The rows of a (sample, key head): row r = query token r / g of query head kh * g + r % g, so that the query heads which
// share a key head share its tiles.  The division by g = group is a multiplication by group_mul = 2^(31 + l) / g + 1 with
// 2^l >= g: n < 2^31 times that, over 2^(31 + l), exceeds n / g by less than 1 / g.
struct RowPlace {
    int tok, head;
};
__device__ __forceinline__ RowPlace row_place(const DiffArgs& a, int kh, int r) {
    if (a.group == 1) return RowPlace{r, kh};
    const int t = (int)(__umulhi((unsigned)r, a.group_mul) >> a.group_shift);
    return RowPlace{t, kh * a.group + (r - t * a.group)};
}

// Waits for every load so far.  Before a loop that loads ahead: what was loaded before it and is used in it would otherwise be
// waited for inside, and the loop's own loads with it.
__device__ __forceinline__ void loads_done() { __builtin_amdgcn_s_waitcnt(0x0F70); }       // vmcnt(0), other counters free

// keys that a query token sees: those below the result
__device__ __forceinline__ int key_limit(const DiffArgs& a, int len, int tok) {
    if (!a.causal) return len;
    const int lim = tok + a.nk - a.nq + 1;
    return lim < len ? (lim > 0 ? lim : 0) : len;
}

constexpr int pow2_below(int n) { return n >= 32 ? 32 : n >= 16 ? 16 : n >= 8 ? 8 : n >= 4 ? 4 : n >= 2 ? 2 : 1; }

// Staging of a chunk of C rows of two tensors side by side, [2 maps x d] and [2 d] (K and V, or Q and dO), through
// registers into an LDS buffer of two tiles: 4 DPC neighbouring lanes move a row's chunks.  Columns past the head's d are
// zeroed once in both buffers and left alone; rows past the last one are the last one again (nothing behind it is read),
// which the caller masks.
template <class T, int DP, int NT, int C>
struct Stage {
    static constexpr int PER = Op<T>::kPer, DPC = DP / PER, RB = row_bytes<T, 2 * DP>(), TILE = C * RB;
    static constexpr int LANES = 4 * DPC, ROWS = pow2_below(NT / LANES < C ? NT / LANES : C), PASSES = C / ROWS;
    int row, col;          // within the chunk; chunk of the LDS row
    bool second, on;
    int map, e;            // first tensor: map and chunk within it
    u32x4 held[PASSES];
    __device__ __forceinline__ void init(int tid, int dc, char* bufs) {
        row = tid / LANES;
        const int c = tid - row * LANES;
        second = c >= 2 * DPC;
        col = second ? c - 2 * DPC : c;
        map = !second && col >= DPC ? 1 : 0;
        e = col - map * DPC;
        const bool mine = row < ROWS;
        on = mine && (second ? col < 2 * dc : e < dc);
        if (mine && !on)
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int i = 0; i < PASSES; ++i) *reinterpret_cast<u32x4*>(bufs + k * 2 * TILE + at(i)) = u32x4{0u, 0u, 0u, 0u};
    }
    __device__ __forceinline__ int at(int i) const {
        const int lr = row + i * ROWS;
        return (second ? TILE : 0) + lr * RB + ((col ^ swz<RB>(lr)) << 4);
    }
    // addr(row): where the row of this lane's tensor, map and chunk lies
    template <class F>
    __device__ __forceinline__ void fetch(int row0, int rows, F&& addr) {
        if (!on) return;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int r = row0 + row + i * ROWS;
            held[i] = *reinterpret_cast<const u32x4*>(addr(r < rows ? r : rows - 1));
        }
    }
    __device__ __forceinline__ void put(char* buf) const {
        if (!on) return;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) *reinterpret_cast<u32x4*>(buf + at(i)) = held[i];
    }
};

// w_h = exp(lam0 . lam1) - exp(lam2 . lam3) + lambda_init; the half-waves share the sums of a lane's head, all loads at once
template <int DP>
__device__ __forceinline__ float map_weight(const DiffArgs& a, int head, int hh) {
    const float* p = a.lam + (a.lam_heads == 1 ? 0 : (int64_t)head * a.d);
    const int64_t vs = (int64_t)a.lam_heads * a.d;
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int t = 0; t < DP / 8; ++t) {
        if (8 * t >= a.d) break;
        const f32x4* e = reinterpret_cast<const f32x4*>(p + 8 * t + 4 * hh);
        const f32x4 x = e[0], y = *reinterpret_cast<const f32x4*>(p + vs + 8 * t + 4 * hh);
        const f32x4 z = *reinterpret_cast<const f32x4*>(p + 2 * vs + 8 * t + 4 * hh);
        const f32x4 u = *reinterpret_cast<const f32x4*>(p + 3 * vs + 8 * t + 4 * hh);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            s1 = fmaf(x[j], y[j], s1);
            s2 = fmaf(z[j], u[j], s2);
        }
    }
    return expf(both_sum(s1)) - expf(both_sum(s2)) + a.lambda_init;
}

}  // namespace diff
}  // namespace vitk
