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
// row0 is a multiple of 16, col0 of 8.
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
    // the rounding to bf16 of a probability or of its gradient: up to 2^-8 of it, of terms that are then added in f32.  The two
    // maps' probabilities are rounded apart, also for dV, where one rounding of P_1 - w P_2 would do: their products lie in two
    // waves.  The matrix pipe multiplies bf16 at 8 times the rate of f32.
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

// Columns col0 + 8 g + 4 hh ... of a row (a) and the same 8 further (b), as an accumulator's elements hold them, if they lie
// below `limit` (a multiple of 8) and the row is live.  In bf16 the half-waves exchange fours, so that each stores 16 bytes.
__device__ __forceinline__ void store_pair(bf16_t* row, int col, int hh, int limit, bool live, f32x4 a, f32x4 b) {
    const auto s0 = __builtin_amdgcn_permlane32_swap(pack_bf16(a[0], a[1]), pack_bf16(b[0], b[1]), false, false);
    const auto s1 = __builtin_amdgcn_permlane32_swap(pack_bf16(a[2], a[3]), pack_bf16(b[2], b[3]), false, false);
    const u32x4 x = {s0[0], s1[0], s0[1], s1[1]};
    col += 8 * hh;
    if (live && col < limit) *reinterpret_cast<u32x4*>(row + col) = x;
}
__device__ __forceinline__ void store_pair(float* row, int col, int hh, int limit, bool live, f32x4 a, f32x4 b) {
    col += 4 * hh;
    if (live && col < limit) store4(row + col, a);
    if (live && col + 8 < limit) store4(row + col + 8, b);
}
__device__ __forceinline__ f32x4 four(const f32x16& v, int g, float f) {
    return f32x4{v[4 * g] * f, v[4 * g + 1] * f, v[4 * g + 2] * f, v[4 * g + 3] * f};
}

// Chunk c of a row, or zeros (columns past the head, rows past the last one): `row` is always one that can be read
template <class T>
__device__ __forceinline__ typename Op<T>::Chunk chunk_or_zero(const T* row, int c, bool on) {
    typename Op<T>::Chunk x = *reinterpret_cast<const typename Op<T>::Chunk*>(row + (on ? c * Op<T>::kPer : 0));
#pragma unroll
    for (int j = 0; j < Op<T>::kPer; ++j) x[j] = on ? x[j] : (T)0.f;
    return x;
}

__device__ __forceinline__ int quotient(int n, Divisor d) { return d.mul ? (int)(__umulhi((unsigned)n, d.mul) >> d.shift) : n; }

// The rows of a (sample, key head): row r = query token r / g of query head kh * g + r % g, so that the query heads which
// share a key head share its tiles.
struct RowPlace {
    int tok, head;
};
__device__ __forceinline__ RowPlace row_place(const DiffArgs& a, int kh, int r) {
    if (a.group == 1) return RowPlace{r, kh};
    const int t = quotient(r, a.by_group);
    return RowPlace{t, kh * a.group + (r - t * a.group)};
}

// Waits for every load so far.  Before a loop that loads ahead: what was loaded before it and is used in it would otherwise be
// waited for inside, and the loop's own loads with it.
__device__ __forceinline__ void loads_done() { __builtin_amdgcn_s_waitcnt(0x0F70); }       // vmcnt(0), other counters free

// Loads what every workgroup needs of the arguments at once: left to the compiler, each block of the prologue loads and waits
// for its own.
__device__ __forceinline__ void arguments(const DiffArgs& a) {
    asm volatile("" ::"s"(a.q), "s"(a.k), "s"(a.v), "s"(a.qs[0]), "s"(a.qs[1]), "s"(a.qs[2]), "s"(a.qs[3]), "s"(a.ks[0]), "s"(a.ks[1]),
                 "s"(a.ks[2]), "s"(a.ks[3]), "s"(a.vs[0]), "s"(a.vs[1]), "s"(a.vs[2]), "s"(a.lam), "s"(a.key_lens), "s"(a.batch),
                 "s"(a.nq), "s"(a.nk), "s"(a.heads), "s"(a.kv_heads), "s"(a.group), "s"(a.d), "s"(a.lam_heads), "s"(a.causal),
                 "s"(a.by_group.mul), "s"(a.by_kv_heads.mul), "s"(a.by_bks.mul), "s"(a.by_bks.shift), "s"(a.scale));
}

// keys that a query token sees: those below the result
__device__ __forceinline__ int key_limit(const DiffArgs& a, int len, int tok) {
    if (!a.causal) return len;
    const int lim = tok + a.nk - a.nq + 1;
    return lim < len ? (lim > 0 ? lim : 0) : len;
}

// Which element of a column's 16 scores is key first + 8 (i >> 2) + 4 hh + (i & 3): those at `seen` and behind are hidden
__device__ __forceinline__ void hide(f32x16& s, int seen) {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 8 * (i >> 2) + (i & 3) < seen ? s[i] : -__builtin_inff();
}

constexpr int pow2_below(int n) { return n >= 32 ? 32 : n >= 16 ? 16 : n >= 8 ? 8 : n >= 4 ? 4 : n >= 2 ? 2 : 1; }

// Staging of a chunk of C rows of two tensors side by side, [2 maps x d] and [2 d] (K and V, or Q and dO), through
// registers into an LDS buffer of two tiles: the first half of the threads moves the first tensor, 2 DPC neighbouring lanes a
// row's chunks.  Columns past the head's d are zeroed once in both buffers and left alone; rows past the last one are the
// last one again (nothing behind it is read), which the caller masks.
template <class T, int DP, int NT, int C>
struct Stage {
    static constexpr int PER = Op<T>::kPer, DPC = DP / PER, RB = row_bytes<T, 2 * DP>(), TILE = C * RB;
    static constexpr int LANES = 2 * DPC, HALF = NT / 2, ROWS = pow2_below(HALF / LANES < C ? HALF / LANES : C), PASSES = C / ROWS;
    static_assert(HALF % 64 == 0, "a wave moves one tensor");
    int row, col;          // within the chunk; chunk of the LDS row
    bool second, on;       // second: wave-uniform
    int map, e;            // first tensor: map and chunk within it
    u32x4 held[PASSES];
    __device__ __forceinline__ void init(int tid, int dc, char* bufs, int buf_bytes) {
        second = __builtin_amdgcn_readfirstlane(tid >= HALF);
        const int t = second ? tid - HALF : tid;
        row = t / LANES;
        col = t - row * LANES;
        map = !second && col >= DPC ? 1 : 0;
        e = col - map * DPC;
        const bool mine = row < ROWS;
        on = mine && (second ? col < 2 * dc : e < dc);
        if (mine && !on)
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int i = 0; i < PASSES; ++i) *reinterpret_cast<u32x4*>(bufs + k * buf_bytes + at(i)) = u32x4{0u, 0u, 0u, 0u};
    }
    __device__ __forceinline__ int at(int i) const {
        const int lr = row + i * ROWS;
        return (second ? TILE : 0) + lr * RB + ((col ^ swz<RB>(lr)) << 4);
    }
    // Whole chunks: row0 + the thread's row lies (row0 >> shift) `step` behind src (wave-uniform: one addition a load).  addr(r):
    // where row r of this lane's tensor, map and chunk lies, for the last chunk, and for all where shift < 0.
    template <class F>
    __device__ __forceinline__ void fetch(int row0, int rows, const T* src, int64_t step, int shift, F&& addr) {
        if (!on) return;
        if (shift >= 0 && row0 + C <= rows) {
#pragma unroll
            for (int i = 0; i < PASSES; ++i)
                held[i] = *reinterpret_cast<const u32x4*>(src + ((row0 + i * ROWS) >> shift) * step);
            return;
        }
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

// w_h = exp(lam0 . lam1) - exp(lam2 . lam3) + lambda_init, all loads at once.  Where all lanes want the same head (same: they do) the first
// half-wave adds the first product, a column to a lane, and the second the other; else the half-waves share the sums of a
// lane's own head.
template <int DP>
__device__ __forceinline__ float map_weight(const DiffArgs& a, int head, int lane, bool same) {
    const int hh = lane >> 5, col = lane & 31;
    const int64_t vs = (int64_t)a.lam_heads * a.d;
    float s1, s2;
    if (same || a.group == 1 || a.lam_heads == 1) {
        const float* p = a.lam + (a.lam_heads == 1 ? 0 : (int64_t)__builtin_amdgcn_readfirstlane(head) * a.d) + 2 * hh * vs;
        const int e = col < a.d ? col : 0, e2 = DP > 32 && col + 32 < a.d ? col + 32 : 0;
        const float x = p[e], y = p[vs + e], x2 = p[e2], y2 = p[vs + e2];
        float s = col < a.d ? x * y : 0.f;
        if constexpr (DP > 32) s += col + 32 < a.d ? x2 * y2 : 0.f;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) s += __shfl_xor(s, o, 64);
        const unsigned u = __builtin_bit_cast(unsigned, s);
        const auto sw = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        const unsigned lo = sw[0], hi = sw[1];
        s1 = __builtin_bit_cast(float, lo);
        s2 = __builtin_bit_cast(float, hi);
    } else {
        const float* p = a.lam + (int64_t)head * a.d;
        s1 = s2 = 0.f;
        f32x4 v[4][DP / 8];
#pragma unroll
        for (int t = 0; t < DP / 8; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i][t] = *reinterpret_cast<const f32x4*>(p + i * vs + (8 * t < a.d ? 8 * t + 4 * hh : 0));
#pragma unroll
        for (int t = 0; t < DP / 8; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s1 = 8 * t < a.d ? fmaf(v[0][t][j], v[1][t][j], s1) : s1;
                s2 = 8 * t < a.d ? fmaf(v[2][t][j], v[3][t][j], s2) : s2;
            }
        s1 = both_sum(s1);
        s2 = both_sum(s2);
    }
    return expf(s1) - expf(s2) + a.lambda_init;
}

}  // namespace diff
}  // namespace vitk
