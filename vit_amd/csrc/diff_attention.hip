// Differential attention, forward (gfx950 / CDNA4): per query row of a head
//     P_m = softmax over the visible keys of scale q_m . k_m,  m = 1, 2
//     out = (P_1 - w P_2) V,    w = exp(lam0 . lam1) - exp(lam2 . lam3) + lambda_init
//
// One pass over the keys with a running maximum and sum per map.  The two maps share everything but their scores: a
// workgroup stages the keys of both maps and V once, and every transposed V fragment feeds the products of both maps.
// The maps' products with V stay apart until the end because their denominators are known only then.
//
//     S_m^T[key][row]  = K_m Q_m^T       keys on the matrix row, query rows on the lane
//     O_m^T[col][row] += V^T P_m^T       the exponentiated accumulators are the B operand as they lie
//
// Rows of a (sample, key head) are the tokens of all its query heads (diff_attention.h), 32 to a wave.  Two forms:
//   many rows:  a workgroup of 4 waves takes 128 rows and walks all their keys in chunks of 32 through two LDS buffers,
//               the next chunk on its way to registers while the waves work on the one before;
//   few rows:   its waves take the same 32 rows and every fourth block of 32 keys, and the keys are split over so many
//               workgroups that the chip is full; the waves' results are joined in LDS, the workgroups' by a second kernel.
#include <type_traits>

#include "diff_attention.h"

namespace vitk {

using namespace diff;

namespace {

template <class T, int DP>
constexpr int keys_waves() { return row_bytes<T, 2 * DP>() == 512 ? 2 : 4; }

constexpr int pow2_below(int n) { return n >= 16 ? 16 : n >= 8 ? 8 : n >= 4 ? 4 : n >= 2 ? 2 : 1; }

// index of a 4-column piece of a joined row in LDS: [row][2 maps x DV columns] f32, pieces swizzled by the row
template <int DV>
__device__ __forceinline__ int joined(int row, int map, int col) {
    const int c = (map * DV + col) >> 2;
    return row * (2 * DV) + ((c ^ (row & 15)) << 2);
}

template <class T, int DP, int NW, bool KEYS>
__global__ __launch_bounds__(NW * 64, KEYS || sizeof(T) == 4 ? 1 : 2) void diff_fwd(DiffArgs a, DiffOut o, float* __restrict__ ws, int tiles,
                                                                  int splits) {
    constexpr int DV = 2 * DP;
    constexpr int RB = row_bytes<T, DV>();         // of an LDS row: both maps of a key, or one of V
    constexpr int PER = Op<T>::kPer;
    constexpr int DPC = DP / PER;                  // chunks of one map's key
    constexpr int KT = DPC / 2;                    // products of 2 chunks (one per half-wave) of a score
    constexpr int DB = DV / 32;
    constexpr int KC = KEYS ? 32 * NW : 32;        // keys of a chunk
    constexpr int TILE = KC * RB;
    typedef typename Op<T>::Chunk Chunk;
    __shared__ __align__(16) char bufs[2][2 * TILE];
    __shared__ float s_ml[KEYS ? NW : 1][4][32];
    __shared__ float s_w[32];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 31, hh = lane >> 5;
    const int bks = a.batch * a.kv_heads;
    const int bk = blockIdx.x % bks;               // workgroups of one head lie bks apart: one XCD where 8 divides bks
    const int rest = blockIdx.x / bks;
    const int tile = KEYS ? rest % tiles : (a.causal ? tiles - 1 - rest : rest);     // causal: the longest rows first
    const int split = KEYS ? rest / tiles : 0;
    const int b = bk / a.kv_heads, kh = bk - b * a.kv_heads;
    const int nrows = a.nq * a.group;
    const int row0 = KEYS ? tile * 32 : (tile * NW + wave) * 32;
    const int end = KEYS ? tile * 32 + 32 : (tile + 1) * NW * 32;
    int len = a.nk;
    if (a.key_lens) {
        len = a.key_lens[b];
        len = len < 0 ? 0 : (len < a.nk ? len : a.nk);
    }
    const int kmax = key_limit(a, len, row_place(a, kh, (end < nrows ? end : nrows) - 1).tok);

    // Staging: 4 DPC neighbouring lanes move a key's chunks, both maps of K and then V, ROWS keys at a time; what lies past
    // the last visible key or past the head's d columns is written as zeros and never read from memory.
    constexpr int LANES = 4 * DPC;
    constexpr int ROWS = pow2_below(NW * 64 / LANES);
    constexpr int PASSES = KC / ROWS;
    const int dc = a.d / PER;
    const int srow = tid / LANES, scol = tid - srow * LANES;
    const bool s_v = scol >= 2 * DPC;
    const int s_c = s_v ? scol - 2 * DPC : scol;                         // chunk of the LDS row
    const int s_m = !s_v && s_c >= DPC ? 1 : 0, s_e = s_c - s_m * DPC;
    const bool s_on = srow < ROWS && (s_v ? s_c < 2 * dc : s_e < dc);
    const int64_t s_step = s_v ? a.vs[1] : a.ks[1];
    const T* s_src = s_v ? reinterpret_cast<const T*>(a.v) + b * a.vs[0] + kh * a.vs[2] + s_c * PER
                         : reinterpret_cast<const T*>(a.k) + b * a.ks[0] + kh * a.ks[2] + s_m * a.ks[3] + s_e * PER;
    u32x4 held[PASSES];
    auto fetch = [&](int key0) {
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int key = key0 + srow + i * ROWS;
            held[i] = u32x4{0u, 0u, 0u, 0u};
            if (s_on && key < kmax) held[i] = *reinterpret_cast<const u32x4*>(s_src + key * s_step);
        }
    };
    auto put = [&](char* buf) {
        if (srow >= ROWS) return;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int lr = srow + i * ROWS;
            *reinterpret_cast<u32x4*>(buf + (s_v ? TILE : 0) + lr * RB + ((s_c ^ swz<RB>(lr)) << 4)) = held[i];
        }
    };

    int c0 = 0, c1 = (kmax + KC - 1) / KC;
    if constexpr (KEYS) {
        const int per = (c1 + splits - 1) / splits;
        c0 = split * per;
        c1 = c0 + per < c1 ? c0 + per : c1;
    }
    if (c0 < c1) fetch(c0 * KC);

    const int row = row0 + r;
    const RowPlace place = row_place(a, kh, row < nrows ? row : nrows - 1);
    const int lim = key_limit(a, len, place.tok);
    // wave-uniform: no row of the wave sees a key from wave_max on, all of them see those below wave_min
    const int wave_max = key_limit(a, len, row_place(a, kh, (row0 + 32 < nrows ? row0 + 32 : nrows) - 1).tok);
    const int wave_min = key_limit(a, len, row_place(a, kh, row0 < nrows ? row0 : nrows - 1).tok);
    const bool active = row0 < nrows;

    Chunk qf[2][KT];
    {
        const T* qg = reinterpret_cast<const T*>(a.q) + b * a.qs[0] + place.tok * a.qs[1] + place.head * a.qs[2];
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                const int c = 2 * t + hh;
                qf[m][t] = *reinterpret_cast<const Chunk*>(c < dc ? (const void*)(qg + m * a.qs[3] + c * PER) : (const void*)kZeros);
            }
    }
    const float weight = map_weight<DP>(a, place.head, hh);

    f32x16 acc[2][DB];
    float m_run[2] = {kNoScore, kNoScore}, l_run[2] = {0.f, 0.f};
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[m][d] = zero16();
    const float sc = a.scale * kLog2e;
    constexpr float kLazy = 8.0f;     // the accumulators are rescaled only when a maximum grows by more than 2^8

    auto step = [&](const char* kt, const char* vt, int kb, int key0) {
        f32x16 s[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            s[m] = zero16();
#pragma unroll
            for (int t = 0; t < KT; ++t) s[m] = Op<T>::mma(chunk_at<T, RB>(kt, kb * 32 + r, m * DPC + 2 * t + hh), qf[m][t], s[m]);
        }
        if (key0 + 32 > wave_min) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (key0 + 8 * (i >> 2) + 4 * hh + (i & 3) >= lim) s[0][i] = s[1][i] = -__builtin_inff();
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            float mx = fmaxf(s[m][0], s[m][1]);
#pragma unroll
            for (int i = 2; i < 16; i += 2) mx = fmaxf(fmaxf(mx, s[m][i]), s[m][i + 1]);
            mx = both_max(mx) * sc;                                  // scale > 0: the maximum commutes with it
            if (__any(mx > m_run[m] + kLazy)) {
                const float m_new = fmaxf(m_run[m], mx);
                const float alpha = __builtin_amdgcn_exp2f(m_run[m] - m_new);
                m_run[m] = m_new;
                l_run[m] *= alpha;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[m][d][i] *= alpha;
            }
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[m][i] = __builtin_amdgcn_exp2f(fmaf(s[m][i], sc, -m_run[m]));
                sum += s[m][i];
            }
            l_run[m] += sum;
        }
#pragma unroll
        for (int st = 0; st < 2; ++st) {
            Slice<T> p1, p2;
            p1.take(s[0], st);
            p2.take(s[1], st);
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                Trans<T, RB> v;
                v.load(vt, kb * 32 + 16 * st, d * 32, lane);
                acc[0][d] = mma_t(v, p1, acc[0][d]);
                acc[1][d] = mma_t(v, p2, acc[1][d]);
            }
        }
    };
    const int kb = KEYS ? wave : 0;                                  // the wave's block of a chunk
    if (c0 < c1) put(bufs[0]);
    __syncthreads();
    for (int c = c0; c < c1; ++c) {
        const char* buf = bufs[(c - c0) & 1];
        const bool more = c + 1 < c1;
        if (more) fetch((c + 1) * KC);
        const int key0 = c * KC + kb * 32;
        if (active && key0 < wave_max) step(buf, buf + TILE, kb, key0);
        if (more) put(bufs[(c - c0 + 1) & 1]);
        __syncthreads();
    }

    const float l_tot[2] = {both_sum(l_run[0]), both_sum(l_run[1])};
    const int64_t orow = (((int64_t)b * a.nq + place.tok) * a.heads + place.head) * 2 * a.d;
    const int64_t lrow = ((int64_t)b * a.heads + place.head) * a.nq + place.tok;
    const int64_t lmap = (int64_t)a.batch * a.heads * a.nq;
    T* out = reinterpret_cast<T*>(o.out);
    T* out2 = reinterpret_cast<T*>(o.out2);

    if constexpr (!KEYS) {
        if (row >= nrows) return;
        const float i1 = l_tot[0] > 0.f || l_tot[0] != l_tot[0] ? 1.0f / l_tot[0] : 0.f;
        const float i2 = l_tot[1] > 0.f || l_tot[1] != l_tot[1] ? 1.0f / l_tot[1] : 0.f;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int col = d * 32 + 8 * g + 4 * hh;
                if (col >= 2 * a.d) continue;
                f32x4 x, y;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    y[j] = acc[1][d][4 * g + j] * i2;
                    x[j] = fmaf(-weight, y[j], acc[0][d][4 * g + j] * i1);
                }
                store4(out + orow + col, x);
                if (out2) store4(out2 + orow + col, y);
            }
        if (out2 && hh == 0) {
            o.stats[lrow] = l_tot[0] == 0.f ? 0.f : m_run[0];
            o.stats[lmap + lrow] = l_tot[1] == 0.f ? 0.f : m_run[1];
            o.stats[2 * lmap + lrow] = i1;
            o.stats[3 * lmap + lrow] = i2;
            if (b == 0 && place.tok == 0) o.weight[place.head] = weight;
        }
    } else {
        // join the waves' keys
        if (hh == 0) {
            s_ml[wave][0][r] = m_run[0];
            s_ml[wave][1][r] = l_tot[0];
            s_ml[wave][2][r] = m_run[1];
            s_ml[wave][3][r] = l_tot[1];
            if (wave == 0) s_w[r] = weight;
        }
        __syncthreads();
        float top[2], sum[2] = {0.f, 0.f};
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            top[m] = s_ml[0][2 * m][r];
#pragma unroll
            for (int w = 1; w < NW; ++w) top[m] = fmaxf(top[m], s_ml[w][2 * m][r]);
#pragma unroll
            for (int w = 0; w < NW; ++w) sum[m] += s_ml[w][2 * m + 1][r] * __builtin_amdgcn_exp2f(s_ml[w][2 * m][r] - top[m]);
        }
        constexpr int HALF = NW / 2;
        float* mine = reinterpret_cast<float*>(bufs[wave < HALF ? 0 : 1]) + (wave % HALF) * 32 * 2 * DV;
        static_assert(HALF * 32 * 2 * DV * 4 <= 2 * TILE, "the waves' rows fit the buffers");
        if (row < nrows) {
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const float f = __builtin_amdgcn_exp2f(m_run[m] - top[m]);
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        f32x4 x;
#pragma unroll
                        for (int j = 0; j < 4; ++j) x[j] = acc[m][d][4 * g + j] * f;
                        *reinterpret_cast<f32x4*>(mine + joined<DV>(r, m, d * 32 + 8 * g + 4 * hh)) = x;
                    }
            }
        }
        __syncthreads();
        if (wave == 0 && hh == 0) {                                  // the joined maximum and sum take the first wave's place
            s_ml[0][0][r] = top[0];
            s_ml[0][1][r] = sum[0];
            s_ml[0][2][r] = top[1];
            s_ml[0][3][r] = sum[1];
        }
        __syncthreads();
        const int live = nrows - row0 < 32 ? nrows - row0 : 32;
        const int64_t part = ((int64_t)bk * tiles + tile) * splits + split;
        float* wo = ws + part * 32 * (2 * DV + 4);
        for (int i = tid; i < live * (DV / 4); i += NW * 64) {
            const int rr = i / (DV / 4), col = (i - rr * (DV / 4)) * 4;
            f32x4 x[2];
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                x[m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < NW; ++w)
                    x[m] = x[m] + *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(bufs[w < HALF ? 0 : 1]) +
                                                                  (w % HALF) * 32 * 2 * DV + joined<DV>(rr, m, col));
            }
            if (splits > 1) {
                *reinterpret_cast<f32x4*>(wo + rr * 2 * DV + col) = x[0];
                *reinterpret_cast<f32x4*>(wo + rr * 2 * DV + DV + col) = x[1];
                continue;
            }
            if (col >= 2 * a.d) continue;
            const RowPlace pl = row_place(a, kh, row0 + rr);
            const float l1 = s_ml[0][1][rr], l2 = s_ml[0][3][rr];
            const float i1 = l1 > 0.f || l1 != l1 ? 1.0f / l1 : 0.f, i2 = l2 > 0.f || l2 != l2 ? 1.0f / l2 : 0.f;
            const float w = s_w[rr];
            f32x4 y = x[1] * i2, z;
#pragma unroll
            for (int j = 0; j < 4; ++j) z[j] = fmaf(-w, y[j], x[0][j] * i1);
            const int64_t at = (((int64_t)b * a.nq + pl.tok) * a.heads + pl.head) * 2 * a.d + col;
            store4(out + at, z);
            if (out2) store4(out2 + at, y);
        }
        if (wave == 0 && row < nrows && hh == 0) {
            if (splits > 1) {
                float* ml = wo + 32 * 2 * DV + r * 4;
                ml[0] = top[0];
                ml[1] = sum[0];
                ml[2] = top[1];
                ml[3] = sum[1];
            } else if (out2) {
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    o.stats[m * lmap + lrow] = sum[m] == 0.f ? 0.f : top[m];
                    o.stats[(2 + m) * lmap + lrow] = sum[m] == 0.f ? 0.f : 1.0f / sum[m];
                }
                if (b == 0 && place.tok == 0) o.weight[place.head] = weight;
            }
        }
    }
}

// The splits of the keys joined: a workgroup per tile of 32 rows.
template <class T, int DV>
__global__ __launch_bounds__(256) void diff_fwd_join(DiffArgs a, DiffOut o, const float* __restrict__ ws, int tiles,
                                                     int splits) {
    __shared__ float s_top[2][32], s_inv[2][32], s_w[32];
    const int tid = threadIdx.x, lane = tid & 63;
    const int bk = blockIdx.x / tiles, tile = blockIdx.x - bk * tiles;
    const int b = bk / a.kv_heads, kh = bk - b * a.kv_heads;
    const int nrows = a.nq * a.group, row0 = tile * 32;
    const int live = nrows - row0 < 32 ? nrows - row0 : 32;
    constexpr int STRIDE = 32 * (2 * DV + 4);
    const float* base = ws + ((int64_t)bk * tiles + tile) * splits * STRIDE;
    if (tid < 64) {
        const int r = lane & 31, hh = lane >> 5;                     // half-wave m joins map m
        const int rr = r < live ? r : live - 1;
        const RowPlace pl = row_place(a, kh, row0 + rr);
        float top = kNoScore, sum = 0.f;
        for (int s = 0; s < splits; ++s) top = fmaxf(top, base[(int64_t)s * STRIDE + 32 * 2 * DV + rr * 4 + 2 * hh]);
        for (int s = 0; s < splits; ++s) {
            const float* ml = base + (int64_t)s * STRIDE + 32 * 2 * DV + rr * 4 + 2 * hh;
            sum += ml[1] * __builtin_amdgcn_exp2f(ml[0] - top);
        }
        s_top[hh][r] = top;
        s_inv[hh][r] = sum > 0.f || sum != sum ? 1.0f / sum : 0.f;
        const float w = map_weight<DV / 2>(a, pl.head, hh);
        if (hh == 0) s_w[r] = w;
        if (o.out2 && r < live) {
            const int64_t lmap = (int64_t)a.batch * a.heads * a.nq, at = ((int64_t)b * a.heads + pl.head) * a.nq + pl.tok;
            o.stats[hh * lmap + at] = sum == 0.f ? 0.f : top;
            o.stats[(2 + hh) * lmap + at] = s_inv[hh][r];
            if (b == 0 && pl.tok == 0 && hh == 0) o.weight[pl.head] = w;
        }
    }
    __syncthreads();
    for (int i = tid; i < live * (DV / 4); i += 256) {
        const int rr = i / (DV / 4), col = (i - rr * (DV / 4)) * 4;
        if (col >= 2 * a.d) continue;
        f32x4 x[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
        for (int s = 0; s < splits; ++s) {
            const float* p = base + (int64_t)s * STRIDE;
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const float f = __builtin_amdgcn_exp2f(p[32 * 2 * DV + rr * 4 + 2 * m] - s_top[m][rr]);
                const f32x4 v = *reinterpret_cast<const f32x4*>(p + rr * 2 * DV + m * DV + col);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[m][j] = fmaf(v[j], f, x[m][j]);
            }
        }
        const RowPlace pl = row_place(a, kh, row0 + rr);
        const f32x4 y = x[1] * s_inv[1][rr];
        f32x4 z;
#pragma unroll
        for (int j = 0; j < 4; ++j) z[j] = fmaf(-s_w[rr], y[j], x[0][j] * s_inv[0][rr]);
        const int64_t at = (((int64_t)b * a.nq + pl.tok) * a.heads + pl.head) * 2 * a.d + col;
        store4(reinterpret_cast<T*>(o.out) + at, z);
        if (o.out2) store4(reinterpret_cast<T*>(o.out2) + at, y);
    }
}

struct Plan {
    bool keys;
    int tiles, splits;
};

// Which form, and into how many workgroups.  Few rows (at most 32 to a key head), or so few workgroups of 128 rows that
// most of the 256 CUs would have none: the waves share the rows and split the keys.
template <class T, int DP>
Plan plan(const DiffArgs& a) {
    const int64_t nrows = (int64_t)a.nq * a.group, bks = (int64_t)a.batch * a.kv_heads;
    Plan p;
    const int64_t wide = bks * ((nrows + 127) / 128);
    p.keys = nrows <= 32 || wide < 128;
    p.tiles = (int)(p.keys ? (nrows + 31) / 32 : (nrows + 127) / 128);
    p.splits = 1;
    if (p.keys) {
        const int kc = 32 * keys_waves<T, DP>();
        const int64_t chunks = ((int64_t)a.nk + kc - 1) / kc, blocks = bks * p.tiles;
        int64_t s = (256 + blocks - 1) / blocks;
        if (s > chunks) s = chunks;
        if (s > 128) s = 128;
        p.splits = s < 1 ? 1 : (int)s;
    }
    return p;
}

template <class T, int DP>
int64_t workspace(const DiffArgs& a) {
    const Plan p = plan<T, DP>(a);
    return p.splits > 1 ? (int64_t)a.batch * a.kv_heads * p.tiles * p.splits * 32 * (4 * DP + 4) : 0;
}

template <class T, int DP>
hipError_t launch(const DiffArgs& a, const DiffOut& o, float* ws, hipStream_t s) {
    const Plan p = plan<T, DP>(a);
    const int64_t blocks = (int64_t)a.batch * a.kv_heads * p.tiles * p.splits;
    if (blocks > 0x7FFFFFFF) return hipErrorInvalidValue;
    constexpr int NK = keys_waves<T, DP>();
    if (p.keys) hipLaunchKernelGGL((diff_fwd<T, DP, NK, true>), dim3((int)blocks), dim3(NK * 64), 0, s, a, o, ws, p.tiles, p.splits);
    else hipLaunchKernelGGL((diff_fwd<T, DP, 4, false>), dim3((int)blocks), dim3(256), 0, s, a, o, ws, p.tiles, 1);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits == 1) return e;
    hipLaunchKernelGGL((diff_fwd_join<T, 2 * DP>), dim3(a.batch * a.kv_heads * p.tiles), dim3(256), 0, s, a, o, ws, p.tiles, p.splits);
    return hipGetLastError();
}

template <class F>
auto by_size(int d, bool bf16, F&& f) {
    if (bf16) {
        if (d <= 32) return f(bf16_t{}, std::integral_constant<int, 32>{});
        if (d <= 48) return f(bf16_t{}, std::integral_constant<int, 48>{});
        return f(bf16_t{}, std::integral_constant<int, 64>{});
    }
    if (d <= 32) return f(float{}, std::integral_constant<int, 32>{});
    if (d <= 48) return f(float{}, std::integral_constant<int, 48>{});
    return f(float{}, std::integral_constant<int, 64>{});
}

}  // namespace

// f32 values of scratch of the forward
int64_t diff_attention_workspace(const DiffArgs& a, bool bf16) {
    return by_size(a.d, bf16, [&](auto t, auto dp) { return workspace<decltype(t), decltype(dp)::value>(a); });
}

hipError_t launch_diff_attention(const DiffArgs& a, const DiffOut& o, float* ws, bool bf16, hipStream_t s) {
    return by_size(a.d, bf16, [&](auto t, auto dp) { return launch<decltype(t), decltype(dp)::value>(a, o, ws, s); });
}

}  // namespace vitk
