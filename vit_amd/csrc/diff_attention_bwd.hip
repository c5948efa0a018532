// Differential attention, backward (gfx950 / CDNA4).  With P_m rebuilt from the scores and the forward's denominators
// (P_m = exp2(scale log2(e) q_m . k_m - m_m) / l_m with the reference point and the sum that the forward leaves: the
// exponent is small where the probability is large, so a probability is exact to a few 2^-24):
//     dA   = dO V^T                         the gradient of P_1 - w P_2
//     D_m  = sum over keys of P_m dA = dO . (P_m V):   D_2 = dO . O_2,  D_1 = dO . O + w D_2
//     dS_1 = P_1 (dA - D_1),  dS_2 = -w P_2 (dA - D_2)
//     dQ_m = scale dS_m K_m,  dK_m = scale dS_m^T Q_m,  dV = (P_1 - w P_2)^T dO
//     dw_h = - sum over the head's rows and keys of P_2 dA
// Two kernels, so that nothing is added by atomics and results are reproducible: one walks the keys for 128 rows (dQ, and
// the row's share of dw), one walks the rows for 128 keys (dK, dV; the rows of all query heads of a key head, so that shared
// heads need no sum of their own).  dw is added from f32 probabilities and f32 accumulators, not from the rounded O_2.
#include <type_traits>

#include "diff_attention.h"

#ifndef KVOCC
#define KVOCC 1
#endif
#ifndef KVRC
#define KVRC 32
#endif

namespace vitk {

using namespace diff;

namespace {

constexpr int kNW = 4;                        // waves of a workgroup, 32 rows or keys each
constexpr int kBlock = 32 * kNW;

constexpr int pow2_below(int n) { return n >= 16 ? 16 : n >= 8 ? 8 : n >= 4 ? 4 : n >= 2 ? 2 : 1; }

__device__ __forceinline__ int sample_len(const DiffArgs& a, int b) {
    if (!a.key_lens) return a.nk;
    const int n = a.key_lens[b];
    return n < 0 ? 0 : (n < a.nk ? n : a.nk);
}

template <class T>
__device__ __forceinline__ float dot(typename Op<T>::Chunk x, typename Op<T>::Chunk y) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < Op<T>::kPer; ++j) s = fmaf((float)x[j], (float)y[j], s);
    return s;
}

// dQ of 128 rows, their D_m (ws_d [2, batch, heads, nq]) and the workgroup's share of every head's dw (ws_w)
template <class T, int DP>
__global__ __launch_bounds__(256, sizeof(T) == 4 ? 1 : 2) void diff_bwd_q(DiffArgs a, DiffGrads g, float* __restrict__ ws_d,
                                                                          float* __restrict__ ws_w, int tiles) {
    constexpr int DV = 2 * DP;
    constexpr int RB = row_bytes<T, DV>();
    constexpr int PER = Op<T>::kPer;
    constexpr int DPC = DP / PER, KT = DPC / 2;
    constexpr int EB = (DP + 31) / 32;
    constexpr int KC = 32, TILE = KC * RB;
    typedef typename Op<T>::Chunk Chunk;
    __shared__ __align__(16) char bufs[2][2 * TILE];
    __shared__ float s_dw[kBlock];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 31, hh = lane >> 5;
    const int bks = a.batch * a.kv_heads;
    const int bk = blockIdx.x % bks, rest = blockIdx.x / bks;
    const int tile = a.causal ? tiles - 1 - rest : rest;
    const int b = bk / a.kv_heads, kh = bk - b * a.kv_heads;
    const int nrows = a.nq * a.group;
    const int row0 = tile * kBlock + wave * 32, end = (tile + 1) * kBlock;
    const int len = sample_len(a, b);
    const int kmax = key_limit(a, len, row_place(a, kh, (end < nrows ? end : nrows) - 1).tok);

    constexpr int LANES = 4 * DPC;
    constexpr int ROWS = pow2_below(256 / LANES);
    constexpr int PASSES = KC / ROWS;
    const int dc = a.d / PER;
    const int srow = tid / LANES, scol = tid - srow * LANES;
    const bool s_v = scol >= 2 * DPC;
    const int s_c = s_v ? scol - 2 * DPC : scol;
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
    const int c1 = (kmax + KC - 1) / KC;
    if (c1 > 0) fetch(0);

    const int row = row0 + r;
    const RowPlace place = row_place(a, kh, row < nrows ? row : nrows - 1);
    const int lim = key_limit(a, len, place.tok);
    const int wave_max = key_limit(a, len, row_place(a, kh, (row0 + 32 < nrows ? row0 + 32 : nrows) - 1).tok);
    const int wave_min = key_limit(a, len, row_place(a, kh, row0 < nrows ? row0 : nrows - 1).tok);
    const bool active = row0 < nrows;
    const int64_t lrow = ((int64_t)b * a.heads + place.head) * a.nq + place.tok;
    const int64_t lmap = (int64_t)a.batch * a.heads * a.nq;
    const float weight = g.weight[place.head];
    const float ref[2] = {g.stats[lrow], g.stats[lmap + lrow]};
    const float inv[2] = {g.stats[2 * lmap + lrow], g.stats[3 * lmap + lrow]};

    Chunk qf[2][KT], of[2 * KT];
    float dd[2];
    {
        const T* qg = reinterpret_cast<const T*>(a.q) + b * a.qs[0] + place.tok * a.qs[1] + place.head * a.qs[2];
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                const int c = 2 * t + hh;
                qf[m][t] = *reinterpret_cast<const Chunk*>(c < dc ? (const void*)(qg + m * a.qs[3] + c * PER) : (const void*)kZeros);
            }
        const int64_t orow = (((int64_t)b * a.nq + place.tok) * a.heads + place.head) * 2 * a.d;
        float d0 = 0.f, d2 = 0.f;
#pragma unroll
        for (int t = 0; t < 2 * KT; ++t) {
            const int c = 2 * t + hh;
            const bool on = c < 2 * dc;
            auto at = [&](const void* p) {
                return *reinterpret_cast<const Chunk*>(on ? (const void*)(reinterpret_cast<const T*>(p) + orow + c * PER) : (const void*)kZeros);
            };
            of[t] = at(g.dout);
            d0 += dot<T>(of[t], at(g.out));
            d2 += dot<T>(of[t], at(g.out2));
        }
        dd[1] = both_sum(d2);
        dd[0] = fmaf(weight, dd[1], both_sum(d0));
        if (row < nrows && hh == 0) {
            ws_d[lrow] = dd[0];
            ws_d[lmap + lrow] = dd[1];
        }
    }

    f32x16 dq[2][EB];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int e = 0; e < EB; ++e) dq[m][e] = zero16();
    float dw = 0.f;
    const float sc = a.scale * kLog2e;

    if (c1 > 0) put(bufs[0]);
    __syncthreads();
    for (int c = 0; c < c1; ++c) {
        const char* kt = bufs[c & 1];
        const char* vt = kt + TILE;
        const bool more = c + 1 < c1;
        if (more) fetch((c + 1) * KC);
        const int key0 = c * KC;
        if (active && key0 < wave_max) {
            f32x16 s[2], da = zero16();
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                s[m] = zero16();
#pragma unroll
                for (int t = 0; t < KT; ++t) s[m] = Op<T>::mma(chunk_at<T, RB>(kt, r, m * DPC + 2 * t + hh), qf[m][t], s[m]);
            }
#pragma unroll
            for (int t = 0; t < 2 * KT; ++t) da = Op<T>::mma(chunk_at<T, RB>(vt, r, 2 * t + hh), of[t], da);
            if (key0 + 32 > wave_min) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (key0 + 8 * (i >> 2) + 4 * hh + (i & 3) >= lim) s[0][i] = s[1][i] = -__builtin_inff();
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float p1 = __builtin_amdgcn_exp2f(fmaf(s[0][i], sc, -ref[0]));       // times 1 / l at the end
                const float p2 = __builtin_amdgcn_exp2f(fmaf(s[1][i], sc, -ref[1]));
                dw = fmaf(p2, da[i], dw);
                s[0][i] = p1 * (da[i] - dd[0]);
                s[1][i] = p2 * (da[i] - dd[1]);
            }
#pragma unroll
            for (int st = 0; st < 2; ++st)
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    Slice<T> ds;
                    ds.take(s[m], st);
#pragma unroll
                    for (int e = 0; e < EB; ++e) {
                        Trans<T, RB> k;
                        k.load(kt, 16 * st, m * DP + e * 32, lane);
                        dq[m][e] = mma_t(k, ds, dq[m][e]);
                    }
                }
        }
        if (more) put(bufs[(c + 1) & 1]);
        __syncthreads();
    }

    dw = both_sum(dw) * inv[1];
    if (hh == 0) s_dw[wave * 32 + r] = row < nrows ? -dw : 0.f;
    __syncthreads();
    for (int h = tid; h < a.group; h += 256) {
        // rows of the workgroup that belong to the group's head h
        const int first = tile * kBlock;
        float t = 0.f;
        for (int i = (h - first % a.group + a.group) % a.group; i < kBlock; i += a.group) t += s_dw[i];
        ws_w[((int64_t)bk * tiles + tile) * a.group + h] = t;
    }
    if (row >= nrows) return;
    T* out = reinterpret_cast<T*>(g.dq) + b * g.dqs[0] + place.tok * g.dqs[1] + place.head * g.dqs[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const float f = m == 0 ? inv[0] * a.scale : -weight * inv[1] * a.scale;
#pragma unroll
        for (int e = 0; e < EB; ++e)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int col = e * 32 + 8 * q + 4 * hh;
                if (col >= a.d) continue;
                store4(out + m * g.dqs[3] + col,
                       f32x4{dq[m][e][4 * q] * f, dq[m][e][4 * q + 1] * f, dq[m][e][4 * q + 2] * f, dq[m][e][4 * q + 3] * f});
            }
    }
}

// dK and dV of 128 keys
template <class T, int DP, int RC>
__global__ __launch_bounds__(256, KVOCC) void diff_bwd_kv(DiffArgs a, DiffGrads g, const float* __restrict__ ws_d, int tiles) {
    constexpr int DV = 2 * DP;
    constexpr int RB = row_bytes<T, DV>();
    constexpr int PER = Op<T>::kPer;
    constexpr int DPC = DP / PER, KT = DPC / 2;
    constexpr int DB = DV / 32, EB = (DP + 31) / 32;
    constexpr int TILE = RC * RB;                                     // RC: rows of a chunk
    typedef typename Op<T>::Chunk Chunk;
    __shared__ __align__(16) char bufs[2][2 * TILE];                  // Q of both maps, dO
    __shared__ __align__(16) float s_row[2][6][RC];                   // m_1, m_2, 1 / l_1, w / l_2, D_1, D_2 of the rows
    __shared__ __align__(16) int s_lim[2][RC];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 31, hh = lane >> 5;
    const int bks = a.batch * a.kv_heads;
    const int bk = blockIdx.x % bks, tile = blockIdx.x / bks;
    const int b = bk / a.kv_heads, kh = bk - b * a.kv_heads;
    const int nrows = a.nq * a.group;
    const int len = sample_len(a, b);
    const int block0 = tile * kBlock, key0 = block0 + wave * 32, key = key0 + r;
    // rows from the first one that sees a key of this workgroup
    int first = 0;
    if (a.causal) {
        const int t = block0 - (a.nk - a.nq);
        first = t > 0 ? t * a.group / RC : 0;
    }
    const int c1 = block0 < len ? (nrows + RC - 1) / RC : 0;

    constexpr int LANES = 4 * DPC;
    constexpr int ROWS = pow2_below(256 / LANES);
    constexpr int PASSES = RC / ROWS;
    const int dc = a.d / PER;
    const int srow = tid / LANES, scol = tid - srow * LANES;
    const bool s_o = scol >= 2 * DPC;
    const int s_c = s_o ? scol - 2 * DPC : scol;
    const int s_m = !s_o && s_c >= DPC ? 1 : 0, s_e = s_c - s_m * DPC;
    const bool s_on = srow < ROWS && (s_o ? s_c < 2 * dc : s_e < dc);
    const T* qg = reinterpret_cast<const T*>(a.q) + b * a.qs[0] + s_m * a.qs[3] + s_e * PER;
    const T* og = reinterpret_cast<const T*>(g.dout) + (int64_t)b * a.nq * a.heads * 2 * a.d + s_c * PER;
    const int64_t lmap = (int64_t)a.batch * a.heads * a.nq;
    u32x4 held[PASSES];
    float held_r[6];
    int held_l = 0;
    auto fetch = [&](int c) {
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int row = c * RC + srow + i * ROWS;
            held[i] = u32x4{0u, 0u, 0u, 0u};
            if (s_on && row < nrows) {
                const RowPlace pl = row_place(a, kh, row);
                const T* src = s_o ? og + ((int64_t)pl.tok * a.heads + pl.head) * 2 * a.d : qg + pl.tok * a.qs[1] + pl.head * a.qs[2];
                held[i] = *reinterpret_cast<const u32x4*>(src);
            }
        }
        if (tid < RC) {
            const int row = c * RC + tid;
            held_l = 0;
#pragma unroll
            for (int j = 0; j < 6; ++j) held_r[j] = 0.f;
            if (row < nrows) {
                const RowPlace pl = row_place(a, kh, row);
                const int64_t at = ((int64_t)b * a.heads + pl.head) * a.nq + pl.tok;
                held_r[0] = g.stats[at];
                held_r[1] = g.stats[lmap + at];
                held_r[2] = g.stats[2 * lmap + at];
                held_r[3] = g.stats[3 * lmap + at] * g.weight[pl.head];
                held_r[4] = ws_d[at];
                held_r[5] = ws_d[lmap + at];
                held_l = key_limit(a, len, pl.tok);
            }
        }
    };
    auto put = [&](int k) {
        if (srow < ROWS) {
#pragma unroll
            for (int i = 0; i < PASSES; ++i) {
                const int lr = srow + i * ROWS;
                *reinterpret_cast<u32x4*>(bufs[k] + (s_o ? TILE : 0) + lr * RB + ((s_c ^ swz<RB>(lr)) << 4)) = held[i];
            }
        }
        if (tid < RC) {
#pragma unroll
            for (int j = 0; j < 6; ++j) s_row[k][j][tid] = held_r[j];
            s_lim[k][tid] = held_l;
        }
    };
    if (first < c1) fetch(first);

    Chunk kf[2][KT], vf[2 * KT];
    {
        const bool on = key < len;
        const T* kg = reinterpret_cast<const T*>(a.k) + b * a.ks[0] + kh * a.ks[2] + (int64_t)(on ? key : 0) * a.ks[1];
        const T* vg = reinterpret_cast<const T*>(a.v) + b * a.vs[0] + kh * a.vs[2] + (int64_t)(on ? key : 0) * a.vs[1];
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                const int c = 2 * t + hh;
                kf[m][t] = *reinterpret_cast<const Chunk*>(on && c < dc ? (const void*)(kg + m * a.ks[3] + c * PER) : (const void*)kZeros);
            }
#pragma unroll
        for (int t = 0; t < 2 * KT; ++t) {
            const int c = 2 * t + hh;
            vf[t] = *reinterpret_cast<const Chunk*>(on && c < 2 * dc ? (const void*)(vg + c * PER) : (const void*)kZeros);
        }
    }

    f32x16 dk[2][EB], dv[DB];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int e = 0; e < EB; ++e) dk[m][e] = zero16();
#pragma unroll
    for (int d = 0; d < DB; ++d) dv[d] = zero16();
    const float sc = a.scale * kLog2e;

    auto work = [&](const char* qt, const char* ot, int k, int rb, bool masked) {
                    f32x16 s[2], da = zero16();
        #pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        s[m] = zero16();
        #pragma unroll
                        for (int t = 0; t < KT; ++t) s[m] = Op<T>::mma(chunk_at<T, RB>(qt, rb + r, m * DPC + 2 * t + hh), kf[m][t], s[m]);
                    }
        #pragma unroll
                    for (int t = 0; t < 2 * KT; ++t) da = Op<T>::mma(chunk_at<T, RB>(ot, rb + r, 2 * t + hh), vf[t], da);
                    f32x16 pa;
        #pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int at = rb + 8 * q + 4 * hh;
                        auto row4 = [&](int j) { return *reinterpret_cast<const f32x4*>(&s_row[k][j][at]); };
                        const f32x4 m1 = row4(0), m2 = row4(1), i1 = row4(2), w2 = row4(3), d1 = row4(4), d2 = row4(5);
        #pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int i = 4 * q + j;
                            float p1 = __builtin_amdgcn_exp2f(fmaf(s[0][i], sc, -m1[j])) * i1[j];
                            float wp2 = __builtin_amdgcn_exp2f(fmaf(s[1][i], sc, -m2[j])) * w2[j];
                            if (masked && key >= s_lim[k][at + j]) p1 = wp2 = 0.f;
                            pa[i] = p1 - wp2;
                            s[0][i] = p1 * (da[i] - d1[j]);
                            s[1][i] = wp2 * (d2[j] - da[i]);
                        }
                    }
        #pragma unroll
                    for (int st = 0; st < 2; ++st) {
                        Slice<T> p, d0, d1;
                        p.take(pa, st);
                        d0.take(s[0], st);
                        d1.take(s[1], st);
        #pragma unroll
                        for (int d = 0; d < DB; ++d) {
                            Trans<T, RB> o;
                            o.load(ot, rb + 16 * st, d * 32, lane);
                            dv[d] = mma_t(o, p, dv[d]);
                        }
        #pragma unroll
                        for (int e = 0; e < EB; ++e) {
                            Trans<T, RB> q0, q1;
                            q0.load(qt, rb + 16 * st, e * 32, lane);
                            q1.load(qt, rb + 16 * st, DP + e * 32, lane);
                            dk[0][e] = mma_t(q0, d0, dk[0][e]);
                            dk[1][e] = mma_t(q1, d1, dk[1][e]);
                        }
                    }
    };
    if (first < c1) put(0);
    __syncthreads();
    for (int c = first; c < c1; ++c) {
        const int k = (c - first) & 1;
        const char* qt = bufs[k];
        const char* ot = qt + TILE;
        const bool more = c + 1 < c1;
        if (more) fetch(c + 1);
#pragma unroll
        for (int rb = 0; rb < RC; rb += 32) {
            // the block's last row sees most: nothing to do where that is below the wave's keys
            const int at0 = c * RC + rb, last = at0 + 32 < nrows ? at0 + 32 : nrows;
            const int most = at0 < nrows ? key_limit(a, len, row_place(a, kh, last - 1).tok) : 0;
            const int least = at0 < nrows ? key_limit(a, len, row_place(a, kh, at0).tok) : 0;
            if (key0 < most) work(qt, ot, k, rb, key0 + 32 > least);
        }
        if (more) put(k ^ 1);
        __syncthreads();
    }

    if (key >= a.nk) return;
    T* ko = reinterpret_cast<T*>(g.dk) + b * g.dks[0] + (int64_t)key * g.dks[1] + kh * g.dks[2];
    T* vo = reinterpret_cast<T*>(g.dv) + b * g.dvs[0] + (int64_t)key * g.dvs[1] + kh * g.dvs[2];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int e = 0; e < EB; ++e)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int col = e * 32 + 8 * q + 4 * hh;
                if (col >= a.d) continue;
                store4(ko + m * g.dks[3] + col, f32x4{dk[m][e][4 * q] * a.scale, dk[m][e][4 * q + 1] * a.scale,
                                                      dk[m][e][4 * q + 2] * a.scale, dk[m][e][4 * q + 3] * a.scale});
            }
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int col = d * 32 + 8 * q + 4 * hh;
            if (col >= 2 * a.d) continue;
            store4(vo + col, f32x4{dv[d][4 * q], dv[d][4 * q + 1], dv[d][4 * q + 2], dv[d][4 * q + 3]});
        }
}

// dlam of one lam head from the workgroups' shares of dw: dlam_0 = dw e_1 lam_1, dlam_1 = dw e_1 lam_0, and the second
// pair with -e_2; a lam that all heads share collects all of them.
__global__ __launch_bounds__(256) void diff_bwd_lam(DiffArgs a, const float* __restrict__ ws_w, int tiles, float* __restrict__ dlam) {
    __shared__ double red[256];
    const int lh = blockIdx.x, tid = threadIdx.x;
    const int64_t per = (int64_t)tiles * a.group, total = (int64_t)a.batch * a.kv_heads * per;
    double t = 0.0;
    if (a.lam_heads == 1) {
        for (int64_t i = tid; i < total; i += 256) t += ws_w[i];
    } else {
        const int kh = lh / a.group, h = lh - kh * a.group;
        for (int64_t i = tid; i < (int64_t)a.batch * tiles; i += 256) {
            const int64_t b = i / tiles, tl = i - b * tiles;
            t += ws_w[((b * a.kv_heads + kh) * tiles + tl) * a.group + h];
        }
    }
    red[tid] = t;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
        if (tid < o) red[tid] += red[tid + o];
        __syncthreads();
    }
    if (tid >= 64) return;
    const float dw = (float)red[0];
    const int64_t vs = (int64_t)a.lam_heads * a.d, at = (int64_t)lh * a.d;
    const float* p = a.lam + at;
    float s1 = 0.f, s2 = 0.f;
    for (int e = tid; e < a.d; e += 64) {
        s1 = fmaf(p[e], p[vs + e], s1);
        s2 = fmaf(p[2 * vs + e], p[3 * vs + e], s2);
    }
    const float f1 = dw * expf(wave_sum(s1)), f2 = -dw * expf(wave_sum(s2));
    for (int e = tid; e < a.d; e += 64) {
        dlam[at + e] = f1 * p[vs + e];
        dlam[vs + at + e] = f1 * p[e];
        dlam[2 * vs + at + e] = f2 * p[3 * vs + e];
        dlam[3 * vs + at + e] = f2 * p[2 * vs + e];
    }
}

template <class T, int DP>
hipError_t launch(const DiffArgs& a, const DiffGrads& g, float* ws, hipStream_t s) {
    const int64_t bks = (int64_t)a.batch * a.kv_heads;
    const int qt = (int)(((int64_t)a.nq * a.group + kBlock - 1) / kBlock), kt = (a.nk + kBlock - 1) / kBlock;
    if (bks * qt > 0x7FFFFFFF || bks * kt > 0x7FFFFFFF) return hipErrorInvalidValue;
    float* ws_d = ws;
    float* ws_w = ws + 2 * (int64_t)a.batch * a.heads * a.nq;
    hipLaunchKernelGGL((diff_bwd_q<T, DP>), dim3((int)(bks * qt)), dim3(256), 0, s, a, g, ws_d, ws_w, qt);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((diff_bwd_kv<T, DP, KVRC>), dim3((int)(bks * kt)), dim3(256), 0, s, a, g, ws_d, kt);
    e = hipGetLastError();
    if (e != hipSuccess || !g.dlam) return e;
    hipLaunchKernelGGL(diff_bwd_lam, dim3(a.lam_heads), dim3(256), 0, s, a, ws_w, qt, g.dlam);
    return hipGetLastError();
}

}  // namespace

// f32 values of scratch of the backward
int64_t diff_attention_bwd_workspace(const DiffArgs& a, bool) {
    const int64_t rows = (int64_t)a.nq * a.group;
    return 2 * (int64_t)a.batch * a.heads * a.nq + (int64_t)a.batch * a.kv_heads * ((rows + kBlock - 1) / kBlock) * a.group;
}

hipError_t launch_diff_attention_backward(const DiffArgs& a, const DiffGrads& g, float* ws, bool bf16, hipStream_t s) {
    if (bf16) {
        if (a.d <= 32) return launch<bf16_t, 32>(a, g, ws, s);
        if (a.d <= 48) return launch<bf16_t, 48>(a, g, ws, s);
        return launch<bf16_t, 64>(a, g, ws, s);
    }
    if (a.d <= 32) return launch<float, 32>(a, g, ws, s);
    if (a.d <= 48) return launch<float, 48>(a, g, ws, s);
    return launch<float, 64>(a, g, ws, s);
}

}  // namespace vitk
