// Differential attention, backward (gfx950 / CDNA4).  With P_m rebuilt from the scores and the forward's denominators
// (P_m = exp2(scale log2(e) q_m . k_m - m_m) / l_m with the reference point and the sum that the forward leaves: the
// exponent is small where the probability is large, so a probability is exact to a few 2^-24):
//     dA   = dO V^T                         the gradient of P_1 - w P_2
//     D_m  = sum over keys of P_m dA = dO . (P_m V):   D_2 = dO . O_2,  D_1 = dO . O + w D_2
//     dS_1 = P_1 (dA - D_1),  dS_2 = -w P_2 (dA - D_2)
//     dQ_m = scale dS_m K_m,  dK_m = scale dS_m^T Q_m,  dV = (P_1 - w P_2)^T dO
//     dw_h = - sum over the head's rows and keys of P_2 dA
// Two kernels, so that nothing is added by atomics and results are reproducible: one walks the keys for 64 rows (dQ, and the
// row's share of dw), one walks the rows for 128 keys (64 in f32: dK, dV; the rows of all query heads of a key head, so that
// shared heads need no sum of their own).  Where that leaves CUs without work the keys or rows are split too, and kernels of
// their own add the parts.  dw is added from f32 probabilities and f32 accumulators, not from the rounded O_2.
// As in the forward a pair of waves shares 32 rows or keys, one map each: dA is computed by both, everything else once, and
// the registers that leaves allow two waves and more to a SIMD, which hide each other's waiting (one wave with both maps
// took 2.3 times as long at 577 tokens of head size 48, most of it waiting).
// At head size 64 dK / dV fills its 256 registers and spills 7 (1 where no heads share keys).
// Bound by the matrix pipe, the exponentials' arithmetic and the LDS reads that feed the products, which overlap in part: at
// 4096 causal tokens (batch 2, 8 heads of 64, 4 key heads) dQ takes 190 us and 145 of them without its staging, 165 without
// its exponentials, 115 with the products and the transposed reads alone; the products at the matrix pipe's rate are 65.
#include <type_traits>

#include "diff_attention.h"

namespace vitk {

using namespace diff;

namespace {

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

// dQ of 32 NP rows, their D_m (ws_d [2, batch, heads, nq]) and the workgroup's share of every head's dw (ws_w)
// NP: pairs of waves in a workgroup, 32 rows each; OCC: waves to a SIMD that the registers have to allow
template <class T, int DP, int NP, int NB, int OCC>
__global__ __launch_bounds__(NP * 128, OCC) void diff_bwd_q(DiffArgs a, DiffGrads g, float* __restrict__ ws_d,
                                                             float* __restrict__ ws_w, float* __restrict__ parts, int tiles,
                                                             int splits) {
    constexpr int kThreads = NP * 128, kBlock = NP * 32;
    constexpr int DV = 2 * DP;
    constexpr int RB = row_bytes<T, DV>();
    constexpr int PER = Op<T>::kPer;
    constexpr int DPC = DP / PER, KT = DPC / 2;
    constexpr int EB = (DP + 31) / 32;
    constexpr int KC = 32 * NB, TILE = KC * RB;                       // KC: keys of a chunk
    typedef typename Op<T>::Chunk Chunk;
    __shared__ __align__(16) char bufs[2][2 * TILE];
    __shared__ float s_dw[kBlock], s_dot[NP][2][32];

    arguments(a);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), map = wave & 1, grp = wave >> 1;
    const int r = lane & 31, hh = lane >> 5;
    const int bks = a.batch * a.kv_heads;
    const int rest = quotient(blockIdx.x, a.by_bks), bk = blockIdx.x - rest * bks;
    const int turn = rest / splits, split = rest - turn * splits;
    const int tile = a.causal ? tiles - 1 - turn : turn;
    const int b = quotient(bk, a.by_kv_heads), kh = bk - b * a.kv_heads;
    const int nrows = a.nq * a.group;
    const int row0 = tile * kBlock + grp * 32, end = (tile + 1) * kBlock;
    const int len = sample_len(a, b);
    const int kmax = key_limit(a, len, row_place(a, kh, (end < nrows ? end : nrows) - 1).tok);

    const int dc = a.d / PER;
    Stage<T, DP, kThreads, KC> stage;
    stage.init(tid, dc, bufs[0], 2 * TILE);
    const int64_t s_step = stage.second ? a.vs[1] : a.ks[1];
    const T* s_src = stage.row * s_step + (stage.second ? reinterpret_cast<const T*>(a.v) + b * a.vs[0] + kh * a.vs[2] + stage.col * PER
                                                        : reinterpret_cast<const T*>(a.k) + b * a.ks[0] + kh * a.ks[2] + stage.map * a.ks[3] + stage.e * PER);
    auto fetch = [&](int key0) { stage.fetch(key0, kmax, s_src, s_step, 0, [&](int key) { return s_src + (key - stage.row) * s_step; }); };
    int c0 = 0, c1 = (kmax + KC - 1) / KC;
    if (splits > 1) {                                                 // this workgroup's share of the keys
        const int per = (c1 + splits - 1) / splits;
        c0 = split * per;
        c1 = c0 + per < c1 ? c0 + per : c1;
    }
    if (c0 < c1) fetch(c0 * KC);

    const int row = row0 + r;
    const RowPlace place = row_place(a, kh, row < nrows ? row : nrows - 1);
    const int lim = key_limit(a, len, place.tok);
    const int wave_max = key_limit(a, len, row_place(a, kh, (row0 + 32 < nrows ? row0 + 32 : nrows) - 1).tok);
    const int wave_min = key_limit(a, len, row_place(a, kh, row0 < nrows ? row0 : nrows - 1).tok);
    const bool active = row0 < nrows;
    const int64_t lrow = ((int64_t)b * a.heads + place.head) * a.nq + place.tok;
    const int64_t lmap = (int64_t)a.batch * a.heads * a.nq;
    const float weight = g.weight[place.head];
    const float ref = g.stats[map * lmap + lrow], inv = g.stats[(2 + map) * lmap + lrow];

    Chunk qf[KT], of[2 * KT];
    {
        const T* qg = reinterpret_cast<const T*>(a.q) + b * a.qs[0] + place.tok * a.qs[1] + place.head * a.qs[2] + map * a.qs[3];
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            const int c = 2 * t + hh;
            qf[t] = chunk_or_zero<T>(qg, c, c < dc);
        }
        // dO . O by the first map's wave, dO . O_2 by the second's, all loads at once.  In bf16 both carry the rounding of O and
        // O_2 to their type (they are the forward's outputs, kept as such for half the bytes), so D_m is off by up to 2^-8 of a
        // term; dw is not made of it.
        const int64_t orow = (((int64_t)b * a.nq + place.tok) * a.heads + place.head) * 2 * a.d;
        const T* og = reinterpret_cast<const T*>(map ? g.out2 : g.out) + orow;
        Chunk o[2 * KT];
#pragma unroll
        for (int t = 0; t < 2 * KT; ++t) of[t] = chunk_or_zero<T>(reinterpret_cast<const T*>(g.dout) + orow, 2 * t + hh, 2 * t + hh < 2 * dc);
#pragma unroll
        for (int t = 0; t < 2 * KT; ++t) o[t] = chunk_or_zero<T>(og, 2 * t + hh, 2 * t + hh < 2 * dc);
        float s = 0.f;
#pragma unroll
        for (int t = 0; t < 2 * KT; ++t) s += dot<T>(of[t], o[t]);
        s = both_sum(s);
        if (hh == 0) s_dot[grp][map][r] = s;
        // The matrix pipe's rounding leans to one side by some 1e-9 of dA, which a sum over all rows collects while the rows' own
        // terms cancel (dw off by 1e-5 of itself and more at 16 x 577 rows of 8 heads): every other row goes through it negated.
        if (r & 1) {
#pragma unroll
            for (int t = 0; t < 2 * KT; ++t)
#pragma unroll
                for (int j = 0; j < PER; ++j) of[t][j] = -of[t][j];
        }
    }
    const float sign = r & 1 ? -1.f : 1.f;

    f32x16 dq[EB];
#pragma unroll
    for (int e = 0; e < EB; ++e) dq[e] = zero16();
    double dw = 0.0;      // the terms nearly cancel: what a block of keys adds in f32 is collected in f64
    const float sc = a.scale * kLog2e;

    if (c0 < c1) stage.put(bufs[0]);
    loads_done();
    __syncthreads();
    float dd = map ? s_dot[grp][1][r] : fmaf(weight, s_dot[grp][1][r], s_dot[grp][0][r]);
    if (row < nrows && hh == 0 && split == 0) ws_d[map * lmap + lrow] = dd;
    dd *= sign;
    auto chunk = [&](int c, auto which) __attribute__((always_inline)) {                            // the buffer is known when compiled: no address arithmetic
        const char* kt = bufs[decltype(which)::value];
        const char* vt = kt + TILE;
        const bool more = c + 1 < c1;
        if (more) fetch((c + 1) * KC);
#pragma unroll
        for (int kb = 0; kb < KC; kb += 32) {
            const int key0 = c * KC + kb;
            if (!active || key0 >= wave_max) continue;
            f32x16 s = zero16(), da = zero16();
#pragma unroll
            for (int t = 0; t < KT; ++t) s = Op<T>::mma(chunk_at<T, RB>(kt, kb + r, map * DPC + 2 * t + hh), qf[t], s);
#pragma unroll
            for (int t = 0; t < 2 * KT; ++t) da = Op<T>::mma(chunk_at<T, RB>(vt, kb + r, 2 * t + hh), of[t], da);
            if (key0 + 32 > wave_min) hide(s, lim - key0 - 4 * hh);
            float part = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float p = __builtin_amdgcn_exp2f(fmaf(s[i], sc, -ref));     // times 1 / l at the end
                part = fmaf(p, da[i], part);
                s[i] = p * (da[i] - dd);
            }
            dw += (double)part;
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                Slice<T> ds;
                ds.take(s, st);
#pragma unroll
                for (int e = 0; e < EB; ++e) {
                    Trans<T, RB> k;
                    k.load(kt, kb + 16 * st, map * DP + e * 32, lane);
                    dq[e] = mma_t(k, ds, dq[e]);
                }
            }
        }
        if (more) stage.put(bufs[decltype(which)::value ^ 1]);
        __syncthreads();
    };
    for (int c = c0; c < c1; c += 2) {
        chunk(c, std::integral_constant<int, 0>{});
        if (c + 1 < c1) chunk(c + 1, std::integral_constant<int, 1>{});
    }

    const float row_dw = both_sum((float)dw) * inv * sign;
    if (map == 1 && hh == 0) s_dw[grp * 32 + r] = row < nrows ? -row_dw : 0.f;
    __syncthreads();
    for (int h = tid; h < a.group; h += kThreads) {
        // rows of the workgroup that belong to the group's head h
        const int first = tile * kBlock;
        double t = 0.0;
        for (int i = (h - first % a.group + a.group) % a.group; i < kBlock; i += a.group) t += s_dw[i];
        ws_w[(((int64_t)bk * tiles + tile) * splits + split) * a.group + h] = (float)t;
    }
    // [split][sample, head, token][map][d]
    float* part = splits > 1 ? parts + ((split * lmap + lrow) * 2 + map) * a.d : nullptr;
    T* out = reinterpret_cast<T*>(g.dq) + b * g.dqs[0] + place.tok * g.dqs[1] + place.head * g.dqs[2] + map * g.dqs[3];
    const float f = sign * (map == 0 ? inv * a.scale : -weight * inv * a.scale);
#pragma unroll
    for (int e = 0; e < EB; ++e)
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
            const f32x4 x = four(dq[e], q, f), y = four(dq[e], q + 1, f);
            if (part) store_pair(part, e * 32 + 8 * q, hh, a.d, row < nrows, x, y);
            else store_pair(out, e * 32 + 8 * q, hh, a.d, row < nrows, x, y);
        }
}

// dlam of one lam head from the dQ workgroups' shares of dw: dlam_0 = dw e_1 lam_1, dlam_1 = dw e_1 lam_0, and the second
// pair with -e_2; a lam that all heads share collects all of them.  By a workgroup of NT threads, red: NT doubles.
template <int NT>
__device__ __forceinline__ void lam_gradient(const DiffArgs& a, const float* __restrict__ ws_w, int tiles, float* __restrict__ dlam,
                                             int lh, double* red) {
    const int tid = threadIdx.x;
    const int64_t per = (int64_t)tiles * a.group, total = (int64_t)a.batch * a.kv_heads * per;
    double t = 0.0;
    if (a.lam_heads == 1) {
        for (int64_t i = tid; i < total; i += NT) t += ws_w[i];
    } else {
        const int kh = lh / a.group, h = lh - kh * a.group;
        for (int64_t i = tid; i < (int64_t)a.batch * tiles; i += NT) {
            const int64_t b = i / tiles, tl = i - b * tiles;
            t += ws_w[((b * a.kv_heads + kh) * tiles + tl) * a.group + h];
        }
    }
    red[tid] = t;
    __syncthreads();
#pragma unroll
    for (int o = NT / 2; o > 0; o >>= 1) {
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

// dK and dV of 32 NP keys.  What a row contributes beside its Q and dO is folded into the products' initial accumulators:
//     S_m starts at -lse_m / (scale log2 e), so that P_m = exp2(scale log2(e) S_m);  dA starts at -D_m.
// In f32 it starts at the reference point alone and 1 / l_m is multiplied on: lse is the larger number, and its rounding
// would be most of the probability's error (1.1e-6 against 5e-7 in dV at 257 tokens).
// ONE: one query head to a key head, so that w is the workgroup's and can wait until the end (else the rows bring theirs).
template <class T, int DP, bool ONE, int NP, int NB, int OCC>
__global__ __launch_bounds__(NP * 128, OCC) void diff_bwd_kv(DiffArgs a, DiffGrads g, const float* __restrict__ ws_d,
                                                             float* __restrict__ parts, int splits,
                                                             const float* __restrict__ ws_w, int row_tiles, unsigned blocks) {
    constexpr int kThreads = NP * 128, kBlock = NP * 32;
    constexpr int DV = 2 * DP;
    constexpr int RB = row_bytes<T, DV>();
    constexpr int PER = Op<T>::kPer;
    constexpr int DPC = DP / PER, KT = DPC / 2;
    constexpr int DB = DV / 32, EB = (DP + 31) / 32;
    constexpr int RC = 32 * NB, TILE = RC * RB;                       // RC: rows of a chunk
    constexpr bool APART = sizeof(T) == 4;                            // 1 / l apart from the exponent
    constexpr int NS = 4 + (APART ? 2 : 0) + (ONE ? 0 : 1);
    typedef typename Op<T>::Chunk Chunk;
    constexpr int BUF = 2 * TILE > NP * DB * 2048 ? 2 * TILE : NP * DB * 2048;              // DB sums of a pair fit
    __shared__ __align__(16) char bufs[2][BUF];                       // Q of both maps, dO
    __shared__ __align__(16) float s_row[2][NS][RC];                  // -lse_1 / sc, -lse_2 / sc, -D_1, -D_2, 1 / l_1, 1 / l_2, w
    __shared__ __align__(16) int s_lim[2][RC];

    // The last workgroups add up the learned weight's gradient from the shares that the dQ kernel has left: a few sums, not
    // worth a launch
    static_assert(kThreads * 8 <= 2 * BUF, "the sums fit the buffers");
    if (blockIdx.x >= blocks) {
        lam_gradient<kThreads>(a, ws_w, row_tiles, g.dlam, blockIdx.x - blocks, reinterpret_cast<double*>(bufs[0]));
        return;
    }
    arguments(a);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), map = wave & 1, grp = wave >> 1;
    const int r = lane & 31, hh = lane >> 5;
    const int bks = a.batch * a.kv_heads;
    const int rest = quotient(blockIdx.x, a.by_bks), bk = blockIdx.x - rest * bks, tile = rest / splits;      // causal: the first keys have the most rows
    const int b = quotient(bk, a.by_kv_heads), kh = bk - b * a.kv_heads;
    const int nrows = a.nq * a.group;
    const int len = sample_len(a, b);
    const int block0 = tile * kBlock, key0 = block0 + grp * 32, key = key0 + r;
    const float sc = a.scale * kLog2e, rsc = 1.0f / sc;
    // rows from the first one that sees a key of this workgroup
    int first = 0;
    if (a.causal) {
        const int t = block0 - (a.nk - a.nq);
        first = t > 0 ? t * a.group / RC : 0;
    }
    int c1 = block0 < len ? (nrows + RC - 1) / RC : 0;
    if (splits > 1) {                                                 // this workgroup's share of them
        const int per = (c1 - first + splits - 1) / splits;
        first += (rest - tile * splits) * per;
        c1 = first + per < c1 ? first + per : c1;
    }

    const int dc = a.d / PER;
    Stage<T, DP, kThreads, RC> stage;
    stage.init(tid, dc, bufs[0], BUF);
    const int64_t s_tok = stage.second ? (int64_t)a.heads * 2 * a.d : a.qs[1], s_head = stage.second ? 2 * a.d : a.qs[2];
    const T* s_base = stage.second ? reinterpret_cast<const T*>(g.dout) + (int64_t)b * a.nq * a.heads * 2 * a.d + stage.col * PER
                                   : reinterpret_cast<const T*>(a.q) + b * a.qs[0] + stage.map * a.qs[3] + stage.e * PER;
    auto addr = [&](int row) {
        const RowPlace pl = ONE ? RowPlace{row, kh} : row_place(a, kh, row);
        return s_base + pl.tok * s_tok + pl.head * s_head;
    };
    // a group of heads that divides the rows of a pass: the token moves on alike for all of them
    const int s_shift = ONE ? 0 : (a.group & (a.group - 1)) == 0 && a.group <= stage.ROWS ? 31 - __builtin_clz(a.group) : -1;
    const T* s_src = addr(stage.row);
    const int64_t lmap = (int64_t)a.batch * a.heads * a.nq;
    static_assert(4 * RC <= kThreads, "four values of a row have a thread each");
    // the rows' values: a thread brings one to four of them, raw; what is computed from them waits until they are put
    const int role = tid / RC, s_at = tid % RC;                       // 0, 1: -lse of a map;  2, 3: -D of a map
    const float* s_from = role < 2 ? g.stats + role * lmap : ws_d + (role - 2) * lmap;
    float held0 = 0.f, held1 = 0.f, held_w = 0.f;
    auto fetch = [&](int c) {
        stage.fetch(c * RC, nrows, s_src, s_tok, s_shift, addr);
        const int row = c * RC + s_at;
        if (role < 4 && row < nrows) {
            const RowPlace pl = ONE ? RowPlace{row, kh} : row_place(a, kh, row);
            const int64_t at = ((int64_t)b * a.heads + pl.head) * a.nq + pl.tok;
            held0 = s_from[at];
            if (role < 2) held1 = s_from[2 * lmap + at];
            if (!ONE && role == 1) held_w = g.weight[pl.head];
        }
    };
    auto put = [&](int k, int c) {
        stage.put(bufs[k]);
        if (role >= 4) return;
        const int row = c * RC + s_at;
        const bool on = row < nrows;                                  // a row past the last one: P = 0
        float x = role < 2 ? -__builtin_inff() : 0.f;
        if (on) x = role >= 2 ? -held0 : APART ? -held0 * rsc : (__builtin_amdgcn_logf(held1) - held0) * rsc;
        s_row[k][role][s_at] = x;
        if (APART && role < 2) s_row[k][4 + role][s_at] = on ? held1 : 0.f;
        if (!ONE && role == 1) s_row[k][NS - 1][s_at] = on ? held_w : 0.f;
        if (role == 0) s_lim[k][s_at] = on ? key_limit(a, len, ONE ? row : row_place(a, kh, row).tok) : 0;
    };
    if (first < c1) fetch(first);

    Chunk kf[KT], vf[2 * KT];
    {
        const bool on = key < len;
        const T* kg = reinterpret_cast<const T*>(a.k) + b * a.ks[0] + kh * a.ks[2] + map * a.ks[3] + (int64_t)(on ? key : 0) * a.ks[1];
        const T* vg = reinterpret_cast<const T*>(a.v) + b * a.vs[0] + kh * a.vs[2] + (int64_t)(on ? key : 0) * a.vs[1];
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            const int c = 2 * t + hh;
            kf[t] = chunk_or_zero<T>(kg, c, on && c < dc);
        }
#pragma unroll
        for (int t = 0; t < 2 * KT; ++t) {
            const int c = 2 * t + hh;
            vf[t] = chunk_or_zero<T>(vg, c, on && c < 2 * dc);
        }
    }

    f32x16 dk[EB], dv[DB];
#pragma unroll
    for (int e = 0; e < EB; ++e) dk[e] = zero16();
#pragma unroll
    for (int d = 0; d < DB; ++d) dv[d] = zero16();

    if (first < c1) put(0, first);
    loads_done();
    __syncthreads();
    auto chunk = [&](int c, auto which) __attribute__((always_inline)) {
        const int k = which;
        const char* qt = bufs[k];
        const char* ot = qt + TILE;
        const bool more = c + 1 < c1;
        if (more) fetch(c + 1);
        // what the chunk's rows see grows with the row: nothing to do where a block's last one sees none of the wave's keys
#pragma unroll 1
        for (int rb = 0; rb < RC; rb += 32) {
            const int at0 = c * RC + rb, last = at0 + 32 < nrows ? at0 + 32 : nrows;
            if (at0 >= nrows) continue;
            if (key0 >= key_limit(a, len, row_place(a, kh, last - 1).tok)) continue;
            auto rows16 = [&](int j) {                                // row values in the accumulators' layout
                f32x16 v;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f32x4 x = *reinterpret_cast<const f32x4*>(&s_row[k][j][rb + 8 * q + 4 * hh]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[4 * q + i] = x[i];
                }
                return v;
            };
            f32x16 s = rows16(map), da = rows16(2 + map);
#pragma unroll
            for (int t = 0; t < KT; ++t) s = Op<T>::mma(chunk_at<T, RB>(qt, rb + r, map * DPC + 2 * t + hh), kf[t], s);
#pragma unroll
            for (int t = 0; t < 2 * KT; ++t) da = Op<T>::mma(chunk_at<T, RB>(ot, rb + r, 2 * t + hh), vf[t], da);
            if (key0 + 32 > key_limit(a, len, row_place(a, kh, at0).tok)) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (key >= s_lim[k][rb + 8 * (i >> 2) + 4 * hh + (i & 3)]) s[i] = -__builtin_inff();
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(s[i] * sc);
            if constexpr (APART) s = s * rows16(4 + map);
            if constexpr (!ONE) {
                if (map == 1) s = s * rows16(NS - 1);
            }
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                Slice<T> p, ds;
                p.take(s, st);
                f32x16 x;
#pragma unroll
                for (int i = 8 * st; i < 8 * st + 8; ++i) x[i] = s[i] * da[i];
                ds.take(x, st);
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    Trans<T, RB> o;
                    o.load(ot, rb + 16 * st, d * 32, lane);
                    dv[d] = mma_t(o, p, dv[d]);
                }
#pragma unroll
                for (int e = 0; e < EB; ++e) {
                    Trans<T, RB> q;
                    q.load(qt, rb + 16 * st, map * DP + e * 32, lane);
                    dk[e] = mma_t(q, ds, dk[e]);
                }
            }
        }
        if (more) put(k ^ 1, c + 1);
        __syncthreads();
    };
    if constexpr (sizeof(T) == 4) {                                   // twice the body costs f32 more than the addresses: 138 / 134 us, 167 / 159
        for (int c = first; c < c1; ++c) chunk(c, (c - first) & 1);
    } else {
        for (int c = first; c < c1; c += 2) {
            chunk(c, std::integral_constant<int, 0>{});
            if (c + 1 < c1) chunk(c + 1, std::integral_constant<int, 1>{});
        }
    }

    const bool live = key < a.nk;
    const float f = map == 0 ? 1.f : ONE ? -g.weight[kh] : -1.f;      // the second map's part
    // [split][sample, key head][key][dK of both maps, dV]
    float* part = splits > 1 ? parts + (((int64_t)(rest - tile * splits) * bks + bk) * a.nk + key) * 4 * a.d : nullptr;
    {
        T* ko = reinterpret_cast<T*>(g.dk) + b * g.dks[0] + (int64_t)key * g.dks[1] + kh * g.dks[2] + map * g.dks[3];
        const float fk = f * a.scale;
#pragma unroll
        for (int e = 0; e < EB; ++e)
#pragma unroll
            for (int q = 0; q < 4; q += 2) {
                const f32x4 x = four(dk[e], q, fk), y = four(dk[e], q + 1, fk);
                if (part) store_pair(part + map * a.d, e * 32 + 8 * q, hh, a.d, live, x, y);
                else store_pair(ko, e * 32 + 8 * q, hh, a.d, live, x, y);
            }
    }
    // the pair's waves exchange their parts of dV: the first finishes the first D0 blocks of 32 columns, the second the others
    T* vo = reinterpret_cast<T*>(g.dv) + b * g.dvs[0] + (int64_t)key * g.dvs[1] + kh * g.dvs[2];
    constexpr int D0 = (DB + 1) / 2;
    f32x4* box = reinterpret_cast<f32x4*>(bufs[0]) + grp * DB * 256 + lane;
#pragma unroll
    for (int d = 0; d < DB; ++d) {
        if ((d < D0) == (map == 0)) continue;
#pragma unroll
        for (int q = 0; q < 4; ++q) box[d * 256 + q * 64] = four(dv[d], q, f);
    }
    __syncthreads();
#pragma unroll
    for (int d = 0; d < DB; ++d) {
        if ((d < D0) != (map == 0)) continue;
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
            const f32x4 x = four(dv[d], q, f) + box[d * 256 + q * 64], y = four(dv[d], q + 1, f) + box[d * 256 + (q + 1) * 64];
            if (part) store_pair(part + 2 * a.d, d * 32 + 8 * q, hh, 2 * a.d, live, x, y);
            else store_pair(vo, d * 32 + 8 * q, hh, 2 * a.d, live, x, y);
        }
    }
}

// The key splits' dQ added, four columns of a row to a lane.
template <class T>
__global__ __launch_bounds__(256) void diff_bwd_q_join(DiffArgs a, DiffGrads g, const float* __restrict__ parts, int splits) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, rows = (int64_t)a.batch * a.heads * a.nq;
    const int per = a.d / 2;                                          // lanes of a row
    const int64_t row = i / per;
    if (row >= rows) return;
    const int col = (int)(i - row * per) * 4;
    const float* p = parts + row * 2 * a.d + col;
    f32x4 x = *reinterpret_cast<const f32x4*>(p);
    for (int s = 1; s < splits; ++s) x = x + *reinterpret_cast<const f32x4*>(p + s * rows * 2 * a.d);
    const int64_t bh = row / a.nq, tok = row - bh * a.nq, b = bh / a.heads, head = bh - b * a.heads;
    const int map = col >= a.d;
    store4(reinterpret_cast<T*>(g.dq) + b * g.dqs[0] + tok * g.dqs[1] + head * g.dqs[2] + map * g.dqs[3] + col - map * a.d, x);
}

// The row splits' dK and dV added, four columns of a key to a lane.
template <class T>
__global__ __launch_bounds__(256) void diff_bwd_join(DiffArgs a, DiffGrads g, const float* __restrict__ parts, int splits) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, keys = (int64_t)a.batch * a.kv_heads * a.nk;
    const int64_t row = i / a.d;
    if (row >= keys) return;
    const int col = (int)(i - row * a.d) * 4;
    const float* p = parts + row * 4 * a.d + col;
    f32x4 x = *reinterpret_cast<const f32x4*>(p);
    for (int s = 1; s < splits; ++s) x = x + *reinterpret_cast<const f32x4*>(p + s * keys * 4 * a.d);
    const int64_t bk = row / a.nk, key = row - bk * a.nk, b = bk / a.kv_heads, kh = bk - b * a.kv_heads;
    const int map = col >= a.d;
    T* to = col < 2 * a.d ? reinterpret_cast<T*>(g.dk) + b * g.dks[0] + key * g.dks[1] + kh * g.dks[2] + map * g.dks[3] + col - map * a.d
                          : reinterpret_cast<T*>(g.dv) + b * g.dvs[0] + key * g.dvs[1] + kh * g.dvs[2] + col - 2 * a.d;
    store4(to, x);
}

// Pairs of a workgroup.  dK and dV: four share the staged tiles in bf16 (with two 577 tokens of size 48 take 95 instead of 100
// us, 1500 of 64 189 instead of 172); in f32 a lane holds twice the bytes, and two pairs leave it all 512 registers.  dQ: two,
// so that a CU holds several workgroups, whose prologues (Q, dO, O) and loops overlap (85 against 101 us, 117 against 131).
template <class T>
constexpr int pairs() { return sizeof(T) == 4 ? 2 : 4; }
constexpr int kRowPairs = 2;

int64_t row_tiles(const DiffArgs& a, int np) { return ((int64_t)a.nq * a.group + 32 * np - 1) / (32 * np); }
int64_t key_tiles(const DiffArgs& a, int np) { return ((int64_t)a.nk + 32 * np - 1) / (32 * np); }

// Into how many parts the rows of a key tile (or the keys of a row tile) are split: so many that there are two workgroups to
// a CU, where most CUs would have none, or where they are long enough to pay for adding the parts (under a causal mask the
// first keys' workgroups have twice the average work).  Measured with / without, the addition included, dK and dV: 10000
// causal rows, 20 workgroups 66 / 621 us; 1800, 45: 31 / 95; 600, 80: 27 / 30; 8192, 256: 305 / 452;  1500 unmasked rows, 384
// workgroups 183 / 183, 1200 causal ones, 240: 64 / 55.  dQ: 10000 causal rows on 2500 keys, 157 workgroups 40 / 67; one f32
// token on 6614 keys, 6 workgroups: the whole step 141 / 993.  f32 takes eight times as long for the same rows and splits earlier (1200 causal rows and
// keys, 152 workgroups: the whole step 302 / 578).
int splits_of(int64_t blocks, int64_t length, bool bf16) {
    if (blocks >= 128 && length < (bf16 ? 2048 : 1024)) return 1;
    int64_t s = 511 / blocks + 1, most = length / 256;
    s = s < most ? s : most;
    return (int)(s < 1 ? 1 : s > 32 ? 32 : s);
}
int row_splits(const DiffArgs& a, int np, bool bf16) {
    return splits_of((int64_t)a.batch * a.kv_heads * key_tiles(a, np), (int64_t)a.nq * a.group, bf16);
}
int key_splits(const DiffArgs& a, bool bf16) { return splits_of((int64_t)a.batch * a.kv_heads * row_tiles(a, kRowPairs), a.nk, bf16); }

// f32 values of the parts, of one kernel after the other
int64_t parts_floats(const DiffArgs& a, int np, bool bf16) {
    const int64_t r = row_splits(a, np, bf16), k = key_splits(a, bf16);
    const int64_t kv = r > 1 ? r * a.batch * a.kv_heads * a.nk * 4 * a.d : 0, q = k > 1 ? k * a.batch * a.heads * a.nq * 2 * a.d : 0;
    return kv > q ? kv : q;
}

template <class T, int DP>
hipError_t launch(const DiffArgs& a, const DiffGrads& g, float* ws, hipStream_t s) {
    constexpr int NP = pairs<T>(), OCC = sizeof(T) == 4 && DP > 32 ? 1 : 2;
    // blocks of 32 that are staged between two barriers, measured with one / two.  dQ at 577 tokens (batch 16, 8 heads of 48)
    // 70 / 81 us, at 197 (64, 12 of 32) 55 / 59: the smaller buffers leave room for a third workgroup on a CU;  at 4096
    // causal ones (2, 8 heads of 64, 4 key heads) 195 / 192, at 1500 (2, 16 of 64) 119 / 115: there the registers do not.
    // dK and dV 100 / 102, 75 / -, 280 / 319;  in f32 at 257 tokens (4, 16 heads of 40) 140 / 134, at 577 (2, 12 of 64) 175 / 159.
    constexpr int NBQ = sizeof(T) == 2 && DP == 64 ? 2 : 1, NBK = sizeof(T) == 4 ? 2 : 1;
    const int64_t bks = (int64_t)a.batch * a.kv_heads;
    const int64_t qt = row_tiles(a, kRowPairs), kt = key_tiles(a, NP), keys = (int64_t)a.batch * a.kv_heads * a.nk;
    const int splits = row_splits(a, NP, sizeof(T) == 2), ksplits = key_splits(a, sizeof(T) == 2);
    const int64_t rows = (int64_t)a.batch * a.heads * a.nq;
    if (bks * qt * ksplits > 0x7FFFFFFF || rows * a.d / 512 > 0x7FFFFFF0 || bks * kt * splits + a.lam_heads > 0x7FFFFFFF || keys * a.d / 256 > 0x7FFFFFF0) return hipErrorInvalidValue;
    float* parts = ws;
    float* ws_d = ws + parts_floats(a, NP, sizeof(T) == 2);
    float* ws_w = ws_d + 2 * (int64_t)a.batch * a.heads * a.nq;
    hipLaunchKernelGGL((diff_bwd_q<T, DP, kRowPairs, NBQ, OCC>), dim3((int)(bks * qt * ksplits)), dim3(kRowPairs * 128), 0, s, a, g, ws_d, ws_w,
                       parts, (int)qt, ksplits);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (ksplits > 1) {
        hipLaunchKernelGGL((diff_bwd_q_join<T>), dim3((int)((rows * (a.d / 2) + 255) / 256)), dim3(256), 0, s, a, g, parts, ksplits);
        e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    const int blocks = (int)(bks * kt * splits);
    const dim3 grid(blocks + (g.dlam ? a.lam_heads : 0)), block(NP * 128);
    if (a.group == 1) hipLaunchKernelGGL((diff_bwd_kv<T, DP, true, NP, NBK, OCC>), grid, block, 0, s, a, g, ws_d, parts, splits, ws_w, (int)qt * ksplits, blocks);
    else hipLaunchKernelGGL((diff_bwd_kv<T, DP, false, NP, NBK, OCC>), grid, block, 0, s, a, g, ws_d, parts, splits, ws_w, (int)qt * ksplits, blocks);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (splits > 1) {
        hipLaunchKernelGGL((diff_bwd_join<T>), dim3((int)((keys * a.d + 255) / 256)), dim3(256), 0, s, a, g, parts, splits);
        e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace

// f32 values of scratch of the backward
int64_t diff_attention_bwd_workspace(const DiffArgs& a, bool bf16) {
    const int np = bf16 ? pairs<bf16_t>() : pairs<float>();
    return parts_floats(a, np, bf16) + 2 * (int64_t)a.batch * a.heads * a.nq + (int64_t)a.batch * a.heads * row_tiles(a, kRowPairs) * key_splits(a, bf16);
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
