// Differential attention, forward (gfx950 / CDNA4): per query row of a head
//     P_m = softmax over the visible keys of scale q_m . k_m,  m = 1, 2
//     out = (P_1 - w P_2) V,    w = exp(lam0 . lam1) - exp(lam2 . lam3) + lambda_init
//
// One pass over the keys with a running maximum and sum per map.  The two maps of a head share V and little else, and
// their products with V stay apart until the end, because their denominators are known only then; so a pair of waves takes
// 32 query rows, one map each, which halves what a wave holds (its accumulators above all) and doubles the waves that hide
// each other's waiting.  They meet once, for P_1 V - w P_2 V.
//
//     S_m^T[key][row]  = K_m Q_m^T       keys on the matrix row, query rows on the lane
//     O_m^T[col][row] += V^T P_m^T       the exponentiated accumulators are the B operand as they lie
//
// Rows of a (sample, key head) are the tokens of all its query heads (diff_attention.h).  Two forms:
//   many rows:  the pairs of a workgroup take 32 rows each and walk all their keys in chunks of 32 through two LDS buffers,
//               the next chunk on its way to registers while the waves work on the one before;
//   few rows:   the pairs (four, in f32 from size 33 on two) take the same 32 rows and a block of 32 keys in turn, and the keys
//               are split over so many workgroups that the chip is full; the pairs' results are joined in LDS, the workgroups'
//               by a second kernel.
#include <type_traits>

#include "diff_attention.h"

namespace vitk {

using namespace diff;

namespace {

// Pairs of waves in a workgroup.  Few rows: as many as LDS has room for with two buffers of 32 keys each.  Many rows: four in f32
// and at size 32, two else, measured with two / four: 197 tokens of 32 (64 x 12 heads) 37.4 / 37.2 us, 197 of 64 (64 x 6)
// 40.6 / 43.5, 4096 causal ones of 64 151 / 161, f32 55 / 55.
template <class T, int DP>
constexpr int keys_pairs() { return row_bytes<T, 2 * DP>() == 512 ? 2 : 4; }

template <class T, int DP>
constexpr int rows_pairs() { return sizeof(T) == 4 || DP == 32 ? 4 : 2; }

// index of a 4-column piece of a joined row in LDS: [row][2 maps x DV columns] f32, pieces swizzled by the row
template <int DV>
__device__ __forceinline__ int joined(int row, int map, int col) {
    const int c = (map * DV + col) >> 2;
    return row * (2 * DV) + ((c ^ (row & 15)) << 2);
}

// OCC: waves to a SIMD that the registers have to allow (at size 64 the form for many rows without TRAIN spills 5).  TRAIN: the sums for the backward are written too, and the
// denominators are added from the probabilities before their rounding to bf16 (16 additions a block and lane); without it
// the matrix pipe adds the rounded ones, which are what the product with V uses, beside that product.
template <class T, int DP, int NG, bool KEYS, bool TRAIN, int OCC>
__global__ __launch_bounds__(NG * 128, OCC) void diff_fwd(DiffArgs a, DiffOut o, float* __restrict__ ws, int tiles, int splits) {
    constexpr int DV = 2 * DP;
    constexpr int NT = NG * 128;
    constexpr int RB = row_bytes<T, DV>();         // of an LDS row: both maps of a key, or one of V
    constexpr int PER = Op<T>::kPer;
    constexpr int DPC = DP / PER;                  // chunks of one map's key
    constexpr int KT = DPC / 2;                    // products of 2 chunks (one per half-wave) of a score
    constexpr int DB = DV / 32;
    constexpr int KC = 32 * (KEYS ? NG : 1);       // keys of a chunk; 64 for many rows: 3 to 9 % slower
    constexpr int TILE = KC * RB;
    typedef typename Op<T>::Chunk Chunk;
    constexpr int BUF = KEYS || 2 * TILE > NG * DB * 2048 ? 2 * TILE : NG * DB * 2048;      // many rows: DB sums of a pair fit
    __shared__ __align__(16) char bufs[2][BUF];
    __shared__ float s_ml[KEYS ? NG : 1][4][32];
    __shared__ float s_w[KEYS ? 32 : 1];

    arguments(a);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), map = wave & 1, grp = wave >> 1;
    const int r = lane & 31, hh = lane >> 5;
    const int bks = a.batch * a.kv_heads;
    const int rest = quotient(blockIdx.x, a.by_bks);
    const int bk = blockIdx.x - rest * bks;        // workgroups of one head lie bks apart: one XCD where 8 divides bks
    const int split = KEYS ? rest / tiles : 0;
    const int tile = KEYS ? rest - split * tiles : (a.causal ? tiles - 1 - rest : rest);     // causal: the longest rows first
    const int b = quotient(bk, a.by_kv_heads), kh = bk - b * a.kv_heads;
    const int nrows = a.nq * a.group;
    const int row0 = KEYS ? tile * 32 : (tile * NG + grp) * 32;
    const int end = KEYS ? tile * 32 + 32 : (tile + 1) * NG * 32;
    int len = a.nk;
    if (a.key_lens) {
        len = a.key_lens[b];
        len = len < 0 ? 0 : (len < a.nk ? len : a.nk);
    }
    const int kmax = key_limit(a, len, row_place(a, kh, (end < nrows ? end : nrows) - 1).tok);

    const int dc = a.d / PER;
    Stage<T, DP, NT, KC> stage;
    stage.init(tid, dc, bufs[0], BUF);
    const int64_t s_step = stage.second ? a.vs[1] : a.ks[1];
    const T* s_src = stage.row * s_step + (stage.second ? reinterpret_cast<const T*>(a.v) + b * a.vs[0] + kh * a.vs[2] + stage.col * PER
                                                        : reinterpret_cast<const T*>(a.k) + b * a.ks[0] + kh * a.ks[2] + stage.map * a.ks[3] + stage.e * PER);
    auto fetch = [&](int key0) { stage.fetch(key0, kmax, s_src, s_step, 0, [&](int key) { return s_src + (key - stage.row) * s_step; }); };

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

    Chunk qf[KT];
    {
        const T* qg = reinterpret_cast<const T*>(a.q) + b * a.qs[0] + place.tok * a.qs[1] + place.head * a.qs[2] + map * a.qs[3];
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            const int c = 2 * t + hh;
            qf[t] = chunk_or_zero<T>(qg, c, c < dc);
        }
    }
    // few rows: the first wave's, and none where the second kernel joins the splits
    const float weight = KEYS && (wave != 0 || splits > 1) ? 0.f : map_weight<DP>(a, place.head, lane, false);

    constexpr bool MSUM = !TRAIN && sizeof(T) == 2;
    f32x16 acc[DB], l_acc = zero16();
    float m_run = kNoScore, l_run = 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[d] = zero16();
    const float sc = a.scale * kLog2e;
    constexpr float kLazy = 8.0f;     // the accumulators are rescaled only when a maximum grows by more than 2^8

    auto step = [&](const char* kt, const char* vt, int kb, int key0, bool fresh) __attribute__((always_inline)) {
        // A wave at its products goes first, so that the others of its SIMD fall behind it and compute while it multiplies:
        // 7 % at head size 64 (1500 tokens 84.4 -> 78.1 us), nothing at 32
        f32x16 s = zero16();
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int t = 0; t < KT; ++t) s = Op<T>::mma(chunk_at<T, RB>(kt, kb * 32 + r, map * DPC + 2 * t + hh), qf[t], s);
        __builtin_amdgcn_s_setprio(0);
        if (key0 + 32 > wave_min) hide(s, lim - key0 - 4 * hh);
        float mx = fmaxf(s[0], s[1]);
#pragma unroll
        for (int i = 2; i < 16; i += 2) mx = fmaxf(fmaxf(mx, s[i]), s[i + 1]);
        mx = both_max(mx) * sc;                                      // scale > 0: the maximum commutes with it
        if (__any(mx > m_run + kLazy)) {
            const float m_new = fmaxf(m_run, mx);
            const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
            m_run = m_new;
            if (!fresh) {                                            // nothing to rescale before the first block
                if constexpr (MSUM) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) l_acc[i] *= alpha;
                } else {
                    l_run *= alpha;
                }
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[d][i] *= alpha;
            }
        }
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], sc, -m_run));
            if constexpr (!MSUM) sum += s[i];
        }
        l_run += sum;
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int st = 0; st < 2; ++st) {
            Slice<T> p;
            p.take(s, st);
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                Trans<T, RB> v;
                v.load(vt, kb * 32 + 16 * st, d * 32, lane);
                acc[d] = mma_t(v, p, acc[d]);
            }
            if constexpr (MSUM) l_acc = ones_t(p, l_acc);
        }
        __builtin_amdgcn_s_setprio(0);
    };
    if (c0 < c1) stage.put(bufs[0]);
    loads_done();
    __syncthreads();
    auto chunk = [&](int c, auto which) __attribute__((always_inline)) {                            // the buffer is known when compiled: no address arithmetic
        const char* buf = bufs[decltype(which)::value];
        const bool more = c + 1 < c1;
        if (more) fetch((c + 1) * KC);
        const int key0 = c * KC + (KEYS ? grp * 32 : 0);             // few rows: the pair's block of the chunk
        if (active && key0 < wave_max) step(buf, buf + TILE, KEYS ? grp : 0, key0, c == c0);
        if (more) stage.put(bufs[decltype(which)::value ^ 1]);
        __syncthreads();
    };
    for (int c = c0; c < c1; c += 2) {
        chunk(c, std::integral_constant<int, 0>{});
        if (c + 1 < c1) chunk(c + 1, std::integral_constant<int, 1>{});
    }

    const float l_tot = MSUM ? l_acc[0] : both_sum(l_run);           // each element of l_acc holds the lane's whole sum
    const float inv = l_tot > 0.f || l_tot != l_tot ? 1.0f / l_tot : 0.f;
    const int64_t orow = (((int64_t)b * a.nq + place.tok) * a.heads + place.head) * 2 * a.d;
    const int64_t lrow = ((int64_t)b * a.heads + place.head) * a.nq + place.tok;
    const int64_t lmap = (int64_t)a.batch * a.heads * a.nq;
    T* out = reinterpret_cast<T*>(o.out);
    T* out2 = reinterpret_cast<T*>(o.out2);

    if constexpr (!KEYS) {
        const bool live = row < nrows;
        if (TRAIN && live && hh == 0) {
            o.stats[map * lmap + lrow] = l_tot == 0.f ? 0.f : m_run;
            o.stats[(2 + map) * lmap + lrow] = inv;
            if (map == 0 && b == 0 && place.tok == 0) o.weight[place.head] = weight;
        }
        // the pair's waves exchange sums: the first finishes the first D0 blocks of 32 columns, the second the others
        constexpr int D0 = (DB + 1) / 2;
        f32x4* box = reinterpret_cast<f32x4*>(bufs[0]) + grp * DB * 256 + lane;
#pragma unroll
        for (int d = 0; d < DB; ++d) {
            if ((d < D0) == (map == 0)) continue;
#pragma unroll
            for (int g = 0; g < 4; ++g) box[d * 256 + g * 64] = four(acc[d], g, inv);
        }
        __syncthreads();
#pragma unroll
        for (int d = 0; d < DB; ++d) {
            if ((d < D0) != (map == 0)) continue;
#pragma unroll
            for (int g = 0; g < 4; g += 2) {
                f32x4 x[2], y[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const f32x4 mine = four(acc[d], g + i, inv), other = box[d * 256 + (g + i) * 64];
                    y[i] = map ? mine : other;
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[i][j] = fmaf(-weight, y[i][j], map ? other[j] : mine[j]);
                }
                store_pair(out + orow, d * 32 + 8 * g, hh, 2 * a.d, live, x[0], x[1]);
                if (TRAIN) store_pair(out2 + orow, d * 32 + 8 * g, hh, 2 * a.d, live, y[0], y[1]);
            }
        }
    } else {
        // join the pairs' keys
        if (hh == 0) {
            s_ml[grp][2 * map][r] = m_run;
            s_ml[grp][2 * map + 1][r] = l_tot;
            if (wave == 0) s_w[r] = weight;
        }
        __syncthreads();
        float top = s_ml[0][2 * map][r], sum = 0.f;
#pragma unroll
        for (int w = 1; w < NG; ++w) top = fmaxf(top, s_ml[w][2 * map][r]);
#pragma unroll
        for (int w = 0; w < NG; ++w) sum += s_ml[w][2 * map + 1][r] * __builtin_amdgcn_exp2f(s_ml[w][2 * map][r] - top);
        constexpr int HALF = NG / 2;
        static_assert(HALF * 32 * 2 * DV * 4 <= 2 * TILE, "the pairs' rows fit the buffers");
        float* mine = reinterpret_cast<float*>(bufs[grp < HALF ? 0 : 1]) + (grp % HALF) * 32 * 2 * DV;
        if (row < nrows) {
            const float f = __builtin_amdgcn_exp2f(m_run - top);
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x4 x = {acc[d][4 * g] * f, acc[d][4 * g + 1] * f, acc[d][4 * g + 2] * f, acc[d][4 * g + 3] * f};
                    *reinterpret_cast<f32x4*>(mine + joined<DV>(r, map, d * 32 + 8 * g + 4 * hh)) = x;
                }
        }
        __syncthreads();
        if (grp == 0 && hh == 0) {                                   // the joined maximum and sum take the first pair's place
            s_ml[0][2 * map][r] = top;
            s_ml[0][2 * map + 1][r] = sum;
        }
        __syncthreads();
        const int live = nrows - row0 < 32 ? nrows - row0 : 32;
        const int64_t part = ((int64_t)bk * tiles + tile) * splits + split;
        float* wo = ws + part * 32 * (2 * DV + 4);
        for (int i = tid; i < live * (DV / 4); i += NT) {
            const int rr = i / (DV / 4), col = (i - rr * (DV / 4)) * 4;
            f32x4 x[2];
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                x[m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < NG; ++w)
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
            if (TRAIN) store4(out2 + at, y);
        }
        if (grp == 0 && row < nrows && hh == 0) {
            if (splits > 1) {
                float* ml = wo + 32 * 2 * DV + r * 4;
                ml[2 * map] = top;
                ml[2 * map + 1] = sum;
            } else if (TRAIN) {
                o.stats[map * lmap + lrow] = sum == 0.f ? 0.f : top;
                o.stats[(2 + map) * lmap + lrow] = sum == 0.f ? 0.f : 1.0f / sum;
                if (map == 0 && b == 0 && place.tok == 0) o.weight[place.head] = weight;
            }
        }
    }
}

// The splits of the keys joined: a workgroup per row, 4 columns to a lane, the splits shared among as many lanes as are
// left, two maps side by side.
template <class T, int DV>
__global__ __launch_bounds__(256) void diff_fwd_join(DiffArgs a, DiffOut o, const float* __restrict__ ws, int tiles,
                                                     int splits) {
    constexpr int CH = DV / 4, NP = 256 / (2 * CH);                  // pieces of a row, lanes that share a piece's splits
    constexpr int STRIDE = 32 * (2 * DV + 4);
    __shared__ f32x4 s_part[NP][2][CH];
    __shared__ float s_f[2][128];                                    // what a split's sums are scaled by
    __shared__ float s_inv[2], s_w;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int nrows = a.nq * a.group;
    const int bk = blockIdx.x / nrows, row = blockIdx.x - bk * nrows, tile = row >> 5, rr = row & 31;
    const int b = quotient(bk, a.by_kv_heads), kh = bk - b * a.kv_heads;
    const RowPlace pl = row_place(a, kh, row);
    const float* base = ws + ((int64_t)bk * tiles + tile) * splits * STRIDE;
    // the splits' values are on their way while the factors are computed
    const int m = tid / (CH * NP), c = tid % CH, part = tid / CH % NP;
    const float* p = base + (int64_t)part * STRIDE + rr * 2 * DV + m * DV + c * 4;
    constexpr int U = 4;                                             // loads on their way at once
    auto batch = [&](int s0, f32x4 (&v)[U]) {                         // splits past the last one: the last one again
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u && u * NP >= splits) break;                        // the same for all
            const int s = s0 + u * NP < splits ? s0 + u * NP : splits - 1;
            v[u] = *reinterpret_cast<const f32x4*>(p + (int64_t)(s - part) * STRIDE);
        }
    };
    f32x4 v[U];
    if (tid < 2 * CH * NP) batch(part, v);
    if (wave < 2) {                                                  // wave m joins map m's maxima and sums
        float mx[2], l[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int s = lane + 64 * j;
            const float* ml = base + (int64_t)s * STRIDE + 32 * 2 * DV + rr * 4 + 2 * wave;
            mx[j] = s < splits ? ml[0] : kNoScore;
            l[j] = s < splits ? ml[1] : 0.f;
        }
        float top = fmaxf(mx[0], mx[1]);
#pragma unroll
        for (int sh = 32; sh > 0; sh >>= 1) top = fmaxf(top, __shfl_xor(top, sh, 64));
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float f = __builtin_amdgcn_exp2f(mx[j] - top);
            s_f[wave][lane + 64 * j] = f;
            sum = fmaf(l[j], f, sum);
        }
        sum = wave_sum(sum);
        const float inv = sum > 0.f || sum != sum ? 1.0f / sum : 0.f;
        if (lane == 0) {
            s_inv[wave] = inv;
            if (o.out2) {
                const int64_t lmap = (int64_t)a.batch * a.heads * a.nq, at = ((int64_t)b * a.heads + pl.head) * a.nq + pl.tok;
                o.stats[wave * lmap + at] = sum == 0.f ? 0.f : top;
                o.stats[(2 + wave) * lmap + at] = inv;
            }
        }
    } else if (wave == 2) {
        const float w = map_weight<DV / 2>(a, pl.head, lane, true);
        if (lane == 0) {
            s_w = w;
            if (o.out2 && b == 0 && pl.tok == 0) o.weight[pl.head] = w;
        }
    }
    __syncthreads();
    if (tid < 2 * CH * NP) {
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
        for (int s0 = part; s0 < splits; s0 += U * NP) {
            if (s0 != part) batch(s0, v);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (u && u * NP >= splits) break;
                const float f = s0 + u * NP < splits ? s_f[m][s0 + u * NP] : 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = s0 + u * NP < splits ? fmaf(v[u][j], f, x[j]) : x[j];
            }
        }
        s_part[part][m][c] = x;
    }
    __syncthreads();
    if (tid >= CH || 4 * tid >= 2 * a.d) return;
    f32x4 x1 = s_part[0][0][tid], x2 = s_part[0][1][tid];
#pragma unroll
    for (int j = 1; j < NP; ++j) {
        x1 = x1 + s_part[j][0][tid];
        x2 = x2 + s_part[j][1][tid];
    }
    const f32x4 y = x2 * s_inv[1];
    f32x4 z;
#pragma unroll
    for (int j = 0; j < 4; ++j) z[j] = fmaf(-s_w, y[j], x1[j] * s_inv[0]);
    const int64_t at = (((int64_t)b * a.nq + pl.tok) * a.heads + pl.head) * 2 * a.d + 4 * tid;
    store4(reinterpret_cast<T*>(o.out) + at, z);
    if (o.out2) store4(reinterpret_cast<T*>(o.out2) + at, y);
}

struct Plan {
    bool keys;
    int tiles, splits;
};

// Which form, and into how many workgroups.  At most 32 rows to a key head, or at most one block of 32 rows to each of the
// 256 CUs (two in f32, whose products take eight times as long): the pairs share the rows and split the keys.  Measured, keys split / not: 64 rows, 2048 keys, 128 key heads of
// size 64 (256 blocks) 50 / 105 us, 256 heads (512 blocks) 105 / 108; 577 rows and keys, 16 heads of 64 (304) 29.2 / 27.4;  in f32
// 577 tokens, 24 heads of 64 (456) 101 / 133, 257, 64 of 64 (576) 84 / 72.
template <class T, int DP>
Plan plan(const DiffArgs& a) {
    const int64_t nrows = (int64_t)a.nq * a.group, bks = (int64_t)a.batch * a.kv_heads;
    Plan p;
    p.keys = nrows <= 32 || bks * ((nrows + 31) / 32) <= (sizeof(T) == 4 ? 512 : 256);
    constexpr int R = 32 * rows_pairs<T, DP>();
    p.tiles = (int)(p.keys ? (nrows + 31) / 32 : (nrows + R - 1) / R);
    p.splits = 1;
    if (p.keys) {
        const int kc = 32 * keys_pairs<T, DP>();
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
    constexpr int NK = keys_pairs<T, DP>(), OCCK = NK == 4 ? 2 : 1;
    constexpr int NG = rows_pairs<T, DP>(), OCC = sizeof(T) == 4 ? 2 : DP == 32 ? 4 : 3;
    const dim3 grid((int)blocks), kb(NK * 128), rb(NG * 128);
    if (p.keys && o.out2) hipLaunchKernelGGL((diff_fwd<T, DP, NK, true, true, OCCK>), grid, kb, 0, s, a, o, ws, p.tiles, p.splits);
    else if (p.keys) hipLaunchKernelGGL((diff_fwd<T, DP, NK, true, false, OCCK>), grid, kb, 0, s, a, o, ws, p.tiles, p.splits);
    else if (o.out2) hipLaunchKernelGGL((diff_fwd<T, DP, NG, false, true, OCC>), grid, rb, 0, s, a, o, ws, p.tiles, 1);
    else hipLaunchKernelGGL((diff_fwd<T, DP, NG, false, false, OCC>), grid, rb, 0, s, a, o, ws, p.tiles, 1);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits == 1) return e;
    const int64_t rows = (int64_t)a.batch * a.heads * a.nq;
    if (rows > 0x7FFFFFFF) return hipErrorInvalidValue;
    hipLaunchKernelGGL((diff_fwd_join<T, 2 * DP>), dim3((int)rows), dim3(256), 0, s, a, o, ws, p.tiles, p.splits);
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
