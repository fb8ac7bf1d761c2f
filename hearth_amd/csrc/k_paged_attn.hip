/*
 * k_paged_attn.hip — attention over a paged cache: few query rows a kv head (single tokens,
 * chains), split over the cache's length and joined.
 *
 * The products run transposed: S^T = K Q^T (rows: cache rows, columns: query rows, one column
 * a (token, head) pair of the kv head's group) and O^T = V^T P^T. In the 16 x 16 result of the
 * first a lane holds four cache rows of one column, which is, two tiles together, the operand
 * that the second product takes for the same column: the probabilities never leave the
 * registers. V comes in by rows (8 elements of 8 cache rows a lane) and is transposed there,
 * a byte permutation a pair of elements.
 * It is bound by the cache's bytes: 268 MB of one token over 131071 rows in 49.7 us (5.4 TB/s), 178
 * MB of 32 tokens over 8-bit rows in 44 us (4.1 TB/s), the joins 5 us each. Nothing of the cache
 * goes through LDS (no row is read by two waves), V is under way before the scores and the next K
 * before the sums (32 tokens over 8-bit rows with each load where it is used: 114 us, not 48).
 *
 * Scores, maxima, sums of probabilities and of rows are float32. The probabilities alone are rounded
 * to the 16-bit type, in this kernel and the two for many rows: the matrix units take both factors in
 * 16 bits, and split into two 16-bit parts they would double the second product. Each rounding is
 * off by half a step at most, which is as much as the result's own (relative error of 2000 tokens
 * over 4048 rows against 64 bits: 0.0022 where the result's rounding alone gives 0.0017); float16
 * takes those below 2^-25 of the maximum they are taken against as 0. Their sum is taken before.
 */
#include "hx_paged.h"

#include <algorithm>

namespace hxp {

namespace {

constexpr int FEW_WAVES = 4, FEW_STEP = 32;   /* a wave takes 32 cache rows at a time, the workgroup 128 */

__device__ __forceinline__ unsigned lo16(unsigned a, unsigned b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ unsigned hi16(unsigned a, unsigned b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

template <class T, bool MX, int D>
struct Few {
    using v8 = typename T::v8;
    static constexpr int KS = D / 32;                    /* matrix steps of the score */
    static constexpr int BD = D < 128 ? D : 128;        /* elements of a V block: 16 lanes x PL */
    static constexpr int NB = D / BD, PL = BD / 16;      /* blocks; elements of a row a lane takes */
    static constexpr int ES = MX ? 1 : 2;                 /* bytes of a stored element */

    static constexpr int KL = MX ? D / 64 : KS;           /* 16-byte loads of a row for the score */
    static constexpr int VW = MX ? PL / 4 : PL / 2;       /* words of a row and block for the sum */
    static constexpr int SW = D / 32 < 4 ? 1 : D / 128;   /* words that hold a row's scales */

    struct K { u4 w[2][KL]; unsigned s[2][SW]; };         /* a lane's row of either tile of 16 */
    struct V { unsigned w[NB][8][VW]; unsigned s[2][D / 32]; };   /* eight rows; scales of the four rows of either tile */

    /* row: first of the tile in its page (a multiple of 16) */
    static __device__ __forceinline__ void load_k(K &k, int u, const uint8_t *page, const uint8_t *sc, int row, int g, int lc) {
        const uint8_t *p = page + (row + lc) * (D * ES) + 16 * g;
#pragma unroll
        for (int i = 0; i < KL; i++) k.w[u][i] = *(const u4 *)(p + 64 * i);
        if constexpr (MX) {
            const uint8_t *q = sc + (row + lc) * (D / MX_BLOCK);
            if constexpr (D == 64) k.s[u][0] = *(const ushort_any *)q;
            else
#pragma unroll
                for (int i = 0; i < SW; i++) k.s[u][i] = ((const unsigned_any *)q)[i];
        }
    }
    static __device__ __forceinline__ void load_v(V &v, int u, const uint8_t *page, const uint8_t *sc, int row, int g, int lc) {
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint8_t *p = page + (row + 4 * g + j) * (D * ES) + (b * BD + lc * PL) * ES;
                if constexpr (VW == 4) {
                    const u4 x = *(const u4 *)p;
#pragma unroll
                    for (int i = 0; i < 4; i++) v.w[b][4 * u + j][i] = x[i];
                } else if constexpr (VW == 2) {
                    const u2 x = *(const u2 *)p;
                    v.w[b][4 * u + j][0] = x[0]; v.w[b][4 * u + j][1] = x[1];
                } else {
                    v.w[b][4 * u + j][0] = *(const unsigned *)p;
                }
            }
        if constexpr (MX) {   /* four rows' scales lie side by side */
            const uint8_t *q = sc + (row + 4 * g) * (D / MX_BLOCK);
#pragma unroll
            for (int i = 0; i < D / 32; i += D / 32 >= 4 ? 4 : 2)
                if constexpr (D / 32 >= 4) {
                    const u4 x = *(const u4_any *)(q + 4 * i);
#pragma unroll
                    for (int j = 0; j < 4; j++) v.s[u][i + j] = x[j];
                } else {
                    const u2 x = *(const u2_any *)(q + 4 * i);
                    v.s[u][i] = x[0]; v.s[u][i + 1] = x[1];
                }
        }
    }
    /* scores of the 16 rows of tile u */
    static __device__ __forceinline__ void scores(const K &k, int u, int g, const v8 (&q)[KS], f4 &s) {
#pragma unroll
        for (int i = 0; i < KL; i++) {
            if constexpr (MX) {
                /* block 2 i + g / 2 */
                const float f = mx_scale(k.s[u][i >> 1] >> (16 * (i & 1) + 8 * (g >> 1)));
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const unsigned a = k.w[u][i][2 * h], b = k.w[u][i][2 * h + 1];
                    const u4 w = {T::template from_mx8<false>(a, f), T::template from_mx8<true>(a, f),
                                  T::template from_mx8<false>(b, f), T::template from_mx8<true>(b, f)};
                    s = T::mfma16(__builtin_bit_cast(v8, w), q[2 * i + h], s);
                }
            } else {
                s = T::mfma16(__builtin_bit_cast(v8, k.w[u][i]), q[i], s);
            }
        }
    }
    /* PL elements of row j, block b, as 16-bit pairs */
    static __device__ __forceinline__ void v_row(const V &v, int b, int j, int lc, unsigned (&w)[PL / 2]) {
        if constexpr (MX) {
            const int jj = j & 3;
            unsigned x;
            if constexpr (D == 64) x = v.s[j >> 2][jj >> 1] >> (16 * (jj & 1) + 8 * (lc >> 3));
            else x = v.s[j >> 2][jj * (D / 128) + b] >> (8 * (lc >> 2));
            const float f = mx_scale(x);
#pragma unroll
            for (int i = 0; i < VW; i++) {
                w[2 * i] = T::template from_mx8<false>(v.w[b][j][i], f);
                w[2 * i + 1] = T::template from_mx8<true>(v.w[b][j][i], f);
            }
        } else {
#pragma unroll
            for (int i = 0; i < VW; i++) w[i] = v.w[b][j][i];
        }
    }
};

template <class T, bool MX, int D>
__global__ __launch_bounds__(64 * FEW_WAVES) void k_attend_few(AttendArgs a) {
    using F = Few<T, MX, D>;
    using v8 = typename T::v8;
    constexpr int PL = F::PL, NB = F::NB, BD = F::BD, ES = F::ES, CT = 16;
    __shared__ float lds_o[FEW_WAVES][16][BD + 4];
    __shared__ float lds_m[FEW_WAVES][CT], lds_l[FEW_WAVES][CT];
    __shared__ unsigned lds_some[FEW_WAVES];   /* bit c: column c attends a row of the wave's */

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int g = lane >> 4, lc = lane & 15;
    int bx = blockIdx.x;
    const int sp = bx % a.n_splits;
    bx /= a.n_splits;
    const int kvh = bx % a.kv_heads, tile = bx / a.kv_heads;
    const int seq = blockIdx.z;
    const Seq q = seq_of(a.b, seq);
    const int cols = min(q.n, a.b.max_q) * a.group;
    if (tile * CT >= cols) return;
    const int n_sp = max(1, (q.kv + a.chunk - 1) / a.chunk);
    if (sp >= n_sp) return;

    /* this lane's column */
    v8 qf[F::KS];
    const int c = tile * CT + lc;
    const bool on = c < cols;
    const int tok = on ? c / a.group : 0, head = kvh * a.group + (on ? c % a.group : 0);
    /* rows it attends without a mask (causal), or rows before the call's */
    const int lim = !on ? 0 : a.b.mask ? min(q.base, q.kv) : min(q.base + tok + 1, q.kv);
    const uint8_t *qp = a.q + (int64_t)(q.q0 + tok) * a.qt + (int64_t)head * a.qh;
#pragma unroll
    for (int i = 0; i < F::KS; i++) {
        const int d = MX ? 64 * (i / 2) + 16 * g + 8 * (i % 2) : 32 * i + 8 * g;
        const unsigned short *p = (const unsigned short *)qp + d;
        u4 w = {0, 0, 0, 0};
        if (on) w = *(const u4_any *)p;
        qf[i] = __builtin_bit_cast(v8, w);
    }
    /* rows [lo, hi) of this split that some column of the tile may attend; below `full` every
     * valid column attends every row */
    const int t_first = tile * CT / a.group, t_last = min(cols - 1, tile * CT + CT - 1) / a.group;
    const int hi = min(min(q.kv, a.b.mask ? q.kv : q.base + t_last + 1), (sp + 1) * a.chunk);
    const int full = a.b.mask ? q.base : q.base + t_first + 1;

    /* which of the 64 rows from t0 on this lane's column attends (where their pages exist) */
    auto attended = [&](int t0) {
        return step_mask(t0, lim, hi, q.base,
                         a.b.mask && on ? a.b.mask + (int64_t)(q.q0 + tok) * a.b.mask_words : nullptr,
                         a.b.mask_words);
    };

    f4 acc[NB * PL];
    float m = -__builtin_huge_valf(), l = 0.0f;
    bool some = false;  /* this lane's column attends a row of the wave's */
    bool odd = false;   /* V held an infinity or NaN in a row that some column does not attend */
#pragma unroll
    for (int i = 0; i < NB * PL; i++) acc[i] = (f4){0, 0, 0, 0};
    const int *pages = a.b.pages + (int64_t)seq * a.b.ld_pages;
    const int page_rows = 1 << a.b.page_shift;
    const uint8_t *kbase = a.k.data + (int64_t)kvh * a.k.head_stride, *vbase = a.v.data + (int64_t)kvh * a.v.head_stride;
    const uint8_t *ksb = MX ? a.k.scales + (int64_t)kvh * a.k.scale_head_stride : nullptr;
    const uint8_t *vsb = MX ? a.v.scales + (int64_t)kvh * a.v.scale_head_stride : nullptr;

    /* Pages of the two tiles of 16 rows (-1: none). Every load goes to a row of the cache: rows past hi
     * lie in the same page, those of a page that is not there are taken from page 0; both are
     * masked, and cleared in V. */
    auto page_at = [&](int t) __attribute__((always_inline)) {
        const int id = t < hi ? word_of(pages, t >> a.b.page_shift) : -1;
        return page_ok(a.b, id) ? id : -1;
    };
    typename F::K kr;
    typename F::V vw;
    auto load_k = [&](int t0, const int (&id)[2]) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int64_t i = max(id[u], 0);
            F::load_k(kr, u, kbase + i * a.k.page_stride, MX ? ksb + i * a.k.scale_page_stride : nullptr, (t0 + 16 * u) & (page_rows - 1), g, lc);
        }
    };
    auto load_v = [&](int t0, const int (&id)[2]) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int64_t i = max(id[u], 0);
            F::load_v(vw, u, vbase + i * a.v.page_stride, MX ? vsb + i * a.v.scale_page_stride : nullptr, (t0 + 16 * u) & (page_rows - 1), g, lc);
        }
    };
    const int first = sp * a.chunk + FEW_STEP * wave;
    int pid[2] = {-1, -1}, next[2] = {page_at(first), page_at(first + 16)};
    arrived();
    if (first < hi) load_k(first, next);
    /* a step: V on its way before the scores, the next step's K as soon as these have taken K */
    for (int t0 = first; t0 < hi; t0 += FEW_STEP * FEW_WAVES) {
        bool ok[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            pid[u] = next[u];
            ok[u] = pid[u] >= 0;
            next[u] = page_at(t0 + FEW_STEP * FEW_WAVES + 16 * u);
        }
        load_v(t0, pid);
        in_order();
        f4 s[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            s[u] = (f4){0, 0, 0, 0};
            F::scores(kr, u, g, qf, s[u]);
        }
        in_order();
        if (t0 + FEW_STEP * FEW_WAVES < hi) load_k(t0 + FEW_STEP * FEW_WAVES, next);
        in_order();
        const bool whole = t0 + FEW_STEP <= full && t0 + FEW_STEP <= hi && ok[0] && ok[1];
        v8 pf;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = s[j >> 2][j & 3] * a.scale2;
        if (whole) {
            some = true;
        } else {
            const unsigned long long at = attended(t0) & group_rows((ok[0] ? 1u : 0u) | (ok[1] ? 2u : 0u)), vis = at >> (4 * g);
            some = some || at;
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = vis >> (16 * (j >> 2) + (j & 3)) & 1 ? x[j] : -__builtin_huge_valf();
        }
        float mx = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
        mx = fmaxf(m, max16(max32(mx)));
        const float ms = mx == -__builtin_huge_valf() ? 0.0f : mx;
        if (__any(mx > m)) {
            const float al = exp2_hw(m - ms);
            l *= al;
#pragma unroll
            for (int i = 0; i < NB * PL; i++) acc[i] *= al;
            m = mx;
        }
        float p[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            p[j] = exp2_hw(x[j] - ms);
            l += p[j];
        }
        const u4 w = {T::pack(p[0], p[1]), T::pack(p[2], p[3]), T::pack(p[4], p[5]), T::pack(p[6], p[7])};
        pf = __builtin_bit_cast(v8, w);
#pragma unroll
        for (int b = 0; b < NB; b++) {
            unsigned w[8][PL / 2];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int u = j >> 2, t = t0 + 16 * u + 4 * g + (j & 3);
                F::v_row(vw, b, j, lc, w[j]);
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < PL / 2; i++) {
                        w[j][i] = t < hi && ok[u] ? w[j][i] : 0u;
                        odd = odd || T::odd(w[j][i]);
                        w[j][i] = T::clean(w[j][i]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < PL / 2; i++) {
                const u4 e = {lo16(w[0][i], w[1][i]), lo16(w[2][i], w[3][i]), lo16(w[4][i], w[5][i]), lo16(w[6][i], w[7][i])};
                const u4 o = {hi16(w[0][i], w[1][i]), hi16(w[2][i], w[3][i]), hi16(w[4][i], w[5][i]), hi16(w[6][i], w[7][i])};
                acc[b * PL + 2 * i] = T::mfma16(__builtin_bit_cast(v8, e), pf, acc[b * PL + 2 * i]);
                acc[b * PL + 2 * i + 1] = T::mfma16(__builtin_bit_cast(v8, o), pf, acc[b * PL + 2 * i + 1]);
            }
        }
    }
    /* an infinity or NaN among rows that some columns do not attend would reach them as 0 * inf:
     * left out above, added here to the columns that do attend it */
    if (__any(odd)) {
        for (int t0 = sp * a.chunk + FEW_STEP * wave; t0 < hi; t0 += FEW_STEP * FEW_WAVES) {
#pragma unroll 1
            for (int t = t0; t < min(t0 + FEW_STEP, hi); t++) {
                const int id = word_of(pages, t >> a.b.page_shift);
                if (t0 + FEW_STEP <= full && t0 + FEW_STEP <= hi && page_ok(a.b, word_of(pages, t0 >> a.b.page_shift)) &&
                    page_ok(a.b, word_of(pages, (t0 + 16) >> a.b.page_shift))) break;   /* a step taken as it is */
                if (!page_ok(a.b, id)) continue;
                const uint8_t *row = vbase + (int64_t)id * a.v.page_stride + (int64_t)(t & (page_rows - 1)) * (D * ES);
                const uint8_t *sc = MX ? vsb + (int64_t)id * a.v.scale_page_stride + (t & (page_rows - 1)) * (D / MX_BLOCK) : nullptr;
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int j = 0; j < PL; j++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const unsigned x = row_elem<T, MX>(row, sc, b * BD + (4 * g + i) * PL + j);
                            acc[b * PL + j][i] += T::odd(x) && (attended(t) & 1) ? T::wide(x) : 0.0f;
                        }
            }
        }
    }

    /* the four waves' columns together: a lane's sums cover its own rows of each step only */
    l = sum16(sum32(l));
    if (g == 0) { lds_m[wave][lc] = m; lds_l[wave][lc] = l; }
    const unsigned mine = (unsigned)__ballot(some);
    if (lane == 0) lds_some[wave] = mine;
    __syncthreads();
    const bool direct = n_sp == 1;
    const int oc = threadIdx.x >> 4, od = (threadIdx.x & 15) * PL;   /* output column and element of this thread */
    float M = lds_m[0][lc];
#pragma unroll
    for (int w = 1; w < FEW_WAVES; w++) M = fmaxf(M, lds_m[w][lc]);
    const float f = m == -__builtin_huge_valf() ? (l == 0.0f ? 0.0f : 1.0f) : exp2_hw(m - M);
    /* the output thread's column */
    float Mo = lds_m[0][oc], Lo = 0.0f;
#pragma unroll
    for (int w = 1; w < FEW_WAVES; w++) Mo = fmaxf(Mo, lds_m[w][oc]);
#pragma unroll
    for (int w = 0; w < FEW_WAVES; w++) {
        const float mw = lds_m[w][oc], lw = lds_l[w][oc];
        Lo += mw == -__builtin_huge_valf() ? lw : lw * exp2_hw(mw - Mo);
    }
    static_assert(FEW_WAVES == 4);
    const bool undefined = Lo == 0.0f && ((lds_some[0] | lds_some[1] | lds_some[2] | lds_some[3]) >> oc & 1);
    const int co = tile * CT + oc;
    const bool here = co < cols;
    const int ot = here ? co / a.group : 0, oh = kvh * a.group + (here ? co % a.group : 0);
    const int64_t row = (int64_t)(q.q0 + ot) * a.heads + oh;
#pragma unroll
    for (int b = 0; b < NB; b++) {
        if (b) __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < PL; j += 4)
                *(f4 *)&lds_o[wave][lc][(4 * g + i) * PL + j] =
                    (f4){acc[b * PL + j][i] * f, acc[b * PL + j + 1][i] * f, acc[b * PL + j + 2][i] * f, acc[b * PL + j + 3][i] * f};
        __syncthreads();
        if (!here) continue;
        float o[PL];
#pragma unroll
        for (int j = 0; j < PL; j++) {
            o[j] = 0.0f;
#pragma unroll
            for (int w = 0; w < FEW_WAVES; w++) o[j] += lds_o[w][oc][od + j];
        }
        if (direct) {
            const float inv = undefined ? UNDEFINED : Lo == 0.0f ? 0.0f : 1.0f / Lo;
            uint8_t *out = a.out + (int64_t)(q.q0 + ot) * a.ot + (int64_t)oh * a.oh + 2 * (b * BD + od);
#pragma unroll
            for (int j = 0; j < PL; j += 4)
                *(u2_any *)(out + 2 * j) = (u2){T::pack(o[j] * inv, o[j + 1] * inv), T::pack(o[j + 2] * inv, o[j + 3] * inv)};
        } else if (!(Lo == 0.0f)) {
            float *po = a.part + (row * a.n_splits + sp) * D + b * BD + od;
#pragma unroll
            for (int j = 0; j < PL; j += 4) *(f4 *)(po + j) = (f4){o[j], o[j + 1], o[j + 2], o[j + 3]};
        }
    }
    if (here && (threadIdx.x & 15) == 0) {
        if (!direct) {
            float *ml = a.part + (int64_t)a.b.n_tokens * a.heads * a.n_splits * D + (row * a.n_splits + sp) * 2;
            ml[0] = undefined ? UNDEFINED : Mo;
            ml[1] = Lo;
        } else if (a.lse) a.lse[row] = Lo == 0.0f ? -__builtin_huge_valf() : (Mo + __log2f(Lo)) * 0.69314718055994531f;
    }
}

/* The splits of a query row joined: out = sum_i o_i 2^(m_i - M) / sum_i l_i 2^(m_i - M). DV / 4
 * threads take a row, four elements each, so a workgroup holds JOIN_THREADS / (DV / 4) groups of
 * threads: with few splits each group has a row of its own; with many (MANY) they share one row's
 * splits and meet in LDS, since one group's loads of 256 splits, one after the other, took 86 us
 * where the attention over 131071 rows took 59. A split whose sum is 0 holds no sums; its maximum is
 * -infinity where the row attends nothing of it, NaN where scores were all -infinity. */
constexpr int JOIN_THREADS = 256, JOIN_MANY = 16;

template <class T, int DV, bool MANY>
__global__ __launch_bounds__(JOIN_THREADS) void k_attend_join(AttendArgs a) {
    constexpr int TPR = DV / 4, NG = JOIN_THREADS / TPR;
    constexpr float NINF = -__builtin_huge_valf();
    __shared__ __align__(16) f4 lds_o[MANY ? JOIN_THREADS : 1];
    __shared__ float lds_l[NG], lds_m[JOIN_THREADS / 64];
    __shared__ bool lds_some[JOIN_THREADS / 64];
    const int seq = blockIdx.z, grp = threadIdx.x / TPR, e = threadIdx.x % TPR * 4;
    const Seq q = seq_of(a.b, seq);
    const int r = MANY ? blockIdx.x : blockIdx.x * NG + grp;
    const int t = r / a.heads, h = r % a.heads;
    const int n_sp = max(1, (q.kv + a.chunk - 1) / a.chunk);
    if (n_sp == 1) return;
    const bool on = t < min(q.n, a.b.max_q);
    if (!on) return;   /* MANY: the whole workgroup */
    const int64_t row = (int64_t)(q.q0 + t) * a.heads + h;
    const float *po = a.part + row * a.n_splits * DV + e;
    const float *ml = a.part + (int64_t)a.b.n_tokens * a.heads * a.n_splits * DV + row * a.n_splits * 2;
    float M = NINF;
    bool some = false;   /* a split whose scores were all -infinity */
    auto take = [&](float m) __attribute__((always_inline)) {
        some = some || m != m;
        M = fmaxf(M, m);   /* not the NaN */
    };
    if constexpr (MANY) {
        for (int i = threadIdx.x; i < n_sp; i += JOIN_THREADS) take(ml[2 * i]);
#pragma unroll
        for (int d = 32; d; d >>= 1) M = fmaxf(M, __shfl_xor(M, d));
        some = __any(some);
        if ((threadIdx.x & 63) == 0) {
            lds_m[threadIdx.x >> 6] = M;
            lds_some[threadIdx.x >> 6] = some;
        }
        __syncthreads();
        M = fmaxf(fmaxf(lds_m[0], lds_m[1]), fmaxf(lds_m[2], lds_m[3]));
        some = lds_some[0] || lds_some[1] || lds_some[2] || lds_some[3];
    } else {
        for (int i = 0; i < n_sp; i++) take(ml[2 * i]);
    }
    float L = 0.0f;
    f4 o = {0, 0, 0, 0};
#pragma unroll 4
    for (int i = MANY ? grp : 0; i < n_sp; i += MANY ? NG : 1) {
        const float mi = ml[2 * i], li = ml[2 * i + 1];
        const f4 x = *(const f4 *)(po + (int64_t)i * DV);      /* within the workspace whether written or not */
        const float f = mi == NINF ? 1.0f : exp2_hw(mi - M);
        const bool some = !(li == 0.0f);
        L += some ? li * f : 0.0f;
#pragma unroll
        for (int j = 0; j < 4; j++) o[j] += some ? x[j] * f : 0.0f;
    }
    if constexpr (MANY) {
        lds_o[threadIdx.x] = o;
        if (e == 0) lds_l[grp] = L;
        __syncthreads();
        if (grp) return;
#pragma unroll
        for (int k = 1; k < NG; k++) {
            o += lds_o[k * TPR + threadIdx.x];
            L += lds_l[k];
        }
    }
    const float inv = L == 0.0f ? (some ? UNDEFINED : 0.0f) : 1.0f / L;
    uint8_t *out = a.out + (int64_t)(q.q0 + t) * a.ot + (int64_t)h * a.oh + 2 * e;
    *(u2_any *)out = (u2){T::pack(o[0] * inv, o[1] * inv), T::pack(o[2] * inv, o[3] * inv)};
    if (a.lse && e == 0) a.lse[row] = L == 0.0f ? NINF : (M + __log2f(L)) * 0.69314718055994531f;
}

template <class T, bool MX, int D>
void few_t(const AttendArgs &a, hipStream_t st) {
    const int tiles = (a.b.max_q * a.group + 15) / 16;
    const dim3 grid((unsigned)a.n_splits * a.kv_heads * tiles, 1, a.b.n_seqs);
    hipLaunchKernelGGL((k_attend_few<T, MX, D>), grid, dim3(64 * FEW_WAVES), 0, st, a);
}

template <class T, int DV>
void join_t(const AttendArgs &a, hipStream_t st) {
    const int rows = a.b.max_q * a.heads, ng = JOIN_THREADS / (DV / 4);
    if (a.n_splits > JOIN_MANY)
        hipLaunchKernelGGL((k_attend_join<T, DV, true>), dim3(rows, 1, a.b.n_seqs), dim3(JOIN_THREADS), 0, st, a);
    else
        hipLaunchKernelGGL((k_attend_join<T, DV, false>), dim3((rows + ng - 1) / ng, 1, a.b.n_seqs), dim3(JOIN_THREADS), 0, st, a);
}

} // namespace

/* Columns (query rows of a kv head) up to which the kernel of few rows is taken, 16 of them a
 * workgroup: past 32 its further passes over the cache cost more than the other's idle columns. 32
 * sequences of 4096 rows, width 128, few against many: 8-bit rows 42 and 51 us at 32 columns, 82
 * and 51 at 40; 16-bit ones 47 and 44 at 32, 111 and 46 at 48; of width 256 108 and 132 at 24. */
static bool takes_many(int64_t cols) { return cols > 32; }

/* Rows a split takes: enough workgroups for the 256 units, two each (one of the latent form, which
 * fills a unit; with four of few rows a unit 32 tokens over 2048 to 8192 8-bit rows took 51 us, not
 * 45, and one over 131071 16-bit rows 59, not 55: more partial sums to write and join). Few query
 * rows are not split below 512 rows: one launch of 500 rows takes 10 us where a split one and its
 * join take 12.5; at 1000 rows two splits take 16 us and eight 15. Many are split down to 192 rows (85 tokens over 2132 rows:
 * 26 us, at 128 rows 31; 64 over 500: 17 us, at 256 rows 20), the latent form down to 128 (1 token
 * over 500 rows: 21 us, at 256 rows 26; 1 over 8192: 30 us, at 64 rows 35). */
Split attend_split(int n_seqs, int max_q, int kv_cap, int heads, int kv_heads, bool latent) {
    const int64_t cols = (int64_t)max_q * (heads / kv_heads);
    const bool many = !latent && takes_many(cols);
    const int tile = latent ? 64 : many ? 128 : 16, step = latent ? 64 : FEW_STEP * FEW_WAVES, at_once = latent ? 256 : 512;
    const int64_t wgs = std::max<int64_t>((int64_t)n_seqs * kv_heads * ((cols + tile - 1) / tile), 1);
    const int64_t want = std::max<int64_t>(1, at_once / wgs);
    int64_t chunk = (kv_cap + want - 1) / want;
    chunk = std::max<int64_t>((chunk + step - 1) / step * step, latent ? 128 : many ? 192 : 512);
    return {(int)chunk, std::max(1, (int)((kv_cap + chunk - 1) / chunk)), many};
}

void attend(const AttendArgs &a, int q_dtype, int cache_dtype, int width, bool many, hipStream_t st) {
    const bool mx = cache_dtype == DT_MX8;
#define HXP_BY(F, T) (width == 64 ? F(T, 64) : width == 128 ? F(T, 128) : F(T, 256))
#define HXP_FEW(T, D) (mx ? few_t<T, true, D>(a, st) : few_t<T, false, D>(a, st))
#define HXP_JOIN(T, D) join_t<T, D>(a, st)
    if (many) attend_many(a, q_dtype, cache_dtype, width, st);
    else if (q_dtype == DT_BF16) HXP_BY(HXP_FEW, Bf16);
    else HXP_BY(HXP_FEW, F16);
    if (a.n_splits == 1) return;
    if (q_dtype == DT_BF16) HXP_BY(HXP_JOIN, Bf16);
    else HXP_BY(HXP_JOIN, F16);
#undef HXP_JOIN
#undef HXP_FEW
#undef HXP_BY
}

void attend_latent(const AttendArgs &a, int q_dtype, int cache_dtype, hipStream_t st) {
    latent_rows(a, q_dtype, cache_dtype == DT_MX8, st);
    if (a.n_splits == 1) return;
    if (q_dtype == DT_BF16) join_t<Bf16, 512>(a, st);
    else join_t<F16, 512>(a, st);
}

} // namespace hxp
