/*
 * k_paged_latent.hip — absorbed latent attention over a paged cache: every query head of a token
 * reads the same rows [c (512) | pe (64)], s = scale (q . c + q_pe . pe), out = softmax(s) c.
 *
 * With 2 x 1088 flops a (column, row) against 1152 bytes a row it is bound by the matrix units
 * from about 150 columns a sequence on, and by the rows' bytes below. The products run transposed
 * as in k_paged_many.hip: S^T = K Q^T, O^T = C^T P^T. A workgroup takes 64 columns and 32 rows a
 * step. Its eight waves, two a SIMD, have two roles: four take the scores of a step (each 16 rows
 * and 32 columns, whose queries fill 144 registers) and write its probabilities to LDS; the other
 * four take the sums of the step before (each a quarter of the latent and all columns, 128
 * registers). So one role's exponentials, reads and waits run under the other's matrix
 * instructions, with one barrier a step and four steps' rows in LDS (one summed, one scored, two
 * arriving). 9 tokens of 128 heads over 131072 16-bit rows take 380 us (865 TFLOP/s) and over 8-bit
 * ones 390 us; four waves that did both in turn, 64 rows a step, took 478 and 504 (where this took
 * 400 and 430). A step of 32 rows
 * takes 2600 cycles, its products 1088; the rest is the way from a barrier to the first product
 * (page, addresses, LDS: 400) and from the last to the next barrier (exponentials, packing: 700).
 * The rows of a step lie in LDS once, row-major, for both products: the score reads them along
 * the row, the sum through the transposing LDS load. The eight 16-byte pieces of each 128 bytes are
 * exchanged by row (piece p of row r at p ^ swz(r)) so that neither read meets a bank conflict.
 * 16-bit rows go from memory to LDS directly, 8-bit rows through registers, where they become
 * 16-bit ones. A wave brings in half of eight rows, which lie in one page whatever its size.
 */
#include "hx_paged.h"

#include <algorithm>

namespace hxp {

namespace {

constexpr int LW = 576, LC = 512;                   /* row width (latent, rotated part), latent */
constexpr int L_WAVES = 8, L_THREADS = 64 * L_WAVES, L_COLS = 64, L_ROWS = 32;
constexpr int L_TILE = L_ROWS * LW * 2;             /* bytes of a step in LDS */
constexpr int L_CHUNKS = LW / 64;                   /* 128-byte chunks of a 16-bit row: 8 pieces of 16 bytes */
constexpr int L_BUFS = 4, L_LDS = L_BUFS * L_TILE;  /* steps in LDS; first the queries are in two of them, last the sums in all */
static_assert(2 * L_TILE == L_COLS * LW * 2 && L_LDS >= L_COLS * LC * 4);

/* The sums' four aligned rows need positions that differ in bit 2; the scores' 16 lanes that LDS serves
 * together are not neighbours (rows 0-3 and 12-15 of one piece with rows 4-11 of the piece beside
 * it), so rows 0-3 and 12-15 take positions in pairs that differ in bit 0: with an order that only
 * kept 16 rows of one piece apart, reads took twice as long and a call 3% more. */
__device__ __forceinline__ int swz(int r) {
    const int k = r >> 1 & 7;
    return (k & 1) << 2 | (-(k >> 1) & 3);
}
/* A step in LDS: blocks of 8 rows x one chunk (1 KiB), the chunks of 8 rows side by side, so that one
 * load instruction's 64 pieces of 16 bytes are a block and its addresses one lane constant plus the
 * block's */
__device__ __forceinline__ int piece_at(int r, int p) {
    return ((r >> 3) * L_CHUNKS + (p >> 3)) * 1024 + (r & 7) * 128 + ((p & 7) ^ swz(r)) * 16;
}

template <class T, bool MX>
__global__ __launch_bounds__(L_THREADS) void k_attend_latent(AttendArgs a) {
    using v8 = typename T::v8;
    constexpr float NINF = -__builtin_huge_valf();
    __shared__ __align__(16) uint8_t lds[L_LDS];
    __shared__ __align__(16) uint8_t lds_p[2][4][L_COLS * 16];   /* step, group of 8 rows: 8 probabilities a column */
    __shared__ float lds_m[2][L_COLS], lds_l[2][L_COLS];
    __shared__ int lds_flags[4];   /* of step s in s % 4: GROW, NO_ROOM, ODD */
    enum { GROW = 1, NO_ROOM = 2, ODD = 4 };

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const bool scorer = wave < 4;
    /* workgroup i runs on XCD i % 8: each XCD takes an eighth of the (sequence, split, column tile)
     * list, in which the column tiles of the same rows follow each other and share its L2 */
    const int tiles = (int)(((int64_t)a.b.max_q * a.heads + L_COLS - 1) / L_COLS);
    const int64_t total = (int64_t)a.b.n_seqs * a.n_splits * tiles, w = (blockIdx.x & 7) * ((total + 7) / 8) + (blockIdx.x >> 3);
    if ((int64_t)(blockIdx.x >> 3) >= (total + 7) / 8 || w >= total) return;
    const int pair = (int)(w / tiles), tile = (int)(w % tiles);
    const int seq = pair / a.n_splits, sp = pair % a.n_splits;
    const Seq q = seq_of(a.b, seq);
    const int cols = min(q.n, a.b.max_q) * a.heads;
    if (tile * L_COLS >= cols) return;
    const int n_sp = max(1, (q.kv + a.chunk - 1) / a.chunk);
    if (sp >= n_sp) return;

    const int t_last = min(cols - 1, tile * L_COLS + L_COLS - 1) / a.heads;
    const int hi = min(min(q.kv, a.b.mask ? q.kv : q.base + t_last + 1), (sp + 1) * a.chunk);
    const int full = a.b.mask ? q.base : q.base + tile * L_COLS / a.heads + 1;
    const int lo = sp * a.chunk;
    const int steps = lo < hi ? (hi - lo + L_ROWS - 1) / L_ROWS : 0;
    /* a column of the tile: its token, head, the rows it attends without a mask word, its mask row */
    struct Col { int tok, head, lim; bool on; const unsigned long long *words; };
    auto column = [&](int c) __attribute__((always_inline)) {
        Col r;
        c += tile * L_COLS;
        r.on = c < cols;
        r.tok = r.on ? c / a.heads : 0;
        r.head = r.on ? c % a.heads : 0;
        r.lim = !r.on ? 0 : a.b.mask ? min(q.base, q.kv) : min(q.base + r.tok + 1, q.kv);
        r.words = a.b.mask && r.on ? a.b.mask + (int64_t)(q.q0 + r.tok) * a.b.mask_words : nullptr;
        return r;
    };
    /* which of the 64 rows from t0 on it attends (where their pages exist) */
    auto attended = [&](const Col &c, int t0) __attribute__((always_inline)) { return step_mask(t0, c.lim, hi, q.base, c.words, a.b.mask_words); };

    const int *pages = a.b.pages + (int64_t)seq * a.b.ld_pages;
    const int rmask = (1 << a.b.page_shift) - 1;
    int pid[2];                        /* pages of the two groups of 16 rows, -1: none */
    auto load_pages = [&](int t0) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int t = t0 + 16 * u;
            const int id = t < hi ? word_of(pages, t >> a.b.page_shift) : -1;
            pid[u] = page_ok(a.b, id) ? id : -1;
        }
    };
    auto have = [&]() __attribute__((always_inline)) { return (pid[0] >= 0 ? 1u : 0u) | (pid[1] >= 0 ? 2u : 0u); };
    /* whether the step has rows that only some columns attend; that some column may not attend each
     * of its rows (h: bit u where group u of 16 has a page) */
    auto some_at = [&](int t0) __attribute__((always_inline)) { return full < min(hi, t0 + L_ROWS); };
    auto edge_at = [&](int t0, unsigned h) __attribute__((always_inline)) { return !(t0 + L_ROWS <= full && t0 + L_ROWS <= hi && h == 3u); };

    /* Waves w and w + 4 bring in rows 8 w .. 8 w + 7 of a step: chunks 0-3 and 4-8. 8-bit rows: 8 codes
     * (a piece) a lane. Every load goes to a row of the cache: rows past hi lie in the same page,
     * those of a page that is not there are taken from page 0; settle clears both. */
    const int oct = wave & 3, lr = 8 * oct + (lane >> 3), lp = lane & 7;
    u2 sw[MX ? 5 : 1];
    unsigned ss[MX ? 5 : 1];
    const uint8_t *from = nullptr, *from_s = nullptr;
    auto aim = [&](int t0) __attribute__((always_inline)) {
        const int64_t id = max(oct < 2 ? pid[0] : pid[1], 0);
        const int row = (t0 + 8 * oct) & rmask;
        if constexpr (MX) {
            from = a.k.data + id * a.k.page_stride + (row + (lane >> 3)) * LW + 8 * lp;
            from_s = a.k.scales + id * a.k.scale_page_stride + (row + (lane >> 3)) * (LW / MX_BLOCK) + (lp >> 2);
        } else {
            from = same(a.k.data + id * a.k.page_stride + (int64_t)row * (2 * LW));
        }
    };
    const int off8 = (lane >> 3) * (2 * LW) + (lp ^ swz(lr)) * 16;
    auto load = [&](auto first, auto j, uint8_t *dst) __attribute__((always_inline)) {   /* chunk first + j, constants */
        constexpr int i = first.value + j.value;
        if constexpr (MX) {
            sw[j.value] = *(const u2 *)(from + 64 * i);
            ss[j.value] = from_s[2 * i];
        } else {
            to_lds<128 * i>(from, off8, dst + (oct * L_CHUNKS + i) * 1024);
        }
    };
    /* This wave's chunks of the step s, which have arrived, made ready in LDS; ODD where rows that only
     * some columns attend hold an infinity or NaN */
    auto settle = [&](auto first, auto count, int s, uint8_t *dst, unsigned h) __attribute__((always_inline)) {
        const int t0 = lo + s * L_ROWS;
        const bool edge = edge_at(t0, h), some = some_at(t0), ok = !edge || (t0 + lr < hi && (h >> (lr >> 4) & 1));
        bool odd = false;
        if constexpr (MX) {
            each<count.value>([&](auto j) __attribute__((always_inline)) {
                const float f = mx_scale(ss[j.value]);
                const unsigned x = sw[j.value][0], y = sw[j.value][1];
                u4 w = {T::template from_mx8<false>(x, f), T::template from_mx8<true>(x, f),
                        T::template from_mx8<false>(y, f), T::template from_mx8<true>(y, f)};
                if (edge) {
                    w = ok ? w : (u4){0, 0, 0, 0};
                    odd = odd || (some && (T::odd(w[0]) || T::odd(w[1]) || T::odd(w[2]) || T::odd(w[3])));
                }
                *(u4 *)(dst + piece_at(lr, 8 * (first.value + j.value) + lp)) = w;
            });
        } else {
            if (edge)
#pragma unroll 1
                for (int i = first.value; i < first.value + count.value; i++) {
                    u4 *p = (u4 *)(dst + (oct * L_CHUNKS + i) * 1024 + lane * 16);
                    if (!ok) *p = (u4){0, 0, 0, 0};
                    else if (some) {
                        const u4 w = *p;
                        odd = odd || T::odd(w[0]) || T::odd(w[1]) || T::odd(w[2]) || T::odd(w[3]);
                    }
                }
        }
        if (some && __any(odd) && lane == 0) atomicOr(&lds_flags[s & 3], ODD);
    };
    const std::integral_constant<int, 0> c0;
    const std::integral_constant<int, 4> c4;
    const std::integral_constant<int, 5> c5;
    auto buffer = [&](int s) __attribute__((always_inline)) { return lds + s % L_BUFS * L_TILE; };
    unsigned have0 = 0, have1 = 0, have2 = 0;   /* pages of the groups of 16 rows: of a step and the two behind it */
    /* The first step's loads. From then on 16-bit rows are sent for two steps ahead and waited for at
     * the end of the step before theirs; 8-bit ones, which wait in registers, go to LDS as that
     * step begins, and the next are sent for then. */
    auto start = [&](auto first, auto count) __attribute__((always_inline)) {
        if (!steps) return;
        load_pages(lo);
        have0 = have();
        aim(lo);
        each<count.value>([&](auto j) __attribute__((always_inline)) { load(first, j, lds); });
        if (steps > 1) load_pages(lo + L_ROWS);
    };
    auto send = [&](int s) __attribute__((always_inline)) {   /* where step s lies; the pages of the next */
        const unsigned h = have();
        aim(lo + s * L_ROWS);
        if (s + 1 < steps) load_pages(lo + (s + 1) * L_ROWS);
        return h;
    };
    auto begin = [&](auto first, auto count) __attribute__((always_inline)) {
        if (steps) {
            if constexpr (MX) settle(first, count, 0, lds, have0);
            if (steps > 1) {
                have1 = send(1);
                each<count.value>([&](auto j) __attribute__((always_inline)) { load(first, j, buffer(1)); });
            }
            if constexpr (!MX) {
                if (steps > 1) vm_wait<count.value>();
                else vm_wait<0>();
                settle(first, count, 0, lds, have0);
            }
        }
        __syncthreads();
    };
    /* as step s begins; returns whether the step after the next is to be sent for (16-bit) */
    auto ahead = [&](auto first, auto count, int s) __attribute__((always_inline)) {
        if constexpr (MX)
            if (s + 1 < steps) settle(first, count, s + 1, buffer(s + 1), have1);
        if (s + 2 >= steps) return false;
        have2 = send(s + 2);
        if constexpr (MX) each<count.value>([&](auto j) __attribute__((always_inline)) { load(first, j, nullptr); });
        return true;
    };
    /* as it ends */
    auto finish = [&](auto first, auto count, int s, bool more) __attribute__((always_inline)) {
        if constexpr (!MX)
            if (s + 1 < steps) {
                if (more) vm_wait<count.value>();
                else vm_wait<0>();
                settle(first, count, s + 1, buffer(s + 1), have1);
            }
        have0 = have1;
        have1 = have2;
        __syncthreads();
    };
    /* The scores are done with step s: an infinity or NaN among rows that some columns do not attend
     * would reach them as 0 * inf in the sums, so it is taken out of LDS and added at the end to the
     * columns that attend it */
    auto clean = [&](int s) __attribute__((always_inline)) {
        unsigned *p = (unsigned *)buffer(s);
        for (int i = threadIdx.x; i < L_TILE / 4; i += L_THREADS) p[i] = T::clean(p[i]);
    };

    if (threadIdx.x < 4) lds_flags[threadIdx.x] = 0;
    __syncthreads();
    if (scorer) start(c0, c4);
    else start(c4, c5);
    /* The queries come in by rows, eight lanes 128 bytes, and go to the waves' operands through the
     * other buffers: read as operands, 32 rows of 32 bytes an instruction, they took 10000 cycles. */
    {
        const int r = 8 * wave + (lane >> 3), qc = tile * L_COLS + r;
        const int qt = qc < cols ? qc / a.heads : 0, qh = qc < cols ? qc % a.heads : 0;
        const uint8_t *qp = a.q + (int64_t)(q.q0 + qt) * a.qt + (int64_t)qh * a.qh + 16 * lp;
        const uint8_t *pp = a.q_pe + (int64_t)(q.q0 + qt) * a.pt + (int64_t)qh * a.ph + 16 * lp;
        u4 x[L_CHUNKS];
#pragma unroll
        for (int i = 0; i < L_CHUNKS; i++) {
            x[i] = *(const u4_any *)(i < LC / 64 ? qp + 128 * i : pp);
            if (qc >= cols) x[i] = (u4){0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < L_CHUNKS; i++) *(u4 *)(lds + 2 * L_TILE + piece_at(r, 8 * i + lp)) = x[i];
        __syncthreads();
    }

    bool odd_any = false, again = false;
    if (scorer) {
        /* 16 x 16 x 32: lane (g, c) has piece g of 64 bytes of row c, and rows 4 g .. 4 g + 3 of column c
         * of the result */
        constexpr int KS = LW / 32;
        const int g = lane >> 4, c = lane & 15, r0 = 16 * (wave >> 1), first = 32 * (wave & 1);
        const Col col[2] = {column(first + c), column(first + 16 + c)};
        v8 qf[KS][2];
#pragma unroll
        for (int i = 0; i < KS; i++)
#pragma unroll
            for (int n = 0; n < 2; n++) qf[i][n] = *(const v8 *)(lds + 2 * L_TILE + piece_at(first + 16 * n + c, 4 * i + g));
        arrived();
        const int k_at = piece_at(r0 + c, g);
        float m[2] = {NINF, NINF}, l[2];
        unsigned some = 0;   /* bit n: the column attends a row of the split (as truth values they took scalars, which ran out) */
        /* Scores of step s, scaled; rows that are not attended -infinity. The rows two steps on are
         * sent for among the products: the address units take 64 bytes a cycle of all waves' together. */
        f4 s[2];
        auto scores = [&](int step, bool more, unsigned h) __attribute__((always_inline)) {
            const uint8_t *tl = buffer(step);
            uint8_t *nx = buffer(step + 2);
            f4 x[2][2];   /* two sums a column: an instruction that adds to the one before it waits for it */
#pragma unroll
            for (int i = 0; i < 4; i++) x[i >> 1][i & 1] = (f4){0, 0, 0, 0};
            /* reads run five pairs of instructions ahead of their use, in this order: left to itself the
             * compiler puts each read right before its instruction and waits for it */
            constexpr int AHEAD = 5;
            v8 kr[AHEAD + 1];
            auto read_k = [&](int i) __attribute__((always_inline)) { return *(const v8 *)(tl + (k_at ^ 64 * (i & 1)) + 1024 * (i >> 1)); };
#pragma unroll
            for (int i = 0; i < AHEAD; i++) kr[i] = read_k(i);
            in_order();
            each<KS>([&](auto k_) __attribute__((always_inline)) {
                constexpr int k = k_.value;
                if constexpr (k + AHEAD < KS) kr[(k + AHEAD) % (AHEAD + 1)] = read_k(k + AHEAD);
                in_order();
                x[k & 1][0] = T::mfma16(kr[k % (AHEAD + 1)], qf[k][0], x[k & 1][0]);
                x[k & 1][1] = T::mfma16(kr[k % (AHEAD + 1)], qf[k][1], x[k & 1][1]);
                in_order();
                if constexpr (!MX && k % 4 == 1 && k / 4 < 4) {
                    if (more) load(c0, std::integral_constant<int, k / 4>{}, nx);
                    in_order();
                }
            });
            const int t0 = lo + step * L_ROWS;
#pragma unroll
            for (int n = 0; n < 2; n++) s[n] = (x[0][n] + x[1][n]) * a.scale2;
            if (!edge_at(t0, h)) some = 3;
            else
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    const unsigned long long at = attended(col[n], t0) & group_rows(h), vis = at >> (r0 + 4 * g);
                    some |= at ? 1u << n : 0u;
#pragma unroll
                    for (int j = 0; j < 4; j++) s[n][j] = vis >> j & 1 ? s[n][j] : NINF;
                }
        };
        auto largest = [&](int n) __attribute__((always_inline)) { return fmaxf(fmaxf(s[n][0], s[n][1]), fmaxf(s[n][2], s[n][3])); };
        auto exchange = [&](const float (&x)[2]) __attribute__((always_inline)) {   /* over a column's lanes, to lds_m */
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const float y = max16(max32(x[n]));
                if (g == 0) lds_m[wave >> 1][first + 16 * n + c] = y;
            }
        };
        auto common = [&](int n) __attribute__((always_inline)) { return fmaxf(lds_m[0][first + 16 * n + c], lds_m[1][first + 16 * n + c]); };
        float sum[2];
        auto weigh = [&](int step) __attribute__((always_inline)) {
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const float ms = m[n] == NINF ? 0.0f : m[n];
                float x[4];
#pragma unroll
                for (int j = 0; j < 4; j++) x[j] = exp2_hw(s[n][j] - ms);
                sum[n] = (x[0] + x[1]) + (x[2] + x[3]);
                *(u2 *)(lds_p[step & 1][r0 / 8 + (g >> 1)] + (first + 16 * n + c) * 16 + 8 * (g & 1)) = (u2){T::pack(x[0], x[1]), T::pack(x[2], x[3])};
            }
        };
        /* The maximum that probabilities are taken against is that of the first step in which a column
         * attends something; they may exceed 1 by 2^14, which costs no accuracy in either 16-bit type.
         * Where a later score exceeds it by more, the rows are gone through for the maxima alone and
         * then once more: the sums are never rescaled. So a call's time depends on its scores: queries
         * three times as wide as those of the 380 us above, whose scores do so, take 930 us. */
        constexpr float ROOM = 14.0f;
        auto pass = [&]() __attribute__((always_inline)) {
            l[0] = l[1] = 0.0f;
            begin(c0, c4);
            for (int step = 0; step < steps; step++) {
                const bool more = ahead(c0, c4, step);
                scores(step, more, have0);
                const float mx[2] = {largest(0), largest(1)};
                const bool up[2] = {mx[0] > m[0] + ROOM, mx[1] > m[1] + ROOM};
                if (__any(up[0] || up[1])) {
                    const bool none = __any((up[0] && m[0] != NINF) || (up[1] && m[1] != NINF));
                    if (lane == 0) atomicOr(&lds_flags[step & 3], none ? GROW | NO_ROOM : GROW);
                }
                weigh(step);
                finish(c0, c4, step, more);
                const int flags = lds_flags[step & 3];
                if (flags) {
                    again = again || (flags & NO_ROOM);
                    odd_any = odd_any || (flags & ODD);
                    if (flags & ODD) clean(step);
                    exchange(mx);
                    __syncthreads();
#pragma unroll
                    for (int n = 0; n < 2; n++)
                        if (m[n] == NINF) m[n] = common(n);
                    weigh(step);
                    if (threadIdx.x == 0) lds_flags[step & 3] = 0;
                    __syncthreads();
                }
                l[0] += sum[0];
                l[1] += sum[1];
            }
        };
        for (int round = 0;; round++) {
            pass();
            if (!again || round) break;
            __syncthreads();   /* (A) the last sums are done with their rows */
            start(c0, c4);
            begin(c0, c4);
            for (int step = 0; step < steps; step++) {
                const bool more = ahead(c0, c4, step);
                scores(step, more, have0);
                m[0] = fmaxf(m[0], largest(0));
                m[1] = fmaxf(m[1], largest(1));
                finish(c0, c4, step, more);
            }
            if (threadIdx.x < 4) lds_flags[threadIdx.x] = 0;   /* odd rows' */
            exchange(m);
            __syncthreads();   /* (B) */
            m[0] = common(0);
            m[1] = common(1);
            odd_any = false;
            start(c0, c4);
        }
        /* a column's sum of probabilities over its lanes, and over the two waves through LDS */
#pragma unroll
        for (int n = 0; n < 2; n++) {
            const float y = sum16(sum32(l[n]));
            if (g == 0) {
                lds_l[wave >> 1][first + 16 * n + c] = y;
                if (!(wave >> 1)) lds_m[0][first + 16 * n + c] = m[n] == NINF && (some >> n & 1) ? UNDEFINED : m[n];
            }
        }
        __syncthreads();   /* (C) */
    } else {
        /* 32 x 32 x 16: 128 elements of the latent (four tiles) by 64 columns */
        const int part = wave - 4, half = lane >> 5, lc = lane & 31;
        const int vr = 8 * half + ((lane & 15) >> 2), vp = 16 * part + 2 * (lane >> 4 & 1) + (lane >> 1 & 1);
        const int v_at[2] = {piece_at(vr, vp) + 8 * (lane & 1), piece_at(vr + 4, vp) + 8 * (lane & 1)};
        f16v acc[4][2];
        auto sums = [&](int step, bool more, uint8_t *nx) __attribute__((always_inline)) {
            const uint8_t *tl = buffer(step);
            v8 pf[2][2], vr8[2][4];
            auto read_v = [&](int i, int u) __attribute__((always_inline)) {   /* tile i of the latent, group u of the rows */
                const u2 x = read_tr(tl + (v_at[0] ^ 64 * (i & 1)) + 1024 * (i >> 1) + u * (2048 * L_CHUNKS));
                const u2 y = read_tr(tl + (v_at[1] ^ 64 * (i & 1)) + 1024 * (i >> 1) + u * (2048 * L_CHUNKS));
                return __builtin_bit_cast(v8, (u4){x[0], x[1], y[0], y[1]});
            };
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int n = 0; n < 2; n++) pf[u][n] = *(const v8 *)(lds_p[step & 1][2 * u + half] + (32 * n + lc) * 16);
#pragma unroll
            for (int i = 0; i < 4; i++) vr8[0][i] = read_v(i, 0);
            in_order();
            each<2>([&](auto u_) __attribute__((always_inline)) {
                constexpr int u = u_.value;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (u == 0) vr8[1][i] = read_v(i, 1);
                in_order();
                each<4>([&](auto i_) __attribute__((always_inline)) {
                    constexpr int i = i_.value, k = 4 * u + i;
                    acc[i][0] = T::mfma32(vr8[u][i], pf[u][0], acc[i][0]);
                    acc[i][1] = T::mfma32(vr8[u][i], pf[u][1], acc[i][1]);
                    in_order();
                    if constexpr (!MX && k < 5) {
                        if (more) load(c4, std::integral_constant<int, k>{}, nx);
                        in_order();
                    }
                });
            });
        };
        auto pass = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int j = 0; j < 16; j++) acc[i][n][j] = 0.0f;
            begin(c4, c5);
            for (int step = 0; steps; step++) {   /* the sums are a step behind */
                const bool more = ahead(c4, c5, step);
                uint8_t *nx = buffer(step + 2);
                if (step) sums(step - 1, more, nx);
                if (step == steps) break;
                if constexpr (!MX)
                    if (step == 0 && more) each<5>([&](auto j) __attribute__((always_inline)) { load(c4, j, nx); });
                finish(c4, c5, step, more);
                const int flags = lds_flags[step & 3];
                if (flags) {
                    again = again || (flags & NO_ROOM);
                    odd_any = odd_any || (flags & ODD);
                    if (flags & ODD) clean(step);
                    __syncthreads();
                    __syncthreads();
                }
            }
        };
        for (int round = 0;; round++) {
            pass();
            if (!again || round) break;
            __syncthreads();   /* (A) */
            start(c4, c5);
            begin(c4, c5);
            for (int step = 0; step < steps; step++) {
                const bool more = ahead(c4, c5, step);
                if constexpr (!MX)
                    if (more) each<5>([&](auto j) __attribute__((always_inline)) { load(c4, j, buffer(step + 2)); });
                finish(c4, c5, step, more);
            }
            __syncthreads();   /* (B) */
            odd_any = false;
            start(c4, c5);
        }
        __syncthreads();   /* (C) every wave is done with the rows */
        /* The sums go out by rows, through the steps' LDS (column c's 16-byte unit u at u ^ c mod 32, so
         * that neither the columns' writes nor the rows' reads meet a bank conflict): 16 bytes a lane
         * and row straight from the registers took 8000 cycles. */
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int k = 0; k < 4; k++)
                    *((f4 *)lds + (32 * n + lc) * (LC / 4) + ((32 * part + 8 * i + 2 * k + half) ^ lc)) =
                        (f4){acc[i][n][4 * k], acc[i][n][4 * k + 1], acc[i][n][4 * k + 2], acc[i][n][4 * k + 3]};
    }
    auto unit = [&](int c, int u) __attribute__((always_inline)) { return (f4 *)lds + c * (LC / 4) + (u ^ (c & 31)); };
    __syncthreads();
    if (odd_any) {   /* what was taken out of LDS above: column `lane`, an eighth of the latent a wave */
        const Col col = column(lane);
#pragma unroll 1
        for (int t = max(lo, full / L_ROWS * L_ROWS); t < hi; t++) {
            const int id = word_of(pages, t >> a.b.page_shift);
            if (!page_ok(a.b, id) || !(attended(col, t) & 1)) continue;
            const uint8_t *rp = a.k.data + (int64_t)id * a.k.page_stride + (int64_t)(t & rmask) * (LW * (MX ? 1 : 2));
            const uint8_t *sc = MX ? a.k.scales + (int64_t)id * a.k.scale_page_stride + (t & rmask) * (LW / MX_BLOCK) : nullptr;
#pragma unroll 1
            for (int e = 0; e < 64; e++) {
                const unsigned v = row_elem<T, MX ? 8 : 16>(rp, sc, 64 * wave + e);
                if (T::odd(v)) ((float *)unit(lane, 16 * wave + (e >> 2)))[e & 3] += T::wide(v);
            }
        }
        __syncthreads();
    }
    const bool direct = n_sp == 1;
    for (int r = wave; r < L_COLS; r += L_WAVES) {   /* a row a wave at a time */
        const Col col = column(r);
        if (!col.on) break;
        const float L = lds_l[0][r] + lds_l[1][r], m = lds_m[0][r];
        const int64_t row = (int64_t)(q.q0 + col.tok) * a.heads + col.head;
        if (direct) {
            const float f = L == 0.0f ? (m == m ? 0.0f : UNDEFINED) : 1.0f / L;
            const f4 x = *unit(r, 2 * lane) * f, y = *unit(r, 2 * lane + 1) * f;
            *(u4_any *)(a.out + (int64_t)(q.q0 + col.tok) * a.ot + (int64_t)col.head * a.oh + 16 * lane) =
                (u4){T::pack(x[0], x[1]), T::pack(x[2], x[3]), T::pack(y[0], y[1]), T::pack(y[2], y[3])};
            if (a.lse && lane == 0) a.lse[row] = L == 0.0f ? NINF : (m + __log2f(L)) * 0.69314718055994531f;
        } else {
            if (!(L == 0.0f)) {
                f4 *po = (f4 *)(a.part + (row * a.n_splits + sp) * LC);
                po[lane] = *unit(r, lane);
                po[64 + lane] = *unit(r, 64 + lane);
            }
            if (lane == 0) {
                float *ml = a.part + (int64_t)a.b.n_tokens * a.heads * a.n_splits * LC + (row * a.n_splits + sp) * 2;
                ml[0] = m;
                ml[1] = L;
            }
        }
    }
}

template <class T, bool MX>
void latent_t(const AttendArgs &a, hipStream_t st) {
    const int64_t tiles = ((int64_t)a.b.max_q * a.heads + L_COLS - 1) / L_COLS;
    const int64_t total = (int64_t)a.b.n_seqs * a.n_splits * tiles;
    hipLaunchKernelGGL((k_attend_latent<T, MX>), dim3((unsigned)((total + 7) / 8 * 8)), dim3(L_THREADS), 0, st, a);
}

} // namespace

void latent_rows(const AttendArgs &a, int q_dtype, bool mx, hipStream_t st) {
    if (q_dtype == DT_BF16) mx ? latent_t<Bf16, true>(a, st) : latent_t<Bf16, false>(a, st);
    else mx ? latent_t<F16, true>(a, st) : latent_t<F16, false>(a, st);
}

} // namespace hxp
