/*
 * k_paged_latent.hip — absorbed latent attention over a paged cache: every query head of a token
 * reads the same rows [c (512) | pe (64)], s = scale (q . c + q_pe . pe), out = softmax(s) c.
 *
 * With 2 x 1088 flops a (column, row) against 1152 bytes a row it is bound by the matrix units
 * from about 150 columns a sequence on, and by the rows' bytes below. The products run transposed
 * as in k_paged_many.hip (S^T = K Q^T, O^T = C^T P^T, 32 x 32 x 16). A workgroup of four waves, one
 * a SIMD, takes 64 columns and 64 rows a step; for the scores a wave has 32 columns (their queries
 * in 144 registers) and 32 rows, for the sums its 32 columns, all 64 rows and half of the latent
 * (128 registers): the two waves of a column pair exchange probabilities through LDS (2 KiB each,
 * in the operand's layout). Eight waves of 16 columns and 256 registers had none left to read LDS
 * ahead and took 14400 cycles a step where the products take 2200; all 512 latent elements in one
 * wave (256 registers of sums) spilled.
 * The rows of a step lie in LDS once, row-major, for both products: the score reads them along
 * the row, the sum through the transposing LDS load. The eight 16-byte pieces of each 128 bytes are
 * exchanged by row (piece p of row r at p ^ swz(r)), so that neither read meets a bank conflict.
 * 16-bit rows go from memory to LDS directly, 8-bit rows through registers, where they become
 * 16-bit ones; the next step's are in flight meanwhile. A wave brings in 16 rows, which lie in one
 * page whatever its size.
 */
#include "hx_paged.h"

#include <algorithm>

namespace hxp {

namespace {

constexpr int LW = 576, LC = 512;                   /* row width (latent, rotated part), latent */
constexpr int L_WAVES = 4, L_THREADS = 64 * L_WAVES, L_COLS = 64, L_ROWS = 64;
constexpr int L_TILE = L_ROWS * LW * 2;             /* bytes of a step in LDS */
constexpr int L_CHUNKS = LW / 64;                   /* 128-byte chunks of a 16-bit row: 8 pieces of 16 bytes */

__device__ __forceinline__ int swz(int r) {
    const int k = r >> 1 & 7;
    return (k & 1) << 2 | k >> 1;
}
/* A step in LDS: blocks of 8 rows x one chunk (1 KiB), the chunks of 8 rows side by side, so that one
 * load instruction's 64 pieces of 16 bytes are a block and its addresses one lane constant plus the
 * block's */
__device__ __forceinline__ int piece_at(int r, int p) {
    return ((r >> 3) * L_CHUNKS + (p >> 3)) * 1024 + (r & 7) * 128 + ((p & 7) ^ swz(r)) * 16;
}

typedef short s4v __attribute__((ext_vector_type(4)));

/* four rows of one element each a lane (transposing LDS load): lane i of 16 gives the address of 4
 * elements of row i / 4 and gets element i of the four rows */
__device__ __forceinline__ u2 read_tr(const uint8_t *p) {
    return __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v *)p));
}

template <class T, bool MX>
__global__ __launch_bounds__(L_THREADS, 1) void k_attend_latent(AttendArgs a) {
    using v8 = typename T::v8;
    constexpr int KS = LW / 16, DT = LC / 64;   /* score steps; tiles of 32 latent elements of a wave */
    constexpr float NINF = -__builtin_huge_valf();
    __shared__ __align__(16) uint8_t lds[2][L_TILE];
    __shared__ float lds_m[2][L_COLS];
    __shared__ __align__(16) u4 lds_p[2][2][2][64];   /* column pair, half of the rows, group of 16 */
    __shared__ int lds_grow;

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int half = lane >> 5, lc = lane & 31, wc = wave & 1, wt = wave >> 1;
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

    const int c = tile * L_COLS + 32 * wc + lc;
    const bool on = c < cols;
    const int tok = on ? c / a.heads : 0, head = on ? c % a.heads : 0;
    const int lim = !on ? 0 : a.b.mask ? min(q.base, q.kv) : min(q.base + tok + 1, q.kv);
    const int t_last = min(cols - 1, tile * L_COLS + L_COLS - 1) / a.heads;
    const int hi = min(min(q.kv, a.b.mask ? q.kv : q.base + t_last + 1), (sp + 1) * a.chunk);
    const int full = a.b.mask ? q.base : q.base + tile * L_COLS / a.heads + 1;
    const int lo = sp * a.chunk;
    /* which of the 64 rows from t0 on this lane's column attends (where their pages exist) */
    const unsigned long long *words = a.b.mask && on ? a.b.mask + (int64_t)(q.q0 + tok) * a.b.mask_words : nullptr;
    auto attended = [&](int t0) __attribute__((always_inline)) { return step_mask(t0, lim, hi, q.base, words, a.b.mask_words); };

    f16v acc[DT];
    float m = NINF, l = 0.0f;

    const int *pages = a.b.pages + (int64_t)seq * a.b.ld_pages;
    const int rmask = (1 << a.b.page_shift) - 1;
    int pid[4];
    auto load_pages = [&](int t0) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int t = t0 + 16 * u;
            const int id = t < hi ? word_of(pages, t >> a.b.page_shift) : -1;
            pid[u] = page_ok(a.b, id) ? id : -1;
        }
    };
    auto have = [&]() __attribute__((always_inline)) { return (pid[0] >= 0 ? 1u : 0u) | (pid[1] >= 0 ? 2u : 0u) | (pid[2] >= 0 ? 4u : 0u) | (pid[3] >= 0 ? 8u : 0u); };
    /* whether the step has rows that only some columns attend; that some column may not attend each
     * of its 64 rows (pages: bit u where group u of 16 has one) */
    auto some_at = [&](int t0) __attribute__((always_inline)) { return full < min(hi, t0 + L_ROWS); };
    auto edge_at = [&](int t0, unsigned h) __attribute__((always_inline)) { return !(t0 + L_ROWS <= full && t0 + L_ROWS <= hi && h == 15u); };

    /* 8-bit: 16 codes of row 16 wave + lane / 4, four lanes a chunk */
    u4 sw[MX ? L_CHUNKS : 1];
    unsigned ss[MX ? L_CHUNKS : 1];
    const int mr = 16 * wave + (lane >> 2), mc = lane & 3;
    /* The loads of the step at t0, to LDS (16-bit) or to registers (8-bit). Every load goes to a row
     * of the cache: rows past hi lie in the same page, those of a page that is not there are taken
     * from page 0; settle clears both. */
    const uint8_t *from = nullptr, *from_s = nullptr;   /* where this wave's 16 rows of the next step lie; 8-bit: this lane's codes and scales */
    auto aim = [&](int t0) __attribute__((always_inline)) {
        const int64_t id = max(wave == 0 ? pid[0] : wave == 1 ? pid[1] : wave == 2 ? pid[2] : pid[3], 0);
        const int row = (t0 + 16 * wave) & rmask;
        if constexpr (MX) {
            from = a.k.data + id * a.k.page_stride + (row + (lane >> 2)) * LW + 16 * mc;
            from_s = a.k.scales + id * a.k.scale_page_stride + (row + (lane >> 2)) * (LW / MX_BLOCK) + (mc >> 1);
        } else {
            from = same(a.k.data + id * a.k.page_stride + (int64_t)row * (2 * LW));
        }
    };
    constexpr int LOADS = MX ? L_CHUNKS : 2 * L_CHUNKS;
    const int off8[2] = {(lane >> 3) * (2 * LW) + ((lane & 7) ^ swz(lane >> 3)) * 16, (lane >> 3) * (2 * LW) + ((lane & 7) ^ swz(8 + (lane >> 3))) * 16};
    auto load = [&](auto j, uint8_t *dst) __attribute__((always_inline)) {   /* the j-th load of a step, j a constant */
        constexpr int h = j.value / L_CHUNKS, i = j.value % L_CHUNKS;
        if constexpr (MX) {
            sw[i] = *(const u4 *)(from + 64 * i);
            ss[i] = from_s[2 * i];
        } else {
            to_lds<128 * i>(from + h * 8 * (2 * LW), off8[h], dst + ((2 * wave + h) * L_CHUNKS + i) * 1024);
        }
    };
    /* The loaded step made ready in LDS; true where it has rows that only some columns attend and an
     * element of it is infinite or NaN. */
    auto settle = [&](int t0, uint8_t *dst, unsigned h, bool edge) __attribute__((always_inline)) {
        bool odd = false;
        if constexpr (MX) {
            const bool ok = !edge || (t0 + mr < hi && (h >> wave & 1)), some = some_at(t0);
            const int at0 = piece_at(mr, 2 * mc), at1 = piece_at(mr, 2 * mc + 1);
#pragma unroll
            for (int i = 0; i < L_CHUNKS; i++) {
                const float f = mx_scale(ss[i]);
                u4 w[2];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    w[k >> 1][2 * (k & 1)] = T::template from_mx8<false>(sw[i][k], f);
                    w[k >> 1][2 * (k & 1) + 1] = T::template from_mx8<true>(sw[i][k], f);
                }
                if (edge)
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        w[k] = ok ? w[k] : (u4){0, 0, 0, 0};
                        odd = odd || (some && (T::odd(w[k][0]) || T::odd(w[k][1]) || T::odd(w[k][2]) || T::odd(w[k][3])));
                    }
                *(u4 *)(dst + at0 + 1024 * i) = w[0];
                *(u4 *)(dst + at1 + 1024 * i) = w[1];
            }
        } else {
            vm_wait();   /* this thread's pieces have arrived */
            if (!(h >> wave & 1) || t0 + 16 * wave + 16 > hi)
                for (int i = 0; i < 2 * L_CHUNKS; i++)
                    if (!(h >> wave & 1) || t0 + 16 * wave + (i >= L_CHUNKS ? 8 : 0) + (lane >> 3) >= hi)
                        *(u4 *)(dst + (2 * wave * L_CHUNKS + i) * 1024 + lane * 16) = (u4){0, 0, 0, 0};
            if (some_at(t0))
#pragma unroll 6
                for (int i = 0; i < 2 * L_CHUNKS; i++) {
                    const u4 w = *(const u4 *)(dst + (2 * wave * L_CHUNKS + i) * 1024 + lane * 16);
                    odd = odd || T::odd(w[0]) || T::odd(w[1]) || T::odd(w[2]) || T::odd(w[3]);
                }
        }
        return odd;
    };

    unsigned have_now = 0, have_next = 0;
    bool odd_now = false, odd_next = false, odd_any = false;
    if (threadIdx.x == 0) lds_grow = 0;
    /* the first step's loads go out before the queries', which arrive with them */
    auto start = [&]() __attribute__((always_inline)) {
        if (lo < hi) {
            load_pages(lo);
            have_next = have();
            aim(lo);
            each<LOADS>([&](auto j) { load(j, lds[0]); });
        }
    };
    start();
    /* The queries come in by rows, eight lanes 128 bytes, and go to the waves' operands through the
     * second buffer: read as operands, 32 rows of 32 bytes an instruction, they took 10000 cycles. */
    v8 qf[KS];
    {
        u4 w[2 * L_CHUNKS];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int r = 8 * (2 * wave + h) + (lane >> 3), qc = tile * L_COLS + r;
            const int qt = qc < cols ? qc / a.heads : 0, qh = qc < cols ? qc % a.heads : 0;
            const uint8_t *qp = a.q + (int64_t)(q.q0 + qt) * a.qt + (int64_t)qh * a.qh + 16 * (lane & 7);
            const uint8_t *pp = a.q_pe + (int64_t)(q.q0 + qt) * a.pt + (int64_t)qh * a.ph + 16 * (lane & 7);
#pragma unroll
            for (int i = 0; i < L_CHUNKS; i++) {
                w[L_CHUNKS * h + i] = *(const u4_any *)(i < LC / 64 ? qp + 128 * i : pp);
                if (qc >= cols) w[L_CHUNKS * h + i] = (u4){0, 0, 0, 0};
            }
        }
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < L_CHUNKS; i++)
                *(u4 *)(lds[1] + piece_at(8 * (2 * wave + h) + (lane >> 3), 8 * i + (lane & 7))) = w[L_CHUNKS * h + i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < KS; i++) qf[i] = *(const v8 *)(lds[1] + piece_at(32 * wc + lc, 2 * i + half));
    }
    arrived();

    /* Byte addresses in a step: scores read row 32 wt + lc, pieces 2 i + half; sums read rows 16 g +
     * 4 half .. + 3 and 8 further, elements 256 wt + 32 i .. + 31; the exchange of pieces is an
     * exclusive or with a constant */
    const int r0 = 32 * wt, vr = 4 * half + ((lane & 15) >> 2), vp = 2 * (lane >> 4 & 1) + (lane >> 1 & 1);
    const int k_at = piece_at(r0 + lc, half);
    const int v_at[2] = {piece_at(vr, vp + 32 * wt) + 8 * (lane & 1), piece_at(vr + 8, vp + 32 * wt) + 8 * (lane & 1)};
    /* the first step's rows; then, a step: the next one's under way */
    auto begin = [&]() __attribute__((always_inline)) {
        if (lo < hi) {
            odd_next = settle(lo, lds[0], have_next, edge_at(lo, have_next));
            if (lo + L_ROWS < hi) load_pages(lo + L_ROWS);
        }
        __syncthreads();
    };
    auto ahead = [&](int t0) __attribute__((always_inline)) {
        have_now = have_next;
        odd_now = odd_next;
        if (t0 + L_ROWS < hi) {
            have_next = have();
            aim(t0 + L_ROWS);
            if (t0 + 2 * L_ROWS < hi) load_pages(t0 + 2 * L_ROWS);
        }
    };
    auto finish = [&](int t0, uint8_t *nx) __attribute__((always_inline)) {
        if (t0 + L_ROWS < hi) odd_next = settle(t0 + L_ROWS, nx, have_next, edge_at(t0 + L_ROWS, have_next));
        __syncthreads();
    };
    /* Scores of this wave's rows, scaled; rows that are not attended -infinity. The next step's loads go
     * out among the products: 18 in a row take 1800 cycles to issue, since the address units take 64
     * bytes a cycle of the four waves' together. */
    auto scores = [&](int t0, const uint8_t *tl, uint8_t *nx) __attribute__((always_inline)) {
        const bool more = t0 + L_ROWS < hi;
        f16v s, s1;   /* two sums: an instruction that adds to the one before it waits for it */
#pragma unroll
        for (int j = 0; j < 16; j++) s[j] = s1[j] = 0.0f;
        /* Six instructions' reads ahead of their use, in this order: left to itself the compiler puts
         * each read right before its instruction and waits for it. */
        constexpr int KB = 6, BATCHES = KS / KB;
        v8 kr[2][KB];
        auto read_k = [&](int i) __attribute__((always_inline)) { return *(const v8 *)(tl + (k_at ^ 32 * (i & 3)) + 1024 * (i >> 2)); };
#pragma unroll
        for (int i = 0; i < KB; i++) kr[0][i] = read_k(i);
        in_order();
        each<BATCHES>([&](auto n_) {
            constexpr int n = n_.value, from_j = LOADS * n / BATCHES, to_j = LOADS * (n + 1) / BATCHES;
#pragma unroll
            for (int i = 0; i < KB; i++)
                if (n + 1 < BATCHES) kr[(n + 1) & 1][i] = read_k((n + 1) * KB + i);
            in_order();
            each<KB / 2>([&](auto i_) {
                constexpr int i = 2 * i_.value;
                s = T::mfma32(kr[n & 1][i], qf[n * KB + i], s);
                s1 = T::mfma32(kr[n & 1][i + 1], qf[n * KB + i + 1], s1);
                in_order();
                if constexpr (from_j + i_.value < to_j) {
                    if (more) load(std::integral_constant<int, from_j + i_.value>{}, nx);
                    in_order();
                }
            });
        });
        s = (s + s1) * a.scale2;
        if (edge_at(t0, have_now)) {
            const unsigned long long vis = (attended(t0) & group_rows(have_now)) >> (r0 + 4 * half);
#pragma unroll
            for (int j = 0; j < 16; j++) s[j] = vis >> (8 * (j >> 2) + (j & 3)) & 1 ? s[j] : NINF;
        }
        return s;
    };
    auto largest = [&](const f16v &s) __attribute__((always_inline)) {
        float x = s[0];
#pragma unroll
        for (int j = 1; j < 16; j++) x = fmaxf(x, s[j]);
        return max32(x);
    };
    /* The maximum that probabilities are taken against is the first step's, common to the two waves of
     * a column; they may exceed 1 by 2^14, which costs no accuracy in either 16-bit type. Where a
     * later score exceeds it by more, the rows are gone through for the maxima alone and then once
     * more: the sums are never rescaled. (The compiler keeps them in registers that only the matrix
     * unit can work on; scaling them inside the loop took 128 more, and the loop spilled.) Returns
     * whether that happened. */
    constexpr float ROOM = 14.0f;
    auto attend = [&]() __attribute__((always_inline)) {
        bool again = false;
        begin();
        for (int t0 = lo, buf = 0; t0 < hi; t0 += L_ROWS, buf ^= 1) {
            uint8_t *tl = lds[buf], *nx = lds[buf ^ 1];
            ahead(t0);
            const f16v s = scores(t0, tl, nx);
            if (some_at(t0) && __syncthreads_or(odd_now)) {
                /* an infinity or NaN among rows that some columns do not attend would reach them as
                 * 0 * inf: the scores are done with the rows, so it is taken out of LDS and added at
                 * the end to the columns that attend it */
                odd_any = true;
                for (int i = threadIdx.x; i < L_TILE / 4; i += L_THREADS) {
                    unsigned *p = (unsigned *)tl + i;
                    *p = T::clean(*p);
                }
                __syncthreads();
            }
            const float mx = largest(s);
            float ms = m == NINF ? 0.0f : m;
            if (half == 0) lds_m[wt][32 * wc + lc] = mx;
            if (__any(mx > m + ROOM)) {   /* 1: a column without a maximum yet has one; 2: no room above a maximum */
                const int grow = __any(mx > m + ROOM && m != NINF) ? 3 : 1;
                if (lane == 0) atomicOr(&lds_grow, grow);
            }
            v8 pf[2][2];
            auto weigh = [&]() __attribute__((always_inline)) {
                float x[16], sum = 0.0f;
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    x[j] = exp2_hw(s[j] - ms);
                    sum += x[j];
                }
#pragma unroll
                for (int g = 0; g < 2; g++) {
                    const u4 w = {T::pack(x[8 * g], x[8 * g + 1]), T::pack(x[8 * g + 2], x[8 * g + 3]),
                                  T::pack(x[8 * g + 4], x[8 * g + 5]), T::pack(x[8 * g + 6], x[8 * g + 7])};
                    lds_p[wc][wt][g][lane] = w;
                }
                return sum;
            };
            float sum = weigh();
            __syncthreads();
            const int grow = lds_grow;
            if (grow) {
                again = again || (grow & 2);   /* and on: leaving the loop here costs 256 register moves a step */
                if (m == NINF) m = fmaxf(lds_m[0][32 * wc + lc], lds_m[1][32 * wc + lc]);
                ms = m == NINF ? 0.0f : m;
                sum = weigh();
                __syncthreads();
                if (threadIdx.x == 0) lds_grow = 0;
            }
            l += sum;
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int g = 0; g < 2; g++) pf[h][g] = __builtin_bit_cast(v8, lds_p[wc][h][g][lane]);
            v8 vr8[2][4];
            auto read_v = [&](int i, int g) __attribute__((always_inline)) {
                const u2 x = read_tr(tl + (v_at[0] ^ 64 * (i & 1)) + 1024 * (i >> 1) + g * (2048 * L_CHUNKS));
                const u2 y = read_tr(tl + (v_at[1] ^ 64 * (i & 1)) + 1024 * (i >> 1) + g * (2048 * L_CHUNKS));
                return __builtin_bit_cast(v8, (u4){x[0], x[1], y[0], y[1]});
            };
#pragma unroll
            for (int i = 0; i < 4; i++) vr8[0][i] = read_v(i, 0);
            in_order();
#pragma unroll
            for (int n = 0; n < DT; n++) {   /* four tiles of the latent at a time, the rows' groups outside */
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (n + 1 < DT) vr8[(n + 1) & 1][i] = read_v(((n + 1) & 1) * 4 + i, (n + 1) >> 1);
                in_order();
#pragma unroll
                for (int i = 0; i < 4; i++)
                    acc[(n & 1) * 4 + i] = T::mfma32(vr8[n & 1][i], pf[n >> 2][n >> 1 & 1], acc[(n & 1) * 4 + i]);
                in_order();
            }
            finish(t0, nx);
        }
        return again;
    };
    for (int pass = 0; pass < 2; pass++) {
        l = 0.0f;
        odd_any = false;
#pragma unroll
        for (int i = 0; i < DT; i++)
#pragma unroll
            for (int j = 0; j < 16; j++) acc[i][j] = 0.0f;
        if (!attend() || pass) break;
        start();
        begin();
        for (int t0 = lo, buf = 0; t0 < hi; t0 += L_ROWS, buf ^= 1) {
            ahead(t0);
            m = fmaxf(m, largest(scores(t0, lds[buf], lds[buf ^ 1])));
            finish(t0, lds[buf ^ 1]);
        }
        if (half == 0) lds_m[wt][32 * wc + lc] = m;
        __syncthreads();
        m = fmaxf(lds_m[0][32 * wc + lc], lds_m[1][32 * wc + lc]);
        __syncthreads();
        start();
    }

    /* the pair's sums of probabilities; each wave has its half of the latent whole */
    l = sum32(l);
    if (half == 0) lds_m[wt][32 * wc + lc] = l;
    __syncthreads();
    const float L = lds_m[0][32 * wc + lc] + lds_m[1][32 * wc + lc];
    const int64_t row = (int64_t)(q.q0 + tok) * a.heads + head;
    const bool direct = n_sp == 1;
    /* The sums go out by rows, through the steps' LDS (column c's 16-byte unit u at u ^ c mod 32, so that
     * neither the columns' writes nor the rows' reads meet a bank conflict): 16 bytes a lane and row
     * straight from the registers took 8000 cycles. */
    auto unit = [&](int c, int u) __attribute__((always_inline)) { return (f4 *)lds[0] + c * (LC / 4) + (u ^ (c & 31)); };
#pragma unroll
    for (int i = 0; i < DT * 4; i++) {
        const f16v &x = acc[i >> 2];
        const int k = 4 * (i & 3);
        *unit(32 * wc + lc, 64 * wt + 2 * i + half) = (f4){x[k], x[k + 1], x[k + 2], x[k + 3]};
    }
    if (odd_any) {   /* what was taken out of LDS above, added to this wave's half of its columns' latents */
#pragma unroll 1
        for (int t = max(lo, full / L_ROWS * L_ROWS); t < hi; t++) {
            const int id = word_of(pages, t >> a.b.page_shift);
            if (!page_ok(a.b, id) || !(attended(t) & 1)) continue;
            const uint8_t *rp = a.k.data + (int64_t)id * a.k.page_stride + (int64_t)(t & rmask) * (LW * (MX ? 1 : 2));
            const uint8_t *sc = MX ? a.k.scales + (int64_t)id * a.k.scale_page_stride + (t & rmask) * (LW / MX_BLOCK) : nullptr;
#pragma unroll 1
            for (int e = 0; e < 128; e++) {
                const int u = 64 * wt + 2 * (e >> 2) + half;
                const unsigned v = row_elem<T, MX>(rp, sc, 4 * u + (e & 3));
                if (T::odd(v)) ((float *)unit(32 * wc + lc, u))[e & 3] += T::wide(v);
            }
        }
    }
    float *lds_l = (float *)lds_p;
    if (wt == 0 && half == 0) lds_l[32 * wc + lc] = L;
    __syncthreads();
    for (int r = wave; r < L_COLS; r += L_WAVES) {   /* a row a wave at a time */
        const int rc = tile * L_COLS + r;
        if (rc >= cols) break;
        const int rt = rc / a.heads, rh = rc % a.heads;
        const float Lr = lds_l[r];
        if (direct) {
            const float f = Lr == 0.0f ? 0.0f : 1.0f / Lr;
            const f4 x = *unit(r, 2 * lane) * f, y = *unit(r, 2 * lane + 1) * f;
            *(u4_any *)(a.out + (int64_t)(q.q0 + rt) * a.ot + (int64_t)rh * a.oh + 16 * lane) =
                (u4){T::pack(x[0], x[1]), T::pack(x[2], x[3]), T::pack(y[0], y[1]), T::pack(y[2], y[3])};
        } else if (!(Lr == 0.0f)) {
            f4 *po = (f4 *)(a.part + (((int64_t)(q.q0 + rt) * a.heads + rh) * a.n_splits + sp) * LC);
            po[lane] = *unit(r, lane);
            po[64 + lane] = *unit(r, 64 + lane);
        }
    }
    if (half || wt || !on) return;
    if (direct) {
        if (a.lse) a.lse[row] = L == 0.0f ? NINF : (m + __log2f(L)) * 0.69314718055994531f;
    } else {
        float *ml = a.part + (int64_t)a.b.n_tokens * a.heads * a.n_splits * LC + (row * a.n_splits + sp) * 2;
        ml[0] = m;
        ml[1] = L;
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
