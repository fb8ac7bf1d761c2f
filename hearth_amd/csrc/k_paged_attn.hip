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
 * goes through LDS (no row is read by two waves) but the keys of blocks that many tokens choose (BY_LDS),
 * V is under way before the scores and the next K before the sums (32 tokens over 8-bit rows with each
 * load where it is used: 114 us, not 48). Rows of 4 bits: one token over 131071 rows, 71 MB in 17.3 us (4.1
 * TB/s); 32 tokens up to 8192 rows, 92 MB in 25 us (3.7 TB/s), wait for the longest sequences: the split goes by
 * the longest, so that 388 of 512 workgroups have rows, up to 2048 where an equal share is 1314. A wave takes
 * about 500 vector instructions for 64 rows (139 of them conversions), four cycles each: 7 and 8 us of
 * the two, spread evenly.
 * Chosen blocks: 32 tokens over 32 blocks of 64 16-bit rows each 27.7 us (134 MB, 4.8 TB/s), 600
 * tokens over 16 blocks of 8-bit rows each 60 (from the chip's caches). The latter is bound by vector
 * instructions, 22.5 M: 22000 a SIMD are 37 us at 4 cycles each. 5.2 M of them are conversions; the others
 * are the softmax, for 16 columns of which 8 are in use with 8 heads a kv head, scale bytes taken out
 * row by row, V's byte permutations, masks and addresses.
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

constexpr int FEW_WAVES = 4;
/* Tiles of 16 cache rows that a wave takes at a time. Rows of 4 bits: twice as many, or too few bytes are under way */
constexpr int few_tiles(int bits) { return bits == 4 ? 4 : 2; }

__device__ __forceinline__ unsigned lo16(unsigned a, unsigned b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ unsigned hi16(unsigned a, unsigned b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

template <class T, int BITS, int D>
struct Few {
    using v8 = typename T::v8;
    static constexpr bool MX = BITS < 16;
    static constexpr int NT = few_tiles(BITS), STEP = 16 * NT;
    static constexpr int KS = D / 32;                    /* matrix steps of the score */
    static constexpr int BD = D < 128 ? D : 128;        /* elements of a V block: 16 lanes x PL */
    static constexpr int NB = D / BD, PL = BD / 16;      /* blocks; elements of a row a lane takes */
    static constexpr int RB = D * BITS / 8;               /* bytes of a row */

    /* Score: the four lanes of a row take LB bytes each a load, LE elements, SL matrix steps */
    static constexpr int LB = RB / 4 < 16 ? RB / 4 : 16, KL = RB / (4 * LB), LE = LB * 8 / BITS, SL = LE / 8;
    static constexpr int VB = PL * BITS / 8;              /* bytes of a row and block for the sum */
    static constexpr int VW = VB < 4 ? 1 : VB / 4;
    static constexpr int SW = D / 32 < 4 ? 1 : D / 128;   /* words that hold a row's scales */

    struct K { unsigned w[NT][KL][LB / 4]; unsigned s[NT][SW]; };             /* a lane's row of each tile of 16 */
    struct V { unsigned w[NB][4 * NT][VW]; unsigned s[NT][D / 32]; };   /* four rows of each tile; their scales */

    /* first element that a lane multiplies in matrix step i */
    static __device__ __forceinline__ int at(int i, int g) { return 4 * LE * (i / SL) + LE * g + 8 * (i % SL); }

    /* BYTES at p (a multiple of 16, 8, 4 or 2) */
    template <int BYTES> static __device__ __forceinline__ void words(const uint8_t *p, unsigned *w) {
        if constexpr (BYTES == 16) {
            const u4 x = *(const u4 *)p;
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = x[i];
        } else if constexpr (BYTES == 8) {
            const u2 x = *(const u2 *)p;
            w[0] = x[0]; w[1] = x[1];
        } else if constexpr (BYTES == 4) w[0] = *(const unsigned *)p;
        else w[0] = *(const unsigned short *)p;
    }
    /* rows, sc: a tile's first row and its scales, the same for the wave; a lane's bytes from there on are a 32-bit
     * offset, so that no load needs an address of its own */
    static __device__ __forceinline__ void load_k(K &k, int u, const uint8_t *rows, int g, int lc) {
        const unsigned at = lc * RB + LB * g;
#pragma unroll
        for (int i = 0; i < KL; i++) words<LB>(rows + at + 4 * LB * i, k.w[u][i]);
    }
    static __device__ __forceinline__ void load_ks(K &k, int u, const uint8_t *sc, int lc) {
        if constexpr (MX) {
            const uint8_t *q = sc + (unsigned)(lc * (D / MX_BLOCK));
            if constexpr (D == 64) k.s[u][0] = *(const ushort_any *)q;
            else
#pragma unroll
                for (int i = 0; i < SW; i++) k.s[u][i] = ((const unsigned_any *)q)[i];
        }
    }
    /* K by way of LDS: 64 lanes bring in 1 KiB of whole rows an instruction, where 16 lanes that read 16 bytes
     * of 16 rows each touch 16 cache lines. The 16-byte pieces of a row are exchanged by row, so that those 16
     * lanes meet 16 different columns of the 256 bytes of banks. */
    static constexpr int P = RB / 16, RI = 1024 / RB, N = STEP * RB / 1024;   /* pieces of a row, rows an instruction, instructions */
    static __device__ __forceinline__ int swz(int r) { return P >= 16 ? r & 15 : r / (16 / P) & (P - 1); }
    /* z: instruction; rows: the first of its rows */
    static __device__ __forceinline__ void send_k(uint8_t *lds, int z, const uint8_t *rows, int lane) {
        const int r = lane / P;
        const unsigned at = r * RB + ((lane % P) ^ swz((z * RI + r) & 15)) * 16;
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(rows + at), (__attribute__((address_space(3))) void *)(lds + 1024 * z), 16, 0, 0);
    }
    static __device__ __forceinline__ void read_k(K &k, const uint8_t *lds, int g, int lc) {
#pragma unroll
        for (int u = 0; u < NT; u++)
#pragma unroll
            for (int i = 0; i < KL; i++) {
                const int byte = 4 * LB * i + LB * g;
                words<LB>(lds + (16 * u + lc) * RB + ((byte / 16) ^ swz(lc)) * 16 + byte % 16, k.w[u][i]);
            }
    }
    static __device__ __forceinline__ void load_v(V &v, int u, const uint8_t *rows, const uint8_t *sc, int g, int lc) {
        const unsigned at = 4 * g * RB + lc * VB;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int j = 0; j < 4; j++) words<VB>(rows + at + (j * RB + b * BD * BITS / 8), v.w[b][4 * u + j]);
        if constexpr (MX) {   /* four rows' scales lie side by side */
            const uint8_t *q = sc + (unsigned)(4 * g * (D / MX_BLOCK));
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
    /* scores of the tiles' rows; the tiles take turns, since an instruction that adds to the one before waits for it */
    static __device__ __forceinline__ void scores(const K &k, int g, const v8 (&q)[KS], f4 (&s)[NT]) {
#pragma unroll
        for (int u = 0; u < NT; u++) s[u] = (f4){0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < KL; i++)
#pragma unroll
            for (int h = 0; h < SL; h++)
#pragma unroll
                for (int u = 0; u < NT; u++) {
                    const unsigned *x = k.w[u][i];
                    u4 w;
                    if constexpr (MX) {
                        /* block LE i / 8 + LE g / 32, which does not leave the word */
                        const float f = mx_scale_at(k.s[u][LE * i / 32], 8 * (LE * i / 8 % 4) + 8 * (LE * g / 32));
                        if constexpr (BITS == 4)
                            w = (u4){T::template from_mx4<0>(x[h], f), T::template from_mx4<1>(x[h], f), T::template from_mx4<2>(x[h], f),
                                     T::template from_mx4<3>(x[h], f)};
                        else
                            w = (u4){T::template from_mx8<false>(x[2 * h], f), T::template from_mx8<true>(x[2 * h], f),
                                     T::template from_mx8<false>(x[2 * h + 1], f), T::template from_mx8<true>(x[2 * h + 1], f)};
                    } else w = (u4){x[0], x[1], x[2], x[3]};
                    s[u] = T::mfma16(__builtin_bit_cast(v8, w), q[SL * i + h], s[u]);
                }
    }
    /* The softmax of a lane's scores x in base 2, against the running maximum m: x become the probabilities,
     * packed into pf, l their sum; sums and l are rescaled where a maximum has grown by more than GROWTH. */
    template <int GROWTH>
    static __device__ __forceinline__ void weights(float (&x)[4 * NT], v8 (&pf)[NT / 2], f4 (&acc)[NB * PL], float &m, float &l) {
        float mx = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
#pragma unroll
        for (int j = 8; j < 4 * NT; j += 4) mx = fmaxf(mx, fmaxf(fmaxf(x[j], x[j + 1]), fmaxf(x[j + 2], x[j + 3])));
        mx = max16(max32(mx));
        if (__any(mx > m + (float)GROWTH)) {
            mx = fmaxf(m, mx);
            const float al = exp2_hw(m - (mx == -__builtin_huge_valf() ? 0.0f : mx));
            l *= al;
#pragma unroll
            for (int i = 0; i < NB * PL; i++) acc[i] *= al;
            m = mx;
        }
        const float ms = m == -__builtin_huge_valf() ? 0.0f : m;
#pragma unroll
        for (int j = 0; j < 4 * NT; j++) {
            x[j] = exp2_hw(x[j] - ms);
            l += x[j];
        }
#pragma unroll
        for (int k = 0; k < NT / 2; k++) {
            const float *p = x + 8 * k;
            pf[k] = __builtin_bit_cast(v8, (u4){T::pack(p[0], p[1]), T::pack(p[2], p[3]), T::pack(p[4], p[5]), T::pack(p[6], p[7])});
        }
    }
    /* acc += V^T P^T. ALL: every row counts as it is; otherwise rows for which there(tile, row of the tile) is
     * false are taken as zeros, and so are infinities and NaN, which `odd` tells of */
    template <bool ALL, class THERE>
    static __device__ __forceinline__ void add(f4 (&acc)[NB * PL], const V &v, const v8 (&pf)[NT / 2], int lc, bool &odd, THERE there) {
#pragma unroll
        for (int bk = 0; bk < NB * NT / 2; bk++) {
            const int b = bk / (NT / 2), k = bk % (NT / 2);   /* block of elements, pair of tiles */
            unsigned w[8][PL / 2];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                v_row(v, b, 8 * k + j, lc, w[j]);
                if constexpr (!ALL) {
                    const unsigned keep = there(2 * k + (j >> 2), j & 3) ? ~0u : 0u;
#pragma unroll
                    for (int i = 0; i < PL / 2; i++) {
                        w[j][i] &= keep;
                        odd = odd || T::odd(w[j][i]);
                        w[j][i] = T::clean(w[j][i]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < PL / 2; i++) {
                const u4 e = {lo16(w[0][i], w[1][i]), lo16(w[2][i], w[3][i]), lo16(w[4][i], w[5][i]), lo16(w[6][i], w[7][i])};
                const u4 o = {hi16(w[0][i], w[1][i]), hi16(w[2][i], w[3][i]), hi16(w[4][i], w[5][i]), hi16(w[6][i], w[7][i])};
                acc[b * PL + 2 * i] = T::mfma16(__builtin_bit_cast(v8, e), pf[k], acc[b * PL + 2 * i]);
                acc[b * PL + 2 * i + 1] = T::mfma16(__builtin_bit_cast(v8, o), pf[k], acc[b * PL + 2 * i + 1]);
            }
        }
    }
    /* the infinities and NaN of one row, to the columns that attend it */
    static __device__ __forceinline__ void add_odd(f4 (&acc)[NB * PL], const uint8_t *row, const uint8_t *sc, int g, bool mine) {
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int j = 0; j < PL; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const unsigned x = row_elem<T, BITS>(row, sc, b * BD + (4 * g + i) * PL + j);
                    acc[b * PL + j][i] += T::odd(x) && mine ? T::wide(x) : 0.0f;
                }
    }
    /* PL elements of row j, block b, as 16-bit pairs */
    static __device__ __forceinline__ void v_row(const V &v, int b, int j, int lc, unsigned (&w)[PL / 2]) {
        if constexpr (MX) {
            const int jj = j & 3;
            float f;
            if constexpr (D == 64) f = mx_scale_at(v.s[j >> 2][jj >> 1], 16 * (jj & 1) + 8 * (lc >> 3));
            else f = mx_scale_at(v.s[j >> 2][jj * (D / 128) + b], 8 * (lc >> 2));
            if constexpr (BITS == 4)
                each<PL / 2>([&](auto i) { w[i] = T::template from_mx4<i.value>(v.w[b][j][0], f); });
            else
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

/* BLOCKS: of the rows of chosen blocks, which stand one after the other in the place of the
 * sequence's. A workgroup's columns are then heads of one token, since every token has blocks of its own.
 * ONE: a step's rows lie in one page (and block), which is looked up once.
 * BY_LDS: K by way of LDS. Blocks that many tokens choose come from the chip's caches, where the
 * lines that K's loads touch bound the kernel (a row of 16 lanes' loads at a time from as many rows;
 * by LDS whole rows): 600 tokens over 16 blocks of 64 rows each, by LDS and straight, 16-bit rows 66 and
 * 95 us, 8-bit 62 and 77; 4-bit, whose rows are a quarter of a line's, 61 and 57. Single tokens'
 * blocks come from memory, where neither way is faster in general (32 of them over 32 blocks each, 16-bit
 * rows: 29.5 and 27.7 us once, 31.3 and 31.2 in other calls; of width 256 61 and 60). */
template <class T, int BITS, int D, bool BLOCKS, bool ONE, bool BY_LDS>
__global__ __launch_bounds__(64 * FEW_WAVES, D <= 128 ? 2 : 1) void k_attend_few(AttendArgs a) {
    using F = Few<T, BITS, D>;
    using v8 = typename T::v8;
    constexpr bool MX = F::MX;
    /* Rows of 4 bits and few rows in all have most to do beside the loads: the sums are rescaled only where a maximum
     * has grown by more than 2^8, below which the probabilities lose no accuracy in either 16-bit type. */
    constexpr int GROWTH = BITS == 4 || BLOCKS ? 8 : 0;
    constexpr int PL = F::PL, NB = F::NB, BD = F::BD, CT = 16, NT = F::NT, STEP = F::STEP;
    constexpr int PER = ONE ? NT : 1, NL = NT / PER, RUN = 16 * PER;   /* tiles of a look-up, look-ups of a step, their rows */
    __shared__ float lds_o[FEW_WAVES][16][BD + 4];
    __shared__ __align__(16) uint8_t lds_k[BY_LDS ? FEW_WAVES : 1][BY_LDS ? STEP * F::RB : 16];
    __shared__ float lds_m[FEW_WAVES][CT], lds_l[FEW_WAVES][CT];
    __shared__ unsigned lds_some[FEW_WAVES];   /* bit c: column c attends a row of the wave's */

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int g = lane >> 4, lc = lane & 15;
    int bx = blockIdx.x;
    const int sp = bx % a.n_splits;
    bx /= a.n_splits;
    const int kvh = bx % a.kv_heads;
    bx /= a.kv_heads;
    const int seq = blockIdx.z;
    const Seq q = seq_of(a.b, seq);
    const int head_tiles = (a.group + CT - 1) / CT;
    /* BLOCKS: the token, and its columns from c0 on; otherwise columns are (token, head) pairs */
    const int only = BLOCKS ? bx / head_tiles : 0, c0 = (BLOCKS ? bx % head_tiles : bx) * CT;
    if (BLOCKS && only >= min(q.n, a.b.max_q)) return;
    const int cols = BLOCKS ? a.group : min(q.n, a.b.max_q) * a.group;
    if (c0 >= cols) return;
    const int n_sp = BLOCKS ? a.n_splits : max(1, (q.kv + a.chunk - 1) / a.chunk);
    if (sp >= n_sp) return;

    /* this lane's column */
    v8 qf[F::KS];
    const int c = c0 + lc;
    const bool on = c < cols;
    const int tok = BLOCKS ? only : on ? c / a.group : 0, head = kvh * a.group + (!on ? 0 : BLOCKS ? c : c % a.group);
    /* rows it attends without a mask (causal), or rows before the call's */
    const int lim = !on ? 0 : a.b.mask ? min(q.base, q.kv) : min(q.base + tok + 1, q.kv);
    const uint8_t *qp = a.q + (int64_t)(q.q0 + tok) * a.qt + (int64_t)head * a.qh;
#pragma unroll
    for (int i = 0; i < F::KS; i++) {
        const unsigned short *p = (const unsigned short *)qp + F::at(i, g);
        u4 w = {0, 0, 0, 0};
        if (on) w = *(const u4_any *)p;
        qf[i] = __builtin_bit_cast(v8, w);
    }
    /* rows below hi some column of the tile may attend (without BLOCKS: of this split); below `full` every
     * valid column attends every row */
    const int t_first = BLOCKS ? only : c0 / a.group, t_last = BLOCKS ? only : min(cols - 1, c0 + CT - 1) / a.group;
    const int end = a.b.mask ? q.kv : min(q.kv, q.base + t_last + 1);
    const int hi = BLOCKS ? end : min(end, (sp + 1) * a.chunk);
    const int full = a.b.mask ? q.base : q.base + t_first + 1;
    const int *list = BLOCKS ? a.chosen + (int64_t)(q.q0 + only) * a.ct + (int64_t)kvh * a.ch : nullptr;
    const int stop = BLOCKS ? min(a.top << a.block_shift, (sp + 1) * a.chunk) : hi;   /* of the steps */

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

    /* RUN rows from `row` on in a page (-1: none). Every load goes to a row of the cache: rows past hi
     * lie in the same page, those of a page that is not there are taken from page 0; both are
     * masked, and cleared in V. */
    struct Run { int row, page; };
    /* in two or three steps, each of which waits for the one before: the block at t, its rows with what the page table
     * says, the page checked */
    auto block_at = [&](int t) __attribute__((always_inline)) { return BLOCKS && t < stop ? word_of(list, t >> a.block_shift) : -1; };
    auto look = [&](int t, int blk) __attribute__((always_inline)) {
        Run x = {t, -1};
        if constexpr (BLOCKS) {
            const int64_t row = ((int64_t)blk << a.block_shift) + (t & ((1 << a.block_shift) - 1));
            x.row = blk >= 0 && row < hi ? (int)row : -1;
            if (x.row >= 0) x.page = word_of(pages, x.row >> a.b.page_shift);
        } else if (t < hi) x.page = word_of(pages, t >> a.b.page_shift);
        return x;
    };
    auto checked = [&](Run x) __attribute__((always_inline)) {
        if (!page_ok(a.b, x.page)) x.page = -1;
        return x;
    };
    /* whether every valid column attends every row of a step */
    auto whole_at = [&](const Run (&x)[NL]) __attribute__((always_inline)) {
        const int below = min(full, hi);
        bool all = true;
#pragma unroll
        for (int z = 0; z < NL; z++) all = all && x[z].page >= 0 && x[z].row + RUN <= below;
        return all;
    };
    typename F::K kr;
    typename F::V vw;
    auto load_k = [&](const Run (&x)[NL]) __attribute__((always_inline)) {
        const uint8_t *rows[NL];
#pragma unroll
        for (int z = 0; z < NL; z++) {
            const int64_t i = max(x[z].page, 0), row = x[z].row & (page_rows - RUN);
            rows[z] = same_global(kbase + i * a.k.page_stride + row * F::RB);
            if constexpr (MX) {
                const uint8_t *sc = same_global(ksb + i * a.k.scale_page_stride + row * (D / MX_BLOCK));
#pragma unroll
                for (int u = 0; u < PER; u++) F::load_ks(kr, z * PER + u, sc + 16 * u * (D / MX_BLOCK), lc);
            }
        }
        if constexpr (!BY_LDS) {
#pragma unroll
            for (int u = 0; u < NT; u++) F::load_k(kr, u, rows[u / PER] + 16 * (u % PER) * F::RB, g, lc);
        } else {
#pragma unroll
            for (int z = 0; z < F::N; z++) {
                constexpr int RI = F::RI;
                const int r = z * RI;                       /* first row of the instruction's */
                static_assert(RI <= 16);                    /* of one run */
                F::send_k(lds_k[wave], z, rows[r / RUN] + (r % RUN) * F::RB, lane);
            }
        }
    };
    auto load_v = [&](const Run (&x)[NL]) __attribute__((always_inline)) {
#pragma unroll
        for (int z = 0; z < NL; z++) {
            const int64_t i = max(x[z].page, 0), row = x[z].row & (page_rows - RUN);
            const uint8_t *rows = same_global(vbase + i * a.v.page_stride + row * F::RB);
            const uint8_t *sc = MX ? same_global(vsb + i * a.v.scale_page_stride + row * (D / MX_BLOCK)) : nullptr;
#pragma unroll
            for (int u = 0; u < PER; u++) F::load_v(vw, z * PER + u, rows + 16 * u * F::RB, MX ? sc + 16 * u * (D / MX_BLOCK) : nullptr, g, lc);
        }
    };
    constexpr int ROUND = STEP * FEW_WAVES;
    const int first = sp * a.chunk + STEP * wave;
    Run now[NL], next[NL];
    int blk[NL];
#pragma unroll
    for (int z = 0; z < NL; z++) blk[z] = block_at(first + RUN * z);
#pragma unroll
    for (int z = 0; z < NL; z++) {
        next[z] = look(first + RUN * z, blk[z]);
        blk[z] = block_at(first + ROUND + RUN * z);
    }
    arrived();
#pragma unroll
    for (int z = 0; z < NL; z++) next[z] = checked(next[z]);
    if (first < stop) load_k(next);
    /* a step: V on its way before the scores, the next step's K as soon as these have taken K */
    for (int t0 = first; t0 < stop; t0 += ROUND) {
#pragma unroll
        for (int z = 0; z < NL; z++) now[z] = next[z];
        /* lists of early tokens end in entries that are none */
        bool none = BLOCKS;
#pragma unroll
        for (int z = 0; z < NL; z++) none = none && now[z].page < 0;
        if (!none) load_v(now);
#pragma unroll
        for (int z = 0; z < NL; z++) {
            next[z] = look(t0 + ROUND + RUN * z, blk[z]);
            blk[z] = block_at(t0 + 2 * ROUND + RUN * z);
        }
        in_order();
        f4 s[NT];
        if constexpr (BY_LDS) F::read_k(kr, lds_k[wave], g, lc);
        if (!none) F::scores(kr, g, qf, s);
        in_order();
#pragma unroll
        for (int z = 0; z < NL; z++) next[z] = checked(next[z]);
        if (t0 + ROUND < stop) load_k(next);
        if (none) continue;
        in_order();
        const bool whole = whole_at(now);
        v8 pf[NT / 2];
        float x[4 * NT];
#pragma unroll
        for (int j = 0; j < 4 * NT; j++) x[j] = s[j >> 2][j & 3] * a.scale2;
        if (whole) {
            some = true;
        } else {
            unsigned long long at = 0;
            if constexpr (BLOCKS && !ONE) {
#pragma unroll
                for (int z = 0; z < NL; z++) at |= now[z].page >= 0 ? (attended(now[z].row) & 0xffff) << (16 * z) : 0;
            } else {
                unsigned have = 0;
#pragma unroll
                for (int u = 0; u < NT; u++) have |= now[u / PER].page >= 0 ? 1u << u : 0u;
                at = attended(now[0].row) & group_rows(have);
            }
            const unsigned long long vis = at >> (4 * g);
            some = some || at;
#pragma unroll
            for (int j = 0; j < 4 * NT; j++) x[j] = vis >> (16 * (j >> 2) + (j & 3)) & 1 ? x[j] : -__builtin_huge_valf();
        }
        F::template weights<GROWTH>(x, pf, acc, m, l);
        /* two ways, so that the one of most steps has no branches in it */
        auto there = [&](int u, int r) { return now[u / PER].row + 16 * (u % PER) + 4 * g + r < hi && now[u / PER].page >= 0; };
        if (whole) F::template add<true>(acc, vw, pf, lc, odd, there);
        else F::template add<false>(acc, vw, pf, lc, odd, there);
    }
    /* an infinity or NaN among rows that some columns do not attend would reach them as 0 * inf:
     * left out above, added here to the columns that do attend it */
    if (__any(odd)) {
        auto run_at = [&](int t) { return checked(look(t, block_at(t))); };
        for (int t0 = first; t0 < stop; t0 += ROUND) {
            Run x[NL];
#pragma unroll
            for (int z = 0; z < NL; z++) x[z] = run_at(t0 + RUN * z);
            if (whole_at(x)) continue;   /* a step taken as it is */
#pragma unroll 1
            for (int z = 0; z < STEP; z++) {
                const Run y = run_at(t0 + (z & -RUN));
                const int id = y.page, t = y.row + (z & (RUN - 1));
                if (id < 0 || t >= hi) continue;
                const uint8_t *row = vbase + (int64_t)id * a.v.page_stride + (int64_t)(t & (page_rows - 1)) * F::RB;
                const uint8_t *sc = MX ? vsb + (int64_t)id * a.v.scale_page_stride + (t & (page_rows - 1)) * (D / MX_BLOCK) : nullptr;
                F::add_odd(acc, row, sc, g, attended(t) & 1);
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
    const int co = c0 + oc;
    const bool here = co < cols;
    const int ot = BLOCKS ? only : here ? co / a.group : 0, oh = kvh * a.group + (!here ? 0 : BLOCKS ? co : co % a.group);
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
    const int n_sp = a.top ? a.n_splits : max(1, (q.kv + a.chunk - 1) / a.chunk);
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

/* Tokens of a sequence from which on K goes by LDS (see BY_LDS). By LDS and straight, us, 8 heads a kv head:
 * one sequence, 16 blocks a token of width 128: 16 tokens 10.3 and 11.4, 128 17.4 and 24.4; 32 sequences, 32 blocks
 * a token, 4, 8, 16 tokens each: 16-bit rows of width 64 28 / 29, 40 / 53, 67 / 93, of 128 55 / 56, 75 / 90, 119 /
 * 164, of 256 107 / 111, 167 / 181, 299 / 337; 8-bit rows of 128 37 / 36, 63 / 65, 96 / 121. 8-bit rows of widths 64
 * and 256 lose by it (24 / 23, 33 / 32, 56 / 55; 88 / 87, 159 / 157, 294 / 291), one sequence of them up to 6%. */
constexpr int SHARING = 16;

template <class T, int BITS, int D, bool BLOCKS>
void few_t(const AttendArgs &a, hipStream_t st) {
    const int tiles = BLOCKS ? a.b.max_q * ((a.group + 15) / 16) : (a.b.max_q * a.group + 15) / 16;
    const dim3 grid((unsigned)a.n_splits * a.kv_heads * tiles, 1, a.b.n_seqs);
    constexpr int STEP = 16 * few_tiles(BITS);
    const bool one = 1 << a.b.page_shift >= STEP && (!BLOCKS || 1 << a.block_shift >= STEP);
    auto launch = [&](auto one, auto lds) {
        hipLaunchKernelGGL((k_attend_few<T, BITS, D, BLOCKS, one.value, lds.value>), grid, dim3(64 * FEW_WAVES), 0, st, a);
    };
    constexpr std::true_type yes;
    constexpr std::false_type no;
    if constexpr (BLOCKS && BITS > 4)
        if (one && a.b.max_q >= SHARING) return launch(yes, yes);
    if constexpr (BITS == 4 || BLOCKS)   /* of two look-ups a step one makes no difference to the others, which wait for memory */
        if (one) return launch(yes, no);
    launch(no, no);
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
/* of 4-bit rows, whose bytes are few: passes over the cache cost less than rows made 16 bits in LDS. 32 sequences of
 * 4096 rows, few and many, us at 32, 64, 96 and 128 columns: width 64 22 / 37, 31 / 39, 38 / 40, 48 / 41; 128 28 / 48,
 * 38 / 50, 54 / 54, 70 / 59; 256 62 / 134, 92 / 141, 128 / 148, 168 / 154. One sequence of 32768 (128: 16 / 22, 20 / 25,
 * 24 / 28, 28 / 30) and four of 2048 are faster by few at 128 columns too. */
static bool takes_many4(int64_t cols) { return cols > 96; }

/* Rows a split takes: enough workgroups for the 256 units, two each (one of the latent form, which fills a
 * unit; with four of few rows a unit 32 tokens over 2048 to 8192 8-bit rows took 51 us, not 45, and one over
 * 131071 16-bit rows 59, not 55: more partial sums to write and join). Few query rows are not split below 512
 * rows: one launch of 500 rows takes 10 us where a split one and its join take 12.5; at 1000 rows two splits
 * take 16 us and eight 15. Many are split down to 192 rows (85 tokens over 2132 rows: 26 us, at 128 rows 31; 64
 * over 500: 17 us, at 256 rows 20), the latent form down to 128 (1 token over 500 rows: 21 us, at 256 rows 26;
 * 1 over 8192: 30 us, at 64 rows 35). */
Split attend_split(int n_seqs, int max_q, int kv_cap, int heads, int kv_heads, bool latent, bool four) {
    const int64_t cols = (int64_t)max_q * (heads / kv_heads);
    const bool many = !latent && (four ? takes_many4(cols) : takes_many(cols));
    const int tile = latent ? 64 : many ? 128 : 16, step = latent ? 64 : 128, at_once = latent ? 256 : 512;
    const int64_t wgs = std::max<int64_t>((int64_t)n_seqs * kv_heads * ((cols + tile - 1) / tile), 1);
    const int64_t want = std::max<int64_t>(1, at_once / wgs);
    int64_t chunk = (kv_cap + want - 1) / want;
    chunk = std::max<int64_t>((chunk + step - 1) / step * step, latent ? 128 : many ? 192 : 512);
    return {(int)chunk, std::max(1, (int)((kv_cap + chunk - 1) / chunk)), many};
}

/* As attend_split; a unit is a token and 16 of a kv head's query heads */
Split blocks_split(int n_seqs, int max_q, int rows, int heads, int kv_heads) {
    const int64_t wgs = std::max<int64_t>((int64_t)n_seqs * kv_heads * max_q * ((heads / kv_heads + 15) / 16), 1);
    const int64_t want = std::max<int64_t>(1, 512 / wgs), step = 128;
    int64_t chunk = (rows + want - 1) / want;
    chunk = std::max<int64_t>((chunk + step - 1) / step * step, 512);
    return {(int)chunk, (int)((rows + chunk - 1) / chunk), false};
}

#define HXP_BY(F, T) (width == 64 ? F(T, 64) : width == 128 ? F(T, 128) : F(T, 256))
template <bool BLOCKS>
static void few(const AttendArgs &a, int q_dtype, int cache_dtype, int width, hipStream_t st) {
    const int bits = bits_of(cache_dtype);
#define HXP_FEW(T, D) (bits == 16 ? few_t<T, 16, D, BLOCKS>(a, st) : bits == 8 ? few_t<T, 8, D, BLOCKS>(a, st) : few_t<T, 4, D, BLOCKS>(a, st))
    if (q_dtype == DT_BF16) HXP_BY(HXP_FEW, Bf16);
    else HXP_BY(HXP_FEW, F16);
#undef HXP_FEW
}

static void join(const AttendArgs &a, int q_dtype, int width, hipStream_t st) {
    if (a.n_splits == 1) return;
#define HXP_JOIN(T, D) join_t<T, D>(a, st)
    if (q_dtype == DT_BF16) HXP_BY(HXP_JOIN, Bf16);
    else HXP_BY(HXP_JOIN, F16);
#undef HXP_JOIN
}
#undef HXP_BY

void attend(const AttendArgs &a, int q_dtype, int cache_dtype, int width, bool many, hipStream_t st) {
    if (many) attend_many(a, q_dtype, cache_dtype, width, st);
    else few<false>(a, q_dtype, cache_dtype, width, st);
    join(a, q_dtype, width, st);
}

void attend_blocks(const AttendArgs &a, int q_dtype, int cache_dtype, int width, hipStream_t st) {
    few<true>(a, q_dtype, cache_dtype, width, st);
    join(a, q_dtype, width, st);
}

void attend_latent(const AttendArgs &a, int q_dtype, int cache_dtype, hipStream_t st) {
    latent_rows(a, q_dtype, cache_dtype == DT_MX8, st);
    if (a.n_splits == 1) return;
    if (q_dtype == DT_BF16) join_t<Bf16, 512>(a, st);
    else join_t<F16, 512>(a, st);
}

} // namespace hxp
