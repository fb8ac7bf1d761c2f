/*
 * k_paged_select.hip — which blocks of a paged cache a query is to look at: bounds of each block's
 * keys, scores of the blocks from them, the best of each token.
 *
 * For a block of rows the least and the greatest value of every key element, lo_d and hi_d, bound
 * the score of all its rows: q . k <= sum_d max(q_d lo_d, q_d hi_d) = q+ . hi + q- . lo, with q's
 * positive and negative parts. Bounds and queries are rounded to whole numbers of up to 127 steps of
 * a power of two, one step for a block and one for a query head, which makes the sum two 8-bit matrix
 * products, exact in 32 bits (at most 127 * 127 * 256 < 2^24, so that its float32 is exact too, and
 * the product with the steps but past float32's range at either end): the order of the blocks does
 * not depend on how the sums are split, and ties go to the lowest block.
 */
#include "hx_paged.h"

#include <algorithm>

namespace hxp {

namespace {

typedef int i4 __attribute__((ext_vector_type(4)));
typedef unsigned short us2 __attribute__((ext_vector_type(2)));

/* The step of whole numbers up to 127 for magnitudes up to m, as exponent + 127: the least with m <= 127 *
 * 2^e = 1.984375 * 2^(e + 6) */
__device__ __forceinline__ int step_byte(float m) {
    const int bits = (int)__float_as_uint(m);
    return max((bits >> 23) - 6 + ((bits & 0x7fffff) > 0x7e0000), 1);
}
/* 1 / step */
__device__ __forceinline__ float per_step(int byte) { return __uint_as_float((unsigned)(254 - byte) << 23); }

__device__ __forceinline__ float finite_or_0(float x) { return __builtin_fabsf(x) < __builtin_huge_valf() ? x : 0.0f; }

/* eight stored elements from element `el` on of a head's rows in a page (data, sc) */
template <int DT>
__device__ __forceinline__ void load8(const uint8_t *data, const uint8_t *sc, int el, float (&v)[8]) {
    if constexpr (DT == DT_MX4) {
        const unsigned c = *(const unsigned *)(data + el / 2);
        const float s = mx_scale(sc[el / MX_BLOCK]);
        each<4>([&](auto j) {
            const f2 x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, j);
            v[2 * j] = x[0]; v[2 * j + 1] = x[1];
        });
    } else if constexpr (DT == DT_MX8) {
        const u2 c = *(const u2 *)(data + el);
        const float s = mx_scale(sc[el / MX_BLOCK]);
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[j], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[j], true);
            v[4 * j] = lo[0] * s; v[4 * j + 1] = lo[1] * s; v[4 * j + 2] = hi[0] * s; v[4 * j + 3] = hi[1] * s;
        }
    } else {
        using T = std::conditional_t<DT == DT_BF16, Bf16, F16>;
        const typename T::v8 x = *(const typename T::v8 *)(data + 2 * el);
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = (float)x[j];
    }
}

/* ---------------------------------------------------------------- bounds
 *
 * A workgroup takes one block and head: D / 8 threads a row, eight elements each, 2048 / D rows at
 * once; the rows' minima and maxima meet across lanes and then through LDS. The blocks are those that
 * hold rows of the call's tokens, taken over all of their rows that exist. One block of 64 rows (16 KiB of
 * 16-bit ones) is a chain of latencies: length, page, rows, LDS, 4.3 us and a launch's own 2; the blocks of a
 * prompt run side by side. */
constexpr int BOUND_THREADS = 256;

template <int DT, int D>
__global__ __launch_bounds__(BOUND_THREADS) void k_key_bounds(BoundsArgs a) {
    constexpr int TPR = D / 8, ROWS = BOUND_THREADS / TPR, WAVES = BOUND_THREADS / 64;
    __shared__ float ends[WAVES][2][D];
    __shared__ float tops[WAVES];
    const int h = blockIdx.x % a.heads, z = blockIdx.x / a.heads;
    const Seq q = seq_of(a.b, blockIdx.z);
    const int from = max(q.base, 0), to = min((int64_t)q.base + min(q.n, a.b.max_q), (int64_t)q.kv);
    const int64_t blk = (int64_t)(from >> a.s.block_shift) + z;
    const int64_t row0 = blk << a.s.block_shift;
    if (from >= to || row0 >= to) return;
    const int page = word_of(a.b.pages, (int64_t)blockIdx.z * a.b.ld_pages + (row0 >> a.b.page_shift));
    if (!page_ok(a.b, page)) return;
    const int in_page = (int)(row0 & ((1 << a.b.page_shift) - 1)), rows = min(1 << a.s.block_shift, q.kv - (int)row0);
    const uint8_t *data = a.k.data + (int64_t)page * a.k.page_stride + (int64_t)h * a.k.head_stride;
    const uint8_t *sc = bits_of(DT) == 16 ? nullptr : a.k.scales + (int64_t)page * a.k.scale_page_stride + (int64_t)h * a.k.scale_head_stride;

    const int e = threadIdx.x % TPR * 8, r0 = threadIdx.x / TPR;
    float lo[8], hi[8];
#pragma unroll
    for (int j = 0; j < 8; j++) { lo[j] = __builtin_huge_valf(); hi[j] = -__builtin_huge_valf(); }
#pragma unroll 4
    for (int r = r0; r < rows; r += ROWS) {
        float v[8];
        load8<DT>(data, sc, (in_page + r) * D + e, v);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            v[j] = finite_or_0(v[j]);
            lo[j] = fminf(lo[j], v[j]);
            hi[j] = fmaxf(hi[j], v[j]);
        }
    }
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
    for (int d = TPR; d < 64; d <<= 1)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            lo[j] = fminf(lo[j], __shfl_xor(lo[j], d));
            hi[j] = fmaxf(hi[j], __shfl_xor(hi[j], d));
        }
    if (lane < TPR)
#pragma unroll
        for (int j = 0; j < 8; j++) { ends[wave][0][e + j] = lo[j]; ends[wave][1][e + j] = hi[j]; }
    __syncthreads();
    /* thread t: element t */
    const int t = threadIdx.x;
    float l = 0.0f, u = 0.0f;
    if (t < D) {
        l = ends[0][0][t]; u = ends[0][1][t];
#pragma unroll
        for (int w = 1; w < WAVES; w++) { l = fminf(l, ends[w][0][t]); u = fmaxf(u, ends[w][1][t]); }
    }
    float m = fmaxf(__builtin_fabsf(l), __builtin_fabsf(u));
#pragma unroll
    for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    if (lane == 0) tops[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    static_assert(WAVES == 4);
    const int byte = step_byte(m);
    const int sub = (int)blk & (a.s.blocks - 1);
    if (t < D) {
        uint8_t *out = a.s.codes + (int64_t)page * a.s.page_stride + (int64_t)h * a.s.head_stride + (int64_t)sub * (2 * D) + t;
        out[0] = (uint8_t)(int)rintf(l * per_step(byte));
        out[D] = (uint8_t)(int)rintf(u * per_step(byte));
    }
    if (t == 0) a.s.scales[(int64_t)page * a.s.scale_page_stride + (int64_t)h * a.s.scale_head_stride + sub] = (uint8_t)byte;
}

/* ---------------------------------------------------------------- scores
 *
 * S = Q B^T, 16 rows a workgroup: the (token, head) pairs of one kv head, each token's heads padded to a power of two P
 * (the last once more, which changes no maximum), so 16 / P tokens, or one token of more than 16 heads, 16 at a time from
 * LDS. Columns are blocks, 16 a matrix instruction: a lane ends with four rows of one block, whose maximum over a
 * token's heads is taken in its registers and with the lanes 16 and 32 further. A wave's instructions bound
 * it (rows and columns the other way round, with the maximum between neighbouring lanes, took 21 us for 600 tokens
 * over 313 blocks, k_block_scores_many takes 12.7); one token over 2048 blocks, 4.9 us, waits for latencies. */
constexpr int SCORE_WAVES = 4, MAX_CHUNKS = 8;

/* heads of a token in a tile of 16 rows */
__host__ __device__ inline int padded(int group) { return group > 8 ? 16 : group > 4 ? 8 : group > 2 ? 4 : group; }

/* Sixteen rows of queries as whole numbers: a lane's row lc, 16 elements of each 64 (from 16 g on), positive
 * and negative parts, and the step */
template <int KS> struct Rows16 { i4 up[KS], down[KS]; int byte; };

/* p: a lane's row. v * r + 3 * 2^22 rounds v / step to nearest even into the low byte of the float's bits (two's
 * complement, |v| * r <= 127). */
template <class T, int KS>
__device__ __forceinline__ Rows16<KS> quantise(const uint8_t *p, int g, bool on) {
    Rows16<KS> c;
    u4 w[KS][2];
#pragma unroll
    for (int i = 0; i < KS; i++)
#pragma unroll
        for (int z = 0; z < 2; z++) {
            w[i][z] = (u4){0, 0, 0, 0};
            if (on) w[i][z] = *(const u4_any *)(p + 2 * (64 * i + 16 * g + 8 * z));
        }
    /* magnitudes of 16-bit floats order like their bits: two at once */
    us2 top = {0, 0};
    auto largest = [&] {
        top = (us2){0, 0};
#pragma unroll
        for (int i = 0; i < KS; i++)
#pragma unroll
            for (int z = 0; z < 8; z++) top = __builtin_elementwise_max(top, __builtin_bit_cast(us2, w[i][z >> 2][z & 3] & 0x7fff7fffu));
    };
    largest();
    constexpr unsigned short INF = std::is_same_v<T, Bf16> ? 0x7f80 : 0x7c00;
    if (__any(top[0] >= INF || top[1] >= INF)) {
#pragma unroll
        for (int i = 0; i < KS; i++)
#pragma unroll
            for (int z = 0; z < 8; z++) w[i][z >> 2][z & 3] = T::clean(w[i][z >> 2][z & 3]);
        largest();
    }
    const float m = max16(max32(T::wide(max(top[0], top[1]))));
    c.byte = step_byte(m);
    const float r = per_step(c.byte);
#pragma unroll
    for (int i = 0; i < KS; i++)
#pragma unroll
        for (int z = 0; z < 4; z++) {
            unsigned b[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const unsigned x = w[i][z >> 1][2 * (z & 1) + (j >> 1)];
                const float v = T::wide(j & 1 ? x >> 16 : x);
                b[j] = __float_as_uint(__builtin_fmaf(v, r, 12582912.0f));
            }
            const unsigned lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu), x = lo | hi;
            const unsigned sign = x >> 7 & 0x01010101u, below = (sign << 8) - sign;   /* 255 in the bytes below 0 */
            c.up[i][z] = (int)(x & ~below);
            c.down[i][z] = (int)(x & below);
        }
    return c;
}

/* What becomes of a lane's four rows (rows 4 g .. of tokens of `pad` heads each) of one block: the token's
 * maxima into `out`, the first token's place of this block. -infinity tells a block whose page is not there; an
 * overflow stays above it. */
struct Put {
    float *out;
    int64_t ld_tok;
    int pad, left;      /* tokens from the lane's first one on */
    bool writes;
    __device__ __forceinline__ Put(const SelectArgs &a, const Seq &q, int h, int pad, int t0, int n, int g) : pad(pad) {
        const int tl = 4 * g / pad, each_g = pad <= 4 ? 1 : pad / 4;
        ld_tok = (int64_t)a.kv_heads * a.ld_score;
        out = a.score + (int64_t)(q.q0 + t0 + tl) * ld_tok + (int64_t)h * a.ld_score;
        left = n - t0 - tl;
        writes = g % each_g == 0 && left > 0;
    }
    __device__ __forceinline__ void operator()(int blk, bool there, bool inside, const float (&s)[4]) const {
        auto put = [&](int t, float x) __attribute__((always_inline)) {
            if (inside) out[t * ld_tok + blk] = there ? fmaxf(x, -3.4028234e38f) : -__builtin_huge_valf();
        };
        if (pad >= 4) {
            float m = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
            if (pad >= 8) m = max16(m);
            if (pad == 16) m = max32(m);
            if (writes) put(0, m);
        } else if (writes) {
            if (pad == 2) {
                put(0, fmaxf(s[0], s[1]));
                if (left > 1) put(1, fmaxf(s[2], s[3]));
            } else
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (left > j) put(j, s[j]);
        }
    }
};

/* 16 rows against 16 blocks; step: of the lane's four rows, byte: of its block */
template <int KS>
__device__ __forceinline__ void score16(const i4 (&up)[KS], const i4 (&down)[KS], const i4 (&high)[KS], const i4 (&low)[KS], const int (&step)[4], int byte,
                                        float (&s)[4]) {
    i4 acc = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < KS; i++) {
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(up[i], high[i], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(down[i], low[i], acc, 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < 4; j++) s[j] = __builtin_ldexpf((float)acc[j], byte + step[j] - 254);
}

template <class T, int D, bool ONE>
__global__ __launch_bounds__(64 * SCORE_WAVES) void k_block_scores(SelectArgs a) {
    constexpr int KS = D / 64;
    __shared__ __align__(16) i4 lds_q[ONE ? 1 : MAX_CHUNKS][ONE ? 1 : 2 * KS][ONE ? 1 : 64];
    __shared__ int lds_b[ONE ? 1 : MAX_CHUNKS][16];

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4, lc = lane & 15;
    int bx = blockIdx.x;
    const int chunk = bx % a.n_chunks;
    bx /= a.n_chunks;
    const int h = bx % a.kv_heads, tile = bx / a.kv_heads;
    const int seq = blockIdx.z;
    const Seq q = seq_of(a.b, seq);
    const int n = min(q.n, a.b.max_q), pad = ONE ? padded(a.group) : 16, tpt = 16 / pad, t0 = tile * tpt;
    if (t0 >= n) return;
    const int64_t last = min((int64_t)q.base + min(t0 + tpt, n) - 1, (int64_t)q.kv - 1);   /* the last token's last row */
    if (last < 0) return;
    const int nb = (int)(last >> a.s.block_shift) + 1;
    const int lo = chunk * a.chunk, hi = min(nb, lo + a.chunk);
    if (lo >= hi) return;

    const int *pages = a.b.pages + (int64_t)seq * a.b.ld_pages;
    const int per_page = a.b.page_shift - a.s.block_shift;
    constexpr int STEP = 16 * SCORE_WAVES;
    const int first = lo + 16 * wave;
    /* page of this lane's block of the sixteen from b0 on (-1: none); its bounds */
    auto page_of = [&](int b0) __attribute__((always_inline)) { return b0 + lc < hi ? pages[(b0 + lc) >> per_page] : -1; };
    struct Codes { i4 low[KS], high[KS]; int byte; } next;
    const uint8_t *codes = a.s.codes + (int64_t)h * a.s.head_stride, *scales = a.s.scales + (int64_t)h * a.s.scale_head_stride;
    auto load = [&](int b0, int id) __attribute__((always_inline)) {
        const bool there = page_ok(a.b, id);
        const int64_t page = there ? id : 0;
        const int sub = (b0 + lc) & (a.s.blocks - 1);
        const uint8_t *p = codes + page * a.s.page_stride + sub * (2 * D) + 16 * g;
#pragma unroll
        for (int i = 0; i < KS; i++) { next.low[i] = *(const i4 *)(p + 64 * i); next.high[i] = *(const i4 *)(p + D + 64 * i); }
        const int byte = scales[page * a.s.scale_page_stride + sub];
        next.byte = there ? byte : -1;
    };
    const int id0 = page_of(first), id1 = page_of(first + STEP);

    Rows16<KS> mine;
    const uint8_t *qp = a.q + (int64_t)(q.q0 + t0) * a.qt + (int64_t)(h * a.group) * a.qh;
    const int chunks = (a.group + 15) / 16;
    if constexpr (ONE) {
        const int tl = lc / pad;
        const bool on = t0 + tl < n;
        mine = quantise<T, KS>(qp + (on ? tl : 0) * a.qt + min(lc % pad, a.group - 1) * a.qh, g, on);
    } else {
        for (int c = wave; c < chunks; c += SCORE_WAVES) {
            const Rows16<KS> x = quantise<T, KS>(qp + min(16 * c + lc, a.group - 1) * a.qh, g, true);
#pragma unroll
            for (int i = 0; i < KS; i++) { lds_q[c][i][lane] = x.up[i]; lds_q[c][KS + i][lane] = x.down[i]; }
            if (g == 0) lds_b[c][lc] = x.byte;
        }
        __syncthreads();
    }
    if (first < hi) load(first, id0);
    int id = id1;
    int eq[4];
#pragma unroll
    for (int j = 0; j < 4; j++) eq[j] = ONE ? __shfl(mine.byte, 4 * g + j) : 0;
    const Put put(a, q, h, pad, t0, n, g);
    /* a step's bounds are sent for a step ahead, its page ids two */
    for (int b0 = first; b0 < hi; b0 += STEP) {
        const Codes now = next;
        if (b0 + STEP < hi) load(b0 + STEP, id);
        id = page_of(b0 + 2 * STEP);
        float s[4];
        if constexpr (ONE) score16<KS>(mine.up, mine.down, now.high, now.low, eq, now.byte, s);
        else
            for (int c = 0; c < chunks; c++) {
                i4 up[KS], down[KS];
                int step[4];
                float x[4];
#pragma unroll
                for (int i = 0; i < KS; i++) { up[i] = lds_q[c][i][lane]; down[i] = lds_q[c][KS + i][lane]; }
#pragma unroll
                for (int j = 0; j < 4; j++) step[j] = lds_b[c][4 * g + j];
                score16<KS>(up, down, now.high, now.low, step, now.byte, x);
#pragma unroll
                for (int j = 0; j < 4; j++) s[j] = c ? fmaxf(s[j], x[j]) : x[j];
            }
        put(b0 + lc, now.byte >= 0, b0 + lc < hi, s);
    }
}

/* Many tokens: four waves with 16 rows each share the bounds of 64 blocks a step, which come in by whole rows of
 * codes (16 lanes a row of width 128) and through LDS: read by each wave for itself, 16 bytes of a row a lane, they
 * were bound by the cache lines that a load touches (600 tokens over 313 blocks: 20 us, so 12.7). Pieces of 16 bytes are
 * exchanged by row, so that 16 lanes that read one piece of 16 rows meet no bank conflict. The next step's
 * are in flight meanwhile (two buffers). */
template <class T, int D>
__global__ __launch_bounds__(64 * SCORE_WAVES) void k_block_scores_many(SelectArgs a) {
    constexpr int KS = D / 64, PIECES = D / 8, STEP = 16 * SCORE_WAVES, RI = 64 / PIECES, N = 16 / RI;   /* pieces of a row, rows a load instruction, instructions */
    __shared__ __align__(16) u4 lds[2][STEP * PIECES];
    __shared__ int lds_b[2][STEP];

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4, lc = lane & 15;
    int bx = blockIdx.x;
    const int chunk = bx % a.n_chunks;
    bx /= a.n_chunks;
    const int h = bx % a.kv_heads, tile = bx / a.kv_heads;
    const int seq = blockIdx.z;
    const Seq q = seq_of(a.b, seq);
    const int n = min(q.n, a.b.max_q), pad = padded(a.group), tpt = 16 / pad, first = tile * tpt * SCORE_WAVES, t0 = first + tpt * wave;
    if (first >= n) return;
    const int64_t last = min((int64_t)q.base + min(first + tpt * SCORE_WAVES, n) - 1, (int64_t)q.kv - 1);   /* the last token's last row */
    if (last < 0) return;
    const int nb = (int)(last >> a.s.block_shift) + 1;
    const int lo = chunk * a.chunk, hi = min(nb, lo + a.chunk);
    if (lo >= hi) return;

    const int *pages = a.b.pages + (int64_t)seq * a.b.ld_pages;
    const int per_page = a.b.page_shift - a.s.block_shift;
    /* lanes 0 to 15 look up the pages of the wave's 16 blocks of a step; each load takes its row's from them */
    auto page_of = [&](int b0) __attribute__((always_inline)) {
        const int blk = b0 + 16 * wave + lc;
        const int id = blk < hi ? pages[blk >> per_page] : -1;
        return page_ok(a.b, id) ? id : -1;
    };
    const uint8_t *codes = a.s.codes + (int64_t)h * a.s.head_stride, *scales = a.s.scales + (int64_t)h * a.s.scale_head_stride;
    const int row = lane / PIECES, piece = lane % PIECES;
    u4 w[N];
    int byte;
    auto load = [&](int b0, int id) __attribute__((always_inline)) {
#pragma unroll
        for (int z = 0; z < N; z++) {
            const int r = z * RI + row;
            const int64_t page = max(__shfl(id, r), 0);
            const int sub = (b0 + 16 * wave + r) & (a.s.blocks - 1);
            w[z] = *(const u4 *)(codes + page * a.s.page_stride + sub * (2 * D) + 16 * piece);
        }
        const int sub = (b0 + 16 * wave + lc) & (a.s.blocks - 1);
        const int x = scales[(int64_t)max(id, 0) * a.s.scale_page_stride + sub];
        byte = id >= 0 ? x : -1;
    };
    auto at = [](int r, int p) { return r * PIECES + (D == 64 ? p ^ (r >> 1 & 7) : p ^ (r & 15)); };
    auto settle = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int z = 0; z < N; z++) lds[buf][at(16 * wave + z * RI + row, piece)] = w[z];
        if (g == 0) lds_b[buf][16 * wave + lc] = byte;
    };
    int id = page_of(lo);
    load(lo, id);
    id = page_of(lo + STEP);
    const int tl = lc / pad;
    const bool on = t0 + tl < n;
    const Rows16<KS> mine = quantise<T, KS>(a.q + (int64_t)(q.q0 + (on ? t0 + tl : first)) * a.qt + (int64_t)(h * a.group + min(lc % pad, a.group - 1)) * a.qh, g, on);
    int eq[4];
#pragma unroll
    for (int j = 0; j < 4; j++) eq[j] = __shfl(mine.byte, 4 * g + j);
    const Put put(a, q, h, pad, t0, n, g);
    settle(0);
    __syncthreads();
    int buf = 0;
    for (int b0 = lo; b0 < hi; b0 += STEP, buf ^= 1) {
        const bool more = b0 + STEP < hi;
        if (more) load(b0 + STEP, id);
        id = page_of(b0 + 2 * STEP);
#pragma unroll
        for (int u = 0; u < SCORE_WAVES; u++) {
            const int r = 16 * u + lc;
            i4 low[KS], high[KS];
#pragma unroll
            for (int i = 0; i < KS; i++) {
                low[i] = __builtin_bit_cast(i4, lds[buf][at(r, 4 * i + g)]);
                high[i] = __builtin_bit_cast(i4, lds[buf][at(r, PIECES / 2 + 4 * i + g)]);
            }
            const int eb = lds_b[buf][r];
            float s[4];
            score16<KS>(mine.up, mine.down, high, low, eq, eb, s);
            put(b0 + r, eb >= 0, b0 + r < hi, s);
        }
        if (more) settle(buf ^ 1);
        __syncthreads();
    }
}

/* f over all lanes, in every lane: lanes ^ 1, ^ 2, the halves of 8 and of 16 turned round, lanes ^ 16, ^ 32 */
template <class F>
__device__ __forceinline__ unsigned over_wave(unsigned x, F f) {
    auto with = [&](auto ctrl) __attribute__((always_inline)) { x = f(x, (unsigned)__builtin_amdgcn_update_dpp((int)x, (int)x, ctrl.value, 0xF, 0xF, false)); };
    with(std::integral_constant<int, 0xB1>{});
    with(std::integral_constant<int, 0x4E>{});
    with(std::integral_constant<int, 0x141>{});
    with(std::integral_constant<int, 0x140>{});
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = f(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return f(b[0], b[1]);
}
/* the sum of the lanes up to this one: within 16 lanes by shifts of 1, 2, 4, 8, then lane 15's to the row behind it
 * and lane 31's to the upper half */
__device__ __forceinline__ unsigned sum_upto(unsigned x) {
    auto with = [&](auto ctrl, auto rows) __attribute__((always_inline)) { x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, ctrl.value, rows.value, 0xF, false); };
    using std::integral_constant;
    with(integral_constant<int, 0x111>{}, integral_constant<int, 0xF>{});
    with(integral_constant<int, 0x112>{}, integral_constant<int, 0xF>{});
    with(integral_constant<int, 0x114>{}, integral_constant<int, 0xF>{});
    with(integral_constant<int, 0x118>{}, integral_constant<int, 0xF>{});
    with(integral_constant<int, 0x142>{}, integral_constant<int, 0xA>{});
    with(integral_constant<int, 0x143>{}, integral_constant<int, 0xC>{});
    return x;
}

/* ---------------------------------------------------------------- the best of a token
 *
 * W waves take one token and kv head, each its share of the blocks, in order: four waves, or one where the keys of all
 * blocks fit its registers, which then waits for no other (2400 rows of 313 blocks: 7.4 us, four waves 9.4). Keys are the
 * scores' bits in an order of unsigned numbers, the greatest for blocks that are kept in any case, 0 for those that
 * cannot be taken. Keys of one row lie close together, so the top-th greatest is looked for within their range: 256
 * bins over it, then over the bin that holds it, until the bin is taken whole or holds one value (two rounds in most rows).
 * Then every wave counts what it takes (keys above, and of those equal the first ones) and writes it behind
 * the waves before. R: keys of a lane that stay in registers (0: they are read again each time). */
constexpr int PICK_THREADS = 256, PICK_ALONE = 8;   /* keys of a lane of one wave */

template <int R, int W>
__global__ __launch_bounds__(PICK_THREADS) void k_block_pick(SelectArgs a) {
    constexpr int ROWS = PICK_THREADS / 64 / W;      /* of a workgroup */
    static_assert(W == 1 || ROWS == 1);
    __shared__ unsigned lds_bins[ROWS][2][256];
    __shared__ unsigned lds_lo[W], lds_hi[W];
    __shared__ int lds_can[W], lds_kept[W], above[W], equal[W];
    const int wave = W == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int mine_of = W == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0, id = W == 1 ? lane : threadIdx.x;
    auto meet = [] {
        if constexpr (W == 1) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        else __syncthreads();
    };
    unsigned (*bins)[256] = lds_bins[mine_of];
    const int unit = blockIdx.x * ROWS + mine_of, seq = blockIdx.z;
    const int h = unit % a.kv_heads, tok = unit / a.kv_heads;
    const Seq q = seq_of(a.b, seq);
    if (tok >= min(q.n, a.b.max_q)) return;          /* the row's waves alike */
    const int64_t row = min((int64_t)q.base + tok, (int64_t)q.kv - 1);
    const int n = row < 0 ? 0 : (int)(row >> a.s.block_shift) + 1;
    int tail = max(n - a.last, 0);                       /* blocks from here on are kept */
    if (a.b.mask) tail = min(tail, max(q.base, 0) >> a.s.block_shift);
    const float *score = a.score + ((int64_t)(q.q0 + tok) * a.kv_heads + h) * a.ld_score;
    const int per = (n + W - 1) / W, from = min(wave * per, n), to = min(from + per, n);
    auto fetch = [&](int i) __attribute__((always_inline)) -> unsigned {   /* of block from + i of the wave */
        if (from + i >= to) return 0u;
        const float s = score[from + i];
        const unsigned u = s == 0.0f ? 0u : __float_as_uint(s);   /* a sum below 0 times steps whose product underflows is -0, which is no less than 0 */
        if (s == -__builtin_huge_valf()) return 0u;
        return from + i < a.first || from + i >= tail ? ~0u : u & 0x80000000u ? ~u : u | 0x80000000u;
    };
    unsigned mine[R ? R : 1];
    if constexpr (R != 0) {
#pragma unroll
        for (int i = 0; i < R; i++) mine[i] = fetch(64 * i + lane);
    }
    auto keys = [&](auto f) __attribute__((always_inline)) {   /* f(index in the wave's share, key), 64 lanes at once */
        if constexpr (R != 0) {
#pragma unroll
            for (int i = 0; i < R; i++) f(64 * i, mine[i]);
        } else
            for (int i = 0; from + i < to; i += 64) f(i, fetch(i + lane));
    };
    for (int i = id; i < 2 * 256; i += 64 * W) bins[i >> 8][i & 255] = 0;
    unsigned lo = ~0u, hi = 0;
    int can = 0, kept = 0;
    keys([&](int, unsigned k) {
        can += __popcll(__ballot(k != 0));
        kept += __popcll(__ballot(k == ~0u));
        if (k && k != ~0u) { lo = min(lo, k); hi = max(hi, k); }
    });
    lo = over_wave(lo, [](unsigned x, unsigned y) { return min(x, y); });
    hi = over_wave(hi, [](unsigned x, unsigned y) { return max(x, y); });
    if constexpr (W > 1) {
        if (lane == 0) { lds_lo[wave] = lo; lds_hi[wave] = hi; lds_can[wave] = can; lds_kept[wave] = kept; }
        can = kept = 0;
        meet();
#pragma unroll
        for (int w = 0; w < W; w++) {
            lo = min(lo, lds_lo[w]);
            hi = max(hi, lds_hi[w]);
            can += lds_can[w];
            kept += lds_kept[w];
        }
    } else meet();
    unsigned limit = 0;          /* keys above it are taken, and `ties` of those equal to it */
    int ties = 0, left = a.top - kept;   /* to be taken within [lo, hi] */
    if (can > a.top) {
        if (left <= 0) limit = ~0u - 1;
        else
            for (int z = 0; z < 4; z++) {   /* shifts of up to 24, 16, 8 and 0: the fourth round ends it */
                const int round = z & 1;
                const int shift = max(24 - __builtin_clz(hi - lo | 1u), 0);   /* (hi - lo) >> shift < 256 */
                keys([&](int, unsigned k) {
                    if (k >= lo && k <= hi) atomicAdd(&bins[round][(k - lo) >> shift], 1u);
                });
                meet();
                /* every wave alike: four bins a lane, the greatest first */
                unsigned c[4], sum = 0;
#pragma unroll
                for (int j = 0; j < 4; j++) { c[j] = bins[round][255 - 4 * lane - j]; sum += c[j]; }
                const unsigned upto = sum_upto(sum);
                unsigned before = upto - sum, bin = 0, over = 0, in = 0;
                bool here = false;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if (before < (unsigned)left && before + c[j] >= (unsigned)left) { here = true; bin = 255 - 4 * lane - j; over = before; in = c[j]; }
                    before += c[j];
                }
                const int who = __ffsll((long long)__ballot(here)) - 1;
                bin = (unsigned)__builtin_amdgcn_readlane((int)bin, who);
                left -= __builtin_amdgcn_readlane((int)over, who);
                in = (unsigned)__builtin_amdgcn_readlane((int)in, who);
                lo += bin << shift;
                if (in == (unsigned)left) { limit = lo - 1; break; }
                if (shift == 0) { limit = lo; ties = left; break; }
                hi = lo + min(hi - lo, (1u << shift) - 1);   /* lo + 2^24 may pass 32 bits */
                /* the other set of bins is clear; this one is for the round after the next */
                meet();
                for (int i = id; i < 256; i += 64 * W) bins[round][i] = 0;
            }
    }
    int na = 0, ne = 0;
    keys([&](int, unsigned k) {
        na += __popcll(__ballot(k > limit));
        ne += __popcll(__ballot(k == limit && k));
    });
    int *out = a.chosen + (int64_t)(q.q0 + tok) * a.ct + (int64_t)h * a.ch;
    int at = 0, eq = 0, total = na, same = ne;
    if constexpr (W > 1) {
        if (lane == 0) { above[wave] = na; equal[wave] = ne; }
        meet();
        total = same = 0;
#pragma unroll
        for (int w = 0; w < W; w++) {
            if (w < wave) { at += above[w]; eq += equal[w]; }
            total += above[w];
            same += equal[w];
        }
    }
    total += min(ties, same);
    const unsigned long long before = (1ull << lane) - 1;
    keys([&](int i, unsigned k) {
        const unsigned long long ma = __ballot(k > limit), me = __ballot(k == limit && k);
        const int e = eq + __popcll(me & before);
        if (k > limit || (k == limit && k && e < ties)) out[at + __popcll(ma & before) + min(e, ties)] = from + i + lane;
        at += __popcll(ma);
        eq += __popcll(me);
    });
    for (int i = total + id; i < a.top; i += 64 * W) out[i] = -1;
}

template <int DT>
void bounds_t(const BoundsArgs &a, int width, hipStream_t st) {
    const dim3 grid((unsigned)(a.per_seq * a.heads), 1, a.b.n_seqs), block(BOUND_THREADS);
    if (width == 64) hipLaunchKernelGGL((k_key_bounds<DT, 64>), grid, block, 0, st, a);
    else if (width == 128) hipLaunchKernelGGL((k_key_bounds<DT, 128>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((k_key_bounds<DT, 256>), grid, block, 0, st, a);
}

template <class T, int D>
void scores_t(const SelectArgs &a, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)a.tiles * a.n_chunks * a.kv_heads), 1, a.b.n_seqs), block(64 * SCORE_WAVES);
    if (a.many) hipLaunchKernelGGL((k_block_scores_many<T, D>), grid, block, 0, st, a);
    else if (a.group <= 16) hipLaunchKernelGGL((k_block_scores<T, D, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((k_block_scores<T, D, false>), grid, block, 0, st, a);
}

} // namespace

void key_bounds(const BoundsArgs &a, int cache_dtype, int width, hipStream_t st) {
    if (cache_dtype == DT_F16) bounds_t<DT_F16>(a, width, st);
    else if (cache_dtype == DT_BF16) bounds_t<DT_BF16>(a, width, st);
    else if (cache_dtype == DT_MX8) bounds_t<DT_MX8>(a, width, st);
    else bounds_t<DT_MX4>(a, width, st);
}

int select_group_limit() { return 16 * MAX_CHUNKS; }

/* Blocks are shared out among workgroups until four are there for each unit, 64 at least each (16 a wave; 600
 * tokens over 313 blocks: 12.7 us, with two 15). Tokens that fill the rows of four waves share their blocks'
 * bounds. */
void score_split(SelectArgs &a) {
    int tpt = a.group <= 16 ? 16 / padded(a.group) : 1;
    a.many = a.group <= 16 && a.b.max_q >= SCORE_WAVES * tpt;
    if (a.many) tpt *= SCORE_WAVES;
    a.tiles = (a.b.max_q + tpt - 1) / tpt;
    const int64_t wgs = (int64_t)a.b.n_seqs * a.kv_heads * a.tiles;
    const int64_t want = std::max<int64_t>(1, 1024 / wgs);
    a.chunk = (int)std::max<int64_t>(((a.ld_score + want - 1) / want + 63) / 64 * 64, 64);   /* no blocks: no shares */
    a.n_chunks = (int)((a.ld_score + a.chunk - 1) / a.chunk);
}

void select_blocks(const SelectArgs &a, int q_dtype, int width, hipStream_t st) {
    if (a.n_chunks) {
        if (q_dtype == DT_BF16) width == 64 ? scores_t<Bf16, 64>(a, st) : width == 128 ? scores_t<Bf16, 128>(a, st) : scores_t<Bf16, 256>(a, st);
        else width == 64 ? scores_t<F16, 64>(a, st) : width == 128 ? scores_t<F16, 128>(a, st) : scores_t<F16, 256>(a, st);
    }
    const int64_t n_blocks = a.ld_score;
    const int64_t rows = (int64_t)a.b.max_q * a.kv_heads;
    const bool alone = n_blocks <= 64 * PICK_ALONE;
    const dim3 grid((unsigned)(alone ? (rows + 3) / 4 : rows), 1, a.b.n_seqs), threads(PICK_THREADS);
    if (alone) hipLaunchKernelGGL((k_block_pick<PICK_ALONE, 1>), grid, threads, 0, st, a);
    else if (n_blocks <= 8 * PICK_THREADS) hipLaunchKernelGGL((k_block_pick<8, 4>), grid, threads, 0, st, a);
    else if (n_blocks <= 32 * PICK_THREADS) hipLaunchKernelGGL((k_block_pick<32, 4>), grid, threads, 0, st, a);
    else hipLaunchKernelGGL((k_block_pick<0, 4>), grid, threads, 0, st, a);
}

} // namespace hxp
