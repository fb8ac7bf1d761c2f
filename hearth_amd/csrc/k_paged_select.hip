/*
 * k_paged_select.hip — which blocks of a paged cache a query is to look at: bounds of each block's
 * keys, scores of the blocks from them, the best of each token.
 *
 * For a block of rows the least and the greatest value of every key element, lo_d and hi_d, bound
 * the score of all its rows: q . k <= sum_d max(q_d lo_d, q_d hi_d) = q+ . hi + q- . lo, with q's
 * positive and negative parts. Bounds and queries are rounded to whole numbers of up to 127 steps of
 * a power of two, one step for a block and one for a query head, which makes the sum two 8-bit matrix
 * products, exact in 32 bits (at most 127 * 127 * 256 < 2^24, so that its float32 is exact too): the
 * order of the blocks does not depend on how the sums are split, and ties go to the lowest block.
 */
#include "hx_paged.h"

#include <algorithm>

namespace hxp {

namespace {

typedef int i4 __attribute__((ext_vector_type(4)));

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
 * hold rows of the call's tokens, taken over all of their rows that exist. */
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
 * S = B Q^T: rows are blocks, a matrix instruction takes 16, columns (token, head) pairs of a kv head's group,
 * 16 a workgroup (TPT tokens of up to 16 heads, or one token of more, 16 heads at a time from LDS). A lane
 * ends with four blocks of one column; the maximum over a token's columns goes through LDS. */
constexpr int SCORE_WAVES = 4, MAX_CHUNKS = 8;

template <class T, int D, bool ONE>
__global__ __launch_bounds__(64 * SCORE_WAVES) void k_block_scores(SelectArgs a) {
    constexpr int KS = D / 64;
    constexpr float NINF = -__builtin_huge_valf();
    struct Cols { i4 up[KS], down[KS]; int byte; };
    __shared__ __align__(16) float lds_s[SCORE_WAVES][16][20];
    __shared__ __align__(16) i4 lds_q[ONE ? 1 : MAX_CHUNKS][ONE ? 1 : 2 * KS][ONE ? 1 : 64];
    __shared__ int lds_b[ONE ? 1 : MAX_CHUNKS][16];

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4, lc = lane & 15;
    int bx = blockIdx.x;
    const int chunk = bx % a.n_chunks;
    bx /= a.n_chunks;
    const int h = bx % a.kv_heads, tile = bx / a.kv_heads;
    const int seq = blockIdx.z;
    const Seq q = seq_of(a.b, seq);
    const int n = min(q.n, a.b.max_q), cols = ONE ? a.group : 16, tpt = ONE ? 16 / a.group : 1, t0 = tile * tpt;
    if (t0 >= n) return;
    const int64_t last = min((int64_t)q.base + min(t0 + tpt, n) - 1, (int64_t)q.kv - 1);   /* the last token's last row */
    if (last < 0) return;
    const int nb = (int)(last >> a.s.block_shift) + 1;
    const int lo = chunk * a.chunk, hi = min(nb, lo + a.chunk);
    if (lo >= hi) return;

    /* lane's column of heads h0 .. */
    auto quantise = [&](int tl, int head, bool on) {
        Cols c;
        const int tok = on ? t0 + tl : 0;
        const uint8_t *p = a.q + (int64_t)(q.q0 + tok) * a.qt + (int64_t)(h * a.group + head) * a.qh;
        float v[KS][16];
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < KS; i++)
#pragma unroll
            for (int z = 0; z < 2; z++) {
                u4 w = {0, 0, 0, 0};
                if (on) w = *(const u4_any *)(p + 2 * (64 * i + 16 * g + 8 * z));
                const typename T::v8 x = __builtin_bit_cast(typename T::v8, w);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    v[i][8 * z + j] = finite_or_0((float)x[j]);
                    m = fmaxf(m, __builtin_fabsf(v[i][8 * z + j]));
                }
            }
        m = max16(max32(m));
        c.byte = step_byte(m);
        const float r = per_step(c.byte);
#pragma unroll
        for (int i = 0; i < KS; i++)
#pragma unroll
            for (int z = 0; z < 4; z++) {
                unsigned up = 0, down = 0;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int x = (int)rintf(v[i][4 * z + j] * r);
                    up |= (unsigned)max(x, 0) << (8 * j);
                    down |= ((unsigned)min(x, 0) & 255u) << (8 * j);
                }
                c.up[i][z] = (int)up;
                c.down[i][z] = (int)down;
            }
        return c;
    };
    Cols mine;
    const int chunks = (a.group + 15) / 16;
    if constexpr (ONE) {
        const int tl = lc / cols;
        mine = quantise(tl, lc % cols, tl < tpt && t0 + tl < n);
    } else {
        for (int c = wave; c < chunks; c += SCORE_WAVES) {
            const int head = 16 * c + lc;
            const Cols x = quantise(0, min(head, a.group - 1), true);   /* heads past the group: the last once more */
#pragma unroll
            for (int i = 0; i < KS; i++) { lds_q[c][i][lane] = x.up[i]; lds_q[c][KS + i][lane] = x.down[i]; }
            if (g == 0) lds_b[c][lc] = x.byte;
        }
        __syncthreads();
    }

    const int *pages = a.b.pages + (int64_t)seq * a.b.ld_pages;
    const int per_page = a.b.page_shift - a.s.block_shift;
    for (int b0 = lo + 16 * wave; b0 < hi; b0 += 16 * SCORE_WAVES) {
        const int blk = b0 + lc;
        int page = blk < hi ? pages[blk >> per_page] : -1;
        const bool there = page_ok(a.b, page);
        page = there ? page : 0;
        const int sub = blk & (a.s.blocks - 1);
        const uint8_t *p = a.s.codes + (int64_t)page * a.s.page_stride + (int64_t)h * a.s.head_stride + (int64_t)sub * (2 * D) + 16 * g;
        i4 low[KS], high[KS];
#pragma unroll
        for (int i = 0; i < KS; i++) { low[i] = *(const i4 *)(p + 64 * i); high[i] = *(const i4 *)(p + D + 64 * i); }
        const int eb = there ? (int)a.s.scales[(int64_t)page * a.s.scale_page_stride + (int64_t)h * a.s.scale_head_stride + sub] : -1;
        int e[4];
#pragma unroll
        for (int j = 0; j < 4; j++) e[j] = __shfl(eb, 4 * g + j);
        f4 s = {NINF, NINF, NINF, NINF};
        auto take = [&](const i4 (&up)[KS], const i4 (&down)[KS], int byte) {
            i4 acc = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < KS; i++) {
                acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(high[i], up[i], acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(low[i], down[i], acc, 0, 0, 0);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) s[j] = fmaxf(s[j], __builtin_ldexpf((float)acc[j], e[j] + byte - 254));
        };
        if constexpr (ONE) take(mine.up, mine.down, mine.byte);
        else
            for (int c = 0; c < chunks; c++) {
                i4 up[KS], down[KS];
#pragma unroll
                for (int i = 0; i < KS; i++) { up[i] = lds_q[c][i][lane]; down[i] = lds_q[c][KS + i][lane]; }
                take(up, down, lds_b[c][lc]);
            }
        *(f4 *)&lds_s[wave][lc][4 * g] = s;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        for (int o = lane; o < 16 * tpt; o += 64) {
            const int tl = o >> 4, b = o & 15;
            if (t0 + tl >= n || b0 + b >= hi) continue;
            float m = lds_s[wave][tl * cols][b];
            for (int c = 1; c < cols; c++) m = fmaxf(m, lds_s[wave][tl * cols + c][b]);
            /* -infinity tells a block whose page is not there; an overflow stays above it */
            m = eb < 0 ? NINF : fmaxf(m, -3.4028234e38f);   /* b is lc: this lane's block */
            a.score[((int64_t)(q.q0 + t0 + tl) * a.kv_heads + h) * a.ld_score + b0 + b] = m;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

/* ---------------------------------------------------------------- the best of a token
 *
 * A workgroup takes one token and kv head. Keys are the scores' bits in an order of unsigned numbers, the
 * greatest for blocks that are kept in any case, 0 for those that cannot be taken. The top-th greatest key is found
 * eight bits at a time by counting; then every wave counts what it takes of its quarter of the blocks
 * (keys above, and of those equal the first ones) and writes it behind the quarters before. */
constexpr int PICK_THREADS = 256;

__global__ __launch_bounds__(PICK_THREADS) void k_block_pick(SelectArgs a) {
    __shared__ unsigned bins[256];
    __shared__ unsigned found[2];                        /* bin, keys above it */
    __shared__ int above[4], equal[4];
    const int h = blockIdx.x % a.kv_heads, tok = blockIdx.x / a.kv_heads, seq = blockIdx.z;
    const Seq q = seq_of(a.b, seq);
    if (tok >= min(q.n, a.b.max_q)) return;
    const int64_t row = min((int64_t)q.base + tok, (int64_t)q.kv - 1);
    const int n = row < 0 ? 0 : (int)(row >> a.s.block_shift) + 1;
    int kept = max(n - a.last, 0);                       /* blocks from here on are kept */
    if (a.b.mask) kept = min(kept, max(q.base, 0) >> a.s.block_shift);
    const float *score = a.score + ((int64_t)(q.q0 + tok) * a.kv_heads + h) * a.ld_score;
    auto key = [&](int i) -> unsigned {
        const float s = score[i];
        if (s == -__builtin_huge_valf()) return 0u;
        if (i < a.first || i >= kept) return ~0u;
        const unsigned u = __float_as_uint(s);
        return u & 0x80000000u ? ~u : u | 0x80000000u;
    };
    unsigned limit = 0;          /* keys above it are taken, and `ties` of those equal to it */
    int ties = 0;
    if (n > a.top) {
        unsigned prefix = 0, mask = 0;
        int left = a.top;        /* to be taken of the keys with the prefix */
        for (int shift = 24; shift >= 0; shift -= 8) {
            bins[threadIdx.x] = 0;
            __syncthreads();
            for (int i = threadIdx.x; i < n; i += PICK_THREADS) {
                const unsigned k = key(i);
                if ((k & mask) == prefix) atomicAdd(&bins[k >> shift & 255u], 1u);
            }
            __syncthreads();
            if (threadIdx.x < 64) {   /* four bins a lane, the greatest first */
                const int l = threadIdx.x;
                unsigned c[4], sum = 0;
#pragma unroll
                for (int j = 0; j < 4; j++) { c[j] = bins[255 - 4 * l - j]; sum += c[j]; }
                unsigned upto = sum;
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) {
                    const unsigned x = __shfl_up(upto, d);
                    if (l >= d) upto += x;
                }
                unsigned before = upto - sum;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if (before < (unsigned)left && before + c[j] >= (unsigned)left) { found[0] = 255 - 4 * l - j; found[1] = before; }
                    before += c[j];
                }
            }
            __syncthreads();
            prefix |= found[0] << shift;
            mask |= 255u << shift;
            left -= (int)found[1];
            __syncthreads();
        }
        limit = prefix;
        ties = limit ? left : 0;   /* keys of 0 are not taken */
    }
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int per = (n + 3) / 4, from = min(wave * per, n), to = min(from + per, n);
    int na = 0, ne = 0;
    for (int i = from; i < to; i += 64) {
        const unsigned k = i + lane < to ? key(i + lane) : 0u;
        na += __popcll(__ballot(k > limit));
        ne += __popcll(__ballot(k == limit && k && i + lane < to));
    }
    if (lane == 0) { above[wave] = na; equal[wave] = ne; }
    __syncthreads();
    int *out = a.chosen + (int64_t)(q.q0 + tok) * a.ct + (int64_t)h * a.ch;
    int at = 0, eq = 0, total = 0;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        if (w < wave) { at += above[w]; eq += equal[w]; }
        total += above[w];
    }
    total += min(ties, equal[0] + equal[1] + equal[2] + equal[3]);
    const unsigned long long before = (1ull << lane) - 1;
    for (int i = from; i < to; i += 64) {
        const unsigned k = i + lane < to ? key(i + lane) : 0u;
        const unsigned long long ma = __ballot(k > limit), me = __ballot(k == limit && k && i + lane < to);
        const int e = eq + __popcll(me & before);
        const bool take = k > limit || ((me >> lane & 1) && e < ties);
        if (take) out[at + __popcll(ma & before) + min(e, ties)] = i + lane;
        at += __popcll(ma);
        eq += __popcll(me);
    }
    for (int i = total + (int)threadIdx.x; i < a.top; i += PICK_THREADS) out[i] = -1;
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
    const int tiles = a.group <= 16 ? (a.b.max_q + 16 / a.group - 1) / (16 / a.group) : a.b.max_q;
    const dim3 grid((unsigned)((int64_t)tiles * a.n_chunks * a.kv_heads), 1, a.b.n_seqs), block(64 * SCORE_WAVES);
    if (a.group <= 16) hipLaunchKernelGGL((k_block_scores<T, D, true>), grid, block, 0, st, a);
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

/* Blocks are shared out among workgroups until two are there for each unit, 64 at least each (16 a wave) */
void select_blocks(SelectArgs a, int q_dtype, int width, int n_blocks, hipStream_t st) {
    const int tpt = a.group <= 16 ? 16 / a.group : 1;
    const int64_t wgs = (int64_t)a.b.n_seqs * a.kv_heads * ((a.b.max_q + tpt - 1) / tpt);
    const int64_t want = std::max<int64_t>(1, 512 / wgs);
    a.chunk = (int)(((n_blocks + want - 1) / want + 63) / 64 * 64);
    a.n_chunks = (n_blocks + a.chunk - 1) / a.chunk;
    if (q_dtype == DT_BF16) width == 64 ? scores_t<Bf16, 64>(a, st) : width == 128 ? scores_t<Bf16, 128>(a, st) : scores_t<Bf16, 256>(a, st);
    else width == 64 ? scores_t<F16, 64>(a, st) : width == 128 ? scores_t<F16, 128>(a, st) : scores_t<F16, 256>(a, st);
    hipLaunchKernelGGL(k_block_pick, dim3((unsigned)((int64_t)a.b.max_q * a.kv_heads), 1, a.b.n_seqs), dim3(PICK_THREADS), 0, st, a);
}

} // namespace hxp
