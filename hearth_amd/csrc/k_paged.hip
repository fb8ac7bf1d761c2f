/*
 * k_paged.hip — rotary positions and the writes and reads of a paged cache. All three move
 * each element once and are bound by HBM for prompts and by launch latency for single tokens:
 * rotating 64 of 192 elements of 2001 tokens of 128 heads (66 MB) takes 13.9 us (4.8 TB/s, near a
 * large copy's 4.9). Rows of 4 heads of 128, keys and values: quantising three prompts of up to 4093 rows,
 * 10012 in all, into 8 bits (31 MB) 10 us, reading eight sequences of up to 4095, 22927 in all, back (71 MB)
 * 15 us (4.7 TB/s), the rows of 32 single tokens 3.2 us; with their rotation and 32 query heads' the three
 * prompts into 16-bit pages (205 MB) 40 us (5.1 TB/s), three of 9819 rows into 8 and 4 bits (191 and 186 MB) 41
 * and 40, 9819 latent rows with 16 query heads 15 us (63 MB), into 8 and 4 bits 17.
 */
#include "hx_paged.h"

#include <algorithm>
#include <type_traits>

namespace hxp {

namespace {

/* ---------------------------------------------------------------- element conversions */

template <int DT> struct Elem;
template <> struct Elem<DT_F32> {
    static constexpr int size = 4;
    static __device__ __forceinline__ void load8(const uint8_t *p, bool wide, float (&v)[8]) {
        if (wide) {
            const f4 a = ((const f4 *)p)[0], b = ((const f4 *)p)[1];
#pragma unroll
            for (int i = 0; i < 4; i++) { v[i] = a[i]; v[4 + i] = b[i]; }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = ((const float *)p)[i];
        }
    }
    static __device__ __forceinline__ void store8(uint8_t *p, bool wide, const float (&v)[8]) {
        if (wide) {
            ((f4 *)p)[0] = (f4){v[0], v[1], v[2], v[3]};
            ((f4 *)p)[1] = (f4){v[4], v[5], v[6], v[7]};
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) ((float *)p)[i] = v[i];
        }
    }
    static __device__ __forceinline__ float load(const uint8_t *p) { return *(const float *)p; }
    static __device__ __forceinline__ void store(uint8_t *p, float v) { *(float *)p = v; }
    template <bool> static __device__ __forceinline__ float rounded(float v) { return v; }
};
template <class T> struct Elem16 {
    static constexpr int size = 2;
    using e = typename T::e;
    static __device__ __forceinline__ void load8(const uint8_t *p, bool wide, float (&v)[8]) {
        if (wide) {
            const typename T::v8 x = *(const typename T::v8 *)p;
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = (float)x[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = (float)((const e *)p)[i];
        }
    }
    static __device__ __forceinline__ void store8(uint8_t *p, bool wide, const float (&v)[8]) {
        if (wide) {
            *(u4 *)p = (u4){T::pack(v[0], v[1]), T::pack(v[2], v[3]), T::pack(v[4], v[5]), T::pack(v[6], v[7])};
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) ((e *)p)[i] = (e)v[i];
        }
    }
    static __device__ __forceinline__ float load(const uint8_t *p) { return (float)*(const e *)p; }
    static __device__ __forceinline__ void store(uint8_t *p, float v) { *(e *)p = (e)v; }
    /* to float32 and then to e, as the pairs of store8 are; ALONE: as store, where the compiler may round a
     * float16's product and sum once */
    template <bool ALONE> static __device__ __forceinline__ float rounded(float v) {
        if constexpr (!ALONE) asm("" : "+v"(v));
        return (float)(e)v;
    }
};
template <> struct Elem<DT_F16> : Elem16<F16> {};
template <> struct Elem<DT_BF16> : Elem16<Bf16> {};

/* ---------------------------------------------------------------- rotary positions
 *
 * y = f (u cos a - v sin a), f (v cos a + u sin a), a = pos * freq. The angle is taken in
 * turns in float64 (pos * freq / 2 pi, less its nearest whole number: exact), so that a
 * position of 10^6 still has its fraction to 1e-10; sine and cosine of the fraction are
 * float32. One workgroup takes `TOK` tokens: cosines and sines once into LDS (n_freqs a
 * token), then all heads of both tensors, eight elements of each half a thread (16 bytes of the
 * 16-bit types). */
constexpr int ROPE_THREADS = 256;
constexpr int ROPE_GROUPS = 1 << 20;   /* at most; longer calls go round */

/* cosine and sine of pos * freq, times factor */
__device__ __forceinline__ f2 turn_of(double pos, double freq, float factor, float sign) {
    const double turns = pos * (freq * 0.15915494309189533577);
    const float r = 2.0f * (float)(turns - rint(turns));
    float s, c;
    sincospif(r, &s, &c);
    return (f2){c * factor, s * factor * sign};
}

/* nt tokens from t0 on of one tensor, their cosines and sines in cs */
template <int DT, bool HALF, bool WIDE>
__device__ __forceinline__ void rope_rows(const RopeArgs::Pair &p, int64_t t0, int nt, const f2 *cs, int n_freqs, int offset, int width, bool in_place) {
    using E = Elem<DT>;
    constexpr int S = E::size;
    /* an item is 8 elements of each half (HALF), 16 consecutive ones (interleaved), or, WIDE
     * false, one pair; then the elements outside the rotated part, one at a time */
    constexpr int PER = WIDE ? 8 : 1;
    const int items = n_freqs / PER;
    const int per_tok = p.heads * items;
    for (int i = threadIdx.x; i < nt * per_tok; i += ROPE_THREADS) {
        const int tl = i / per_tok, rem = i % per_tok, h = rem / items, j = rem % items * PER;
        const uint8_t *x = p.x + (t0 + tl) * p.xt + (int64_t)h * p.xh + offset * S;
        uint8_t *y = p.y + (t0 + tl) * p.yt + (int64_t)h * p.yh + offset * S;
        const f2 *w = cs + tl * n_freqs + j;
        if constexpr (WIDE) {
            const int o0 = HALF ? j * S : 2 * j * S, o1 = HALF ? (j + n_freqs) * S : (2 * j + 8) * S;
            float u[8], v[8], ru[8], rv[8];
            E::load8(x + o0, true, u);
            E::load8(x + o1, true, v);
            if constexpr (HALF) {
#pragma unroll
                for (int i8 = 0; i8 < 8; i8++) {
                    ru[i8] = __builtin_fmaf(u[i8], w[i8][0], -(v[i8] * w[i8][1]));
                    rv[i8] = __builtin_fmaf(v[i8], w[i8][0], u[i8] * w[i8][1]);
                }
            } else {
#pragma unroll
                for (int i4 = 0; i4 < 4; i4++) {
                    ru[2 * i4] = __builtin_fmaf(u[2 * i4], w[i4][0], -(u[2 * i4 + 1] * w[i4][1]));
                    ru[2 * i4 + 1] = __builtin_fmaf(u[2 * i4 + 1], w[i4][0], u[2 * i4] * w[i4][1]);
                    rv[2 * i4] = __builtin_fmaf(v[2 * i4], w[4 + i4][0], -(v[2 * i4 + 1] * w[4 + i4][1]));
                    rv[2 * i4 + 1] = __builtin_fmaf(v[2 * i4 + 1], w[4 + i4][0], v[2 * i4] * w[4 + i4][1]);
                }
            }
            E::store8(y + o0, true, ru);
            E::store8(y + o1, true, rv);
        } else {
            const int o0 = HALF ? j * S : 2 * j * S, o1 = HALF ? (j + n_freqs) * S : (2 * j + 1) * S;
            const float u = E::load(x + o0), v = E::load(x + o1);
            E::store(y + o0, __builtin_fmaf(u, w[0][0], -(v * w[0][1])));
            E::store(y + o1, __builtin_fmaf(v, w[0][0], u * w[0][1]));
        }
    }
    if (!in_place) {
        const int rest = width - 2 * n_freqs;
        for (int i = threadIdx.x; i < nt * p.heads * rest; i += ROPE_THREADS) {
            const int tl = i / (p.heads * rest), rem = i % (p.heads * rest), h = rem / rest;
            int d = rem % rest;
            if (d >= offset) d += 2 * n_freqs;
            const uint8_t *x = p.x + (t0 + tl) * p.xt + (int64_t)h * p.xh + (int64_t)d * S;
            uint8_t *y = p.y + (t0 + tl) * p.yt + (int64_t)h * p.yh + (int64_t)d * S;
            if constexpr (S == 4) *(unsigned *)y = *(const unsigned *)x;
            else *(unsigned short *)y = *(const unsigned short *)x;
        }
    }
}

template <int DT, bool HALF, bool WIDE>
__global__ __launch_bounds__(ROPE_THREADS) void k_rope(RopeArgs a, int tok) {
    extern __shared__ f2 cs[];   /* [tok][n_freqs] */
    for (int64_t t0 = (int64_t)blockIdx.x * tok; t0 < a.n_tokens; t0 += (int64_t)gridDim.x * tok) {
        const int nt = (int)min((int64_t)tok, a.n_tokens - t0);
        for (int i = threadIdx.x; i < nt * a.n_freqs; i += ROPE_THREADS) {
            const int64_t t = t0 + i / a.n_freqs;
            const double pos = a.pos64 ? (double)((const int64_t *)a.pos)[t] : (double)((const int *)a.pos)[t];
            cs[i] = turn_of(pos, a.freqs[i % a.n_freqs], a.factor, a.sign);
        }
        __syncthreads();
        for (int z = 0; z < a.n_pairs; z++)
            rope_rows<DT, HALF, WIDE>(a.p[z], t0, nt, cs, a.n_freqs, a.offset, a.width, a.in_place);
        __syncthreads();   /* the next tokens' cosines go where these lie */
    }
}

/* ---------------------------------------------------------------- cache writes
 *
 * A thread takes eight elements of one token, head and piece. MX8: four neighbouring lanes
 * hold a block of 32 and take its maximum with two lane exchanges; e is the least exponent
 * with amax * 2^-e <= 448 = 1.75 * 2^8, read off the bits of amax = m * 2^x: x - 8 where
 * m <= 1.75, else x - 7. Dividing by 2^e is exact; the hardware conversion rounds to nearest
 * even. Where rounding up would leave the range of the source type (its largest exponent, m
 * above 1.9375) the code is cut to 240: off by up to the step below it, 2^-4 of the value. MX4
 * alike, with amax * 2^-e <= 7 = 1.75 * 2^2: a value between 6, the largest code, and 7 rounds to 6 and
 * is off by no more than half the step of the codes above 4; at the range's end (m above 1.75) the
 * code is cut to 3, off by up to the step to 4, 2^-2 of the value. e2m1 has no NaN, so a block that holds one, or an
 * infinity, gets the scale byte 255, which the conversions back turn into NaN. Looking at every element for these took
 * 12 us for the 10012 rows of three prompts, 4 heads of 128, into 4 bits (26 MB, 5.1 us at a large copy's rate), a look at
 * the block's largest bits 9.1. */
__device__ __forceinline__ bool fin(float x) { return __builtin_fabsf(x) < __builtin_huge_valf(); }

/* over four neighbouring lanes */
__device__ __forceinline__ unsigned max_of4(unsigned m) {
    m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, true));
    return max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, true));
}

/* The eight elements that a thread of either kernel takes of each of its tokens: octs threads a
 * token (grid.z of them where that is more than a workgroup), several tokens a workgroup where it is
 * less; which piece, head and element they are is worked out once for COPY_TOKENS tokens (16 prompts of
 * up to 4093 rows, 42348 in all, of 4 heads of 128 into 8 bits: 37 us, one by one 44; eight at once 15% more
 * than four on three such prompts). The four tokens' page ids, then their rows, are under way together. */
constexpr int COPY_TOKENS = 4;
struct Place {
    const Piece *p;
    int h, d;          /* head; element in the piece's row */
    int tok, step;     /* first token, tokens a round; tok < 0: none */
};
__device__ __forceinline__ Place place_of(const CopyArgs &a) {
    Place r;
    const int per = min(a.octs, 256), tpb = 256 / per;   /* threads of a token, tokens a round of the workgroup */
    int o = threadIdx.x % per + blockIdx.z * 256;
    const int tl = threadIdx.x / per, o0 = a.p[0].heads * (a.p[0].width / 8);
    const bool second = o >= o0;
    r.p = &a.p[second ? 1 : 0];
    if (second) o -= o0;
    r.h = o / (r.p->width / 8);
    r.d = o % (r.p->width / 8) * 8;
    r.tok = tl < tpb && o + (second ? o0 : 0) < a.octs ? (int)blockIdx.x * tpb * COPY_TOKENS + tl : -1;
    r.step = tpb;
    return r;
}

/* where a token's row lies: its head's rows of a page and the row's number in it; page < 0: nowhere */
struct Spot { int page, row; };
__device__ __forceinline__ Spot spot_of(const Batch &b, const Seq &q, int tok) {
    const int pos = q.base + tok;
    if (pos < 0 || pos >= q.kv) return {-1, 0};
    const int page = b.pages[(int64_t)blockIdx.y * b.ld_pages + (pos >> b.page_shift)];
    return {page_ok(b, page) ? page : -1, pos & ((1 << b.page_shift) - 1)};
}

/* Eight values, which SRC holds, into a row of the cache. Lanes of one block of 32 come here together:
 * octs and every piece's width / 8 are multiples of 4. */
template <int SRC, int DST>
__device__ __forceinline__ void put8(const Piece &p, const Spot &at, int h, int d, const float (&v)[8]) {
    uint8_t *dst = p.rows.data + (int64_t)at.page * p.rows.page_stride + (int64_t)h * p.rows.head_stride;
    const int64_t el = (int64_t)at.row * p.row_width + p.col + d;
    if constexpr (bits_of(DST) == 16) {
        Elem<DST>::store8(dst + el * 2, true, v);
    } else {
        /* Both largest magnitudes of a scale of 1 are 1.75 * 2^TOP_E: 448, and 7 = 6 and half the step above it */
        constexpr int TOP_E = DST == DT_MX4 ? 2 : 8, FULL = (SRC == DT_F16 ? 15 : 127) + 127 + 1 - TOP_E;
        auto byte_of = [](unsigned m) { return max((int)(m >> 23) - TOP_E + ((m & 0x7fffff) > 0x600000), 1); };
        /* magnitudes of floats order like their bits, infinities and NaN above all */
        unsigned m = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
        m = max_of4(m);
        int byte = byte_of(m);
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = v[j];
        unsigned odd = 0;            /* elements whose code is NaN */
        if (__any(m >= 0x7f800000u || byte == FULL)) {   /* rare: checked element by element, otherwise none can leave the codes' range */
            const bool whole = m < 0x7f800000u;
            if constexpr (DST == DT_MX4) {
                if (!whole) byte = 255;                  /* a block of NaN */
            } else {
                unsigned f = 0;                          /* the largest of the finite ones */
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    if (!fin(v[j])) odd |= 1u << j;
                    f = max(f, fin(v[j]) ? __float_as_uint(v[j]) & 0x7fffffffu : 0u);
                }
                byte = byte_of(max_of4(f));
            }
            /* the code above these would leave the source type's range: they are off by up to the step to it */
            const float top = byte == FULL ? (DST == DT_MX4 ? 3.0f : 240.0f) * mx_scale(byte) : __builtin_huge_valf();
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = (DST == DT_MX4 ? whole : fin(v[j])) ? fminf(fmaxf(v[j], -top), top) : 0.0f;
        }
        if constexpr (DST == DT_MX4) {
            const float scale = mx_scale(byte == 255 ? 127 : byte);
            unsigned c = 0;
            each<4>([&](auto j) { c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2 * j], x[2 * j + 1], scale, j); });   /* to nearest even, above 6 to 6 */
            *(unsigned *)(dst + el / 2) = c;
        } else {
            const float inv = __uint_as_float((unsigned)(254 - byte) << 23);
            u2 c;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j] * inv, x[4 * j + 1] * inv, 0, false);
                c[j] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j + 2] * inv, x[4 * j + 3] * inv, w, true);
            }
            if (__any(odd))
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (odd >> j & 1) c[j >> 2] = (c[j >> 2] & ~(255u << (8 * (j & 3)))) | 0x7fu << (8 * (j & 3));
            *(u2 *)(dst + el) = c;
        }
        if ((d & 31) == 0)
            p.rows.scales[(int64_t)at.page * p.rows.scale_page_stride + (int64_t)h * p.rows.scale_head_stride + el / MX_BLOCK] = (uint8_t)byte;
    }
}

/* Eight elements on their way from a caller's row into the cache: as they are where the types are the same */
template <int SRC, int DST, bool WIDE>
struct Eight {
    using E = Elem<SRC>;
    u4 raw;
    float v[8];
    __device__ __forceinline__ void load(const uint8_t *src) {
        if constexpr (DST != SRC) E::load8(src, WIDE, v);
        else if constexpr (WIDE) raw = *(const u4 *)src;
        else {
            unsigned short w[8];
#pragma unroll
            for (int j = 0; j < 8; j++) w[j] = ((const unsigned short *)src)[j];
            raw = (u4){w[0] | (unsigned)w[1] << 16, w[2] | (unsigned)w[3] << 16, w[4] | (unsigned)w[5] << 16, w[6] | (unsigned)w[7] << 16};
        }
    }
    __device__ __forceinline__ void store(const Piece &p, const Spot &at, int h, int d) const {
        if constexpr (DST != SRC) put8<SRC, DST>(p, at, h, d, v);
        else
            *(u4 *)(p.rows.data + (int64_t)at.page * p.rows.page_stride + (int64_t)h * p.rows.head_stride + ((int64_t)at.row * p.row_width + p.col + d) * 2) = raw;
    }
};

template <int SRC, int DST, bool WIDE>
__device__ __forceinline__ void append_item(const CopyArgs &a, const Seq &q, const Piece &p, int tok, int h, int d) {
    const Spot at = spot_of(a.b, q, tok);
    if (at.page < 0) return;
    Eight<SRC, DST, WIDE> x;
    x.load(p.arr + (int64_t)(q.q0 + tok) * p.at + (int64_t)h * p.ah + (int64_t)d * Elem<SRC>::size);
    x.store(p, at, h, d);
}

template <int SRC, int DST, bool WIDE>
__global__ __launch_bounds__(256) void k_kv_append(CopyArgs a) {
    const Seq q = seq_of(a.b, blockIdx.y);
    const int n = min(q.n, a.b.max_q);
    const Place r = place_of(a);
    if (r.tok < 0) return;
    const Piece p = *r.p;
    const uint8_t *src = p.arr + (int64_t)q.q0 * p.at + (int64_t)r.h * p.ah + (int64_t)r.d * Elem<SRC>::size;
    Spot at[COPY_TOKENS];
    Eight<SRC, DST, WIDE> x[COPY_TOKENS];
#pragma unroll
    for (int i = 0; i < COPY_TOKENS; i++) {
        const int tok = r.tok + i * r.step;
        at[i] = tok < n ? spot_of(a.b, q, tok) : Spot{-1, 0};
        if (tok < n) x[i].load(src + (int64_t)tok * p.at);
    }
#pragma unroll
    for (int i = 0; i < COPY_TOKENS; i++)
        if (at[i].page >= 0) x[i].store(p, at[i], r.h, r.d);
}

/* ---------------------------------------------------------------- writes of rotated rows
 *
 * Rope and append in one pass: the queries as k_rope takes them, the keys on their way into the pages,
 * which saves a launch and the keys' way to memory and back. A rotated key is rounded to its array's
 * type before it is stored, so that the cache holds the bits that the two calls, one after the other,
 * leave there. A key's thread takes eight elements of the row that it writes and reads the eight that
 * they are turned against as well (the second read of a line that its neighbour brings in). */
template <int SRC, bool HALF, bool EIGHTS>
__device__ __forceinline__ void rotated8(const uint8_t *row, int d, const f2 *cs, int n_freqs, int offset, float (&v)[8]) {
    using E = Elem<SRC>;
    constexpr int S = E::size;
    if constexpr (EIGHTS) {   /* all within the rotated part's one half, or all outside of it; on 16 bytes */
        E::load8(row + d * S, true, v);
        const int j = d - offset;
        if (j < 0 || j >= 2 * n_freqs) return;
        if constexpr (HALF) {
            const bool second = j >= n_freqs;
            const f2 *w = cs + (second ? j - n_freqs : j);
            float x[8];
            E::load8(row + (second ? d - n_freqs : d + n_freqs) * S, true, x);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float t = x[i] * w[i][1];
                v[i] = E::template rounded<false>(__builtin_fmaf(v[i], w[i][0], second ? t : -t));
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const f2 w = cs[j / 2 + i];
                const float x = v[2 * i], y = v[2 * i + 1];
                v[2 * i] = E::template rounded<false>(__builtin_fmaf(x, w[0], -(y * w[1])));
                v[2 * i + 1] = E::template rounded<false>(__builtin_fmaf(y, w[0], x * w[1]));
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int j = d + i - offset;
            v[i] = E::load(row + (d + i) * S);
            if (j < 0 || j >= 2 * n_freqs) continue;
            const bool second = HALF ? j >= n_freqs : j & 1;
            const f2 w = cs[HALF ? (second ? j - n_freqs : j) : j / 2];
            const int o = HALF ? n_freqs : 1;
            const float t = E::load(row + (second ? d + i - o : d + i + o) * S) * w[1];
            v[i] = E::template rounded<true>(__builtin_fmaf(v[i], w[0], second ? t : -t));
        }
    }
}

template <int SRC, int DST, bool HALF, bool WIDE>
__global__ __launch_bounds__(ROPE_THREADS) void k_kv_append_rotated(RotatedArgs a, int tok) {
    extern __shared__ f2 cs[];   /* [tok][n_freqs] */
    const Seq q = seq_of(a.c.b, blockIdx.y);
    const int n = min(q.n, a.c.b.max_q);
    const int64_t first = (int64_t)blockIdx.x * tok;
    if (first >= n) return;
    const int t0 = (int)first, nt = min(tok, n - t0);
    for (int i = threadIdx.x; i < nt * a.n_freqs; i += ROPE_THREADS) {
        const int t = t0 + i / a.n_freqs;
        const int64_t at = q.q0 + t;
        const double pos = !a.pos ? (double)(q.base + t) : a.pos64 ? (double)((const int64_t *)a.pos)[at] : (double)((const int *)a.pos)[at];
        cs[i] = turn_of(pos, a.freqs[i % a.n_freqs], a.factor, 1.0f);
    }
    __syncthreads();
    if (a.q.heads) rope_rows<SRC, HALF, WIDE>(a.q, q.q0 + t0, nt, cs, a.n_freqs, a.offset, a.width, a.in_place);
    const int o0 = a.c.p[0].heads * (a.c.p[0].width / 8);
    for (int i = threadIdx.x; i < nt * a.c.octs; i += ROPE_THREADS) {
        const int tl = i / a.c.octs;
        int o = i % a.c.octs;
        const int z = o >= o0 ? 1 : 0;
        if (z) o -= o0;
        const Piece &p = a.c.p[z];
        const int h = o / (p.width / 8), d = o % (p.width / 8) * 8;
        if (z != a.rotated) {
            append_item<SRC, DST, WIDE>(a.c, q, p, t0 + tl, h, d);
            continue;
        }
        const Spot at = spot_of(a.c.b, q, t0 + tl);
        if (at.page < 0) continue;
        float v[8];
        rotated8<SRC, HALF, WIDE>(p.arr + (int64_t)(q.q0 + t0 + tl) * p.at + (int64_t)h * p.ah, d, cs + tl * a.n_freqs, a.n_freqs, a.offset, v);
        put8<SRC, DST>(p, at, h, d, v);
    }
}

/* ---------------------------------------------------------------- cache reads */
template <int DST, int SRC, bool WIDE>
__global__ __launch_bounds__(256) void k_kv_read(CopyArgs a) {
    using E = Elem<DST>;
    const Seq q = seq_of(a.b, blockIdx.y);
    const int n = min(q.n, a.b.max_q);
    const Place r = place_of(a);
    if (r.tok < 0) return;
    const Piece p = *r.p;
    uint8_t *dst = p.arr + (int64_t)q.q0 * p.at + (int64_t)r.h * p.ah + (int64_t)r.d * E::size;
    Spot at[COPY_TOKENS];
    u4 w[COPY_TOKENS];              /* 8 stored elements: 16, 8 or 4 bytes */
    unsigned sc[COPY_TOKENS];
#pragma unroll
    for (int i = 0; i < COPY_TOKENS; i++) {
        const int tok = r.tok + i * r.step;
        at[i] = tok < n ? spot_of(a.b, q, tok) : Spot{-1, 0};
    }
#pragma unroll
    for (int i = 0; i < COPY_TOKENS; i++) {
        w[i] = (u4){0, 0, 0, 0};    /* zeros for rows that are not there, in every format */
        sc[i] = 127;
        if (at[i].page < 0) continue;
        const uint8_t *src = p.rows.data + (int64_t)at[i].page * p.rows.page_stride + (int64_t)r.h * p.rows.head_stride;
        const int64_t el = (int64_t)at[i].row * p.row_width + p.col + r.d;
        if constexpr (bits_of(SRC) == 16) w[i] = *(const u4 *)(src + el * 2);
        else {
            if constexpr (SRC == DT_MX4) w[i][0] = *(const unsigned *)(src + el / 2);
            else {
                const u2 c = *(const u2 *)(src + el);
                w[i][0] = c[0]; w[i][1] = c[1];
            }
            sc[i] = p.rows.scales[(int64_t)at[i].page * p.rows.scale_page_stride + (int64_t)r.h * p.rows.scale_head_stride + el / MX_BLOCK];
        }
    }
#pragma unroll
    for (int i = 0; i < COPY_TOKENS; i++) {
        const int tok = r.tok + i * r.step;
        if (tok >= n) return;
        uint8_t *to = dst + (int64_t)tok * p.at;
        if constexpr (SRC == DST) {
            if (WIDE) *(u4 *)to = w[i];
            else
#pragma unroll
                for (int j = 0; j < 8; j++) ((unsigned short *)to)[j] = (unsigned short)(w[i][j >> 1] >> (16 * (j & 1)));
        } else {
            float v[8];
            const float s = mx_scale(sc[i]);
            if constexpr (SRC == DT_MX4)
                each<4>([&](auto j) {
                    const f2 x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i][0], s, j);
                    v[2 * j] = x[0]; v[2 * j + 1] = x[1];
                });
            else if constexpr (SRC == DT_MX8)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i][j], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i][j], true);
                    v[4 * j] = lo[0] * s; v[4 * j + 1] = lo[1] * s; v[4 * j + 2] = hi[0] * s; v[4 * j + 3] = hi[1] * s;
                }
            else Elem<SRC>::load8((const uint8_t *)&w[i], true, v);
            E::store8(to, WIDE, v);
        }
    }
}

} // namespace

/* grid of place_of */
int64_t copy_groups(const CopyArgs &a) {
    const int tokens = 256 / std::min(a.octs, 256) * COPY_TOKENS;
    return ((int64_t)a.b.max_q + tokens - 1) / tokens;
}
static dim3 copy_grid(const CopyArgs &a) { return dim3((unsigned)copy_groups(a), a.b.n_seqs, (a.octs + 255) / 256); }

template <int DT, bool HALF>
static void rope_t(const RopeArgs &a, bool wide, int tok, hipStream_t st) {
    const dim3 grid(std::min((a.n_tokens - 1) / tok + 1, ROPE_GROUPS)), block(ROPE_THREADS);
    const size_t lds = sizeof(f2) * (size_t)tok * a.n_freqs;
    if (wide) hipLaunchKernelGGL((k_rope<DT, HALF, true>), grid, block, lds, st, a, tok);
    else hipLaunchKernelGGL((k_rope<DT, HALF, false>), grid, block, lds, st, a, tok);
}

void rope(const RopeArgs &a, int dtype, hipStream_t st) {
    const int es = dtype == DT_F32 ? 4 : 2;
    /* eight elements a thread where every piece of 8 starts on 16 bytes */
    bool wide = a.n_freqs % 8 == 0 && a.offset * es % 16 == 0;
    for (int z = 0; z < a.n_pairs; z++) {
        const auto &p = a.p[z];
        wide = wide && (((uintptr_t)p.x | (uintptr_t)p.y | (uint64_t)p.xt | (uint64_t)p.xh | (uint64_t)p.yt | (uint64_t)p.yh) & 15) == 0;
    }
    /* four tokens a workgroup where one does not fill it (64000 tokens, 9 heads of 64: 31 us, one by one
     * 85; 36 heads of 128: 200 us one by one, 217 in fours), and enough of them to fill the card */
    int64_t items = 0;
    for (int z = 0; z < a.n_pairs; z++) items += (int64_t)a.p[z].heads * (a.n_freqs / (wide ? 8 : 1));
    const int tok = a.n_tokens >= 1024 && items < ROPE_THREADS ? 4 : 1;
#define HXP_ROPE(DT) (a.interleaved ? rope_t<DT, false>(a, wide, tok, st) : rope_t<DT, true>(a, wide, tok, st))
    if (dtype == DT_F32) HXP_ROPE(DT_F32);
    else if (dtype == DT_F16) HXP_ROPE(DT_F16);
    else HXP_ROPE(DT_BF16);
#undef HXP_ROPE
}

/* calls f with the two dtypes as constants (arr: the caller's array, rows: the cache) */
template <class F>
static void by_types(int arr, int rows, F f) {
    auto with = [&](auto a) {
        if (rows == DT_F16) f(a, std::integral_constant<int, DT_F16>{});
        else if (rows == DT_BF16) f(a, std::integral_constant<int, DT_BF16>{});
        else if (rows == DT_MX8) f(a, std::integral_constant<int, DT_MX8>{});
        else f(a, std::integral_constant<int, DT_MX4>{});
    };
    if (arr == DT_F32) with(std::integral_constant<int, DT_F32>{});
    else if (arr == DT_F16) with(std::integral_constant<int, DT_F16>{});
    else with(std::integral_constant<int, DT_BF16>{});
}

void kv_append(const CopyArgs &a, int src_dtype, int cache_dtype, bool aligned, hipStream_t st) {
    const dim3 grid = copy_grid(a), block(256);
    by_types(src_dtype, cache_dtype, [&](auto s, auto c) {
        if (aligned) hipLaunchKernelGGL((k_kv_append<s.value, c.value, true>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((k_kv_append<s.value, c.value, false>), grid, block, 0, st, a);
    });
}

/* Tokens a workgroup takes where it does not fill it: as in rope. wide: q's and the keys' pieces of 8
 * start on 16 bytes, and none crosses a border of the rotated part. */
void kv_append_rotated(const RotatedArgs &a, int src_dtype, int cache_dtype, bool aligned, hipStream_t st) {
    bool wide = aligned && a.n_freqs % 8 == 0 && a.offset % 8 == 0;
    if (a.q.heads) wide = wide && (((uintptr_t)a.q.x | (uintptr_t)a.q.y | (uint64_t)a.q.xt | (uint64_t)a.q.xh | (uint64_t)a.q.yt | (uint64_t)a.q.yh) & 15) == 0;
    const int64_t items = (int64_t)a.q.heads * (a.n_freqs / (wide ? 8 : 1)) + a.c.octs;
    const int tok = a.c.b.max_q >= 1024 && items < ROPE_THREADS ? 4 : 1;
    const dim3 grid((unsigned)((a.c.b.max_q - 1) / tok + 1), a.c.b.n_seqs), block(ROPE_THREADS);
    const size_t lds = sizeof(f2) * (size_t)tok * a.n_freqs;
    by_types(src_dtype, cache_dtype, [&](auto s, auto c) {
        if (a.interleaved) {
            if (wide) hipLaunchKernelGGL((k_kv_append_rotated<s.value, c.value, false, true>), grid, block, lds, st, a, tok);
            else hipLaunchKernelGGL((k_kv_append_rotated<s.value, c.value, false, false>), grid, block, lds, st, a, tok);
        } else {
            if (wide) hipLaunchKernelGGL((k_kv_append_rotated<s.value, c.value, true, true>), grid, block, lds, st, a, tok);
            else hipLaunchKernelGGL((k_kv_append_rotated<s.value, c.value, true, false>), grid, block, lds, st, a, tok);
        }
    });
}

void kv_read(const CopyArgs &a, int dst_dtype, int cache_dtype, bool aligned, hipStream_t st) {
    const dim3 grid = copy_grid(a), block(256);
    by_types(dst_dtype, cache_dtype, [&](auto d, auto c) {
        if (aligned) hipLaunchKernelGGL((k_kv_read<d.value, c.value, true>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((k_kv_read<d.value, c.value, false>), grid, block, 0, st, a);
    });
}

} // namespace hxp
