/*
 * k_paged.hip — rotary positions and the writes and reads of a paged cache. All three move
 * each element once and are bound by HBM for prompts and by launch latency for single tokens:
 * rotating 64 of 192 elements of 2001 tokens of 128 heads (66 MB) takes 13.9 us (4.8 TB/s, near a
 * large copy's 4.9), quantising 3 x 4093 rows (31 MB) 13.2 us, reading 8 x 4095 back (71 MB) 19 us
 * (3.7 TB/s), the rows of 32 single tokens 3.5 us.
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

template <int DT, bool HALF, bool WIDE>
__global__ __launch_bounds__(ROPE_THREADS) void k_rope(RopeArgs a, int tok) {
    extern __shared__ f2 cs[];   /* [tok][n_freqs] */
    using E = Elem<DT>;
    constexpr int S = E::size;
    for (int64_t t0 = (int64_t)blockIdx.x * tok; t0 < a.n_tokens; t0 += (int64_t)gridDim.x * tok) {
        const int nt = (int)min((int64_t)tok, a.n_tokens - t0);
        for (int i = threadIdx.x; i < nt * a.n_freqs; i += ROPE_THREADS) {
            const int64_t t = t0 + i / a.n_freqs;
            const int j = i % a.n_freqs;
            const double pos = a.pos64 ? (double)((const int64_t *)a.pos)[t] : (double)((const int *)a.pos)[t];
            const double turns = pos * (a.freqs[j] * 0.15915494309189533577);
            const float r = 2.0f * (float)(turns - rint(turns));
            float s, c;
            sincospif(r, &s, &c);
            cs[i] = (f2){c * a.factor, s * a.factor * a.sign};
        }
        __syncthreads();
        /* an item is 8 elements of each half (HALF), 16 consecutive ones (interleaved), or, WIDE
         * false, one pair; then the elements outside the rotated part, one at a time */
        constexpr int PER = WIDE ? 8 : 1;
        const int items = a.n_freqs / PER;
        for (int z = 0; z < a.n_pairs; z++) {
            const auto &p = a.p[z];
            const int per_tok = p.heads * items;
            for (int i = threadIdx.x; i < nt * per_tok; i += ROPE_THREADS) {
                const int tl = i / per_tok, rem = i % per_tok, h = rem / items, j = rem % items * PER;
                const uint8_t *x = p.x + (t0 + tl) * p.xt + (int64_t)h * p.xh + a.offset * S;
                uint8_t *y = p.y + (t0 + tl) * p.yt + (int64_t)h * p.yh + a.offset * S;
                const f2 *w = cs + tl * a.n_freqs + j;
                if constexpr (WIDE) {
                    const int o0 = HALF ? j * S : 2 * j * S, o1 = HALF ? (j + a.n_freqs) * S : (2 * j + 8) * S;
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
                    const int o0 = HALF ? j * S : 2 * j * S, o1 = HALF ? (j + a.n_freqs) * S : (2 * j + 1) * S;
                    const float u = E::load(x + o0), v = E::load(x + o1);
                    E::store(y + o0, __builtin_fmaf(u, w[0][0], -(v * w[0][1])));
                    E::store(y + o1, __builtin_fmaf(v, w[0][0], u * w[0][1]));
                }
            }
            if (!a.in_place) {
                const int rest = a.width - 2 * a.n_freqs;
                for (int i = threadIdx.x; i < nt * p.heads * rest; i += ROPE_THREADS) {
                    const int tl = i / (p.heads * rest), rem = i % (p.heads * rest), h = rem / rest;
                    int d = rem % rest;
                    if (d >= a.offset) d += 2 * a.n_freqs;
                    const uint8_t *x = p.x + (t0 + tl) * p.xt + (int64_t)h * p.xh + (int64_t)d * S;
                    uint8_t *y = p.y + (t0 + tl) * p.yt + (int64_t)h * p.yh + (int64_t)d * S;
                    if constexpr (S == 4) *(unsigned *)y = *(const unsigned *)x;
                    else *(unsigned short *)y = *(const unsigned short *)x;
                }
            }
        }
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
 * above 1.9375) the code is cut to 240, which is within half a step (2^-4) of the value. */
__device__ __forceinline__ bool fin(float x) { return __builtin_fabsf(x) < __builtin_huge_valf(); }

/* The eight elements that a thread of either kernel takes of each of its tokens: octs threads a
 * token (grid.z of them where that is more than a workgroup), several tokens a workgroup where it is
 * less; which piece, head and element they are is worked out once for COPY_TOKENS tokens (16 x 4093
 * rows of 4 heads of 128 into 8 bits: 37 us, one by one 44, eight at once 15% more than four on 3 x
 * 4093). The piece's addresses and strides are read from the arguments again for each token, so the
 * four tokens' way from page id to store is walked one after the other: that bounds prompts. */
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

/* lanes of one block of 32 come here together: octs and every piece's width / 8 are multiples of 4 */
template <int SRC, int DST, bool WIDE>
__device__ __forceinline__ void append_item(const CopyArgs &a, const Seq &q, const Piece &p, int tok, int h, int d) {
    using E = Elem<SRC>;
    const int pos = q.base + tok;
    if (pos < 0 || pos >= q.kv) return;
    const int page = a.b.pages[(int64_t)blockIdx.y * a.b.ld_pages + (pos >> a.b.page_shift)];
    if (!page_ok(a.b, page)) return;
    const int row = pos & ((1 << a.b.page_shift) - 1);
    const uint8_t *src = p.arr + (int64_t)(q.q0 + tok) * p.at + (int64_t)h * p.ah + (int64_t)d * E::size;
    uint8_t *dst = p.rows.data + (int64_t)page * p.rows.page_stride + (int64_t)h * p.rows.head_stride;
    const int64_t el = (int64_t)row * p.row_width + p.col + d;
    if constexpr (DST == SRC && DST != DT_MX8) {
        if (WIDE) *(u4 *)(dst + el * 2) = *(const u4 *)src;
        else {
            unsigned short w[8];
#pragma unroll
            for (int j = 0; j < 8; j++) w[j] = ((const unsigned short *)src)[j];
            *(u4 *)(dst + el * 2) = (u4){w[0] | (unsigned)w[1] << 16, w[2] | (unsigned)w[3] << 16,
                                         w[4] | (unsigned)w[5] << 16, w[6] | (unsigned)w[7] << 16};
        }
    } else {
        float v[8];
        E::load8(src, WIDE, v);
        if constexpr (DST != DT_MX8) {
            Elem<DST>::store8(dst + el * 2, true, v);
        } else {
            float m = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) m = fmaxf(m, fin(v[j]) ? __builtin_fabsf(v[j]) : 0.0f);
            m = fmaxf(m, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(m), 0xB1, 0xF, 0xF, true)));
            m = fmaxf(m, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(m), 0x4E, 0xF, 0xF, true)));
            const int bits = (int)__float_as_uint(m);
            const int byte = max((bits >> 23) - 8 + ((bits & 0x7fffff) > 0x600000), 1);   /* e + 127 */
            const float inv = __uint_as_float((unsigned)(254 - byte) << 23);
            const float top = (SRC == DT_F16 ? byte == 127 + 8 : byte == 127 + 120) ? 240.0f : 448.0f;
            unsigned c[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float s = v[j] * inv;
                const float t = fin(v[j]) ? fminf(fmaxf(s, -top), top) : 0.0f;
                unsigned code = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(t, t, 0, false) & 255u;
                if (!fin(v[j])) code = 0x7f;
                c[j >> 2] |= code << (8 * (j & 3));
            }
            *(u2 *)(dst + el) = (u2){c[0], c[1]};
            if ((d & 31) == 0)
                p.rows.scales[(int64_t)page * p.rows.scale_page_stride + (int64_t)h * p.rows.scale_head_stride +
                              el / MX_BLOCK] = (uint8_t)byte;
        }
    }
}

template <int SRC, int DST, bool WIDE>
__global__ __launch_bounds__(256) void k_kv_append(CopyArgs a) {
    const Seq q = seq_of(a.b, blockIdx.y);
    const int n = min(q.n, a.b.max_q);
    const Place r = place_of(a);
    if (r.tok < 0) return;
#pragma unroll
    for (int i = 0; i < COPY_TOKENS; i++) {
        const int tok = r.tok + i * r.step;
        if (tok < n) append_item<SRC, DST, WIDE>(a, q, *r.p, tok, r.h, r.d);
    }
}

/* ---------------------------------------------------------------- cache reads */
template <int DST, int SRC, bool WIDE>
__device__ __forceinline__ void read_item(const CopyArgs &a, const Seq &q, const Piece &p, int tok, int h, int d) {
    using E = Elem<DST>;
    const int pos = q.base + tok;
    int page = -1;
    if (pos >= 0 && pos < q.kv) page = a.b.pages[(int64_t)blockIdx.y * a.b.ld_pages + (pos >> a.b.page_shift)];
    const int row = pos & ((1 << a.b.page_shift) - 1);
    uint8_t *dst = p.arr + (int64_t)(q.q0 + tok) * p.at + (int64_t)h * p.ah + (int64_t)d * E::size;
    float v[8] = {};
    if (page_ok(a.b, page)) {
        const uint8_t *src = p.rows.data + (int64_t)page * p.rows.page_stride + (int64_t)h * p.rows.head_stride;
        const int64_t el = (int64_t)row * p.row_width + p.col + d;
        if constexpr (SRC == DT_MX8) {
            const u2 c = *(const u2 *)(src + el);
            const float s = mx_scale(p.rows.scales[(int64_t)page * p.rows.scale_page_stride +
                                                   (int64_t)h * p.rows.scale_head_stride + el / MX_BLOCK]);
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[j], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[j], true);
                v[4 * j] = lo[0] * s; v[4 * j + 1] = lo[1] * s; v[4 * j + 2] = hi[0] * s; v[4 * j + 3] = hi[1] * s;
            }
        } else {
            if constexpr (SRC == DST) {
                const u4 w = *(const u4 *)(src + el * 2);
                if (WIDE) *(u4 *)dst = w;
                else {
#pragma unroll
                    for (int j = 0; j < 8; j++) ((unsigned short *)dst)[j] = (unsigned short)(w[j >> 1] >> (16 * (j & 1)));
                }
                return;
            }
            Elem<SRC>::load8(src + el * 2, true, v);
        }
    }
    E::store8(dst, WIDE, v);
}

template <int DST, int SRC, bool WIDE>
__global__ __launch_bounds__(256) void k_kv_read(CopyArgs a) {
    const Seq q = seq_of(a.b, blockIdx.y);
    const int n = min(q.n, a.b.max_q);
    const Place r = place_of(a);
    if (r.tok < 0) return;
#pragma unroll
    for (int i = 0; i < COPY_TOKENS; i++) {
        const int tok = r.tok + i * r.step;
        if (tok < n) read_item<DST, SRC, WIDE>(a, q, *r.p, tok, r.h, r.d);
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
        else f(a, std::integral_constant<int, DT_MX8>{});
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

void kv_read(const CopyArgs &a, int dst_dtype, int cache_dtype, bool aligned, hipStream_t st) {
    const dim3 grid = copy_grid(a), block(256);
    by_types(dst_dtype, cache_dtype, [&](auto d, auto c) {
        if (aligned) hipLaunchKernelGGL((k_kv_read<d.value, c.value, true>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((k_kv_read<d.value, c.value, false>), grid, block, 0, st, a);
    });
}

} // namespace hxp
