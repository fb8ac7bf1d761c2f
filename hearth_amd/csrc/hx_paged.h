/*
 * hx_paged.h — argument blocks, device helpers and launchers of the paged-cache operators
 * (rotary positions, cache writes and reads, attention over pages). api_paged.cpp checks
 * every host-side field before a launch; lengths and page ids live in device memory and are
 * cut or checked in the kernels (seq_of, page_ok).
 */
#pragma once

#include "hx_host.h"

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

namespace hxp {

enum { DT_F32 = HEARTH_F32, DT_F16 = HEARTH_F16, DT_BF16 = HEARTH_BF16, DT_MX8 = HEARTH_GPU_MX8, DT_MX4 = HEARTH_GPU_MX4 };
constexpr int MX_BLOCK = 32;
/* bits of a stored element; below 16: codes with a scale byte for each MX_BLOCK */
constexpr int bits_of(int dtype) { return dtype == DT_MX4 ? 4 : dtype == DT_MX8 ? 8 : 16; }

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef short s4v __attribute__((ext_vector_type(4)));

/* hearth_gpu_batch with the bounds of every sequence's rows folded in */
struct Batch {
    const int *pages, *kv_len, *q_start;
    const unsigned long long *mask;
    int64_t ld_pages;
    int n_seqs, n_tokens, max_q, mask_words;
    int kv_cap;       /* min(max_kv, pages_per_seq * page): rows past it do not exist for the call */
    int n_pages, page_shift;
};

struct Rows {
    uint8_t *data;    /* bytes */
    uint8_t *scales;
    int64_t page_stride, head_stride;               /* bytes */
    int64_t scale_page_stride, scale_head_stride;   /* bytes */
};

/* ---- rotary positions ---- */
struct RopeArgs {
    struct Pair { const uint8_t *x; uint8_t *y; int64_t xt, xh, yt, yh; int heads; } p[2];   /* strides in bytes */
    const void *pos;
    const double *freqs;
    int n_tokens, width, n_freqs, offset, pos64, interleaved, n_pairs;
    float factor, sign;
    bool in_place;    /* the elements outside the rotated part are where they belong */
};

/* ---- cache writes and reads: up to two pieces of a row (k and v, or latent and rotated part) ---- */
struct Piece {
    uint8_t *arr;             /* the caller's rows */
    int64_t at, ah;           /* its strides, bytes */
    Rows rows;
    int col, width, row_width, heads;   /* elements [col, col + width) of cache rows of row_width */
};
struct CopyArgs {
    Batch b;
    Piece p[2];
    int n_pieces, octs;       /* groups of 8 elements of a token over all pieces and heads */
};

/* ---- writes of rotated rows ---- */
struct RotatedArgs {
    CopyArgs c;
    RopeArgs::Pair q;         /* heads 0: none */
    const void *pos;          /* NULL: a token's row in its sequence */
    const double *freqs;
    int rotated;              /* which piece is: the keys, or a latent row's second part */
    int width, n_freqs, offset, pos64, interleaved;
    float factor;
    bool in_place;
};

/* ---- attention ---- */
struct AttendArgs {
    Batch b;
    Rows k, v;
    const uint8_t *q, *q_pe;
    uint8_t *out;
    float *lse;
    int64_t qt, qh, pt, ph, ot, oh;   /* strides of q, q_pe, out; bytes */
    int heads, kv_heads, group;       /* group: query heads per kv head */
    float scale2;                     /* scale * log2(e): probabilities are powers of two */
    int chunk, n_splits;              /* rows of a split (a multiple of the kernels' row step); splits of the longest */
    float *part;                      /* [n_tokens][heads][n_splits][DV] sums, then [..][2] maximum and sum */
    /* attend_blocks: the rows are those of the chosen blocks, one after the other */
    const int *chosen;
    int64_t ct, ch;                   /* elements */
    int top, block_shift;             /* top 0: every row */
};

/* ---- blocks of rows, their bounds and their choice ---- */
struct Bounds {
    uint8_t *codes, *scales;
    int64_t page_stride, head_stride, scale_page_stride, scale_head_stride;   /* bytes */
    int block_shift, blocks;          /* log2 of a block's rows; blocks of a page */
};
struct BoundsArgs {
    Batch b;
    Rows k;
    Bounds s;
    int heads;
    int64_t per_seq;                  /* blocks that a sequence's tokens may touch */
};
struct SelectArgs {
    Batch b;
    Bounds s;
    const uint8_t *q;
    int64_t qt, qh;                   /* bytes */
    int *chosen;
    int64_t ct, ch;                   /* elements */
    int kv_heads, group, top, first, last;
    float *score;                     /* [n_tokens][kv_heads][ld_score] */
    int64_t ld_score;
    int tiles, chunk, n_chunks;       /* of the scores: workgroups of tokens, blocks a workgroup, its shares (0: no blocks) */
    bool many;                        /* tokens share their blocks' bounds */
};

/* device of a call made current while the object lives */
struct DeviceGuard {
    int old = -1;
    bool ok = false;
    explicit DeviceGuard(int dev) {
        if (hipGetDevice(&old) != hipSuccess) return;
        ok = old == dev || hipSetDevice(dev) == hipSuccess;
        if (old == dev) old = -1;
    }
    ~DeviceGuard() { if (ok && old >= 0) (void)hipSetDevice(old); }
};

void rope(const RopeArgs &a, int dtype, hipStream_t st);
int64_t copy_groups(const CopyArgs &a);   /* workgroups of a sequence's tokens */
void kv_append(const CopyArgs &a, int src_dtype, int cache_dtype, bool aligned, hipStream_t st);
void kv_append_rotated(const RotatedArgs &a, int src_dtype, int cache_dtype, bool aligned, hipStream_t st);
void kv_read(const CopyArgs &a, int dst_dtype, int cache_dtype, bool aligned, hipStream_t st);

/* Split of the rows axis: rows per split and splits of the longest sequence, and whether the
 * kernel of many query rows takes the call. Depends on the host-side fields only, and not on the
 * call's token count. latent: the kernels of attend_latent. */
struct Split { int chunk, n; bool many; };
Split attend_split(int n_seqs, int max_q, int kv_cap, int heads, int kv_heads, bool latent, bool four);
void attend(const AttendArgs &a, int q_dtype, int cache_dtype, int width, bool many, hipStream_t st);
Split blocks_split(int n_seqs, int max_q, int rows, int heads, int kv_heads);
void attend_blocks(const AttendArgs &a, int q_dtype, int cache_dtype, int width, hipStream_t st);
void attend_many(const AttendArgs &a, int q_dtype, int cache_dtype, int width, hipStream_t st);   /* k_paged_many.hip */
void latent_rows(const AttendArgs &a, int q_dtype, bool mx, hipStream_t st);                         /* k_paged_latent.hip */
void attend_latent(const AttendArgs &a, int q_dtype, int cache_dtype, hipStream_t st);

void key_bounds(const BoundsArgs &a, int cache_dtype, int width, hipStream_t st);   /* k_paged_select.hip */
int select_group_limit();   /* query heads of a kv head */
void score_split(SelectArgs &a);
void select_blocks(const SelectArgs &a, int q_dtype, int width, hipStream_t st);

/* ------------------------------------------------------------------ device helpers */

/* A word that the whole workgroup reads and no kernel of the call writes, through the scalar cache:
 * a vector load's wait would wait for every row load issued before it as well. */
__device__ __forceinline__ int word_of(const int *p, int64_t i) { return ((const __attribute__((address_space(4))) int *)p)[i]; }

struct Seq {
    int q0, n;       /* first token of the call, tokens */
    int kv;          /* rows that exist */
    int base;        /* position of its first token of the call (negative: more tokens than rows) */
};

__device__ __forceinline__ Seq seq_of(const Batch &b, int s) {
    Seq r;
    const int lo = min(max(word_of(b.q_start, s), 0), b.n_tokens);
    const int hi = min(max(word_of(b.q_start, s + 1), lo), b.n_tokens);
    const int len = max(word_of(b.kv_len, s), 0);
    r.q0 = lo;
    r.n = hi - lo;
    r.kv = min(len, b.kv_cap);
    r.base = len - r.n;
    return r;
}

__device__ __forceinline__ bool page_ok(const Batch &b, int id) { return (unsigned)id < (unsigned)b.n_pages; }

/* Which of the 64 rows from t0 on a column attends: those below lim and, in a tree, the call's
 * tokens of its mask row `words` (token j is row base + j); none from hi on. Two words are read a
 * step: a load a score cost a tree's last steps 30 us. */
__device__ __forceinline__ unsigned long long step_mask(int t0, int lim, int hi, int base, const unsigned long long *words, int n_words) {
    const int n = lim - t0, h = hi - t0;
    unsigned long long x = n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1;
    if (words) {
        const int64_t off = (int64_t)t0 - base;
        if (off > -64 && off < 64 * (int64_t)n_words) {
            const int k = (int)(off >> 6), sh = (int)(off & 63);   /* floor: k = -1 where the call's tokens begin inside the step */
            const unsigned long long a = k >= 0 ? words[k] : 0, b = k + 1 < n_words ? words[k + 1] : 0;
            x |= sh ? a >> sh | b << (64 - sh) : a;
        }
    }
    return h >= 64 ? x : h <= 0 ? 0ull : x & ((1ull << h) - 1);
}

/* The sum of exponentials is 0 where a column attends nothing, and where it attends rows whose scores
 * are all -infinity. The first result is 0, the second 0 / 0: NaN, as in the formula. */
constexpr float UNDEFINED = __builtin_nanf("");

/* bits of 16 rows a page group each, from bits of groups */
__device__ __forceinline__ unsigned long long group_rows(unsigned have) {
    unsigned long long x = 0;
#pragma unroll
    for (int u = 0; u < 4; u++) x |= have >> u & 1 ? 0xffffull << (16 * u) : 0;
    return x;
}

/* 16-bit types: the matrix instructions and conversions of one type */
struct Bf16 {
    using v8 = b8;
    using e = __bf16;
    static __device__ __forceinline__ f4 mfma16(v8 a, v8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ f16v mfma32(v8 a, v8 b, f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    /* codes (two bytes of x, the upper two with HI) times a power of two; exact but for underflow */
    template <bool HI> static __device__ __forceinline__ unsigned from_mx8(unsigned x, float s) {
        return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, s, HI));
    }
    /* two 4-bit codes (byte B of x, the lower half first) likewise */
    template <int B> static __device__ __forceinline__ unsigned from_mx4(unsigned x, float s) {
        return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, s, B));
    }
    /* round to nearest even, both halves */
    static __device__ __forceinline__ unsigned pack(float a, float b) { return __builtin_bit_cast(unsigned, __builtin_convertvector((f2){a, b}, b2)); }
    static __device__ __forceinline__ float wide(unsigned x) { return __uint_as_float(x << 16); }   /* of the lower half */
    /* x with infinite and NaN halves as zeros */
    static __device__ __forceinline__ unsigned clean(unsigned x) {
        return ((x & 0x7f80u) == 0x7f80u ? 0u : x & 0xffffu) | ((x & 0x7f800000u) == 0x7f800000u ? 0u : x & 0xffff0000u);
    }
    /* true where a half of x is infinite or NaN */
    static __device__ __forceinline__ bool odd(unsigned x) { return (x & 0x7f80u) == 0x7f80u || (x & 0x7f800000u) == 0x7f800000u; }
};
struct F16 {
    using v8 = h8;
    using e = _Float16;
    static __device__ __forceinline__ f4 mfma16(v8 a, v8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ f16v mfma32(v8 a, v8 b, f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    template <bool HI> static __device__ __forceinline__ unsigned from_mx8(unsigned x, float s) {
        return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, s, HI));
    }
    template <int B> static __device__ __forceinline__ unsigned from_mx4(unsigned x, float s) {
        return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x, s, B));
    }
    static __device__ __forceinline__ unsigned pack(float a, float b) { return __builtin_bit_cast(unsigned, __builtin_convertvector((f2){a, b}, h2)); }
    static __device__ __forceinline__ float wide(unsigned x) { return (float)__builtin_bit_cast(_Float16, (unsigned short)x); }
    static __device__ __forceinline__ unsigned clean(unsigned x) {
        return ((x & 0x7c00u) == 0x7c00u ? 0u : x & 0xffffu) | ((x & 0x7c000000u) == 0x7c000000u ? 0u : x & 0xffff0000u);
    }
    static __device__ __forceinline__ bool odd(unsigned x) { return (x & 0x7c00u) == 0x7c00u || (x & 0x7c000000u) == 0x7c000000u; }
};

/* Element d of a stored row (row: its first byte, sc: its first scale byte) in T's format */
template <class T, int BITS>
__device__ __forceinline__ unsigned row_elem(const uint8_t *row, const uint8_t *sc, int d) {
    if constexpr (BITS == 4)
        return T::template from_mx4<0>((unsigned)row[d >> 1] >> (4 * (d & 1)), __uint_as_float((unsigned)sc[d / MX_BLOCK] << 23)) & 0xffffu;
    else if constexpr (BITS == 8)
        return T::template from_mx8<false>((unsigned)row[d], __uint_as_float((unsigned)sc[d / MX_BLOCK] << 23)) & 0xffffu;
    else
        return ((const unsigned short *)row)[d];
}

/* 16, 8, 4 and 2 bytes at any address (the memory system takes each as one access) */
typedef u4 u4_any __attribute__((aligned(1)));
typedef u2 u2_any __attribute__((aligned(1)));
typedef unsigned unsigned_any __attribute__((aligned(1)));
typedef unsigned short ushort_any __attribute__((aligned(1)));

/* the scale of a block from its byte (1 to 254; 255, of a 4-bit block that holds a NaN or an infinity, makes
 * every conversion of its codes a NaN) */
__device__ __forceinline__ float mx_scale(unsigned byte) { return __uint_as_float((byte & 255u) << 23); }

/* of the byte at bit `at` of a word */
__device__ __forceinline__ float mx_scale_at(unsigned word, unsigned at) { return __uint_as_float(__builtin_amdgcn_ubfe(word, at, 8) << 23); }

/* maximum / sum of a value over the lanes l, l ^ 32 */
__device__ __forceinline__ float max32(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum32(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
/* ... over the lanes l, l ^ 16 */
__device__ __forceinline__ float max16(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum16(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

/* 16 bytes a lane from memory straight to LDS: lane l's, at base + off + OFS, to dst + 16 l (base and
 * dst: the same for the wave). Written out because the compiler, which cannot tell the buffers of a
 * double buffer apart, lets every later LDS read wait for the builtin's loads. The LDS address is
 * handed over in m0, which the compiler writes, so that it knows of it (it takes m0 for no clobber);
 * no register is written here. The loads have arrived after vm_wait(), and are there for the other
 * waves after a barrier behind it. */
template <int OFS>
__device__ __forceinline__ void to_lds(const uint8_t *base, int off, uint8_t *dst) {
    const unsigned at = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)dst) - OFS;   /* the instruction adds OFS here too */
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 offset:%3" ::"{m0}"(at), "v"(off), "s"(base), "n"(OFS)
                 : "memory");
}
/* N instructions of the same kind, the z-th 1 KiB further in memory (from off[z]) and in LDS */
template <int N>
__device__ __forceinline__ void to_lds_rows(const uint8_t *base, const int (&off)[N], uint8_t *dst) {
    static_assert(N == 2 || N == 4);
    const unsigned at = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)dst);
    if constexpr (N == 2)
        asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %3\n\t"
                     "global_load_lds_dwordx4 %2, %3 offset:%4" ::"{m0}"(at), "v"(off[0]), "v"(off[1]), "s"(base), "n"(1 << 10) : "memory");
    else
        asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %5\n\t"
                     "global_load_lds_dwordx4 %2, %5 offset:%6\n\tglobal_load_lds_dwordx4 %3, %5 offset:%7\n\t"
                     "global_load_lds_dwordx4 %4, %5 offset:%8"
                     ::"{m0}"(at), "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(base), "n"(1 << 10), "n"(2 << 10), "n"(3 << 10)
                     : "memory");
}
/* transposing LDS load: lane i of 16 gives the address of 4 elements of row i / 4 and gets element
 * i of the four rows */
__device__ __forceinline__ u2 read_tr(const uint8_t *p) {
    return __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v *)p));
}

/* the same address for the whole wave, in scalar registers */
__device__ __forceinline__ const uint8_t *same(const uint8_t *p) {
    const uint64_t x = (uint64_t)p;
    return (const uint8_t *)((uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 |
                             (unsigned)__builtin_amdgcn_readfirstlane((int)x));
}
/* likewise, for loads: an address of device memory to which a lane adds a 32-bit offset of its own */
__device__ __forceinline__ const uint8_t *same_global(const uint8_t *p) {
    return (const uint8_t *)(const __attribute__((address_space(1))) uint8_t *)(uint64_t)same(p);
}
template <int N, class F> __device__ __forceinline__ void each(F f) {   /* f(constant 0) .. f(constant N - 1) */
    if constexpr (N > 0) {
        each<N - 1>(f);
        f(std::integral_constant<int, N - 1>{});
    }
}
/* all but the wave's last N loads have arrived */
template <int N = 0> __device__ __forceinline__ void vm_wait() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

/* Every load has arrived and the compiler knows it: without this the first use inside a loop of a
 * value loaded before it waits, in every round, for all loads under way. */
__device__ __forceinline__ void arrived() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0f70);   /* vmcnt(0) */
    __builtin_amdgcn_sched_barrier(0);
}

/* keeps what stands before it in the source before what stands behind it */
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0); }

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

} // namespace hxp
