/*
 * api_paged.cpp — the paged-cache operators of hearth_gpu.h: host-side checks, then one or two
 * launches on the caller's stream. Every field that a kernel uses as a bound or an index is
 * checked here; what lies in device memory (page ids, lengths) is checked in the kernels.
 */
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "hx_host.h"
#include "hx_paged.h"

using namespace hx;
using namespace hxp;

namespace {

constexpr int64_t MAX_STRIDE = (int64_t)1 << 46;   /* elements: past any memory, and far from 64 bits in bytes */
constexpr int MAX_ROWS = 0x3fff0000;                /* rows of a sequence that an attention takes: split ends stay within 31 bits */
constexpr int64_t MAX_LATENT_TILES = 0x7ffff0;      /* workgroups of 512 threads in one dimension of a grid (below 2^32 threads) */
constexpr int64_t MAX_COPY_GROUPS = 0xffffff;       /* workgroups of 256 likewise */
constexpr int64_t MAX_PICKS = 1 << 23;              /* workgroups of 256 that choose blocks, likewise */
constexpr int MAX_HEADS = 65536;                    /* of an array */
constexpr int64_t MAX_ROPE_ROW = 1 << 24;           /* elements of a token: four of them count within 31 bits */

bool pow2(int x) { return x > 0 && (x & (x - 1)) == 0; }

bool rows_ok(const hearth_gpu_rows &r, const hearth_gpu_cache &c) {
    const int bits = bits_of(c.dtype);
    const int es = bits == 16 ? 2 : 1;                                              /* bytes of a stride's element */
    const int64_t els = (int64_t)c.page * c.width, block = bits == 4 ? els / 2 : els;
    if (!r.data || (uintptr_t)r.data % 16) return false;
    if (r.head_stride < (c.n_heads > 1 ? block : 0) || r.page_stride < (c.n_pages > 1 ? block : 0)) return false;
    if (r.head_stride > MAX_STRIDE || r.page_stride > MAX_STRIDE) return false;
    if (r.head_stride * es % 16 || r.page_stride * es % 16) return false;
    if (bits == 16) return true;
    if (!r.scales || r.scale_head_stride < (c.n_heads > 1 ? els / MX_BLOCK : 0) || r.scale_head_stride > MAX_STRIDE) return false;
    return r.scale_page_stride >= (c.n_pages > 1 ? els / MX_BLOCK : 0) && r.scale_page_stride <= MAX_STRIDE;
}

bool cache_ok(const hearth_gpu_cache *c) {
    if (!c || (c->dtype != HEARTH_F16 && c->dtype != HEARTH_BF16 && c->dtype != HEARTH_GPU_MX8 && c->dtype != HEARTH_GPU_MX4)) return false;
    if (c->n_pages < 1 || c->n_heads < 1 || c->n_heads > 4096 || !pow2(c->page) || c->page < 16 || c->page > 4096) return false;
    if (c->width < 32 || c->width > 1024 || c->width % 32) return false;
    return rows_ok(c->k, *c) && (!c->v.data || rows_ok(c->v, *c));
}

bool batch_ok(const hearth_gpu_batch *b) {
    if (!b || b->n_seqs < 0 || b->n_seqs > 65535 || b->n_tokens < 0 || b->max_q < 0 || b->max_kv < 0 || b->pages_per_seq < 0) return false;
    if (b->n_seqs && (!b->kv_len || !b->q_start || (b->pages_per_seq && !b->pages))) return false;
    if (b->ld_pages < b->pages_per_seq && b->n_seqs > 1) return false;
    if (b->ld_pages < 0 || b->ld_pages > MAX_STRIDE) return false;
    if (((uintptr_t)b->pages | (uintptr_t)b->kv_len | (uintptr_t)b->q_start) % 4 || (uintptr_t)b->mask % 8) return false;
    return !b->mask || (b->mask_words >= 1 && (int64_t)b->mask_words * 64 >= b->max_q);
}

int elem(int dtype) { return dtype == HEARTH_F32 ? 4 : dtype == HEARTH_F16 || dtype == HEARTH_BF16 ? 2 : 0; }

/* n: tokens; without any, data may be NULL */
bool array_ok(const hearth_gpu_array *x, int n) {
    if (!x || (n && !x->data) || !elem(x->dtype) || x->n_heads < 1 || x->n_heads > MAX_HEADS || x->width < 1 || x->width > 65536) return false;
    if ((uintptr_t)x->data % elem(x->dtype)) return false;
    return std::llabs(x->token_stride) <= MAX_STRIDE && std::llabs(x->head_stride) <= MAX_STRIDE;
}

/* of an array that is written: neighbouring rows share no element (broadcast ones do) */
bool apart(const hearth_gpu_array &x, int n) {
    return (x.n_heads < 2 || std::llabs(x.head_stride) >= x.width) && (n < 2 || std::llabs(x.token_stride) >= x.width);
}

/* pointer and strides on 16 bytes */
bool on16(const hearth_gpu_array &x) {
    const int64_t es = elem(x.dtype);
    return (uintptr_t)x.data % 16 == 0 && x.token_stride * es % 16 == 0 && x.head_stride * es % 16 == 0;
}

Rows rows_of(const hearth_gpu_rows &r, int dtype) {
    const int64_t es = bits_of(dtype) == 16 ? 2 : 1;
    return {(uint8_t *)r.data, r.scales, r.page_stride * es, r.head_stride * es, r.scale_page_stride, r.scale_head_stride};
}

Batch batch_of(const hearth_gpu_batch &b, const hearth_gpu_cache &c) {
    Batch o{};
    o.pages = b.pages; o.kv_len = b.kv_len; o.q_start = b.q_start;
    o.mask = (const unsigned long long *)b.mask;
    o.ld_pages = b.ld_pages; o.n_seqs = b.n_seqs; o.n_tokens = b.n_tokens;
    o.max_q = std::min(b.max_q, b.n_tokens); o.mask_words = b.mask_words;
    o.kv_cap = (int)std::min<int64_t>(b.max_kv, std::min<int64_t>((int64_t)b.pages_per_seq * c.page, 0x7fffff00));
    o.n_pages = c.n_pages;
    o.page_shift = __builtin_ctz((unsigned)c.page);
    return o;
}

Batch batch_of(const hearth_gpu_batch &b, int n_pages, int page) {
    hearth_gpu_cache c{};
    c.n_pages = n_pages; c.page = page;
    return batch_of(b, c);
}

bool bounds_ok(const hearth_gpu_bounds *s) {
    if (!s || !s->codes || (uintptr_t)s->codes % 16 || !s->scales) return false;
    if (s->n_pages < 1 || s->n_heads < 1 || s->n_heads > 4096 || !pow2(s->block) || s->block < 16 || !pow2(s->blocks)) return false;
    if ((int64_t)s->block * s->blocks > 4096 || (s->width != 64 && s->width != 128 && s->width != 256)) return false;
    const int64_t els = (int64_t)s->blocks * 2 * s->width;
    if (s->head_stride < (s->n_heads > 1 ? els : 0) || s->page_stride < (s->n_pages > 1 ? els : 0)) return false;
    if (s->head_stride > MAX_STRIDE || s->page_stride > MAX_STRIDE || s->head_stride % 16 || s->page_stride % 16) return false;
    if (s->scale_head_stride < (s->n_heads > 1 ? s->blocks : 0) || s->scale_page_stride < (s->n_pages > 1 ? s->blocks : 0)) return false;
    return s->scale_head_stride <= MAX_STRIDE && s->scale_page_stride <= MAX_STRIDE;
}

Bounds bounds_of(const hearth_gpu_bounds &s) {
    return {(uint8_t *)s.codes, s.scales, s.page_stride, s.head_stride, s.scale_page_stride, s.scale_head_stride,
            __builtin_ctz((unsigned)s.block), s.blocks};
}

int64_t blocks_of(int rows, int block) { return ((int64_t)rows + block - 1) / block; }

/* of the blocks chosen for n tokens and so many heads; written: rows share no element */
bool blocks_ok(const hearth_gpu_blocks *x, int n, int heads, bool written) {
    if (!x || (n && !x->chosen) || (uintptr_t)x->chosen % 4 || x->top < 1 || x->top > (1 << 20) || !pow2(x->block) || x->block < 16 || x->block > 4096) return false;
    if (std::llabs(x->token_stride) > MAX_STRIDE || std::llabs(x->head_stride) > MAX_STRIDE) return false;
    return !written || ((heads < 2 || std::llabs(x->head_stride) >= x->top) && (n < 2 || std::llabs(x->token_stride) >= x->top));
}

int finish() { return hipGetLastError() == hipSuccess ? OK : E_IO; }   /* this call's launches only */

/* The call's own error, read so that the thread's next call does not take it for the caller's. */
int no_device() {
    (void)hipGetLastError();
    return E_IO;
}

/* Checked arguments of a write or read; a.b.max_q 0: nothing to do. wide: every array's pieces of 8 lie on 16 bytes. */
int copy_args(bool write, const hearth_gpu_cache *c, const hearth_gpu_batch *b, const hearth_gpu_array *k,
              const hearth_gpu_array *v, int dev, CopyArgs &a, bool &wide) {
    if (!cache_ok(c) || !batch_ok(b) || dev < 0) return E_ARG;
    const bool latent = !c->v.data;
    const int n = b->n_tokens;
    if (v && !v->data && n) v = nullptr;
    if (!array_ok(k, n) || (v && !array_ok(v, n)) || (!latent && !v)) return E_ARG;
    if (v && v->dtype != k->dtype) return E_ARG;
    a = {};
    a.b = batch_of(*b, *c);
    a.n_pieces = v ? 2 : 1;
    int col = 0;
    wide = true;
    for (int i = 0; i < a.n_pieces; i++) {
        const hearth_gpu_array &x = i ? *v : *k;
        if (x.n_heads != c->n_heads || x.width % 32 || (!write && !apart(x, n))) return E_ARG;
        Piece &p = a.p[i];
        const int es = elem(x.dtype);
        p.arr = (uint8_t *)x.data; p.at = x.token_stride * es; p.ah = x.head_stride * es;
        p.rows = rows_of(i && !latent ? c->v : c->k, c->dtype);
        p.col = latent ? col : 0; p.width = x.width; p.row_width = c->width; p.heads = x.n_heads;
        col += x.width;
        if (!latent && x.width != c->width) return E_ARG;
        a.octs += p.heads * (p.width / 8);
        wide = wide && on16(x);
    }
    if (latent && (col != c->width || (v && c->n_heads != 1))) return E_ARG;
    if (!a.b.n_seqs) a.b.max_q = 0;
    return OK;
}

int copy_call(bool write, const hearth_gpu_cache *c, const hearth_gpu_batch *b, const hearth_gpu_array *k,
              const hearth_gpu_array *v, int dev, void *stream) {
    CopyArgs a;
    bool wide;
    if (const int rc = copy_args(write, c, b, k, v, dev, a, wide)) return rc;
    if (!a.b.max_q) return OK;
    if (copy_groups(a) > MAX_COPY_GROUPS) return E_ARG;
    if (hipPeekAtLastError() != hipSuccess) return E_IO;
    DeviceGuard g(dev);
    if (!g.ok) return no_device();
    if (write) kv_append(a, k->dtype, c->dtype, wide, (hipStream_t)stream);
    else kv_read(a, k->dtype, c->dtype, wide, (hipStream_t)stream);
    return finish();
}

/* arguments that both attentions share */
bool attend_shape_ok(const hearth_gpu_cache *c, const hearth_gpu_batch *b, int heads) {
    if (!cache_ok(c) || !batch_ok(b)) return false;
    if (heads < 1 || heads > MAX_HEADS || heads % c->n_heads) return false;
    const Batch o = batch_of(*b, *c);
    if ((int64_t)o.max_q * heads > (1 << 26) || o.kv_cap > MAX_ROWS) return false;
    if (!c->v.data && ((int64_t)o.max_q * heads + 63) / 64 * o.n_seqs > MAX_LATENT_TILES) return false;
    if (c->v.data) return c->width == 64 || c->width == 128 || c->width == 256;
    return c->width == 576 && c->n_heads == 1 && c->dtype != HEARTH_GPU_MX4;
}

int64_t part_bytes(const hearth_gpu_cache &c, const hearth_gpu_batch &b, int heads, Split &s) {
    const Batch o = batch_of(b, c);
    if (!o.n_seqs || !o.max_q) { s = {0x40000000, 1, false}; return 0; }
    s = attend_split(o.n_seqs, b.max_q, o.kv_cap, heads, c.n_heads, !c.v.data, c.dtype == HEARTH_GPU_MX4);
    const int64_t dv = c.v.data ? c.width : 512;
    return s.n == 1 ? 0 : (int64_t)o.n_tokens * heads * s.n * (dv + 2) * (int64_t)sizeof(float);
}

/* the split of an attention over chosen blocks, and its bytes; -1 for arguments that it refuses */
int64_t blocks_part_bytes(const hearth_gpu_cache *c, const hearth_gpu_batch *b, int heads, int top, int block, Split &s) {
    if (!attend_shape_ok(c, b, heads) || !c->v.data || top < 1 || top > (1 << 20) || !pow2(block) || block < 16 || block > c->page) return E_ARG;
    const Batch o = batch_of(*b, *c);
    if ((int64_t)top * block > MAX_ROWS || (int64_t)o.max_q * c->n_heads * ((heads / c->n_heads + 15) / 16) > MAX_COPY_GROUPS) return E_ARG;
    s = {0x40000000, 1, false};
    if (!o.n_seqs || !o.max_q) return 0;
    s = blocks_split(o.n_seqs, b->max_q, top * block, heads, c->n_heads);
    return s.n == 1 ? 0 : (int64_t)o.n_tokens * heads * s.n * (c->width + 2) * (int64_t)sizeof(float);
}

int attend_call(const hearth_gpu_cache *c, const hearth_gpu_batch *b, const hearth_gpu_array *q, const hearth_gpu_array *q_pe,
                const hearth_gpu_blocks *blocks, const hearth_gpu_array *out, float *lse, float scale, void *work, size_t work_bytes,
                int dev, void *stream) {
    if (!q || !attend_shape_ok(c, b, q->n_heads) || !array_ok(q, b->n_tokens) || !array_ok(out, b->n_tokens) || dev < 0) return E_ARG;
    const bool latent = q_pe != nullptr;
    if (latent != !c->v.data || (uintptr_t)lse % 4 || !std::isfinite(scale * 1.44269504088896340736f)) return E_ARG;
    if ((q->dtype != HEARTH_F16 && q->dtype != HEARTH_BF16) || out->dtype != q->dtype || !apart(*out, b->n_tokens)) return E_ARG;
    if (bits_of(c->dtype) == 16 && c->dtype != q->dtype) return E_ARG;
    const int width = latent ? 512 : c->width;
    if (q->width != width || out->width != width || out->n_heads != q->n_heads) return E_ARG;
    if (latent && (!array_ok(q_pe, b->n_tokens) || q_pe->dtype != q->dtype || q_pe->n_heads != q->n_heads || q_pe->width != 64)) return E_ARG;
    if (blocks && !blocks_ok(blocks, b->n_tokens, c->n_heads, false)) return E_ARG;
    Split s;
    const int64_t need = blocks ? blocks_part_bytes(c, b, q->n_heads, blocks->top, blocks->block, s) : part_bytes(*c, *b, q->n_heads, s);
    if (need < 0 || (need && ((uintptr_t)work % 16 || !work))) return E_ARG;
    if ((uint64_t)need > work_bytes) return E_CAPACITY;
    AttendArgs a{};
    a.b = batch_of(*b, *c);
    if (!a.b.n_seqs || !a.b.max_q) return OK;
    a.k = rows_of(c->k, c->dtype);
    if (!latent) a.v = rows_of(c->v, c->dtype);
    a.q = (const uint8_t *)q->data; a.qt = 2 * q->token_stride; a.qh = 2 * q->head_stride;
    a.out = (uint8_t *)out->data; a.ot = 2 * out->token_stride; a.oh = 2 * out->head_stride;
    if (latent) {
        a.q_pe = (const uint8_t *)q_pe->data; a.pt = 2 * q_pe->token_stride; a.ph = 2 * q_pe->head_stride;
    }
    a.lse = lse;
    a.heads = q->n_heads; a.kv_heads = c->n_heads; a.group = a.heads / a.kv_heads;
    a.scale2 = scale * 1.44269504088896340736f;
    a.chunk = s.chunk; a.n_splits = s.n;
    a.part = (float *)work;
    if (blocks) {
        a.chosen = blocks->chosen; a.ct = blocks->token_stride; a.ch = blocks->head_stride;
        a.top = blocks->top; a.block_shift = __builtin_ctz((unsigned)blocks->block);
    }
    if (hipPeekAtLastError() != hipSuccess) return E_IO;
    DeviceGuard g(dev);
    if (!g.ok) return no_device();
    if (latent) attend_latent(a, q->dtype, c->dtype, (hipStream_t)stream);
    else if (blocks) attend_blocks(a, q->dtype, c->dtype, c->width, (hipStream_t)stream);
    else attend(a, q->dtype, c->dtype, c->width, s.many, (hipStream_t)stream);
    return finish();
}

/* bytes of scores, or -1 for arguments that the selection refuses */
int64_t score_bytes(const hearth_gpu_bounds *s, const hearth_gpu_batch *b) {
    if (!bounds_ok(s) || !batch_ok(b)) return E_ARG;
    const Batch o = batch_of(*b, s->n_pages, s->block * s->blocks);
    if (o.kv_cap > MAX_ROWS || (int64_t)o.max_q * s->n_heads > MAX_PICKS) return E_ARG;
    if (!o.n_seqs || !o.max_q) return 0;
    int64_t bytes;   /* up to 2^71: few query rows a sequence say nothing of all tokens */
    if (__builtin_mul_overflow((int64_t)o.n_tokens * s->n_heads, blocks_of(o.kv_cap, s->block) * (int64_t)sizeof(float), &bytes)) return E_ARG;
    return bytes;
}

} // namespace

extern "C" {

HEARTH_API int hearth_gpu_rope(const hearth_gpu_array *x, const hearth_gpu_array *out, const hearth_gpu_array *k,
                               const hearth_gpu_array *k_out, int n_tokens, const void *pos, int pos64,
                               const double *freqs, int n_freqs, int offset, int interleaved, int inverse,
                               double factor, int dev, void *stream) {
    if (k && !k->data && n_tokens) k = nullptr;
    if (k_out && !k_out->data && n_tokens) k_out = nullptr;
    if (!array_ok(x, n_tokens) || !array_ok(out, n_tokens) || !k != !k_out || n_tokens < 0 || (n_tokens && !pos) || !freqs || dev < 0) return E_ARG;
    if (n_freqs < 1 || n_freqs > 512 || offset < 0 || (int64_t)offset + 2 * n_freqs > x->width) return E_ARG;
    if ((int64_t)x->n_heads * x->width > MAX_ROPE_ROW || (k && (int64_t)k->n_heads * x->width > MAX_ROPE_ROW)) return E_ARG;
    if (k && n_tokens && (k->data == x->data || k_out->data == out->data)) return E_ARG;
    if (!std::isfinite(factor) || (uintptr_t)pos % (pos64 ? 8 : 4) || (uintptr_t)freqs % 8) return E_ARG;
    RopeArgs a{};
    a.in_place = true;
    a.n_pairs = k ? 2 : 1;
    for (int i = 0; i < a.n_pairs; i++) {
        const hearth_gpu_array *s = i ? k : x, *d = i ? k_out : out;
        if (!array_ok(s, n_tokens) || !array_ok(d, n_tokens) || s->dtype != x->dtype || d->dtype != x->dtype || s->width != x->width ||
            d->width != x->width || s->n_heads != d->n_heads || !apart(*d, n_tokens)) return E_ARG;
        const int64_t es = elem(s->dtype);
        a.p[i] = {(const uint8_t *)s->data, (uint8_t *)d->data, s->token_stride * es, s->head_stride * es,
                  d->token_stride * es, d->head_stride * es, s->n_heads};
        const bool same = s->data == d->data;
        if (same && (s->token_stride != d->token_stride || s->head_stride != d->head_stride)) return E_ARG;
        a.in_place = a.in_place && same;
    }
    a.pos = pos; a.pos64 = pos64 != 0; a.freqs = freqs;
    a.n_tokens = n_tokens; a.width = x->width; a.n_freqs = n_freqs; a.offset = offset; a.interleaved = interleaved != 0;
    a.factor = (float)factor; a.sign = inverse ? -1.0f : 1.0f;
    if (!n_tokens) return OK;
    if (hipPeekAtLastError() != hipSuccess) return E_IO;
    DeviceGuard g(dev);
    if (!g.ok) return no_device();
    rope(a, x->dtype, (hipStream_t)stream);
    return finish();
}

HEARTH_API int hearth_gpu_kv_append(const hearth_gpu_cache *c, const hearth_gpu_batch *b, const hearth_gpu_array *k,
                                    const hearth_gpu_array *v, int dev, void *stream) {
    return copy_call(true, c, b, k, v, dev, stream);
}

HEARTH_API int hearth_gpu_kv_append_rotated(const hearth_gpu_cache *c, const hearth_gpu_batch *b, const hearth_gpu_array *q,
                                            const hearth_gpu_array *q_out, const hearth_gpu_array *k, const hearth_gpu_array *v,
                                            const void *pos, int pos64, const double *freqs, int n_freqs, int offset,
                                            int interleaved, double factor, int dev, void *stream) {
    RotatedArgs a{};
    bool wide;
    if (const int rc = copy_args(true, c, b, k, v, dev, a.c, wide)) return rc;
    const int n = b->n_tokens;
    if (q && !q->data && n) q = nullptr;
    if (q_out && !q_out->data && n) q_out = nullptr;
    const bool latent = !c->v.data;
    if (!q != !q_out || (latent && a.c.n_pieces != 2) || !freqs) return E_ARG;
    a.rotated = latent ? 1 : 0;
    a.width = a.c.p[a.rotated].width;
    if (n_freqs < 1 || n_freqs > 512 || offset < 0 || (int64_t)offset + 2 * n_freqs > a.width) return E_ARG;
    if (!std::isfinite(factor) || (uintptr_t)pos % (pos64 ? 8 : 4) || (uintptr_t)freqs % 8) return E_ARG;
    if (q) {
        if (!array_ok(q, n) || !array_ok(q_out, n) || q->dtype != k->dtype || q_out->dtype != q->dtype || q->width != a.width ||
            q_out->width != a.width || q_out->n_heads != q->n_heads || !apart(*q_out, n)) return E_ARG;
        if ((int64_t)q->n_heads * q->width > MAX_ROPE_ROW) return E_ARG;
        a.in_place = q->data == q_out->data;
        if (a.in_place && (q->token_stride != q_out->token_stride || q->head_stride != q_out->head_stride)) return E_ARG;
        if (n && (q_out->data == k->data || (v && q_out->data == v->data))) return E_ARG;   /* read by some threads, written by others */
        const int64_t es = elem(q->dtype);
        a.q = {(const uint8_t *)q->data, (uint8_t *)q_out->data, q->token_stride * es, q->head_stride * es,
               q_out->token_stride * es, q_out->head_stride * es, q->n_heads};
    }
    if ((int64_t)c->n_heads * c->width > MAX_ROPE_ROW / 2 || a.c.b.max_q > MAX_COPY_GROUPS) return E_ARG;
    a.pos = pos; a.pos64 = pos64 != 0; a.freqs = freqs; a.n_freqs = n_freqs; a.offset = offset;
    a.interleaved = interleaved != 0; a.factor = (float)factor;
    if (!a.c.b.max_q) return OK;
    if (hipPeekAtLastError() != hipSuccess) return E_IO;
    DeviceGuard g(dev);
    if (!g.ok) return no_device();
    kv_append_rotated(a, k->dtype, c->dtype, wide, (hipStream_t)stream);
    return finish();
}

HEARTH_API int hearth_gpu_kv_read(const hearth_gpu_cache *c, const hearth_gpu_batch *b, const hearth_gpu_array *k,
                                  const hearth_gpu_array *v, int dev, void *stream) {
    return copy_call(false, c, b, k, v, dev, stream);
}

HEARTH_API int64_t hearth_gpu_attend_workspace(const hearth_gpu_cache *c, const hearth_gpu_batch *b, int n_heads) {
    if (!attend_shape_ok(c, b, n_heads)) return E_ARG;
    Split s;
    return part_bytes(*c, *b, n_heads, s);
}

HEARTH_API int hearth_gpu_attend(const hearth_gpu_cache *c, const hearth_gpu_batch *b, const hearth_gpu_array *q,
                                 const hearth_gpu_array *out, float *lse, float scale, void *work, size_t work_bytes,
                                 int dev, void *stream) {
    return attend_call(c, b, q, nullptr, nullptr, out, lse, scale, work, work_bytes, dev, stream);
}

HEARTH_API int hearth_gpu_attend_latent(const hearth_gpu_cache *c, const hearth_gpu_batch *b,
                                        const hearth_gpu_array *q, const hearth_gpu_array *q_pe,
                                        const hearth_gpu_array *out, float *lse, float scale, void *work,
                                        size_t work_bytes, int dev, void *stream) {
    if (!q_pe) return E_ARG;
    return attend_call(c, b, q, q_pe, nullptr, out, lse, scale, work, work_bytes, dev, stream);
}

HEARTH_API int hearth_gpu_key_bounds(const hearth_gpu_cache *c, const hearth_gpu_batch *b, const hearth_gpu_bounds *s, int dev,
                                     void *stream) {
    if (!cache_ok(c) || !batch_ok(b) || !bounds_ok(s) || dev < 0) return E_ARG;
    if (!c->v.data || s->n_pages != c->n_pages || s->n_heads != c->n_heads || s->width != c->width || s->block * s->blocks != c->page) return E_ARG;
    BoundsArgs a{};
    a.b = batch_of(*b, *c);
    if (!a.b.n_seqs || !a.b.max_q) return OK;
    a.k = rows_of(c->k, c->dtype);
    a.s = bounds_of(*s);
    a.heads = c->n_heads;
    a.per_seq = std::min<int64_t>((int64_t)a.b.max_q / s->block + 2, blocks_of(a.b.kv_cap, s->block));
    if (a.per_seq * a.heads > MAX_COPY_GROUPS) return E_ARG;
    if (!a.per_seq) return OK;
    if (hipPeekAtLastError() != hipSuccess) return E_IO;
    DeviceGuard g(dev);
    if (!g.ok) return no_device();
    key_bounds(a, c->dtype, c->width, (hipStream_t)stream);
    return finish();
}

HEARTH_API int64_t hearth_gpu_select_workspace(const hearth_gpu_bounds *s, const hearth_gpu_batch *b) { return score_bytes(s, b); }

HEARTH_API int hearth_gpu_select_blocks(const hearth_gpu_bounds *s, const hearth_gpu_batch *b, const hearth_gpu_array *q,
                                        const hearth_gpu_blocks *out, int first, int last, void *work, size_t work_bytes, int dev,
                                        void *stream) {
    const int64_t need = score_bytes(s, b);
    if (need < 0 || dev < 0 || !array_ok(q, b->n_tokens) || !blocks_ok(out, b->n_tokens, s->n_heads, true)) return E_ARG;
    if ((q->dtype != HEARTH_F16 && q->dtype != HEARTH_BF16) || q->width != s->width || q->n_heads % s->n_heads || out->block != s->block) return E_ARG;
    const int group = q->n_heads / s->n_heads;
    if (group > select_group_limit() || first < 0 || last < 1 || first > out->top || last > out->top) return E_ARG;
    SelectArgs a{};
    a.b = batch_of(*b, s->n_pages, s->block * s->blocks);
    /* blocks that a tree's node keeps: from the one of the call's first token on */
    const int64_t tail = b->mask ? std::max<int64_t>(last, a.b.max_q ? blocks_of(a.b.max_q - 1, s->block) + 1 : 0) : last;
    if (first + tail > out->top) return E_ARG;
    if (!a.b.n_seqs || !a.b.max_q) return OK;
    if (need && (!work || (uintptr_t)work % 16)) return E_ARG;
    if ((uint64_t)need > work_bytes) return E_CAPACITY;
    a.s = bounds_of(*s);
    a.q = (const uint8_t *)q->data; a.qt = 2 * q->token_stride; a.qh = 2 * q->head_stride;
    a.chosen = out->chosen; a.ct = out->token_stride; a.ch = out->head_stride;
    a.kv_heads = s->n_heads; a.group = group; a.top = out->top; a.first = first; a.last = last;
    a.score = (float *)work;
    a.ld_score = blocks_of(a.b.kv_cap, s->block);
    score_split(a);
    if (hipPeekAtLastError() != hipSuccess) return E_IO;
    DeviceGuard g(dev);
    if (!g.ok) return no_device();
    select_blocks(a, q->dtype, s->width, (hipStream_t)stream);
    return finish();
}

HEARTH_API int hearth_gpu_attend_blocks(const hearth_gpu_cache *c, const hearth_gpu_batch *b, const hearth_gpu_array *q,
                                        const hearth_gpu_blocks *blocks, const hearth_gpu_array *out, float *lse, float scale,
                                        void *work, size_t work_bytes, int dev, void *stream) {
    if (!blocks) return E_ARG;
    return attend_call(c, b, q, nullptr, blocks, out, lse, scale, work, work_bytes, dev, stream);
}

HEARTH_API int64_t hearth_gpu_attend_blocks_workspace(const hearth_gpu_cache *c, const hearth_gpu_batch *b, int n_heads, int top, int block) {
    Split s;
    return blocks_part_bytes(c, b, n_heads, top, block, s);
}

} // extern "C"
