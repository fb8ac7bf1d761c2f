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
constexpr int64_t MAX_ROPE_ROW = 1 << 24;           /* elements of a token: four of them count within 31 bits */

bool pow2(int x) { return x > 0 && (x & (x - 1)) == 0; }

bool rows_ok(const hearth_gpu_rows &r, const hearth_gpu_cache &c) {
    const bool mx = c.dtype == HEARTH_GPU_MX8;
    const int es = mx ? 1 : 2;
    const int64_t block = (int64_t)c.page * c.width;
    if (!r.data || (uintptr_t)r.data % 16) return false;
    if (r.head_stride < (c.n_heads > 1 ? block : 0) || r.page_stride < (c.n_pages > 1 ? block : 0)) return false;
    if (r.head_stride > MAX_STRIDE || r.page_stride > MAX_STRIDE) return false;
    if (r.head_stride * es % 16 || r.page_stride * es % 16) return false;
    if (!mx) return true;
    if (!r.scales || r.scale_head_stride < (c.n_heads > 1 ? block / MX_BLOCK : 0) || r.scale_head_stride > MAX_STRIDE) return false;
    return r.scale_page_stride >= (c.n_pages > 1 ? block / MX_BLOCK : 0) && r.scale_page_stride <= MAX_STRIDE;
}

bool cache_ok(const hearth_gpu_cache *c) {
    if (!c || (c->dtype != HEARTH_F16 && c->dtype != HEARTH_BF16 && c->dtype != HEARTH_GPU_MX8)) return false;
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
    if (!x || (n && !x->data) || !elem(x->dtype) || x->n_heads < 1 || x->n_heads > 65536 || x->width < 1 || x->width > 65536) return false;
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
    const int64_t es = dtype == HEARTH_GPU_MX8 ? 1 : 2;
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

int finish() { return hipGetLastError() == hipSuccess ? OK : E_IO; }   /* this call's launches only */

/* The call's own error, read so that the thread's next call does not take it for the caller's. */
int no_device() {
    (void)hipGetLastError();
    return E_IO;
}

int copy_call(bool write, const hearth_gpu_cache *c, const hearth_gpu_batch *b, const hearth_gpu_array *k,
              const hearth_gpu_array *v, int dev, void *stream) {
    if (!cache_ok(c) || !batch_ok(b) || dev < 0) return E_ARG;
    const bool latent = !c->v.data;
    const int n = b->n_tokens;
    if (v && !v->data && n) v = nullptr;
    if (!array_ok(k, n) || (v && !array_ok(v, n)) || (!latent && !v)) return E_ARG;
    if (v && v->dtype != k->dtype) return E_ARG;
    CopyArgs a{};
    a.b = batch_of(*b, *c);
    a.n_pieces = v ? 2 : 1;
    int col = 0;
    bool wide = true;
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
    if (!a.b.n_seqs || !a.b.max_q) return OK;
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
    if (heads < 1 || heads % c->n_heads) return false;
    const Batch o = batch_of(*b, *c);
    if ((int64_t)o.max_q * heads > (1 << 26) || o.kv_cap > MAX_ROWS) return false;
    if (!c->v.data && ((int64_t)o.max_q * heads + 63) / 64 * o.n_seqs > MAX_LATENT_TILES) return false;
    if (c->v.data) return c->width == 64 || c->width == 128 || c->width == 256;
    return c->width == 576 && c->n_heads == 1;
}

int64_t part_bytes(const hearth_gpu_cache &c, const hearth_gpu_batch &b, int heads, Split &s) {
    const Batch o = batch_of(b, c);
    if (!o.n_seqs || !o.max_q) { s = {0x40000000, 1, false}; return 0; }
    s = attend_split(o.n_seqs, b.max_q, o.kv_cap, heads, c.n_heads, !c.v.data);
    const int64_t dv = c.v.data ? c.width : 512;
    return s.n == 1 ? 0 : (int64_t)o.n_tokens * heads * s.n * (dv + 2) * (int64_t)sizeof(float);
}

int attend_call(const hearth_gpu_cache *c, const hearth_gpu_batch *b, const hearth_gpu_array *q, const hearth_gpu_array *q_pe,
                const hearth_gpu_array *out, float *lse, float scale, void *work, size_t work_bytes, int dev, void *stream) {
    if (!q || !attend_shape_ok(c, b, q->n_heads) || !array_ok(q, b->n_tokens) || !array_ok(out, b->n_tokens) || dev < 0) return E_ARG;
    const bool latent = q_pe != nullptr;
    if (latent != !c->v.data || (uintptr_t)lse % 4 || !std::isfinite(scale * 1.44269504088896340736f)) return E_ARG;
    if ((q->dtype != HEARTH_F16 && q->dtype != HEARTH_BF16) || out->dtype != q->dtype || !apart(*out, b->n_tokens)) return E_ARG;
    if (c->dtype != HEARTH_GPU_MX8 && c->dtype != q->dtype) return E_ARG;
    const int width = latent ? 512 : c->width;
    if (q->width != width || out->width != width || out->n_heads != q->n_heads) return E_ARG;
    if (latent && (!array_ok(q_pe, b->n_tokens) || q_pe->dtype != q->dtype || q_pe->n_heads != q->n_heads || q_pe->width != 64)) return E_ARG;
    Split s;
    const int64_t need = part_bytes(*c, *b, q->n_heads, s);
    if (need && ((uintptr_t)work % 16 || !work)) return E_ARG;
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
    if (hipPeekAtLastError() != hipSuccess) return E_IO;
    DeviceGuard g(dev);
    if (!g.ok) return no_device();
    if (latent) attend_latent(a, q->dtype, c->dtype, (hipStream_t)stream);
    else attend(a, q->dtype, c->dtype, c->width, s.many, (hipStream_t)stream);
    return finish();
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
    return attend_call(c, b, q, nullptr, out, lse, scale, work, work_bytes, dev, stream);
}

HEARTH_API int hearth_gpu_attend_latent(const hearth_gpu_cache *c, const hearth_gpu_batch *b,
                                        const hearth_gpu_array *q, const hearth_gpu_array *q_pe,
                                        const hearth_gpu_array *out, float *lse, float scale, void *work,
                                        size_t work_bytes, int dev, void *stream) {
    if (!q_pe) return E_ARG;
    return attend_call(c, b, q, q_pe, out, lse, scale, work, work_bytes, dev, stream);
}

} // extern "C"
