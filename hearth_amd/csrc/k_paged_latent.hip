/*
 * k_paged_latent.hip — absorbed latent attention over a paged cache: every query head of a token
 * reads the same rows [c (512) | pe (64)], s = scale (q . c + q_pe . pe), out = softmax(s) c.
 *
 * With 2 x 1088 flops a (column, row) against 1152 bytes a row it is bound by the matrix units
 * from about 150 columns a sequence on, and by the rows' bytes below. The products run transposed
 * as in k_paged_attn.hip (S^T = K Q^T, O^T = C^T P^T, 16 x 16 x 32): a wave keeps 16 columns'
 * queries (72 registers) and sums (128) and takes 32 rows of a step of 64; four waves side by
 * side cover 64 columns, the other four the step's other 32 rows (joined at the end through LDS).
 * The rows of a step lie in LDS once, row-major, for both products: the score reads them along
 * the row, the sum through the transposing LDS load. Of the 16-byte pieces of a row, the eight of
 * each 128 bytes are exchanged by row (piece p of row r at p ^ swz(r)), so that neither read meets
 * a bank conflict although a row is 1152 bytes. 16-bit rows go from memory to LDS directly, 8-bit
 * rows through registers, where they become 16-bit ones; the next step's are in flight meanwhile.
 */
#include "hx_paged.h"

#include <algorithm>

namespace hxp {

namespace {

constexpr int LW = 576, LC = 512;                   /* row width (latent, rotated part), latent */
constexpr int L_WAVES = 8, L_THREADS = 64 * L_WAVES, L_COLS = 64, L_ROWS = 64;
constexpr int L_PIECES = LW / 8;                    /* 16-byte pieces of a 16-bit row */
constexpr int L_TILE = L_ROWS * LW * 2;             /* bytes of a step in LDS */

__device__ __forceinline__ int swz(int r) {
    const int k = r >> 1 & 7;
    return (k & 3) << 1 | k >> 2;
}
__device__ __forceinline__ int piece_at(int r, int p) { return (r * L_PIECES + (p ^ swz(r))) * 16; }

typedef short s4v __attribute__((ext_vector_type(4)));

/* four rows of one element each a lane (transposing LDS load): lane i of 16 gives the address of 4
 * elements of row i / 4 and gets element i of the four rows */
__device__ __forceinline__ u2 read_tr(const uint8_t *p) {
    return __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v *)p));
}

template <class T, bool MX>
__global__ __launch_bounds__(L_THREADS, 2) void k_attend_latent(AttendArgs a) {
    using v8 = typename T::v8;
    constexpr int KS = LW / 32, DT = LC / 16;
    constexpr float NINF = -__builtin_huge_valf();
    constexpr int N = MX ? (L_ROWS * LW / 16 + L_THREADS - 1) / L_THREADS : L_ROWS * L_PIECES / L_THREADS;   /* pieces a thread brings in */
    __shared__ __align__(16) uint8_t lds[2][L_TILE];
    __shared__ float lds_m[2][L_COLS], lds_l[2][L_COLS];

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int g = lane >> 4, lc = lane & 15, wc = wave & 3, wt = wave >> 2;
    /* the column tiles of one (sequence, split) follow each other on one XCD (workgroup i runs on
     * XCD i % 8), whose L2 then holds their rows */
    const int tiles = (int)(((int64_t)a.b.max_q * a.heads + L_COLS - 1) / L_COLS);
    const int pair = (int)(blockIdx.x / (8 * tiles)) * 8 + (int)(blockIdx.x & 7), tile = (int)(blockIdx.x >> 3) % tiles;
    if (pair >= a.b.n_seqs * a.n_splits) return;
    const int seq = pair / a.n_splits, sp = pair % a.n_splits;
    const Seq q = seq_of(a.b, seq);
    const int cols = min(q.n, a.b.max_q) * a.heads;
    if (tile * L_COLS >= cols) return;
    const int n_sp = max(1, (q.kv + a.chunk - 1) / a.chunk);
    if (sp >= n_sp) return;

    const int c = tile * L_COLS + 16 * wc + lc;
    const bool on = c < cols;
    const int tok = on ? c / a.heads : 0, head = on ? c % a.heads : 0;
    const int lim = !on ? 0 : a.b.mask ? min(q.base, q.kv) : min(q.base + tok + 1, q.kv);
    v8 qf[KS];
    {
        const uint8_t *qp = a.q + (int64_t)(q.q0 + tok) * a.qt + (int64_t)head * a.qh;
        const uint8_t *pp = a.q_pe + (int64_t)(q.q0 + tok) * a.pt + (int64_t)head * a.ph;
#pragma unroll
        for (int i = 0; i < KS; i++) {
            const int d = 32 * i + 8 * g;
            const unsigned short *p = d < LC ? (const unsigned short *)qp + d : (const unsigned short *)pp + (d - LC);
            u4 w = {0, 0, 0, 0};
            if (on) {
                if (a.aligned) w = *(const u4 *)p;
                else
#pragma unroll
                    for (int k = 0; k < 4; k++) w[k] = p[2 * k] | (unsigned)p[2 * k + 1] << 16;
            }
            qf[i] = __builtin_bit_cast(v8, w);
        }
    }
    const int t_last = min(cols - 1, tile * L_COLS + L_COLS - 1) / a.heads;
    const int hi = min(min(q.kv, a.b.mask ? q.kv : q.base + t_last + 1), (sp + 1) * a.chunk);
    const int full = a.b.mask ? q.base : q.base + tile * L_COLS / a.heads + 1;
    const int lo = sp * a.chunk;
    /* which of the 64 rows from t0 on this lane's column attends (where their pages exist) */
    const unsigned long long *words = a.b.mask && on ? a.b.mask + (int64_t)(q.q0 + tok) * a.b.mask_words : nullptr;
    auto attended = [&](int t0) { return step_mask(t0, lim, hi, q.base, words, a.b.mask_words); };

    f4 acc[DT];
#pragma unroll
    for (int i = 0; i < DT; i++) acc[i] = (f4){0, 0, 0, 0};
    float m = NINF, l = 0.0f;

    const int *pages = a.b.pages + (int64_t)seq * a.b.ld_pages;
    const int rmask = (1 << a.b.page_shift) - 1;
    int pid[4];
    auto load_pages = [&](int t0) {
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int t = t0 + 16 * u;
            const int id = t < hi ? word_of(pages, t >> a.b.page_shift) : -1;
            pid[u] = page_ok(a.b, id) ? id : -1;
        }
    };
    auto page_of = [&](int r) {
        const int u = r >> 4;
        return u == 0 ? pid[0] : u == 1 ? pid[1] : u == 2 ? pid[2] : pid[3];
    };
    auto have = [&] { return (pid[0] >= 0 ? 1u : 0u) | (pid[1] >= 0 ? 2u : 0u) | (pid[2] >= 0 ? 4u : 0u) | (pid[3] >= 0 ? 8u : 0u); };
    auto edge_at = [&](int t0, unsigned h) { return !(t0 + L_ROWS <= full && t0 + L_ROWS <= hi && h == 15u); };

    u4 sw[MX ? N : 1];
    unsigned ss[MX ? N : 1];
    /* the loads of the step at t0: to LDS (16-bit; rows that are not there take the cache's first
     * row and are cleared in settle) or to registers (8-bit) */
    auto load = [&](int t0, int buf) {
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));   /* the pieces' places are worked out anew: held, they cost registers */
        if constexpr (MX) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int idx = tid + L_THREADS * i, r = idx / (LW / 16), p = idx % (LW / 16);
                sw[i] = (u4){0, 0, 0, 0};
                ss[i] = 127;
                const int id = page_of(r);
                if (idx < L_ROWS * (LW / 16) && id >= 0 && t0 + r < hi) {
                    const int row = (t0 + r) & rmask;
                    sw[i] = *(const u4 *)(a.k.data + (int64_t)id * a.k.page_stride + row * LW + 16 * p);
                    ss[i] = a.k.scales[(int64_t)id * a.k.scale_page_stride + row * (LW / MX_BLOCK) + (p >> 1)];
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int at = (wave * N + i) * 64, idx = at + (tid & 63), r = idx / L_PIECES, p = idx % L_PIECES;
                const int id = page_of(r);
                const bool ok = id >= 0 && t0 + r < hi;
                const uint8_t *src = a.k.data + (ok ? (int64_t)id * a.k.page_stride + (int64_t)(((t0 + r) & rmask) * LW + 8 * (p ^ swz(r))) * 2 : 0);
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)src,
                                                 (__attribute__((address_space(3))) void *)(lds[buf] + at * 16), 16, 0, 0);
            }
        }
    };
    /* The loaded step made ready in LDS; in edge steps true where a latent element that some
     * column does not attend is infinite or NaN. */
    auto settle = [&](int t0, int buf, unsigned h, bool edge) {
        bool odd = false;
        if constexpr (MX) {
            int tid = threadIdx.x;
            asm volatile("" : "+v"(tid));
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int idx = tid + L_THREADS * i, r = idx / (LW / 16), p = idx % (LW / 16);
                if (idx < L_ROWS * (LW / 16)) {
                    const float f = mx_scale(ss[i]);
                    u4 w[2];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        w[k >> 1][2 * (k & 1)] = T::template from_mx8<false>(sw[i][k], f);
                        w[k >> 1][2 * (k & 1) + 1] = T::template from_mx8<true>(sw[i][k], f);
                    }
#pragma unroll
                    for (int k = 0; k < 2; k++) *(u4 *)(lds[buf] + piece_at(r, 2 * p + k)) = w[k];
                    if (edge)
#pragma unroll
                        for (int k = 0; k < 8; k++) odd = odd || T::odd(w[k >> 2][k & 3]);
                }
            }
        } else {
            __builtin_amdgcn_s_waitcnt(0x0f70);   /* vmcnt(0): this thread's pieces have arrived */
            if (edge)
#pragma unroll 1
                for (int i = 0; i < N; i++) {
                    const int idx = (wave * N + i) * 64 + lane, r = idx / L_PIECES;
                    u4 *p = (u4 *)(lds[buf] + idx * 16);
                    if (!(h >> (r >> 4) & 1) || t0 + r >= hi) *p = (u4){0, 0, 0, 0};
                    else {
                        const u4 w = *p;
                        odd = odd || T::odd(w[0]) || T::odd(w[1]) || T::odd(w[2]) || T::odd(w[3]);
                    }
                }
        }
        return odd && t0 + L_ROWS > full;
    };

    unsigned have_now = 0, have_next = 0;
    bool odd_now = false, odd_next = false, odd_any = false;
    if (lo < hi) {
        load_pages(lo);
        have_next = have();
        load(lo, 0);
        odd_next = settle(lo, 0, have_next, edge_at(lo, have_next));
        if (lo + L_ROWS < hi) load_pages(lo + L_ROWS);
    }
    __syncthreads();

    /* Byte addresses in a step's tile. A row is nine times 128 bytes, so the exchange of pieces is
     * an exclusive or with a constant: scores read row 16 u + lc, pieces 4 i + g; sums read rows
     * 4 g .. 4 g + 3 of either tile of 16, elements 16 i .. 16 i + 15 */
    const int r0 = 32 * wt, ra = r0 + 4 * g + (lc >> 2);
    const int k_at[2] = {piece_at(r0 + lc, g), piece_at(r0 + 16 + lc, g)};
    const int v_at[2] = {piece_at(ra, lc >> 1 & 1) + 8 * (lc & 1), piece_at(ra + 16, lc >> 1 & 1) + 8 * (lc & 1)};
    int buf = 0;
    for (int t0 = lo; t0 < hi; t0 += L_ROWS, buf ^= 1) {
        const bool more = t0 + L_ROWS < hi;
        have_now = have_next;
        odd_now = odd_next;
        if (more) {
            have_next = have();
            load(t0 + L_ROWS, buf ^ 1);
            if (t0 + 2 * L_ROWS < hi) load_pages(t0 + 2 * L_ROWS);
        }
        f4 s[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
        const uint8_t *tl = lds[buf];
#pragma unroll
        for (int i = 0; i < KS; i++)
#pragma unroll
            for (int u = 0; u < 2; u++)
                s[u] = T::mfma16(*(const v8 *)(tl + (k_at[u] ^ 64 * (i & 1)) + 128 * (i >> 1)), qf[i], s[u]);

        const bool edge = edge_at(t0, have_now);
        float x[8], mx = NINF;
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = s[j >> 2][j & 3] * a.scale2;
        if (edge) {
            const unsigned long long vis = (attended(t0) & group_rows(have_now)) >> (r0 + 4 * g);
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = vis >> (16 * (j >> 2) + (j & 3)) & 1 ? x[j] : NINF;
            if (__syncthreads_or(odd_now)) {
                /* an infinity or NaN among rows that some columns do not attend would reach them as
                 * 0 * inf: the scores are done with the rows, so it is taken out of LDS and added
                 * at the end to the columns that attend it */
                odd_any = true;
                for (int i = threadIdx.x; i < L_TILE / 4; i += L_THREADS) {
                    unsigned *p = (unsigned *)lds[buf] + i;
                    *p = T::clean(*p);
                }
                __syncthreads();
            }
        }
#pragma unroll
        for (int j = 0; j < 8; j++) mx = fmaxf(mx, x[j]);
        mx = fmaxf(m, max16(max32(mx)));
        const float ms = mx == NINF ? 0.0f : mx;
        if (__any(mx > m)) {
            const float al = exp2_hw(m - ms);
            l *= al;
#pragma unroll
            for (int i = 0; i < DT; i++) acc[i] *= al;
            m = mx;
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            x[j] = exp2_hw(x[j] - ms);
            l += x[j];
        }
        const u4 pw = {T::pack(x[0], x[1]), T::pack(x[2], x[3]), T::pack(x[4], x[5]), T::pack(x[6], x[7])};
        const v8 pf = __builtin_bit_cast(v8, pw);
#pragma unroll
        for (int i = 0; i < DT; i++) {
            const u2 va = read_tr(tl + (v_at[0] ^ 32 * (i & 3)) + 128 * (i >> 2));
            const u2 vb = read_tr(tl + (v_at[1] ^ 32 * (i & 3)) + 128 * (i >> 2));
            acc[i] = T::mfma16(__builtin_bit_cast(v8, (u4){va[0], va[1], vb[0], vb[1]}), pf, acc[i]);
        }
        if (more) odd_next = settle(t0 + L_ROWS, buf ^ 1, have_next, edge_at(t0 + L_ROWS, have_next));
        __syncthreads();
    }
    /* the two halves of the rows together, through the steps' LDS */
    l = sum16(sum32(l));
    if (g == 0) { lds_m[wt][16 * wc + lc] = m; lds_l[wt][16 * wc + lc] = l; }
    __syncthreads();
    const float m0 = lds_m[0][16 * wc + lc], m1 = lds_m[1][16 * wc + lc];
    const float M = fmaxf(m0, m1);
    const float f0 = m0 == NINF ? 1.0f : exp2_hw(m0 - M), f1 = m1 == NINF ? 1.0f : exp2_hw(m1 - M);
    const float L = lds_l[0][16 * wc + lc] * f0 + lds_l[1][16 * wc + lc] * f1;
    f4 *half = (f4 *)lds[0] + wc * (DT * 64);     /* 4 x 32 KiB of the 144 KiB */
    if (wt == 1) {
#pragma unroll
        for (int i = 0; i < DT; i++) half[i * 64 + lane] = acc[i] * f1;
    }
    __syncthreads();
    if (odd_any) {   /* what was taken out of LDS above */
#pragma unroll 1
        for (int t = max(lo, full / L_ROWS * L_ROWS); t < hi; t++) {
            const int id = word_of(pages, t >> a.b.page_shift);
            if (!page_ok(a.b, id) || !(attended(t) & 1)) continue;
            const uint8_t *row = a.k.data + (int64_t)id * a.k.page_stride + (int64_t)(t & rmask) * (LW * (MX ? 1 : 2));
            const uint8_t *sc = MX ? a.k.scales + (int64_t)id * a.k.scale_page_stride + (t & rmask) * (LW / MX_BLOCK) : nullptr;
#pragma unroll 1
            for (int e = 0; e < DT / 2 * 4; e++) {
                const int i = wt * (DT / 2) + (e >> 2), j = e & 3;
                const unsigned v = row_elem<T, MX>(row, sc, 16 * i + 4 * g + j);
                if (T::odd(v)) ((float *)&half[i * 64 + lane])[j] += T::wide(v);
            }
        }
        __syncthreads();
    }
    if (wt == 1 || !on) return;
    const int64_t row = (int64_t)(q.q0 + tok) * a.heads + head;
    if (n_sp == 1) {
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        uint8_t *out = a.out + (int64_t)(q.q0 + tok) * a.ot + (int64_t)head * a.oh;
#pragma unroll
        for (int i = 0; i < DT; i++) {
            const f4 o = (acc[i] * f0 + half[i * 64 + lane]) * inv;
            uint8_t *p = out + 2 * (16 * i + 4 * g);
            if (a.aligned) *(u2 *)p = (u2){T::pack(o[0], o[1]), T::pack(o[2], o[3])};
            else
#pragma unroll
                for (int j = 0; j < 4; j++) ((typename T::e *)p)[j] = (typename T::e)o[j];
        }
        if (a.lse && g == 0) a.lse[row] = L == 0.0f ? NINF : (M + __log2f(L)) * 0.69314718055994531f;
    } else {
        float *po = a.part + (row * a.n_splits + sp) * LC;
        if (!(L == 0.0f))
#pragma unroll
            for (int i = 0; i < DT; i++) *(f4 *)(po + 16 * i + 4 * g) = acc[i] * f0 + half[i * 64 + lane];
        if (g == 0) {
            float *ml = a.part + (int64_t)a.b.n_tokens * a.heads * a.n_splits * LC + (row * a.n_splits + sp) * 2;
            ml[0] = M;
            ml[1] = L;
        }
    }
}

template <class T, bool MX>
void latent_t(const AttendArgs &a, hipStream_t st) {
    const int64_t tiles = ((int64_t)a.b.max_q * a.heads + L_COLS - 1) / L_COLS;
    const int64_t pairs = ((int64_t)a.b.n_seqs * a.n_splits + 7) / 8 * 8;
    hipLaunchKernelGGL((k_attend_latent<T, MX>), dim3((unsigned)(pairs * tiles)), dim3(L_THREADS), 0, st, a);
}

} // namespace

void latent_rows(const AttendArgs &a, int q_dtype, bool mx, hipStream_t st) {
    if (q_dtype == DT_BF16) mx ? latent_t<Bf16, true>(a, st) : latent_t<Bf16, false>(a, st);
    else mx ? latent_t<F16, true>(a, st) : latent_t<F16, false>(a, st);
}

} // namespace hxp
