/*
 * k_paged_many.hip — attention over a paged cache for many query rows a kv head: prompts and
 * draft trees.
 *
 * As in k_paged_attn.hip the products run transposed, S^T = K Q^T and O^T = V^T P^T, here with
 * the 32 x 32 x 16 matrix instruction: a wave owns 32 columns ((token, head) pairs of the kv
 * head's group), a lane half of one column's scores, so the softmax needs one exchange between
 * lanes l and l ^ 32, and the scores' registers, packed, are the second product's operand.
 * Four waves (128 columns) share 64 cache rows (32 of width 256) at a time through LDS, K and V as
 * they lie in memory: the scores read K along its rows, the sums read V through the transposing
 * LDS load. The 16-byte pieces of a row are exchanged by row (piece p of row r at p ^ swz(r)), so
 * that neither read meets a bank conflict. 16-bit rows go from memory to LDS directly, 8-bit rows
 * through registers, where they become 16-bit ones once for the four waves; the next step's are
 * in flight while this one is worked on (two buffers).
 * It is bound by the products and by what a wave does between them: 8000 tokens at the end of 16384
 * rows, 32 heads of 128 over 4 of 16 bits take 1640 us (990 TFLOP/s; 8-bit rows 1820), 2000 over 4048
 * 113 us (890); 4000 tokens of width 256 (one workgroup a unit) take 2720 us. A step of the two
 * workgroups of a unit takes 4000 cycles of which the matrix units are busy 54%; the exponentials,
 * maxima and packing of a wave take about as long as its products. Rows through registers into LDS
 * took 166 us for the 2000 tokens, page ids loaded where they are used 30 more.
 */
#include "hx_paged.h"

#include <algorithm>

namespace hxp {

namespace {

constexpr int MANY_WAVES = 4, MANY_COLS = 32 * MANY_WAVES;

template <int D>
struct Many {
    static constexpr int ROWS = D <= 128 ? 64 : 32;        /* cache rows of a step */
    static constexpr int PIECES = D / 8;                   /* 16-byte pieces of a row in LDS */
    static constexpr int TILE = ROWS * D * 2;              /* bytes of K or V of a step */
    static constexpr int GROUPS = ROWS / 16, TILES = ROWS / 32;

    /* Exchange of a row's pieces. Scores: 16 lanes read the same piece of 16 rows, which must fall
     * into 16 different 16-byte columns of the 256 bytes of banks. Sums: 32 lanes read 4 pieces
     * (aligned) of 4 rows, whose groups of 4 must differ. Rows of 128 bytes alternate between the
     * halves of the banks by themselves. */
    static __device__ __forceinline__ int swz(int r) {
        if constexpr (D == 64) { const int k = r >> 1 & 7; return (k & 1) << 2 | k >> 1; }
        else return (r & 3) << 2 | (r >> 2 & 3);
    }
    static __device__ __forceinline__ int at(int r, int p) { return (r * PIECES + (p ^ swz(r))) * 16; }
};

template <class T, bool MX, int D>
__global__ __launch_bounds__(64 * MANY_WAVES, D <= 128 ? 2 : 1) void k_attend_many(AttendArgs a) {
    using M = Many<D>;
    using v8 = typename T::v8;
    constexpr int KS = D / 16, DT = D / 32;
    constexpr float NINF = -__builtin_huge_valf();
    __shared__ __align__(16) uint8_t lds[2][2][M::TILE];   /* buffer, K or V */
    __shared__ int odd_flag;

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int half = lane >> 5, lc = lane & 31;
    int bx = blockIdx.x;
    const int kvh = bx % a.kv_heads;
    bx /= a.kv_heads;
    const int sp = bx % a.n_splits;
    const int tiles = gridDim.x / (a.kv_heads * a.n_splits), tile = tiles - 1 - bx / a.n_splits;   /* the longest first */
    const int seq = blockIdx.z;
    const Seq q = seq_of(a.b, seq);
    const int cols = min(q.n, a.b.max_q) * a.group;
    if (tile * MANY_COLS >= cols) return;
    const int n_sp = max(1, (q.kv + a.chunk - 1) / a.chunk);
    if (sp >= n_sp) return;

    const int c = tile * MANY_COLS + 32 * wave + lc;
    const bool on = c < cols;
    const int tok = on ? c / a.group : 0, head = kvh * a.group + (on ? c % a.group : 0);
    const int lim = !on ? 0 : a.b.mask ? min(q.base, q.kv) : min(q.base + tok + 1, q.kv);
    const unsigned flip = a.scale2 < 0.0f ? 0x80008000u : 0u;   /* a negative scale turns q's signs */
    const float scale2 = __builtin_fabsf(a.scale2);
    v8 qf[KS];
    {
        const uint8_t *qp = a.q + (int64_t)(q.q0 + tok) * a.qt + (int64_t)head * a.qh;
#pragma unroll
        for (int i = 0; i < KS; i++) {
            const unsigned short *p = (const unsigned short *)qp + 16 * i + 8 * half;
            u4 w = {0, 0, 0, 0};
            if (on) w = *(const u4_any *)p;
            qf[i] = __builtin_bit_cast(v8, w ^ flip);
        }
    }
    arrived();
    const int t_last = min(cols - 1, tile * MANY_COLS + MANY_COLS - 1) / a.group;
    const int hi = min(min(q.kv, a.b.mask ? q.kv : q.base + t_last + 1), (sp + 1) * a.chunk);
    const int full = a.b.mask ? q.base : q.base + tile * MANY_COLS / a.group + 1;
    const int lo = sp * a.chunk;

    /* which of the 64 rows from t0 on this lane's column attends (where their pages exist) */
    const unsigned long long *words = a.b.mask && on ? a.b.mask + (int64_t)(q.q0 + tok) * a.b.mask_words : nullptr;
    auto attended = [&](int t0) { return step_mask(t0, lim, hi, q.base, words, a.b.mask_words); };

    f16v acc[DT];
#pragma unroll
    for (int i = 0; i < DT; i++)
#pragma unroll
        for (int j = 0; j < 16; j++) acc[i][j] = 0.0f;
    float m = NINF, l = 0.0f;
    bool some = false;   /* this lane's column attends a row of the split */

    const int *pages = a.b.pages + (int64_t)seq * a.b.ld_pages;
    const int rmask = (1 << a.b.page_shift) - 1;
    const uint8_t *kbase = a.k.data + (int64_t)kvh * a.k.head_stride, *vbase = a.v.data + (int64_t)kvh * a.v.head_stride;
    const uint8_t *ksb = MX ? a.k.scales + (int64_t)kvh * a.k.scale_head_stride : nullptr;
    const uint8_t *vsb = MX ? a.v.scales + (int64_t)kvh * a.v.scale_head_stride : nullptr;

    /* Page ids of a step's groups of 16 rows, one a lane (its number in the group of 16 lanes past
     * GROUPS: none). They are loaded a step before their use, when every load has been waited for;
     * by scalar instructions, checks included, they took a third of a wave's instructions. */
    int pv = -1;
    auto load_pages = [&](int t0) __attribute__((always_inline)) {
        const int t = t0 + 16 * lane;
        pv = lane < M::GROUPS && t < hi ? pages[t >> a.b.page_shift] : -1;
    };
    unsigned have_now = 0, have_next = 0;   /* bit u: group u has a page */
    int id_next = 0;                        /* the page of this wave's rows, 0 where there is none */
    auto look = [&]() __attribute__((always_inline)) {
        const bool ok = page_ok(a.b, pv);
        have_next = (unsigned)__ballot(ok);
        id_next = __builtin_amdgcn_readlane(ok ? pv : 0, wave * (M::ROWS / 4) / 16);
    };
    /* A wave brings in a quarter of the step's rows of K and of V; they lie in one page. 16-bit: 1 KiB
     * of LDS an instruction, 16 bytes a lane; 8-bit: 16 codes a lane, two pieces. */
    constexpr int RW = M::ROWS / 4, LANES = MX ? M::PIECES / 2 : M::PIECES, RI = 64 / LANES, N = RW / RI;   /* lanes of a row, rows an instruction, instructions */
    const int my = wave * RW, lr = lane / LANES, lp = lane % LANES;
    /* 16-bit: byte of a lane's pieces in memory (the z-th instruction's 1 KiB further, there and in LDS) */
    int off[N];
#pragma unroll
    for (int z = 0; z < N; z++) off[z] = lr * (2 * D) + (lp ^ M::swz(my + z * RI + lr)) * 16;
    u4 sw[MX ? 2 * N : 1];
    unsigned ss[MX ? 2 * N : 1];
    /* Every load goes to a row of the cache: rows past hi lie in the same page, those of a page that
     * is not there are taken from page 0; settle clears both. */
    auto load = [&](int t0, int buf) {
        const int64_t id = id_next;
        const int row = (t0 + my) & rmask;
        if constexpr (MX) {
            const uint8_t *kp = kbase + id * a.k.page_stride + row * D, *vp = vbase + id * a.v.page_stride + row * D;
            const uint8_t *kq = ksb + id * a.k.scale_page_stride + row * (D / MX_BLOCK), *vq = vsb + id * a.v.scale_page_stride + row * (D / MX_BLOCK);
#pragma unroll
            for (int z = 0; z < 2 * N; z++) {
                const int r = z % N * RI + lr;
                sw[z] = *(const u4 *)((z < N ? kp : vp) + r * D + 16 * lp);
                ss[z] = (z < N ? kq : vq)[r * (D / MX_BLOCK) + (lp >> 1)];
            }
        } else {
            const uint8_t *kp = same(kbase + id * a.k.page_stride + (int64_t)row * (2 * D)), *vp = same(vbase + id * a.v.page_stride + (int64_t)row * (2 * D));
            to_lds_rows<N>(kp, off, lds[buf][0] + my * (2 * D));
            to_lds_rows<N>(vp, off, lds[buf][1] + my * (2 * D));
        }
    };
    /* whether some column of the workgroup may not attend every row of the step at t0 (pages: bit
     * u where group u has one) */
    auto edge_at = [&](int t0, unsigned have) {
        return !(t0 + M::ROWS <= full && t0 + M::ROWS <= hi && have == (1u << M::GROUPS) - 1);
    };
    /* The loaded step made ready in LDS. Past `full` (rows that some columns do not attend) an
     * infinity or NaN of V would reach those columns as 0 * inf, so it is left out and added at the
     * end; rows that do not exist are cleared. */
    auto settle = [&](int buf, int t0, unsigned have) {
        const bool edge = edge_at(t0, have), some = t0 + M::ROWS > full;
        bool odd = false;
        auto clear = [&](int r, const u4 x) {
            const bool ok = t0 + r < hi && (have >> (r >> 4) & 1);
            odd = odd || (ok && some && (T::odd(x[0]) || T::odd(x[1]) || T::odd(x[2]) || T::odd(x[3])));
            const u4 y = some ? (u4){T::clean(x[0]), T::clean(x[1]), T::clean(x[2]), T::clean(x[3])} : x;
            return ok ? y : (u4){0, 0, 0, 0};
        };
        if constexpr (MX) {
#pragma unroll
            for (int z = 0; z < 2 * N; z++) {
                const int r = my + z % N * RI + lr;
                const float f = mx_scale(ss[z]);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const unsigned x = sw[z][2 * h], y = sw[z][2 * h + 1];
                    u4 w = {T::template from_mx8<false>(x, f), T::template from_mx8<true>(x, f),
                            T::template from_mx8<false>(y, f), T::template from_mx8<true>(y, f)};
                    if (z >= N && edge) w = clear(r, w);
                    *(u4 *)(lds[buf][z >= N] + M::at(r, 2 * lp + h)) = w;
                }
            }
        } else {
            vm_wait();   /* this thread's pieces have arrived */
            if (edge)
#pragma unroll 1
                for (int z = 0; z < N; z++) {
                    u4 *x = (u4 *)(lds[buf][1] + (my + z * RI) * (2 * D) + lane * 16);
                    *x = clear(my + z * RI + lr, *x);
                }
        }
        if (odd) odd_flag = 1;
    };
    if (threadIdx.x == 0) odd_flag = 0;
    __syncthreads();
    if (lo < hi) {
        load_pages(lo);
        look();
        load(lo, 0);
        settle(0, lo, have_next);
        load_pages(lo + M::ROWS);
    }
    __syncthreads();

    /* Byte addresses in K and V of a step: scores read row 32 u + lc, pieces 2 i + half (an exclusive
     * or with 32 i); sums read rows 16 g + 4 half .. + 3 and 8 further, elements 32 i .. 32 i + 31
     * (with 64 i) */
    const int vr = 4 * half + ((lane & 15) >> 2), vp = 2 * (lane >> 4 & 1) + (lane >> 1 & 1);
    const int k_at = M::at(lc, half), v_at[2] = {M::at(vr, vp) + 8 * (lane & 1), M::at(vr + 8, vp) + 8 * (lane & 1)};
    int buf = 0;
    for (int t0 = lo; t0 < hi; t0 += M::ROWS, buf ^= 1) {
        const bool more = t0 + M::ROWS < hi;
        have_now = have_next;
        const uint8_t *kb = lds[buf][0], *vb = lds[buf][1];
        f16v s[M::TILES];
#pragma unroll
        for (int u = 0; u < M::TILES; u++)
#pragma unroll
            for (int j = 0; j < 16; j++) s[u][j] = 0.0f;
        /* four instructions' reads ahead of their use, in this order: left to itself the compiler puts
         * each read right before its instruction */
        constexpr int KN = KS * M::TILES, AHEAD = 4;
        v8 kr[2][AHEAD];
        auto read_k = [&](int n) __attribute__((always_inline)) {
            return *(const v8 *)(kb + (k_at ^ 32 * (n / M::TILES)) + 32 * (n % M::TILES) * (2 * D));
        };
#pragma unroll
        for (int n = 0; n < AHEAD; n++) kr[0][n] = read_k(n);
        in_order();
        if (more) {   /* the next step's rows are sent for while the first reads are on their way */
            look();
            load(t0 + M::ROWS, buf ^ 1);
            load_pages(t0 + 2 * M::ROWS);
        }
        in_order();
#pragma unroll
        for (int b = 0; b < KN / AHEAD; b++) {
#pragma unroll
            for (int n = 0; n < AHEAD; n++)
                if (b + 1 < KN / AHEAD) kr[(b + 1) & 1][n] = read_k((b + 1) * AHEAD + n);
            in_order();
#pragma unroll
            for (int n = 0; n < AHEAD; n++) {
                const int z = b * AHEAD + n;
                s[z % M::TILES] = T::mfma32(kr[b & 1][n], qf[z / M::TILES], s[z % M::TILES]);
            }
            in_order();
        }

        const bool edge = edge_at(t0, have_now);
        v8 pf[M::GROUPS];
        float mx;
        if (!edge) {
            some = true;
            mx = s[0][0];
#pragma unroll
            for (int u = 0; u < M::TILES; u++)
#pragma unroll
                for (int j = 0; j < 16; j++) mx = fmaxf(mx, s[u][j]);
            mx = max32(mx) * scale2;
        } else {
            mx = NINF;
            const unsigned long long at = attended(t0) & group_rows(have_now), vis = at >> (4 * half);
            some = some || at;
#pragma unroll
            for (int u = 0; u < M::TILES; u++)
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    s[u][j] = vis >> (32 * u + 8 * (j >> 2) + (j & 3)) & 1 ? s[u][j] * scale2 : NINF;
                    mx = fmaxf(mx, s[u][j]);
                }
            mx = max32(mx);
        }
        /* the sums are rescaled only where a maximum has grown by more than 2^8: until then the
         * probabilities stay below 2^8, which costs no accuracy in either 16-bit type */
        if (__any(mx > m + 8.0f)) {
            mx = fmaxf(mx, m);
            const float al = mx == NINF ? 0.0f : exp2_hw(m - mx);
            l *= al;
#pragma unroll
            for (int i = 0; i < DT; i++) acc[i] *= al;
            m = mx;
        }
        const float ms = m == NINF ? 0.0f : m;
        const float sc = edge ? 1.0f : scale2;
        float ls = 0.0f;
#pragma unroll
        for (int u = 0; u < M::TILES; u++)
#pragma unroll
            for (int j = 0; j < 16; j++) {
                s[u][j] = exp2_hw(__builtin_fmaf(s[u][j], sc, -ms));
                ls += s[u][j];
            }
        l += ls;
#pragma unroll
        for (int g = 0; g < M::GROUPS; g++) {
            const f16v &x = s[g >> 1];
            const int o = 8 * (g & 1);
            const u4 w = {T::pack(x[o], x[o + 1]), T::pack(x[o + 2], x[o + 3]), T::pack(x[o + 4], x[o + 5]), T::pack(x[o + 6], x[o + 7])};
            pf[g] = __builtin_bit_cast(v8, w);
        }
        constexpr int VN = M::GROUPS * DT, VAHEAD = VN < 8 ? 2 : 4;
        v8 vr8[2][VAHEAD];
        auto read_v = [&](int n) __attribute__((always_inline)) {
            const int g = n / DT, i = n % DT;
            const u2 x = read_tr(vb + (v_at[0] ^ 64 * i) + 16 * g * (2 * D)), y = read_tr(vb + (v_at[1] ^ 64 * i) + 16 * g * (2 * D));
            return __builtin_bit_cast(v8, (u4){x[0], x[1], y[0], y[1]});
        };
#pragma unroll
        for (int n = 0; n < VAHEAD; n++) vr8[0][n] = read_v(n);
        in_order();
#pragma unroll
        for (int b = 0; b < VN / VAHEAD; b++) {
#pragma unroll
            for (int n = 0; n < VAHEAD; n++)
                if (b + 1 < VN / VAHEAD) vr8[(b + 1) & 1][n] = read_v((b + 1) * VAHEAD + n);
            in_order();
#pragma unroll
            for (int n = 0; n < VAHEAD; n++) {
                const int z = b * VAHEAD + n;
                acc[z % DT] = T::mfma32(vr8[b & 1][n], pf[z / DT], acc[z % DT]);
            }
            in_order();
        }
        if (more) settle(buf ^ 1, t0 + M::ROWS, have_next);
        __syncthreads();
    }

    if (odd_flag) {
#pragma unroll 1
        for (int t = max(lo, full / M::ROWS * M::ROWS); t < hi; t++) {
            const int id = word_of(pages, t >> a.b.page_shift);
            if (!page_ok(a.b, id)) continue;
            const bool add = attended(t) & 1;
            const uint8_t *row = vbase + (int64_t)id * a.v.page_stride + (int64_t)(t & rmask) * (D * (MX ? 1 : 2));
            const uint8_t *sc = MX ? vsb + (int64_t)id * a.v.scale_page_stride + (t & rmask) * (D / MX_BLOCK) : nullptr;
#pragma unroll
            for (int i = 0; i < DT; i++)
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    const unsigned x = row_elem<T, MX>(row, sc, 32 * i + 8 * (j >> 2) + 4 * half + (j & 3));
                    acc[i][j] += add && T::odd(x) ? T::wide(x) : 0.0f;
                }
        }
    }

    l = sum32(l);
    if (!on) return;
    const int64_t row = (int64_t)(q.q0 + tok) * a.heads + head;
    if (n_sp == 1) {
        const float inv = l == 0.0f ? (some ? UNDEFINED : 0.0f) : 1.0f / l;
        uint8_t *out = a.out + (int64_t)(q.q0 + tok) * a.ot + (int64_t)head * a.oh;
#pragma unroll
        for (int i = 0; i < DT; i++)
#pragma unroll
            for (int b = 0; b < 4; b += 2) {
                /* lanes l and l ^ 32 hold elements 0-3 8-11 and 4-7 12-15 of these 16: after the
                 * exchange each has 8 consecutive ones */
                unsigned x[2][2];
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int w = 0; w < 2; w++)
                        x[k][w] = T::pack(acc[i][4 * (b + k) + 2 * w] * inv, acc[i][4 * (b + k) + 2 * w + 1] * inv);
                u4 o;
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    const auto r = __builtin_amdgcn_permlane32_swap(x[0][w], x[1][w], false, false);
                    o[w] = r[0];
                    o[2 + w] = r[1];
                }
                uint8_t *p = out + 2 * (32 * i + 8 * b + 8 * half);
                *(u4_any *)p = o;
            }
        if (a.lse && half == 0) a.lse[row] = l == 0.0f ? NINF : (m + __log2f(l)) * 0.69314718055994531f;
    } else {
        float *po = a.part + (row * a.n_splits + sp) * D;
        if (!(l == 0.0f))
#pragma unroll
            for (int i = 0; i < DT; i++)
#pragma unroll
                for (int b = 0; b < 4; b++)
                    *(f4 *)(po + 32 * i + 8 * b + 4 * half) = (f4){acc[i][4 * b], acc[i][4 * b + 1], acc[i][4 * b + 2], acc[i][4 * b + 3]};
        if (half == 0) {
            float *ml = a.part + (int64_t)a.b.n_tokens * a.heads * a.n_splits * D + (row * a.n_splits + sp) * 2;
            ml[0] = l == 0.0f && some ? UNDEFINED : m;
            ml[1] = l;
        }
    }
}

template <class T, bool MX, int D>
void many_t(const AttendArgs &a, hipStream_t st) {
    const int64_t tiles = ((int64_t)a.b.max_q * a.group + MANY_COLS - 1) / MANY_COLS;
    const dim3 grid((unsigned)(tiles * a.n_splits * a.kv_heads), 1, a.b.n_seqs);
    hipLaunchKernelGGL((k_attend_many<T, MX, D>), grid, dim3(64 * MANY_WAVES), 0, st, a);
}

} // namespace

void attend_many(const AttendArgs &a, int q_dtype, int cache_dtype, int width, hipStream_t st) {
    const bool mx = cache_dtype == DT_MX8;
#define HXP_MANY(T, D) (mx ? many_t<T, true, D>(a, st) : many_t<T, false, D>(a, st))
    if (q_dtype == DT_BF16) width == 64 ? HXP_MANY(Bf16, 64) : width == 128 ? HXP_MANY(Bf16, 128) : HXP_MANY(Bf16, 256);
    else width == 64 ? HXP_MANY(F16, 64) : width == 128 ? HXP_MANY(F16, 128) : HXP_MANY(F16, 256);
#undef HXP_MANY
}

} // namespace hxp
