// kv4_attend.cu -- attention over the paged 4-bit KV cache.
//
// For row r of a sequence at position p, query head h of KV head h / G:
//     s_t = scale * q . k_t,   ctx = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m)   over t in (p - window, p],
// k_t and v_t the values held (code * step), positions of absent pages (table entry -1) left out, 0 where nothing is left.
#include "kv4_frag.cuh"
#include "kv4_attend.cuh"
#include <type_traits>

namespace {

// ---- few rows a sequence (decode) ------------------------------------------------------------------------------------
// A CTA takes one KV head of one sequence, up to 4 or 8 (row, query head) pairs of it ("columns"), and a span of pages.
// Warp w owns positions 16 w .. 16 w + 15 of every page of the span: it brings their codes and steps to its own ring in
// shared memory (three or four pages deep, 16-byte asynchronous copies, no barrier beyond the warp) and multiplies
//     scores  [16 positions x columns] = codes [16 x 32] (a group) * q pieces, times the position's step, group by group
//     output  [32 dims x columns]     += codes [dims x 16 positions] * (weight * value step) pieces
// PAIR (up to four columns): hi and lo piece of a column are neighbouring columns of one product and land in the same
// thread, which adds them.  Otherwise eight columns, and hi and lo are two products into the same sums: the same matrix
// work a column, half the piece arithmetic.  Every warp keeps its own exponent of the largest value step, and for each column a
// reference that weights are scaled by: the first page's largest weight is 2^10 exactly (a row that sees one position is that
// position's values, unless its score's own rounding shows), and where that of a page leaves 2^6 .. 2^15 the reference is
// moved by a whole number of base-2 units to put that one at 2^10, up or down (at 2^15 where others of the page lie 10 below
// it), for the lower piece ends at 2^-24, and one position that holds nearly all the weight must not take the bits of those beside and after it (that
// costs 2 %: 64 sequences of up to 8192 103.2 -> 105.5 us; a look at every column's largest on every page, and less
// room above, 5 %).  Warps join in shared memory, spans
// through `part` ({m, l, acc[hd]} per (row, head, split)): up to DEC_JOIN of them by the CTA of a tile that ends last
// (1000 positions, 16 heads on 8: 7 us, with a second launch a microsecond more; 2 sequences of 8000 at hd 64, 17 to 32
// spans: 9.7 us, 13.3 us with a second launch), others by the merge kernels below.  A join is a chain of waits, so it asks
// for the sums of its spans before it knows their weights (7.8 -> 6.8 us; one sequence of 131072 39.8 -> 33.7 us).
// What bounds it: instructions and the waits between them.  A warp's 16 positions of 128 dims against 4 columns take about 400
// (32 matrix products, the rest unpacking codes, the two pieces of weight * step, softmax), issued in 64 of 100 cycles by four
// warps a scheduler (eight columns: 49 of 100 by three, whose registers leave no room for a fourth); memory is not the limit:
// 64 sequences of up to 8192 positions, 32 heads on 8, 369 MB: 105 us, 3.5 TB/s; one sequence of 131072, 32 heads on 4: 34.6
// us; 13 sequences, window 1024, hd 256: 17.9 us.  Where pages' largest weights differ much the reference moves often: scores
// of twice that spread (2.4 units) 112 and 37.7 us, of four times 120 and 39.0.  The steps measured at the first of these, which
// are without all that: codes straight from memory to
// fragments 188 us, the ring 107 us, weight * step in f16 pairs and the joins in the launch 103 us.
constexpr int DEC_W = 4, DEC_NP = 256, DEC_JOIN = 32, DEC_F = 16;      // warps a CTA, the most pages of a span, the most spans joined in the launch itself, pages of a matrix unit's sum
// exponents of a page's largest weight: the range it may have (DEC_LOW: where each four positions have one as large), where it is
// put, and how far below the highest reference so far one may be
constexpr float DEC_HI = 15.f, DEC_LO = 6.f, DEC_LOW = 4.f, DEC_AT = 10.f, DEC_DOWN = 60.f;

// the most pages of a span whose sums stay in the matrix unit (one or two products a page)
constexpr int kv4_decode_long(bool pair) { return pair ? 32 : 20; }
// CTAs an SM holds (registers)
constexpr int kv4_decode_ctas(int NG, bool pair) { return NG <= 2 ? 4 : NG <= 4 ? (pair ? 4 : 3) : NG <= 6 ? (pair ? 3 : 2) : pair ? 3 : 2; }
template <int NG, bool PAIR> struct DecL {
    static constexpr int HD = NG * 32, NC = PAIR ? 4 : 8, STAGE = 18 * HD;       // bytes of 16 positions: codes 2 x 8 HD, steps 2 x HD
    static constexpr int CTAS = kv4_decode_ctas(NG, PAIR);
    static constexpr int ST = NG >= 7 ? 3 : 4;               // ring depth in pages
    static constexpr int RING = DEC_W * ST * STAGE, JOIN = DEC_W * NC * HD * 4;
    static constexpr int BODY = RING > JOIN ? RING : JOIN;
    static constexpr int SMEM = BODY + NC * HD * 4 + (2 * DEC_W * NC + 4 * NC + DEC_NP) * 4;
};

// LONG: spans of more pages than the matrix unit's own sums are good for (see tot below).
template <int NG, bool PAIR, bool LONG>
__global__ void __launch_bounds__(DEC_W * 32, DecL<NG, PAIR>::CTAS) kv4_decode_kernel(Kv4Attend a, int ntile, int nsplit, int span, float *part, int *count) {
    using Lay = DecL<NG, PAIR>;
    constexpr int HD = NG * 32, NC = Lay::NC, UNIT = 72 * HD, STAGE = Lay::STAGE, NS = PAIR ? 1 : 2, NCP = (36 * NG + 31) / 32, DEC_ST = Lay::ST;
    extern __shared__ __align__(128) uint8_t sm_kv4[];
    float *js = reinterpret_cast<float *>(sm_kv4);           // the ring, then acc[DEC_W][NC][HD]
    float *qs = reinterpret_cast<float *>(sm_kv4 + Lay::BODY);   // the query rows [NC][HD]
    float *ml = qs + NC * HD;                                // m, then factor, [DEC_W][NC]; l [DEC_W][NC]; descale [NC]
    int *col = reinterpret_cast<int *>(ml + 2 * DEC_W * NC + NC);   // row of a column, its query head, its position [NC] each
    int *list = col + 3 * NC;                                // page ids of the span, -1: not there
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = lane >> 2, j = lane & 3;
    const int split = blockIdx.x % nsplit;
    const int u = blockIdx.x / nsplit, tile = u % ntile, head = (u / ntile) % a.geo.KV, seq = u / ntile / a.geo.KV;
    pdl_trigger();
    pdl_wait();
    const Kv4Seq sq = kv4_load_seq(a, seq);
    if (!sq.ok) {
        if ((nsplit == 1 || (count && split == 0)) && tile == 0) kv4_zero_rows(a, sq, head);
        return;
    }
    const int c0 = tile * NC, ncol = sq.n * a.G - c0 < NC ? sq.n * a.G - c0 : NC;
    if (ncol <= 0) return;
    const int pos0 = sq.len - sq.n;                          // position of the sequence's first row
    const int row_a = c0 / a.G, row_z = (c0 + ncol - 1) / a.G;
    const Kv4Range cr = kv4_range(a, pos0 + row_a, pos0 + row_z);
    const int t_lo = (cr.lo_any & ~(KV4_PAGE - 1)) + split * span, t_hi = cr.hi_any - t_lo < span ? cr.hi_any : t_lo + span;
    if (t_lo >= cr.hi_any && nsplit > 1) return;             // nothing in this span: the merge does not look at it
    const int np = t_hi > t_lo ? (t_hi - t_lo + KV4_PAGE - 1) / KV4_PAGE : 0;
    const int *tab = a.b.table + (size_t)seq * a.b.ld + t_lo / KV4_PAGE;
    for (int i = tid; i < np; i += DEC_W * 32) {
        const int id = tab[i];
        const bool ok = kv4_page_ok(a.geo, id);
        if (!ok && id != -1) atomicExch(a.err, 1);
        list[i] = ok ? id : -1;
    }
    if (tid < NC) {
        const int cc = c0 + tid, row = cc / a.G;
        col[tid] = sq.r0 + row; col[NC + tid] = head * a.G + cc - row * a.G; col[2 * NC + tid] = tid < ncol ? pos0 + row : -1;
    }
    __syncthreads();
    // this lane's 16-byte pieces of a stage: [K codes | V codes | K steps | V steps] of positions 16 warp ..
    uint8_t *ring = sm_kv4 + warp * (DEC_ST * STAGE);
    const uint8_t *base = a.mem + (size_t)(a.layer * a.geo.KV + head) * UNIT;
    // chunk c = lane + 32 i of a stage; a round of 32 that lies within one part has the same offset to `mine` in every lane
    const uint8_t *mine = base + warp * (8 * HD) + lane * 16;
    constexpr int KC = 16 * NG;                              // chunks of one part's codes
    int off[NCP];
#pragma unroll
    for (int i = 0; i < NCP; i++) {
        const int c = lane + 32 * i;
        const int o = c < KC ? warp * (8 * HD) + c * 16
                    : c < 2 * KC ? kv4_v_code_off(HD) + warp * (8 * HD) + (c - KC) * 16
                    : c < 34 * NG ? kv4_k_step_off(HD) + warp * HD + (c - 32 * NG) * 16
                                  : kv4_v_step_off(HD) + warp * HD + (c - 34 * NG) * 16;
        off[i] = o - warp * (8 * HD) - lane * 16;
        if (32 * i + 31 < KC) off[i] = 512 * i;
        else if (32 * i >= KC && 32 * i + 31 < 2 * KC) off[i] = kv4_v_code_off(HD) + 512 * i - KC * 16;
    }
    const bool last = lane + 32 * (NCP - 1) < 36 * NG;       // the lane has a chunk in the last round
    const unsigned page_bytes = (unsigned)kv4_page_bytes(a.geo);     // (65535 units of 18 KB at most)
    auto issue = [&](int i, int slot) {                      // page i of the span to ring slot `slot`
        if (i < np) {
            const int id = list[i];
            if (id >= 0) {
                const uint8_t *src = mine + (size_t)(unsigned)id * page_bytes;
                uint8_t *dst = ring + slot * STAGE + lane * 16;
#pragma unroll
                for (int k = 0; k < NCP; k++)
                    if (k < NCP - 1 || last) cp_async16(dst + k * 512, src + off[k]);
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < DEC_ST - 1; i++) issue(i, i);
    // query rows, scaled by a power of two so that |q| 2^k < 2^14; a row that is not finite has NaN scores
    for (int c = warp; c < NC; c += DEC_W) {
        float x[NG];
        unsigned mb = 0;
        const float *src = a.q + (size_t)col[c] * a.q_ld + (size_t)col[NC + c] * HD;
#pragma unroll
        for (int g = 0; g < NG; g++) x[g] = c < ncol ? src[g * 32 + lane] : 0.f;
#pragma unroll
        for (int g = 0; g < NG; g++) mb = max(mb, __float_as_uint(fabsf(x[g])));
        mb = __reduce_max_sync(0xffffffffu, mb);
        const bool fin = mb < 0x7f800000u;
        const int k = fin ? kv4_q_shift(mb) : 0;
#pragma unroll
        for (int g = 0; g < NG; g++) qs[c * HD + g * 32 + lane] = fin ? kv4_scale2(x[g], k) : 0.f;
        if (lane == 0) ml[2 * DEC_W * NC + c] = fin ? kv4_scale2(a.scale * 1.44269504f, -k) : __int_as_float(0x7fffffff);
    }
    __syncthreads();
    // operand column r: PAIR: pair r / 2, piece r & 1; else column r, both pieces
    unsigned qf[NS][NG][4];
    const unsigned short sel = (r & 1) ? KV4_HM1 : KV4_H0;
    {
        const float *qc = qs + (PAIR ? r >> 1 : r) * HD;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            const float4 x = *reinterpret_cast<const float4 *>(qc + g * 32 + 8 * j), z = *reinterpret_cast<const float4 *>(qc + g * 32 + 8 * j + 4);
            const float xs[4] = {x.x, x.y, x.z, x.w}, zs[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (PAIR) qf[0][g][i] = kv4_piece(xs[i], zs[i], sel);
                else kv4_pieces(xs[i], zs[i], qf[0][g][i], qf[NS - 1][g][i]);
            }
        }
    }
    // the columns whose scores this thread holds: PAIR: j; else 2 j and 2 j + 1
    float desc[NS];
    int clo[NS], chi[NS];
#pragma unroll
    for (int k = 0; k < NS; k++) {
        const int c = PAIR ? j : 2 * j + k, p = col[2 * NC + c];
        desc[k] = ml[2 * DEC_W * NC + c];
        chi[k] = p;
        clo[k] = a.window > 0 && p - a.window + 1 > 0 ? p - a.window + 1 : 0;
    }
    const int phi = col[2 * NC + (PAIR ? r >> 1 : r)], plo = a.window > 0 ? phi - a.window + 1 : 0;      // limits of operand column r
    float m[NS], mh[NS], l[NS], acc[NG][2][4];
    float vth = 0.f;                                         // 2^(e + 1) for the exponent e of the largest value step so far
    int dk = 0;                                              // exponent of the steps' factor; see below
#pragma unroll
    for (int k = 0; k < NS; k++) { m[k] = mh[k] = -INFINITY; l[k] = 0.f; }   // m: the reference, mh: the highest so far; l: weights over 2^m; acc: times 2^dk too
#pragma unroll
    for (int g = 0; g < NG; g++)
#pragma unroll
        for (int i = 0; i < 8; i++) acc[g][i >> 2][i & 3] = 0.f;
    // The matrix unit cuts its sums off, it does not round them, 1.6e-8 of a result a product: with 99 pages to a span and two
    // products a page results were 3.2e-6 off, with kv4_decode_long pages 0.6e-6 at most.  Of longer spans what acc holds is
    // added to rounded sums every DEC_F pages.  These lie in local memory, with the reference and the steps' factor that they
    // were left with, and the code beside the loop costs 10 % (64 sequences of up to 8192: 114 us), so shorter spans have a
    // kernel without.
    volatile float tot[LONG ? NG * 8 : 1], mt[NS];
    volatile int dkt;
    auto tot_factors = [&](float (&f)[NS]) {                 // what brings tot to the present ones
#pragma unroll
        for (int k = 0; k < NS; k++) f[k] = (mt[k] == m[k] ? 1.f : kv4_exp2(mt[k] - m[k])) * kv4_pow2(dk - dkt);
    };
    int pages = 0;                                           // (tot holds nothing before DEC_F of them)
    for (int it = 0, slot = 0; it < np; it++) {
        cp_async_wait<DEC_ST - 2>();
        __syncwarp();                                        // everyone's pieces of page `it` are here, and page it - 1 is done with
        issue(it + DEC_ST - 1, slot ? slot - 1 : DEC_ST - 1);
        const uint8_t *sg = ring + slot * STAGE;
        slot = slot == DEC_ST - 1 ? 0 : slot + 1;
        const int t0 = t_lo + it * KV4_PAGE + warp * 16;
        if (list[it] < 0 || t0 >= cr.hi_any || t0 + 16 <= cr.lo_any) continue;
        // two copies of the body: every position seen by every column, or limits to look at (columns past ncol hold zero
        // rows, and are not written)
        auto body = [&](auto in) {
        constexpr bool inside = decltype(in)::value;
        // scores of positions t0 + r and t0 + r + 8
        float s[NS][2];
#pragma unroll
        for (int k = 0; k < NS; k++) s[k][0] = s[k][1] = 0.f;
        {
            unsigned ka[NG], kb[NG], sa[(NG + 1) / 2], sb[(NG + 1) / 2];
            kv4_ldsw<NG>(ka, sg + r * (HD / 2) + j * (4 * NG));
            kv4_ldsw<NG>(kb, sg + (r + 8) * (HD / 2) + j * (4 * NG));
            kv4_ldsteps<NG>(sa, sg + 16 * HD + r * (2 * NG));
            kv4_ldsteps<NG>(sb, sg + 16 * HD + (r + 8) * (2 * NG));
            // the groups' products are independent of one another: their chains are written side by side
            constexpr int GB = NG <= 4 ? NG : NG % 4 == 0 ? 4 : NG % 3 == 0 ? 3 : NG == 5 ? 5 : 7;
#pragma unroll
            for (int g0 = 0; g0 < NG; g0 += GB) {
                unsigned ea[GB][4], eb[GB][4];
                float c[GB][4];
#pragma unroll
                for (int g = 0; g < GB; g++) {
                    kv4_codes(ka[g0 + g], ea[g]);
                    kv4_codes(kb[g0 + g], eb[g]);
                }
#pragma unroll
                for (int pc = NS - 1; pc >= 0; pc--)
#pragma unroll
                    for (int st = 0; st < 2; st++)
#pragma unroll
                        for (int g = 0; g < GB; g++)
                            if (pc == NS - 1 && st == 0)
                                kv4_mma0(c[g], ea[g][0], eb[g][0], ea[g][1], eb[g][1], qf[pc][g0 + g][0], qf[pc][g0 + g][1]);
                            else kv4_mma(c[g], ea[g][2 * st], eb[g][2 * st], ea[g][2 * st + 1], eb[g][2 * st + 1], qf[pc][g0 + g][2 * st], qf[pc][g0 + g][2 * st + 1]);
#pragma unroll
                for (int g = 0; g < GB; g++) {
                    const int gg = g0 + g;
                    const float da = kv4_half_of(sa[gg >> 1], gg & 1), db = kv4_half_of(sb[gg >> 1], gg & 1);
                    if (PAIR) {
                        s[0][0] = fmaf(da, c[g][0] + c[g][1], s[0][0]); s[0][1] = fmaf(db, c[g][2] + c[g][3], s[0][1]);
                    } else {
#pragma unroll
                        for (int k = 0; k < NS; k++) { s[k][0] = fmaf(da, c[g][k], s[k][0]); s[k][1] = fmaf(db, c[g][2 + k], s[k][1]); }
                    }
                }
            }
        }
        unsigned see = 0xffffffffu;                          // bit 2 k + half: that score is seen
        if (!inside) {
#pragma unroll
            for (int k = 0; k < NS; k++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int t = t0 + r + 8 * h;
                    if (t < clo[k] || t > chi[k]) { see &= ~(1u << (2 * k + h)); s[k][h] = 0.f; }
                }
        }
        // Weights stay below 2^15.  Where the largest value step so far (NaN left aside), of exponent e, is 1 or more or below
        // 2^-4, steps are scaled by 2^dk, dk = -1 - e: weight * step stays below 2^15, and a page's largest weight (2^4 or
        // more, see below) times that step is 1 or more: pieces end at 2^-25 of it, and at 2^-19 in a group whose steps are 64
        // times smaller.
        {
            __half2 mx = __halves2half2(__ushort_as_half(0), __ushort_as_half(0));
#pragma unroll
            for (int i = 0; i < (8 * NG + 31) / 32; i++) {
                const int w = lane + 32 * i;                 // one word each: steps 2 w and 2 w + 1 of the 16 x NG
                if (w < 8 * NG) {
                    unsigned v = *reinterpret_cast<const unsigned *>(sg + 17 * HD + 4 * w);
                    if (!inside) {
                        const int ta = t0 + 2 * w / NG, tb = t0 + (2 * w + 1) / NG;
                        v &= (ta >= cr.lo_any && ta < cr.hi_any ? 0xffffu : 0u) | (tb >= cr.lo_any && tb < cr.hi_any ? 0xffff0000u : 0u);
                    }
                    mx = __hmax2(mx, __habs2(*reinterpret_cast<const __half2 *>(&v)));
                }
            }
            const float big = fmaxf(__low2float(mx), __high2float(mx));
            if (__any_sync(0xffffffffu, big >= vth)) {
                const unsigned b = __reduce_max_sync(0xffffffffu, __float_as_uint(big)) >> 23;           // e + 127
                if (b) {                                     // (f16 subnormals are normal f32; all steps 0: nothing to add, any scale does)
                    const int e = (int)b - 127, k = e > -1 || e < -4 ? -1 - e : 0;                       // -16 .. 23
                    const float f = kv4_pow2(k - dk);
                    vth = kv4_pow2(e + 1); dk = k;
#pragma unroll
                    for (int g = 0; g < NG; g++)
#pragma unroll
                        for (int i = 0; i < 8; i++) acc[g][i >> 2][i & 3] *= f;
                }
            }
        }
        float e[NS][2];                                      // base-2 exponents of the scaled weights
        bool odd = false;                                    // a cheap look first: the largest of each four positions within the range
        float big[NS];
#pragma unroll
        for (int k = 0; k < NS; k++) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                e[k][h] = fmaf(s[k][h], desc[k], -m[k]);
                if (!inside && !(see >> (2 * k + h) & 1)) e[k][h] = -INFINITY;
            }
            big[k] = fmaxf(e[k][0], e[k][1]);
            big[k] = fmaxf(big[k], __shfl_xor_sync(0xffffffffu, big[k], 16));
            odd |= !(big[k] > DEC_LOW && big[k] <= DEC_HI);
        }
        bool move = __any_sync(0xffffffffu, odd);
        if (move) {
            move = false;
#pragma unroll
            for (int k = 0; k < NS; k++) {                   // (a column is lane j of every quad; its largest decides)
                const unsigned large = __ballot_sync(0xffffffffu, big[k] > DEC_LO) & 0x11111111u << j;
                move |= big[k] > DEC_HI;
                move |= !large && m[k] > mh[k] - DEC_DOWN;
            }
            move = __any_sync(0xffffffffu, move);
        }
        if (move) {
#pragma unroll
            for (int k = 0; k < NS; k++) {
                float mx = -INFINITY, mn = INFINITY;
#pragma unroll
                for (int h = 0; h < 2; h++) if (see >> (2 * k + h) & 1) { mx = fmaxf(mx, s[k][h] * desc[k]); mn = fminf(mn, s[k][h] * desc[k]); }
                for (int o = 4; o < 32; o <<= 1) {
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
                }
                // one far above the others of its own page: no room above it, for their bits; within the range or nothing seen:
                // the reference is left where it is
                const float at = mx - mn > DEC_AT ? DEC_HI : DEC_AT;
                float to = m[k] == -INFINITY ? mx - at : m[k] + ceilf(mx - m[k] - at);
                if (mx == -INFINITY || (mx - m[k] > DEC_LO && mx - m[k] <= DEC_HI)) to = m[k];
                to = fmaxf(to, mh[k] - DEC_DOWN);
                const float f = to == m[k] ? 1.f : kv4_exp2(m[k] - to);
                m[k] = to; mh[k] = fmaxf(mh[k], to); l[k] *= f;
#pragma unroll
                for (int h = 0; h < 2; h++) e[k][h] = see >> (2 * k + h) & 1 ? fmaf(s[k][h], desc[k], -to) : -INFINITY;
#pragma unroll
                for (int g = 0; g < NG; g++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {            // the thread's output columns are its score columns
                        const int at = PAIR ? (i & 1) * 2 : (i & 1) * 2 + k;
                        acc[g][i >> 1][at] *= f;
                        if (PAIR) acc[g][i >> 1][at + 1] *= f;
                    }
            }
        }
        // scaled weights of positions 2 j, 2 j + 1, 2 j + 8, 2 j + 9 for column r
        float y[4];
        bool hide[4];
        {
            float p[NS][2];
#pragma unroll
            for (int k = 0; k < NS; k++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    p[k][h] = kv4_exp2(e[k][h]);
                    if (!inside && !(see >> (2 * k + h) & 1)) p[k][h] = 0.f;
                    l[k] += p[k][h];
                }
            // score column c sits in lane 4 row + c (PAIR) or 4 row + c / 2, register c & 1
            const int src = 8 * j + (r >> 1);
            if (PAIR) {
                y[0] = __shfl_sync(0xffffffffu, p[0][0], src); y[1] = __shfl_sync(0xffffffffu, p[0][0], src + 4);
                y[2] = __shfl_sync(0xffffffffu, p[0][1], src); y[3] = __shfl_sync(0xffffffffu, p[0][1], src + 4);
            } else {
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const float a0 = __shfl_sync(0xffffffffu, p[0][h], src), a1 = __shfl_sync(0xffffffffu, p[NS - 1][h], src);
                    const float b0 = __shfl_sync(0xffffffffu, p[0][h], src + 4), b1 = __shfl_sync(0xffffffffu, p[NS - 1][h], src + 4);
                    y[2 * h] = r & 1 ? a1 : a0; y[2 * h + 1] = r & 1 ? b1 : b0;
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) hide[i] = false;
            if (!inside) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int t = t0 + 2 * j + (i & 1) + 8 * (i >> 1);
                    hide[i] = t < plo || t > phi;
                }
            }
        }
        {
            unsigned va[NG], vb[NG], wa[NG], wb[NG];
            kv4_ldsw<NG>(va, sg + 8 * HD + lane * (4 * NG));
            kv4_ldsw<NG>(vb, sg + 12 * HD + lane * (4 * NG));
            kv4_ldsw<NG>(wa, sg + 17 * HD + 2 * j * (2 * NG));
            kv4_ldsw<NG>(wb, sg + 17 * HD + (8 + 2 * j) * (2 * NG));
            if (dk) {                                        // (f16 ends at 2^15: the rest in a second step)
                const __half2 f1 = __float2half2_rn(kv4_pow2(dk < 15 ? dk : 15)), f2 = __float2half2_rn(kv4_pow2(dk < 15 ? 0 : dk - 15));
                const unsigned u1 = *reinterpret_cast<const unsigned *>(&f1), u2 = *reinterpret_cast<const unsigned *>(&f2);
#pragma unroll
                for (int g = 0; g < NG; g++) { wa[g] = kv4_hmul2(kv4_hmul2(wa[g], u1), u2); wb[g] = kv4_hmul2(kv4_hmul2(wb[g], u1), u2); }
            }
            // weight * step in f16 pairs of positions: with y = yh + yl, hi = round(yh d), lo = round(yl d + (yh d - hi)); the
            // remainder of hi is exact, lo's rounding is 2^-22 of the product
            unsigned yh[2], yl[2];
            kv4_pieces(y[0], y[1], yh[0], yl[0]);
            kv4_pieces(y[2], y[3], yh[1], yl[1]);
            unsigned b[NS][NG][2];                           // operand columns: PAIR: this lane's piece; else hi and lo
#pragma unroll
            for (int g = 0; g < NG; g++)
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    const unsigned *w = q ? wb : wa;
                    const int i1 = NG + g;                   // steps of positions 2 j (+ 8 q) and the next: halves g and NG + g
                    const unsigned d = __byte_perm(w[g >> 1], w[i1 >> 1], (g & 1 ? 0x32 : 0x10) | (i1 & 1 ? 0x7600 : 0x5400));
                    unsigned hi, lo;
                    kv4_scaled_pieces(yh[q], yl[q], d, hi, lo);
                    if (!inside) {                           // a position that is not seen adds nothing, whatever its step holds
                        const unsigned keep = (hide[2 * q] ? 0u : 0xffffu) | (hide[2 * q + 1] ? 0u : 0xffff0000u);
                        hi &= keep; lo &= keep;
                    }
                    if (PAIR) b[0][g][q] = r & 1 ? lo : hi;
                    else { b[0][g][q] = hi; b[NS - 1][g][q] = lo; }
                }
            constexpr int GB = NG % 2 == 0 ? 2 : NG == 3 ? 3 : 1;
#pragma unroll
            for (int g0 = 0; g0 < NG; g0 += GB) {
                unsigned ea[GB][4], eb[GB][4];
#pragma unroll
                for (int g = 0; g < GB; g++) { kv4_codes(va[g0 + g], ea[g]); kv4_codes(vb[g0 + g], eb[g]); }
#pragma unroll
                for (int pc = NS - 1; pc >= 0; pc--)
#pragma unroll
                    for (int g = 0; g < GB; g++)
#pragma unroll
                        for (int h = 0; h < 2; h++)
                            kv4_mma(acc[g0 + g][h], ea[g][2 * h], ea[g][2 * h + 1], eb[g][2 * h], eb[g][2 * h + 1], b[pc][g0 + g][0], b[pc][g0 + g][1]);
            }
        }
        };
        if (t0 >= cr.lo_all && t0 + 15 < cr.hi_all) body(std::true_type{});
        else body(std::false_type{});
        if (LONG && ++pages % DEC_F == 0) {
            const bool first = pages == DEC_F;
            float f[NS];
#pragma unroll
            for (int k = 0; k < NS; k++) f[k] = 1.f;
            if (!first) tot_factors(f);
#pragma unroll
            for (int g = 0; g < NG; g++) {                   // (a group's loads together)
                float old[8];
#pragma unroll
                for (int i = 0; i < 8; i++) old[i] = first ? 0.f : tot[LONG ? 8 * g + i : 0];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    tot[LONG ? 8 * g + i : 0] = fmaf(old[i], f[PAIR ? 0 : i & (NS - 1)], acc[g][i >> 2][i & 3]);
                    acc[g][i >> 2][i & 3] = 0.f;
                }
            }
#pragma unroll
            for (int k = 0; k < NS; k++) mt[k] = m[k];
            dkt = dk;
        }
    }
    if (LONG && pages >= DEC_F) {
        float f[NS];
        tot_factors(f);
#pragma unroll
        for (int g = 0; g < NG; g++)
#pragma unroll
            for (int i = 0; i < 8; i++) acc[g][i >> 2][i & 3] = fmaf(tot[LONG ? 8 * g + i : 0], f[PAIR ? 0 : i & (NS - 1)], acc[g][i >> 2][i & 3]);
    }
    // join the warps: a thread holds dims 32 g + 4 r + 0 .. 3 of its score columns
    cp_async_wait<0>();
    __syncthreads();
    const float vs = kv4_pow2(-dk);
#pragma unroll
    for (int k = 0; k < NS; k++) {
        for (int o = 4; o < 32; o <<= 1) l[k] += __shfl_xor_sync(0xffffffffu, l[k], o);
        const int c = PAIR ? j : 2 * j + k;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            float o[4];
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] = (PAIR ? acc[g][i >> 1][(i & 1) * 2] + acc[g][i >> 1][(i & 1) * 2 + 1] : acc[g][i >> 1][(i & 1) * 2 + k]) * vs;
            *reinterpret_cast<float4 *>(js + ((size_t)warp * NC + c) * HD + g * 32 + 4 * r) = make_float4(o[0], o[1], o[2], o[3]);
        }
        if (r == 0) { ml[warp * NC + c] = m[k]; ml[DEC_W * NC + warp * NC + c] = l[k]; }
    }
    __syncthreads();
    if (warp == 0 && lane < NC) {                            // the factor of each warp's sums; m and l of all
        float M = -INFINITY, L = 0.f, f[DEC_W];
#pragma unroll
        for (int w = 0; w < DEC_W; w++) M = fmaxf(M, ml[w * NC + lane]);
#pragma unroll
        for (int w = 0; w < DEC_W; w++) {
            const float lw = ml[DEC_W * NC + w * NC + lane];
            f[w] = kv4_factor(lw, ml[w * NC + lane], M);
            L = fmaf(lw, f[w], L);
        }
#pragma unroll
        for (int w = 0; w < DEC_W; w++) ml[w * NC + lane] = f[w];
        ml[DEC_W * NC + lane] = L; ml[2 * DEC_W * NC + lane] = M;
    }
    __syncthreads();
    for (int i = tid; i < ncol * (HD / 4); i += DEC_W * 32) {
        const int c = i / (HD / 4), d = (i - c * (HD / 4)) * 4;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < DEC_W; w++) {
            const float f = ml[w * NC + c];
            const float4 v = *reinterpret_cast<const float4 *>(js + ((size_t)w * NC + c) * HD + d);
            if (f != 0.f) { o.x = fmaf(v.x, f, o.x); o.y = fmaf(v.y, f, o.y); o.z = fmaf(v.z, f, o.z); o.w = fmaf(v.w, f, o.w); }
        }
        const float L = ml[DEC_W * NC + c];
        const size_t rh = (size_t)col[c] * a.H + col[NC + c];
        if (nsplit == 1) {
            *reinterpret_cast<float4 *>(a.ctx + rh * HD + d) = kv4_times(o, kv4_over(L));
        } else {
            float *p = part + (rh * nsplit + split) * (HD + 4);
            *reinterpret_cast<float4 *>(p + 4 + d) = o;
            if (d == 0) { p[0] = ml[2 * DEC_W * NC + c]; p[1] = L; }
        }
    }
    if (!count) return;
    // few spans: the CTA that finishes last joins them, in the spans' order (the same sums whichever it is)
    int live = (cr.hi_any - (cr.lo_any & ~(KV4_PAGE - 1)) + span - 1) / span;
    if (live > nsplit) live = nsplit;
    __threadfence();
    __syncthreads();
    if (tid == 0) col[0] = atomicAdd(&count[u], 1) == live - 1 ? col[0] : -1;
    __syncthreads();
    if (col[0] < 0) return;
    __threadfence();
    for (int c = warp; c < ncol; c += DEC_W) {               // a warp a column, lane k the span k's {m, l}
        const size_t rh = (size_t)col[c] * a.H + col[NC + c];
        const float *p = part + rh * nsplit * (HD + 4);
        const float2 e = lane < live ? __ldcg(reinterpret_cast<const float2 *>(p + (size_t)lane * (HD + 4))) : make_float2(-INFINITY, 0.f);
        float4 v[16];                                        // the first spans' values on their way beside the {m, l}
        auto fetch = [&](int k0, int d) {
#pragma unroll
            for (int k = 0; k < 16; k++)
                if (k0 + k < live && d < HD) v[k] = __ldcg(reinterpret_cast<const float4 *>(p + (size_t)(k0 + k) * (HD + 4) + 4 + d));
        };
        fetch(0, 4 * lane);
        const float M = warp_max_f32(e.x), f = kv4_factor(e.y, e.x, M);
        float L = e.y * f;
        for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
        const float over = kv4_over(L);
#pragma unroll
        for (int d0 = 0; d0 < HD; d0 += 128) {
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
            for (int k0 = 0; k0 < live; k0 += 16) {
                if (d0 + k0 > 0) fetch(k0, d0 + 4 * lane);
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    const float fk = __shfl_sync(0xffffffffu, f, k0 + k);
                    if (k0 + k < live && fk != 0.f) { o.x = fmaf(v[k].x, fk, o.x); o.y = fmaf(v[k].y, fk, o.y); o.z = fmaf(v[k].z, fk, o.z); o.w = fmaf(v[k].w, fk, o.w); }
                }
            }
            if (d0 + 4 * lane < HD) *reinterpret_cast<float4 *>(a.ctx + rh * HD + d0 + 4 * lane) = kv4_times(o, over);
        }
    }
    if (tid == 0) count[u] = 0;                              // as the next launch finds it
}

// What the join of a row's heads needs of its sequence: r0 < 0: no sequence has the row; n == 0: the row is refused and
// reads as zeros.
struct Kv4Join { int r0, n, len; };
__device__ __forceinline__ Kv4Join kv4_join_row(const Kv4Attend &a, int row) {
    int seq, pos;
    const int st = kv4_row<32>(a.b, row, &seq, &pos);
    Kv4Join r{-1, 0, 0};
    if (st == KV4_ROW_NONE || st == KV4_ROW_STRAY) return r;
    r.r0 = 0;
    if (st == KV4_ROW_BAD) return r;
    const int r0 = a.b.row0[seq], n = a.b.row0[seq + 1] - r0, len = a.b.len[seq];
    if (n <= a.max_rows && len <= a.max_len) r = {r0, n, len};
    return r;
}
// how many spans of a (row, head) hold something (the row's column tile decides)
__device__ __forceinline__ int kv4_live_spans(const Kv4Attend &a, const Kv4Plan &pl, const Kv4Join &j, int row, int h) {
    if (j.n == 0) return 0;
    const int c0 = ((row - j.r0) * a.G + h % a.G) & -pl.cols, last = j.n * a.G - 1;      // (cols: a power of two)
    const int cz = c0 + pl.cols - 1 < last ? c0 + pl.cols - 1 : last;
    const Kv4Range cr = kv4_range(a, j.len - j.n + c0 / a.G, j.len - j.n + cz / a.G);
    const int live = (cr.hi_any - (cr.lo_any & ~(KV4_PAGE - 1)) + pl.span - 1) / pl.span;
    return live < pl.nsplit ? live : pl.nsplit;
}

// Joins up to 32 spans of a (row, head): a warp each, a span's {m, l} a lane.  A chain of loads (the row's sequence, {m, l},
// sums), so what counts is how many warps wait at once: 1568 rows x 20 heads x 96 dims in two spans 22 us, 34 us with half the
// warps, and 1024 rows x 32 heads x 128 dims in two 140 us when a CTA took a (row, head); with more spans than lanes a CTA does (kv4_merge_kernel).
constexpr int MG_T = 256;
__global__ void __launch_bounds__(MG_T, 3) kv4_merge_few_kernel(Kv4Attend a, Kv4Plan pl, const float *part) {
    const int hd = a.geo.hd, lane = threadIdx.x & 31, q4 = hd >> 2;
    const unsigned item = blockIdx.x * (MG_T / 32) + (threadIdx.x >> 5);
    pdl_trigger();
    pdl_wait();
    const int row = (int)(item / (unsigned)a.H), h = (int)item - row * a.H;
    if (row >= a.b.rows) return;
    const Kv4Join j = kv4_join_row(a, row);
    if (j.r0 < 0) return;
    const int live = kv4_live_spans(a, pl, j, row, h);
    const float *p = part + (size_t)item * pl.nsplit * (hd + 4);
    const float2 ml = lane < live ? *reinterpret_cast<const float2 *>(p + (size_t)lane * (hd + 4)) : make_float2(-INFINITY, 0.f);
    float4 v[8];                                             // the first spans' values on their way beside the {m, l}
    auto fetch = [&](int i0, int d) {
#pragma unroll
        for (int u = 0; u < 8; u++)
            if (i0 + u < live && d < q4) v[u] = reinterpret_cast<const float4 *>(p + (size_t)(i0 + u) * (hd + 4) + 4)[d];
    };
    fetch(0, lane);
    const float M = warp_max_f32(ml.x), f = kv4_factor(ml.y, ml.x, M);
    float L = ml.y * f;
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    const float over = kv4_over(L);
#pragma unroll 1
    for (int d0 = 0; d0 < q4; d0 += 32) {
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (int i0 = 0; i0 < live; i0 += 8) {
            if (d0 + i0 > 0) fetch(i0, d0 + lane);
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const float fi = __shfl_sync(0xffffffffu, f, i0 + u);
                if (fi != 0.f) { o.x = fmaf(v[u].x, fi, o.x); o.y = fmaf(v[u].y, fi, o.y); o.z = fmaf(v[u].z, fi, o.z); o.w = fmaf(v[u].w, fi, o.w); }
            }
        }
        if (d0 + lane < q4) reinterpret_cast<float4 *>(a.ctx + (size_t)item * hd)[d0 + lane] = kv4_times(o, over);
    }
}

// joins the many spans of one (row, head): the same sums over {m, l, acc}, a CTA each
__global__ void __launch_bounds__(MG_T) kv4_merge_kernel(Kv4Attend a, Kv4Plan pl, const float *part) {
    __shared__ float red[MG_T / 32], ls[MG_T / 8];
    __shared__ float4 os[MG_T];
    const int row = blockIdx.x, h = blockIdx.y, hd = a.geo.hd, tid = threadIdx.x;
    pdl_trigger();
    pdl_wait();
    const Kv4Join j = kv4_join_row(a, row);
    if (j.r0 < 0) return;
    const int live = kv4_live_spans(a, pl, j, row, h);
    float *out = a.ctx + ((size_t)row * a.H + h) * hd;
    const float *p = part + ((size_t)row * a.H + h) * pl.nsplit * (hd + 4);
    // thread group k takes spans k, k + ng, ...: four dims a thread, group order fixed; the first eight of its spans are
    // fetched beside the maxima
    const int q4 = hd / 4, ng = MG_T / q4, k = tid / q4, d = tid - k * q4, mine = k < ng ? live : 0;
    auto span = [&](int i) { return p + (size_t)i * (hd + 4); };
    float2 e[8];
    float4 v[8];
#pragma unroll
    for (int u = 0; u < 8; u++)
        if (k + u * ng < mine) {
            e[u] = *reinterpret_cast<const float2 *>(span(k + u * ng));
            v[u] = reinterpret_cast<const float4 *>(span(k + u * ng) + 4)[d];
        }
    float M = -INFINITY;
    for (int i = tid; i < live; i += MG_T) M = fmaxf(M, span(i)[0]);
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    if ((tid & 31) == 0) red[tid >> 5] = M;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < MG_T / 32; w++) M = fmaxf(M, red[w]);
    float L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](const float2 &ml, const float4 &x) {
        const float f = kv4_factor(ml.y, ml.x, M);
        L = fmaf(ml.y, f, L);
        if (ml.y != 0.f) { o.x = fmaf(x.x, f, o.x); o.y = fmaf(x.y, f, o.y); o.z = fmaf(x.z, f, o.z); o.w = fmaf(x.w, f, o.w); }
    };
#pragma unroll
    for (int u = 0; u < 8; u++) if (k + u * ng < mine) add(e[u], v[u]);
    for (int i = k + 8 * ng; i < mine; i += ng) add(*reinterpret_cast<const float2 *>(span(i)), reinterpret_cast<const float4 *>(span(i) + 4)[d]);
    if (k < ng) { os[k * q4 + d] = o; if (d == 0) ls[k] = L; }
    __syncthreads();
    if (k == 0) {
        for (int i = 1; i < ng; i++) {
            const float4 v = os[i * q4 + d];
            L += ls[i]; o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
        }
        *reinterpret_cast<float4 *>(out + 4 * d) = kv4_times(o, kv4_over(L));
    }
}

}  // namespace

// How a call is cut.  Host numbers only (the limits the caller gave), so a captured call stays valid for any batch within
// them.  Which kernel, by (row, query head) pairs of a KV head ("columns"):
//   decode, which re-reads the pages for every 8 columns, up to 48 of them (8 sequences of 4096, 4 KV heads, 48 columns: hd 128
//     48 us against 51 us of the matrix-instruction prompt kernel, hd 64 30 against 33, hd 256 86 against 103); up to 64 at
//     the narrowest and widest heads (56 columns: hd 32 31 against 38 us, hd 256 98 against 107; but
//     hd 64 41 against 34, hd 128 60 against 52, hd 160 74 against 67), and where there are six pages of 64 columns an SM or
//     fewer (one sequence of 1024, 56 columns: hd 64 9.3 against 10.8 us, hd 128 10.7 against 13.8, hd 160 11.9 against 17.1);
//   tensor memory above 64 columns at hd 64, 96, 128 when there are more than those six pages: below that its set-up (13 us) is
//     more than the matrix work it saves (one sequence of 1024, 8 KV heads, hd 128, 256 columns: 25 us against 21 us of
//     the other; of 4096: 33 us against 52 us; 8 of 4096: 119 us against 336 us).
// Spans of decode: with `units` (sequence, KV head, tile) triples of P pages on `slots` resident CTAs, a CTA costs its pages
// plus about FIX pages' time of set-up and join.  When all CTAs are resident at once the longest one counts; otherwise the
// total work over the slots plus a last CTA (lengths of a ragged batch are taken as 0.6 of the limit).  The cut with the
// least of that (64 sequences of up to 8192 positions, 32 heads on 8: 105 us).  A prompt is cut only to fill the GPU: the
// joins move rows x heads x hd x spans f32 values (4096 rows at 4096 positions, 16 heads: 175 us whole, 250 us in two spans;
// nine ragged sequences of up to 333 rows and 2900 positions 104 us whole, 124 us in two).
Kv4Plan kv4_plan(const Kv4Attend &a, int sms) {
    Kv4Plan p{};
    const long long cols = (long long)a.max_rows * a.G;
    const int NG = a.geo.hd / 32;
    const long long seen = a.window > 0 && a.window + 2LL * KV4_PAGE < a.max_len ? a.window + 2LL * KV4_PAGE : a.max_len;
    const long long pages64 = (long long)a.b.nseq * a.geo.KV * ((cols + 63) / 64) * ((seen + KV4_PAGE - 1) / KV4_PAGE);
    const bool many = pages64 > 6LL * sms;
    p.decode = cols <= 48 || (cols <= 64 && (NG == 1 || NG >= 6 || !many));
    p.tc = a.tc && cols > KV4_LINES && NG >= 2 && NG <= 4 && many;
    p.cols = p.tc ? KV4_TC_LINES : !p.decode ? KV4_LINES : cols > 4 ? 8 : 4;
    p.ntile = (int)((cols + p.cols - 1) / p.cols);
    if (p.ntile < 1) p.ntile = 1;
    // the longest stretch of positions a CTA's columns see together, from a page's first on
    long long range = a.max_len;
    const long long rows_a_tile = p.cols / a.G + 2 < a.max_rows ? p.cols / a.G + 2 : a.max_rows;
    if (a.window > 0 && (long long)a.window + rows_a_tile + KV4_PAGE < range) range = (long long)a.window + rows_a_tile + KV4_PAGE;
    const int occ = p.tc ? 1 : !p.decode ? 2 : p.cols == 4 ? kv4_decode_ctas(NG, true) : kv4_decode_ctas(NG, false);
    const double units = (double)a.b.nseq * a.geo.KV * p.ntile, slots = (double)sms * occ, FIX = 6;
    const long long P = (range + KV4_PAGE - 1) / KV4_PAGE, least = p.decode ? (P + DEC_NP - 1) / DEC_NP : p.tc ? (P + KV4_TC_PAGES - 1) / KV4_TC_PAGES : 1;
    const double w = a.b.nseq > 1 ? 0.6 : 1.0;
    long long best = least > 0 ? least : 1;
    double cost = 1e300;
    for (long long n = best; n <= P && n <= 1024 + best;) {
        const long long pages = (P + n - 1) / n;
        const double c = (units * n <= slots ? pages + FIX : units * (w * P + FIX * n) / slots + pages + FIX) + (n > 1 ? 2 : 0);
        if (c < cost) { cost = c; best = n; }
        if (pages == 1) break;
        n = (P + pages - 2) / (pages - 1);                     // the next that makes the spans shorter
    }
    if (!p.decode) best = units < slots ? (long long)(slots / units) : 1;
    if (best < least) best = least;
    if (best > P) best = P > 0 ? P : 1;
    const long long pages = P ? (P + best - 1) / best : 1;
    p.span = (int)(pages * KV4_PAGE);
    p.nsplit = (int)((range + p.span - 1) / p.span);
    if (p.nsplit < 1) p.nsplit = 1;
    return p;
}

size_t kv4_attend_scratch_bytes(const Kv4Attend &a, const Kv4Plan &p) {
    return p.nsplit > 1 ? (size_t)a.b.rows * a.H * p.nsplit * (a.geo.hd + 4) * 4 : 0;
}
// CTAs that count their spans' ends, when few spans are joined in the launch itself
size_t kv4_attend_counters(const Kv4Attend &a, const Kv4Plan &p) {
    return p.decode && p.nsplit > 1 && p.nsplit <= DEC_JOIN ? (size_t)a.b.nseq * a.geo.KV * p.ntile : 0;
}

template <int NG, bool PAIR, bool LONG>
static int kv4_decode_go(const Kv4Attend &a, const Kv4Plan &p, float *part, int *count, cudaStream_t st) {
    constexpr size_t smem = DecL<NG, PAIR>::SMEM;
    static bool attr[MOTY_MAX_DEV];
    int dev = 0;
    CK(cudaGetDevice(&dev));
    if (dev < 0 || dev >= MOTY_MAX_DEV) return moty_set_error(MOTY_CUDA_EARG, "kv4_attend: device %d", dev);
    if (!attr[dev]) {
        CK(cudaFuncSetAttribute(kv4_decode_kernel<NG, PAIR, LONG>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        attr[dev] = true;
    }
    const long long grid = (long long)a.b.nseq * a.geo.KV * p.ntile * p.nsplit;
    if (grid > 0x7fffffffLL) return moty_set_error(MOTY_CUDA_ELIMIT, "kv4_attend: %lld CTAs", grid);
    CK(moty_launch_pdl(kv4_decode_kernel<NG, PAIR, LONG>, dim3((unsigned)grid), dim3(DEC_W * 32), smem, st, a, p.ntile, p.nsplit, p.span, part, count));
    return 0;
}
template <int NG>
static int kv4_decode_go(const Kv4Attend &a, const Kv4Plan &p, float *part, int *count, cudaStream_t st) {
    const bool pair = p.cols == 4;
    if (p.span / KV4_PAGE > kv4_decode_long(pair)) return pair ? kv4_decode_go<NG, true, true>(a, p, part, count, st) : kv4_decode_go<NG, false, true>(a, p, part, count, st);
    return pair ? kv4_decode_go<NG, true, false>(a, p, part, count, st) : kv4_decode_go<NG, false, false>(a, p, part, count, st);
}

// part: scratch of kv4_attend_scratch_bytes; count: kv4_attend_counters ints, all zero (and left so)
int launch_kv4_attend(const Kv4Attend &a, const Kv4Plan &p, float *part, int *count, cudaStream_t st) {
    if (p.nsplit > 1 && !part) return moty_set_error(MOTY_CUDA_EARG, "kv4_attend: scratch for %d spans missing", p.nsplit);
    int rc = 0;
    if (p.tc) rc = launch_kv4_prompt_tc(a, p, part, st);
    else if (!p.decode) rc = launch_kv4_prompt(a, p, part, st);
    else switch (a.geo.hd / 32) {
        case 1: rc = kv4_decode_go<1>(a, p, part, count, st); break;
        case 2: rc = kv4_decode_go<2>(a, p, part, count, st); break;
        case 3: rc = kv4_decode_go<3>(a, p, part, count, st); break;
        case 4: rc = kv4_decode_go<4>(a, p, part, count, st); break;
        case 5: rc = kv4_decode_go<5>(a, p, part, count, st); break;
        case 6: rc = kv4_decode_go<6>(a, p, part, count, st); break;
        case 7: rc = kv4_decode_go<7>(a, p, part, count, st); break;
        default: rc = kv4_decode_go<8>(a, p, part, count, st); break;
    }
    CKR(rc);
    if (p.nsplit > 1 && !count) {
        if (p.nsplit <= 32)
            CK(moty_launch_pdl(kv4_merge_few_kernel, dim3((unsigned)(((long long)a.b.rows * a.H + MG_T / 32 - 1) / (MG_T / 32))), dim3(MG_T), (size_t)0, st, a, p, (const float *)part));
        else CK(moty_launch_pdl(kv4_merge_kernel, dim3(a.b.rows, a.H), dim3(MG_T), (size_t)0, st, a, p, (const float *)part));
    }
    return 0;
}
