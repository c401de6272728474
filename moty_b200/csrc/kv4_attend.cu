// kv4_attend.cu -- attention over the paged 4-bit KV cache.
//
// For row r of a sequence at position p, query head h of KV head h / G:
//     s_t = scale * q . k_t,   ctx = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m)   over t in (p - window, p],
// k_t and v_t the values held (code * step), positions of absent pages (table entry -1) left out, 0 where nothing is left.
#include "kv4_frag.cuh"
#include "kv4_attend.cuh"

namespace {

// ---- few rows a sequence (decode) ------------------------------------------------------------------------------------
// A CTA takes one KV head of one sequence, up to 4 NT (row, query head) pairs of it ("columns"), and a span of positions;
// its warps walk the span 16 positions at a time, straight from global memory into matrix operands:
//     scores  [16 positions x 2 columns a pair] = codes [16 x 32] (a group) * q pieces, times the position's step, group by group
//     output  [32 dims x 2 columns a pair]     += codes [dims x 16 positions] * (weight * value step) pieces
// The two columns of a pair are the hi and lo piece of its f32 operand and land in the same thread, which adds them.  Every
// warp keeps its own running maximum (moved only when a score passes it by 8 in base-2 units, so weights stay below 256)
// and exponent of the largest value step (so that weight * step fits f16); warps join in shared memory, spans through
// `part` ({m, l, acc[hd]} per (row, head, split)) and kv4_merge_kernel.
constexpr int DEC_W = 4;                                     // warps a CTA

template <int NG, int NT>
__global__ void __launch_bounds__(DEC_W * 32) kv4_decode_kernel(Kv4Attend a, int ntile, int nsplit, int span, float *part) {
    constexpr int HD = NG * 32, NC = NT * 4;                 // columns (pairs) of the CTA
    extern __shared__ float sm_kv4[];
    float *qs = sm_kv4;                                      // [NC][HD] the query rows; later acc[DEC_W][NC][HD]
    float *ml = sm_kv4 + DEC_W * NC * HD;                    // m, l [DEC_W][NC], then descale [NC]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = lane >> 2, j = lane & 3;
    const int split = blockIdx.x % nsplit;
    const int u = blockIdx.x / nsplit, tile = u % ntile, head = (u / ntile) % a.geo.KV, seq = u / ntile / a.geo.KV;
    pdl_trigger();
    pdl_wait();
    const Kv4Seq sq = kv4_load_seq(a, seq);
    if (!sq.ok) {
        if (nsplit == 1 && tile == 0) kv4_zero_rows(a, sq, head);
        return;
    }
    const int c0 = tile * NC, ncol = sq.n * a.G - c0 < NC ? sq.n * a.G - c0 : NC;
    if (ncol <= 0) return;
    const int pos0 = sq.len - sq.n;                          // position of the sequence's first row
    const int row_a = c0 / a.G, row_z = (c0 + ncol - 1) / a.G;
    const Kv4Range cr = kv4_range(a, pos0 + row_a, pos0 + row_z);
    const int t_lo = (cr.lo_any & ~15) + split * span, t_hi = cr.hi_any - t_lo < span ? cr.hi_any : t_lo + span;
    if (t_lo >= cr.hi_any && nsplit > 1) return;             // nothing in this span: the merge does not look at it
    // query rows, then their two pieces as operands: column 2 c + piece, k = the dims of a word's nibble pairs
    for (int c = warp; c < NC; c += DEC_W) {
        float am = 0.f, x[NG];
        unsigned mb = 0;
        const int cc = c0 + c;
        if (c < ncol) {
            const float *src = a.q + (size_t)(sq.r0 + cc / a.G) * a.q_ld + (size_t)(head * a.G + cc % a.G) * HD;
#pragma unroll
            for (int g = 0; g < NG; g++) { x[g] = src[g * 32 + lane]; const unsigned b = __float_as_uint(fabsf(x[g])); mb = b > mb ? b : mb; }
        } else {
#pragma unroll
            for (int g = 0; g < NG; g++) x[g] = 0.f;
        }
        for (int off = 16; off > 0; off >>= 1) { const unsigned o = __shfl_xor_sync(0xffffffffu, mb, off); mb = o > mb ? o : mb; }
        am = __uint_as_float(mb);
        // |q| 2^k < 2^14; a row that is not finite has NaN scores
        const bool fin = mb < 0x7f800000u;
        const int k = fin && am > 0.f ? 13 - ilogbf(am) : 0;
#pragma unroll
        for (int g = 0; g < NG; g++) qs[c * HD + g * 32 + lane] = fin ? scalbnf(x[g], k) : 0.f;
        if (lane == 0) ml[2 * DEC_W * NC + c] = fin ? (float)ldexp((double)a.scale * 1.4426950408889634, -k) : __int_as_float(0x7fffffff);
    }
    __syncthreads();
    unsigned qf[NT][NG][4];
    float desc[NT];
    int clo[NT], chi[NT];
    const float sel = (r & 1) ? 1.f : 0.f;                   // operand column r: pair r / 2, piece r & 1
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const float *qc = qs + (nt * 4 + (r >> 1)) * HD;
#pragma unroll
        for (int g = 0; g < NG; g++)
#pragma unroll
            for (int i = 0; i < 4; i++) qf[nt][g][i] = kv4_piece(qc[g * 32 + 8 * j + i], qc[g * 32 + 8 * j + i + 4], sel);
        const int cc = c0 + nt * 4 + j;                      // the pair whose scores this thread holds
        desc[nt] = ml[2 * DEC_W * NC + nt * 4 + j];
        const int p = pos0 + cc / a.G;
        chi[nt] = nt * 4 + j < ncol ? p : -1;
        clo[nt] = a.window > 0 && p - a.window + 1 > 0 ? p - a.window + 1 : 0;
    }
    __syncthreads();                                         // qs is reused for the join
    float m[NT], l[NT], acc[NT][NG][2][4];
    int ve = -24;                                            // exponent of the largest value step so far
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        m[nt] = -INFINITY; l[nt] = 0.f;
#pragma unroll
        for (int g = 0; g < NG; g++)
#pragma unroll
            for (int i = 0; i < 8; i++) acc[nt][g][i >> 2][i & 3] = 0.f;
    }
    const int *tab = a.b.table + (size_t)seq * a.b.ld;
    for (int t0 = t_lo + warp * 16; t0 < t_hi; t0 += DEC_W * 16) {
        const int page = tab[t0 / KV4_PAGE];
        if (!kv4_page_ok(a.geo, page)) { if (page != -1 && lane == 0) atomicExch(a.err, 1); continue; }
        const uint8_t *unit = a.mem + kv4_unit_off(a.geo, page, a.layer, head);
        const int tp = t0 % KV4_PAGE;                        // 16 positions of one block
        unsigned ka[NG], kb[NG], va[NG], vb[NG], sa[(NG + 1) / 2], sb[(NG + 1) / 2], wa[NG], wb[NG];
        kv4_ldw<NG>(ka, unit + (tp + r) * (HD / 2) + j * (4 * NG));
        kv4_ldw<NG>(kb, unit + (tp + r + 8) * (HD / 2) + j * (4 * NG));
        kv4_ldsteps<NG>(sa, unit + kv4_k_step_off(HD) + (tp + r) * (2 * NG));
        kv4_ldsteps<NG>(sb, unit + kv4_k_step_off(HD) + (tp + r + 8) * (2 * NG));
        kv4_ldw<NG>(va, unit + kv4_v_code_off(HD) + (tp >> 4) * (8 * HD) + lane * (4 * NG));
        kv4_ldw<NG>(vb, unit + kv4_v_code_off(HD) + (tp >> 4) * (8 * HD) + 4 * HD + lane * (4 * NG));
        kv4_ldw<NG>(wa, unit + kv4_v_step_off(HD) + (tp + 2 * j) * (2 * NG));
        kv4_ldw<NG>(wb, unit + kv4_v_step_off(HD) + (tp + 8 + 2 * j) * (2 * NG));
        // scores of positions t0 + r and t0 + r + 8 for the thread's pairs
        float s[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) s[nt][0] = s[nt][1] = 0.f;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            unsigned ea[4], eb[4];
            kv4_codes(ka[g], ea);
            kv4_codes(kb[g], eb);
            const float da = kv4_half_of(sa[g >> 1], g & 1), db = kv4_half_of(sb[g >> 1], g & 1);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float c[4] = {0.f, 0.f, 0.f, 0.f};
                kv4_mma(c, ea[0], eb[0], ea[1], eb[1], qf[nt][g][0], qf[nt][g][1]);
                kv4_mma(c, ea[2], eb[2], ea[3], eb[3], qf[nt][g][2], qf[nt][g][3]);
                s[nt][0] = fmaf(da, c[0] + c[1], s[nt][0]);
                s[nt][1] = fmaf(db, c[2] + c[3], s[nt][1]);
            }
        }
        const bool inside = t0 >= cr.lo_all && t0 + 15 < cr.hi_all;      // (columns past ncol hold zero rows, and are not written)
        bool up = false;
        bool see[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            s[nt][0] *= desc[nt]; s[nt][1] *= desc[nt];
            see[nt][0] = inside || (t0 + r >= clo[nt] && t0 + r <= chi[nt]);
            see[nt][1] = inside || (t0 + r + 8 >= clo[nt] && t0 + r + 8 <= chi[nt]);
            if (!see[nt][0]) s[nt][0] = -INFINITY;
            if (!see[nt][1]) s[nt][1] = -INFINITY;
            up |= fmaxf(s[nt][0], s[nt][1]) > m[nt] + 8.f;
        }
        if (__any_sync(0xffffffffu, up)) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float mx = fmaxf(s[nt][0], s[nt][1]);
                for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
                const float mn = fmaxf(m[nt], mx), f = mn == -INFINITY ? 1.f : kv4_exp2(m[nt] - mn);
                m[nt] = mn; l[nt] *= f;
#pragma unroll
                for (int g = 0; g < NG; g++)
#pragma unroll
                    for (int i = 0; i < 8; i++) acc[nt][g][i >> 2][i & 3] *= f;
            }
        }
        if (!inside) {
            kv4_mask_steps<NG>(wa, t0 + 2 * j, cr.lo_any, cr.hi_any);
            kv4_mask_steps<NG>(wb, t0 + 8 + 2 * j, cr.lo_any, cr.hi_any);
        }
        // the largest value step (NaN left aside) decides the power of two that weight * step is scaled by
        {
            __half2 mx = __halves2half2(__ushort_as_half(0), __ushort_as_half(0));
#pragma unroll
            for (int g = 0; g < NG; g++) {
                mx = __hmax2(mx, __habs2(*reinterpret_cast<const __half2 *>(&wa[g])));
                mx = __hmax2(mx, __habs2(*reinterpret_cast<const __half2 *>(&wb[g])));
            }
            const float big = fmaxf(__low2float(mx), __high2float(mx));
            if (__any_sync(0xffffffffu, big >= scalbnf(2.f, ve))) {
                unsigned b = __float_as_uint(big);
                for (int off = 16; off > 0; off >>= 1) { const unsigned o = __shfl_xor_sync(0xffffffffu, b, off); b = o > b ? o : b; }
                const int e = (int)(b >> 23) - 127;          // (f16 subnormals are normal f32)
                const float f = scalbnf(1.f, ve - e);
                ve = e;
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int g = 0; g < NG; g++)
#pragma unroll
                        for (int i = 0; i < 8; i++) acc[nt][g][i >> 2][i & 3] *= f;
            }
        }
        const float vn = scalbnf(64.f, -ve);                 // weight * step * vn < 256 * 2 * 64 = 2^15
        float y[NT][4];                                      // scaled weights of positions 2 j, 2 j + 1, 2 j + 8, 2 j + 9 for column r; < 0: not seen
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float p0 = kv4_exp2(s[nt][0] - m[nt]), p1 = kv4_exp2(s[nt][1] - m[nt]);
            if (!see[nt][0]) p0 = 0.f;
            if (!see[nt][1]) p1 = 0.f;
            l[nt] += p0 + p1;
            p0 = see[nt][0] ? p0 * vn : -1.f; p1 = see[nt][1] ? p1 * vn : -1.f;
            const int src = 8 * j + (r >> 1);
            y[nt][0] = __shfl_sync(0xffffffffu, p0, src); y[nt][1] = __shfl_sync(0xffffffffu, p0, src + 4);
            y[nt][2] = __shfl_sync(0xffffffffu, p1, src); y[nt][3] = __shfl_sync(0xffffffffu, p1, src + 4);
        }
#pragma unroll
        for (int g = 0; g < NG; g++) {
            unsigned ea[4], eb[4];
            kv4_codes(va[g], ea);
            kv4_codes(vb[g], eb);
            const float d0 = kv4_half_of(wa[g >> 1], g & 1), d1 = kv4_half_of(wa[(NG + g) >> 1], (NG + g) & 1);
            const float d2 = kv4_half_of(wb[g >> 1], g & 1), d3 = kv4_half_of(wb[(NG + g) >> 1], (NG + g) & 1);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                // a position that is not seen adds nothing, whatever its step holds
                const float x0 = y[nt][0] < 0.f ? 0.f : y[nt][0] * d0, x1 = y[nt][1] < 0.f ? 0.f : y[nt][1] * d1;
                const float x2 = y[nt][2] < 0.f ? 0.f : y[nt][2] * d2, x3 = y[nt][3] < 0.f ? 0.f : y[nt][3] * d3;
                const unsigned b0 = kv4_piece(x0, x1, sel), b1 = kv4_piece(x2, x3, sel);
                kv4_mma(acc[nt][g][0], ea[0], ea[1], eb[0], eb[1], b0, b1);
                kv4_mma(acc[nt][g][1], ea[2], ea[3], eb[2], eb[3], b0, b1);
            }
        }
    }
    // join the warps: every thread holds, for pair j of each tile, dims 32 g + 4 r + 0 .. 3
    const float vs = scalbnf(1.f / 64.f, ve);
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        for (int off = 4; off < 32; off <<= 1) l[nt] += __shfl_xor_sync(0xffffffffu, l[nt], off);
        const int c = nt * 4 + j;
#pragma unroll
        for (int g = 0; g < NG; g++)
            *reinterpret_cast<float4 *>(qs + ((size_t)warp * NC + c) * HD + g * 32 + 4 * r) =
                make_float4((acc[nt][g][0][0] + acc[nt][g][0][1]) * vs, (acc[nt][g][0][2] + acc[nt][g][0][3]) * vs,
                            (acc[nt][g][1][0] + acc[nt][g][1][1]) * vs, (acc[nt][g][1][2] + acc[nt][g][1][3]) * vs);
        if (r == 0) { ml[warp * NC + c] = m[nt]; ml[DEC_W * NC + warp * NC + c] = l[nt]; }
    }
    __syncthreads();
    for (int i = tid; i < ncol * HD; i += DEC_W * 32) {
        const int c = i / HD, d = i - c * HD, cc = c0 + c;
        float M = -INFINITY, L = 0.f, o = 0.f;
#pragma unroll
        for (int w = 0; w < DEC_W; w++) M = fmaxf(M, ml[w * NC + c]);
#pragma unroll
        for (int w = 0; w < DEC_W; w++) {
            const float lw = ml[DEC_W * NC + w * NC + c], f = lw == 0.f ? 0.f : kv4_exp2(ml[w * NC + c] - M);
            L = fmaf(lw, f, L);
            o = fmaf(lw == 0.f ? 0.f : qs[((size_t)w * NC + c) * HD + d], f, o);
        }
        const size_t rh = (size_t)(sq.r0 + cc / a.G) * a.H + head * a.G + cc % a.G;
        if (nsplit == 1) a.ctx[rh * HD + d] = L == 0.f ? 0.f : __fdiv_rn(o, L);
        else {
            float *p = part + (rh * nsplit + split) * (HD + 4);
            p[4 + d] = o;
            if (d == 0) { p[0] = M; p[1] = L; }
        }
    }
}

// joins the spans of one (row, head): the same sums over {m, l, acc} with the maximum over all spans
__global__ void __launch_bounds__(256) kv4_merge_kernel(Kv4Attend a, Kv4Plan pl, const float *part) {
    const int row = blockIdx.x, h = blockIdx.y, hd = a.geo.hd, d = threadIdx.x;
    pdl_trigger();
    pdl_wait();
    int seq, pos;
    const int st = kv4_row(a.b, row, &seq, &pos);
    if (st == KV4_ROW_NONE) return;
    float *out = a.ctx + ((size_t)row * a.H + h) * hd + d;
    const int n = st == KV4_ROW_OK ? a.b.row0[seq + 1] - a.b.row0[seq] : 0;
    if (st == KV4_ROW_BAD || n > a.max_rows || a.b.len[seq] > a.max_len) { *out = 0.f; return; }
    // the spans that hold anything for this row's column tile
    const long long c = (long long)(row - a.b.row0[seq]) * a.G + h % a.G, c0 = c / pl.cols * pl.cols, last = (long long)n * a.G - 1;
    const long long cz = c0 + pl.cols - 1 < last ? c0 + pl.cols - 1 : last;
    const int pos0 = a.b.len[seq] - n;
    const Kv4Range cr = kv4_range(a, pos0 + (int)(c0 / a.G), pos0 + (int)(cz / a.G));
    int live = (cr.hi_any - (cr.lo_any & ~(pl.align - 1)) + pl.span - 1) / pl.span;
    if (live > pl.nsplit) live = pl.nsplit;
    const float *p = part + ((size_t)row * a.H + h) * pl.nsplit * (hd + 4);
    float M = -INFINITY, L = 0.f, o = 0.f;
    for (int i = 0; i < live; i++) M = fmaxf(M, p[(size_t)i * (hd + 4)]);
    for (int i = 0; i < live; i++) {
        const float li = p[(size_t)i * (hd + 4) + 1], f = li == 0.f ? 0.f : kv4_exp2(p[(size_t)i * (hd + 4)] - M);
        L = fmaf(li, f, L);
        o = fmaf(li == 0.f ? 0.f : p[(size_t)i * (hd + 4) + 4 + d], f, o);
    }
    *out = L == 0.f ? 0.f : __fdiv_rn(o, L);
}

}  // namespace

// how a call is cut
static Kv4Plan kv4_plan(const Kv4Attend &a, int sms) {
    Kv4Plan p{};
    const long long cols = (long long)a.max_rows * a.G;
    p.decode = cols <= 32;
    p.nt = cols > 4 && a.geo.hd <= 128 ? 2 : 1;
    p.cols = p.decode ? 4 * p.nt : KV4_LINES;
    p.align = p.decode ? 16 : KV4_PAGE;
    p.ntile = (int)((cols + p.cols - 1) / p.cols);
    if (p.ntile < 1) p.ntile = 1;
    // the longest stretch of positions a CTA's columns see together, from a multiple of `align` on
    long long range = a.max_len;
    const long long rows_a_tile = p.cols / a.G + 2 < a.max_rows ? p.cols / a.G + 2 : a.max_rows;
    if (a.window > 0 && (long long)a.window + rows_a_tile + p.align < range) range = (long long)a.window + rows_a_tile + p.align;
    const long long units = (long long)a.b.nseq * a.geo.KV * p.ntile, most = (range + 63) / 64;
    long long n = p.decode ? (6LL * sms + units - 1) / units : units < 2LL * sms ? (3LL * sms + units - 1) / units : 1;
    if (n > most) n = most;
    if (n < 1) n = 1;
    long long span = (range + n - 1) / n;
    span = (span + 63) / 64 * 64;
    if (span < 64) span = 64;
    p.span = (int)span;
    p.nsplit = (int)((range + span - 1) / span);
    if (p.nsplit < 1) p.nsplit = 1;
    return p;
}

size_t kv4_attend_scratch_bytes(const Kv4Attend &a, int sms) {
    const Kv4Plan p = kv4_plan(a, sms);
    return p.nsplit > 1 ? (size_t)a.b.rows * a.H * p.nsplit * (a.geo.hd + 4) * 4 : 0;
}

template <int NG, int NT>
static int kv4_decode_go(const Kv4Attend &a, const Kv4Plan &p, float *part, cudaStream_t st) {
    constexpr size_t smem = ((size_t)DEC_W * NT * 4 * NG * 32 + 2 * DEC_W * NT * 4 + NT * 4) * 4;
    static_assert(smem <= 48 * 1024, "fits without an attribute");
    const long long grid = (long long)a.b.nseq * a.geo.KV * p.ntile * p.nsplit;
    if (grid > 0x7fffffffLL) return moty_set_error(MOTY_CUDA_ELIMIT, "kv4_attend: %lld CTAs", grid);
    CK(moty_launch_pdl(kv4_decode_kernel<NG, NT>, dim3((unsigned)grid), dim3(DEC_W * 32), smem, st, a, p.ntile, p.nsplit, p.span, part));
    return 0;
}

int launch_kv4_attend(const Kv4Attend &a, float *part, int sms, cudaStream_t st) {
    const Kv4Plan p = kv4_plan(a, sms);
    if (p.nsplit > 1 && !part) return moty_set_error(MOTY_CUDA_EARG, "kv4_attend: scratch for %d spans missing", p.nsplit);
    int rc = 0;
    if (!p.decode) rc = launch_kv4_prompt(a, p, part, st);
    else switch (a.geo.hd / 32) {
        case 1: rc = p.nt == 2 ? kv4_decode_go<1, 2>(a, p, part, st) : kv4_decode_go<1, 1>(a, p, part, st); break;
        case 2: rc = p.nt == 2 ? kv4_decode_go<2, 2>(a, p, part, st) : kv4_decode_go<2, 1>(a, p, part, st); break;
        case 3: rc = p.nt == 2 ? kv4_decode_go<3, 2>(a, p, part, st) : kv4_decode_go<3, 1>(a, p, part, st); break;
        case 4: rc = p.nt == 2 ? kv4_decode_go<4, 2>(a, p, part, st) : kv4_decode_go<4, 1>(a, p, part, st); break;
        case 5: rc = kv4_decode_go<5, 1>(a, p, part, st); break;
        case 6: rc = kv4_decode_go<6, 1>(a, p, part, st); break;
        case 7: rc = kv4_decode_go<7, 1>(a, p, part, st); break;
        default: rc = kv4_decode_go<8, 1>(a, p, part, st); break;
    }
    CKR(rc);
    if (p.nsplit > 1)
        CK(moty_launch_pdl(kv4_merge_kernel, dim3(a.b.rows, a.H), dim3(a.geo.hd), (size_t)0, st, a, p, (const float *)part));
    return 0;
}
