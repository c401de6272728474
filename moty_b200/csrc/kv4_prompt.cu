// kv4_prompt.cu -- attention over the paged 4-bit KV cache for many rows a sequence (prompts).
//
// A CTA takes 16 PR_W (row, query head) pairs ("lines") of one KV head of one sequence, 16 a warp, and walks the pages of
// its span; a page's unit (codes and steps, 72 hd bytes) is brought to shared memory as it is, the next one while this one
// is used.  As in the decode kernel the codes go into the 16-bit matrix instruction as exact small integers and the f32
// operand (query, then weight * value step) as two f16 pieces, here the wide operand:
//     scores [16 lines x 8 positions] += (q hi + q lo) [16 x 32 dims of a group] * codes, then times the positions' steps
//     output [16 lines x 8 dims]      += (x hi + x lo) [16 x 16 positions] * codes,   x = weight * step of the dims' group
// The score fragment of two 8-position tiles is the weight fragment of the second product, so weights never leave the
// thread.  Query pieces stay in shared memory in fragment order.  The weights' reference is moved up and down as in the decode
// kernel, so that a line's largest weight of a pass (8 PT positions) lies between 2^-6 and 2^5; x, scaled by the exponent of the
// largest value step so far and 2^9, then lies below 2^15, and its pieces end at 2^-28 of those two's product at worst.
// It serves the head widths that the tensor-memory kernel has no operand tiles for, and calls too short for that kernel's
// set-up.  What bounds it: two pieces make two matrix instructions of half the rate a product, and turning codes into
// operands is done by every warp for itself; 4096 rows at 4096 positions, 16 heads on 8, hd 128: 586 us (tensor memory:
// 175 us), one sequence of 1024, 64 rows, 32 heads on 8: 21 us (25 us); 2048 rows, 16 heads on 4: hd 32 110 us, 160 213,
// 192 248, 224 291, 256 334.
#include "kv4_frag.cuh"
#include "kv4_attend.cuh"

namespace {

constexpr int PR_W = KV4_LINES / 16, PR_F = 16;              // warps a CTA; pages of a lower sum
// exponents of a line's largest weight of a pass: the range it may have (PR_LOW: where every lane has one as large), where it is
// put, and how far below the highest reference so far one may be
constexpr float PR_HI = 5.f, PR_LO = -4.f, PR_LOW = -6.f, PR_AT = 0.f, PR_DOWN = 60.f;

template <int NG> struct PrL {
    static constexpr int HD = NG * 32, UNIT = 72 * HD, PT = NG <= 4 ? 4 : 2;
    static constexpr size_t SMEM = (size_t)PR_W * NG * 4 * 512 + 2 * UNIT;
};

template <int NG>
__global__ void __launch_bounds__(PR_W * 32, NG == 1 ? 5 : 2) kv4_prompt_kernel(Kv4Attend a, int ntile, int nsplit, int span, float *part) {
    constexpr int HD = NG * 32, UNIT = PrL<NG>::UNIT, PT = PrL<NG>::PT, NL = 16 * PR_W;
    extern __shared__ __align__(128) uint8_t sm_kv4p[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = lane >> 2, j = lane & 3;
    uint8_t *qw = sm_kv4p + (size_t)warp * NG * 4 * 512;     // this warp's query pieces [g][step][piece][lane] x 16 bytes
    uint8_t *stage = sm_kv4p + (size_t)PR_W * NG * 4 * 512;
    // (head, sequence) pairs of the last line tiles first: under a causal mask they see the most positions
    const int split = blockIdx.x % nsplit, u = blockIdx.x / nsplit;
    const int tile = ntile - 1 - u / (a.geo.KV * a.b.nseq), hs = u % (a.geo.KV * a.b.nseq), head = hs % a.geo.KV, seq = hs / a.geo.KV;
    pdl_trigger();
    pdl_wait();
    const Kv4Seq sq = kv4_load_seq(a, seq);
    if (!sq.ok) {
        if (nsplit == 1 && tile == 0) kv4_zero_rows(a, sq, head);
        return;
    }
    const int lines = sq.n * a.G, c0 = tile * NL;            // (rows * heads of a call stay below 2^31)
    if (c0 >= lines) return;
    const int ncol = lines - c0 < NL ? lines - c0 : NL;
    const int pos0 = sq.len - sq.n, row_a = c0 / a.G, row_z = (c0 + ncol - 1) / a.G;
    const Kv4Range cr = kv4_range(a, pos0 + row_a, pos0 + row_z);
    const int t_lo = (cr.lo_any & ~(KV4_PAGE - 1)) + split * span, t_hi = cr.hi_any - t_lo < span ? cr.hi_any : t_lo + span;
    if (t_lo >= cr.hi_any && nsplit > 1) return;
    // the warp's own lines
    const int w0 = warp * 16, wn = ncol - w0 < 16 ? ncol - w0 : 16;          // valid lines of the warp (may be <= 0)
    Kv4Range wr = kv4_range(a, 0, 0);
    if (wn > 0) wr = kv4_range(a, pos0 + (c0 + w0) / a.G, pos0 + (c0 + w0 + wn - 1) / a.G);
    float desc[2];
    int clo[2], chi[2];
#pragma unroll
    for (int hlf = 0; hlf < 2; hlf++) {
        const int line = r + 8 * hlf;
        const int cc = c0 + w0 + line;
        const bool have = line < wn;
        const int row = have ? cc / a.G : 0, g0 = have ? cc % a.G : 0;
        const float *src = a.q + (size_t)(sq.r0 + row) * a.q_ld + (size_t)(head * a.G + g0) * HD;
        unsigned mb = 0;
        if (have) {
#pragma unroll
            for (int g = 0; g < NG; g++)
#pragma unroll
                for (int h4 = 0; h4 < 2; h4++) {
                    const uint4 v = *reinterpret_cast<const uint4 *>(src + g * 32 + 8 * j + 4 * h4);
                    mb = max(max(max(v.x & 0x7fffffffu, v.y & 0x7fffffffu), max(v.z & 0x7fffffffu, v.w & 0x7fffffffu)), mb);
                }
        }
        mb = max(mb, __shfl_xor_sync(0xffffffffu, mb, 1));
        mb = max(mb, __shfl_xor_sync(0xffffffffu, mb, 2));
        const bool fin = mb < 0x7f800000u;                   // |q| 2^k < 2^14; a line that is not finite has NaN scores
        const int k = fin ? kv4_q_shift(mb) : 0;
        desc[hlf] = fin ? kv4_scale2(a.scale * 1.44269504f, -k) : __int_as_float(0x7fffffff);
        const int p = pos0 + row;
        chi[hlf] = have ? p : -1;
        clo[hlf] = a.window > 0 && p - a.window + 1 > 0 ? p - a.window + 1 : 0;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = 0.f;
            if (have && fin) {
                const float4 v0 = *reinterpret_cast<const float4 *>(src + g * 32 + 8 * j), v1 = *reinterpret_cast<const float4 *>(src + g * 32 + 8 * j + 4);
                x[0] = v0.x; x[1] = v0.y; x[2] = v0.z; x[3] = v0.w; x[4] = v1.x; x[5] = v1.y; x[6] = v1.z; x[7] = v1.w;
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = kv4_scale2(x[i], k);
            }
            // step s covers nibbles 2 s and 2 s + 1 of a word and their partners 4 on: registers 0, 2 (line r) and 1, 3 (line r + 8)
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int pc = 0; pc < 2; pc++) {
                    unsigned *dst = reinterpret_cast<unsigned *>(qw + ((g * 2 + s) * 2 + pc) * 512 + lane * 16);
                    dst[hlf] = kv4_piece(x[2 * s], x[2 * s + 4], pc ? KV4_HM1 : KV4_H0);
                    dst[2 + hlf] = kv4_piece(x[2 * s + 1], x[2 * s + 5], pc ? KV4_HM1 : KV4_H0);
                }
        }
    }
    __syncwarp();
    float m[2] = {-INFINITY, -INFINITY}, mh[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, acc[NG][4][4];    // m: the reference, mh: the highest so far
#pragma unroll
    for (int g = 0; g < NG; g++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[g][i >> 2][i & 3] = 0.f;
    // Sums over a long span are made in two levels: l and acc take PR_F pages and are then added to lt and tot (in local
    // memory), which keep the maximum and the scale that they were left with.  One level alone: 131072 flat weights 1e-4 off.
    volatile float lt[2] = {0.f, 0.f}, mt[2] = {-INFINITY, -INFINITY}, vnt = 0.f, tot[NG * 16];
    int passes = 0;                                          // (tot holds nothing before PR_F pages of them)
    float vth = 0.f, vn = 0.f;                               // 2^(e + 1) and 2^9 * 2^-e for the exponent e of the largest value step so far
    const int *tab = a.b.table + (size_t)seq * a.b.ld;
    const uint8_t *base = a.mem + (size_t)(a.layer * a.geo.KV + head) * UNIT;
    const size_t page_bytes = kv4_page_bytes(a.geo);
    // factors that bring lt (of a line) and tot to the present maximum and scale
    auto total_factors = [&](float (&fl)[2], float (&fa)[2]) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            fl[h] = mt[h] == m[h] ? 1.f : kv4_exp2(mt[h] - m[h]);
            fa[h] = vnt == vn ? fl[h] : vnt == 0.f ? 0.f : fl[h] * (vn / vnt);
        }
    };
    auto fetch = [&](int t, int buf) {                       // the unit of position t's page to a stage; false: absent
        bool ok = false;
        if (t < t_hi) {
            const int page = tab[t / KV4_PAGE];
            ok = kv4_page_ok(a.geo, page);
            if (ok) {
                const uint8_t *src = base + (size_t)page * page_bytes;
                for (int i = tid; i < UNIT / 16; i += PR_W * 32) cp_async16(stage + buf * UNIT + i * 16, src + i * 16);
            } else if (page != -1 && tid == 0) atomicExch(a.err, 1);
        }
        cp_async_commit();
        return ok;
    };
    bool have_next = fetch(t_lo, 0);
    for (int t0 = t_lo, buf = 0; t0 < t_hi; t0 += KV4_PAGE, buf ^= 1) {
        const bool have = have_next;
        cp_async_wait<0>();
        __syncthreads();                                     // the page is there for all; the other stage is free
        have_next = fetch(t0 + KV4_PAGE, buf ^ 1);
        if (!have || wn <= 0) continue;
        const uint8_t *unit = stage + buf * UNIT;
        for (int pp = 0; pp < KV4_PAGE / (8 * PT); pp++) {
            const int tp = pp * 8 * PT, tb = t0 + tp;        // 8 PT positions from tb on
            if (tb >= wr.hi_any || tb >= t_hi) break;
            if (tb + 8 * PT <= wr.lo_any) continue;
            float s[PT][4];
#pragma unroll
            for (int nt = 0; nt < PT; nt++)
#pragma unroll
                for (int i = 0; i < 4; i++) s[nt][i] = 0.f;
            {
                unsigned kw[PT][NG], ks[PT][NG];             // codes of position 8 nt + r; steps of positions 8 nt + 2 j, + 1
#pragma unroll
                for (int nt = 0; nt < PT; nt++) {
                    kv4_ldsw<NG>(kw[nt], unit + (tp + nt * 8 + r) * (HD / 2) + j * (4 * NG));
                    kv4_ldsw<NG>(ks[nt], unit + kv4_k_step_off(HD) + (tp + nt * 8 + 2 * j) * (2 * NG));
                }
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    uint4 qf[2][2];
#pragma unroll
                    for (int i = 0; i < 4; i++) qf[i >> 1][i & 1] = *reinterpret_cast<const uint4 *>(qw + (g * 4 + i) * 512 + lane * 16);
#pragma unroll
                    for (int nt = 0; nt < PT; nt++) {
                        unsigned e[4];
                        kv4_codes(kw[nt][g], e);
                        float c[4];
#pragma unroll
                        for (int st = 0; st < 2; st++) {
                            if (st == 0) kv4_mma0(c, qf[st][1].x, qf[st][1].y, qf[st][1].z, qf[st][1].w, e[2 * st], e[2 * st + 1]);
                            else kv4_mma(c, qf[st][1].x, qf[st][1].y, qf[st][1].z, qf[st][1].w, e[2 * st], e[2 * st + 1]);
                            kv4_mma(c, qf[st][0].x, qf[st][0].y, qf[st][0].z, qf[st][0].w, e[2 * st], e[2 * st + 1]);
                        }
                        const float d0 = kv4_half_of(ks[nt][g >> 1], g & 1), d1 = kv4_half_of(ks[nt][(NG + g) >> 1], (NG + g) & 1);
                        s[nt][0] = fmaf(d0, c[0], s[nt][0]); s[nt][1] = fmaf(d1, c[1], s[nt][1]);
                        s[nt][2] = fmaf(d0, c[2], s[nt][2]); s[nt][3] = fmaf(d1, c[3], s[nt][3]);
                    }
                }
            }
            const bool inside = tb >= wr.lo_all && tb + 8 * PT <= wr.hi_all;
            unsigned see = 0xffffffffu;                      // bit 4 nt + i: that score is seen
#pragma unroll
            for (int nt = 0; nt < PT; nt++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    s[nt][i] *= desc[i >> 1];
                    if (!inside) {
                        const int t = tb + nt * 8 + 2 * j + (i & 1);
                        if (t < clo[i >> 1] || t > chi[i >> 1]) { s[nt][i] = -INFINITY; see &= ~(1u << (4 * nt + i)); }
                    }
                }
            bool odd = false;                                // a cheap look first: each lane's largest weight within the range
            float top[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                top[h] = -INFINITY;
#pragma unroll
                for (int nt = 0; nt < PT; nt++) top[h] = fmaxf(top[h], fmaxf(s[nt][2 * h], s[nt][2 * h + 1]));
                top[h] -= m[h];
                odd |= !(top[h] > PR_LOW && top[h] <= PR_HI);
            }
            bool move = __any_sync(0xffffffffu, odd);
            if (move) {
                move = false;
#pragma unroll
                for (int h = 0; h < 2; h++) {                // (a line is a quad; its largest decides)
                    const unsigned large = __ballot_sync(0xffffffffu, top[h] > PR_LO) & 0xfu << 4 * r;
                    move |= top[h] > PR_HI;
                    move |= !large && m[h] > mh[h] - PR_DOWN;
                }
                move = __any_sync(0xffffffffu, move);
            }
            if (move) {
                float f[2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float mx = -INFINITY, mn = INFINITY;
#pragma unroll
                    for (int i = 0; i < 2 * PT; i++)
                        if (see >> (4 * (i >> 1) + 2 * h + (i & 1)) & 1) { mx = fmaxf(mx, s[i >> 1][2 * h + (i & 1)]); mn = fminf(mn, s[i >> 1][2 * h + (i & 1)]); }
#pragma unroll
                    for (int o = 1; o < 4; o <<= 1) {
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                        mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
                    }
                    // one far above the others of its own pass: no room above it, for their bits; within the range or nothing
                    // seen: the reference is left where it is
                    const float at = mx - mn > 10.f ? PR_HI : PR_AT;
                    float to = m[h] == -INFINITY ? mx - at : m[h] + ceilf(mx - m[h] - at);
                    if (mx == -INFINITY || (mx - m[h] > PR_LO && mx - m[h] <= PR_HI)) to = m[h];
                    to = fmaxf(to, mh[h] - PR_DOWN);
                    f[h] = to == m[h] ? 1.f : kv4_exp2(m[h] - to);
                    m[h] = to; mh[h] = fmaxf(mh[h], to); l[h] *= f[h];
                }
#pragma unroll
                for (int g = 0; g < NG; g++)
#pragma unroll
                    for (int i = 0; i < 16; i++) acc[g][i >> 2][i & 3] *= f[(i & 3) >> 1];
            }
            float lp[2] = {0.f, 0.f};
#pragma unroll
            for (int nt = 0; nt < PT; nt++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float p = kv4_exp2(s[nt][i] - m[i >> 1]);
                    if (!inside && !(see >> (4 * nt + i) & 1)) p = 0.f;
                    lp[i >> 1] += p;
                    s[nt][i] = p;
                }
            l[0] += lp[0]; l[1] += lp[1];
            // The pass's own sums start from zero and are added to acc by an ordinary f32 addition: the matrix unit cuts a
            // sum off instead of rounding it, and over a long prompt a sum kept in it drifts (4096 positions: 1.9e-6 off,
            // this way 6e-7, as the f32 torch form is).
            unsigned va[PT / 2][NG], vb[PT / 2][NG], wa[PT / 2][NG], wb[PT / 2][NG];
            __half2 mx = __halves2half2(__ushort_as_half(0), __ushort_as_half(0));
#pragma unroll
            for (int b = 0; b < PT / 2; b++) {               // 16 positions of one block at a time
                const int tq = tp + 16 * b;
                kv4_ldsw<NG>(va[b], unit + kv4_v_code_off(HD) + (tq >> 4) * (8 * HD) + lane * (4 * NG));
                kv4_ldsw<NG>(vb[b], unit + kv4_v_code_off(HD) + (tq >> 4) * (8 * HD) + 4 * HD + lane * (4 * NG));
                kv4_ldsw<NG>(wa[b], unit + kv4_v_step_off(HD) + (tq + 2 * j) * (2 * NG));
                kv4_ldsw<NG>(wb[b], unit + kv4_v_step_off(HD) + (tq + 8 + 2 * j) * (2 * NG));
                if (!inside) {
                    kv4_mask_steps<NG>(wa[b], tb + 16 * b + 2 * j, wr.lo_any, wr.hi_any);
                    kv4_mask_steps<NG>(wb[b], tb + 16 * b + 8 + 2 * j, wr.lo_any, wr.hi_any);
                }
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    mx = __hmax2(mx, __habs2(*reinterpret_cast<const __half2 *>(&wa[b][g])));
                    mx = __hmax2(mx, __habs2(*reinterpret_cast<const __half2 *>(&wb[b][g])));
                }
            }
            // the largest value step (NaN left aside) decides the power of two that weight * step is scaled by
            const float big = fmaxf(__low2float(mx), __high2float(mx));
            if (__any_sync(0xffffffffu, big >= vth)) {
                const unsigned bb = __reduce_max_sync(0xffffffffu, __float_as_uint(big)) & 0x7f800000u;   // 2^e
                if (bb) {
                    const float nn = 512.f / __uint_as_float(bb), f = vn == 0.f ? 1.f : nn / vn;
                    vth = 2.f * __uint_as_float(bb); vn = nn;
#pragma unroll
                    for (int g = 0; g < NG; g++)
#pragma unroll
                        for (int i = 0; i < 16; i++) acc[g][i >> 2][i & 3] *= f;
                }
            }
#pragma unroll
            for (int nt = 0; nt < PT; nt++)                  // block b: line r: positions 2j, 2j+1 | line r+8 | the same 8 positions on
#pragma unroll
                for (int i = 0; i < 4; i++) s[nt][i] *= vn;
#pragma unroll
            for (int g = 0; g < NG; g++) {
                float c[4][4];
#pragma unroll
                for (int b = 0; b < PT / 2; b++) {
                    const float d[4] = {kv4_half_of(wa[b][g >> 1], g & 1), kv4_half_of(wa[b][(NG + g) >> 1], (NG + g) & 1),
                                        kv4_half_of(wb[b][g >> 1], g & 1), kv4_half_of(wb[b][(NG + g) >> 1], (NG + g) & 1)};
                    float x[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) x[i] = s[2 * b + (i >> 2)][i & 3] * d[(i & 1) + 2 * (i >> 2)];
                    if (!inside) {                           // a position that is not seen adds nothing, whatever its step holds
#pragma unroll
                        for (int i = 0; i < 8; i++) if (!(see >> (8 * b + i) & 1)) x[i] = 0.f;
                    }
                    unsigned h[4], lo[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) kv4_pieces(x[2 * i], x[2 * i + 1], h[i], lo[i]);
                    unsigned ea[4], eb[4];
                    kv4_codes(va[b][g], ea);
                    kv4_codes(vb[b][g], eb);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        if (b == 0) kv4_mma0(c[i], lo[0], lo[1], lo[2], lo[3], ea[i], eb[i]);
                        else kv4_mma(c[i], lo[0], lo[1], lo[2], lo[3], ea[i], eb[i]);
                        kv4_mma(c[i], h[0], h[1], h[2], h[3], ea[i], eb[i]);
                    }
                }
#pragma unroll
                for (int i = 0; i < 16; i++) acc[g][i >> 2][i & 3] += c[i >> 2][i & 3];
            }
            if (++passes % (PR_F * KV4_PAGE / (8 * PT)) == 0) {
                float fl[2], fa[2];
                total_factors(fl, fa);
#pragma unroll
                for (int h = 0; h < 2; h++) { lt[h] = fmaf(lt[h], fl[h], l[h]); l[h] = 0.f; mt[h] = m[h]; }
                vnt = vn;
                const bool first = passes == PR_F * KV4_PAGE / (8 * PT);
#pragma unroll
                for (int g = 0; g < NG; g++) {               // (a group's loads together: one by one they were a fifth of the kernel's time)
                    float old[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) old[i] = first ? 0.f : tot[16 * g + i];
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        float &x = acc[g][i >> 2][i & 3];
                        tot[16 * g + i] = fmaf(old[i], fa[(i & 3) >> 1], x);
                        x = 0.f;
                    }
                }
            }
        }
    }
    // a thread holds, for lines r and r + 8, dims 32 g + 8 j + 0 .. 7: dim i + 4 k of them in acc[g][i][line half * 2 + k]
    if (passes >= PR_F * KV4_PAGE / (8 * PT)) {
        float fl[2], fa[2];
        total_factors(fl, fa);
        l[0] = fmaf(lt[0], fl[0], l[0]); l[1] = fmaf(lt[1], fl[1], l[1]);
#pragma unroll
        for (int i = 0; i < 16 * NG; i++) acc[i >> 4][i >> 2 & 3][i & 3] = fmaf(tot[i], fa[(i & 3) >> 1], acc[i >> 4][i >> 2 & 3][i & 3]);
    }
    const float vs = vn == 0.f ? 1.f : 1.f / vn;             // (a power of two)
#pragma unroll
    for (int hlf = 0; hlf < 2; hlf++) {
        l[hlf] += __shfl_xor_sync(0xffffffffu, l[hlf], 1);
        l[hlf] += __shfl_xor_sync(0xffffffffu, l[hlf], 2);
        const int line = r + 8 * hlf;
        if (line >= wn) continue;
        const int cc = c0 + w0 + line;
        const size_t rh = (size_t)(sq.r0 + cc / a.G) * a.H + head * a.G + cc % a.G;
        float *out;
        float f = vs;
        if (nsplit == 1) {
            out = a.ctx + rh * HD;
            f = vs * kv4_over(l[hlf]);
        } else {
            out = part + (rh * nsplit + split) * (HD + 4) + 4;
            if (j == 0) { out[-4] = m[hlf]; out[-3] = l[hlf]; }
        }
#pragma unroll
        for (int g = 0; g < NG; g++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
                float o[4];
#pragma unroll
                for (int i = 0; i < 4; i++) o[i] = acc[g][i][2 * hlf + k] * f;
                *reinterpret_cast<float4 *>(out + g * 32 + 8 * j + 4 * k) = make_float4(o[0], o[1], o[2], o[3]);
            }
    }
}

template <int NG>
int go(const Kv4Attend &a, const Kv4Plan &p, float *part, cudaStream_t st) {
    static bool attr[MOTY_MAX_DEV];
    int dev = 0;
    CK(cudaGetDevice(&dev));
    if (dev < 0 || dev >= MOTY_MAX_DEV) return moty_set_error(MOTY_CUDA_EARG, "kv4_attend: device %d", dev);
    if (!attr[dev]) {
        CK(cudaFuncSetAttribute(kv4_prompt_kernel<NG>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PrL<NG>::SMEM));
        attr[dev] = true;
    }
    const long long grid = (long long)a.b.nseq * a.geo.KV * p.ntile * p.nsplit;
    if (grid > 0x7fffffffLL) return moty_set_error(MOTY_CUDA_ELIMIT, "kv4_attend: %lld CTAs", grid);
    CK(moty_launch_pdl(kv4_prompt_kernel<NG>, dim3((unsigned)grid), dim3(PR_W * 32), PrL<NG>::SMEM, st, a, p.ntile, p.nsplit, p.span, part));
    return 0;
}

}  // namespace

int launch_kv4_prompt(const Kv4Attend &a, const Kv4Plan &p, float *part, cudaStream_t st) {
    switch (a.geo.hd / 32) {
        case 1: return go<1>(a, p, part, st);
        case 2: return go<2>(a, p, part, st);
        case 3: return go<3>(a, p, part, st);
        case 4: return go<4>(a, p, part, st);
        case 5: return go<5>(a, p, part, st);
        case 6: return go<6>(a, p, part, st);
        case 7: return go<7>(a, p, part, st);
        default: return go<8>(a, p, part, st);
    }
}
