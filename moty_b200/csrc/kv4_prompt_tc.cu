// kv4_prompt_tc.cu -- attention over the paged 4-bit KV cache for prompts, on the 5th-generation tensor cores.
//
// A CTA takes 256 lines ((row, query head) pairs of one KV head of one sequence) as two tiles of 128 that share a page's
// operand tiles, and walks the pages of its span, 64 positions a step:
//     S = Q K^T   [128 x 64]     three products: q lo * k hi, q hi * k lo, q hi * k hi
//     O = P V     [128 x hd]     three products: p lo * v hi, p hi * v lo, p hi * v hi
// f32 accuracy from f16 operands: an operand is hi + lo, f16 each.  A value held is code * step, 4 x 11 bits, so k and v are
// exact as hi + lo (the rest of an f16 product is a multiple of the smallest f16); q (scaled by a power of two a line) and
// the softmax weights (scaled by a power of two a line and page) carry 22 bits down to an end: 2^-38 of the line's largest
// query value, 2^-39 of its largest weight on the page; the dropped lo * lo term is 2^-22 of a product.  Steps of 4096 and more would overflow
// f16: a page that has one is brought down by 2^4.  O starts from zero at every page and is added to f32 registers, because
// the tensor core's own sum drifts over a long prompt.
//   warps 0-3, 4-7   softmax of a tile, a thread a line: S from TMEM, running maximum (moved when passed by 8 in base-2
//               units), weights back to TMEM over the scores as the A operand of the second product, then
//               the O of the page before added to the registers
//   warps 8-11, 12-14   keys and values of a page: bulk copies of codes and steps into shared memory (two pages deep), then k
//               and v^T operand tiles (K-major, 128-byte swizzle): eight key dims of a position, or eight positions of a
//               value dim, are one 16-byte piece
//   warp 15     issues the products: both S of page j + 1, then both O of page j, so that a tile's softmax of a page has the
//               time of three products, and each operand tile is rebuilt during the two products that do not read it
// TMEM (512 columns): scores / weights two buffers a tile, O one a tile.  What bounds it, at hd = 128: the products of a page
// and two tiles take 3900 cycles of tensor core (scores 48 K-steps of 49 cycles, which reading both operands from shared
// memory costs at N = 64, where the matrix unit alone would need 33; output 24 of 65), and a page takes 2.1 us where few SMs
// work, 2.6 us where all do and the power limit lowers the clock.  Beside that a CTA spends 13 us: 8 on its query rows (13 from
// memory), 2 on its first page, 3 on its results.  4096 rows at 4096 positions, 16 heads on 8: 175 us back to back, 195 us by
// itself (41 us at the tensor peak for one product each, 124 for three); one tile a CTA 416 us, when staging was longer than a tile's products; unrolled loops in the roles 227 us
// (their code outgrew the instruction cache); division instead of a reciprocal for the results 3 us a CTA.
// Every wait is bounded; on expiry all roles leave and the error word is set.
// An infinity or NaN of a key makes its scores NaN; a NaN step of a value is taken out of the product (a weight of 0 would
// spread it to lines that do not see it) and set in the result of the lines that do.
#include "kv4_frag.cuh"
#include "kv4_attend.cuh"
#include "tc_common.cuh"
#include <type_traits>

namespace {

constexpr int PT_M = 128, PT_NP = KV4_TC_PAGES, PT_T = 512, PT_KT = 128, PT_VT = 96;     // lines a tile, pages a span, threads: all, keys, values
constexpr int PT_REGS = 128, PT_REGS_SOFT = 184, PT_REGS_REST = 72;
static_assert(KV4_TC_LINES == 2 * PT_M && 256 * PT_REGS_SOFT + 256 * PT_REGS_REST <= PT_T * PT_REGS, "lines; register shares");
constexpr uint32_t TM_S = 0, TM_O = 256;                     // TMEM columns: scores / weights [tile][page & 1] x 64, O [tile] x 128

template <int NG> struct PtL {
    static constexpr int HD = NG * 32, NSUB = (NG + 1) / 2;
    static constexpr int VS = 4 * HD + 16;                   // bytes between staged value halves (eight positions)
    static constexpr int RK = 32 * HD, RV = 8 * VS, RST = 4 * HD, RAW = RK + RV + 2 * RST;       // staged: key codes, key steps, value halves, value steps
    static constexpr int Q = NSUB * PT_M * 128, K = NSUB * 64 * 128, V = HD * 128;      // one piece (hi or lo) of an operand
    static constexpr int OFF_K = 4 * Q, OFF_V = OFF_K + 2 * K, OFF_RAW = OFF_V + 2 * V, OFF_LIST = OFF_RAW + 2 * RAW;
    static constexpr int SMEM = OFF_LIST + PT_NP * 8 + 1024;
};

struct PtShared {
    uint64_t kfull, vfull, sfull[2][2], pfull[2][2], pvdone[2], oempty[2];   // [tile][page & 1]; the others one phase a page
    uint64_t rawk[2], rawv[2];                               // [page & 1]
    uint32_t tmem;
    int abort, n;
    float fk[8], fv[8];                                      // by page (the staging warps run ahead): what scores and outputs are to be multiplied by
    unsigned long long nan[8][4];                            // by page and group: positions whose value step is NaN
    int anynan[8];
    int big[2];                                              // a step of the staged keys / values that would overflow
};

__device__ __forceinline__ void mbar_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// D [tmem] (+)= A * B^T, f16 in, f32 sums; A from shared memory or from TMEM.  The whole warp runs the issuing code with
// uniform values and one lane issues (`lead`), so that addresses and descriptors stay in uniform registers: formed by a
// single lane they took 75 cycles a product.  A descriptor is its constant high word and an address word.
constexpr uint32_t DESC_HI = (uint32_t)(1024 >> 4) | 1u << 14 | 2u << 29;     // umma_desc's upper half: rows of 8 x 128 bytes, version 1, 128-byte swizzle
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr) { return (saddr >> 4 & 0x3fffu) | 1u << 16; }
__device__ __forceinline__ void umma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc, uint32_t lead) {
    asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "mov.b64 x, {%1, %6};\n\tmov.b64 y, {%2, %6};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(lead), "r"(DESC_HI) : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc, uint32_t lead) {
    asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "mov.b64 y, {%2, %6};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(lead), "r"(DESC_HI) : "memory");
}
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r;
}
// 32 columns of this warp's 32 lanes
__device__ __forceinline__ void tm_ld32(float (&v)[32], uint32_t addr) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,"
        "%26,%27,%28,%29,%30,%31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr) : "memory");
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tm_ld16(float (&v)[16], uint32_t addr) {
    uint32_t r[16];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(addr) : "memory");
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tm_st8(uint32_t addr, const unsigned (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// bounded (a page is about a microsecond; each poll may itself wait a while)
constexpr uint32_t PT_LIMIT = 1u << 22;
__device__ __forceinline__ bool pt_wait(uint64_t *bar, uint32_t parity, volatile int *abort_flag) {
    return moty_mbar_wait_abortable(smem_u32(bar), parity, abort_flag, PT_LIMIT);
}
// the whole warp waits, or leaves, together
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, volatile int *abort_flag) {
    const bool ok = pt_wait(bar, parity, abort_flag);
    return __all_sync(0xffffffffu, ok);
}
// a warpgroup's registers a thread (all four warps run it)
template <bool MORE, int N> __device__ __forceinline__ void role_registers() {
    if constexpr (MORE) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
// the warps of one role: a barrier of their own (1 keys, 2 values), and whether all of them say yes
template <int ID, int N> __device__ __forceinline__ void role_sync() { asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(N) : "memory"); }
template <int ID, int N> __device__ __forceinline__ bool role_and(bool ok) {
    int all;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.s32 q, %1, 0;\n\tbarrier.cta.red.and.pred p, %2, %3, q;\n\tselp.s32 %0, 1, 0, p;\n\t}"
                 : "=r"(all) : "r"((int)ok), "n"(ID), "n"(N) : "memory");
    return all != 0;
}
__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

// the word's values times the step pair d (one step twice for keys, two positions' steps for values): 4 pairs hi, 4 pairs lo
__device__ __forceinline__ void kv4_values_hl(unsigned w, __half2 d, unsigned (&hi)[4], unsigned (&lo)[4]) {
    unsigned e[4];
    kv4_codes(w, e);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const __half2 c = *reinterpret_cast<__half2 *>(&e[i]), h = __hmul2(c, d), l = __hfma2(c, d, __hneg2(h));
        hi[i] = *reinterpret_cast<const unsigned *>(&h);
        lo[i] = *reinterpret_cast<const unsigned *>(&l);
    }
}

template <int NG>
__global__ void __launch_bounds__(PT_T, 1) kv4_prompt_tc_kernel(Kv4Attend a, int ntile, int nsplit, int span, float *part, int *err_wait) {
    using L = PtL<NG>;
    constexpr int HD = L::HD, UNIT = 72 * HD;
    extern __shared__ uint8_t sm_raw_[];
    uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(sm_raw_) + 1023) & ~(uintptr_t)1023);
    __shared__ PtShared sh;
    int2 *list = reinterpret_cast<int2 *>(sm + L::OFF_LIST);                 // {page, first position} of the pages that are there
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int split = blockIdx.x % nsplit, u = blockIdx.x / nsplit;
    const int tile = ntile - 1 - u / (a.geo.KV * a.b.nseq), hs = u % (a.geo.KV * a.b.nseq), head = hs % a.geo.KV, seq = hs / a.geo.KV;
    pdl_trigger();
    pdl_wait();
    const Kv4Seq sq = kv4_load_seq(a, seq);
    if (!sq.ok) {
        if (nsplit == 1 && tile == 0) kv4_zero_rows(a, sq, head);
        return;
    }
    const int lines = sq.n * a.G, c0 = tile * KV4_TC_LINES;  // (rows * heads of a call stay below 2^31)
    if (c0 >= lines) return;
    const int ncol = lines - c0 < KV4_TC_LINES ? lines - c0 : KV4_TC_LINES, nx = ncol > PT_M ? 2 : 1;      // lines, tiles
    const int pos0 = sq.len - sq.n;
    const Kv4Range cr = kv4_range(a, pos0 + c0 / a.G, pos0 + (c0 + ncol - 1) / a.G);
    const int t_lo = (cr.lo_any & ~(KV4_PAGE - 1)) + split * span, t_hi = cr.hi_any - t_lo < span ? cr.hi_any : t_lo + span;
    if (t_lo >= cr.hi_any && nsplit > 1) return;

    if (tid == 0) {
        sh.abort = 0;
        mbar_init(&sh.kfull, PT_KT); mbar_init(&sh.vfull, PT_VT);
        for (int x = 0; x < 2; x++) {
            for (int i = 0; i < 2; i++) { mbar_init(&sh.sfull[x][i], 1); mbar_init(&sh.pfull[x][i], PT_M); }
            mbar_init(&sh.pvdone[x], 1); mbar_init(&sh.oempty[x], PT_M);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 15) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // pages as they lie in memory, two in flight
    const uint8_t *base = a.mem + (size_t)(a.layer * a.geo.KV + head) * UNIT;
    const size_t page_bytes = kv4_page_bytes(a.geo);
    auto load_k = [&](int j) {                               // key codes and steps are one run of bytes
        mbar_expect_tx(&sh.rawk[j & 1], 36 * HD);
        bulk_load(sm + L::OFF_RAW + (j & 1) * L::RAW, base + (size_t)list[j].x * page_bytes, 36 * HD, &sh.rawk[j & 1]);
    };
    auto load_v = [&](int j) {
        uint8_t *dst = sm + L::OFF_RAW + (j & 1) * L::RAW + L::RK + L::RST;
        const uint8_t *src = base + (size_t)list[j].x * page_bytes + kv4_v_code_off(HD);
        mbar_expect_tx(&sh.rawv[j & 1], 36 * HD);
        for (int o = 0; o < 8; o++) bulk_load(dst + o * L::VS, src + o * (4 * HD), 4 * HD, &sh.rawv[j & 1]);     // apart by 16 bytes: eight halves, eight bank groups
        bulk_load(dst + L::RV, src + 32 * HD, 4 * HD, &sh.rawv[j & 1]);
    };
    if (warp == 8) {                                         // the pages of the span that are there, in order
        const int np = t_hi > t_lo ? (t_hi - t_lo + KV4_PAGE - 1) / KV4_PAGE : 0;
        const int *tab = a.b.table + (size_t)seq * a.b.ld + t_lo / KV4_PAGE;
        int n = 0;
        for (int i0 = 0; i0 < np; i0 += 32) {
            const int i = i0 + lane, id = i < np ? tab[i] : -1;
            const bool ok = kv4_page_ok(a.geo, id);
            if (!ok && id != -1) atomicExch(a.err, 1);
            const unsigned m = __ballot_sync(0xffffffffu, ok);
            if (ok) list[n + __popc(m & ((1u << lane) - 1))] = make_int2(id, t_lo + i * KV4_PAGE);
            n += __popc(m);
        }
        __syncwarp();
        if (lane == 0) {
            sh.n = n;
            for (int i = 0; i < 2; i++) { mbar_init(&sh.rawk[i], 1); mbar_init(&sh.rawv[i], 1); }
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            for (int j = 0; j < 2 && j < n; j++) { load_k(j); load_v(j); }         // on their way while the queries are prepared
        }
    }
    // a softmax thread's line: its query row, limits, scale; the row goes to shared memory in two pieces
    float desc = 0.f;
    bool fin = true;                                         // a row that is not finite scores 0, and is NaN in the end where it saw anything
    int clo = 0, chi = 0x7fffffff;                           // (lines that are not there see everything, and are not written)
    size_t rh = 0;
    const int x = warp >> 2;                                 // the tile of a softmax warp
    if (x < nx) {
        const bool have = tid < ncol;
        const float *src = a.q;
        if (have) {
            const int cc = c0 + tid, row = cc / a.G, g0 = cc - row * a.G, p = pos0 + row;
            src = a.q + (size_t)(sq.r0 + row) * a.q_ld + (size_t)(head * a.G + g0) * HD;
            rh = (size_t)(sq.r0 + row) * a.H + head * a.G + g0;
#pragma unroll
            for (int i = 0; i < NG; i++) asm volatile("prefetch.global.L2 [%0];" ::"l"(src + 32 * i));       // all of the tile's rows at once
            chi = p;
            clo = a.window > 0 && p - a.window + 1 > 0 ? p - a.window + 1 : 0;
        }
        // LPR lanes bring a row (a lane the eight dims of a piece), so that a warp's loads touch few lines of memory
        constexpr int LPR = NG == 2 ? 8 : 16, RPI = 32 / LPR;
        const int c = lane % LPR, sub = lane / LPR;          // piece c = 4 g + j: dims 8 c + 0, 4, 1, 5, 2, 6, 3, 7 (the order of a code word's pairs)
        unsigned mb = 0;
#pragma unroll 4
        for (int i0 = 0; i0 < 32; i0 += RPI) {
            const int line = (warp & 3) * 32 + i0 + sub;     // of the tile
            const float *from = reinterpret_cast<const float *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src), i0 + sub));
            float4 v0 = make_float4(0.f, 0.f, 0.f, 0.f), v1 = v0;
            if (x * PT_M + line < ncol && c < 4 * NG) {
                v0 = reinterpret_cast<const float4 *>(from)[2 * c];
                v1 = reinterpret_cast<const float4 *>(from)[2 * c + 1];
            }
            const float y[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
            unsigned m = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) m = max(m, __float_as_uint(y[i]) & 0x7fffffffu);
#pragma unroll
            for (int o = 1; o < LPR; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            const unsigned own = __shfl_sync(0xffffffffu, m, lane % RPI * LPR);
            if (lane / RPI * RPI == i0) mb = own;
            const bool fin = m < 0x7f800000u;
            const int k = fin ? kv4_q_shift(m) : 0;
            unsigned h[4], l[4];
#pragma unroll
            for (int i = 0; i < 4; i++) kv4_pieces(fin ? kv4_scale2(y[i], k) : 0.f, fin ? kv4_scale2(y[i + 4], k) : 0.f, h[i], l[i]);
            if (c < 4 * NG) {
                uint8_t *dst = sm + 2 * x * L::Q + (c >> 3) * (PT_M * 128) + line * 128 + (((c & 7) ^ (line & 7)) << 4);
                *reinterpret_cast<uint4 *>(dst) = make_uint4(h[0], h[1], h[2], h[3]);
                *reinterpret_cast<uint4 *>(dst + L::Q) = make_uint4(l[0], l[1], l[2], l[3]);
            }
        }
        fin = mb < 0x7f800000u;
        // (not below the smallest normal number: -infinity times it has to stay -infinity)
        desc = fin ? fmaxf(kv4_scale2(a.scale * 1.44269504f, -kv4_q_shift(mb)), 1.17549435e-38f) : 1.f;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = sh.tmem;
    const int n = sh.n;
    volatile int *abort_flag = &sh.abort;

    // ---- pages into shared memory, then as operand tiles ----
    const __half2 down = __half2half2(__ushort_as_half(0x2c00));         // 1 / 16
    // Steps of a staged part: positions that no line sees become 0 (their memory may hold anything), steps that would
    // overflow and NaN steps of values are noted; all of it rare, and looked for two steps at a time.  Returns what
    // the part's values have been divided by.  (The barrier in it also says that all have left the page before.)
    auto look = [&](auto keys_, int w, int j, uint32_t *st) {
        constexpr bool keys = decltype(keys_)::value;
        constexpr int ID = keys ? 1 : 2, N = keys ? PT_KT : PT_VT;
        const int t0 = list[j].y;
        bool odd = t0 < cr.lo_any || t0 + KV4_PAGE > cr.hi_any;
        for (int i = w; i < 32 * NG; i += N) odd |= (((st[i] & 0x7fff7fffu) + 0x14001400u) & 0x80008000u) != 0;      // |step| >= 4096, infinity, NaN
        if (role_and<ID, N>(!odd)) return 1.f;
        if (w == 0) sh.big[keys] = 0;
        role_sync<ID, N>();
        uint16_t *h = reinterpret_cast<uint16_t *>(st);
        for (int i = w; i < 64 * NG; i += N) {
            const int t = i / NG, g = i - t * NG;
            uint16_t v = h[i];
            if (t0 + t < cr.lo_any || t0 + t >= cr.hi_any) v = 0;
            if ((v & 0x7fff) >= 0x7c00) {
                if (!keys) { atomicOr(&sh.nan[j & 7][g], 1ull << t); sh.anynan[j & 7] = 1; v = 0; }
            } else if ((v & 0x7fff) >= 0x6c00) sh.big[keys] = 1;
            h[i] = v;
        }
        role_sync<ID, N>();
        const float f = sh.big[keys] ? 16.f : 1.f;
        role_sync<ID, N>();
        return f;
    };
    // The roles by warpgroup; each takes its registers first thing in its own branch, so that what the compiler gives a role's
    // code is bounded by the number the role holds (512 x 128 at launch).
    if (warp >= 12) {
        role_registers<false, PT_REGS_REST>();
        if (warp == 15) {
            // ---- the products ----
            const uint32_t id_s = (1u << 4) | (64u >> 3) << 17 | (uint32_t)(PT_M >> 4) << 24;
            const uint32_t id_o = (1u << 4) | ((uint32_t)HD >> 3) << 17 | (uint32_t)(PT_M >> 4) << 24;
            const uint32_t q0 = __shfl_sync(0xffffffffu, smem_u32(sm), 0), tm = __shfl_sync(0xffffffffu, tmem, 0);
            const uint32_t dq = desc_lo(q0), dk = desc_lo(q0 + L::OFF_K), dv = desc_lo(q0 + L::OFF_V);     // (offsets below do not leave 14 bits)
            const uint32_t lead = elect_one();
            bool ok = true;
            for (int j = 0; j <= n && ok; j++) {
                if (j < n) {                                     // S of page j (its buffer: the O of page j - 2 was issued before)
                    ok = warp_wait(&sh.kfull, j & 1, abort_flag);
                    if (!ok) break;
                    tc_after();
#pragma unroll 1
                    for (int y = 0; y < nx; y++) {
                        const uint32_t d = tm + TM_S + (y * 2 + (j & 1)) * 64, q = dq + y * (2 * L::Q >> 4);
#pragma unroll
                        for (int term = 0; term < 3; term++)     // q lo * k hi, q hi * k lo, q hi * k hi
#pragma unroll
                            for (int s = 0; s < 2 * NG; s++)
                                umma_ss(d, q + (((term == 0 ? L::Q : 0) + (s >> 2) * (PT_M * 128) + (s & 3) * 32) >> 4),
                                        dk + (((term == 1 ? L::K : 0) + (s >> 2) * (64 * 128) + (s & 3) * 32) >> 4), id_s, (term | s) != 0, lead);
                        if (lead) umma_commit(&sh.sfull[y][j & 1]);
                        __syncwarp();
                    }
                }
                if (j > 0) {                                     // O of page j - 1
                    const int i = j - 1;
                    ok = warp_wait(&sh.vfull, i & 1, abort_flag);
#pragma unroll 1
                    for (int y = 0; y < nx && ok; y++) {
                        ok = warp_wait(&sh.pfull[y][i & 1], i >> 1 & 1, abort_flag) && warp_wait(&sh.oempty[y], (i & 1) ^ 1, abort_flag);
                        if (!ok) break;
                        tc_after();
                        const uint32_t d = tm + TM_O + y * 128, p = tm + TM_S + (y * 2 + (i & 1)) * 64;
#pragma unroll
                        for (int term = 0; term < 3; term++)     // p lo * v hi, p hi * v lo, p hi * v hi
#pragma unroll
                            for (int s = 0; s < 4; s++)
                                umma_ts(d, p + s * 16 + (term == 0 ? 8 : 0), dv + (((term == 1 ? L::V : 0) + s * 32) >> 4), id_o,
                                        (term | s) != 0, lead);
                        if (lead) umma_commit(&sh.pvdone[y]);
                        __syncwarp();
                    }
                }
            }
        } else {
            // ---- values of a page ----
            bool ok = true;
            const int w = tid - 384;
            for (int j = 0; j < n; j++) {
                uint8_t *raw = sm + L::OFF_RAW + (j & 1) * L::RAW + L::RK + L::RST;
                ok = warp_wait(&sh.rawv[j & 1], j >> 1 & 1, abort_flag);
                if (!role_and<2, PT_VT>(ok)) break;
                if (w == 0 && j > 0 && j + 1 < n) load_v(j + 1);
                if (w < NG) sh.nan[j & 7][w] = 0ull;
                if (w == 4) sh.anynan[j & 7] = 0;
                const float f = look(std::false_type{}, w, j, reinterpret_cast<uint32_t *>(raw + L::RV));
                if (w == 0) sh.fv[j & 7] = f;
                if (j > 0 && !warp_wait(&sh.pvdone[nx - 1], (j - 1) & 1, abort_flag)) continue;  // the values of page j - 1 are done with
                const uint16_t *vst = reinterpret_cast<const uint16_t *>(raw + L::RV);
#pragma unroll 1
                for (int it = w; it < 64 * NG; it += PT_VT) {        // eight positions 8 o .., dims 32 g + 4 r + 0 .. 3
                    const int o = it & 7, r = it >> 3 & 7, g = it >> 6;
                    unsigned h[4][4], l[4][4];
#pragma unroll
                    for (int q = 0; q < 4; q++) {            // positions 8 o + 2 q, + 1
                        const unsigned vw = *reinterpret_cast<const unsigned *>(raw + o * L::VS + (r * 4 + q) * (4 * NG) + 4 * g);
                        const int t = 8 * o + 2 * q;
                        __half2 d = __halves2half2(__ushort_as_half(vst[t * NG + g]), __ushort_as_half(vst[(t + 1) * NG + g]));
                        if (f != 1.f) d = __hmul2(d, down);
                        unsigned hh[4], ll[4];
                        kv4_values_hl(vw, d, hh, ll);
#pragma unroll
                        for (int i = 0; i < 4; i++) { h[i][q] = hh[i]; l[i][q] = ll[i]; }
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int dim = 32 * g + 4 * r + i;
                        uint8_t *dst = sm + L::OFF_V + dim * 128 + ((o ^ (dim & 7)) << 4);
                        *reinterpret_cast<uint4 *>(dst) = make_uint4(h[i][0], h[i][1], h[i][2], h[i][3]);
                        *reinterpret_cast<uint4 *>(dst + L::V) = make_uint4(l[i][0], l[i][1], l[i][2], l[i][3]);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(&sh.vfull);
            }
        }
    } else if (warp >= 8) {
        role_registers<false, PT_REGS_REST>();
        // ---- keys of a page ----
        bool ok = true;
        const int w = tid - 256;
        for (int j = 0; j < n; j++) {
            uint8_t *raw = sm + L::OFF_RAW + (j & 1) * L::RAW;
            ok = warp_wait(&sh.rawk[j & 1], j >> 1 & 1, abort_flag);
            if (!role_and<1, PT_KT>(ok)) break;
            if (w == 0 && j > 0 && j + 1 < n) load_k(j + 1);
            const float f = look(std::true_type{}, w, j, reinterpret_cast<uint32_t *>(raw + L::RK));
            if (w == 0) sh.fk[j & 7] = f;
            // the keys of page j - 1 are done with (a warp that gives up goes on to the next barrier, where all leave)
            if (j > 0 && !warp_wait(&sh.sfull[nx - 1][(j - 1) & 1], (j - 1) >> 1 & 1, abort_flag)) continue;
#pragma unroll 1
            for (int it = w; it < 256; it += PT_KT) {    // position t, piece jj of a group's four
                const int t = (it >> 5) * 8 + (it & 7), jj = it >> 3 & 3;
                unsigned kw[NG], st[(NG + 1) / 2];
                kv4_ldsw<NG>(kw, raw + t * (HD / 2) + jj * (4 * NG));
                kv4_ldsteps<NG>(st, raw + L::RK + t * (2 * NG));
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    __half2 d = __half2half2(__ushort_as_half((unsigned short)(g & 1 ? st[g >> 1] >> 16 : st[g >> 1])));
                    if (f != 1.f) d = __hmul2(d, down);
                    unsigned h[4], l[4];
                    kv4_values_hl(kw[g], d, h, l);
                    const int c = 4 * g + jj;
                    uint8_t *dst = sm + L::OFF_K + (c >> 3) * (64 * 128) + t * 128 + (((c & 7) ^ (t & 7)) << 4);
                    *reinterpret_cast<uint4 *>(dst) = make_uint4(h[0], h[1], h[2], h[3]);
                    *reinterpret_cast<uint4 *>(dst + L::K) = make_uint4(l[0], l[1], l[2], l[3]);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_arrive(&sh.kfull);
        }
    } else {
        role_registers<true, PT_REGS_SOFT>();
        if (x < nx) {
            // ---- softmax: a thread a line ----
            const uint32_t mine = tmem + ((uint32_t)((warp & 3) * 32) << 16);
            float m = -INFINITY, l = 0.f, lt = 0.f, o[HD];       // lt: the weights' total of whole 16 pages, l: of those after them
            unsigned nanbits = 0;
#pragma unroll
            for (int i = 0; i < HD; i++) o[i] = 0.f;
            float f = 1.f, b = 0.f;                              // what the O of the page before is still to be multiplied by: m's move, its weights' scale
            bool ok = true;
            for (int j = 0; j <= n; j++) {
                const int t0 = j < n ? list[j].y : 0;
                const float before = b;
                if (j < n) {
                    ok = warp_wait(&sh.sfull[x][j & 1], j >> 1 & 1, abort_flag);
                    if (!ok) break;
                    tc_after();
                    const float ds = desc * sh.fk[j & 7];
                    const bool inside = t0 >= cr.lo_all && t0 + KV4_PAGE <= cr.hi_all;
                    const uint32_t at = mine + TM_S + (x * 2 + (j & 1)) * 64;
                    float mx = -INFINITY;
                    // (loops kept rolled: unrolled, the roles' code together outgrew the instruction cache)
#pragma unroll 1
                    for (int q = 0; q < 2; q++) {
                        float v[32];
                        tm_ld32(v, at + q * 32);
                        if (!inside) {
#pragma unroll
                            for (int i = 0; i < 32; i++) { const int t = t0 + q * 32 + i; if (t < clo || t > chi) v[i] = -INFINITY; }
                        }
#pragma unroll
                        for (int i = 0; i < 32; i += 2) mx = fmaxf(mx, fmaxf(v[i], v[i + 1]));
                    }
                    mx *= ds;                                    // (the scale is positive)
                    const bool up = mx > m + 8.f;
                    f = 1.f;
                    if (__any_sync(0xffffffffu, up)) {
                        if (up) { f = kv4_exp2(m - mx); m = mx; }
                        __syncwarp();
                        l *= f; lt *= f;
#pragma unroll
                        for (int i = 0; i < HD; i++) o[i] *= f;
                    }
                    // weights as hi and lo pairs of consecutive positions, over the scores: 16 columns become 8 of hi and 8 of
                    // lo.  They are brought up to 2^15 by the largest of the line on THIS page (lo ends at 2^-24, which
                    // then is 2^-39 of it), not by the largest so far, which one position may hold; bn takes it back.  Both are
                    // a whole number of base-2 units apart: a line that sees one position is that position's values,
                    // unless its score's own rounding shows.
                    const float mm = mx == -INFINITY ? 0.f : m + ceilf(mx - m) - 15.f, bn = mx == -INFINITY ? 0.f : kv4_exp2(mm - m);
                    float s0 = 0.f, s1 = 0.f;
#pragma unroll 1
                    for (int q = 0; q < 4; q++) {
                        float v[16];
                        tm_ld16(v, at + q * 16);
                        if (!inside) {
#pragma unroll
                            for (int i = 0; i < 16; i++) { const int t = t0 + q * 16 + i; if (t < clo || t > chi) v[i] = -INFINITY; }
                        }
                        unsigned ph[8], pl[8];
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const float p0 = kv4_exp2(fmaf(v[2 * i], ds, -mm)), p1 = kv4_exp2(fmaf(v[2 * i + 1], ds, -mm));
                            s0 += p0; s1 += p1;
                            kv4_pieces(p0, p1, ph[i], pl[i]);
                        }
                        tm_st8(at + q * 16, ph);
                        tm_st8(at + q * 16 + 8, pl);
                    }
                    l = fmaf(s0 + s1, bn, l);
                    if ((j & 15) == 15) { lt += l; l = 0.f; }    // (one sum of 512 even pages: 3e-6 off)
                    b = bn;
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    tc_before();
                    mbar_arrive(&sh.pfull[x][j & 1]);
                } else f = 1.f;
                if (j > 0) {                                     // O of page j - 1 to the registers
                    const int i0 = j - 1;
                    ok = warp_wait(&sh.pvdone[x], i0 & 1, abort_flag);
                    if (!ok) break;
                    tc_after();
                    const float g = f * before * sh.fv[i0 & 7];
#pragma unroll
                    for (int c = 0; c < HD; c += 32) {
                        float v[32];
                        tm_ld32(v, mine + TM_O + x * 128 + c);
#pragma unroll
                        for (int i = 0; i < 32; i++) o[c + i] = fmaf(v[i], g, o[c + i]);
                    }
                    tc_before();
                    mbar_arrive(&sh.oempty[x]);
                    if (sh.anynan[i0 & 7]) {
                        const int tn = list[i0].y;
                        for (int gg = 0; gg < NG; gg++)
                            for (unsigned long long mk = sh.nan[i0 & 7][gg]; mk; mk &= mk - 1) {
                                const int t = tn + __ffsll((long long)mk) - 1;
                                if (t >= clo && t <= chi) nanbits |= 1u << gg;
                            }
                        __syncwarp();
                    }
                }
            }
            // out through the tile's query rows (their products are done), so that a warp writes whole lines: a thread puts its
            // line there in pieces of four dims, turned by the line so that eight lanes meet eight bank groups
            if (__all_sync(0xffffffffu, ok)) {
                l += lt;
                if (!fin && l != 0.f) l = __int_as_float(0x7fffffff);
                float4 *box = reinterpret_cast<float4 *>(sm + 2 * x * L::Q) + (warp & 3) * (32 * HD / 4);
                if (tid < ncol && nsplit > 1) *reinterpret_cast<float2 *>(part + (rh * nsplit + split) * (HD + 4)) = make_float2(m, l);
                const float over = nsplit > 1 ? 1.f : kv4_over(l);
#pragma unroll
                for (int c = 0; c < HD / 4; c++) {
                    const float no = nanbits >> (c >> 3) & 1 ? __int_as_float(0x7fffffff) : 0.f;
                    box[lane * (HD / 4) + (c ^ (lane & 7))] = make_float4(fmaf(o[4 * c], over, no), fmaf(o[4 * c + 1], over, no), fmaf(o[4 * c + 2], over, no), fmaf(o[4 * c + 3], over, no));
                }
                __syncwarp();
                float *const to = nsplit == 1 ? a.ctx + rh * HD : part + (rh * nsplit + split) * (HD + 4) + 4;
#pragma unroll 8
                for (int i = 0; i < HD / 4; i++) {
                    const int at = i * 32 + lane, line = at / (HD / 4), c = at - line * (HD / 4);
                    float4 *dst = reinterpret_cast<float4 *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(to), line));
                    if ((warp & 3) * 32 + line + x * PT_M < ncol) dst[c] = box[line * (HD / 4) + (c ^ (line & 7))];
                }
            }
        }
    }
    // (behind the roles nothing is kept in registers from before them: what is needed is read anew)
    tc_before();
    __syncthreads();
    tc_after();
    if (sh.abort) {                                          // products still on their way are given time before their memory goes
        if (threadIdx.x == 0) atomicExch(err_wait, 1);
        for (int i = 0; i < 1000; i++) __nanosleep(1000);
        __syncthreads();
    }
    if (threadIdx.x >> 5 == 15) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(sh.tmem), "r"(512));
    }
}

// The roles' register shares (setmaxnreg) must add up to what the threads are launched with, which the compiler decides: where
// it gave another number the other prompt kernel serves the call.  Looked at once a device.
template <int NG> bool ready(int dev) {
    static signed char state[MOTY_MAX_DEV];                  // 0: not looked at yet, 1: yes, -1: no
    if (dev < 0 || dev >= MOTY_MAX_DEV) return false;
    if (!state[dev]) {
        cudaFuncAttributes fa;
        const bool ok = cudaFuncGetAttributes(&fa, kv4_prompt_tc_kernel<NG>) == cudaSuccess && fa.numRegs == PT_REGS &&
                        cudaFuncSetAttribute(kv4_prompt_tc_kernel<NG>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PtL<NG>::SMEM) == cudaSuccess;
        if (!ok) cudaGetLastError();
        state[dev] = ok ? 1 : -1;
    }
    return state[dev] > 0;
}

template <int NG>
int go(const Kv4Attend &a, const Kv4Plan &p, float *part, int *err_wait, cudaStream_t st) {
    const long long grid = (long long)a.b.nseq * a.geo.KV * p.ntile * p.nsplit;
    if (grid > 0x7fffffffLL) return moty_set_error(MOTY_CUDA_ELIMIT, "kv4_attend: %lld CTAs", grid);
    CK(moty_launch_pdl(kv4_prompt_tc_kernel<NG>, dim3((unsigned)grid), dim3(PT_T), (size_t)PtL<NG>::SMEM, st, a, p.ntile, p.nsplit, p.span, part, err_wait));
    return 0;
}

}  // namespace

bool kv4_prompt_tc_ready(int hd, int device) { return hd == 64 ? ready<2>(device) : hd == 96 ? ready<3>(device) : hd == 128 ? ready<4>(device) : false; }

int launch_kv4_prompt_tc(const Kv4Attend &a, const Kv4Plan &p, float *part, cudaStream_t st) {
    int *err_wait = a.err - 4;                               // the library's error words: [0] tensor-core pipeline waits, [4] this cache's batches
    switch (a.geo.hd / 32) {
        case 2: return go<2>(a, p, part, err_wait, st);
        case 3: return go<3>(a, p, part, err_wait, st);
        default: return go<4>(a, p, part, err_wait, st);
    }
}
