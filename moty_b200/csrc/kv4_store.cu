// kv4_store.cu -- rows into and out of the paged 4-bit KV cache.
//
// A group of 32 dims of a row shares one signed f16 step, chosen as the Q4R4 weight packer chooses it
// (nn/quant.c:157-179): big = the first value of largest magnitude, other = the largest magnitude of the opposite sign,
//     step = max(|big| / 8, other / 7),  d = f16(big > 0 ? -step : step),  code = clamp(rint(x / d), -8, 7).
// Two differences from the weights: the code comes from the correctly rounded quotient x / d, not from x * (1 / d) -- x is
// f32 and d has 11 bits, and then rint of the f32 quotient IS rint of the exact one (d (k + 1/2) is representable, so x
// differs from it by an ulp of x at least, which is more than half an ulp of the quotient): the codes follow from the
// formula alone.  And activations, unlike weights, may be anything: d saturates at 65504, and a group that holds an
// infinity or a NaN gets the step NaN, so that it reads as NaN instead of as some finite row.
#include "kv4.cuh"

namespace {

// a warp holds one group, a value a lane: returns the lane's nibble (code + 8), *d = the step's bits
__device__ __forceinline__ unsigned kv4_quant_lane(float x, int lane, unsigned short *d) {
    const float a = fabsf(x);
    const unsigned ab = __float_as_uint(a);                    // non-negative floats order like their bits, NaN above all
    unsigned m = ab;
    for (int off = 16; off > 0; off >>= 1) { const unsigned o = __shfl_xor_sync(0xffffffffu, m, off); m = o > m ? o : m; }
    if (m >= 0x7f800000u) { *d = 0x7fff; return 8; }
    const int src = __ffs(__ballot_sync(0xffffffffu, ab == m)) - 1;
    const float big = __shfl_sync(0xffffffffu, x, src);
    const float other = warp_max_f32(((x > 0.f) != (big > 0.f)) ? a : 0.f);
    const float step = fminf(fmaxf(__fmul_rn(fabsf(big), 0.125f), __fdiv_rn(other, 7.f)), 65504.f);
    const __half h = __float2half_rn(big > 0.f ? -step : step);
    const float df = __half2float(h);
    *d = __half_as_ushort(h);
    if (df == 0.f) return 8;
    int c = __float2int_rn(__fdiv_rn(x, df));
    c = c < -8 ? -8 : c > 7 ? 7 : c;
    return (unsigned)(c + 8);
}
// store group g of key / value row t of a unit from the lanes' nibbles
__device__ __forceinline__ void kv4_put_k(uint8_t *unit, int hd, int t, int g, int lane, unsigned nib, unsigned short d) {
    unsigned w = nib << (4 * (lane & 7));
    for (int off = 1; off < 8; off <<= 1) w |= __shfl_xor_sync(0xffffffffu, w, off);
    if ((lane & 7) == 0) *reinterpret_cast<unsigned *>(unit + kv4_k_word(hd, t, g, lane >> 3)) = w;
    if (lane == 0) reinterpret_cast<unsigned short *>(unit + kv4_k_step_off(hd))[t * (hd >> 5) + g] = d;
}
__device__ __forceinline__ void kv4_put_v(uint8_t *unit, int hd, int t, int g, int lane, unsigned nib, unsigned short d) {
    unsigned w = nib << (4 * (lane & 3));
    for (int off = 1; off < 4; off <<= 1) w |= __shfl_xor_sync(0xffffffffu, w, off);
    if ((lane & 3) == 0) *reinterpret_cast<unsigned short *>(unit + kv4_v_piece(hd, t, g, lane >> 2)) = (unsigned short)w;
    if (lane == 0) reinterpret_cast<unsigned short *>(unit + kv4_v_step_off(hd))[t * (hd >> 5) + g] = d;
}

// ---- many rows at once -----------------------------------------------------------------------------------------------
// A CTA takes ST_ROWS rows of one KV head, a thread eight dims of a row at a time: a group is the four threads of a quad
// (two shuffles a reduction), eight key codes are one word of the page, the value codes go through shared memory so that
// two positions of a pair leave as one word and neighbouring threads write neighbouring bytes.  A warp a group, a value a
// lane (as the single-row kernel below has it) spent 188 us on 3 sequences' 4096-row prompts of 16 heads, hd 128 (append and
// fetch: 248 MB, 38 us at the copy rate); this 75 us, 47 of them the append, which issues instructions four cycles of five:
// two exact maxima, a correctly rounded step and eight codes a thread.  64 single rows: 6.6 us both, launch and look-up latency.
constexpr int ST_ROWS = 16, ST_T = 256;

// The quad's step for x[8] a thread: *d = its bits, returns it (0 for a group of zeros, NaN for one that is not finite).
__device__ __forceinline__ float kv4_quad_step(const float (&x)[8], unsigned short *d) {
    int pb = 0, nb = 0;                                        // largest positive value and largest magnitude of a negative one, as bits
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int b = __float_as_int(x[i]);
        pb = max(pb, b);
        nb = max(nb, b ^ (int)0x80000000);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        pb = max(pb, __shfl_xor_sync(0xffffffffu, pb, o));
        nb = max(nb, __shfl_xor_sync(0xffffffffu, nb, o));
    }
    const bool bad = pb >= 0x7f800000 || nb >= 0x7f800000;
    bool neg = nb > pb;                                        // the sign of the first value of largest magnitude
    if (__any_sync(0xffffffffu, pb == nb && pb > 0)) {         // both signs reach it: look which comes first
        int first = 64;                                        // 2 * dim + (negative)
#pragma unroll
        for (int i = 7; i >= 0; i--) {
            const int b = __float_as_int(x[i]);
            if (b == pb) first = 2 * i;
            if ((b ^ (int)0x80000000) == nb) first = 2 * i + 1;
        }
        first += first < 64 ? 16 * (threadIdx.x & 3) : 0;
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
        if (pb == nb) neg = first & 1;
    }
    const float big = __int_as_float(neg ? nb : pb), other = __int_as_float(neg ? pb : nb);
    const float step = fminf(fmaxf(__fmul_rn(big, 0.125f), __fdiv_rn(other, 7.f)), 65504.f);
    const __half h = __float2half_rn(neg || big == 0.f ? step : -step);
    *d = bad ? (unsigned short)0x7fff : __half_as_ushort(h);
    return bad ? 0.f : __half2float(h);                        // codes of a bad group are 0, as with a step of 0
}
// The eight nibbles (code + 8) of x for step d.  y = 1.5 * 2^23 + x / d approximately, which rounds to an integer t in the low
// bits; the remainder x - t d is exact, and where one is half a step or more (a tie, or the approximation on the wrong side of
// one) the eight quotients are divided out.  (One look for all eight: one each cost 5 us of a prompt's 47.)
__device__ __forceinline__ unsigned kv4_quant8(const float (&x)[8], float d) {
    constexpr float MAGIC = 12582912.f;                        // 1.5 * 2^23
    const float inv = d == 0.f ? 0.f : __frcp_rn(d), half = d == 0.f ? INFINITY : 0.5f * fabsf(d);
    float y[8];
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        y[i] = __fmaf_rn(x[i], inv, MAGIC);
        odd |= !(fabsf(__fmaf_rn(-__fsub_rn(y[i], MAGIC), d, x[i])) < half);
    }
    if (odd) {
#pragma unroll
        for (int i = 0; i < 8; i++) y[i] = d == 0.f ? MAGIC : __fadd_rn(MAGIC, fminf(fmaxf(rintf(__fdiv_rn(x[i], d)), -8.f), 7.f));
    }
    unsigned w = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) w |= (__float_as_uint(fminf(fmaxf(y[i], MAGIC - 8.f), MAGIC + 7.f)) & 15u) << (4 * i);
    return w ^ 0x88888888u;
}
// what the rows of a CTA are: unit (null: skip) and position in the page
struct Kv4Rows { uint8_t *unit[ST_ROWS]; int t[ST_ROWS], seq[ST_ROWS]; };
__device__ __forceinline__ void kv4_rows(Kv4Rows &s, const Kv4Geom &geo, uint8_t *mem, const Kv4Batch &b, int row0, int layer, int head, int *err,
                                         bool absent_ok) {
    // 16 lanes look for a row where there are many sequences (64: 6.7 us for their rows stored and fetched, 7.5 us with four
    // lanes), else four, which is two warps instead of all (3 prompts of up to 4096 rows: 75.0 us, 76.6 us with 16)
    const int w = b.nseq > 16 ? 4 : 2, i = threadIdx.x >> w, r = row0 + i;
    int seq, pos, st = KV4_ROW_NONE;
    if (w == 4) st = kv4_row<16>(b, r, &seq, &pos);
    else if (i < ST_ROWS) st = kv4_row<4>(b, r, &seq, &pos);   // (whole warps)
    if (i < ST_ROWS && (threadIdx.x & ((1 << w) - 1)) == 0) {
        uint8_t *unit = nullptr;
        if (r >= b.rows) { seq = -1; pos = 0; }
        else {
            if (st == KV4_ROW_BAD || st == KV4_ROW_STRAY) atomicExch(err, 1);
            if (st == KV4_ROW_OK) {
                const int page = b.table[(size_t)seq * b.ld + pos / KV4_PAGE];
                if (kv4_page_ok(geo, page)) unit = mem + kv4_unit_off(geo, page, layer, head);
                else if (!(absent_ok && page == -1)) atomicExch(err, 1);
            }
            else seq = -1;                                     // (nothing is stored or fetched for it)
        }
        s.unit[i] = unit; s.t[i] = pos % KV4_PAGE; s.seq[i] = seq;
    }
    __syncthreads();
}

__global__ void __launch_bounds__(ST_T) kv4_append_kernel(Kv4Geom geo, uint8_t *mem, int layer, const float *k, const float *v, long long ld,
                                                          Kv4Batch b, int *err) {
    __shared__ Kv4Rows rs;
    __shared__ unsigned short vp[ST_ROWS][64 + 2];             // value pieces of four dims: [row][g * 8 + r]
    const int tid = threadIdx.x, hd = geo.hd, NG = hd >> 5, row0 = blockIdx.x * ST_ROWS, head = blockIdx.y;
    pdl_trigger();
    pdl_wait();
    const int per = hd >> 3, items = ST_ROWS * per;            // eight dims an item; a quad never leaves its group
    const unsigned nth = 65535u / (unsigned)NG + 1;            // n / NG = n nth >> 16 for n < 65536 / NG: here n <= 1024
    float kx[8], vx[8];
    auto load = [&](int it) {
        const int i = (int)((unsigned)(it >> 2) * nth >> 16), d8 = it - i * per;
#pragma unroll
        for (int e = 0; e < 8; e++) kx[e] = vx[e] = 0.f;
        if (it < items && row0 + i < b.rows) {
            const size_t at = (size_t)(row0 + i) * ld + (size_t)head * hd + d8 * 8;
            *reinterpret_cast<float4 *>(kx) = *reinterpret_cast<const float4 *>(k + at);
            *reinterpret_cast<float4 *>(kx + 4) = *reinterpret_cast<const float4 *>(k + at + 4);
            *reinterpret_cast<float4 *>(vx) = *reinterpret_cast<const float4 *>(v + at);
            *reinterpret_cast<float4 *>(vx + 4) = *reinterpret_cast<const float4 *>(v + at + 4);
        }
    };
    load(tid);                                                 // on its way while the rows are looked up
    kv4_rows(rs, geo, mem, b, row0, layer, head, err, false);
    for (int it = tid; it < (items + ST_T - 1) / ST_T * ST_T; it += ST_T) {
        const int i = (int)((unsigned)(it >> 2) * nth >> 16), d8 = it - i * per, g = d8 >> 2, j = d8 & 3;
        uint8_t *unit = it < items ? rs.unit[i] : nullptr;
        if (it != tid) load(it);
        unsigned short kd, vd;
        const float ks = kv4_quad_step(kx, &kd), vs = kv4_quad_step(vx, &vd);
        if (unit) {
            const int t = rs.t[i];
            *reinterpret_cast<unsigned *>(unit + kv4_k_word(hd, t, g, j)) = kv4_quant8(kx, ks);
            const unsigned w = kv4_quant8(vx, vs);
            vp[i][g * 8 + 2 * j] = (unsigned short)w; vp[i][g * 8 + 2 * j + 1] = (unsigned short)(w >> 16);
            if (j == 0) reinterpret_cast<unsigned short *>(unit + kv4_k_step_off(hd))[t * NG + g] = kd;
            if (j == 1) reinterpret_cast<unsigned short *>(unit + kv4_v_step_off(hd))[t * NG + g] = vd;
        }
    }
    __syncthreads();
    for (int it = tid; it < ST_ROWS * NG * 8; it += ST_T) {    // [r][row][g]: consecutive threads, consecutive bytes of a block
        const int q = (int)((unsigned)it * nth >> 16), g = it - q * NG, i = q % ST_ROWS, r = q / ST_ROWS;
        uint8_t *unit = rs.unit[i];
        if (!unit) continue;
        const int t = rs.t[i];
        const unsigned lo = vp[i][g * 8 + r];
        if (t & 1) {
            if (i > 0 && rs.unit[i - 1] == unit && rs.seq[i - 1] == rs.seq[i]) continue;             // stored with its partner
        } else if (i + 1 < ST_ROWS && rs.unit[i + 1] == unit && rs.seq[i + 1] == rs.seq[i]) {
            *reinterpret_cast<unsigned *>(unit + kv4_v_piece(hd, t, g, r)) = lo | (unsigned)vp[i + 1][g * 8 + r] << 16;
            continue;
        }
        *reinterpret_cast<unsigned short *>(unit + kv4_v_piece(hd, t, g, r)) = (unsigned short)lo;
    }
}

__device__ __forceinline__ double kv4_block_sum(double v, double *red) {
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    const int nw = blockDim.x >> 5;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    double s = 0;
    for (int i = 0; i < nw; i++) s += red[i];
    return s;
}

// One CTA per (row, head slot), a dim a thread, a group a warp: the norm and rotation of attn_prep_kernel (attn.cu) at the
// row's own position, q and k written back in place, then k and v quantised as above.
__global__ void __launch_bounds__(256) kv4_append_rope_kernel(Kv4Geom geo, uint8_t *mem, int layer, int H, float *q, long long q_ld, float *k,
                                                              const float *v, long long ld, Kv4Rope a, Kv4Batch b, int *err) {
    __shared__ double red64[8];
    __shared__ float xs[256];
    const int r = blockIdx.x, slot = blockIdx.y, i = threadIdx.x, hd = geo.hd;
    pdl_trigger();
    pdl_wait();
    const bool isq = slot < H;
    const int hh = isq ? slot : slot - H;
    int seq, pos;
    const int st = kv4_row<32>(b, r, &seq, &pos);
    if (st != KV4_ROW_OK) { if (st != KV4_ROW_NONE && i == 0) atomicExch(err, 1); return; }      // (the whole CTA)
    float *row = (isq ? q + (size_t)r * q_ld : k + (size_t)r * ld) + (size_t)hh * hd;
    const float *nw = isq ? a.qn : a.kn;
    float x = row[i];
    if (nw) {                                                  // hw/hw_ops.h:14-18
        const double ms = kv4_block_sum((double)x * (double)x, red64);
        const float rr = __fdiv_rn(1.f, __fsqrt_rn(__fadd_rn((float)(ms / hd), a.eps)));
        x = __fmul_rn(__fmul_rn(x, rr), nw[i]);
    }
    xs[i] = x;
    __syncthreads();
    // nn/rope.c:39-49 (half-split pairs) or engines/gemma.c:287-297 (p-RoPE), as attn_prep_kernel has them
    const int half = a.gemma ? hd / 2 : a.rot / 2, nang = a.gemma ? a.rot : a.rot / 2;
    if (i < 2 * half) {
        const int j = i < half ? i : i - half;
        if (j < nang) {
            const float angle = a.gemma ? __fmul_rn((float)pos, powf(a.theta, __fdiv_rn(__fmul_rn(-2.0f, (float)j), (float)hd)))
                                        : __fdiv_rn((float)pos, powf(a.theta, __fdiv_rn((float)(2 * j), (float)a.rot)));
            const float c = cosf(angle), sn = sinf(angle);
            const float lo = xs[j], hi = xs[j + half];
            x = i < half ? __fsub_rn(__fmul_rn(lo, c), __fmul_rn(hi, sn)) : __fadd_rn(__fmul_rn(lo, sn), __fmul_rn(hi, c));
        }
    }
    row[i] = x;
    if (isq) return;
    float vv = v[(size_t)r * ld + (size_t)hh * hd + i];
    if (a.vn) {                                                // engines/gemma.c:320-324
        const double ms = kv4_block_sum((double)vv * (double)vv, red64);
        const float rr = __fdiv_rn(1.f, __fsqrt_rn(__fadd_rn((float)(ms / hd), a.eps)));
        vv = __fmul_rn(__fmul_rn(vv, rr), a.vn[i]);
    }
    const int page = b.table[(size_t)seq * b.ld + pos / KV4_PAGE];
    if (!kv4_page_ok(geo, page)) { if (i == 0) atomicExch(err, 1); return; }
    uint8_t *unit = mem + kv4_unit_off(geo, page, layer, hh);
    const int lane = i & 31, g = i >> 5, t = pos % KV4_PAGE;
    unsigned short d;
    unsigned nib = kv4_quant_lane(x, lane, &d);
    kv4_put_k(unit, hd, t, g, lane, nib, d);
    nib = kv4_quant_lane(vv, lane, &d);
    kv4_put_v(unit, hd, t, g, lane, nib, d);
}

// the batch's own positions back as f32: k, v [rows][KV * hd]; 0 where the page is absent
__device__ __forceinline__ void kv4_values8(float *out, unsigned w, float d) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = __fmul_rn((float)((int)(w >> (4 * e) & 15u) - 8), d);
    *reinterpret_cast<float4 *>(out) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4 *>(out + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
__global__ void __launch_bounds__(ST_T) kv4_fetch_kernel(Kv4Geom geo, const uint8_t *mem, int layer, float *k, float *v, Kv4Batch b, int *err) {
    __shared__ Kv4Rows rs;
    const int tid = threadIdx.x, hd = geo.hd, NG = hd >> 5, row0 = blockIdx.x * ST_ROWS, head = blockIdx.y;
    pdl_trigger();
    pdl_wait();
    kv4_rows(rs, geo, const_cast<uint8_t *>(mem), b, row0, layer, head, err, true);
    const int per = hd >> 3;
    for (int it = tid; it < ST_ROWS * per; it += ST_T) {
        const int i = it / per, d8 = it - i * per, g = d8 >> 2, j = d8 & 3, t = rs.t[i];
        if (rs.seq[i] < 0) continue;
        const uint8_t *unit = rs.unit[i];
        unsigned kw = 0, vw = 0;
        float kd = 0.f, vd = 0.f;
        if (unit) {
            kw = *reinterpret_cast<const unsigned *>(unit + kv4_k_word(hd, t, g, j));
            vw = *reinterpret_cast<const unsigned short *>(unit + kv4_v_piece(hd, t, g, 2 * j)) |
                 (unsigned)*reinterpret_cast<const unsigned short *>(unit + kv4_v_piece(hd, t, g, 2 * j + 1)) << 16;
            kd = f16bits_to_f32(reinterpret_cast<const uint16_t *>(unit + kv4_k_step_off(hd))[t * NG + g]);
            vd = f16bits_to_f32(reinterpret_cast<const uint16_t *>(unit + kv4_v_step_off(hd))[t * NG + g]);
        }
        const size_t at = ((size_t)(row0 + i) * geo.KV + head) * hd + d8 * 8;
        kv4_values8(k + at, kw, kd);
        kv4_values8(v + at, vw, vd);
    }
}

}  // namespace

int launch_kv4_append(const Kv4Geom &geo, uint8_t *mem, int layer, const float *k, const float *v, long long ld, const Kv4Batch &b,
                      int *err, cudaStream_t st) {
    if (b.rows <= 0) return 0;
    CK(moty_launch_pdl(kv4_append_kernel, dim3((unsigned)((b.rows + (long long)ST_ROWS - 1) / ST_ROWS), geo.KV), dim3(ST_T), (size_t)0, st, geo, mem, layer, k, v, ld, b, err));
    return 0;
}

int launch_kv4_append_rope(const Kv4Geom &geo, uint8_t *mem, int layer, int H, float *q, long long q_ld, float *k, const float *v, long long ld,
                           const Kv4Rope &rope, const Kv4Batch &b, int *err, cudaStream_t st) {
    if (b.rows <= 0) return 0;
    if (H + geo.KV > 65535) return moty_set_error(MOTY_CUDA_ELIMIT, "kv4_append_rope: %d heads", H + geo.KV);
    CK(moty_launch_pdl(kv4_append_rope_kernel, dim3(b.rows, H + geo.KV), dim3(geo.hd), (size_t)0, st, geo, mem, layer, H, q, q_ld, k, v, ld, rope, b, err));
    return 0;
}

int launch_kv4_fetch(const Kv4Geom &geo, const uint8_t *mem, int layer, float *k, float *v, const Kv4Batch &b, int *err, cudaStream_t st) {
    if (b.rows <= 0) return 0;
    CK(moty_launch_pdl(kv4_fetch_kernel, dim3((unsigned)((b.rows + (long long)ST_ROWS - 1) / ST_ROWS), geo.KV), dim3(ST_T), (size_t)0, st, geo, mem, layer, k, v, b, err));
    return 0;
}
