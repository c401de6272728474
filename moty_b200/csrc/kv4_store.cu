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
    const float step = fminf(fmaxf(__fdiv_rn(fabsf(big), 8.f), __fdiv_rn(other, 7.f)), 65504.f);
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

// the unit and slot of batch row r for (layer, head), or null (a row behind the last sequence; a bad one sets *err)
__device__ __forceinline__ uint8_t *kv4_find(const Kv4Geom &geo, uint8_t *mem, const Kv4Batch &b, int r, int layer, int head, int *t,
                                             int *pos, int *err, bool absent_ok) {
    int seq;
    const int st = kv4_row(b, r, &seq, pos);
    if (st == KV4_ROW_NONE) return nullptr;
    if (st == KV4_ROW_BAD) { atomicExch(err, 1); return nullptr; }
    const int page = b.table[(size_t)seq * b.ld + *pos / KV4_PAGE];
    if (!kv4_page_ok(geo, page)) { if (!(absent_ok && page == -1)) atomicExch(err, 1); return nullptr; }
    *t = *pos % KV4_PAGE;
    return mem + kv4_unit_off(geo, page, layer, head);
}

__global__ void __launch_bounds__(256) kv4_append_kernel(Kv4Geom geo, uint8_t *mem, int layer, const float *k, const float *v, long long ld,
                                                         Kv4Batch b, int *err) {
    const int lane = threadIdx.x & 31;
    const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);      // one warp per (row, head)
    pdl_trigger();
    pdl_wait();
    if (w >= (long long)b.rows * geo.KV) return;
    const int r = (int)(w / geo.KV), head = (int)(w % geo.KV);
    int t = 0, pos;
    uint8_t *unit = kv4_find(geo, mem, b, r, layer, head, &t, &pos, err, false);
    if (!unit) return;
    for (int g = 0; g < geo.hd >> 5; g++) {
        unsigned short d;
        const size_t at = (size_t)r * ld + head * geo.hd + g * 32 + lane;
        unsigned nib = kv4_quant_lane(k[at], lane, &d);
        kv4_put_k(unit, geo.hd, t, g, lane, nib, d);
        nib = kv4_quant_lane(v[at], lane, &d);
        kv4_put_v(unit, geo.hd, t, g, lane, nib, d);
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
    const int st = kv4_row(b, r, &seq, &pos);
    if (st != KV4_ROW_OK) { if (st == KV4_ROW_BAD && i == 0) atomicExch(err, 1); return; }       // (the whole CTA)
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
__global__ void __launch_bounds__(256) kv4_fetch_kernel(Kv4Geom geo, const uint8_t *mem, int layer, float *k, float *v, Kv4Batch b, int *err) {
    const int lane = threadIdx.x & 31, hd = geo.hd, NG = hd >> 5;
    const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);      // one warp per (row, head)
    pdl_trigger();
    pdl_wait();
    if (w >= (long long)b.rows * geo.KV) return;
    const int r = (int)(w / geo.KV), head = (int)(w % geo.KV);
    int seq, pos, t = 0, p2;
    if (kv4_row(b, r, &seq, &pos) == KV4_ROW_NONE) return;
    const uint8_t *unit = kv4_find(geo, const_cast<uint8_t *>(mem), b, r, layer, head, &t, &p2, err, true);
    for (int g = 0; g < NG; g++) {
        const size_t at = ((size_t)r * geo.KV + head) * hd + g * 32 + lane;
        float kx = 0.f, vx = 0.f;
        if (unit) {
            const unsigned kw = *reinterpret_cast<const unsigned *>(unit + kv4_k_word(hd, t, g, lane >> 3));
            const unsigned vw = *reinterpret_cast<const unsigned short *>(unit + kv4_v_piece(hd, t, g, lane >> 2));
            kx = __fmul_rn((float)((int)((kw >> (4 * (lane & 7))) & 15u) - 8), f16bits_to_f32(reinterpret_cast<const uint16_t *>(unit + kv4_k_step_off(hd))[t * NG + g]));
            vx = __fmul_rn((float)((int)((vw >> (4 * (lane & 3))) & 15u) - 8), f16bits_to_f32(reinterpret_cast<const uint16_t *>(unit + kv4_v_step_off(hd))[t * NG + g]));
        }
        k[at] = kx; v[at] = vx;
    }
}

}  // namespace

int launch_kv4_append(const Kv4Geom &geo, uint8_t *mem, int layer, const float *k, const float *v, long long ld, const Kv4Batch &b,
                      int *err, cudaStream_t st) {
    const long long warps = (long long)b.rows * geo.KV;
    if (warps <= 0) return 0;
    if ((warps + 7) / 8 > 0x7fffffffLL) return moty_set_error(MOTY_CUDA_ELIMIT, "kv4_append: %d rows", b.rows);
    CK(moty_launch_pdl(kv4_append_kernel, dim3((unsigned)((warps + 7) / 8)), dim3(256), (size_t)0, st, geo, mem, layer, k, v, ld, b, err));
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
    const long long warps = (long long)b.rows * geo.KV;
    if (warps <= 0) return 0;
    if ((warps + 7) / 8 > 0x7fffffffLL) return moty_set_error(MOTY_CUDA_ELIMIT, "kv4_fetch: %d rows", b.rows);
    CK(moty_launch_pdl(kv4_fetch_kernel, dim3((unsigned)((warps + 7) / 8)), dim3(256), (size_t)0, st, geo, mem, layer, k, v, b, err));
    return 0;
}
