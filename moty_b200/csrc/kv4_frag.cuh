// kv4_frag.cuh -- operand fragments of the 16-bit matrix instruction (mma.sync m16n8k16, f16 in, f32 sums) taken straight
// from a unit of the paged 4-bit KV cache, and the two-piece form of its f32 operands.
//
// A code of -8 .. 7 is exact in f16.  The other operand (a query value, or a softmax weight times a value step) is f32: it
// goes in as hi + lo, two f16 of 11 bits each, in neighbouring columns of the narrow operand: 2^-23 of a term, down to
// the smallest f16, 2^-24, where lo ends.  Both are first scaled by a power of two so that hi fits and the terms that count lie
// far above that end: a query row by its largest value (the end is 2^-38 of it), weights by the largest of a page and not of all
// (each kernel says what its end is).
#pragma once
#include "kv4.cuh"

// N words from shared memory, 4 N byte aligned
template <int N>
__device__ __forceinline__ void kv4_ldsw(unsigned (&w)[N], const uint8_t *p) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const uint4 v = *reinterpret_cast<const uint4 *>(p + 16 * i);
            w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
        }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            const uint2 v = *reinterpret_cast<const uint2 *>(p + 8 * i);
            w[2 * i] = v.x; w[2 * i + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) w[i] = *reinterpret_cast<const unsigned *>(p + 4 * i);
    }
}

// NG f16 steps of one key row (2 NG bytes aligned), two to a word
template <int NG>
__device__ __forceinline__ void kv4_ldsteps(unsigned (&w)[(NG + 1) / 2], const uint8_t *p) {
    if constexpr (NG % 2) {
#pragma unroll
        for (int i = 0; i < NG / 2; i++) {
            const unsigned short a = reinterpret_cast<const unsigned short *>(p)[2 * i], b = reinterpret_cast<const unsigned short *>(p)[2 * i + 1];
            w[i] = (unsigned)a | (unsigned)b << 16;
        }
        w[NG / 2] = reinterpret_cast<const unsigned short *>(p)[NG - 1];
    } else {
        if constexpr (NG % 4 == 0) {
#pragma unroll
            for (int i = 0; i < NG / 4; i++) {
                const uint2 v = *reinterpret_cast<const uint2 *>(p + 8 * i);
                w[2 * i] = v.x; w[2 * i + 1] = v.y;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NG / 2; i++) w[i] = *reinterpret_cast<const unsigned *>(p + 4 * i);
        }
    }
}
__device__ __forceinline__ float kv4_half_of(unsigned w, int hi) {
    return __half2float(__ushort_as_half((unsigned short)(hi ? w >> 16 : w & 0xffffu)));
}

// steps of positions t and t + 1, NG each, two to a word: those outside [lo, hi) become 0 (a page's memory behind the last
// position may hold anything)
template <int NG>
__device__ __forceinline__ void kv4_mask_steps(unsigned (&w)[NG], int t, int lo, int hi) {
    const bool s0 = t >= lo && t < hi, s1 = t + 1 >= lo && t + 1 < hi;
#pragma unroll
    for (int i = 0; i < NG; i++) {
        const unsigned a = 2 * i < NG ? (s0 ? 0xffffu : 0u) : (s1 ? 0xffffu : 0u), b = 2 * i + 1 < NG ? (s0 ? 0xffff0000u : 0u) : (s1 ? 0xffff0000u : 0u);
        w[i] &= a | b;
    }
}

// (The bare bits are n in f16 subnormals and need four operations less a word, with -8 sum(q) as the sum's start; but the
// matrix unit cuts sums off, and there the larger terms left 1.9e-6 instead of 2e-7.)
constexpr unsigned KV4_C = 0x64006400u;
// nibbles i and i + 4 of a word as f16 pairs of code values (n - 8): 0x6400 | n is 1024 + n, 0x6400 | 16 n is 1024 + 16 n
__device__ __forceinline__ void kv4_codes(unsigned w, unsigned (&e)[4]) {
    constexpr unsigned M0 = 0x000f000fu, M1 = 0x00f000f0u;
    const unsigned C = KV4_C;
    const unsigned s = w >> 8;
    const __half2 b0 = __halves2half2(__ushort_as_half(0x6408), __ushort_as_half(0x6408));      // 1032
    const __half2 c1 = __halves2half2(__ushort_as_half(0x2c00), __ushort_as_half(0x2c00));      // 1 / 16
    const __half2 b1 = __halves2half2(__ushort_as_half(0xd480), __ushort_as_half(0xd480));      // -72 = -(1024 / 16 + 8)
    unsigned r[4];                                           // (w & M) | C in one operation: C in a register, M in the instruction
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r[0]) : "r"(w), "n"(M0), "r"(C));
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r[1]) : "r"(w), "n"(M1), "r"(C));
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r[2]) : "r"(s), "n"(M0), "r"(C));
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r[3]) : "r"(s), "n"(M1), "r"(C));
    __half2 h;
    h = __hsub2(*reinterpret_cast<__half2 *>(&r[0]), b0); e[0] = *reinterpret_cast<unsigned *>(&h);
    h = __hfma2(*reinterpret_cast<__half2 *>(&r[1]), c1, b1); e[1] = *reinterpret_cast<unsigned *>(&h);
    h = __hsub2(*reinterpret_cast<__half2 *>(&r[2]), b0); e[2] = *reinterpret_cast<unsigned *>(&h);
    h = __hfma2(*reinterpret_cast<__half2 *>(&r[3]), c1, b1); e[3] = *reinterpret_cast<unsigned *>(&h);
}

__device__ __forceinline__ void kv4_mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same with a sum that starts from zero
__device__ __forceinline__ void kv4_mma0(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ unsigned kv4_pack_f16(float lo_half, float hi_half) {                // two f32, rounded, low half first
    const __half2 h = __floats2half2_rn(lo_half, hi_half);
    return *reinterpret_cast<const unsigned *>(&h);
}
// x0 + s h.low and x1 + s h.high for a pair h and a factor s of f16 (s h is exact here: s is 0 or -1)
__device__ __forceinline__ void kv4_rest(float &x0, float &x1, unsigned h, unsigned short s) {
    asm("{.reg .f16 l, u; mov.b32 {l, u}, %2; fma.rn.f32.f16 %0, l, %3, %0; fma.rn.f32.f16 %1, u, %3, %1;}" : "+f"(x0), "+f"(x1) : "r"(h), "h"(s));
}
constexpr unsigned short KV4_H0 = 0x8000, KV4_HM1 = 0xbc00;  // -0 and -1
// the pair (x0, x1) as f16: its leading pieces (s = -0) or what they leave over (s = -1)
__device__ __forceinline__ unsigned kv4_piece(float x0, float x1, unsigned short s) {
    kv4_rest(x0, x1, kv4_pack_f16(x0, x1), s);
    return kv4_pack_f16(x0, x1);
}
// both: x = h + lo
__device__ __forceinline__ void kv4_pieces(float x0, float x1, unsigned &h, unsigned &lo) {
    h = kv4_pack_f16(x0, x1);
    kv4_rest(x0, x1, h, KV4_HM1);
    lo = kv4_pack_f16(x0, x1);
}
__device__ __forceinline__ unsigned kv4_hmul2(unsigned a, unsigned b) {
    const __half2 h = __hmul2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const unsigned *>(&h);
}
// (yh + yl) d as hi + lo, pairs of f16
__device__ __forceinline__ void kv4_scaled_pieces(unsigned yh, unsigned yl, unsigned d, unsigned &hi, unsigned &lo) {
    const __half2 a = *reinterpret_cast<const __half2 *>(&yh), b = *reinterpret_cast<const __half2 *>(&yl), c = *reinterpret_cast<const __half2 *>(&d);
    const __half2 h = __hmul2(a, c), l = __hfma2(b, c, __hfma2(a, c, __hneg2(h)));
    hi = *reinterpret_cast<const unsigned *>(&h);
    lo = *reinterpret_cast<const unsigned *>(&l);
}
// 2^k for -126 <= k <= 127, and x 2^k for any k of the f32 range (two factors, each a normal number)
__device__ __forceinline__ float kv4_pow2(int k) { return __int_as_float((k + 127) << 23); }
__device__ __forceinline__ float kv4_scale2(float x, int k) { const int h = k >> 1; return x * kv4_pow2(h) * kv4_pow2(k - h); }
// the power of two that brings a query row whose largest magnitude has the bits mb below 2^14 (0 for a row of zeros)
__device__ __forceinline__ int kv4_q_shift(unsigned mb) { return mb ? 13 + 127 - (int)(mb >> 23 ? mb >> 23 : 1) : 0; }
__device__ __forceinline__ float kv4_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
