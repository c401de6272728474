// kv4_frag.cuh -- operand fragments of the 16-bit matrix instruction (mma.sync m16n8k16, f16 in, f32 sums) taken straight
// from a unit of the paged 4-bit KV cache, and the two-piece form of its f32 operands.
//
// A code of -8 .. 7 is exact in f16.  The other operand (a query value, or a softmax weight times a value step) is f32: it
// goes in as hi + lo, two f16 of 11 bits each, in neighbouring columns of the narrow operand, so that products and sums
// are f32's own to within 2^-23 of each term.  Both are first scaled by a power of two so that hi fits and lo keeps its bits.
#pragma once
#include "kv4.cuh"

// Pages are written by the launch before (append), which a chained launch may overlap until pdl_wait: plain loads, not the
// read-only path.  They are read once: not kept in L1.
__device__ __forceinline__ int4 kv4_ld16(const uint8_t *p) {
    int4 v;
    asm volatile("ld.global.L1::no_allocate.v4.s32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
// N 32-bit words from a 4 N byte aligned address (16-, 8- or 4-byte loads as N allows)
template <int N>
__device__ __forceinline__ void kv4_ldw(unsigned (&w)[N], const uint8_t *p) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const int4 v = kv4_ld16(p + 16 * i);
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

// nibbles i and i + 4 of a word as f16 pairs of code values (n - 8): 0x6400 | n is 1024 + n, 0x6400 | 16 n is 1024 + 16 n
__device__ __forceinline__ void kv4_codes(unsigned w, unsigned (&e)[4]) {
    constexpr unsigned M0 = 0x000f000fu, M1 = 0x00f000f0u, C = 0x64006400u;
    const unsigned s = w >> 8;
    const __half2 b0 = __halves2half2(__ushort_as_half(0x6408), __ushort_as_half(0x6408));      // 1032
    const __half2 c1 = __halves2half2(__ushort_as_half(0x2c00), __ushort_as_half(0x2c00));      // 1 / 16
    const __half2 b1 = __halves2half2(__ushort_as_half(0xd480), __ushort_as_half(0xd480));      // -72 = -(1024 / 16 + 8)
    unsigned r[4] = {(w & M0) | C, (w & M1) | C, (s & M0) | C, (s & M1) | C};
    __half2 h;
    h = __hsub2(*reinterpret_cast<__half2 *>(&r[0]), b0); e[0] = *reinterpret_cast<unsigned *>(&h);
    h = __hfma2(*reinterpret_cast<__half2 *>(&r[1]), c1, b1); e[1] = *reinterpret_cast<unsigned *>(&h);
    h = __hsub2(*reinterpret_cast<__half2 *>(&r[2]), b0); e[2] = *reinterpret_cast<unsigned *>(&h);
    h = __hfma2(*reinterpret_cast<__half2 *>(&r[3]), c1, b1); e[3] = *reinterpret_cast<unsigned *>(&h);
}

__device__ __forceinline__ void kv4_mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned kv4_pack_f16(float lo_half, float hi_half) {                // two f32, rounded, low half first
    const __half2 h = __floats2half2_rn(lo_half, hi_half);
    return *reinterpret_cast<const unsigned *>(&h);
}
// the pair (x0, x1) as f16: its leading pieces (sel = 0) or what they leave over (sel = 1)
__device__ __forceinline__ unsigned kv4_piece(float x0, float x1, float sel) {
    const __half2 h = __floats2half2_rn(x0, x1);
    const float2 f = __half22float2(h);
    return kv4_pack_f16(fmaf(-sel, f.x, x0), fmaf(-sel, f.y, x1));
}
__device__ __forceinline__ float kv4_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
