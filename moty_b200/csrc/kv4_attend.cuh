// kv4_attend.cuh -- how an attention call over the paged 4-bit KV cache is cut, and what its kernels share.
#pragma once
#include "kv4.cuh"

constexpr int KV4_LINES = 64;             // (row, query head) pairs a CTA of the prompt kernel takes
constexpr int KV4_TC_LINES = 256, KV4_TC_PAGES = 512;       // the same of the tensor-memory prompt kernel, and the most pages of its spans
int launch_kv4_prompt(const Kv4Attend &a, const Kv4Plan &p, float *part, cudaStream_t st);
int launch_kv4_prompt_tc(const Kv4Attend &a, const Kv4Plan &p, float *part, cudaStream_t st);

#ifdef __CUDACC__
// what a CTA of sequence `seq` works on
struct Kv4Seq { int r0, n, len; bool ok; };
__device__ __forceinline__ Kv4Seq kv4_load_seq(const Kv4Attend &a, int seq) {
    Kv4Seq q;
    const int st = kv4_seq(a.b, seq, &q.r0, &q.n, &q.len);
    q.ok = st == KV4_ROW_OK && q.n <= a.max_rows && q.len <= a.max_len;
    if (st != KV4_ROW_NONE && !q.ok && threadIdx.x == 0) atomicExch(a.err, 1);
    if (st == KV4_ROW_NONE) q.n = 0;
    return q;
}
// rows of a sequence that is refused are zero (one CTA per KV head does it)
__device__ __forceinline__ void kv4_zero_rows(const Kv4Attend &a, const Kv4Seq &q, int head) {
    const int lo = q.r0 > 0 ? q.r0 : 0;
    const long long hi = (long long)q.r0 + q.n < a.b.rows ? (long long)q.r0 + q.n : a.b.rows;
    const int w = a.G * a.geo.hd;
    for (long long r = lo; r < hi; r++)
        for (int i = threadIdx.x; i < w; i += blockDim.x) a.ctx[r * a.H * a.geo.hd + (size_t)head * w + i] = 0.f;
}
// a finished row: its sums over the weights' total l, zeros where nothing was seen (times a reciprocal: half a step of f32
// more than the quotient, and a prompt's CTA spends 3 us less on its rows)
__device__ __forceinline__ float kv4_over(float l) { return l == 0.f ? 0.f : __frcp_rn(l); }
__device__ __forceinline__ float4 kv4_times(const float4 &o, float f) { return make_float4(o.x * f, o.y * f, o.z * f, o.w * f); }
// What sums over a part with maximum m count where the whole's is M; never 0 where the part saw anything (l > 0), for a NaN
// among its values has to stay one however small its weight.
__device__ __forceinline__ float kv4_factor(float l, float m, float M) { return l == 0.f ? 0.f : fmaxf(kv4_exp2(m - M), 1.17549435e-38f); }
// rows at positions p_a .. p_z: [lo_any, hi_any) is seen by some of them, [lo_all, hi_all) by all
struct Kv4Range { int lo_any, hi_any, lo_all, hi_all; };
__device__ __forceinline__ Kv4Range kv4_range(const Kv4Attend &a, int p_a, int p_z) {
    Kv4Range r;
    r.lo_any = a.window > 0 && p_a - a.window + 1 > 0 ? p_a - a.window + 1 : 0;
    r.lo_all = a.window > 0 && p_z - a.window + 1 > 0 ? p_z - a.window + 1 : 0;
    r.hi_any = p_z + 1;
    r.hi_all = p_a + 1;
    return r;
}
#endif
