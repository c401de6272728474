// kv4_attend.cu -- attention over the paged 4-bit KV cache.
//
// For row r of a sequence at position p, query head h of KV head h / G:
//     s_t = scale * q . k_t,   ctx = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m)   over t in (p - window, p],
// k_t and v_t the values held (code * step), positions of absent pages (table entry -1) left out, 0 where nothing is left.
#include "kv4.cuh"

namespace {

// One warp per (row, query head), lane = dim of a group; one pass with the running maximum and sum.
__global__ void __launch_bounds__(128) kv4_attend_simple_kernel(Kv4Attend a) {
    const int lane = threadIdx.x & 31, hd = a.geo.hd, NG = hd >> 5;
    const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    pdl_trigger();
    pdl_wait();
    if (w >= (long long)a.b.rows * a.H) return;
    const int r = (int)(w / a.H), h = (int)(w % a.H);
    int seq, pos;
    const int st = kv4_row(a.b, r, &seq, &pos);
    if (st == KV4_ROW_NONE) return;
    float acc[8], q[8], m = -INFINITY, l = 0.f;
    for (int g = 0; g < 8; g++) { acc[g] = 0.f; q[g] = 0.f; }
    int n = 0;
    if (st == KV4_ROW_BAD || a.b.len[seq] > a.max_len || a.b.row0[seq + 1] - a.b.row0[seq] > a.max_rows) {
        if (lane == 0) atomicExch(a.err, 1);
    } else {
        n = pos + 1;
        for (int g = 0; g < 8; g++) if (g < NG) q[g] = a.q[(size_t)r * a.q_ld + (size_t)h * hd + g * 32 + lane];
    }
    for (int t = a.window > 0 && n > a.window ? n - a.window : 0; t < n; t++) {
        const int page = a.b.table[(size_t)seq * a.b.ld + t / KV4_PAGE];
        if (!kv4_page_ok(a.geo, page)) { if (page != -1 && lane == 0) atomicExch(a.err, 1); continue; }
        const uint8_t *u = a.mem + kv4_unit_off(a.geo, page, a.layer, h / a.G);
        const int tt = t % KV4_PAGE;
        float s = 0.f;
        for (int g = 0; g < 8; g++)
            if (g < NG) {
                const unsigned kw = *reinterpret_cast<const unsigned *>(u + kv4_k_word(hd, tt, g, lane >> 3));
                const float d = f16bits_to_f32(reinterpret_cast<const uint16_t *>(u + kv4_k_step_off(hd))[tt * NG + g]);
                s = fmaf(q[g], (float)((int)((kw >> (4 * (lane & 7))) & 15u) - 8) * d, s);
            }
        for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
        s *= a.scale;
        const float mn = fmaxf(m, s), f = mn == -INFINITY ? 1.f : expf(m - mn), e = mn == -INFINITY ? s : expf(s - mn);
        m = mn; l = fmaf(l, f, e);
        for (int g = 0; g < 8; g++)
            if (g < NG) {
                const unsigned vw = *reinterpret_cast<const unsigned short *>(u + kv4_v_piece(hd, tt, g, lane >> 2));
                const float d = f16bits_to_f32(reinterpret_cast<const uint16_t *>(u + kv4_v_step_off(hd))[tt * NG + g]);
                acc[g] = fmaf(acc[g], f, e * ((float)((int)((vw >> (4 * (lane & 3))) & 15u) - 8) * d));
            }
    }
    for (int g = 0; g < 8; g++)
        if (g < NG) a.ctx[((size_t)r * a.H + h) * hd + g * 32 + lane] = l == 0.f ? 0.f : acc[g] / l;
}

}  // namespace

size_t kv4_attend_scratch_bytes(const Kv4Attend &a, int sms) { return 0; }

int launch_kv4_attend(const Kv4Attend &a, float *part, int sms, cudaStream_t st) {
    const long long warps = (long long)a.b.rows * a.H;
    if (warps <= 0) return 0;
    if ((warps + 3) / 4 > 0x7fffffffLL) return moty_set_error(MOTY_CUDA_ELIMIT, "kv4_attend: %d rows of %d heads", a.b.rows, a.H);
    CK(moty_launch_pdl(kv4_attend_simple_kernel, dim3((unsigned)((warps + 3) / 4)), dim3(128), (size_t)0, st, a));
    return 0;
}
