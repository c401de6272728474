// kv4_api.cu -- C entries of the paged 4-bit KV cache: argument checks, the page bookkeeping, launches.
#include "kv4.cuh"
#include <math.h>
#include <new>
#include <string.h>

struct MotyCudaKv4 {
    Kv4Geom geo;
    int device;
    uint8_t *mem;
    bool owned;
    Kv4Pages pages;
};

static cudaStream_t kv4_stream(DevCtx *c, void *stream) { return stream ? (cudaStream_t)stream : c->stream; }
static bool kv4_aligned(const void *p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

static int kv4_shape(const char *who, int layers, int KV, int hd) {
    if (layers <= 0 || KV <= 0 || hd < 32 || hd > 256 || hd % 32 || (long long)layers * KV > 65535)
        return moty_set_error(MOTY_CUDA_EARG, "%s: layers=%d kv_heads=%d head_dim=%d (a multiple of 32, at most 256)", who, layers, KV, hd);
    return 0;
}

extern "C" int64_t moty_cuda_kv4_page_bytes(int layers, int n_kv_heads, int head_dim) {
    const int r = kv4_shape("kv4_page_bytes", layers, n_kv_heads, head_dim);
    if (r) return r;
    const Kv4Geom g{layers, n_kv_heads, head_dim, 1};
    return (int64_t)kv4_page_bytes(g);
}

extern "C" int moty_cuda_kv4_create(MotyCudaKv4 **out, int layers, int n_kv_heads, int head_dim, int pages, void *mem_dev, int device) {
    if (!out) return moty_set_error(MOTY_CUDA_EARG, "kv4_create: null argument");
    CKR(kv4_shape("kv4_create", layers, n_kv_heads, head_dim));
    if (pages <= 0 || pages > (1 << 25)) return moty_set_error(MOTY_CUDA_EARG, "kv4_create: pages=%d", pages);
    if (!kv4_aligned(mem_dev, 128)) return moty_set_error(MOTY_CUDA_EARG, "kv4_create: the pages' memory must be 128-byte aligned");
    DevCtx *c = moty_ctx(device);
    if (!c) return moty_set_error(MOTY_CUDA_EINIT, "device %d not initialised", device);
    MOTY_USE_DEVICE(device);
    if (mem_dev) {
        cudaPointerAttributes at;
        if (cudaPointerGetAttributes(&at, mem_dev) != cudaSuccess) { cudaGetLastError(); at.type = cudaMemoryTypeUnregistered; }
        if (at.type != cudaMemoryTypeDevice || at.device != device)
            return moty_set_error(MOTY_CUDA_EARG, "kv4_create: the pages' memory is not on device %d", device);
    }
    MotyCudaKv4 *h = nullptr;
    try {
        h = new MotyCudaKv4();
        h->pages.init(pages);
    } catch (const std::bad_alloc &) {
        delete h;
        return moty_set_error(MOTY_CUDA_ENOMEM, "kv4_create: host allocation for %d pages", pages);
    }
    h->geo = Kv4Geom{layers, n_kv_heads, head_dim, pages};
    h->device = device; h->mem = (uint8_t *)mem_dev; h->owned = !mem_dev;
    if (!mem_dev) {
        const size_t bytes = kv4_page_bytes(h->geo) * (size_t)pages;
        cudaError_t e = cudaMalloc(&h->mem, bytes);
        // positions never written read as zero rows
        if (e == cudaSuccess) {
            e = cudaMemsetAsync(h->mem, 0, bytes, c->stream);
            if (e == cudaSuccess) e = cudaStreamSynchronize(c->stream);
            if (e != cudaSuccess) cudaFree(h->mem);
        }
        if (e != cudaSuccess) {
            cudaGetLastError();
            delete h;
            return moty_set_error(MOTY_CUDA_ENOMEM, "kv4_create: %zu bytes: %s", bytes, cudaGetErrorString(e));
        }
    }
    *out = h;
    return 0;
}

extern "C" int moty_cuda_kv4_free(MotyCudaKv4 *kv) {
    if (!kv) return 0;
    if (kv->owned) {
        MotyDevGuard g;
        if (g.set(kv->device) == cudaSuccess) cudaFree(kv->mem);       // (waits for the device's work)
    }
    delete kv;
    return 0;
}

extern "C" int moty_cuda_kv4_alloc(MotyCudaKv4 *kv, int n, int *ids) {
    if (!kv || n < 0 || (n && !ids)) return moty_set_error(MOTY_CUDA_EARG, "kv4_alloc: null argument or n=%d", n);
    if (!kv->pages.alloc(n, ids)) return moty_set_error(MOTY_CUDA_ELIMIT, "kv4_alloc: %d pages asked, %d free", n, kv->pages.free_count());
    return 0;
}
extern "C" int moty_cuda_kv4_retain(MotyCudaKv4 *kv, int n, const int *ids) {
    if (!kv || n < 0 || (n && !ids)) return moty_set_error(MOTY_CUDA_EARG, "kv4_retain: null argument or n=%d", n);
    if (!kv->pages.retain(ids, n)) return moty_set_error(MOTY_CUDA_EARG, "kv4_retain: a page of the list is not in use");
    return 0;
}
extern "C" int moty_cuda_kv4_release(MotyCudaKv4 *kv, int n, const int *ids) {
    if (!kv || n < 0 || (n && !ids)) return moty_set_error(MOTY_CUDA_EARG, "kv4_release: null argument or n=%d", n);
    if (!kv->pages.release(ids, n)) return moty_set_error(MOTY_CUDA_EARG, "kv4_release: a page of the list is not in use (or listed more often than it is owned)");
    return 0;
}
extern "C" int moty_cuda_kv4_free_pages(const MotyCudaKv4 *kv) {
    if (!kv) return moty_set_error(MOTY_CUDA_EARG, "kv4_free_pages: null argument");
    return kv->pages.free_count();
}
extern "C" int moty_cuda_kv4_compact_plan(MotyCudaKv4 *kv, int cap, int *src, int *dst, int *n) {
    if (!kv || !n || cap < 0 || (cap && (!src || !dst))) return moty_set_error(MOTY_CUDA_EARG, "kv4_compact_plan: null argument or cap=%d", cap);
    try {
        std::vector<int> s, d;
        kv->pages.plan(&s, &d);
        *n = (int)s.size();
        if ((int)s.size() > cap) return moty_set_error(MOTY_CUDA_ELIMIT, "kv4_compact_plan: %d moves, room for %d", (int)s.size(), cap);
        if (!s.empty()) {
            memcpy(src, s.data(), s.size() * 4);
            memcpy(dst, d.data(), d.size() * 4);
            kv->pages.moved(s, d);
        }
    } catch (const std::bad_alloc &) {
        return moty_set_error(MOTY_CUDA_ENOMEM, "kv4_compact_plan: host allocation");
    }
    return 0;
}

static int kv4_batch(const char *who, const MotyCudaKv4 *kv, int layer, const MotyKv4Batch *b, Kv4Batch *out) {
    if (!kv || !b) return moty_set_error(MOTY_CUDA_EARG, "%s: null argument", who);
    if (layer < 0 || layer >= kv->geo.layers) return moty_set_error(MOTY_CUDA_EARG, "%s: layer %d of %d", who, layer, kv->geo.layers);
    if (b->nseq < 0 || b->rows < 0 || b->table_ld <= 0 || !b->row0_dev || !b->len_dev || !b->table_dev)
        return moty_set_error(MOTY_CUDA_EARG, "%s: batch of nseq=%d rows=%d table_ld=%d, or a null array", who, b->nseq, b->rows, b->table_ld);
    *out = Kv4Batch{b->nseq, b->rows, b->table_ld, b->row0_dev, b->len_dev, b->table_dev};
    return 0;
}
// row strides: 0 = contiguous
static int kv4_ld(const char *who, int ld, long long width, long long *out) {
    if (ld < 0 || (ld && ld < width) || ld % 4) return moty_set_error(MOTY_CUDA_EARG, "%s: row stride %d for rows of %lld values", who, ld, width);
    *out = ld ? ld : width;
    return 0;
}

extern "C" int moty_cuda_kv4_append_dev(MotyCudaKv4 *kv, int layer, const float *k_dev, const float *v_dev, int kv_ld,
                                        const MotyKv4Batch *batch, void *stream) {
    Kv4Batch b;
    CKR(kv4_batch("kv4_append_dev", kv, layer, batch, &b));
    long long ld;
    CKR(kv4_ld("kv4_append_dev", kv_ld, (long long)kv->geo.KV * kv->geo.hd, &ld));
    if (!k_dev || !v_dev || !kv4_aligned(k_dev, 16) || !kv4_aligned(v_dev, 16))
        return moty_set_error(MOTY_CUDA_EARG, "kv4_append_dev: k or v null or not 16-byte aligned");
    DevCtx *c = moty_ctx(kv->device);
    if (!c) return moty_set_error(MOTY_CUDA_EINIT, "device %d not initialised", kv->device);
    if (!b.nseq || !b.rows) return 0;
    MOTY_USE_DEVICE(kv->device);
    return launch_kv4_append(kv->geo, kv->mem, layer, k_dev, v_dev, ld, b, c->err_dev + 4, kv4_stream(c, stream));
}

extern "C" int moty_cuda_kv4_append_rope_dev(MotyCudaKv4 *kv, int layer, int n_heads, float *q_dev, int q_ld, float *k_dev, const float *v_dev,
                                             int kv_ld, const MotyKv4Rope *rope, const MotyKv4Batch *batch, void *stream) {
    Kv4Batch b;
    CKR(kv4_batch("kv4_append_rope_dev", kv, layer, batch, &b));
    if (!rope || n_heads < 0 || (n_heads && !q_dev) || !k_dev || !v_dev) return moty_set_error(MOTY_CUDA_EARG, "kv4_append_rope_dev: null argument");
    const int hd = kv->geo.hd;
    if (rope->rot < 0 || (rope->gemma ? rope->rot > hd / 2 : rope->rot > hd || (rope->rot & 1)) || !(rope->theta > 0.f) || !(rope->eps >= 0.f))
        return moty_set_error(MOTY_CUDA_EARG, "kv4_append_rope_dev: rot=%d of head_dim=%d, theta=%g, eps=%g", rope->rot, hd, (double)rope->theta, (double)rope->eps);
    if (n_heads + (long long)kv->geo.KV > 65535) return moty_set_error(MOTY_CUDA_ELIMIT, "kv4_append_rope_dev: %d heads", n_heads);
    long long ld, qld;
    CKR(kv4_ld("kv4_append_rope_dev", kv_ld, (long long)kv->geo.KV * hd, &ld));
    CKR(kv4_ld("kv4_append_rope_dev", q_ld, (long long)n_heads * hd, &qld));
    if (!kv4_aligned(q_dev, 16) || !kv4_aligned(k_dev, 16) || !kv4_aligned(v_dev, 16))
        return moty_set_error(MOTY_CUDA_EARG, "kv4_append_rope_dev: q, k or v not 16-byte aligned");
    DevCtx *c = moty_ctx(kv->device);
    if (!c) return moty_set_error(MOTY_CUDA_EINIT, "device %d not initialised", kv->device);
    if (!b.nseq || !b.rows) return 0;
    MOTY_USE_DEVICE(kv->device);
    const Kv4Rope r{rope->rot, rope->gemma, rope->theta, rope->eps, rope->qn_dev, rope->kn_dev, rope->vn_dev};
    return launch_kv4_append_rope(kv->geo, kv->mem, layer, n_heads, q_dev, qld, k_dev, v_dev, ld, r, b, c->err_dev + 4, kv4_stream(c, stream));
}

extern "C" int moty_cuda_kv4_fetch_dev(MotyCudaKv4 *kv, int layer, float *k_dev, float *v_dev, const MotyKv4Batch *batch, void *stream) {
    Kv4Batch b;
    CKR(kv4_batch("kv4_fetch_dev", kv, layer, batch, &b));
    if (!k_dev || !v_dev || !kv4_aligned(k_dev, 16) || !kv4_aligned(v_dev, 16))
        return moty_set_error(MOTY_CUDA_EARG, "kv4_fetch_dev: k or v null or not 16-byte aligned");
    DevCtx *c = moty_ctx(kv->device);
    if (!c) return moty_set_error(MOTY_CUDA_EINIT, "device %d not initialised", kv->device);
    if (!b.nseq || !b.rows) return 0;
    MOTY_USE_DEVICE(kv->device);
    return launch_kv4_fetch(kv->geo, kv->mem, layer, k_dev, v_dev, b, c->err_dev + 4, kv4_stream(c, stream));
}

extern "C" int moty_cuda_kv4_attend_dev(MotyCudaKv4 *kv, int layer, float *ctx_dev, const float *q_dev, int q_ld, int n_heads, int window,
                                        float scale, const MotyKv4Batch *batch, void *stream) {
    Kv4Attend a;
    CKR(kv4_batch("kv4_attend_dev", kv, layer, batch, &a.b));
    a.geo = kv->geo; a.mem = kv->mem; a.layer = layer;
    if (n_heads <= 0 || n_heads % kv->geo.KV || n_heads > 65535)
        return moty_set_error(MOTY_CUDA_EARG, "kv4_attend_dev: %d query heads on %d KV heads", n_heads, kv->geo.KV);
    if (window < 0 || !(scale >= 0.f) || isinf(scale)) return moty_set_error(MOTY_CUDA_EARG, "kv4_attend_dev: window=%d scale=%g", window, (double)scale);
    if (batch->max_rows < 0 || batch->max_rows > batch->rows || batch->max_len < 0 || batch->max_len > (long long)batch->table_ld * KV4_PAGE)
        return moty_set_error(MOTY_CUDA_EARG, "kv4_attend_dev: max_rows=%d of %d rows, max_len=%d with %d pages a sequence", batch->max_rows, batch->rows,
                              batch->max_len, batch->table_ld);
    if (batch->max_len > 1 << 30) return moty_set_error(MOTY_CUDA_ELIMIT, "kv4_attend_dev: max_len=%d (2^30 at most)", batch->max_len);
    if ((long long)batch->rows * n_heads > 0x7fffff00LL)       // (512 GB of context rows)
        return moty_set_error(MOTY_CUDA_ELIMIT, "kv4_attend_dev: %d rows of %d heads", batch->rows, n_heads);
    CKR(kv4_ld("kv4_attend_dev", q_ld, (long long)n_heads * kv->geo.hd, &a.q_ld));
    if (!ctx_dev || !q_dev || !kv4_aligned(ctx_dev, 16) || !kv4_aligned(q_dev, 16))
        return moty_set_error(MOTY_CUDA_EARG, "kv4_attend_dev: ctx or q null or not 16-byte aligned");
    DevCtx *c = moty_ctx(kv->device);
    if (!c) return moty_set_error(MOTY_CUDA_EINIT, "device %d not initialised", kv->device);
    if (!a.b.nseq || !a.b.rows) return 0;
    MOTY_USE_DEVICE(kv->device);
    a.H = n_heads; a.G = n_heads / kv->geo.KV; a.q = q_dev; a.ctx = ctx_dev; a.max_rows = batch->max_rows; a.max_len = batch->max_len;
    a.window = window; a.scale = scale > 0.f ? scale : 1.f / sqrtf((float)kv->geo.hd); a.err = c->err_dev + 4;
    a.tc = kv4_prompt_tc_ready(kv->geo.hd, kv->device);
    const Kv4Plan p = kv4_plan(a, c->sms);
    const size_t sb = kv4_attend_scratch_bytes(a, p), nc = kv4_attend_counters(a, p) * 4;
    if (sb) CKR(moty_grow(c, &c->attn, sb));
    if (nc) CKR(moty_grow_zero(c, &c->kv4n, nc));
    return launch_kv4_attend(a, p, sb ? (float *)c->attn.p : nullptr, nc ? (int *)c->kv4n.p : nullptr, kv4_stream(c, stream));
}

extern "C" int moty_cuda_kv4_fork_dev(MotyCudaKv4 *kv, int n, const int *src_dev, const int *dst_dev, const int *fresh_dev, int nseq,
                                      int *len_dev, int *table_dev, int table_ld, void *stream) {
    if (!kv || n < 0 || nseq < 0 || table_ld <= 0 || !src_dev || !dst_dev || !fresh_dev || !len_dev || !table_dev)
        return moty_set_error(MOTY_CUDA_EARG, "kv4_fork_dev: null argument, or n=%d nseq=%d table_ld=%d", n, nseq, table_ld);
    DevCtx *c = moty_ctx(kv->device);
    if (!c) return moty_set_error(MOTY_CUDA_EINIT, "device %d not initialised", kv->device);
    MOTY_USE_DEVICE(kv->device);
    return launch_kv4_fork(kv->geo, kv->mem, n, src_dev, dst_dev, fresh_dev, nseq, len_dev, table_dev, table_ld, c->err_dev + 4, kv4_stream(c, stream));
}

extern "C" int moty_cuda_kv4_compact_dev(MotyCudaKv4 *kv, int n, const int *src_dev, const int *dst_dev, int64_t count, const int *table_dev,
                                         int *out_dev, void *stream) {
    if (!kv || n < 0 || count < 0 || (n && (!src_dev || !dst_dev)) || (count && (!table_dev || !out_dev)))
        return moty_set_error(MOTY_CUDA_EARG, "kv4_compact_dev: null argument, or n=%d count=%lld", n, (long long)count);
    if (n > kv->geo.pages) return moty_set_error(MOTY_CUDA_EARG, "kv4_compact_dev: %d moves in a pool of %d pages", n, kv->geo.pages);
    DevCtx *c = moty_ctx(kv->device);
    if (!c) return moty_set_error(MOTY_CUDA_EINIT, "device %d not initialised", kv->device);
    MOTY_USE_DEVICE(kv->device);
    return launch_kv4_compact(kv->geo, kv->mem, n, src_dev, dst_dev, count, table_dev, out_dev, c->err_dev + 4, c->sms, kv4_stream(c, stream));
}
