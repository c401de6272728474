// kv4_pages.cu -- moves of whole pages of the paged 4-bit KV cache: forks (copy on write of the last partial page) and
// compaction.  A page is contiguous over its layers and heads, so both are copies of long runs of bytes; each does its
// table work in the same launch.  Bound by memory: a page of 28 layers, 8 KV heads, hd 128 is 2 MB; 180 of them moved 126 us
// (743 MB read and written, 5.9 TB/s), 48 forks with partial pages 29 us (the bytes alone 26.5 us at the copy rate), four
// forks 8 us (16 MB, 2.5 us at the copy rate: launch, table look-ups, and a CTA's eight copies one after the other, for a load
// is not moved over the store before it), five pages of 100 KB 3 us.  A page is cut into chunks of
// about 32 KB, a CTA each, so that a few pages fill the GPU.
#include "kv4.cuh"

namespace {

constexpr int PG_THREADS = 256;

__device__ __forceinline__ void kv4_copy_chunk(uint8_t *mem, size_t page_bytes, int src, int dst, int chunk, int nchunk) {
    const size_t n16 = page_bytes / 16, per = (n16 + nchunk - 1) / nchunk;
    const size_t lo = per * chunk, hi = lo + per < n16 ? lo + per : n16;
    const int4 *s = reinterpret_cast<const int4 *>(mem + (size_t)src * page_bytes);
    int4 *d = reinterpret_cast<int4 *>(mem + (size_t)dst * page_bytes);
    for (size_t i = lo + threadIdx.x; i < hi; i += PG_THREADS) d[i] = s[i];
}

// fork f: sequence dst[f] becomes a copy of sequence src[f].  Full pages are shared (their ids copied), a partial last
// page is copied to page fresh[f].
__global__ void __launch_bounds__(PG_THREADS) kv4_fork_kernel(Kv4Geom geo, uint8_t *mem, int n, const int *src, const int *dst, const int *fresh,
                                                              int nseq, int *len, int *table, int ld, int *err) {
    __shared__ int bad;
    const int f = blockIdx.x, tid = threadIdx.x;
    if (tid == 0) bad = 0;
    pdl_trigger();
    pdl_wait();
    __syncthreads();
    const int s = src[f], d = dst[f], to = fresh[f];
    // the partial last page of a source, -1: none (no fork writes a source's row or length: a target that is one is refused)
    auto last_page = [&](int r) {
        const int L = r >= 0 && r < nseq ? len[r] : 0;
        return L > 0 && L % KV4_PAGE && L / KV4_PAGE < ld ? table[(size_t)r * ld + L / KV4_PAGE] : -1;
    };
    const int from = last_page(s);
    // a target (row or page) that some fork reads, or another one writes too: refused, and reported
    if (s < 0 || s >= nseq || d < 0 || d >= nseq) bad = 1;
    else
        for (int i = tid; i < n; i += PG_THREADS)
            if (src[i] == d || (i != f && (dst[i] == d || (fresh[i] == to && to >= 0))) || (from >= 0 && to >= 0 && last_page(src[i]) == to)) bad = 1;
    __syncthreads();
    if (bad) { if (tid == 0) atomicExch(err, 1); return; }
    const int L = len[s], full = L / KV4_PAGE, tail = L % KV4_PAGE;
    if (L < 0 || (long long)L > (long long)ld * KV4_PAGE || (tail && (!kv4_page_ok(geo, from) || !kv4_page_ok(geo, to)))) {
        if (tid == 0) atomicExch(err, 1);
        return;
    }
    if (blockIdx.y == 0) {
        for (int i = tid; i < ld; i += PG_THREADS) table[(size_t)d * ld + i] = i < full ? table[(size_t)s * ld + i] : i == full && tail ? to : -1;
        if (tid == 0) len[d] = L;
    }
    if (tail) kv4_copy_chunk(mem, kv4_page_bytes(geo), from, to, blockIdx.y, gridDim.y);
}

// the index of `id` in the ascending list, or -1
__device__ __forceinline__ int kv4_find_id(const int *list, int n, int id) {
    int lo = 0, hi = n - 1;
    while (lo <= hi) {
        const int mid = (lo + hi) >> 1, x = list[mid];
        if (x == id) return mid;
        if (x < id) lo = mid + 1; else hi = mid - 1;
    }
    return -1;
}

// Whether move i may be made: ids in the pool, its place in both lists, and a target that is no source.
__device__ __forceinline__ bool kv4_move_ok(const Kv4Geom &geo, const int *src, const int *dst, int n, int i) {
    const int s = src[i], d = dst[i];
    return kv4_page_ok(geo, s) && kv4_page_ok(geo, d) && (i == 0 || (src[i - 1] < s && dst[i - 1] < d)) && kv4_find_id(src, n, d) < 0;
}

// CTAs 0 .. n * nchunk - 1 copy pages src[i] -> dst[i]; the others rename the table's entries.  Both lists must be
// strictly ascending and share no id, which makes every copy's target distinct from every page that is read; each CTA
// checks what it relies on (its neighbours in the lists, its target against the sources).  An entry keeps its id where the
// move is refused.
__global__ void __launch_bounds__(PG_THREADS) kv4_compact_kernel(Kv4Geom geo, uint8_t *mem, int n, const int *src, const int *dst, int nchunk,
                                                                 long long count, const int *table, int *out, int *err) {
    const int tid = threadIdx.x;
    pdl_trigger();
    pdl_wait();
    const long long ncopy = (long long)n * nchunk;
    if (blockIdx.x < ncopy) {
        const int i = blockIdx.x / nchunk, chunk = blockIdx.x - i * nchunk;
        if (!kv4_move_ok(geo, src, dst, n, i)) {
            if (tid == 0) atomicExch(err, 1);
            return;
        }
        kv4_copy_chunk(mem, kv4_page_bytes(geo), src[i], dst[i], chunk, nchunk);
        return;
    }
    for (long long i = (blockIdx.x - ncopy) * PG_THREADS + tid; i < count; i += (gridDim.x - ncopy) * PG_THREADS) {
        const int id = table[i], at = id < 0 ? -1 : kv4_find_id(src, n, id);
        out[i] = at >= 0 && kv4_move_ok(geo, src, dst, n, at) ? dst[at] : id;
    }
}

}  // namespace

int launch_kv4_fork(const Kv4Geom &geo, uint8_t *mem, int n, const int *src, const int *dst, const int *fresh, int nseq, int *len,
                    int *table, int ld, int *err, cudaStream_t st) {
    if (n <= 0) return 0;
    size_t nchunk = (kv4_page_bytes(geo) + 32767) / 32768;
    if (nchunk > 65535) nchunk = 65535;
    CK(moty_launch_pdl(kv4_fork_kernel, dim3(n, (unsigned)nchunk), dim3(PG_THREADS), (size_t)0, st, geo, mem, n, src, dst, fresh, nseq, len, table, ld, err));
    return 0;
}

int launch_kv4_compact(const Kv4Geom &geo, uint8_t *mem, int n, const int *src, const int *dst, long long count, const int *table,
                       int *out, int *err, int sms, cudaStream_t st) {
    if (n <= 0 && count <= 0) return 0;
    size_t nchunk = (kv4_page_bytes(geo) + 32767) / 32768;
    if ((long long)n * (long long)nchunk > 0x3fffffffLL) nchunk = 1;
    long long names = (count + PG_THREADS - 1) / PG_THREADS;
    if (names > 2 * sms) names = 2 * sms;
    CK(moty_launch_pdl(kv4_compact_kernel, dim3((unsigned)(n * (long long)nchunk + names)), dim3(PG_THREADS), (size_t)0, st, geo, mem, n, src, dst,
                       (int)nchunk, count, table, out, err));
    return 0;
}
