// kv4.cuh -- shared pieces of the paged 4-bit KV cache (kv4_store.cu, kv4_attend.cu, kv4_pages.cu, kv4_api.cu).
#pragma once
#include "kernels.cuh"
#include "kv4_index.h"

struct Kv4Rope {                         // what is done to q and k before they are used (attn_prep_kernel's statements)
    int rot, gemma;
    float theta, eps;
    const float *qn, *kn, *vn;           // per head dimension, device, or null
};

struct Kv4Attend {
    Kv4Geom geo; Kv4Batch b;
    const uint8_t *mem;
    int layer, H, G;                     // G = H / KV query heads per KV head
    const float *q; long long q_ld; float *ctx;
    int max_rows, max_len, window;
    float scale;
    bool tc;                             // the tensor-memory prompt kernel may run (kv4_prompt_tc_ready)
    int *err;                            // device word set when the batch arrays or the table are out of range
};

// ---- kv4_store.cu ----
int launch_kv4_append(const Kv4Geom &geo, uint8_t *mem, int layer, const float *k, const float *v, long long ld, const Kv4Batch &b,
                      int *err, cudaStream_t st);
int launch_kv4_append_rope(const Kv4Geom &geo, uint8_t *mem, int layer, int H, float *q, long long q_ld, float *k, const float *v, long long ld,
                           const Kv4Rope &rope, const Kv4Batch &b, int *err, cudaStream_t st);
int launch_kv4_fetch(const Kv4Geom &geo, const uint8_t *mem, int layer, float *k, float *v, const Kv4Batch &b, int *err, cudaStream_t st);
// ---- kv4_attend.cu ----
// how an attention call is cut.  decode: the kernel for few rows; tc: the tensor-memory prompt kernel; a CTA takes `cols`
// (row, query head) pairs of one KV head of one sequence, ntile such tiles a sequence at most, and one of nsplit spans of
// `span` positions
struct Kv4Plan { bool decode, tc; int cols, ntile, nsplit, span; };
Kv4Plan kv4_plan(const Kv4Attend &a, int sms);
// kv4_prompt_tc.cu: whether that kernel was built with the registers that its roles share out (head width hd, the current device)
bool kv4_prompt_tc_ready(int hd, int device);
size_t kv4_attend_scratch_bytes(const Kv4Attend &a, const Kv4Plan &p);
size_t kv4_attend_counters(const Kv4Attend &a, const Kv4Plan &p);
int launch_kv4_attend(const Kv4Attend &a, const Kv4Plan &p, float *part, int *count, cudaStream_t st);
// ---- kv4_pages.cu ----
int launch_kv4_fork(const Kv4Geom &geo, uint8_t *mem, int n, const int *src, const int *dst, const int *fresh, int nseq, int *len,
                    int *table, int ld, int *err, cudaStream_t st);
int launch_kv4_compact(const Kv4Geom &geo, uint8_t *mem, int n, const int *src, const int *dst, long long count, const int *table,
                       int *out, int *err, int sms, cudaStream_t st);
