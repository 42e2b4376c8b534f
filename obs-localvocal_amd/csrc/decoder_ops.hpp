// decoder_ops.hpp — the decoder operators on device memory (paged key / value cache, attention over it, sampler): what
// kv_cache.hip, kv_attend.hip and sampler.hip share.  Argument structures: include/mi355_whisper.h.
#pragma once

#include "../../include/mi355_whisper.h"
#include "common.hpp"

namespace mw {

void launch_kv_write(const mw_kv_cache &c, const mw_kv_batch &b, int dtype, const void *k, const void *v, int64_t row_stride,
                     int64_t head_stride, hipStream_t st);
void launch_kv_read(const mw_kv_cache &c, const mw_kv_batch &b, int dtype, void *k, void *v, int64_t row_stride, int64_t head_stride,
                    hipStream_t st);
struct KvAttendArgs {
    int n_heads = 0;
    const void *q = nullptr;
    int64_t q_row = 0, q_head = 0;
    void *out = nullptr;
    int64_t o_row = 0, o_head = 0;
    float scale = 0.0f;
    int window = 0, sinks = 0;
    void *ws = nullptr;
    size_t ws_bytes = 0;
};
size_t kv_attend_workspace(int n_cus, const mw_kv_cache &c, const mw_kv_batch &b, int n_heads, int window, int sinks);
void launch_kv_attend(int n_cus, const mw_kv_cache &c, const mw_kv_batch &b, const KvAttendArgs &a, hipStream_t st);
struct SampleArgs {
    const void *logits = nullptr;
    int dtype = 0, n_rows = 0, n_vocab = 0;
    int64_t row_stride = 0;
    const float *temperature = nullptr;
    const int32_t *top_k = nullptr;
    const float *top_p = nullptr, *min_p = nullptr;
    const double *u = nullptr;
    int32_t *ids = nullptr;
    float *logprobs = nullptr;
};
void launch_sample(const SampleArgs &a, hipStream_t st);

// the checks of the arguments, on the host alone (throw with the reason)
void check_kv(const mw_kv_cache &c, const mw_kv_batch &b);
void check_kv_rows(const mw_kv_cache &c, const mw_kv_batch &b, int dtype, const void *k, const void *v, int64_t row_stride, int64_t head_stride,
                   bool write);
void check_kv_attend(const mw_kv_cache &c, const mw_kv_batch &b, const KvAttendArgs &a);
void check_sample(const SampleArgs &a);

#ifdef __HIPCC__
// ---- device view -----------------------------------------------------------------------------------------------------
// Every index that is read from device memory (cu_rows, kv_len, block_table) is checked against the bounds given by the host
// before it addresses anything: a table with wrong contents gives wrong rows, never an access outside the buffers.
struct KvView {
    char *k, *v;
    float *ks, *vs;
    int n_pages, shift, mask, n_kv_heads;
    int64_t page_stride, head_stride, row_stride, s_page, s_head, s_row;
    const int *cu, *kv_len, *table;
    int64_t table_stride;
    int table_cols, n_seqs, n_rows;
};
inline KvView make_view(const mw_kv_cache &c, const mw_kv_batch &b) {
    int shift = 0;
    while ((1 << shift) < c.page_size) ++shift;
    return KvView{(char *)c.k, (char *)c.v, c.k_scale, c.v_scale, c.n_pages, shift, c.page_size - 1, c.n_kv_heads, c.page_stride, c.head_stride,
                  c.row_stride, c.scale_page_stride, c.scale_head_stride, c.scale_row_stride, b.cu_rows, b.kv_len, b.block_table, b.table_stride,
                  b.table_cols, b.n_seqs, b.n_rows};
}
// first row of sequence b, inside 0 .. n_rows whatever cu holds
__device__ __forceinline__ int kv_cu(const KvView &V, int b) { return min(max(V.cu[b], 0), V.n_rows); }
// the sequence that owns row t (the last one that starts at or before it), or -1
__device__ __forceinline__ int kv_seq_of_row(const KvView &V, int t) {
    int lo = 0, hi = V.n_seqs;  // cu[lo] <= t < cu[hi], once both are checked
    if (V.n_seqs <= 0 || t < V.cu[0] || t >= V.cu[V.n_seqs]) return -1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (V.cu[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}
// page of position p (>= 0) of sequence b, or -1
__device__ __forceinline__ int kv_page(const KvView &V, int b, int64_t p) {
    const int64_t col = p >> V.shift;
    if (col >= V.table_cols) return -1;
    const int page = V.table[b * V.table_stride + col];
    return (unsigned)page < (unsigned)V.n_pages ? page : -1;
}
#endif

}  // namespace mw
