// Paged 8-bit key/value cache: addressing and checks shared by rns_kv_sm100.cu and
// rns_kv_attention_sm100.cu.
//
// A cache holds `pages` pages; page p of head h is `page_tokens` rows of `head_dim` bytes at
// ((p * kv_heads + h) * page_tokens) * head_dim of d_k and d_v, and its values stand for
// byte * scale[p * kv_heads + h].  Token t of sequence b lies in row t % page_tokens of page
// table[b * table_stride + t / page_tokens].
#pragma once

#include "rns_common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace rns {

// What the kernels read of rns_kv_cache, by value.
struct KvView {
    int8_t* data[2];               // keys, values
    float* scale[2];
    int64_t pages;
    int page_shift, page_tokens;
    int kv_heads, head_dim;
    const int32_t* table;
    int64_t table_stride;
    int table_pages, sequences;
    int32_t* status;
};

// The queries of one attention call.
struct KvQuery {
    const void* q;
    int type;                      // RNS_F16 or RNS_BF16
    int heads, group;              // group: query heads that share a head of the cache
    int64_t tokens, q_token_stride, q_head_stride;
    const int32_t *lens, *starts;
    int causal, window;
    float scale_log2;              // softmax scale / ln 2
    void* out;
    int64_t out_token_stride, out_head_stride;
    float* lse;
};

// Streaming multiprocessors of the current device.
int sm_count(int* out);

// rns_kv_prompt_sm100.cu: sequences with at least min_rows_tokens new tokens, heads of up to 128.
bool kv_prompt_supported(const KvView& c);
int64_t kv_prompt_workspace(const KvView& c);
int kv_prompt(const KvView& c, const KvQuery& a, int format, int min_rows_tokens, void* workspace, cudaStream_t st);

// rns_kv_decode_sm100.cu.  Serves the sequences with at most max_rows_tokens new tokens; max_new sizes the row tiles.
int64_t kv_decode_workspace(const KvView& c, const KvQuery& a, int max_new);
int kv_decode(const KvView& c, const KvQuery& a, int format, int max_new, int max_rows_tokens, void* workspace,
              cudaStream_t st);

// Checks everything the host can see; RNS_OK fills `view`.
int make_kv_view(const rns_kv_cache* cache, KvView* view);

constexpr float kKvEps = 1.1920928955078125e-07f;   // floor of a block's largest magnitude, as for weights

// The addressing compiles for the host as well (rns_host_kv_rows), so that CPU tests can run it on
// bad lengths, starts and pages.
RNS_HD void kv_flag(const KvView& c) {
    if (c.status != nullptr) *c.status = RNS_ERR_BAD_INDEX;
}

// New tokens of sequence b: rows [begin, begin + count) of the packed token axis, at positions
// [length - count, length).  Starts that do not ascend inside [0, tokens] or a length beyond the
// page table set the status word and leave an empty sequence.
struct KvSpan {
    int64_t begin;
    int count, length;
};
RNS_HD KvSpan kv_span(const KvView& c, const int32_t* lens, const int32_t* starts,
                                          int64_t tokens, int b) {
    KvSpan s;
    const int64_t first = starts[b], last = starts[b + 1];
    s.begin = first;
    s.count = (int)(last - first);
    s.length = lens[b];
    if (first < 0 || last < first || last > tokens || s.length < 0 ||
        (int64_t)s.length > (int64_t)c.table_pages * c.page_tokens) {
        kv_flag(c);
        s.begin = 0; s.count = 0; s.length = 0;
    }
    return s;
}
// Entry `nth` of sequence b's row of the page table, and the page it names: -1 (status word set) when the
// cache has no such page.
RNS_HD int32_t kv_entry(const KvView& c, int b, int nth) { return c.table[(int64_t)b * c.table_stride + nth]; }
RNS_HD int kv_named(const KvView& c, int32_t page) {
    if (page < 0 || (int64_t)page >= c.pages) {
        kv_flag(c);
        return -1;
    }
    return page;
}
RNS_HD int kv_page(const KvView& c, int b, int nth) { return kv_named(c, kv_entry(c, b, nth)); }

#ifdef __CUDACC__
template <typename T> __device__ __forceinline__ float kv_to_float(T v);
template <> __device__ __forceinline__ float kv_to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float kv_to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float kv_to_float<float>(float v) { return v; }
template <typename T> __device__ __forceinline__ T kv_from_float(float v);
template <> __device__ __forceinline__ __half kv_from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 kv_from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ float kv_from_float<float>(float v) { return v; }

// One cached byte <-> float.  Rounding to the grid is to nearest, ties to even, clamped.
template <int FORMAT> __device__ __forceinline__ float kv_decode(int8_t byte) {
    if (FORMAT == RNS_KV_INT8) return (float)byte;
    __nv_fp8_e4m3 v;
    v.__x = (__nv_fp8_storage_t)byte;
    return (float)v;
}
template <int FORMAT> __device__ __forceinline__ uint8_t kv_encode(float x) {
    if (FORMAT == RNS_KV_INT8) return (uint8_t)(int8_t)max(-127, min(127, __float2int_rn(x)));
    return (uint8_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}
#endif

}  // namespace rns
