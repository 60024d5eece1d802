// Paged 8-bit key/value cache: addressing, checks and conversions shared by the files that write and read it
// (rns_kv_sm100.cu) and attend to it (rns_kv_attention_sm100.cu and its kernels, rns_kv_decode_sm100.cu and
// rns_kv_prompt_sm100.cu).
//
// A cache holds `pages` pages; page p of head h is `page_tokens` rows of `head_dim` bytes at
// ((p * kv_heads + h) * page_tokens) * head_dim of d_k and d_v, and its values stand for
// byte * scale[p * kv_heads + h].  Token t of sequence b lies in row t % page_tokens of page
// table[b * table_stride + t / page_tokens].
#pragma once

#include "rns_common.cuh"

#include <atomic>

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

// Streaming multiprocessors of the current device; the dynamic shared memory of a kernel, asked for once per
// device (bits of *done).
int sm_count(int* out);
int allow_smem(const void* kernel, int bytes, std::atomic<uint64_t>* done);

// rns_kv_prompt_sm100.cu: sequences with at least min_rows_tokens new tokens.
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

// First key that a query at `position` sees.  A position before the first token sees nothing; it counts as the
// first here, so that it less a window stays within 32 bits.
RNS_HD int kv_first_key(const KvQuery& a, int position) {
    return a.window > 0 ? (position > 0 ? position : 0) + 1 - a.window : 0;
}

#ifdef __CUDACC__
template <typename T> __device__ __forceinline__ float kv_to_float(T v);
template <> __device__ __forceinline__ float kv_to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float kv_to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float kv_to_float<float>(float v) { return v; }
// Two neighbouring elements of a 16-bit type in one word <-> floats.
template <typename T> __device__ __forceinline__ float2 kv_unpack(uint32_t w);
template <> __device__ __forceinline__ float2 kv_unpack<__half>(uint32_t w) {
    return make_float2(__half2float(__ushort_as_half((unsigned short)w)), __half2float(__ushort_as_half((unsigned short)(w >> 16))));
}
template <> __device__ __forceinline__ float2 kv_unpack<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <typename T> __device__ __forceinline__ uint32_t kv_pack(float x, float y);
template <> __device__ __forceinline__ uint32_t kv_pack<__half>(float x, float y) {
    return (uint32_t)__half_as_ushort(__float2half_rn(x)) | (uint32_t)__half_as_ushort(__float2half_rn(y)) << 16;
}
template <> __device__ __forceinline__ uint32_t kv_pack<__nv_bfloat16>(float x, float y) {
    return (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(x)) | (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(y)) << 16;
}

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
// Four cached bytes -> floats, exactly.  An integer byte becomes the low mantissa byte of 2^23 + 128 + value: the
// conversion unit has a quarter of the rate of these.
template <int FORMAT> __device__ __forceinline__ void kv_decode4(uint32_t w, float (&v)[4]) {
    if (FORMAT == RNS_KV_INT8) {
        const uint32_t u = w ^ 0x80808080u;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __fadd_rn(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7540u + i)), -8388736.0f);
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * i)), __NV_E4M3);
            const float2 f = __half22float2(__half2(h));
            v[2 * i] = f.x; v[2 * i + 1] = f.y;
        }
    }
}
// A page's value scale s as 2^exponent * weight, and 2^-exponent.  Attention keeps a row's softmax weights in
// units of 2^M, where M is a whole number near the largest (score + exponent) that the row has met:
//     w_j = 2^(t_j + exponent - M) * weight          what is rounded to fp16 and meets the bytes
//     l   = sum 2^(t_j + exponent - M) * 2^-exponent the softmax's sum, fp32
// so fp16's range lies where the row's own contributions are, whatever the scales of pages that it does not
// see or heed (a unit near the largest scale met lost the other pages: a scale 2^14 above theirs cost 5 % of
// an output, one 2^26 above all of it).  M - exponent is a difference of whole numbers, exact.  The exponent is
// kept within [-64, 126]: its powers of two are normal numbers and l does not overflow; smaller scales (zeros
// among them) have weights below one.  l loses terms only where scales within a row differ by more than 2^100.
// A scale that is not finite has weight NaN, which reaches the rows that see it.
struct KvValueScale {
    float exponent, weight, back;
};
__device__ __forceinline__ KvValueScale kv_value_scale(float s) {
    const bool finite = fabsf(s) <= 3.0e38f;
    const int e = finite ? max(63, min(253, (int)(__float_as_uint(s) >> 23 & 255u))) : 127;
    KvValueScale v;
    v.back = __uint_as_float((uint32_t)(254 - e) << 23);
    v.weight = finite ? s * v.back : __uint_as_float(0x7fc00000u);
    v.exponent = __uint_as_float(0x4B000000u + (uint32_t)e) - (8388608.0f + 127.0f);
    return v;
}
// x / scale on the grid, eight values -> bytes; inverse = 1 / scale.  The quotient is the correctly rounded
// one: the product with the inverse is off by at most two units in the last place, so only values that
// close to the middle between two grid points need the division.
template <int FORMAT> __device__ __forceinline__ uint2 kv_encode8(const float (&x)[8], float scale, float inverse) {
    uint32_t out[2];
    bool close = false;
    if (FORMAT == RNS_KV_INT8) {
        float far = 0.0f;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            uint32_t bits[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float y = __fmul_rn(x[4 * w + i], inverse), t = __fadd_rn(y, kMagic);   // |y| < 128: t's low byte is rint(y)
                far = fmaxf(far, fabsf(__fsub_rn(y, __fsub_rn(t, kMagic))));
                bits[i] = __float_as_uint(t);
            }
            out[w] = __byte_perm(__byte_perm(bits[0], bits[1], 0x0040), __byte_perm(bits[2], bits[3], 0x0040), 0x5410);
        }
        close = far > 0.4999f;
    } else {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            uint32_t lo = 0, hi = 0;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float a = __fmul_rn(x[4 * w + 2 * i], inverse), b = __fmul_rn(x[4 * w + 2 * i + 1], inverse);
                lo |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a * (1.0f - 0x1p-21f), b * (1.0f - 0x1p-21f)), __NV_SATFINITE, __NV_E4M3) << (16 * i);
                hi |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a * (1.0f + 0x1p-21f), b * (1.0f + 0x1p-21f)), __NV_SATFINITE, __NV_E4M3) << (16 * i);
            }
            close = close || lo != hi;
            out[w] = lo;
        }
    }
    if (close) {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            out[w] = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) out[w] |= (uint32_t)kv_encode<FORMAT>(__fdiv_rn(x[4 * w + i], scale)) << (8 * i);
        }
    }
    return make_uint2(out[0], out[1]);
}
#endif

}  // namespace rns
