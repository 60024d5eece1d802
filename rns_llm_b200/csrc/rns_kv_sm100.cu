// Paged 8-bit key/value cache: quantise as it is written, read it back.
//
// A block of the cache is one page of one head: `page_tokens` tokens share a scale.  Writing
// computes, per touched block and in fp32 with IEEE division,
//     a     = max |x| over the block's new tokens
//     s     = max(a, eps) / Q                        Q = 127 (int8) or 448 (e4m3)
//     s     = max(s, s_old)                          where the block already holds tokens
//     q_old = round(q_old * (s_old / s))             where the scale grew
//     q     = round(x / s)                           ties to even, clamped
// A block has one owner (a CTA), so nothing is exchanged between CTAs and the result does not
// depend on any order.
//
// Both directions are bound by memory: writing 4096 tokens x 32 heads x 128 (fp16 to int8) takes 26 us, 0.59 of
// the copy rate (a CTA's load, reduction and store follow one another, so the number of CTAs in flight counts:
// 55 us with the block held as floats); reading 65537 x 8 x 128 to bf16 78 us, 0.79 of it.
#include "rns_kv.cuh"

#include <algorithm>

namespace rns {

int make_kv_view(const rns_kv_cache* c, KvView* v) {
    if (c == nullptr) return fail(RNS_ERR_INVALID_ARGUMENT, "cache is NULL");
    if (!c->d_k || !c->d_v || !c->d_k_scale || !c->d_v_scale)
        return fail(RNS_ERR_INVALID_ARGUMENT, "the cache has a NULL pointer");
    if ((reinterpret_cast<uintptr_t>(c->d_k) | reinterpret_cast<uintptr_t>(c->d_v)) & 15)
        return fail(RNS_ERR_INVALID_ARGUMENT, "cache pages must be 16-byte aligned");
    if (c->format != RNS_KV_INT8 && c->format != RNS_KV_E4M3)
        return fail(RNS_ERR_INVALID_ARGUMENT, "unknown cache format %d", (int)c->format);
    if (c->page_tokens != 16 && c->page_tokens != 32 && c->page_tokens != 64 && c->page_tokens != 128)
        return fail(RNS_ERR_UNSUPPORTED, "page_tokens must be 16, 32, 64 or 128");
    if (c->head_dim < 16 || c->head_dim > 256 || c->head_dim % 16 != 0)
        return fail(RNS_ERR_UNSUPPORTED, "head_dim must be a multiple of 16 in [16, 256]");
    if (c->kv_heads < 1 || c->kv_heads > 4096) return fail(RNS_ERR_INVALID_ARGUMENT, "kv_heads must be in [1, 4096]");
    if (c->pages < 1 || c->pages > INT32_MAX) return fail(RNS_ERR_INVALID_ARGUMENT, "pages must be in [1, 2^31)");
    if (c->sequences < 0 || c->sequences > 65535) return fail(RNS_ERR_INVALID_ARGUMENT, "sequences must be in [0, 65535]");
    if (c->table_pages < 0 || c->table_stride < c->table_pages)
        return fail(RNS_ERR_INVALID_ARGUMENT, "the page table's row stride is below its width");
    if ((int64_t)c->table_pages * c->page_tokens > INT32_MAX - 4096)
        return fail(RNS_ERR_UNSUPPORTED, "a sequence holds fewer than 2^31 - 4096 tokens");
    if (c->sequences > 0 && c->table_pages > 0 && !c->d_page_table)
        return fail(RNS_ERR_INVALID_ARGUMENT, "d_page_table is NULL");
    v->data[0] = c->d_k; v->data[1] = c->d_v;
    v->scale[0] = c->d_k_scale; v->scale[1] = c->d_v_scale;
    v->pages = c->pages;
    v->page_tokens = c->page_tokens;
    v->page_shift = c->page_tokens == 16 ? 4 : c->page_tokens == 32 ? 5 : c->page_tokens == 64 ? 6 : 7;
    v->kv_heads = c->kv_heads; v->head_dim = c->head_dim;
    v->table = c->d_page_table; v->table_stride = c->table_stride;
    v->table_pages = c->table_pages; v->sequences = c->sequences;
    v->status = c->d_status;
    return RNS_OK;
}

// ---------------------------------------------------------------------------
// write
// ---------------------------------------------------------------------------
struct KvSource {
    const void* x[2];
    int64_t token_stride[2], head_stride[2];      // elements
};

// 8 consecutive elements as they lie in memory; VECTOR: 16-byte loads (addresses are 16-byte aligned).  A
// thread holds its share of a block in this form, half the registers of floats.  `most` gathers the largest
// magnitude as bits of the type (they order like the numbers, with infinities and NaN on top).
template <typename T> struct Raw8 {
    uint32_t w[4];
    __device__ __forceinline__ void clear() { w[0] = w[1] = w[2] = w[3] = 0; }
    template <bool VECTOR> __device__ __forceinline__ void load(const T* p) {
        if (VECTOR) {
            const uint4 a = *reinterpret_cast<const uint4*>(p);
            w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
        } else {
            const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = h[2 * i] | (uint32_t)h[2 * i + 1] << 16;
        }
    }
    __device__ __forceinline__ void most(uint32_t& m) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
    }
    // the gathered magnitudes -> bits of the largest as a float
    static __device__ __forceinline__ uint32_t float_bits(uint32_t m) {
        return __float_as_uint(kv_unpack<T>(max(m & 0xffffu, m >> 16)).x);
    }
    __device__ __forceinline__ void expand(float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = kv_unpack<T>(w[i]);
            v[2 * i] = f.x; v[2 * i + 1] = f.y;
        }
    }
};
template <> struct Raw8<float> {
    float w[8];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = 0.0f;
    }
    template <bool VECTOR> __device__ __forceinline__ void load(const float* p) {
        if (VECTOR) {
            const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
            w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = p[i];
        }
    }
    __device__ __forceinline__ void most(uint32_t& m) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(w[i]) & 0x7fffffffu);
    }
    static __device__ __forceinline__ uint32_t float_bits(uint32_t m) { return m; }
    __device__ __forceinline__ void expand(float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = w[i];
    }
};
// 16 floats to 16 consecutive elements at a 16-byte boundary.
template <typename T> __device__ __forceinline__ void store16(T* p, const float (&v)[16]) {
    uint4* o = reinterpret_cast<uint4*>(p);
#pragma unroll
    for (int i = 0; i < 2; ++i)
        o[i] = make_uint4(kv_pack<T>(v[8 * i], v[8 * i + 1]), kv_pack<T>(v[8 * i + 2], v[8 * i + 3]),
                          kv_pack<T>(v[8 * i + 4], v[8 * i + 5]), kv_pack<T>(v[8 * i + 6], v[8 * i + 7]));
}
template <> __device__ __forceinline__ void store16<float>(float* p, const float (&v)[16]) {
    float4* o = reinterpret_cast<float4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
}

constexpr int kWriteVectors = 8;                  // groups of 8 elements a thread holds

// (registers for 1024 threads an SM where the block is held in 16-bit words)
template <typename T, int FORMAT, bool VECTOR, int THREADS>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 2 && VECTOR ? 1024 / THREADS : 1) kv_write_kernel(KvView c, KvSource src, const int32_t* lens,
                                                           const int32_t* starts, int64_t tokens, int max_new) {
    const int b = blockIdx.z, head = blockIdx.y >> 1, which = blockIdx.y & 1, t = threadIdx.x;
    const KvSpan s = kv_span(c, lens, starts, tokens, b);
    if (s.count > max_new) { kv_flag(c); return; }
    const int from = max(s.length - s.count, 0);                  // tokens before position 0 have no place
    if (s.length <= from) return;
    const int nth = (from >> c.page_shift) + blockIdx.x;
    if (nth > (s.length - 1) >> c.page_shift) return;              // (page numbers: a position there may pass 2^31)
    const int page_from = nth << c.page_shift;
    const int32_t named = kv_entry(c, b, nth);                     // looked at when the new tokens are on their way
    const int row0 = max(from - page_from, 0), row1 = min(s.length - page_from, c.page_tokens);
    const int groups = c.head_dim >> 3;                            // groups of 8 elements in a row
    // (selects, not indices: an indexed parameter is copied to local memory first)
    const int64_t token_stride = which ? src.token_stride[1] : src.token_stride[0];
    // element 0 of the block's row 0 (which may lie before the first new token: never read there)
    const T* x = static_cast<const T*>(which ? src.x[1] : src.x[0]) + head * (which ? src.head_stride[1] : src.head_stride[0]) +
                 (s.begin + page_from - (s.length - s.count)) * token_stride;

    Raw8<T> v[kWriteVectors];
    uint32_t most = 0;
    const int first = row0 * groups, last = row1 * groups;
#pragma unroll
    for (int i = 0; i < kWriteVectors; ++i) {
        const int g = first + t + i * THREADS;
        v[i].clear();
        if (g < last) {
            const int row = g / groups;
            v[i].template load<VECTOR>(x + row * token_stride + (g - row * groups) * 8);
        }
    }
#pragma unroll
    for (int i = 0; i < kWriteVectors; ++i) v[i].most(most);
    uint32_t top = __reduce_max_sync(0xffffffffu, Raw8<T>::float_bits(most));
    const int page = kv_named(c, named);
    if (page < 0) return;                                          // the whole CTA's page
    const int64_t block = (int64_t)page * c.kv_heads + head;
    int8_t* data = (which ? c.data[1] : c.data[0]) + block * c.page_tokens * c.head_dim;
    float* scale = (which ? c.scale[1] : c.scale[0]) + block;
    __shared__ uint32_t warp_top[THREADS / 32];
    if ((t & 31) == 0) warp_top[t >> 5] = top;
    const float old_scale = row0 > 0 ? *scale : 0.0f;
    __syncthreads();                                               // also: every thread has read the old scale
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) top = max(top, warp_top[w]);
    // Bit patterns of magnitudes order like the numbers, with infinities and NaN on top: a block
    // that was given one gets the scale NaN, so that it never reads back as something else, and bytes of zero:
    // attention multiplies the bytes that a row does not see by zero, which removes no NaN.
    float s_new = __fdiv_rn(fmaxf(__uint_as_float(top), kKvEps), FORMAT == RNS_KV_INT8 ? 127.0f : 448.0f);
    if (top >= 0x7f800000u || old_scale != old_scale) s_new = __uint_as_float(0x7fc00000u);
    else s_new = fmaxf(s_new, old_scale);
    if (t == 0) *scale = s_new;
    if (s_new != s_new) {
        for (int g = t; g < last; g += THREADS) *reinterpret_cast<uint2*>(data + (int64_t)g * 8) = make_uint2(0, 0);
        return;
    }
    if (row0 > 0 && s_new != old_scale) {                          // the scale grew: the tokens that stay follow
        const float ratio = __fdiv_rn(old_scale, s_new);
        uint32_t* words = reinterpret_cast<uint32_t*>(data);
        for (int g = t; g < row0 * groups * 2; g += THREADS) {
            const uint32_t w = words[g];
            uint32_t r = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                r |= (uint32_t)kv_encode<FORMAT>(__fmul_rn(kv_decode<FORMAT>((int8_t)(w >> (8 * e))), ratio)) << (8 * e);
            words[g] = r;
        }
    }
    const float inverse = __fdiv_rn(1.0f, s_new);
#pragma unroll
    for (int i = 0; i < kWriteVectors; ++i) {
        const int g = first + t + i * THREADS;
        if (g < last) {
            float f[8];
            v[i].expand(f);
            *reinterpret_cast<uint2*>(data + (int64_t)g * 8) = kv_encode8<FORMAT>(f, s_new, inverse);
        }
    }
}

template <typename T, int FORMAT>
static int launch_write(const KvView& c, const KvSource& src, const int32_t* lens, const int32_t* starts,
                        int64_t tokens, int max_new, bool vector, cudaStream_t st) {
    const dim3 grid((unsigned)(((int64_t)max_new + c.page_tokens - 2) / c.page_tokens + 1), (unsigned)(2 * c.kv_heads),
                    (unsigned)c.sequences);
    // A CTA holds its block in registers, eight groups of eight elements a thread: the fewest threads that can,
    // so that an SM has many blocks in flight (pages of 32 x 128, bf16 to e4m3: 43 us with 128 threads, 36 with 64).
    const int groups = c.page_tokens * c.head_dim / 8;
#define RNS_KV_WRITE_LAUNCH(V, N) kv_write_kernel<T, FORMAT, V, N><<<grid, N, 0, st>>>(c, src, lens, starts, tokens, max_new)
    if (!vector) RNS_KV_WRITE_LAUNCH(false, 512);
    else if (groups <= 64 * kWriteVectors) RNS_KV_WRITE_LAUNCH(true, 64);
    else if (groups <= 128 * kWriteVectors) RNS_KV_WRITE_LAUNCH(true, 128);
    else RNS_KV_WRITE_LAUNCH(true, 512);
#undef RNS_KV_WRITE_LAUNCH
    RNS_CUDA_OK(cudaGetLastError());
    return RNS_OK;
}

// ---------------------------------------------------------------------------
// read
// ---------------------------------------------------------------------------
// 16 bytes each: 8 KB of the cache per CTA.  8 x 640 tokens of 12 heads / 65537 of 8 take 8.3 / 78 us; with 256
// threads 10.1 / 80, with 8 groups of those a thread 14.4 / 104, with 2 of 128 8.3 / 82.
constexpr int kReadThreads = 128, kReadVectors = 4;

template <typename T, int FORMAT>
__global__ void __launch_bounds__(kReadThreads) kv_read_kernel(KvView c, const int32_t* first, const int32_t* row_starts,
                                                               int64_t rows, int max_rows, T* out_k, T* out_v,
                                                               int chunk_rows) {
    const int b = blockIdx.z, head = blockIdx.y >> 1, which = blockIdx.y & 1;
    const int64_t begin = row_starts[b], end = row_starts[b + 1];
    const int position = first[b];
    if (begin < 0 || end < begin || end > rows || position < 0 || end - begin > max_rows ||
        position + (end - begin) > (int64_t)c.table_pages * c.page_tokens) {
        kv_flag(c);
        return;
    }
    const int count = (int)(end - begin);
    const int at = blockIdx.x * chunk_rows;
    if (at >= count) return;
    const int chunks = c.head_dim >> 4, total = min(chunk_rows, count - at) * chunks;
    T* out = (which ? out_v : out_k) + ((begin + at) * c.kv_heads + head) * c.head_dim;
    // pages first, then bytes and scales, then the arithmetic: what is independent is in flight together
    int32_t named[kReadVectors];
    uint4 q[kReadVectors];
    float s[kReadVectors];
#pragma unroll
    for (int i = 0; i < kReadVectors; ++i) {
        const int g = threadIdx.x + i * kReadThreads;
        named[i] = g < total ? kv_entry(c, b, (position + at + g / chunks) >> c.page_shift) : 0;
    }
#pragma unroll
    for (int i = 0; i < kReadVectors; ++i) {
        const int g = threadIdx.x + i * kReadThreads;
        q[i] = make_uint4(0, 0, 0, 0);
        s[i] = 0.0f;
        if (g >= total) continue;
        const int page = kv_named(c, named[i]);
        if (page >= 0) {
            const int row = g / chunks, token = position + at + row;
            const int64_t block = (int64_t)page * c.kv_heads + head;
            q[i] = *reinterpret_cast<const uint4*>(
                (which ? c.data[1] : c.data[0]) + (block * c.page_tokens + (token & (c.page_tokens - 1))) * c.head_dim + (g - row * chunks) * 16);
            s[i] = (which ? c.scale[1] : c.scale[0])[block];
        }
    }
#pragma unroll
    for (int i = 0; i < kReadVectors; ++i) {
        const int g = threadIdx.x + i * kReadThreads;
        if (g >= total) continue;
        const int row = g / chunks, col = g - row * chunks;
        float v[16];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float f[4];
            kv_decode4<FORMAT>(e == 0 ? q[i].x : e == 1 ? q[i].y : e == 2 ? q[i].z : q[i].w, f);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[4 * e + k] = __fmul_rn(f[k], s[i]);
        }
        store16<T>(out + (int64_t)row * c.kv_heads * c.head_dim + col * 16, v);
    }
}

template <typename T, int FORMAT>
static int launch_read(const KvView& c, const int32_t* first, const int32_t* row_starts, int64_t rows, int max_rows,
                       void* k, void* v, cudaStream_t st) {
    const int chunk_rows = kReadThreads * kReadVectors * 16 / c.head_dim;
    const dim3 grid((unsigned)std::max<int64_t>(1, ((int64_t)max_rows + chunk_rows - 1) / chunk_rows), (unsigned)(2 * c.kv_heads), (unsigned)c.sequences);
    kv_read_kernel<T, FORMAT><<<grid, kReadThreads, 0, st>>>(c, first, row_starts, rows, max_rows, static_cast<T*>(k),
                                                             static_cast<T*>(v), chunk_rows);
    RNS_CUDA_OK(cudaGetLastError());
    return RNS_OK;
}

}  // namespace rns

using namespace rns;

extern "C" int rns_host_kv_rows(const rns_kv_cache* cache, const int32_t* seq_lens, const int32_t* query_starts,
                                int64_t tokens, int64_t* row_offsets) {
    KvView c;
    if (int rc = make_kv_view(cache, &c)) return rc;
    if (tokens < 0 || !seq_lens || !query_starts || !row_offsets) return fail(RNS_ERR_INVALID_ARGUMENT, "a pointer is NULL");
    for (int64_t t = 0; t < tokens; ++t) row_offsets[t] = -1;
    for (int b = 0; b < c.sequences; ++b) {
        const KvSpan s = kv_span(c, seq_lens, query_starts, tokens, b);
        for (int i = 0; i < s.count; ++i) {
            const int position = s.length - s.count + i;
            const int page = position < 0 ? -1 : kv_page(c, b, position >> c.page_shift);
            if (page < 0) continue;
            row_offsets[s.begin + i] = ((int64_t)page * c.kv_heads * c.page_tokens + (position & (c.page_tokens - 1))) * c.head_dim;
        }
    }
    return RNS_OK;
}

extern "C" int rns_kv_write(const rns_kv_cache* cache, const void* d_k_new, const void* d_v_new, rns_float_type type,
                            int64_t tokens, int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride,
                            int64_t v_head_stride, const int32_t* d_seq_lens, const int32_t* d_query_starts,
                            int max_new, rns_stream_t stream) {
    KvView c;
    if (int rc = make_kv_view(cache, &c)) return rc;
    if (tokens < 0 || tokens > INT32_MAX || max_new < 0) return fail(RNS_ERR_INVALID_ARGUMENT, "token counts must be in [0, 2^31)");
    if (type != RNS_F16 && type != RNS_BF16 && type != RNS_F32) return fail(RNS_ERR_INVALID_ARGUMENT, "unknown float type %d", (int)type);
    if (c.sequences == 0 || tokens == 0) return RNS_OK;              // (a bound of zero: what exceeds it is flagged)
    if (!d_k_new || !d_v_new || !d_seq_lens || !d_query_starts) return fail(RNS_ERR_INVALID_ARGUMENT, "a pointer is NULL");
    if (max_new > tokens) max_new = (int)tokens;
    const KvSource src = {{d_k_new, d_v_new}, {k_token_stride, v_token_stride}, {k_head_stride, v_head_stride}};
    const int size = type == RNS_F32 ? 4 : 2;
    bool vector = true;
    for (int i = 0; i < 2; ++i)
        vector = vector && (reinterpret_cast<uintptr_t>(src.x[i]) & 15) == 0 && src.token_stride[i] * size % 16 == 0 &&
                 src.head_stride[i] * size % 16 == 0;
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
#define RNS_KV_WRITE(T)                                                                                           \
    (cache->format == RNS_KV_INT8                                                                                 \
         ? launch_write<T, RNS_KV_INT8>(c, src, d_seq_lens, d_query_starts, tokens, max_new, vector, st)          \
         : launch_write<T, RNS_KV_E4M3>(c, src, d_seq_lens, d_query_starts, tokens, max_new, vector, st))
    if (type == RNS_F16) return RNS_KV_WRITE(__half);
    if (type == RNS_BF16) return RNS_KV_WRITE(__nv_bfloat16);
    return RNS_KV_WRITE(float);
#undef RNS_KV_WRITE
}

extern "C" int rns_kv_read(const rns_kv_cache* cache, const int32_t* d_first, const int32_t* d_row_starts, int64_t rows,
                           int max_rows, void* d_k_out, void* d_v_out, rns_float_type type, rns_stream_t stream) {
    KvView c;
    if (int rc = make_kv_view(cache, &c)) return rc;
    if (rows < 0 || rows > INT32_MAX || max_rows < 0) return fail(RNS_ERR_INVALID_ARGUMENT, "row counts must be in [0, 2^31)");
    if (type != RNS_F16 && type != RNS_BF16 && type != RNS_F32) return fail(RNS_ERR_INVALID_ARGUMENT, "unknown float type %d", (int)type);
    if (c.sequences == 0 || rows == 0) return RNS_OK;
    if (!d_first || !d_row_starts || !d_k_out || !d_v_out) return fail(RNS_ERR_INVALID_ARGUMENT, "a pointer is NULL");
    if ((reinterpret_cast<uintptr_t>(d_k_out) | reinterpret_cast<uintptr_t>(d_v_out)) & 15)
        return fail(RNS_ERR_INVALID_ARGUMENT, "outputs must be 16-byte aligned");
    if (max_rows > rows) max_rows = (int)rows;
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
#define RNS_KV_READ(T)                                                                                               \
    (cache->format == RNS_KV_INT8 ? launch_read<T, RNS_KV_INT8>(c, d_first, d_row_starts, rows, max_rows, d_k_out, d_v_out, st) \
                                  : launch_read<T, RNS_KV_E4M3>(c, d_first, d_row_starts, rows, max_rows, d_k_out, d_v_out, st))
    if (type == RNS_F16) return RNS_KV_READ(__half);
    if (type == RNS_BF16) return RNS_KV_READ(__nv_bfloat16);
    return RNS_KV_READ(float);
#undef RNS_KV_READ
}
