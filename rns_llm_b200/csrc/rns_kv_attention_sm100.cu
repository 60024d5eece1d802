// Attention of new query tokens over the paged 8-bit cache.
//
// One pass over the keys a query sees, with the running maximum m and sum l of the softmax:
//     t_j = scale * s_k * (q . k_j) / ln 2,   m' = max(m, t),   l' = l 2^(m - m') + sum 2^(t_j - m')
//     o'  = o 2^(m - m') + sum 2^(t_j - m') s_v v_j
// and out = o / l, lse = (m + log2 l) ln 2.
//
// One warp per (query token, head); a lane scores one key of 32, then owns up to eight
// dimensions of the output.
#include "rns_kv.cuh"

#include <cmath>

namespace rns {

struct KvQuery {
    const void* q;
    int heads, group;
    int64_t tokens, q_token_stride, q_head_stride;
    const int32_t *lens, *starts;
    int max_new, causal, window;
    float scale_log2;              // softmax scale / ln 2
    void* out;
    int64_t out_token_stride, out_head_stride;
    float* lse;
};

constexpr int kWarps = 4;

template <typename T, int FORMAT>
__global__ void __launch_bounds__(kWarps * 32) kv_attention_rows_kernel(KvView c, KvQuery a) {
    __shared__ float q_rows[kWarps][256];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head = blockIdx.y;
    const int64_t token = (int64_t)blockIdx.x * kWarps + warp;
    if (token >= a.tokens) return;
    int b = -1;
    KvSpan s{};
    for (int i = 0; i < c.sequences; ++i) {
        const KvSpan t = kv_span(c, a.lens, a.starts, a.tokens, i);
        if (token >= t.begin && token < t.begin + t.count) { b = i; s = t; }
    }
    if (b < 0) return;
    const int position = s.length - s.count + (int)(token - s.begin);
    int last = a.causal ? position + 1 : s.length;
    int first = a.window > 0 ? max(0, position - a.window + 1) : 0;
    if (position < 0) last = 0;                                    // no place in the sequence
    const T* q = static_cast<const T*>(a.q) + token * a.q_token_stride + head * a.q_head_stride;
    for (int d = lane; d < c.head_dim; d += 32) q_rows[warp][d] = kv_to_float<T>(q[d]);
    __syncwarp();
    const int kv_head = head / a.group;
    float m = -INFINITY, l = 0.0f, o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = 0.0f;
    for (int base = first; base < last; base += 32) {
        const int key = base + lane;
        float t = -INFINITY, v_scale = 0.0f;
        int64_t row = -1;
        if (key < last) {
            const int page = kv_page(c, b, key >> c.page_shift);
            t = 0.0f;
            if (page >= 0) {
                const int64_t block = (int64_t)page * c.kv_heads + kv_head;
                row = block * c.page_tokens + (key & (c.page_tokens - 1));
                v_scale = c.scale[1][block];
                float dot = 0.0f;
                for (int d = 0; d < c.head_dim; ++d)
                    dot = fmaf(q_rows[warp][d], kv_decode<FORMAT>(c.data[0][row * c.head_dim + d]), dot);
                t = dot * c.scale[0][block] * a.scale_log2;
            }
        }
        float top = t;
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        const float m_new = fmaxf(m, top);
        const float keep = m == -INFINITY ? 0.0f : exp2f(m - m_new);
        const float p = key < last ? exp2f(t - m_new) : 0.0f;
        float sum = p;
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        l = l * keep + sum;
        m = m_new;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] *= keep;
        const float weight = p * v_scale;
        for (int j = 0; j < min(32, last - base); ++j) {
            const float w = __shfl_sync(0xffffffffu, weight, j);
            const int64_t r = __shfl_sync(0xffffffffu, row, j);
            if (r < 0) continue;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int d = lane + i * 32;
                if (d < c.head_dim) o[i] = fmaf(w, kv_decode<FORMAT>(c.data[1][r * c.head_dim + d]), o[i]);
            }
        }
    }
    T* out = static_cast<T*>(a.out) + token * a.out_token_stride + head * a.out_head_stride;
    const float inv = last > first ? 1.0f / l : 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int d = lane + i * 32;
        if (d < c.head_dim) out[d] = kv_from_float<T>(o[i] * inv);
    }
    if (a.lse != nullptr && lane == 0)
        a.lse[token * a.heads + head] = last > first ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
}

static int check_attention(const rns_kv_cache* cache, const rns_kv_attention_args* a, KvView* c) {
    if (int rc = make_kv_view(cache, c)) return rc;
    if (a == nullptr) return fail(RNS_ERR_INVALID_ARGUMENT, "args is NULL");
    if (a->type != RNS_F16 && a->type != RNS_BF16)
        return fail(RNS_ERR_UNSUPPORTED, "queries are F16 or BF16");
    if (a->heads < 1 || a->heads > 65535 || a->heads % c->kv_heads != 0)
        return fail(RNS_ERR_INVALID_ARGUMENT, "heads must be a multiple of kv_heads, at most 65535");
    if (a->tokens < 0 || a->tokens > INT32_MAX || a->max_new < 0)
        return fail(RNS_ERR_INVALID_ARGUMENT, "token counts must be in [0, 2^31)");
    if (a->window < 0 || (a->window > 0 && !a->causal))
        return fail(RNS_ERR_INVALID_ARGUMENT, "window must not be negative and needs causal");
    if (!(std::fabs(a->softmax_scale) <= 3.0e38f)) return fail(RNS_ERR_INVALID_ARGUMENT, "softmax_scale must be finite");
    if (a->tokens > 0 && c->sequences > 0 && (!a->d_q || !a->d_out || !a->d_seq_lens || !a->d_query_starts))
        return fail(RNS_ERR_INVALID_ARGUMENT, "a pointer is NULL");
    return RNS_OK;
}

}  // namespace rns

using namespace rns;

extern "C" int64_t rns_kv_attention_workspace(const rns_kv_cache* cache, const rns_kv_attention_args* args) {
    KvView c;
    if (int rc = check_attention(cache, args, &c)) return -rc;
    return 0;
}

extern "C" int rns_kv_attention(const rns_kv_cache* cache, const rns_kv_attention_args* a, rns_stream_t stream) {
    KvView c;
    if (int rc = check_attention(cache, a, &c)) return rc;
    if (c.sequences == 0 || a->tokens == 0) return RNS_OK;
    KvQuery p;
    p.q = a->d_q; p.heads = a->heads; p.group = a->heads / c.kv_heads;
    p.tokens = a->tokens; p.q_token_stride = a->q_token_stride; p.q_head_stride = a->q_head_stride;
    p.lens = a->d_seq_lens; p.starts = a->d_query_starts;
    p.max_new = a->max_new; p.causal = a->causal; p.window = a->window;
    p.scale_log2 = a->softmax_scale * 1.4426950408889634f;
    p.out = a->d_out; p.out_token_stride = a->out_token_stride; p.out_head_stride = a->out_head_stride;
    p.lse = a->d_lse;
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)((a->tokens + kWarps - 1) / kWarps), (unsigned)a->heads);
#define RNS_KV_ROWS(T, F) kv_attention_rows_kernel<T, F><<<grid, kWarps * 32, 0, st>>>(c, p)
    if (a->type == RNS_F16) {
        if (cache->format == RNS_KV_INT8) RNS_KV_ROWS(__half, RNS_KV_INT8);
        else RNS_KV_ROWS(__half, RNS_KV_E4M3);
    } else {
        if (cache->format == RNS_KV_INT8) RNS_KV_ROWS(__nv_bfloat16, RNS_KV_INT8);
        else RNS_KV_ROWS(__nv_bfloat16, RNS_KV_E4M3);
    }
#undef RNS_KV_ROWS
    RNS_CUDA_OK(cudaGetLastError());
    return RNS_OK;
}
