// Attention of new query tokens over the paged 8-bit cache: argument checks and the choice of kernel.
//
// One pass over the keys a query sees, with the running maximum m and sum l of the softmax:
//     t_j = scale * s_k * (q . k_j) / ln 2,   m' = max(m, t),   l' = l 2^(m - m') + sum 2^(t_j - m')
//     o'  = o 2^(m - m') + sum 2^(t_j - m') s_v v_j
// and out = o / l, lse = (m + log2 l) ln 2.  The kernels take m near the largest t + log2 s_v, so that o's weights
// with their scales stay in fp16's range (kv_value_scale); any m gives the same out and lse.
#include "rns_kv.cuh"

#include <cmath>

namespace rns {

static int check_attention(const rns_kv_cache* cache, const rns_kv_attention_args* a, KvView* c, KvQuery* p) {
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
    if (!(std::fabs(a->softmax_scale) <= 2.0e38f)) return fail(RNS_ERR_INVALID_ARGUMENT, "softmax_scale must be finite");
    if (a->tokens > 0 && c->sequences > 0 && (!a->d_q || !a->d_out || !a->d_seq_lens || !a->d_query_starts))
        return fail(RNS_ERR_INVALID_ARGUMENT, "a pointer is NULL");
    memset(p, 0, sizeof(*p));
    p->q = a->d_q; p->type = a->type; p->heads = a->heads; p->group = a->heads / c->kv_heads;
    p->tokens = a->tokens; p->q_token_stride = a->q_token_stride; p->q_head_stride = a->q_head_stride;
    p->lens = a->d_seq_lens; p->starts = a->d_query_starts;
    // a window as long as the longest sequence there can be hides nothing
    p->causal = a->causal != 0; p->window = a->window >= (int64_t)c->table_pages * c->page_tokens ? 0 : a->window;
    p->scale_log2 = a->softmax_scale * 1.4426950408889634f;
    p->out = a->d_out; p->out_token_stride = a->out_token_stride; p->out_head_stride = a->out_head_stride;
    p->lse = a->d_lse;
    return RNS_OK;
}

// Which kernel serves which sequences: tiles of the rows kernel hold up to 32 query rows (new tokens x
// heads that share one of the cache), those of the prompt kernel 256 (128 of heads above 128).  Beyond 32 rows
// the rows kernel reads a sequence's keys once for every tile (8 prompts of 512: 182 us there, 39 us in the
// prompt kernel; 48 rows of heads of 256, four sequences of 8000 tokens: 83 and 70 us).
struct Routing {
    bool rows, prompt;
    int rows_most;                 // new tokens of a sequence that the rows kernel takes, at most
    int rows_new;                  // and those its tiles (and so its workspace) are made for
    int64_t rows_bytes, prompt_bytes;
};
static int route(const KvView& c, const KvQuery& a, int max_new, Routing* r) {
    r->rows = r->prompt = false;
    r->rows_bytes = r->prompt_bytes = 0;
    r->rows_most = INT32_MAX;
    if (max_new > a.tokens) max_new = (int)a.tokens;
    if ((int64_t)max_new * a.group > 32) {
        r->prompt = true;
        r->rows_most = 32 / a.group;
        // few sequences can be much shorter than the longest: the prompt kernel takes them all
        r->rows = r->rows_most > 0 && a.tokens * 4 < (int64_t)c.sequences * max_new * 3;
        if (!r->rows) r->rows_most = 0;
    } else {
        r->rows = true;
    }
    r->rows_new = r->prompt ? r->rows_most : max_new;
    if (r->rows) r->rows_bytes = kv_decode_workspace(c, a, r->rows_new);
    if (r->prompt) r->prompt_bytes = kv_prompt_workspace(c);
    if (r->rows_bytes < 0 || r->prompt_bytes < 0) return RNS_ERR_CUDA;
    return RNS_OK;
}

}  // namespace rns

using namespace rns;

extern "C" int64_t rns_kv_attention_workspace(const rns_kv_cache* cache, const rns_kv_attention_args* args) {
    KvView c;
    KvQuery p;
    Routing r;
    if (int rc = check_attention(cache, args, &c, &p)) return -rc;
    if (c.sequences == 0 || p.tokens == 0) return 0;
    if (int rc = route(c, p, args->max_new, &r)) return -rc;
    return r.rows_bytes > r.prompt_bytes ? r.rows_bytes : r.prompt_bytes;
}

extern "C" int rns_kv_attention(const rns_kv_cache* cache, const rns_kv_attention_args* a, rns_stream_t stream) {
    KvView c;
    KvQuery p;
    Routing r;
    if (int rc = check_attention(cache, a, &c, &p)) return rc;
    if (c.sequences == 0 || p.tokens == 0) return RNS_OK;
    if (int rc = route(c, p, a->max_new, &r)) return rc;
    if ((reinterpret_cast<uintptr_t>(a->d_workspace) & 15) || a->d_workspace == nullptr ||
        a->workspace_bytes < r.rows_bytes || a->workspace_bytes < r.prompt_bytes)
        return fail(RNS_ERR_INVALID_ARGUMENT, "the workspace is missing, misaligned or too small");
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    // the two may share the workspace: the second starts when the first has finished
    if (r.prompt)
        if (int rc = kv_prompt(c, p, cache->format, r.rows ? r.rows_most + 1 : 0, a->d_workspace, st)) return rc;
    if (r.rows)
        return kv_decode(c, p, cache->format, r.rows_new, r.rows_most, a->d_workspace, st);
    return RNS_OK;
}
