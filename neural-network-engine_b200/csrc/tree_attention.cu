// Tree attention over the paged cache: argument checks and dispatch (tree_attention.cuh has the kernel).
#include "tree_attention.cuh"

#include <math.h>

#include <new>

using namespace nne;

extern "C" int nne_tree_attention_dev(nne_kv_cache *c, const nne_tree_attention *a, void *stream) {
    NNE_GUARD_BEGIN
    NNE_TRY(check_cache(c));
    if (!a) return fail(NNE_ERR_INVALID_ARGUMENT, "null arguments");
    if (a->q_heads < 1 || a->q_heads % c->kv_heads)
        return fail(NNE_ERR_INVALID_ARGUMENT, "q_heads %d is not a multiple of kv_heads %d", a->q_heads, c->kv_heads);
    if (a->max_nodes < 0 || a->max_nodes > 64) return fail(NNE_ERR_INVALID_ARGUMENT, "max_nodes must be from 0 to 64, got %d", a->max_nodes);
    const size_t width = (size_t)a->q_heads * c->d;
    if (a->q_stride < width || a->out_stride < width) return fail(NNE_ERR_INVALID_ARGUMENT, "q_stride or out_stride below q_heads * head_dim");
    if (a->tokens > 0x7fffffffu || a->sequences < 0 || a->max_context < 0) return fail(NNE_ERR_INVALID_ARGUMENT, "a size is out of range");
    if (!isfinite(a->scale)) return fail(NNE_ERR_INVALID_ARGUMENT, "scale is not finite");
    if ((size_t)a->max_nodes * (a->q_heads / c->kv_heads) > (1 << 20)) return fail(NNE_ERR_INVALID_ARGUMENT, "too many query heads a key head");
    if (a->tokens == 0 || a->sequences == 0 || a->max_nodes == 0) return NNE_OK;
    if (!a->q || !a->out || !a->node_start || !a->context || !a->page_table)
        return fail(NNE_ERR_INVALID_ARGUMENT, "null device pointer");
    if (a->table_stride == 0) return fail(NNE_ERR_INVALID_ARGUMENT, "table_stride is 0");
    const uintptr_t bits = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->out) | reinterpret_cast<uintptr_t>(a->node_start) |
                           reinterpret_cast<uintptr_t>(a->context) | reinterpret_cast<uintptr_t>(a->page_table);
    if ((bits & 3) || (reinterpret_cast<uintptr_t>(a->visible) & 7))
        return fail(NNE_ERR_INVALID_ARGUMENT, "a pointer is not aligned to its type");
    NNE_TRY(use_ctx(c->ctx));
    TreeArgs t = {};
    t.q = a->q, t.out = a->out, t.q_stride = a->q_stride, t.out_stride = a->out_stride;
    t.group = a->q_heads / c->kv_heads, t.kv_heads = c->kv_heads;
    t.tokens = (int)a->tokens, t.max_nodes = a->max_nodes;
    t.node_start = a->node_start, t.context = a->context, t.visible = a->visible;
    t.page_table = a->page_table, t.table_stride = a->table_stride, t.pages = c->pages, t.page_shift = c->page_shift;
    t.scale = a->scale * 1.44269504088896340736f;
    t.k = c->k, t.v = c->v;
    t.vec_out = (reinterpret_cast<uintptr_t>(a->out) & 15) == 0 && a->out_stride % 4 == 0;
    const long long keys = (long long)a->max_context + a->max_nodes;
    if (c->dtype == NNE_F16) return launch_tree_f16(c->ctx, c->d, t, a->sequences, keys, (cudaStream_t)stream);
    return launch_tree_bf16(c->ctx, c->d, t, a->sequences, keys, (cudaStream_t)stream);
    NNE_GUARD_END
}
