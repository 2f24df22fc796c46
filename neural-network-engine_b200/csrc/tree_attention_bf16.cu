// Tree attention over a bf16 cache.
#include "tree_attention.cuh"

namespace nne {
int launch_tree_bf16(nne_ctx *ctx, int d, const TreeArgs &a, int sequences, long long max_keys, cudaStream_t s) {
    return launch_tree<__nv_bfloat16>(ctx, d, a, sequences, max_keys, s);
}
}  // namespace nne
