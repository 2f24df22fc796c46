// Tree attention over an f16 cache.
#include "tree_attention.cuh"

namespace nne {
int launch_tree_f16(nne_ctx *ctx, int d, const TreeArgs &a, int sequences, long long max_keys, cudaStream_t s) {
    return launch_tree<__half>(ctx, d, a, sequences, max_keys, s);
}
}  // namespace nne
