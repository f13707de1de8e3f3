// Cache attention: FP16 caches, plain scores.
#include "kv_launch.cuh"

template int voom::kv::launch_attention<__half, false>(const voom::kv::Attn&, cudaStream_t);
template int voom::kv::launch_sums<__half, false>(const voom::kv::Attn&, cudaStream_t);
