// Cache attention: BF16 caches, plain scores.
#include "kv_launch.cuh"

template int voom::kv::launch_attention<__nv_bfloat16, false>(const voom::kv::Attn&, cudaStream_t);
template int voom::kv::launch_sums<__nv_bfloat16, false>(const voom::kv::Attn&, cudaStream_t);
