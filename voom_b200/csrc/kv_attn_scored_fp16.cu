// Cache attention: FP16 caches, capped, biased or windowed scores.
#include "kv_launch.cuh"

template int voom::kv::launch_attention<__half, true>(const voom::kv::Attn&, cudaStream_t);
template int voom::kv::launch_sums<__half, true>(const voom::kv::Attn&, cudaStream_t);
