// Attention of chunks over a cache of type Q4: the kernel's instantiations.
#include "krk_attn_chunk.cuh"

namespace krk_cuda {

int launch_attn_chunk_q4(const attn::ChunkParams &p, int head_dim, int half, cudaStream_t st) {
    return half ? attn::launch_chunk_type<KRK_CUDA_KV_Q4, true>(p, head_dim, st) : attn::launch_chunk_type<KRK_CUDA_KV_Q4, false>(p, head_dim, st);
}

} // namespace krk_cuda
