// Attention of chunks over a cache of type Q8: the kernel's instantiations.
#include "krk_attn_chunk.cuh"

namespace krk_cuda {

int launch_attn_chunk_q8(const attn::ChunkParams &p, int head_dim, int half, cudaStream_t st) {
    return half ? attn::launch_chunk_type<KRK_CUDA_KV_Q8, true>(p, head_dim, st) : attn::launch_chunk_type<KRK_CUDA_KV_Q8, false>(p, head_dim, st);
}

} // namespace krk_cuda
