// Attention of chunks over a cache of type F16: the kernel's instantiations.
#include "krk_attn_chunk.cuh"

namespace krk_cuda {

int launch_attn_chunk_f16(const attn::ChunkParams &p, int head_dim, int half, cudaStream_t st) {
    return half ? launch_attn_chunk_f16_half(p, head_dim, st) : attn::launch_chunk_type<KRK_CUDA_KV_F16, false>(p, head_dim, st);
}

} // namespace krk_cuda
