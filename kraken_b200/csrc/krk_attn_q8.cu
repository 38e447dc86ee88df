// Attention over a cache of type Q8: the kernel's instantiations.
#include "krk_attn_kernel.cuh"

namespace krk_cuda {

int launch_attn_q8(const attn::Params &p, int head_dim, int rows, cudaStream_t st) {
    return attn::launch_type<KRK_CUDA_KV_Q8>(p, head_dim, rows, st);
}
int attn_ctas_q8(int head_dim, int rows) { return attn::ctas_per_sm(KRK_CUDA_KV_Q8, head_dim, rows); }

} // namespace krk_cuda
