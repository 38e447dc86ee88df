// Attention of many rows to a key head over a cache of type F16, on tcgen05: the kernel's instantiations.
#include "krk_attn_wide.cuh"

namespace krk_cuda {

int launch_attn_wide_f16(const attn::Params &p, int head_dim, cudaStream_t st) {
    return head_dim == 96 ? attn::launch_wide<96>(p, st) : attn::launch_wide<128>(p, st);
}

} // namespace krk_cuda
