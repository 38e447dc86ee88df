// krk_cuda_attention_chunk, its simplest form: a warp for each (token, query head), one position after the other with the running maximum and sum.
#include "krk_attn_kernel.cuh"

namespace krk_cuda {
namespace attn {
namespace {

struct ChunkParams {
    const void *q;
    void *out;
    int64_t q_stride, out_stride;
    const uint8_t *k, *v;
    const __half *k_scale, *v_scale;
    const int32_t *table, *q_start, *kv_len;
    const float *sinks;
    int64_t n_pages;
    int table_width, page_size, max_len, n_seq, n_heads, n_kv, group, max_q, window, type, q_half, out_half;
    float scale, softcap;
};

template <int D>
__device__ __forceinline__ void row_values(float (&x)[D / 32], const uint8_t *pool, const __half *scale, int type, int64_t row) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int c = 0; c < D / 32; c++) {
        if (type == KRK_CUDA_KV_F16) x[c] = __half2float(reinterpret_cast<const __half *>(pool)[row * D + 32 * c + lane]);
        else {
            const float d = __half2float(scale[row * (D / 32) + c]);
            if (type == KRK_CUDA_KV_Q8) x[c] = d * (float)(int8_t)pool[row * D + 32 * c + lane];
            else {
                const int b = pool[row * (D / 2) + 16 * c + (lane & 15)];
                x[c] = d * (float)((lane < 16 ? b & 15 : b >> 4) - 8);
            }
        }
    }
}

template <int D>
__global__ void __launch_bounds__(128)
attn_chunk_simple(const __grid_constant__ ChunkParams p) {
    constexpr int NB = D / 32;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31, head = blockIdx.y, s = blockIdx.z, i = blockIdx.x * 4 + (threadIdx.x >> 5);
    const int q0 = p.q_start[s], n_q = min(max(p.q_start[s + 1] - q0, 0), p.max_q);
    if (i >= n_q) return;
    const int len = min(max(p.kv_len[s], 0), 1 << 30), own = len - n_q + i, kvh = head / p.group;
    float q[NB], o[NB], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int c = 0; c < NB; c++) {
        const int64_t at = (int64_t)(q0 + i) * p.q_stride + head * D + 32 * c + lane;
        q[c] = p.q_half ? __half2float(static_cast<const __half *>(p.q)[at]) : static_cast<const float *>(p.q)[at];
        o[c] = 0.0f;
    }
    const int end = min(min(own + 1, len), p.max_len);
    for (int pos = p.window > 0 ? max(0, own - p.window + 1) : 0; pos < end; pos++) {
        const int page = p.table[(size_t)s * p.table_width + pos / p.page_size];
        if (page < 0 || page >= p.n_pages) continue;
        const int64_t row = ((int64_t)page * p.n_kv + kvh) * p.page_size + pos % p.page_size;
        float x[NB], sum = 0.0f;
        row_values<D>(x, p.k, p.k_scale, p.type, row);
#pragma unroll
        for (int c = 0; c < NB; c++) sum = fmaf(q[c], x[c], sum);
#pragma unroll
        for (int b = 16; b > 0; b >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, b);
        sum *= p.scale;
        sum = p.softcap > 0.0f ? capped(sum, p.softcap) : sum * 1.44269504f;
        const float top = fmaxf(m, sum);
        if (top == -INFINITY) continue;
        const float corr = exp2f(m - top), w = exp2f(sum - top);
        m = top;
        l = l * corr + w;
        row_values<D>(x, p.v, p.v_scale, p.type, row);
#pragma unroll
        for (int c = 0; c < NB; c++) o[c] = o[c] * corr + w * x[c];
    }
    float keep = 1.0f;
    if (p.sinks) {
        const float sink = p.sinks[head] * 1.44269504f, top = fmaxf(m, sink);
        keep = m == -INFINITY ? 0.0f : exp2f(m - top);
        l = l * keep + (sink == -INFINITY ? 0.0f : exp2f(sink - top));
    }
    const float f = l == 0.0f ? 0.0f : keep / l;
#pragma unroll
    for (int c = 0; c < NB; c++) {
        const int64_t at = (int64_t)(q0 + i) * p.out_stride + head * D + 32 * c + lane;
        if (p.out_half) static_cast<__half *>(p.out)[at] = __float2half_rn(o[c] * f);
        else static_cast<float *>(p.out)[at] = o[c] * f;
    }
}

}   // namespace
}   // namespace attn

size_t attention_chunk_workspace_bytes(const krk_cuda_kv_cache &, const krk_cuda_attention &, int) { return 0; }

int launch_attention_chunk(void *out, int out_dtype, const void *q, int q_dtype, const krk_cuda_kv_cache &cache, const krk_cuda_attention &a, void *, cudaStream_t st) {
    attn::ChunkParams p;
    p.q = q, p.out = out, p.q_stride = a.q_stride, p.out_stride = a.out_stride;
    p.k = static_cast<const uint8_t *>(cache.k), p.v = static_cast<const uint8_t *>(cache.v);
    p.k_scale = static_cast<const __half *>(cache.k_scale), p.v_scale = static_cast<const __half *>(cache.v_scale);
    p.table = static_cast<const int32_t *>(a.page_table), p.q_start = static_cast<const int32_t *>(a.q_start), p.kv_len = static_cast<const int32_t *>(a.kv_len);
    p.sinks = static_cast<const float *>(a.sinks);
    p.n_pages = cache.n_pages, p.table_width = a.table_width, p.page_size = cache.page_size, p.max_len = (int)a.max_kv_len, p.n_seq = a.n_seq, p.n_heads = a.n_heads;
    p.n_kv = cache.n_kv_heads, p.group = a.n_heads / cache.n_kv_heads, p.max_q = a.max_q, p.window = a.window, p.type = cache.type;
    p.q_half = q_dtype == KRK_CUDA_X_F16, p.out_half = out_dtype == KRK_CUDA_X_F16, p.scale = a.scale, p.softcap = a.softcap;
    if (a.n_seq > 65535 || a.n_heads > 65535) return KRK_CUDA_ESHAPE;
    const int d = cache.head_dim;
    auto kernel = d == 64 ? attn::attn_chunk_simple<64> : d == 96 ? attn::attn_chunk_simple<96> : d == 128 ? attn::attn_chunk_simple<128> : d == 192 ? attn::attn_chunk_simple<192> : attn::attn_chunk_simple<256>;
    return launched(launch_overlapped(kernel, dim3((unsigned)((a.max_q + 3) / 4), (unsigned)a.n_heads, (unsigned)a.n_seq), dim3(128), st, p));
}

} // namespace krk_cuda
