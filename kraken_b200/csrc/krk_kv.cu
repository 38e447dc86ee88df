// From the q/k/v projections to the cache: norm and rotation of query and key heads, and the paged cache that new keys and values
// are written into in f16, 8 or 4 bits a value, and read back out of.
#include "krk_common.cuh"

namespace krk_cuda {

namespace {

// ---- krk_cuda_qk_norm_rope ---------------------------------------------------------------------------------------
//
//   x' = R(pos) (w . x / sqrt(mean(x^2) + eps)),   R: pairs (a, b) -> (a cos - b sin, b cos + a sin), angle = pos * inv_freq
//
// Bound: reading and writing x once; for a few tokens a launch's latency. A lane has eight values of a head, four pairs (or eight
// values that are not rotated), so a group of 8, 16 or 32 lanes has a head, the sum of squares is a few shuffles, and
// a lane's four angles serve all heads that its group walks: angles take 64 bits (a far position's fraction of a turn is
// lost in 32), and are as dear as the rest of a head.
struct RopeParams {
    const float *x[2];
    float *y[2];
    const float *w[2];
    int64_t x_stride[2], y_stride[2];
    const int32_t *pos;
    const float *inv_freq;
    int64_t n_tok;
    int heads[2], d, rot, interleaved, norm, chunks;
    float eps;
};

__device__ __forceinline__ float4 ld4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
__device__ __forceinline__ void st4(float *p, const float v[4]) { *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]); }

template <int L>
__global__ void __launch_bounds__(256)
qk_norm_rope_kernel(const __grid_constant__ RopeParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int j = threadIdx.x % L, pairs = p.rot / 8, half = p.rot / 2;
    const int64_t group = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    const int64_t tok = group / p.chunks;
    const int chunk = (int)(group - tok * p.chunks), all = p.heads[0] + p.heads[1];
    const bool mine = tok < p.n_tok && 8 * j < p.d, turns = j < pairs;
    // first values of the lane's two runs of four
    const int a0 = !turns ? p.rot + 8 * (j - pairs) : p.interleaved ? 8 * j : 4 * j, b0 = turns && !p.interleaved ? half + 4 * j : a0 + 4;
    float cs[4], sn[4];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (mine && turns) {
        const double at = (double)p.pos[tok] * 0.15915494309189535;   // turns per unit of frequency
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const double turn = at * (double)p.inv_freq[4 * j + i];
            sincospif((float)(2.0 * (turn - rint(turn))), &sn[i], &cs[i]);
        }
    }
    // heads in equal runs
    const int h0 = (int)((int64_t)all * chunk / p.chunks), h1 = (int)((int64_t)all * (chunk + 1) / p.chunks);
#pragma unroll 2
    for (int h = h0; h < h1; h++) {
        const int which = h >= p.heads[0], head = h - (which ? p.heads[0] : 0);
        const float *x = p.x[which] + tok * p.x_stride[which] + (int64_t)head * p.d;
        float v[8] = {};
        if (mine) {
            const float4 a = ld4(x + a0), b = ld4(x + b0);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        }
        if (p.norm) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) sum += v[i] * v[i];
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
            const float r = 1.0f / sqrtf(sum / (float)p.d + p.eps);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] *= r;
            if (mine && p.w[which]) {
                const float4 a = ld4(p.w[which] + a0), b = ld4(p.w[which] + b0);
                v[0] *= a.x, v[1] *= a.y, v[2] *= a.z, v[3] *= a.w, v[4] *= b.x, v[5] *= b.y, v[6] *= b.z, v[7] *= b.w;
            }
        }
        if (!mine) continue;
        if (turns) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float &a = v[p.interleaved ? 2 * i : i], &b = v[p.interleaved ? 2 * i + 1 : i + 4];
                const float u = a * cs[i] - b * sn[i];
                b = b * cs[i] + a * sn[i];
                a = u;
            }
        }
        float *y = p.y[which] + tok * p.y_stride[which] + (int64_t)head * p.d;
        st4(y + a0, v);
        st4(y + b0, v + 4);
    }
}

// ---- the cache ----------------------------------------------------------------------------------------------------

struct CacheParams {
    uint8_t *pool[2];       // keys, values
    __half *scale[2];
    const float *x[2];      // append: [token][kv head][d]
    float *y[2];            // read
    int64_t x_stride[2];    // floats from a token to the next
    const int64_t *slots;
    int64_t n, n_slots;
    int heads, d, page_size, per_block;
};

// Where a row of the pools lies: (page, head, slot of the page).
__device__ __forceinline__ int64_t pool_row(const CacheParams &p, int64_t slot, int head) {
    const int64_t page = slot / p.page_size;
    return (page * p.heads + head) * p.page_size + (slot - page * p.page_size);
}

// Append: reads x once, writes the rows. A lane has eight values, four lanes a block of 32, whose largest value is two
// shuffles. Of tokens with the same slot the last one stays: a block of threads looks through the slots behind its tokens while its
// first values are on their way (from 1184 tokens on, a block has more than one token, which share the look).
template <int CT>
__global__ void __launch_bounds__(256)
kv_append_kernel(const __grid_constant__ CacheParams p) {
    constexpr int kMost = 32;
    __shared__ int64_t s_slot[kMost];
    __shared__ int s_drop[kMost];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, of_row = p.d / 8, of_tok = 2 * p.heads * of_row;
    const int64_t t0 = (int64_t)blockIdx.x * p.per_block;
    const int n_tok = (int)min((int64_t)p.per_block, p.n - t0), total = n_tok * of_tok;
    auto load = [&](int u, float x[8]) {
        if (u >= total) return;
        const int tok = u / of_tok, in_tok = u - tok * of_tok, kv = in_tok >= of_tok / 2, at = in_tok - (kv ? of_tok / 2 : 0);
        const float *from = p.x[kv] + (t0 + tok) * p.x_stride[kv] + 8 * at;
        const float4 a = ld4(from), b = ld4(from + 4);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    };
    float x[8] = {};
    load(tid, x);
    if (tid < n_tok) {
        const int64_t slot = p.slots[t0 + tid];
        s_slot[tid] = slot;
        s_drop[tid] = slot < 0 || slot >= p.n_slots;
    }
    __syncthreads();
    for (int64_t j = t0 + 1 + tid; j < p.n; j += 256) {
        const int64_t slot = p.slots[j];
        for (int i = 0; i < n_tok; i++)
            if (slot == s_slot[i] && t0 + i < j) s_drop[i] = 1;
    }
    __syncthreads();
    for (int base = 0; base < total; base += 256) {
        const int u = base + tid;
        if (base) load(u, x);
        const int uu = min(u, total - 1), tok = uu / of_tok, in_tok = uu - tok * of_tok, kv = in_tok >= of_tok / 2, at = in_tok - (kv ? of_tok / 2 : 0);
        const int head = at / of_row, c = at - head * of_row;
        const bool keep = u < total && !s_drop[tok];
        const int64_t row = keep ? pool_row(p, s_slot[tok], head) : 0;
        if constexpr (CT == KRK_CUDA_KV_F16) {
            __half2 h[4];
#pragma unroll
            for (int i = 0; i < 4; i++) h[i] = __halves2half2(half_sat(x[2 * i]), half_sat(x[2 * i + 1]));
            if (keep) *reinterpret_cast<uint4 *>(p.pool[kv] + (row * p.d + 8 * c) * 2) = *reinterpret_cast<uint4 *>(h);
        } else {
            float hi = x[0], lo = x[0];
            bool odd = false;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                hi = fmaxf(hi, x[i]);
                lo = fminf(lo, x[i]);
                odd |= !(fabsf(x[i]) <= 3.4028234e38f);
            }
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) {
                hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
                lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
                odd |= __shfl_xor_sync(0xFFFFFFFFu, odd, o);
            }
            // a block that holds an infinity or a NaN reads back as NaN
            constexpr bool k8 = CT == KRK_CUDA_KV_Q8;
            const __half dh = odd ? __ushort_as_half(0x7FFF) : half_sat(__fdiv_rn(k8 ? fmaxf(hi, -lo) : hi >= -lo ? hi : lo, k8 ? 127.0f : -8.0f));
            const float d = __half2float(dh);
            uint32_t w[2] = {};
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float r = d == 0.0f || odd ? 0.0f : rintf(__fdiv_rn(x[i], d));
                if constexpr (k8)
                    w[i >> 2] |= ((uint32_t)(int)fminf(fmaxf(r, -127.0f), 127.0f) & 255u) << (8 * (i & 3));
                else
                    w[i >> 2] |= (uint32_t)(int)(fminf(fmaxf(r, -8.0f), 7.0f) + 8.0f) << (8 * (i & 3));
            }
            if constexpr (k8) {
                if (keep) *reinterpret_cast<uint2 *>(p.pool[kv] + row * p.d + 8 * c) = make_uint2(w[0], w[1]);
            } else {
                // values 16 .. 31 of a block (lanes 2, 3 of its four) are the high halves of the bytes of values 0 .. 15
                const uint32_t h0 = __shfl_down_sync(0xFFFFFFFFu, w[0], 2), h1 = __shfl_down_sync(0xFFFFFFFFu, w[1], 2);
                if (keep && (c & 3) < 2) *reinterpret_cast<uint2 *>(p.pool[kv] + row * (p.d / 2) + 16 * (c >> 2) + 8 * (c & 3)) = make_uint2(w[0] | h0 << 4, w[1] | h1 << 4);
            }
            if (keep && (c & 3) == 0) p.scale[kv][row * (p.d / 32) + (c >> 2)] = dh;
        }
    }
}

// Read: the rows of the slots as f32; a slot that the cache does not have is a row of zeros. A lane has eight values.
template <int CT>
__global__ void __launch_bounds__(256)
kv_read_kernel(const __grid_constant__ CacheParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int of_row = p.d / 8, of_tok = p.heads * of_row;
    const int64_t total = 2 * p.n * of_tok;
    for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < total; u += (int64_t)gridDim.x * 256) {
        const int64_t tk = u / of_tok, tok = tk >> 1;
        const int kv = (int)(tk & 1), at = (int)(u - tk * of_tok), head = at / of_row, c = at - head * of_row;
        const int64_t slot = p.slots[tok];
        float x[8] = {};
        if (slot >= 0 && slot < p.n_slots) {
            const int64_t row = pool_row(p, slot, head);
            if constexpr (CT == KRK_CUDA_KV_F16) {
                const uint4 w = *reinterpret_cast<const uint4 *>(p.pool[kv] + (row * p.d + 8 * c) * 2);
                const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&ws[i]));
                    x[2 * i] = f.x, x[2 * i + 1] = f.y;
                }
            } else {
                const float d = __half2float(p.scale[kv][row * (p.d / 32) + (c >> 2)]);
                const uint2 w = CT == KRK_CUDA_KV_Q8 ? *reinterpret_cast<const uint2 *>(p.pool[kv] + row * p.d + 8 * c)
                                                     : *reinterpret_cast<const uint2 *>(p.pool[kv] + row * (p.d / 2) + 16 * (c >> 2) + 8 * (c & 1));
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const uint32_t byte = (i < 4 ? w.x : w.y) >> (8 * (i & 3)) & 255u;
                    x[i] = __fmul_rn(d, CT == KRK_CUDA_KV_Q8 ? (float)(int8_t)byte : (float)((int)((c & 2) ? byte >> 4 : byte & 15u) - 8));
                }
            }
        }
        float *to = p.y[kv] + tok * (int64_t)of_tok * 8 + 8 * at;
        st4(to, x);
        st4(to + 4, x + 4);
    }
}

CacheParams cache_params(const krk_cuda_kv_cache &cache, const int64_t *slots, int64_t n) {
    CacheParams p = {};
    p.pool[0] = static_cast<uint8_t *>(cache.k);
    p.pool[1] = static_cast<uint8_t *>(cache.v);
    p.scale[0] = static_cast<__half *>(cache.k_scale);
    p.scale[1] = static_cast<__half *>(cache.v_scale);
    p.slots = slots;
    p.n = n;
    p.n_slots = cache.n_pages * cache.page_size;
    p.heads = cache.n_kv_heads;
    p.d = cache.head_dim;
    p.page_size = cache.page_size;
    return p;
}

#define KRK_DISPATCH_KV(type, kernel) \
    ((type) == KRK_CUDA_KV_F16 ? kernel<KRK_CUDA_KV_F16> : (type) == KRK_CUDA_KV_Q8 ? kernel<KRK_CUDA_KV_Q8> : kernel<KRK_CUDA_KV_Q4>)

} // namespace

int launch_qk_norm_rope(float *q_out, float *k_out, const float *q, const float *k, const krk_cuda_rope &r, cudaStream_t st) {
    RopeParams p;
    p.x[0] = q, p.x[1] = k, p.y[0] = q_out, p.y[1] = k_out;
    p.w[0] = static_cast<const float *>(r.q_weight), p.w[1] = static_cast<const float *>(r.k_weight);
    p.x_stride[0] = r.q_stride, p.x_stride[1] = r.k_stride, p.y_stride[0] = r.q_out_stride, p.y_stride[1] = r.k_out_stride;
    p.pos = static_cast<const int32_t *>(r.pos);
    p.inv_freq = static_cast<const float *>(r.inv_freq);
    p.n_tok = r.n_tok;
    p.heads[0] = r.n_heads, p.heads[1] = r.n_kv_heads;
    p.d = r.head_dim, p.rot = r.rot_dim, p.interleaved = r.interleaved, p.norm = r.norm;
    p.eps = r.eps;
    const int lanes = r.head_dim <= 64 ? 8 : r.head_dim <= 128 ? 16 : 32, all = r.n_heads + r.n_kv_heads;
    // Groups for about 1024 threads an SM, each with as many heads of a token as that leaves; a head each for few tokens.
    const int64_t groups = (int64_t)sm_count() * 1024 / lanes, want = (groups + r.n_tok - 1) / r.n_tok;
    p.chunks = (int)(want < all ? want : all);
    const int64_t blocks = (r.n_tok * p.chunks + 256 / lanes - 1) / (256 / lanes);
    if (blocks > INT32_MAX) return KRK_CUDA_ESHAPE;
    auto kernel = lanes == 8 ? qk_norm_rope_kernel<8> : lanes == 16 ? qk_norm_rope_kernel<16> : qk_norm_rope_kernel<32>;
    return launched(launch_overlapped(kernel, dim3((unsigned)blocks), dim3(256), st, p));
}

int launch_kv_append(const krk_cuda_kv_cache &cache, const float *k, const float *v, int64_t k_stride, int64_t v_stride, const int64_t *slots, int64_t n, cudaStream_t st) {
    CacheParams p = cache_params(cache, slots, n);
    p.x[0] = k, p.x[1] = v;
    p.x_stride[0] = k_stride, p.x_stride[1] = v_stride;
    const int64_t per = n / (8 * (int64_t)sm_count());
    p.per_block = (int)(per < 1 ? 1 : per > 32 ? 32 : per);
    const int64_t blocks = (n + p.per_block - 1) / p.per_block;
    if (blocks > INT32_MAX) return KRK_CUDA_ESHAPE;
    return launched(launch_overlapped(KRK_DISPATCH_KV(cache.type, kv_append_kernel), dim3((unsigned)blocks), dim3(256), st, p));
}

int launch_kv_read(const krk_cuda_kv_cache &cache, float *k, float *v, const int64_t *slots, int64_t n, cudaStream_t st) {
    CacheParams p = cache_params(cache, slots, n);
    p.y[0] = k, p.y[1] = v;
    const int64_t want = (2 * n * cache.n_kv_heads * (cache.head_dim / 8) + 255) / 256, fill = (int64_t)sm_count() * 16;
    return launched(launch_overlapped(KRK_DISPATCH_KV(cache.type, kv_read_kernel), dim3((unsigned)(want < fill ? want : fill)), dim3(256), st, p));
}

} // namespace krk_cuda
