// From the q/k/v projections to the cache: norm and rotation of query and key heads, and the paged cache that new keys and values
// are written into in f16, 8 or 4 bits a value, and read back out of.
#include "krk_common.cuh"

#include <algorithm>

namespace krk_cuda {

namespace {

// ---- krk_cuda_qk_norm_rope ---------------------------------------------------------------------------------------
//
//   x' = R(pos) (w . x / sqrt(mean(x^2) + eps)),   R: pairs (a, b) -> (a cos - b sin, b cos + a sin), angle = pos * inv_freq
//
// Bound: reading and writing x once; for a few tokens a launch's latency. A lane has eight values of a head, four pairs (or eight
// values that are not rotated), so a group of 8, 16 or 32 lanes has a head, the sum of squares is a few shuffles, and
// a lane's four angles serve all heads that its group walks: angles take 64 bits (a far position's fraction of a turn is
// lost in 32), and are as dear as the rest of a head. 2048 tokens of 40 heads of 128 values: 16.6 us, 0.77 of the copy bandwidth.
struct RopeParams {
    const float *x[2];
    float *y[2];
    const float *w[2];
    int64_t x_stride[2], y_stride[2];
    const int32_t *pos;
    const float *inv_freq;
    int64_t n_tok;
    int heads[2], d, rot, norm, chunks, trips;   // chunks: runs of a token's heads; trips: of the loop over the longest of them
    float eps;
};

__device__ __forceinline__ float4 ld4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
__device__ __forceinline__ void st4(float *p, const float v[4]) { *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]); }

constexpr int kRopeHeads = 2;

template <int L, bool INTERLEAVED>
__global__ void __launch_bounds__(256, 4)
qk_norm_rope_kernel(const __grid_constant__ RopeParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int j = threadIdx.x % L, pairs = p.rot / 8, half = p.rot / 2;
    const int64_t group = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    const int64_t tok = group / p.chunks;
    const int chunk = (int)(group - tok * p.chunks), all = p.heads[0] + p.heads[1];
    const bool mine = tok < p.n_tok && 8 * j < p.d, turns = j < pairs;
    // first values of the lane's two runs of four
    const int a0 = !turns ? p.rot + 8 * (j - pairs) : INTERLEAVED ? 8 * j : 4 * j, b0 = turns && !INTERLEAVED ? half + 4 * j : a0 + 4;
    // heads in equal runs, kRopeHeads at a time: the next ones' values are on their way while some are worked on
    const int h0 = (int)((int64_t)all * chunk / p.chunks), h1 = (int)((int64_t)all * (chunk + 1) / p.chunks);
    auto load = [&](int hb, float (&v)[kRopeHeads][8]) {
#pragma unroll
        for (int u = 0; u < kRopeHeads; u++) {
            const int h = hb + u, which = h >= p.heads[0], head = h - (which ? p.heads[0] : 0);
            const float *x = p.x[which] + tok * p.x_stride[which] + head * p.d;
            if (mine && h < h1) {
                const float4 a = ld4(x + a0), b = ld4(x + b0);
                v[u][0] = a.x, v[u][1] = a.y, v[u][2] = a.z, v[u][3] = a.w, v[u][4] = b.x, v[u][5] = b.y, v[u][6] = b.z, v[u][7] = b.w;
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) v[u][i] = 0.0f;
            }
        }
    };
    asm volatile("griddepcontrol.wait;" ::: "memory");
    float v[kRopeHeads][8], next[kRopeHeads][8];
    load(h0, next);
    float cs[4], sn[4];
    if (mine && turns) {
        const double at = (double)p.pos[tok] * 0.15915494309189535;   // turns per unit of frequency
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const double turn = at * (double)p.inv_freq[4 * j + i];
            // halves of a turn; what f32 leaves of them goes to the sine and cosine by the first term of their series
            const double angle = 2.0 * (turn - rint(turn));
            const float first = (float)angle, rest = (float)(angle - (double)first) * 3.14159265f;
            float s, c;
            sincospif(first, &s, &c);
            sn[i] = fmaf(rest, c, s), cs[i] = fmaf(-rest, s, c);
        }
    }
    // (The runs of a warp's groups may differ by a head, and the sums below name all lanes of the warp: every group makes as many trips as
    // the longest run takes; heads behind its own are zeros that are not written. 2048 tokens: 16.5 us, 16.4 with a trip count for each group.)
    for (int trip = p.trips, hb = h0; trip > 0; trip--, hb += kRopeHeads) {
#pragma unroll
        for (int u = 0; u < kRopeHeads; u++)
#pragma unroll
            for (int i = 0; i < 8; i++) v[u][i] = next[u][i];
        load(hb + kRopeHeads, next);
        if (p.norm) {
            float sum[kRopeHeads];
#pragma unroll
            for (int u = 0; u < kRopeHeads; u++) {
                sum[u] = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) sum[u] += v[u][i] * v[u][i];
            }
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1)
#pragma unroll
                for (int u = 0; u < kRopeHeads; u++) sum[u] += __shfl_xor_sync(0xFFFFFFFFu, sum[u], o);
#pragma unroll
            for (int u = 0; u < kRopeHeads; u++) {
                const int which = hb + u >= p.heads[0];
                const float r = 1.0f / sqrtf(sum[u] / (float)p.d + p.eps);
#pragma unroll
                for (int i = 0; i < 8; i++) v[u][i] *= r;
                if (mine && p.w[which]) {
                    const float4 a = ld4(p.w[which] + a0), b = ld4(p.w[which] + b0);
                    v[u][0] *= a.x, v[u][1] *= a.y, v[u][2] *= a.z, v[u][3] *= a.w, v[u][4] *= b.x, v[u][5] *= b.y, v[u][6] *= b.z, v[u][7] *= b.w;
                }
            }
        }
#pragma unroll
        for (int u = 0; u < kRopeHeads; u++) {
            const int h = hb + u, which = h >= p.heads[0], head = h - (which ? p.heads[0] : 0);
            if (!mine || h >= h1) continue;
            if (turns) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float &a = INTERLEAVED ? v[u][2 * i] : v[u][i], &b = INTERLEAVED ? v[u][2 * i + 1] : v[u][i + 4];
                    const float z = a * cs[i] - b * sn[i];
                    b = b * cs[i] + a * sn[i];
                    a = z;
                }
            }
            float *y = p.y[which] + tok * p.y_stride[which] + head * p.d;
            st4(y + a0, v[u]);
            st4(y + b0, v[u] + 4);
        }
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
    uint32_t of_row_inv;    // see part
};
constexpr int kMostTokens = 32;   // of a block of threads
constexpr int64_t kAppended = 4096;   // tokens of a launch of append, see launch_kv_append

// u / by for u * by < 2^32, inv = ceil(2^32 / by): u inv / 2^32 is too large by less than u / 2^32, and a quotient's distance to the next whole
// number is at least 1 / by.
__device__ __forceinline__ int part(int u, uint32_t inv) { return (int)__umulhi((uint32_t)u, inv); }

// Where the rows of a block's tokens lie: row of the pools of head 0 (heads are page_size rows apart), or -1. Dividing by the page size takes
// longer than what is done with eight values, so a token's slot is looked at once.
__device__ __forceinline__ void find_rows(const CacheParams &p, int64_t t0, int n_tok, int *rows) {
    if ((int)threadIdx.x < n_tok) {
        const int64_t slot = p.slots[t0 + threadIdx.x];
        const int64_t page = slot / p.page_size;
        rows[threadIdx.x] = slot < 0 || slot >= p.n_slots ? -1 : (int)(page * p.heads * p.page_size + (slot - page * p.page_size));
    }
}

// Append: reads x once, writes the rows. A lane has eight values, four lanes a block of 32, whose largest value is two shuffles; its place
// in a token stays, and the block's tokens follow each other there, the next one's values on their way. Of tokens with the same slot the last
// one stays: a block of threads looks through the slots of the launch behind its tokens while its first values are on their way.
template <int CT>
__global__ void __launch_bounds__(256)
kv_append_kernel(const __grid_constant__ CacheParams p) {
    __shared__ int64_t s_slot[kMostTokens];
    __shared__ int s_row[kMostTokens];
    __shared__ uint32_t s_met[64];   // bit slot % 2048 of the block's slots
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, of_row = p.d / 8, of_tok = 2 * p.heads * of_row;
    const int64_t t0 = (int64_t)blockIdx.x * p.per_block;
    const int n_tok = (int)min((int64_t)p.per_block, p.n - t0);
    struct Place {
        bool there;
        int kv, head, c;
        const float *from;
    };
    auto place = [&](int at) {
        Place w;
        w.there = at < of_tok;
        at = min(at, of_tok - 1);
        w.kv = at >= of_tok / 2;
        if (w.kv) at -= of_tok / 2;
        w.head = part(at, p.of_row_inv);
        w.c = at - w.head * of_row;
        w.from = p.x[w.kv] + t0 * p.x_stride[w.kv] + w.head * p.d + 8 * w.c;
        return w;
    };
    auto load = [&](const Place &w, int tok, float x[8]) {
        if (!w.there || tok >= n_tok) return;
        const float *from = w.from + tok * p.x_stride[w.kv];
        const float4 a = ld4(from), b = ld4(from + 4);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    };
    Place w = place(tid);
    float next[8] = {};
    load(w, 0, next);
    if (tid < n_tok) s_slot[tid] = p.slots[t0 + tid];
    if (tid < 64) s_met[tid] = 0u;
    find_rows(p, t0, n_tok, s_row);
    __syncthreads();
    if (tid < n_tok) atomicOr(&s_met[(s_slot[tid] >> 5) & 63], 1u << (s_slot[tid] & 31));
    __syncthreads();
#pragma unroll 4
    for (int64_t j = t0 + 1 + tid; j < p.n; j += 256) {
        const int64_t slot = p.slots[j];
        if ((s_met[(slot >> 5) & 63] >> (slot & 31)) & 1)   // (8191 tokens: 31 us; each against every later one 55)
            for (int i = 0; i < n_tok; i++)
                if (slot == s_slot[i] && t0 + i < j) s_row[i] = -1;
    }
    __syncthreads();
    for (int base = 0, tok = 0; base < of_tok;) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = next[i];
        const int kv = w.kv, head = w.head, c = w.c;
        const int first = s_row[tok], row = first + head * p.page_size;
        const bool keep = w.there && first >= 0;
        if (++tok == n_tok) {   // the next place
            tok = 0;
            base += 256;
            w = place(base + tid);
        }
        load(w, tok, next);
        if constexpr (CT == KRK_CUDA_KV_F16) {
            __half2 h[4];
#pragma unroll
            for (int i = 0; i < 4; i++) h[i] = __halves2half2(half_sat(x[2 * i]), half_sat(x[2 * i + 1]));
            if (keep) *reinterpret_cast<uint4 *>(p.pool[kv] + ((int64_t)row * p.d + 8 * c) * 2) = *reinterpret_cast<uint4 *>(h);
        } else {
            float hi = x[0], lo = x[0], all = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                hi = fmaxf(hi, x[i]);
                lo = fminf(lo, x[i]);
                all = fmaf(x[i], 0.0f, all);   // (NaN where an infinity or a NaN is)
            }
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) {
                hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
                lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
                all += __shfl_xor_sync(0xFFFFFFFFu, all, o);
            }
            // a block that holds an infinity or a NaN reads back as NaN
            constexpr bool k8 = CT == KRK_CUDA_KV_Q8;
            const bool odd = all != all;
            const __half dh = odd ? __ushort_as_half(0x7FFF) : half_sat(__fdiv_rn(k8 ? fmaxf(hi, -lo) : hi >= -lo ? hi : lo, k8 ? 127.0f : -8.0f));
            const float d = __half2float(dh), inv = 1.0f / d;
            const bool none = d == 0.0f || odd;
            // rint(x / d) as x / d rounds to f32: the product with the reciprocal is off by less than 2^-16 of up to 128, so only quotients that
            // near to a half are divided. A whole number is in the low bits of 1.5 * 2^23 more.
            constexpr float kMagic = 12582912.0f, kLeast = k8 ? -127.0f : -8.0f, kMost = k8 ? 127.0f : 7.0f;
            uint32_t u[8];
            bool near = none;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float q = fminf(fmaxf(x[i] * inv, kLeast), kMost), f = q + kMagic;   // (beyond the limits nothing is near)
                near |= !(fabsf(q - (f - kMagic)) < 0.49998f);
                u[i] = __float_as_uint(f);
            }
            if (near) {
#pragma unroll
                for (int i = 0; i < 8; i++) u[i] = __float_as_uint((none ? 0.0f : fminf(fmaxf(rintf(__fdiv_rn(x[i], d)), kLeast), kMost)) + kMagic);
            }
            uint32_t b[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                b[i] = __byte_perm(__byte_perm(u[4 * i], u[4 * i + 1], 0x0040), __byte_perm(u[4 * i + 2], u[4 * i + 3], 0x0040), 0x5410);
                if constexpr (!k8) b[i] = (b[i] ^ 0x08080808u) & 0x0F0F0F0Fu;   // (-8 .. 7 in four bits to 0 .. 15)
            }
            if constexpr (k8) {
                if (keep) *reinterpret_cast<uint2 *>(p.pool[kv] + (int64_t)row * p.d + 8 * c) = make_uint2(b[0], b[1]);
            } else {
                // values 16 .. 31 of a block (lanes 2, 3 of its four) are the high halves of the bytes of values 0 .. 15
                const uint32_t h0 = __shfl_down_sync(0xFFFFFFFFu, b[0], 2), h1 = __shfl_down_sync(0xFFFFFFFFu, b[1], 2);
                if (keep && (c & 3) < 2) *reinterpret_cast<uint2 *>(p.pool[kv] + (int64_t)row * (p.d / 2) + 16 * (c >> 2) + 8 * (c & 3)) = make_uint2(b[0] | h0 << 4, b[1] | h1 << 4);
            }
            if (keep && (c & 3) == 0) p.scale[kv][(int64_t)row * (p.d / 32) + (c >> 2)] = dh;
        }
    }
}

// Read: the rows of the slots as f32; a slot that the cache does not have is a row of zeros. A lane has four values of a row of keys and
// of the row of values (eight, written 32 bytes apart, wrote each sector of level 2 twice); its place in a token stays, and
// the block's tokens follow each other there, two at a time.
template <int CT>
__global__ void __launch_bounds__(256)
kv_read_kernel(const __grid_constant__ CacheParams p) {
    __shared__ int s_row[kMostTokens];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, of_row = p.d / 4, of_tok = p.heads * of_row;
    const int64_t t0 = (int64_t)blockIdx.x * p.per_block;
    const int n_tok = (int)min((int64_t)p.per_block, p.n - t0);
    find_rows(p, t0, n_tok, s_row);
    __syncthreads();
    for (int at = tid; at < of_tok; at += 256) {
        const int head = part(at, p.of_row_inv), c = at - head * of_row;
        const int in_head = head * p.page_size;
        const int of_pool = CT == KRK_CUDA_KV_F16 ? 2 * p.d : CT == KRK_CUDA_KV_Q8 ? p.d : p.d / 2;   // bytes of a row
        const int in_row = CT == KRK_CUDA_KV_F16 ? 8 * c : CT == KRK_CUDA_KV_Q8 ? 4 * c : 16 * (c >> 3) + 4 * (c & 3);
#pragma unroll 2
        for (int tok = 0; tok < n_tok; tok++) {
            const int first = s_row[tok], row = first + in_head;
#pragma unroll
            for (int kv = 0; kv < 2; kv++) {
                float x[4] = {};
                if (first >= 0) {
                    const uint8_t *from = p.pool[kv] + (int64_t)row * of_pool + in_row;
                    if constexpr (CT == KRK_CUDA_KV_F16) {
                        const uint2 w = *reinterpret_cast<const uint2 *>(from);
                        const float2 f0 = __half22float2(*reinterpret_cast<const __half2 *>(&w.x)), f1 = __half22float2(*reinterpret_cast<const __half2 *>(&w.y));
                        x[0] = f0.x, x[1] = f0.y, x[2] = f1.x, x[3] = f1.y;
                    } else {
                        const uint32_t w = *reinterpret_cast<const uint32_t *>(from);
                        const float d = __half2float(p.scale[kv][(int64_t)row * (p.d / 32) + (c >> 3)]);
                        // a byte under the exponent of 2^23 is 2^23 more than its value
                        const uint32_t q = CT == KRK_CUDA_KV_Q8 ? w ^ 0x80808080u : ((c & 4) ? w >> 4 : w) & 0x0F0F0F0Fu;
                        const float off = CT == KRK_CUDA_KV_Q8 ? 8388608.0f + 128.0f : 8388608.0f + 8.0f;
#pragma unroll
                        for (int i = 0; i < 4; i++) x[i] = __fmul_rn(d, __fsub_rn(__uint_as_float(__byte_perm(q, 0x4B000000u, 0x7650u | i)), off));
                    }
                }
                st4(p.y[kv] + ((t0 + tok) * of_tok + at) * 4, x);
            }
        }
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
// Tokens of a block: a block for each up to `blocks` blocks an SM, then equal shares.
void set_per_block(CacheParams &p, int blocks, int values) {
    const int64_t of_row = p.d / values, per = p.n / (blocks * (int64_t)sm_count());
    p.per_block = (int)std::max<int64_t>(1, std::min<int64_t>(per, kMostTokens));
    p.of_row_inv = (uint32_t)((0x100000000ll + of_row - 1) / of_row);
}

#define KRK_DISPATCH_KV(type, kernel) \
    ((type) == KRK_CUDA_KV_F16 ? kernel<KRK_CUDA_KV_F16> : (type) == KRK_CUDA_KV_Q8 ? kernel<KRK_CUDA_KV_Q8> : kernel<KRK_CUDA_KV_Q4>)

} // namespace

int launch_qk_norm_rope(float *q_out, float *k_out, const float *q, const float *k, const krk_cuda_rope &r, cudaStream_t st) {
    RopeParams p;
    p.x[0] = q, p.x[1] = k, p.y[0] = q_out, p.y[1] = k_out;
    p.w[0] = static_cast<const float *>(r.q_weight), p.w[1] = r.n_kv_heads > 0 ? static_cast<const float *>(r.k_weight) : nullptr;   // (an odd last head's partner is the first key head, there or not)
    p.x_stride[0] = r.q_stride, p.x_stride[1] = r.k_stride, p.y_stride[0] = r.q_out_stride, p.y_stride[1] = r.k_out_stride;
    p.pos = static_cast<const int32_t *>(r.pos);
    p.inv_freq = static_cast<const float *>(r.inv_freq);
    p.n_tok = r.n_tok;
    p.heads[0] = r.n_heads, p.heads[1] = r.n_kv_heads;
    p.d = r.head_dim, p.rot = r.rot_dim, p.norm = r.norm;
    p.eps = r.eps;
    const int lanes = r.head_dim <= 64 ? 8 : r.head_dim <= 128 ? 16 : 32, all = r.n_heads + r.n_kv_heads;
    // At most as many groups as run at once, 1024 threads an SM, each with as many heads of a token as that leaves; a head each for few tokens.
    const int64_t groups = (int64_t)sm_count() * 1024 / lanes, want = groups / r.n_tok;
    p.chunks = (int)(want < 1 ? 1 : want < all ? want : all);
    p.trips = ((all + p.chunks - 1) / p.chunks + kRopeHeads - 1) / kRopeHeads;
    const int64_t blocks = (r.n_tok * p.chunks + 256 / lanes - 1) / (256 / lanes);
    if (blocks > INT32_MAX) return KRK_CUDA_ESHAPE;
    auto kernel = r.interleaved ? (lanes == 8 ? qk_norm_rope_kernel<8, true> : lanes == 16 ? qk_norm_rope_kernel<16, true> : qk_norm_rope_kernel<32, true>)
                                : (lanes == 8 ? qk_norm_rope_kernel<8, false> : lanes == 16 ? qk_norm_rope_kernel<16, false> : qk_norm_rope_kernel<32, false>);
    return launched(launch_overlapped(kernel, dim3((unsigned)blocks), dim3(256), st, p));
}

int launch_kv_append(const krk_cuda_kv_cache &cache, const float *k, const float *v, int64_t k_stride, int64_t v_stride, const int64_t *slots, int64_t n, cudaStream_t st) {
    // The look through the later slots grows with the square of the tokens: from twice kAppended on, equal pieces of about kAppended tokens one after
    // the other, of which a later one overwrites what an earlier one wrote. 8 heads of 128 values in f16, one launch and pieces: 8500 tokens
    // 27.9 us and 27.4, 9216 31.0 and 29.4 (8 bits 35.1 and 31.5), 16,384 74 and 52 (pieces of 8192: 55), 131,072 1625 and 410 (471); but 6144 17.7 and 19.7.
    const int64_t pieces = n < 2 * kAppended ? 1 : (n + kAppended / 2) / kAppended, share = (n + pieces - 1) / pieces;
    for (int64_t t = 0; t < n; t += share) {
        CacheParams p = cache_params(cache, slots + t, std::min(n - t, share));
        p.x[0] = k + t * k_stride, p.x[1] = v + t * v_stride;
        p.x_stride[0] = k_stride, p.x_stride[1] = v_stride;
        set_per_block(p, 4, 8);
        const int64_t blocks = (p.n + p.per_block - 1) / p.per_block;
        const int rc = launched(launch_overlapped(KRK_DISPATCH_KV(cache.type, kv_append_kernel), dim3((unsigned)blocks), dim3(256), st, p));
        if (rc != KRK_CUDA_OK) return rc;
    }
    return KRK_CUDA_OK;
}

int launch_kv_read(const krk_cuda_kv_cache &cache, float *k, float *v, const int64_t *slots, int64_t n, cudaStream_t st) {
    CacheParams p = cache_params(cache, slots, n);
    p.y[0] = k, p.y[1] = v;
    set_per_block(p, 16, 4);
    const int64_t blocks = (n + p.per_block - 1) / p.per_block;
    if (blocks > INT32_MAX) return KRK_CUDA_ESHAPE;
    return launched(launch_overlapped(KRK_DISPATCH_KV(cache.type, kv_read_kernel), dim3((unsigned)blocks), dim3(256), st, p));
}

} // namespace krk_cuda
