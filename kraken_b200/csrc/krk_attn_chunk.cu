// krk_cuda_attention_chunk: the choice of a launch's form, and the kernel that adds up the partial sums of divided items.
#include "krk_attn_chunk.cuh"

#include <algorithm>
#include <cfloat>

namespace krk_cuda {
namespace attn {
namespace {

// CTA (b, y): the item that CTA b + 1 of the first kernel went on with as the second one to have a part of it, if there is one; a warp a row. The parts are
// added in the order of the CTAs.
template <int D, bool HALF>
__global__ void __launch_bounds__(128)
chunk_merge_kernel(const __grid_constant__ ChunkParams p, int R) {   // R: rows of an item
    constexpr int NB = D / 32;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31, b = blockIdx.x + 1;
    const Shared it = p.shared[b];
    if (it.parts == 0) return;
    const size_t pitch = (size_t)2 * R * (D + 2);   // from a CTA's parts to the next one's
    for (int r = blockIdx.y * 4 + (threadIdx.x >> 5); r < it.n_rows; r += gridDim.y * 4) {
        const float *others = p.part + (size_t)(b - 1) * pitch, *first = others + (size_t)R * (D + 2);   // of part 0, of the others
        float x[NB], m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int c = 0; c < NB; c++) x[c] = 0.0f;
#pragma unroll 2
        for (int i = 0; i < it.parts; i++) {
            const float *from = i == 0 ? first : others + i * pitch;
            float y[NB];
#pragma unroll
            for (int c = 0; c < NB; c++) y[c] = from[r * D + 32 * c + lane];
            const float2 ml = reinterpret_cast<const float2 *>(from + R * D)[r];
            if (ml.x == -INFINITY) continue;
            const float top = fmaxf(m, ml.x), old = m == -INFINITY ? 0.0f : exp2f(m - top), now = exp2f(ml.x - top);
            m = top;
            l = l * old + ml.y * now;
#pragma unroll
            for (int c = 0; c < NB; c++) x[c] = x[c] * old + y[c] * now;
        }
        const int rr = it.row0 + r, token = rr / p.group, head = it.kvh * p.group + rr % p.group;
        float keep = 1.0f;
        if (p.sinks) {
            const float sink = p.sinks[head] * 1.44269504f, top = fmaxf(m, sink);
            keep = m == -INFINITY ? 0.0f : exp2f(m - top);
            l = l * keep + (sink == -INFINITY ? 0.0f : sink == top ? 1.0f : exp2f(sink - top));
        }
        const float f = l == 0.0f ? 0.0f : keep / l;
        const int64_t to = (int64_t)(it.q0 + token) * p.out_stride + (int64_t)head * D + lane;
#pragma unroll
        for (int c = 0; c < NB; c++) {
            if constexpr (HALF) static_cast<__half *>(p.out)[to + 32 * c] = __float2half_rn(x[c] * f);
            else static_cast<float *>(p.out)[to + 32 * c] = x[c] * f;
        }
    }
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {   // looked up once: the library does not link the driver
    static const EncodeTiled fn = [] {
        void *ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) ptr = nullptr;
        return reinterpret_cast<EncodeTiled>(ptr);
    }();
    return fn;
}
// The rows of an f16 pool, in boxes of 64 values (the 128-byte swizzle) of as many positions of a tile as lie in one page.
bool encode_pools(ChunkParams &p, int d) {
    const EncodeTiled encode = encode_tiled();
    if (!encode) return false;
    p.box_rows = chunk_positions(d, 1);
    while (p.page_size % p.box_rows) p.box_rows /= 2;
    // (a cache without pages has no memory: a row of the queries, which no copy names)
    const int64_t rows = p.n_pages * p.n_kv * p.page_size;
    p.pool_rows = (int)(rows > 0 ? rows : 1);
    for (int kv = 0; kv < 2; kv++) {
        const cuuint64_t dims[2] = {(cuuint64_t)d, (cuuint64_t)p.pool_rows}, strides[1] = {(cuuint64_t)(2 * d)};
        const cuuint32_t box[2] = {64, (cuuint32_t)p.box_rows}, step[2] = {1, 1};
        const void *from = rows > 0 ? static_cast<const void *>(kv ? p.v : p.k) : p.q;
        if (encode(kv ? &p.v_map : &p.k_map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void *>(from), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return false;
    }
    return true;
}

// The queries as [token][head][value], in boxes of 128 bytes of the group's heads of so many tokens as are 128 rows. f16 in the 128-byte swizzle.
void encode_queries(ChunkParams &p, int d, bool half) {
    const EncodeTiled encode = encode_tiled();
    p.q_boxes = 0;
    if (!encode || 128 % p.group != 0) return;
    const int bytes = half ? 2 : 4;
    // (no box names a token that no sequence has: their number is not known here)
    const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)p.n_heads, 1ull << 30}, strides[2] = {(cuuint64_t)(d * bytes), (cuuint64_t)(p.q_stride * bytes)};
    const cuuint32_t box[3] = {(cuuint32_t)(128 / bytes), (cuuint32_t)p.group, (cuuint32_t)(128 / p.group)}, step[3] = {1, 1, 1};
    p.q_boxes = encode(&p.q_map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<void *>(p.q), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                       half ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int launch_chunk_merge(const ChunkParams &p, int d, bool half, int r, int rows, cudaStream_t st) {
    auto kernel = half ? (d == 64 ? chunk_merge_kernel<64, true> : d == 96 ? chunk_merge_kernel<96, true> : d == 128 ? chunk_merge_kernel<128, true>
                          : d == 192 ? chunk_merge_kernel<192, true> : chunk_merge_kernel<256, true>)
                       : (d == 64 ? chunk_merge_kernel<64, false> : d == 96 ? chunk_merge_kernel<96, false> : d == 128 ? chunk_merge_kernel<128, false>
                          : d == 192 ? chunk_merge_kernel<192, false> : chunk_merge_kernel<256, false>);
    return launched(launch_overlapped(kernel, dim3((unsigned)(p.grid - 1), (unsigned)(rows < 32 ? (rows + 3) / 4 : 8)), dim3(128), st, p, r));
}

// One piece of 64 tokens of every sequence that has so many is a sequence of tree attention.
krk_cuda_attention pieces_of(const krk_cuda_attention &a, int parts) {
    krk_cuda_attention t = a;
    t.n_seq = (int)((int64_t)a.n_seq * parts < INT32_MAX ? (int64_t)a.n_seq * parts : INT32_MAX);   // (more are refused)
    t.max_q = a.max_q < KRK_CUDA_MAX_DRAFT ? a.max_q : KRK_CUDA_MAX_DRAFT;
    return t;
}

struct ChunkForm {
    bool chunk, tree;   // the kernel of chunks; that of attention_tree, over pieces of 64 tokens. Both: the second one where the first one met what it cannot hold
    int terms;          // of keys and values
    int grid, whole, rows, parts;   // parts: pieces of a sequence at most
    size_t bytes, runs_at, beyond_at;
};
ChunkForm form_of(const krk_cuda_kv_cache &cache, const krk_cuda_attention &a, int out_dtype) {
    ChunkForm f = {};
    f.tree = out_dtype == KRK_CUDA_X_F32 && cache.type != KRK_CUDA_KV_F16;
    f.terms = f.tree ? 2 : 1;
    const int d = cache.head_dim, r = chunk_rows(d, f.terms), tp = chunk_positions(d, f.terms);
    const int64_t rows = (int64_t)a.max_q * (a.n_heads / cache.n_kv_heads), blocks = (rows + r - 1) / r;
    // f32 results over 8 and 4 bits: few rows go to the kernel of attention_tree, as all rows of heads longer than 128 (two terms of queries, keys and values have no
    // room). Behind 2000 positions, eight sequences of 64 tokens (256 rows of 128 values, 8 bits): 61 us here, 68 there, one sequence 57 and 39; of 128 tokens 76 and
    // 120, 58 and 67; 4 bits and 64 values, 128 tokens 73 and 77, 56 and 45; 300 tokens 124 and 164, 75 and 85; one token 38 and 13.
    f.chunk = !f.tree || (d <= 128 && rows * d > 256 * 128);
    // f32 results over 8- and 4-bit caches: keys and values of 18 bits, which the products of tree attention take as whole numbers and scales
    if (f.tree) {
        f.parts = (a.max_q + KRK_CUDA_MAX_DRAFT - 1) / KRK_CUDA_MAX_DRAFT;
        f.bytes = attention_tree_workspace_bytes(cache, pieces_of(a, f.parts));
        if (!f.chunk) return f;
    }
    f.whole = a.max_kv_len <= (int64_t)kChunkWholeTiles * tp / 2;
    const int64_t items = (int64_t)a.n_seq * cache.n_kv_heads * blocks, units = f.whole ? items : items * ((a.max_kv_len + tp - 1) / tp);
    f.grid = (int)(units < sm_count() ? units : sm_count());
    f.rows = (int)(rows < r ? rows : r);
    size_t bytes = f.whole ? 0 : shared_bytes(f.grid) + 32 + (size_t)f.grid * 2 * r * (d + 2) * sizeof(float);
    f.runs_at = (bytes + 15) / 16 * 16;
    if (!f.whole && out_dtype == KRK_CUDA_X_F32) bytes = f.runs_at + (size_t)f.grid * r * (d + 1) * sizeof(float);
    f.beyond_at = ((f.bytes > bytes ? f.bytes : bytes) + 15) / 16 * 16;
    f.bytes = f.tree ? f.beyond_at + f.grid * sizeof(int) : bytes;
    return f;
}
}   // namespace
}   // namespace attn

size_t attention_chunk_workspace_bytes(const krk_cuda_kv_cache &cache, const krk_cuda_attention &a, int out_dtype) {
    const attn::ChunkForm f = attn::form_of(cache, a, out_dtype);
    return f.bytes;
}

int launch_attention_chunk(void *out, int out_dtype, const void *q, int q_dtype, const krk_cuda_kv_cache &cache, const krk_cuda_attention &a, void *workspace, cudaStream_t st) {
    const attn::ChunkForm f = attn::form_of(cache, a, out_dtype);
    const int d = cache.head_dim, r = attn::chunk_rows(d, f.terms);
    attn::ChunkParams p;
    p.beyond = reinterpret_cast<int *>(static_cast<uint8_t *>(workspace) + f.beyond_at);
    if (f.tree && (int64_t)a.n_seq * f.parts > INT32_MAX) return KRK_CUDA_ESHAPE;
    auto pieces = [&]() {
        return launch_attention_pieces(static_cast<float *>(out), static_cast<const float *>(q), cache, attn::pieces_of(a, f.parts), f.parts, a.max_q, f.chunk ? p.beyond : nullptr, f.grid, workspace, st);
    };
    if (!f.chunk) return pieces();
    p.q = q, p.out = out, p.q_stride = a.q_stride, p.out_stride = a.out_stride;
    p.k = static_cast<const uint8_t *>(cache.k), p.v = static_cast<const uint8_t *>(cache.v);
    p.k_scale = static_cast<const __half *>(cache.k_scale), p.v_scale = static_cast<const __half *>(cache.v_scale);
    p.table = static_cast<const int32_t *>(a.page_table), p.q_start = static_cast<const int32_t *>(a.q_start), p.kv_len = static_cast<const int32_t *>(a.kv_len);
    p.sinks = static_cast<const float *>(a.sinks);
    p.shared = static_cast<attn::Shared *>(workspace);
    p.part = f.whole ? nullptr : reinterpret_cast<float *>((reinterpret_cast<uintptr_t>(workspace) + attn::shared_bytes(f.grid) + 31) & ~(uintptr_t)31);
    p.runs = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + f.runs_at), p.run_tops = p.runs + (size_t)f.grid * r * d;
    p.n_pages = cache.n_pages, p.table_width = a.table_width, p.page_size = cache.page_size, p.max_len = (int)a.max_kv_len, p.n_seq = a.n_seq, p.n_heads = a.n_heads;
    p.n_kv = cache.n_kv_heads, p.group = a.n_heads / cache.n_kv_heads, p.max_q = a.max_q, p.window = a.window, p.whole = f.whole, p.grid = f.grid;
    p.out_wide = (reinterpret_cast<uintptr_t>(out) | (uintptr_t)(a.out_stride * (out_dtype == KRK_CUDA_X_F16 ? 2 : 4))) % 32 == 0;
    p.q_half = q_dtype == KRK_CUDA_X_F16, p.out_half = out_dtype == KRK_CUDA_X_F16, p.scale = a.scale, p.softcap = a.softcap;
    // Scores are masked before they are multiplied by the row's factor, which therefore must not be 0 (-infinity times 0). Under a soft limit they are multiplied first, and
    // those of 0 stay 0, whatever the limit is.
    if (p.scale == 0.0f && p.softcap == 0.0f) p.softcap = 1.0f;
    // (finite, so that a score of 0 stays 0 under the smallest limits)
    p.per_cap = p.softcap > 0.0f ? std::min(1.0f / p.softcap, FLT_MAX) : 0.0f;
    attn::divide_by(p.group, p.group_mul, p.group_shift);
    p.status = device_status_word();
    if (!p.status) return KRK_CUDA_EDEVICE;
    if (cache.type == KRK_CUDA_KV_F16 && !attn::encode_pools(p, d)) return KRK_CUDA_ELAUNCH;
    attn::encode_queries(p, d, p.q_half);
    // units of work are counted in 64 bits
    const double blocks = ((double)a.max_q * p.group + r - 1) / r, all = (double)a.n_seq * p.n_kv * blocks * 4.0 * p.group * ((double)a.max_kv_len + 2.0 * r + 1024.0);
    if (all > 4e18) return KRK_CUDA_ESHAPE;
    int rc = cache.type == KRK_CUDA_KV_F16 ? launch_attn_chunk_f16(p, d, p.out_half, st) : cache.type == KRK_CUDA_KV_Q8 ? launch_attn_chunk_q8(p, d, p.out_half, st) : launch_attn_chunk_q4(p, d, p.out_half, st);
    if (rc == KRK_CUDA_OK && !f.whole && f.grid > 1) rc = attn::launch_chunk_merge(p, d, p.out_half, r, f.rows, st);
    return rc == KRK_CUDA_OK && f.tree ? pieces() : rc;
}

} // namespace krk_cuda
