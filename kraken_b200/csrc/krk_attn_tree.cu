// krk_cuda_attention_tree: the choice of a launch's form, and the kernel that adds up the partial sums of divided items.
#include "krk_attn_tree.cuh"

namespace krk_cuda {
namespace attn {
namespace {

// CTA (b, y): the item that CTA b of the first kernel went on with as the second one to have a part of it, if there is one; rows y,
// y + gridDim.y, ... of it. Four warps take the parts in turn, in the order of the CTAs; their sums are added in the order of the warps.
template <int D>
__global__ void __launch_bounds__(kThreads)
merge_kernel(const __grid_constant__ Params p, int r_block) {
    constexpr int NB = D / 32;
    __shared__ float s_sum[kWarps][D];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (!called_for(p)) return;
    const int b = blockIdx.x + 1;
    const Shared it = p.shared[b];
    if (it.parts == 0) return;
    const size_t pitch = (size_t)2 * r_block * (D + 2);   // from a CTA's parts to the next one's
    for (int r = blockIdx.y; r < it.n_rows; r += gridDim.y) {
        // part 0: CTA b - 1, place 1; part i: CTA b - 1 + i, place 0
        const float *first = p.part + (size_t)(b - 1) * pitch + (size_t)(r_block + r) * (D + 2), *others = p.part + (size_t)(b - 1) * pitch + (size_t)r * (D + 2);
        auto part = [&](int i) { return i == 0 ? first : others + i * pitch; };
        float2 ml = lane < it.parts ? *reinterpret_cast<const float2 *>(part(lane) + D) : make_float2(-INFINITY, 0.0f);
        for (int i = lane + 32; i < it.parts; i += 32) {
            const float2 more = *reinterpret_cast<const float2 *>(part(i) + D);
            const float top = fmaxf(ml.x, more.x);
            ml.y = (ml.x == -INFINITY ? 0.0f : ml.y * exp2f(ml.x - top)) + (more.x == -INFINITY ? 0.0f : more.y * exp2f(more.x - top));
            ml.x = top;
        }
        float top = ml.x;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        float all = ml.x == -INFINITY ? 0.0f : ml.y * exp2f(ml.x - top);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xFFFFFFFFu, all, o);
        float x[NB];
#pragma unroll
        for (int j = 0; j < NB; j++) x[j] = 0.0f;
#pragma unroll 4
        for (int i = warp; i < it.parts; i += kWarps) {
            const float *from = part(i);
            const float m = from[D], f = m == -INFINITY ? 0.0f : exp2f(m - top);
#pragma unroll
            for (int j = 0; j < NB; j++) x[j] += f * from[32 * j + lane];
        }
#pragma unroll
        for (int j = 0; j < NB; j++) s_sum[warp][32 * j + lane] = x[j];
        __syncthreads();
        const int rr = it.row0 + r, head = it.kvh * p.group + rr % p.group;
        float keep;
        const float f = norm_of(p, head, top, all, keep);
        float *to = p.out + (int64_t)(it.q0 + rr / p.group) * p.out_stride + head * D;
        for (int c = tid; c < D; c += kThreads) {
            float sum = s_sum[0][c];
#pragma unroll
            for (int w = 1; w < kWarps; w++) sum += s_sum[w][c];
            to[c] = sum * f;
        }
        __syncthreads();
    }
}

int launch_merge(const Params &p, int d, int r_block, int rows, cudaStream_t st) {
    auto kernel = d == 64 ? merge_kernel<64> : d == 96 ? merge_kernel<96> : d == 128 ? merge_kernel<128> : d == 192 ? merge_kernel<192> : merge_kernel<256>;
    return launched(launch_overlapped(kernel, dim3((unsigned)(p.grid - 1), (unsigned)(rows < 8 ? rows : 8)), dim3(kThreads), st, p, r_block));
}

struct Form {
    int block, grid, rows, whole;   // rows of a block, CTAs, rows of an item at most, items not divided
};
Form form_of(const krk_cuda_kv_cache &cache, const krk_cuda_attention &a) {
    Form f;
    const int type = cache.type, d = cache.head_dim;
    const int64_t rows = (int64_t)a.max_q * (a.n_heads / cache.n_kv_heads);
    // Short contexts: a CTA walks a whole item, which costs less than the second kernel.
    f.whole = a.max_kv_len <= kWholeTiles * kTile;
    // Blocks as small as the rows, 16 of them at most: 32 with their outputs in 128 registers of a lane took longer than two blocks of 16 (48
    // ragged sequences of 4 to 32 rows, heads of 128 in 8 bits: 214 us against 157; blocks of 8: 207; windows over heads of 64 in 4 bits: 29 against 24.6, blocks of 8 25.1).
    // The longest sequence is not known here: by max_kv_len, or the table's width, short contexts under a wide table are divided (one token, 300
    // positions, f16, a table for 131,072: 9.1 us, 8.0 with the limit given; 8 bits 8.6 and 8.4). Over f16 caches more than 32 rows go to the
    // tensor memory's form, heads of 96 and 128 values over contexts that are divided (4 sequences of 16,000, 64 rows: 99 us against 145, 128
    // rows 166 against 296; 32 rows 80 against 94 there, but 27 against 23 at 2000; heads of 64: 91 against 87, 152 against 157).
    // A cache without pages has no memory: that form's copies of rows that are not there have a row's address all the same.
    const bool wide = type == KRK_CUDA_KV_F16 && rows > 32 && (d == 96 || d == 128) && !f.whole && cache.n_pages > 0;
    f.block = wide ? kWideRows : rows <= 4 ? 4 : rows <= 8 ? 8 : 16;
    f.rows = (int)(rows < f.block ? rows : f.block);
    const int64_t tiles = (a.max_kv_len + tile_of(f.block) - 1) / tile_of(f.block);
    const int64_t items = (int64_t)a.n_seq * cache.n_kv_heads * ((rows + f.block - 1) / f.block);
    const int64_t units = f.whole ? items : items * tiles;   // (a tile or more to a CTA)
    const int ctas = f.block == kWideRows ? 1 : type == KRK_CUDA_KV_F16 ? attn_ctas_f16(d, f.block) : type == KRK_CUDA_KV_Q8 ? attn_ctas_q8(d, f.block) : attn_ctas_q4(d, f.block);
    const int64_t fill = (int64_t)ctas * sm_count();
    f.grid = (int)(units < fill ? units : fill);
    return f;
}

}   // namespace
}   // namespace attn

size_t attention_tree_workspace_bytes(const krk_cuda_kv_cache &cache, const krk_cuda_attention &a) {
    const attn::Form f = attn::form_of(cache, a);
    return f.whole ? 0 : attn::shared_bytes(f.grid) + (size_t)f.grid * 2 * f.block * (cache.head_dim + 2) * sizeof(float);
}

int launch_attention_pieces(float *out, const float *q, const krk_cuda_kv_cache &cache, const krk_cuda_attention &a, int pieces, int piece_q, const int *only_if, int only_ifs, void *workspace, cudaStream_t st) {
    const attn::Form f = attn::form_of(cache, a);
    attn::Params p;
    p.q = q;
    p.out = out;
    p.q_stride = a.q_stride;
    p.out_stride = a.out_stride;
    p.k = static_cast<const uint8_t *>(cache.k);
    p.v = static_cast<const uint8_t *>(cache.v);
    p.k_scale = static_cast<const __half *>(cache.k_scale);
    p.v_scale = static_cast<const __half *>(cache.v_scale);
    p.table = static_cast<const int32_t *>(a.page_table);
    p.q_start = static_cast<const int32_t *>(a.q_start);
    p.kv_len = static_cast<const int32_t *>(a.kv_len);
    p.tree = static_cast<const uint64_t *>(a.tree);
    p.sinks = static_cast<const float *>(a.sinks);
    p.shared = static_cast<attn::Shared *>(workspace);
    p.part = f.whole ? nullptr : reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + attn::shared_bytes(f.grid));
    p.n_pages = cache.n_pages;
    p.table_width = a.table_width;
    p.page_size = cache.page_size;
    p.max_len = (int)a.max_kv_len;
    p.n_seq = a.n_seq;
    p.n_heads = a.n_heads;
    p.n_kv = cache.n_kv_heads;
    p.group = a.n_heads / cache.n_kv_heads;
    p.max_q = a.max_q;
    p.window = a.window;
    p.pieces = pieces;
    p.piece_q = piece_q;
    p.only_if = only_if;
    p.only_ifs = only_ifs;
    p.whole = f.whole;
    p.grid = f.grid;
    p.scale = a.scale;
    p.softcap = a.softcap;
    p.status = device_status_word();
    if (!p.status) return KRK_CUDA_EDEVICE;
    int rc = f.block == attn::kWideRows ? launch_attn_wide_f16(p, cache.head_dim, st) : cache.type == KRK_CUDA_KV_F16 ? launch_attn_f16(p, cache.head_dim, f.block, st)
             : cache.type == KRK_CUDA_KV_Q8 ? launch_attn_q8(p, cache.head_dim, f.block, st) : launch_attn_q4(p, cache.head_dim, f.block, st);
    if (rc == KRK_CUDA_OK && !f.whole && f.grid > 1) rc = attn::launch_merge(p, cache.head_dim, f.block, f.rows, st);
    return rc;
}

int launch_attention_tree(float *out, const float *q, const krk_cuda_kv_cache &cache, const krk_cuda_attention &a, void *workspace, cudaStream_t st) {
    return launch_attention_pieces(out, q, cache, a, 1, 0, nullptr, 0, workspace, st);
}

} // namespace krk_cuda
