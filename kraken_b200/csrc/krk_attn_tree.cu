// krk_cuda_attention_tree: the choice of a launch's form, and the kernel that adds up the partial sums of divided items.
#include "krk_attn_tree.cuh"

namespace krk_cuda {
namespace attn {
namespace {

// CTA (b, y): the item that CTA b - 1 of the first kernel began and CTA b went on with, if there is one; rows y, y + gridDim.y, ...
// of it. Four warps take the parts in turn, in the order of the CTAs; their sums are added in the order of the warps.
template <int D, int BM>
__global__ void __launch_bounds__(kThreads)
merge_kernel(const __grid_constant__ Params p) {
    constexpr int NB = D / 32;
    __shared__ float s_sum[kWarps][D];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int b = blockIdx.x + 1;
    const Place place = find_place<BM>(p, b);
    if (place.at >= place.total) return;
    const Seq sq = sequence<BM>(p, place.seq);
    const int64_t in_seq = place.at - place.before;
    const int per_item = item_units(p, sq), item = (int)(in_seq / per_item);
    // the item's tiles, as units
    const int64_t first = place.at - (in_seq - (int64_t)item * per_item) + kSetup, item_end = first + sq.tiles;
    const int64_t prev = first_unit(place.total, p.grid, b - 1);
    if (place.at <= first || prev == place.at || prev > first) return;
    // CTAs b .. last - 1 went on with the item: those that begin before its end
    const int last = (int)min((int64_t)p.grid, (item_end * p.grid + place.total - 1) / place.total);
    const int parts = last - b + 1;
    const bool all_there = place.total >= p.grid;
    const int kvh = item / sq.blocks, block = item - kvh * sq.blocks;
    const int n_rows = min(BM, sq.n_q * p.group - block * BM);
    for (int r = blockIdx.y; r < n_rows; r += gridDim.y) {
        // part i: CTA b - 1 + i; a CTA without units has none
        auto part = [&](int i) -> const float * { return part_row<D, BM>(p, b - 1 + i, i == 0 ? 1 : 0, r); };
        auto there = [&](int i) { return all_there || first_unit(place.total, p.grid, b - 1 + i) < first_unit(place.total, p.grid, b + i); };
        float top = -INFINITY, all = 0.0f;
        for (int i = lane; i < parts; i += 32)
            if (there(i)) top = fmaxf(top, part(i)[D]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        for (int i = lane; i < parts; i += 32)
            if (there(i)) {
                const float2 ml = *reinterpret_cast<const float2 *>(part(i) + D);
                if (ml.x != -INFINITY) all += ml.y * exp2f(ml.x - top);
            }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xFFFFFFFFu, all, o);
        float x[NB];
#pragma unroll
        for (int j = 0; j < NB; j++) x[j] = 0.0f;
#pragma unroll 4
        for (int i = warp; i < parts; i += kWarps) {
            if (!there(i)) continue;
            const float *from_part = part(i);
            const float m = from_part[D], f = m == -INFINITY ? 0.0f : exp2f(m - top);
#pragma unroll
            for (int j = 0; j < NB; j++) x[j] += f * from_part[32 * j + lane];
        }
#pragma unroll
        for (int j = 0; j < NB; j++) s_sum[warp][32 * j + lane] = x[j];
        __syncthreads();
        const int rr = block * BM + r, head = kvh * p.group + rr % p.group;
        float keep;
        const float f = norm_of(p, head, top, all, keep);
        float *to = p.out + (int64_t)(sq.q0 + rr / p.group) * p.out_stride + head * D;
        for (int c = tid; c < D; c += kThreads) {
            float sum = s_sum[0][c];
#pragma unroll
            for (int w = 1; w < kWarps; w++) sum += s_sum[w][c];
            to[c] = sum * f;
        }
        __syncthreads();
    }
}

template <int D, int BM>
int merge_one(const Params &p, int rows, cudaStream_t st) {
    return launched(launch_overlapped(merge_kernel<D, BM>, dim3((unsigned)(p.grid - 1), (unsigned)(rows < 8 ? rows : 8)), dim3(kThreads), st, p));
}

int launch_merge(const Params &p, int d, int mt, int rows, cudaStream_t st) {
    switch (d) {
    case 64: return mt == 2 ? merge_one<64, 32>(p, rows, st) : merge_one<64, 16>(p, rows, st);
    case 96: return mt == 2 ? merge_one<96, 32>(p, rows, st) : merge_one<96, 16>(p, rows, st);
    case 128: return mt == 2 ? merge_one<128, 32>(p, rows, st) : merge_one<128, 16>(p, rows, st);
    case 192: return merge_one<192, 16>(p, rows, st);
    default: return merge_one<256, 16>(p, rows, st);
    }
}

struct Form {
    int mt, grid, rows, whole;   // row tiles of a block, CTAs, rows of an item at most, items not divided
};
Form form_of(const krk_cuda_kv_cache &cache, const krk_cuda_attention &a) {
    Form f;
    const int type = cache.type, d = cache.head_dim;
    const int64_t rows = (int64_t)a.max_q * (a.n_heads / cache.n_kv_heads);
    f.mt = rows > 16 && d <= 128 ? 2 : 1;
    const int bm = 16 * f.mt;
    f.rows = (int)(rows < bm ? rows : bm);
    const int64_t tiles = (a.max_kv_len + kTile - 1) / kTile;
    // Short contexts: a CTA walks a whole item, which costs less than the second kernel.
    f.whole = tiles <= kWholeTiles;
    const int64_t items = (int64_t)a.n_seq * cache.n_kv_heads * ((rows + bm - 1) / bm);
    const int64_t units = f.whole ? items : items * (tiles + kSetup);
    const int ctas = type == KRK_CUDA_KV_F16 ? attn_ctas_f16(d, f.mt) : type == KRK_CUDA_KV_Q8 ? attn_ctas_q8(d, f.mt) : attn_ctas_q4(d, f.mt);
    const int64_t fill = (int64_t)ctas * sm_count();
    f.grid = (int)(units < fill ? units : fill);
    return f;
}

}   // namespace
}   // namespace attn

size_t attention_tree_workspace_bytes(const krk_cuda_kv_cache &cache, const krk_cuda_attention &a) {
    const attn::Form f = attn::form_of(cache, a);
    return f.whole ? 0 : (size_t)f.grid * 2 * 16 * f.mt * (cache.head_dim + 2) * sizeof(float);
}

int launch_attention_tree(float *out, const float *q, const krk_cuda_kv_cache &cache, const krk_cuda_attention &a, void *workspace, cudaStream_t st) {
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
    p.part = static_cast<float *>(workspace);
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
    p.whole = f.whole;
    p.grid = f.grid;
    p.scale = a.scale;
    p.softcap = a.softcap;
    int rc = cache.type == KRK_CUDA_KV_F16 ? launch_attn_f16(p, cache.head_dim, f.mt, st)
             : cache.type == KRK_CUDA_KV_Q8 ? launch_attn_q8(p, cache.head_dim, f.mt, st) : launch_attn_q4(p, cache.head_dim, f.mt, st);
    if (rc == KRK_CUDA_OK && !f.whole && f.grid > 1) rc = attn::launch_merge(p, cache.head_dim, f.mt, f.rows, st);
    return rc;
}

} // namespace krk_cuda
