// Attention of drafted tokens over a paged cache (krk_cuda_attention_tree): declarations shared by the kernel, which is
// instantiated per cache type in krk_attn_f16.cu / _q8.cu / _q4.cu, and the entry point in krk_attn_tree.cu.
//
//   out[r] = sum_p w_rp v_p / sum_p w_rp,   w_rp = exp(score_rp - max),   score = scale * q_r . k_p
//
// over the positions p that row r sees: all before its sequence's drafted tokens (inside the window), and of the drafted
// tokens those in its mask. A row is a (drafted token, query head) pair; the `group` query heads of a key head are rows of
// one product, so that a cached row is read once for all of them.
#pragma once

#include "krk_common.cuh"

namespace krk_cuda {
namespace attn {

constexpr int kWarps = 4;                 // of a CTA; each takes chunks of its own
constexpr int kThreads = 32 * kWarps;
constexpr int kChunk = 16;                // positions of a step of a warp; pages hold whole chunks
constexpr int kTile = kChunk * kWarps;    // positions the warps of a CTA take together
constexpr int kSetup = 3;                 // what an item costs beside its tiles, in tiles (queries, joining the warps' sums, latencies)
constexpr int kWholeTiles = 8;            // up to so many tiles an item is not divided, see launch

// An item that several CTAs have parts of, noted by the second one of them: parts 0 elsewhere.
struct Shared {
    int parts, n_rows, kvh, row0;   // row0: of the item's first row among its key head's
    int q0, pad[3];
};
inline size_t shared_bytes(int grid) { return (size_t)grid * sizeof(Shared); }

struct Params {
    const float *q;
    float *out;
    int64_t q_stride, out_stride;         // floats from a token to the next
    const uint8_t *k, *v;
    const __half *k_scale, *v_scale;
    const int32_t *table;                 // [n_seq][table_width] pages
    const int32_t *q_start, *kv_len;
    const uint64_t *tree;
    const float *sinks;
    Shared *shared;                       // [grid]
    float *part;                          // [grid][2][R][D + 2]: see part_row
    int64_t n_pages;
    int table_width, page_size, max_len, n_seq, n_heads, n_kv, group, max_q, window, whole, grid;
    float scale, softcap;
};

// The work, in the order of its units: sequences, their key heads, blocks of R rows, tiles of positions. A unit is a tile, and each
// item, all tiles of a block of rows, has kSetup more at its beginning (without them a CTA whose share was 40 items of one tile
// took four times as long as the others); or, where items are not divided (Params::whole), a unit is an item. The CTAs take equal shares of
// the units, whatever the lengths are, so at most a CTA's first and last items are shared with others; those leave partial
// sums, which a second kernel adds up in the order of the CTAs (the same bits every time; finding the items anew in that kernel took it 14 to 24 us).
struct Seq {
    int q0, n_q, len, before;   // first row of q, drafted tokens, positions, positions before the drafted ones (may be negative)
    int blocks, tile0, tiles;   // blocks of rows; first tile that any row sees, tiles from there on (at least one where there are rows)
};
template <int R>
__device__ __forceinline__ Seq sequence(const Params &p, int s) {
    Seq q;
    q.q0 = p.q_start[s];
    q.n_q = min(max(p.q_start[s + 1] - q.q0, 0), p.max_q);
    q.len = min(max(p.kv_len[s], 0), p.max_len);
    q.before = q.len - q.n_q;
    q.blocks = (q.n_q * p.group + R - 1) / R;
    const int first = p.window > 0 ? max(0, q.before - p.window) : 0;   // (the shallowest row is at `before`, or a position less where its mask is empty)
    q.tile0 = min(first, max(q.len - 1, 0)) / kTile;
    q.tiles = max(1, (q.len + kTile - 1) / kTile - q.tile0);
    return q;
}
__device__ __forceinline__ int item_units(const Params &p, const Seq &q) { return p.whole ? 1 : q.tiles + kSetup; }
__device__ __forceinline__ int64_t units_of(const Params &p, const Seq &q) { return (int64_t)p.n_kv * q.blocks * item_units(p, q); }

// Units [first(b), first(b + 1)) are CTA b's.
__device__ __forceinline__ int64_t first_unit(int64_t total, int grid, int b) { return total * min(b, grid) / grid; }

// By a whole CTA of 128 threads: the number of all units, the CTAs that share them (no more than there are units, so that each has some),
// and the sequence that CTA b's first one lies in (n_seq where it has none) with the units before that sequence.
struct Place {
    int64_t total, at, before;
    int grid, seq;
};
template <int R>
__device__ __forceinline__ Place find_place(const Params &p, int b) {
    __shared__ int64_t s_sum[kWarps];
    __shared__ int64_t s_before;
    __shared__ int s_found;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    Place r;
    r.total = 0;
    int64_t lo = 0, mine = 0;   // of this thread's sequence of the last 128
    auto scan = [&](int s0, int64_t base) {
        const int s = s0 + tid;
        mine = s < p.n_seq ? units_of(p, sequence<R>(p, s)) : 0;
        int64_t upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
            if (lane >= o) upto += v;
        }
        if (lane == 31) s_sum[warp] = upto;
        __syncthreads();
        int64_t all = 0;
        lo = base + upto - mine;
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            if (w < warp) lo += s_sum[w];
            all += s_sum[w];
        }
        __syncthreads();
        return all;
    };
    for (int s0 = 0; s0 < p.n_seq; s0 += kThreads) r.total += scan(s0, r.total);
    r.grid = (int)max(min((int64_t)p.grid, r.total), (int64_t)1);
    r.at = first_unit(r.total, r.grid, b);
    if (tid == 0) {
        s_found = p.n_seq;
        s_before = r.total;
    }
    __syncthreads();
    int64_t base = 0;
    for (int s0 = 0; s0 < p.n_seq; s0 += kThreads) {
        if (p.n_seq > kThreads) base += scan(s0, base);   // (up to 128 sequences the first scan's values stand)
        if (r.at >= lo && r.at < lo + mine) {
            s_found = s0 + tid;
            s_before = lo;
        }
    }
    __syncthreads();
    r.seq = s_found;
    r.before = s_before;
    return r;
}

// Rows of partial sums of CTA b: place 0 its first item's, where that began before the CTA; place 1 its last item's, where that
// goes on behind it and place 0 is not it. A row: D sums, the maximum (log2 domain), the sum of weights.
template <int D, int R>
__device__ __forceinline__ float *part_row(const Params &p, int b, int place, int row) {
    return p.part + (((size_t)b * 2 + place) * R + row) * (D + 2);
}

// out = sums / weights, with the sink's weight among the latter. Nothing seen: zero.
__device__ __forceinline__ float norm_of(const Params &p, int head, float m, float l, float &keep) {
    keep = 1.0f;
    if (p.sinks) {
        const float sink = p.sinks[head] * 1.44269504f;
        const float top = fmaxf(m, sink);
        keep = m == -INFINITY ? 0.0f : exp2f(m - top);
        l = l * keep + (sink == -INFINITY ? 0.0f : exp2f(sink - top));
    }
    return l == 0.0f ? 0.0f : keep / l;
}

}   // namespace attn

int launch_attn_f16(const attn::Params &p, int head_dim, int rows, cudaStream_t st);
int launch_attn_q8(const attn::Params &p, int head_dim, int rows, cudaStream_t st);
int launch_attn_q4(const attn::Params &p, int head_dim, int rows, cudaStream_t st);
// CTAs that an SM holds at once
int attn_ctas_f16(int head_dim, int rows);
int attn_ctas_q8(int head_dim, int rows);
int attn_ctas_q4(int head_dim, int rows);

}   // namespace krk_cuda
